// sb_gnorm.cu -- the end of one transformer block and the start of the next in one pass:
//   n = Npost(z),  y = x + scale * gate * n,  h = Npre(y)
// (each norm optional, RMS or layer norm, fp32 statistics), and its gradients.
//
// Forward, per row v of D values: RMS norm v r w with r = (mean v^2 + eps)^-1/2; layer norm
// (v - m) r w + b with r = (mean (v - m)^2 + eps)^-1/2 (the mean first, then the centred squares, no
// cancellation; the backward kernel for aligned rows takes both at once around values of the row, and
// again around its mean where those lie far from it).
// Apart, the norms and the residual sum would read and write the rows five times; here x and z are
// read and y and h written once, which bounds the kernel.
//
// Backward, with hats the normalised rows and e = d * w:
//   dyt = dy + r_y (e - yhat mean(e yhat) [- mean(e)]),  e = dh * w_pre        -> dx = dyt
//   dn = dyt * scale * gate,  dz = r_z (e - zhat mean(e zhat) [- mean(e)]),  e = dn * w_post
// The rows' statistics are taken again from x and z (they are in registers anyway) instead of
// being kept by the forward pass.  With f = dyt (times the gate where each row has its own), all
// column sums follow from four: Z = sum f zhat, Y = sum f, H = sum dh yhat, S = sum dh, per image
// where the gate is an image's:
//   d post_w = scale gate Z,  d post_b = scale gate Y,  d scale = gate (w Z + b Y),
//   d gate = scale (w Z + b Y),  d pre_w = H,  d pre_b = S.
// Each CTA keeps its columns' sums in registers over its rows and writes them once; a second
// kernel adds the CTAs' sums in a fixed order (no atomics: the same inputs give the same bits).
//
// A row belongs to a team: one warp, or all of a CTA's threads; a thread has NV vectors of eight
// columns.  Rows reach shared memory by bulk copies (x, z, dy, dh and a row's own gate), several rows
// ahead, so what is in flight does not cost registers and the reductions' latency is hidden.
// Element types are compile-time for the usual pairs.  Rows that are not 16-byte aligned or not a
// multiple of eight columns take plain loads, one row ahead (the kernels named `_any`).
//
// Forward, 65,280 rows of 2048 bf16 columns, RMS: 198 us, 83 % of the copy rate.  Backward, 65,280 rows of
// 1024, x fp32, z bf16, layer norms: 331 us, 56 %: 1100 instructions a warp and step of two rows, three
// dependent reductions, and registers for twelve warps an SM (a warp issues every 7 clocks; four CTAs an SM
// spill, 503 us of a run whose three took 384; a third stage of rows ahead took 426).
#include <algorithm>

#include "sb_xattn.cuh"

namespace sb {
namespace {

constexpr int kMaxD = 8192;
constexpr int kSums = 4;  // Z, Y, H, S

struct Rows {
  const void* p;
  long long row, img;
};

struct NormArgs {
  Rows x, z, gate, dy, dh;
  int xdt, zdt;
  const float *scale, *post_w, *post_b, *pre_w, *pre_b;
  int layer;
  float eps;
  int T, D, tpr, per;  // threads a row, rows a CTA takes at once (several: a warp each)
  long long rows;      // B * T
  long long step_b;    // forward, any alignment: from row to row as (items, rows), no division in the loop
  int step_t;
  void *y, *h;         // forward
  long long y_row, y_img, h_row, h_img;
  void *dx, *dz, *dgate_rows;  // backward
  float* part;                 // [groups * chunks][kSums][D]
  long long group_rows;        // rows that share their column sums (T for an image's gate, B * T else)
  int chunks, gate_is_row;     // CTAs a group
  int stages, stage_bytes;     // of a team's ring
  int row_bytes, copy_bytes;   // room of a row in it, what is copied of one
  int pitch;                   // columns that a row has room for
  long long team_rows;         // forward: rows of a team
};

// Sum of a pair of values over the threads of a row; the two halves of the buffer alternate, so one
// barrier a reduction is enough.
struct RowSum {
  float2* buf;  // [2][32]; as floats, [2][64]: K sums of up to 64 / K warps
  int warps, half;
  SB_DEV float2 operator()(float a, float b) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
      b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    if (warps == 1) return make_float2(a, b);
    float2* mine = buf + half * 32;
    half ^= 1;
    if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
    for (int i = 0; i < warps; ++i) {
      const float2 t = mine[i];
      s.x += t.x;
      s.y += t.y;
    }
    return s;
  }
  SB_DEV float operator()(float a) {
#pragma unroll
    for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
    if (warps == 1) return a;
    float2* mine = buf + half * 32;
    half ^= 1;
    if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5].x = a;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < warps; ++i) s += mine[i].x;
    return s;
  }
};

// A thread's columns: vector j begins at c0 + j * pitch; n(j) of its eight columns exist.
template <int NV>
struct Cols {
  int c0, pitch, D;
  SB_DEV int at(int j) const { return c0 + j * pitch; }
  SB_DEV int n(int j) const { return max(0, min(8, D - at(j))); }
};

SB_DEV void columns(const float* w, int c, int n, float other, float (&v)[8]) {
  if (!w) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = other;
    return;
  }
  unpack8(load_raw8_tail(w, SB_F32, c, n), SB_F32, v);
}

// mean and 1 / deviation of a row whose columns past D hold zeros
template <int NV>
SB_DEV void stats_of(const float (&v)[NV][8], const Cols<NV>& cols, int layer, float inv_d, float eps, RowSum& sum,
                     float& mean, float& r) {
  mean = 0.f;
  if (layer) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[j][u];
    mean = sum(s) * inv_d;
  }
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int n = cols.n(j);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float d = v[j][u] - mean;
      q += u < n ? d * d : 0.f;
    }
  }
  r = rsqrtf(sum(q) * inv_d + eps);
}

// ---------------------------------------------------------------- rows through shared memory
// The same value in every lane: whether all of the team's threads say yes (a barrier of the team).
SB_DEV bool team_all(bool yes, int warps) {
  return warps == 1 ? __all_sync(0xFFFFFFFFu, yes) : __syncthreads_and(yes) != 0;
}
// 8 fp32 column weights (16-byte aligned, read-only), `other` without any
SB_DEV void weights8(const float* w, int c, bool on, float other, float (&v)[8]) {
  if (w && on) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(w + c)), y = __ldg(reinterpret_cast<const float4*>(w + c) + 1);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = other;
  }
}
template <int DT>
SB_DEV void from_smem(const uint8_t* row, int dt, int c, float (&v)[8]) {
  unpack8(load_raw8(row, DT < 0 ? dt : DT, c), DT < 0 ? dt : DT, v);
}
template <int DT>
SB_DEV void from_smem(const uint8_t* row, int dt, int c, bool on, float (&v)[8]) {
  if (on) {
    unpack8(load_raw8(row, DT < 0 ? dt : DT, c), DT < 0 ? dt : DT, v);
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = 0.f;
  }
}
// Sums of K = 1, 2, 4 or 8 values over a team, in every thread.  A warp halves the values with its
// lanes (each half of the lanes goes on with half of the values), so eight values take 9 shuffles, not 40.
// WARPS: as many as a team can have, each with STRIDE floats in the buffer, zero where there is no such
// warp (a loop of known length); 0: the team's own number.
template <int K, int WARPS = 0, int STRIDE = K>
SB_DEV void team_sum(float (&v)[K], RowSum& sum) {
  static_assert(K == 1 || K == 2 || K == 4 || K == 8, "values");
  static_assert(WARPS * STRIDE <= 64 && STRIDE >= K, "half of the buffer");
  const int lane = threadIdx.x & 31;
  int o = 16;
#pragma unroll
  for (int n = K / 2; n; n >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int k = 0; k < n; ++k)
      v[k] = (up ? v[k + n] : v[k]) + __shfl_xor_sync(0xFFFFFFFFu, up ? v[k] : v[k + n], o);
  }
  float x = v[0];
#pragma unroll
  for (o = 16 / K; o; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
  constexpr int per = 32 / K;  // lanes that hold the same value: value k in lanes k * per ..
  if (sum.warps == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = K == 1 ? x : __shfl_sync(0xFFFFFFFFu, x, k * per);
    return;
  }
  float* mine = reinterpret_cast<float*>(sum.buf) + sum.half * 64;
  sum.half ^= 1;
  if (lane % per == 0) mine[(threadIdx.x >> 5) * STRIDE + lane / per] = x;
  __syncthreads();
  if constexpr (K == 1) {
    v[0] = 0.f;
    const int warps = WARPS ? WARPS : sum.warps;
#pragma unroll WARPS ? WARPS : 1
    for (int i = 0; i < warps; ++i) v[0] += mine[i * STRIDE];
  } else {
    uint64_t t[K / 2];
#pragma unroll
    for (int k = 0; k < K / 2; ++k) t[k] = 0;
    const int warps = WARPS ? WARPS : sum.warps;
#pragma unroll WARPS ? WARPS : 1
    for (int i = 0; i < warps; ++i) {
      if constexpr (K == 2) {
        t[0] = add2(t[0], *reinterpret_cast<const uint64_t*>(mine + i * STRIDE));
      } else {
#pragma unroll
        for (int k = 0; k < K; k += 4) {
          const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(mine + i * STRIDE + k);
          t[k / 2] = add2(t[k / 2], w.x);
          t[k / 2 + 1] = add2(t[k / 2 + 1], w.y);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < K / 2; ++k) split2(t[k], v[2 * k], v[2 * k + 1]);
  }
}

// 1 / deviation r and -mean r of R rows, so that their hats are v r + shift; `on[j]`: vector j of a row
// exists (the others hold zeros)
template <bool LAYER, int R, int NV>
SB_DEV void stats8(const float (&v)[R][NV][8], const bool (&on)[NV], float inv_d, float eps, RowSum& sum, float (&r)[R],
                   float (&shift)[R]) {
  float mean[R], q[R];
#pragma unroll
  for (int x = 0; x < R; ++x) mean[x] = q[x] = 0.f;
  if (LAYER) {
#pragma unroll
    for (int x = 0; x < R; ++x)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int u = 0; u < 8; ++u) mean[x] += v[x][j][u];
    team_sum(mean, sum);
#pragma unroll
    for (int x = 0; x < R; ++x) mean[x] *= inv_d;
  }
#pragma unroll
  for (int x = 0; x < R; ++x)
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (on[j]) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float d = LAYER ? v[x][j][u] - mean[x] : v[x][j][u];
          q[x] = fmaf(d, d, q[x]);
        }
      }
  team_sum(q, sum);
#pragma unroll
  for (int x = 0; x < R; ++x) {
    r[x] = rsqrtf(q[x] * inv_d + eps);
    shift[x] = LAYER ? -mean[x] * r[x] : 0.f;
  }
}

// A team's ring of rows.  Operand o of a row lies `off[o]` bytes into its stage; an operand that is
// not streamed has no bytes.
struct Ring {
  uint8_t* base;
  uint64_t* full;
  int stages, stage_bytes;
};
// A place in the ring: stage and the parity of its use.
struct Place {
  int st = 0;
  uint32_t parity = 0;
  SB_DEV void next(const Ring& r) {
    if (++st == r.stages) {
      st = 0;
      parity ^= 1u;
    }
  }
};
constexpr int kMaxStages = 8;

// A row as (b, t); the team's rows follow each other.
struct Walk {
  long long b;
  int t, T;
  SB_DEV void next() {
    if (++t == T) {
      t = 0;
      ++b;
    }
  }
};

// The copies of `rows` rows from `ahead` on into stage st, by the team's first thread.
template <bool BACK>
SB_DEV void fill(const NormArgs& a, const Ring& ring, int st, Walk& ahead, int rows) {
  uint64_t* bar = &ring.full[st];
  mbar_arrive_expect_tx(bar, (uint32_t)(rows * a.copy_bytes));
  const int xs = a.xdt == SB_F32 ? 4 : 2, zs = a.zdt == SB_F32 ? 4 : 2;
  for (int i = 0; i < rows; ++i, ahead.next()) {
    uint8_t* dst = ring.base + st * ring.stage_bytes + i * a.row_bytes;
    auto copy = [&](const Rows& r, int size) {
      bulk_load(dst, static_cast<const uint8_t*>(r.p) + (ahead.b * r.img + ahead.t * r.row) * size, a.D * size, bar);
      dst += a.pitch * size;
    };
    copy(a.z, zs);
    if (a.gate_is_row) copy(a.gate, zs);
    if (BACK ? a.dh.p != nullptr : true) copy(a.x, xs);
    if (BACK && a.dy.p) copy(a.dy, xs);
    if (BACK && a.dh.p) copy(a.dh, zs);
  }
}

__device__ int g_gnorm_error;

// A copy did not come: note it, and wait (bounded too) for those in flight before the CTA ends.
SB_DEV void give_up(const Ring& ring, Place at, int left, int me) {
  if (me != 0) return;
  atomicOr(&g_gnorm_error, SB_ERR_TIMEOUT_FULL);
  for (; left > 0; --left, at.next(ring)) bounded_wait(&ring.full[at.st], at.parity);
}

// XD, ZD: dtype codes of x and z, -1: as the arguments say.  Each team walks rows that follow each
// other, so that what depends on the columns alone (and an image's gate) stays in registers:
// y = x + hat A + B with A = scale gate post_w, B = scale gate post_b.
template <int XD, int ZD, bool LAYER, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 128 ? 4 : 1) gated_norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ __align__(16) float2 buf[64];
  __shared__ uint64_t bars[8 * kMaxStages];
  extern __shared__ __align__(16) uint8_t rows_smem[];
  const int xdt = XD < 0 ? a.xdt : XD, zdt = ZD < 0 ? a.zdt : ZD;
  const int warps = a.tpr >> 5;
  RowSum sum{buf, warps, 0};
  const int sub = a.per > 1 ? threadIdx.x >> 5 : 0, me = a.per > 1 ? threadIdx.x & 31 : threadIdx.x;
  const Ring ring{rows_smem + (size_t)sub * a.stages * a.stage_bytes, bars + sub * a.stages, a.stages, a.stage_bytes};
  const float inv_d = 1.f / (float)a.D;
  int c[NV];
  bool on[NV];
  float w[NV][8], o[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    c[j] = (me + j * a.tpr) * 8;
    on[j] = c[j] < a.D;
    weights8(a.pre_w, c[j], on[j], 1.f, w[j]);
    if (LAYER) weights8(a.pre_b, c[j], on[j], 0.f, o[j]);
  }
  if (me == 0)
    for (int i = 0; i < a.stages; ++i) mbar_init(&ring.full[i], 1);
  fence_mbar_init();
  __syncthreads();
  const long long begin = min(((long long)blockIdx.x * a.per + sub) * a.team_rows, a.rows);
  const int n = (int)(min(begin + a.team_rows, a.rows) - begin);
  Walk at{begin / a.T, (int)(begin % a.T), a.T}, ahead = at;
  Place here, there;
  int filled = 0;
  if (me == 0)
    for (; filled < min(n, a.stages); ++filled, there.next(ring)) fill<false>(a, ring, there.st, ahead, 1);
  const int go = a.pitch * (zdt == SB_F32 ? 4 : 2), xo = a.gate_is_row ? 2 * go : go;  // places in a stage: z, gate, x
  float A[NV][8], B[NV][8];
  long long gate_of = -1;
  for (int i = 0; i < n; ++i, at.next(), here.next(ring)) {
    if (!team_all(bounded_wait(&ring.full[here.st], here.parity), warps)) {
      give_up(ring, here, filled - i, me);
      break;
    }
    // the team has left row i - 1: its stage is free
    if (me == 0 && i > 0 && filled < n) {
      fill<false>(a, ring, there.st, ahead, 1);
      ++filled;
      there.next(ring);
    }
    if (at.b != gate_of) {
      gate_of = at.b;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        weights8(a.scale, c[j], on[j], 1.f, A[j]);
        if (a.gate.p && !a.gate_is_row && on[j]) {
          float g[8];
          unpack8(load_raw8(a.gate.p, zdt, at.b * a.gate.img + c[j]), zdt, g);
#pragma unroll
          for (int u = 0; u < 8; ++u) A[j][u] *= g[u];
        }
        if (LAYER) {
          weights8(a.post_b, c[j], on[j], 0.f, B[j]);
#pragma unroll
          for (int u = 0; u < 8; ++u) B[j][u] *= A[j][u];
        }
        float pw[8];
        weights8(a.post_w, c[j], on[j], 1.f, pw);
#pragma unroll
        for (int u = 0; u < 8; ++u) A[j][u] *= pw[u];
      }
    }
    const uint8_t* row = ring.base + here.st * a.stage_bytes;
    float v1[1][NV][8], y1[1][NV][8], r1[1] = {1.f}, shift1[1] = {0.f};
    float(&v)[NV][8] = v1[0];
    float(&y)[NV][8] = y1[0];
    float &r = r1[0], &shift = shift1[0];
#pragma unroll
    for (int j = 0; j < NV; ++j) from_smem<ZD>(row, zdt, c[j], on[j], v[j]);
    if (a.post_w) stats8<LAYER>(v1, on, inv_d, a.eps, sum, r1, shift1);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      from_smem<XD>(row + xo, xdt, c[j], on[j], y[j]);
      if (!on[j]) continue;
      if (a.gate_is_row) {
        float g[8];
        from_smem<ZD>(row + go, zdt, c[j], true, g);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float hat = fmaf(v[j][u], r, shift);
          y[j][u] = fmaf(g[u], LAYER ? fmaf(hat, A[j][u], B[j][u]) : hat * A[j][u], y[j][u]);
        }
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float hat = LAYER ? fmaf(v[j][u], r, shift) : v[j][u] * r;
          y[j][u] = fmaf(hat, A[j][u], LAYER ? y[j][u] + B[j][u] : y[j][u]);
        }
      }
      store8(a.y, xdt, at.b * a.y_img + at.t * a.y_row + c[j], y[j]);
    }
    if (a.h) {
      stats8<LAYER>(y1, on, inv_d, a.eps, sum, r1, shift1);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!on[j]) continue;
#pragma unroll
        for (int u = 0; u < 8; ++u)
          y[j][u] = LAYER ? fmaf(fmaf(y[j][u], r, shift), w[j][u], o[j][u]) : y[j][u] * r * w[j][u];
        store8(a.h, zdt, at.b * a.h_img + at.t * a.h_row + c[j], y[j]);
      }
    }
  }
}

// Pairs of fp32 values, two operations an instruction
SB_DEV float both(uint64_t v) {
  float lo, hi;
  split2(v, lo, hi);
  return lo + hi;
}
SB_DEV uint64_t twice(float v) { return pair2(v, v); }
SB_DEV void pairs(const float (&v)[8], uint64_t (&p)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) p[u] = pair2(v[2 * u], v[2 * u + 1]);
}
template <int DT>
SB_DEV void pairs_from(const uint8_t* row, int dt, int c, uint64_t (&p)[4]) {
  float v[8];
  from_smem<DT>(row, dt, c, v);
  pairs(v, p);
}
SB_DEV void store_pairs(void* p, int dt, long long i, const uint64_t (&v)[4]) {
  float f[8];
#pragma unroll
  for (int u = 0; u < 4; ++u) split2(v[u], f[2 * u], f[2 * u + 1]);
  store8(p, dt, i, f);
}
// Whether the squares of one of R rows were summed around a point more than four deviations from its mean
// (`squares` and `values`: sums over the row's columns; the same in all of a team's threads).
template <int R>
SB_DEV bool far_off(const float* squares, const float* values, float inv_d) {
  bool far = false;
#pragma unroll
  for (int x = 0; x < R; ++x) {
    const float m = values[x] * inv_d;
    far = far || 17.f * m * m > 16.f * (squares[x] * inv_d);
  }
  return far;
}
// The mean of four values: of equal ones exactly their value.
SB_DEV float mean4(float a, float b, float c, float d) { return ((a + b) + (c + d)) * 0.25f; }

// R rows of a team at once, in three reductions that their rows share:
//   1. z - c and its square,  2. y - c', its square, e and e (y - c') with e = dh w_pre,
//   3. e and e zhat with e = dn w_post  (RMS norm: the squares and the products alone).
// Layer norm's c and c' are the mean of the row's first four values, so that no pass for the mean comes
// first, and var = E (v - c)^2 - (E v - c)^2 loses nothing in rows of values alike, however large
// their mean.  Where c is more than four deviations off (the first values are the row's outliers), the row's
// mean takes its place and the sums are taken once more, a fourth reduction for those rows: what
// cancels is at most 16 var of 17.  Asking costs all rows 3 % (65,280 rows of 1024: 322 -> 331 us; as a loop
// over both blocks 25 %).  With the means first it was six reductions a step, whose latency bounded
// the kernel: 387 us.
// With A = scale gate w_post and B = scale gate b_post (of a row's own gate: without it),
// y = x + zhat A + B and dn w_post = dyt A.
// A row in shared memory has room for all of the team's columns, zero past D, and a row past the
// team's last is zeroed before its step, so the loop has no selects: lanes past D hold zeros in
// x, z, dy, dh, A and B and subtract nothing from them, which makes every term they add zero.
template <int XD, int ZD, bool LAYER, int R, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 128 ? 3 : 1) gated_norm_back_kernel(const __grid_constant__ NormArgs a) {
  __shared__ __align__(16) float2 buf[64];
  __shared__ uint64_t bars[8 * kMaxStages];
  __shared__ __align__(16) float first[2][4];  // A and B of the first four columns
  extern __shared__ __align__(16) uint8_t rows_smem[];
  const int xdt = XD < 0 ? a.xdt : XD, zdt = ZD < 0 ? a.zdt : ZD;
  const int warps = a.tpr >> 5;
  RowSum sum{buf, warps, 0};
  const int sub = a.per > 1 ? threadIdx.x >> 5 : 0, me = a.per > 1 ? threadIdx.x & 31 : threadIdx.x;
  const Ring ring{rows_smem + (size_t)sub * a.stages * a.stage_bytes, bars + sub * a.stages, a.stages, a.stage_bytes};
  const float inv_d = 1.f / (float)a.D;
  int c[NV], cw[NV];  // columns; of the weights (any for a lane past D)
  bool on[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    c[j] = (me + j * a.tpr) * 8;
    on[j] = c[j] < a.D;
    cw[j] = on[j] ? c[j] : 0;
  }
  constexpr int kWarps = MAXT / 32, kStride = (LAYER ? 4 : 2) * R;
  for (int i = threadIdx.x; i < 64; i += blockDim.x) buf[i] = make_float2(0.f, 0.f);
  if (me == 0)
    for (int i = 0; i < a.stages; ++i) mbar_init(&ring.full[i], 1);
  fence_mbar_init();
  for (int i = threadIdx.x; i < a.per * a.stages * a.stage_bytes / 16; i += blockDim.x)
    reinterpret_cast<uint4*>(rows_smem)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncthreads();
  const long long group = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const long long each = (a.group_rows + a.chunks - 1) / a.chunks;
  const long long last = group * a.group_rows + min((chunk + 1) * each, a.group_rows);
  const long long part = (each + a.per - 1) / a.per;  // a team's rows
  const long long begin = min(group * a.group_rows + min(chunk * each, a.group_rows) + sub * part, last);
  const int rows = (int)(min(begin + part, last) - begin), n = (rows + R - 1) / R;
  Walk ahead{begin / a.T, (int)(begin % a.T), a.T};
  Place here, there;
  int filled = 0;
  if (me == 0)
    for (; filled < min(n, a.stages); ++filled, there.next(ring))
      fill<true>(a, ring, there.st, ahead, min(R, rows - filled * R));
  // places in a row of a stage: z, gate, x, dy, dh
  const int zb = a.pitch * (zdt == SB_F32 ? 4 : 2), xb = a.pitch * (xdt == SB_F32 ? 4 : 2);
  const int xo = a.gate_is_row ? 2 * zb : zb, dyo = a.dh.p ? xo + xb : xo, dho = a.dy.p ? dyo + xb : dyo;
  // A, B and w_pre in registers where a thread has one vector, else from the cache each time
  float sg[NV][8];  // scale x gate of the CTA's rows (scale alone where every row has its gate)
  uint64_t acc[kSums][NV][4], keep[3][4];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    weights8(a.scale, c[j], on[j], on[j] ? 1.f : 0.f, sg[j]);
    if (a.gate.p && !a.gate_is_row && on[j]) {
      float g[8];
      unpack8(load_raw8(a.gate.p, zdt, group * a.gate.img + c[j]), zdt, g);
#pragma unroll
      for (int u = 0; u < 8; ++u) sg[j][u] *= g[u];
    }
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[k][j][u] = 0;
  }
  enum { kA, kB, kW };
  auto column = [&](int which, int j, uint64_t(&v)[4]) {
    float w[8];
    weights8(which == kA ? a.post_w : which == kB ? a.post_b : a.pre_w, cw[j], true, which == kB ? 0.f : 1.f, w);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (which != kW) w[u] *= sg[j][u];
    pairs(w, v);
  };
  auto take = [&](int which, int j, uint64_t(&v)[4]) {
    if constexpr (NV == 1) {
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = keep[which][u];
    } else {
      column(which, j, v);
    }
  };
  if constexpr (NV == 1) {
    column(kA, 0, keep[kA]);
    if (LAYER) column(kB, 0, keep[kB]);
    column(kW, 0, keep[kW]);
  }
  if (LAYER) {
    if (threadIdx.x == 0) {
      uint64_t v[4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        take(k, 0, v);
        split2(v[0], first[k][0], first[k][1]);
        split2(v[1], first[k][2], first[k][3]);
      }
    }
    __syncthreads();
  }
  // where the thread's columns of the step's first row go
  const int xe = xdt == SB_F32 ? 4 : 2, ze = zdt == SB_F32 ? 4 : 2;
  uint8_t* dx = static_cast<uint8_t*>(a.dx) + (begin * a.D + c[0]) * xe;
  uint8_t* dz = static_cast<uint8_t*>(a.dz) + (begin * a.D + c[0]) * ze;
  const intptr_t to_gates = reinterpret_cast<intptr_t>(a.dgate_rows) - reinterpret_cast<intptr_t>(a.dz);
  for (int i = 0; i < n; ++i, dx += R * a.D * xe, dz += R * a.D * ze, here.next(ring)) {
    if (!team_all(bounded_wait(&ring.full[here.st], here.parity), warps)) {
      give_up(ring, here, filled - i, me);
      break;
    }
    // the team has left step i - 1: its stage is free
    if (me == 0 && i > 0 && filled < n) {
      fill<true>(a, ring, there.st, ahead, min(R, rows - filled * R));
      ++filled;
      there.next(ring);
    }
    uint8_t* stage = ring.base + here.st * a.stage_bytes;
    const bool odd = R > 1 && (i + 1) * R > rows;  // the last row of this step does not exist
    if (odd) {
      for (int o = 0; o < a.row_bytes; o += 16 * a.tpr)
        if (o + 16 * me < a.row_bytes) *reinterpret_cast<uint4*>(stage + a.row_bytes + o + 16 * me) = make_uint4(0, 0, 0, 0);
      team_all(true, warps);
    }
    uint64_t zh[R][NV][4];
    float zr[R], zs[R], zc[R];  // zhat = (z - zc) zr + zs
#pragma unroll
    for (int x = 0; x < R; ++x) {
      zr[x] = 1.f;
      zs[x] = zc[x] = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) pairs_from<ZD>(stage + x * a.row_bytes, zdt, c[j], zh[x][j]);
    }
    if (a.post_w) {
      float s[LAYER ? 2 * R : R];  // squares, then (layer norm) values
#pragma unroll
      for (int x = 0; x < R; ++x) {
        if (LAYER) {
          float f[8];
          from_smem<ZD>(stage + x * a.row_bytes, zdt, 0, f);
          zc[x] = mean4(f[0], f[1], f[2], f[3]);
        }
        uint64_t q = 0, t = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const uint64_t off = twice(on[j] ? -zc[x] : 0.f);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint64_t& v = zh[x][j][u];
            if (LAYER) {
              v = add2(v, off);
              t = add2(t, v);
            }
            q = fma2(v, v, q);
          }
        }
        s[x] = both(q);
        if (LAYER) s[R + x] = both(t);
      }
      team_sum<sizeof(s) / 4, kWarps, kStride>(s, sum);
      if (LAYER && far_off<R>(s, s + R, inv_d)) {
#pragma unroll
        for (int x = 0; x < R; ++x) {
          const float m = s[R + x] * inv_d;
          zc[x] += m;
          uint64_t q = 0, t = 0;
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const uint64_t off = twice(on[j] ? -m : 0.f);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint64_t& v = zh[x][j][u];
              v = add2(v, off);
              t = add2(t, v);
              q = fma2(v, v, q);
            }
          }
          s[x] = both(q);
          s[R + x] = both(t);
        }
        team_sum<sizeof(s) / 4, kWarps, kStride>(s, sum);
      }
#pragma unroll
      for (int x = 0; x < R; ++x) {
        float var = s[x] * inv_d;
        if (LAYER) {
          const float m = s[R + x] * inv_d;
          var = fmaf(-m, m, var);
          if (var < 0.f) var = 0.f;  // (NaN stays)
          zr[x] = rsqrtf(var + a.eps);
          zs[x] = -m * zr[x];
        } else {
          zr[x] = rsqrtf(var + a.eps);
        }
        if (odd && x == R - 1) zr[x] = zs[x] = 0.f;
        const uint64_t r2 = twice(zr[x]), s2 = twice(zs[x]);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int u = 0; u < 4; ++u) zh[x][j][u] = LAYER ? fma2(zh[x][j][u], r2, s2) : mul2(zh[x][j][u], r2);
      }
    }
    uint64_t d[R][NV][4];
    float rs[R], m1[R], m0[R];
    if (a.dh.p) {
      constexpr int K = LAYER ? 4 : 2;  // squares, products of e, (layer norm) values, e
      float s[K * R];
      uint64_t dh[R][NV][4];
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const uint8_t* row = stage + x * a.row_bytes;
        float cy = 0.f;
        if (LAYER) {
          float z8[8], x8[8], g8[8], y4[4];
          from_smem<ZD>(row, zdt, 0, z8);
          from_smem<XD>(row + xo, xdt, 0, x8);
          if (a.gate_is_row) from_smem<ZD>(row + zb, zdt, 0, g8);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float t = fmaf(fmaf(z8[u] - zc[x], zr[x], zs[x]), first[0][u], first[1][u]);
            y4[u] = a.gate_is_row ? fmaf(g8[u], t, x8[u]) : x8[u] + t;
          }
          cy = mean4(y4[0], y4[1], y4[2], y4[3]);
        }
        uint64_t q = 0, p = 0, t = 0, te = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const uint64_t off = twice(on[j] ? -cy : 0.f);
          uint64_t A[4], B[4], W[4], g[4];
          take(kA, j, A);
          if (LAYER) take(kB, j, B);
          take(kW, j, W);
          if (a.gate_is_row) pairs_from<ZD>(row + zb, zdt, c[j], g);
          pairs_from<XD>(row + xo, xdt, c[j], d[x][j]);  // x, then y - c', then yhat
          pairs_from<ZD>(row + dho, zdt, c[j], dh[x][j]);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint64_t& y = d[x][j][u];
            if (a.gate_is_row) y = fma2(g[u], LAYER ? fma2(zh[x][j][u], A[u], B[u]) : mul2(zh[x][j][u], A[u]), y);
            else if (LAYER) y = add2(fma2(zh[x][j][u], A[u], B[u]), y);
            else y = fma2(zh[x][j][u], A[u], y);
            const uint64_t e = mul2(dh[x][j][u], W[u]);
            if (LAYER) {
              y = add2(y, off);
              t = add2(t, y);
              te = add2(te, e);
            }
            q = fma2(y, y, q);
            p = fma2(e, y, p);
          }
        }
        s[x] = both(q);
        s[R + x] = both(p);
        if (LAYER) {
          s[2 * R + x] = both(t);
          s[3 * R + x] = both(te);
        }
      }
      team_sum<sizeof(s) / 4, kWarps, kStride>(s, sum);
      if (LAYER && far_off<R>(s, s + 2 * R, inv_d)) {
#pragma unroll
        for (int x = 0; x < R; ++x) {
          const float m = s[2 * R + x] * inv_d;
          uint64_t q = 0, p = 0, t = 0, te = 0;
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const uint64_t off = twice(on[j] ? -m : 0.f);
            uint64_t W[4];
            take(kW, j, W);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint64_t& y = d[x][j][u];
              const uint64_t e = mul2(dh[x][j][u], W[u]);
              y = add2(y, off);
              t = add2(t, y);
              te = add2(te, e);
              q = fma2(y, y, q);
              p = fma2(e, y, p);
            }
          }
          s[x] = both(q);
          s[R + x] = both(p);
          s[2 * R + x] = both(t);
          s[3 * R + x] = both(te);
        }
        team_sum<sizeof(s) / 4, kWarps, kStride>(s, sum);
      }
#pragma unroll
      for (int x = 0; x < R; ++x) {
        float var = s[x] * inv_d, shift = 0.f, p = s[R + x];  // p: sum of e yhat
        if (LAYER) {
          const float m = s[2 * R + x] * inv_d;
          var = fmaf(-m, m, var);
          if (var < 0.f) var = 0.f;
          rs[x] = rsqrtf(var + a.eps);
          shift = -m * rs[x];
          p = rs[x] * fmaf(-m, s[3 * R + x], p);
          m0[x] = -s[3 * R + x] * inv_d * rs[x];
        } else {
          rs[x] = rsqrtf(var + a.eps);
          p *= rs[x];
        }
        m1[x] = -p * inv_d;
        if (odd && x == R - 1) rs[x] = shift = m1[x] = m0[x] = 0.f;
        const uint64_t r2 = twice(rs[x]), s2 = twice(shift);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          uint64_t W[4], dy[4];
          take(kW, j, W);
          if (a.dy.p) pairs_from<XD>(stage + x * a.row_bytes + dyo, xdt, c[j], dy);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint64_t& v = d[x][j][u];
            const uint64_t dd = dh[x][j][u], y = LAYER ? fma2(v, r2, s2) : mul2(v, r2);
            acc[2][j][u] = fma2(dd, y, acc[2][j][u]);
            if (LAYER) acc[3][j][u] = add2(acc[3][j][u], dd);
            v = fma2(y, twice(m1[x]), mul2(dd, W[u]));
            if (LAYER) v = fma2(v, r2, twice(m0[x]));
            else v = mul2(v, r2);
            if (a.dy.p) v = add2(v, dy[u]);
          }
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < R; ++x)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (a.dy.p) {
            pairs_from<XD>(stage + x * a.row_bytes + dyo, xdt, c[j], d[x][j]);
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) d[x][j][u] = 0;
          }
        }
    }
    float s[LAYER ? 2 * R : R];  // sums of e zhat, then (layer norm) of e
#pragma unroll
    for (int x = 0; x < R; ++x) {
      const bool there_is = !(x == R - 1 && odd);
      uint64_t p = 0, te = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        uint64_t A[4];
        take(kA, j, A);
        if (there_is && on[j]) store_pairs(dx, xdt, x * a.D + j * a.tpr * 8, d[x][j]);
        if (a.gate_is_row) {
          uint64_t g[4];
          pairs_from<ZD>(stage + x * a.row_bytes + zb, zdt, c[j], g);
          if (a.dgate_rows && there_is && on[j]) {
            uint64_t B[4], dg[4];
            if (LAYER) take(kB, j, B);
#pragma unroll
            for (int u = 0; u < 4; ++u)
              dg[u] = mul2(d[x][j][u], LAYER ? fma2(zh[x][j][u], A[u], B[u]) : mul2(zh[x][j][u], A[u]));
            store_pairs(dz + to_gates, zdt, x * a.D + j * a.tpr * 8, dg);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) d[x][j][u] = mul2(d[x][j][u], g[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint64_t& dd = d[x][j][u];
          acc[0][j][u] = fma2(dd, zh[x][j][u], acc[0][j][u]);
          if (LAYER) acc[1][j][u] = add2(acc[1][j][u], dd);
          dd = mul2(dd, A[u]);
          p = fma2(dd, zh[x][j][u], p);
          if (LAYER) te = add2(te, dd);
        }
      }
      s[x] = both(p);
      if (LAYER) s[R + x] = both(te);
    }
    if (a.post_w) {
      team_sum<sizeof(s) / 4, kWarps, kStride>(s, sum);
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const uint64_t n1 = twice(-s[x] * inv_d * zr[x]), n0 = twice(LAYER ? -s[R + x] * inv_d * zr[x] : 0.f);
        const uint64_t r2 = twice(zr[x]);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint64_t t = LAYER ? fma2(zh[x][j][u], n1, n0) : mul2(zh[x][j][u], n1);
            d[x][j][u] = fma2(d[x][j][u], r2, t);
          }
      }
    }
#pragma unroll
    for (int x = 0; x < R; ++x)
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (on[j] && !(x == R - 1 && odd)) store_pairs(dz, zdt, x * a.D + j * a.tpr * 8, d[x][j]);
  }
  if (!a.part) return;
  float* mine = a.part + (long long)blockIdx.x * kSums * a.D;
  if (a.per == 1) {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (on[j]) store_pairs(mine, SB_F32, (long long)k * a.D + c[j], acc[k][j]);
    return;
  }
  // the CTA's warps one after the other, over the rings (every copy has been waited for)
  float* fold = reinterpret_cast<float*>(rows_smem);
  const int width = a.tpr * 8 * NV;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        reinterpret_cast<uint64_t*>(fold)[((sub * kSums + k) * width + c[j]) / 2 + u] = acc[k][j][u];
  __syncthreads();
  for (int i = threadIdx.x; i < kSums * a.D; i += blockDim.x) {
    const int k = i / a.D, col = i - k * a.D;
    float s = 0.f;
    for (int q = 0; q < a.per; ++q) s += fold[(q * kSums + k) * width + col];
    mine[i] = s;
  }
}

// ---------------------------------------------------------------- any alignment, any D
template <int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_any_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 buf[64];
  const int xdt = a.xdt, zdt = a.zdt;
  RowSum sum{buf, a.tpr >> 5, 0};
  const int sub = a.per > 1 ? threadIdx.x >> 5 : 0;
  const Cols<NV> cols{(int)(a.per > 1 ? threadIdx.x & 31 : threadIdx.x) * 8, a.tpr * 8, a.D};
  const float inv_d = 1.f / (float)a.D;
  const long long step = (long long)gridDim.x * a.per;
  long long r = (long long)blockIdx.x * a.per + sub;
  long long b = r / a.T;
  int t = (int)(r - b * a.T);
  Raw8 rx[NV], rz[NV], rg[NV];
  auto load = [&](bool ok, long long bb, int tt) {
    const long long xo = bb * a.x.img + tt * a.x.row, zo = bb * a.z.img + tt * a.z.row;
    const long long go = bb * a.gate.img + tt * a.gate.row;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = cols.at(j), m = ok ? cols.n(j) : 0;
      rx[j] = load_raw8_tail(a.x.p, xdt, xo + c, m);
      rz[j] = load_raw8_tail(a.z.p, zdt, zo + c, m);
      if (a.gate.p) rg[j] = load_raw8_tail(a.gate.p, zdt, go + c, m);
    }
  };
  load(r < a.rows, b, t);
  // every warp of a row's CTA walks the same rows; with a warp a row there is no barrier
  for (; r < a.rows; r += step) {
    float v[NV][8], y[NV][8], g[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack8(rz[j], zdt, v[j]);
      unpack8(rx[j], xdt, y[j]);
      if (a.gate.p) {
        unpack8(rg[j], zdt, g[j]);
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) g[j][u] = 1.f;
      }
    }
    long long nb = b + a.step_b;
    int nt = t + a.step_t;
    if (nt >= a.T) {
      nt -= a.T;
      ++nb;
    }
    load(r + step < a.rows, nb, nt);
    float mean = 0.f, rs = 1.f;
    if (a.post_w) stats_of(v, cols, a.layer, inv_d, a.eps, sum, mean, rs);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = cols.at(j), n = cols.n(j);
      float s[8], w[8], o[8];
      columns(a.scale, c, n, 1.f, s);
      if (a.post_w) {
        columns(a.post_w, c, n, 1.f, w);
        columns(a.post_b, c, n, 0.f, o);
#pragma unroll
        for (int u = 0; u < 8; ++u) v[j][u] = fmaf((v[j][u] - mean) * rs, w[u], o[u]);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) y[j][u] = u < n ? fmaf(s[u] * g[j][u], v[j][u], y[j][u]) : 0.f;
      store8_tail(a.y, xdt, b * a.y_img + t * a.y_row + c, y[j], n);
    }
    if (a.h) {
      stats_of(y, cols, a.layer, inv_d, a.eps, sum, mean, rs);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = cols.at(j), n = cols.n(j);
        float w[8], o[8];
        columns(a.pre_w, c, n, 1.f, w);
        columns(a.pre_b, c, n, 0.f, o);
#pragma unroll
        for (int u = 0; u < 8; ++u) y[j][u] = fmaf((y[j][u] - mean) * rs, w[u], o[u]);
        store8_tail(a.h, zdt, b * a.h_img + t * a.h_row + c, y[j], n);
      }
    }
    b = nb;
    t = nt;
  }
}

template <int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) gated_norm_back_any_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 buf[64];
  extern __shared__ float fold[];  // [per][kSums][D padded]: several rows' warps meet here
  const int xdt = a.xdt, zdt = a.zdt;
  RowSum sum{buf, a.tpr >> 5, 0};
  const int sub = a.per > 1 ? threadIdx.x >> 5 : 0;
  const Cols<NV> cols{(int)(a.per > 1 ? threadIdx.x & 31 : threadIdx.x) * 8, a.tpr * 8, a.D};
  const float inv_d = 1.f / (float)a.D;
  const long long group = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const long long each = (a.group_rows + a.chunks - 1) / a.chunks;
  const long long first = group * a.group_rows + min(chunk * each, a.group_rows);
  const long long last = group * a.group_rows + min((chunk + 1) * each, a.group_rows);
  float acc[kSums][NV][8];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int u = 0; u < 8; ++u) acc[k][j][u] = 0.f;
  long long r = first + sub, b = r / a.T;
  int t = (int)(r - b * a.T);
  Raw8 rx[NV], rz[NV], rg[NV], rdy[NV], rdh[NV];
  auto load = [&](bool ok, long long bb, int tt) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = cols.at(j), m = ok ? cols.n(j) : 0;
      rz[j] = load_raw8_tail(a.z.p, zdt, bb * a.z.img + tt * a.z.row + c, m);
      rdy[j] = load_raw8_tail(a.dy.p, xdt, bb * a.dy.img + tt * a.dy.row + c, a.dy.p ? m : 0);
      if (a.dh.p) {
        rx[j] = load_raw8_tail(a.x.p, xdt, bb * a.x.img + tt * a.x.row + c, m);
        rdh[j] = load_raw8_tail(a.dh.p, zdt, bb * a.dh.img + tt * a.dh.row + c, m);
      }
      if (a.gate.p) rg[j] = load_raw8_tail(a.gate.p, zdt, bb * a.gate.img + tt * a.gate.row + c, m);
    }
  };
  load(r < last, b, t);
  for (; r < last; r += a.per) {
    float zh[NV][8], g[NV][8], d[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack8(rz[j], zdt, zh[j]);
      unpack8(rdy[j], xdt, d[j]);
      if (a.gate.p) {
        unpack8(rg[j], zdt, g[j]);
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) g[j][u] = 1.f;
      }
    }
    float y[NV][8], dh[NV][8];
    if (a.dh.p) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        unpack8(rx[j], xdt, y[j]);
        unpack8(rdh[j], zdt, dh[j]);
      }
    }
    t += a.per;
    if (t >= a.T) {  // T < per: the division below
      const int over = t / a.T;
      t -= over * a.T;
      b += over;
    }
    load(r + a.per < last, b, t);
    float zr = 1.f;
    if (a.post_w) {
      float mean;
      stats_of(zh, cols, a.layer, inv_d, a.eps, sum, mean, zr);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int u = 0; u < 8; ++u) zh[j][u] = u < cols.n(j) ? (zh[j][u] - mean) * zr : 0.f;
    }
    if (a.dh.p) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = cols.at(j), n = cols.n(j);
        float s[8], w[8], o[8];
        columns(a.scale, c, n, 1.f, s);
        columns(a.post_w, c, n, 1.f, w);
        columns(a.post_b, c, n, 0.f, o);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          y[j][u] = u < n ? fmaf(s[u] * g[j][u], fmaf(zh[j][u], w[u], o[u]), y[j][u]) : 0.f;
      }
      float mean, rs, e0 = 0.f, e1 = 0.f;
      stats_of(y, cols, a.layer, inv_d, a.eps, sum, mean, rs);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float w[8];
        columns(a.pre_w, cols.at(j), cols.n(j), 1.f, w);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          y[j][u] = u < cols.n(j) ? (y[j][u] - mean) * rs : 0.f;
          acc[2][j][u] = fmaf(dh[j][u], y[j][u], acc[2][j][u]);
          acc[3][j][u] += dh[j][u];
          dh[j][u] *= w[u];
          e0 += dh[j][u];
          e1 = fmaf(dh[j][u], y[j][u], e1);
        }
      }
      const float2 m = sum(e0, e1);
      const float m0 = a.layer ? m.x * inv_d : 0.f, m1 = m.y * inv_d;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int u = 0; u < 8; ++u) d[j][u] += rs * (dh[j][u] - y[j][u] * m1 - m0);
    }
    float e0 = 0.f, e1 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = cols.at(j), n = cols.n(j);
      store8_tail(a.dx, xdt, r * a.D + c, d[j], n);
      float s[8], w[8];
      columns(a.scale, c, n, 1.f, s);
      columns(a.post_w, c, n, 1.f, w);
      if (a.dgate_rows) {
        float o[8], dg[8];
        columns(a.post_b, c, n, 0.f, o);
#pragma unroll
        for (int u = 0; u < 8; ++u) dg[u] = d[j][u] * s[u] * fmaf(zh[j][u], w[u], o[u]);
        store8_tail(a.dgate_rows, zdt, r * a.D + c, dg, n);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float f = a.gate_is_row ? d[j][u] * g[j][u] : d[j][u];
        acc[0][j][u] = fmaf(f, zh[j][u], acc[0][j][u]);
        acc[1][j][u] += f;
        d[j][u] = u < n ? d[j][u] * s[u] * g[j][u] * w[u] : 0.f;
        e0 += d[j][u];
        e1 = fmaf(d[j][u], zh[j][u], e1);
      }
    }
    float m0 = 0.f, m1 = 0.f;
    if (a.post_w) {
      const float2 m = sum(e0, e1);
      m0 = a.layer ? m.x * inv_d : 0.f;
      m1 = m.y * inv_d;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (a.post_w) {
#pragma unroll
        for (int u = 0; u < 8; ++u) d[j][u] = zr * (d[j][u] - zh[j][u] * m1 - m0);
      }
      store8_tail(a.dz, zdt, r * a.D + cols.at(j), d[j], cols.n(j));
    }
  }
  if (!a.part) return;
  float* mine = a.part + (long long)blockIdx.x * kSums * a.D;
  if (a.per == 1) {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int j = 0; j < NV; ++j) store8_tail(mine, SB_F32, (long long)k * a.D + cols.at(j), acc[k][j], cols.n(j));
    return;
  }
  // the CTA's warps one after the other
  const int width = a.tpr * 8 * NV;
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int u = 0; u < 8; ++u) fold[(sub * kSums + k) * width + cols.at(j) + u] = acc[k][j][u];
  __syncthreads();
  for (int i = threadIdx.x; i < kSums * a.D; i += blockDim.x) {
    const int k = i / a.D, col = i - k * a.D;
    float s = 0.f;
    for (int q = 0; q < a.per; ++q) s += fold[(q * kSums + k) * width + col];
    mine[i] = s;
  }
}

struct FoldArgs {
  const float* part;
  int groups, chunks, D, gate_mode;
  Rows gate;  // of the group's rows
  int zdt, gate_is_row;
  const float *scale, *post_w, *post_b;
  float *dscale, *dgate, *dpost_w, *dpost_b, *dpre_w, *dpre_b;
};

// 32 columns a CTA; 16 threads a column add the partial sums of a group, in a fixed order
__global__ void __launch_bounds__(512) gated_norm_fold_kernel(const __grid_constant__ FoldArgs a) {
  __shared__ float sh[16][kSums][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float tot[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // scale, gate, post_w, post_b, pre_w, pre_b
  for (int g = 0; g < a.groups; ++g) {
    float s[kSums] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.D)
      for (int k = part; k < a.chunks; k += 16) {
        const float* p = a.part + ((long long)g * a.chunks + k) * kSums * a.D + c;
#pragma unroll
        for (int q = 0; q < kSums; ++q) s[q] += p[(long long)q * a.D];
      }
#pragma unroll
    for (int q = 0; q < kSums; ++q) sh[part][q][lane] = s[q];
    __syncthreads();
    if (part == 0 && c < a.D) {
#pragma unroll
      for (int q = 0; q < kSums; ++q) {
        s[q] = 0.f;
        for (int k = 0; k < 16; ++k) s[q] += sh[k][q][lane];
      }
      const float sc = a.scale ? a.scale[c] : 1.f;
      const float gt = a.gate.p && !a.gate_is_row ? one_of(a.gate.p, a.zdt, g * a.gate.img + c) : 1.f;
      const float n = s[0] * (a.post_w ? a.post_w[c] : 1.f) + s[1] * (a.post_b ? a.post_b[c] : 0.f);
      if (a.gate_mode == 2) a.dgate[(long long)g * a.D + c] = sc * n;
      tot[0] += gt * n;
      tot[1] += sc * n;
      tot[2] += sc * gt * s[0];
      tot[3] += sc * gt * s[1];
      tot[4] += s[2];
      tot[5] += s[3];
    }
    __syncthreads();
  }
  if (part != 0 || c >= a.D) return;
  if (a.dscale) a.dscale[c] = tot[0];
  if (a.gate_mode == 1) a.dgate[c] = tot[1];
  if (a.dpost_w) a.dpost_w[c] = tot[2];
  if (a.dpost_b) a.dpost_b[c] = tot[3];
  if (a.dpre_w) a.dpre_w[c] = tot[4];
  if (a.dpre_b) a.dpre_b[c] = tot[5];
}

int sm_count() {
  static int of[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  int n = of[dev & 63];
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    of[dev & 63] = n;
  }
  return n;
}

// Up to 256 channels a warp takes a row with one vector a lane, eight (backward: four) teams a CTA;
// above, a CTA is a team: forward with two vectors a thread, backward with two rows of one vector
// (twice the independent work of a row, half the registers that two vectors' column sums take) up to
// 2048 channels, and one row of two vectors above.
struct Plan {
  int kind;  // of the launch tables
  int tpr, per, threads, at_once;
};
Plan plan_of(int D, bool back) {
  Plan p;
  const int vecs = (D + 7) / 8;
  p.at_once = back && vecs <= 256 ? 2 : 1;
  p.per = 1;
  if (vecs <= 32) {
    p.kind = 0;
    p.tpr = 32;
    p.per = back ? 4 : 8;
  } else if (p.at_once == 2) {
    p.tpr = (vecs + 31) / 32 * 32;
    p.kind = p.tpr <= 128 ? 1 : 2;
  } else {
    p.tpr = ((vecs + 1) / 2 + 31) / 32 * 32;
    p.kind = p.tpr <= 128 ? 1 : p.tpr <= 256 ? 2 : 3;
    if (back) p.kind += 1;  // 3, 4
  }
  p.threads = p.tpr * p.per;
  return p;
}

using NormKernel = void (*)(const NormArgs);

template <int XD, int ZD, bool LAYER>
NormKernel ring_kernel(bool back, int kind) {
  if (back) {
    if (kind == 0) return gated_norm_back_kernel<XD, ZD, LAYER, 2, 1, 128>;
    if (kind == 1) return gated_norm_back_kernel<XD, ZD, LAYER, 2, 1, 128>;
    if (kind == 2) return gated_norm_back_kernel<XD, ZD, LAYER, 2, 1, 256>;
    return kind == 3 ? gated_norm_back_kernel<-1, -1, LAYER, 1, 2, 256> : gated_norm_back_kernel<-1, -1, LAYER, 1, 2, 512>;
  }
  if (kind == 0) return gated_norm_kernel<XD, ZD, LAYER, 1, 256>;
  if (kind == 1) return gated_norm_kernel<XD, ZD, LAYER, 2, 128>;
  return kind == 2 ? gated_norm_kernel<XD, ZD, LAYER, 2, 256> : gated_norm_kernel<-1, -1, LAYER, 2, 512>;
}
template <int XD, int ZD>
NormKernel ring_kernel(bool back, int kind, bool layer) {
  return layer ? ring_kernel<XD, ZD, true>(back, kind) : ring_kernel<XD, ZD, false>(back, kind);
}
NormKernel pick(bool back, int xdt, int zdt, bool vec, int kind, bool layer) {
  if (!vec) {
    if (back) return kind <= 2 ? gated_norm_back_any_kernel<1, 256> : gated_norm_back_any_kernel<2, 512>;
    return kind == 0 ? gated_norm_any_kernel<1, 256> : gated_norm_any_kernel<2, 512>;
  }
  if (xdt == SB_F32 && zdt == SB_F16) return ring_kernel<SB_F32, SB_F16>(back, kind, layer);
  if (xdt == SB_F32 && zdt == SB_BF16) return ring_kernel<SB_F32, SB_BF16>(back, kind, layer);
  if (xdt == SB_F16 && zdt == SB_F16) return ring_kernel<SB_F16, SB_F16>(back, kind, layer);
  if (xdt == SB_BF16 && zdt == SB_BF16) return ring_kernel<SB_BF16, SB_BF16>(back, kind, layer);
  return ring_kernel<-1, -1>(back, kind, layer);
}

// CTAs an SM: as many as have 512 threads (backward, with its registers: 384), four (three) at least.  65,280
// rows of bf16, RMS: with four CTAs whatever their size 1024 columns take 154 us instead of 97; with 640
// threads, whose registers then spill, 137, and 2048 columns 277 instead of 193.
int ctas_of(const Plan& p, bool back) { return back ? std::max(3, 384 / p.threads) : std::max(4, 512 / p.threads); }

// The ring of each team (as many rows as its part of an SM's bytes holds, two to eight) and a CTA's shared
// memory, which the backward kernels' last sums share.  More rows ahead than these do not help: with 184 KB of
// forward rings 65,280 rows of 256 to 2048 columns take as long, or up to 5 % longer.
int ring_bytes(bool back) { return (back ? 138 : 96) * 1024; }
int ring_of(NormArgs& a, const Plan& p, bool back, bool& vec) {
  const int xs = dtype_bytes(a.xdt), zs = dtype_bytes(a.zdt);
  a.pitch = back ? p.tpr * 8 * (p.at_once == 2 || p.kind == 0 ? 1 : 2) : a.D;
  const int elem = zs + (a.gate_is_row ? zs : 0) + (back ? (a.dh.p ? xs + zs : 0) + (a.dy.p ? xs : 0) : xs);
  a.copy_bytes = a.D * elem;
  a.row_bytes = a.pitch * elem;
  a.stage_bytes = a.row_bytes * p.at_once;
  a.stages = std::max(2, std::min(kMaxStages, ring_bytes(back) / ctas_of(p, back) / (p.per * a.stage_bytes)));
  vec = vec && 2 * p.per * a.stage_bytes <= 200 * 1024;  // else the widest fp32 rows: no room for two
  const int ring = vec ? p.per * a.stages * a.stage_bytes : 0;
  const int fold = back && p.per > 1 ? p.per * kSums * p.tpr * 8 * 4 : 0;
  return std::max(ring, fold);
}
cudaError_t launch_norm(NormKernel kernel, unsigned grid, int threads, int smem, const NormArgs& a, cudaStream_t st) {
  if (smem > 46 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  kernel<<<grid, threads, smem, st>>>(a);
  return cudaGetLastError();
}

// CTAs a group of rows: about ctas_of an SM over all groups, at least eight rows a warp or CTA
int chunks_of(int groups, long long group_rows, const Plan& p, int sms) {
  const long long want = std::max(1, ctas_of(p, true) * sms / groups);
  return (int)std::max(1ll, std::min(want, (group_rows + 8 * p.per - 1) / (8 * p.per)));
}

bool rows_aligned(const void* p, int dt, long long row, long long img) {
  const int e = dtype_bytes(dt);
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row * e % 16 == 0 && img * e % 16 == 0;
}
bool cols_aligned(const float* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int gnorm_error(int clear, int* flags) {
  const int zero = 0;
  if (cudaMemcpyFromSymbol(flags, g_gnorm_error, sizeof(int)) != cudaSuccess) return -1;
  return clear && cudaMemcpyToSymbol(g_gnorm_error, &zero, sizeof(int)) != cudaSuccess ? -1 : 0;
}

}  // namespace sb

using namespace sb;

extern "C" int sb_gated_norm(const void* x, long long x_row, long long x_img, int x_dtype, const void* z, long long z_row,
                             long long z_img, int z_dtype, const void* gate, long long gate_row, long long gate_img,
                             const float* scale, const float* post_w, const float* post_b, const float* pre_w,
                             const float* pre_b, int layer, float eps, int B, int T, int D, void* y, long long y_row,
                             long long y_img, void* h, long long h_row, long long h_img, void* stream) {
  if (B < 0 || T < 0 || D < 1 || D > kMaxD || !rows_dtype_ok(x_dtype) || !rows_dtype_ok(z_dtype) || !(eps >= 0.f))
    return record_error(SB_EINVAL, "sb_gated_norm: sizes (1 <= D <= 8192), dtype or eps");
  if (B == 0 || T == 0) return SB_OK;
  if (!x || !z || !y || (pre_w != nullptr) != (h != nullptr) || (post_b && !(post_w && layer)) || (pre_b && !(pre_w && layer)))
    return record_error(SB_EINVAL, "sb_gated_norm: null argument (h with pre_w, biases with their weights)");
  const Plan p = plan_of(D, false);
  NormArgs a{};
  a.x = {x, x_row, x_img};
  a.z = {z, z_row, z_img};
  a.gate = {gate, gate_row, gate_img};
  a.xdt = x_dtype; a.zdt = z_dtype;
  a.scale = scale; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
  a.layer = layer != 0; a.eps = eps; a.T = T; a.D = D; a.tpr = p.tpr; a.per = p.per;
  a.rows = (long long)B * T;
  a.y = y; a.y_row = y_row; a.y_img = y_img;
  a.h = h; a.h_row = h_row; a.h_img = h_img;
  bool vec = D % 8 == 0 && rows_aligned(x, x_dtype, x_row, x_img) && rows_aligned(z, z_dtype, z_row, z_img) &&
                   (!gate || rows_aligned(gate, z_dtype, gate_row, gate_img)) &&
                   rows_aligned(y, x_dtype, y_row, y_img) && (!h || rows_aligned(h, z_dtype, h_row, h_img)) &&
                   cols_aligned(scale) && cols_aligned(post_w) && cols_aligned(post_b) && cols_aligned(pre_w) &&
                   cols_aligned(pre_b);
  const int sms = sm_count();
  if (sms == 0) return record_error(SB_ECUDA, "sb_gated_norm: device");
  a.gate_is_row = gate && gate_row != 0;
  const int smem = ring_of(a, p, false, vec);
  const NormKernel kernel = pick(false, x_dtype, z_dtype, vec, p.kind, layer != 0);
  const long long grid = std::min((a.rows + p.per - 1) / p.per, (long long)sms * ctas_of(p, false));
  const long long step = grid * p.per;
  a.step_b = step / T;
  a.step_t = (int)(step % T);
  a.team_rows = (a.rows + step - 1) / step;
  const cudaError_t e = launch_norm(kernel, (unsigned)grid, p.threads, smem, a, (cudaStream_t)stream);
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}

extern "C" int sb_gated_norm_work(int B, int T, int D, long long* bytes) {
  if (!bytes || B < 0 || T < 0 || D < 1 || D > kMaxD) return record_error(SB_EINVAL, "sb_gated_norm_work: arguments");
  const int sms = sm_count();
  if (sms == 0) return record_error(SB_ECUDA, "sb_gated_norm_work: device");
  const Plan p = plan_of(D, true);
  // enough for one group of all rows and for a group an item
  const long long one = chunks_of(1, (long long)B * T, p, sms), each = (long long)B * chunks_of(std::max(1, B), T, p, sms);
  *bytes = std::max(one, each) * kSums * D * 4;
  return SB_OK;
}

extern "C" int sb_gated_norm_backward(const void* dy, long long dy_row, long long dy_img, const void* dh, long long dh_row,
                                      long long dh_img, const void* x, long long x_row, long long x_img, int x_dtype,
                                      const void* z, long long z_row, long long z_img, int z_dtype, const void* gate,
                                      long long gate_row, long long gate_img, const float* scale, const float* post_w,
                                      const float* post_b, const float* pre_w, const float* pre_b, int layer, float eps,
                                      int B, int T, int D, void* dx, void* dz, float* dscale, void* dgate, int dgate_mode,
                                      float* dpost_w, float* dpost_b, float* dpre_w, float* dpre_b, void* work,
                                      long long work_bytes, void* stream) {
  if (B < 1 || T < 1 || D < 1 || D > kMaxD || !rows_dtype_ok(x_dtype) || !rows_dtype_ok(z_dtype) || !(eps >= 0.f))
    return record_error(SB_EINVAL, "sb_gated_norm_backward: sizes (1 <= D <= 8192), dtype or eps");
  if (!x || !z || !dx || !dz || (dh && !pre_w) || (post_b && !(post_w && layer)) || (pre_b && !(pre_w && layer)) || dgate_mode < 0 ||
      dgate_mode > 3 || (dgate_mode != 0 && (!dgate || !gate)) || (dscale && !scale) || ((dpost_w || dpost_b) && !post_w) ||
      ((dpre_w || dpre_b) && !pre_w))
    return record_error(SB_EINVAL, "sb_gated_norm_backward: null argument or a gradient without its input");
  const bool by_row = gate && gate_row != 0 && T > 1;
  const bool by_img = gate && gate_img != 0 && B > 1;
  if ((dgate_mode == 1 && (by_row || by_img)) || (dgate_mode == 2 && by_row))
    return record_error(SB_EINVAL, "sb_gated_norm_backward: dgate_mode does not fit the gate's strides");
  const Plan p = plan_of(D, true);
  NormArgs a{};
  a.x = {x, x_row, x_img};
  a.z = {z, z_row, z_img};
  a.gate = {gate, gate_row, gate_img};
  a.dy = {dy, dy_row, dy_img};
  a.dh = {dh, dh_row, dh_img};
  a.xdt = x_dtype; a.zdt = z_dtype;
  a.scale = scale; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
  a.layer = layer != 0; a.eps = eps; a.T = T; a.D = D; a.tpr = p.tpr; a.per = p.per;
  a.rows = (long long)B * T;
  a.dx = dx; a.dz = dz;
  a.dgate_rows = dgate_mode == 3 ? dgate : nullptr;
  a.gate_is_row = by_row || dgate_mode == 3;
  const bool sums = dscale || dgate_mode == 1 || dgate_mode == 2 || dpost_w || dpost_b || dpre_w || dpre_b;
  const int sms = sm_count();
  if (sms == 0) return record_error(SB_ECUDA, "sb_gated_norm_backward: device");
  const int groups = !a.gate_is_row && (by_img || dgate_mode == 2) ? B : 1;
  a.group_rows = groups == 1 ? a.rows : T;
  a.chunks = chunks_of(groups, a.group_rows, p, sms);
  const long long need = (long long)groups * a.chunks * kSums * D * 4;
  if (sums) {
    if (!work || work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15) != 0)
      return record_error(SB_EINVAL, "sb_gated_norm_backward: workspace (sb_gated_norm_work bytes, 16-byte aligned)");
    a.part = static_cast<float*>(work);
  }
  bool vec = D % 8 == 0 && rows_aligned(x, x_dtype, x_row, x_img) && rows_aligned(z, z_dtype, z_row, z_img) &&
                   (!gate || rows_aligned(gate, z_dtype, gate_row, gate_img)) &&
                   (!dy || rows_aligned(dy, x_dtype, dy_row, dy_img)) &&
                   (!dh || rows_aligned(dh, z_dtype, dh_row, dh_img)) && rows_aligned(dx, x_dtype, 0, 0) &&
                   rows_aligned(dz, z_dtype, 0, 0) && (dgate_mode != 3 || rows_aligned(dgate, z_dtype, 0, 0)) &&
                   cols_aligned(scale) && cols_aligned(post_w) && cols_aligned(post_b) && cols_aligned(pre_w) &&
                   cols_aligned(pre_b);
  const int smem = ring_of(a, p, true, vec);
  const NormKernel kernel = pick(true, x_dtype, z_dtype, vec, p.kind, layer != 0);
  if ((long long)groups * a.chunks > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_gated_norm_backward: too many items");
  cudaError_t e = launch_norm(kernel, (unsigned)(groups * a.chunks), p.threads, smem, a, (cudaStream_t)stream);
  if (e == cudaSuccess && sums) {
    FoldArgs f{};
    f.part = a.part;
    f.groups = groups; f.chunks = a.chunks; f.D = D; f.gate_mode = dgate_mode;
    f.gate = a.gate; f.zdt = z_dtype; f.gate_is_row = a.gate_is_row;
    f.scale = scale; f.post_w = post_w; f.post_b = post_b;
    f.dscale = dscale; f.dgate = static_cast<float*>(dgate);
    f.dpost_w = dpost_w; f.dpost_b = dpost_b; f.dpre_w = dpre_w; f.dpre_b = dpre_b;
    gated_norm_fold_kernel<<<(unsigned)((D + 31) / 32), 512, 0, (cudaStream_t)stream>>>(f);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}
