// sb_gnorm.cu -- the end of one transformer block and the start of the next in one pass:
//   n = Npost(z),  y = x + scale * gate * n,  h = Npre(y)
// (each norm optional, RMS or layer norm, fp32 statistics), and its gradients.
//
// Forward, per row v of D values: RMS norm v r w with r = (mean v^2 + eps)^-1/2; layer norm
// (v - m) r w + b with r = (mean (v - m)^2 + eps)^-1/2 (the mean first, then the centred
// squares: no cancellation).  Apart, the norms and the residual sum would read and write the
// rows five times; here x and z are read and y and h written once, which bounds the kernel.
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
// A row belongs to one warp, or to all of a CTA's threads, NV vectors of eight columns each; a
// CTA walks its rows with the next row's loads issued before the current row's reductions.  Element
// types are compile-time for the usual pairs (DT of the template), so a row costs few registers
// and no selects.
#include <algorithm>

#include "sb_rows.cuh"

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
  long long step_b;    // a CTA's step from row to row as (items, rows): no division in the loop
  int step_t;
  void *y, *h;         // forward
  long long y_row, y_img, h_row, h_img;
  void *dx, *dz, *dgate_rows;  // backward
  float* part;                 // [groups * chunks][kSums][D]
  long long group_rows;        // rows that share their column sums (T for an image's gate, B * T else)
  int chunks, gate_is_row;     // CTAs a group
};

// Sum of a pair of values over the threads of a row; the two halves of the buffer alternate, so one
// barrier a reduction is enough.
struct RowSum {
  float2* buf;  // [2][32]
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

template <bool VEC>
SB_DEV Raw8 fetch(const void* p, int dt, long long i, int n) {
  if constexpr (VEC) return n > 0 ? load_raw8(p, dt, i) : Raw8{};
  else return load_raw8_tail(p, dt, i, n);
}
template <bool VEC>
SB_DEV void put(void* p, int dt, long long i, const float (&v)[8], int n) {
  if constexpr (VEC) {
    if (n > 0) store8(p, dt, i, v);
  } else {
    store8_tail(p, dt, i, v, n);
  }
}
template <bool VEC>
SB_DEV void columns(const float* w, int c, int n, float other, float (&v)[8]) {
  if (!w) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = other;
    return;
  }
  unpack8(fetch<VEC>(w, SB_F32, c, n), SB_F32, v);
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

// XD, ZD: dtype codes of x and z, -1: as the arguments say
template <int XD, int ZD, bool VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 buf[64];
  const int xdt = XD < 0 ? a.xdt : XD, zdt = ZD < 0 ? a.zdt : ZD;
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
      rx[j] = fetch<VEC>(a.x.p, xdt, xo + c, m);
      rz[j] = fetch<VEC>(a.z.p, zdt, zo + c, m);
      if (a.gate.p) rg[j] = fetch<VEC>(a.gate.p, zdt, go + c, m);
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
      columns<VEC>(a.scale, c, n, 1.f, s);
      if (a.post_w) {
        columns<VEC>(a.post_w, c, n, 1.f, w);
        columns<VEC>(a.post_b, c, n, 0.f, o);
#pragma unroll
        for (int u = 0; u < 8; ++u) v[j][u] = fmaf((v[j][u] - mean) * rs, w[u], o[u]);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) y[j][u] = u < n ? fmaf(s[u] * g[j][u], v[j][u], y[j][u]) : 0.f;
      put<VEC>(a.y, xdt, b * a.y_img + t * a.y_row + c, y[j], n);
    }
    if (a.h) {
      stats_of(y, cols, a.layer, inv_d, a.eps, sum, mean, rs);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = cols.at(j), n = cols.n(j);
        float w[8], o[8];
        columns<VEC>(a.pre_w, c, n, 1.f, w);
        columns<VEC>(a.pre_b, c, n, 0.f, o);
#pragma unroll
        for (int u = 0; u < 8; ++u) y[j][u] = fmaf((y[j][u] - mean) * rs, w[u], o[u]);
        put<VEC>(a.h, zdt, b * a.h_img + t * a.h_row + c, y[j], n);
      }
    }
    b = nb;
    t = nt;
  }
}

template <int XD, int ZD, bool VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) gated_norm_back_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 buf[64];
  extern __shared__ float fold[];  // [per][kSums][D padded]: several rows' warps meet here
  const int xdt = XD < 0 ? a.xdt : XD, zdt = ZD < 0 ? a.zdt : ZD;
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
      rz[j] = fetch<VEC>(a.z.p, zdt, bb * a.z.img + tt * a.z.row + c, m);
      rdy[j] = fetch<VEC>(a.dy.p, xdt, bb * a.dy.img + tt * a.dy.row + c, a.dy.p ? m : 0);
      if (a.dh.p) {
        rx[j] = fetch<VEC>(a.x.p, xdt, bb * a.x.img + tt * a.x.row + c, m);
        rdh[j] = fetch<VEC>(a.dh.p, zdt, bb * a.dh.img + tt * a.dh.row + c, m);
      }
      if (a.gate.p) rg[j] = fetch<VEC>(a.gate.p, zdt, bb * a.gate.img + tt * a.gate.row + c, m);
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
        columns<VEC>(a.scale, c, n, 1.f, s);
        columns<VEC>(a.post_w, c, n, 1.f, w);
        columns<VEC>(a.post_b, c, n, 0.f, o);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          y[j][u] = u < n ? fmaf(s[u] * g[j][u], fmaf(zh[j][u], w[u], o[u]), y[j][u]) : 0.f;
      }
      float mean, rs, e0 = 0.f, e1 = 0.f;
      stats_of(y, cols, a.layer, inv_d, a.eps, sum, mean, rs);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float w[8];
        columns<VEC>(a.pre_w, cols.at(j), cols.n(j), 1.f, w);
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
      put<VEC>(a.dx, xdt, r * a.D + c, d[j], n);
      float s[8], w[8];
      columns<VEC>(a.scale, c, n, 1.f, s);
      columns<VEC>(a.post_w, c, n, 1.f, w);
      if (a.dgate_rows) {
        float o[8], dg[8];
        columns<VEC>(a.post_b, c, n, 0.f, o);
#pragma unroll
        for (int u = 0; u < 8; ++u) dg[u] = d[j][u] * s[u] * fmaf(zh[j][u], w[u], o[u]);
        put<VEC>(a.dgate_rows, zdt, r * a.D + c, dg, n);
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
      put<VEC>(a.dz, zdt, r * a.D + cols.at(j), d[j], cols.n(j));
    }
  }
  if (!a.part) return;
  float* mine = a.part + (long long)blockIdx.x * kSums * a.D;
  if (a.per == 1) {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int j = 0; j < NV; ++j) put<VEC>(mine, SB_F32, (long long)k * a.D + cols.at(j), acc[k][j], cols.n(j));
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

// Up to 256 channels a warp takes a row with one vector a lane, eight (backward: four) rows a CTA;
// above, a CTA takes a row: two vectors a thread forward and, with its column sums in registers, one
// backward up to 2048 channels and two above.
struct Plan {
  int kind;  // of the launch tables
  int tpr, per, threads;
};
Plan plan_of(int D, bool back) {
  Plan p;
  const int vecs = (D + 7) / 8;
  if (vecs <= 32) {
    p = {0, 32, back ? 4 : 8, 0};
  } else if (!back) {
    p.tpr = ((vecs + 1) / 2 + 31) / 32 * 32;
    p.kind = p.tpr <= 128 ? 1 : 2;
    p.per = 1;
  } else {
    p.kind = vecs <= 256 ? 1 : 2;
    p.tpr = (p.kind == 1 ? vecs + 31 : (vecs + 1) / 2 + 31) / 32 * 32;
    p.per = 1;
  }
  p.threads = p.tpr * p.per;
  return p;
}

using NormKernel = void (*)(const NormArgs);

template <int XD, int ZD, bool VEC>
NormKernel norm_kernel(int kind) {
  return kind == 0 ? gated_norm_kernel<XD, ZD, VEC, 1, 256> : kind == 1 ? gated_norm_kernel<XD, ZD, VEC, 2, 128>
                                                                        : gated_norm_kernel<XD, ZD, VEC, 2, 512>;
}
template <int XD, int ZD, bool VEC>
NormKernel back_kernel(int kind) {
  return kind == 0 ? gated_norm_back_kernel<XD, ZD, VEC, 1, 128> : kind == 1 ? gated_norm_back_kernel<XD, ZD, VEC, 1, 256>
                                                                             : gated_norm_back_kernel<XD, ZD, VEC, 2, 512>;
}
NormKernel pick(bool back, int xdt, int zdt, bool vec, int kind) {
#define SB_PICK(X, Z, V) (back ? back_kernel<X, Z, V>(kind) : norm_kernel<X, Z, V>(kind))
  if (!vec) return SB_PICK(-1, -1, false);
  if (xdt == SB_F32 && zdt == SB_F16) return SB_PICK(SB_F32, SB_F16, true);
  if (xdt == SB_F32 && zdt == SB_BF16) return SB_PICK(SB_F32, SB_BF16, true);
  if (xdt == SB_F16 && zdt == SB_F16) return SB_PICK(SB_F16, SB_F16, true);
  if (xdt == SB_BF16 && zdt == SB_BF16) return SB_PICK(SB_BF16, SB_BF16, true);
  return SB_PICK(-1, -1, true);
#undef SB_PICK
}

// CTAs a group of rows: about `kBackCtas` a SM over all groups, at least eight rows a warp or CTA
constexpr int kBackCtas = 3;
int chunks_of(int groups, long long group_rows, const Plan& p, int sms) {
  const long long want = std::max(1, kBackCtas * sms / groups);
  return (int)std::max(1ll, std::min(want, (group_rows + 8 * p.per - 1) / (8 * p.per)));
}

bool rows_aligned(const void* p, int dt, long long row, long long img) {
  const int e = dtype_bytes(dt);
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row * e % 16 == 0 && img * e % 16 == 0;
}
bool cols_aligned(const float* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
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
  if (!x || !z || !y || (pre_w != nullptr) != (h != nullptr) || (post_b && !post_w) || (pre_b && !pre_w))
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
  const bool vec = D % 8 == 0 && rows_aligned(x, x_dtype, x_row, x_img) && rows_aligned(z, z_dtype, z_row, z_img) &&
                   (!gate || rows_aligned(gate, z_dtype, gate_row, gate_img)) &&
                   rows_aligned(y, x_dtype, y_row, y_img) && (!h || rows_aligned(h, z_dtype, h_row, h_img)) &&
                   cols_aligned(scale) && cols_aligned(post_w) && cols_aligned(post_b) && cols_aligned(pre_w) &&
                   cols_aligned(pre_b);
  const int sms = sm_count();
  if (sms == 0) return record_error(SB_ECUDA, "sb_gated_norm: device");
  const NormKernel kernel = pick(false, x_dtype, z_dtype, vec, p.kind);
  int ctas = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, p.threads, 0) != cudaSuccess || ctas < 1)
    return record_error(SB_ECUDA, "sb_gated_norm: occupancy");
  const long long grid = std::min((a.rows + p.per - 1) / p.per, (long long)sms * ctas);
  const long long step = grid * p.per;
  a.step_b = step / T;
  a.step_t = (int)(step % T);
  kernel<<<(unsigned)grid, p.threads, 0, (cudaStream_t)stream>>>(a);
  const cudaError_t e = cudaGetLastError();
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
  if (!x || !z || !dx || !dz || (dh && !pre_w) || (post_b && !post_w) || (pre_b && !pre_w) || dgate_mode < 0 ||
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
  const bool vec = D % 8 == 0 && rows_aligned(x, x_dtype, x_row, x_img) && rows_aligned(z, z_dtype, z_row, z_img) &&
                   (!gate || rows_aligned(gate, z_dtype, gate_row, gate_img)) &&
                   (!dy || rows_aligned(dy, x_dtype, dy_row, dy_img)) &&
                   (!dh || rows_aligned(dh, z_dtype, dh_row, dh_img)) && rows_aligned(dx, x_dtype, 0, 0) &&
                   rows_aligned(dz, z_dtype, 0, 0) && (dgate_mode != 3 || rows_aligned(dgate, z_dtype, 0, 0)) &&
                   cols_aligned(scale) && cols_aligned(post_w) && cols_aligned(post_b) && cols_aligned(pre_w) &&
                   cols_aligned(pre_b);
  const NormKernel kernel = pick(true, x_dtype, z_dtype, vec, p.kind);
  const int smem = sums && p.per > 1 ? p.per * kSums * p.tpr * 8 * 4 : 0;
  if ((long long)groups * a.chunks > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_gated_norm_backward: too many items");
  kernel<<<(unsigned)(groups * a.chunks), p.threads, smem, (cudaStream_t)stream>>>(a);
  if (sums) {
    FoldArgs f{};
    f.part = a.part;
    f.groups = groups; f.chunks = a.chunks; f.D = D; f.gate_mode = dgate_mode;
    f.gate = a.gate; f.zdt = z_dtype; f.gate_is_row = a.gate_is_row;
    f.scale = scale; f.post_w = post_w; f.post_b = post_b;
    f.dscale = dscale; f.dgate = static_cast<float*>(dgate);
    f.dpost_w = dpost_w; f.dpost_b = dpost_b; f.dpre_w = dpre_w; f.dpre_b = dpre_b;
    gated_norm_fold_kernel<<<(unsigned)((D + 31) / 32), 512, 0, (cudaStream_t)stream>>>(f);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}
