// sb_xattn_few.cu -- attention of up to 16 query rows an (item, key head): single tokens, and few
// queries of heads that share their keys.
//
// K and V are read once and 4 rows x 4 flops a value do not load the tensor pipe, so memory bounds
// it: what matters is that many bytes are on their way and nothing waits for anything else.  So
// each warp works alone: it streams its own chunks of keys (8 KB of K and V together) by TMA into
// its own three-stage ring, multiplies them with mma.sync m16n8k16 (the 16 rows are the fragment's,
// in registers; the 128-row tiles of tcgen05 would be mostly empty and cost a dozen barriers a tile:
// measured 166 us for 64 x 16 heads of 128 on 8160 ragged states, this kernel 114, 89 % of the copy rate), keeps its own
// running maximum, sum and output, and meets the CTA's other warps once, at the end.  The key range
// is split over CTAs (fp32 partial rows, joined by a second kernel) so that ragged lengths even out.
#include <algorithm>

#include "sb_xattn.cuh"

namespace sb {
namespace {

__device__ int g_few_error;

constexpr int kWarps = 4, kStages = 3;

template <int DH>
struct Few {
  static constexpr int CK = 2048 / DH;  // keys a chunk: 4 KB of K, 4 KB of V
  static constexpr int HALF = Tile<DH>::bytes(CK), STAGE = 2 * HALF;
  static constexpr int RING = kWarps * kStages * STAGE;
  static constexpr int SMEM = 1024 + RING;
  static_assert(HALF == 4096 && RING >= kWarps * 16 * DH * 4, "ring");
};

template <int DH, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, 2)
    attend_few_kernel(const __grid_constant__ FwdArgs a, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap) {
  using C = Few<DH>;
  using T = Tile<DH>;
  constexpr int CK = C::CK, NT = CK / 8, KS = DH / 16, WORDS = (CK + 31) / 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ float2 ml[kWarps][16];
  __shared__ int failed;
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, tig = lane & 3;
  int idx = blockIdx.x;
  const int split = idx % a.splits;
  idx /= a.splits;
  const int kvh = idx % a.Hkv, b = idx / a.Hkv;
  const int count = a.mask.count(b);
  // the item's own keys are split evenly, in whole chunks
  const int chunks = (count + CK - 1) / CK, each = (chunks + a.splits - 1) / a.splits;
  const int first = min(split * each, chunks), n = min(first + each, chunks) - first;
  const int mine = n > warp ? (n - warp + kWarps - 1) / kWarps : 0;  // chunks first + warp, + kWarps ...
  uint8_t* ring = smem + warp * kStages * C::STAGE;

  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int i = 0; i < kStages; ++i) mbar_init(&full[w][i], 1);
    failed = 0;
    fence_mbar_init();
  }
  __syncthreads();
  auto load = [&](int i) {  // the warp's chunk i, by one lane
    const int st = i % kStages, j0 = (first + warp + i * kWarps) * CK;
    uint8_t* dst = ring + st * C::STAGE;
    mbar_arrive_expect_tx(&full[warp][st], C::STAGE);
    for (int x = 0; x < T::BOXES; ++x) {
      tma_load_4d(dst + x * T::box_bytes(CK), &kmap, &full[warp][st], x * T::COLS, j0, kvh, b * a.k_item);
      tma_load_4d(dst + C::HALF + x * T::box_bytes(CK), &vmap, &full[warp][st], x * T::COLS, j0, kvh, b * a.v_item);
    }
  };
  int filled = min(mine, kStages);
  if (lane == 0)
    for (int i = 0; i < filled; ++i) load(i);

  // Q fragments: rows g and g + 8, channels 16 ks + 2 tig (+ 8)
  uint32_t q[KS][4];
  {
    const uint16_t* base = static_cast<const uint16_t*>(a.q.p) + b * a.q.img;
    auto row = [&](int r) -> const uint16_t* {
      const int t = r / a.group;
      return base + t * a.q.row + (long long)(kvh * a.group + r - t * a.group) * DH;
    };
    const uint16_t *q0 = row(g), *q1 = row(g + 8);
    const bool has0 = g < a.rows, has1 = g + 8 < a.rows;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c = ks * 16 + 2 * tig;
      q[ks][0] = has0 ? *reinterpret_cast<const uint32_t*>(q0 + c) : 0u;
      q[ks][1] = has1 ? *reinterpret_cast<const uint32_t*>(q1 + c) : 0u;
      q[ks][2] = has0 ? *reinterpret_cast<const uint32_t*>(q0 + c + 8) : 0u;
      q[ks][3] = has1 ? *reinterpret_cast<const uint32_t*>(q1 + c + 8) : 0u;
    }
  }
  float o[DH / 8][4];
#pragma unroll
  for (int i = 0; i < DH / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  constexpr float lift = kLift<BF16>;
  const float sl = a.scale_log2;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const int krow = lane & 7, kc = lane >> 3;
  const int vrow = ((lane >> 3) & 1) * 8 + (lane & 7), vc = lane >> 4;
  const uint8_t* valid = a.mask.row(b);
  uint32_t next[WORDS];
  auto ask = [&](int i) {
#pragma unroll
    for (int x = 0; x < WORDS; ++x) next[x] = ask_keys(valid, (first + warp + i * kWarps) * CK + 32 * x, count);
  };
  if (valid) ask(0);
  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    const int st = i % kStages, j0 = (first + warp + i * kWarps) * CK;
    uint32_t w[WORDS];
    bool all = true;
#pragma unroll
    for (int x = 0; x < WORDS; ++x) {
      w[x] = valid ? told_keys(next[x]) : bits_below(j0 + 32 * x, count);
      if (CK < 32) w[x] |= 0xFFFFFFFFu << (CK & 31);  // keys of the next chunk
      all = all && w[x] == 0xFFFFFFFFu;
    }
    if (valid) ask(i + 1);
    ok = __all_sync(0xFFFFFFFFu, bounded_wait(&full[warp][st], (i / kStages) & 1));
    if (!ok) break;
    uint8_t* stage = ring + st * C::STAGE;
    const uint32_t kb = smem_u32(stage), vb = kb + C::HALF;
    if (!all) {  // V of keys that take no part may be NaN: zero it (0 x NaN is NaN)
#pragma unroll
      for (int x = 0; x < (CK + 31) / 32; ++x)
        if (32 * x + lane < CK && !(w[x] >> lane & 1u))
          for (int c = 0; c < DH / 8; ++c)
            *reinterpret_cast<uint4*>(stage + C::HALF + T::chunk(CK, 32 * x + lane, c)) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int p = 0; p < KS / 2; ++p) {
        uint32_t f[4];
        ldsm4(kb + T::chunk(CK, nt * 8 + krow, p * 4 + kc), f);
        mma16816<BF16>(s[nt], q[2 * p], f[0], f[1]);
        mma16816<BF16>(s[nt], q[2 * p + 1], f[2], f[3]);
      }
    }
    if (!all) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint32_t bits = w[nt * 8 / 32] >> ((nt * 8 & 31) + 2 * tig);
        if (!(bits & 1u)) s[nt][0] = s[nt][2] = -INFINITY;
        if (!(bits & 2u)) s[nt][1] = s[nt][3] = -INFINITY;
      }
    }
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      t0 = max3(t0, s[nt][0], s[nt][1]);
      t1 = max3(t1, s[nt][2], s[nt][3]);
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      const float u0 = __shfl_xor_sync(0xFFFFFFFFu, t0, x), u1 = __shfl_xor_sync(0xFFFFFFFFu, t1, x);
      t0 = max3(t0, u0, u0);
      t1 = max3(t1, u1, u1);
    }
    // a new reference point with the first keys, and where a maximum grew by more than 2^8 (or is NaN)
    // (what is compared is the exponent that a row's largest P would get)
    float r0 = fmaf(-m0, sl, lift), r1 = fmaf(-m1, sl, lift);
    if (__any_sync(0xFFFFFFFFu, !(fmaf(t0, sl, r0) <= lift + 8.f) || !(fmaf(t1, sl, r1) <= lift + 8.f))) {
      const float n0 = max3(m0, t0, t0), n1 = max3(m1, t1, t1);
      const float c0 = m0 == n0 ? 1.f : exp2_hw((m0 - n0) * sl), c1 = m1 == n1 ? 1.f : exp2_hw((m1 - n1) * sl);
      m0 = n0;
      m1 = n1;
      r0 = fmaf(-m0, sl, lift);
      r1 = fmaf(-m1, sl, lift);
      l0 *= c0;
      l1 *= c1;
#pragma unroll
      for (int x = 0; x < DH / 8; ++x) {
        o[x][0] *= c0;
        o[x][1] *= c0;
        o[x][2] *= c1;
        o[x][3] *= c1;
      }
    }
    if (m0 == -INFINITY) r0 = 0.f;
    if (m1 == -INFINITY) r1 = 0.f;
    uint32_t p[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float p0 = exp2_hw(fmaf(s[nt][0], sl, r0)), p1 = exp2_hw(fmaf(s[nt][1], sl, r0));
      const float p2 = exp2_hw(fmaf(s[nt][2], sl, r1)), p3 = exp2_hw(fmaf(s[nt][3], sl, r1));
      l0 += p0 + p1;
      l1 += p2 + p3;
      p[nt][0] = pack16<BF16>(p0, p1);
      p[nt][1] = pack16<BF16>(p2, p3);
    }
#pragma unroll
    for (int ks = 0; ks < CK / 16; ++ks) {
      const uint32_t pa[4] = {p[2 * ks][0], p[2 * ks][1], p[2 * ks + 1][0], p[2 * ks + 1][1]};
#pragma unroll
      for (int y = 0; y < DH / 16; ++y) {
        uint32_t f[4];
        ldsm4_t(vb + T::chunk(CK, ks * 16 + vrow, y * 2 + vc), f);
        mma16816<BF16>(o[2 * y], pa, f[0], f[1]);
        mma16816<BF16>(o[2 * y + 1], pa, f[2], f[3]);
      }
    }
    __syncwarp();  // every lane has read the stage
    if (filled < mine) {
      if (lane == 0) {
        fence_proxy_async_smem();
        load(filled);
      }
      ++filled;
    }
    __syncwarp();
  }
  if (!ok) {
    if (lane == 0) {
      failed = 1;
      atomicOr(&g_few_error, SB_ERR_TIMEOUT_FULL);
      for (int i = max(0, filled - kStages); i < filled; ++i) bounded_wait(&full[warp][i % kStages], (i / kStages) & 1);
    }
    __syncwarp();
  }
#pragma unroll
  for (int x = 1; x <= 2; x <<= 1) {
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, x);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, x);
  }
  // the warps' outputs meet in shared memory, rows [warp][16][DH], over the rings
  __syncthreads();
  float* all_o = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int x = 0; x < DH / 8; ++x) {
    float* d0 = all_o + (warp * 16 + g) * DH + x * 8 + 2 * tig;
    *reinterpret_cast<float2*>(d0) = make_float2(o[x][0], o[x][1]);
    *reinterpret_cast<float2*>(d0 + 8 * DH) = make_float2(o[x][2], o[x][3]);
  }
  if (tig == 0) {
    ml[warp][g] = make_float2(m0, l0);
    ml[warp][g + 8] = make_float2(m1, l1);
  }
  __syncthreads();
  if (failed) return;
  constexpr int per = DH / 8;
  for (int i = threadIdx.x; i < a.rows * per; i += kWarps * 32) {
    const int r = i / per, c = (i - r * per) * 8;
    float top = -INFINITY, l = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max3(top, ml[w][r].x, ml[w][r].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = ml[w][r].x, k = mw == top ? 1.f : exp2_hw((mw - top) * sl);
      l = fmaf(k, ml[w][r].y, l);
      const float4* src = reinterpret_cast<const float4*>(all_o + (w * 16 + r) * DH + c);
      const float4 x = src[0], y = src[1];
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] = fmaf(k, v[u], f[u]);
    }
    const bool none = top == -INFINITY;  // no keys
    const float inv = none ? 0.f : 1.f / l;
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] = none ? 0.f : f[u] * inv;
    const float lse = none ? -INFINITY : fmaf(top, sl, -lift) * 0.69314718055994531f + logf(l);
    const int t = r / a.group, h = kvh * a.group + r - t * a.group;
    const long long rr = ((long long)b * a.H + h) * a.Tq + t;
    if (a.splits > 1) {
      if (!none) store8(a.part_o, SB_F32, (split * a.all_rows + rr) * DH + c, f);
      if (c == 0) a.part_l[split * a.all_rows + rr] = lse;
    } else {
      store8(a.o.p, BF16 ? SB_BF16 : SB_F16, b * a.o.img + t * a.o.row + (long long)h * DH + c, f);
      if (a.lse && c == 0) a.lse[rr] = lse;
    }
  }
}

// Joins the splits' rows: out = sum_s e^(L_s - L) O_s, L = log sum_s e^L_s.  A warp takes a row: its lanes
// find the largest L_s, then take eight channels each of several splits at once (there may be 128).  A
// split without keys (L_s = -inf) has not written its O_s.
template <int DH, bool BF16>
__global__ void __launch_bounds__(128) few_join_kernel(const __grid_constant__ FwdArgs a) {
  constexpr int per = DH / 8, lanes = 32 / per;  // threads of a split's row, splits at once
  const int lane = lane_id();
  const long long rr = (long long)blockIdx.x * 4 + warp_id();
  if (rr >= a.all_rows) return;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, a.part_l[s * a.all_rows + rr]);
#pragma unroll
  for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
  const int c = lane % per * 8, s0 = lane / per;
  float f[9] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // channels, sum of weights
#pragma unroll 4
  for (int s = s0; s < a.splits; s += lanes) {
    const float ls = a.part_l[s * a.all_rows + rr];
    if (ls == -INFINITY) continue;
    const float w = expf(ls - top);
    float v[8];
    unpack8(load_raw8(a.part_o, SB_F32, (s * a.all_rows + rr) * DH + c), SB_F32, v);
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] = fmaf(w, v[u], f[u]);
    f[8] += w;
  }
#pragma unroll
  for (int x = per; x < 32; x <<= 1)
#pragma unroll
    for (int u = 0; u < 9; ++u) f[u] += __shfl_xor_sync(0xFFFFFFFFu, f[u], x);
  if (s0 != 0) return;
  const float inv = f[8] != 0.f ? 1.f / f[8] : 0.f;
  float v[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) v[u] = f[u] * inv;
  const int t = (int)(rr % a.Tq), h = (int)(rr / a.Tq % a.H);
  const long long b = rr / a.Tq / a.H;
  store8(a.o.p, BF16 ? SB_BF16 : SB_F16, b * a.o.img + t * a.o.row + (long long)h * DH + c, v);
  if (a.lse && c == 0) a.lse[rr] = f[8] != 0.f ? top + logf(f[8]) : -INFINITY;
}

template <int DH, bool BF16>
cudaError_t launch(const FwdArgs& a, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  static bool ready[64];
  const cudaError_t e = xattn_smem(reinterpret_cast<const void*>(&attend_few_kernel<DH, BF16>), Few<DH>::SMEM, ready);
  if (e != cudaSuccess) return e;
  attend_few_kernel<DH, BF16>
      <<<(unsigned)((long long)a.B * a.Hkv * a.splits), kWarps * 32, Few<DH>::SMEM, st>>>(a, k, v);
  return cudaGetLastError();
}
template <int DH, bool BF16>
cudaError_t join(const FwdArgs& a, cudaStream_t st) {
  few_join_kernel<DH, BF16><<<(unsigned)((a.all_rows + 3) / 4), 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

int few_keys(int dh) { return 2048 / dh; }

// About three CTAs a place (two an SM), so that ragged lengths even out, but a split for each 256 keys begun
// at most.
int few_splits(long long units, int Tk, int sms) {
  const long long want = (3ll * 2 * sms + units - 1) / units;
  return (int)std::max(1ll, std::min({want, ((long long)Tk + 255) / 256, 128ll}));
}

cudaError_t few_launch(const FwdArgs& a, int dh, bool bf16, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  if (bf16) return dh == 32 ? launch<32, true>(a, k, v, st) : dh == 64 ? launch<64, true>(a, k, v, st) : launch<128, true>(a, k, v, st);
  return dh == 32 ? launch<32, false>(a, k, v, st) : dh == 64 ? launch<64, false>(a, k, v, st) : launch<128, false>(a, k, v, st);
}
cudaError_t few_join(const FwdArgs& a, int dh, bool bf16, cudaStream_t st) {
  if (bf16) return dh == 32 ? join<32, true>(a, st) : dh == 64 ? join<64, true>(a, st) : join<128, true>(a, st);
  return dh == 32 ? join<32, false>(a, st) : dh == 64 ? join<64, false>(a, st) : join<128, false>(a, st);
}

int few_error(int clear, int* flags) {
  const int zero = 0;
  if (cudaMemcpyFromSymbol(flags, g_few_error, sizeof(int)) != cudaSuccess) return -1;
  return clear && cudaMemcpyToSymbol(g_few_error, &zero, sizeof(int)) != cudaSuccess ? -1 : 0;
}

}  // namespace sb
