// sb_xattn_bwd.cu -- gradients of the attention of queries to an encoder's states.
//
// With P = exp(scale q k^T - L), dP = dout v^T, D_i = dout_i.out_i and dS = P (dP - D):
//   dq = scale dS k,   dk = scale dS^T q,   dv = P^T dout   (dk, dv summed over the query heads that
// share a key head).  Two kernels of one form, each owning its results, so that no sum needs an
// atomic and the same inputs give the same bits:
//   SIDE 0 (dq)      a CTA holds 128 query rows (q, dout) and streams 128-row tiles of k, v
//   SIDE 1 (dk, dv)  a CTA holds 128 keys (k, v) and streams 128-row tiles of q, dout, head by head
// Per step, with X the held and Y the streamed operands:
//   S = X1 Y1^T, R = X2 Y2^T (128 x 128; X in TMEM where its 512 columns have room)
//   sixteen softmax warps, four threads a held row: P from S and dS from P and R, rounded to the operands'
//   type, to TMEM (SIDE 1: over S and R, which they replace)
//   acc1 += dS Y1 (dq, dk),  SIDE 1: acc2 += P Y2 (dv)     (A in TMEM, B the rows as they lie)
// Steps of 64 streamed rows (two buffers each of S and R) were half as fast: a product of 64 columns
// takes as long as one of 128, 60 of 68 clocks.  So there is one buffer, and what overlaps is the halves
// of a step: one warp issues S and acc2, another R and acc1 (in SIDE 1 acc2 of a step, then the next S;
// acc1, then the next R), so P's half runs while dS is computed, and the next S while dS's half runs.
// S and R are computed on both sides (7 products instead of 5): against one kernel that adds up dq in
// global memory this costs 2 of 7 products and saves the atomics.
//
// fp16 gradients: P and dS may be far below fp16's smallest normal number (long memories, small
// losses).  P is held as 2^14 P, and dS as F dS with F the power of two that the bound |dS_i| <= 2 P_i
// |dout_i| max|v_j| (norms from a first kernel that also forms D, the largest over the item and key head) keeps
// below 2^15; both factors leave at the end.  For dq each row has its own F, so that one query with a
// gradient 2^23 times the others' takes nothing from theirs; dk and dv add rows up and have one F of the largest
// |dout_i| of an item and key head.  bf16 has fp32's range and needs neither.
//
// A range of steps may be split over CTAs (few rows against many): these write fp32 partial
// results, which a last kernel adds in order.
//
// 2 x 16 heads of 128 channels (4 key heads), 2040 queries, 8160 keys: 1126 us, 606 TFLOP/s of the five
// products' operations, 848 of the seven that are done; what is left is waits, as in the forward kernel.
// 8 x 8 heads of 64 channels, 300 queries, up to 2040 keys: 136 us, of them 12 for the first kernel, 42 for
// dq and 84 for dk and dv, whose CTAs have three steps each: starting and ending take most of theirs.
#include <algorithm>
#include <cmath>

#include "sb_xattn.cuh"

namespace sb {
namespace {

__device__ int g_xattn_bwd_error;

constexpr int kStep = 128;  // streamed rows a step
constexpr int kSoft = 16;   // softmax warps: 32 streamed rows (w / 4), TMEM lanes (w % 4)

struct BackArgs {
  View q, k, v, out, dout;
  OutView dq, dk, dv;
  const float* lse;
  KeyMask mask;
  int dt, B, H, Hkv, group, Tq, Tk;
  int x_tiles, splits, steps;  // held tiles of an (item, key head); splits of its steps
  int y1_item, y2_item;  // 0: one memory for every item
  int masked;
  float scale, scale_log2;
  float* lse2;   // [B][H][Tq] L log2 e, +inf for a row without keys
  float* delta;  // [B][H][Tq]
  float* norm;   // [B][H][Tq] |dout_i| (fp16 only)
  unsigned* top;  // [B][Hkv][2] bits of max |dout_i|, max |v_j| (fp16 only)
  float* part;   // [splits][held rows of all][DH] (SIDE 1: dk, then dv)
  long long part_rows;
};

// ---------------------------------------------------------------- D, L log2 e and the norms
// blockIdx.x < B * H: rows of a head (DH / 8 threads each); above: keys of a key head
template <int DH>
__global__ void __launch_bounds__(256) attend_back_rows_kernel(const __grid_constant__ BackArgs a) {
  constexpr int per = DH / 8, rows = 256 / per;
  const int c = (threadIdx.x % per) * 8, sub = threadIdx.x / per;
  const bool keys = blockIdx.x >= (unsigned)(a.B * a.H);
  const int who = keys ? blockIdx.x - a.B * a.H : blockIdx.x;
  const int heads = keys ? a.Hkv : a.H;
  const int b = who / heads, h = who % heads;
  const int n = keys ? a.mask.count(b) : a.Tq;
  float top = 0.f;
  for (int t = blockIdx.y * rows + sub; t - sub < n; t += gridDim.y * rows) {
    float d = 0.f, sq = 0.f;
    bool use = t < n;
    if (keys && use && a.mask.valid) use = a.mask.valid[b * a.mask.valid_img + t] != 0;
    if (use) {
      const View& src = keys ? a.v : a.dout;
      float g[8], o[8];
      unpack8(load_raw8(src.p, a.dt, b * src.img + t * src.row + (long long)h * DH + c), a.dt, g);
      if (!keys) unpack8(load_raw8(a.out.p, a.dt, b * a.out.img + t * a.out.row + (long long)h * DH + c), a.dt, o);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (!keys) d = fmaf(g[u], o[u], d);
        sq = fmaf(g[u], g[u], sq);
      }
    }
#pragma unroll
    for (int x = per / 2; x; x >>= 1) {
      d += __shfl_xor_sync(0xFFFFFFFFu, d, x);
      sq += __shfl_xor_sync(0xFFFFFFFFu, sq, x);
    }
    top = fmaxf(top, sqrtf(sq));
    if (!keys && use && c == 0) {
      const long long r = (long long)who * a.Tq + t;
      const float l = a.lse[r];
      a.delta[r] = l == -INFINITY ? 0.f : d;
      a.lse2[r] = l == -INFINITY ? INFINITY : l * 1.4426950408889634f;
      if (a.dt == SB_F16) a.norm[r] = sqrtf(sq);
    }
  }
  if (a.dt != SB_F16) return;
#pragma unroll
  for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
  __shared__ float sh[8];
  if (lane_id() == 0) sh[warp_id()] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) top = fmaxf(top, sh[i]);
    const int kvh = keys ? h : h / a.group;
    // a maximum does not depend on the order
    atomicMax(&a.top[(b * a.Hkv + kvh) * 2 + keys], __float_as_uint(top));
  }
}

// ---------------------------------------------------------------- the products
template <int DH, int SIDE>
struct Back {
  // TMEM columns: S, R (SIDE 1: P and dS over them), dS (SIDE 0), acc1, acc2, X1, X2 (XT of them)
  static constexpr int R0 = kStep, D0 = 2 * kStep, ACC = D0 + (SIDE == 0 ? kStep / 2 : 0), X0 = ACC + (1 + SIDE) * DH;
  static constexpr int XT = DH < 128 ? 2 : SIDE == 0 ? 1 : 0;
  static constexpr int XS = Tile<DH>::bytes(128);    // a held operand in shared memory
  static constexpr int XB = (2 - XT) * XS;
  static constexpr int YB = Tile<DH>::bytes(kStep);  // a streamed operand
  static constexpr int SB = 2 * YB;                  // a stage
  static constexpr int STAT = SIDE ? kSoft * 2 * 64 * 4 : 0;  // L and D of a step's queries, a warp each
  static constexpr int ROOM = 224 * 1024 - XB - STAT;
  static constexpr int STAGES = ROOM / SB < 8 ? ROOM / SB : 8;
  static constexpr int SMEM = 1024 + XB + STAGES * SB + STAT + 512;
  static constexpr int THREADS = (kSoft + 4) * 32;
  static_assert(STAGES >= 2 && X0 + XT * DH / 2 <= 512, "ring and TMEM");
};

template <int DH, bool BF16, int SIDE>
__global__ void __launch_bounds__(Back<DH, SIDE>::THREADS, 1)
    attend_back_kernel(const __grid_constant__ BackArgs a, const __grid_constant__ CUtensorMap y1map,
                       const __grid_constant__ CUtensorMap y2map) {
  using C = Back<DH, SIDE>;
  using T = Tile<DH>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + C::XB;
  float* stat = reinterpret_cast<float*>(ring + ST * C::SB);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + ST * C::SB + C::STAT);
  uint64_t* empty = full + ST;
  uint64_t* clean = empty + ST;  // [ST]
  uint64_t* x_full = clean + ST;
  uint64_t* s_full = x_full + 1;  // S computed
  uint64_t* r_full = s_full + 1;
  uint64_t* s_free = r_full + 1;  // SIDE 0: S taken into registers
  uint64_t* r_free = s_free + 1;
  uint64_t* p_full = r_free + 1;  // SIDE 1: P written
  uint64_t* d_full = p_full + 1;  // dS written
  uint64_t* d_free = d_full + 1;  // SIDE 0: and read by the accumulation
  uint64_t* acc_full = d_free + 1;
  uint64_t* dbar = acc_full + 1;  // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(dbar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = warp_id(), lane = lane_id();

  int idx = blockIdx.x;
  const int tile = idx % a.x_tiles;
  idx /= a.x_tiles;
  const int split = idx % a.splits;
  idx /= a.splits;
  const int kvh = idx % a.Hkv, b = idx / a.Hkv;
  const int count = a.mask.count(b);
  const int q_tiles = (a.Tq + kStep - 1) / kStep;  // SIDE 1: steps a head
  // steps with anything to do, split evenly: key tiles that begin before the item's end; all, if the held
  // keys do
  const int all = SIDE == 0 ? (count + kStep - 1) / kStep : tile * 128 < count ? a.steps : 0;
  const int each = (all + a.splits - 1) / a.splits, first = min(split * each, all), n = min(first + each, all) - first;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);  // both issuers
      mbar_init(&clean[i], 1);
    }
    for (uint64_t* bar : {x_full, s_free, r_free, p_full, d_full}) mbar_init(bar, kSoft);
    for (uint64_t* bar : {s_full, r_full, d_free, &dbar[0], &dbar[1]}) mbar_init(bar, 1);
    mbar_init(acc_full, 1 + SIDE);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kSoft) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  auto give_up = [&](int code) {
    *abort_flag = 1;
    atomicOr(&g_xattn_bwd_error, code);
  };

  if (warp == kSoft + 2) {
    if (lane == 0 && n > 0) {  // loader
      int p = 0;
      for (; p < n; ++p) {
        const int st = p % ST;
        if (p >= ST && !mbar_wait(&empty[st], ((p / ST) - 1) & 1, abort_flag)) {
          give_up(SB_ERR_TIMEOUT_EMPTY);
          break;
        }
        mbar_arrive_expect_tx(&full[st], C::SB);
        const int step = first + p;
        const int row = SIDE == 0 ? step * kStep : step % q_tiles * kStep;
        const int head = SIDE == 0 ? kvh : kvh * a.group + step / q_tiles;
        for (int x = 0; x < T::BOXES; ++x) {
          uint8_t* dst = ring + st * C::SB + x * T::box_bytes(kStep);
          tma_load_4d(dst, &y1map, &full[st], x * T::COLS, row, head, b * a.y1_item);
          tma_load_4d(dst + C::YB, &y2map, &full[st], x * T::COLS, row, head, b * a.y2_item);
        }
      }
      if (*abort_flag)
        for (int i = max(0, p - ST); i < p; ++i) bounded_wait(&full[i % ST], (i / ST) & 1);
    }
  } else if (warp == kSoft || warp == kSoft + 1) {
    if (lane == 0 && n > 0) {  // issuers: of S and acc2, of R and acc1
      const bool second = warp == kSoft + 1;
      const uint32_t xb = smem_u32(smem), rb = smem_u32(ring);
      constexpr uint32_t id_s = idesc_16bit(BF16, 128, kStep, false), id_a = idesc_16bit(BF16, 128, DH, true);
      auto landed = [&](int i) { return mbar_wait(&full[i % ST], (i / ST) & 1, abort_flag); };
      // S or R of step i
      auto scores = [&](int i) {
        tc_fence_after();
        const uint32_t y = rb + i % ST * C::SB + (second ? C::YB : 0), d = tmem + (second ? C::R0 : 0);
#pragma unroll
        for (int ks = 0; ks < T::KSTEPS; ++ks) {
          const uint64_t yd = T::k_major(y, kStep, ks);
          if (C::XT == 2 || (C::XT == 1 && !second))
            mma_f16_ts(d, tmem + C::X0 + (second ? DH / 2 : 0) + ks * 8, yd, id_s, ks > 0);
          else
            mma_f16_ss(d, T::k_major(xb + (second && C::XT == 0 ? C::XS : 0), 128, ks), yd, id_s, ks > 0);
        }
        mma_commit(second ? r_full : s_full);
      };
      // acc2 += P Y2 or acc1 += dS Y1 of step i; rows 16 k .. of P and dS (SIDE 1: each warp's over its scores)
      auto accumulate = [&](int i) {
        tc_fence_after();
        const uint32_t y = rb + i % ST * C::SB + (second ? 0 : C::YB);
        const uint32_t from = tmem + (second ? (SIDE == 0 ? C::D0 : C::R0) : 0), to = tmem + C::ACC + (second ? 0 : DH);
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          mma_f16_ts(to, from + (SIDE == 0 ? k * 8 : (k >> 1) * 32 + (k & 1) * 8), T::mn_major(y, kStep, k), id_a,
                     i > 0 || k > 0);
        if (SIDE == 0) mma_commit(d_free);
        mma_commit(&empty[i % ST]);
      };
      bool ok = mbar_wait(x_full, 0, abort_flag) && landed(0);
      if (ok) scores(0);
      if (SIDE == 0 && !second) {
        if (ok) mma_commit(&empty[0]);
        for (int i = 1; i < n && ok; ++i) {
          ok = landed(i) && mbar_wait(s_free, (i - 1) & 1, abort_flag);
          if (!ok) break;
          scores(i);
          mma_commit(&empty[i % ST]);
        }
      } else if (SIDE == 0) {
        for (int i = 0; i < n && ok; ++i) {
          if (i + 1 < n) {
            ok = landed(i + 1) && mbar_wait(r_free, i & 1, abort_flag);
            if (!ok) break;
            scores(i + 1);
          }
          ok = (!a.masked || mbar_wait(&clean[i % ST], (i / ST) & 1, abort_flag)) && mbar_wait(d_full, i & 1, abort_flag);
          if (!ok) break;
          accumulate(i);
        }
        if (ok) mma_commit(acc_full);
      } else {
        for (int i = 0; i < n && ok; ++i) {
          ok = (i + 1 == n || ST == 1 || landed(i + 1)) && mbar_wait(second ? d_full : p_full, i & 1, abort_flag);
          if (!ok) break;
          accumulate(i);
          if (i + 1 < n) scores(i + 1);
        }
        if (ok) mma_commit(acc_full);
      }
      if (!ok) {
        give_up(SB_ERR_TIMEOUT_FULL);
        mma_commit(&dbar[second]);
        bounded_wait(&dbar[second], 0);
      }
    }
  } else if (warp == kSoft + 3) {
    if (SIDE == 0 && a.masked) {  // cleaner: k's rows of keys that take no part, mask bytes two tiles ahead
      const uint8_t* vrow = a.mask.row(b);
      uint32_t next[2][kStep / 32];
      if (vrow) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int x = 0; x < kStep / 32; ++x) next[y][x] = ask_keys(vrow, (first + y) * kStep + 32 * x, count);
      }
#pragma unroll 2
      for (int i = 0; i < n; ++i) {
        const int st = i % ST, j0 = (first + i) * kStep;
        uint32_t w[kStep / 32];
#pragma unroll
        for (int x = 0; x < kStep / 32; ++x) {
          if (vrow) {
            w[x] = told_keys(next[i & 1][x]);
            next[i & 1][x] = ask_keys(vrow, j0 + 2 * kStep + 32 * x, count);
          } else {
            w[x] = bits_below(j0 + 32 * x, count);
          }
        }
        if (!warp_wait(&full[st], (i / ST) & 1, abort_flag)) {
          if (lane == 0) give_up(SB_ERR_TIMEOUT_FULL);
          break;
        }
        bool touched = false;
#pragma unroll
        for (int x = 0; x < kStep / 32; ++x) {
          if (w[x] == 0xFFFFFFFFu) continue;
          touched = true;
          if (!(w[x] >> lane & 1u))
            for (int c = 0; c < DH / 8; ++c)
              *reinterpret_cast<uint4*>(ring + st * C::SB + T::chunk(kStep, 32 * x + lane, c)) = make_uint4(0, 0, 0, 0);
        }
        if (touched) fence_proxy_async_smem();
        warp_arrive(&clean[st]);
      }
    }
  } else {
    const int cg = warp >> 2, quad = warp & 3;  // streamed rows 32 cg .., held rows 32 quad ..
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_at = tmem + lanes + cg * 32, r_at = s_at + C::R0;
    const uint32_t p_at = s_at, d_at = SIDE == 0 ? tmem + lanes + C::D0 + cg * 16 : r_at;
    const int u = cg >> 1, hf = cg & 1;  // what it loads and stores: operand or accumulator, half of its channels
    const int x = tile * 128 + quad * 32 + lane;  // held row: query row of the group, or key
    const int rows = SIDE == 0 ? a.group * a.Tq : a.Tk;
    const int tq = SIDE == 0 ? x / a.group : 0, h = kvh * a.group + (SIDE == 0 ? x - tq * a.group : 0);
    const bool live = x < rows;
    bool takes = true;  // SIDE 1: this key takes part
    if (SIDE == 1) takes = x < count && (!a.mask.valid || a.mask.valid[b * a.mask.valid_img + x] != 0);
    {  // the held rows: X1 by the first group of warps, X2 by the second, half of the channels a warp
      const View& src = SIDE == 0 ? (u == 0 ? a.q : a.dout) : u == 0 ? a.k : a.v;
      const long long at = SIDE == 0 ? tq * src.row + (long long)h * DH : x * src.row + (long long)kvh * DH;
      const uint4* from = reinterpret_cast<const uint4*>(static_cast<const __half*>(src.p) + b * src.img + at) +
                          hf * (DH / 16);
      uint4 v[DH / 16];
#pragma unroll
      for (int c = 0; c < DH / 16; ++c) v[c] = live ? from[c] : make_uint4(0, 0, 0, 0);
      if (u < C::XT) {
        const uint32_t to = tmem + lanes + C::X0 + u * (DH / 2) + hf * (DH / 4);
        const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
        __syncwarp();
        if constexpr (DH == 128) tmem_st32(to, w);
        else if constexpr (DH == 64) tmem_st16(to, w);
        else tmem_st8(to, w);
        tmem_st_wait();
        tc_fence_before();
      } else {
#pragma unroll
        for (int c = 0; c < DH / 16; ++c)
          *reinterpret_cast<uint4*>(smem + (u - C::XT) * C::XS + T::chunk(128, quad * 32 + lane, hf * (DH / 16) + c)) = v[c];
        fence_proxy_async_smem();
      }
      warp_arrive(x_full);
    }
    // P is held as 2^lift P, dS as F dS with F = f 2^lift
    constexpr float lift = BF16 ? 0.f : 14.f;
    float f = 1.f;
    const long long qrow = ((long long)b * a.H + h) * a.Tq + tq;  // SIDE 0: the held row
    if constexpr (!BF16) {
      const unsigned* top = a.top + (b * a.Hkv + kvh) * 2;
      const float bound = (SIDE == 1 ? __uint_as_float(top[0]) : live ? a.norm[qrow] : 0.f) * __uint_as_float(top[1]);
      if (bound > 0.f && bound < INFINITY) f = exp2f(-(float)(ilogbf(bound) + 1));
    }
    const float sl = a.scale_log2;
    float l2 = INFINITY, df = 0.f;
    if (SIDE == 0 && live) {
      l2 = a.lse2[qrow] - lift;
      df = a.delta[qrow] * f;
    }
    float* mine = stat + warp * 128;  // [2][L, D][32]
    float next[2];
    auto fetch = [&](int i) {  // SIDE 1: L and D of step i's queries, one a lane
      const int step = first + i, t = step % q_tiles * kStep + cg * 32 + lane;
      const long long at = ((long long)b * a.H + kvh * a.group + step / q_tiles) * a.Tq + t;
      next[0] = t < a.Tq ? a.lse2[at] - lift : INFINITY;
      next[1] = t < a.Tq ? a.delta[at] * f : 0.f;
    };
    if (SIDE == 1 && n > 0) fetch(0);
    const uint8_t* vrow = SIDE == 0 ? a.mask.row(b) : nullptr;
    uint32_t byte = vrow ? ask_keys(vrow, first * kStep + cg * 32, count) : 0u;
    // D comes from the rounded out.  Its error is the sum of a row's dS, which is 0 otherwise, and shows beside
    // dS's own rounding where few keys share a row (2 keys: gradients 2.5 times as far off as their rounding,
    // 30 keys: 1.6, from 100 on 1.45).  So where one step has all keys of an item, D is put right there, for
    // the other side too, which runs later.
    const bool one = SIDE == 0 && all == 1 && n == 1;
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(kSoft * 32) : "memory"); };  // all softmax warps, once
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      uint32_t w = takes ? 0xFFFFFFFFu : 0u;
      const float* st = mine + (i & 1) * 64;
      if constexpr (SIDE == 0) {
        const int j0 = (first + i) * kStep + cg * 32;
        if (vrow) {
          w = told_keys(byte);
          byte = ask_keys(vrow, j0 + kStep, count);
        } else {
          w = bits_below(j0, count);
        }
      } else {
        float* put = mine + (i & 1) * 64;
        put[lane] = next[0];
        put[32 + lane] = next[1];
        __syncwarp();
        if (i + 1 < n) fetch(i + 1);
      }
      ok = warp_wait(s_full, i & 1, abort_flag);
      if (!ok) {
        if (one) meet();
        break;
      }
      tc_fence_after();
      uint32_t s[32];
      tmem_ld32(s_at, s);
      tmem_ld_wait();
      if (SIDE == 0) {
        tc_fence_before();
        warp_arrive(s_free);
      }
      float p[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) p[j] = exp2_hw(fmaf(__uint_as_float(s[j]), sl, -(SIDE == 0 ? l2 : st[j])));
      if (w != 0xFFFFFFFFu) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!(w >> j & 1u)) p[j] = 0.f;
      }
      if (SIDE == 1) {
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) pk[j] = pack16<BF16>(p[2 * j], p[2 * j + 1]);
        __syncwarp();
        tmem_st16(p_at, pk);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(p_full);
      }
      ok = warp_wait(r_full, i & 1, abort_flag);
      if (!ok) {
        if (one) meet();
        break;
      }
      tc_fence_after();
      tmem_ld32(r_at, s);
      tmem_ld_wait();
      if (SIDE == 0) {
        tc_fence_before();
        warp_arrive(r_free);
      }
      if (one) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (w >> j & 1u) sum = fmaf(p[j], fmaf(__uint_as_float(s[j]), f, -df), sum);
        // the second stage is not used by a single step
        float* told = reinterpret_cast<float*>(ring + C::SB) + quad * 32 + lane;
        told[cg * 128] = sum;
        meet();
        df += ((told[0] + told[128]) + (told[256] + told[384])) * exp2f(-lift);
        if (live && cg == 0) a.delta[qrow] = df / f;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) p[j] *= fmaf(__uint_as_float(s[j]), f, -(SIDE == 0 ? df : st[32 + j]));
      if (w != 0xFFFFFFFFu) {  // R may be NaN there
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!(w >> j & 1u)) p[j] = 0.f;
      }
      uint32_t pk[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) pk[j] = pack16<BF16>(p[2 * j], p[2 * j + 1]);
      if (SIDE == 0 && i > 0) {  // the last step's accumulation has read its dS
        ok = warp_wait(d_free, (i - 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
      }
      __syncwarp();
      tmem_st16(d_at, pk);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(d_full);
    }
    if (ok && n > 0) ok = warp_wait(acc_full, 0, abort_flag);
    if (!ok) {
      if (lane == 0) give_up(SB_ERR_TIMEOUT_ACC);
    } else {
      tc_fence_after();
      // a warp writes half of dq's channels (SIDE 0, four of a row's warps idle) or of dk's or dv's
      constexpr int cols = DH / 2;
      const int c0 = (SIDE == 0 ? u : hf) * cols;
      const bool writes = live && (SIDE == 1 || hf == 0);
      const uint32_t from = tmem + lanes + C::ACC + (SIDE == 0 ? 0 : u * DH) + c0;
      const float by = SIDE == 1 && u == 1 ? exp2f(-lift) : a.scale * exp2f(-lift) / f;
      const OutView& o = SIDE == 0 ? a.dq : u == 0 ? a.dk : a.dv;
      const long long prow = SIDE == 0 ? qrow
                                       : (((long long)u * a.B + b) * a.Hkv + kvh) * a.Tk + x;
#pragma unroll
      for (int c = 0; c < cols; c += 16) {
        uint32_t v[16];
        __syncwarp();
        if (n > 0) {
          tmem_ld16(from + c, v);
          tmem_ld_wait();
        }
        if (!writes) continue;
        float y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = n > 0 && takes ? __uint_as_float(v[j]) * by : 0.f;
        if (a.splits > 1) {
          float4* dst = reinterpret_cast<float4*>(a.part + (split * a.part_rows + prow) * DH + c0 + c);
#pragma unroll
          for (int j = 0; j < 4; ++j) dst[j] = make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
        } else {
          const long long at = SIDE == 0 ? b * o.img + tq * o.row + (long long)h * DH
                                         : b * o.img + (long long)x * o.row + (long long)kvh * DH;
          uint4* dst = reinterpret_cast<uint4*>(static_cast<__half*>(o.p) + at + c0 + c);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            dst[j] = make_uint4(pack16<BF16>(y[8 * j], y[8 * j + 1]), pack16<BF16>(y[8 * j + 2], y[8 * j + 3]),
                                pack16<BF16>(y[8 * j + 4], y[8 * j + 5]), pack16<BF16>(y[8 * j + 6], y[8 * j + 7]));
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kSoft) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the splits' partial rows in order; a thread holds eight channels of a row.
template <int DH, int SIDE>
__global__ void __launch_bounds__(256) attend_back_join_kernel(const __grid_constant__ BackArgs a) {
  constexpr int per = DH / 8;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long rr = i / per;
  const int c = (int)(i % per) * 8;
  if (rr >= a.part_rows) return;
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    float v[8];
    unpack8(load_raw8(a.part, SB_F32, (s * a.part_rows + rr) * DH + c), SB_F32, v);
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] += v[u];
  }
  const int len = SIDE == 0 ? a.Tq : a.Tk, heads = SIDE == 0 ? a.H : a.Hkv;
  const long long t = rr % len, h = rr / len % heads, ub = rr / len / heads, b = ub % a.B;
  const OutView& o = SIDE == 0 ? a.dq : ub < a.B ? a.dk : a.dv;
  store8(o.p, a.dt, b * o.img + t * o.row + h * DH + c, f);
}

struct SidePlan {
  int x_tiles, steps, splits;
  long long units, part_rows;
};
struct BackPlan {
  SidePlan side[2];
  long long rows, bytes;  // B * H * Tq; the workspace
};

// Steps are split where the CTAs' last wave would leave more SMs idle than the splits cost (about
// kStart steps a CTA to start and end, as much again for the join).
SidePlan side_plan(long long items, long long x_rows, long long steps, long long part_rows, int sms) {
  constexpr int kStart = 4, kMost = 64;
  SidePlan p;
  p.x_tiles = (int)((x_rows + 127) / 128);
  p.steps = (int)steps;
  p.units = items * p.x_tiles;
  p.part_rows = part_rows;
  p.splits = 1;
  double best = 1e300;
  for (int s = 1; s <= std::min<long long>(kMost, steps); ++s) {
    const long long each = (steps + s - 1) / s;
    if ((steps + each - 1) / each != s) continue;
    const double cost = (double)((p.units * s + sms - 1) / sms) * (each + kStart) + (s > 1 ? kStart : 0);
    if (cost < 0.95 * best) {
      best = cost;
      p.splits = s;
    }
  }
  return p;
}
// lse2, delta, norm and top
long long stats_bytes(long long rows, long long items) { return (rows * 12 + items * 8 + 15) / 16 * 16; }
BackPlan back_plan(int B, int H, int Hkv, int dh, int Tq, int Tk, int sms) {
  BackPlan p;
  const long long group = H / Hkv, items = (long long)B * Hkv;
  p.rows = (long long)B * H * Tq;
  p.side[0] = side_plan(items, group * Tq, (Tk + kStep - 1) / kStep, p.rows, sms);
  p.side[1] = side_plan(items, Tk, group * ((Tq + kStep - 1) / kStep), 2 * items * Tk, sms);
  long long part = 0;  // the sides run one after the other and share it
  for (const SidePlan& s : p.side)
    if (s.splits > 1) part = std::max(part, (long long)s.splits * s.part_rows * dh * 4);
  p.bytes = stats_bytes(p.rows, items) + part;
  return p;
}

template <int DH, bool BF16, int SIDE>
cudaError_t launch_side(BackArgs a, const SidePlan& p, const CUtensorMap& y1, const CUtensorMap& y2, cudaStream_t st) {
  using C = Back<DH, SIDE>;
  static bool ready[64];
  cudaError_t e = xattn_smem(reinterpret_cast<const void*>(&attend_back_kernel<DH, BF16, SIDE>), C::SMEM, ready);
  if (e != cudaSuccess) return e;
  a.x_tiles = p.x_tiles;
  a.splits = p.splits;
  a.steps = p.steps;
  a.part_rows = p.part_rows;
  attend_back_kernel<DH, BF16, SIDE><<<(unsigned)(p.units * p.splits), C::THREADS, C::SMEM, st>>>(a, y1, y2);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  const long long threads = p.part_rows * (DH / 8);
  attend_back_join_kernel<DH, SIDE><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <int DH, bool BF16>
int launch_back(BackArgs& a, const BackPlan& p, int* counts, cudaStream_t st) {
  // all maps before the first launch: a call that is refused has done nothing
  CUtensorMap km, vm, qm, dm;
  if (!xattn_tensor_map(&km, a.k, a.dt, a.B, a.Tk, a.Hkv, DH, kStep) ||
      !xattn_tensor_map(&vm, a.v, a.dt, a.B, a.Tk, a.Hkv, DH, kStep) ||
      !xattn_tensor_map(&qm, a.q, a.dt, a.B, a.Tq, a.H, DH, kStep) ||
      !xattn_tensor_map(&dm, a.dout, a.dt, a.B, a.Tq, a.H, DH, kStep))
    return record_error(SB_EINVAL, "sb_cross_attention_backward: tensor map of k, v, q or dout");
  if (a.mask.valid) {
    const cudaError_t e = count_keys(a.mask, a.B, counts, st);
    if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
    a.mask.lens = counts;
  }
  constexpr int per = 256 / (DH / 8);
  const int most = std::max(a.Tq, BF16 ? 0 : a.Tk);
  // sixteen CTAs an SM over all heads (8 x 8 heads of 300 queries and up to 2040 keys: 5 us less than with
  // 64 a head)
  const int heads = a.B * a.H + (BF16 ? 0 : a.B * a.Hkv), each = std::max(1, 16 * xattn_sms() / heads);
  const dim3 grid((unsigned)heads, (unsigned)std::min({(most + per - 1) / per, each, 64}));
  if (!BF16 && cudaMemsetAsync(a.top, 0, (size_t)a.B * a.Hkv * 8, st) != cudaSuccess)
    return record_error(SB_ECUDA, "sb_cross_attention_backward: memset");
  attend_back_rows_kernel<DH><<<grid, 256, 0, st>>>(a);
  a.y1_item = a.k.img != 0;
  a.y2_item = a.v.img != 0;
  cudaError_t e = launch_side<DH, BF16, 0>(a, p.side[0], km, vm, st);
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  a.y1_item = a.q.img != 0;
  a.y2_item = a.dout.img != 0;
  e = launch_side<DH, BF16, 1>(a, p.side[1], qm, dm, st);
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}

// Zero rows of a gradient whose other side is empty.
__global__ void zero_rows_kernel(OutView o, int T, int width, long long n) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const long long c = i % width, row = i / width;
  static_cast<uint16_t*>(o.p)[row / T * o.img + row % T * o.row + c] = 0;
}
void zero_rows(const OutView& o, int B, int T, int width, cudaStream_t st) {
  const long long n = (long long)B * T * width;
  zero_rows_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(o, T, width, n);
}

}  // namespace

int xattn_back_error(int clear, int* flags) {
  const int zero = 0;
  if (cudaMemcpyFromSymbol(flags, g_xattn_bwd_error, sizeof(int)) != cudaSuccess) return -1;
  return clear && cudaMemcpyToSymbol(g_xattn_bwd_error, &zero, sizeof(int)) != cudaSuccess ? -1 : 0;
}

long long xattn_back_work(int B, int H, int Hkv, int dh, int Tq, int Tk, int sms) {
  return back_plan(B, H, Hkv, dh, Tq, Tk, sms).bytes;
}

}  // namespace sb

using namespace sb;

extern "C" int sb_cross_attention_backward(const void* dout, long long do_row, long long do_img, const void* q,
                                           long long q_row, long long q_img, const void* k, long long k_row,
                                           long long k_img, const void* v, long long v_row, long long v_img, const void* out,
                                           long long o_row, long long o_img, const float* lse, int dtype, int B, int H,
                                           int Hkv, int dh, int Tq, int Tk, float scale, const int* lens, const void* valid,
                                           long long valid_img, void* dq, long long dq_row, long long dq_img, void* dk,
                                           long long dk_row, long long dk_img, void* dv, long long dv_row, long long dv_img,
                                           void* work, long long work_bytes, void* stream) {
  if (!xattn_sizes_ok(dtype, B, H, Hkv, dh, Tq, Tk) || !(scale > 0.f) || !std::isfinite(scale))
    return record_error(SB_EINVAL,
                        "sb_cross_attention_backward: sizes (dh 32, 64 or 128, H a multiple of Hkv), dtype or scale");
  if (B == 0 || (Tq == 0 && Tk == 0)) return SB_OK;
  if ((Tq > 0 && (!lse || !xattn_map_ok(dout, do_row, do_img, Tq) || !xattn_map_ok(q, q_row, q_img, Tq) ||
                  !xattn_view_ok(out, o_row, o_img) || !xattn_view_ok(dq, dq_row, dq_img))) ||
      (Tk > 0 && (!xattn_map_ok(k, k_row, k_img, Tk) || !xattn_map_ok(v, v_row, v_img, Tk) ||
                  !xattn_view_ok(dk, dk_row, dk_img) || !xattn_view_ok(dv, dv_row, dv_img))))
    return record_error(SB_EINVAL, "sb_cross_attention_backward: rows (16-byte aligned, strides multiples of 8, dout's, q's, "
                                   "k's and v's not 0) or lse");
  BackArgs a{};
  a.q = {q, q_row, q_img}; a.k = {k, k_row, k_img}; a.v = {v, v_row, v_img};
  a.out = {out, o_row, o_img}; a.dout = {dout, do_row, do_img};
  a.dq = {dq, dq_row, dq_img}; a.dk = {dk, dk_row, dk_img}; a.dv = {dv, dv_row, dv_img};
  a.lse = lse;
  a.mask = {lens, static_cast<const uint8_t*>(valid), valid_img, Tk};
  a.dt = dtype; a.B = B; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.Tq = Tq; a.Tk = Tk;
  a.masked = lens || valid;
  a.scale = scale;
  a.scale_log2 = scale * 1.4426950408889634f;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (Tq == 0 || Tk == 0) {
    if (Tq > 0) {
      zero_rows(a.dq, B, Tq, H * dh, st);
    } else {
      zero_rows(a.dk, B, Tk, Hkv * dh, st);
      zero_rows(a.dv, B, Tk, Hkv * dh, st);
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
  }
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_cross_attention_backward: device");
  const BackPlan p = back_plan(B, H, Hkv, dh, Tq, Tk, sms);
  const long long counts = counts_bytes(valid != nullptr, B);
  if (!work || work_bytes < counts + p.bytes || (reinterpret_cast<uintptr_t>(work) & 15) != 0)
    return record_error(SB_EINVAL,
                        "sb_cross_attention_backward: workspace (sb_cross_attention_work bytes, 16-byte aligned)");
  for (const SidePlan& s : p.side)
    if (s.units * s.splits > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_cross_attention_backward: too many items");
  if ((long long)B * (H + Hkv) > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_cross_attention_backward: too many items");
  int* counts_at = static_cast<int*>(work);
  a.lse2 = reinterpret_cast<float*>(static_cast<char*>(work) + counts);
  a.delta = a.lse2 + p.rows;
  a.norm = a.delta + p.rows;
  a.top = reinterpret_cast<unsigned*>(a.norm + p.rows);
  a.part = reinterpret_cast<float*>(static_cast<char*>(work) + counts + stats_bytes(p.rows, (long long)B * Hkv));
  if (dtype == SB_BF16)
    return dh == 32 ? launch_back<32, true>(a, p, counts_at, st) : dh == 64 ? launch_back<64, true>(a, p, counts_at, st)
                                                                 : launch_back<128, true>(a, p, counts_at, st);
  return dh == 32 ? launch_back<32, false>(a, p, counts_at, st) : dh == 64 ? launch_back<64, false>(a, p, counts_at, st)
                                                                : launch_back<128, false>(a, p, counts_at, st);
}
