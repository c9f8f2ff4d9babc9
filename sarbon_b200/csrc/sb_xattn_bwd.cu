// sb_xattn_bwd.cu -- gradients of the attention of queries to an encoder's states.
//
// With P = exp(scale q k^T - L), dP = dout v^T, D_i = dout_i.out_i and dS = P (dP - D):
//   dq = scale dS k,   dk = scale dS^T q,   dv = P^T dout   (dk, dv summed over the query heads that
// share a key head).  Two kernels of one form, each owning its results, so that no sum needs an
// atomic and the same inputs give the same bits:
//   SIDE 0 (dq)      a CTA holds 128 query rows (q, dout) and streams 64-row tiles of k, v
//   SIDE 1 (dk, dv)  a CTA holds 128 keys (k, v) and streams 64-row tiles of q, dout, head by head
// Per step, with X the held and Y the streamed operands:
//   S = X1 Y1^T, R = X2 Y2^T (128 x 64, operands in shared memory)
//   thread = held row: takes S and R into registers at once (their buffer is then free for the next
//   step's), P and dS from them, rounded to the operands' type, back to TMEM
//   acc1 += dS Y1 (dq, dk),  SIDE 1: acc2 += P Y2 (dv)     (A in TMEM, B the rows as they lie)
// Steps alternate between two groups of eight softmax warps (two threads a held row, 32 streamed rows
// each) with their own P and dS; S and R have two buffers, or one where two accumulators of 128 columns
// leave no room.  One warp issues S and R while another issues the accumulations: the products of one step run
// while the other's softmax does, and an issuer's waits on barriers do not idle the tensor pipe.  S and R are computed on both sides (7 products instead of 5): against
// one kernel that adds up dq in global memory this costs 2 of 7 products and saves the atomics.
//
// fp16 gradients: P and dS may be far below fp16's smallest normal number (long memories, small
// losses).  P is held as 2^14 P, and dS as F dS with F the power of two that the bound |dS| <= 2 P
// max|dout_i| max|v_j| (norms over the item and key head, from a first kernel that also forms D)
// keeps below 2^15; both factors leave at the end.  bf16 has fp32's range and needs neither.
//
// A range of steps may be split over CTAs (few rows against many): these write fp32 partial
// results, which a last kernel adds in order.
#include <algorithm>
#include <cmath>

#include "sb_xattn.cuh"

namespace sb {
namespace {

__device__ int g_xattn_bwd_error;

constexpr int kStep = 64;  // streamed rows a step
constexpr int kSoft = 16;  // softmax warps: buffer (w / 8), half of a step's rows (w / 4 % 2), TMEM lanes (w % 4)

struct BackArgs {
  View q, k, v, out, dout;
  OutView dq, dk, dv;
  const float* lse;
  KeyMask mask;
  int dt, B, H, Hkv, group, Tq, Tk;
  int x_tiles, splits, steps;  // held tiles of an (item, key head); splits of its steps
  int y1_item, y2_item, x1_item, x2_item;  // 0: one memory for every item
  int masked;
  float scale, scale_log2;
  float* lse2;   // [B][H][Tq] L log2 e, +inf for a row without keys
  float* delta;  // [B][H][Tq]
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
  static constexpr int XB = Tile<DH>::bytes(128);    // a held operand
  static constexpr int YB = Tile<DH>::bytes(kStep);  // a streamed one
  static constexpr int SB = 2 * YB;                  // a stage
  static constexpr int STAT = SIDE ? kSoft * 2 * 64 * 4 : 0;  // L and D of a step's queries, a warp each
  static constexpr int ROOM = 224 * 1024 - 2 * XB - STAT;
  static constexpr int STAGES = ROOM / SB < 8 ? ROOM / SB : 8;
  static constexpr int SMEM = 1024 + 2 * XB + STAGES * SB + STAT + 512;
  static constexpr int THREADS = (kSoft + 4) * 32;
  // TMEM columns: S and R (64 + 64, NB times), P and dS of each group (32 + 32), acc1, acc2
  static constexpr int NB = SIDE == 1 && DH == 128 ? 1 : 2;
  static constexpr int PD = NB * 128, ACC = PD + 128;
  static_assert(STAGES >= 4 && ACC + (1 + SIDE) * DH <= 512, "ring and TMEM");
};

template <int DH, bool BF16, int SIDE>
__global__ void __launch_bounds__(Back<DH, SIDE>::THREADS, 1)
    attend_back_kernel(const __grid_constant__ BackArgs a, const __grid_constant__ CUtensorMap x1map,
                       const __grid_constant__ CUtensorMap x2map, const __grid_constant__ CUtensorMap y1map,
                       const __grid_constant__ CUtensorMap y2map) {
  using C = Back<DH, SIDE>;
  using T = Tile<DH>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * C::XB;
  float* stat = reinterpret_cast<float*>(ring + ST * C::SB);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + ST * C::SB + C::STAT);
  uint64_t* empty = full + ST;
  uint64_t* clean = empty + ST;  // [ST]
  uint64_t* x_full = clean + ST;
  uint64_t* s_full = x_full + 1;  // [2] each, a group: S and R computed
  uint64_t* s_free = s_full + 2;  // S and R taken into registers
  uint64_t* p_full = s_free + 2;  // P and dS written
  uint64_t* p_free = p_full + 2;  // and read by the accumulations
  uint64_t* acc_full = p_free + 2;
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
  const int each = (a.steps + a.splits - 1) / a.splits, first = split * each;
  // steps with anything to do: key tiles that begin before the item's end; all, if the held keys do
  const int all = SIDE == 0 ? min(a.steps, (count + kStep - 1) / kStep) : tile * 128 < count ? a.steps : 0;
  const int n = max(0, min(first + each, all) - first);

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&clean[i], 1);
    }
    mbar_init(x_full, SIDE == 0 ? kSoft : 1);
    for (int u = 0; u < 2; ++u) {
      mbar_init(&s_full[u], 1);
      mbar_init(&s_free[u], kSoft / 2);
      mbar_init(&p_full[u], kSoft / 2);
      mbar_init(&p_free[u], 1);
      mbar_init(&dbar[u], 1);
    }
    mbar_init(acc_full, 1);
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
      if constexpr (SIDE == 1) {
        mbar_arrive_expect_tx(x_full, 2 * C::XB);
        for (int x = 0; x < T::BOXES; ++x) {
          tma_load_4d(smem + x * T::box_bytes(128), &x1map, x_full, x * T::COLS, tile * 128, kvh, b * a.x1_item);
          tma_load_4d(smem + C::XB + x * T::box_bytes(128), &x2map, x_full, x * T::COLS, tile * 128, kvh, b * a.x2_item);
        }
      }
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
      if (*abort_flag) {
        for (int i = max(0, p - ST); i < p; ++i) bounded_wait(&full[i % ST], (i / ST) & 1);
        if (SIDE == 1) bounded_wait(x_full, 0);
      }
    }
  } else if (warp == kSoft) {
    if (lane == 0 && n > 0) {  // issuer of S and R
      const uint32_t xb = smem_u32(smem), rb = smem_u32(ring);
      constexpr uint32_t id_s = idesc_16bit(BF16, 128, kStep, false);
      bool ok = mbar_wait(x_full, 0, abort_flag);
      for (int i = 0; i < n && ok; ++i) {
        const int st = i % ST, u = i & 1;
        ok = mbar_wait(&full[st], (i / ST) & 1, abort_flag) &&
             (SIDE == 1 || !a.masked || mbar_wait(&clean[st], (i / ST) & 1, abort_flag)) &&
             (i < C::NB || mbar_wait(&s_free[(i - C::NB) & 1], ((i - C::NB) >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t y = rb + st * C::SB, s = tmem + (C::NB == 2 ? u * 128 : 0);
#pragma unroll
        for (int ks = 0; ks < T::KSTEPS; ++ks)
          mma_f16_ss(s, T::k_major(xb, 128, ks), T::k_major(y, kStep, ks), id_s, ks > 0);
#pragma unroll
        for (int ks = 0; ks < T::KSTEPS; ++ks)
          mma_f16_ss(s + 64, T::k_major(xb + C::XB, 128, ks), T::k_major(y + C::YB, kStep, ks), id_s, ks > 0);
        mma_commit(&s_full[u]);
      }
      if (!ok) {
        give_up(SB_ERR_TIMEOUT_FULL);
        mma_commit(&dbar[0]);
        bounded_wait(&dbar[0], 0);
      }
    }
  } else if (warp == kSoft + 1) {
    if (lane == 0 && n > 0) {  // issuer of the accumulations
      const uint32_t rb = smem_u32(ring);
      constexpr uint32_t id_a = idesc_16bit(BF16, 128, DH, true);
      bool ok = true;
      for (int i = 0; i < n; ++i) {
        const int st = i % ST, u = i & 1;
        ok = mbar_wait(&p_full[u], (i >> 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t y = rb + st * C::SB, p = tmem + C::PD + u * 64;
        if constexpr (SIDE == 1) {
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
            mma_f16_ts(tmem + C::ACC + DH, p + k * 8, T::mn_major(y + C::YB, kStep, k), id_a, i > 0 || k > 0);
        }
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          mma_f16_ts(tmem + C::ACC, p + 32 + k * 8, T::mn_major(y, kStep, k), id_a, i > 0 || k > 0);
        mma_commit(&p_free[u]);
        mma_commit(&empty[st]);
      }
      if (ok) {
        mma_commit(acc_full);
      } else {
        give_up(SB_ERR_TIMEOUT_FULL);
        mma_commit(&dbar[1]);
        bounded_wait(&dbar[1], 0);
      }
    }
  } else if (warp == kSoft + 3) {
    if (SIDE == 0 && a.masked) {  // cleaner: k's rows of keys that take no part
      for (int i = 0; i < n; ++i) {
        const int st = i % ST, j0 = (first + i) * kStep;
        if (!warp_wait(&full[st], (i / ST) & 1, abort_flag)) {
          if (lane == 0) give_up(SB_ERR_TIMEOUT_FULL);
          break;
        }
        bool touched = false;
#pragma unroll 1
        for (int x = 0; x < kStep / 32; ++x) {
          const uint32_t w = a.mask.word(b, j0 + 32 * x, count);
          if (w == 0xFFFFFFFFu) continue;
          touched = true;
          if (!(w >> lane & 1u))
            for (int c = 0; c < DH / 8; ++c)
              *reinterpret_cast<uint4*>(ring + st * C::SB + T::chunk(kStep, 32 * x + lane, c)) = make_uint4(0, 0, 0, 0);
        }
        if (touched) fence_proxy_async_smem();
        warp_arrive(&clean[st]);
      }
    }
  } else {
    const int u = warp >> 3, hf = warp >> 2 & 1, quad = warp & 3;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_at = tmem + lanes + (C::NB == 2 ? u * 128 : 0) + hf * 32, r_at = s_at + 64;
    const uint32_t p_at = tmem + lanes + C::PD + u * 64 + hf * 16, d_at = p_at + 32;
    const int x = tile * 128 + quad * 32 + lane;  // held row: query row of the group, or key
    const int rows = SIDE == 0 ? a.group * a.Tq : a.Tk;
    const int tq = SIDE == 0 ? x / a.group : 0, h = kvh * a.group + (SIDE == 0 ? x - tq * a.group : 0);
    const bool live = x < rows;
    bool takes = true;  // SIDE 1: this key takes part
    if (SIDE == 1) takes = x < count && (!a.mask.valid || a.mask.valid[b * a.mask.valid_img + x] != 0);
    if constexpr (SIDE == 0) {
      const View& src = u == 0 ? a.q : a.dout;
      const uint4* from = reinterpret_cast<const uint4*>(static_cast<const __half*>(src.p) + b * src.img + tq * src.row +
                                                         (long long)h * DH);
#pragma unroll
      for (int c = hf * (DH / 16); c < (hf + 1) * (DH / 16); ++c)
        *reinterpret_cast<uint4*>(smem + u * C::XB + T::chunk(128, quad * 32 + lane, c)) =
            live ? from[c] : make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      warp_arrive(x_full);
    }
    // P is held as 2^lift P, dS as F dS with F = f 2^lift
    constexpr float lift = BF16 ? 0.f : 14.f;
    float f = 1.f;
    if constexpr (!BF16) {
      const unsigned* top = a.top + (b * a.Hkv + kvh) * 2;
      const float bound = __uint_as_float(top[0]) * __uint_as_float(top[1]);
      if (bound > 0.f && bound < INFINITY) f = exp2f(-(float)(ilogbf(bound) + 1));
    }
    const float sl = a.scale_log2;
    float l2 = INFINITY, df = 0.f;
    if (SIDE == 0 && live) {
      const long long r = ((long long)b * a.H + h) * a.Tq + tq;
      l2 = a.lse2[r] - lift;
      df = a.delta[r] * f;
    }
    float* mine = stat + warp * 128;  // [2][L, D][32]
    float next[2];
    auto fetch = [&](int i) {  // SIDE 1: L and D of step i's queries, one a lane
      const int step = first + i, t = step % q_tiles * kStep + hf * 32 + lane;
      const long long at = ((long long)b * a.H + kvh * a.group + step / q_tiles) * a.Tq + t;
      next[0] = t < a.Tq ? a.lse2[at] - lift : INFINITY;
      next[1] = t < a.Tq ? a.delta[at] * f : 0.f;
    };
    if (SIDE == 1 && u < n) fetch(u);
    uint32_t byte = SIDE == 0 ? a.mask.ask(b, (first + u) * kStep + hf * 32, count) : 0u;
    bool ok = true;
    for (int i = u; i < n; i += 2) {
      uint32_t w = 0xFFFFFFFFu;
      const float* st = mine + ((i >> 1) & 1) * 64;
      if constexpr (SIDE == 0) {
        const int j0 = (first + i) * kStep + hf * 32;
        w = a.mask.told(byte, j0, count);
        byte = a.mask.ask(b, j0 + 2 * kStep, count);
      } else {
        float* put = mine + ((i >> 1) & 1) * 64;
        put[lane] = next[0];
        put[32 + lane] = next[1];
        __syncwarp();
        if (i + 2 < n) fetch(i + 2);
      }
      ok = warp_wait(&s_full[u], (i >> 1) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[2][16], r[2][16];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        tmem_ld16(s_at + 16 * q, s[q]);
        tmem_ld16(r_at + 16 * q, r[q]);
      }
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(&s_free[u]);
      uint32_t pp[2][8], pd[2][8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          float p[2], d[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int at = 16 * q + j + y;
            const float lj = SIDE == 0 ? l2 : st[at], dj = SIDE == 0 ? df : st[32 + at];
            p[y] = exp2_hw(fmaf(__uint_as_float(s[q][j + y]), sl, -lj));
            d[y] = p[y] * fmaf(__uint_as_float(r[q][j + y]), f, -dj);
          }
          if (SIDE == 0 ? w != 0xFFFFFFFFu : !takes) {
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (SIDE == 1 || !(w >> (16 * q + j + y) & 1u)) p[y] = d[y] = 0.f;
          }
          if (SIDE == 1) pp[q][j / 2] = pack16<BF16>(p[0], p[1]);
          pd[q][j / 2] = pack16<BF16>(d[0], d[1]);
        }
        if (q == 0 && i > 1) {  // the accumulations of the group's last step have read P and dS
          ok = warp_wait(&p_free[u], ((i >> 1) - 1) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
        }
        __syncwarp();
        if (SIDE == 1) tmem_st8(p_at + 8 * q, pp[q]);
        tmem_st8(d_at + 8 * q, pd[q]);
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&p_full[u]);
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
      const long long prow = SIDE == 0 ? ((long long)b * a.H + h) * a.Tq + tq
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
  constexpr int kStart = 8, kMost = 64;
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
BackPlan back_plan(int B, int H, int Hkv, int dh, int Tq, int Tk, int sms) {
  BackPlan p;
  const long long group = H / Hkv, items = (long long)B * Hkv;
  p.rows = (long long)B * H * Tq;
  p.side[0] = side_plan(items, group * Tq, (Tk + kStep - 1) / kStep, p.rows, sms);
  p.side[1] = side_plan(items, Tk, group * ((Tq + kStep - 1) / kStep), 2 * items * Tk, sms);
  long long part = 0;  // the sides run one after the other and share it
  for (const SidePlan& s : p.side)
    if (s.splits > 1) part = std::max(part, (long long)s.splits * s.part_rows * dh * 4);
  p.bytes = (p.rows * 8 + items * 8 + 15) / 16 * 16 + part;
  return p;
}

template <int DH, bool BF16, int SIDE>
cudaError_t launch_side(BackArgs a, const SidePlan& p, const CUtensorMap (&m)[4], cudaStream_t st) {
  using C = Back<DH, SIDE>;
  static bool ready[64];
  cudaError_t e = xattn_smem(reinterpret_cast<const void*>(&attend_back_kernel<DH, BF16, SIDE>), C::SMEM, ready);
  if (e != cudaSuccess) return e;
  a.x_tiles = p.x_tiles;
  a.splits = p.splits;
  a.steps = p.steps;
  a.part_rows = p.part_rows;
  attend_back_kernel<DH, BF16, SIDE><<<(unsigned)(p.units * p.splits), C::THREADS, C::SMEM, st>>>(a, m[0], m[1], m[2], m[3]);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  const long long threads = p.part_rows * (DH / 8);
  attend_back_join_kernel<DH, SIDE><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <int DH, bool BF16>
int launch_back(BackArgs& a, const BackPlan& p, cudaStream_t st) {
  constexpr int per = 256 / (DH / 8);
  const int most = std::max(a.Tq, BF16 ? 0 : a.Tk);
  const dim3 grid((unsigned)(a.B * a.H + (BF16 ? 0 : a.B * a.Hkv)), (unsigned)std::min((most + per - 1) / per, 64));
  if (!BF16 && cudaMemsetAsync(a.top, 0, (size_t)a.B * a.Hkv * 8, st) != cudaSuccess)
    return record_error(SB_ECUDA, "sb_cross_attention_backward: memset");
  attend_back_rows_kernel<DH><<<grid, 256, 0, st>>>(a);
  CUtensorMap m[4];
  // SIDE 0 streams k, v (its held rows are gathered by threads); SIDE 1 holds k, v and streams q, dout
  if (!xattn_tensor_map(&m[2], a.k, a.dt, a.B, a.Tk, a.Hkv, DH, kStep) ||
      !xattn_tensor_map(&m[3], a.v, a.dt, a.B, a.Tk, a.Hkv, DH, kStep))
    return record_error(SB_EINVAL, "sb_cross_attention_backward: tensor map of k or v");
  m[0] = m[2];
  m[1] = m[3];
  a.y1_item = a.k.img != 0;
  a.y2_item = a.v.img != 0;
  cudaError_t e = launch_side<DH, BF16, 0>(a, p.side[0], m, st);
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  if (!xattn_tensor_map(&m[0], a.k, a.dt, a.B, a.Tk, a.Hkv, DH, 128) ||
      !xattn_tensor_map(&m[1], a.v, a.dt, a.B, a.Tk, a.Hkv, DH, 128) ||
      !xattn_tensor_map(&m[2], a.q, a.dt, a.B, a.Tq, a.H, DH, kStep) ||
      !xattn_tensor_map(&m[3], a.dout, a.dt, a.B, a.Tq, a.H, DH, kStep))
    return record_error(SB_EINVAL, "sb_cross_attention_backward: tensor map of q, dout, k or v");
  a.x1_item = a.y1_item;
  a.x2_item = a.y2_item;
  a.y1_item = a.q.img != 0;
  a.y2_item = a.dout.img != 0;
  e = launch_side<DH, BF16, 1>(a, p.side[1], m, st);
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
  if ((Tq > 0 && (!lse || !xattn_view_ok(dout, do_row, do_img) || !xattn_view_ok(q, q_row, q_img) ||
                  !xattn_view_ok(out, o_row, o_img) || !xattn_view_ok(dq, dq_row, dq_img))) ||
      (Tk > 0 && (!xattn_view_ok(k, k_row, k_img) || !xattn_view_ok(v, v_row, v_img) ||
                  !xattn_view_ok(dk, dk_row, dk_img) || !xattn_view_ok(dv, dv_row, dv_img))))
    return record_error(SB_EINVAL, "sb_cross_attention_backward: rows (16-byte aligned, strides multiples of 8) or lse");
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
  if (!work || work_bytes < p.bytes || (reinterpret_cast<uintptr_t>(work) & 15) != 0)
    return record_error(SB_EINVAL,
                        "sb_cross_attention_backward: workspace (sb_cross_attention_work bytes, 16-byte aligned)");
  for (const SidePlan& s : p.side)
    if (s.units * s.splits > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_cross_attention_backward: too many items");
  if ((long long)B * (H + Hkv) > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_cross_attention_backward: too many items");
  a.lse2 = static_cast<float*>(work);
  a.delta = a.lse2 + p.rows;
  a.top = reinterpret_cast<unsigned*>(a.delta + p.rows);
  a.part = reinterpret_cast<float*>(static_cast<char*>(work) + (p.rows * 8 + (long long)B * Hkv * 8 + 15) / 16 * 16);
  if (dtype == SB_BF16)
    return dh == 32 ? launch_back<32, true>(a, p, st) : dh == 64 ? launch_back<64, true>(a, p, st)
                                                                 : launch_back<128, true>(a, p, st);
  return dh == 32 ? launch_back<32, false>(a, p, st) : dh == 64 ? launch_back<64, false>(a, p, st)
                                                                : launch_back<128, false>(a, p, st);
}
