// sb_xattn.cu -- attention of queries to an encoder's states of another length.
//
// Per head and query i over the keys j that take part: s_ij = scale q_i.k_j, L_i = log sum_j exp s_ij,
// out_i = sum_j exp(s_ij - L_i) v_j; a query without keys gets zeros and L_i = -inf.
//
// The query heads that share a key head are one list of rows (token-major, head-minor): a tile is
// 128 of them, whatever the group's size.  A CTA has two streams of 128-row tiles, each with an
// accumulator, eight softmax warps and a warp that issues its products, over a range of 128-key tiles:
//   two tiles of rows left   a tile a stream, both over every key tile
//   one                      both streams on it, over alternate key tiles, joined at the end (the
//                            last tile of an odd number)
//   loader warp   K and V tiles by TMA into a ring each, in the order in which they are used.  A stage's
//                 barrier is only waited for by roles that see each of its uses (a parity says
//                 nothing about a use before the last)
//   issuer warps  S_t = Q_t K^T (operands in shared memory); O_t += P_t V with P_t in TMEM as the A
//                 operand.  With a tile a stream there is an issuer a stream: a wait on a barrier costs
//                 one a few hundred clocks, in which the other keeps the tensor pipe fed.  Alternate
//                 tiles have one issuer
//   8 warps a stream  two threads a query row, 64 keys each (one thread a row left two warps a
//                 scheduler, too few to cover the arithmetic's latency): scores from TMEM into registers
//                 at once, so that the next tile's are computed meanwhile (one buffer for both
//                 streams with 128 channels, which the accumulators leave no room beside; one each
//                 below); P = 2^(s scale log2 e - m), rounded to the operands' type, back to TMEM.  The
//                 reference point m moves, and O is rescaled, only when a row's maximum grew by more
//                 than 2^8 since the last time (P stays below 2^8, in fp16 times 2^7 below 2^15; m and the
//                 factor cancel in O / l), so the two threads need each other's maximum only then:
//                 otherwise one barrier with the OR of "grew" is all that a tile costs them
//   cleaner warp  with masks: zeroes V's rows of keys that take no part (0 x NaN is NaN), before
//                 the product reads them
// What bounds it is the chain of a tile: P stored, its product, the wait for it, the next P.  A wait costs
// 100 to 400 clocks whatever its form (polls, suspended or with sleeps, measured alike), a tile of a stream
// 2400 with the arithmetic and all but one of its products left out, 4400 with them; two streams overlap,
// and with P beside the scores TMEM has no room for a third or for two P.  2 x 16 heads of 128 channels (4 key heads), 4096
// queries, 8160 keys: 545 us, 1005 TFLOP/s, where the products alone would take 336 and the exponentials
// (16 a clock and SM) 238.  16 x 8 heads of 32 channels, 300 queries, 28,900 of 42,840 keys: 842 us, of them
// 215 for the 44 rows behind the second tile, which load two of an SM's four schedulers.  A polynomial for
// part of the exponentials was slower: the issue slots are as scarce.
// The key range is split over CTAs where the rows alone leave SMs idle: these write fp32 partial rows
// with their L, and a second kernel joins them.  Up to 16 rows (single tokens) have a kernel of their
// own, which reads K and V once at memory speed.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "sb_xattn.cuh"

namespace sb {

namespace {

__device__ int g_xattn_error;

constexpr int KT = 128;      // keys a tile
constexpr int kSoft = 16;     // softmax warps: stream (w / 8), half of a tile's keys (w / 4 % 2), TMEM lanes (w % 4)
constexpr int kThreads = (kSoft + 4) * 32;

template <int DH>
struct Fwd {
  static constexpr int QB = Tile<DH>::bytes(128);  // a tile of queries
  static constexpr int SB = Tile<DH>::bytes(KT);   // a stage: one K or V tile
  // K and V stages with two tiles of queries and with one
  static constexpr int ROOM2 = (224 * 1024 - 2 * QB) / SB, ROOM1 = (224 * 1024 - QB) / SB;
  static constexpr int K2 = ROOM2 < 12 ? (ROOM2 + 1) / 2 : 6, V2 = ROOM2 < 12 ? ROOM2 / 2 : 6;
  static constexpr int K1 = ROOM1 < 12 ? (ROOM1 + 1) / 2 : 6, V1 = ROOM1 < 12 ? ROOM1 / 2 : 6;
  static constexpr int TILES = 224 * 1024, SMEM = 1024 + TILES + 512 + 1024;
  // TMEM columns: scores (shared by the streams or one each), P, accumulators
  static constexpr bool SHARED = DH == 128;
  static constexpr int SSTEP = SHARED ? 0 : KT, P0 = SHARED ? KT : 2 * KT, O0 = P0 + KT;
  static_assert(V2 >= 2 && K2 <= 6 && K1 <= 6 && O0 + 2 * DH <= 512, "rings and TMEM");
};

// A place in a ring of `stages`: stage and the parity of its use.
struct Place {
  int stages, st = 0;
  uint32_t parity = 0;
  SB_DEV explicit Place(int n) : stages(n) {}
  SB_DEV void next() {
    if (++st == stages) {
      st = 0;
      parity ^= 1u;
    }
  }
};

// P of 32 columns: 2^(s sl + ms), their sum added to `sum`, rounded into 16 words
template <bool BF16>
SB_DEV void probabilities(const uint32_t* s, uint64_t sl, uint64_t ms, uint64_t (&sum)[2], uint32_t (&pk)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    float a, b;
    split2(fma2(pair2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), sl, ms), a, b);
    a = exp2_hw(a);
    b = exp2_hw(b);
    sum[j & 1] = add2(sum[j & 1], pair2(a, b));
    pk[j] = pack16<BF16>(a, b);
  }
}

template <int DH, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ FwdArgs a, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  using C = Fwd<DH>;
  using T = Tile<DH>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::TILES);  // [6] each
  uint64_t* v_full = k_full + 6;
  uint64_t* k_empty = v_full + 6;
  uint64_t* v_empty = k_empty + 6;
  uint64_t* clean = v_empty + 6;  // V tile ready for its product (with masks)
  uint64_t* q_full = clean + 6;   // [2] each, a stream
  uint64_t* s_full = q_full + 2;  // scores computed
  uint64_t* s_free = s_full + 2;  // scores taken into registers
  uint64_t* p_full = s_free + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* dbar = o_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(dbar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  // what threads of a row tell each other: [stream][row] a maximum or a sum; at the end [row] both of the
  // second stream's
  float* told = reinterpret_cast<float*>(smem + C::TILES + 512);
  float2* ml = reinterpret_cast<float2*>(told);
  const int warp = warp_id(), lane = lane_id();

  int idx = blockIdx.x;
  const int pair = idx % a.pairs;
  idx /= a.pairs;
  const int split = idx % a.splits;
  idx /= a.splits;
  const int kvh = idx % a.Hkv, b = idx / a.Hkv;
  const bool two = pair * 256 + 128 < a.rows;  // two tiles of rows
  const int count = a.mask.count(b);
  // the item's own key tiles, split evenly
  const int all_tiles = (count + KT - 1) / KT, each = (all_tiles + a.splits - 1) / a.splits;
  const int first = min(split * each, all_tiles), n = min(first + each, all_tiles) - first;
  const int KS = two ? C::K2 : C::K1, VS = two ? C::V2 : C::V1;
  uint8_t* k_ring = smem + (two ? 2 : 1) * C::QB;
  uint8_t* v_ring = k_ring + KS * C::SB;
  // tiles are used, and loaded, in the order K0 .. K(ahead - 1) V0 K(ahead) V1 ...
  const int ahead = two || C::SHARED ? 2 : 3;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 6; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&k_empty[i], two ? 2 : 1);  // the streams that read a tile
      mbar_init(&v_empty[i], two ? 2 : 1);
      mbar_init(&clean[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], kSoft / 2);
      mbar_init(&s_full[t], 1);
      mbar_init(&s_free[t], kSoft / 2);
      mbar_init(&p_full[t], kSoft / 2);
      mbar_init(&o_full[t], 1);
      mbar_init(&dbar[t], 1);
    }
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
    atomicOr(&g_xattn_error, code);
  };

  // softmax threads: their row, reference point (of the raw scores) and sum over their half of the keys
  const int t = warp >> 3, hf = warp >> 2 & 1, quad = warp & 3;
  const int lr = quad * 32 + lane;
  const int tile = pair * 2 + (two ? t : 0);
  const int r = tile * 128 + lr;
  const bool some = warp < kSoft && tile * 128 + quad * 32 < a.rows;  // the warp has rows
  const int tq = r / a.group, h = kvh * a.group + (r - tq * a.group);
  const int mine = two ? n : (n - t + 1) / 2;  // key tiles of the stream
  const uint32_t lanes = (uint32_t)(quad * 32) << 16;
  const uint32_t s_at = tmem + lanes + t * C::SSTEP + hf * 64, p_at = tmem + lanes + C::P0 + t * (KT / 2) + hf * 32;
  const uint32_t o_at = tmem + lanes + C::O0 + t * DH + hf * (DH / 2);
  const int bar_id = 1 + t * 4 + quad;  // of the two warps of these rows
  float* tell = told + t * 128 + lr;
  const float sl = a.scale_log2;
  constexpr float lift = kLift<BF16>;
  float m = -INFINITY, l = 0.f;
  bool ok = true;

  if (warp == kSoft + 2) {
    if (lane == 0) {  // loader
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
      int ki = 0, vi = 0;
      Place kp(KS), vp(VS);
      while (vi < n) {
        const bool v = ki == min(n, vi + ahead);
        const int i = v ? vi : ki;
        Place& at = v ? vp : kp;
        // (the first use of a stage passes: its barrier's phase before the first counts as done)
        if (!mbar_wait((v ? v_empty : k_empty) + at.st, at.parity ^ 1u, abort_flag)) {
          give_up(SB_ERR_TIMEOUT_EMPTY);
          break;
        }
        uint64_t* bar = (v ? v_full : k_full) + at.st;
        mbar_arrive_expect_tx(bar, C::SB);
        const CUtensorMap* map = v ? &vmap : &kmap;
        uint8_t* dst = (v ? v_ring : k_ring) + at.st * C::SB;
        const int item = b * (v ? a.v_item : a.k_item);
        for (int x = 0; x < T::BOXES; ++x)
          tma_load_4d(dst + x * T::box_bytes(KT), map, bar, x * T::COLS, (first + i) * KT, kvh, item);
        if (v) ++vi;
        else ++ki;
        at.next();
      }
      if (*abort_flag) {
        for (int i = max(0, ki - KS); i < ki; ++i) bounded_wait(&k_full[i % KS], (i / KS) & 1);
        for (int i = max(0, vi - VS); i < vi; ++i) bounded_wait(&v_full[i % VS], (i / VS) & 1);
      }
    }
  } else if (warp == kSoft || warp == kSoft + 1) {
    const int u0 = warp - kSoft;
    if (lane == 0 && n > 0 && (two || u0 == 0)) {  // issuer of stream u0, or of both
      const uint32_t kb = smem_u32(k_ring), vb = smem_u32(v_ring), qb = smem_u32(smem) + u0 * C::QB;
      constexpr uint32_t id_s = idesc_16bit(BF16, 128, KT, false), id_o = idesc_16bit(BF16, 128, DH, true);
      Place kp(KS), vp(VS);
      auto k_ready = [&]() { return mbar_wait(&k_full[kp.st], kp.parity, abort_flag); };
      auto v_ready = [&]() {
        return mbar_wait(&v_full[vp.st], vp.parity, abort_flag) &&
               (!a.masked || mbar_wait(&clean[vp.st], vp.parity, abort_flag));
      };
      auto scores = [&](int u) {  // of stream u with the next K tile
        const uint32_t k = kb + kp.st * C::SB;
#pragma unroll
        for (int ks = 0; ks < T::KSTEPS; ++ks)
          mma_f16_ss(tmem + u * C::SSTEP, T::k_major(qb, 128, ks), T::k_major(k, KT, ks), id_s, ks > 0);
        mma_commit(&s_full[u]);
        mma_commit(&k_empty[kp.st]);
        kp.next();
      };
      auto values = [&](int u, int c) {  // P of stream u's tile c with the next V tile
        const uint32_t v = vb + vp.st * C::SB;
#pragma unroll
        for (int k = 0; k < KT / 16; ++k)
          mma_f16_ts(tmem + C::O0 + u * DH, tmem + C::P0 + u * (KT / 2) + k * 8, T::mn_major(v, KT, k), id_o,
                     c > 0 || k > 0);
        mma_commit(&o_full[u]);
        mma_commit(&v_empty[vp.st]);
        vp.next();
      };
      auto p_ready = [&](int u, int c) { return mbar_wait(&p_full[u], c & 1, abort_flag); };
      // stream u has taken the scores of its tile c into registers
      auto taken = [&](int u, int c) { return mbar_wait(&s_free[u], c & 1, abort_flag); };
      ok = mbar_wait(&q_full[u0], 0, abort_flag);
      if (two) {
        // the scores' buffer is free when this stream has taken its last tile's, a shared one when the other
        // stream has taken the tile before
        ok = ok && k_ready() && (!C::SHARED || u0 == 0 || taken(0, 0));
        if (ok) {
          tc_fence_after();
          scores(u0);
        }
        for (int c = 0; c < n && ok; ++c) {
          if (c + 1 < n) {
            ok = k_ready() && (C::SHARED ? taken(1 - u0, c + u0) : taken(u0, c));
            if (!ok) break;
            tc_fence_after();
            scores(u0);
          }
          ok = v_ready() && p_ready(u0, c);
          if (!ok) break;
          tc_fence_after();
          values(u0, c);
        }
      } else {
        // tile i belongs to stream i % 2; before its values come the scores of the next tile, or of the one
        // after where the streams have a buffer each
        constexpr int more = C::SHARED ? 1 : 2;
        for (int i = 0; i < min(n, more) && ok; ++i) {
          ok = k_ready();
          if (!ok) break;
          tc_fence_after();
          scores(i);
        }
        for (int i = 0; i < n && ok; ++i) {
          const int u = i & 1, c = i >> 1;
          if (i + more < n) {
            ok = k_ready() && taken(u, c);
            if (!ok) break;
            tc_fence_after();
            scores((i + more) & 1);
          }
          ok = v_ready() && p_ready(u, c);
          if (!ok) break;
          tc_fence_after();
          values(u, c);
        }
      }
      if (!ok) {
        give_up(SB_ERR_TIMEOUT_FULL);
        mma_commit(&dbar[u0]);
        bounded_wait(&dbar[u0], 0);
      }
    }
  } else if (warp == kSoft + 3) {
    if (a.masked) {  // cleaner, its mask bytes two tiles ahead
      const uint8_t* vrow = a.mask.row(b);
      uint32_t next[2][KT / 32];
      if (vrow) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int x = 0; x < KT / 32; ++x) next[y][x] = ask_keys(vrow, (first + y) * KT + 32 * x, count);
      }
      Place vp(VS);
#pragma unroll 2
      for (int i = 0; i < n; ++i, vp.next()) {
        const int j0 = (first + i) * KT;
        uint8_t* v = v_ring + vp.st * C::SB;
        uint32_t w[KT / 32];
#pragma unroll
        for (int x = 0; x < KT / 32; ++x) {
          if (vrow) {
            w[x] = told_keys(next[i & 1][x]);
            next[i & 1][x] = ask_keys(vrow, j0 + 2 * KT + 32 * x, count);
          } else {
            w[x] = bits_below(j0 + 32 * x, count);
          }
        }
        if (!warp_wait(&v_full[vp.st], vp.parity, abort_flag)) {
          if (lane == 0) give_up(SB_ERR_TIMEOUT_FULL);
          break;
        }
        bool touched = false;
#pragma unroll
        for (int x = 0; x < KT / 32; ++x) {
          if (w[x] == 0xFFFFFFFFu) continue;
          touched = true;
          if (!(w[x] >> lane & 1u))
            for (int c = 0; c < DH / 8; ++c)
              *reinterpret_cast<uint4*>(v + T::chunk(KT, 32 * x + lane, c)) = make_uint4(0, 0, 0, 0);
        }
        if (touched) fence_proxy_async_smem();
        warp_arrive(&clean[vp.st]);
      }
    }
  } else {
    if (two || t == 0) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __half*>(a.q.p) + b * a.q.img + tq * a.q.row +
                                                        (long long)h * DH);
      uint8_t* dst = smem + t * C::QB;
#pragma unroll
      for (int c = hf * (DH / 16); c < (hf + 1) * (DH / 16); ++c)
        *reinterpret_cast<uint4*>(dst + T::chunk(128, lr, c)) = r < a.rows ? src[c] : make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      warp_arrive(&q_full[t]);
    }
    const uint64_t sl2 = pair2(sl, sl);
    const int jstep = two ? KT : 2 * KT;
    int j0 = (first + (two ? 0 : t)) * KT + hf * 64;
    const uint8_t* vrow = a.mask.row(b);
    uint32_t b0 = 0, b1 = 0;
    if (vrow) {
      b0 = ask_keys(vrow, j0, count);
      b1 = ask_keys(vrow, j0 + 32, count);
    }
    // A warp whose wait failed goes on to the next barrier with its partner, which then leaves too.
    for (int i = 0; i < mine; ++i, j0 += jstep) {
      uint32_t w0 = 0xFFFFFFFFu, w1 = 0xFFFFFFFFu;
      if (vrow) {
        w0 = told_keys(b0);
        w1 = told_keys(b1);
        b0 = ask_keys(vrow, j0 + jstep, count);
        b1 = ask_keys(vrow, j0 + jstep + 32, count);
      } else if (j0 + 64 > count) {
        w0 = bits_below(j0, count);
        w1 = bits_below(j0 + 32, count);
      }
      ok = ok && warp_wait(&s_full[t], i & 1, abort_flag);
      if (!some) {  // P of lanes without rows is never looked at
        if (!ok) break;
        warp_arrive(&s_free[t]);
        ok = i == 0 || warp_wait(&o_full[t], (i - 1) & 1, abort_flag);
        if (!ok) break;
        warp_arrive(&p_full[t]);
        continue;
      }
      tc_fence_after();
      uint32_t s[64];
      tmem_ld32(s_at, s);
      tmem_ld32(s_at + 32, s + 32);
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(&s_free[t]);
      if ((w0 & w1) != 0xFFFFFFFFu) {
        // 16 keys at a time: masks of images and lengths leave most groups whole
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t g = (x < 2 ? w0 : w1) >> (16 * (x & 1)) & 0xFFFFu;
          if (g == 0xFFFFu) continue;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (!(g >> j & 1u)) s[16 * x + j] = 0xFF800000u;  // -inf
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 64; j += 2)
        mx[j / 2 & 3] = max3(mx[j / 2 & 3], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
      float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
      // a new reference point: with the first tile, and where the maximum grew (or is NaN).  What is compared
      // is the exponent that the row's largest P would get, so no score's rounding carries one past 2^15.
      float ms = fmaf(-m, sl, lift);
      const bool grew = pair_or(bar_id, !ok || i == 0 || !(fmaf(top, sl, ms) <= lift + 8.f));
      float c = 1.f;
      if (grew) {
        if (hf == 1) *tell = top;
        if (pair_or(bar_id, !ok)) {
          ok = false;
          break;
        }
        if (hf == 0) *tell = top = max3(top, *tell, m);
        pair_or(bar_id, false);
        if (hf == 1) top = *tell;
        c = m == top ? 1.f : exp2_hw((m - top) * sl);
        m = top;
        ms = fmaf(-m, sl, lift);
        l *= c;
      }
      // masked scores give 0; a row whose reference is still -inf has had no keys
      if (m == -INFINITY) ms = 0.f;
      const uint64_t ms2 = pair2(ms, ms);
      uint64_t sum[2] = {0, 0};
      // All exponentials before the last product is waited for, or the second half after the first has
      // gone to TMEM: 2 x 16 heads, 4096 queries, 8160 keys: 440 against 473 us with 64 channels, 493 against
      // 503 with 128; with 32, whose products are short, 447 against 433 in bf16 (420 against 438 in fp16).
      constexpr bool kAll = DH >= 64;
      uint32_t pk[16], pl[16];
      probabilities<BF16>(s, sl2, ms2, sum, pk);
      if constexpr (kAll) probabilities<BF16>(s + 32, sl2, ms2, sum, pl);
      // the last tile's product has read its P and added to O
      if (i > 0) {
        ok = warp_wait(&o_full[t], (i - 1) & 1, abort_flag);
        tc_fence_after();
      }
      if (grew && i > 0) {
#pragma unroll
        for (int y = 0; y < DH / 32; ++y) {
          uint32_t o[16];
          tmem_ld16(o_at + 16 * y, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * c);
          tmem_st16(o_at + 16 * y, o);
        }
      }
      tmem_st16(p_at, pk);
      if constexpr (!kAll) probabilities<BF16>(s + 32, sl2, ms2, sum, pl);
      tmem_st16(p_at + 16, pl);
      float s0, s1;
      split2(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tmem_st_wait();
      tc_fence_before();
      if (ok) warp_arrive(&p_full[t]);
    }
    if (ok && mine > 0) ok = warp_wait(&o_full[t], (mine - 1) & 1, abort_flag);
    if (!ok && lane == 0) give_up(SB_ERR_TIMEOUT_ACC);
    tc_fence_after();
    if (some) {  // the row's sum
      pair_or(bar_id, false);
      if (hf == 1) *tell = l;
      pair_or(bar_id, false);
      if (hf == 0) *tell = l += *tell;
      pair_or(bar_id, false);
      if (hf == 1) l = *tell;
      if (m == -INFINITY) l = 0.f;
    }
  }

  float m1 = -INFINITY, l1 = 0.f;  // of the other stream on the same rows
  float4* other = reinterpret_cast<float4*>(smem);  // [128][DH / 4] its O, in the queries' place
  constexpr int per = DH / 4;
  const bool join = !two && n > 1;
  if (join) {
    __syncthreads();  // both streams' products are done: the queries are no longer read
    if (t == 1 && some && !*abort_flag) {
      if (hf == 0) ml[lr] = make_float2(m, l);
#pragma unroll
      for (int x = 0; x < DH / 32; ++x) {
        uint32_t o[16];
        tmem_ld16(o_at + 16 * x, o);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 4; ++c)
          other[lr * per + ((hf * (DH / 8) + 4 * x + c) ^ (lr & 7))] =
              make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]), __uint_as_float(o[4 * c + 2]),
                          __uint_as_float(o[4 * c + 3]));
      }
    }
    __syncthreads();
  }
  if (some && (two || t == 0) && !*abort_flag) {
    float w0 = 1.f, w1 = 0.f;
    if (join) {
      m1 = ml[lr].x;
      l1 = ml[lr].y;
      const float top = max3(m, m1, m1);
      w0 = m == top ? 1.f : exp2_hw((m - top) * sl);
      w1 = m1 == top ? 1.f : exp2_hw((m1 - top) * sl);
      m = top;
      l = l * w0 + l1 * w1;
    }
    const float lse = l == 0.f ? -INFINITY : fmaf(m, sl, -lift) * 0.69314718055994531f + logf(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    w0 *= inv;
    w1 *= inv;
    const long long rr = ((long long)b * a.H + h) * a.Tq + tq;
    const bool live = r < a.rows;
#pragma unroll
    for (int x = 0; x < DH / 32; ++x) {
      const int col = hf * (DH / 2) + 16 * x;
      uint32_t o[16];
      float f[16];
      __syncwarp();
      if (mine > 0) {
        tmem_ld16(o_at + 16 * x, o);
        tmem_ld_wait();
      }
      if (!live || (a.splits > 1 && n == 0)) continue;
#pragma unroll
      for (int j = 0; j < 16; ++j) f[j] = mine > 0 ? __uint_as_float(o[j]) * w0 : 0.f;
      if (join) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 e = other[lr * per + ((hf * (DH / 8) + 4 * x + c) ^ (lr & 7))];
          f[4 * c] = fmaf(e.x, w1, f[4 * c]);
          f[4 * c + 1] = fmaf(e.y, w1, f[4 * c + 1]);
          f[4 * c + 2] = fmaf(e.z, w1, f[4 * c + 2]);
          f[4 * c + 3] = fmaf(e.w, w1, f[4 * c + 3]);
        }
      }
      if (a.splits > 1) {
        float4* dst = reinterpret_cast<float4*>(a.part_o + (split * a.all_rows + rr) * DH + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
      } else {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<__half*>(a.o.p) + b * a.o.img + tq * a.o.row +
                                              (long long)h * DH + col);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          dst[j] = make_uint4(pack16<BF16>(f[8 * j], f[8 * j + 1]), pack16<BF16>(f[8 * j + 2], f[8 * j + 3]),
                              pack16<BF16>(f[8 * j + 4], f[8 * j + 5]), pack16<BF16>(f[8 * j + 6], f[8 * j + 7]));
      }
    }
    if (live && hf == 0) {
      if (a.splits > 1) a.part_l[split * a.all_rows + rr] = n > 0 ? lse : -INFINITY;
      else if (a.lse) a.lse[rr] = n > 0 ? lse : -INFINITY;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoft) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the splits' rows: out = sum_s e^(L_s - L) O_s, L = log sum_s e^L_s.  A thread holds eight
// channels of a row; a split without keys (L_s = -inf) has not written its O_s.
template <int DH, bool BF16>
__global__ void __launch_bounds__(256) attend_join_kernel(const __grid_constant__ FwdArgs a) {
  constexpr int per = DH / 8;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long rr = i / per;
  const int c = (int)(i % per) * 8;
  if (rr >= a.all_rows) return;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_l[s * a.all_rows + rr]);
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float ls = a.part_l[s * a.all_rows + rr];
    if (ls == -INFINITY) continue;
    const float w = expf(ls - top);
    const float4* src = reinterpret_cast<const float4*>(a.part_o + (s * a.all_rows + rr) * DH + c);
    const float4 x = src[0], y = src[1];
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    sum += w;
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] = fmaf(w, v[u], f[u]);
  }
  if (sum != 0.f) {
    const float inv = 1.f / sum;
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] *= inv;
  }
  const int t = (int)(rr % a.Tq), h = (int)(rr / a.Tq % a.H);
  const long long b = rr / a.Tq / a.H;
  store8(a.o.p, BF16 ? SB_BF16 : SB_F16, b * a.o.img + t * a.o.row + (long long)h * DH + c, f);
  if (a.lse && c == 0) a.lse[rr] = sum != 0.f ? top + logf(sum) : -INFINITY;
}

// One CTA an item, from the end on: images are padded behind, cameras are off.
__global__ void __launch_bounds__(1024) count_keys_kernel(KeyMask mask, int* counts) {
  constexpr int kEach = 8;
  const int b = blockIdx.x;
  __shared__ int last;
  if (threadIdx.x == 0) last = 0;
  __syncthreads();
  for (int end = mask.count(b); end > 0; end -= 1024 * kEach) {
    int mine = 0;
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int j = end - 1 - u * 1024 - (int)threadIdx.x;
      if (j >= 0 && mask.valid[b * mask.valid_img + j] != 0) mine = max(mine, j + 1);
    }
    if (mine > 0) atomicMax(&last, mine);
    if (__syncthreads_or(mine > 0)) break;
  }
  if (threadIdx.x == 0) counts[b] = last;
}

// No keys at all: zero rows and L = -inf.
__global__ void attend_none_kernel(OutView o, float* lse, int H, int Tq, int dh, long long n) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int c = (int)(i % ((long long)H * dh));
  const long long row = i / ((long long)H * dh), b = row / Tq, t = row % Tq;
  static_cast<uint16_t*>(o.p)[b * o.img + t * o.row + c] = 0;
  if (lse && c % dh == 0) lse[(b * H + c / dh) * Tq + t] = -INFINITY;
}

struct FwdPlan {
  int pairs, splits;
  long long units;
  bool few;
};

// CTAs take two tiles of rows each; a last single tile takes half of a CTA's time (its streams share
// the key tiles).  The key range is split where that shortens the longest CTA or evens out the SMs by
// more than it costs: a CTA spends about `kStart` key tiles on starting and ending, and joining costs
// about as much again.
FwdPlan fwd_plan(int B, int H, int Hkv, int Tq, int Tk, int sms) {
  constexpr int kStart = 4, kMost = 64;
  FwdPlan p;
  const long long tiles = ((long long)(H / Hkv) * Tq + 127) / 128;
  p.few = (long long)(H / Hkv) * Tq <= kFewRows;
  if (p.few) {
    p.pairs = 1;
    p.units = (long long)B * Hkv;
    p.splits = few_splits(p.units, Tk, sms);
    return p;
  }
  p.pairs = (int)((tiles + 1) / 2);
  const int key_tiles = (Tk + KT - 1) / KT;
  p.units = (long long)B * Hkv * p.pairs;
  const double twos = (double)B * Hkv * (tiles / 2), ones = (double)B * Hkv * (tiles % 2);
  p.splits = 1;
  double best = 1e300;
  for (int s = 1; s <= std::min(kMost, key_tiles); ++s) {
    const int each = (key_tiles + s - 1) / s;
    if ((key_tiles + each - 1) / each != s) continue;  // some split would be empty
    const double t2 = each + kStart, t1 = 0.5 * each + kStart, longest = tiles > 1 ? t2 : t1;
    // SMs take CTAs as they come: the even share, and about half of a CTA's time until the last ends
    const double share = s * (twos * t2 + ones * t1) / sms;
    const double cost = std::max(longest, share + 0.5 * longest) + (s > 1 ? kStart : 0);
    if (cost < 0.97 * best) {
      best = cost;
      p.splits = s;
    }
  }
  return p;
}

typedef CUresult (*PFN_encodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

PFN_encodeTiled encode_fn() {
  static PFN_encodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_encodeTiled>(p);
  });
  return fn;
}

template <int DH, bool BF16>
cudaError_t launch_fwd(const FwdArgs& a, const FwdPlan& p, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  using C = Fwd<DH>;
  static bool ready[64];
  cudaError_t e = xattn_smem(reinterpret_cast<const void*>(&attend_kernel<DH, BF16>), C::SMEM, ready);
  if (e != cudaSuccess) return e;
  attend_kernel<DH, BF16><<<(unsigned)(p.units * p.splits), kThreads, C::SMEM, st>>>(a, k, v);
  e = cudaGetLastError();
  if (e != cudaSuccess || a.splits == 1) return e;
  const long long threads = a.all_rows * (DH / 8);
  attend_join_kernel<DH, BF16><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a);
  return cudaGetLastError();
}
template <int DH>
cudaError_t launch_fwd(const FwdArgs& a, const FwdPlan& p, bool bf16, const CUtensorMap& k, const CUtensorMap& v,
                       cudaStream_t st) {
  return bf16 ? launch_fwd<DH, true>(a, p, k, v, st) : launch_fwd<DH, false>(a, p, k, v, st);
}

}  // namespace

bool xattn_sizes_ok(int dtype, int B, int H, int Hkv, int dh, int Tq, int Tk) {
  return (dtype == SB_F16 || dtype == SB_BF16) && (dh == 32 || dh == 64 || dh == 128) && B >= 0 && Tq >= 0 && Tk >= 0 &&
         H >= 1 && Hkv >= 1 && H % Hkv == 0 && (long long)H * dh <= 65536 &&
         (long long)(H / Hkv) * Tq < (1ll << 30) && Tk < (1 << 30);
}
bool xattn_view_ok(const void* p, long long row, long long img) {
  return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row >= 0 && img >= 0 && row % 8 == 0 && img % 8 == 0 &&
         row < (1ll << 38) && img < (1ll << 38);
}
bool xattn_map_ok(const void* p, long long row, long long img, int T) {
  return xattn_view_ok(p, row, img) && (row > 0 || T == 1);
}

bool xattn_tensor_map(CUtensorMap* map, const View& v, int dtype, int B, int T, int heads, int dh, int rows) {
  PFN_encodeTiled enc = encode_fn();
  if (!enc) return false;
  const bool one = v.img == 0;
  const cuuint64_t row = (cuuint64_t)v.row * 2, img = one ? 16 : (cuuint64_t)v.img * 2;
  cuuint64_t dims[4] = {(cuuint64_t)dh, (cuuint64_t)T, (cuuint64_t)heads, one ? 1u : (cuuint64_t)B};
  cuuint64_t strides[3] = {row == 0 ? 16 : row, (cuuint64_t)dh * 2, img};  // (a single row's is never used)
  cuuint32_t box[4] = {(cuuint32_t)std::min(dh, 64), (cuuint32_t)rows, 1u, 1u};
  cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  return enc(map, dtype == SB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void*>(v.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             dh < 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t count_keys(const KeyMask& mask, int B, int* counts, cudaStream_t st) {
  count_keys_kernel<<<(unsigned)B, 1024, 0, st>>>(mask, counts);
  return cudaGetLastError();
}

int xattn_error(int clear, int* flags) {
  const int zero = 0;
  if (cudaMemcpyFromSymbol(flags, g_xattn_error, sizeof(int)) != cudaSuccess) return -1;
  return clear && cudaMemcpyToSymbol(g_xattn_error, &zero, sizeof(int)) != cudaSuccess ? -1 : 0;
}

cudaError_t xattn_smem(const void* kernel, int bytes, bool (&ready)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || ready[dev & 63]) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  ready[dev & 63] = e == cudaSuccess;
  return e;
}

int xattn_sms() {
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

}  // namespace sb

using namespace sb;

extern "C" int sb_cross_attention_work(int backward, int masked, int B, int H, int Hkv, int dh, int Tq, int Tk, long long* bytes) {
  if (!bytes || !xattn_sizes_ok(SB_F16, B, H, Hkv, dh, Tq, Tk))
    return record_error(SB_EINVAL, "sb_cross_attention_work: arguments");
  *bytes = 0;
  if (B == 0 || Tq == 0 || Tk == 0) return SB_OK;
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_cross_attention_work: device");
  if (backward) {
    *bytes = counts_bytes(masked, B) + xattn_back_work(B, H, Hkv, dh, Tq, Tk, sms);
    return SB_OK;
  }
  const FwdPlan p = fwd_plan(B, H, Hkv, Tq, Tk, sms);
  *bytes = counts_bytes(masked, B) + (p.splits > 1 ? (long long)p.splits * B * H * Tq * (dh + 1) * 4 : 0);
  return SB_OK;
}

extern "C" int sb_cross_attention(const void* q, long long q_row, long long q_img, const void* k, long long k_row,
                                  long long k_img, const void* v, long long v_row, long long v_img, int dtype, int B, int H,
                                  int Hkv, int dh, int Tq, int Tk, float scale, const int* lens, const void* valid,
                                  long long valid_img, void* out, long long o_row, long long o_img, float* lse, void* work,
                                  long long work_bytes, void* stream) {
  if (!xattn_sizes_ok(dtype, B, H, Hkv, dh, Tq, Tk) || !(scale > 0.f) || !std::isfinite(scale))
    return record_error(SB_EINVAL, "sb_cross_attention: sizes (dh 32, 64 or 128, H a multiple of Hkv), dtype or scale");
  if (B == 0 || Tq == 0) return SB_OK;
  if (!xattn_view_ok(q, q_row, q_img) || !xattn_view_ok(out, o_row, o_img) ||
      (Tk > 0 && (!xattn_map_ok(k, k_row, k_img, Tk) || !xattn_map_ok(v, v_row, v_img, Tk))))
    return record_error(SB_EINVAL, "sb_cross_attention: rows (16-byte aligned, strides multiples of 8, k's and v's not 0)");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (Tk == 0) {
    const long long n = (long long)B * Tq * H * dh;
    attend_none_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>({out, o_row, o_img}, lse, H, Tq, dh, n);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
  }
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_cross_attention: device");
  const FwdPlan p = fwd_plan(B, H, Hkv, Tq, Tk, sms);
  const long long counts = counts_bytes(valid != nullptr, B);
  const long long need = counts + (p.splits > 1 ? (long long)p.splits * B * H * Tq * (dh + 1) * 4 : 0);
  if (need > 0 && (!work || work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15) != 0))
    return record_error(SB_EINVAL, "sb_cross_attention: workspace (sb_cross_attention_work bytes, 16-byte aligned)");
  if (p.units * p.splits > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_cross_attention: too many items");
  FwdArgs a{};
  a.q = {q, q_row, q_img};
  a.o = {out, o_row, o_img};
  a.lse = lse;
  a.mask = {lens, static_cast<const uint8_t*>(valid), valid_img, Tk};
  a.B = B; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.Tq = Tq; a.rows = a.group * Tq;
  a.pairs = p.pairs; a.splits = p.splits;
  a.k_item = k_img != 0; a.v_item = v_img != 0;
  a.masked = lens || valid;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.all_rows = (long long)B * H * Tq;
  // (before the first launch: a call that is refused has done nothing)
  CUtensorMap km, vm;
  const int box = p.few ? few_keys(dh) : KT;
  if (!xattn_tensor_map(&km, {k, k_row, k_img}, dtype, B, Tk, Hkv, dh, box) ||
      !xattn_tensor_map(&vm, {v, v_row, v_img}, dtype, B, Tk, Hkv, dh, box))
    return record_error(SB_EINVAL, "sb_cross_attention: tensor map of k or v");
  if (valid) {
    int* last = static_cast<int*>(work);
    const cudaError_t e = count_keys(a.mask, B, last, st);
    if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
    a.mask.lens = last;
  }
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(work) + counts);
  a.part_l = a.part_o + (long long)p.splits * a.all_rows * dh;
  const bool bf16 = dtype == SB_BF16;
  if (p.few) {
    cudaError_t e = few_launch(a, dh, bf16, km, vm, st);
    if (e == cudaSuccess && p.splits > 1) e = few_join(a, dh, bf16, st);
    return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
  }
  const cudaError_t e = dh == 32 ? launch_fwd<32>(a, p, bf16, km, vm, st)
                        : dh == 64 ? launch_fwd<64>(a, p, bf16, km, vm, st) : launch_fwd<128>(a, p, bf16, km, vm, st);
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}
