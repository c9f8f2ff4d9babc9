// sb_xattn.cu -- attention of queries to an encoder's states of another length.
//
// Per head and query i over the keys j that take part: s_ij = scale q_i.k_j, L_i = log sum_j exp s_ij,
// out_i = sum_j exp(s_ij - L_i) v_j; a query without keys gets zeros and L_i = -inf.
//
// The query heads that share a key head are one list of rows (token-major, head-minor): a tile is
// 128 of them, whatever the group's size.  A CTA takes NT tiles of one (item, key head) and a range
// of key tiles (KT keys), walked once with the softmax's running maximum and sum:
//   loader warp   K and V tiles by TMA into one ring, in the order K0 V0 K1 V1 ...
//   MMA warp      S_t = Q_t K^T (operands in shared memory), O_t += P_t V with P_t in TMEM as the A
//                 operand; the NT tiles alternate, so one tile's products run while the other's
//                 softmax does
//   4 warps/tile  thread = query row: reads its scores from TMEM, 2^(s scale log2 e - m), rounds P to
//                 the operands' type and writes it over the scores.  O is rescaled only when the
//                 maximum grew by more than 2^8 since the last time (P stays below 2^8, far from
//                 fp16's limit; the reference point cancels in O / l)
//   cleaner warp  with masks: zeroes V's rows of keys that take no part (0 x NaN is NaN), before
//                 the product reads them
// Few rows (a token a stream, NT = 1) leave SMs idle: the key range is split over CTAs, which write
// fp32 partial rows with their L, and a second kernel joins them.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "sb_xattn.cuh"

namespace sb {

namespace {

__device__ int g_xattn_error;

struct FwdArgs {
  View q;
  OutView o;
  float* lse;
  KeyMask mask;
  int B, H, Hkv, group, Tq, rows;  // rows = group * Tq of an (item, key head)
  int pairs, splits, key_tiles;    // CTAs a (item, key head) and split; key tiles in all
  int k_item, v_item;              // 0: one memory for every item
  int masked;                      // lens or valid given: the cleaner runs
  float scale_log2;
  float* part_o;  // [splits][B * H * Tq][DH]
  float* part_l;  // [splits][B * H * Tq]
  long long all_rows;
};

template <int DH, int NT>
struct Fwd {
  static constexpr int KT = NT == 2 ? 128 : 64;
  static constexpr int QB = Tile<DH>::bytes(128);  // one tile of queries
  static constexpr int SB = Tile<DH>::bytes(KT);   // a stage: one K or V tile
  static constexpr int ROOM = (NT == 2 ? 224 : 109) * 1024 - NT * QB;
  static constexpr int STAGES = ROOM / SB < 8 ? ROOM / SB : 8;
  static constexpr int SMEM = 1024 + NT * QB + STAGES * SB + 512;
  static constexpr int THREADS = (NT * 4 + 3) * 32;
  static constexpr uint32_t TMEM = NT == 2 ? 512 : 256;
  static constexpr int O0 = NT * KT;  // TMEM column of the first accumulator
  static_assert(STAGES >= 3 && NT * (KT + DH) <= (int)TMEM, "ring and TMEM");
};
constexpr int kClean = 8;  // more V tiles than the ring can hold at once

template <int DH, bool BF16, int NT>
__global__ void __launch_bounds__(Fwd<DH, NT>::THREADS, NT == 2 ? 1 : 2)
    attend_kernel(const __grid_constant__ FwdArgs a, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  using C = Fwd<DH, NT>;
  using T = Tile<DH>;
  constexpr int KT = C::KT, ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + NT * C::QB;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + ST * C::SB);
  uint64_t* empty = full + ST;
  uint64_t* clean = empty + ST;     // [kClean]
  uint64_t* q_full = clean + kClean;  // [NT] each
  uint64_t* s_full = q_full + NT;
  uint64_t* p_full = s_full + NT;
  uint64_t* o_full = p_full + NT;
  uint64_t* dbar = o_full + NT;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(dbar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = warp_id(), lane = lane_id();

  int idx = blockIdx.x;
  const int pair = idx % a.pairs;
  idx /= a.pairs;
  const int split = idx % a.splits;
  idx /= a.splits;
  const int kvh = idx % a.Hkv, b = idx / a.Hkv;
  const int tiles = (a.rows + 127) / 128;
  const int na = min(NT, tiles - pair * NT);  // tiles of this CTA
  const int count = a.mask.count(b);
  const int each = (a.key_tiles + a.splits - 1) / a.splits;
  const int first = split * each;
  const int n = max(0, min(min(first + each, a.key_tiles), (count + KT - 1) / KT) - first);

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kClean; ++i) mbar_init(&clean[i], 1);
    for (int t = 0; t < NT; ++t) {
      mbar_init(&q_full[t], 4);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(dbar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == NT * 4) {
    tmem_alloc(tmem_holder, C::TMEM);
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

  if (warp == NT * 4 + 1) {
    if (lane == 0) {  // loader
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
      int p = 0;
      for (; p < 2 * n; ++p) {
        const int st = p % ST;
        if (p >= ST && !mbar_wait(&empty[st], ((p / ST) - 1) & 1, abort_flag)) {
          give_up(SB_ERR_TIMEOUT_EMPTY);
          break;
        }
        mbar_arrive_expect_tx(&full[st], C::SB);
        const CUtensorMap* map = p & 1 ? &vmap : &kmap;
        const int item = b * (p & 1 ? a.v_item : a.k_item);
        for (int x = 0; x < T::BOXES; ++x)
          tma_load_4d(ring + st * C::SB + x * T::box_bytes(KT), map, &full[st], x * T::COLS, (first + p / 2) * KT, kvh,
                      item);
      }
      if (*abort_flag)
        for (int i = max(0, p - ST); i < p; ++i) bounded_wait(&full[i % ST], (i / ST) & 1);
    }
  } else if (warp == NT * 4) {
    if (lane == 0 && n > 0) {  // MMA
      const uint32_t qb = smem_u32(smem), rb = smem_u32(ring);
      constexpr uint32_t id_s = idesc_16bit(BF16, 128, KT, false), id_o = idesc_16bit(BF16, 128, DH, true);
      auto scores = [&](int t, int st) {
#pragma unroll
        for (int ks = 0; ks < T::KSTEPS; ++ks)
          mma_f16_ss(tmem + t * KT, T::k_major(qb + t * C::QB, 128, ks), T::k_major(rb + st * C::SB, KT, ks), id_s, ks > 0);
        mma_commit(&s_full[t]);
      };
      bool ok = true;
      for (int t = 0; t < na && ok; ++t) ok = mbar_wait(&q_full[t], 0, abort_flag);
      ok = ok && mbar_wait(&full[0], 0, abort_flag);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < na; ++t) scores(t, 0);
        mma_commit(&empty[0]);
      }
      for (int i = 0; i < n && ok; ++i) {
        const int vp = 2 * i + 1, vs = vp % ST, kp = 2 * i + 2, ks = kp % ST;
        for (int t = 0; t < na; ++t) {
          ok = mbar_wait(&p_full[t], i & 1, abort_flag);
          if (t == 0 && ok)
            ok = mbar_wait(&full[vs], (vp / ST) & 1, abort_flag) &&
                 (!a.masked || mbar_wait(&clean[i % kClean], (i / kClean) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < KT / 16; ++k)
            mma_f16_ts(tmem + C::O0 + t * DH, tmem + t * KT + k * 8, T::mn_major(rb + vs * C::SB, KT, k), id_o,
                       i > 0 || k > 0);
          mma_commit(&o_full[t]);
          if (t == na - 1) mma_commit(&empty[vs]);
          if (i + 1 < n) {
            if (t == 0) ok = mbar_wait(&full[ks], (kp / ST) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            scores(t, ks);
            if (t == na - 1) mma_commit(&empty[ks]);
          }
        }
      }
      if (!ok) {
        give_up(SB_ERR_TIMEOUT_FULL);
        mma_commit(dbar);
        bounded_wait(dbar, 0);
      }
    }
  } else if (warp == NT * 4 + 2) {
    if (a.masked) {  // cleaner
      for (int i = 0; i < n; ++i) {
        const int vp = 2 * i + 1, vs = vp % ST, j0 = (first + i) * KT;
        if (!warp_wait(&full[vs], (vp / ST) & 1, abort_flag)) {
          if (lane == 0) give_up(SB_ERR_TIMEOUT_FULL);
          break;
        }
        bool touched = false;
#pragma unroll 1
        for (int x = 0; x < KT / 32; ++x) {
          const uint32_t w = a.mask.word(b, j0 + 32 * x, count);
          if (w == 0xFFFFFFFFu) continue;
          touched = true;
          if (!(w >> lane & 1u))
            for (int c = 0; c < DH / 8; ++c)
              *reinterpret_cast<uint4*>(ring + vs * C::SB + T::chunk(KT, 32 * x + lane, c)) = make_uint4(0, 0, 0, 0);
        }
        if (touched) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&clean[i % kClean]);
      }
    }
  } else if (warp < na * 4) {
    const int t = warp >> 2, quad = warp & 3;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * KT, o_at = tmem + lanes + C::O0 + t * DH;
    const int r = (pair * NT + t) * 128 + quad * 32 + lane;  // row of the (item, key head)
    const bool some = (pair * NT + t) * 128 + quad * 32 < a.rows;  // the warp has rows
    const int tq = r / a.group, h = kvh * a.group + (r - tq * a.group);
    {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __half*>(a.q.p) + b * a.q.img + tq * a.q.row +
                                                        (long long)h * DH);
      uint8_t* dst = smem + t * C::QB;
#pragma unroll 8
      for (int c = 0; c < DH / 8; ++c)
        *reinterpret_cast<uint4*>(dst + T::chunk(128, quad * 32 + lane, c)) =
            r < a.rows ? src[c] : make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[t]);
    }
    const float sl = a.scale_log2, slack = 8.f / sl;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      uint32_t w[KT / 32];
      bool all = true;
#pragma unroll
      for (int x = 0; x < KT / 32; ++x) {
        w[x] = a.mask.word(b, (first + i) * KT + 32 * x, count);
        all = all && w[x] == 0xFFFFFFFFu;
      }
      ok = warp_wait(&s_full[t], i & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (some) {
        uint32_t s[KT];
#pragma unroll
        for (int x = 0; x < KT / 32; ++x) tmem_ld32(s_at + 32 * x, s + 32 * x);
        tmem_ld_wait();
        if (!all) {
#pragma unroll
          for (int j = 0; j < KT; ++j)
            if (!(w[j >> 5] >> (j & 31) & 1u)) s[j] = 0xFF800000u;  // -inf
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < KT; ++j) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(s[j]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (i == 0) {
          m = top;  // nothing accumulated yet
        } else if (__any_sync(0xFFFFFFFFu, top > m + slack)) {
          ok = warp_wait(&o_full[t], (i - 1) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const float mn = fmaxf(m, top);
          const float c = m == mn ? 1.f : exp2_hw((m - mn) * sl);
          m = mn;
          l *= c;
#pragma unroll
          for (int x = 0; x < DH / 16; ++x) {
            uint32_t o[16];
            tmem_ld16(o_at + 16 * x, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * c);
            tmem_st16(o_at + 16 * x, o);
          }
        }
        const float ms = m == -INFINITY ? 0.f : m * sl;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < KT / 32; ++x) {
          uint32_t pk[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float p0 = exp2_hw(fmaf(__uint_as_float(s[32 * x + 2 * j]), sl, -ms));
            const float p1 = exp2_hw(fmaf(__uint_as_float(s[32 * x + 2 * j + 1]), sl, -ms));
            sum[j & 3] += p0 + p1;
            pk[j] = pack16<BF16>(p0, p1);
          }
          tmem_st16(s_at + 16 * x, pk);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok && n > 0) ok = warp_wait(&o_full[t], (n - 1) & 1, abort_flag);
    if (!ok) {
      if (lane == 0) give_up(SB_ERR_TIMEOUT_ACC);
    } else if (some) {
      tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : NAN;
      const float lse = l == 0.f ? -INFINITY : m * sl * 0.69314718055994531f + logf(l);
      const long long rr = ((long long)b * a.H + h) * a.Tq + tq;
      const bool live = r < a.rows;
#pragma unroll
      for (int x = 0; x < DH / 32; ++x) {
        uint32_t o[32];
        __syncwarp();
        if (n > 0) {
          tmem_ld32(o_at + 32 * x, o);
          tmem_ld_wait();
        }
        if (!live || (a.splits > 1 && n == 0)) continue;
        float f[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = n > 0 && l != 0.f ? __uint_as_float(o[j]) * inv : 0.f;
        if (a.splits > 1) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + (split * a.all_rows + rr) * DH + 32 * x);
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<__half*>(a.o.p) + b * a.o.img + tq * a.o.row +
                                                (long long)h * DH + 32 * x);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            dst[j] = make_uint4(pack16<BF16>(f[8 * j], f[8 * j + 1]), pack16<BF16>(f[8 * j + 2], f[8 * j + 3]),
                                pack16<BF16>(f[8 * j + 4], f[8 * j + 5]), pack16<BF16>(f[8 * j + 6], f[8 * j + 7]));
        }
      }
      if (live) {
        if (a.splits > 1) a.part_l[split * a.all_rows + rr] = n > 0 ? lse : -INFINITY;
        else if (a.lse) a.lse[rr] = n > 0 ? lse : -INFINITY;
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == NT * 4) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
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
  int nt, kt, pairs, splits, key_tiles;
  long long units;
};

// Two tiles of rows a CTA where there are two (one CTA an SM), one otherwise (two CTAs an SM).  The
// key range is split where the CTAs' last wave would leave more SMs idle than the splits cost: a CTA
// spends about `kStart` key tiles on starting and ending, and joining costs about as much again.
FwdPlan fwd_plan(int B, int H, int Hkv, int Tq, int Tk, int sms) {
  constexpr int kStart = 4, kMost = 64;
  FwdPlan p;
  const int rows_tiles = (int)(((long long)(H / Hkv) * Tq + 127) / 128);
  p.nt = rows_tiles >= 2 ? 2 : 1;
  p.kt = p.nt == 2 ? 128 : 64;
  p.pairs = (rows_tiles + p.nt - 1) / p.nt;
  p.key_tiles = (Tk + p.kt - 1) / p.kt;
  p.units = (long long)B * Hkv * p.pairs;
  const long long slots = (long long)sms * (p.nt == 2 ? 1 : 2);
  p.splits = 1;
  double best = 1e300;
  for (int s = 1; s <= std::min(kMost, p.key_tiles); ++s) {
    const long long each = (p.key_tiles + s - 1) / s;
    if ((p.key_tiles + each - 1) / each != s) continue;  // some split would be empty
    const double cost = (double)((p.units * s + slots - 1) / slots) * (each + kStart) + (s > 1 ? kStart : 0);
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

template <int DH, bool BF16, int NT>
cudaError_t launch_fwd(const FwdArgs& a, long long grid, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  using C = Fwd<DH, NT>;
  cudaError_t e = cudaFuncSetAttribute(attend_kernel<DH, BF16, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  attend_kernel<DH, BF16, NT><<<(unsigned)grid, C::THREADS, C::SMEM, st>>>(a, k, v);
  e = cudaGetLastError();
  if (e != cudaSuccess || a.splits == 1) return e;
  const long long threads = a.all_rows * (DH / 8);
  attend_join_kernel<DH, BF16><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a);
  return cudaGetLastError();
}
template <int DH>
cudaError_t launch_fwd(const FwdArgs& a, const FwdPlan& p, bool bf16, const CUtensorMap& k, const CUtensorMap& v,
                       cudaStream_t st) {
  const long long grid = p.units * p.splits;
  if (p.nt == 2) return bf16 ? launch_fwd<DH, true, 2>(a, grid, k, v, st) : launch_fwd<DH, false, 2>(a, grid, k, v, st);
  return bf16 ? launch_fwd<DH, true, 1>(a, grid, k, v, st) : launch_fwd<DH, false, 1>(a, grid, k, v, st);
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

bool xattn_tensor_map(CUtensorMap* map, const View& v, int dtype, int B, int T, int heads, int dh, int rows) {
  PFN_encodeTiled enc = encode_fn();
  if (!enc) return false;
  const bool one = v.img == 0;
  const cuuint64_t row = (cuuint64_t)v.row * 2, img = one ? 16 : (cuuint64_t)v.img * 2;
  cuuint64_t dims[4] = {(cuuint64_t)dh, (cuuint64_t)T, (cuuint64_t)heads, one ? 1u : (cuuint64_t)B};
  cuuint64_t strides[3] = {row == 0 ? 16 : row, (cuuint64_t)dh * 2, img};
  cuuint32_t box[4] = {(cuuint32_t)std::min(dh, 64), (cuuint32_t)rows, 1u, 1u};
  cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  if (row == 0 && T > 1) return false;
  return enc(map, dtype == SB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void*>(v.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             dh < 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int xattn_error(int clear, int* flags) {
  const int zero = 0;
  if (cudaMemcpyFromSymbol(flags, g_xattn_error, sizeof(int)) != cudaSuccess) return -1;
  return clear && cudaMemcpyToSymbol(g_xattn_error, &zero, sizeof(int)) != cudaSuccess ? -1 : 0;
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

extern "C" int sb_cross_attention_work(int backward, int B, int H, int Hkv, int dh, int Tq, int Tk, long long* bytes) {
  if (!bytes || !xattn_sizes_ok(SB_F16, B, H, Hkv, dh, Tq, Tk))
    return record_error(SB_EINVAL, "sb_cross_attention_work: arguments");
  *bytes = 0;
  if (B == 0 || Tq == 0 || Tk == 0) return SB_OK;
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_cross_attention_work: device");
  if (backward) {
    *bytes = xattn_back_work(B, H, Hkv, dh, Tq, Tk, sms);
    return SB_OK;
  }
  const FwdPlan p = fwd_plan(B, H, Hkv, Tq, Tk, sms);
  if (p.splits > 1) *bytes = (long long)p.splits * B * H * Tq * (dh + 1) * 4;
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
      (Tk > 0 && (!xattn_view_ok(k, k_row, k_img) || !xattn_view_ok(v, v_row, v_img))))
    return record_error(SB_EINVAL, "sb_cross_attention: rows (16-byte aligned, strides multiples of 8)");
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
  const long long need = p.splits > 1 ? (long long)p.splits * B * H * Tq * (dh + 1) * 4 : 0;
  if (need > 0 && (!work || work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15) != 0))
    return record_error(SB_EINVAL, "sb_cross_attention: workspace (sb_cross_attention_work bytes, 16-byte aligned)");
  if (p.units * p.splits > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_cross_attention: too many items");
  FwdArgs a{};
  a.q = {q, q_row, q_img};
  a.o = {out, o_row, o_img};
  a.lse = lse;
  a.mask = {lens, static_cast<const uint8_t*>(valid), valid_img, Tk};
  a.B = B; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.Tq = Tq; a.rows = a.group * Tq;
  a.pairs = p.pairs; a.splits = p.splits; a.key_tiles = p.key_tiles;
  a.k_item = k_img != 0; a.v_item = v_img != 0;
  a.masked = lens || valid;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.all_rows = (long long)B * H * Tq;
  a.part_o = static_cast<float*>(work);
  a.part_l = a.part_o + (long long)p.splits * a.all_rows * dh;
  CUtensorMap km, vm;
  if (!xattn_tensor_map(&km, {k, k_row, k_img}, dtype, B, Tk, Hkv, dh, p.kt) ||
      !xattn_tensor_map(&vm, {v, v_row, v_img}, dtype, B, Tk, Hkv, dh, p.kt))
    return record_error(SB_EINVAL, "sb_cross_attention: tensor map of k or v");
  const bool bf16 = dtype == SB_BF16;
  const cudaError_t e = dh == 32 ? launch_fwd<32>(a, p, bf16, km, vm, st)
                        : dh == 64 ? launch_fwd<64>(a, p, bf16, km, vm, st) : launch_fwd<128>(a, p, bf16, km, vm, st);
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}
