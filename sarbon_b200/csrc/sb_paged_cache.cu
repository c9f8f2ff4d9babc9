// sb_paged_cache.cu -- a paged memory's upkeep: new states into their pages, and eviction of those that were
// looked at least.
#include <algorithm>
#include <cmath>

#include "sb_paged.cuh"

namespace sb {
namespace {

// ---------------------------------------------------------------- write
// Row (b, t), t < count[b], goes to position at[b] + t of item b.  Copies, bound by memory: a warp takes the
// rows of a group (their pages are looked up once, by a lane a row) and keeps four vectors of K and four of V a lane
// in flight (two where 32 bytes become 16 of e4m3).  e4m3 pages get the code of x / scale, a true division, or
// where both scales are powers of two the product with their reciprocals, which is the quotient.
struct WriteArgs {
  const void *k, *v;
  long long k_row, k_img, v_row, v_img;  // elements
  int dt;
  Pool kp, vp;
  PageTable pages;
  const int *at, *count, *stamp;
  long long stamp_img, stamp_row;
  int B, T, Hkv;
  float k_scale, v_scale;
  float* weight;
  int *born, *after;
  FastDiv vecs;  // 16-byte vectors a row of the pool
  int group;     // rows a warp
  long long rows, row_blocks, marks;  // marks: what else is written, one a thread
  SB_DEV int start(int b) const { return pages.clamp(at[b]); }
  SB_DEV int fresh(int b) const { return count ? min(max(count[b], 0), T) : T; }
};

constexpr int kWriteWarps = 8;

// The 16 bytes of a pool's vector from row element i on: eight values, or sixteen as e4m3.
template <bool E4M3>
struct Vec {
  Raw8 r[E4M3 ? 2 : 1];
};
template <bool E4M3, bool ALIGNED>
SB_DEV Vec<E4M3> load_vec(const void* p, int dt, long long i) {
  Vec<E4M3> v;
#pragma unroll
  for (int x = 0; x < (E4M3 ? 2 : 1); ++x)
    v.r[x] = ALIGNED ? load_raw8(p, dt, i + 8 * x) : load_raw8_tail(p, dt, i + 8 * x, 8);
  return v;
}
// MODE 0: as they are; 1: e4m3 of x * scale; 2: e4m3 of x / scale
template <int MODE>
SB_DEV uint4 pool_vec(const Vec<(MODE > 0)>& v, int dt, float scale) {
  if constexpr (MODE == 0) {
    return v.r[0].lo;
  } else {
    uint32_t w[4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float f[8];
      unpack8(v.r[x], dt, f);
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] = MODE == 1 ? f[u] * scale : __fdiv_rn(f[u], scale);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        w[2 * x + u] = (uint32_t)e4m3x2_of(f[4 * u], f[4 * u + 1]) | (uint32_t)e4m3x2_of(f[4 * u + 2], f[4 * u + 3]) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int MODE, bool ALIGNED>
__global__ void __launch_bounds__(kWriteWarps * 32) paged_write_kernel(const __grid_constant__ WriteArgs a) {
  constexpr bool E4M3 = MODE > 0;
  constexpr int kAhead = E4M3 ? 2 : 4;
  if (blockIdx.x >= a.row_blocks) {  // new lengths, then weights and stamps, neighbours along t
    long long i = (blockIdx.x - a.row_blocks) * (kWriteWarps * 32) + threadIdx.x;
    if (i >= a.marks) return;
    if (i < a.B) {
      a.after[i] = min(a.start((int)i) + a.fresh((int)i), a.pages.cap);
      return;
    }
    i -= a.B;
    const int t = (int)(i % a.T);
    const long long unit = i / a.T;
    const int b = (int)(unit / a.Hkv), pos = a.start(b) + t;
    if (t >= a.fresh(b) || pos >= a.pages.cap) return;
    if (a.weight) a.weight[unit * a.pages.cap + pos] = 0.f;
    if (a.born) a.born[unit * a.pages.cap + pos] = a.stamp ? a.stamp[b * a.stamp_img + t * a.stamp_row] : 0;
    return;
  }
  __shared__ ulonglong2 to[kWriteWarps][32];  // addresses in the pools (0: nowhere)
  __shared__ longlong2 from[kWriteWarps][32];  // elements
  const int warp = warp_id(), lane = lane_id();
  const long long r0 = ((long long)blockIdx.x * kWriteWarps + warp) * a.group;
  if (r0 >= a.rows) return;
  const int rows = (int)min((long long)a.group, a.rows - r0);
  if (lane < rows) {
    const long long r = r0 + lane;
    const int b = (int)(r / a.T), t = (int)(r - (long long)b * a.T), pos = a.start(b) + t;
    ulonglong2 where = make_ulonglong2(0, 0);
    if (t < a.fresh(b) && pos < a.pages.cap) {
      uint32_t row;
      const int p = a.pages.entry(b, (uint32_t)pos, row);
      if (a.pages.has(p)) where = make_ulonglong2(a.kp.row_at(p, row), a.vp.row_at(p, row));
    }
    to[warp][lane] = where;
    from[warp][lane] = make_longlong2(b * a.k_img + t * a.k_row, b * a.v_img + t * a.v_row);
  }
  __syncwarp();
  const int total = rows * (int)a.vecs.d;
  constexpr int per = E4M3 ? 16 : 8;
  for (int i0 = lane; i0 < total; i0 += 32 * kAhead) {
    Vec<E4M3> k[kAhead], v[kAhead];
    ulonglong2 where[kAhead];
    int c[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      const int i = i0 + 32 * x;
      where[x] = make_ulonglong2(0, 0);
      if (i < total) {
        const int r = (int)a.vecs.div((uint32_t)i);
        c[x] = i - r * (int)a.vecs.d;
        where[x] = to[warp][r];
        if (where[x].x) {
          const longlong2 s = from[warp][r];
          k[x] = load_vec<E4M3, ALIGNED>(a.k, a.dt, s.x + c[x] * per);
          v[x] = load_vec<E4M3, ALIGNED>(a.v, a.dt, s.y + c[x] * per);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kAhead; ++x)
      if (where[x].x) {
        *reinterpret_cast<uint4*>(where[x].x + c[x] * 16) = pool_vec<MODE>(k[x], a.dt, a.k_scale);
        *reinterpret_cast<uint4*>(where[x].y + c[x] * 16) = pool_vec<MODE>(v[x], a.dt, a.v_scale);
      }
  }
}

// ---------------------------------------------------------------- evict
// Of the len states of an (item, key head), the keep largest by (born >= since, weight, -index) stay; the i-th freed
// place below keep takes the i-th kept state from keep on.  So what moves is only what has to, and no row is both
// read and written.
//
// A first kernel, a cluster of CTAs an (item, key head), finds the weight of the last state that stays by radix
// selection (11, 11 and 10 bits; each CTA counts its own states in shared memory and all add up the others'
// counts) and pairs places with states; the second moves the rows.  The weights, as integers of the same
// order, are kept in shared memory where they fit.
struct EvictArgs {
  Pool k, v;
  PageTable pages;
  const int *lens, *keep, *since;
  int keep_all;  // where keep is null
  const float* weight;
  float* weight_out;
  const int* born;
  int* born_out;
  int* after;
  int B, Hkv, row_bytes, half, parts, ctas;
  int *to, *from, *moves;  // workspace: [units][half], [units][half], [units]
  uint32_t* bits;          // [units][2][cap / 32]: states that are protected, that stay, where shared memory has no room
  SB_DEV int budget(int b) const { return pages.clamp(keep ? keep[b] : keep_all); }
};

constexpr int kSelect = 512, kSelectWarps = kSelect / 32, kBins = 2048, kMostCtas = 8;
constexpr int kSelectRoom = 92 * 1024;  // shared memory for weights and bits, two CTAs an SM
// words of 32 states of a CTA, one of `ctas`
inline int select_words(int cap, int ctas) {
  const int words = (cap + 31) / 32, warps = kSelectWarps * ctas;
  return (words + warps - 1) / warps * kSelectWarps;
}
inline long long select_bytes(int cap, int ctas) { return select_words(cap, ctas) * (32ll * 4 + 8); }

// Integers in the order of the weights; NaN is the least, both zeros are one.
SB_DEV uint32_t ordered(float w) {
  if (w != w) return 0u;
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums over the warps before this one and over all, of the CTA.  `room`: 33 ints; begins and ends with a barrier.
SB_DEV int warps_before(int v, int* room, int& total) {
  const int lane = lane_id(), warp = warp_id();
  __syncthreads();
  if (lane == 0) room[warp] = v;
  __syncthreads();
  int w = lane < kSelectWarps ? room[lane] : 0, s = w;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, s, x);
    if (lane >= x) s += u;
  }
  total = __shfl_sync(0xFFFFFFFFu, s, 31);
  const int before = __shfl_sync(0xFFFFFFFFu, s - w, warp);
  return before;
}
// The same over the warps of all CTAs of the cluster; `mine`: an int of its own for each call.
SB_DEV int warps_before_all(int v, int* room, int* mine, int ctas, uint32_t rank, int& total) {
  int before = warps_before(v, room, total);
  if (ctas > 1) {
    if (threadIdx.x == 0) *mine = total;
    cluster_sync();
    int all = 0;
    for (uint32_t r = 0; r < (uint32_t)ctas; ++r) {
      const int t = (int)peer_word(mine, r);
      if (r < rank) before += t;
      all += t;
    }
    total = all;
  }
  return before;
}

// A warp's states lie behind one another, so that places come out in order; kAtOnce times 32 at a time.
// HELD: the weights and bits are in shared memory.
template <bool HELD>
__global__ void __launch_bounds__(kSelect, 2) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  constexpr int kAtOnce = 8;
  extern __shared__ __align__(16) uint32_t held[];  // the CTA's ordered weights; words of protected states and of those that stay
  __shared__ int bins[kBins], sums[kBins];
  __shared__ int room[33], totals[4], found[2];
  const int warp = warp_id(), lane = lane_id(), cap = a.pages.cap, ctas = a.ctas;
  const uint32_t rank = ctas > 1 ? cluster_ctarank() : 0u;
  const long long unit = blockIdx.x / ctas;
  const int b = (int)(unit / a.Hkv);
  const int len = a.pages.clamp(a.lens[b]), keep = a.budget(b), left = min(len, keep);
  const float* weight = a.weight + unit * cap;
  float* weight_out = a.weight_out + unit * cap;
  const int* born = a.born ? a.born + unit * cap : nullptr;
  int* born_out = a.born ? a.born_out + unit * cap : nullptr;
  const bool guard = born && a.since;
  const int since = guard ? a.since[b] : 0;
  int* to = a.to + unit * a.half;
  int* from = a.from + unit * a.half;
  const int warps = kSelectWarps * ctas, words = (len + 31) / 32, steps = (words + warps - 1) / warps;
  const int w_first = min(((int)rank * kSelectWarps + warp) * steps, words), w_end = min(w_first + steps, words);
  // words of this CTA, from its first on; in memory, of the unit
  const int base = HELD ? (int)rank * kSelectWarps * steps : 0, all_words = (cap + 31) / 32;
  uint32_t* guarded = HELD ? held + kSelectWarps * steps * 32 : a.bits + unit * 2 * all_words;
  uint32_t* stay = HELD ? guarded + kSelectWarps * steps : guarded + all_words;
  int moves = 0;
  auto cta_sync = [&] {
    if (ctas > 1) cluster_sync();
    else __syncthreads();
  };

  if (len > keep) {
    // what the passes look at: the ordered weight of state j (below len, else 0) and the bits of its word
    auto key_of = [&](int w) {
      const int j = w * 32 + lane;
      return HELD ? held[(w - base) * 32 + lane] : j < len ? ordered(weight[j]) : 0u;
    };
    int n = 0;
    for (int w0 = w_first; w0 < w_end; w0 += kAtOnce) {
      float f[kAtOnce];
      int s[kAtOnce];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) {
        const int j = (w0 + x) * 32 + lane;
        const bool in = w0 + x < w_end && j < len;
        f[x] = HELD && in ? weight[j] : 0.f;
        s[x] = guard && in ? born[j] : 0;
      }
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) {
        const int j = (w0 + x) * 32 + lane;
        if (w0 + x < w_end) {
          const uint32_t word = __ballot_sync(0xFFFFFFFFu, guard && j < len && s[x] >= since);
          if (HELD) held[(w0 + x - base) * 32 + lane] = ordered(f[x]);
          if (lane == 0) guarded[w0 + x - base] = word;
          n += __popc(word);
        }
      }
    }
    int all;
    warps_before_all(n, room, &totals[0], ctas, rank, all);
    // the states among which weights decide: the protected ones where they alone are too many, else the others
    const bool inner = all >= keep;
    const uint32_t flip = inner ? 0u : 0xFFFFFFFFu;
    int need = inner ? keep : keep - all, same = 0;
    uint32_t last = 0xFFFFFFFFu;  // the ordered weight of the last state that stays; `need` of that weight do
    if (need > 0) {
      last = 0;
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xFFE00000u : 0xFFFFFC00u;
        for (int x = threadIdx.x; x < kBins; x += kSelect) bins[x] = 0;
        __syncthreads();
        for (int w0 = w_first; w0 < w_end; w0 += kAtOnce) {
          uint32_t key[kAtOnce], who[kAtOnce];
#pragma unroll
          for (int x = 0; x < kAtOnce; ++x) {
            const int w = w0 + x;
            key[x] = w < w_end ? key_of(w) : 0u;
            who[x] = w < w_end ? (guarded[w - base] ^ flip) & bits_below(w * 32, len) : 0u;
          }
#pragma unroll
          for (int x = 0; x < kAtOnce; ++x) {
            const bool mine = (who[x] >> lane & 1u) && (key[x] & mask) == last;
            const uint32_t some = __ballot_sync(0xFFFFFFFFu, mine);
            if (some == 0) continue;
            const int bin = key[x] >> shift & (pass == 2 ? 1023 : 2047);
            // many states of one weight (new ones have 0): one count for the warp
            const int one = __shfl_sync(0xFFFFFFFFu, bin, __ffs(some) - 1);
            if (__all_sync(0xFFFFFFFFu, !mine || bin == one)) {
              if (lane == 0) atomicAdd(&bins[one], __popc(some));
            } else if (mine) {
              atomicAdd(&bins[bin], 1);
            }
          }
        }
        cta_sync();
        // four bins a thread, from the top
        const int top = kBins - 1 - 4 * (int)threadIdx.x;
        int c[4], four = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          c[x] = 0;
          if (ctas > 1)
            for (uint32_t r = 0; r < (uint32_t)ctas; ++r) c[x] += (int)peer_word(&bins[top - x], r);
          else c[x] = bins[top - x];
          sums[top - x] = c[x];
          four += c[x];
        }
        if (ctas > 1) cluster_sync();  // bins are written again
        int s = four, total;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const int u = __shfl_up_sync(0xFFFFFFFFu, s, x);
          if (lane >= x) s += u;
        }
        int above = warps_before(__shfl_sync(0xFFFFFFFFu, s, 31), room, total) + s - four;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (above < need && need <= above + c[x]) {
            found[0] = top - x;
            found[1] = above;
          }
          above += c[x];
        }
        __syncthreads();
        last |= (uint32_t)found[0] << shift;
        need -= found[1];
        same = sums[found[0]];
        __syncthreads();  // sums and found are written again
      }
    }
    // where more states have the last weight than may stay, the first of them do
    const bool some = need > 0, choose = same > need;
    int ties = 0;
    if (choose) {
      n = 0;
      for (int w = w_first; w < w_end; ++w) {
        const uint32_t who = (guarded[w - base] ^ flip) & bits_below(w * 32, len);
        n += __popc(__ballot_sync(0xFFFFFFFFu, key_of(w) == last) & who);
      }
      int total;
      ties = warps_before_all(n, room, &totals[1], ctas, rank, total);
    }
    int free = 0, move = 0;
    for (int w0 = w_first; w0 < w_end; w0 += kAtOnce) {
      uint32_t key[kAtOnce], g[kAtOnce];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) {
        const int w = w0 + x;
        key[x] = w < w_end ? key_of(w) : 0u;
        g[x] = w < w_end ? guarded[w - base] : 0u;
      }
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) {
        const int w = w0 + x;
        if (w < w_end) {
          const uint32_t here = bits_below(w * 32, len), low = bits_below(w * 32, keep), who = (g[x] ^ flip) & here;
          const uint32_t more = __ballot_sync(0xFFFFFFFFu, key[x] > last) & who;
          uint32_t tied = some ? __ballot_sync(0xFFFFFFFFu, key[x] == last) & who : 0u;
          uint32_t first = tied;
          if (choose) {
            first = __ballot_sync(0xFFFFFFFFu, (tied >> lane & 1u) && ties + __popc(tied & ((1u << lane) - 1u)) < need);
            ties += __popc(tied);
          }
          const uint32_t stays = more | first | (inner ? 0u : g[x] & here);
          if (lane == 0) stay[w - base] = stays;
          free += __popc(~stays & low & here);
          move += __popc(stays & ~low);
        }
      }
    }
    int total;
    int at_free = warps_before_all(free, room, &totals[2], ctas, rank, total);
    int at_move = warps_before_all(move, room, &totals[3], ctas, rank, moves);
    for (int w = w_first; w < w_end; ++w) {
      const int j = w * 32 + lane;
      const uint32_t s = stay[w - base], low = bits_below(w * 32, keep), below = (1u << lane) - 1u;
      const uint32_t f = ~s & low & bits_below(w * 32, len), m = s & ~low;
      if (f >> lane & 1u) to[at_free + __popc(f & below)] = j;
      if (m >> lane & 1u) from[at_move + __popc(m & below)] = j;
      if (weight_out != weight && (s & low) >> lane & 1u) weight_out[j] = weight[j];
      if (born_out != born && (s & low) >> lane & 1u) born_out[j] = born[j];
      at_free += __popc(f);
      at_move += __popc(m);
    }
    cta_sync();
    for (int i = (int)rank * kSelect + threadIdx.x; i < moves; i += ctas * kSelect) {
      const int d = to[i], s = from[i];
      weight_out[d] = weight[s];
      if (born) born_out[d] = born[s];
    }
    cta_sync();  // where the results lie on the operands: read before they are cleared
  } else {
    for (int j = (int)rank * kSelect + threadIdx.x; j < len; j += ctas * kSelect) {
      if (weight_out != weight) weight_out[j] = weight[j];
      if (born_out != born) born_out[j] = born[j];
    }
  }
  for (int j = left + (int)rank * kSelect + threadIdx.x; j < cap; j += ctas * kSelect) {
    weight_out[j] = 0.f;
    if (born) born_out[j] = 0;
  }
  if (threadIdx.x == 0 && rank == 0) a.moves[unit] = moves;
  if (ctas > 1) cluster_sync();  // no CTA ends while another reads its counts
}

// Rows of the pairs: a warp takes 32 pairs, a lane looks up where a pair's rows lie, then all copy them, 16 bytes a lane,
// four loads of K and four of V in flight.  And the new lengths, which may lie on the old ones: nothing but the
// thread that writes an item's reads it here.
constexpr int kMoveWarps = 4, kMoveAhead = 4;
template <int LANES>
__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ ulonglong2 source[kMoveWarps][32], target[kMoveWarps][32];  // addresses of K and V; 0: nowhere
  const int warp = warp_id(), lane = lane_id();
  const int part = blockIdx.x % a.parts;
  const long long unit = blockIdx.x / a.parts;
  const int b = (int)(unit / a.Hkv), h = (int)(unit - (long long)b * a.Hkv);
  grid_dep_wait();
  if (h == 0 && part == 0 && threadIdx.x == 0) a.after[b] = min(a.pages.clamp(a.lens[b]), a.budget(b));
  const int moves = a.moves[unit];
  const long long c = (long long)h * a.row_bytes + lane % LANES * 16;
  const int *to = a.to + unit * a.half, *from = a.from + unit * a.half;
  constexpr int AT_ONCE = 32 / LANES;
  for (int i0 = (part * kMoveWarps + warp) * 32; i0 < moves; i0 += a.parts * kMoveWarps * 32) {
    ulonglong2 p = make_ulonglong2(0, 0), q = p;
    if (i0 + lane < moves) {
      uint32_t dr, sr;
      const int d = to[i0 + lane], s = from[i0 + lane];
      const int dp = a.pages.entry(b, (uint32_t)d, dr), sp = a.pages.entry(b, (uint32_t)s, sr);
      if (a.pages.has(dp) && a.pages.has(sp)) {
        p = make_ulonglong2(a.k.row_at(sp, sr), a.v.row_at(sp, sr));
        q = make_ulonglong2(a.k.row_at(dp, dr), a.v.row_at(dp, dr));
      }
    }
    __syncwarp();
    source[warp][lane] = p;
    target[warp][lane] = q;
    __syncwarp();
#pragma unroll
    for (int x0 = 0; x0 < LANES; x0 += kMoveAhead) {
      if (i0 + x0 * AT_ONCE >= moves) break;
      uint4 k[kMoveAhead], v[kMoveAhead];
#pragma unroll
      for (int x = 0; x < kMoveAhead; ++x)
        if (x0 + x < LANES) {
          const ulonglong2 at = source[warp][(x0 + x) * AT_ONCE + lane / LANES];
          if (at.x) {
            k[x] = *reinterpret_cast<const uint4*>(at.x + c);
            v[x] = *reinterpret_cast<const uint4*>(at.y + c);
          }
        }
#pragma unroll
      for (int x = 0; x < kMoveAhead; ++x)
        if (x0 + x < LANES) {
          const ulonglong2 at = target[warp][(x0 + x) * AT_ONCE + lane / LANES];
          if (at.x) {
            *reinterpret_cast<uint4*>(at.x + c) = k[x];
            *reinterpret_cast<uint4*>(at.y + c) = v[x];
          }
        }
    }
  }
}

struct EvictPlan {
  int half, words, ctas, parts;
  bool held;
  long long lists, moves, bits;  // ints
  long long bytes() const { return (lists + moves + bits) * 4; }
};
// CTAs an (item, key head): doubled while all are resident at once (two an SM) and each still has 2048 places, or until
// the weights fit shared memory.
EvictPlan evict_plan(int B, int Hkv, int cap, int sms) {
  const long long units = (long long)B * Hkv;
  EvictPlan p{};
  p.half = std::max(1, cap / 2);  // at most min(keep, len - keep) states move
  p.words = (cap + 31) / 32;
  p.ctas = 1;
  while (p.ctas < kMostCtas &&
         ((2 * units * p.ctas <= 2 * sms && cap / p.ctas > 2048) || select_bytes(cap, p.ctas) > kSelectRoom))
    p.ctas *= 2;
  p.held = select_bytes(cap, p.ctas) <= kSelectRoom;
  p.parts = (int)std::max(1ll, std::min(((long long)p.half + kMoveWarps * 32 - 1) / (kMoveWarps * 32), (16ll * sms + units - 1) / units));
  p.lists = 2 * units * p.half;
  p.moves = units;
  p.bits = p.held ? 0 : 2 * units * p.words;
  return p;
}

template <bool HELD>
cudaError_t evict_select(const EvictArgs& a, long long units, cudaStream_t st) {
  static bool ready[64];
  const size_t room = HELD ? (size_t)select_bytes(a.pages.cap, a.ctas) : 0;
  const cudaError_t e = xattn_smem(reinterpret_cast<const void*>(&evict_select_kernel<HELD>), kSelectRoom, ready);
  return e != cudaSuccess ? e : launch_after(evict_select_kernel<HELD>, units * a.ctas, kSelect, room, st, a, a.ctas, false);
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_paged_write(const sb_paged_memory* memory, const void* k, long long k_row, long long k_img, const void* v,
                              long long v_row, long long v_img, int dtype, const int* at, const int* count, int T,
                              float k_scale, float v_scale, float* weight, int* born, const int* stamp, long long stamp_img,
                              long long stamp_row, int* after, void* stream) {
  const sb_paged_memory* const m = memory;
  if (!paged_memory_ok(m) || T < 0 || T >= (1 << 30) || (dtype != SB_F16 && dtype != SB_BF16) ||
      (m->dtype != dtype && m->dtype != SB_F8))
    return record_error(SB_EINVAL, "sb_paged_write: sizes (dh 32, 64 or 128) or dtypes");
  if (!scales_ok(m, k_scale, v_scale)) return record_error(SB_EINVAL, "sb_paged_write: scales, or scales of pages that are not e4m3");
  if (m->B == 0) return SB_OK;
  const bool some = T > 0 && m->P > 0 && m->N > 0;
  if (!at || !after || !paged_pools_ok(m) || (some && (!k || !v || k_row < 0 || k_img < 0 || v_row < 0 || v_img < 0)))
    return record_error(SB_EINVAL, "sb_paged_write: rows (pools 16-byte aligned, strides multiples of 16 bytes) or null argument");
  WriteArgs a{};
  a.k = k; a.k_row = k_row; a.k_img = k_img;
  a.v = v; a.v_row = v_row; a.v_img = v_img;
  a.dt = dtype;
  a.kp = k_pool(m);
  a.vp = v_pool(m);
  a.pages = page_table(m);
  a.at = at; a.count = count; a.stamp = stamp; a.stamp_img = stamp_img; a.stamp_row = stamp_row;
  a.B = m->B; a.T = T; a.Hkv = m->Hkv;
  a.k_scale = k_scale; a.v_scale = v_scale;
  a.weight = weight; a.born = born; a.after = after;
  const bool e4m3 = m->dtype == SB_F8;
  const int vecs = m->Hkv * m->dh * (e4m3 ? 1 : 2) / 16;
  a.vecs = fast_div((uint32_t)vecs);
  a.group = std::min(32, std::max(1, 128 / vecs));
  a.rows = some ? (long long)m->B * T : 0;
  const long long warps = (a.rows + a.group - 1) / a.group;
  a.row_blocks = (warps + kWriteWarps - 1) / kWriteWarps;
  a.marks = m->B + (T > 0 && m->N > 0 && (weight || born) ? (long long)m->B * m->Hkv * T : 0);
  const long long blocks = a.row_blocks + (a.marks + kWriteWarps * 32 - 1) / (kWriteWarps * 32);
  if (blocks > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_paged_write: too many rows");
  auto aligned = [](const void* p, long long row, long long img) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row % 8 == 0 && img % 8 == 0;
  };
  const bool vec = aligned(k, k_row, k_img) && aligned(v, v_row, v_img);
  int bits;
  const bool exact = std::frexp(k_scale, &bits) == 0.5f && std::abs(bits) < 120 && std::frexp(v_scale, &bits) == 0.5f && std::abs(bits) < 120;
  if (exact) {
    a.k_scale = 1.f / k_scale;
    a.v_scale = 1.f / v_scale;
  }
  auto kernel = !e4m3  ? (vec ? paged_write_kernel<0, true> : paged_write_kernel<0, false>)
                : exact ? (vec ? paged_write_kernel<1, true> : paged_write_kernel<1, false>)
                        : (vec ? paged_write_kernel<2, true> : paged_write_kernel<2, false>);
  kernel<<<(unsigned)blocks, kWriteWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}

extern "C" int sb_paged_evict_work(int B, int Hkv, int page, int N, long long* bytes) {
  if (!bytes || !paged_sizes_ok(B, Hkv, 32, 0, page, N)) return record_error(SB_EINVAL, "sb_paged_evict_work: arguments");
  *bytes = 0;
  if (B == 0) return SB_OK;
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_evict_work: device");
  *bytes = evict_plan(B, Hkv, N * page, sms).bytes();
  return SB_OK;
}

extern "C" int sb_paged_evict(const sb_paged_memory* memory, const int* lens, const int* keep, int keep_all, const int* since,
                              const float* weight, const int* born, float* weight_out, int* born_out, int* after, void* work,
                              long long work_bytes, void* stream) {
  const sb_paged_memory* const m = memory;
  if (!paged_memory_ok(m)) return record_error(SB_EINVAL, "sb_paged_evict: sizes (dh 32, 64 or 128) or dtype");
  if (m->B == 0) return SB_OK;
  if (!lens || !after || (m->N > 0 && (!weight || !weight_out)) || (since && !born) || (!born) != (!born_out) || !paged_pools_ok(m))
    return record_error(SB_EINVAL, "sb_paged_evict: rows (16-byte aligned, strides multiples of 16 bytes) or null argument");
  if (!work || (reinterpret_cast<uintptr_t>(work) & 15) != 0)
    return record_error(SB_EINVAL, "sb_paged_evict: workspace (sb_paged_evict_work bytes, 16-byte aligned)");
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_evict: device");
  EvictArgs a{};
  a.pages = page_table(m);
  const EvictPlan p = evict_plan(m->B, m->Hkv, a.pages.cap, sms);
  if (work_bytes < p.bytes()) return record_error(SB_EINVAL, "sb_paged_evict: workspace (sb_paged_evict_work bytes, 16-byte aligned)");
  a.k = k_pool(m);
  a.v = v_pool(m);
  a.lens = lens; a.keep = keep; a.keep_all = keep_all; a.since = since;
  a.weight = weight; a.weight_out = weight_out; a.born = born; a.born_out = born_out; a.after = after;
  a.B = m->B; a.Hkv = m->Hkv; a.row_bytes = m->dh * page_dtype_bytes(m->dtype); a.half = p.half;
  a.ctas = p.ctas; a.parts = p.parts;
  const long long units = (long long)m->B * m->Hkv;
  if (units * std::max(p.ctas, p.parts) > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_paged_evict: too many items");
  a.to = static_cast<int*>(work);
  a.from = a.to + units * p.half;
  a.moves = a.from + units * p.half;
  a.bits = reinterpret_cast<uint32_t*>(a.moves + units);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = p.held ? evict_select<true>(a, units, st) : evict_select<false>(a, units, st);
  if (e == cudaSuccess) {
    auto move = a.row_bytes == 32   ? evict_move_kernel<2>
                : a.row_bytes == 64 ? evict_move_kernel<4> : a.row_bytes == 128 ? evict_move_kernel<8> : evict_move_kernel<16>;
    e = launch_after(move, units * a.parts, kMoveWarps * 32, 0, st, a);
  }
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}
