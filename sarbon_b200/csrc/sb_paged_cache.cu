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
// in flight.  e4m3 pages get round(x / scale), a true division, so that the codes are those of the quotient.
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

constexpr int kWriteWarps = 8, kAhead = 4;

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
template <bool E4M3>
SB_DEV uint4 pool_vec(const Vec<E4M3>& v, int dt, float scale) {
  if constexpr (!E4M3) {
    return v.r[0].lo;
  } else {
    uint32_t w[4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float f[8];
      unpack8(v.r[x], dt, f);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        w[2 * x + u] = (uint32_t)e4m3x2_of(__fdiv_rn(f[4 * u], scale), __fdiv_rn(f[4 * u + 1], scale)) |
                       (uint32_t)e4m3x2_of(__fdiv_rn(f[4 * u + 2], scale), __fdiv_rn(f[4 * u + 3], scale)) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool E4M3, bool ALIGNED>
__global__ void __launch_bounds__(kWriteWarps * 32) paged_write_kernel(const __grid_constant__ WriteArgs a) {
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
  __shared__ longlong2 to[kWriteWarps][32], from[kWriteWarps][32];  // byte offsets in the pools (-1: nowhere), elements
  const int warp = warp_id(), lane = lane_id();
  const long long r0 = ((long long)blockIdx.x * kWriteWarps + warp) * a.group;
  if (r0 >= a.rows) return;
  const int rows = (int)min((long long)a.group, a.rows - r0);
  if (lane < rows) {
    const long long r = r0 + lane;
    const int b = (int)(r / a.T), t = (int)(r - (long long)b * a.T), pos = a.start(b) + t;
    longlong2 where = make_longlong2(-1, -1);
    if (t < a.fresh(b) && pos < a.pages.cap) {
      uint32_t row;
      const long long p = a.pages.entry(b, (uint32_t)pos, row);
      if (a.pages.has((int)p)) where = make_longlong2(p * a.kp.page + row * a.kp.row, p * a.vp.page + row * a.vp.row);
    }
    to[warp][lane] = where;
    from[warp][lane] = make_longlong2(b * a.k_img + t * a.k_row, b * a.v_img + t * a.v_row);
  }
  __syncwarp();
  const int total = rows * (int)a.vecs.d;
  constexpr int per = E4M3 ? 16 : 8;
  for (int i0 = lane; i0 < total; i0 += 32 * kAhead) {
    Vec<E4M3> k[kAhead], v[kAhead];
    longlong2 where[kAhead];
    int c[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      const int i = i0 + 32 * x;
      where[x] = make_longlong2(-1, -1);
      if (i < total) {
        const int r = (int)a.vecs.div((uint32_t)i);
        c[x] = i - r * (int)a.vecs.d;
        where[x] = to[warp][r];
        if (where[x].x >= 0) {
          const longlong2 s = from[warp][r];
          k[x] = load_vec<E4M3, ALIGNED>(a.k, a.dt, s.x + c[x] * per);
          v[x] = load_vec<E4M3, ALIGNED>(a.v, a.dt, s.y + c[x] * per);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kAhead; ++x)
      if (where[x].x >= 0) {
        *reinterpret_cast<uint4*>(a.kp.p + where[x].x + c[x] * 16) = pool_vec<E4M3>(k[x], a.dt, a.k_scale);
        *reinterpret_cast<uint4*>(a.vp.p + where[x].y + c[x] * 16) = pool_vec<E4M3>(v[x], a.dt, a.v_scale);
      }
  }
}

// ---------------------------------------------------------------- evict
// Of the len states of an (item, key head), the keep largest by (born >= since, weight, -index) stay; the i-th freed
// place below keep takes the i-th kept state from keep on.  So what moves is only what has to, and no row is both
// read and written.
//
// A first kernel, a CTA an (item, key head), finds the weight of the last state that stays by radix selection
// (11, 11 and 10 bits, counts in shared memory) and pairs places with states; the second moves the rows.  The
// weights, as integers of the same order, are kept in shared memory where they fit.
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
  int B, Hkv, row_bytes, half, parts;
  int *to, *from, *moves;  // workspace: [units][half], [units][half], [units]
  uint32_t* bits;          // [units][cap / 32]: states that stay, where shared memory has no room
  SB_DEV int budget(int b) const { return pages.clamp(keep ? keep[b] : keep_all); }
};

constexpr int kSelect = 1024, kBins = 2048;
constexpr int kSelectRoom = 200 * 1024;  // shared memory for weights and bits
inline long long select_bytes(int cap) { return ((long long)cap + 31) / 32 * 32 * 4 + ((long long)cap + 31) / 32 * 8; }

// Integers in the order of the weights; NaN is the least, both zeros are one.
SB_DEV uint32_t ordered(float w) {
  if (w != w) return 0u;
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the CTA's threads, and the total.  `room`: 33 ints; ends with a barrier.
SB_DEV int sum_before(int v, int* room, int& total) {
  const int lane = lane_id(), warp = warp_id();
  int s = v;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, s, x);
    if (lane >= x) s += u;
  }
  if (lane == 31) room[warp] = s;
  __syncthreads();
  if (warp == 0) {
    const int w = room[lane];
    int t = w;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, t, x);
      if (lane >= x) t += u;
    }
    room[lane] = t - w;
    if (lane == 31) room[32] = t;
  }
  __syncthreads();
  const int before = room[warp] + s - v;
  total = room[32];
  __syncthreads();
  return before;
}
static_assert(kSelect == 1024, "sum_before: 32 warps");

// A warp's states lie behind one another, so that places come out in order; 32 at a time.
// HELD: the weights and bits are in shared memory.
template <bool HELD>
__global__ void __launch_bounds__(kSelect, 1) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ __align__(16) uint32_t held[];  // [cap] ordered weights, [cap / 32] protected, [cap / 32] stay
  __shared__ int bins[kBins];
  __shared__ int room[33], found[2];
  const int warp = warp_id(), lane = lane_id(), cap = a.pages.cap, words = (cap + 31) / 32;
  const long long unit = blockIdx.x;
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
  uint32_t* guarded = held + words * 32;
  uint32_t* stay = HELD ? guarded + words : a.bits + unit * words;
  const int steps = ((len + 31) / 32 + 31) / 32, j_first = warp * steps * 32, j_end = min(j_first + steps * 32, len);
  int moves = 0;

  if (len > keep) {
    auto key_of = [&](int j) { return HELD ? held[j] : ordered(weight[j]); };
    auto word_of = [&](int j, bool in) {  // protected states j .. of the warp, as bits
      return HELD ? guarded[j >> 5] : __ballot_sync(0xFFFFFFFFu, in && guard && born[j + lane] >= since);
    };
    int n = 0;
    for (int j = j_first; j < j_end; j += 32) {
      const bool in = j + lane < j_end;
      const uint32_t w = __ballot_sync(0xFFFFFFFFu, in && guard && born[j + lane] >= since);
      if (HELD) {
        if (in) held[j + lane] = ordered(weight[j + lane]);
        if (lane == 0) guarded[j >> 5] = w;
      }
      n += __popc(w);
    }
    int all;
    sum_before(lane == 0 ? n : 0, room, all);
    // the states among which weights decide: the protected ones where they alone are too many, else the others
    const bool inner = all >= keep;
    int need = inner ? keep : keep - all, same = 0;
    uint32_t last = 0xFFFFFFFFu;  // the ordered weight of the last state that stays; `need` of that weight do
    if (need > 0) {
      last = 0;
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xFFE00000u : 0xFFFFFC00u;
        bins[threadIdx.x] = bins[threadIdx.x + kSelect] = 0;
        __syncthreads();
        for (int j = j_first; j < j_end; j += 32) {
          const bool in = j + lane < j_end;
          const uint32_t w = word_of(j, in), key = in ? key_of(j + lane) : 0u;
          const bool mine = in && (w >> lane & 1u) == (uint32_t)inner && (key & mask) == last;
          const uint32_t some = __ballot_sync(0xFFFFFFFFu, mine);
          if (some == 0) continue;
          const int bin = key >> shift & (pass == 2 ? 1023 : 2047);
          // many states of one weight (new ones have 0): one count for the warp
          const int one = __shfl_sync(0xFFFFFFFFu, bin, __ffs(some) - 1);
          if (__all_sync(0xFFFFFFFFu, !mine || bin == one)) {
            if (lane == 0) atomicAdd(&bins[one], __popc(some));
          } else if (mine) {
            atomicAdd(&bins[bin], 1);
          }
        }
        __syncthreads();
        const int top = kBins - 1 - 2 * threadIdx.x, c0 = bins[top], c1 = bins[top - 1];
        int total;
        const int above = sum_before(c0 + c1, room, total);
        if (above < need && need <= above + c0 + c1) {
          const bool upper = need <= above + c0;
          found[0] = upper ? top : top - 1;
          found[1] = upper ? above : above + c0;
        }
        __syncthreads();
        last |= (uint32_t)found[0] << shift;
        need -= found[1];
        same = bins[found[0]];
        __syncthreads();  // bins and found are written again
      }
    }
    // where more states have the last weight than may stay, the first of them do
    const bool choose = same > need;
    auto is_last = [&](int j, bool in, uint32_t w, uint32_t key) {
      return in && (w >> lane & 1u) == (uint32_t)inner && key == last && need > 0;
    };
    int ties = 0;
    if (choose) {
      n = 0;
      for (int j = j_first; j < j_end; j += 32) {
        const bool in = j + lane < j_end;
        const uint32_t w = word_of(j, in);
        n += __popc(__ballot_sync(0xFFFFFFFFu, is_last(j, in, w, in ? key_of(j + lane) : 0u)));
      }
      int total;
      ties = __shfl_sync(0xFFFFFFFFu, sum_before(lane == 0 ? n : 0, room, total), 0);
    }
    int free = 0, move = 0;
    for (int j = j_first; j < j_end; j += 32) {
      const bool in = j + lane < j_end;
      const uint32_t w = word_of(j, in), key = in ? key_of(j + lane) : 0u;
      const bool safe = w >> lane & 1u, tie = is_last(j, in, w, key);
      const uint32_t tied = __ballot_sync(0xFFFFFFFFu, tie);
      bool stays = in && (safe == inner ? key > last : safe);
      if (tie) stays = !choose || ties + __popc(tied & ((1u << lane) - 1u)) < need;
      ties += __popc(tied);
      const uint32_t s = __ballot_sync(0xFFFFFFFFu, stays);
      if (lane == 0) stay[j >> 5] = s;
      const uint32_t low = bits_below(j, keep), here = bits_below(j, j_end);
      free += __popc(~s & low & here);
      move += __popc(s & ~low);
    }
    int total;
    int at_free = __shfl_sync(0xFFFFFFFFu, sum_before(lane == 0 ? free : 0, room, total), 0);
    int at_move = __shfl_sync(0xFFFFFFFFu, sum_before(lane == 0 ? move : 0, room, moves), 0);
    for (int j = j_first; j < j_end; j += 32) {
      const uint32_t s = stay[j >> 5], low = bits_below(j, keep), below = (1u << lane) - 1u;
      const uint32_t f = ~s & low & bits_below(j, j_end), m = s & ~low;
      if (f >> lane & 1u) to[at_free + __popc(f & below)] = j + lane;
      if (m >> lane & 1u) from[at_move + __popc(m & below)] = j + lane;
      if (weight_out != weight && (s & low) >> lane & 1u) weight_out[j + lane] = weight[j + lane];
      if (born_out != born && (s & low) >> lane & 1u) born_out[j + lane] = born[j + lane];
      at_free += __popc(f);
      at_move += __popc(m);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moves; i += kSelect) {
      const int d = to[i], s = from[i];
      weight_out[d] = weight[s];
      if (born) born_out[d] = born[s];
    }
    __syncthreads();  // where the results lie on the operands: read before they are cleared
  } else {
    for (int j = threadIdx.x; j < len; j += kSelect) {
      if (weight_out != weight) weight_out[j] = weight[j];
      if (born_out != born) born_out[j] = born[j];
    }
  }
  for (int j = left + threadIdx.x; j < cap; j += kSelect) {
    weight_out[j] = 0.f;
    if (born) born_out[j] = 0;
  }
  if (threadIdx.x == 0) a.moves[unit] = moves;
}

// Rows of the pairs, 16 bytes a lane, K and V; the new lengths.  The lengths may lie on the old ones: nothing reads
// an item's but the thread that writes it.
constexpr int kMoveWarps = 4;
__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  const int part = blockIdx.x % a.parts;
  const long long unit = blockIdx.x / a.parts;
  const int b = (int)(unit / a.Hkv), h = (int)(unit - (long long)b * a.Hkv);
  if (h == 0 && part == 0 && threadIdx.x == 0) a.after[b] = min(a.pages.clamp(a.lens[b]), a.budget(b));
  const int moves = a.moves[unit], lanes = a.row_bytes / 16, at_once = 32 / lanes;
  const long long c = (long long)h * a.row_bytes + lane_id() % lanes * 16;
  const int *to = a.to + unit * a.half, *from = a.from + unit * a.half;
  for (int i = (part * kMoveWarps + (int)warp_id()) * at_once + (int)lane_id() / lanes; i < moves;
       i += a.parts * kMoveWarps * at_once) {
    uint32_t dr, sr;
    const long long d = a.pages.entry(b, (uint32_t)to[i], dr), s = a.pages.entry(b, (uint32_t)from[i], sr);
    if (!a.pages.has((int)d) || !a.pages.has((int)s)) continue;
    const uint4 k = *reinterpret_cast<const uint4*>(a.k.p + s * a.k.page + sr * a.k.row + c);
    const uint4 v = *reinterpret_cast<const uint4*>(a.v.p + s * a.v.page + sr * a.v.row + c);
    *reinterpret_cast<uint4*>(a.k.p + d * a.k.page + dr * a.k.row + c) = k;
    *reinterpret_cast<uint4*>(a.v.p + d * a.v.page + dr * a.v.row + c) = v;
  }
}

struct EvictPlan {
  int half, words;
  bool held;
  long long lists, moves, bits;  // ints
  long long bytes() const { return (lists + moves + bits) * 4; }
};
EvictPlan evict_plan(int B, int Hkv, int cap) {
  const long long units = (long long)B * Hkv;
  EvictPlan p{};
  p.half = std::max(1, cap / 2);  // at most min(keep, len - keep) states move
  p.words = (cap + 31) / 32;
  p.held = select_bytes(cap) <= kSelectRoom;
  p.lists = 2 * units * p.half;
  p.moves = units;
  p.bits = p.held ? 0 : units * p.words;
  return p;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_paged_write(const void* k, long long k_row, long long k_img, const void* v, long long v_row, long long v_img,
                              int dtype, void* k_pages, long long kp_row, long long kp_page, void* v_pages,
                              long long vp_row, long long vp_page, int page_dtype, int P, int page, const int* table,
                              long long table_row, int N, const int* at, const int* count, int B, int T, int Hkv, int dh,
                              float k_scale, float v_scale, float* weight, int* born, const int* stamp,
                              long long stamp_img, long long stamp_row, int* after, void* stream) {
  if (!paged_sizes_ok(B, Hkv, dh, P, page, N) || T < 0 || T >= (1 << 30) || (dtype != SB_F16 && dtype != SB_BF16) ||
      (page_dtype != dtype && page_dtype != SB_F8))
    return record_error(SB_EINVAL, "sb_paged_write: sizes (dh 32, 64 or 128) or dtypes");
  if (!(k_scale > 0.f) || !std::isfinite(k_scale) || !(v_scale > 0.f) || !std::isfinite(v_scale) ||
      (page_dtype != SB_F8 && (k_scale != 1.f || v_scale != 1.f)))
    return record_error(SB_EINVAL, "sb_paged_write: scales, or scales of pages that are not e4m3");
  if (B == 0) return SB_OK;
  const int es = page_dtype_bytes(page_dtype);
  const bool some = T > 0 && P > 0 && N > 0;
  if (!at || !after || (N > 0 && (!table || table_row < 0)) ||
      (some && (!k || !v || k_row < 0 || k_img < 0 || v_row < 0 || v_img < 0 || !pool_ok(k_pages, kp_row, kp_page, es) ||
                !pool_ok(v_pages, vp_row, vp_page, es))))
    return record_error(SB_EINVAL, "sb_paged_write: rows (pools 16-byte aligned, strides multiples of 16 bytes) or null argument");
  WriteArgs a{};
  a.k = k; a.k_row = k_row; a.k_img = k_img;
  a.v = v; a.v_row = v_row; a.v_img = v_img;
  a.dt = dtype;
  a.kp = pool_of(k_pages, kp_row, kp_page, es);
  a.vp = pool_of(v_pages, vp_row, vp_page, es);
  a.pages = page_table(table, table_row, P, page, N);
  a.at = at; a.count = count; a.stamp = stamp; a.stamp_img = stamp_img; a.stamp_row = stamp_row;
  a.B = B; a.T = T; a.Hkv = Hkv;
  a.k_scale = k_scale; a.v_scale = v_scale;
  a.weight = weight; a.born = born; a.after = after;
  const int vecs = Hkv * dh * es / 16;
  a.vecs = fast_div((uint32_t)vecs);
  a.group = std::min(32, std::max(1, 128 / vecs));
  a.rows = some ? (long long)B * T : 0;
  const long long warps = (a.rows + a.group - 1) / a.group;
  a.row_blocks = (warps + kWriteWarps - 1) / kWriteWarps;
  a.marks = B + (T > 0 && N > 0 && (weight || born) ? (long long)B * Hkv * T : 0);
  const long long blocks = a.row_blocks + (a.marks + kWriteWarps * 32 - 1) / (kWriteWarps * 32);
  if (blocks > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_paged_write: too many rows");
  auto aligned = [](const void* p, long long row, long long img) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row % 8 == 0 && img % 8 == 0;
  };
  const bool vec = aligned(k, k_row, k_img) && aligned(v, v_row, v_img);
  auto kernel = page_dtype == SB_F8 ? (vec ? paged_write_kernel<true, true> : paged_write_kernel<true, false>)
                                    : (vec ? paged_write_kernel<false, true> : paged_write_kernel<false, false>);
  kernel<<<(unsigned)blocks, kWriteWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}

extern "C" int sb_paged_evict_work(int B, int Hkv, int page, int N, long long* bytes) {
  if (!bytes || !paged_sizes_ok(B, Hkv, 32, 0, page, N)) return record_error(SB_EINVAL, "sb_paged_evict_work: arguments");
  *bytes = B == 0 ? 0 : evict_plan(B, Hkv, N * page).bytes();
  return SB_OK;
}

extern "C" int sb_paged_evict(void* k_pages, long long k_row, long long k_page, void* v_pages, long long v_row,
                              long long v_page, int page_dtype, int P, int page, const int* table, long long table_row, int N,
                              const int* lens, const int* keep, int keep_all, const int* since, int B, int Hkv, int dh,
                              const float* weight, const int* born, float* weight_out, int* born_out, int* after, void* work,
                              long long work_bytes, void* stream) {
  if (!paged_sizes_ok(B, Hkv, dh, P, page, N) || !page_dtype_ok(page_dtype))
    return record_error(SB_EINVAL, "sb_paged_evict: sizes (dh 32, 64 or 128) or dtype");
  if (B == 0) return SB_OK;
  const int es = page_dtype_bytes(page_dtype);
  if (!lens || !after || (N > 0 && (!table || table_row < 0 || !weight || !weight_out)) || (since && !born) || (!born) != (!born_out) ||
      (P > 0 && N > 0 && (!pool_ok(k_pages, k_row, k_page, es) || !pool_ok(v_pages, v_row, v_page, es))))
    return record_error(SB_EINVAL, "sb_paged_evict: rows (16-byte aligned, strides multiples of 16 bytes) or null argument");
  const EvictPlan p = evict_plan(B, Hkv, N * page);
  if (!work || work_bytes < p.bytes() || (reinterpret_cast<uintptr_t>(work) & 15) != 0)
    return record_error(SB_EINVAL, "sb_paged_evict: workspace (sb_paged_evict_work bytes, 16-byte aligned)");
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_evict: device");
  EvictArgs a{};
  a.k = pool_of(k_pages, k_row, k_page, es);
  a.v = pool_of(v_pages, v_row, v_page, es);
  a.pages = page_table(table, table_row, P, page, N);
  a.lens = lens; a.keep = keep; a.keep_all = keep_all; a.since = since;
  a.weight = weight; a.weight_out = weight_out; a.born = born; a.born_out = born_out; a.after = after;
  a.B = B; a.Hkv = Hkv; a.row_bytes = dh * es; a.half = p.half;
  const long long units = (long long)B * Hkv;
  // about eight CTAs an SM over the units, each with at least one round of pairs in the worst case
  const int round = kMoveWarps * (32 / (a.row_bytes / 16));
  a.parts = (int)std::max(1ll, std::min((8ll * sms + units - 1) / units, ((long long)p.half + round - 1) / round));
  if (units * a.parts > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_paged_evict: too many items");
  a.to = static_cast<int*>(work);
  a.from = a.to + units * p.half;
  a.moves = a.from + units * p.half;
  a.bits = reinterpret_cast<uint32_t*>(a.moves + units);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (p.held) {
    static bool ready[64];
    e = xattn_smem(reinterpret_cast<const void*>(&evict_select_kernel<true>), kSelectRoom, ready);
    if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
    evict_select_kernel<true><<<(unsigned)units, kSelect, (size_t)select_bytes(N * page), st>>>(a);
  } else {
    evict_select_kernel<false><<<(unsigned)units, kSelect, 0, st>>>(a);
  }
  e = cudaGetLastError();
  if (e == cudaSuccess) {
    evict_move_kernel<<<(unsigned)(units * a.parts), kMoveWarps * 32, 0, st>>>(a);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}
