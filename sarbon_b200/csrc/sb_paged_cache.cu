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
// in flight: 16 x 2040 ragged rows of 8 x 128 channels of K and of V in bf16 37 us, 224 MB, 93 % of the copy rate; 8 x
// 8160 of 8 x 64 from fp16 to e4m3 35.5 us, 205 MB, 88 % (57 with divisions).  e4m3 pages get the code of x / scale, a true division, or
// where both scales are powers of two the product with their reciprocals, which is the quotient.
struct WriteArgs {
  const void *k, *v;
  long long k_row, k_img, v_row, v_img;  // elements
  Pool kp, vp;
  PageTable pages;
  const int *at, *count, *stamp;
  long long stamp_img, stamp_row;
  int B, T, Hkv;
  float k_scale, v_scale;
  float* weight;
  int *born, *after;
  FastDiv vecs;  // vectors of eight elements a row
  int group;     // rows a warp
  long long rows, row_blocks, marks;  // marks: what else is written, one a thread
  SB_DEV int start(int b) const { return pages.clamp(at[b]); }
  SB_DEV int fresh(int b) const { return count ? min(max(count[b], 0), T) : T; }
};

constexpr int kWriteWarps = 8;

// Eight elements as a pool holds them.  MODE 0: as they are; 1: e4m3 of x * scale; 2: e4m3 of x / scale
template <int MODE, bool BF16>
SB_DEV void put_vec(uint64_t to, const uint4& r, float scale) {
  if constexpr (MODE == 0) {
    *reinterpret_cast<uint4*>(to) = r;
  } else {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float2 f = pair_of(w[u], BF16 ? SB_BF16 : SB_F16);
      c[u] = MODE == 1 ? e4m3x2_of(f.x * scale, f.y * scale) : e4m3x2_of(__fdiv_rn(f.x, scale), __fdiv_rn(f.y, scale));
    }
    *reinterpret_cast<uint2*>(to) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
  }
}
// Eight 16-bit elements from element i on.
template <bool ALIGNED>
SB_DEV uint4 load_vec(const void* p, long long i) {
  const uint16_t* q = static_cast<const uint16_t*>(p) + i;
  if constexpr (ALIGNED) {
    return *reinterpret_cast<const uint4*>(q);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = (uint32_t)q[2 * u] | (uint32_t)q[2 * u + 1] << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int MODE, bool ALIGNED, bool BF16>
__global__ void __launch_bounds__(kWriteWarps * 32, MODE == 2 ? 2 : 4)
    paged_write_kernel(const __grid_constant__ WriteArgs a) {
  constexpr int kAhead = 4, bytes = MODE ? 8 : 16;  // vectors of K and V at once, bytes of one in the pool
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
  for (int i0 = lane; i0 < total; i0 += 32 * kAhead) {
    uint4 k[kAhead], v[kAhead];
    ulonglong2 where[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      const int i = i0 + 32 * x;
      where[x] = make_ulonglong2(0, 0);
      if (i < total) {
        const int r = (int)a.vecs.div((uint32_t)i), c = i - r * (int)a.vecs.d;
        where[x] = to[warp][r];
        if (where[x].x) {
          where[x].x += c * bytes;
          where[x].y += c * bytes;
          const longlong2 s = from[warp][r];
          k[x] = load_vec<ALIGNED>(a.k, s.x + c * 8);
          v[x] = load_vec<ALIGNED>(a.v, s.y + c * 8);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kAhead; ++x)
      if (where[x].x) {
        put_vec<MODE, BF16>(where[x].x, k[x], a.k_scale);
        put_vec<MODE, BF16>(where[x].y, v[x], a.v_scale);
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
//
// What bounds it: the chain of passes, each with an exchange of counts.  16 x 8 units of 18,360 states, 2040 of them to
// go, rows of 256 bytes: 24 us for the selection, 13.5 for the rows (82 MB, 93 % of the copy rate); 2 x 8 of 130,560, half
// of them, rows of 64 bytes: 34.7 and 40 (150 MB in pieces of 64 bytes: 58 %).  Each pass looks at all keys again, though after
// the first only one bin's matter, and a few hundred places take the bins and barriers of many: 8.8 us for 241.  At 64
// registers (two CTAs an SM) the selection spills 100 bytes a thread, as many with four stamps' loads at once as with nine.
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
  int B, Hkv, row_bytes, half, parts, ctas;  // parts: CTAs a unit of the second kernel; 0: none, the first does it all
  int *to, *from, *moves;  // workspace: [units][half], [units][half], [units]
  uint32_t* bits;          // [units][2][cap / 32]: states that are protected, that stay, where shared memory has no room
  SB_DEV int budget(int b) const { return pages.clamp(keep ? keep[b] : keep_all); }
};

constexpr int kSelect = 512, kSelectWarps = kSelect / 32, kBins = 2048, kMostCtas = 8;

// Integers in the order of the weights; NaN is the least, both zeros are one.
SB_DEV uint32_t ordered(float w) {
  if (w != w) return 0u;
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// A pass's bits of a key, and those of the passes before it.
SB_DEV int bin_of(uint32_t key, int pass) { return pass == 0 ? key >> 21 : pass == 1 ? key >> 10 & 2047u : key & 1023u; }
SB_DEV uint32_t prefix_of(uint32_t key, int pass) {
  return pass == 0 ? 0u : pass == 1 ? key & 0xFFE00000u : key & 0xFFFFFC00u;
}
SB_DEV uint32_t as_prefix(int bin, int pass) { return (uint32_t)bin << (pass == 0 ? 21 : pass == 1 ? 10 : 0); }

// What the CTAs of an (item, key head) tell each other; bins and counts are never written twice.
struct Told {
  int bins[4][kBins];  // the first pass's of the protected and of the others, the second's, the third's
  int groups[4][kBins / 32];  // their sums by 32
  int counts[3][2];
  int room[2][kSelectWarps], found[3];
};
SB_DEV void all_sync(int ctas) {
  __syncwarp();
  if (ctas > 1) cluster_sync();
  else __syncthreads();
}

// Sums of two numbers over the threads before this one and over all of the CTA.
SB_DEV void before_and_all(int (&v)[2], int (&total)[2], Told& told) {
  const int lane = lane_id(), warp = warp_id();
  int s[2] = {v[0], v[1]};
#pragma unroll
  for (int x = 1; x < 32; x <<= 1)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, s[y], x);
      if (lane >= x) s[y] += u;
    }
  __syncthreads();
  if (lane == 31) {
    told.room[0][warp] = s[0];
    told.room[1][warp] = s[1];
  }
  __syncthreads();
#pragma unroll
  for (int y = 0; y < 2; ++y) {  // (a lane a warp)
    const int t = lane < kSelectWarps ? told.room[y][lane] : 0;
    v[y] = s[y] - v[y] + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? t : 0);
    total[y] = __reduce_add_sync(0xFFFFFFFFu, t);
  }
}
// The same over all CTAs; the c-th such sum.  base: what the CTAs before this one have.
SB_DEV void before_and_all(int (&v)[2], int (&total)[2], int (&base)[2], Told& told, int c, int ctas, uint32_t rank) {
  before_and_all(v, total, told);
  base[0] = base[1] = 0;
  if (ctas > 1) {
    if (threadIdx.x == 0) {
      told.counts[c][0] = total[0];
      told.counts[c][1] = total[1];
    }
    all_sync(ctas);
    const uint32_t lane = lane_id();
    int t[2] = {0, 0};  // (a lane a CTA: one trip to the others)
    if (lane < (uint32_t)ctas) {
      t[0] = (int)peer_word(&told.counts[c][0], lane);
      t[1] = (int)peer_word(&told.counts[c][1], lane);
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      base[y] = __reduce_add_sync(0xFFFFFFFFu, lane < rank ? t[y] : 0);
      total[y] = __reduce_add_sync(0xFFFFFFFFu, t[y]);
      v[y] += base[y];
    }
  }
}

// Inclusive sums over lanes of `width`, in order.
SB_DEV int scan_of(int v, int width) {
  for (int x = 1; x < width; x <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, x, width);
    if ((lane_id() & (width - 1)) >= x) v += u;
  }
  return v;
}
// Where among four numbers a lane, of which `above` lie before, the need-th is: x, what lies before it and it; -1: not here.
struct Found {
  int x, above, same;
};
SB_DEV Found find_in(const int (&c)[4], int above, int need) {
  Found f{-1, 0, 0};
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (above < need && need <= above + c[x]) f = {x, above, c[x]};
    above += c[x];
  }
  return f;
}

// What the CTAs of a cluster tell: the sums of their bins by 32.
SB_DEV void tell_groups(Told& told, int which) {
  const uint4 u = reinterpret_cast<const uint4*>(told.bins[which])[threadIdx.x];
  int sum = (int)(u.x + u.y + u.z + u.w);
#pragma unroll
  for (int x = 1; x < 8; x <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
  if (lane_id() % 8 == 0) told.groups[which][threadIdx.x / 8] = sum;
}

// After a pass over a CTA's states.
SB_DEV void counted(Told& told, int which, int ctas) {
  if (ctas > 1) {
    __syncthreads();
    tell_groups(told, which);
  }
  all_sync(ctas);
}

// The bin of all CTAs' bins, which they have told, that holds the need-th number from the top; need becomes its place in
// the bin, same how many the bin holds.  In a cluster one warp looks at the groups of all CTAs and then at the bins
// of one group (for eight CTAs 0.9 us, where all threads looked at all bins 2.7).
SB_DEV int find_bin(Told& told, int which, int& need, int& same, int ctas) {
  static_assert(kBins == 4 * kSelect && kBins / 32 == 64, "four bins a thread, four groups a lane of 16");
  const int lane = lane_id(), warp = warp_id();
  auto add = [](int (&c)[4], const uint4& u) {  // from the top
    c[0] += (int)u.w;
    c[1] += (int)u.z;
    c[2] += (int)u.y;
    c[3] += (int)u.x;
  };
  int c[4] = {0, 0, 0, 0};
  if (ctas > 1) {
    if (warp == 0) {
#pragma unroll
      for (int r = 0; r < kMostCtas; r += 2)
        if (r + lane / 16 < ctas) add(c, peer_words(&told.groups[which][60 - lane % 16 * 4], (uint32_t)(r + lane / 16)));
#pragma unroll
      for (int x = 0; x < 4; ++x) c[x] += __shfl_xor_sync(0xFFFFFFFFu, c[x], 16);
      int sum = c[0] + c[1] + c[2] + c[3];
      const Found g = find_in(c, scan_of(sum, 16) - sum, need);
      const int holds = max(__ffs(__ballot_sync(0xFFFFFFFFu, g.x >= 0)) - 1, 0);
      const int group = 63 - __shfl_sync(0xFFFFFFFFu, lane % 16 * 4 + g.x, holds), above = __shfl_sync(0xFFFFFFFFu, g.above, holds);
      const int first = group * 32 + 28 - lane % 8 * 4;
      c[0] = c[1] = c[2] = c[3] = 0;
#pragma unroll
      for (int r = 0; r < kMostCtas; r += 4)
        if (r + lane / 8 < ctas) add(c, peer_words(&told.bins[which][first], (uint32_t)(r + lane / 8)));
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        c[x] += __shfl_xor_sync(0xFFFFFFFFu, c[x], 8);
        c[x] += __shfl_xor_sync(0xFFFFFFFFu, c[x], 16);
      }
      sum = c[0] + c[1] + c[2] + c[3];
      const Found f = find_in(c, above + scan_of(sum, 8) - sum, need);
      if (lane < 8 && f.x >= 0) {
        told.found[0] = first + 3 - f.x;
        told.found[1] = f.above;
        told.found[2] = f.same;
      }
    }
  } else {
    const int first = kBins - 4 * (1 + (int)threadIdx.x);
    add(c, *reinterpret_cast<const uint4*>(&told.bins[which][first]));
    const int sum = c[0] + c[1] + c[2] + c[3], of_warp = __reduce_add_sync(0xFFFFFFFFu, sum);
    if (lane == 0) told.room[0][warp] = of_warp;  // (all_sync came after what it held before was read)
    __syncthreads();
    // every warp finds the warp whose bins hold it, and that warp the bin
    const int t = lane < kSelectWarps ? told.room[0][lane] : 0, upto = scan_of(t, 32);
    const uint32_t holds = __ballot_sync(0xFFFFFFFFu, upto - t < need && need <= upto);
    const int above = __shfl_sync(0xFFFFFFFFu, upto - t, max(__ffs(holds) - 1, 0));
    if (holds >> warp & 1u) {
      const Found f = find_in(c, above + scan_of(sum, 32) - sum, need);
      if (f.x >= 0) {
        told.found[0] = first + 3 - f.x;
        told.found[1] = f.above;
        told.found[2] = f.same;
      }
    }
  }
  __syncthreads();
  need -= told.found[1];
  same = told.found[2];
  return told.found[0];
}

// An item within its budget stays as it is.  Places from the new length on are cleared here where the results lie in
// memory of their own; where they lie on the operands, those of states that go are, and the second
// kernel clears those of states that move once it has read them.
SB_DEV void keep_all_of(const EvictArgs& a, long long at, int len, int ctas, uint32_t rank) {
  for (int j = (int)rank * kSelect + (int)threadIdx.x; j < len; j += ctas * kSelect) {
    if (a.weight_out != a.weight) a.weight_out[at + j] = a.weight[at + j];
    if (a.born_out != a.born) a.born_out[at + j] = a.born[at + j];
  }
}
SB_DEV void finish(const EvictArgs& a, long long unit, int moves, int len, int left, int ctas, uint32_t rank) {
  const long long at = unit * a.pages.cap;
  const int w_from = a.weight_out != a.weight ? left : len, b_from = a.born_out != a.born ? left : len;
  for (int j = left + (int)rank * kSelect + (int)threadIdx.x; j < a.pages.cap; j += ctas * kSelect) {
    if (j >= w_from) a.weight_out[at + j] = 0.f;
    if (a.born && j >= b_from) a.born_out[at + j] = 0;
  }
  if (a.parts && threadIdx.x == 0 && rank == 0) a.moves[unit] = moves;
  if (ctas > 1) all_sync(ctas);  // no CTA ends while another reads what it told
}
// A state that goes from its place, which nothing fills.
SB_DEV void clear_own(const EvictArgs& a, long long at) {
  if (a.weight_out == a.weight) a.weight_out[at] = 0.f;
  if (a.born && a.born_out == a.born) a.born_out[at] = 0;
}

// Rows, weights and stamps of the pairs: a warp takes 32 of them from i0 on, then those `stride` on; a lane looks up where
// a pair's rows lie, then all copy them, 16 bytes a lane, four loads of K and four of V in flight.
constexpr int kMoveWarps = 4, kMoveAhead = 4;
struct Pairs {
  ulonglong2 source[32], target[32];  // addresses of K and V; 0: nowhere
};
template <int LANES>
SB_DEV void move_pairs(const EvictArgs& a, long long unit, const int* to, const int* from, int moves, int i0, int stride,
                       Pairs& pairs) {
  constexpr int AT_ONCE = 32 / LANES;
  const int lane = lane_id(), b = (int)(unit / a.Hkv), h = (int)(unit - (long long)b * a.Hkv);
  const long long c = (long long)h * a.row_bytes + lane % LANES * 16, at = unit * a.pages.cap;
  // a lane's pair: its places, the pages and rows they are on, weight and stamp; asked for two rounds and one ahead
  int d = -1, s = 0, dp = -1, sp = -1, r = 0;
  uint32_t dr = 0, sr = 0;
  float w = 0.f;
  auto places = [&](int i) {
    d = i < moves ? to[i] : -1;
    s = d < 0 ? 0 : from[i];
  };
  auto look_up = [&] {
    if (d >= 0) {
      dp = a.pages.entry(b, (uint32_t)d, dr);
      sp = a.pages.entry(b, (uint32_t)s, sr);
      w = a.weight[at + s];
      if (a.born) r = a.born[at + s];
    }
  };
  places(i0 + lane);
  look_up();
  int d_now = d, s_now = s;
  places(i0 + stride + lane);
  for (; i0 < moves; i0 += stride) {
    ulonglong2 p = make_ulonglong2(0, 0), q = p;
    if (d_now >= 0) {
      if (a.pages.has(dp) && a.pages.has(sp)) {
        p = make_ulonglong2(a.k.row_at(sp, sr), a.v.row_at(sp, sr));
        q = make_ulonglong2(a.k.row_at(dp, dr), a.v.row_at(dp, dr));
      }
      a.weight_out[at + d_now] = w;
      if (a.born) a.born_out[at + d_now] = r;
      clear_own(a, at + s_now);
    }
    __syncwarp();
    pairs.source[lane] = p;
    pairs.target[lane] = q;
    __syncwarp();
    look_up();
    d_now = d;
    s_now = s;
    places(i0 + 2 * stride + lane);
#pragma unroll
    for (int x0 = 0; x0 < LANES; x0 += kMoveAhead) {
      if (i0 + x0 * AT_ONCE >= moves) break;
      uint4 k[kMoveAhead], v[kMoveAhead];
#pragma unroll
      for (int x = 0; x < kMoveAhead; ++x)
        if (x0 + x < LANES) {
          const ulonglong2 from_row = pairs.source[(x0 + x) * AT_ONCE + lane / LANES];
          if (from_row.x) {
            k[x] = *reinterpret_cast<const uint4*>(from_row.x + c);
            v[x] = *reinterpret_cast<const uint4*>(from_row.y + c);
          }
        }
#pragma unroll
      for (int x = 0; x < kMoveAhead; ++x)
        if (x0 + x < LANES) {
          const ulonglong2 to_row = pairs.target[(x0 + x) * AT_ONCE + lane / LANES];
          if (to_row.x) {
            *reinterpret_cast<uint4*>(to_row.x + c) = k[x];
            *reinterpret_cast<uint4*>(to_row.y + c) = v[x];
          }
        }
    }
  }
}

// To shared memory, asynchronously: `bytes` of 16, zeros behind them; 0: a word.
SB_DEV void copy_in(const void* to, const void* from, int bytes) {
  if (bytes)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
SB_DEV void copies_in() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Selection with the CTA's ordered weights in shared memory: a thread has a run of states, an odd number of fours, so that
// neighbours' 16-byte reads fall in distinct banks, and their bits (protected, staying) in registers; no pass
// needs a word with another thread but the counts.  (1024 threads, one CTA an SM, took half as long again for clusters of
// eight: not all of them find their SMs at once.)
constexpr int kMostFours = 15, kFoursOfTwo = 9;  // states a thread: 60; up to 36 (109 KB of shared memory) two CTAs an SM
inline int held_fours(int cap, int ctas) { return ((cap + ctas * kSelect * 4 - 1) / (ctas * kSelect * 4)) | 1; }
inline int held_bytes(int fours) { return kSelect * 4 * fours * 4 + kSelect * fours; }
// A memory of up to this many places is evicted from by one kernel: at most half of them move, 1 MB a CTA.
constexpr int kFewPlaces = 4096;
static_assert(sizeof(Told) >= kSelectWarps * sizeof(Pairs), "room for the pairs");

__global__ void __launch_bounds__(kSelect, 2) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ __align__(16) uint32_t held[];  // weights of the CTA's states, then bits of the protected ones, a byte four
  __shared__ __align__(16) Told told;
  const int warp = warp_id(), lane = lane_id(), ctas = a.ctas;
  const uint32_t rank = ctas > 1 ? cluster_ctarank() : 0u;
  const long long unit = blockIdx.x / ctas, at = unit * a.pages.cap;
  const int b = (int)(unit / a.Hkv);
  const int len = a.pages.clamp(a.lens[b]), keep = a.budget(b);
  int moves = 0;
  if (len <= keep) {
    keep_all_of(a, at, len, ctas, rank);
  } else {
    const bool guard = a.born && a.since;
    const int since = guard ? a.since[b] : 0;
    const int fours = ((len + ctas * kSelect * 4 - 1) / (ctas * kSelect * 4)) | 1, run = fours * 4, mine = kSelect * run;
    const int j_cta = (int)rank * mine, here = min(max(len - j_cta, 0), mine);  // the CTA's states
    uint8_t* const nibbles = reinterpret_cast<uint8_t*>(held + mine);
    // weights arrive in shared memory by themselves, sixteen bytes at once where they lie so, while stamps are looked at
    const float* const from_w = a.weight + at + j_cta;
    float* const to_w = a.weight_out + at + j_cta;
    const int* const from_b = a.born + at + j_cta;
    int* const to_b = a.born_out + at + j_cta;
    const bool copied = a.weight_out != a.weight, copied_b = a.born_out != a.born;
    const uintptr_t all_at = reinterpret_cast<uintptr_t>(from_w) | reinterpret_cast<uintptr_t>(to_w) |
                             (a.born ? reinterpret_cast<uintptr_t>(from_b) | reinterpret_cast<uintptr_t>(to_b) : 0);
    const bool wide = (all_at & 15) == 0;
    const int step = wide ? 4 : 1, kept = min(keep - j_cta, here);  // as if all of those below keep stayed
    for (int j = (int)threadIdx.x * step; j < here; j += kSelect * step) copy_in(held + j, from_w + j, wide ? min(16, (here - j) * 4) : 0);
    for (int x = threadIdx.x; x < kBins; x += kSelect) reinterpret_cast<uint4*>(told.bins)[x] = make_uint4(0, 0, 0, 0);
    if (!a.born) {
      for (int x = threadIdx.x; x * 16 < here; x += kSelect) reinterpret_cast<uint32_t*>(nibbles)[x] = 0;
    } else if (wide) {
      constexpr int kAtOnce = kFoursOfTwo;
      for (int j0 = (int)threadIdx.x * 4; j0 < here; j0 += kAtOnce * kSelect * 4) {
        int4 s[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
          const int j = j0 + x * kSelect * 4;
          s[x] = make_int4(0, 0, 0, 0);
          if (j + 3 < here) {
            s[x] = *reinterpret_cast<const int4*>(from_b + j);
          } else if (j < here) {
            s[x].x = from_b[j];
            if (j + 1 < here) s[x].y = from_b[j + 1];
            if (j + 2 < here) s[x].z = from_b[j + 2];
          }
        }
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
          const int j = j0 + x * kSelect * 4;
          if (j >= here) break;
          const int low = copied_b ? kept - j : 0;
          nibbles[j >> 2] = guard ? (s[x].x >= since) | (s[x].y >= since) << 1 | (s[x].z >= since) << 2 | (s[x].w >= since) << 3 : 0;
          if (low >= 4) {
            *reinterpret_cast<int4*>(to_b + j) = s[x];
          } else {
            if (low > 0) to_b[j] = s[x].x;
            if (low > 1) to_b[j + 1] = s[x].y;
            if (low > 2) to_b[j + 2] = s[x].z;
          }
        }
      }
    } else {
      constexpr int kAtOnce = 8;
      for (int j0 = warp * 32; j0 < here; j0 += kAtOnce * kSelect) {
        int s[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
          const int j = j0 + x * kSelect + lane;
          s[x] = j < here ? from_b[j] : 0;
        }
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
          const int j = j0 + x * kSelect + lane;
          if (j0 + x * kSelect >= here) break;
          const uint32_t word = __ballot_sync(0xFFFFFFFFu, guard && s[x] >= since);
          if (lane % 4 == 0) nibbles[j >> 2] = word >> lane & 15u;
          if (copied_b && j < kept) to_b[j] = s[x];
        }
      }
    }
    copies_in();
    for (int j = (int)threadIdx.x * step; j < here; j += kSelect * step) {  // what this thread has copied
      const int low = copied ? kept - j : 0;
      if (wide) {
        uint4 u = *reinterpret_cast<const uint4*>(held + j);
        if (low >= 4) {
          *reinterpret_cast<uint4*>(to_w + j) = u;
        } else {
          if (low > 0) to_w[j] = __uint_as_float(u.x);
          if (low > 1) to_w[j + 1] = __uint_as_float(u.y);
          if (low > 2) to_w[j + 2] = __uint_as_float(u.z);
        }
        u = make_uint4(ordered(__uint_as_float(u.x)), ordered(__uint_as_float(u.y)), ordered(__uint_as_float(u.z)),
                       ordered(__uint_as_float(u.w)));
        *reinterpret_cast<uint4*>(held + j) = u;
      } else {
        const float f = __uint_as_float(held[j]);
        if (low > 0) to_w[j] = f;
        held[j] = ordered(f);
      }
    }
    __syncthreads();
    // this thread's run, its protected states, and those of all
    const int j_run = (int)threadIdx.x * run, states = min(max(here - j_run, 0), run), my_fours = (states + 3) / 4;
    const uint64_t valid = states > 0 ? ~0ull >> (64 - states) : 0ull;
    uint64_t safe = 0;
    for (int i = 0; i < my_fours; ++i) safe |= (uint64_t)nibbles[(j_run >> 2) + i] << (4 * i);
    safe &= valid;
    const int n = __reduce_add_sync(0xFFFFFFFFu, __popcll(safe));
    if (lane == 0) told.room[1][warp] = n;
    const uint4* const keys = reinterpret_cast<const uint4*>(held + j_run);
    {  // the first pass for both classes, before it is known which of them weights decide among
      // (many states may have one weight, new ones 0: runs of a bin are counted before they are added)
      int bin = -1, count = 0;
      for (int i = 0; i < my_fours; ++i) {
        const uint4 k = keys[i];
        const uint32_t key[4] = {k.x, k.y, k.z, k.w}, is = (uint32_t)(valid >> (4 * i)), other = (uint32_t)(~safe >> (4 * i));
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (is >> y & 1u) {
            const int x = bin_of(key[y], 0) + (other >> y & 1u ? kBins : 0);
            if (x != bin) {
              if (count) atomicAdd(&told.bins[0][bin], count);
              bin = x;
              count = 0;
            }
            ++count;
          }
      }
      if (count) atomicAdd(&told.bins[0][bin], count);
    }
    __syncthreads();
    int protect = __reduce_add_sync(0xFFFFFFFFu, lane < kSelectWarps ? told.room[1][lane] : 0);
    if (ctas > 1) {
      if (threadIdx.x == 0) told.counts[0][0] = protect;
      tell_groups(told, 0);
      tell_groups(told, 1);
      all_sync(ctas);
      protect = __reduce_add_sync(0xFFFFFFFFu, lane < ctas ? (int)peer_word(&told.counts[0][0], (uint32_t)lane) : 0);
    }
    // the states among which weights decide: the protected ones where they alone are too many, else the others
    const bool inner = protect >= keep;
    const uint64_t who = inner ? safe : valid & ~safe;
    int need = inner ? keep : keep - protect, same = 0;
    uint32_t last = 0xFFFFFFFFu;  // the ordered weight of the last state that stays; `need` of that weight do
    if (need > 0) {
      last = as_prefix(find_bin(told, inner ? 0 : 1, need, same, ctas), 0);
      for (int pass = 1; pass < 3; ++pass) {
        int bin = -1, count = 0;
        for (int i = 0; i < my_fours; ++i) {
          const uint4 k = keys[i];
          const uint32_t key[4] = {k.x, k.y, k.z, k.w}, nibble = (uint32_t)(who >> (4 * i));
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if ((nibble >> y & 1u) && prefix_of(key[y], pass) == last) {
              const int x = bin_of(key[y], pass);
              if (x != bin) {
                if (count) atomicAdd(&told.bins[1 + pass][bin], count);
                bin = x;
                count = 0;
              }
              ++count;
            }
        }
        if (count) atomicAdd(&told.bins[1 + pass][bin], count);
        counted(told, 1 + pass, ctas);
        last |= as_prefix(find_bin(told, 1 + pass, need, same, ctas), pass);
      }
    }
    uint64_t more = 0, tied = 0;
    for (int i = 0; i < my_fours; ++i) {
      const uint4 k = keys[i];
      const uint32_t key[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        more |= (uint64_t)(key[y] > last) << (4 * i + y);
        tied |= (uint64_t)(key[y] == last) << (4 * i + y);
      }
    }
    more &= who;
    tied &= need > 0 ? who : 0ull;
    if (same > need) {  // more states have the last weight than may stay: the first of them do
      int ties[2] = {__popcll(tied), 0}, total[2], base[2];
      before_and_all(ties, total, base, told, 1, ctas, rank);
      for (int extra = ties[0] + __popcll(tied) - max(need, ties[0]); extra > 0; --extra)
        tied &= ~(1ull << (63 - __clzll(tied)));
    }
    const uint64_t stays = more | tied | (inner ? 0ull : safe);
    const int low_n = min(max(keep - j_cta - j_run, 0), states);  // states of the run below keep
    const uint64_t low = low_n > 0 ? ~0ull >> (64 - low_n) : 0ull;
    uint64_t free = low & ~stays, move = stays & ~low;
    int put[2] = {__popcll(free), __popcll(move)}, total[2], base[2];
    before_and_all(put, total, base, told, 2, ctas, rank);
    moves = total[1];
    // one kernel: the pairs in shared memory, behind the nibbles
    int* const to = a.parts ? a.to + unit * a.half : reinterpret_cast<int*>(held + mine + mine / 16);
    int* const from = a.parts ? a.from + unit * a.half : to + a.half;
    if (a.parts) {
      // through shared memory, over the weights, from both ends, and out in whole lines
      int* const list = reinterpret_cast<int*>(held);
      int f = put[0] - base[0], m = mine - 1 - (put[1] - base[1]);
      for (; free; free &= free - 1) list[f++] = j_cta + j_run + __ffsll(free) - 1;
      for (; move; move &= move - 1) list[m--] = j_cta + j_run + __ffsll(move) - 1;
      if (threadIdx.x == kSelect - 1) {  // how many of each this CTA has
        told.found[0] = f;
        told.found[1] = mine - 1 - m;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < told.found[0]; i += kSelect) to[base[0] + i] = list[i];
      for (int i = threadIdx.x; i < told.found[1]; i += kSelect) from[base[1] + i] = list[mine - 1 - i];
    } else {
      for (; free; free &= free - 1) to[put[0]++] = j_cta + j_run + __ffsll(free) - 1;
      for (; move; move &= move - 1) from[put[1]++] = j_cta + j_run + __ffsll(move) - 1;
    }
    if (a.weight_out == a.weight || (a.born && a.born_out == a.born))
      for (uint64_t gone = valid & ~low & ~stays; gone; gone &= gone - 1)
        clear_own(a, at + j_cta + j_run + __ffsll(gone) - 1);
    if (a.parts == 0) {
      __syncthreads();
      Pairs& pairs = reinterpret_cast<Pairs*>(&told)[warp];  // (the counts are not looked at again)
      if (a.row_bytes == 32) move_pairs<2>(a, unit, to, from, moves, warp * 32, kSelect, pairs);
      else if (a.row_bytes == 64) move_pairs<4>(a, unit, to, from, moves, warp * 32, kSelect, pairs);
      else if (a.row_bytes == 128) move_pairs<8>(a, unit, to, from, moves, warp * 32, kSelect, pairs);
      else move_pairs<16>(a, unit, to, from, moves, warp * 32, kSelect, pairs);
    }
  }
  if (a.parts == 0 && threadIdx.x == 0 && unit % a.Hkv == 0) a.after[b] = min(len, keep);
  finish(a, unit, moves, len, min(len, keep), ctas, rank);
}

// The same for longer ones, from memory: a warp's states lie behind one another, 32 at a time, their bits in memory too.
__global__ void __launch_bounds__(kSelect, 2) evict_select_long_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ __align__(16) Told told;
  const int warp = warp_id(), lane = lane_id(), ctas = a.ctas;
  const uint32_t rank = ctas > 1 ? cluster_ctarank() : 0u;
  const long long unit = blockIdx.x / ctas, at = unit * a.pages.cap;
  const int b = (int)(unit / a.Hkv);
  const int len = a.pages.clamp(a.lens[b]), keep = a.budget(b);
  int moves = 0;
  if (len <= keep) {
    keep_all_of(a, at, len, ctas, rank);
  } else {
    constexpr int kAtOnce = 8;
    const bool guard = a.born && a.since;
    const int since = guard ? a.since[b] : 0;
    const int warps = kSelectWarps * ctas, words = (len + 31) / 32, steps = (words + warps - 1) / warps;
    const int w_first = min(((int)rank * (kSelectWarps) + warp) * steps, words), w_end = min(w_first + steps, words);
    uint32_t* const guarded = a.bits + unit * 2 * ((a.pages.cap + 31) / 32);
    uint32_t* const stay = guarded + (a.pages.cap + 31) / 32;
    auto key_of = [&](int w) { return w < w_end && w * 32 + lane < len ? ordered(a.weight[at + w * 32 + lane]) : 0u; };
    for (int x = threadIdx.x; x < kBins; x += kSelect) reinterpret_cast<uint4*>(told.bins)[x] = make_uint4(0, 0, 0, 0);
    int all[2], n[2] = {0, 0};
    for (int w0 = w_first; w0 < w_end; w0 += kAtOnce) {
      int s[kAtOnce];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) {
        const int j = (w0 + x) * 32 + lane;
        s[x] = a.born && w0 + x < w_end && j < len ? a.born[at + j] : 0;
      }
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) {
        const int j = (w0 + x) * 32 + lane;
        if (w0 + x < w_end) {
          const uint32_t word = __ballot_sync(0xFFFFFFFFu, guard && j < len && s[x] >= since);
          if (lane == 0) {
            guarded[w0 + x] = word;
            n[0] += __popc(word);
          }
          if (j < keep) {  // as if all of these stayed
            if (a.weight_out != a.weight) a.weight_out[at + j] = a.weight[at + j];
            if (a.born_out != a.born) a.born_out[at + j] = s[x];
          }
        }
      }
    }
    int base[2];
    before_and_all(n, all, base, told, 0, ctas, rank);
    const bool inner = all[0] >= keep;
    const uint32_t flip = inner ? 0u : 0xFFFFFFFFu;
    int need = inner ? keep : keep - all[0], same = 0;
    uint32_t last = 0xFFFFFFFFu;
    auto class_of = [&](int w) { return w < w_end ? (guarded[w] ^ flip) & bits_below(w * 32, len) : 0u; };
    if (need > 0) {
      last = 0;
      for (int pass = 0; pass < 3; ++pass) {
        for (int w0 = w_first; w0 < w_end; w0 += kAtOnce) {
          uint32_t key[kAtOnce], who[kAtOnce];
#pragma unroll
          for (int x = 0; x < kAtOnce; ++x) {
            key[x] = key_of(w0 + x);
            who[x] = class_of(w0 + x);
          }
#pragma unroll
          for (int x = 0; x < kAtOnce; ++x) {
            const bool mine = (who[x] >> lane & 1u) && prefix_of(key[x], pass) == last;
            const uint32_t some = __ballot_sync(0xFFFFFFFFu, mine);
            if (some == 0) continue;
            const int bin = bin_of(key[x], pass);
            const int one = __shfl_sync(0xFFFFFFFFu, bin, __ffs(some) - 1);
            if (__all_sync(0xFFFFFFFFu, !mine || bin == one)) {
              if (lane == 0) atomicAdd(&told.bins[pass][one], __popc(some));
            } else if (mine) {
              atomicAdd(&told.bins[pass][bin], 1);
            }
          }
        }
        counted(told, pass, ctas);
        last |= as_prefix(find_bin(told, pass, need, same, ctas), pass);
      }
    }
    const bool some = need > 0, choose = same > need;
    int ties = 0;
    if (choose) {
      int t[2] = {0, 0}, total[2];
      for (int w = w_first; w < w_end; ++w) {
        const uint32_t tied = __ballot_sync(0xFFFFFFFFu, key_of(w) == last) & class_of(w);
        if (lane == 0) t[0] += __popc(tied);
      }
      before_and_all(t, total, base, told, 1, ctas, rank);
      ties = __shfl_sync(0xFFFFFFFFu, t[0], 0);
    }
    int put[2] = {0, 0}, total[2];
    for (int w0 = w_first; w0 < w_end; w0 += kAtOnce) {
      uint32_t key[kAtOnce];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) key[x] = key_of(w0 + x);
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) {
        const int w = w0 + x;
        if (w < w_end) {
          const uint32_t here = bits_below(w * 32, len), low = bits_below(w * 32, keep), who = class_of(w);
          const uint32_t more = __ballot_sync(0xFFFFFFFFu, key[x] > last) & who;
          const uint32_t tied = __ballot_sync(0xFFFFFFFFu, key[x] == last) & (some ? who : 0u);
          uint32_t first = tied;
          if (choose) {
            first = __ballot_sync(0xFFFFFFFFu, (tied >> lane & 1u) && ties + __popc(tied & ((1u << lane) - 1u)) < need);
            ties += __popc(tied);
          }
          const uint32_t stays = more | first | (inner ? 0u : guarded[w] & here);
          if (lane == 0) {
            stay[w] = stays;
            put[0] += __popc(~stays & low & here);
            put[1] += __popc(stays & ~low);
          }
        }
      }
    }
    before_and_all(put, total, base, told, 2, ctas, rank);
    moves = total[1];
    int* const to = a.to + unit * a.half;
    int* const from = a.from + unit * a.half;
    int at_free = __shfl_sync(0xFFFFFFFFu, put[0], 0), at_move = __shfl_sync(0xFFFFFFFFu, put[1], 0);
    for (int w = w_first; w < w_end; ++w) {
      const uint32_t s = stay[w], low = bits_below(w * 32, keep), here = bits_below(w * 32, len), below = (1u << lane) - 1u;
      const uint32_t f = ~s & low & here, m = s & ~low;
      if (f >> lane & 1u) to[at_free + __popc(f & below)] = w * 32 + lane;
      if (m >> lane & 1u) from[at_move + __popc(m & below)] = w * 32 + lane;
      if ((here & ~low & ~s) >> lane & 1u) clear_own(a, at + w * 32 + lane);
      at_free += __popc(f);
      at_move += __popc(m);
    }
  }
  finish(a, unit, moves, len, min(len, keep), ctas, rank);
}

// The pairs of longer memories, and the new lengths, which may lie on the old ones: nothing but the thread that writes
// an item's reads it here.
template <int LANES>
__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ Pairs pairs[kMoveWarps];
  const int part = blockIdx.x % a.parts, warp = warp_id();
  const long long unit = blockIdx.x / a.parts;
  grid_dep_wait();
  if (part == 0 && threadIdx.x == 0 && unit % a.Hkv == 0) {
    const int b = (int)(unit / a.Hkv);
    a.after[b] = min(a.pages.clamp(a.lens[b]), a.budget(b));
  }
  move_pairs<LANES>(a, unit, a.to + unit * a.half, a.from + unit * a.half, a.moves[unit], (part * kMoveWarps + warp) * 32,
                    a.parts * kMoveWarps * 32, pairs[warp]);
}

struct EvictPlan {
  int half, words, ctas, parts;
  bool held;
  long long lists, moves, bits;  // ints
  long long bytes() const { return (lists + moves + bits) * 4; }
};
// Clusters of `ctas` that find an SM for each of their CTAs at once (the SMs come in groups, and not all divide evenly).
int clusters_at_once(int ctas, int sms) {
  static int of[64][kMostCtas + 1];
  int dev = 0;
  if (ctas == 1 || cudaGetDevice(&dev) != cudaSuccess) return sms / ctas;
  int& known = of[dev & 63][ctas];
  if (known == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kSelect);
    cfg.dynamicSmemBytes = (size_t)held_bytes(kMostFours);  // no room for another
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    static bool ready[64];
    if (xattn_smem(reinterpret_cast<const void*>(&evict_select_kernel), held_bytes(kMostFours), ready) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, evict_select_kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = std::max(1, sms / ctas * 7 / 8);
    }
    known = n;
  }
  return known;
}

// CTAs an (item, key head): those with the least estimated time.  A CTA takes about 4.8 us and, by how its weights spread over
// the bins, 1.8 to 2.9 for each four states of a thread, 1.2 to 1.5 times that where it shares its SM; one of a cluster of
// c 8.3 + 0.17 c.  Measured, us of the first kernel with 1, 2, 4, 6, 8: 4 units of 4000 places 10.1, 10.6, 11.0, 11.2, 11.3; of
// 8000 13.6, 13.7, 10.9, 11.1, 11.4; of 16,000 20.5, 17.1, 14.3, 14.6, 11.5; 64 of 8000 13.9, 14.2, 13.7, 23.5, 26.9; 128 of
// 18,360, whose weights spread, 34.3, 24.0, 37, 42.6, 71; 16 of 130,560, alike, -, -, -, 34.7, 41.7.
// One kernel where there are few places (us in kernels, one and two: 256 units of 1000 places 12.1 and 16.7, of 2000 14.0
// and 20.5, of 4000 22.0 and 26.4, of 8000 45.8 and 45.2; 4 units 10.2 and 11.8, 10.7 and 12.3, 14.2 and 15.3, 20.1 and
// 15.5), unless the new lengths lie on the old ones, which its CTAs read at any time.
EvictPlan evict_plan(int B, int Hkv, int cap, bool apart, int sms) {
  const long long units = (long long)B * Hkv;
  EvictPlan p{};
  p.half = std::max(1, cap / 2);  // at most min(keep, len - keep) states move
  p.words = (cap + 31) / 32;
  p.ctas = 1;
  if (cap <= kFewPlaces && apart) {  // (its pairs lie in one CTA's shared memory)
    p.held = true;
    return p;
  }
  p.held = held_fours(cap, kMostCtas) <= kMostFours;
  if (!p.held) p.ctas = kMostCtas;
  double best = 1e300;
  for (int c = 1; p.held && c <= kMostCtas; ++c) {
    const int fours = held_fours(cap, c);
    if (fours > kMostFours) continue;
    const long long room = clusters_at_once(c, sms), resident = fours <= kFoursOfTwo ? 2 * room : room;
    const double us = (double)((units + resident - 1) / resident) *
                      ((c > 1 ? 8.3 + 0.17 * c : 4.8) + 2.7 * fours * (units > room ? 1.4 : 1.0));
    if (us < best) {
      best = us;
      p.ctas = c;
    }
  }
  constexpr int each = kMoveWarps * 32;
  p.parts = (int)std::max(1ll, std::min(((long long)p.half + each - 1) / each, (16ll * sms + units - 1) / units));
  p.lists = 2 * units * p.half;
  p.moves = units;
  p.bits = p.held ? 0 : 2 * units * p.words;
  return p;
}

cudaError_t evict_select(const EvictArgs& a, bool held, long long units, cudaStream_t st) {
  if (!held) return launch_after(evict_select_long_kernel, units * a.ctas, kSelect, 0, st, a, a.ctas, false);
  static bool ready[64];
  const cudaError_t e = xattn_smem(reinterpret_cast<const void*>(&evict_select_kernel), held_bytes(kMostFours), ready);
  if (e != cudaSuccess) return e;
  const int room = held_bytes(held_fours(a.pages.cap, a.ctas)) + (a.parts ? 0 : 2 * a.half * 4);
  return launch_after(evict_select_kernel, units * a.ctas, kSelect, (size_t)room, st, a, a.ctas, false);
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_paged_write(const sb_paged_append* call, void* stream) {
  if (!call) return record_error(SB_EINVAL, "sb_paged_write: null argument");
  const sb_paged_append& c = *call;
  const sb_paged_memory* const m = &c.memory;
  const void *const k = c.k, *const v = c.v;
  const long long k_row = c.k_row, k_img = c.k_img, v_row = c.v_row, v_img = c.v_img;
  const int T = c.T, dtype = c.dtype;
  const float k_scale = c.k_scale, v_scale = c.v_scale;
  if (!paged_memory_ok(m) || T < 0 || T >= (1 << 30) || (dtype != SB_F16 && dtype != SB_BF16) ||
      (m->dtype != dtype && m->dtype != SB_F8))
    return record_error(SB_EINVAL, "sb_paged_write: sizes (dh 32, 64 or 128) or dtypes");
  if (!scales_ok(m, k_scale, v_scale)) return record_error(SB_EINVAL, "sb_paged_write: scales, or scales of pages that are not e4m3");
  if (m->B == 0) return SB_OK;
  const bool some = T > 0 && m->P > 0 && m->N > 0;
  if (!c.at || !c.after || !paged_pools_ok(m) || (some && (!k || !v || k_row < 0 || k_img < 0 || v_row < 0 || v_img < 0)))
    return record_error(SB_EINVAL, "sb_paged_write: rows (pools 16-byte aligned, strides multiples of 16 bytes) or null argument");
  WriteArgs a{};
  a.k = k; a.k_row = k_row; a.k_img = k_img;
  a.v = v; a.v_row = v_row; a.v_img = v_img;
  a.kp = k_pool(m);
  a.vp = v_pool(m);
  a.pages = page_table(m);
  a.at = c.at; a.count = c.count; a.stamp = c.stamp; a.stamp_img = c.stamp_img; a.stamp_row = c.stamp_row;
  a.B = m->B; a.T = T; a.Hkv = m->Hkv;
  a.k_scale = k_scale; a.v_scale = v_scale;
  a.weight = c.weight; a.born = c.born; a.after = c.after;
  const bool e4m3 = m->dtype == SB_F8;
  const int vecs = m->Hkv * m->dh / 8;
  a.vecs = fast_div((uint32_t)vecs);
  a.group = std::min(32, std::max(1, 128 / vecs));
  a.rows = some ? (long long)m->B * T : 0;
  const long long warps = (a.rows + a.group - 1) / a.group;
  a.row_blocks = (warps + kWriteWarps - 1) / kWriteWarps;
  a.marks = m->B + (T > 0 && m->N > 0 && (c.weight || c.born) ? (long long)m->B * m->Hkv * T : 0);
  const long long blocks = a.row_blocks + (a.marks + kWriteWarps * 32 - 1) / (kWriteWarps * 32);
  if (blocks > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_paged_write: too many rows");
  auto aligned = [](const void* p, long long row, long long img) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row % 8 == 0 && img % 8 == 0;
  };
  const bool vec = aligned(k, k_row, k_img) && aligned(v, v_row, v_img);
  int bits;
  auto power = [&](float x) { return std::frexp(x, &bits) == 0.5f && std::abs(bits) < 120; };
  const bool exact = power(k_scale) && power(v_scale);
  if (exact) {
    a.k_scale = 1.f / k_scale;
    a.v_scale = 1.f / v_scale;
  }
  const bool bf16 = dtype == SB_BF16;
  auto kernel = !e4m3   ? (vec ? paged_write_kernel<0, true, false> : paged_write_kernel<0, false, false>)
                : exact ? (bf16 ? (vec ? paged_write_kernel<1, true, true> : paged_write_kernel<1, false, true>)
                                : (vec ? paged_write_kernel<1, true, false> : paged_write_kernel<1, false, false>))
                        : (bf16 ? (vec ? paged_write_kernel<2, true, true> : paged_write_kernel<2, false, true>)
                                : (vec ? paged_write_kernel<2, true, false> : paged_write_kernel<2, false, false>));
  kernel<<<(unsigned)blocks, kWriteWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}

extern "C" int sb_paged_evict_work(int B, int Hkv, int page, int N, int in_place, long long* bytes) {
  if (!bytes || !paged_sizes_ok(B, Hkv, 32, 0, page, N)) return record_error(SB_EINVAL, "sb_paged_evict_work: arguments");
  *bytes = 0;
  if (B == 0) return SB_OK;
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_evict_work: device");
  *bytes = evict_plan(B, Hkv, N * page, !in_place, sms).bytes();
  return SB_OK;
}

extern "C" int sb_paged_evict(const sb_paged_cut* call, void* stream) {
  if (!call) return record_error(SB_EINVAL, "sb_paged_evict: null argument");
  const sb_paged_cut& c = *call;
  const sb_paged_memory* const m = &c.memory;
  if (!paged_memory_ok(m)) return record_error(SB_EINVAL, "sb_paged_evict: sizes (dh 32, 64 or 128) or dtype");
  if (m->B == 0) return SB_OK;
  // (without places an account is an empty tensor, whose address is null)
  if (!c.lens || !c.after || (m->N > 0 && (!c.weight || !c.weight_out || (c.since && !c.born))) || (!c.born) != (!c.born_out) ||
      !paged_pools_ok(m))
    return record_error(SB_EINVAL, "sb_paged_evict: rows (16-byte aligned, strides multiples of 16 bytes) or null argument");
  EvictArgs a{};
  a.pages = page_table(m);
  if ((a.pages.cap > kFewPlaces || c.after == c.lens) && (!c.work || (reinterpret_cast<uintptr_t>(c.work) & 15) != 0))
    return record_error(SB_EINVAL, "sb_paged_evict: workspace (sb_paged_evict_work bytes, 16-byte aligned)");
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_evict: device");
  const EvictPlan p = evict_plan(m->B, m->Hkv, a.pages.cap, c.after != c.lens, sms);
  if (c.work_bytes < p.bytes()) return record_error(SB_EINVAL, "sb_paged_evict: workspace (sb_paged_evict_work bytes)");
  a.k = k_pool(m);
  a.v = v_pool(m);
  a.lens = c.lens; a.keep = c.keep; a.keep_all = c.keep_all; a.since = c.since;
  a.weight = c.weight; a.weight_out = c.weight_out; a.born = c.born; a.born_out = c.born_out; a.after = c.after;
  a.B = m->B; a.Hkv = m->Hkv; a.row_bytes = m->dh * page_dtype_bytes(m->dtype); a.half = p.half;
  a.ctas = p.ctas; a.parts = p.parts;
  const long long units = (long long)m->B * m->Hkv;
  if (units * std::max(p.ctas, p.parts) > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_paged_evict: too many items");
  a.to = static_cast<int*>(c.work);
  a.from = a.to + units * p.half;
  a.moves = a.from + units * p.half;
  a.bits = reinterpret_cast<uint32_t*>(a.moves + units);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = evict_select(a, p.held, units, st);
  if (e == cudaSuccess && p.parts) {
    auto move = a.row_bytes == 32    ? evict_move_kernel<2>
                : a.row_bytes == 64  ? evict_move_kernel<4>
                : a.row_bytes == 128 ? evict_move_kernel<8> : evict_move_kernel<16>;
    e = launch_after(move, units * a.parts, kMoveWarps * 32, 0, st, a);
  }
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}
