// sb_paged_attn.cu -- attention of new tokens over a paged memory:
//   s_rj = scale q_r . k_j,  out_r = sum_j p_rj v_j,  p_rj = e^(s_rj - L_r),  L_r = log sum_j e^s_rj,
// and, where the memory keeps account of what is looked at, weight_j = decay weight_j + sum_r p_rj.
//
// K and V are read once and memory bounds it, so each warp works alone on its own chunks of states (up to 4 KB of
// K and of V, 16 to 64 states): cp.async brings their rows, wherever their pages lie, into the warp's own ring,
// which copes with any page size and costs no barrier; states that take no part arrive as zeros.  The
// products are mma.sync m16n8k16 (a 128-row tile of tcgen05 would be mostly empty) with the states as the 16 rows of
// S^T = K Q^T and the channels as those of O^T = V^T P^T: one token's query heads (up to eight a key head) are then
// one column tile, half of what the rows of S = Q K^T would take, and movmatrix turns P^T around in registers.  e4m3
// pages are widened to fp16 in registers; the channels' order inside a step is free, so it is the one that the bytes
// lie in.  P is multiplied as the sum of two 16-bit parts, so that nothing but the result's own rounding shows; a
// product more, and the tensor pipe has room for it.
//
// As many CTAs as are resident share the chunks of all (item, key head)s evenly, whatever their lengths, and a second
// kernel joins the fp32 partial rows; smaller calls take a CTA or a cluster of them an (item, key head), joined through
// the cluster's shared memory, and no second kernel.  The account needs L, which is there only after the last piece, so
// the scores are kept (fp32) and the second kernel, or the CTA itself, reads them back: 8 bytes a state and row
// beside 4 dim bytes of K and V, most of them from the L2.
//
// 64 x 1 token on 8160 ragged states of 4 key heads of 128, 16 query heads, with the account: bf16 165 to 172 us (157 for
// 961 MB with the scores, 6.1 TB/s, 94 % of the copy rate; 11 the second kernel), e4m3 97 to 100 (84 for 495 MB, 90 %; 11 the
// second kernel and its launch).  One stream of 130,560 states 56 (47 for 267 MB: start and end; 7 the second kernel).  16 x 8
// causal tokens on 42,840 of 4 heads of 64: 173 to 180; the scores of 16 rows a state, written and read, are 350 MB
// beside 601 of K and V.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "sb_paged.cuh"

namespace sb {
namespace {

constexpr int kWarps = 4;

struct PagedArgs {
  const void* q;
  long long q_row, q_img;  // elements
  Pool k, v;
  PageTable pages;
  const int* lens;
  int B, H, Hkv, group, Tq, rows, blocks;  // rows = group * Tq of an (item, key head), blocks of 16
  int shares;                              // CTAs that share the chunks of all units; 0: CTAs of a unit's own
  int cluster;                             // of them, then: 1 to 8
  int ends;                                // CTAs an (item, key head) of the last kernel; 0: none
  int chunk;                               // states
  int q_bf16, causal;
  float scale_log2, v_scale;  // scale * k_scale * log2(e)
  OutView o;
  float* lse;
  float* weight;
  float decay;
  float* scores;  // [B * Hkv][blocks][places][score_rows], log2 units
  int places, score_rows;  // cap and a block's rows, up to a multiple of 4 and a power of two
  float* part_l;  // [units + shares][part_rows], log2 of the sum: what CTA i finds of unit u at i + u
  float* part_o;  // [2 shares][part_rows][dh]: a CTA's piece of a unit that began before, of one that goes on behind
  int part_rows;  // min(rows, 16)
  SB_DEV int chunks(int b) const { return (pages.clamp(lens[b]) + chunk - 1) / chunk; }
  SB_DEV int units() const { return Hkv * blocks; }  // of an item
  SB_DEV float* plane(int head, int block) const {
    return scores + ((long long)head * blocks + block) * places * score_rows;
  }
};

// How the chunks of all units, one unit after the other, are shared: CTA i gets `each` of them from i * each on.
// (Along the chunks i or u grows from one piece to the next, so i + u is a place of its own.)
struct Shares {
  long long total, each;
  int item;            // the item that position `at` lies in (B: none)
  long long before;    // chunks of one unit of every item before it
};
constexpr long long kLeast = 16;  // chunks a CTA, four a warp

// Looks up the shares and position `at` of the chunks, with all `THREADS` of the CTA; item >= 0: that item instead.
template <int THREADS>
SB_DEV Shares look_up(const PagedArgs& a, long long cta, int item, long long (&room)[THREADS / 32 + 2], int& found) {
  const int lane = lane_id(), warp = warp_id();
  Shares s;
  if (a.B <= 32) {  // each warp for itself: a lane an item, no barrier (fewer than 2^27 chunks an item)
    const uint32_t n = lane < a.B ? (uint32_t)a.chunks(lane) : 0u;
    s.total = (long long)__reduce_add_sync(0xFFFFFFFFu, n) * a.units();
    s.each = max((s.total + a.shares - 1) / a.shares, kLeast);
    if (item >= 0) {
      s.item = item;
      s.before = __reduce_add_sync(0xFFFFFFFFu, lane < item ? n : 0u);
      return s;
    }
    uint32_t upto = n;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, upto, x);
      if (lane >= x) upto += u;
    }
    const long long at = cta * s.each < s.total ? cta * s.each / a.units() : -1;
    const uint32_t here = __ballot_sync(0xFFFFFFFFu, (long long)(upto - n) <= at && at < (long long)upto);
    const int lane_of = here ? __ffs(here) - 1 : 0;
    s.item = here ? lane_of : a.B;
    s.before = __shfl_sync(0xFFFFFFFFu, upto - n, lane_of);
    return s;
  }
  long long sum = 0, before = 0;
  for (int b = threadIdx.x; b < a.B; b += THREADS) {
    const int n = a.chunks(b);
    sum += n;
    if (b < item) before += n;
  }
#pragma unroll
  for (int x = 16; x; x >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
    before += __shfl_xor_sync(0xFFFFFFFFu, before, x);
  }
  s.total = s.before = 0;
  __syncthreads();
  if (lane == 0) room[warp] = sum;
  __syncthreads();
  for (int w = 0; w < THREADS / 32; ++w) s.total += room[w];
  s.total *= a.units();
  s.each = max((s.total + a.shares - 1) / a.shares, kLeast);
  s.item = item;
  if (item >= 0) {
    __syncthreads();
    if (lane == 0) room[warp] = before;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) s.before += room[w];
    return s;
  }
  s.item = a.B;
  if (cta * s.each >= s.total) return s;
  const long long at = cta * s.each / a.units();
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {  // ends with the tile of items that holds it
    const int b = b0 + (int)threadIdx.x;
    const int n = b < a.B ? a.chunks(b) : 0;
    long long upto = n;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const long long u = __shfl_up_sync(0xFFFFFFFFu, upto, x);
      if (lane >= x) upto += u;
    }
    __syncthreads();
    if (lane == 31) room[warp] = upto;
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    long long base = s.before, all = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) base += room[w];
      all += room[w];
    }
    const long long from = base + upto - n;
    if (from <= at && at < from + n) {
      found = b;
      room[THREADS / 32] = from;
    }
    __syncthreads();
    if (found >= 0) {
      s.item = found;
      s.before = room[THREADS / 32];
      break;
    }
    s.before += all;
  }
  return s;
}

template <int DH, int PT, int NB>
struct Paged {
  static constexpr bool E4M3 = PT == SB_F8, BF16 = PT == SB_BF16;
  static constexpr int RB = DH * (E4M3 ? 1 : 2);                // bytes a state and head
  // Two CTAs an SM, 24 KB a warp on their way.  e4m3 has twice the instructions a byte (41 % of the issue slots): three
  // CTAs (83 us for the 64 x 8160 states above, 92 with two).
  static constexpr int OCC = E4M3 && NB == 1 ? 3 : 2;
  static constexpr int kRing = OCC == 3 ? 16 * 1024 : 24 * 1024;  // bytes a warp
  static constexpr int CK = 4096 / RB < 64 ? 4096 / RB : 64;      // states a chunk
  static constexpr int HALF = CK * RB, STAGE = 2 * HALF, STAGES = kRing / STAGE;
  static constexpr int LANES = RB / 16, AT_ONCE = 32 / LANES;   // lanes a row, rows a copy
  static constexpr int SMEM = kWarps * kRing;
  static_assert(8 * NB * DH * 4 <= STAGE && STAGES >= 2, "ring");
  // Byte of 16-byte chunk c of a row: eight rows of a chunk fall in distinct banks.  Bits of the row are bits of
  // what its chunks are turned by, so rows x + l that share none are l's place, turned by x's.
  SB_DEV static constexpr uint32_t turn(int row) {
    return (RB >= 128 ? row & 7 : RB == 64 ? (row >> 1) & 3 : (row >> 2) & 1) << 4;
  }
  SB_DEV static uint32_t at(int row, int c) { return row * RB + (c << 4 ^ turn(row)); }
};

// What states that take no part are read from.
__device__ uint4 g_zeros[16];

// K and V that are read once pass through the L2 as what goes first: scores written meanwhile are still there for the
// account (64 x 8160 states in bf16: 176 -> 171 us), and nothing else is driven out.
SB_DEV uint64_t passing(bool once) {
  uint64_t p;
  if (once) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  else asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}
SB_DEV void copy16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
SB_DEV void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
SB_DEV void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// An 8 x 8 matrix of 16-bit values, a pair of a row a thread, turned around.
SB_DEV uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// Four e4m3 codes as two pairs of fp16 values (exact)
SB_DEV void widen(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}

// Query row r of an (item, key head): token r / group, head r % group.
struct Row {
  int t, h;
  SB_DEV Row(const PagedArgs& a, int kvh, int r) : t(r / a.group), h(kvh * a.group + r - t * a.group) {}
};

// Where a warp is among the chunks: item, unit of the item, chunk of the unit.
struct Cursor {
  int b, unit, c, n, count;
  SB_DEV void item(const PagedArgs& a) {
    count = a.pages.clamp(a.lens[b]);
    n = (count + a.chunk - 1) / a.chunk;
  }
  // `by` chunks on, of which there are as many
  SB_DEV void advance(const PagedArgs& a, int by) {
    c += by;
    while (c >= n) {
      c -= n;
      if (++unit == a.units()) {
        unit = 0;
        do {
          ++b;
          item(a);
        } while (n == 0);
      }
    }
  }
};

constexpr int kHeldScores = 1536;  // floats: 6 KB, as many CTAs an SM as without

// The rows of a unit from those of its cluster's CTAs, out = sum_s 2^(L_s - L) O_s, CTA by CTA every cluster-th of them, and
// L of all into fin.  A group of lanes takes a row's eight channels, a lane a CTA.
template <int DH>
SB_DEV void join_cluster(const PagedArgs& a, int b, int kvh, int unit, int r0, int rows, const float* own, const float* own_l,
                         float* fin) {
  constexpr int per = DH / 8;
  const int n = a.cluster, rank = (int)cluster_ctarank(), lane = lane_id(), s = lane % n;
  auto sums_of = [&](int r, float& l, float& all) {  // L of this lane's CTA and of the cluster, for row r
    l = __uint_as_float(peer_word(own_l + r, (uint32_t)s));
    float top = l;
    for (int x = 1; x < n; x <<= 1) {
      const float u = __shfl_xor_sync(0xFFFFFFFFu, top, x);
      top = max3(top, u, u);
    }
    float sum = l == top ? 1.f : exp2_hw(l - top);
    for (int x = 1; x < n; x <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
    all = top == -INFINITY ? -INFINITY : top + log2f(sum);
  };
  for (int r = threadIdx.x / n; r < 16; r += kWarps * 32 / n) {  // (16 rows: whole warps)
    float l, all;
    sums_of(min(r, rows - 1), l, all);
    if (s == 0 && r < rows) {
      fin[r] = all;
      if (rank == 0 && a.ends > 0) a.part_l[((long long)b * a.units() + unit) * a.part_rows + r] = all;
    }
  }
  const int mine = rows > rank ? (rows - rank + n - 1) / n : 0, work = mine * per;
  for (int e0 = 0; e0 < work; e0 += kWarps * 32 / n) {
    const int e = e0 + (int)threadIdx.x / n, at = min(e, work - 1), r = rank + at / per * n, c = at % per * 8;
    float l, all;
    sums_of(r, l, all);
    const uint4 x = peer_words(own + r * DH + c, (uint32_t)s), y = peer_words(own + r * DH + c + 4, (uint32_t)s);
    const uint32_t v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    const float k = l == -INFINITY ? 0.f : exp2_hw(l - all);
    float f[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float x = __uint_as_float(v[u]);
      f[u] = fabsf(x) == INFINITY ? x : k * x;  // (however small its share)
      for (int z = 1; z < n; z <<= 1) f[u] += __shfl_xor_sync(0xFFFFFFFFu, f[u], z);
    }
    if (s == 0 && e < work) {
      const Row w(a, kvh, r0 + r);
      store8(a.o.p, a.q_bf16 ? SB_BF16 : SB_F16, b * a.o.img + w.t * a.o.row + (long long)w.h * DH + c, f);
      if (c == 0 && a.lse) a.lse[((long long)b * a.H + w.h) * a.Tq + w.t] = all * 0.69314718055994531f;
    }
  }
}

// A 16-bit value that is infinite is lost where a probability is multiplied in two parts (inf - inf where they differ in
// sign, 0 x inf where the second is 0).  So a row's channels c .. c + 7 that came out as no number, `lost` as bits, are asked
// here what states j0 .. j1 - 1 make of them: bits 0 .. 7 where one has +inf, 8 .. 15 -inf, 16 .. 23 no number (NaN, or an infinite
// value of a state whose score is -inf).  A share that rounds to 0 is taken for what it stands for.  Looked at only
// then, so that the loop over the states knows nothing of it; a walk of waits, eight states together (64 x 8160 states of 4
// key heads, one row of infinities an item: 195 us become 1384, one state after the other 5810).
template <int DH, bool BF16>
__device__ __noinline__ uint32_t odd_values(const PagedArgs& a, int b, int kvh, int t, int h, int c, uint32_t lost, int j0,
                                            int j1) {
  constexpr int type = BF16 ? SB_BF16 : SB_F16;
  const uint16_t* const q = static_cast<const uint16_t*>(a.q) + b * a.q_img + t * a.q_row + (long long)h * DH;
  uint32_t odd = 0;
  constexpr int kAtOnce = 8;  // states: what they wait for is asked for together
  for (int j = j0; j < j1; j += kAtOnce) {
    int page[kAtOnce];
    uint32_t row[kAtOnce];
    uint4 v[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) page[i] = a.pages.entry(b, (uint32_t)min(j + i, j1 - 1), row[i]);  // (the last one twice: no matter)
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint64_t at = a.pages.has(page[i]) ? a.v.row_at(page[i], row[i]) + (kvh * DH + c) * 2 : reinterpret_cast<uint64_t>(g_zeros);
      v[i] = *reinterpret_cast<const uint4*>(at);
    }
    // (an exponent of ones, and one more in its lowest bit, is the sign's bit)
    constexpr uint32_t ones = BF16 ? 0x7F807F80u : 0x7C007C00u, one = BF16 ? 0x00800080u : 0x04000400u;
    uint32_t some = 0;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      some |= ((v[i].x & ones) + one) | ((v[i].y & ones) + one) | ((v[i].z & ones) + one) | ((v[i].w & ones) + one);
    if (!(some & 0x80008000u)) continue;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t here = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float2 f = pair_of(w[u], type);
        here |= (f.x == INFINITY ? 1u : f.x == -INFINITY ? 1u << 8 : f.x != f.x ? 1u << 16 : 0u) << (2 * u) |
                (f.y == INFINITY ? 1u : f.y == -INFINITY ? 1u << 8 : f.y != f.y ? 1u << 16 : 0u) << (2 * u + 1);
      }
      if (here & 0xFFFFu) {
        const void* const k = reinterpret_cast<const void*>(a.k.row_at(page[i], row[i]));
        float s = 0.f;
        for (int x = 0; x < DH; ++x) s = fmaf(one_of(q, type, x), one_of(k, type, kvh * DH + x), s);
        if (s == -INFINITY) here = ((here | here >> 8 | here >> 16) & 0xFFu) << 16;
      }
      odd |= here;
    }
    if (((odd >> 16 | (odd & odd >> 8)) & lost) == lost) break;  // none of them can be anything else
  }
  return odd;
}

// NB: column tiles of eight query rows
template <int DH, int PT, int NB>
__global__ void __launch_bounds__(kWarps * 32, Paged<DH, PT, NB>::OCC)
    paged_attend_kernel(const __grid_constant__ PagedArgs a) {
  using C = Paged<DH, PT, NB>;
  constexpr bool E4M3 = C::E4M3, BF16 = C::BF16;
  constexpr int CK = C::CK, KT = CK / 16, KS = DH / 16, R = CK > 32 ? 2 : 1;
  constexpr float lift = kLift<BF16>;
  // bf16 values reach fp32's end, and a sum of them beyond it (p up to 2^8 a state): P meets V 2^40 times smaller, which is
  // exact down to p = 2^-86 and leaves room for 2^30 states
  constexpr float room_for = BF16 ? 0x1p-40f : 1.f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ ulonglong2 place[kWarps][CK];      // addresses of a chunk's rows of K and V
  __shared__ uint64_t there[kWarps][C::STAGES];  // a stage's rows that take part, as bits
  __shared__ float2 ml[kWarps][16];
  __shared__ float fin[16], found_l[16];
  __shared__ long long room[kWarps + 2];
  __shared__ int area[kWarps], found;
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, tig = lane & 3;

  // this CTA's chunks: `left` from cursor `at` on
  Cursor at;
  long long left;
  if (a.shares) {
    const Shares s = look_up<kWarps * 32>(a, blockIdx.x, -1, room, found);
    if (s.item == a.B) return;
    at.b = s.item;
    at.item(a);
    const long long in = blockIdx.x * s.each - s.before * a.units();
    at.unit = (int)(in / at.n);
    at.c = (int)(in - (long long)at.unit * at.n);
    left = min(s.each, s.total - blockIdx.x * s.each);
  } else {
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;  // (a cluster's CTAs lie side by side)
    at.b = unit / a.units();
    at.unit = unit - at.b * a.units();
    at.item(a);
    const int each = (at.n + a.cluster - 1) / a.cluster;
    at.c = min(rank * each, at.n);
    left = min(each, at.n - at.c);
  }
  const int mine = left > warp ? (int)((left - warp + kWarps - 1) / kWarps) : 0;  // chunks warp, warp + kWarps, ... of them
  uint8_t* const ring = smem + warp * C::kRing;
  const uint32_t ring_at = smem_u32(ring);

  // table entries of the next chunk to be copied, asked for a chunk ahead
  Cursor ahead = at;
  if (mine > 0 && warp > 0) ahead.advance(a, warp);
  int entry[R], asked = 0, head = 0;
  uint32_t within[R];
  auto ask = [&] {
    if (asked < mine) {
      if (asked) ahead.advance(a, kWarps);
      head = ahead.unit / a.blocks;
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const int r = lane + 32 * x, j = ahead.c * CK + r;
        entry[x] = -1;
        within[x] = 0;
        if (r < CK && j < ahead.count) entry[x] = a.pages.entry(ahead.b, (uint32_t)j, within[x]);
      }
    }
    ++asked;
  };
  const uint64_t policy = passing(a.blocks == 1);
  const uint32_t own16 = lane % C::LANES * 16, own_at = ring_at + C::at(lane / C::LANES, lane % C::LANES);
  auto copy = [&](int i) {  // the warp's chunk i, whose entries are there
    if (i < mine) {
      const int st = i % C::STAGES;
      uint64_t bits = 0;
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const bool ok = a.pages.has(entry[x]);
        const uint64_t none = reinterpret_cast<uint64_t>(g_zeros);
        if (lane + 32 * x < CK)
          place[warp][lane + 32 * x] =
              make_ulonglong2(ok ? a.k.row_at(entry[x], within[x]) + head * C::RB : none,
                              ok ? a.v.row_at(entry[x], within[x]) + head * C::RB : none);
        bits |= (uint64_t)__ballot_sync(0xFFFFFFFFu, ok) << (32 * x);
      }
      if (lane == 0) there[warp][st] = bits;
      __syncwarp();
      const uint32_t dst = own_at + st * C::STAGE;
#pragma unroll
      for (int x = 0; x < CK; x += C::AT_ONCE) {
        const ulonglong2 from = place[warp][x + lane / C::LANES];
        const uint32_t to = (dst ^ C::turn(x)) + x * C::RB;
        copy16(to, reinterpret_cast<const void*>(from.x + own16), policy);
        copy16(to + C::HALF, reinterpret_cast<const void*>(from.y + own16), policy);
      }
    }
    copies_done();
  };
  ask();
#pragma unroll 1
  for (int i = 0; i < C::STAGES; ++i) {
    copy(i);
    ask();
    __syncwarp();  // place is written again
  }

  // behind the rings: this CTA's states' scores, where they are held, and its rows of a cluster
  float* const held = reinterpret_cast<float*>(smem + C::SMEM);
  float* const rows_of_cluster = held + kHeldScores;

  int i = 0;  // the warp's chunk
  long long done = 0;
  do {  // a piece: this CTA's chunks of a unit
    const int b = at.b, kvh = at.unit / a.blocks, block = at.unit - kvh * a.blocks, count = at.count;
    const int r0 = block * 16, rows = min(16, a.rows - r0);
    const int piece = (int)min((long long)at.n - at.c, left - done);
    const bool whole = piece == at.n;
    const int i_end = done + piece > warp ? (int)((done + piece - warp + kWarps - 1) / kWarps) : 0;

    // Q as the second operand: rows g (+ 8), channels 16 ks + 2 tig (+ 8), or for e4m3 16 ks + 4 tig (+ 2).  e4m3 is
    // multiplied as fp16: bf16 rows are then brought to at most 2^14 by a power of two, and what falls
    // below fp16's 2^-24 is less than 2^-37 of the row's largest.
    uint32_t q[KS][NB][2];
    float factor[NB][2];  // of rows 2 tig, 2 tig + 1 (+ 8): scores times it are exponents of 2
    int limit[NB][2];     // states that those rows see
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      const bool has = g + 8 * y < rows;
      const Row w(a, kvh, has ? r0 + g + 8 * y : 0);
      const uint16_t* p = static_cast<const uint16_t*>(a.q) + b * a.q_img + w.t * a.q_row + (long long)w.h * DH;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int c = E4M3 ? ks * 16 + 4 * tig : ks * 16 + 2 * tig;
        q[ks][y][0] = has ? *reinterpret_cast<const uint32_t*>(p + c) : 0u;
        q[ks][y][1] = has ? *reinterpret_cast<const uint32_t*>(p + c + (E4M3 ? 2 : 8)) : 0u;
      }
      int up = 0;
      if (E4M3 && a.q_bf16) {
        uint32_t top = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) top = max(top, max(q[ks][y][x] & 0x7FFFu, q[ks][y][x] >> 16 & 0x7FFFu));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const int e = (int)(top >> 7);  // the largest's exponent, biased by 127
        up = e == 255 ? 0 : min(max(140 - e, -126), 126);
        const float by = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 f = pair_of(q[ks][y][x], SB_BF16);
            q[ks][y][x] = pack_pair(f.x * by, f.y * by, SB_F16);
          }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int down = __shfl_sync(0xFFFFFFFFu, up, (2 * tig + x) * 4), r = r0 + 8 * y + 2 * tig + x;
        // (neither 0 nor infinite: -inf, which states that take no part score, has to stay so, and 0 too)
        factor[y][x] = fminf(fmaxf(a.scale_log2 * __uint_as_float((uint32_t)(127 - down) << 23), FLT_MIN), FLT_MAX);
        limit[y][x] = a.causal && r < a.rows ? max(count - a.Tq + 1 + r / a.group, 0) : count;
      }
    }
    const int seen_by_all = a.causal ? max(count - a.Tq + 1 + r0 / a.group, 0) : count;

    float o[KS][NB][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      m[y][0] = m[y][1] = -INFINITY;
      l[y][0] = l[y][1] = 0.f;
#pragma unroll
      for (int x = 0; x < KS; ++x) o[x][y][0] = o[x][y][1] = o[x][y][2] = o[x][y][3] = 0.f;
    }
    float* const scores = a.scores   ? a.plane(b * a.Hkv + kvh, block)
                          : a.weight ? held - (long long)at.c * CK * a.score_rows : nullptr;
    const int chunk0 = at.c - (int)done;  // of the unit: chunk0 + warp + i * kWarps

    const int i_first = i;
    for (; i < i_end; ++i) {
      copies_wait<C::STAGES - 1>();
      __syncwarp();
      const int st = i % C::STAGES, j0 = (chunk0 + warp + i * kWarps) * CK;
      const uint32_t kb = ring_at + st * C::STAGE, vb = kb + C::HALF;
      const uint64_t bits = there[warp][st];
      const bool mixed = j0 + CK > seen_by_all;  // (or the last chunk)
      const bool all = bits == (~0ull >> (64 - CK)) && !mixed;

      float s[KT][NB][4];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int y = 0; y < NB; ++y) s[kt][y][0] = s[kt][y][1] = s[kt][y][2] = s[kt][y][3] = 0.f;
        const int row = kt * 16 + (lane >> 3 & 1) * 8 + (lane & 7);
        if constexpr (E4M3) {
#pragma unroll
          for (int p = 0; p < KS / 2; ++p) {
            uint32_t f[4];
            ldsm4(kb + C::at(row, 2 * p + (lane >> 4)), f);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              uint32_t w[4];
              widen(f[2 * z], w[0], w[2]);
              widen(f[2 * z + 1], w[1], w[3]);
#pragma unroll
              for (int y = 0; y < NB; ++y) mma16816<false>(s[kt][y], w, q[2 * p + z][y][0], q[2 * p + z][y][1]);
            }
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t f[4];
            ldsm4(kb + C::at(row, 2 * ks + (lane >> 4)), f);
#pragma unroll
            for (int y = 0; y < NB; ++y) mma16816<BF16>(s[kt][y], f, q[ks][y][0], q[ks][y][1]);
          }
        }
      }
      if (!all) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int k = kt * 16 + g + 8 * x;
            const bool in = bits >> k & 1u;
#pragma unroll
            for (int y = 0; y < NB; ++y)
#pragma unroll
              for (int z = 0; z < 2; ++z)
                if (!in || j0 + k >= limit[y][z]) s[kt][y][2 * x + z] = -INFINITY;
          }
      }
      if (scores) {
        float* to8 = scores + (long long)(j0 + g) * a.score_rows + 2 * tig;  // of every eighth state
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int x = 0; x < 2; ++x, to8 += 8 * a.score_rows) {
            if (j0 + kt * 16 + 8 * x + g < count) {
#pragma unroll
              for (int y = 0; y < NB; ++y) {
                const float u = s[kt][y][2 * x] * factor[y][0], w = s[kt][y][2 * x + 1] * factor[y][1];
                if (a.score_rows == 1) {
                  if (tig == 0 && y == 0) *to8 = u;
                } else if (8 * y + 2 * tig < rows) {  // (the row after an odd last one is room of its own)
                  *reinterpret_cast<float2*>(to8 + 8 * y) = make_float2(u, w);
                }
              }
            }
          }
      }
      // a new reference point with the first states, and where a maximum grew by more than 2^8 (or is NaN)
      bool grew = false;
      float base[NB][2];
#pragma unroll
      for (int y = 0; y < NB; ++y)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          float top = s[0][y][z];
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) top = max3(top, s[kt][y][z], s[kt][y][2 + z]);
          base[y][z] = fmaf(-m[y][z], factor[y][z], lift);
          grew = grew || !(fmaf(top, factor[y][z], base[y][z]) <= lift + 8.f);
        }
      if (__any_sync(0xFFFFFFFFu, grew)) {
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            float top = m[y][z];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) top = max3(top, s[kt][y][z], s[kt][y][2 + z]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              const float u = __shfl_xor_sync(0xFFFFFFFFu, top, x);
              top = max3(top, u, u);
            }
            const float c = m[y][z] == top ? 1.f : exp2_hw((m[y][z] - top) * factor[y][z]);
            m[y][z] = top;
            base[y][z] = fmaf(-top, factor[y][z], lift);
            l[y][z] *= c;
#pragma unroll
            for (int x = 0; x < KS; ++x) {
              o[x][y][z] *= c;
              o[x][y][2 + z] *= c;
            }
          }
      }
#pragma unroll
      for (int y = 0; y < NB; ++y)
#pragma unroll
        for (int z = 0; z < 2; ++z)
          if (m[y][z] == -INFINITY) base[y][z] = 0.f;
      // probabilities in place of the scores
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float p = exp2_hw(fmaf(s[kt][y][x], factor[y][x & 1], base[y][x & 1]));
            s[kt][y][x] = p;
            l[y][x & 1] += p;
          }
      // a causal call's last states are seen by some rows only; where one's V is no number, 0 x V is not 0
      bool odd = false;
      if (a.causal && mixed) {
        for (int x = lane; x < C::HALF / 16; x += 32) {
          const uint4 w = *reinterpret_cast<const uint4*>(ring + st * C::STAGE + C::HALF + x * 16);
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            if constexpr (E4M3) odd = odd || (__vcmpeq4(u[z] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0);
            else {
              constexpr uint32_t e = BF16 ? 0x7F807F80u : 0x7C007C00u;
              odd = odd || (__vcmpeq2(u[z] & e, e) != 0);
            }
          }
        }
        odd = __any_sync(0xFFFFFFFFu, odd);
      }
      if (!odd) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          uint32_t hi[NB][2], lo[NB][2];
#pragma unroll
          for (int y = 0; y < NB; ++y)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float u = s[kt][y][2 * x] * room_for, w = s[kt][y][2 * x + 1] * room_for;
              const uint32_t h = pack16<BF16>(u, w);
              const float2 f = pair_of(h, BF16 ? SB_BF16 : SB_F16);
              hi[y][x] = transposed(h);
              lo[y][x] = transposed(pack16<BF16>(u - f.x, w - f.y));
            }
          if constexpr (E4M3) {
            const int row = kt * 16 + (lane >> 3 & 1) * 8 + (lane & 7);
#pragma unroll
            for (int p = 0; p < KS / 2; ++p) {
              uint32_t f[4];
              ldsm4_t(vb + C::at(row, 2 * p + (lane >> 4)), f);
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                // a register: channels 2g, 2g + 1 of a state, then of the next
                uint32_t w[4];
                widen(__byte_perm(f[2 * z], 0, 0x3120), w[0], w[1]);
                widen(__byte_perm(f[2 * z + 1], 0, 0x3120), w[2], w[3]);
#pragma unroll
                for (int y = 0; y < NB; ++y) {
                  mma16816<false>(o[2 * p + z][y], w, hi[y][0], hi[y][1]);
                  mma16816<false>(o[2 * p + z][y], w, lo[y][0], lo[y][1]);
                }
              }
            }
          } else {
            const int row = kt * 16 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
            for (int x = 0; x < KS; ++x) {
              uint32_t f[4];
              ldsm4_t(vb + C::at(row, 2 * x + (lane >> 3 & 1)), f);
#pragma unroll
              for (int y = 0; y < NB; ++y) {
                mma16816<BF16>(o[x][y], f, hi[y][0], hi[y][1]);
                mma16816<BF16>(o[x][y], f, lo[y][0], lo[y][1]);
              }
            }
          }
        }
      } else {  // state by state, rows that do not see it left alone
        const uint8_t* v = ring + st * C::STAGE + C::HALF;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
            const int row = kt * 16 + k;
            float p[NB][2];
#pragma unroll
            for (int y = 0; y < NB; ++y)
#pragma unroll
              for (int z = 0; z < 2; ++z)
                p[y][z] = room_for * __shfl_sync(0xFFFFFFFFu, k < 8 ? s[kt][y][z] : s[kt][y][2 + z], (k & 7) * 4 + tig);
#pragma unroll
            for (int x = 0; x < KS; ++x)
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                const int c = E4M3 ? x * 16 + 2 * g + w : x * 16 + g + 8 * w;
                float f;
                if constexpr (E4M3) f = float2_of_e4m3x2(v[C::at(row, c >> 4) + (c & 15)]).x;
                else f = one_of(v + C::at(row, c >> 3), PT, c & 7);
#pragma unroll
                for (int y = 0; y < NB; ++y)
#pragma unroll
                  for (int z = 0; z < 2; ++z)
                    if (j0 + row < limit[y][z]) o[x][y][2 * w + z] = fmaf(p[y][z], f, o[x][y][2 * w + z]);
              }
          }
      }
      __syncwarp();  // every lane has read the stage
      if (i + 1 < i_end) {
        copy(i + C::STAGES);
        ask();
        __syncwarp();
      }
    }
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[y][z] += __shfl_xor_sync(0xFFFFFFFFu, l[y][z], x);
    // the warps' outputs meet in shared memory: rows of DH floats in the stage that a warp has just read (and fills
    // again afterwards), groups of eight floats turned so that no two lanes meet in a bank; maxima as exponents of 2
    const bool some = i > i_first;
    const int last = some ? warp * C::kRing + (i - 1) % C::STAGES * C::STAGE : -1;
    if (some) {
      float* own = reinterpret_cast<float*>(smem + last);
#pragma unroll
      for (int x = 0; x < KS; ++x)
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const int c = E4M3 ? x * 16 + 2 * g + (z >> 1) : x * 16 + g + 8 * (z >> 1);
            own[(8 * y + 2 * tig + (z & 1)) * DH + (c ^ tig << 3)] = o[x][y][z];
          }
    }
    if (lane == 0) area[warp] = last;
    if (g == 0) {
#pragma unroll
      for (int y = 0; y < NB; ++y)
#pragma unroll
        for (int z = 0; z < 2; ++z)
          ml[warp][8 * y + 2 * tig + z] = make_float2(m[y][z] == -INFINITY ? -INFINITY : m[y][z] * factor[y][z], l[y][z]);
    }
    __syncthreads();
    const long long slot = a.shares ? (long long)blockIdx.x + (long long)b * a.units() + at.unit : 0;
    constexpr int per = DH / 8;
    for (int e = threadIdx.x; e < rows * per; e += kWarps * 32) {
      const int r = e / per, c = (e - r * per) * 8;
      float top = -INFINITY, sum = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = max3(top, ml[w][r].x, ml[w][r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (area[w] < 0) continue;
        const float mw = ml[w][r].x, k = mw == top ? 1.f : exp2_hw(mw - top);
        sum = fmaf(k, ml[w][r].y, sum);
        const float4* src = reinterpret_cast<const float4*>(smem + area[w]) + (r * DH + (c ^ (r >> 1 & 3) << 3)) / 4;
        const float4 x = src[0], y = src[1];
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int u = 0; u < 8; ++u) f[u] = fmaf(k, v[u], f[u]);
      }
      const bool none = top == -INFINITY;  // no states
      const float inv = none ? 0.f : a.v_scale / room_for / sum;
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] = none ? 0.f : f[u] * inv;
      const float log_sum = none ? -INFINITY : top - lift + log2f(sum);
      const Row w(a, kvh, r0 + r);
      if constexpr (!E4M3) {  // (e4m3 has no infinities)
        uint32_t lost = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) lost |= (uint32_t)(f[u] != f[u]) << u;
        if (lost && sum == sum) {
          const int seen = a.causal ? max(count - a.Tq + 1 + w.t, 0) : count;
          const uint32_t odd = odd_values<DH, BF16>(a, b, kvh, w.t, w.h, c, lost, at.c * CK, min(seen, (at.c + piece) * CK));
          lost &= (odd ^ odd >> 8) & ~(odd >> 16);  // of one sign
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (lost >> u & 1u) f[u] = odd >> u & 1u ? INFINITY : -INFINITY;
        }
      }
      if (a.cluster > 1) {
        store8(rows_of_cluster, SB_F32, r * DH + c, f);
        if (c == 0) found_l[r] = log_sum;
        continue;
      }
      if (a.shares && !whole) {
        const long long place = 2ll * blockIdx.x + (at.c == 0);
        store8(a.part_o, SB_F32, (place * a.part_rows + r) * DH + c, f);
      } else {
        store8(a.o.p, a.q_bf16 ? SB_BF16 : SB_F16, b * a.o.img + w.t * a.o.row + (long long)w.h * DH + c, f);
        if (c == 0 && a.lse) a.lse[((long long)b * a.H + w.h) * a.Tq + w.t] = log_sum * 0.69314718055994531f;
      }
      if (c == 0) {
        if (a.ends > 0) a.part_l[(a.shares ? slot : (long long)b * a.units() + at.unit) * a.part_rows + r] = log_sum;
        fin[r] = log_sum;
      }
    }
    if (a.cluster > 1) {  // (one piece a CTA)
      __syncwarp();
      cluster_sync();
      join_cluster<DH>(a, b, kvh, at.unit, r0, rows, rows_of_cluster, found_l, fin);
    }
    __syncthreads();
    if (a.weight && a.ends == 0) {  // the scores are this CTA's own, and all of the sums are here
      float* weight = a.weight + ((long long)b * a.Hkv + kvh) * a.pages.cap;
      const int j_end = min(count, (at.c + piece) * CK);
      for (int j = at.c * CK + (int)threadIdx.x; j < j_end; j += kWarps * 32) {
        float w = 0.f;
        for (int r = 0; r < rows; ++r)
          if (fin[r] != -INFINITY) w += exp2_hw(scores[(long long)j * a.score_rows + r] - fin[r]);
        weight[j] = fmaf(a.decay, weight[j], w);
      }
    }
    if (some) {
      copy(i - 1 + C::STAGES);
      ask();
      __syncwarp();
    }
    done += piece;
    if (done < left) at.advance(a, piece);
  } while (done < left);
  copies_wait<0>();
  __syncwarp();
  if (a.cluster > 1) cluster_sync();  // no CTA ends while another reads its rows
}

// What is left after the last piece, a CTA a part of an (item, key head): its share of the rows is joined from the
// unit's pieces,
//   out = sum_s 2^(L_s - L) O_s,  L = log2 sum_s 2^L_s,
// and its share of the states gets its account, weight = decay weight + sum over the rows of 2^(score - L).  Every CTA
// finds L of the rows by itself, 16 at a time.  A unit in one piece has its rows already, one without states gets
// zeros.
constexpr int kEndThreads = 256, kEndOcc = 4, kEndEach = 4;  // threads, CTAs an SM, states a thread at once

// The account of states j_first (a multiple of 4) .. j_end - 1 from a plane of scores, ROWS a state: neighbouring threads
// take neighbouring 16 bytes, four at once, and those of a state add up among themselves.
template <int ROWS>
SB_DEV void account(const float4* scores, const float* fin, float* weight, float decay, int j_first, int j_end) {
  constexpr int lanes = ROWS > 4 ? ROWS / 4 : 1, states = ROWS < 4 ? 4 / ROWS : 1;  // threads a state, states a thread
  constexpr int step = kEndThreads / lanes * states;
  const int quad = threadIdx.x % lanes * 4, j_mine = j_first + (int)threadIdx.x / lanes * states;
  float l[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) l[y] = fin[ROWS < 4 ? y % ROWS : quad + y];
  for (int j0 = j_first; j0 < j_end; j0 += step * kEndEach) {  // (all threads take part in the sums)
    float4 v[kEndEach];
    float w[kEndEach][states];
#pragma unroll
    for (int x = 0; x < kEndEach; ++x) {
      const int j = j_mine + (j0 - j_first) + x * step;
      v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j < j_end) v[x] = scores[(long long)j * ROWS / 4 + (ROWS > 4 ? (int)threadIdx.x % lanes : 0)];
#pragma unroll
      for (int z = 0; z < states; ++z) w[x][z] = j + z < j_end && quad == 0 ? weight[j + z] : 0.f;
    }
#pragma unroll
    for (int x = 0; x < kEndEach; ++x) {
      const int j = j_mine + (j0 - j_first) + x * step;
      const float u[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
      float sum[states];
#pragma unroll
      for (int z = 0; z < states; ++z) sum[z] = 0.f;
#pragma unroll
      for (int y = 0; y < 4; ++y) sum[y / (4 / states)] += l[y] == -INFINITY ? 0.f : exp2_hw(u[y] - l[y]);
#pragma unroll
      for (int z = 1; z < lanes; z <<= 1) sum[0] += __shfl_xor_sync(0xFFFFFFFFu, sum[0], z);
#pragma unroll
      for (int z = 0; z < states; ++z)
        if (j + z < j_end && quad == 0) weight[j + z] = fmaf(decay, w[x][z], sum[z]);
    }
  }
}

template <int DH>
__global__ void __launch_bounds__(kEndThreads, kEndOcc) paged_end_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int per = DH / 8, at_once = kEndThreads / per;  // threads of a piece's row, pieces at once
  __shared__ float fin[16];
  __shared__ float part[at_once][DH + 4];
  __shared__ long long room[kEndThreads / 32 + 2];
  __shared__ int found;
  const int warp = warp_id(), lane = lane_id();
  const int p = blockIdx.x % a.ends, head = blockIdx.x / a.ends;
  const int b = head / a.Hkv, kvh = head - b * a.Hkv;
  const int count = a.pages.clamp(a.lens[b]), n = a.chunks(b);
  // this CTA's states
  const int share = ((count + a.ends - 1) / a.ends + 3) / 4 * 4, j_first = p * share, j_end = min(j_first + share, count);
  // pieces of a unit: slots first .. first + pieces - 1
  Shares s{};
  if (a.shares) s = look_up<kEndThreads>(a, 0, b, room, found);
  grid_dep_wait();
  for (int block = 0; block < a.blocks; ++block) {
    const int r0 = block * 16, rows = min(16, a.rows - r0), unit = kvh * a.blocks + block;
    long long first = (long long)b * a.units() + unit, cta = 0;
    int pieces = 1;
    if (a.shares) {
      const long long from = s.before * a.units() + (long long)unit * n;
      cta = from / s.each;
      pieces = n == 0 ? 0 : (int)((from + n - 1) / s.each - cta) + 1;
      first += cta;
    }
    __syncthreads();
    for (int r = warp; r < 16; r += kEndThreads / 32) {
      if (r >= rows) {
        if (lane == 0) fin[r] = -INFINITY;
        continue;
      }
      float top = -INFINITY, sum = 0.f;
      for (int x = lane; x < pieces; x += 32) {
        const float u = a.part_l[(first + x) * a.part_rows + r], t = max3(top, u, u);
        if (t != -INFINITY) sum = sum * (top == t ? 1.f : exp2_hw(top - t)) + (u == t ? 1.f : exp2_hw(u - t));
        top = t;
      }
#pragma unroll
      for (int x = 16; x; x >>= 1) {
        const float u = __shfl_xor_sync(0xFFFFFFFFu, top, x), y = __shfl_xor_sync(0xFFFFFFFFu, sum, x), t = max3(top, u, u);
        if (t != -INFINITY) sum = sum * (top == t ? 1.f : exp2_hw(top - t)) + y * (u == t ? 1.f : exp2_hw(u - t));
        top = t;
      }
      if (lane == 0) fin[r] = top == -INFINITY ? -INFINITY : top + log2f(sum);
    }
    __syncthreads();
    if (pieces != 1) {
      for (int r = (p + a.ends - r0 % a.ends) % a.ends; r < rows; r += a.ends) {  // rows p, p + ends, ... of all
        const float l = fin[r];
        const int c = threadIdx.x % per * 8;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
        for (int x = threadIdx.x / per; x < pieces; x += at_once) {
          const float ls = a.part_l[(first + x) * a.part_rows + r];
          if (ls == -INFINITY) continue;
          const float k = exp2_hw(ls - l);
          float v[8];
          const long long place = 2 * (cta + x) + (x == 0);  // the first of them goes on behind its CTA
          unpack8(load_raw8(a.part_o, SB_F32, (place * a.part_rows + r) * DH + c), SB_F32, v);
#pragma unroll
          for (int u = 0; u < 8; ++u) f[u] = fmaf(fabsf(v[u]) == INFINITY ? 1.f : k, v[u], f[u]);  // (however small its share)
        }
        float4* to = reinterpret_cast<float4*>(&part[threadIdx.x / per][c]);
        to[0] = make_float4(f[0], f[1], f[2], f[3]);
        to[1] = make_float4(f[4], f[5], f[6], f[7]);
        __syncthreads();
        if (threadIdx.x < DH / 2) {  // two channels a thread
          float x = 0.f, y = 0.f;
          const int some = min(at_once, pieces);
          for (int z = 0; z < some; ++z) {
            x += part[z][2 * threadIdx.x];
            y += part[z][2 * threadIdx.x + 1];
          }
          const Row q(a, kvh, r0 + r);
          uint16_t* o = static_cast<uint16_t*>(a.o.p) + b * a.o.img + q.t * a.o.row + (long long)q.h * DH;
          reinterpret_cast<uint32_t*>(o)[threadIdx.x] = pack_pair(x, y, a.q_bf16 ? SB_BF16 : SB_F16);
          if (threadIdx.x == 0 && a.lse) a.lse[((long long)b * a.H + q.h) * a.Tq + q.t] = l * 0.69314718055994531f;
        }
        __syncthreads();
      }
    }
    if (!a.weight) continue;
    float* const weight = a.weight + (long long)head * a.pages.cap;
    const float4* const scores = reinterpret_cast<const float4*>(a.plane(head, block));
    const float decay = block == 0 ? a.decay : 1.f;
    if (a.score_rows == 1) account<1>(scores, fin, weight, decay, j_first, j_end);
    else if (a.score_rows == 2) account<2>(scores, fin, weight, decay, j_first, j_end);
    else if (a.score_rows == 4) account<4>(scores, fin, weight, decay, j_first, j_end);
    else if (a.score_rows == 8) account<8>(scores, fin, weight, decay, j_first, j_end);
    else account<16>(scores, fin, weight, decay, j_first, j_end);
  }
}

// The account of a call without queries, `ends` CTAs an (item, key head): decay times the weight of the states that are there.
__global__ void __launch_bounds__(kEndThreads) paged_age_kernel(const __grid_constant__ PagedArgs a) {
  const int part = blockIdx.x % a.ends, head = blockIdx.x / a.ends, count = a.pages.clamp(a.lens[head / a.Hkv]);
  float* const weight = a.weight + (long long)head * a.pages.cap;
  for (int j = part * kEndThreads + (int)threadIdx.x; j < count; j += a.ends * kEndThreads) weight[j] *= a.decay;
}

template <int DH, int PT>
void shape_of(int rows, int& chunk, int& occ) {
  chunk = rows <= 8 ? Paged<DH, PT, 1>::CK : Paged<DH, PT, 2>::CK;
  occ = rows <= 8 ? Paged<DH, PT, 1>::OCC : Paged<DH, PT, 2>::OCC;
}
template <int DH>
void shape_of(int pt, int rows, int& chunk, int& occ) {
  return pt == SB_F8     ? shape_of<DH, SB_F8>(rows, chunk, occ)
         : pt == SB_BF16 ? shape_of<DH, SB_BF16>(rows, chunk, occ) : shape_of<DH, SB_F16>(rows, chunk, occ);
}

struct PagedPlan {
  int rows, blocks, shares, cluster, ends, chunk, part_rows, places, score_rows;
  bool held;  // scores in shared memory
  long long units, scores, part_o, part_l;  // floats of the workspace
  long long bytes() const { return (scores + part_o + part_l) * 4; }
};

// Either a CTA or a cluster of up to eight a unit, and one kernel; or as many CTAs as are resident at once share all chunks
// evenly, whatever the items' lengths, and a second kernel joins the pieces.  What they take is estimated from
// the places (lengths are on the device): a CTA of a unit about 3 us to start and end (5 in a cluster) and 6 ns and 35 ps a
// byte for a state; shared chunks 14 us for both kernels and the rate of all.  Measured, us in kernels, for a CTA a unit, the
// cluster taken, and shared chunks: 2 x 8 units of 1000, 2000, 4000, 8000 states of 32 channels 12, 8, 20; 21, 9, 18;
// 40, 12, 18; 83, 16, 19; 1 x 4 of 512, 1024, 2048, 4096 of 128 14, 8, 15; 25, 10, 14; 47, 12, 14; -, 18, 14; 64 x 4 of
// 1024, 2048, 8160 30, -, 38; 54, -, 54; 203, -, 171; 640 x 4 of 1000 of 64 142, -, 127.
PagedPlan paged_plan(int B, int H, int Hkv, int dh, int Tq, int pt, int cap, bool account, int sms) {
  PagedPlan p{};
  int occ;
  p.rows = H / Hkv * Tq;
  if (dh == 32) shape_of<32>(pt, p.rows, p.chunk, occ);
  else if (dh == 64) shape_of<64>(pt, p.rows, p.chunk, occ);
  else shape_of<128>(pt, p.rows, p.chunk, occ);
  p.blocks = (p.rows + 15) / 16;
  p.part_rows = std::min(p.rows, 16);
  p.units = (long long)B * Hkv * p.blocks;
  const long long resident = (long long)occ * sms;
  const double unit_us = 2.0 * cap * dh * page_dtype_bytes(pt) / 6.2e6;  // at the rate of all
  const double state_us = 0.006 + 35e-6 * 2.0 * dh * page_dtype_bytes(pt);
  double best = 1e300;
  for (int c = 1; c <= 8; c *= 2) {
    if (c > 1 && cap < c * kWarps * p.chunk) break;  // a chunk a warp
    const double us = (double)((p.units * c + resident - 1) / resident) * ((c > 1 ? 5.0 : 3.0) + cap * state_us / c);
    if (us < best) {
      best = us;
      p.cluster = c;
    }
  }
  const bool apart = best > 14.0 + p.units * unit_us;
  p.shares = apart ? (int)resident : 0;
  if (apart) p.cluster = 1;
  account = account && cap > 0;
  // one wave of the last kernel's CTAs, each with 256 places or a row
  const long long heads = (long long)B * Hkv, wave = std::max(1ll, (long long)kEndOcc * sms / std::max(heads, 1ll));
  if (account && (apart || p.blocks > 1)) p.ends = (int)std::min(wave, ((long long)cap + 255) / 256);
  else if (apart) p.ends = (int)std::min(wave, (long long)p.rows);
  auto even = [](long long n) { return (n + 3) / 4 * 4; };
  p.places = (cap + 3) / 4 * 4;
  for (p.score_rows = 1; p.score_rows < p.part_rows;) p.score_rows *= 2;
  const int chunks = (cap + p.chunk - 1) / p.chunk, most = (chunks + p.cluster - 1) / p.cluster * p.chunk;  // of a CTA
  p.held = account && p.ends == 0 && (p.cluster > 1 ? most : p.places) * p.score_rows <= kHeldScores;
  p.scores = account && !p.held ? (long long)B * Hkv * p.blocks * p.places * p.score_rows : 0;
  p.part_l = p.ends > 0 ? even((p.units + p.shares) * p.part_rows) : 0;
  p.part_o = 2ll * p.shares * p.part_rows * dh;
  return p;
}

template <int DH, int PT, int NB>
cudaError_t launch(const PagedArgs& a, long long ctas, cudaStream_t st) {
  static bool ready[64];
  constexpr int room = Paged<DH, PT, NB>::SMEM, scores = kHeldScores * 4, rows = 8 * NB * DH * 4;
  auto* const kernel = paged_attend_kernel<DH, PT, NB>;
  const cudaError_t e = xattn_smem(reinterpret_cast<const void*>(kernel), room + scores + rows, ready);
  if (e != cudaSuccess) return e;
  const int bytes = room + (a.cluster > 1 ? scores + rows : a.weight && !a.scores ? scores : 0);
  return launch_after(kernel, ctas, kWarps * 32, (size_t)bytes, st, a, a.cluster, false);
}
// One column tile for up to eight rows: e4m3 above 83 us and with two tiles 116, fp16 heads of 32 158 and 162, bf16 heads of
// 128, which wait for memory alone, 156 and 152.
template <int DH, int PT>
cudaError_t launch(const PagedArgs& a, long long ctas, cudaStream_t st) {
  return a.rows <= 8 ? launch<DH, PT, 1>(a, ctas, st) : launch<DH, PT, 2>(a, ctas, st);
}
template <int DH>
cudaError_t launch(const PagedArgs& a, int pt, long long ctas, long long ends, cudaStream_t st) {
  const cudaError_t e = pt == SB_F8     ? launch<DH, SB_F8>(a, ctas, st)
                        : pt == SB_BF16 ? launch<DH, SB_BF16>(a, ctas, st) : launch<DH, SB_F16>(a, ctas, st);
  return e != cudaSuccess || ends == 0 ? e : launch_after(paged_end_kernel<DH>, ends, kEndThreads, 0, st, a);
}

bool paged_attention_sizes_ok(int B, int H, int Hkv, int dh, int Tq, int P, int page, int N) {
  return paged_sizes_ok(B, Hkv, dh, P, page, N) && H >= 1 && H % Hkv == 0 && (long long)H * dh <= 65536 && Tq >= 0 &&
         (long long)(H / Hkv) * Tq < (1ll << 30) && (long long)B * H * Tq < (1ll << 33);
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_paged_attention_work(int B, int H, int Hkv, int dh, int Tq, int page_dtype, int page, int N, int account,
                                       long long* bytes) {
  if (!bytes || !paged_attention_sizes_ok(B, H, Hkv, dh, Tq, 0, page, N) || !page_dtype_ok(page_dtype))
    return record_error(SB_EINVAL, "sb_paged_attention_work: arguments");
  *bytes = 0;
  if (B == 0 || Tq == 0) return SB_OK;
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_attention_work: device");
  *bytes = paged_plan(B, H, Hkv, dh, Tq, page_dtype, N * page, account != 0, sms).bytes();
  return SB_OK;
}

extern "C" int sb_paged_attention(const sb_paged_attend* call, void* stream) {
  if (!call) return record_error(SB_EINVAL, "sb_paged_attention: null argument");
  const sb_paged_attend& c = *call;
  const sb_paged_memory* const m = &c.memory;
  const int H = c.H, Tq = c.Tq;
  if (!paged_memory_ok(m) || !paged_attention_sizes_ok(m->B, H, m->Hkv, m->dh, Tq, m->P, m->page, m->N) ||
      (c.q_dtype != SB_F16 && c.q_dtype != SB_BF16) || (m->dtype != c.q_dtype && m->dtype != SB_F8))
    return record_error(SB_EINVAL, "sb_paged_attention: sizes (dh 32, 64 or 128, H a multiple of Hkv) or dtypes");
  if (!(c.scale > 0.f) || !scales_ok(m, c.k_scale, c.v_scale) || !std::isnormal(c.scale * c.k_scale * 1.4426950408889634f))
    return record_error(SB_EINVAL, "sb_paged_attention: scale, or scales of pages that are not e4m3");
  if (c.weight && !(c.decay >= 0.f && c.decay <= 1.f)) return record_error(SB_EINVAL, "sb_paged_attention: decay from 0 to 1");
  if (m->B == 0 || (Tq == 0 && (!c.weight || m->N == 0))) return SB_OK;
  if (Tq == 0 && c.lens) {
    PagedArgs a{};
    a.pages = page_table(m);
    a.lens = c.lens; a.Hkv = m->Hkv; a.weight = c.weight; a.decay = c.decay;
    const long long heads = (long long)m->B * m->Hkv;
    a.ends = (int)std::min((a.pages.cap + kEndThreads - 1ll) / kEndThreads, std::max(1ll, 2048 / heads));
    const cudaError_t e = launch_after(paged_age_kernel, heads * a.ends, kEndThreads, 0, static_cast<cudaStream_t>(stream), a, 1, false);
    return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
  }
  if (!c.lens || !xattn_view_ok(c.q, c.q_row, c.q_img) || !xattn_view_ok(c.out, c.out_row, c.out_img) || !paged_pools_ok(m))
    return record_error(SB_EINVAL, "sb_paged_attention: rows (16-byte aligned, strides multiples of 16 bytes) or null argument");
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_attention: device");
  PagedArgs a{};
  a.pages = page_table(m);
  const PagedPlan p = paged_plan(m->B, H, m->Hkv, m->dh, Tq, m->dtype, a.pages.cap, c.weight != nullptr, sms);
  if (p.bytes() > 0 && (!c.work || c.work_bytes < p.bytes() || (reinterpret_cast<uintptr_t>(c.work) & 15) != 0))
    return record_error(SB_EINVAL, "sb_paged_attention: workspace (sb_paged_attention_work bytes, 16-byte aligned)");
  const long long ctas = p.shares ? p.shares : p.units * p.cluster, ends = (long long)p.ends * m->B * m->Hkv;
  if (ctas > 0x7FFFFFFFll || ends > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_paged_attention: too many items");
  a.q = c.q; a.q_row = c.q_row; a.q_img = c.q_img;
  a.k = k_pool(m);
  a.v = v_pool(m);
  a.lens = c.lens;
  a.B = m->B; a.H = H; a.Hkv = m->Hkv; a.group = H / m->Hkv; a.Tq = Tq;
  a.rows = p.rows; a.blocks = p.blocks; a.shares = p.shares; a.cluster = p.cluster; a.ends = p.ends; a.chunk = p.chunk; a.part_rows = p.part_rows;
  a.places = p.places; a.score_rows = p.score_rows;
  a.q_bf16 = c.q_dtype == SB_BF16; a.causal = c.causal != 0;
  a.scale_log2 = c.scale * c.k_scale * 1.4426950408889634f;
  a.v_scale = c.v_scale;
  a.o = {c.out, c.out_row, c.out_img};
  a.lse = c.lse;
  a.weight = p.scores > 0 || p.held ? c.weight : nullptr;  // (no places: no account)
  a.decay = c.decay;
  float* w = static_cast<float*>(c.work);
  a.scores = p.scores > 0 ? w : nullptr;
  a.part_l = w + p.scores;
  a.part_o = a.part_l + p.part_l;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = m->dh == 32   ? launch<32>(a, m->dtype, ctas, ends, st)
                        : m->dh == 64 ? launch<64>(a, m->dtype, ctas, ends, st) : launch<128>(a, m->dtype, ctas, ends, st);
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}
