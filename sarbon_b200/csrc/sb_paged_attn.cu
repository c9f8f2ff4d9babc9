// sb_paged_attn.cu -- attention of new tokens over a paged memory:
//   s_rj = scale q_r . k_j,  out_r = sum_j p_rj v_j,  p_rj = e^(s_rj - L_r),  L_r = log sum_j e^s_rj,
// and, where the memory keeps account of what is looked at, weight_j = decay weight_j + sum_r p_rj.
//
// K and V are read once and memory bounds it, so each warp works alone on its own chunks of states (4 KB of
// K and of V, 16 to 64 states): cp.async brings their rows, wherever their pages lie, into the warp's own ring,
// which copes with any page size and costs no barrier; states that take no part arrive as zeros.  The
// products are mma.sync m16n8k16 with the states as the 16 rows of S^T = K Q^T and the channels as those of
// O^T = V^T P^T: one token's query heads (up to eight a key head) are then one column tile, half of what the
// rows of S = Q K^T would take, and movmatrix turns P^T around in registers.  e4m3 pages are widened to fp16
// in registers; the channels' order inside a step is free, so it is the one that the bytes lie in.  P is
// multiplied as the sum of two 16-bit halves: a product more, and the tensor pipe has room for it.
//
// The states of an (item, key head) are split over CTAs; fp32 partial rows are joined by a second kernel.
// The account needs L, which is there only after the last split, so the scores are kept (fp32) and a last kernel
// reads them back: 8 bytes a state and row against 4 dim bytes of K and V; a call of one split does it itself.
#include <algorithm>
#include <cmath>

#include "sb_paged.cuh"

namespace sb {
namespace {

constexpr int kWarps = 4;
constexpr int kRing = 24 * 1024;  // bytes a warp

struct PagedArgs {
  const void* q;
  long long q_row, q_img;  // elements
  Pool k, v;
  PageTable pages;
  const int* lens;
  int B, H, Hkv, group, Tq, rows, blocks, splits;  // rows = group * Tq of an (item, key head), blocks of 16
  int q_bf16, causal;
  float scale_log2, v_scale;  // scale * k_scale * log2(e)
  OutView o;
  float* lse;
  float* weight;
  float decay;
  float* scores;  // [B * Hkv][cap][rows], log2 units
  float* part_o;  // [splits][B * H * Tq][dh]
  float* part_l;  // [splits][B * H * Tq], log2 of the sum
  float* log_sum;  // [B * H * Tq], log2
  long long all_rows;
};

template <int DH, int PT>
struct Paged {
  static constexpr bool E4M3 = PT == SB_F8, BF16 = PT == SB_BF16;
  static constexpr int RB = DH * (E4M3 ? 1 : 2);                // bytes a state and head
  static constexpr int CK = 4096 / RB < 64 ? 4096 / RB : 64;    // states a chunk
  static constexpr int HALF = CK * RB, STAGE = 2 * HALF, STAGES = kRing / STAGE;
  static constexpr int LANES = RB / 16, AT_ONCE = 32 / LANES;   // lanes a row, rows a copy
  static constexpr int PITCH = DH + 4;                          // floats a row of the warps' outputs
  static constexpr int SMEM = kWarps * kRing;
  static_assert(kWarps * 16 * PITCH * 4 <= SMEM && STAGES >= 3, "ring");
  // byte of 16-byte chunk c of a row: eight rows of a chunk fall in distinct banks
  SB_DEV static uint32_t at(int row, int c) {
    const int x = RB >= 128 ? row & 7 : RB == 64 ? (row >> 1) & 3 : (row >> 2) & 1;
    return row * RB + ((c ^ x) << 4);
  }
};

SB_DEV void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
SB_DEV void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
SB_DEV void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool BF16>
SB_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
SB_DEV void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
SB_DEV void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// An 8 x 8 matrix of 16-bit values, a pair of a row a thread, turned around.
SB_DEV uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// Two e4m3 codes as two fp16 values (exact)
SB_DEV uint32_t widen(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  return (uint32_t)h.x | (uint32_t)h.y << 16;
}

// Query row r of an (item, key head): token r / group, head r % group.
struct Row {
  int t, h;
  SB_DEV Row(const PagedArgs& a, int kvh, int r) : t(r / a.group), h(kvh * a.group + r - t * a.group) {}
};

// NB: column tiles of eight query rows
template <int DH, int PT, int NB>
__global__ void __launch_bounds__(kWarps * 32, 2) paged_attend_kernel(const __grid_constant__ PagedArgs a) {
  using C = Paged<DH, PT>;
  constexpr bool E4M3 = C::E4M3, BF16 = C::BF16;
  constexpr int CK = C::CK, KT = CK / 16, KS = DH / 16, R = CK > 32 ? 2 : 1;
  constexpr float lift = kLift<BF16>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ longlong2 place[kWarps][CK];       // where a chunk's rows lie in the pools; -1: nowhere
  __shared__ uint64_t there[kWarps][C::STAGES];  // a stage's rows that take part, as bits
  __shared__ float2 ml[kWarps][16];
  __shared__ float fin[16];
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, tig = lane & 3;
  int idx = blockIdx.x;
  const int block = idx % a.blocks;
  idx /= a.blocks;
  const int split = idx % a.splits;
  idx /= a.splits;
  const int kvh = idx % a.Hkv, b = idx / a.Hkv, unit = idx;
  const int r0 = block * 16, rows = min(16, a.rows - r0);
  const int count = a.pages.clamp(a.lens[b]);
  // the item's own states are split evenly, in whole chunks
  const int chunks = (count + CK - 1) / CK, each = (chunks + a.splits - 1) / a.splits;
  const int first = min(split * each, chunks), n = min(first + each, chunks) - first;
  const int mine = n > warp ? (n - warp + kWarps - 1) / kWarps : 0;  // chunks first + warp, + kWarps ...
  uint8_t* const ring = smem + warp * kRing;
  const uint32_t ring_at = smem_u32(ring);
  const uint8_t* const kp = a.k.p + (long long)kvh * C::RB;
  const uint8_t* const vp = a.v.p + (long long)kvh * C::RB;

  // table entries of the next chunk to be copied, asked for a chunk ahead
  int entry[R];
  uint32_t within[R];
  auto ask = [&](int i) {
#pragma unroll
    for (int x = 0; x < R; ++x) {
      const int r = lane + 32 * x, j = (first + warp + i * kWarps) * CK + r;
      entry[x] = -1;
      within[x] = 0;
      if (r < CK && i < mine && j < count) entry[x] = a.pages.entry(b, (uint32_t)j, within[x]);
    }
  };
  auto copy = [&](int i) {  // the warp's chunk i, whose entries are there
    if (i < mine) {
      const int st = i % C::STAGES;
      uint64_t bits = 0;
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const bool ok = a.pages.has(entry[x]);
        const long long w = within[x], e = entry[x];
        if (lane + 32 * x < CK)
          place[warp][lane + 32 * x] = ok ? make_longlong2(e * a.k.page + w * a.k.row, e * a.v.page + w * a.v.row)
                                          : make_longlong2(-1, -1);
        bits |= (uint64_t)__ballot_sync(0xFFFFFFFFu, ok) << (32 * x);
      }
      if (lane == 0) there[warp][st] = bits;
      __syncwarp();
      const int c = lane % C::LANES;
      const uint32_t dst = ring_at + st * C::STAGE;
#pragma unroll
      for (int x = 0; x < CK / C::AT_ONCE; ++x) {
        const int r = x * C::AT_ONCE + lane / C::LANES;
        const longlong2 from = place[warp][r];
        const bool ok = from.x >= 0;
        const uint32_t to = dst + C::at(r, c);
        copy16(to, ok ? kp + from.x + c * 16 : static_cast<const uint8_t*>(a.q), ok);
        copy16(to + C::HALF, ok ? vp + from.y + c * 16 : static_cast<const uint8_t*>(a.q), ok);
      }
    }
    copies_done();
  };
  ask(0);
#pragma unroll 1
  for (int i = 0; i < C::STAGES; ++i) {
    copy(i);
    ask(i + 1);
    __syncwarp();  // place is written again
  }

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
      up = e == 0 || e == 255 ? 0 : min(max(140 - e, -126), 126);
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
      factor[y][x] = a.scale_log2 * __uint_as_float((uint32_t)(127 - down) << 23);
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
  float* const scores = a.scores ? a.scores + (long long)unit * a.pages.cap * a.rows + r0 : nullptr;

  for (int i = 0; i < mine; ++i) {
    copies_wait<C::STAGES - 1>();
    __syncwarp();
    const int st = i % C::STAGES, j0 = (first + warp + i * kWarps) * CK;
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
            const uint32_t w[4] = {widen(f[2 * z] & 0xFFFFu), widen(f[2 * z + 1] & 0xFFFFu), widen(f[2 * z] >> 16),
                                   widen(f[2 * z + 1] >> 16)};
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
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int j = j0 + kt * 16 + g + 8 * x;
          if (j < count) {
#pragma unroll
            for (int y = 0; y < NB; ++y) {
              const int r = 8 * y + 2 * tig;
              float* to = scores + (long long)j * a.rows + r;
              const float u = s[kt][y][2 * x] * factor[y][0], w = s[kt][y][2 * x + 1] * factor[y][1];
              if (a.rows % 2 == 0) {
                if (r < rows) *reinterpret_cast<float2*>(to) = make_float2(u, w);
              } else {
                if (r < rows) to[0] = u;
                if (r + 1 < rows) to[1] = w;
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
            const float u = s[kt][y][2 * x], w = s[kt][y][2 * x + 1];
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
              const uint32_t u = __byte_perm(f[2 * z], 0, 0x3120), v = __byte_perm(f[2 * z + 1], 0, 0x3120);
              const uint32_t w[4] = {widen(u & 0xFFFFu), widen(u >> 16), widen(v & 0xFFFFu), widen(v >> 16)};
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
              p[y][z] = __shfl_sync(0xFFFFFFFFu, k < 8 ? s[kt][y][z] : s[kt][y][2 + z], (k & 7) * 4 + tig);
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
    copy(i + C::STAGES);
    ask(i + C::STAGES + 1);
    __syncwarp();
  }
  copies_wait<0>();
#pragma unroll
  for (int y = 0; y < NB; ++y)
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[y][z] += __shfl_xor_sync(0xFFFFFFFFu, l[y][z], x);
  // the warps' outputs meet in shared memory, rows [warp][8 NB][PITCH], over the rings; maxima as exponents of 2
  __syncthreads();
  float* all_o = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int x = 0; x < KS; ++x)
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const int c = E4M3 ? x * 16 + 2 * g + (z >> 1) : x * 16 + g + 8 * (z >> 1);
        all_o[(warp * 8 * NB + 8 * y + 2 * tig + (z & 1)) * C::PITCH + c] = o[x][y][z];
      }
  if (g == 0) {
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int z = 0; z < 2; ++z)
        ml[warp][8 * y + 2 * tig + z] = make_float2(m[y][z] == -INFINITY ? -INFINITY : m[y][z] * factor[y][z], l[y][z]);
  }
  __syncthreads();
  constexpr int per = DH / 8;
  for (int i = threadIdx.x; i < rows * per; i += kWarps * 32) {
    const int r = i / per, c = (i - r * per) * 8;
    float top = -INFINITY, sum = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max3(top, ml[w][r].x, ml[w][r].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = ml[w][r].x, k = mw == top ? 1.f : exp2_hw(mw - top);
      sum = fmaf(k, ml[w][r].y, sum);
      const float4* src = reinterpret_cast<const float4*>(all_o + (w * 8 * NB + r) * C::PITCH + c);
      const float4 x = src[0], y = src[1];
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] = fmaf(k, v[u], f[u]);
    }
    const bool none = top == -INFINITY;  // no states
    const float inv = none ? 0.f : a.v_scale / sum;
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] = none ? 0.f : f[u] * inv;
    const float log_sum = none ? -INFINITY : top - lift + log2f(sum);
    const Row w(a, kvh, r0 + r);
    const long long rr = ((long long)b * a.H + w.h) * a.Tq + w.t;
    if (a.splits > 1) {
      if (!none) store8(a.part_o, SB_F32, (split * a.all_rows + rr) * DH + c, f);
      if (c == 0) a.part_l[split * a.all_rows + rr] = log_sum;
    } else {
      store8(a.o.p, a.q_bf16 ? SB_BF16 : SB_F16, b * a.o.img + w.t * a.o.row + (long long)w.h * DH + c, f);
      if (c == 0) {
        if (a.lse) a.lse[rr] = log_sum * 0.69314718055994531f;
        if (a.log_sum) a.log_sum[rr] = log_sum;
        fin[r] = log_sum;
      }
    }
  }
  if (a.weight && a.splits == 1 && a.blocks == 1) {  // all of the scores and sums are this CTA's own
    __syncthreads();
    float* weight = a.weight + (long long)unit * a.pages.cap;
    for (int j = threadIdx.x; j < count; j += kWarps * 32) {
      float w = 0.f;
      for (int r = 0; r < rows; ++r)
        if (fin[r] != -INFINITY) w += exp2_hw(scores[(long long)j * a.rows + r] - fin[r]);
      weight[j] = fmaf(a.decay, weight[j], w);
    }
  }
}

// Joins the splits' rows: out = sum_s 2^(L_s - L) O_s, L = log2 sum_s 2^L_s.  A warp takes a row: its lanes
// find the largest L_s, then take eight channels each of several splits at once.  A split without states
// (L_s = -inf) has not written its O_s.
template <int DH>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int per = DH / 8, lanes = 32 / per;  // threads of a split's row, splits at once
  const int lane = lane_id();
  const long long rr = (long long)blockIdx.x * 4 + warp_id();
  if (rr >= a.all_rows) return;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) {
    const float u = a.part_l[s * a.all_rows + rr];
    top = max3(top, u, u);
  }
#pragma unroll
  for (int x = 16; x; x >>= 1) {
    const float u = __shfl_xor_sync(0xFFFFFFFFu, top, x);
    top = max3(top, u, u);
  }
  const int c = lane % per * 8, s0 = lane / per;
  float f[9] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // channels, sum of weights
#pragma unroll 4
  for (int s = s0; s < a.splits; s += lanes) {
    const float ls = a.part_l[s * a.all_rows + rr];
    if (ls == -INFINITY) continue;
    const float w = exp2_hw(ls - top);
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
  store8(a.o.p, a.q_bf16 ? SB_BF16 : SB_F16, b * a.o.img + t * a.o.row + (long long)h * DH + c, v);
  if (c == 0) {
    const float log_sum = f[8] != 0.f ? top + log2f(f[8]) : -INFINITY;
    if (a.lse) a.lse[rr] = log_sum * 0.69314718055994531f;
    if (a.log_sum) a.log_sum[rr] = log_sum;
  }
}

// weight = decay weight + sum over the rows of 2^(score - L): a thread a state.
__global__ void __launch_bounds__(256) paged_account_kernel(const __grid_constant__ PagedArgs a) {
  const int parts = (a.pages.cap + 255) / 256;
  const int unit = blockIdx.x / parts, j = (blockIdx.x - unit * parts) * 256 + threadIdx.x;
  const int b = unit / a.Hkv, kvh = unit - b * a.Hkv;
  if (j >= a.pages.clamp(a.lens[b])) return;
  const float* s = a.scores + ((long long)unit * a.pages.cap + j) * a.rows;
  float w = 0.f;
  for (int r = 0; r < a.rows; ++r) {
    const Row q(a, kvh, r);
    const float l = a.log_sum[((long long)b * a.H + q.h) * a.Tq + q.t];
    if (l != -INFINITY) w += exp2_hw(s[r] - l);
  }
  float* to = a.weight + (long long)unit * a.pages.cap + j;
  *to = fmaf(a.decay, *to, w);
}

struct PagedPlan {
  int rows, blocks, splits;
  bool apart;  // the account by a kernel of its own
  long long units, scores, part_o, part_l, sums;  // floats of the workspace
  long long bytes() const { return (scores + part_o + part_l + sums) * 4; }
};

PagedPlan paged_plan(int B, int H, int Hkv, int dh, int Tq, int cap, bool account, int sms) {
  PagedPlan p{};
  p.rows = H / Hkv * Tq;
  p.blocks = (p.rows + 15) / 16;
  p.units = (long long)B * Hkv * p.blocks;
  p.splits = few_splits(p.units, cap, sms);
  p.apart = account && (p.splits > 1 || p.blocks > 1);
  const long long all = (long long)B * H * Tq;
  auto even = [](long long n) { return (n + 3) / 4 * 4; };
  p.scores = account ? even((long long)B * Hkv * cap * p.rows) : 0;
  p.part_o = p.splits > 1 ? p.splits * all * dh : 0;
  p.part_l = p.splits > 1 ? even(p.splits * all) : 0;
  p.sums = p.apart ? even(all) : 0;
  return p;
}

template <int DH, int PT, int NB>
cudaError_t launch(const PagedArgs& a, long long ctas, cudaStream_t st) {
  static bool ready[64];
  const cudaError_t e = xattn_smem(reinterpret_cast<const void*>(&paged_attend_kernel<DH, PT, NB>), Paged<DH, PT>::SMEM, ready);
  if (e != cudaSuccess) return e;
  paged_attend_kernel<DH, PT, NB><<<(unsigned)ctas, kWarps * 32, Paged<DH, PT>::SMEM, st>>>(a);
  return cudaGetLastError();
}
template <int DH, int PT>
cudaError_t launch(const PagedArgs& a, long long ctas, cudaStream_t st) {
  return a.rows <= 8 ? launch<DH, PT, 1>(a, ctas, st) : launch<DH, PT, 2>(a, ctas, st);
}
template <int DH>
cudaError_t launch(const PagedArgs& a, int pt, long long ctas, cudaStream_t st) {
  const cudaError_t e = pt == SB_F8     ? launch<DH, SB_F8>(a, ctas, st)
                        : pt == SB_BF16 ? launch<DH, SB_BF16>(a, ctas, st) : launch<DH, SB_F16>(a, ctas, st);
  if (e != cudaSuccess || a.splits == 1) return e;
  paged_join_kernel<DH><<<(unsigned)((a.all_rows + 3) / 4), 128, 0, st>>>(a);
  return cudaGetLastError();
}

bool paged_attention_sizes_ok(int B, int H, int Hkv, int dh, int Tq, int P, int page, int N) {
  return paged_sizes_ok(B, Hkv, dh, P, page, N) && H >= 1 && H % Hkv == 0 && (long long)H * dh <= 65536 && Tq >= 0 &&
         (long long)(H / Hkv) * Tq < (1ll << 30) && (long long)B * H * Tq < (1ll << 33);
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_paged_attention_work(int B, int H, int Hkv, int dh, int Tq, int page, int N, int account, long long* bytes) {
  if (!bytes || !paged_attention_sizes_ok(B, H, Hkv, dh, Tq, 0, page, N))
    return record_error(SB_EINVAL, "sb_paged_attention_work: arguments");
  *bytes = 0;
  if (B == 0 || Tq == 0) return SB_OK;
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_attention_work: device");
  *bytes = paged_plan(B, H, Hkv, dh, Tq, N * page, account != 0, sms).bytes();
  return SB_OK;
}

extern "C" int sb_paged_attention(const void* q, long long q_row, long long q_img, int q_dtype, const void* k_pages,
                                  long long k_row, long long k_page, const void* v_pages, long long v_row,
                                  long long v_page, int page_dtype, int P, int page, const int* table, long long table_row,
                                  int N, const int* lens, int B, int H, int Hkv, int dh, int Tq, float scale, float k_scale,
                                  float v_scale, int causal, void* out, long long o_row, long long o_img, float* lse,
                                  float* weight, float decay, void* work, long long work_bytes, void* stream) {
  if (!paged_attention_sizes_ok(B, H, Hkv, dh, Tq, P, page, N) || (q_dtype != SB_F16 && q_dtype != SB_BF16) ||
      (page_dtype != q_dtype && page_dtype != SB_F8))
    return record_error(SB_EINVAL, "sb_paged_attention: sizes (dh 32, 64 or 128, H a multiple of Hkv) or dtypes");
  if (!(scale > 0.f) || !std::isfinite(scale) || !(k_scale > 0.f) || !std::isfinite(k_scale) || !(v_scale > 0.f) ||
      !std::isfinite(v_scale) || !std::isfinite(scale * k_scale) || (page_dtype != SB_F8 && (k_scale != 1.f || v_scale != 1.f)))
    return record_error(SB_EINVAL, "sb_paged_attention: scale, or scales of pages that are not e4m3");
  if (weight && !(decay >= 0.f && decay <= 1.f)) return record_error(SB_EINVAL, "sb_paged_attention: decay from 0 to 1");
  if (B == 0 || Tq == 0) return SB_OK;
  const int es = page_dtype_bytes(page_dtype);
  const bool some = P > 0 && N > 0;  // states there may be
  if (!lens || (N > 0 && (!table || table_row < 0)) || !xattn_view_ok(q, q_row, q_img) || !xattn_view_ok(out, o_row, o_img) ||
      (some && (!pool_ok(k_pages, k_row, k_page, es) || !pool_ok(v_pages, v_row, v_page, es))))
    return record_error(SB_EINVAL, "sb_paged_attention: rows (16-byte aligned, strides multiples of 16 bytes) or null argument");
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_paged_attention: device");
  const PagedPlan p = paged_plan(B, H, Hkv, dh, Tq, N * page, weight != nullptr, sms);
  if (p.bytes() > 0 && (!work || work_bytes < p.bytes() || (reinterpret_cast<uintptr_t>(work) & 15) != 0))
    return record_error(SB_EINVAL, "sb_paged_attention: workspace (sb_paged_attention_work bytes, 16-byte aligned)");
  const long long ctas = p.units * p.splits, parts = (N * (long long)page + 255) / 256 * B * Hkv;
  if (ctas > 0x7FFFFFFFll || parts > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_paged_attention: too many items");
  PagedArgs a{};
  a.q = q; a.q_row = q_row; a.q_img = q_img;
  a.k = pool_of(k_pages, k_row, k_page, es);
  a.v = pool_of(v_pages, v_row, v_page, es);
  a.pages = page_table(table, table_row, P, page, N);
  a.lens = lens;
  a.B = B; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.Tq = Tq; a.rows = p.rows; a.blocks = p.blocks; a.splits = p.splits;
  a.q_bf16 = q_dtype == SB_BF16; a.causal = causal != 0;
  a.scale_log2 = scale * k_scale * 1.4426950408889634f;
  a.v_scale = v_scale;
  a.o = {out, o_row, o_img};
  a.lse = lse;
  a.weight = p.scores > 0 ? weight : nullptr;  // (no places: no account)
  a.decay = decay;
  a.all_rows = (long long)B * H * Tq;
  float* w = static_cast<float*>(work);
  a.scores = p.scores > 0 ? w : nullptr;
  a.part_o = w + p.scores;
  a.part_l = a.part_o + p.part_o;
  a.log_sum = p.sums > 0 ? a.part_l + p.part_l : nullptr;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = dh == 32   ? launch<32>(a, page_dtype, ctas, st)
                  : dh == 64 ? launch<64>(a, page_dtype, ctas, st) : launch<128>(a, page_dtype, ctas, st);
  if (e == cudaSuccess && p.apart && parts > 0) {
    paged_account_kernel<<<(unsigned)parts, 256, 0, st>>>(a);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? SB_OK : record_error(SB_ECUDA, cudaGetErrorString(e));
}
