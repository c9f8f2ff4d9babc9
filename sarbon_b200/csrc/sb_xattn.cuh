// sb_xattn.cuh -- what the forward and backward attention kernels of the memory-reading block
// share: operand views, key masks as bits, tcgen05 forms and swizzled rows.
#pragma once
#include "sb_rows.cuh"

namespace sb {

struct View {
  const void* p;
  long long row, img;  // elements between rows, between items
};
struct OutView {
  void* p;
  long long row, img;
};

// Which keys of item b take part: j < lens[b] and valid[b * valid_img + j] != 0.
struct KeyMask {
  const int* lens;
  const uint8_t* valid;
  long long valid_img;
  int Tk;
  SB_DEV int count(int b) const { return lens ? min(max(lens[b], 0), Tk) : Tk; }
  // the item's row of valid, kept in registers by what uses it in a loop
  SB_DEV const uint8_t* row(int b) const { return valid ? valid + b * valid_img : nullptr; }
};

// Keys j0 .. j0 + 31 below n, as bits.
SB_DEV uint32_t bits_below(int j0, int n) {
  const int left = n - j0;
  return left >= 32 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << left) - 1u;
}
// A lane's byte of keys j0 .. j0 + 31 of row (KeyMask::row, not null) and, a tile later, the warp's
// bits: the bytes are on their way while another tile is worked on.
SB_DEV uint32_t ask_keys(const uint8_t* row, int j0, int n) {
  const int j = j0 + (int)lane_id();
  return j < n ? row[j] : 0u;
}
SB_DEV uint32_t told_keys(uint32_t byte) { return __ballot_sync(0xFFFFFFFFu, byte != 0); }

// Arguments of the forward kernels.
struct FwdArgs {
  View q;
  OutView o;
  float* lse;
  KeyMask mask;
  int B, H, Hkv, group, Tq, rows;  // rows = group * Tq of an (item, key head)
  int pairs, splits;               // CTAs a (item, key head) and split
  int k_item, v_item;              // 0: one memory for every item
  int masked;                      // lens or valid given: the cleaner runs
  float scale_log2;
  float* part_o;  // [splits][B * H * Tq][DH]
  float* part_l;  // [splits][B * H * Tq]
  long long all_rows;
};

// fp16 probabilities are held times 2^kLift: the reference point keeps them below 2^8, so fp16 has seven more
// powers of two above, and what a long memory's many small ones add up to is not lost (42,839 keys at
// 2^-25 of the one on top: 0 instead of 1.3e-3 without).  A value below 2^-14 is off by 2^-25, so Tk keys are
// off by Tk 2^-32 of the row's sum at most, less than fp16's own half step up to two million of them.
// The sum is taken of the same values, so the factor leaves with it.  bf16 has fp32's range.
template <bool BF16>
constexpr float kLift = BF16 ? 0.f : 7.f;

// ---------------------------------------------------------------- tcgen05 forms
// D[tmem] (+)= A[tmem] * B[smem]: A holds 16-bit pairs, k and k + 1 in a 32-bit column.
SB_DEV void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accum)
      : "memory");
}
// 32 lanes x 32 bit, 32 consecutive columns: thread i of the warp holds lane (base + i).
SB_DEV void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
SB_DEV void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
SB_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
SB_DEV void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
SB_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two fp32 values in one register pair: one instruction works on both.
SB_DEV uint64_t pair2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
SB_DEV void split2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
SB_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
SB_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SB_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The largest of three; NaN if one is.
SB_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
SB_DEV float exp2_hw(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One arrival for a warp.  The barrier after it matters: without it lanes 1 .. 31 may run ahead into the
// next wait, which suspends the warp for its whole time limit before lane 0 gets to arrive.
SB_DEV void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(bar);
  __syncwarp();
}

// Barrier `id` (1 ..) of 64 threads, two warps, with the OR of their predicates.
SB_DEV bool pair_or(int id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred.aligned q, %2, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)p), "r"(id)
      : "memory");
  return r != 0;
}

// ---------------------------------------------------------------- operand tiles in shared memory
// A tile of rows x DH 16-bit values lies as DH / COLS boxes of rows x COLS (COLS = min(DH, 64)),
// each row of a box SPAN = 2 COLS bytes, 16-byte chunks swizzled over SPAN bytes (the TMA modes
// SWIZZLE_128B and SWIZZLE_64B).  As a K-major operand (contraction over the channels) a step of
// 16 channels is 32 bytes inside a row; as an MN-major one (contraction over the rows) a step of 16
// rows is 16 SPAN bytes, and the next 64 channels are a box away.
template <int DH>
struct Tile {
  static constexpr int COLS = DH < 64 ? DH : 64;
  static constexpr int BOXES = DH / COLS;
  static constexpr int SPAN = COLS * 2;
  static constexpr uint32_t SWZ = SPAN == 128 ? 2u : 4u;
  static constexpr int KSTEPS = DH / 16;
  __host__ __device__ static constexpr int box_bytes(int rows) { return rows * SPAN; }
  __host__ __device__ static constexpr int bytes(int rows) { return rows * DH * 2; }

  // contraction over channels, step ks of 16
  SB_DEV static uint64_t k_major(uint32_t base, int rows, int ks) {
    constexpr int per = COLS / 16;
    return smem_desc(base + (ks / per) * box_bytes(rows) + (ks % per) * 32, SPAN * 8, SWZ);
  }
  // contraction over rows, step ks of 16
  SB_DEV static uint64_t mn_major(uint32_t base, int rows, int ks) {
    uint64_t d = smem_desc(base + ks * 16 * SPAN, SPAN * 8, SWZ);
    d &= ~((uint64_t)0x3FFF << 16);
    return d | (uint64_t)((box_bytes(rows) & 0x3FFFF) >> 4) << 16;
  }
  // byte offset of 16-byte chunk c (of DH / 8) of a row
  SB_DEV static uint32_t chunk(int rows, int row, int c) {
    constexpr int per = COLS / 8;
    const int box = c / per, x = c % per;
    const int s = SPAN == 128 ? x ^ (row & 7) : x ^ ((row >> 1) & 3);
    return box * box_bytes(rows) + row * SPAN + s * 16;
  }
};

// kind::f16 with fp32 accumulation: fp16 or bf16 operands, B K-major or (mn) MN-major
__host__ __device__ constexpr uint32_t idesc_16bit(bool bf16, int M, int N, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

template <bool BF16>
SB_DEV uint32_t pack16(float lo, float hi) {
  return pack_pair(lo, hi, BF16 ? SB_BF16 : SB_F16);
}

// ---------------------------------------------------------------- host
// One [B][T][heads * dh] operand as a 4-D tensor map; its box is `rows` rows of one head of one item, and
// rows past T arrive as zeros.  img = 0 (one memory for every item) makes the item dimension 1: kernels
// multiply the item by 0 then.
bool xattn_tensor_map(CUtensorMap* map, const View& v, int dtype, int B, int T, int heads, int dh, int rows);
bool xattn_sizes_ok(int dtype, int B, int H, int Hkv, int dh, int Tq, int Tk);
// 16-byte rows whose strides fit a tensor map; where one is made, several rows may not be one and the same
bool xattn_view_ok(const void* p, long long row, long long img);
bool xattn_map_ok(const void* p, long long row, long long img, int T);
// counts[b] = 1 + the last key of item b that takes part (0: none): keys behind it are never looked at.
constexpr long long counts_bytes(int masked, int B) { return masked ? ((long long)B * 4 + 15) / 16 * 16 : 0; }
cudaError_t count_keys(const KeyMask& mask, int B, int* counts, cudaStream_t st);
// Few query rows an (item, key head): the key splits of its kernel, its launch (partial rows where splits
// > 1), and the join of the partial rows.
constexpr int kFewRows = 16;
int few_splits(long long units, int Tk, int sms);
cudaError_t few_launch(const FwdArgs& a, int dh, bool bf16, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st);
int few_keys(int dh);  // rows of its tensor maps' boxes
cudaError_t few_join(const FwdArgs& a, int dh, bool bf16, cudaStream_t st);
// Sticky SB_ERR_* flags of the attention kernels, cleared on request.
int xattn_error(int clear, int* flags);  // 0, or -1 when the device could not be read
int xattn_back_error(int clear, int* flags);
int few_error(int clear, int* flags);
int gnorm_error(int clear, int* flags);  // of the gated norms
long long xattn_back_work(int B, int H, int Hkv, int dh, int Tq, int Tk, int sms);
// SMs of the current device, 0 on error
int xattn_sms();
// Lets `kernel` use `bytes` of dynamic shared memory on the current device, once a device (`ready`).
cudaError_t xattn_smem(const void* kernel, int bytes, bool (&ready)[64]);

}  // namespace sb
