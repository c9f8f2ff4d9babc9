// sb_rope.cu -- rotary positions with several axes (time, height, width).
//
// Pair p of a head is turned by angle(t, p) = pos[t, axis[p]] * freq[p]:
//   u' = u cos - v sin,  v' = u sin + v cos,
// and by the opposite angle for the gradient (the rotation's transpose).  A camera's frame
// numbers reach millions, where an fp32 product is off by a tenth of a radian, so the angle is
// taken in fp64 as turns (pos * freq / 2 pi), its whole turns are dropped there, and only the
// remainder in [-1/2, 1/2] goes to fp32 and to sincospi; what that rounds off, up to 1.6 2^-24 of an
// angle, is added to first order.
//
// A thread owns eight pairs of one token: it computes their sines and cosines once and applies
// them to every head of its chunk, so that the trigonometry is paid once a token and the pass is
// bound by reading and writing x.  The heads are split over blockIdx.y only where the tokens
// alone would leave SMs idle.  2 x 65,280 tokens of 8 x 128 channels in bf16: 90 us, 91 % of the copy rate;
// 3 x 8161 of 12 x 64 in fp32: 35 us, 66 % (one wave of CTAs, so starting and ending show).
#include <algorithm>

#include "sb_xattn.cuh"

namespace sb {
namespace {

struct RopeArgs {
  const void* x;
  long long x_row, x_img;
  void* out;
  long long o_row, o_img;
  const void* pos;
  long long pos_img;
  const double* freq;
  const int* axis;
  int dt, pos_f32, A, R, T, H, dh, heads_per, pairs, inverse, copy;
  long long units;  // B * T * slots
  int slots;        // threads a token: groups of pairs, then groups of channels to copy
};

// sine and cosine of pair p for token row `at` of pos
SB_DEV void turn_of(const RopeArgs& a, long long at, int p, float& sn, float& cs) {
  const int ax = a.axis[p];
  sn = 0.f;
  cs = 1.f;
  if (ax < 0 || ax >= a.A) return;
  const double where = a.pos_f32 ? (double)static_cast<const float*>(a.pos)[at + ax]
                                 : (double)static_cast<const int*>(a.pos)[at + ax];
  double turns = where * a.freq[p] * 0.15915494309189533576888;  // 1 / (2 pi)
  turns = 2.0 * (turns - rint(turns));
  const float near = (float)turns, rest = 3.14159265f * (float)(turns - (double)near);
  sincospif(near, &sn, &cs);
  const float s0 = sn;
  sn = fmaf(cs, rest, sn);
  cs = fmaf(-s0, rest, cs);
  if (a.inverse) sn = -sn;
}

constexpr int kAhead = 2;

// VEC: rows in vectors of eight, of type DT; otherwise element by element.  Four blocks an SM: with
// three, or the five that 48 registers allow, 5 to 50 % slower.
template <bool VEC, int DT>
__global__ void __launch_bounds__(256, 4) rope_kernel(const __grid_constant__ RopeArgs a) {
  const int dt = VEC ? DT : a.dt;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.units) return;
  int slot, t;
  long long b;
  if (a.units <= 0x7FFFFFFF) {  // a 64-bit division costs as much as a pair's trigonometry
    const uint32_t token = (uint32_t)i / (uint32_t)a.slots;
    slot = (int)((uint32_t)i - token * (uint32_t)a.slots);
    b = token / (uint32_t)a.T;
    t = (int)(token - (uint32_t)b * (uint32_t)a.T);
  } else {
    const long long token = i / a.slots;
    slot = (int)(i - token * a.slots);
    b = token / a.T;
    t = (int)(token - b * a.T);
  }
  const long long xr = b * a.x_img + t * a.x_row, orow = b * a.o_img + t * a.o_row;
  const long long at = b * a.pos_img + (long long)t * a.A;
  const int h0 = blockIdx.y * a.heads_per, h1 = min(a.H, h0 + a.heads_per);
  if constexpr (VEC) {
    const int groups = a.R >> 3;
    if (slot >= groups) {  // channels that no pair covers
      const int c = 2 * a.R + (slot - groups) * 8;
      for (int h = h0; h < h1; h += 2 * kAhead) {
        Raw8 r[2 * kAhead];
#pragma unroll
        for (int y = 0; y < 2 * kAhead; ++y)
          if (h + y < h1) r[y] = load_raw8(a.x, dt, xr + (long long)(h + y) * a.dh + c);
#pragma unroll
        for (int y = 0; y < 2 * kAhead; ++y)
          if (h + y < h1) store_raw8(a.out, dt, orow + (long long)(h + y) * a.dh + c, r[y]);
      }
      return;
    }
    const int p0 = slot * 8;
    float sn[8], cs[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) turn_of(a, at, p0 + u, sn[u], cs[u]);
    // the eight pairs' first and second vectors: (p0.., R + p0..) or the 16 channels from 2 p0 on
    const int c0 = a.pairs ? 2 * p0 : p0, c1 = a.pairs ? 2 * p0 + 8 : a.R + p0;
    // two heads' loads before the first store: x and out may be the same rows, so the compiler keeps
    // the order of what is written here
    for (int h = h0; h < h1; h += kAhead) {
      Raw8 r0[kAhead], r1[kAhead];
#pragma unroll
      for (int y = 0; y < kAhead; ++y)
        if (h + y < h1) {
          const long long xo = xr + (long long)(h + y) * a.dh;
          r0[y] = load_raw8(a.x, dt, xo + c0);
          r1[y] = load_raw8(a.x, dt, xo + c1);
        }
#pragma unroll
      for (int y = 0; y < kAhead; ++y) {
        if (h + y >= h1) break;
        const long long oo = orow + (long long)(h + y) * a.dh;
        float u[8], v[8], y0[8], y1[8];
        unpack8(r0[y], dt, u);
        unpack8(r1[y], dt, v);
        if (a.pairs) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            y0[2 * k] = u[2 * k] * cs[k] - u[2 * k + 1] * sn[k];
            y0[2 * k + 1] = u[2 * k] * sn[k] + u[2 * k + 1] * cs[k];
            y1[2 * k] = v[2 * k] * cs[4 + k] - v[2 * k + 1] * sn[4 + k];
            y1[2 * k + 1] = v[2 * k] * sn[4 + k] + v[2 * k + 1] * cs[4 + k];
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            y0[k] = u[k] * cs[k] - v[k] * sn[k];
            y1[k] = u[k] * sn[k] + v[k] * cs[k];
          }
        }
        store8(a.out, dt, oo + c0, y0);
        store8(a.out, dt, oo + c1, y1);
      }
    }
  } else {
    if (slot >= a.R) {
      const int c = 2 * a.R + slot - a.R;
      for (int h = h0; h < h1; ++h)
        put_one(a.out, a.dt, orow + (long long)h * a.dh + c, one_of(a.x, a.dt, xr + (long long)h * a.dh + c));
      return;
    }
    float sn, cs;
    turn_of(a, at, slot, sn, cs);
    const int c0 = a.pairs ? 2 * slot : slot, c1 = a.pairs ? 2 * slot + 1 : a.R + slot;
    for (int h = h0; h < h1; ++h) {
      const long long xo = xr + (long long)h * a.dh, oo = orow + (long long)h * a.dh;
      const float u = one_of(a.x, a.dt, xo + c0), v = one_of(a.x, a.dt, xo + c1);
      put_one(a.out, a.dt, oo + c0, u * cs - v * sn);
      put_one(a.out, a.dt, oo + c1, u * sn + v * cs);
    }
  }
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_rope_axes(const void* x, long long x_row, long long x_img, int dtype, int B, int T, int H, int dh,
                            const void* pos, int pos_f32, long long pos_img, int A, const double* freq, const int* axis, int R,
                            int pairs, int inverse, void* out, long long o_row, long long o_img, void* stream) {
  if (B < 0 || T < 0 || H < 1 || dh < 1 || A < 1 || R < 0 || 2 * (long long)R > dh || !rows_dtype_ok(dtype))
    return record_error(SB_EINVAL, "sb_rope_axes: sizes (2 R <= dh) or dtype");
  if (B == 0 || T == 0) return SB_OK;
  if (!x || !out || !pos || (R > 0 && (!freq || !axis))) return record_error(SB_EINVAL, "sb_rope_axes: null argument");
  if (x_row < 0 || x_img < 0 || o_row < 0 || o_img < 0 || pos_img < 0)
    return record_error(SB_EINVAL, "sb_rope_axes: negative strides");
  const int esz = dtype_bytes(dtype);
  auto aligned = [&](const void* p, long long row, long long img) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row * esz % 16 == 0 && img * esz % 16 == 0;
  };
  const bool vec = R % 8 == 0 && dh % 8 == 0 && aligned(x, x_row, x_img) && aligned(out, o_row, o_img);
  RopeArgs a{};
  a.x = x; a.x_row = x_row; a.x_img = x_img;
  a.out = out; a.o_row = o_row; a.o_img = o_img;
  a.pos = pos; a.pos_img = pos_img;
  a.freq = freq; a.axis = axis;
  a.dt = dtype; a.pos_f32 = pos_f32; a.A = A; a.R = R; a.T = T; a.H = H; a.dh = dh;
  a.pairs = pairs != 0; a.inverse = inverse != 0;
  a.copy = !(x == out && x_row == o_row && x_img == o_img);  // channels without a pair are there already when the rows are the same
  const int g = vec ? 8 : 1;
  a.slots = R / g + (a.copy ? (dh - 2 * R) / g : 0);
  if (a.slots == 0) return SB_OK;
  a.units = (long long)B * T * a.slots;
  const long long blocks = (a.units + 255) / 256;
  if (blocks > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_rope_axes: too many rows");
  // split the heads until every SM has its four blocks; more of them pay the trigonometry again (eight an SM:
  // 41 against 38 us for 3 x 8161 tokens of 12 x 64 in fp16, as long for fp32)
  const int sms = xattn_sms();
  if (sms == 0) return record_error(SB_ECUDA, "sb_rope_axes: device");
  int parts = 1;
  while (parts < H && parts < 32 && blocks * parts < 4ll * sms) ++parts;
  a.heads_per = (H + parts - 1) / parts;
  const dim3 grid((unsigned)blocks, (unsigned)((H + a.heads_per - 1) / a.heads_per));
  auto kernel = !vec               ? rope_kernel<false, 0>
                : dtype == SB_F32 ? rope_kernel<true, SB_F32>
                : dtype == SB_F16 ? rope_kernel<true, SB_F16> : rope_kernel<true, SB_BF16>;
  kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}
