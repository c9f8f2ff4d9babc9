// sb_xattn_bwd.cu -- gradients of the attention of queries to an encoder's states.
//
// Per head and query i over the keys j that take part: s_ij = scale q_i.k_j, L_i = log sum_j exp s_ij,
// out_i = sum_j exp(s_ij - L_i) v_j; a query without keys gets zeros and L_i = -inf.  Gradients with
// P = exp(s - L), dP = dout v^T, D_i = dout_i.out_i, dS = P (dP - D):
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout   (dk, dv summed over the query heads that
// share a key head).
//
// A warp takes one query row (one key row for dk, dv), its channels spread over the lanes, and
// walks the other side once with the running maximum and sum of the softmax.
#include <cmath>

#include "sb_xattn.cuh"

namespace sb {
namespace {

struct AttnArgs {
  View q, k, v, out, dout;
  OutView o, dq, dk, dv;
  float* lse;
  const int* lens;
  const uint8_t* valid;
  long long valid_img;
  int dt, B, H, Hkv, dh, Tq, Tk;
  float scale;
};

constexpr int kWarps = 8;

SB_DEV float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
  return x;
}
// 4 channels a lane (dh <= 128)
SB_DEV void lane_load(const View& v, int dt, int b, long long t, int c0, int dh, float (&x)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int c = lane + 32 * u;
    x[u] = c < dh ? one_of(v.p, dt, b * v.img + t * v.row + c0 + c) : 0.f;
  }
}
SB_DEV void lane_store(const OutView& v, int dt, int b, long long t, int c0, int dh, const float (&x)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int c = lane + 32 * u;
    if (c < dh) put_one(v.p, dt, b * v.img + t * v.row + c0 + c, x[u]);
  }
}
SB_DEV float dot4(const float (&a)[4], const float (&b)[4]) {
  return warp_sum(a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3]);
}
SB_DEV int keys_of(const AttnArgs& a, int b) { return a.lens ? min(max(a.lens[b], 0), a.Tk) : a.Tk; }
SB_DEV bool takes_part(const AttnArgs& a, int b, int j) { return !a.valid || a.valid[b * a.valid_img + j] != 0; }

__global__ void __launch_bounds__(32 * kWarps) attend_dq_kernel(const __grid_constant__ AttnArgs a) {
  const long long r = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= (long long)a.B * a.H * a.Tq) return;
  const int t = (int)(r % a.Tq), h = (int)(r / a.Tq % a.H), b = (int)(r / a.Tq / a.H);
  const int kc = h / (a.H / a.Hkv) * a.dh;
  float q[4], k[4], v[4], g[4], o[4], dq[4] = {0.f, 0.f, 0.f, 0.f};
  lane_load(a.q, a.dt, b, t, h * a.dh, a.dh, q);
  lane_load(a.dout, a.dt, b, t, h * a.dh, a.dh, g);
  lane_load(a.out, a.dt, b, t, h * a.dh, a.dh, o);
  const float d = dot4(g, o), lse = a.lse[r];
  const int n = lse == -INFINITY ? 0 : keys_of(a, b);
  for (int j = 0; j < n; ++j) {
    if (!takes_part(a, b, j)) continue;
    lane_load(a.k, a.dt, b, j, kc, a.dh, k);
    lane_load(a.v, a.dt, b, j, kc, a.dh, v);
    const float ds = expf(dot4(q, k) * a.scale - lse) * (dot4(g, v) - d) * a.scale;
#pragma unroll
    for (int u = 0; u < 4; ++u) dq[u] += ds * k[u];
  }
  lane_store(a.dq, a.dt, b, t, h * a.dh, a.dh, dq);
}

__global__ void __launch_bounds__(32 * kWarps) attend_dkv_kernel(const __grid_constant__ AttnArgs a) {
  const long long r = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= (long long)a.B * a.Hkv * a.Tk) return;
  const int j = (int)(r % a.Tk), hk = (int)(r / a.Tk % a.Hkv), b = (int)(r / a.Tk / a.Hkv);
  const int group = a.H / a.Hkv;
  float q[4], k[4], v[4], g[4], o[4], dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
  if (j < keys_of(a, b) && takes_part(a, b, j)) {
    lane_load(a.k, a.dt, b, j, hk * a.dh, a.dh, k);
    lane_load(a.v, a.dt, b, j, hk * a.dh, a.dh, v);
    for (int h = hk * group; h < (hk + 1) * group; ++h)
      for (int t = 0; t < a.Tq; ++t) {
        const float lse = a.lse[((long long)b * a.H + h) * a.Tq + t];
        lane_load(a.q, a.dt, b, t, h * a.dh, a.dh, q);
        lane_load(a.dout, a.dt, b, t, h * a.dh, a.dh, g);
        lane_load(a.out, a.dt, b, t, h * a.dh, a.dh, o);
        const float p = expf(dot4(q, k) * a.scale - lse);
        const float ds = p * (dot4(g, v) - dot4(g, o)) * a.scale;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          dk[u] += ds * q[u];
          dv[u] += p * g[u];
        }
      }
  }
  lane_store(a.dk, a.dt, b, j, hk * a.dh, a.dh, dk);
  lane_store(a.dv, a.dt, b, j, hk * a.dh, a.dh, dv);
}

unsigned blocks_of(long long rows) { return (unsigned)((rows + kWarps - 1) / kWarps); }

}  // namespace
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
  if ((Tq > 0 && (!lse || !xattn_view_ok(dout, do_row, do_img) || !xattn_view_ok(q, q_row, q_img) || !xattn_view_ok(out, o_row, o_img) ||
                  !xattn_view_ok(dq, dq_row, dq_img))) ||
      (Tk > 0 && (!xattn_view_ok(k, k_row, k_img) || !xattn_view_ok(v, v_row, v_img) || !xattn_view_ok(dk, dk_row, dk_img) ||
                  !xattn_view_ok(dv, dv_row, dv_img))))
    return record_error(SB_EINVAL, "sb_cross_attention_backward: rows (16-byte aligned, strides multiples of 8) or lse");
  (void)work;
  (void)work_bytes;
  AttnArgs a{};
  a.q = {q, q_row, q_img}; a.k = {k, k_row, k_img}; a.v = {v, v_row, v_img};
  a.out = {out, o_row, o_img}; a.dout = {dout, do_row, do_img};
  a.dq = {dq, dq_row, dq_img}; a.dk = {dk, dk_row, dk_img}; a.dv = {dv, dv_row, dv_img};
  a.lse = const_cast<float*>(lse); a.lens = lens; a.valid = static_cast<const uint8_t*>(valid); a.valid_img = valid_img;
  a.dt = dtype; a.B = B; a.H = H; a.Hkv = Hkv; a.dh = dh; a.Tq = Tq; a.Tk = Tk; a.scale = scale;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (Tq > 0) attend_dq_kernel<<<blocks_of((long long)B * H * Tq), 32 * kWarps, 0, st>>>(a);
  if (Tk > 0) attend_dkv_kernel<<<blocks_of((long long)B * Hkv * Tk), 32 * kWarps, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}
