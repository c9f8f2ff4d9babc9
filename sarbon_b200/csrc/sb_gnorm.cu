// sb_gnorm.cu -- the end of one transformer block and the start of the next in one pass:
//   n = Npost(z),  y = x + scale * gate * n,  h = Npre(y)
// (each norm optional, RMS or layer norm, fp32 statistics), and its gradients.
//
// Forward, per row v of D values: RMS norm v r w with r = (mean v^2 + eps)^-1/2; layer norm
// (v - m) r w + b with r = (mean (v - m)^2 + eps)^-1/2 (the mean first, then the centred
// squares: no cancellation).  Apart, the norms and the residual sum would read and write the
// rows five times; here x and z are read and y and h written once, which bounds the kernel.
//
// Backward, with hats the normalised rows and e = d * w:
//   dyt = dy + r_y (e - yhat mean(e yhat) [- mean(e)]),  e = dh * w_pre        -> dx = dyt
//   dn = dyt * scale * gate,  dz = r_z (e - zhat mean(e zhat) [- mean(e)]),  e = dn * w_post
// The rows' statistics are taken again from x and z (they are in registers anyway) instead of
// being kept by the forward pass.  With f = dyt (times the gate where each row has its own), all
// column sums follow from four: Z = sum f zhat, Y = sum f, H = sum dh yhat, S = sum dh, per image
// where the gate is an image's:
//   d post_w = scale gate Z,  d post_b = scale gate Y,  d scale = gate (w Z + b Y),
//   d gate = scale (w Z + b Y),  d pre_w = H,  d pre_b = S.
// Each CTA keeps its columns' sums in registers over its rows and writes them once; a second
// kernel adds the CTAs' sums in a fixed order (no atomics: the same inputs give the same bits).
//
// A row belongs to `tpr` threads (a multiple of a warp, eight columns each), a CTA of at least
// 256 threads handles several short rows at once, and the next rows' loads are issued before the
// current rows' reductions.
#include <algorithm>

#include "sb_rows.cuh"

namespace sb {
namespace {

constexpr int kMaxD = 8192;
constexpr int kSums = 4;  // Z, Y, H, S

struct Rows {
  const void* p;
  long long row, img;
};

struct NormArgs {
  Rows x, z, gate, dy, dh;
  int xdt, zdt;
  const float *scale, *post_w, *post_b, *pre_w, *pre_b;
  int layer;
  float eps;
  int T, D, tpr, per;  // threads a row, rows a CTA takes at once
  long long rows;      // B * T
  void *y, *h;         // forward
  long long y_row, y_img, h_row, h_img;
  void *dx, *dz, *dgate_rows;  // backward
  float* part;                 // [groups * chunks][kSums][D]
  long long group_rows;        // rows that share their column sums (T for an image's gate, B * T else)
  int chunks, gate_is_row;     // CTAs a group
};

// Sums of two values over the threads of a row; `slot` alternates between two halves of the
// buffer, so one barrier a reduction is enough.
struct RowSum {
  float2* buf;  // [2][per * warps a row]
  int warps, half;
  SB_DEV float2 operator()(float a, float b) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
      b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    if (warps == 1) return make_float2(a, b);
    float2* mine = buf + half * 32;
    half ^= 1;
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) mine[w] = make_float2(a, b);
    __syncthreads();
    const int w0 = w / warps * warps;
    float2 s = make_float2(0.f, 0.f);
    for (int i = 0; i < warps; ++i) {
      const float2 t = mine[w0 + i];
      s.x += t.x;
      s.y += t.y;
    }
    return s;
  }
};

template <bool VEC>
SB_DEV Raw8 fetch(const void* p, int dt, long long i, int n) {
  if constexpr (VEC) return n > 0 ? load_raw8(p, dt, i) : Raw8{};
  else return load_raw8_tail(p, dt, i, n);
}
template <bool VEC>
SB_DEV void put(void* p, int dt, long long i, const float (&v)[8], int n) {
  if constexpr (VEC) {
    if (n > 0) store8(p, dt, i, v);
  } else {
    store8_tail(p, dt, i, v, n);
  }
}
template <bool VEC>
SB_DEV void columns(const float* w, int c, int n, float other, float (&v)[8]) {
  if (!w) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = other;
    return;
  }
  unpack8(fetch<VEC>(w, SB_F32, c, n), SB_F32, v);
}

// mean and 1 / deviation of a row; columns from n on do not count
SB_DEV void stats_of(const float (&v)[8], int n, int layer, float inv_d, float eps, RowSum& sum, float& mean, float& r) {
  float s = 0.f, q = 0.f;
  if (layer) {
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u];  // zero from n on
    mean = sum(s, 0.f).x * inv_d;
  } else {
    mean = 0.f;
  }
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const float d = v[u] - mean;
    q += u < n ? d * d : 0.f;
  }
  r = rsqrtf(sum(q, 0.f).x * inv_d + eps);
}

template <bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 buf[64];
  RowSum sum{buf, a.tpr >> 5, 0};
  const int sub = threadIdx.x / a.tpr;
  const int c = (threadIdx.x - sub * a.tpr) * 8;
  const int n = max(0, min(8, a.D - c));
  const float inv_d = 1.f / (float)a.D;
  const long long step = (long long)gridDim.x * a.per;
  Raw8 rx, rz, rg;
  auto load = [&](long long r) {
    const bool ok = r < a.rows;
    const long long b = ok ? r / a.T : 0, t = ok ? r - b * a.T : 0;
    const int m = ok ? n : 0;
    rx = fetch<VEC>(a.x.p, a.xdt, b * a.x.img + t * a.x.row + c, m);
    rz = fetch<VEC>(a.z.p, a.zdt, b * a.z.img + t * a.z.row + c, m);
    if (a.gate.p) rg = fetch<VEC>(a.gate.p, a.zdt, b * a.gate.img + t * a.gate.row + c, m);
  };
  float scale[8], post_w[8], pre_w[8];
  columns<VEC>(a.scale, c, n, 1.f, scale);
  columns<VEC>(a.post_w, c, n, 1.f, post_w);
  columns<VEC>(a.pre_w, c, n, 1.f, pre_w);
  long long r0 = (long long)blockIdx.x * a.per;
  load(r0 + sub);
  for (; r0 < a.rows; r0 += step) {
    const long long r = r0 + sub;
    const bool ok = r < a.rows;
    float v[8], y[8], g[8];
    unpack8(rz, a.zdt, v);
    unpack8(rx, a.xdt, y);
    if (a.gate.p) {
      unpack8(rg, a.zdt, g);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) g[u] = 1.f;
    }
    load(r + step);
    if (a.post_w) {
      float mean, rs, post_b[8];
      stats_of(v, n, a.layer, inv_d, a.eps, sum, mean, rs);
      columns<VEC>(a.post_b, c, n, 0.f, post_b);
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = (v[u] - mean) * rs * post_w[u] + post_b[u];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) y[u] = u < n ? fmaf(scale[u] * g[u], v[u], y[u]) : 0.f;
    const long long b = r / a.T, t = r - b * a.T;
    if (ok) put<VEC>(a.y, a.xdt, b * a.y_img + t * a.y_row + c, y, n);
    if (a.h) {
      float mean, rs, pre_b[8];
      stats_of(y, n, a.layer, inv_d, a.eps, sum, mean, rs);
      columns<VEC>(a.pre_b, c, n, 0.f, pre_b);
#pragma unroll
      for (int u = 0; u < 8; ++u) y[u] = (y[u] - mean) * rs * pre_w[u] + pre_b[u];
      if (ok) put<VEC>(a.h, a.zdt, b * a.h_img + t * a.h_row + c, y, n);
    }
  }
}

template <bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_back_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 buf[64];
  extern __shared__ float fold[];  // [per][kSums][tpr * 8] sums of the rows a CTA takes at once
  RowSum sum{buf, a.tpr >> 5, 0};
  const int sub = threadIdx.x / a.tpr;
  const int c = (threadIdx.x - sub * a.tpr) * 8;
  const int n = max(0, min(8, a.D - c));
  const float inv_d = 1.f / (float)a.D;
  const long long group = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const long long each = (a.group_rows + a.chunks - 1) / a.chunks;
  const long long first = group * a.group_rows + min(chunk * each, a.group_rows);
  const long long last = group * a.group_rows + min((chunk + 1) * each, a.group_rows);
  float acc[kSums][8];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int u = 0; u < 8; ++u) acc[k][u] = 0.f;
  Raw8 rx, rz, rg, rdy, rdh;
  auto load = [&](long long r) {
    const bool ok = r < last;
    const long long b = ok ? r / a.T : 0, t = ok ? r - b * a.T : 0;
    const int m = ok ? n : 0;
    rx = fetch<VEC>(a.x.p, a.xdt, b * a.x.img + t * a.x.row + c, a.dh.p ? m : 0);
    rz = fetch<VEC>(a.z.p, a.zdt, b * a.z.img + t * a.z.row + c, m);
    rg = fetch<VEC>(a.gate.p, a.zdt, b * a.gate.img + t * a.gate.row + c, a.gate.p ? m : 0);
    rdy = fetch<VEC>(a.dy.p, a.xdt, b * a.dy.img + t * a.dy.row + c, a.dy.p ? m : 0);
    rdh = fetch<VEC>(a.dh.p, a.zdt, b * a.dh.img + t * a.dh.row + c, a.dh.p ? m : 0);
  };
  load(first + sub);
  for (long long r0 = first; r0 < last; r0 += a.per) {
    const long long r = r0 + sub;
    const bool ok = r < last;
    float zh[8], g[8], d[8], y[8], dh[8];
    unpack8(rz, a.zdt, zh);
    unpack8(rx, a.xdt, y);
    unpack8(rdy, a.xdt, d);
    unpack8(rdh, a.zdt, dh);
    if (a.gate.p) {
      unpack8(rg, a.zdt, g);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) g[u] = 1.f;
    }
    load(r + a.per);
    float zr = 1.f, w[8], bb[8], s[8];
    columns<VEC>(a.scale, c, n, 1.f, s);
    if (a.post_w) {
      float mean;
      stats_of(zh, n, a.layer, inv_d, a.eps, sum, mean, zr);
#pragma unroll
      for (int u = 0; u < 8; ++u) zh[u] = u < n ? (zh[u] - mean) * zr : 0.f;
    }
    columns<VEC>(a.post_w, c, n, 1.f, w);
    if (a.dh.p) {
      columns<VEC>(a.post_b, c, n, 0.f, bb);
      float mean, rs;
#pragma unroll
      for (int u = 0; u < 8; ++u) y[u] = u < n ? fmaf(s[u] * g[u], zh[u] * w[u] + bb[u], y[u]) : 0.f;
      stats_of(y, n, a.layer, inv_d, a.eps, sum, mean, rs);
      float pw[8], e0 = 0.f, e1 = 0.f;
      columns<VEC>(a.pre_w, c, n, 1.f, pw);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        y[u] = u < n ? (y[u] - mean) * rs : 0.f;
        acc[2][u] += ok ? dh[u] * y[u] : 0.f;
        acc[3][u] += dh[u];
        dh[u] *= pw[u];
        e0 += dh[u];
        e1 += dh[u] * y[u];
      }
      const float2 m = sum(e0, e1);
      const float m0 = a.layer ? m.x * inv_d : 0.f, m1 = m.y * inv_d;
#pragma unroll
      for (int u = 0; u < 8; ++u) d[u] += rs * (dh[u] - y[u] * m1 - m0);
    }
    if (ok) put<VEC>(a.dx, a.xdt, r * a.D + c, d, n);
    if (a.dgate_rows) {
      float dg[8];
      columns<VEC>(a.post_b, c, n, 0.f, bb);
#pragma unroll
      for (int u = 0; u < 8; ++u) dg[u] = d[u] * s[u] * (zh[u] * w[u] + bb[u]);
      if (ok) put<VEC>(a.dgate_rows, a.zdt, r * a.D + c, dg, n);
    }
    float e0 = 0.f, e1 = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      // rows past the CTA's last hold zeros in d and zh
      const float f = a.gate_is_row ? d[u] * g[u] : d[u];
      acc[0][u] += ok ? f * zh[u] : 0.f;
      acc[1][u] += ok ? f : 0.f;
      d[u] = u < n ? d[u] * s[u] * g[u] * w[u] : 0.f;
      e0 += d[u];
      e1 += d[u] * zh[u];
    }
    if (a.post_w) {
      const float2 m = sum(e0, e1);
      const float m0 = a.layer ? m.x * inv_d : 0.f, m1 = m.y * inv_d;
#pragma unroll
      for (int u = 0; u < 8; ++u) d[u] = zr * (d[u] - zh[u] * m1 - m0);
    }
    if (ok) put<VEC>(a.dz, a.zdt, r * a.D + c, d, n);
  }
  if (!a.part) return;
  // the CTA's sums: over its row groups in order, one group of threads after the other
  const int width = a.tpr * 8;
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int u = 0; u < 8; ++u) fold[(sub * kSums + k) * width + c + u] = acc[k][u];
  __syncthreads();
  float* mine = a.part + (long long)blockIdx.x * kSums * a.D;
  for (int i = threadIdx.x; i < kSums * a.D; i += blockDim.x) {
    const int k = i / a.D, col = i - k * a.D;
    float s = 0.f;
    for (int q = 0; q < a.per; ++q) s += fold[(q * kSums + k) * width + col];
    mine[i] = s;
  }
}

struct FoldArgs {
  const float* part;
  int groups, chunks, D, gate_mode;
  Rows gate;  // of the group's rows
  int zdt, gate_is_row;
  const float *scale, *post_w, *post_b;
  float *dscale, *dgate, *dpost_w, *dpost_b, *dpre_w, *dpre_b;
};

// 32 columns a CTA; 16 threads a column add the partial sums of a group, in a fixed order
__global__ void __launch_bounds__(512) gated_norm_fold_kernel(const __grid_constant__ FoldArgs a) {
  __shared__ float sh[16][kSums][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float tot[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // scale, gate, post_w, post_b, pre_w, pre_b
  for (int g = 0; g < a.groups; ++g) {
    float s[kSums] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.D)
      for (int k = part; k < a.chunks; k += 16) {
        const float* p = a.part + ((long long)g * a.chunks + k) * kSums * a.D + c;
#pragma unroll
        for (int q = 0; q < kSums; ++q) s[q] += p[(long long)q * a.D];
      }
#pragma unroll
    for (int q = 0; q < kSums; ++q) sh[part][q][lane] = s[q];
    __syncthreads();
    if (part == 0 && c < a.D) {
#pragma unroll
      for (int q = 0; q < kSums; ++q) {
        s[q] = 0.f;
        for (int k = 0; k < 16; ++k) s[q] += sh[k][q][lane];
      }
      const float sc = a.scale ? a.scale[c] : 1.f;
      const float gt = a.gate.p && !a.gate_is_row ? one_of(a.gate.p, a.zdt, g * a.gate.img + c) : 1.f;
      const float n = s[0] * (a.post_w ? a.post_w[c] : 1.f) + s[1] * (a.post_b ? a.post_b[c] : 0.f);
      if (a.gate_mode == 2) a.dgate[(long long)g * a.D + c] = sc * n;
      tot[0] += gt * n;
      tot[1] += sc * n;
      tot[2] += sc * gt * s[0];
      tot[3] += sc * gt * s[1];
      tot[4] += s[2];
      tot[5] += s[3];
    }
    __syncthreads();
  }
  if (part != 0 || c >= a.D) return;
  if (a.dscale) a.dscale[c] = tot[0];
  if (a.gate_mode == 1) a.dgate[c] = tot[1];
  if (a.dpost_w) a.dpost_w[c] = tot[2];
  if (a.dpost_b) a.dpost_b[c] = tot[3];
  if (a.dpre_w) a.dpre_w[c] = tot[4];
  if (a.dpre_b) a.dpre_b[c] = tot[5];
}

int sm_count() {
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

struct Plan {
  int tpr, per, threads;
};
Plan plan_of(int D) {
  Plan p;
  p.tpr = ((D + 7) / 8 + 31) / 32 * 32;
  p.per = std::max(1, 256 / p.tpr);
  p.threads = p.tpr * p.per;
  return p;
}

// CTAs a group of rows: about two a SM over all groups, at least eight rows each
int chunks_of(int groups, long long group_rows, const Plan& p, int sms) {
  const long long want = std::max(1, 2 * sms / groups);
  return (int)std::max(1ll, std::min(want, (group_rows + 8 * p.per - 1) / (8 * p.per)));
}

bool rows_aligned(const void* p, int dt, long long row, long long img) {
  const int e = dtype_bytes(dt);
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row * e % 16 == 0 && img * e % 16 == 0;
}
bool cols_aligned(const float* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_gated_norm(const void* x, long long x_row, long long x_img, int x_dtype, const void* z, long long z_row,
                             long long z_img, int z_dtype, const void* gate, long long gate_row, long long gate_img,
                             const float* scale, const float* post_w, const float* post_b, const float* pre_w,
                             const float* pre_b, int layer, float eps, int B, int T, int D, void* y, long long y_row,
                             long long y_img, void* h, long long h_row, long long h_img, void* stream) {
  if (B < 0 || T < 0 || D < 1 || D > kMaxD || !rows_dtype_ok(x_dtype) || !rows_dtype_ok(z_dtype) || !(eps >= 0.f))
    return record_error(SB_EINVAL, "sb_gated_norm: sizes (1 <= D <= 8192), dtype or eps");
  if (B == 0 || T == 0) return SB_OK;
  if (!x || !z || !y || (pre_w != nullptr) != (h != nullptr) || (post_b && !post_w) || (pre_b && !pre_w))
    return record_error(SB_EINVAL, "sb_gated_norm: null argument (h with pre_w, biases with their weights)");
  const Plan p = plan_of(D);
  NormArgs a{};
  a.x = {x, x_row, x_img};
  a.z = {z, z_row, z_img};
  a.gate = {gate, gate_row, gate_img};
  a.xdt = x_dtype; a.zdt = z_dtype;
  a.scale = scale; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
  a.layer = layer != 0; a.eps = eps; a.T = T; a.D = D; a.tpr = p.tpr; a.per = p.per;
  a.rows = (long long)B * T;
  a.y = y; a.y_row = y_row; a.y_img = y_img;
  a.h = h; a.h_row = h_row; a.h_img = h_img;
  const bool vec = D % 8 == 0 && rows_aligned(x, x_dtype, x_row, x_img) && rows_aligned(z, z_dtype, z_row, z_img) &&
                   (!gate || rows_aligned(gate, z_dtype, gate_row, gate_img)) &&
                   rows_aligned(y, x_dtype, y_row, y_img) && (!h || rows_aligned(h, z_dtype, h_row, h_img)) &&
                   cols_aligned(scale) && cols_aligned(post_w) && cols_aligned(post_b) && cols_aligned(pre_w) &&
                   cols_aligned(pre_b);
  const int sms = sm_count();
  if (sms == 0) return record_error(SB_ECUDA, "sb_gated_norm: device");
  const long long grid = std::min((a.rows + p.per - 1) / p.per, (long long)sms * std::max(1, 1536 / p.threads));
  auto kernel = p.threads <= 256   ? vec ? gated_norm_kernel<true, 256> : gated_norm_kernel<false, 256>
                : p.threads <= 512 ? vec ? gated_norm_kernel<true, 512> : gated_norm_kernel<false, 512>
                                   : vec ? gated_norm_kernel<true, 1024> : gated_norm_kernel<false, 1024>;
  kernel<<<(unsigned)grid, p.threads, 0, (cudaStream_t)stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}

extern "C" int sb_gated_norm_work(int B, int T, int D, long long* bytes) {
  if (!bytes || B < 0 || T < 0 || D < 1 || D > kMaxD) return record_error(SB_EINVAL, "sb_gated_norm_work: arguments");
  const int sms = sm_count();
  if (sms == 0) return record_error(SB_ECUDA, "sb_gated_norm_work: device");
  const Plan p = plan_of(D);
  // enough for one group of all rows and for a group an item
  const long long one = chunks_of(1, (long long)B * T, p, sms), each = (long long)B * chunks_of(std::max(1, B), T, p, sms);
  *bytes = std::max(one, each) * kSums * D * 4;
  return SB_OK;
}

extern "C" int sb_gated_norm_backward(const void* dy, long long dy_row, long long dy_img, const void* dh, long long dh_row,
                                      long long dh_img, const void* x, long long x_row, long long x_img, int x_dtype,
                                      const void* z, long long z_row, long long z_img, int z_dtype, const void* gate,
                                      long long gate_row, long long gate_img, const float* scale, const float* post_w,
                                      const float* post_b, const float* pre_w, const float* pre_b, int layer, float eps,
                                      int B, int T, int D, void* dx, void* dz, float* dscale, void* dgate, int dgate_mode,
                                      float* dpost_w, float* dpost_b, float* dpre_w, float* dpre_b, void* work,
                                      long long work_bytes, void* stream) {
  if (B < 1 || T < 1 || D < 1 || D > kMaxD || !rows_dtype_ok(x_dtype) || !rows_dtype_ok(z_dtype) || !(eps >= 0.f))
    return record_error(SB_EINVAL, "sb_gated_norm_backward: sizes (1 <= D <= 8192), dtype or eps");
  if (!x || !z || !dx || !dz || (dh && !pre_w) || (post_b && !post_w) || (pre_b && !pre_w) || dgate_mode < 0 ||
      dgate_mode > 3 || (dgate_mode != 0 && (!dgate || !gate)) || (dscale && !scale) || ((dpost_w || dpost_b) && !post_w) ||
      ((dpre_w || dpre_b) && !pre_w))
    return record_error(SB_EINVAL, "sb_gated_norm_backward: null argument or a gradient without its input");
  const bool by_row = gate && gate_row != 0 && T > 1;
  const bool by_img = gate && gate_img != 0 && B > 1;
  if ((dgate_mode == 1 && (by_row || by_img)) || (dgate_mode == 2 && by_row))
    return record_error(SB_EINVAL, "sb_gated_norm_backward: dgate_mode does not fit the gate's strides");
  const Plan p = plan_of(D);
  NormArgs a{};
  a.x = {x, x_row, x_img};
  a.z = {z, z_row, z_img};
  a.gate = {gate, gate_row, gate_img};
  a.dy = {dy, dy_row, dy_img};
  a.dh = {dh, dh_row, dh_img};
  a.xdt = x_dtype; a.zdt = z_dtype;
  a.scale = scale; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
  a.layer = layer != 0; a.eps = eps; a.T = T; a.D = D; a.tpr = p.tpr; a.per = p.per;
  a.rows = (long long)B * T;
  a.dx = dx; a.dz = dz;
  a.dgate_rows = dgate_mode == 3 ? dgate : nullptr;
  a.gate_is_row = by_row || dgate_mode == 3;
  const bool sums = dscale || dgate_mode == 1 || dgate_mode == 2 || dpost_w || dpost_b || dpre_w || dpre_b;
  const int sms = sm_count();
  if (sms == 0) return record_error(SB_ECUDA, "sb_gated_norm_backward: device");
  const int groups = !a.gate_is_row && (by_img || dgate_mode == 2) ? B : 1;
  a.group_rows = groups == 1 ? a.rows : T;
  a.chunks = chunks_of(groups, a.group_rows, p, sms);
  const long long need = (long long)groups * a.chunks * kSums * D * 4;
  if (sums) {
    if (!work || work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15) != 0)
      return record_error(SB_EINVAL, "sb_gated_norm_backward: workspace (sb_gated_norm_work bytes, 16-byte aligned)");
    a.part = static_cast<float*>(work);
  }
  const bool vec = D % 8 == 0 && rows_aligned(x, x_dtype, x_row, x_img) && rows_aligned(z, z_dtype, z_row, z_img) &&
                   (!gate || rows_aligned(gate, z_dtype, gate_row, gate_img)) &&
                   (!dy || rows_aligned(dy, x_dtype, dy_row, dy_img)) &&
                   (!dh || rows_aligned(dh, z_dtype, dh_row, dh_img)) && rows_aligned(dx, x_dtype, 0, 0) &&
                   rows_aligned(dz, z_dtype, 0, 0) && (dgate_mode != 3 || rows_aligned(dgate, z_dtype, 0, 0)) &&
                   cols_aligned(scale) && cols_aligned(post_w) && cols_aligned(post_b) && cols_aligned(pre_w) &&
                   cols_aligned(pre_b);
  auto kernel = p.threads <= 256   ? vec ? gated_norm_back_kernel<true, 256> : gated_norm_back_kernel<false, 256>
                : p.threads <= 512 ? vec ? gated_norm_back_kernel<true, 512> : gated_norm_back_kernel<false, 512>
                                   : vec ? gated_norm_back_kernel<true, 1024> : gated_norm_back_kernel<false, 1024>;
  const int smem = sums ? p.per * kSums * p.tpr * 8 * 4 : 0;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return record_error(SB_ECUDA, "sb_gated_norm_backward: shared memory");
  if ((long long)groups * a.chunks > 0x7FFFFFFFll) return record_error(SB_EINVAL, "sb_gated_norm_backward: too many items");
  kernel<<<(unsigned)(groups * a.chunks), p.threads, smem, (cudaStream_t)stream>>>(a);
  if (sums) {
    FoldArgs f{};
    f.part = a.part;
    f.groups = groups; f.chunks = a.chunks; f.D = D; f.gate_mode = dgate_mode;
    f.gate = a.gate; f.zdt = z_dtype; f.gate_is_row = a.gate_is_row;
    f.scale = scale; f.post_w = post_w; f.post_b = post_b;
    f.dscale = dscale; f.dgate = static_cast<float*>(dgate);
    f.dpost_w = dpost_w; f.dpost_b = dpost_b; f.dpre_w = dpre_w; f.dpre_b = dpre_b;
    gated_norm_fold_kernel<<<(unsigned)((D + 31) / 32), 512, 0, (cudaStream_t)stream>>>(f);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_error(SB_ECUDA, cudaGetErrorString(e));
  return SB_OK;
}
