// sb_rows.cuh -- rows of fp16, bf16 or fp32 elements as fp32 values: 8-element vectors and
// single elements, for the kernels of the memory-reading block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sb_internal.cuh"
#include "sb_ptx.cuh"

namespace sb {

inline bool rows_dtype_ok(int dt) { return dt == SB_F16 || dt == SB_BF16 || dt == SB_F32; }
inline int dtype_bytes(int dt) { return dt == SB_F32 ? 4 : 2; }

// Eight elements as loaded: 16 bytes of fp16 / bf16 (lo) or 32 bytes of fp32 (lo, hi).  Loads
// and conversions are apart, so that a thread's loads are all in flight before the first
// conversion waits for one.
struct Raw8 {
  uint4 lo, hi;
};

SB_DEV float one_of(const void* p, int dt, long long i) {
  if (dt == SB_F32) return static_cast<const float*>(p)[i];
  if (dt == SB_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
SB_DEV void put_one(void* p, int dt, long long i, float v) {
  if (dt == SB_F32) static_cast<float*>(p)[i] = v;
  else if (dt == SB_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// 8 elements at element offset i (16-byte aligned address)
SB_DEV Raw8 load_raw8(const void* p, int dt, long long i) {
  Raw8 r;
  r.hi = make_uint4(0, 0, 0, 0);
  if (dt == SB_F32) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
    r.lo = q[0];
    r.hi = q[1];
  } else {
    r.lo = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + i);
  }
  return r;
}
// the same, element by element, those from n on as zero (any alignment)
SB_DEV Raw8 load_raw8_tail(const void* p, int dt, long long i, int n) {
  Raw8 r;
  uint32_t w[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) w[u] = 0;
  if (dt == SB_F32) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (u < n) w[u] = __float_as_uint(static_cast<const float*>(p)[i + u]);
  } else {
    const unsigned short* q = static_cast<const unsigned short*>(p) + i;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (u < n) w[u >> 1] |= (uint32_t)q[u] << (16 * (u & 1));
  }
  r.lo = make_uint4(w[0], w[1], w[2], w[3]);
  r.hi = make_uint4(w[4], w[5], w[6], w[7]);
  return r;
}
SB_DEV float2 pair_of(uint32_t w, int dt) {
  if (dt == SB_F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
SB_DEV void unpack8(const Raw8& r, int dt, float (&v)[8]) {
  if (dt == SB_F32) {
    v[0] = __uint_as_float(r.lo.x); v[1] = __uint_as_float(r.lo.y);
    v[2] = __uint_as_float(r.lo.z); v[3] = __uint_as_float(r.lo.w);
    v[4] = __uint_as_float(r.hi.x); v[5] = __uint_as_float(r.hi.y);
    v[6] = __uint_as_float(r.hi.z); v[7] = __uint_as_float(r.hi.w);
  } else {
    const uint32_t w[4] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float2 f = pair_of(w[u], dt);
      v[2 * u] = f.x;
      v[2 * u + 1] = f.y;
    }
  }
}
SB_DEV uint32_t pack_pair(float a, float b, int dt) {
  if (dt == SB_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
SB_DEV void store8(void* p, int dt, long long i, const float (&v)[8]) {
  if (dt == SB_F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<__half*>(p) + i) =
        make_uint4(pack_pair(v[0], v[1], dt), pack_pair(v[2], v[3], dt), pack_pair(v[4], v[5], dt),
                   pack_pair(v[6], v[7], dt));
  }
}
SB_DEV void store_raw8(void* p, int dt, long long i, const Raw8& r) {
  if (dt == SB_F32) {
    uint4* q = reinterpret_cast<uint4*>(static_cast<float*>(p) + i);
    q[0] = r.lo;
    q[1] = r.hi;
  } else {
    *reinterpret_cast<uint4*>(static_cast<__half*>(p) + i) = r.lo;
  }
}
SB_DEV void store8_tail(void* p, int dt, long long i, const float (&v)[8], int n) {
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (u < n) put_one(p, dt, i + u, v[u]);
}

// A bounded wait for an mbarrier's phase that no flag cuts short; false when it ran out.
SB_DEV bool bounded_wait(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  while (!mbar_try_wait(bar, parity))
    if (global_ns() - t0 > SB_WAIT_NS) return false;
  return true;
}

}  // namespace sb
