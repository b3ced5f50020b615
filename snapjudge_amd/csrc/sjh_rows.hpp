// sjh_rows.hpp -- row access and reductions shared by the row-wise kernels.
#pragma once

#include "sjh_common.hpp"

namespace sjh {

namespace {

// Four consecutive values of a row: 16-byte (fp32) or 8-byte (bf16) accesses.
template <typename T>
struct Vec4;
template <>
struct Vec4<float> {
  using Raw = f32x4_t;
  static __device__ __forceinline__ Raw raw(const float* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void cvt(const Raw& v, float (&o)[4]) {
    o[0] = v[0], o[1] = v[1], o[2] = v[2], o[3] = v[3];
  }
  static __device__ __forceinline__ void load(const float* p, float (&o)[4]) {
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(p);
    o[0] = v[0], o[1] = v[1], o[2] = v[2], o[3] = v[3];
  }
  static __device__ __forceinline__ void store(float* p, const float (&o)[4]) {
    *reinterpret_cast<f32x4_t*>(p) = f32x4_t{o[0], o[1], o[2], o[3]};
  }
};
template <>
struct Vec4<bf16_t> {
  using Raw = u32x2_t;
  static __device__ __forceinline__ Raw raw(const bf16_t* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void cvt(const Raw& v, float (&o)[4]) {
    o[0] = __uint_as_float(v[0] << 16), o[1] = __uint_as_float(v[0] & 0xffff0000u);
    o[2] = __uint_as_float(v[1] << 16), o[3] = __uint_as_float(v[1] & 0xffff0000u);
  }
  static __device__ __forceinline__ void load(const bf16_t* p, float (&o)[4]) {
    const u32x2_t v = *reinterpret_cast<const u32x2_t*>(p);
    o[0] = __uint_as_float(v[0] << 16), o[1] = __uint_as_float(v[0] & 0xffff0000u);
    o[2] = __uint_as_float(v[1] << 16), o[3] = __uint_as_float(v[1] & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float (&o)[4]) {
    *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
  }
};

// Sum of a double over the 64 lanes, every lane receiving the total: DPP
// exchanges inside each row of 16 lanes (pairs, quads, mirrored halves,
// mirrored rows), then two shuffles across the rows.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xf, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32) |
                                        static_cast<uint32_t>(lo));
}
__device__ __forceinline__ void wave_sum2(double& a, double& b) {
  a += dpp_f64<0xB1>(a), b += dpp_f64<0xB1>(b);    // quad_perm [1,0,3,2]
  a += dpp_f64<0x4E>(a), b += dpp_f64<0x4E>(b);    // quad_perm [2,3,0,1]
  a += dpp_f64<0x141>(a), b += dpp_f64<0x141>(b);  // row_half_mirror
  a += dpp_f64<0x140>(a), b += dpp_f64<0x140>(b);  // row_mirror
  a += __shfl_xor(a, 16, 64), b += __shfl_xor(b, 16, 64);
  a += __shfl_xor(a, 32, 64), b += __shfl_xor(b, 32, 64);
}

}  // namespace

}  // namespace sjh
