// add_norm.hip -- the norms on both sides of a residual block, fused with its
// gate and scales, for gfx950:
//
//   u = post(r)                                  (nothing, LayerNorm or RMS norm)
//   x' = x_scale x + r_scale gate[row] * u       (fp32 residual stream)
//   y = pre(x')                                  (the next block's input)
//
// Bound by HBM: a row of D columns is read and written once (x 4 D, r and y
// 2 D or 4 D bytes each, x' 4 D) and everything between stays in registers.
// A wave owns a row of up to 1024 columns, a workgroup of four waves a longer
// one; all of a row's loads go out before the first is used.  Measured on inputs
// that no cache holds, bf16, LayerNorm and RMS norm, gates: 18432 x 1024 56.6 us
// (4.0 TB/s; a large copy 5.1), 18432 x 768 43.7, 4000 x 4096 51.0; 17 x 768 4.3.
// Rows at any alignment take the same accesses: 18432 x 771 fp32 55.4 us (4.1
// TB/s), 136.6 with one column per lane and load.
//
// Each norm needs its row's sum and sum of squares: both are taken in double
// (exact products of fp32 values, no overflow at any magnitude), in one
// reduction per norm, for LayerNorm of d = v - v0 with v0 a value of the row
// (or close to one), so that a row's offset, however large against its spread,
// neither cancels in E[d^2] - E[d]^2 nor rounds the mean: y = (d - E[d]) inv.
#include <type_traits>

#include "sjh_common.hpp"
#include "sjh_host.hpp"
#include "sjh_kernels.hpp"
#include "sjh_rows.hpp"

namespace sjh {

namespace {

constexpr int kWpb = 4;          // waves per workgroup of the batch kernels
constexpr int kWaveMaxD = 1024;  // columns of a row that one wave holds
constexpr int kMaxD = 8192;      // ... that a workgroup of four holds
constexpr unsigned kGridX = 1u << 22;  // workgroups of a grid's row: a grid dimension holds fewer than 2^32 threads

// Four consecutive values at any alignment of T: one 16-byte (fp32) or 8-byte
// (bf16) access, which global memory takes at any address.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&o)[4]) {
  typename Vec4<T>::Raw v;
  __builtin_memcpy(&v, p, sizeof(v));
  Vec4<T>::cvt(v, o);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&o)[4]) {
  typename Vec4<T>::Raw v;
  if constexpr (sizeof(T) == 4)
    v = f32x4_t{o[0], o[1], o[2], o[3]};
  else
    v = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
  __builtin_memcpy(p, &v, sizeof(v));
}

// Piece c of a row of D values: columns 4 c to 4 c + 3; where TAIL, D is no
// multiple of four and the last piece has the D % 4 columns that are left (it lies
// among a thread's pieces from tail_from on, by the widths that NV stands for).
template <int NV, int WAVES>
constexpr int tail_from() {
  return WAVES == 1 ? NV - 1 : NV / 2;
}
template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int c, int D, bool tail, float (&o)[4]) {
  if (4 * c + 4 <= D) {
    load4(row + 4 * c, o);
  } else if (tail) {
    // (a clamped address in place of a branch: arrays that branches fill go to scratch)
    const int last = D - 1;
    float v[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] = load_f32(row + min(4 * c + k, last));
#pragma unroll
    for (int k = 0; k < 3; ++k) o[k] = 4 * c + k < D ? v[k] : o[k];
  }
}
template <typename T>
__device__ __forceinline__ void store_piece(T* row, int c, int D, bool tail, const float (&o)[4]) {
  if (4 * c + 4 <= D) {
    store4(row + 4 * c, o);
  } else if (tail) {
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (4 * c + k < D) store_f32(row + 4 * c + k, o[k]);
  }
}

// A row of D values (NV pieces of four per thread) becomes its norm: (v - shift - mean) * inv * w + b for LayerNorm, v * inv * w + b for the
// RMS norm.  WAVES: waves that share the row.
// The weights are read early where the caller has them in w and b.
template <int NV, int WAVES, bool TAIL, bool EARLY>
__device__ __forceinline__ void norm_row(float (&v)[NV][4], float (&w)[NV][4], float (&b)[NV][4], const float* wp, const float* bp,
                                         int kind, float shift, int t, int D, float eps, double* red) {
  const bool layer = kind == NORM_LAYER;
  if (!layer) shift = 0.f;
  double s1 = 0.0, s2 = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[i][k] -= shift;
      const int c = t + 64 * WAVES * i;
      const double d = (TAIL ? 4 * c + k < D : 4 * c < D) ? static_cast<double>(v[i][k]) : 0.0;
      s1 += d;
      s2 += d * d;
    }
  wave_sum2(s1, s2);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) {
      red[2 * (threadIdx.x >> 6)] = s1;
      red[2 * (threadIdx.x >> 6) + 1] = s2;
    }
    __syncthreads();
    s1 = s2 = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      s1 += red[2 * w];
      s2 += red[2 * w + 1];
    }
  }
  const double m = layer ? s1 / D : 0.0;
  const double var = s2 / D - m * m;
  // (a NaN, or an infinity under LayerNorm, makes the whole row NaN)
  const float inv = var == var ? static_cast<float>(1.0 / sqrt(fmax(var, 0.0) + static_cast<double>(eps))) : __builtin_nanf("");
  const float mean = static_cast<float>(m);
  if constexpr (!EARLY) {
    asm volatile("" ::: "memory");  // (keeps the weights' loads, and their registers, behind the sums)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + 64 * WAVES * i;
      if (wp) load_piece(wp, c, D, TAIL && i >= tail_from<NV, WAVES>(), w[i]);
      if (bp) load_piece(bp, c, D, TAIL && i >= tail_from<NV, WAVES>(), b[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[i][k] = (v[i][k] - mean) * inv * w[i][k] + b[i][k];
}

// WAVES 1: WPB rows per workgroup, a wave each; 4: one row per workgroup.  EARLY:
// the weights and the gate are read with the row; else where they are used.
template <int NV, int WAVES, int WPB, bool TAIL, typename T>
__global__ __launch_bounds__(64 * WPB) void add_norm_kernel(AddNormArgs a) {
  static_assert(WAVES == 1 || WAVES == WPB, "a wave or the workgroup owns a row");
  constexpr bool EARLY = WAVES == 1 && (WPB == 1 || NV == 1);
  constexpr int TPR = 64 * WAVES;  // threads per row
  __shared__ double red[2][2 * WPB];
  const int t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  const unsigned wg = blockIdx.y * kGridX + blockIdx.x;
  const int64_t row = __builtin_amdgcn_readfirstlane(WAVES == 1 ? wg * WPB + (threadIdx.x >> 6) : wg);
  if (static_cast<unsigned>(row) >= static_cast<unsigned>(a.M)) return;  // uniform over the wave (WAVES 1) or the workgroup
  const int D = a.D;
  float x[NV][4], u[NV][4], g[NV][4], pw[NV][4], pb[NV][4], w[NV][4], b[NV][4];
  const float* gate = nullptr;
  if (a.gate) {
    const int id = a.gate_row ? min(max(a.gate_row[row], 0), a.n_gates - 1) : 0;
    gate = a.gate + static_cast<int64_t>(id) * D;
  }
  const float* xr = a.x + row * a.ld_x;
  float first_x = WAVES == 1 ? 0.f : xr[0];
  const T* rr = a.r ? static_cast<const T*>(a.r) + row * a.ld_r : nullptr;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + TPR * i;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[i][k] = u[i][k] = 0.f, g[i][k] = pw[i][k] = w[i][k] = 1.f, pb[i][k] = b[i][k] = 0.f;
    if (rr) load_piece(rr, c, D, TAIL && i >= tail_from<NV, WAVES>(), u[i]);
    load_piece(xr, c, D, TAIL && i >= tail_from<NV, WAVES>(), x[i]);
    if constexpr (EARLY) {
      if (a.post_w) load_piece(a.post_w, c, D, TAIL && i >= tail_from<NV, WAVES>(), pw[i]);
      if (a.post_b) load_piece(a.post_b, c, D, TAIL && i >= tail_from<NV, WAVES>(), pb[i]);
      if (gate) load_piece(gate, c, D, TAIL && i >= tail_from<NV, WAVES>(), g[i]);
      if (a.pre_w) load_piece(a.pre_w, c, D, TAIL && i >= tail_from<NV, WAVES>(), w[i]);
      if (a.pre_b) load_piece(a.pre_b, c, D, TAIL && i >= tail_from<NV, WAVES>(), b[i]);
    }
  }
  if (rr) {
    if (a.post_norm != NORM_NONE)
      norm_row<NV, WAVES, TAIL, EARLY>(u, pw, pb, a.post_w, a.post_b, a.post_norm, load_f32(rr), t, D, a.eps, red[0]);
    if constexpr (!EARLY)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (gate) load_piece(gate, t + TPR * i, D, TAIL && i >= tail_from<NV, WAVES>(), g[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) x[i][k] = a.x_scale * x[i][k] + a.r_scale * g[i][k] * u[i][k];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) x[i][k] *= a.x_scale;
  }
  if constexpr (WAVES > 1) {
    // x_out may be x: every wave has read x[0] before any wave writes it
    asm volatile("" : "+v"(first_x));
    __syncthreads();
  }
  if (a.x_out) {
    float* xo = a.x_out + row * a.ld_xo;
#pragma unroll
    for (int i = 0; i < NV; ++i) store_piece(xo, t + TPR * i, D, TAIL && i >= tail_from<NV, WAVES>(), x[i]);
  }
  if (!a.y) return;
  if (a.pre_norm != NORM_NONE) {
    // x'[0] itself where the wave holds it, else the stream's part of it
    const float x0 = WAVES == 1 ? __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x[0][0])))
                                : a.x_scale * first_x;
    norm_row<NV, WAVES, TAIL, EARLY>(x, w, b, a.pre_w, a.pre_b, a.pre_norm, x0, t, D, a.eps, red[1]);
  }
  T* yo = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
  for (int i = 0; i < NV; ++i) store_piece(yo, t + TPR * i, D, TAIL && i >= tail_from<NV, WAVES>(), x[i]);
}

dim3 grid_of(int wgs) {
  const unsigned n = static_cast<unsigned>(wgs);
  return dim3(n < kGridX ? n : kGridX, (n + kGridX - 1) / kGridX);
}

template <int NV, bool TAIL, typename T>
void launch_wave_rows(const AddNormArgs& a, hipStream_t st) {
  // few rows are bound by latency: a workgroup each, with the weights' loads beside
  // the row's (1501 x 768 fp32 8.3 us, 9.3 the other way); many by the bytes in
  // flight: four to a workgroup and the weights late, which leaves room for 7 waves
  // a SIMD in place of 3 (18432 x 1024 56.6 us, 68.0 the other way)
  if (a.M <= 8 * num_cus())
    add_norm_kernel<NV, 1, 1, TAIL, T><<<grid_of(a.M), 64, 0, st>>>(a);
  else
    add_norm_kernel<NV, 1, kWpb, TAIL, T><<<grid_of(a.M / kWpb + (a.M % kWpb != 0)), 64 * kWpb, 0, st>>>(a);
}

template <int NV, bool TAIL, typename T>
void launch_group_rows(const AddNormArgs& a, hipStream_t st) {
  add_norm_kernel<NV, kWpb, kWpb, TAIL, T><<<grid_of(a.M), 64 * kWpb, 0, st>>>(a);
}

template <bool TAIL, typename T>
void launch_typed(const AddNormArgs& a, hipStream_t st) {
  if (a.D <= 256) return launch_wave_rows<1, TAIL, T>(a, st);
  if (a.D <= 512) return launch_wave_rows<2, TAIL, T>(a, st);
  if (a.D <= 768) return launch_wave_rows<3, TAIL, T>(a, st);
  if (a.D <= kWaveMaxD) return launch_wave_rows<4, TAIL, T>(a, st);
  if (a.D <= 2048) return launch_group_rows<2, TAIL, T>(a, st);
  if (a.D <= 4096) return launch_group_rows<4, TAIL, T>(a, st);
  return launch_group_rows<8, TAIL, T>(a, st);
}

}  // namespace

void launch_add_norm(const AddNormArgs& a, hipStream_t st) {
  if (a.M < 0) fail_arg("add_norm: M must not be negative");
  if (a.D < 1 || a.D > kMaxD) fail_arg("add_norm: D must lie in [1, 8192]");
  if (a.dtype != DT_F32 && a.dtype != DT_BF16) fail_arg("add_norm: dtype must be SJH_F32 or SJH_BF16");
  for (int k : {a.post_norm, a.pre_norm})
    if (k != NORM_NONE && k != NORM_LAYER && k != NORM_RMS) fail_arg("add_norm: unknown norm");
  if (a.ld_x < a.D || a.ld_xo < a.D || a.ld_r < a.D || a.ld_y < a.D) fail_arg("add_norm: row stride < D");
  if (!(a.eps >= 0.f) || !(a.eps < INFINITY)) fail_arg("add_norm: eps must be finite and not negative");
  if (a.gate && a.n_gates < 1) fail_arg("add_norm: gates need n_gates >= 1");
  if (a.gate_row && !a.gate) fail_arg("add_norm: gate_row without gates");
  if (a.M == 0) return;
  if (!a.x) fail_arg("add_norm: null x");
  if (!a.x_out && !a.y) fail_arg("add_norm: neither x_out nor y");
  const bool tail = a.D % 4 != 0;
  if (a.dtype == DT_BF16)
    tail ? launch_typed<true, bf16_t>(a, st) : launch_typed<false, bf16_t>(a, st);
  else
    tail ? launch_typed<true, float>(a, st) : launch_typed<false, float>(a, st);
  check_launch("add_norm");
}

}  // namespace sjh
