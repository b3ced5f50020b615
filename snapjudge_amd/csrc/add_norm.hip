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
// one; all of a row's loads go out before the first is used.
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

// V consecutive values of a row, V = 4 (vector accesses) or 1.
template <int V, typename T>
__device__ __forceinline__ void loadv(const T* p, float (&o)[V]) {
  if constexpr (V == 4)
    Vec4<T>::load(p, o);
  else
    o[0] = load_f32(p);
}
template <int V, typename T>
__device__ __forceinline__ void storev(T* p, const float (&o)[V]) {
  if constexpr (V == 4)
    Vec4<T>::store(p, o);
  else
    store_f32(p, o[0]);
}

// A row of D values (NV pieces of V per thread, n of them real) becomes its
// norm: (v - shift - mean) * inv * w + b for LayerNorm, v * inv * w + b for the
// RMS norm.  WAVES: waves that share the row.
template <int NV, int V, int WAVES>
__device__ __forceinline__ void norm_row(float (&v)[NV][V], const float (&w)[NV][V], const float (&b)[NV][V], int kind,
                                         float shift, int t, int np, int D, float eps, double* red) {
  const bool layer = kind == NORM_LAYER;
  if (!layer) shift = 0.f;
  double s1 = 0.0, s2 = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      v[i][k] -= shift;
      const double d = t + 64 * WAVES * i < np ? static_cast<double>(v[i][k]) : 0.0;
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
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) v[i][k] = (v[i][k] - mean) * inv * w[i][k] + b[i][k];
}

// WAVES 1: WPB rows per workgroup, a wave each; 4: one row per workgroup.
template <int NV, int V, int WAVES, int WPB, typename T>
__global__ __launch_bounds__(64 * WPB) void add_norm_kernel(AddNormArgs a) {
  static_assert(WAVES == 1 || WAVES == WPB, "a wave or the workgroup owns a row");
  constexpr int TPR = 64 * WAVES;  // threads per row
  __shared__ double red[2][2 * WPB];
  const int t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  const unsigned wg = blockIdx.y * kGridX + blockIdx.x;
  const int64_t row = __builtin_amdgcn_readfirstlane(WAVES == 1 ? wg * WPB + (threadIdx.x >> 6) : wg);
  if (static_cast<unsigned>(row) >= static_cast<unsigned>(a.M)) return;  // uniform over the wave (WAVES 1) or the workgroup
  const int D = a.D, np = D / V;
  float x[NV][V], u[NV][V], g[NV][V], pw[NV][V], pb[NV][V], w[NV][V], b[NV][V];
  const float* gate = nullptr;
  if (a.gate) {
    const int id = a.gate_row ? min(max(a.gate_row[row], 0), a.n_gates - 1) : 0;
    gate = a.gate + static_cast<int64_t>(id) * D;
  }
  const float* xr = a.x + row * a.ld_x;
  // (read before x_out, which may be x, is written)
  const float first_x = WAVES == 1 ? 0.f : xr[0];
  const T* rr = a.r ? static_cast<const T*>(a.r) + row * a.ld_r : nullptr;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + TPR * i;
#pragma unroll
    for (int k = 0; k < V; ++k) x[i][k] = u[i][k] = 0.f, g[i][k] = pw[i][k] = w[i][k] = 1.f, pb[i][k] = b[i][k] = 0.f;
    if (c < np) {
      if (rr) loadv<V>(rr + V * c, u[i]);
      loadv<V>(xr + V * c, x[i]);
      if (a.post_w) loadv<V>(a.post_w + V * c, pw[i]);
      if (a.post_b) loadv<V>(a.post_b + V * c, pb[i]);
      if (gate) loadv<V>(gate + V * c, g[i]);
      if (a.pre_w) loadv<V>(a.pre_w + V * c, w[i]);
      if (a.pre_b) loadv<V>(a.pre_b + V * c, b[i]);
    }
  }
  if (rr) {
    if (a.post_norm != NORM_NONE)
      norm_row<NV, V, WAVES>(u, pw, pb, a.post_norm, load_f32(rr), t, np, D, a.eps, red[0]);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) x[i][k] = a.x_scale * x[i][k] + a.r_scale * g[i][k] * u[i][k];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) x[i][k] *= a.x_scale;
  }
  if (a.x_out) {
    float* xo = a.x_out + row * a.ld_xo;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + TPR * i < np) storev<V>(xo + V * (t + TPR * i), x[i]);
  }
  if (!a.y) return;
  if (a.pre_norm != NORM_NONE) {
    // x'[0] itself where the wave holds it, else the stream's part of it
    const float x0 = WAVES == 1 ? __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x[0][0])))
                                : a.x_scale * first_x;
    norm_row<NV, V, WAVES>(x, w, b, a.pre_norm, x0, t, np, D, a.eps, red[1]);
  }
  T* yo = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (t + TPR * i < np) storev<V>(yo + V * (t + TPR * i), x[i]);
}

dim3 grid_of(int wgs) {
  const unsigned n = static_cast<unsigned>(wgs);
  return dim3(n < kGridX ? n : kGridX, (n + kGridX - 1) / kGridX);
}

template <int NV, int V, typename T>
void launch_wave_rows(const AddNormArgs& a, hipStream_t st) {
  // one row per workgroup while that leaves CUs without a row, four beyond
  if (a.M <= 2 * num_cus())
    add_norm_kernel<NV, V, 1, 1, T><<<grid_of(a.M), 64, 0, st>>>(a);
  else
    add_norm_kernel<NV, V, 1, kWpb, T><<<grid_of(a.M / kWpb + (a.M % kWpb != 0)), 64 * kWpb, 0, st>>>(a);
}

template <int NV, int V, typename T>
void launch_group_rows(const AddNormArgs& a, hipStream_t st) {
  add_norm_kernel<NV, V, kWpb, kWpb, T><<<grid_of(a.M), 64 * kWpb, 0, st>>>(a);
}

template <typename T>
void launch_typed(const AddNormArgs& a, bool vec, hipStream_t st) {
  const int per_wave = (a.D + 63) / 64;  // columns per lane of a wave-owned row
  if (vec) {
    if (a.D <= 256) return launch_wave_rows<1, 4, T>(a, st);
    if (a.D <= 512) return launch_wave_rows<2, 4, T>(a, st);
    if (a.D <= 768) return launch_wave_rows<3, 4, T>(a, st);
    if (a.D <= 1024) return launch_wave_rows<4, 4, T>(a, st);
    if (a.D <= 2048) return launch_group_rows<2, 4, T>(a, st);
    if (a.D <= 4096) return launch_group_rows<4, 4, T>(a, st);
    return launch_group_rows<8, 4, T>(a, st);
  }
  if (per_wave <= 4) return launch_wave_rows<4, 1, T>(a, st);
  if (a.D <= kWaveMaxD) return launch_wave_rows<16, 1, T>(a, st);
  if (a.D <= 4096) return launch_group_rows<16, 1, T>(a, st);
  return launch_group_rows<32, 1, T>(a, st);
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
  const uintptr_t rb = a.dtype == DT_BF16 ? 7 : 15;  // alignment of four values of r and y
  auto ok = [](const void* p, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) == 0; };
  const bool vec = a.D % 4 == 0 && (a.ld_x | a.ld_xo | a.ld_r | a.ld_y) % 4 == 0 && ok(a.x, 15) && ok(a.x_out, 15) &&
                   ok(a.r, rb) && ok(a.y, rb) && ok(a.post_w, 15) && ok(a.post_b, 15) && ok(a.gate, 15) &&
                   ok(a.pre_w, 15) && ok(a.pre_b, 15);
  if (a.dtype == DT_BF16)
    launch_typed<bf16_t>(a, vec, st);
  else
    launch_typed<float>(a, vec, st);
  check_launch("add_norm");
}

}  // namespace sjh
