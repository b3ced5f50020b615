// lora.hip -- low-rank adapters of many requests beside a shared projection:
//
//   out[m] = act(x[m] W^T + bias + scale_a (x[m] A_a^T) B_a^T),  a = adapter[m]
//
// Two launches.  Here: t[m] = scale_a x[m] A_a^T for every row with an adapter
// (R values of a row).  Then the shared product, whose epilogue adds t B_a^T to
// its accumulators before bias and activation (EPI_LORA): the update never
// leaves the registers, and rows of different adapters share the base's tiles.
//
// For the bf16 and fp8 bases t is rounded to bf16, the second product's operand
// type: one rounding of a sum held in fp32, at most 2^-8 of the adapter's share
// of the output, whose own rounding is as large relative to the whole.  The
// fp32-product base takes t in fp32.
#include <algorithm>

#include "sjh_common.hpp"
#include "sjh_host.hpp"
#include "sjh_kernels.hpp"

namespace sjh {

namespace {

typedef __attribute__((ext_vector_type(4))) float acc4_t;

// t of 16 rows by v_mfma_f32_16x16x32_bf16: the rows' fragments and A_a's come
// straight from memory (16 consecutive values of a row per lane quarter), the
// four waves take every fourth 64-value piece of K and add up through LDS.  The
// adapters of the 16 rows are taken in turn (grid y of them at once), a row
// keeping its own one's product.  Bound by reading x once (M K 2 bytes).
constexpr int kRB = 4;  // 16-rank blocks per sweep over K
__global__ __launch_bounds__(256) void lora_shrink_kernel(GemmArgs g, const bf16_t* A, const float* scale, bf16_t* T) {
  __shared__ float red[4][16][16 * kRB + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = lane & 15, q = lane >> 4;
  const int m0 = blockIdx.x * 16;
  const int m = min(m0 + c, g.M - 1);
  const int ad = g.lora_adapter ? g.lora_adapter[m] : 0;
  const bool has = m0 + c < g.M && static_cast<unsigned>(ad) < static_cast<unsigned>(g.lora_n);
  uint32_t rest = static_cast<uint32_t>(__ballot(has)) & 0xffffu;  // the rows, the same in each quarter
  const bf16_t* x = static_cast<const bf16_t*>(g.A) + static_cast<int64_t>(m) * g.lda + 8 * q;
  const int R = g.lora_r, pieces = g.K / 64;
  for (int turn = 0; rest; ++turn) {  // uniform over the workgroup
    const int a = __builtin_amdgcn_readlane(ad, __builtin_ctz(rest));
    const uint32_t mine = static_cast<uint32_t>(__ballot(has && ad == a)) & 0xffffu;
    rest &= ~mine;
    if (turn % gridDim.y != blockIdx.y) continue;
    const float sc = scale ? scale[a] : 1.f;
    for (int r0 = 0; r0 < g.lora_ld; r0 += 16 * kRB) {
      const bf16_t* w[kRB];
#pragma unroll
      for (int b = 0; b < kRB; ++b)
        w[b] = A + (static_cast<int64_t>(a) * R + min(r0 + 16 * b + c, R - 1)) * g.K + 8 * q;
      const int nb = min(kRB, (g.lora_ld - r0) / 16);
      acc4_t acc[kRB];
#pragma unroll
      for (int b = 0; b < kRB; ++b) acc[b] = acc4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
      for (int p = wave; p < pieces; p += 4) {
        bf16x8_t xf[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) xf[s] = *reinterpret_cast<const bf16x8_t*>(x + 64 * p + 32 * s);
#pragma unroll
        for (int b = 0; b < kRB; ++b)
          if (b < nb)
#pragma unroll
            for (int s = 0; s < 2; ++s)
              acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[s], *reinterpret_cast<const bf16x8_t*>(w[b] + 64 * p + 32 * s),
                                                               acc[b], 0, 0, 0);
      }
      __syncthreads();  // the last sweep's reads
#pragma unroll
      for (int b = 0; b < kRB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][4 * q + e][16 * b + c] = acc[b][e];
      __syncthreads();
      for (int i = tid; i < 16 * 16 * nb; i += 256) {
        const int row = i / (16 * nb), r = i - row * 16 * nb;
        if (!((mine >> row) & 1u)) continue;
        const float v = (red[0][row][r] + red[1][row][r]) + (red[2][row][r] + red[3][row][r]);
        T[static_cast<int64_t>(m0 + row) * g.lora_ld + r0 + r] = r0 + r < R ? f32_to_bf16(sc * v) : bf16_t{0};
      }
    }
  }
}

// t in fp32, any shape: a workgroup per row, a wave per rank in turn.
template <typename T>
__global__ __launch_bounds__(256) void lora_shrink_f32_kernel(GemmArgs g, const T* A, const float* scale, float* t) {
  const int m = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int a = g.lora_adapter ? g.lora_adapter[m] : 0;
  if (static_cast<unsigned>(a) >= static_cast<unsigned>(g.lora_n)) return;
  const T* x = static_cast<const T*>(g.A) + static_cast<int64_t>(m) * g.lda;
  const float sc = scale ? scale[a] : 1.f;
  for (int r = wave; r < g.lora_r; r += 4) {
    const T* w = A + (static_cast<int64_t>(a) * g.lora_r + r) * g.K;
    float s = 0.f;
    for (int k = lane; k < g.K; k += 64) s = __builtin_fmaf(load_f32(x + k), load_f32(w + k), s);
    s = wave_sum(s);
    if (lane == 0) t[static_cast<int64_t>(m) * g.lora_ld + r] = sc * s;
  }
}

}  // namespace

void launch_gemm_lora(const LoraArgs& l, hipStream_t st) {
  GemmArgs g = l.g;
  g.epi = EPI_LORA;
  g.lora_t = l.ws;
  if (g.M > (1 << 24) - 1) fail_arg("gemm_lora: M must be below 2^24");
  const bool mfma = gemm_takes_mfma(g) && (reinterpret_cast<uintptr_t>(l.a) & 15u) == 0;
  if (!mfma && g.w_dtype == DT_FP8) fail_arg("gemm_lora: fp8 weights need 16-byte aligned adapters");
  g.lora_ld = mfma ? (g.lora_r + 15) / 16 * 16 : g.lora_r;
  check_gemm(g);
  if (mfma) {
    const int blocks = (g.M + 15) / 16;
    // few rows: the adapters of a block's rows side by side
    const int side = blocks >= 64 ? 1 : std::min({16, g.M, g.lora_n});
    lora_shrink_kernel<<<dim3(blocks, side), 256, 0, st>>>(g, static_cast<const bf16_t*>(l.a), l.scale, static_cast<bf16_t*>(l.ws));
    check_launch("lora_shrink");
    launch_gemm(g, st);
    return;
  }
  if (g.in_dtype == DT_BF16)
    lora_shrink_f32_kernel<<<g.M, 256, 0, st>>>(g, static_cast<const bf16_t*>(l.a), l.scale, static_cast<float*>(l.ws));
  else
    lora_shrink_f32_kernel<<<g.M, 256, 0, st>>>(g, static_cast<const float*>(l.a), l.scale, static_cast<float*>(l.ws));
  check_launch("lora_shrink_f32");
  launch_gemm_f32(g, st);
  check_launch("gemm_f32");
}

}  // namespace sjh
