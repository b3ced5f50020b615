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

// t of 16 RB rows by v_mfma_f32_16x16x32_bf16.  The four waves take every fourth
// 64-value piece of K, each through an LDS ring of its own (direct-to-LDS loads of
// whole 128-byte row pieces, XOR-swizzled; operands loaded straight into the
// MFMA's layout take 16 rows per quarter wave, which the vector cache serves at a
// fraction of its rate: 4033 x 2624 at rank 32 20 us), and add up through LDS.  The
// adapters of the rows are taken in turn (grid y of them at once), a row keeping
// its own one's product.  Reads x once and A_a once
// per workgroup.  Further workgroups (grid x past row_wgs) list the adapters of
// the second product's tiles of tile_rows rows, a wave each; workgroup 0 also
// writes the 16 zero bytes that its stages read.
__device__ __forceinline__ void lora_tile_list(const GemmArgs& g, int tile, int tile_rows, int lane) {
  const int m0 = tile * tile_rows;
  int* list = const_cast<int*>(lora_list(g)) + m0;
  constexpr int NR = 4;  // up to 256 rows
  int ad[NR];
  uint64_t rest[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = 64 * i + lane;
    ad[i] = r < tile_rows && m0 + r < g.M ? (g.lora_adapter ? g.lora_adapter[m0 + r] : 0) : -1;
    rest[i] = __ballot(static_cast<unsigned>(ad[i]) < static_cast<unsigned>(g.lora_n));
  }
  int n = 0;
#pragma unroll
  for (int i = 0; i < NR; ++i)
    while (rest[i]) {
      const int a = __builtin_amdgcn_readlane(ad[i], __builtin_ctzll(rest[i]));
#pragma unroll
      for (int k = 0; k < NR; ++k) rest[k] &= ~__ballot(ad[k] == a);
      if (lane == 0) list[n] = a;  // (at most one per row)
      ++n;
    }
  if (lane == 0) const_cast<int*>(lora_counts(g))[tile] = n;
}

template <int NB, int RB>
__global__ __launch_bounds__(256) void lora_shrink_kernel(GemmArgs g, const bf16_t* A, const float* scale, bf16_t* T,
                                                          int row_wgs, int tile_rows) {
  constexpr int STAGE = 2048 * (RB + NB), G = 2 * (RB + NB);  // bytes, load instructions: 8 rows of 128 bytes each
  constexpr int NS = 36864 / STAGE < 6 ? 36864 / STAGE : 6;   // ring stages of a wave
  constexpr int LDR = 16 * NB + 1;
  static_assert(NS >= 3 && 4 * 16 * RB * LDR * 4 <= 4 * NS * STAGE && G * (NS - 1) <= 63, "rings");
  __shared__ __attribute__((aligned(16))) char smem[4 * NS * STAGE];
  float* red = reinterpret_cast<float*>(smem);  // [4][16 RB][LDR], over the rings
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = lane & 15, q = lane >> 4;
  if (static_cast<int>(blockIdx.x) >= row_wgs) {
    const int tile = (blockIdx.x - row_wgs) * 4 + wave;
    if (blockIdx.y == 0 && tile < (g.M + tile_rows - 1) / tile_rows) lora_tile_list(g, tile, tile_rows, lane);
    return;
  }
  const int m0 = blockIdx.x * 16 * RB;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid < 8) T[static_cast<int64_t>(g.M) * g.lora_ld + tid] = bf16_t{0};
  int ad[RB];
  uint32_t rest = 0;  // the rows, the same in each lane quarter's vote
  bool has[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const int r = m0 + 16 * i + c, m = min(r, g.M - 1);
    ad[i] = g.lora_adapter ? g.lora_adapter[m] : 0;
    has[i] = r < g.M && static_cast<unsigned>(ad[i]) < static_cast<unsigned>(g.lora_n);
    rest |= (static_cast<uint32_t>(__ballot(has[i])) & 0xffffu) << (16 * i);
  }
  // a lane's row and chunk of each load instruction
  const int lrow = lane >> 3, lchunk = lane & 7;
  auto swz = [](int r) { return (r >> 1) & 7; };
  const bf16_t* x[2 * RB];
#pragma unroll
  for (int i = 0; i < 2 * RB; ++i) {
    const int r = 8 * i + lrow;
    x[i] = static_cast<const bf16_t*>(g.A) + static_cast<int64_t>(min(m0 + r, g.M - 1)) * g.lda + 8 * (lchunk ^ swz(r));
  }
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  char* ring = smem + wave_s * NS * STAGE;
  const int R = g.lora_r, pieces = g.K / 64;
  for (int turn = 0; rest; ++turn) {  // uniform over the workgroup
    const int first = __builtin_ctz(rest);
    const int a = __builtin_amdgcn_readlane(RB == 1 || first < 16 ? ad[0] : ad[RB - 1], first & 15);
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < RB; ++i) mine |= (static_cast<uint32_t>(__ballot(has[i] && ad[i] == a)) & 0xffffu) << (16 * i);
    rest &= ~mine;
    if (turn % gridDim.y != blockIdx.y) continue;
    const float sc = scale ? scale[a] : 1.f;
    for (int r0 = 0; r0 < g.lora_ld; r0 += 16 * NB) {
      const bf16_t* w[2 * NB];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        const int r = 8 * i + lrow;
        w[i] = A + (static_cast<int64_t>(a) * R + min(r0 + r, R - 1)) * g.K + 8 * (lchunk ^ swz(r));
      }
      auto issue = [&](int n) {  // the wave's n-th piece
        const int k = 64 * (wave_s + 4 * n);
        char* base = ring + (n % NS) * STAGE;
#pragma unroll
        for (int i = 0; i < 2 * RB; ++i) load_lds16(x[i] + k, base + 1024 * i);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) load_lds16(w[i] + k, base + 1024 * (2 * RB + i));
      };
      acc4_t acc[RB][NB];
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[i][b] = acc4_t{0.f, 0.f, 0.f, 0.f};
      const int np = (pieces - wave_s + 3) / 4;  // of this wave
#pragma unroll
      for (int s = 0; s < NS - 1; ++s)
        if (s < np) issue(s);
      for (int n = 0; n < np; ++n) {
        // (a wave's own ring: no barriers.  The last piece's reads are above the
        // wait, so the slot that the next loads take is free.)
        wait_lgkm0();
        if (n + NS - 1 < np) {
          issue(n + NS - 1);
          wait_vmcnt<G * (NS - 1)>();
        } else {
          wait_vmcnt<0>();
        }
        const char* sb = ring + (n % NS) * STAGE + c * 128;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int o = ((4 * s + q) ^ swz(c)) * 16;
          bf16x8_t xf[RB], wf[NB];
#pragma unroll
          for (int i = 0; i < RB; ++i) xf[i] = *reinterpret_cast<const bf16x8_t*>(sb + 2048 * i + o);
#pragma unroll
          for (int b = 0; b < NB; ++b) wf[b] = *reinterpret_cast<const bf16x8_t*>(sb + 2048 * (RB + b) + o);
#pragma unroll
          for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[i][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[i], wf[b], acc[i][b], 0, 0, 0);
        }
      }
      __syncthreads();  // every wave is done with its ring
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) red[((wave * RB + i) * 16 + 4 * q + e) * LDR + 16 * b + c] = acc[i][b][e];
      __syncthreads();
      for (int k = tid; k < 16 * RB * 16 * NB; k += 256) {
        const int row = k / (16 * NB), r = k - row * 16 * NB;
        if (!((mine >> row) & 1u) || r0 + r >= g.lora_ld) continue;
        auto part = [&](int w_) { return red[(w_ * 16 * RB + row) * LDR + r]; };
        const float v = (part(0) + part(1)) + (part(2) + part(3));
        T[static_cast<int64_t>(m0 + row) * g.lora_ld + r0 + r] = r0 + r < R ? f32_to_bf16(sc * v) : bf16_t{0};
      }
      __syncthreads();  // before the next sweep's loads
    }
  }
}

template <int NB>
void launch_shrink(const GemmArgs& g, const LoraArgs& l, hipStream_t st) {
  const bf16_t* A = static_cast<const bf16_t*>(l.a);
  bf16_t* T = static_cast<bf16_t*>(l.ws);
  const int rows = g.epi == EPI_LORAK ? gemm_lora_tile_rows(g) : 1;
  const int list_wgs = g.epi == EPI_LORAK ? ((g.M + rows - 1) / rows + 3) / 4 : 0;
  // 32 rows a workgroup (half the reads of A_a) where that still fills the CUs
  if (g.M >= 32 * 2 * num_cus()) {
    const int wgs = (g.M + 31) / 32;
    lora_shrink_kernel<NB, 2><<<wgs + list_wgs, 256, 0, st>>>(g, A, l.scale, T, wgs, rows);
    return;
  }
  const int wgs = (g.M + 15) / 16;
  // few rows: the adapters of a block's rows side by side
  const int side = wgs >= 64 ? 1 : std::min({16, g.M, g.lora_n});
  lora_shrink_kernel<NB, 1><<<dim3(wgs + list_wgs, side), 256, 0, st>>>(g, A, l.scale, T, wgs, rows);
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
  if (mfma && g.w_dtype != DT_FP8 && g.lora_r % 8 == 0 && (reinterpret_cast<uintptr_t>(g.lora_b) & 15u) == 0 &&
      lora_ws_bytes(g.M, g.lora_r) / 2 + 16 < (int64_t{1} << 32) &&
      static_cast<int64_t>(g.lora_n) * g.N * g.lora_r * 2 < (int64_t{1} << 32))
    g.epi = EPI_LORAK;
  check_gemm(g);
  if (mfma) {
    // 16-rank blocks per sweep over K
    if (g.lora_r <= 16)
      launch_shrink<1>(g, l, st);
    else if (g.lora_r <= 32)
      launch_shrink<2>(g, l, st);
    else
      launch_shrink<4>(g, l, st);
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
