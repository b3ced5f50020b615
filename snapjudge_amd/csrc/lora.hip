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

// t of 16 rows by v_mfma_f32_16x16x32_bf16.  The four waves take every fourth
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

template <int NB>
__global__ __launch_bounds__(256) void lora_shrink_kernel(GemmArgs g, const bf16_t* A, const float* scale, bf16_t* T,
                                                          int row_wgs, int tile_rows) {
  constexpr int STAGE = 2048 * (1 + NB), G = 2 * (1 + NB);  // bytes, load instructions: 8 rows of 128 bytes each
  constexpr int NS = 36864 / STAGE < 6 ? 36864 / STAGE : 6;   // ring stages of a wave
  constexpr int LDR = 16 * NB + 1;
  static_assert(NS >= 3 && 4 * 16 * LDR * 4 <= 4 * NS * STAGE && G * (NS - 1) <= 63, "rings");
  __shared__ __attribute__((aligned(16))) char smem[4 * NS * STAGE];
  float* red = reinterpret_cast<float*>(smem);  // [4][16][LDR], over the rings
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = lane & 15, q = lane >> 4;
  if (static_cast<int>(blockIdx.x) >= row_wgs) {
    const int tile = (blockIdx.x - row_wgs) * 4 + wave;
    if (blockIdx.y == 0 && tile < (g.M + tile_rows - 1) / tile_rows) lora_tile_list(g, tile, tile_rows, lane);
    return;
  }
  const int m0 = blockIdx.x * 16;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid < 8) T[static_cast<int64_t>(g.M) * g.lora_ld + tid] = bf16_t{0};
  // the rows, the same in each lane quarter
  const int ad = g.lora_adapter ? g.lora_adapter[min(m0 + c, g.M - 1)] : 0;
  const bool has = m0 + c < g.M && static_cast<unsigned>(ad) < static_cast<unsigned>(g.lora_n);
  uint32_t rest = static_cast<uint32_t>(__ballot(has)) & 0xffffu;
  // a lane's row and chunk of each load instruction
  const int lrow = lane >> 3, lchunk = lane & 7;
  auto swz = [](int r) { return (r >> 1) & 7; };
  const bf16_t* x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 8 * i + lrow;
    x[i] = static_cast<const bf16_t*>(g.A) + static_cast<int64_t>(min(m0 + r, g.M - 1)) * g.lda + 8 * (lchunk ^ swz(r));
  }
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  char* ring = smem + wave_s * NS * STAGE;
  const int R = g.lora_r, pieces = g.K / 64;
  for (int turn = 0; rest; ++turn) {  // uniform over the workgroup
    const int a = __builtin_amdgcn_readlane(ad, __builtin_ctz(rest));
    const uint32_t mine = static_cast<uint32_t>(__ballot(has && ad == a)) & 0xffffu;
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
        for (int i = 0; i < 2; ++i) load_lds16(x[i] + k, base + 1024 * i);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) load_lds16(w[i] + k, base + 1024 * (2 + i));
      };
      acc4_t acc[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = acc4_t{0.f, 0.f, 0.f, 0.f};
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
          const bf16x8_t xf = *reinterpret_cast<const bf16x8_t*>(sb + o);
          bf16x8_t wf[NB];
#pragma unroll
          for (int b = 0; b < NB; ++b) wf[b] = *reinterpret_cast<const bf16x8_t*>(sb + 2048 * (1 + b) + o);
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, wf[b], acc[b], 0, 0, 0);
        }
      }
      __syncthreads();  // every wave is done with its ring
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[(wave * 16 + 4 * q + e) * LDR + 16 * b + c] = acc[b][e];
      __syncthreads();
      for (int k = tid; k < 16 * 16 * NB; k += 256) {
        const int row = k / (16 * NB), r = k - row * 16 * NB;
        if (!((mine >> row) & 1u) || r0 + r >= g.lora_ld) continue;
        auto part = [&](int w_) { return red[(w_ * 16 + row) * LDR + r]; };
        const float v = (part(0) + part(1)) + (part(2) + part(3));
        T[static_cast<int64_t>(m0 + row) * g.lora_ld + r0 + r] = r0 + r < R ? f32_to_bf16(sc * v) : bf16_t{0};
      }
      __syncthreads();  // before the next sweep's loads
    }
  }
}

// t of 64 rows, where there are many: a wave's 16 rows each, all of K, the ranks'
// rows of A_a shared by the four waves in LDS (a ring of four 64-value pieces, three
// of them in flight): a quarter of the reads of A_a and no sums over the waves, at
// two workgroups a CU at least.  The adapters of a block's rows in two turns of grid
// y: a block where two requests meet is not twice as late as the others.  18432 x
// 768 at rank 64: 12.5 us (31 MB read and written, 6 us at a copy's rate; 16 without
// the turns, 18.5 with 32 rows a workgroup and a wave per quarter of K).
template <int NB>
__global__ __launch_bounds__(256) void lora_shrink_rows_kernel(GemmArgs g, const bf16_t* A, const float* scale, bf16_t* T,
                                                               int row_wgs, int tile_rows) {
  constexpr int STAGE = 8192 + 2048 * NB, NS = 4;
  constexpr int NA = NB == 4 ? 2 : 1;  // of a wave's load instructions of A_a (NB 1: two waves load the same)
  constexpr int G = 2 + NA;
  static_assert(NB == 1 || NB == 2 || NB == 4, "two load instructions a rank block, among four waves");
  __shared__ __attribute__((aligned(16))) char smem[NS * STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, q = lane >> 4;
  if (static_cast<int>(blockIdx.x) >= row_wgs) {
    const int tile = (blockIdx.x - row_wgs) * 4 + wave;
    if (blockIdx.y == 0 && tile < (g.M + tile_rows - 1) / tile_rows) lora_tile_list(g, tile, tile_rows, lane);
    return;
  }
  const int m0 = blockIdx.x * 64;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid < 8) T[static_cast<int64_t>(g.M) * g.lora_ld + tid] = bf16_t{0};
  // a lane per row, the same in each wave
  const int ad = g.lora_adapter ? g.lora_adapter[min(m0 + lane, g.M - 1)] : 0;
  const bool has = m0 + lane < g.M && static_cast<unsigned>(ad) < static_cast<unsigned>(g.lora_n);
  uint64_t rest = __ballot(has);
  // a lane's row and chunk of each load instruction
  const int lrow = lane >> 3, lchunk = lane & 7;
  auto swz = [](int r) { return (r >> 1) & 7; };
  const bf16_t* x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 8 * i + lrow;
    x[i] = static_cast<const bf16_t*>(g.A) + static_cast<int64_t>(min(m0 + 16 * wave + r, g.M - 1)) * g.lda + 8 * (lchunk ^ swz(r));
  }
  const int R = g.lora_r, pieces = g.K / 64;
  for (int turn = 0; rest; ++turn) {  // uniform over the workgroup
    const int a = __builtin_amdgcn_readlane(ad, __builtin_ctzll(rest));
    const uint64_t mine = __ballot(has && ad == a);
    rest &= ~mine;
    if (turn % gridDim.y != blockIdx.y) continue;
    const float sc = scale ? scale[a] : 1.f;
    for (int r0 = 0; r0 < g.lora_ld; r0 += 16 * NB) {
      const bf16_t* w[NA];
      int wi[NA];
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        wi[i] = (NA * wave + i) & (2 * NB - 1);
        const int r = 8 * wi[i] + lrow;
        w[i] = A + (static_cast<int64_t>(a) * R + min(r0 + r, R - 1)) * g.K + 8 * (lchunk ^ swz(r));
      }
      auto issue = [&](int n) {
        char* base = smem + (n % NS) * STAGE;
#pragma unroll
        for (int i = 0; i < 2; ++i) load_lds16(x[i] + 64 * n, base + 2048 * wave + 1024 * i);
#pragma unroll
        for (int i = 0; i < NA; ++i) load_lds16(w[i] + 64 * n, base + 8192 + 1024 * wi[i]);
      };
      acc4_t acc[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = acc4_t{0.f, 0.f, 0.f, 0.f};
      __syncthreads();  // every wave is done with the sweep before
#pragma unroll
      for (int s = 0; s < NS - 1; ++s)
        if (s < pieces) issue(s);
      for (int n = 0; n < pieces; ++n) {
        // this wave's loads of the piece, and its reads of the one before, whose
        // slot the next loads take; the barrier says so of the others
        if (n + NS - 2 < pieces)
          wait_vmcnt<G * (NS - 2)>();
        else
          wait_vmcnt<0>();
        wait_lgkm0();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (n + NS - 1 < pieces) issue(n + NS - 1);
        const char* sb = smem + (n % NS) * STAGE + c * 128;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int o = ((4 * s + q) ^ swz(c)) * 16;
          const bf16x8_t xf = *reinterpret_cast<const bf16x8_t*>(sb + 2048 * wave + o);
          bf16x8_t wf[NB];
#pragma unroll
          for (int b = 0; b < NB; ++b) wf[b] = *reinterpret_cast<const bf16x8_t*>(sb + 8192 + 2048 * b + o);
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, wf[b], acc[b], 0, 0, 0);
        }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int r = r0 + 16 * b + c;
        if (r >= g.lora_ld) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = 16 * wave + 4 * q + e;
          if ((mine >> row) & 1u) T[static_cast<int64_t>(m0 + row) * g.lora_ld + r] = r < R ? f32_to_bf16(sc * acc[b][e]) : bf16_t{0};
        }
      }
    }
  }
}

template <int NB>
void launch_shrink(const GemmArgs& g, const LoraArgs& l, hipStream_t st) {
  const bf16_t* A = static_cast<const bf16_t*>(l.a);
  bf16_t* T = static_cast<bf16_t*>(l.ws);
  const int rows = g.epi == EPI_LORAK ? gemm_lora_tile_rows(g) : 1;
  const int list_wgs = g.epi == EPI_LORAK ? ((g.M + rows - 1) / rows + 3) / 4 : 0;
  // 64 rows a workgroup where that leaves a CU half a workgroup or more (sjh_gemm_lora,
  // N 2304, K 768, rank 64, 8192 rows: 62.9 us, 68.2 with 16 or 32 rows each; 4033 rows
  // at K 2624, N 1024, rank 32: 49.7, 42.4)
  if (g.M >= 32 * num_cus()) {
    const int wgs = (g.M + 63) / 64;
    lora_shrink_rows_kernel<NB><<<dim3(wgs + list_wgs, 2), 256, 0, st>>>(g, A, l.scale, T, wgs, rows);
    return;
  }
  const int wgs = (g.M + 15) / 16;
  // few rows: the adapters of a block's rows side by side
  const int side = wgs >= 64 ? 1 : std::min({16, g.M, g.lora_n});
  lora_shrink_kernel<NB><<<dim3(wgs + list_wgs, side), 256, 0, st>>>(g, A, l.scale, T, wgs, rows);
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
