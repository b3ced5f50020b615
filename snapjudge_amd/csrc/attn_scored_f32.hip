// attn_scored_f32.hip -- attention with modified scores (attn_scored.hip) in
// fp32 products: fp32 tensors, and the bf16 shapes and addresses that the bf16
// kernel does not take (values widened exactly; heads of 8, 16, 32, 64, 128).
//
// A workgroup takes 64 queries of one head, 16 per wave, over the 64-key tiles
// its masks need (32 keys at a time at head_dim 128), the next keys' rows in
// flight in registers meanwhile.  S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_16x16x4_f32: lane (c, q) of an accumulator holds query c and keys
// (head dims) 4 q + [0, 4), so P goes into the second product as it is.  Bound
// by the fp32 matrix rate, a sixteenth of bf16's.  Splits of the tile list
// fill the CUs where there are few blocks of queries.
#include <type_traits>

#include "sjh_attn_scored.hpp"
#include "sjh_common.hpp"
#include "sjh_host.hpp"
#include "sjh_kernels.hpp"

namespace sjh {

namespace {

constexpr int kRows = 64;  // queries per workgroup

template <typename T, int DH>
__global__ __launch_bounds__(256) void attn_scored_f32_kernel(AttnScoredArgs a, int vec) {
  constexpr int DP = DH < 16 ? 16 : DH;  // padded with zeros to one MFMA block
  constexpr int KT = DP > 64 ? 32 : 64, HALVES = kTile / KT, NB = KT / 16, ND = DP / 16;
  constexpr int LDR = DP + 4;  // rows 4 q + e of V, and 16 rows of K, on different banks
  constexpr int NL = KT * DP / 4 / 256 > 0 ? KT * DP / 4 / 256 : 1;  // 4-value pieces per thread and operand
  __shared__ __attribute__((aligned(16))) float Ks[KT * LDR], Vs[KT * LDR];
  __shared__ int2 tile_docs[64];
  __shared__ int ids[KT], flag;

  const int qb = blockIdx.x % a.n_blocks, r = blockIdx.x / a.n_blocks;
  const int b = r / a.H, head = r - b * a.H, split = blockIdx.y;
  const int kvh = head / (a.H / a.Hkv);
  const Seq s = load_seq(a, b);
  const int q0 = qb * kRows;
  if (q0 >= s.qlen) return;  // uniform
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
  const int qi = q0 + wave * 16 + c;
  const bool live = qi < s.qlen;
  const int qic = min(qi, s.qlen - 1), pos = s.pos0 + qic;
  const T* Q = static_cast<const T*>(a.q) + static_cast<int64_t>(head) * DH;
  const T* K = static_cast<const T*>(a.k) + s.k_row * a.ld_k + static_cast<int64_t>(kvh) * DH;
  const T* V = static_cast<const T*>(a.v) + s.k_row * a.ld_v + static_cast<int64_t>(kvh) * DH;

  Masks mk;
  mk.klen = s.klen, mk.prefix = s.prefix, mk.window = a.window, mk.causal = a.causal;
  mk.docs = a.k_doc != nullptr;
  QRange wg;
  const int n_wg = min(s.qlen - q0, kRows);
  wg.p0 = s.pos0 + q0, wg.p1 = wg.p0 + n_wg - 1, wg.d0 = wg.d1 = 0;
  if (mk.docs) doc_range(a, s, q0, n_wg, wg.d0, wg.d1);
  const int qdoc = mk.docs ? a.q_doc[s.q_row + qic] : 0;
  const int klo = a.window ? pos - a.window : 0;
  int khi = s.klen;
  if (a.window) khi = min(khi, pos + a.window + 1);
  if (a.causal) khi = min(khi, pos + 1);
  const float slope = a.slopes ? a.slopes[head] : 0.f;

  // four values of a row from head dim d on (zeros past DH)
  auto load4 = [&](const T* p, int d) {
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (DH % 4 == 0 && d >= DH) return v;
    if constexpr (std::is_same<T, float>::value) {
      if (vec) return *reinterpret_cast<const f32x4_t*>(p + d);
    } else {
      if (vec) {
        const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p + d);
        return f32x4_t{__uint_as_float(x[0] << 16), __uint_as_float(x[0] & 0xffff0000u), __uint_as_float(x[1] << 16),
                       __uint_as_float(x[1] & 0xffff0000u)};
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = load_f32(p + d + j);
    return v;
  };
  f32x4_t qf[ND], o[ND];
  const T* qrow = Q + (s.q_row + qic) * a.ld_q;
#pragma unroll
  for (int t = 0; t < ND; ++t) qf[t] = load4(qrow, 16 * t + 4 * q);
  float m_i, l_i;  // l_i: this lane's keys only, until the end

  f32x4_t kr[NL], vr[NL];
  int id_r = 0;
  auto fetch = [&](int kt) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int idx = min(tid + 256 * i, KT * DP / 4 - 1), row = idx / (DP / 4), d = 4 * (idx - row * (DP / 4));
      const int64_t key = min(kt + row, s.klen - 1);
      kr[i] = load4(K + key * a.ld_k, d);
      vr[i] = load4(V + key * a.ld_v, d);
      if (kt + row >= s.klen) vr[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};  // (masked: nothing of the last key's values)
    }
    if (mk.docs && tid < KT) id_r = a.k_doc[s.k_row + min(kt + tid, s.klen - 1)];
  };

  // (modes of a redo as in attn_scored.hip: 0 finite values only, 1 whether
  // not finite, 2 and 3 whether also not +inf, not -inf)
  auto pass = [&](auto nf_tag, int mode) {
    constexpr bool NF = decltype(nf_tag)::value;
#pragma unroll
    for (int t = 0; t < ND; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_i = -INFINITY, l_i = 0.f;
    TileIter<256> it(a, s, mk, wg, tile_docs, a.splits, split);
    int tl = -1, cls = 0, half = HALVES - 1;
    // next step: (key offset, or -1; masks needed)
    auto next = [&](int& kt, int& cl) {
      if (++half < HALVES && tl >= 0 && tl * kTile + half * KT < s.klen) {
        kt = tl * kTile + half * KT, cl = cls;
        return;
      }
      tl = it.next();
      half = 0;
      if (tl >= 0) cls = it.cls(wg, tl);
      kt = tl >= 0 ? tl * kTile : -1, cl = cls;
    };
    int kt, cl;
    next(kt, cl);
    if (kt >= 0) fetch(kt);
    while (kt >= 0) {
      int kn, cn;
      next(kn, cn);
      __syncthreads();  // the previous step's reads
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int idx = min(tid + 256 * i, KT * DP / 4 - 1), row = idx / (DP / 4), d = 4 * (idx - row * (DP / 4));
        *reinterpret_cast<f32x4_t*>(Ks + row * LDR + d) = kr[i];
        if constexpr (NF) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float v = vr[i][j];
            const bool bad = !(fabsf(v) < INFINITY);
            vr[i][j] = mode == 0 ? (bad ? 0.f : v)
                                 : (bad && !(mode == 2 && v == INFINITY) && !(mode == 3 && v == -INFINITY) ? 1.f : 0.f);
          }
        }
        *reinterpret_cast<f32x4_t*>(Vs + row * LDR + d) = vr[i];
      }
      if (mk.docs && tid < KT) ids[tid] = id_r;
      __syncthreads();
      if (kn >= 0) fetch(kn);
      f32x4_t sc[NB];
      float tmax = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        sc[kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          const f32x4_t kf = *reinterpret_cast<const f32x4_t*>(Ks + (kb * 16 + c) * LDR + 16 * t + 4 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qf[t][j], sc[kb], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = kb * 16 + 4 * q + e, key = kt + i;
          float x = sc[kb][e] * a.scale;
          if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
          if (a.slopes) x -= slope * fabsf(static_cast<float>(pos - key));
          if (cl != 1) {
            const bool vis = key < s.prefix || (key >= klo && key < khi && (!mk.docs || ids[i] == qdoc));
            x = vis ? x : -INFINITY;
          }
          sc[kb][e] = x;
          tmax = fmaxf(tmax, x);
        }
      }
      tmax = fmaxf(tmax, __shfl_xor(tmax, 16, 64));
      tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
      const float m_new = fmaxf(m_i, tmax);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = m_i == -INFINITY ? 0.f : expf(m_i - m_use);
      m_i = m_new;
      l_i *= alpha;
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] *= alpha;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = expf(sc[kb][e] - m_use);
          l_i += p;
          const float* vrow = Vs + (kb * 16 + 4 * q + e) * LDR + c;
#pragma unroll
          for (int t = 0; t < ND; ++t) o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(vrow[16 * t], p, o[t], 0, 0, 0);
        }
      kt = kn, cl = cn;
    }
    l_i += __shfl_xor(l_i, 16, 64);
    l_i += __shfl_xor(l_i, 32, 64);
    __syncthreads();
  };

  if (tid == 0) flag = 0;  // ordered before other waves' writes by the pass's last barrier
  pass(std::false_type{}, 0);
  bool bad = false;
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[t][e]) < INFINITY);
  if (__any(bad && live) && lane == 0) flag = 1;
  __syncthreads();
  if (flag) {  // uniform over the workgroup
    uint32_t saw[3] = {};
#pragma unroll 1
    for (int mode = 1; mode <= 3; ++mode) {
      pass(std::true_type{}, mode);
      uint32_t bits = 0;
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) bits |= o[t][e] > 0.f ? 1u << (4 * t + e) : 0u;
      if (mode == 1) saw[0] = bits;
      if (mode == 2) saw[1] = bits;
      if (mode == 3) saw[2] = bits;
    }
    pass(std::true_type{}, 0);
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t bit = 1u << (4 * t + e);
        if (saw[0] & bit) o[t][e] = !(saw[1] & bit) ? INFINITY : !(saw[2] & bit) ? -INFINITY : __builtin_nanf("");
      }
  }
  if (!live) return;
  if (a.splits > 1) {
    float* part = a.part + (static_cast<int64_t>(blockIdx.x) * a.splits + split) * part_floats(kRows, DH);
    const int row = wave * 16 + c;
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (DP == DH || 16 * t + 4 * q + e < DH) part[row * DH + 16 * t + 4 * q + e] = o[t][e];
    if (q == 0) {
      part[kRows * DH + row] = m_i;
      part[kRows * DH + kRows + row] = l_i;
    }
    return;
  }
  const float inv = l_i > 0.f || l_i != l_i ? 1.f / l_i : 0.f;
  T* O = static_cast<T*>(a.o) + (s.q_row + qi) * a.ld_o + static_cast<int64_t>(head) * DH + 4 * q;
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (DP == DH || 16 * t + 4 * q + e < DH) store_f32(O + 16 * t + e, o[t][e] * inv);
}

template <typename T>
void launch_typed(const AttnScoredArgs& a, hipStream_t st) {
  const uintptr_t align = 4 * sizeof(T) - 1;
  auto ok = [&](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & align) == 0 && ld % 4 == 0; };
  const int vec = ok(a.q, a.ld_q) && ok(a.k, a.ld_k) && ok(a.v, a.ld_v);
  const dim3 grid(static_cast<unsigned>(a.B * a.H * a.n_blocks), static_cast<unsigned>(a.splits));
  switch (a.Dh) {
    case 8: attn_scored_f32_kernel<T, 8><<<grid, 256, 0, st>>>(a, vec); break;
    case 16: attn_scored_f32_kernel<T, 16><<<grid, 256, 0, st>>>(a, vec); break;
    case 32: attn_scored_f32_kernel<T, 32><<<grid, 256, 0, st>>>(a, vec); break;
    case 64: attn_scored_f32_kernel<T, 64><<<grid, 256, 0, st>>>(a, vec); break;
    default: attn_scored_f32_kernel<T, 128><<<grid, 256, 0, st>>>(a, vec); break;
  }
}

}  // namespace

void launch_attn_scored_f32(const AttnScoredArgs& a, hipStream_t st) {
  if (a.dtype == DT_BF16)
    launch_typed<bf16_t>(a, st);
  else
    launch_typed<float>(a, st);
}

}  // namespace sjh
