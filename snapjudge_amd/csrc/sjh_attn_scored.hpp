// sjh_attn_scored.hpp -- what the kernels of attention with modified scores
// share: where a work item lies, which key tiles it needs, partial results.
#pragma once

#include "sjh_common.hpp"
#include "sjh_kernels.hpp"

namespace sjh {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;  // keys per tile
constexpr int kMaxPos = 1 << 29;  // rows too: positions and their differences, and a window more, stay in 32 bits

// Row count of a partial result's block, and its floats: O [rows][Dh], then
// the rows' softmax offsets (log2 domain) and weight sums.
__host__ __device__ inline int64_t part_floats(int rows, int Dh) { return static_cast<int64_t>(rows) * (Dh + 2); }

// A sequence, clamped to the rows that the buffers hold and the bounds that
// the grid was sized by: nothing read from device memory is trusted further.
struct Seq {
  int64_t q_row, k_row;
  int qlen, klen, pos0, prefix;
};
__device__ __forceinline__ Seq load_seq(const AttnScoredArgs& a, int b) {
  Seq s;
  const int qs = min(max(a.q_start[b], 0), a.q_rows), ks = min(max(a.k_start[b], 0), a.k_rows);
  s.q_row = qs;
  s.k_row = ks;
  s.qlen = min(max(a.q_len[b], 0), min(a.max_q, a.q_rows - qs));
  s.klen = min(max(a.k_len[b], 0), min(a.max_k, a.k_rows - ks));
  s.pos0 = a.q_pos ? min(max(a.q_pos[b], 0), kMaxPos) : 0;
  s.prefix = a.prefix ? min(max(a.prefix[b], 0), s.klen) : 0;
  return s;
}

// Positions [p0, p1] and documents [d0, d1] of a set of queries.
struct QRange {
  int p0, p1, d0, d1;
};

// The masks of a sequence against tiles of its keys.
struct Masks {
  int klen, prefix, window, causal;
  bool docs;
  // Whether any (need) or every (full) query of r may see a key of tile
  // [k0, k0 + 64), whose documents lie in [t0, t1].  need errs on the side of
  // reading a tile: a range of documents can hold ids that no key has.
  __device__ __forceinline__ bool need(const QRange& r, int k0, int t0, int t1) const {
    if (k0 < prefix) return true;
    const int k1 = min(k0 + kTile, klen) - 1;
    return (!causal || k0 <= r.p1) && (!window || (k0 - r.p1 <= window && r.p0 - k1 <= window)) &&
           (!docs || (t0 <= r.d1 && t1 >= r.d0));
  }
  __device__ __forceinline__ bool full(const QRange& r, int k0, int t0, int t1) const {
    const int k1 = k0 + kTile - 1;
    if (k1 >= klen) return false;
    if (k1 < prefix) return true;
    return (!causal || k1 <= r.p0) && (!window || (r.p1 - k0 <= window && k1 - r.p0 <= window)) &&
           (!docs || (t0 == t1 && r.d0 == r.d1 && t0 == r.d0));
  }
};

// Wave-wide minimum and maximum (every lane takes part).
__device__ __forceinline__ void wave_range(int& lo, int& hi) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    lo = min(lo, __shfl_xor(lo, off, 64));
    hi = max(hi, __shfl_xor(hi, off, 64));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
}

// Documents of queries [q0, q0 + n) of a sequence (n >= 1), the same in every lane.
__device__ __forceinline__ void doc_range(const AttnScoredArgs& a, const Seq& s, int q0, int n, int& d0, int& d1) {
  d0 = 0x7fffffff, d1 = -0x7fffffff - 1;
  for (int i = threadIdx.x & 63; i < n; i += 64) {
    const int d = a.q_doc[s.q_row + q0 + i];
    d0 = min(d0, d);
    d1 = max(d1, d);
  }
  wave_range(d0, d1);
}

// The key tiles that a workgroup's queries need, in order.  64 tiles at a time
// (4096 keys) a lane decides about one, from the positions and, with
// documents, the range of the tile's ids; the wave's vote is the list.  Every
// wave of the workgroup walks the same list in step: with documents a new word
// holds barriers.
template <int NT>
struct TileIter {
  const AttnScoredArgs& a;
  const Seq& s;
  const Masks& m;
  const QRange& wg;  // the workgroup's queries
  int2* tile_docs;   // LDS, 64 entries
  int stride, mine;
  uint64_t mask = 0;
  int word = -1, t0 = 0, t1 = 0;  // lane t: documents of tile 64 word + t
  int before = 0;                 // entries of earlier words

  __device__ __forceinline__ TileIter(const AttnScoredArgs& a_, const Seq& s_, const Masks& m_, const QRange& wg_, int2* td,
                                      int stride_ = 1, int mine_ = 0)
      : a(a_), s(s_), m(m_), wg(wg_), tile_docs(td), stride(stride_), mine(mine_) {}

  __device__ __forceinline__ void eval() {
    const int lane = threadIdx.x & 63;
    const int k0 = (word * 64 + lane) * kTile;
    if (m.docs) {
      // NT / 64 threads per tile, its ids taken in turn; keys past the end
      // repeat the last one
      constexpr int TPT = NT / 64;
      const int t = threadIdx.x / TPT, f = threadIdx.x % TPT;
      const int kt = (word * 64 + t) * kTile;
      int lo = 0x7fffffff, hi = -0x7fffffff - 1;
      if (kt < m.klen) {
        const int* ids = a.k_doc + s.k_row;
#pragma unroll
        for (int i = 0; i < kTile / TPT; ++i) {
          const int d = ids[min(kt + f + TPT * i, m.klen - 1)];
          lo = min(lo, d);
          hi = max(hi, d);
        }
      }
#pragma unroll
      for (int off = 1; off < TPT; off <<= 1) {
        lo = min(lo, __shfl_xor(lo, off, 64));
        hi = max(hi, __shfl_xor(hi, off, 64));
      }
      __syncthreads();  // the last word's reads
      if (f == 0) tile_docs[t] = make_int2(lo, hi);
      __syncthreads();
      const int2 d = tile_docs[lane];
      t0 = d.x, t1 = d.y;
    }
    const bool need = k0 < m.klen && m.need(wg, k0, t0, t1);
    mask = __ballot(need);
    if (stride > 1) {
      const int rank = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                                 __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
      const int total = before + __builtin_popcountll(mask);
      mask = __ballot(need && (before + rank) % stride == mine);
      before = total;
    }
  }
  // Tile of the next entry of its own, or -1.
  __device__ __forceinline__ int next() {
    while (mask == 0) {
      if ((word + 1) * 64 * kTile >= m.klen) return -1;
      ++word;
      eval();
    }
    const int t = __builtin_ctzll(mask);
    mask &= mask - 1;
    return word * 64 + t;
  }
  // How the queries of r stand to the tile last returned: 0 see nothing of it,
  // 1 all of it, 2 some.
  __device__ __forceinline__ int cls(const QRange& r, int tile) const {
    const int l0 = __builtin_amdgcn_readlane(t0, tile & 63), l1 = __builtin_amdgcn_readlane(t1, tile & 63);
    if (!m.need(r, tile * kTile, l0, l1)) return 0;
    return m.full(r, tile * kTile, l0, l1) ? 1 : 2;
  }
};

}  // namespace

}  // namespace sjh
