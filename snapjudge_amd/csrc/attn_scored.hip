// attn_scored.hip -- attention with modified scores for gfx950 (bf16, heads of
// 64 or 128):
//
//   s(p, j) = cap tanh(scale q_p . k_j / cap) - slope_h |p - j|
//   o_p = sum_j softmax_j(s(p, j)) v_j over the visible keys j
//
// with key j visible where j < prefix, or where it is not after p (causal), at
// most `window` away and of p's document.  One pass over the keys with a
// running maximum and sum; nothing of the scores leaves the registers.
//
// A wave owns 32 queries and takes 64-key tiles: S^T = K Q^T by
// v_mfma_f32_32x32x16_bf16 (a lane holds 32 of the tile's scores of one
// query), the scores' cap, bias, masks and exponentials in registers, O^T += V^T
// P^T with P^T straight from the accumulator (its key order is the MFMA's k
// order) and V^T through transposed LDS reads.  K and V tiles come by
// direct-to-LDS loads into a ring, XOR-swizzled.
//
// Which tiles: the mask's positions and each tile's range of documents decide
// before anything of the tile is read (TileIter); a tile that every query of
// a wave sees whole runs without masks.  Two shapes:
//  - four waves of 32 queries share the ring (128 queries a workgroup; three
//    workgroups share a CU at head_dim 64, two at 128), without a running maximum
//    at first: rows whose weight sum or outputs come out of range run again;
//  - few queries: a workgroup owns 32 (with shared key heads, the queries of
//    all heads of the group where they fit), each wave takes every NW-th
//    needed tile through a ring of its own, further workgroups further tiles
//    (splits); sums meet in LDS and, split, in a second launch.
//
// What bounds it: the vector pipe.  A lane's score costs the cap's polynomial (five
// instructions), the exponential (a quarter of the rate), its rounding and its
// share of the sum, about 50 cycles per 64 scores against 16 of the matrix pipe at
// head_dim 64; few queries over long keys are bound by the bytes of K and V.
// Measured, bf16: 16 sequences of 1800 to 2048 tokens of packed documents, 12 heads
// of 64, cap, 156 us; two causal ones of 5000 and 8192 with distance biases 196 us; 3
// sequences of 6000 to 8191 keys, a few queries each, 16 heads of 128 on 4 key
// heads, 17 us and 5 for the join.
//
// A masked key takes no part, whatever its values: its score is replaced, and
// where an infinite or NaN V row met a weight of 0 (the output is then not
// finite), the workgroup runs its tiles again with such values taken out and
// counts apart which sign of them each output really saw (below).
//
// P is rounded to bf16 for the second product, and the weight sum adds the
// rounded weights, so that the weights that V meets sum to one.
#include <algorithm>
#include <type_traits>

#include "sjh_attn_scored.hpp"
#include "sjh_attn_tile.hpp"
#include "sjh_common.hpp"
#include "sjh_host.hpp"
#include "sjh_kernels.hpp"

namespace sjh {

namespace {

constexpr float kLazy = 8.f;  // log2 headroom before the running max is raised
// Ring stages: a workgroup's shared ring, two stages ahead of the one in use where
// three workgroups of them fit a CU (head_dim 64), one ahead else; a wave's own,
// one ahead at head_dim 64, none at 128 (four waves' stages fill the LDS, and
// the waves cover one another: 3 x 8191 keys, 4 key heads, 19.2 us with two waves
// and a stage ahead).
template <int DH, bool KS>
constexpr int ring_stages() {
  return KS ? (DH == 64 ? 2 : 1) : (DH == 64 ? 3 : 2);
}

// tanh(u) = u (c0 + c1 u^2 + c2 u^4 + c3 u^6) + e, |e| < 6e-7 for |u| <= 0.6
// (a least-squares fit over the interval, reweighted to even out the error):
// below the rounding of P by far at any cap whose scores fit fp32.
constexpr float kTanhMax = 0.6f;
constexpr float kTanh0 = 0.99999102f, kTanh1 = -0.33298974f, kTanh2 = 0.12974552f, kTanh3 = -0.039611236f;

// 64 x DH tiles in LDS: 16-byte chunk c of row r at chunk position c ^ swz(r).
// DH 64: kv_swz.  DH 128: a row is all 64 banks, so 16 consecutive rows read
// at one chunk (K fragments) need 16 distinct positions, and the four rows of
// half a wave's transposed V reads (4 chunks of each) distinct groups of four.
template <int DH>
__device__ __forceinline__ int t_swz(int r) {
  return DH == 64 ? kv_swz(r) : ((r & 3) << 2) | ((r >> 2) & 3);
}
template <int DH>
__device__ __forceinline__ int t_off(int row, int col) {
  return row * (DH * 2) + (((col >> 3) ^ t_swz<DH>(row)) << 4) + ((col & 7) << 1);
}

// The V^T fragments of two 32-dim blocks for one 16-key step: transposed reads
// (sjh_attn_tile.hpp's lds_read_tr) at a0 .. a3 + OFF and the wait for them in
// one block, so that no register of theirs is live before it holds its value.
template <int OFF>
__device__ __forceinline__ void lds_read_tr4(s16x4_t (&r)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset field");
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%8\n\tds_read_b64_tr_b16 %1, %5 offset:%8\n\t"
      "ds_read_b64_tr_b16 %2, %6 offset:%8\n\tds_read_b64_tr_b16 %3, %7 offset:%8\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
      : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(OFF)
      : "memory");
}

enum Cap : int { CAP_NONE = 0, CAP_FIXED = 1, CAP_ANY = 2 };
constexpr float kFixedCap = 96.f;

// Redo passes: how a V value enters the product.
enum VMode : int {
  V_FINITE = 0,    // infinities and NaN as 0
  V_BAD = 1,       // 1 where not finite, else 0
  V_NOT_POS = 2,   // 1 where not finite and not +inf
  V_NOT_NEG = 3,   // 1 where not finite and not -inf
};
__device__ __forceinline__ bf16x8_t v_map(bf16x8_t v, int mode) {
  u32x4_t x = __builtin_bit_cast(u32x4_t, v), y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t out = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t b = (x[i] >> (16 * h)) & 0xffffu;
      const bool bad = (b & 0x7f80u) == 0x7f80u;
      uint32_t o;
      if (mode == V_FINITE)
        o = bad ? 0u : b;
      else
        o = bad && !(mode == V_NOT_POS && b == 0x7f80u) && !(mode == V_NOT_NEG && b == 0xff80u) ? 0x3f80u : 0u;
      out |= o << (16 * h);
    }
    y[i] = out;
  }
  return __builtin_bit_cast(bf16x8_t, y);
}

// The work of workgroup (pair of sequence and key head, head of the group,
// query block, split).  NW waves; KS: the waves (and splits) divide the keys.
template <int DH, int NW, bool KS, int CAPM, bool BIAS>
__device__ __forceinline__ void scored_item(const AttnScoredArgs& a, char* smem, int b, int kvh, int g, int qb, int split) {
  constexpr bool CAP = CAPM != CAP_NONE;
  // Capped scores without a bias lie within [-cap, cap]: with the cap at most
  // kFixedCap in log2, weights 2^s need no running maximum: sums of 2^29 of them
  // fit fp32, and rows whose sums or outputs come near its ends run again.
  constexpr bool FIXED = CAPM == CAP_FIXED;
  static_assert(!FIXED || !BIAS, "a bias leaves no lower bound");
  constexpr int ROWB = DH * 2, TILEB = kTile * ROWB;          // bytes of a row, of a K or V tile
  constexpr int STAGE = 2 * TILEB + 256;                      // K, V, the keys' documents
  constexpr int RPI = 1024 / ROWB;                            // rows per load instruction
  constexpr int CPR = ROWB / 16;                              // chunks per row
  constexpr int GRP = kTile / RPI;                            // load instructions per tile
  constexpr int LW = KS ? 1 : NW;                             // waves that share a stage's loads
  constexpr int NL = GRP / LW;                                // ... per wave, K and V each
  constexpr int ST = DH / 16, DB = DH / 32;                   // K steps of QK^T, 32-dim blocks
  constexpr int QB = KS ? 32 : 32 * NW;                       // queries of the workgroup
  constexpr int NS = ring_stages<DH, KS>();
  constexpr int RING = NS * STAGE;                            // bytes of a ring
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  const int l32 = lane & 31, hb = lane >> 5;
  const int G = a.H / a.Hkv;

  const Seq s = load_seq(a, b);
  // this lane's query and head (clamped; lanes without a query store nothing)
  const bool pack = KS && a.pack;
  const int q0 = pack ? 0 : qb * QB;
  if (q0 >= s.qlen) return;  // uniform
  int qi, head;
  bool live;
  if (pack) {
    const int gi = l32 / a.max_q;
    qi = l32 - gi * a.max_q;
    live = gi < G && qi < s.qlen;
    head = kvh * G + min(gi, G - 1);
  } else {
    qi = q0 + (KS ? 0 : wave * 32) + l32;
    live = qi < s.qlen;
    head = kvh * G + g;
  }
  const int qic = min(qi, s.qlen - 1);
  const int pos = s.pos0 + qic;
  const int64_t qrow = s.q_row + qic;

  Masks mk;
  mk.klen = s.klen, mk.prefix = s.prefix, mk.window = a.window, mk.causal = a.causal;
  mk.docs = a.k_doc != nullptr;
  // the workgroup's queries, and the wave's
  QRange wg, wr;
  const int n_wg = min(s.qlen - q0, QB);
  wg.p0 = s.pos0 + q0, wg.p1 = wg.p0 + n_wg - 1, wg.d0 = wg.d1 = 0;
  wr = wg;
  bool wave_active = true;
  if constexpr (!KS) {
    const int w0 = q0 + 32 * wave_s;
    wave_active = w0 < s.qlen;
    const int w0c = min(w0, s.qlen - 1);
    wr.p0 = s.pos0 + w0c, wr.p1 = wr.p0 + min(s.qlen - w0c, 32) - 1;
    if (mk.docs) doc_range(a, s, w0c, min(s.qlen - w0c, 32), wr.d0, wr.d1);
  }
  if (mk.docs) doc_range(a, s, q0, n_wg, wg.d0, wg.d1);
  if constexpr (KS) wr = wg;
  // what masks and biases ask of the lane's query, in LDS: needed by some tiles
  // only, and spilled registers would be reloaded behind the ring's loads
  int4* qinfo = reinterpret_cast<int4*>(smem + (KS ? NW : 1) * RING + 64 * 8 + 16) + wave * 32 + l32;
  {
    // {position, first key and number of keys of the lane's window and past, document}
    const int klo = a.window ? pos - a.window : 0;
    int khi = s.klen;
    if (a.window) khi = min(khi, pos + a.window + 1);
    if (a.causal) khi = min(khi, pos + 1);
    *qinfo = make_int4(pos, klo, max(khi - klo, 0), mk.docs ? a.q_doc[qrow] : 0);
  }

  const bf16_t* Q = static_cast<const bf16_t*>(a.q) + static_cast<int64_t>(head) * DH;
  const bf16_t* K = static_cast<const bf16_t*>(a.k) + s.k_row * a.ld_k + static_cast<int64_t>(kvh) * DH;
  const bf16_t* V = static_cast<const bf16_t*>(a.v) + s.k_row * a.ld_v + static_cast<int64_t>(kvh) * DH;
  const int* kdoc = mk.docs ? a.k_doc + s.k_row : nullptr;
  bf16x8_t qf[ST];
#pragma unroll
  for (int st = 0; st < ST; ++st) qf[st] = *reinterpret_cast<const bf16x8_t*>(Q + qrow * a.ld_q + 16 * st + 8 * hb);

  // Loads: instruction i of a tile carries rows RPI i + [0, RPI); a lane's
  // 16 bytes land at 16 lane, so it reads the logical chunk that belongs there.
  // The buffer descriptor of a tile starts at its first row and ends with the
  // head's values of its last key: rows past the keys land as zeros.
  const uint32_t kstride = static_cast<uint32_t>(a.ld_k) * 2u, vstride = static_cast<uint32_t>(a.ld_v) * 2u;
  uint32_t koffs[NL], voffs[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = RPI * (i * LW + (KS ? 0 : wave)) + lane / CPR;
    const uint32_t c = static_cast<uint32_t>(((lane % CPR) ^ t_swz<DH>(r)) << 4);
    koffs[i] = r * kstride + c;
    voffs[i] = r * vstride + c;
  }
  char* ring = smem + (KS ? wave_s * RING : 0);
  auto issue = [&](int tile, int buf) {
    char* base = ring + buf * STAGE;
    const int k0 = tile * kTile;
    const uint32_t last = static_cast<uint32_t>(min(kTile, s.klen - k0) - 1);
    const __amdgpu_buffer_rsrc_t rk = seq_rsrc(K + static_cast<int64_t>(k0) * a.ld_k, last * kstride + ROWB);
    const __amdgpu_buffer_rsrc_t rv = seq_rsrc(V + static_cast<int64_t>(k0) * a.ld_v, last * vstride + ROWB);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int grp = i * LW + (KS ? 0 : wave_s);
      load_lds16_buf(rk, koffs[i], 0u, base + grp * 1024);
      load_lds16_buf(rv, voffs[i], 0u, base + TILEB + grp * 1024);
    }
    if (kdoc)  // (every wave the same 64: the count of loads per stage is one for all)
      __builtin_amdgcn_global_load_lds(kdoc + min(k0 + lane, s.klen - 1),
                                       (__attribute__((address_space(3))) void*)(base + 2 * TILEB), 4, 0, 0);
  };

  // operand offsets within a stage: K fragments (row 32 jb + l32, chunk 2 st +
  // hb), V^T fragments through transposed reads (lane group tg covers dims 16
  // (tg % 2) + [0, 16) of a 32-dim block and keys 4 (tg / 2) + [0, 4) of an
  // 8-key half step); neither swizzle sees the 32-row block or the 16-row step
  int koff[ST];
  uint32_t vaddr[DB][2];
  {
    const int tq = lane & 3, tk = (lane >> 2) & 3, tg = lane >> 4;
#pragma unroll
    for (int st = 0; st < ST; ++st) koff[st] = t_off<DH>(l32, 16 * st + 8 * hb);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int hl = 0; hl < 2; ++hl)
        vaddr[db][hl] = lds_addr(ring) + TILEB + t_off<DH>(8 * hl + 4 * (tg >> 1) + tk, db * 32 + 16 * (tg & 1) + 4 * tq);
  }

  // constants of the launch (and, but for packed heads, the head's slope) in
  // scalar registers: the vector ones are what the tile's code is short of
  auto uni = [](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); };
  const float slope1 = BIAS && a.slopes ? a.slopes[head] * kLog2e : 0.f;
  const float slope2 = KS ? slope1 : uni(slope1);
  const float c = uni(a.scale * kLog2e);                     // plain scores to log2
  const float cap2 = uni(CAP ? a.softcap * kLog2e : 0.f);    // the cap in log2
  const float ucap = CAP ? a.scale / a.softcap : 0.f;        // u = ucap raw
  // y = raw (A0 + w (A1 + w (A2 + w A3))), w = raw^2
  const float B0 = c, B1 = B0 * ucap * ucap, B2 = B1 * ucap * ucap, B3 = B2 * ucap * ucap;
  const float A0 = uni(B0 * kTanh0), A1 = uni(B1 * kTanh1), A2 = uni(B2 * kTanh2), A3 = uni(B3 * kTanh3);
  const float raw_max = uni(CAP && fabsf(A3) < INFINITY ? kTanhMax / ucap : -1.f);
  const float kexp = uni(2.f * kLog2e * ucap);
  auto cap_exact = [&](float x) {  // cap2 tanh(ucap x), any x
    const float e = __builtin_amdgcn_exp2f(x * kexp);
    return __builtin_fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + e), cap2);
  };
  auto cap_poly = [&](float x) {  // |x| <= raw_max: the factor of x
    const float w = x * x;
    return __builtin_fmaf(w, __builtin_fmaf(w, __builtin_fmaf(w, A3, A2), A1), A0);
  };

  // Bias of a tile that lies on one side of all of the wave's queries: slope (key
  // - pos), or its negative, is linear in the key, so a 16-deep MFMA step adds the
  // part within the tile to the scores: the key's offset (whole numbers up to 63,
  // exact in bf16) times slope / scale as three bf16 summands, and the tile's
  // part joins the softmax offset.  The matrix pipe has the time; on the vector
  // pipe it is two instructions per score.
  constexpr bool LIN = BIAS && !CAP;
  uint32_t sf0 = 0, sf1 = 0;  // the summands, packed; the operands are made from them per tile
  if constexpr (LIN) {
    const float r = (a.slopes ? a.slopes[head] : 0.f) / a.scale;
    const float r1 = r - bf16_to_f32(f32_to_bf16(r)), r2 = r1 - bf16_to_f32(f32_to_bf16(r1));
    if (hb == 0) sf0 = pack_bf16x2(r, r1), sf1 = pack_bf16x2(r2, 0.f);
  }

  f32x16_t o[DB];
  float m_i, l_i, l_j;

  // One tile from ring slot `slot`.  PART: masks.  MAXR: the running maximum; else
  // weights are 2^s as they come (checked after the pass).  NF: V through v_map(mode) where
  // mode >= 0.  side (whole tiles under a linear bias): 1 keys before the queries,
  // 3 after.
  auto tile = [&](auto part_tag, auto max_tag, auto nf_tag, int mode, int slot, int tl, int side) {
    constexpr bool PART = decltype(part_tag)::value, NF = decltype(nf_tag)::value, NOMAX = !decltype(max_tag)::value;
    const char* sb = ring + slot * STAGE;
    const int kt = tl * kTile;
    constexpr bool LINT = LIN && !PART;
    f32x16_t sc[2];
    const f32x16_t zero16 = {};
    if constexpr (LINT) {
      const uint32_t flip = side == 3 ? 0x80008000u : 0u;
      const u32x4_t s4 = {sf0 ^ flip, sf1 ^ flip, 0u, 0u};
#pragma unroll
      for (int jb = 0; jb < 2; ++jb) {
        // (the upper half of the wave meets zeros of s4: only its summands 0 to 2 count)
        const uint32_t o1 = __float_as_uint(static_cast<float>(32 * jb + l32)) >> 16;
        const u32x4_t k4 = {o1 | o1 << 16, o1, 0u, 0u};
        sc[jb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k4), __builtin_bit_cast(bf16x8_t, s4), zero16, 0, 0, 0);
      }
    }
    bf16x8_t kf[2][4];
#pragma unroll
    for (int s0 = 0; s0 < ST; s0 += 4) {
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int st = 0; st < 4; ++st) kf[jb][st] = *reinterpret_cast<const bf16x8_t*>(sb + jb * (32 * ROWB) + koff[s0 + st]);
#pragma unroll
      for (int st = 0; st < 4; ++st)
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
          sc[jb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[jb][st], qf[s0 + st], !LINT && s0 + st == 0 ? zero16 : sc[jb], 0, 0, 0);
    }
    // element (jb, e) is key kt + 4 hb + key_of(jb, e)
    auto key_of = [](int jb, int e) { return 32 * jb + 8 * (e >> 2) + (e & 3); };
    const int base = kt + 4 * hb;
    bool small = true;
    if constexpr (CAP) {
      float amax = 0.f;
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(sc[jb][e]));
      small = !__any(!(amax <= raw_max));
    }
    // FUSED: the cap's last product and the softmax offset meet in one FMA
    constexpr bool FUSED = !PART && (!BIAS || LINT);
    float tb = 0.f;  // the tile's bias
    if constexpr (LINT) {
      const int qp = qinfo->x;
      tb = slope2 * static_cast<float>(side == 3 ? qp - kt : kt - qp);
    }
    float tmax = -INFINITY;
    if constexpr (FUSED && NOMAX) {
    } else if constexpr (FUSED) {
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, sc[jb][e]);
      tmax = wave_max32(tmax);
      // (all rise with the score; the form that the tile's scores take, whose errors
      // a large cap would otherwise set apart)
      tmax = !CAP ? __builtin_fmaf(tmax, c, tb) : small ? tmax * cap_poly(tmax) : cap_exact(tmax);
    } else {
      const int4 qi4 = *qinfo;
      const float d0 = static_cast<float>(qi4.x - base);
      if (!CAP || small) {
        if constexpr (CAP) asm volatile("" ::: "memory");  // a branch, not a select
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sc[jb][e] *= CAP ? cap_poly(sc[jb][e]) : c;
          }
      } else {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sc[jb][e] = cap_exact(sc[jb][e]);
          }
      }
      if constexpr (BIAS) {
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            sc[jb][e] = __builtin_fmaf(-slope2, fabsf(d0 - static_cast<float>(key_of(jb, e))), sc[jb][e]);
      }
      if constexpr (PART) {
        // (no short cuts: each would be a branch per score; a range of keys is
        // one unsigned comparison)
        const uint32_t len = static_cast<uint32_t>(qi4.z);
        const int qdoc = qi4.w;
        auto mask = [&](auto docs_tag, auto pre_tag, auto range_tag) {
          int pre = s.prefix - base, lo = qi4.y - base;
          // (each form's own: the compiler would compute the comparisons that the
          // forms share ahead of the branch and hold 32 of them)
          asm volatile("" : "+v"(lo), "+v"(pre));
#pragma unroll
          for (int jb = 0; jb < 2; ++jb)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              int4 id = {0, 0, 0, 0};
              if constexpr (decltype(docs_tag)::value) id = reinterpret_cast<const int4*>(sb + 2 * TILEB)[hb + 8 * jb + 2 * q];
              const int dv[4] = {id.x, id.y, id.z, id.w};
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                const int k = key_of(jb, 4 * q + t);
                bool vis = true;
                if constexpr (decltype(range_tag)::value) vis = static_cast<uint32_t>(k - lo) < len;
                if constexpr (decltype(docs_tag)::value) vis &= dv[t] == qdoc;
                if constexpr (decltype(pre_tag)::value) vis |= k < pre;
                sc[jb][4 * q + t] = vis ? sc[jb][4 * q + t] : -INFINITY;
              }
            }
        };
        // (uniform) the documents alone decide where nothing else reaches the tile
        const bool range = a.window || a.causal || kt + kTile > s.klen;
        using Y = std::true_type;
        using N = std::false_type;
        if (mk.docs) {
          if (kt < s.prefix)
            mask(Y{}, Y{}, Y{});
          else if (range)
            mask(Y{}, N{}, Y{});
          else
            mask(Y{}, N{}, N{});
        } else if (kt < s.prefix) {
          mask(N{}, Y{}, Y{});
        } else {
          mask(N{}, N{}, Y{});
        }
      }
      if constexpr (!NOMAX) {
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, sc[jb][e]);
        tmax = wave_max32(tmax);
      }
    }
    // the running max, raised only when the tile's exceeds it by more than
    // kLazy (weights stay below 2^kLazy; the quotient is exact either way)
    if constexpr (!NOMAX) {
      const bool bump = tmax > m_i + kLazy;
      if (__any(bump)) {
        asm volatile("" ::: "memory");  // a branch (rarely taken), not a select
        const float m_new = bump ? tmax : m_i;
        const float alpha = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - m_new);
        m_i = m_new;
        l_i *= alpha;
        l_j *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
      }
    }
    const float m_use = NOMAX || m_i == -INFINITY ? 0.f : m_i;
    if constexpr (FUSED) {
      const float off = LINT ? tb - m_use : -m_use;  // (0 under a fixed offset: a product instead of the FMA)
      if (!CAP || small) {
        if constexpr (CAP) asm volatile("" ::: "memory");
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sc[jb][e] = __builtin_amdgcn_exp2f(NOMAX && CAP ? sc[jb][e] * cap_poly(sc[jb][e])
                                               : NOMAX && !LINT ? sc[jb][e] * c
                                                     : __builtin_fmaf(sc[jb][e], CAP ? cap_poly(sc[jb][e]) : c, off));
          }
      } else {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sc[jb][e] = __builtin_amdgcn_exp2f(NOMAX ? cap_exact(sc[jb][e]) : cap_exact(sc[jb][e]) - m_use);
          }
      }
    } else {
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[jb][e] = __builtin_amdgcn_exp2f(NOMAX ? sc[jb][e] : sc[jb][e] - m_use);
    }
    // O^T += V^T P^T.  The MFMA's k index 8 hb + t of 16-key step g stands for
    // key 16 g + 4 hb + t (t < 4) or 16 g + 8 + 4 hb + t - 4, as the S^T
    // accumulator holds them.
    uint32_t vb[DB][2];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int hl = 0; hl < 2; ++hl) vb[db][hl] = vaddr[db][hl] + slot * STAGE;
    static_for<0, 4>([&](auto g_tag) {
      constexpr int gk = decltype(g_tag)::value;
      bf16x8_t pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) pf[e] = static_cast<__bf16>(sc[gk >> 1][8 * (gk & 1) + e]);
      const bf16x2_t ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
      l_i = __builtin_amdgcn_fdot2_f32_bf16((bf16x2_t){pf[0], pf[1]}, ones, l_i, false);
      l_j = __builtin_amdgcn_fdot2_f32_bf16((bf16x2_t){pf[2], pf[3]}, ones, l_j, false);
      l_i = __builtin_amdgcn_fdot2_f32_bf16((bf16x2_t){pf[4], pf[5]}, ones, l_i, false);
      l_j = __builtin_amdgcn_fdot2_f32_bf16((bf16x2_t){pf[6], pf[7]}, ones, l_j, false);
#pragma unroll
      for (int dp = 0; dp < DB / 2; ++dp) {
        s16x4_t vr[4];
        lds_read_tr4<gk * 16 * ROWB>(vr, vb[2 * dp][0], vb[2 * dp][1], vb[2 * dp + 1][0], vb[2 * dp + 1][1]);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const s16x4_t lo = vr[2 * d], hi = vr[2 * d + 1];
          bf16x8_t vf = __builtin_bit_cast(bf16x8_t, (s16x8_t){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
          if constexpr (NF)
            if (mode >= 0) vf = v_map(vf, mode);
          o[2 * dp + d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf, o[2 * dp + d], 0, 0, 0);
        }
      }
    });
  };

  // One pass over the needed tiles.
  int2* tile_docs = reinterpret_cast<int2*>(smem + (KS ? NW : 1) * RING);
  int* flag = reinterpret_cast<int*>(tile_docs + 64);
  // REDO: a pass again, with the running maximum and (mode >= 0) V mapped; it masks
  // every tile, so that it has one body of its own.  Few queries (KS) keep the
  // maximum at first too: what a wave or split holds is not the whole row.
  // WHOLE: the tile needs no masks.
  auto run = [&](int cl, auto whole_tag, auto redo_tag, int mode, int slot, int t) {
    using Y = std::true_type;
    using N = std::false_type;
    using Max = std::integral_constant<bool, KS>;
    if constexpr (decltype(redo_tag)::value)
      tile(Y{}, Y{}, Y{}, mode, slot, t, cl);
    else if constexpr (decltype(whole_tag)::value)
      tile(N{}, Max{}, N{}, mode, slot, t, cl);
    else
      tile(Y{}, Max{}, N{}, mode, slot, t, cl);
  };
  // a tile's class for the wave: 0 nothing, 2 masks, 1 whole (3 whole, behind the
  // queries; under a linear bias only a tile on one side counts as whole)
  auto class_of = [&](const auto& it, int t) {
    if (!wave_active) return 0;
    const int cl = it.cls(wr, t);
    if (!LIN || cl != 1) return cl;
    return t * kTile + kTile - 1 <= wr.p0 ? 1 : t * kTile >= wr.p1 ? 3 : 2;
  };
  auto pass = [&](auto redo_tag, int mode) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] = 0.f;
    constexpr bool kMax = KS || decltype(redo_tag)::value;
    m_i = kMax ? -INFINITY : 0.f, l_i = 0.f, l_j = 0.f;
    TileIter<64 * NW> it(a, s, mk, wg, tile_docs, KS ? a.splits * NW : 1, KS ? split * NW + wave_s : 0);
    if constexpr (!KS) {
      // the tile in use and the NS - 1 after it, with their classes
      int tq[NS], cq[NS], slot = 0;
#pragma unroll
      for (int i = 0; i < NS - 1; ++i) {
        tq[i] = it.next();
        cq[i] = tq[i] >= 0 ? class_of(it, tq[i]) : 0;
        if (tq[i] >= 0) issue(tq[i], i);
      }
      auto step = [&](auto whole_tag) {
        tq[NS - 1] = it.next();  // (its barriers, if any, before the loads are waited for)
        cq[NS - 1] = tq[NS - 1] >= 0 ? class_of(it, tq[NS - 1]) : 0;
        if (NS == 2 || tq[1] < 0)
          wait_vmcnt<0>();
        else if (kdoc)
          wait_vmcnt<(NS - 2) * (2 * NL + 1)>();
        else
          wait_vmcnt<(NS - 2) * 2 * NL>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");  // (the barrier alone orders no reads for the compiler)
        const int last = slot == 0 ? NS - 1 : slot - 1;  // the slot that the tile before was in
        if (tq[NS - 1] >= 0) issue(tq[NS - 1], last);
        if (cq[0] != 0) run(cq[0], whole_tag, redo_tag, mode, slot, tq[0]);
        slot = slot == NS - 1 ? 0 : slot + 1;
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) tq[i] = tq[i + 1], cq[i] = cq[i + 1];
      };
      // runs of whole tiles and of others, a loop each: one loop with a branch
      // between the two bodies copies the accumulators on every tile
      while (tq[0] >= 0) {
        if constexpr (!decltype(redo_tag)::value)
          while (tq[0] >= 0 && (cq[0] & 1)) step(std::true_type{});
        while (tq[0] >= 0 && (decltype(redo_tag)::value || !(cq[0] & 1))) step(std::false_type{});
      }
    } else {
      // this wave's tiles: every (splits * NW)-th of the list
      int t = it.next(), n = 0;
      int cl = t >= 0 ? class_of(it, t) : 0;
      if (t >= 0) issue(t, 0);
      auto step = [&](auto whole_tag) {
        const int tn = it.next();
        const int cn = tn >= 0 ? class_of(it, tn) : 0;
        wait_vmcnt<0>();  // (its memory clobber keeps the last tile's reads above the next loads)
        if (NS > 1 && tn >= 0) issue(tn, (n + 1) % NS);
        run(cl, whole_tag, redo_tag, mode, n % NS, t);
        if (NS == 1 && tn >= 0) {
          wait_lgkm0();  // the tile's reads
          asm volatile("" ::: "memory");
          issue(tn, 0);
        }
        t = tn, cl = cn, ++n;
      };
      while (t >= 0) {
        if constexpr (!decltype(redo_tag)::value)
          while (t >= 0 && (cl & 1)) step(std::true_type{});
        while (t >= 0 && (decltype(redo_tag)::value || !(cl & 1))) step(std::false_type{});
      }
    }
    l_i += l_j;
    l_i += __shfl_xor(l_i, 32, 64);
    __syncthreads();  // every wave is done with the ring and the list
  };
  if (tid == 0) *flag = 0;  // ordered before other waves' writes by the pass's last barrier
  pass(std::false_type{}, -1);
  auto vote = [&](bool bad) {  // whether any wave's
    if (__any(bad && live) && lane == 0) *flag = 1;
    __syncthreads();
    const bool any = *flag != 0;
    __syncthreads();
    if (any && tid == 0) *flag = 0;
    return any;
  };
  // an output that is not finite: a visible key's value, or a masked one's times
  // a weight of 0
  auto unclean = [&] {
    bool bad = false;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) bad |= !(fabsf(o[db][e]) < INFINITY);
    return bad;
  };
  {
    // Without the maximum: every row's weight sum must lie in [2^-60, 2^64].  Then
    // nothing overflowed, and what flushed to zero (weights, and their products
    // with values, below 2^-126) is under 2^-66 per key of the sum.  Else (a row
    // that sees no key among them, but where a cap keeps the sums of others above
    // 0) the workgroup runs again with the maximum, as it does for an output that is
    // not finite.
    bool again = unclean();
    if constexpr (!KS) again |= FIXED ? l_i > 0.f && l_i < 0x1p-60f : !(l_i >= 0x1p-60f && l_i <= 0x1p64f);
    if (vote(again)) {  // uniform over the workgroup
      pass(std::true_type{}, -1);
      again = vote(unclean());
    } else {
      again = false;
    }
    if (again) {
      // which outputs saw a value that is not finite, and whether any but
      // +inf, any but -inf; then the sums of the finite ones
      uint32_t saw[3][DB / 2] = {};
#pragma unroll 1
      for (int mode = V_BAD; mode <= V_NOT_NEG; ++mode) {
        pass(std::true_type{}, mode);
        uint32_t bits[DB / 2] = {};
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) bits[db >> 1] |= o[db][e] > 0.f ? 1u << (16 * (db & 1) + e) : 0u;
#pragma unroll
        for (int i = 0; i < DB / 2; ++i) {
          if (mode == V_BAD) saw[0][i] = bits[i];
          if (mode == V_NOT_POS) saw[1][i] = bits[i];
          if (mode == V_NOT_NEG) saw[2][i] = bits[i];
        }
      }
      pass(std::true_type{}, V_FINITE);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t bit = 1u << (16 * (db & 1) + e);
          if (saw[0][db >> 1] & bit)
            o[db][e] = !(saw[1][db >> 1] & bit) ? INFINITY : !(saw[2][db >> 1] & bit) ? -INFINITY : __builtin_nanf("");
        }
    }
  }

  if constexpr (!KS) {
    if (!live) return;
    const float inv = l_i > 0.f || l_i != l_i ? 1.f / l_i : 0.f;
    bf16_t* O = static_cast<bf16_t*>(a.o) + qrow * a.ld_o + static_cast<int64_t>(head) * DH;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        u32x2_t w;
        w[0] = pack_bf16x2(o[db][4 * gq + 0] * inv, o[db][4 * gq + 1] * inv);
        w[1] = pack_bf16x2(o[db][4 * gq + 2] * inv, o[db][4 * gq + 3] * inv);
        *reinterpret_cast<u32x2_t*>(O + db * 32 + 8 * gq + 4 * hb) = w;
      }
  } else {
    // the waves' sums meet in LDS (the rings are done with): each scales its
    // own by 2^(m - M), M the largest offset, and the threads add them in wave
    // order.  Rows are padded by four floats against bank conflicts.
    constexpr int LDO = DH + 4;
    float* red = reinterpret_cast<float*>(smem);          // [NW][32][LDO]
    float* ml = red + NW * 32 * LDO;                      // [NW][32] offsets
    float* ll = ml + NW * 32;                             // [NW][32] sums
    static_assert((NW * 32 * LDO + 2 * NW * 32) * 4 <= NW * RING, "the sums fit the rings");
    if (hb == 0) {
      ml[wave * 32 + l32] = m_i;
      ll[wave * 32 + l32] = l_i;
    }
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[w * 32 + l32]);
    // (a wave without a tile has offset -inf and sums of 0; a NaN stays in its query)
    const float f = m_i == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_i - M);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq)
        *reinterpret_cast<f32x4_t*>(red + (wave * 32 + l32) * LDO + db * 32 + 8 * gq + 4 * hb) =
            (f32x4_t){o[db][4 * gq] * f, o[db][4 * gq + 1] * f, o[db][4 * gq + 2] * f, o[db][4 * gq + 3] * f};
    __syncthreads();
    const int item = ((b * a.Hkv + kvh) * (pack ? 1 : G) + (pack ? 0 : g)) * a.n_blocks + qb;
    float* part = a.splits > 1 ? a.part + (static_cast<int64_t>(item) * a.splits + split) * part_floats(32, DH) : nullptr;
    constexpr int C4 = DH / 4;
    for (int i = tid; i < 32 * C4; i += 64 * NW) {
      const int q = i / C4, d = 4 * (i - q * C4);
      float Mq = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) Mq = fmaxf(Mq, ml[w * 32 + q]);
      float l = 0.f;
      f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = ml[w * 32 + q];
        l += ll[w * 32 + q] * (mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - Mq));
        x += *reinterpret_cast<const f32x4_t*>(red + (w * 32 + q) * LDO + d);
      }
      if (part) {
        *reinterpret_cast<f32x4_t*>(part + q * DH + d) = x;
        if (d == 0) {
          part[32 * DH + q] = Mq;
          part[32 * DH + 32 + q] = l;
        }
        continue;
      }
      const int gi = pack ? q / a.max_q : 0;
      const int oq = pack ? q - gi * a.max_q : q0 + q;
      if (gi >= G || oq >= s.qlen) continue;
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      const int oh = kvh * G + (pack ? gi : g);
      bf16_t* O = static_cast<bf16_t*>(a.o) + (s.q_row + oq) * a.ld_o + static_cast<int64_t>(oh) * DH + d;
      *reinterpret_cast<u32x2_t*>(O) = (u32x2_t){pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv)};
    }
  }
}

// LDS: the ring or rings, the list's documents, the redo flag, the queries' masks.
template <int DH, int NW, bool KS>
constexpr int lds_bytes() {
  return (KS ? NW : 1) * ring_stages<DH, KS>() * (2 * kTile * DH * 2 + 256) + 64 * 8 + 16 + 32 * NW * 16;
}

// Query blocks of 128.  Workgroup i runs on XCD i % 8: the blocks and heads
// that read one key head go to one XCD, close together, where the pairs fill
// the XCDs evenly enough (a.pack is then 0; -1: blocks in plain order).
template <int DH, int CAP, bool BIAS>
__global__ __launch_bounds__(256, DH == 64 ? 3 : 2) void attn_scored_kernel(AttnScoredArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[lds_bytes<DH, 4, false>()];
  const int G = a.H / a.Hkv, per = G * a.n_blocks;
  int pair, r;
  if (a.pack < 0) {
    const int np = a.B * a.Hkv;  // causal: the longest rows of all pairs first
    pair = a.causal ? blockIdx.x % np : blockIdx.x / per;
    r = a.causal ? blockIdx.x / np : blockIdx.x - pair * per;
  } else if (a.causal) {  // the longest rows of all of the XCD's pairs first
    const int xcd = blockIdx.x & 7, kx = blockIdx.x >> 3, np = (a.B * a.Hkv + 7) / 8;
    r = kx / np;
    pair = xcd + 8 * (kx - r * np);
  } else {
    const int xcd = blockIdx.x & 7, kx = blockIdx.x >> 3;
    pair = xcd + 8 * (kx / per);
    r = kx % per;
  }
  if (pair >= a.B * a.Hkv) return;  // uniform
  const int b = pair / a.Hkv, kvh = pair - b * a.Hkv;
  int qb = r / G;
  const int g = r - qb * G;
  if (a.causal) qb = a.n_blocks - 1 - qb;
  scored_item<DH, 4, false, CAP, BIAS>(a, smem, b, kvh, g, qb, 0);
}

// Few queries: blocks of 32, the four waves and the splits (grid y) divide the keys.
constexpr int kKsWaves = 4;
template <int DH, int CAP, bool BIAS>
__global__ __launch_bounds__(64 * kKsWaves) void attn_scored_few_kernel(AttnScoredArgs a) {
  constexpr int NW = kKsWaves;
  __shared__ __attribute__((aligned(16))) char smem[lds_bytes<DH, NW, true>()];
  const int G = a.pack ? 1 : a.H / a.Hkv;
  const int qb = blockIdx.x % a.n_blocks, r = blockIdx.x / a.n_blocks;
  const int g = r % G, pair = r / G;
  const int b = pair / a.Hkv, kvh = pair - b * a.Hkv;
  scored_item<DH, NW, true, CAP, BIAS>(a, smem, b, kvh, g, qb, blockIdx.y);
}

// Joins the splits of a block: workgroup = block, the rows' sums scaled to the
// largest offset and added in split order.  T: the output's type; NAT: the
// offsets are natural logarithms (the fp32-product kernel's), not log2.
// Grid y: 256 values of the block each.
template <typename T, bool NAT>
__global__ __launch_bounds__(256) void attn_scored_merge_kernel(AttnScoredArgs a, int rows) {
  const int G = a.H / a.Hkv, GB = a.pack > 0 ? 1 : G;
  const int item = blockIdx.x;
  const int qb = item % a.n_blocks, r = item / a.n_blocks;
  const int g = r % GB, pair = r / GB;
  const int b = pair / a.Hkv, kvh = pair - b * a.Hkv;
  const Seq s = load_seq(a, b);
  const int DH = a.Dh;
  const int64_t pf = part_floats(rows, DH);
  const float* part = a.part + static_cast<int64_t>(item) * a.splits * pf;
  const int i = blockIdx.y * 256 + threadIdx.x;
  if (i >= rows * DH) return;
  const int q = i / DH, d = i - q * DH;
  const int gi = a.pack > 0 ? q / a.max_q : 0;
  const int oq = a.pack > 0 ? q - gi * a.max_q : qb * rows + q;
  if (gi >= G || oq >= s.qlen) return;
  // eight splits' loads at a time, the sums rescaled to the larger offset between
  const float* pm = part + static_cast<int64_t>(rows) * DH + q;
  auto ex = [](float y) { return NAT ? expf(y) : __builtin_amdgcn_exp2f(y); };
  float M = -INFINITY, l = 0.f, x = 0.f;
  constexpr int U = 8;
  for (int k0 = 0; k0 < a.splits; k0 += U) {
    float mk[U], lk[U], xk[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t o = min(k0 + u, a.splits - 1) * pf;
      mk[u] = pm[o], lk[u] = pm[o + rows], xk[u] = part[o + i];
    }
    float Mn = M;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u < a.splits) Mn = fmaxf(Mn, mk[u]);
    const float f0 = M == -INFINITY ? 1.f : ex(M - Mn);
    l *= f0, x *= f0, M = Mn;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u < a.splits) {
        const float f = mk[u] == -INFINITY ? 1.f : ex(mk[u] - M);
        l += lk[u] * f, x += xk[u] * f;
      }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int oh = kvh * G + (a.pack > 0 ? gi : g);
  store_f32(static_cast<T*>(a.o) + (s.q_row + oq) * a.ld_o + static_cast<int64_t>(oh) * DH + d, x * inv);
}

// How a launch is cut: from its sizes alone, for a device of 256 CUs.
struct Plan {
  bool mfma, few, pack;
  int n_blocks, splits, rows;  // rows: queries of a block
  int64_t items;
};
constexpr int kCus = 256;
constexpr int64_t kMaxWgs = (int64_t{1} << 24) - 1;  // a grid dimension holds fewer than 2^32 threads

bool al(const void* p, uintptr_t m) { return (reinterpret_cast<uintptr_t>(p) & m) == 0; }

Plan plan_of(const AttnScoredArgs& a) {
  Plan p{};
  p.mfma = a.dtype == DT_BF16 && (a.Dh == 64 || a.Dh == 128) && a.ld_q % 8 == 0 && a.ld_k % 8 == 0 && a.ld_v % 8 == 0 &&
           a.ld_o % 4 == 0 && al(a.q, 15) && al(a.k, 15) && al(a.v, 15) && al(a.o, 7);
  p.splits = 1;
  const int G = a.H / a.Hkv;
  const int64_t heads = static_cast<int64_t>(a.B) * a.H;
  // the most tiles that a query block can need (a prefix adds to a window, but
  // its length is not known here)
  const int64_t keys = a.window ? std::min<int64_t>(a.max_k, 2 * int64_t{a.window} + 64) : a.max_k;
  const int64_t tiles = (keys + kTile - 1) / kTile;
  if (!p.mfma) {
    p.rows = 64;
    p.n_blocks = (a.max_q + 63) / 64;
    p.items = heads * p.n_blocks;
    // one tile list per workgroup: splits fill the CUs, at least two tiles each
    p.splits = static_cast<int>(std::clamp<int64_t>(kCus / std::max<int64_t>(1, p.items), 1, std::max<int64_t>(1, tiles / 2)));
    return p;
  }
  // Blocks of 128 queries, or of 32 whose keys the waves and splits divide.  A CU
  // takes one of the latter at a time, 5.5 us + 0.4 us a tile (head_dim 64, cap), and
  // 64 CUs of them are the work of 64 blocks of 128; those run side by side, 4 us +
  // 1.6 us a tile while there are no more than CUs.  Measured (12 heads, 512-key
  // sequences of 512 queries; 8, 16, 20 blocks of 128 a head): 18.6, 27.7, 34.9 us in
  // 32s, 16.4, 16.9, 18.2 in 128s; (8192 keys; 8 and 16 blocks) 112, 168 in 32s, 201,
  // 206 in 128s.  Where a block of 32 holds the queries of all heads of a key head,
  // keys are read once for them: 64 single tokens of 32 heads on 8 key heads over
  // 2048 keys 60.9 us, 186 in 128s.
  p.pack = G > 1 && static_cast<int64_t>(a.max_q) * G <= 32;
  const int64_t full = heads * ((a.max_q + 127) / 128), rounds = (full + kCus / 4 - 1) / (kCus / 4);
  if (!p.pack && rounds > 1 && rounds * (14 + tiles) >= 10 + 4 * tiles) {
    p.rows = 128;
    p.n_blocks = (a.max_q + 127) / 128;
    p.items = full;
    return p;
  }
  p.few = true;
  p.rows = 32;
  p.n_blocks = p.pack ? 1 : (a.max_q + 31) / 32;
  p.items = (p.pack ? static_cast<int64_t>(a.B) * a.Hkv : heads) * p.n_blocks;
  p.splits = static_cast<int>(std::clamp<int64_t>(kCus / std::max<int64_t>(1, p.items), 1, std::max<int64_t>(1, tiles / kKsWaves)));
  return p;
}

template <int DH, int CAP, bool BIAS>
void launch_mfma(const AttnScoredArgs& a, const Plan& p, hipStream_t st) {
  if (p.few) {
    attn_scored_few_kernel<DH, CAP, BIAS>
        <<<dim3(static_cast<unsigned>(p.items), static_cast<unsigned>(p.splits)), 64 * kKsWaves, 0, st>>>(a);
    return;
  }
  const int64_t pairs = static_cast<int64_t>(a.B) * a.Hkv, pairs8 = (pairs + 7) / 8 * 8;
  AttnScoredArgs b = a;
  int64_t wgs = p.items;
  // Pairs of sequence and key head to an XCD each where that fills 7/8 of them (8192
  // keys, not causal; 3 pairs of 4 heads: 762 us so, 337 in plain order; 10 of one: 428,
  // 319; 12: 438, 332; 192 pairs, 512 keys: 30.2, 32.9)
  if (8 * pairs >= 7 * pairs8)
    wgs = pairs8 * (a.H / a.Hkv) * p.n_blocks;
  else
    b.pack = -1;
  if (wgs > kMaxWgs) fail_arg("attn_scored: too many sequences, heads and query blocks for one launch");
  attn_scored_kernel<DH, CAP, BIAS><<<static_cast<unsigned>(wgs), 256, 0, st>>>(b);
}

template <int DH>
void launch_dh(const AttnScoredArgs& a, const Plan& p, hipStream_t st) {
  if (!(a.softcap > 0.f))
    a.slopes ? launch_mfma<DH, CAP_NONE, true>(a, p, st) : launch_mfma<DH, CAP_NONE, false>(a, p, st);
  else if (!a.slopes && a.softcap * kLog2e <= kFixedCap)
    launch_mfma<DH, CAP_FIXED, false>(a, p, st);
  else
    launch_mfma<DH, CAP_ANY, true>(a, p, st);  // (no slopes: a bias of 0)
}

}  // namespace

int64_t attn_scored_part_bytes(const AttnScoredArgs& a) {
  const Plan p = plan_of(a);
  return p.splits > 1 ? 4 * p.items * p.splits * part_floats(p.rows, a.Dh) : 0;
}

void launch_attn_scored(const AttnScoredArgs& a0, hipStream_t st) {
  AttnScoredArgs a = a0;
  const Plan p = plan_of(a);
  if (p.items > kMaxWgs) fail_arg("attn_scored: too many sequences, heads and query blocks for one launch");
  a.n_blocks = p.n_blocks;
  a.splits = p.splits;
  a.pack = p.pack;
  if (!p.mfma)
    launch_attn_scored_f32(a, st);
  else if (a.Dh == 64)
    launch_dh<64>(a, p, st);
  else
    launch_dh<128>(a, p, st);
  check_launch("attn_scored");
  if (p.splits > 1) {
    const dim3 n(static_cast<unsigned>(p.items), static_cast<unsigned>((p.rows * a.Dh + 255) / 256));
    if (p.mfma)
      attn_scored_merge_kernel<bf16_t, false><<<n, 256, 0, st>>>(a, p.rows);
    else if (a.dtype == DT_BF16)
      attn_scored_merge_kernel<bf16_t, true><<<n, 256, 0, st>>>(a, p.rows);
    else
      attn_scored_merge_kernel<float, true><<<n, 256, 0, st>>>(a, p.rows);
    check_launch("attn_scored_merge");
  }
}

}  // namespace sjh
