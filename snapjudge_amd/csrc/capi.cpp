// capi.cpp -- extern "C" surface of libsnapjudge_hip.so (include/snapjudge_hip.h).
//
// Exceptions never cross the boundary: each entry point catches, stores the
// message in a thread-local slot readable through sjh_last_error(), and
// returns a negative status, the convention of the reference's engine ABI
// (include/snapjudge/capi.h).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <stdexcept>
#include <string>

#include "ckpt.hpp"
#include "engine.hpp"
#include "sjh_host.hpp"
#include "sjh_kernels.hpp"
#include "snapjudge_hip.h"

struct sjh_model {
  sjh::Engine* eng;
};

namespace {

thread_local std::string g_last_error;

template <typename Fn>
int guarded(Fn&& fn) {
  try {
    fn();
    return SJH_OK;
  } catch (const std::bad_alloc&) {
    g_last_error = "snapjudge HIP: host allocation failed";
    return SJH_E_OOM;
  } catch (const sjh::ArgError& e) {
    g_last_error = e.what();
    return SJH_E_INVALID;
  } catch (const std::runtime_error& e) {
    g_last_error = e.what();
    const std::string s = e.what();
    if (s.find("out of device memory") != std::string::npos) return SJH_E_OOM;
    if (s.find("hip") != std::string::npos || s.find("device") != std::string::npos ||
        s.find("launch") != std::string::npos)
      return SJH_E_DEVICE;
    return SJH_E_INVALID;
  } catch (const std::exception& e) {
    g_last_error = e.what();
    return SJH_E_INVALID;
  }
}

hipStream_t as_stream(sjh_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

size_t esize(int32_t dt) { return dt == SJH_BF16 ? 2 : 4; }

// The stream of a call must be one of the current device, whose memory the
// pointers are taken to be in.
void check_stream(sjh_stream_t s) {
  if (!s) return;
  int cur = 0;
  hipDevice_t dev = 0;
  sjh::hip_check(hipGetDevice(&cur), "hipGetDevice");
  sjh::hip_check(hipStreamGetDevice(as_stream(s), &dev), "hipStreamGetDevice");
  if (dev != cur) sjh::fail_arg("the stream belongs to another device than the current one");
}

// sjh_attn_scored's arguments, checked (but for the pointers) and completed.
sjh::AttnScoredArgs scored_args(const sjh_attn_scored_args* p) {
  using sjh::fail_arg;
  if (!p) fail_arg("attn_scored: null arguments");
  constexpr int32_t kMaxRows = 1 << 29;
  if (p->dtype != SJH_F32 && p->dtype != SJH_BF16) fail_arg("attn_scored: dtype must be SJH_F32 or SJH_BF16");
  if (p->B < 0 || p->H < 1 || p->Hkv < 0) fail_arg("attn_scored: bad batch or heads");
  const int32_t hkv = p->Hkv ? p->Hkv : p->H;
  if (p->H % hkv != 0) fail_arg("attn_scored: Hkv must divide H");
  if (p->Dh != 8 && p->Dh != 16 && p->Dh != 32 && p->Dh != 64 && p->Dh != 128)
    fail_arg("attn_scored: head_dim must be 8, 16, 32, 64 or 128");
  if (p->q_rows < 0 || p->k_rows < 0 || p->q_rows > kMaxRows || p->k_rows > kMaxRows)
    fail_arg("attn_scored: q_rows and k_rows must lie in [0, 2^29]");
  if (p->max_q < 0 || p->max_k < 0) fail_arg("attn_scored: negative length bound");
  if (!(p->scale >= 0.f) || !(p->scale < INFINITY)) fail_arg("attn_scored: scale must be finite and not negative");
  if (!(p->softcap >= 0.f) || !(p->softcap < INFINITY)) fail_arg("attn_scored: softcap must be finite and not negative");
  if (p->window < 0) fail_arg("attn_scored: negative window");
  if (!p->q_doc != !p->k_doc) fail_arg("attn_scored: documents of queries and keys, or of neither");
  if (!p->k_start != !p->k_len) fail_arg("attn_scored: k_start and k_len, or neither");
  sjh::AttnScoredArgs a;
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.o = p->o;
  const int64_t qd = static_cast<int64_t>(p->H) * p->Dh, kd = static_cast<int64_t>(hkv) * p->Dh;
  a.ld_q = p->ld_q ? p->ld_q : qd;
  a.ld_k = p->ld_k ? p->ld_k : kd;
  a.ld_v = p->ld_v ? p->ld_v : kd;
  a.ld_o = p->ld_o ? p->ld_o : qd;
  if (a.ld_q < qd || a.ld_o < qd || a.ld_k < kd || a.ld_v < kd) fail_arg("attn_scored: row stride < heads * Dh");
  // (a tile's rows are addressed by 32-bit byte offsets)
  if (a.ld_k > (1 << 23) || a.ld_v > (1 << 23)) fail_arg("attn_scored: key row stride above 2^23");
  a.q_start = p->q_start;
  a.q_len = p->q_len;
  a.k_start = p->k_start ? p->k_start : p->q_start;
  a.k_len = p->k_len ? p->k_len : p->q_len;
  a.q_pos = p->q_pos;
  a.prefix = p->prefix;
  a.q_doc = p->q_doc;
  a.k_doc = p->k_doc;
  a.slopes = p->slopes;
  a.scale = p->scale > 0.f ? p->scale : 1.0f / std::sqrt(static_cast<float>(p->Dh));
  a.softcap = p->softcap;
  // positions differ by less than 2^30: a wider window hides nothing
  a.window = p->window < (1 << 30) - 2 ? p->window : 0;
  a.causal = p->causal != 0;
  a.B = p->B;
  a.H = p->H;
  a.Hkv = hkv;
  a.Dh = p->Dh;
  a.q_rows = p->q_rows;
  a.k_rows = p->k_rows;
  a.max_q = p->max_q < p->q_rows ? p->max_q : p->q_rows;
  a.max_k = p->max_k < p->k_rows ? p->max_k : p->k_rows;
  a.dtype = p->dtype;
  return a;
}

void check_dtype(int32_t dt) {
  if (dt != SJH_F32 && dt != SJH_BF16) sjh::fail("dtype must be SJH_F32 or SJH_BF16");
}

}  // namespace

extern "C" {

const char* sjh_last_error(void) { return g_last_error.c_str(); }

int sjh_version(void) { return 1; }

void sjh_default_options(sjh_options* opt) {
  if (!opt) return;
  opt->precision = SJH_PREC_BF16;
  opt->max_len = 0;
  opt->use_graphs = 1;
  opt->pad_rows = 0;
  opt->device = 0;
  opt->fuse_ln = 1;
  opt->fuse_attn_wo = 1;
}

int sjh_model_create(const sjh_model_desc* desc, const sjh_options* opt, sjh_model** out) {
  return guarded([&] {
    if (!desc || !out) sjh::fail("sjh_model_create: null argument");
    *out = nullptr;
    sjh_options o;
    sjh_default_options(&o);
    if (opt) o = *opt;
    auto* m = new sjh_model{nullptr};
    try {
      m->eng = new sjh::Engine(sjh::source_from_desc(*desc), o);
    } catch (...) {
      delete m;
      throw;
    }
    *out = m;
  });
}

int sjh_model_load(const char* dir, const sjh_options* opt, sjh_model** out) {
  return guarded([&] {
    if (!dir || !out) sjh::fail_arg("sjh_model_load: null argument");
    *out = nullptr;
    sjh_options o;
    sjh_default_options(&o);
    if (opt) o = *opt;
    // the mapping stays open until every tensor is on the device
    std::unique_ptr<sjh::Checkpoint> ck = sjh::read_checkpoint(dir);
    auto* m = new sjh_model{nullptr};
    try {
      m->eng = new sjh::Engine(ck->src, o);
    } catch (...) {
      delete m;
      throw;
    }
    *out = m;
  });
}

void sjh_model_destroy(sjh_model* m) {
  if (!m) return;
  delete m->eng;
  delete m;
}

int sjh_model_encode(sjh_model* m, const int64_t* ids, const int64_t* mask, int32_t B, int32_t L,
                     float* hidden) {
  return guarded([&] {
    if (!m) sjh::fail("null model");
    if (B < 0) sjh::fail("negative batch");
    m->eng->encode(ids, mask, B, L, hidden);
  });
}

int sjh_model_forward(sjh_model* m, const int64_t* ids, const int64_t* mask,
                      const int64_t* marker_pos, const uint8_t* marker_mask, const int64_t* qtype,
                      int32_t B, int32_t L, int32_t K, float* logits, float* act) {
  return guarded([&] {
    if (!m) sjh::fail("null model");
    if (B < 0) sjh::fail("negative batch");
    m->eng->forward(ids, mask, marker_pos, marker_mask, qtype, B, L, K, logits, act);
  });
}

int sjh_model_forward_shared(sjh_model* m, const int64_t* ids, const int64_t* mask, int32_t U,
                             int32_t L, const int32_t* row_seq, const int64_t* marker_pos,
                             const uint8_t* marker_mask, const int64_t* qtype, int32_t B,
                             int32_t K, float* logits, float* act) {
  return guarded([&] {
    if (!m) sjh::fail("null model");
    if (B < 0 || U < 0) sjh::fail("negative batch");
    m->eng->forward_shared(ids, mask, U, L, row_seq, marker_pos, marker_mask, qtype, B, K, logits,
                           act);
  });
}

int sjh_model_encode_device(sjh_model* m, const int32_t* d_ids, const int32_t* h_lens, int32_t B,
                            float* d_hidden, sjh_stream_t stream) {
  return guarded([&] {
    if (!m) sjh::fail("null model");
    if (B < 0) sjh::fail("negative batch");
    m->eng->encode_device(d_ids, h_lens, B, d_hidden, as_stream(stream));
  });
}

int sjh_model_encode_device_noalloc(sjh_model* m, const int32_t* d_ids, const int32_t* h_lens,
                                    int32_t B, float* d_hidden, sjh_stream_t stream) {
  return guarded([&] {
    if (!m) sjh::fail("null model");
    if (B < 0) sjh::fail("negative batch");
    m->eng->encode_device_noalloc(d_ids, h_lens, B, d_hidden, as_stream(stream));
  });
}

int sjh_model_info(const sjh_model* m, int32_t* D, int32_t* H, int32_t* n_act,
                   int32_t* precision) {
  return guarded([&] {
    if (!m) sjh::fail("null model");
    if (D) *D = m->eng->D();
    if (H) *H = m->eng->H();
    if (n_act) *n_act = m->eng->n_act();
    if (precision) *precision = m->eng->precision();
  });
}

int sjh_model_graph_stats(const sjh_model* m, int32_t* cached, int64_t* captures,
                          int64_t* replays) {
  return guarded([&] {
    if (!m) sjh::fail("null model");
    m->eng->graph_stats(cached, captures, replays);
  });
}

int sjh_model_profile(sjh_model* m, int32_t enable) {
  return guarded([&] {
    if (!m) sjh::fail("null model");
    m->eng->set_profile(enable != 0);
  });
}

int sjh_model_profile_read(sjh_model* m, int32_t max_entries, const char** names,
                           double* total_ms, int64_t* launches, int32_t* n_entries) {
  return guarded([&] {
    if (!m || !n_entries) sjh::fail("null argument");
    auto v = m->eng->profile_totals();
    int n = 0;
    for (auto& t : v) {
      if (n >= max_entries) break;
      if (names) names[n] = std::get<0>(t);
      if (total_ms) total_ms[n] = std::get<1>(t);
      if (launches) launches[n] = std::get<2>(t);
      ++n;
    }
    *n_entries = n;
  });
}

// ---------------------------------------------------------------- kernels --
int sjh_gemm(const void* A, const void* W, const float* bias, void* C, int32_t M, int32_t N,
             int32_t K, int32_t act, int32_t dtype, sjh_stream_t stream) {
  return guarded([&] {
    check_dtype(dtype);
    if (act < 0 || act > 2) sjh::fail("act must be 0, 1 or 2");
    sjh::GemmArgs g;
    g.A = A;
    g.lda = K;
    g.W = W;
    g.ldw = K;
    g.M = M;
    g.N = N;
    g.K = K;
    g.in_dtype = dtype;
    g.epi = sjh::EPI_STORE;
    g.out = C;
    g.ldo = N;
    g.out_dtype = dtype;
    g.bias = bias;
    g.act = act;
    sjh::launch_gemm(g, as_stream(stream));
  });
}

int sjh_quantize_fp8(const float* w, int64_t rows, int64_t cols, uint8_t* q, float* scale) {
  return guarded([&] {
    if (rows < 0 || cols < 0) sjh::fail("quantize_fp8: negative shape");
    if (rows > 0 && cols > 0 && (!w || !q || !scale)) sjh::fail("quantize_fp8: null argument");
    sjh::quantize_fp8_rows(w, static_cast<size_t>(rows), static_cast<size_t>(cols), q, scale);
  });
}

int sjh_gemm_fp8w(const void* A, const uint8_t* Wq, const float* w_scale, const float* bias,
                  void* C, int32_t M, int32_t N, int32_t K, int32_t act, sjh_stream_t stream) {
  return guarded([&] {
    if (act < 0 || act > 2) sjh::fail("act must be 0, 1 or 2");
    sjh::GemmArgs g;
    g.A = A;
    g.lda = K;
    g.W = Wq;
    g.ldw = K;
    g.M = M;
    g.N = N;
    g.K = K;
    g.in_dtype = SJH_BF16;
    g.w_dtype = sjh::DT_FP8;
    g.w_scale = w_scale;
    g.epi = sjh::EPI_STORE;
    g.out = C;
    g.ldo = N;
    g.out_dtype = SJH_BF16;
    g.bias = bias;
    g.act = act;
    sjh::launch_gemm(g, as_stream(stream));
  });
}

int64_t sjh_gemm_lora_workspace(int32_t M, int32_t R) {
  if (M < 0 || R < 1 || R > sjh::kLoraMaxRank) {
    g_last_error = "snapjudge HIP: gemm_lora: M must not be negative and R must lie in [1, 256]";
    return SJH_E_INVALID;
  }
  return sjh::lora_ws_bytes(M, R);
}

int sjh_gemm_lora(const sjh_lora_args* p, sjh_stream_t stream) {
  return guarded([&] {
    using sjh::fail_arg;
    if (!p) fail_arg("gemm_lora: null arguments");
    if (p->dtype != SJH_F32 && p->dtype != SJH_BF16) fail_arg("gemm_lora: dtype must be SJH_F32 or SJH_BF16");
    if (p->act < 0 || p->act > 2) fail_arg("gemm_lora: act must be 0, 1 or 2");
    if (p->M < 0 || p->N < 0 || p->K < 1) fail_arg("gemm_lora: bad shape");
    if (p->n_adapters < 0) fail_arg("gemm_lora: negative n_adapters");
    if (p->n_adapters > 0 && (p->R < 1 || p->R > sjh::kLoraMaxRank)) fail_arg("gemm_lora: R must lie in [1, 256]");
    if (p->w_scale && p->dtype != SJH_BF16) fail_arg("gemm_lora: fp8 weights need SJH_BF16 rows");
    const int64_t ldx = p->ld_x ? p->ld_x : p->K, ldo = p->ld_out ? p->ld_out : p->N;
    if (ldx < p->K || ldo < p->N) fail_arg("gemm_lora: row stride < its row");
    if (ldo > (1 << 23)) fail_arg("gemm_lora: output row stride above 2^23");  // (32-bit offsets within a tile)
    if (p->M == 0 || p->N == 0) return;
    if (!p->x || !p->w || !p->out) fail_arg("gemm_lora: null operand");
    sjh::LoraArgs l;
    sjh::GemmArgs& g = l.g;
    g.A = p->x;
    g.lda = ldx;
    g.W = p->w;
    g.ldw = p->K;
    g.M = p->M;
    g.N = p->N;
    g.K = p->K;
    g.in_dtype = p->dtype;
    g.w_dtype = p->w_scale ? sjh::DT_FP8 : p->dtype == SJH_BF16 ? sjh::DT_BF16 : sjh::DT_F32;
    g.w_scale = p->w_scale;
    g.out = p->out;
    g.ldo = ldo;
    g.out_dtype = p->dtype;
    g.bias = p->bias;
    g.act = p->act;
    if (p->n_adapters == 0) {
      check_stream(stream);
      g.epi = sjh::EPI_STORE;
      sjh::launch_gemm(g, as_stream(stream));
      return;
    }
    if (!p->a || !p->b) fail_arg("gemm_lora: null adapters");
    if (!p->workspace || p->workspace_bytes < sjh::lora_ws_bytes(p->M, p->R)) fail_arg("gemm_lora: workspace too small");
    if (reinterpret_cast<uintptr_t>(p->workspace) & 15u) fail_arg("gemm_lora: workspace must be 16-byte aligned");
    g.lora_b = p->b;
    g.lora_adapter = p->adapter;
    g.lora_n = p->n_adapters;
    g.lora_r = p->R;
    l.a = p->a;
    l.scale = p->scale;
    l.ws = p->workspace;
    check_stream(stream);
    sjh::launch_gemm_lora(l, as_stream(stream));
  });
}

int sjh_gemm_geglu(const void* A, const void* Wi, void* C, int32_t M, int32_t F, int32_t K,
                   int32_t dtype, sjh_stream_t stream) {
  return guarded([&] {
    check_dtype(dtype);
    sjh::GemmArgs g;
    g.A = A;
    g.lda = K;
    g.W = Wi;
    g.ldw = K;
    g.M = M;
    g.N = F;
    g.K = K;
    g.in_dtype = dtype;
    g.epi = sjh::EPI_GEGLU;
    g.out = C;
    g.ldo = F;
    g.out_dtype = dtype;
    sjh::launch_gemm(g, as_stream(stream));
  });
}

int sjh_gemm_residual(const void* A, const void* W, float* X, int32_t M, int32_t D, int32_t K,
                      int32_t dtype, sjh_stream_t stream) {
  return guarded([&] {
    check_dtype(dtype);
    sjh::GemmArgs g;
    g.A = A;
    g.lda = K;
    g.W = W;
    g.ldw = K;
    g.M = M;
    g.N = D;
    g.K = K;
    g.in_dtype = dtype;
    g.epi = sjh::EPI_RESID;
    g.X = X;
    g.ldx = D;
    sjh::launch_gemm(g, as_stream(stream));
  });
}

int sjh_gemm_qkv_rope(const void* A, const void* Wqkv, void* qkv, const int32_t* pos,
                      const float* cos_t, const float* sin_t, int32_t max_pos, int32_t M,
                      int32_t H, int32_t Dh, int32_t K, int32_t dtype, sjh_stream_t stream) {
  return guarded([&] {
    check_dtype(dtype);
    if (H <= 0 || Dh <= 0 || Dh % 2 != 0) sjh::fail("gemm_qkv_rope: bad head shape");
    if (!pos || !cos_t || !sin_t) sjh::fail("gemm_qkv_rope: null positions or tables");
    if (max_pos <= 0) sjh::fail("gemm_qkv_rope: max_pos must be positive");
    sjh::GemmArgs g;
    g.A = A;
    g.lda = K;
    g.W = Wqkv;
    g.ldw = K;
    g.M = M;
    g.N = 3 * H * Dh;
    g.K = K;
    g.in_dtype = dtype;
    g.epi = sjh::EPI_ROPE;
    g.out = qkv;
    g.ldo = 3 * H * Dh;
    g.out_dtype = dtype;
    g.pos = pos;
    g.rope_cos = cos_t;
    g.rope_sin = sin_t;
    g.rope_rows = max_pos;
    g.rope_dim = H * Dh;
    g.head_dim = Dh;
    sjh::launch_gemm(g, as_stream(stream));
  });
}

int sjh_add_ln(float* X, const void* R, const float* W, const float* B, void* Y, int32_t M,
               int32_t D, float eps, int32_t residual, int32_t bias, int32_t dtype,
               sjh_stream_t stream) {
  return guarded([&] {
    check_dtype(dtype);
    sjh::LnArgs a;
    a.in = X;
    a.in_dtype = sjh::DT_F32;
    a.ld_in = D;
    if (residual) {
      if (!R) sjh::fail("add_ln: residual requested without R");
      a.resid = R;
      a.resid_dtype = dtype;
      a.xio = X;
    }
    a.w = W;
    a.b = bias ? B : nullptr;
    a.eps = eps;
    a.y_out = Y;
    a.y_dtype = dtype;
    a.ld_y = D;
    a.M = M;
    a.D = D;
    sjh::launch_ln(a, as_stream(stream));
  });
}

int sjh_add_norm(const sjh_add_norm_args* p, sjh_stream_t stream) {
  return guarded([&] {
    if (!p) sjh::fail_arg("add_norm: null arguments");
    sjh::AddNormArgs a;
    a.x = p->x;
    a.r = p->r;
    a.x_out = p->x_out;
    a.y = p->y;
    a.post_w = p->post_w;
    a.post_b = p->post_b;
    a.pre_w = p->pre_w;
    a.pre_b = p->pre_b;
    a.gate = p->gate;
    a.gate_row = p->gate_row;
    a.ld_x = p->ld_x ? p->ld_x : p->D;
    a.ld_r = p->ld_r ? p->ld_r : p->D;
    a.ld_xo = p->ld_xo ? p->ld_xo : p->D;
    a.ld_y = p->ld_y ? p->ld_y : p->D;
    a.x_scale = p->x_scale;
    a.r_scale = p->r_scale;
    a.eps = p->eps;
    a.post_norm = p->post_norm;
    a.pre_norm = p->pre_norm;
    a.n_gates = p->n_gates;
    a.M = p->M;
    a.D = p->D;
    a.dtype = p->dtype;
    if (a.M > 0) check_stream(stream);
    sjh::launch_add_norm(a, as_stream(stream));
  });
}

int sjh_rope(void* qkv, const float* cos_t, const float* sin_t, int64_t M, int32_t L, int32_t H,
             int32_t Dh, int32_t dtype, sjh_stream_t stream) {
  return guarded([&] {
    check_dtype(dtype);
    if (L <= 0) sjh::fail("rope: L must be positive");
    sjh::launch_rope(qkv, dtype, M, static_cast<int64_t>(3) * H * Dh, nullptr, L, H, Dh, cos_t,
                     sin_t, as_stream(stream));
  });
}

int sjh_attn(const void* qkv, const int32_t* lens, void* O, int32_t B, int32_t L, int32_t H,
             int32_t Dh, int32_t window, int32_t dtype, sjh_stream_t stream) {
  return guarded([&] {
    check_dtype(dtype);
    if (L <= 0 || H <= 0 || Dh <= 0) sjh::fail("attn: bad shape");
    const size_t es = esize(dtype);
    const int64_t HD = static_cast<int64_t>(H) * Dh;
    sjh::AttnArgs a;
    a.q = qkv;
    a.k = static_cast<const char*>(qkv) + HD * es;
    a.v = static_cast<const char*>(qkv) + 2 * HD * es;
    a.ld_q = a.ld_k = a.ld_v = 3 * HD;
    a.o = O;
    a.ld_o = HD;
    a.dtype = dtype;
    a.k_len = lens;
    a.uniform_L = L;
    a.B = B;
    a.H = H;
    a.Dh = Dh;
    a.max_q = L;
    a.window = window;
    a.scale = 1.0f / std::sqrt(static_cast<float>(Dh));
    sjh::launch_attn(a, as_stream(stream));
  });
}

int sjh_attn_log2(const void* qkv, const int32_t* lens, void* O, int32_t B, int32_t L, int32_t H,
                  int32_t window, sjh_stream_t stream) {
  return guarded([&] {
    if (L <= 0 || H <= 0) sjh::fail("attn_log2: bad shape");
    const int64_t HD = static_cast<int64_t>(H) * 64;
    sjh::AttnArgs a;
    a.q = qkv;
    a.k = static_cast<const char*>(qkv) + HD * 2;
    a.v = static_cast<const char*>(qkv) + 2 * HD * 2;
    a.ld_q = a.ld_k = a.ld_v = 3 * HD;
    a.o = O;
    a.ld_o = HD;
    a.dtype = sjh::DT_BF16;
    a.k_len = lens;
    a.uniform_L = L;
    a.B = B;
    a.H = H;
    a.Dh = 64;
    a.max_q = L;
    a.window = window;
    a.scale = 0.125f;
    a.q_log2_scaled = true;
    sjh::launch_attn(a, as_stream(stream));
  });
}

int64_t sjh_attn_scored_workspace(const sjh_attn_scored_args* p) {
  int64_t n = 0;
  const int rc = guarded([&] {
    const sjh::AttnScoredArgs a = scored_args(p);
    if (a.B > 0 && a.max_q > 0) n = sjh::attn_scored_part_bytes(a);
  });
  return rc == SJH_OK ? n : rc;
}

int sjh_attn_scored(const sjh_attn_scored_args* p, sjh_stream_t stream) {
  return guarded([&] {
    sjh::AttnScoredArgs a = scored_args(p);
    if (a.B == 0 || a.max_q == 0) return;
    if (!a.q || !a.o || !a.q_start || !a.q_len || (a.max_k > 0 && (!a.k || !a.v)))
      sjh::fail_arg("attn_scored: null pointer");
    const int64_t need = sjh::attn_scored_part_bytes(a);
    if (need > 0) {
      if (!p->workspace || p->workspace_bytes < need) sjh::fail_arg("attn_scored: workspace too small");
      if (reinterpret_cast<uintptr_t>(p->workspace) & 15u) sjh::fail_arg("attn_scored: workspace must be 16-byte aligned");
      a.part = static_cast<float*>(p->workspace);
    }
    check_stream(stream);
    sjh::launch_attn_scored(a, as_stream(stream));
  });
}

int sjh_embed_ln(const void* table, const int32_t* ids, const float* w, float* X, int32_t M,
                 int32_t D, float eps, int32_t dtype, sjh_stream_t stream) {
  return guarded([&] {
    check_dtype(dtype);
    sjh::LnArgs a;
    a.in = table;
    a.in_dtype = dtype;
    a.ld_in = D;
    a.ids = ids;
    a.w = w;
    a.eps = eps;
    a.x_out = X;
    a.ld_x = D;
    a.M = M;
    a.D = D;
    sjh::launch_ln(a, as_stream(stream));
  });
}

}  // extern "C"
