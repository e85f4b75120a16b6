// attn_window_abi.hip -- extern "C" entry points of the window attention (include/metalllm_attn.h).
// Validation happens on the host before any HIP call.
#include <cmath>

#include "../../include/metalllm_attn.h"
#include "attn_window.hpp"
#include "overlap.hpp"

namespace {

constexpr uint32_t kMostRows = 1u << 24;       // positions and row counts stay far inside 32 bits
constexpr uint32_t kMostRowStride = 1u << 22;  // a tile's byte offsets are 24-bit products

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Strides of a [B, T, heads, D] tensor: rows and sequences apart from each other, in either order.
bool strides_ok(const metalllmWindowParams& p, uint64_t T, uint64_t heads, uint64_t row, uint64_t seq) {
  const uint64_t w = heads * p.D;
  if (row % 8 || seq % 8 || row < w || row >= kMostRowStride || seq >= (1ull << 48)) return false;
  if (p.B == 1) return true;
  return seq >= (T - 1) * row + w || (seq >= w && row >= (p.B - 1) * seq + w);
}

mla::WinShape shape_of(const metalllmWindowParams& p, const int32_t* q_len, const int32_t* k_len) {
  mla::WinShape s;
  s.B = (int)p.B, s.TQ = (int)p.TQ, s.TK = (int)p.TK, s.NH = (int)p.NH, s.NKV = (int)p.NKV, s.G = (int)(p.NH / p.NKV);
  s.window = (int)(p.window < (1u << 30) ? p.window : 1u << 30);
  s.sinks = (int)p.sinks;
  s.q_row = (uint32_t)p.q_row, s.k_row = (uint32_t)p.k_row, s.v_row = (uint32_t)p.v_row, s.o_row = (uint32_t)p.o_row;
  s.q_seq = p.q_seq, s.k_seq = p.k_seq, s.v_seq = p.v_seq, s.o_seq = p.o_seq;
  s.q_len = q_len, s.k_len = k_len;
  s.scale = 1.0f / std::sqrt((float)p.D);
  return s;
}

int validate(const metalllmWindowParams* p) {
  if (!p) return METALLLM_ATTN_E_NULL;
  if (p->D != 64 && p->D != 128) return METALLLM_ATTN_E_HEADDIM;
  if (p->TQ == 0 || p->TK == 0) return METALLLM_ATTN_E_LAYOUT;
  if (p->B == 0 || p->NH == 0 || p->NKV == 0 || p->NH % p->NKV) return METALLLM_ATTN_E_LAYOUT;
  if (p->window == 0 || p->sinks > mla::kWinMaxSinks) return METALLLM_ATTN_E_WINDOW;
  if (p->TQ > kMostRows || p->TK > kMostRows) return METALLLM_ATTN_E_SIZE;
  if ((uint64_t)p->B * p->NH > (1u << 24) || !mla::win_grids_fit(shape_of(*p, nullptr, nullptr), (int)p->D))
    return METALLLM_ATTN_E_SIZE;
  if (!strides_ok(*p, p->TQ, p->NH, p->q_row, p->q_seq) || !strides_ok(*p, p->TK, p->NKV, p->k_row, p->k_seq) ||
      !strides_ok(*p, p->TK, p->NKV, p->v_row, p->v_seq) || !strides_ok(*p, p->TQ, p->NH, p->o_row, p->o_seq))
    return METALLLM_ATTN_E_LAYOUT;
  return METALLLM_ATTN_OK;
}

// the memory from a tensor's first element to its last
mla::Span span(const metalllmWindowParams& p, const void* t, uint64_t T, uint64_t heads, uint64_t row, uint64_t seq) {
  return {t, 2 * ((p.B - 1) * seq + (T - 1) * row + heads * p.D)};
}
mla::Span q_span(const metalllmWindowParams& p, const void* t) { return span(p, t, p.TQ, p.NH, p.q_row, p.q_seq); }
mla::Span o_span(const metalllmWindowParams& p, const void* t) { return span(p, t, p.TQ, p.NH, p.o_row, p.o_seq); }
mla::Span k_span(const metalllmWindowParams& p, const void* t) { return span(p, t, p.TK, p.NKV, p.k_row, p.k_seq); }
mla::Span v_span(const metalllmWindowParams& p, const void* t) { return span(p, t, p.TK, p.NKV, p.v_row, p.v_seq); }
mla::Span l_span(const metalllmWindowParams& p, const void* t) { return {t, t ? 4 * (size_t)p.B * p.NH * p.TQ : 0}; }
mla::Span len_span(const metalllmWindowParams& p, const void* t) { return {t, t ? 4 * (size_t)p.B : 0}; }

uint64_t forward_bytes(const mla::WinShape& s, int D) {
  return mla::win_is_token(s, D) ? 4 * (uint64_t)mla::win_token_floats(s, D, mla::win_token_splits(s)) : 0;
}
// l log2(e) and the row sums of dO * O, each rounded up to whole 16 bytes, then the sink keys' parts
uint64_t stat_floats(const mla::WinShape& s) { return (2 * (uint64_t)s.B * s.NH * s.TQ + 3) / 4 * 4; }
uint64_t backward_bytes(const mla::WinShape& s, int D) {
  return 4 * (stat_floats(s) + mla::win_sink_floats(s, D, mla::win_sink_splits(s)));
}

}  // namespace

extern "C" {

int metalllmWindowForwardWorkspaceSize(const metalllmWindowParams* p, uint64_t* bytes) {
  const int rc = validate(p);
  if (rc) return rc;
  if (!bytes) return METALLLM_ATTN_E_NULL;
  *bytes = forward_bytes(shape_of(*p, nullptr, nullptr), (int)p->D);
  return METALLLM_ATTN_OK;
}

int metalllmWindowBackwardWorkspaceSize(const metalllmWindowParams* p, uint64_t* bytes) {
  const int rc = validate(p);
  if (rc) return rc;
  if (!bytes) return METALLLM_ATTN_E_NULL;
  *bytes = backward_bytes(shape_of(*p, nullptr, nullptr), (int)p->D);
  return METALLLM_ATTN_OK;
}

int windowAttentionForward(const uint16_t* q, const uint16_t* k, const uint16_t* v, uint16_t* out, float* l,
                           const int32_t* q_len, const int32_t* k_len, void* workspace, uint64_t workspace_bytes,
                           const metalllmWindowParams* p, metalllm_stream_t stream) {
  const int rc = validate(p);
  if (rc) return rc;
  if (!q || !k || !v || !out) return METALLLM_ATTN_E_NULL;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(l, 16) || !aligned(q_len, 4) ||
      !aligned(k_len, 4))
    return METALLLM_ATTN_E_ALIGN;
  mla::WinFwdArgs a{q, k, v, out, l, shape_of(*p, q_len, k_len), nullptr, 1};
  const int D = (int)p->D;
  const uint64_t need = forward_bytes(a.s, D);
  if (need) {
    if (!workspace) return METALLLM_ATTN_E_NULL;
    if (!aligned(workspace, 16)) return METALLLM_ATTN_E_ALIGN;
    if (workspace_bytes < need) return METALLLM_ATTN_E_SIZE;
  }
  const mla::Span o = o_span(*p, out), ls = l_span(*p, l), ws{need ? workspace : nullptr, (size_t)need};
  if (mla::any_overlap({o, ls, ws}, {q_span(*p, q), k_span(*p, k), v_span(*p, v), len_span(*p, q_len), len_span(*p, k_len)}) ||
      mla::any_overlap({o, ls, ws}))
    return METALLLM_ATTN_E_OVERLAP;
  hipError_t e;
  if (mla::win_is_token(a.s, D)) {
    a.splits = mla::win_token_splits(a.s);
    a.part = (float*)workspace;
    e = mla::launch_window_token(a, D, (hipStream_t)stream);
  } else {
    e = mla::launch_window_forward(a, D, (hipStream_t)stream);
  }
  return e == hipSuccess ? METALLLM_ATTN_OK : METALLLM_ATTN_E_LAUNCH;
}

int windowAttentionBackward(const uint16_t* dO, const uint16_t* O, const float* l, const uint16_t* q, const uint16_t* k,
                            const uint16_t* v, uint16_t* dQ, uint16_t* dK, uint16_t* dV, const int32_t* q_len,
                            const int32_t* k_len, void* workspace, uint64_t workspace_bytes,
                            const metalllmWindowParams* p, metalllm_stream_t stream) {
  const int rc = validate(p);
  if (rc) return rc;
  if (!dO || !O || !l || !q || !k || !v || !dQ || !dK || !dV || !workspace) return METALLLM_ATTN_E_NULL;
  for (const void* t : {(const void*)dO, (const void*)O, (const void*)l, (const void*)q, (const void*)k, (const void*)v,
                        (const void*)dQ, (const void*)dK, (const void*)dV, (const void*)workspace})
    if (!aligned(t, 16)) return METALLLM_ATTN_E_ALIGN;
  if (!aligned(q_len, 4) || !aligned(k_len, 4)) return METALLLM_ATTN_E_ALIGN;
  mla::WinBwdArgs a{dO, O, l, q, k, v, dQ, dK, dV, shape_of(*p, q_len, k_len), (float*)workspace, nullptr, 0, false};
  const int D = (int)p->D;
  a.narrow = mla::win_is_narrow(a.s);
  if (workspace_bytes < backward_bytes(a.s, D)) return METALLLM_ATTN_E_SIZE;
  // dQ, dK and dV may be interleaved with each other (slices of one buffer), not with anything read
  const mla::Span ws{workspace, (size_t)backward_bytes(a.s, D)};
  const std::initializer_list<mla::Span> in = {o_span(*p, dO), o_span(*p, O), l_span(*p, l), q_span(*p, q), k_span(*p, k),
                                               v_span(*p, v), len_span(*p, q_len), len_span(*p, k_len)};
  const mla::Span dq = q_span(*p, dQ), dk = k_span(*p, dK), dv = v_span(*p, dV);
  if (mla::any_overlap({dq, dk, dv, ws}, in) || mla::any_overlap({ws}, {dq, dk, dv}) || dQ == dK || dK == dV || dQ == dV)
    return METALLLM_ATTN_E_OVERLAP;
  a.splits = mla::win_sink_splits(a.s);
  if (a.splits) a.part = a.Dsum + stat_floats(a.s);
  return mla::launch_window_backward(a, D, (hipStream_t)stream) == hipSuccess ? METALLLM_ATTN_OK : METALLLM_ATTN_E_LAUNCH;
}

}  // extern "C"
