// rotary.hip -- rotary positions of q and k (include/metalllm_attn.h), HBM-bound.
//
// Pair i of a token at position pos turns by pos * f_i. The plan holds f_i / 2pi in 64 bits: the angle in
// turns is pos * f_i, reduced to [-1/2, 1/2] in 64 bits (at position 10^6 a 32-bit product would be off by
// 2^-5 of a turn for the fastest pair) and only then rounded to 32, where v_sin_f32 and v_cos_f32 take
// turns. A thread owns 8 pairs of a token: it computes their sines once, then turns them in kHeads heads,
// q and k in one launch.
// Measured: B = 8, T = 2048, 12 + 12 heads of 64 with 48 turned: 25 us, 4.0 TB/s of 101 MB read and written; B = 16, T
// = 4096, 16 + 16 heads of 128: 191 us, 5.6 TB/s. A batch of 32 tokens: 4.5 us, a launch and two dependent reads.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "../../include/metalllm_attn.h"
#include "overlap.hpp"

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct RotArgs {
  const uint16_t* q;
  const uint16_t* k;
  uint16_t* qo;
  uint16_t* ko;
  const int32_t* pos;
  metalllmRotaryParams p;
  metalllmRotaryPlan plan;
};

__device__ __forceinline__ uint32_t pk(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, b2));
}
__device__ __forceinline__ float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

constexpr int kHeads = 4;  // heads per thread: the sines of 8 pairs cost about as much as turning two heads

struct Place {  // what a thread turns: unit c of heads h0 .. h1 - 1 of a token
  uint32_t c, token, t, h0, h1;
  const uint16_t *q, *k;
  uint16_t *qo, *ko;
  __device__ __forceinline__ Place(const RotArgs& a, uint32_t id, uint32_t units, uint32_t parts) {
    const uint32_t rest = id / units;
    c = id - rest * units;
    token = rest / parts;
    h0 = (rest - token * parts) * kHeads;
    h1 = min(h0 + kHeads, a.p.NH + a.p.NKV);
    const uint32_t b = token / a.p.T;
    t = token - b * a.p.T;
    q = a.q + b * a.p.q_seq + t * a.p.q_row;
    k = a.k + b * a.p.k_seq + t * a.p.k_row;
    qo = a.qo + b * a.p.qo_seq + t * a.p.qo_row;
    ko = a.ko + b * a.p.ko_seq + t * a.p.ko_row;
  }
  __device__ __forceinline__ const uint16_t* in(const RotArgs& a, uint32_t h) const {
    return h < a.p.NH ? q + h * a.p.D : k + (h - a.p.NH) * a.p.D;
  }
  __device__ __forceinline__ uint16_t* out(const RotArgs& a, uint32_t h) const {
    return h < a.p.NH ? qo + h * a.p.D : ko + (h - a.p.NH) * a.p.D;
  }
};
// sine and cosine of pair i at a position, times the magnitude
__device__ __forceinline__ void turn_of(const RotArgs& a, double pos, uint32_t i, int back, float& cs, float& sn) {
  double turn = pos * a.plan.turns[i];
  turn -= rint(turn);
  const float f = (float)turn;
  cs = __builtin_amdgcn_cosf(f) * a.plan.magnitude;
  sn = __builtin_amdgcn_sinf(f) * a.plan.magnitude;
  if (back) sn = -sn;
}

// R a multiple of 16: a unit is 8 pairs, two 16-byte chunks of the head in either order; units R/16 .. of a head
// (the part that does not turn) are copied, 16 values each.
__global__ void __launch_bounds__(256) rotary_kernel(RotArgs a, int back, uint32_t units, uint32_t parts, uint32_t work) {
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  if (id >= work) return;
  const Place w(a, id, units, parts);
  const uint32_t R = a.plan.dims, half = R / 2, turning = R / 16;
  const bool copied = w.c >= turning;
  const bool inter = a.plan.interleaved != 0;
  // the chunks: values 16c .. 16c + 15 (neighbours paired, or copied) or 8c .. and half + 8c ..; every load is in
  // flight while the sines are computed
  const uint32_t d0 = copied || inter ? 16 * w.c : 8 * w.c;
  const uint32_t d1 = copied || inter ? d0 + 8 : half + d0;
  const bool two = d1 < a.p.D;
  u4 x0[kHeads], x1[kHeads];
#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    const uint16_t* x = w.in(a, min(w.h0 + n, w.h1 - 1));
    x0[n] = *(const u4*)(x + d0);
    x1[n] = two ? *(const u4*)(x + d1) : u4{0, 0, 0, 0};
  }
  const double pos = a.pos ? (double)a.pos[w.token] : (double)w.t;
  float cs[8], sn[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) turn_of(a, pos, min(8 * w.c + u, half - 1), back, cs[u], sn[u]);
#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    const uint32_t h = w.h0 + n;
    if (h >= w.h1) continue;
    u4 y0, y1;
    if (inter) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float e0 = lo_f(x0[n][v]), o0 = hi_f(x0[n][v]), e1 = lo_f(x1[n][v]), o1 = hi_f(x1[n][v]);
        y0[v] = pk(e0 * cs[v] - o0 * sn[v], e0 * sn[v] + o0 * cs[v]);
        y1[v] = pk(e1 * cs[4 + v] - o1 * sn[4 + v], e1 * sn[4 + v] + o1 * cs[4 + v]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float a0 = lo_f(x0[n][v]), a1 = hi_f(x0[n][v]), b0 = lo_f(x1[n][v]), b1 = hi_f(x1[n][v]);
        y0[v] = pk(a0 * cs[2 * v] - b0 * sn[2 * v], a1 * cs[2 * v + 1] - b1 * sn[2 * v + 1]);
        y1[v] = pk(a0 * sn[2 * v] + b0 * cs[2 * v], a1 * sn[2 * v + 1] + b1 * cs[2 * v + 1]);
      }
    }
    uint16_t* y = w.out(a, h);
    *(u4*)(y + d0) = copied ? x0[n] : y0;
    if (two) *(u4*)(y + d1) = copied ? x1[n] : y1;
  }
}

// Any other R: a unit is one pair, or two values of the rest, so that the lanes of a wave read and write
// beside each other. (8 pairs to a thread, value by value, took 206 us where this takes 53: B = 9, T = 5030, 20
// heads of 64 with 62 turned, neighbours; halves 190 and 64.)
template <bool BESIDE>  // the two values of every unit are one 4-byte word
__global__ void __launch_bounds__(256) rotary_pairs_kernel(RotArgs a, int back, uint32_t units, uint32_t parts, uint32_t work) {
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  if (id >= work) return;
  const Place w(a, id, units, parts);
  const uint32_t half = a.plan.dims / 2;
  const bool copied = w.c >= half;
  const uint32_t e = copied || BESIDE ? 2 * w.c : w.c, o = copied ? e + 1 : half + w.c;
  uint32_t x2[kHeads];
#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    const uint16_t* x = w.in(a, min(w.h0 + n, w.h1 - 1));
    x2[n] = BESIDE ? *(const uint32_t*)(x + e) : x[e] | (uint32_t)x[o] << 16;
  }
  float cs, sn;
  turn_of(a, a.pos ? (double)a.pos[w.token] : (double)w.t, min(w.c, half - 1), back, cs, sn);
#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    if (w.h0 + n >= w.h1) continue;
    const float a0 = lo_f(x2[n]), b0 = hi_f(x2[n]);
    const uint32_t y2 = copied ? x2[n] : pk(a0 * cs - b0 * sn, a0 * sn + b0 * cs);
    uint16_t* y = w.out(a, w.h0 + n);
    if (BESIDE) {
      *(uint32_t*)(y + e) = y2;
    } else {
      y[e] = (uint16_t)y2;
      y[o] = (uint16_t)(y2 >> 16);
    }
  }
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

bool strides_ok(const metalllmRotaryParams& p, uint64_t heads, uint64_t row, uint64_t seq) {
  const uint64_t w = heads * p.D;
  if (row % 8 || seq % 8 || row < w || row >= (1ull << 31) || seq >= (1ull << 48)) return false;
  if (p.B == 1) return true;
  return seq >= (p.T - 1) * row + w || (seq >= w && row >= (p.B - 1) * seq + w);
}

mla::Span span(const metalllmRotaryParams& p, const void* t, uint64_t heads, uint64_t row, uint64_t seq) {
  return {t, 2 * ((p.B - 1) * seq + (p.T - 1) * row + heads * p.D)};
}

int rotary(const uint16_t* q, const uint16_t* k, uint16_t* qo, uint16_t* ko, const int32_t* positions,
           const metalllmRotaryPlan* plan, const metalllmRotaryParams* p, hipStream_t stream, int back) {
  if (!p || !plan) return METALLLM_ATTN_E_NULL;
  if (p->D == 0 || p->D % 8 || p->D > 2 * METALLLM_ROTARY_PAIRS) return METALLLM_ATTN_E_HEADDIM;
  if (p->B == 0 || p->T == 0 || p->NH == 0) return METALLLM_ATTN_E_LAYOUT;
  if (plan->dims == 0 || plan->dims % 2 || plan->dims > p->D) return METALLLM_ATTN_E_LAYOUT;
  if (p->B > (1u << 24) || p->T > (1u << 24) || p->NH > (1u << 16) || p->NKV > (1u << 16)) return METALLLM_ATTN_E_SIZE;
  if (!strides_ok(*p, p->NH, p->q_row, p->q_seq) || !strides_ok(*p, p->NH, p->qo_row, p->qo_seq)) return METALLLM_ATTN_E_LAYOUT;
  if (p->NKV && (!strides_ok(*p, p->NKV, p->k_row, p->k_seq) || !strides_ok(*p, p->NKV, p->ko_row, p->ko_seq)))
    return METALLLM_ATTN_E_LAYOUT;
  if (!q || !qo || (p->NKV && (!k || !ko))) return METALLLM_ATTN_E_NULL;
  if (!aligned(q, 16) || !aligned(qo, 16) || !aligned(positions, 4)) return METALLLM_ATTN_E_ALIGN;
  if (p->NKV && (!aligned(k, 16) || !aligned(ko, 16))) return METALLLM_ATTN_E_ALIGN;
  const bool whole = plan->dims % 16 == 0;
  const uint32_t units = whole ? plan->dims / 16 + (p->D - plan->dims + 15) / 16 : p->D / 2;
  const uint32_t parts = (p->NH + p->NKV + kHeads - 1) / kHeads;
  const uint64_t work = (uint64_t)p->B * p->T * parts * units;
  if (work >= (1ull << 32) - 256) return METALLLM_ATTN_E_SIZE;
  const dim3 grid((unsigned)((work + 255) / 256));
  // A tensor is turned in place (a thread reads and writes the same values) or into memory of its own;
  // in place, q and k may be interleaved slices of one buffer.
  const bool q_in = q == qo, k_in = p->NKV && k == ko;
  if ((q_in && (p->q_row != p->qo_row || p->q_seq != p->qo_seq)) ||
      (k_in && (p->k_row != p->ko_row || p->k_seq != p->ko_seq)) || (p->NKV && (qo == ko || qo == k || ko == q)))
    return METALLLM_ATTN_E_OVERLAP;
  const mla::Span sq = span(*p, q, p->NH, p->q_row, p->q_seq), sqo = span(*p, qo, p->NH, p->qo_row, p->qo_seq);
  const mla::Span sk = p->NKV ? span(*p, k, p->NKV, p->k_row, p->k_seq) : mla::Span{nullptr, 0};
  const mla::Span sko = p->NKV ? span(*p, ko, p->NKV, p->ko_row, p->ko_seq) : mla::Span{nullptr, 0};
  const mla::Span sp{positions, positions ? 4 * (size_t)p->B * p->T : 0};
  if ((!q_in && mla::any_overlap({sqo}, {sq, sk})) || (p->NKV && !k_in && mla::any_overlap({sko}, {sk, sq})) ||
      (positions && mla::any_overlap({sp}, {sqo, sko})))
    return METALLLM_ATTN_E_OVERLAP;
  const RotArgs a{q, k, qo, ko, positions, *p, *plan};
  auto* kernel = whole ? rotary_kernel : plan->interleaved ? rotary_pairs_kernel<true> : rotary_pairs_kernel<false>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a, back, units, parts, (uint32_t)work);
  return hipGetLastError() == hipSuccess ? METALLLM_ATTN_OK : METALLLM_ATTN_E_LAUNCH;
}

}  // namespace

extern "C" {

int metalllmRotaryPlanInit(uint32_t dims, double base, int interleaved, const metalllmRotaryScaling* sc,
                           metalllmRotaryPlan* plan) {
  if (!plan) return METALLLM_ATTN_E_NULL;
  if (dims == 0 || dims % 2 || dims > 2 * METALLLM_ROTARY_PAIRS || !(base > 0.0) || !std::isfinite(base))
    return METALLLM_ATTN_E_LAYOUT;
  const int kind = sc ? sc->kind : METALLLM_ROTARY_PLAIN;
  if (kind < METALLLM_ROTARY_PLAIN || kind > METALLLM_ROTARY_PARTS) return METALLLM_ATTN_E_LAYOUT;
  if (kind != METALLLM_ROTARY_PLAIN && (!(sc->factor > 0.0) || !std::isfinite(sc->factor))) return METALLLM_ATTN_E_LAYOUT;
  if (kind == METALLLM_ROTARY_PARTS && (!(sc->original > 0.0) || !std::isfinite(sc->original) || !std::isfinite(sc->low) ||
                                        !std::isfinite(sc->high) || !(sc->high > sc->low)))
    return METALLLM_ATTN_E_LAYOUT;
  const float magnitude = sc ? sc->magnitude : 1.0f;
  if (!std::isfinite(magnitude)) return METALLLM_ATTN_E_LAYOUT;
  metalllmRotaryPlan r{};
  r.dims = dims, r.interleaved = interleaved != 0, r.magnitude = magnitude;
  const double two_pi = 6.283185307179586476925286766559;
  for (uint32_t i = 0; i < dims / 2; ++i) {
    double f = std::pow(base, -2.0 * i / dims) / two_pi;
    if (!std::isfinite(f)) return METALLLM_ATTN_E_LAYOUT;
    if (kind == METALLLM_ROTARY_LINEAR) f /= sc->factor;
    if (kind == METALLLM_ROTARY_PARTS) {
      const double keep = std::min(1.0, std::max(0.0, (sc->original * f - sc->low) / (sc->high - sc->low)));
      f = f * keep + f / sc->factor * (1.0 - keep);
    }
    r.turns[i] = f;
  }
  *plan = r;
  return METALLLM_ATTN_OK;
}

int rotaryForward(const uint16_t* q, const uint16_t* k, uint16_t* q_out, uint16_t* k_out, const int32_t* positions,
                  const metalllmRotaryPlan* plan, const metalllmRotaryParams* p, metalllm_stream_t stream) {
  return rotary(q, k, q_out, k_out, positions, plan, p, (hipStream_t)stream, 0);
}

int rotaryBackward(const uint16_t* dq, const uint16_t* dk, uint16_t* dq_out, uint16_t* dk_out, const int32_t* positions,
                   const metalllmRotaryPlan* plan, const metalllmRotaryParams* p, metalllm_stream_t stream) {
  return rotary(dq, dk, dq_out, dk_out, positions, plan, p, (hipStream_t)stream, 1);
}

}  // extern "C"
