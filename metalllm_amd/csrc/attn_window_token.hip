// attn_window_token.hip -- windowAttentionForward on gfx950 for few query rows: next tokens over a cache, a prompt's
// part, or a short prompt (win_is_token).
//
// The mathematics is attn_window_fwd.hip's. The bound is reading the visible keys and values once, so
// there is no LDS tile: the G query heads that share a key head, times the query rows, are the 16 columns
// of v_mfma_f32_16x16x32_bf16, and every lane loads its operands from global memory as it needs them.
//   * S^T = K.Q^T: the lane's key row lane%16 (+16), d = 32c + 8g .. +7 with g = lane/16: 64 bytes of each
//     of 16 rows per load.
//   * C gives the lane keys 4g + r and 16 + 4g + r of its query, which are the 8 keys that it holds as the
//     B operand of O^T += V^T.P^T: the order of keys inside a product is free as long as both operands
//     agree, so p needs no exchange.
//   * V rows are loaded whole (16 lanes x 16 or 8 bytes), the lane's 8 keys of its d chunk, and turned in
//     registers: one v_perm per pair of values. The d of an output row is E*(4g + r) + e for product e.
// A step takes 32 keys. Its K registers are loaded again as soon as its scores are formed, its V registers
// as soon as its products are; what one to three waves per SIMD have in flight covers the rest.
//
// Split: the steps are dealt to the waves of a workgroup, and over `splits` workgroups where there are
// too few (sequence, key head) pairs to fill the chip; each part keeps its own reference point and sum, and
// they are joined in LDS, or through the workspace by a second small kernel.
//
// Measured: 64 sequences of 4096 visible keys, 16 heads of 128 over 4, 97 to 104 us by card: 5.2 to 5.5 TB/s of the keys
// and values, above a large copy's 4.7. 12 heads of 64, 512 keys: 6.5 us, of
// which a launch is 2; the rest is three dependent reads (lengths, keys and values, the join).
#include <algorithm>

#include "attn_common.hpp"
#include "attn_window.hpp"

namespace mla {

typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
// over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max_groups(float x) {
  x = max_halves(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
  x = sum_halves(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ bool not_finite(uint32_t pair) {
  return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}

constexpr int kTokWaves = 4;  // to a workgroup

template <int D>
struct WtCfg {
  static constexpr int KC = D / 32;  // products over d of a score
  static constexpr int E = D / 16;   // output products: values of a V row per lane
  static constexpr int VW = E / 2;   // dwords of a V row per lane
  static constexpr int KEYS = 32;    // per step
  static constexpr int PITCH = D + 4;
};

// The rows of one tile of 16 (query row, head of the group) and the keys they visit.
struct WtRange {
  int i_lo, i_hi;  // query rows (i_hi < lq); none where i_lo > i_hi
  int w_lo, end, ns, sink_steps, steps;
};
__device__ __forceinline__ WtRange wt_range(const WinShape& s, const WinSeq& q, int rt) {
  WtRange r{0, -1, 0, 0, 0, 0, 0};
  r.i_lo = rt * kTokRows / s.G;
  r.i_hi = min(min(rt * kTokRows + kTokRows, s.TQ * s.G) - 1, q.lq * s.G - 1) / s.G;
  if (q.lq == 0) r.i_hi = -1;
  if (r.i_lo > r.i_hi || q.off + r.i_hi < 0) return r;
  r.end = q.off + r.i_hi + 1;
  r.w_lo = max(0, q.off + r.i_lo - s.window + 1);
  r.ns = min(s.sinks, r.w_lo);
  r.sink_steps = (r.ns + 31) / 32;
  r.steps = r.sink_steps + (r.end - r.w_lo + 31) / 32;
  return r;
}

// SEVERAL: more than one query row (TQ > 1), which may see different keys of a step; its path for values that
// are not finite takes registers that one row does without.
template <int D, bool SEVERAL>
__global__ void __launch_bounds__(64 * kTokWaves, SEVERAL ? 2 : D == 64 ? 4 : 3) win_token_kernel(WinFwdArgs a) {
  using C = WtCfg<D>;
  __shared__ __attribute__((aligned(16))) float sm_o[kTokWaves][kTokRows][C::PITCH];
  __shared__ float sm_m[kTokWaves][kTokRows], sm_l[kTokWaves][kTokRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n16 = lane & 15;
  const WinShape& s = a.s;
  const int tiles = (s.TQ * s.G + kTokRows - 1) / kTokRows;
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int rt = unit % tiles, group = unit / tiles;
  const int b = group / s.NKV, kvh = group - b * s.NKV;
  const WinSeq sq = win_seq(s, b);
  const WtRange w = wt_range(s, sq, rt);
  if (w.i_lo > w.i_hi) return;  // rows behind the sequence: left as they were (the join too)
  const int parts = kTokWaves * a.splits, part = kTokWaves * split + wave;
  const int t0 = (int)((int64_t)w.steps * part / parts), t1 = (int)((int64_t)w.steps * (part + 1) / parts);

  const int row = rt * kTokRows + n16, qi = row / s.G;
  const bool row_ok = qi <= w.i_hi && row < s.TQ * s.G;
  const int pos = sq.off + qi;
  u32x4 Qr[C::KC];
#pragma unroll
  for (int c = 0; c < C::KC; ++c) Qr[c] = u32x4{0, 0, 0, 0};
  if (row_ok) {
    const uint16_t* qr = a.q + b * s.q_seq + (size_t)qi * s.q_row + (kvh * s.G + row - qi * s.G) * D + 8 * g;
#pragma unroll
    for (int c = 0; c < C::KC; ++c) Qr[c] = *(const u32x4*)(qr + 32 * c);
  }
  const char* Kg = (const char*)(a.k + b * s.k_seq + kvh * D);
  const char* Vg = (const char*)(a.v + b * s.v_seq + kvh * D);
  const uint32_t krs = 2 * s.k_row, vrs = 2 * s.v_row;
  const float c1 = s.scale * kLog2e, slack = 8.0f / c1;

  // first key of step t and one past its last
  auto keys_of = [&](int t, int& base, int& end) {
    const bool sink = t < w.sink_steps;
    base = sink ? 32 * t : w.w_lo + 32 * (t - w.sink_steps);
    end = sink ? w.ns : w.end;
  };
  // V row x of the lane: key 4g + x, or 16 + 4g + x - 4
  auto v_key = [&](int x) { return 4 * g + x + (x >= 4 ? 12 : 0); };
  u32x4 kk[2][C::KC];      // the lane's two K rows of a step
  uint32_t vv[8][C::VW];  // its 8 V rows
  auto load_k = [&](int t) __attribute__((always_inline)) {
    int base, end;
    keys_of(t, base, end);
    const char* kp = Kg + (size_t)base * krs;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t at = __umul24(min(16 * u + n16, end - 1 - base), krs) + 16 * g;
#pragma unroll
      for (int c = 0; c < C::KC; ++c) kk[u][c] = *(const u32x4*)(kp + at + 64 * c);
    }
  };
  auto load_v = [&](int t) __attribute__((always_inline)) {
    int base, end;
    keys_of(t, base, end);
    const char* vp = Vg + (size_t)base * vrs;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const uint32_t at = __umul24(min(v_key(x), end - 1 - base), vrs) + 4 * C::VW * n16;
      if constexpr (C::VW == 4) {
        const u32x4 y = *(const u32x4*)(vp + at);
#pragma unroll
        for (int d = 0; d < 4; ++d) vv[x][d] = y[d];
      } else {
        const u32x2v y = *(const u32x2v*)(vp + at);
        vv[x][0] = y[0];
        vv[x][1] = y[1];
      }
    }
  };

  f32x4 O[C::E];
#pragma unroll
  for (int e = 0; e < C::E; ++e) O[e] = f32x4{0, 0, 0, 0};
  float m_run = -INFINITY, l_run = 0.0f;

  // V^T operand of product e: d = E*lane%16 + e, the lane's 8 keys
  auto turned = [&](int e) {
    u32x4 r;
#pragma unroll
    for (int d = 0; d < 4; ++d)
      r[d] = __builtin_amdgcn_perm(vv[2 * d + 1][e / 2], vv[2 * d][e / 2], (e & 1) ? 0x07060302u : 0x05040100u);
    return r;
  };
  auto step = [&](int t) __attribute__((always_inline)) {
    int base, end;
    keys_of(t, base, end);
    f32x4 S[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
    for (int c = 0; c < C::KC; ++c) {
      S[0] = mfma16(kk[0][c], Qr[c], S[0]);
      S[1] = mfma16(kk[1][c], Qr[c], S[1]);
    }
    if (t + 1 < t1) load_k(t + 1);
    float mt = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = base + 16 * u + 4 * g + r;
        S[u][r] = key < end && win_sees(s, pos, key) ? S[u][r] : -INFINITY;
        mt = fmaxf(mt, S[u][r]);
      }
    mt = max_groups(mt);
    const bool need = mt > m_run + slack;
    if (__any(need)) {
      const float m_new = need ? mt : m_run;
      const float alpha = need ? exp2_hw((m_run - m_new) * c1) : 1.0f;
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int e = 0; e < C::E; ++e) O[e] *= alpha;
    }
    const float mb = m_run == -INFINITY ? 0.0f : m_run * c1;
    float p[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      p[x] = exp2_hw(fmaf(S[x >> 2][x & 3], c1, -mb));
      l_run += p[x];
    }
    const u32x4 P = {pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7])};
    bool odd = false;
    if (SEVERAL) {
#pragma unroll
      for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int d = 0; d < C::VW; ++d) odd |= not_finite(vv[x][d]);
    }
    if (!SEVERAL || !__any(odd)) {
#pragma unroll
      for (int e = 0; e < C::E; ++e) O[e] = mfma16(turned(e), P, O[e]);
    } else {  // values that are not finite: query row by query row, without the keys that it does not see
      for (int i = w.i_lo; i <= w.i_hi; ++i) {
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
          for (int d = 0; d < C::VW; ++d) pin(vv[x][d]);  // (or the turned operands are kept over the loop)
        u32x4 kept;  // of the pairs of keys in an operand
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int k0 = base + v_key(2 * d), k1 = base + v_key(2 * d + 1);
          kept[d] = (k0 < end && win_sees(s, sq.off + i, k0) ? 0xffffu : 0u) |
                    (k1 < end && win_sees(s, sq.off + i, k1) ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int e = 0; e < C::E; ++e) {
          const f32x4 y = mfma16(turned(e) & kept, P, O[e]);
          if (qi == i) O[e] = y;
        }
      }
    }
    if (t + 1 < t1) load_v(t + 1);
  };

  if (t0 < t1) {
    load_k(t0);
    load_v(t0);
    for (int t = t0; t < t1; ++t) step(t);
  }

  // ---- join the waves ----
  l_run = sum_groups(l_run);
  if (g == 0) {
    sm_m[wave][n16] = m_run * c1;
    sm_l[wave][n16] = l_run;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int e = 0; e < C::E; ++e) sm_o[wave][n16][C::E * (4 * g + r) + e] = O[e][r];
  __syncthreads();
  const int jr = tid >> 4, d0 = (tid & 15) * C::E;  // row and columns that this thread joins
  if (jr >= kTokRows) return;
  float M = -INFINITY;
#pragma unroll
  for (int v = 0; v < kTokWaves; ++v) M = fmaxf(M, sm_m[v][jr]);
  float L = 0.0f, acc[C::E];
#pragma unroll
  for (int e = 0; e < C::E; ++e) acc[e] = 0.0f;
#pragma unroll
  for (int v = 0; v < kTokWaves; ++v) {
    const float m = sm_m[v][jr];
    if (m == -INFINITY && sm_l[v][jr] == 0.0f) continue;  // a part without visible keys
    const float f = exp2_hw(m - (M == -INFINITY ? 0.0f : M));
    L = fmaf(sm_l[v][jr], m == -INFINITY ? 1.0f : f, L);
#pragma unroll
    for (int e = 0; e < C::E; ++e) acc[e] = fmaf(sm_o[v][jr][d0 + e], m == -INFINITY ? 1.0f : f, acc[e]);
  }
  if (a.splits > 1) {
    float* out = a.part + (((size_t)unit * a.splits + split) * kTokRows + jr) * (D + 2);
#pragma unroll
    for (int e = 0; e < C::E; e += 2) *(f32x2*)(out + d0 + e) = f32x2{acc[e], acc[e + 1]};
    if ((tid & 15) == 0) *(f32x2*)(out + D) = f32x2{M, L};
    return;
  }
  const int orow = rt * kTokRows + jr, oi = orow / s.G;
  if (oi > w.i_hi || orow >= s.TQ * s.G) return;
  const int head = kvh * s.G + orow - oi * s.G;
  const bool empty = sq.off + oi < 0;
  const float inv = 1.0f / L;
  uint32_t* o = (uint32_t*)(a.out + b * s.o_seq + (size_t)oi * s.o_row + head * D + d0);
#pragma unroll
  for (int e = 0; e < C::E; e += 2) o[e / 2] = empty ? 0u : pack_bf16(acc[e] * inv, acc[e + 1] * inv);
  if (a.l && (tid & 15) == 0)
    a.l[((size_t)b * s.NH + head) * s.TQ + oi] = empty ? -INFINITY : M * (1.0f / kLog2e) + logf(L);
}

// The parts of a tile's rows, in order: 256 threads, 16 to a row.
template <int D>
__global__ void __launch_bounds__(256) win_join_kernel(WinFwdArgs a) {
  using C = WtCfg<D>;
  const int tid = threadIdx.x;
  const WinShape& s = a.s;
  const int tiles = (s.TQ * s.G + kTokRows - 1) / kTokRows;
  const int unit = blockIdx.x, rt = unit % tiles, group = unit / tiles;
  const int b = group / s.NKV, kvh = group - b * s.NKV;
  const WinSeq sq = win_seq(s, b);
  const WtRange w = wt_range(s, sq, rt);
  const int jr = tid >> 4, d0 = (tid & 15) * C::E;
  const int row = rt * kTokRows + jr, qi = row / s.G;
  if (w.i_lo > w.i_hi || qi > w.i_hi || row >= s.TQ * s.G) return;
  const float* in = a.part + ((size_t)unit * a.splits * kTokRows + jr) * (D + 2);
  const size_t step = (size_t)kTokRows * (D + 2);
  float M = -INFINITY;
#pragma unroll 8
  for (int v = 0; v < a.splits; ++v) M = fmaxf(M, in[v * step + D]);
  const float Mb = M == -INFINITY ? 0.0f : M;
  float L = 0.0f, acc[C::E];
#pragma unroll
  for (int e = 0; e < C::E; ++e) acc[e] = 0.0f;
#pragma unroll 4
  for (int v = 0; v < a.splits; ++v) {  // (a part without keys holds m = -inf and zeros)
    const float* p = in + v * step;
    const float m = p[D], l = p[D + 1];
    const float f = m == -INFINITY ? 1.0f : exp2_hw(m - Mb);
    L = fmaf(l, f, L);
#pragma unroll
    for (int e = 0; e < C::E; ++e) acc[e] = fmaf(p[d0 + e], f, acc[e]);
  }
  const int head = kvh * s.G + row - qi * s.G;
  const bool empty = sq.off + qi < 0;
  const float inv = 1.0f / L;
  uint32_t* o = (uint32_t*)(a.out + b * s.o_seq + (size_t)qi * s.o_row + head * D + d0);
#pragma unroll
  for (int e = 0; e < C::E; e += 2) o[e / 2] = empty ? 0u : pack_bf16(acc[e] * inv, acc[e + 1] * inv);
  if (a.l && (tid & 15) == 0)
    a.l[((size_t)b * s.NH + head) * s.TQ + qi] = empty ? -INFINITY : M * (1.0f / kLog2e) + logf(L);
}

// Workgroups to a unit (sequence, key head, row tile), from the steps that a unit has at most: as many as put
// one on each CU, where their waves get 4 steps or more. One workgroup joins its waves in LDS; more take
// the second kernel. us at (B, TQ, TK, NH, NKV, D), all keys visible but (64, ..), which sees 4096:
//                                 this   two for each CU  6 steps or more  never split
//   (4, 1, 4096, 16, 4, 128)      13.2   13.3             16.3             39.8
//   (16, 1, 4096, 16, 4, 128)     26.4   28.1             26.6             42.9
//   (64, 1, 8192, 16, 4, 128)     96.8  107.5             96.8             96.8
// Workgroups of 8 waves, so half as many of them, took 26.0 and 28.7 in the first two.
int win_token_splits(const WinShape& s) {
  const int64_t units = win_token_units(s);
  const int64_t keys = std::min<int64_t>((int64_t)s.window + s.TQ - 1, s.TK) + s.sinks;
  const int64_t steps = (keys + 31) / 32;
  const int64_t want = std::min<int64_t>((kCus + units - 1) / units, steps / (4 * kTokWaves));
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, 64));
}

template <int D>
static hipError_t launch_token(const WinFwdArgs& a, unsigned units, hipStream_t s) {
  const dim3 grid(units * a.splits);
  hipLaunchKernelGGL((a.s.TQ > 1 ? win_token_kernel<D, true> : win_token_kernel<D, false>), grid, dim3(64 * kTokWaves), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL(win_join_kernel<D>, dim3(units), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_window_token(const WinFwdArgs& a, int D, hipStream_t s) {
  const unsigned units = (unsigned)win_token_units(a.s);
  return D == 64 ? launch_token<64>(a, units, s) : launch_token<128>(a, units, s);
}

}  // namespace mla
