// rmsnorm.hip -- root-mean-square norm with the residual's addition (include/metalllm_attn.h), HBM-bound.
//
// Forward, per row: h = x + residual, rstd = 1/sqrt(mean(h^2) + eps), y = h rstd gamma, written as bf16 or
// as e4m3 with one scale per group of columns (the group's largest |y| / 448). h is normed as the fp32 sum;
// bf16(h) is stored for the residual stream. Backward, with xh = h rstd and g = dOut gamma:
// dX = dSum + rstd (g - xh mean(g xh)), dgamma = sum over rows of dOut xh.
//
// A row belongs to a team of 64 or 256 threads that holds it in registers, 16-byte chunks c = thread +
// TEAM j, so it is read once and written once. One wave per row up to 2048 columns: its sum needs no
// barrier. The backward runs one workgroup of up to 1024 threads per CU over many rows; a thread sums dgamma of
// its columns in registers, the teams are joined in LDS, and one row of partial sums per workgroup goes
// to the workspace, where a second kernel adds them in order (no atomics: results repeat bit for bit).
//
// Measured: 16383 rows of 4096 with e4m3 out 81 us, 5.8 TB/s of 472 MB; the backward of 16384 rows of 768 20 us, 5.0
// TB/s, and 4 us for the join (from within one launch to the next); 7 rows of 768 2.4 us, a launch.
// 64 rows of 2048 columns would take 2.6 us instead of 3.1 with 256 threads to a row; 16384 rows take 40.3 either way.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "../../include/metalllm_attn.h"
#include "overlap.hpp"

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float kFp8Max = 448.0f;
constexpr int kBwdBlocks = 256;  // workgroups of the backward: one per CU

__device__ __forceinline__ uint32_t pk(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, b2));
}
__device__ __forceinline__ void unpack(u4 v, float (&f)[8]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[2 * w] = __uint_as_float(v[w] << 16);
    f[2 * w + 1] = __uint_as_float(v[w] & 0xffff0000u);
  }
}
__device__ __forceinline__ u4 pack(const float (&f)[8]) {
  return u4{pk(f[0], f[1]), pk(f[2], f[3]), pk(f[4], f[5]), pk(f[6], f[7])};
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
struct Sum {
  __device__ static float op(float a, float b) { return a + b; }
};
struct Max {
  __device__ static float op(float a, float b) { return fmaxf(a, b); }
};
// Over 4, 8, 16 or 64 lanes beside each other; every lane gets the same result.
template <class Op, int N>
__device__ __forceinline__ float lanes(float v) {
  v = Op::op(v, dpp<0xb1>(v));                      // lane ^ 1
  v = Op::op(v, dpp<0x4e>(v));                      // lane ^ 2
  if (N >= 8) v = Op::op(v, dpp<0x141>(v));         // mirrored in its 8: the other quad
  if (N >= 16) v = Op::op(v, dpp<0x140>(v));        // mirrored in its 16: the other 8
  if (N >= 64) {
    const uint32_t u = __float_as_uint(v);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = Op::op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t w = __float_as_uint(v);
    auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    v = Op::op(__uint_as_float(b[0]), __uint_as_float(b[1]));
  }
  return v;
}
// Over the TEAM threads of a row; slot: 4 floats of LDS per team, used in turn by `turn`
template <class Op, int TEAM>
__device__ __forceinline__ float team(float v, float (*slot)[4]) {
  v = lanes<Op, 64>(v);
  if (TEAM == 64) return v;
  const int t = threadIdx.x / TEAM, w = (threadIdx.x / 64) % (TEAM / 64);
  if ((threadIdx.x & 63) == 0) slot[t][w] = v;
  __syncthreads();
  v = Op::op(Op::op(slot[t][0], slot[t][1]), Op::op(slot[t][2], slot[t][3]));
  return v;
}

struct FwdArgs {
  const uint16_t* x;
  const uint16_t* res;
  uint16_t* sum;
  void* out;
  float* scales;
  const uint16_t* gamma;
  float* rstd;
  uint32_t rows, cols, group;
  float eps;
};

// FP8: 0 = bf16 output, else e4m3
template <int TEAM, int NCH, bool FP8>
__global__ void __launch_bounds__(256) rms_fwd_kernel(FwdArgs a) {
  __shared__ float slots[2][256 / TEAM][4];
  const uint32_t lane = threadIdx.x % TEAM;
  const uint64_t row = (uint64_t)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
  if (row >= a.rows) return;  // TEAM = 256: the whole workgroup
  const uint32_t nchunk = a.cols / 8;
  const u4* x = (const u4*)(a.x + row * a.cols);
  const u4* r = a.res ? (const u4*)(a.res + row * a.cols) : nullptr;
  u4 xv[NCH], rv[NCH], gv[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const uint32_t c = lane + TEAM * j;
    const bool in = c < nchunk;
    xv[j] = in ? x[c] : u4{0, 0, 0, 0};
    rv[j] = in && r ? r[c] : u4{0, 0, 0, 0};
    gv[j] = in ? ((const u4*)a.gamma)[c] : u4{0, 0, 0, 0};
  }
  float h[NCH][8], sq = 0.0f;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    float f[8];
    unpack(xv[j], h[j]);
    if (r) {
      unpack(rv[j], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] += f[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sq = fmaf(h[j][e], h[j][e], sq);
    const uint32_t c = lane + TEAM * j;
    if (a.sum && c < nchunk) ((u4*)(a.sum + row * a.cols))[c] = pack(h[j]);
  }
  sq = team<Sum, TEAM>(sq, slots[0]);
  const float rstd = 1.0f / sqrtf(sq / (float)a.cols + a.eps);
  if (a.rstd && lane == 0) a.rstd[row] = rstd;
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    float f[8];
    unpack(gv[j], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[j][e] = h[j][e] * rstd * f[e];
      if (FP8) amax = fmaxf(amax, fabsf(h[j][e]));
    }
    if (!FP8) {
      const uint32_t c = lane + TEAM * j;
      if (c < nchunk) ((u4*)((uint16_t*)a.out + row * a.cols))[c] = pack(h[j]);
    }
  }
  if (!FP8) return;
  if (a.group == 0) amax = team<Max, TEAM>(amax, slots[1]);
  const uint32_t per = a.group ? a.group / 8 : 1, groups = a.group ? (nchunk + per - 1) / per : 1;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const uint32_t c = lane + TEAM * j;
    float m = amax;
    if (a.group) {
      m = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(h[j][e]));
      m = per == 4 ? lanes<Max, 4>(m) : per == 8 ? lanes<Max, 8>(m) : lanes<Max, 16>(m);
    }
    // all zeros: 1; at least the smallest normal number, so that its reciprocal is finite
    const float scale = m == 0.0f ? 1.0f : fmaxf(m / kFp8Max, 0x1p-126f), inv = 1.0f / scale;
    if (c < nchunk) {
      uint32_t w[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        int v = __builtin_amdgcn_cvt_pk_fp8_f32(h[j][4 * u] * inv, h[j][4 * u + 1] * inv, 0, false);
        w[u] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(h[j][4 * u + 2] * inv, h[j][4 * u + 3] * inv, v, true);
      }
      ((uint2*)((uint8_t*)a.out + row * a.cols))[c] = uint2{w[0], w[1]};
      if (a.group ? c % per == 0 : lane == 0 && j == 0) a.scales[row * groups + (a.group ? c / per : 0)] = scale;
    }
  }
}

struct BwdArgs {
  const uint16_t* dout;
  const uint16_t* dsum;
  const uint16_t* h;
  const uint16_t* gamma;
  const float* rstd;
  uint16_t* dx;
  float* part;  // [blocks][cols]
  uint32_t rows, cols;
};

template <int TEAM, int NCH, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_bwd_kernel(BwdArgs a) {
  constexpr int TEAMS = THREADS / TEAM;
  __shared__ float slots[2][TEAMS][4];
  __shared__ __attribute__((aligned(16))) float joined[TEAMS][TEAM * 8];  // 32 bytes a thread
  const uint32_t lane = threadIdx.x % TEAM, tm = threadIdx.x / TEAM;
  const uint32_t nchunk = a.cols / 8, step = gridDim.x * TEAMS;
  u4 gv[NCH];
  float dg[NCH][8];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const uint32_t c = lane + TEAM * j;
    gv[j] = c < nchunk ? ((const u4*)a.gamma)[c] : u4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[j][e] = 0.0f;
  }
  const uint32_t rounds = (a.rows + step - 1) / step;  // the same for every team: team() may have a barrier
  for (uint32_t n = 0; n < rounds; ++n) {
    const uint64_t row = (uint64_t)n * step + blockIdx.x * TEAMS + tm;
    const bool in = row < a.rows;
    const u4* dy = (const u4*)(a.dout + row * a.cols);
    const u4* hh = (const u4*)(a.h + row * a.cols);
    const u4* ds = a.dsum ? (const u4*)(a.dsum + row * a.cols) : nullptr;
    u4 yv[NCH], hv[NCH], sv[NCH];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const uint32_t c = lane + TEAM * j;
      const bool ok = in && c < nchunk;
      yv[j] = ok ? dy[c] : u4{0, 0, 0, 0};
      hv[j] = ok ? hh[c] : u4{0, 0, 0, 0};
      sv[j] = ok && ds ? ds[c] : u4{0, 0, 0, 0};
    }
    const float rstd = in ? a.rstd[row] : 0.0f;
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      float y[8], x[8], g[8];
      unpack(yv[j], y);
      unpack(hv[j], x);
      unpack(gv[j], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = x[e] * rstd;
        dg[j][e] = fmaf(y[e], xh, dg[j][e]);
        dot = fmaf(y[e] * g[e], xh, dot);
      }
    }
    dot = team<Sum, TEAM>(dot, slots[n & 1]) / (float)a.cols;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const uint32_t c = lane + TEAM * j;
      float y[8], x[8], g[8], s[8];
      unpack(yv[j], y);
      unpack(hv[j], x);
      unpack(gv[j], g);
      unpack(sv[j], s);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = fmaf(rstd, y[e] * g[e] - x[e] * rstd * dot, s[e]);
      if (in && c < nchunk) ((u4*)(a.dx + row * a.cols))[c] = pack(s);
    }
  }
  // the teams' sums of TEAM chunks at a time
  for (int j = 0; j < NCH; ++j) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f4 v;
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (i == j) v = f4{dg[i][4 * u], dg[i][4 * u + 1], dg[i][4 * u + 2], dg[i][4 * u + 3]};
      *(f4*)&joined[tm][8 * lane + 4 * u] = v;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < TEAM * 8; i += THREADS) {
      const uint32_t col = TEAM * 8 * j + i;
      if (col >= a.cols) break;
      float s = 0.0f;
#pragma unroll
      for (int t = 0; t < TEAMS; ++t) s += joined[t][i];
      a.part[(size_t)blockIdx.x * a.cols + col] = s;
    }
  }
}

// dgamma[c] = sum over the workgroups' rows: 16 columns to a workgroup, 16 threads to a column
__global__ void __launch_bounds__(256) rms_join_kernel(const float* part, float* dgamma, uint32_t blocks, uint32_t cols) {
  __shared__ float sums[16][17];
  const uint32_t c = threadIdx.x % 16, s = threadIdx.x / 16, col = blockIdx.x * 16 + c;
  float v = 0.0f;
  if (col < cols) {
#pragma unroll 8
    for (uint32_t b = s; b < blocks; b += 16) v += part[(size_t)b * cols + col];
  }
  sums[s][c] = v;
  __syncthreads();
  if (s == 0 && col < cols) {
    v = 0.0f;
    for (int i = 0; i < 16; ++i) v += sums[i][c];
    dgamma[col] = v;
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int validate(const metalllmRmsnormParams* p) {
  if (!p) return METALLLM_ATTN_E_NULL;
  if (p->rows == 0 || p->cols == 0 || p->cols % 8 || p->cols > METALLLM_RMSNORM_MAX_COLS) return METALLLM_ATTN_E_LAYOUT;
  if (!(p->eps >= 0.0f) || !std::isfinite(p->eps)) return METALLLM_ATTN_E_LAYOUT;
  if (p->group != 0 && p->group != 32 && p->group != 64 && p->group != 128) return METALLLM_ATTN_E_LAYOUT;
  if (p->rows >= (1u << 24)) return METALLLM_ATTN_E_SIZE;  // 256 threads to a row, counted in 32 bits
  return METALLLM_ATTN_OK;
}

// The backward's workgroups: one per CU, of 1024 threads or, where four chunks a thread need more than 128 registers,
// 512 (1024 spill: 16384 rows of 7816 columns 579 us, with 512 194 us; 1000 of 2048 27.8 and 10.0). Up to 32
// workgroups' worth of rows 256 threads: more of them, but more sums to join (16 rows of 4096: 5.8 us against 6.6,
// 100 rows of 4096 8.4 against 6.9).
struct BwdGrid {
  bool few;
  unsigned threads, blocks;
};
BwdGrid bwd_grid(const metalllmRmsnormParams& p) {
  const uint32_t team = p.cols <= 2048 ? 64 : 256;
  if (p.rows <= 32 * (256 / team)) return {true, 256, (p.rows + 256 / team - 1) / (256 / team)};
  const uint32_t threads = p.cols > 4096 || (p.cols > 1024 && p.cols <= 2048) ? 512 : 1024, teams = threads / team;
  return {false, threads, std::min<uint32_t>(kBwdBlocks, (p.rows + teams - 1) / teams)};
}
template <int TEAM, int NCH, int THREADS>
void backward(const BwdGrid& g, const BwdArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((g.few ? rms_bwd_kernel<TEAM, NCH, 256> : rms_bwd_kernel<TEAM, NCH, THREADS>), dim3(g.blocks),
                     dim3(g.threads), 0, s, a);
}

template <bool FP8>
int forward(const FwdArgs& a, hipStream_t s) {
  const uint32_t n = a.cols / 8;
  const dim3 wave((a.rows + 3) / 4), wide(a.rows);
  if (n <= 64)
    hipLaunchKernelGGL((rms_fwd_kernel<64, 1, FP8>), wave, dim3(256), 0, s, a);
  else if (n <= 128)
    hipLaunchKernelGGL((rms_fwd_kernel<64, 2, FP8>), wave, dim3(256), 0, s, a);
  else if (n <= 256)
    hipLaunchKernelGGL((rms_fwd_kernel<64, 4, FP8>), wave, dim3(256), 0, s, a);
  else if (n <= 512)
    hipLaunchKernelGGL((rms_fwd_kernel<256, 2, FP8>), wide, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((rms_fwd_kernel<256, 4, FP8>), wide, dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? METALLLM_ATTN_OK : METALLLM_ATTN_E_LAUNCH;
}

// An output may lie in the memory of an input of its type and size (a team holds a row before it writes
// it), else apart from every input; outputs apart from each other.
bool in_place_or_apart(const mla::Span& out, std::initializer_list<mla::Span> in) {
  for (const mla::Span& i : in)
    if (i.p && mla::overlap(out, i) && !(out.p == i.p && out.bytes == i.bytes)) return false;
  return true;
}

int check_forward(const uint16_t* x, const uint16_t* res, uint16_t* sum, const void* out, size_t out_bytes,
                  const float* scales, size_t scale_bytes, const uint16_t* gamma, const float* rstd,
                  const metalllmRmsnormParams* p) {
  if (!x || !out || !gamma || (res && !sum)) return METALLLM_ATTN_E_NULL;
  for (const void* t : {(const void*)x, (const void*)res, (const void*)sum, out, (const void*)scales, (const void*)gamma,
                        (const void*)rstd})
    if (!aligned16(t)) return METALLLM_ATTN_E_ALIGN;
  const size_t e = (size_t)p->rows * p->cols;
  const mla::Span so{out, out_bytes}, ss{sum, sum ? 2 * e : 0}, sc{scales, scale_bytes}, sr{rstd, rstd ? 4 * (size_t)p->rows : 0};
  const mla::Span sx{x, 2 * e}, sres{res, res ? 2 * e : 0}, sg{gamma, 2 * (size_t)p->cols};
  if (mla::any_overlap({so, ss, sc, sr}) || mla::any_overlap({so, ss, sc, sr}, {sg}) || mla::any_overlap({sc, sr}, {sx, sres}) ||
      !in_place_or_apart(so, {sx, sres}) || !in_place_or_apart(ss, {sx, sres}))
    return METALLLM_ATTN_E_OVERLAP;
  return METALLLM_ATTN_OK;
}

}  // namespace

extern "C" {

int rmsnormForward(const uint16_t* x, const uint16_t* residual, uint16_t* sum, uint16_t* out, const uint16_t* gamma,
                   float* rstd, const metalllmRmsnormParams* p, metalllm_stream_t stream) {
  int rc = validate(p);
  if (rc) return rc;
  rc = check_forward(x, residual, sum, out, 2 * (size_t)p->rows * p->cols, nullptr, 0, gamma, rstd, p);
  if (rc) return rc;
  return forward<false>(FwdArgs{x, residual, sum, out, nullptr, gamma, rstd, p->rows, p->cols, 0, p->eps},
                        (hipStream_t)stream);
}

int rmsnormForwardFp8(const uint16_t* x, const uint16_t* residual, uint16_t* sum, uint8_t* out, float* scales,
                      const uint16_t* gamma, float* rstd, const metalllmRmsnormParams* p, metalllm_stream_t stream) {
  int rc = validate(p);
  if (rc) return rc;
  if (!scales) return METALLLM_ATTN_E_NULL;
  const size_t groups = p->group ? (p->cols + p->group - 1) / p->group : 1;
  rc = check_forward(x, residual, sum, out, (size_t)p->rows * p->cols, scales, 4 * groups * p->rows, gamma, rstd, p);
  if (rc) return rc;
  return forward<true>(FwdArgs{x, residual, sum, out, scales, gamma, rstd, p->rows, p->cols, p->group, p->eps},
                       (hipStream_t)stream);
}

int metalllmRmsnormBackwardWorkspaceSize(const metalllmRmsnormParams* p, uint64_t* bytes) {
  const int rc = validate(p);
  if (rc) return rc;
  if (!bytes) return METALLLM_ATTN_E_NULL;
  *bytes = 4ull * bwd_grid(*p).blocks * p->cols;
  return METALLLM_ATTN_OK;
}

int rmsnormBackward(const uint16_t* dOut, const uint16_t* dSum, const uint16_t* h, const uint16_t* gamma, const float* rstd,
                    uint16_t* dX, float* dgamma, void* workspace, uint64_t workspace_bytes,
                    const metalllmRmsnormParams* p, metalllm_stream_t stream) {
  const int rc = validate(p);
  if (rc) return rc;
  if (!dOut || !h || !gamma || !rstd || !dX || !dgamma || !workspace) return METALLLM_ATTN_E_NULL;
  for (const void* t : {(const void*)dOut, (const void*)dSum, (const void*)h, (const void*)gamma, (const void*)rstd,
                        (const void*)dX, (const void*)dgamma, (const void*)workspace})
    if (!aligned16(t)) return METALLLM_ATTN_E_ALIGN;
  const BwdGrid g = bwd_grid(*p);
  const size_t need = 4ull * g.blocks * p->cols, e = 2 * (size_t)p->rows * p->cols;
  if (workspace_bytes < need) return METALLLM_ATTN_E_SIZE;
  const mla::Span sdx{dX, e}, sdg{dgamma, 4 * (size_t)p->cols}, sw{workspace, need};
  const mla::Span sy{dOut, e}, ss{dSum, dSum ? e : 0}, sh{h, e}, sg{gamma, 2 * (size_t)p->cols}, sr{rstd, 4 * (size_t)p->rows};
  if (mla::any_overlap({sdx, sdg, sw}) || mla::any_overlap({sdg, sw}, {sy, ss, sh}) || mla::any_overlap({sdx, sdg, sw}, {sg, sr}) ||
      !in_place_or_apart(sdx, {sy, ss, sh}))
    return METALLLM_ATTN_E_OVERLAP;
  const BwdArgs a{dOut, dSum, h, gamma, rstd, dX, (float*)workspace, p->rows, p->cols};
  const hipStream_t s = (hipStream_t)stream;
  const uint32_t n = p->cols / 8;
  if (n <= 64)
    backward<64, 1, 1024>(g, a, s);
  else if (n <= 128)
    backward<64, 2, 1024>(g, a, s);
  else if (n <= 256)
    backward<64, 4, 512>(g, a, s);
  else if (n <= 512)
    backward<256, 2, 1024>(g, a, s);
  else
    backward<256, 4, 512>(g, a, s);
  if (hipGetLastError() != hipSuccess) return METALLLM_ATTN_E_LAUNCH;
  hipLaunchKernelGGL(rms_join_kernel, dim3((p->cols + 15) / 16), dim3(256), 0, s, (const float*)workspace, dgamma, g.blocks,
                     p->cols);
  return hipGetLastError() == hipSuccess ? METALLLM_ATTN_OK : METALLLM_ATTN_E_LAUNCH;
}

}  // extern "C"
