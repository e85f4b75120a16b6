// attn_window.hpp -- attention over a window of keys with a few first keys that stay visible
// (attn_window_*.hip): what the kernels share, and their launch interface. Shapes arrive validated.
//
// Sequence b has lq query rows and lk keys. Query row i stands at position pos = lk - lq + i, and sees
// key j where j <= pos and (pos - j < window or j < sinks). Rows at a negative position see nothing.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_common.hpp"
#include "attn_launch.hpp"

namespace mla {

constexpr int kWinMaxSinks = 64;  // one key tile

struct WinShape {
  int B, TQ, TK, NH, NKV, G;  // G = NH / NKV query heads share a key head
  int window, sinks;          // window at most 2^30
  uint32_t q_row, k_row, v_row, o_row;  // elements from a token to the next
  size_t q_seq, k_seq, v_seq, o_seq;    // elements from a sequence to the next
  const int32_t* q_len;       // device [B], or NULL: TQ rows, TK keys each
  const int32_t* k_len;
  float scale;                // 1/sqrt(D)
};

struct WinFwdArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  float* l;  // [B, NH, TQ], or NULL
  WinShape s;
  float* part;  // single-token form: partial results of the splits (win_token_floats)
  int splits;
};

struct WinBwdArgs {
  const uint16_t* dO;
  const uint16_t* O;
  const float* l;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* dQ;
  uint16_t* dK;
  uint16_t* dV;
  WinShape s;
  float* Dsum;  // [B, NH, TQ] workspace, twice: -Dl (Dl = sum over d of dO O), l log2(e)
  float* part;  // workspace: partial dK, dV of the sink keys, or NULL where nothing is split (splits = 0)
  int splits;
  bool narrow;  // win_is_narrow
};

// A sequence's lengths, held inside the buffers whatever the device arrays say.
struct WinSeq {
  int lq, lk, off;  // off = lk - lq: position of query row 0
};
__device__ __forceinline__ WinSeq win_seq(const WinShape& s, int b) {
  int lq = s.q_len ? s.q_len[b] : s.TQ, lk = s.k_len ? s.k_len[b] : s.TK;
  lq = min(max(lq, 0), s.TQ);
  lk = min(max(lk, 0), s.TK);
  return WinSeq{__builtin_amdgcn_readfirstlane(lq), __builtin_amdgcn_readfirstlane(lk),
                __builtin_amdgcn_readfirstlane(lk - lq)};
}

// The 64-key tiles that query rows i0 .. i1 of a sequence (i1 < lq) visit, in order: the sink tile 0
// alone where the window begins behind it, then the window's tiles t0 .. t1.
struct WinTiles {
  int t0, sink, n;  // first window tile, 1 where tile 0 comes before it, number of tiles
  int lo, hi;       // rows of k and v that window tiles may read: every key outside is hidden from all
  __device__ __forceinline__ int tile(int j) const { return j < sink ? 0 : t0 + j - sink; }
};
__device__ __forceinline__ WinTiles win_tiles(const WinShape& s, const WinSeq& q, int i0, int i1) {
  WinTiles w{0, 0, 0, 0, 0};
  const int last = q.off + i1;  // position of the last row
  if (last < 0) return w;
  const int first = max(0, q.off + i0 - s.window + 1);  // first key of the rows' windows
  w.t0 = first / kTile;
  w.sink = s.sinks > 0 && w.t0 > 0 ? 1 : 0;
  w.n = last / kTile - w.t0 + 1 + w.sink;
  w.lo = s.sinks > 0 && w.t0 == 0 ? 0 : first;
  w.hi = last;
  return w;
}

__device__ __forceinline__ int clamp_row(int r, int lo, int hi) { return min(max(r, lo), hi); }

// A wave's 32 rows x D outputs, held as accumulators (lane: row l32, values 32 dt + 8g + 4h + 0..3 in registers
// 4g .. of acc[dt]) -> bf16 rows in memory, through LDS: a lane stores 16 bytes of a row, 64 lanes whole
// rows. Straight from the registers it is twice the instructions, each over 32 rows.
// lds: kRowsOut<D> bytes of the wave's own; live(r): whether row r is written.
template <int D>
constexpr int kRowsOut = 32 * (2 * D + 16);
template <int D, class Acc, class Live>
__device__ __forceinline__ void store_rows(uint32_t lds, int lane, const Acc* acc, float scale, uint16_t* out, uint32_t row,
                                           Live live) {
  typedef uint32_t v2 __attribute__((ext_vector_type(2)));
  typedef uint32_t v4 __attribute__((ext_vector_type(4)));
  constexpr uint32_t P = 2 * D + 16;
  const int h = lane >> 5, l32 = lane & 31;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *(__attribute__((address_space(3))) v2*)(uintptr_t)(lds + l32 * P + 64 * dt + 16 * g + 8 * h) =
          v2{pack_bf16(acc[dt][4 * g] * scale, acc[dt][4 * g + 1] * scale),
             pack_bf16(acc[dt][4 * g + 2] * scale, acc[dt][4 * g + 3] * scale)};
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    const int t = 64 * n + lane, r = t / (D / 8), c = t % (D / 8);
    const v4 x = *(const __attribute__((address_space(3))) v4*)(uintptr_t)(lds + r * P + 16 * c);
    if (live(r)) *(v4*)(out + (size_t)r * row + 8 * c) = x;
  }
}

// Whether query position `pos` sees key j.
__device__ __forceinline__ bool win_sees(const WinShape& s, int pos, int j) {
  return j <= pos && (pos - j < s.window || j < s.sinks);
}

// ---- host ----
// Which kernel a forward call runs. The one for few rows (attn_window_token.hip) takes tiles of kTokRows rows
// (query row, head of the group) and splits their keys over the chip; its time is reading the keys once
// for each tile: units * keys * 4 D bytes at about 6 TB/s. The other (attn_window_fwd.hip) takes blocks of
// 128 rows of a head, each of which runs along its keys by itself, about 1 us to 64 of them at any
// number of blocks that run at once. They meet near units * D = 24576. us, few rows' kernel and the other, at
// (B, TQ, TK, NH, NKV, D), all keys visible:
//   (1, 32, 16384, 8, 8, 128)    units 16    24   266      (1, 128, 8192, 12, 12, 64)   units 96    44   110
//   (1, 64, 16384, 32, 8, 128)         128   96   271      (1, 512, 8192, 12, 12, 64)         384   92   110
//   (4, 32, 4096, 32, 8, 128)          256   83    71      (1, 256, 256, 12, 12, 64)          192  5.6   8.0
// Up to kTokMost rows of a key head the other one would leave half of its block or more empty: 47 and 77 at
// (16, 4, 4096, 32, 4, 128), 81 and 77 at (16, 8, ..), 43 and 62 at (16, 8, 4096, 32, 4, 64).
constexpr int kTokRows = 16;
constexpr int kTokMost = 64;
constexpr int64_t kTokUnitsD = 24576;
inline int64_t win_token_units(const WinShape& s) {
  return (int64_t)s.B * s.NKV * (((int64_t)s.TQ * s.G + kTokRows - 1) / kTokRows);
}
inline bool win_is_token(const WinShape& s, int D) {
  return ((int64_t)s.TQ * s.G <= kTokMost && s.TQ <= kTokRows) || win_token_units(s) * D <= kTokUnitsD;
}
int win_token_splits(const WinShape& s);
inline size_t win_token_floats(const WinShape& s, int D, int splits) {
  const size_t tiles = ((size_t)s.TQ * s.G + kTokRows - 1) / kTokRows;
  return splits > 1 ? (size_t)s.B * s.NKV * tiles * splits * kTokRows * (D + 2) : 0;
}
// Parts that the query tiles (of all heads of a group) beyond the windows of the sink keys' block are dealt to
// (0: there are none): two tiles for each wave of a workgroup, so that they fill the gaps that the key blocks
// leave, and no more than the chip can run of them, since each keeps its sums in the workspace.
inline int win_sink_splits(const WinShape& s) {
  const int64_t far = (int64_t)s.TK - (kBwdBlockN - 1) - s.window;  // rows that see the sinks alone of block 0
  if (s.sinks == 0 || far <= 0) return 0;
  const int64_t n = (s.G * ((far + kTile - 1) / kTile) + 7) / 8, groups = (int64_t)s.B * s.NKV;
  const int64_t most = 4096 / groups < 8 ? 8 : 4096 / groups < 128 ? 4096 / groups : 128;
  return (int)(n < most ? n : most);
}
// Backward with key blocks for a quarter of the CUs or fewer and four query tiles or more to each: blocks of 32
// keys, whose waves take tiles each by itself and join their sums in LDS. Whole backward, us, with blocks of 32
// and of 128, at (B, T, NH, NKV, D), every key visible: (1, 4096, 8, 2, 128) 280, 458; (1, 521, 12, 3, 128) 58, 82;
// (2, 1024, 12, 4, 128) 75, 104; two tiles, (1, 100, 4, 4, 64), 20.5, 19.2. Not with far rows of sinks, which block 0
// would take alone: (1, 4096, 4, 2, 64), window 256, 74, 37.
inline bool win_is_narrow(const WinShape& s) {
  const int64_t blocks = (int64_t)s.B * s.NKV * ((s.TK + kBwdBlockN - 1) / kBwdBlockN);
  const int64_t rows = s.TQ < (int64_t)s.window + kBwdBlockN - 1 ? s.TQ : (int64_t)s.window + kBwdBlockN - 1;
  return blocks <= kCus / 4 && s.G * ((rows + kTile - 1) / kTile) >= 4 && win_sink_splits(s) == 0;
}
inline size_t win_sink_floats(const WinShape& s, int D, int splits) {  // [group][part][dK, dV][sink][D]
  return splits ? (size_t)s.B * s.NKV * (splits + 1) * 2 * s.sinks * D : 0;
}
// Work items of a launch are counted in 32 bits: whether every grid of a call, in threads, fits.
inline bool win_grids_fit(const WinShape& s, int D) {
  const int64_t most = 1ll << 24, heads = (int64_t)s.B * s.NH, groups = (int64_t)s.B * s.NKV;
  const int64_t qb = (s.TQ + kFwdBlockM - 1) / kFwdBlockM, kb = (s.TK + kBwdBlockN - 1) / kBwdBlockN;
  return heads < most / 4 && heads * qb < most && groups * (kb + 128) < most && groups * s.sinks * D < most * 64;
}

hipError_t launch_window_forward(const WinFwdArgs& a, int D, hipStream_t s);
hipError_t launch_window_token(const WinFwdArgs& a, int D, hipStream_t s);
hipError_t launch_window_backward(const WinBwdArgs& a, int D, hipStream_t s);

}  // namespace mla
