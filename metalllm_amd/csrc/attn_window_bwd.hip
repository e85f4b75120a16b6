// attn_window_bwd.hip -- windowAttentionBackward on gfx950.
//
// With s = q.k/sqrt(D), p = exp(s - l) over the visible keys (l the forward's logsumexp), Dl = sum_d dO.O,
// dP = dO.v and dS = p (dP - Dl):  dV = P^T.dO,  dK = dS^T.q/sqrt(D),  dQ = dS.k/sqrt(D).
// Products accumulate in fp32 over all tiles and are rounded once; p and dS are rounded to bf16, the type of
// the matrix cores' operands (half a step of 2^-8 each, as of the outputs; FINE: dS in two such parts). No
// atomics: every output has one owner, and the sum over the query heads of a key head runs in the owner, so
// results repeat bit for bit.
//
// Two kernels, then a small one where there are sinks:
//   win_dq_kernel    query owner: 4 waves x 32 rows of a head, over the key tiles that they see
//                    (attn_window_fwd.hip's order). Also writes Dl and l log2(e) of its rows for the next.
//   win_dkdv_kernel  key owner: 4 waves x 32 keys of a key head, over the query tiles that see them, head
//                    by head of the group. The sinks of block 0 are seen by every later row, so the query
//                    tiles beyond the block's windows are dealt to workgroups of their own, whose waves take
//                    tiles by themselves for the sums of the sink keys, in fp32.
//   win_sink_kernel  dK, dV of the sink keys from those parts, in order.
// A tile that is seen in part is masked by one unsigned compare per score; in the key owner the
// compare's limit belongs to the lane's key and covers window, sinks and the sequence's end. There the
// products of dP begin at -Dl, read from LDS where the accumulators have it, which saves a subtraction per
// score. (In the query owner Dl is the lane's, and 16 registers of it cost more: 135 us against 119 at D = 128.)
//
// Bound: instruction issue and, with a full chip, power. A wave's tile of 64 x 32 scores is 1024 cycles of matrix core
// at D = 64 and 2048 at D = 128 in the key owner, 768 and 1536 in the query owner. The key owner at D = 128 keeps 512
// registers (its sums alone are 128), so one wave per SIMD, which hides nothing of another's: 409 instructions to
// 64 products. Measured, each alone: (B, T, NH, NKV, D) = (8, 2048, 12, 12, 64), window 512: 69 and 73 us,
// 490 and 620 TFLOP/s of visible scores; (2, 4096, 16, 4, 128), window 1024: 114 and 144 us, 790 and 835 TFLOP/s. The
// sinks' last sums: 5 us.
// Tried without gain: reads further ahead (4% slower), other paddings of the tiles (a quarter of the LDS cycles are
// conflicts, but LDS is busy 35% at most), the vector work of two tiles in stages.
#include "attn_common.hpp"
#include "attn_window.hpp"

namespace mla {

typedef __attribute__((address_space(3))) uint16_t lds_u16w;
__device__ __forceinline__ uint32_t lds_at(const void* p) { return (uint32_t)(uintptr_t)(const lds_u16w*)p; }
__device__ __forceinline__ u32x4 lds_b128_w(uint32_t a) {
  return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)a;
}
__device__ __forceinline__ f32x4 lds_f4_w(uint32_t a) {
  return *(const __attribute__((address_space(3))) f32x4*)(uintptr_t)a;
}
__device__ __forceinline__ u32x2 lds_tr_w(uint32_t a) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) i16x4*)(uintptr_t)a));
}
// Global -> LDS copy of 4 bytes per lane to m0 + 4 lane (untracked, as dma16)
__device__ __forceinline__ void dma4_v(const void* src, uint32_t m0) {
  asm volatile("global_load_lds_dword %0, off" ::"v"(src), "{m0}"(m0) : "memory");
}
// sum over 8 pairs of bf16 products, added to x
__device__ __forceinline__ float dot8(u32x4 a, u32x4 b, float x) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    x = fmaf(bf_lo(a[w]), bf_lo(b[w]), x);
    x = fmaf(bf_hi(a[w]), bf_hi(b[w]), x);
  }
  return x;
}

// Tiles of 64 rows of two tensors in LDS, padded: 16-byte row reads and transposing reads.
template <int D>
struct WbCfg {
  static constexpr int P = D == 128 ? D + 24 : D + 8;
  static constexpr int TBYTES = kTile * P * 2;
  static constexpr int SLOTS = P / 8;
  static constexpr int LPW = (SLOTS + 3) / 4;
  static constexpr int STAT = 2 * TBYTES;  // key owner: l log2(e) and Dl of the tile's rows
  static constexpr int STAGE = 2 * TBYTES + 512;
  static constexpr int KC = D / 16;
  static constexpr int DT = D / 32;
  // What a lane copies of a tile's rows: instruction n of the wave covers 16-byte slots 64 (wave + 4n) .. + 63 of
  // the padded tile; slot t is row t / SLOTS, chunk t % SLOTS, pad chunks repeating the row's last one. Part
  // n copies that of two tensors, whose rows are held in [lo, hi].
  struct Slots {
    int wave, row[LPW];
    uint32_t chunk[LPW];
    __device__ __forceinline__ Slots(int wave_, int lane) : wave(wave_) {
#pragma unroll
      for (int n = 0; n < LPW; ++n) {
        const int t = 64 * (wave + 4 * n) + lane;
        row[n] = t / SLOTS;
        chunk[n] = 16 * min(t % SLOTS, D / 8 - 1);
      }
    }
    __device__ __forceinline__ void copy(int n, int lo, int hi, const char* a, uint32_t a_row, const char* b, uint32_t b_row,
                                         uint32_t dst) const {
      if (wave + 4 * n < SLOTS) {
        const int r = clamp_row(row[n], lo, hi);
        dma16(__umul24(r, a_row) + chunk[n], a, dst + 1024 * (wave + 4 * n));
        dma16(__umul24(r, b_row) + chunk[n], b, dst + TBYTES + 1024 * (wave + 4 * n));
      }
    }
  };
};

// Most tiles of a query block whose rows' Dl is summed over the keys: up to here some row sees 128 keys or
// fewer. Relative error of dQ and dK with Dl from the rounded O, and summed: T = 44 2.8e-3 and 2.3e-3 (2.35e-3 is
// what rounding dS and the output leaves), T = 2048 with a window of 512 2.46e-3 and 2.38e-3.
constexpr int kExactTiles = 4;

__device__ __forceinline__ void pin(u32x4& a) { asm volatile("" : "+v"(a)); }

template <int V>
struct IntTag {
  static constexpr int value = V;
};

// FINE: a product more with what rounding to bf16 has left of dS, for calls of few rows, over which such errors
// do not average out: dQ and dK of up to 2176 rows were off by 1.5 times the rounding of the outputs alone, with
// it by 1.0 times. It takes 22 us instead of 18 at (B, T, NH, NKV, D) = (2, 68, 4, 2, 64), 43 instead of 37 at
// (1, 1000, 4, 4, 128), both captured; of longer loops it would take a third.
constexpr int kFineRows = 4096;  // of all heads
constexpr int kFineItems = 8;    // query tiles of a key block
// x - bf16(x); 0 where that is no number, so that an infinite x stays one
__device__ __forceinline__ float rest_bf16(float x) {
  const float d = x - round_bf16(x);
  return d - d == 0.0f ? d : 0.0f;
}

// ---- dQ: query owner ----

template <int D, bool FINE>
__global__ void __launch_bounds__(256, FINE ? 1 : D == 64 ? 3 : 2) win_dq_kernel(WinBwdArgs a) {
  using C = WbCfg<D>;
  constexpr int BM = kDqBlockM;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * C::TBYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  const WinShape& s = a.s;
  const int nqb = (s.TQ + BM - 1) / BM;
  int group, blk;
  decode_workgroup(blockIdx.x, s.B * s.NKV, nqb * s.G, true, kBwdDispatchRound, group, blk);
  const int b = group / s.NKV, kvh = group - b * s.NKV;
  const int qb = blk / s.G, head = kvh * s.G + (blk - qb * s.G);
  const WinSeq sq = win_seq(s, b);
  const int i0 = qb * BM;
  if (i0 >= sq.lq) return;
  const int i1 = min(i0 + BM, sq.lq) - 1;
  const WinTiles wt = win_tiles(s, sq, i0, i1);
  const int i = i0 + 32 * wave + l32, ic = min(i, i1);
  const bool row_ok = i <= i1;
  const int pos = sq.off + i;
  uint16_t* dQg = a.dQ + b * s.q_seq + (size_t)(i0 + 32 * wave) * s.q_row + head * D;  // the wave's rows
  const size_t stat = ((size_t)b * s.NH + head) * s.TQ + ic, stats = (size_t)s.B * s.NH * s.TQ;

  // Q^T and dO^T as B operands: lane holds the row, d = 16c + 8h .. +7. Dl from dO and the rounded O: half a
  // step of O's values, which for rows of many keys are small against dP.
  u32x4 Qr[C::KC], Gr[C::KC];
  const uint16_t* Qg = a.q + b * s.q_seq + (size_t)ic * s.q_row + head * D + 8 * h;
  const size_t o_at = b * s.o_seq + (size_t)ic * s.o_row + head * D + 8 * h;
  float dl = 0.0f;
#pragma unroll
  for (int c = 0; c < C::KC; ++c) {
    Qr[c] = *(const u32x4*)(Qg + 16 * c);
    Gr[c] = *(const u32x4*)(a.dO + o_at + 16 * c);
    dl = dot8(Gr[c], *(const u32x4*)(a.O + o_at + 16 * c), dl);
  }
  dl = sum_halves(dl);
  const float l2 = a.l[stat] * kLog2e;
  const float sl = s.scale * kLog2e;

  const char* Kg = (const char*)(a.k + b * s.k_seq + kvh * D);
  const char* Vg = (const char*)(a.v + b * s.v_seq + kvh * D);
  const uint32_t krs = 2 * s.k_row, vrs = 2 * s.v_row;
  // Copies of the tile aimed at, in C::LPW parts that a step issues among its products (attn_window_fwd.hip)
  const typename C::Slots cp(wave, lane);
  const uint32_t smem_a = lds_at(smem);
  const char *ks = Kg + (size_t)wt.tile(0) * kTile * krs, *vs = Vg + (size_t)wt.tile(0) * kTile * vrs;
  int lo = 0, hi = 0;
  uint32_t dst = 0;
  auto aim = [&](int j) {
    const int kt = wt.tile(j);
    if (j > 0) {
      const int64_t rows = (int64_t)kTile * (kt - wt.tile(j - 1));
      ks += rows * krs;
      vs += rows * vrs;
    }
    lo = j < wt.sink ? 0 : max(wt.lo - kt * kTile, 0);
    hi = j < wt.sink ? s.sinks - 1 : min(wt.hi - kt * kTile, kTile - 1);
    dst = smem_a + (j & 1) * 2 * C::TBYTES;
  };
  auto part = [&](int n) __attribute__((always_inline)) { cp.copy(n, lo, hi, ks, krs, vs, vrs, dst); };
  const uint32_t row_rd = 2 * (l32 * C::P + 8 * h);
  const int g16 = lane >> 4, s16 = lane & 15;
  const uint32_t tr_rd = 2 * ((4 * h + (s16 >> 2)) * C::P + 16 * (g16 & 1) + 4 * (s16 & 3));

  f32x16 dQa[C::DT];
#pragma unroll
  for (int t = 0; t < C::DT; ++t) dQa[t] = zero16();

  // One key tile: the products in order, one per slot: S and dP of keys 0-31 in turn, of keys 32-63, then
  // dQ by 16-key chunk; pair p of half t goes through its three stages (exponent; p and dP - Dl; dS packed)
  // from slot enter(t, p) on, between products that do not need it. A dQ product comes after the slot
  // that packs its chunk's last pair.
  constexpr int PPS = D == 64 ? 2 : 1;
  struct Sched {
    static constexpr int enter(int t, int p) { return (t ? 4 * C::KC : 2 * C::KC) + p / PPS; }
    static constexpr int dq_slot(int k) {
      int slot = 4 * C::KC - 1;
      for (int j = 0; j <= k; ++j) {
        const int c = j / C::DT, ready = enter(c / 2, 4 * (c % 2) + 3) + 2;
        slot = (slot + 1 > ready + 1) ? slot + 1 : ready + 1;
      }
      return slot;
    }
    static constexpr int product_at(int i) {
      if (i < 4 * C::KC) return i;
      for (int k = 0; k < 4 * C::DT; ++k)
        if (dq_slot(k) == i) return 4 * C::KC + k;
      return -1;
    }
  };
  constexpr int NM = 4 * C::KC + 4 * C::DT, NV = Sched::dq_slot(4 * C::DT - 1) + 1;
  auto tile = [&](int j, auto mask_tag, auto part) __attribute__((always_inline)) {
    constexpr int MASK = decltype(mask_tag)::value;
    const uint32_t kb = smem_a + (j & 1) * 2 * C::TBYTES, vb = kb + C::TBYTES;
    int dq = 0, sq_ = 0;
    if (MASK) {
      const int kt = wt.tile(j);
      dq = pos - kt * kTile - 4 * h;
      asm volatile("" : "+v"(dq));
      if (MASK == 2) sq_ = min(s.sinks - kt * kTile - 4 * h, dq + 1);
    }
    auto seen = [&](int off) {
      return (uint32_t)(dq - off) < (uint32_t)s.window || (MASK == 2 && off < sq_);
    };
    f32x16 x0 = zero16(), x1 = zero16(), y0 = zero16(), y1 = zero16();
    uint32_t dS[16], low[16];
    constexpr int RING = 6;
    auto ahead = [](int n) { return n < 2 * C::KC || D == 64 ? 5 : 3; };
    u32x4 ring[RING];
    auto op_of = [&](int n) -> u32x4 {
      if (n < 4 * C::KC) {
        const int t = n / (2 * C::KC), isdp = n & 1, c = (n % (2 * C::KC)) >> 1;
        return lds_b128_w((isdp ? vb : kb) + row_rd + 2 * (32 * t * C::P + 16 * c));
      }
      const int k = n - 4 * C::KC, dt = k % C::DT, c = k / C::DT;
      const u32x2 lo = lds_tr_w(kb + tr_rd + 2 * (16 * c * C::P + 32 * dt));
      const u32x2 hi = lds_tr_w(kb + tr_rd + 2 * ((16 * c + 8) * C::P + 32 * dt));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
#pragma unroll
    for (int n = 0; n <= ahead(0); ++n) ring[n] = op_of(n);
    float ta[16], tb[16], ya[16], yb[16];
    auto stage = [&](int t, int p, int st) {
      f32x16& x = t ? x1 : x0;
      f32x16& y = t ? y1 : y0;
      const int u = 8 * t + p, r = 2 * p;
      if (st == 0) {
        ta[u] = fmaf(x[r], sl, -l2);
        tb[u] = fmaf(x[r + 1], sl, -l2);
        pin(ta[u], tb[u]);
      } else if (st == 1) {
        ta[u] = exp2_hw(ta[u]);
        tb[u] = exp2_hw(tb[u]);
        ya[u] = y[r] - dl;
        yb[u] = y[r + 1] - dl;
        pin(ta[u], tb[u]);
        pin(ya[u], yb[u]);
      } else {
        float d0 = ta[u] * ya[u], d1 = tb[u] * yb[u];
        if (MASK) {
          const int off = 32 * t + 8 * (r >> 2) + (r & 3);
          d0 = seen(off) ? d0 : 0.0f;
          d1 = seen(off + 1) ? d1 : 0.0f;
        }
        uint32_t pk = pack_bf16(d0, d1);
        pin(pk);
        dS[u] = pk;
        if (FINE) low[u] = pack_bf16(rest_bf16(d0), rest_bf16(d1));
      }
    };
#pragma unroll
    for (int slot = 0; slot < NV; ++slot) {
      if ((slot & 1) && slot / 2 < C::LPW) part(slot / 2);
      const int n = Sched::product_at(slot);
      if (n >= 0) {
#pragma unroll
        for (int k = (n ? n - 1 + ahead(n - 1) : ahead(0)) + 1; k <= n + ahead(n) && k < NM; ++k)
          ring[k % RING] = op_of(k);
        const u32x4& op = ring[n % RING];
        if (n < 4 * C::KC) {
          const int t = n / (2 * C::KC), c = (n % (2 * C::KC)) >> 1;
          if (n & 1) {
            if (t) y1 = mfma(op, Gr[c], y1);
            else y0 = mfma(op, Gr[c], y0);
          } else {
            if (t) x1 = mfma(op, Qr[c], x1);
            else x0 = mfma(op, Qr[c], x0);
          }
        } else {
          const int k = n - 4 * C::KC, dt = k % C::DT, c = k / C::DT;
          dQa[dt] = mfma(op, u32x4{dS[4 * c], dS[4 * c + 1], dS[4 * c + 2], dS[4 * c + 3]}, dQa[dt]);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const int st = slot - Sched::enter(t, p);
          if (st >= 0 && st < 3) stage(t, p, st);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (FINE)
#pragma unroll
      for (int k = 0; k < 4 * C::DT; ++k) {
        const int dt = k % C::DT, c = k / C::DT;
        dQa[dt] = mfma(op_of(4 * C::KC + k), u32x4{low[4 * c], low[4 * c + 1], low[4 * c + 2], low[4 * c + 3]}, dQa[dt]);
      }
  };

  // The wave's rows [pw0, pw1] (positions) see tiles of the steps jv0 .. jv1 - 1 (and the sinks in step 0), and
  // those of jw0 .. jw1 - 1 whole: every row every key
  const int pw0 = sq.off + i0 + 32 * wave, pw1 = min(pw0 + 31, sq.off + i1);
  const int j_of = wt.sink - wt.t0;  // step of window tile kt: kt + j_of
  const bool active = i0 + 32 * wave <= i1 && pw1 >= 0;
  const int jv0 = active ? max(0, pw0 - s.window + 1) / kTile + j_of : wt.n, jv1 = active ? pw1 / kTile + j_of + 1 : 0;
  const int jw0 = (max(0, pw1 - s.window + 1) + kTile - 1) / kTile + j_of, jw1 = max(0, pw0 + 1) / kTile + j_of;
  const bool sinks = active && s.sinks > 0;

  // Rows of few keys: there the rounding of O is of the size of dP itself, so Dl = sum_j P_ij dP_ij, in a pass
  // over the tiles of its own (two of the three products again).
  if (wt.n <= kExactTiles) {
    dl = 0.0f;
    for (int j = 0; j < wt.n; ++j) {
      aim(j);
      for (int n = 0; n < C::LPW; ++n) part(n);
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      const uint32_t kb = smem_a + (j & 1) * 2 * C::TBYTES + row_rd;
      const int key0 = wt.tile(j) * kTile + 4 * h;
#pragma unroll 1
      for (int t = 0; t < 2 && ((j >= jv0 && j < jv1) || (j == 0 && sinks)); ++t) {
        f32x16 x = zero16(), y = zero16();
#pragma unroll
        for (int c = 0; c < C::KC; ++c) {
          x = mfma(lds_b128_w(kb + 2 * (32 * t * C::P + 16 * c)), Qr[c], x);
          y = mfma(lds_b128_w(kb + C::TBYTES + 2 * (32 * t * C::P + 16 * c)), Gr[c], y);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (win_sees(s, pos, key0 + 32 * t + 8 * (r >> 2) + (r & 3))) dl = fmaf(exp2_hw(fmaf(x[r], sl, -l2)), y[r], dl);
      }
      __syncthreads();
    }
    dl = sum_halves(dl);
    ks = Kg + (size_t)wt.tile(0) * kTile * krs, vs = Vg + (size_t)wt.tile(0) * kTile * vrs;
  }
  if (row_ok && h == 0) {
    a.Dsum[stat] = -dl;
    a.Dsum[stats + stat] = l2;
  }

  if (wt.n) {
    aim(0);
    for (int n = 0; n < C::LPW; ++n) part(n);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    int j = 0;
    // Step j copies tile j + 1 (the last one its own again, to where nothing reads: its parts need no branch)
    auto run = [&](auto tag) __attribute__((always_inline)) {
      if (j + 1 < wt.n)
        aim(j + 1);
      else
        dst = smem_a + ((j + 1) & 1) * 2 * C::TBYTES;
      if constexpr (decltype(tag)::value >= 0)
        tile(j, tag, part);
      else
        for (int n = 0; n < C::LPW; ++n) part(n);
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      ++j;
    };
    if (sinks) run(IntTag<2>());
    while (j < wt.n) {
      while (j < wt.n && (j < jv0 || j >= jv1)) run(IntTag<-1>());
      while (j < jv1 && (j < jw0 || j >= jw1)) run(IntTag<1>());
      while (j < jw1 && j >= jw0 && j < jv1) run(IntTag<0>());
    }
  }

  // a hidden key whose row is not finite has added 0 * NaN to the rows of its tile: such rows are summed
  // again over the keys that they see
  float bad = 0.0f;
#pragma unroll
  for (int t = 0; t < C::DT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad = fmaf(dQa[t][r], 0.0f, bad);
  const bool again = row_ok && (pos < 0 || (dl - dl == 0.0f && l2 - l2 == 0.0f)) && sum_halves(bad) != 0.0f;
  if (__any(again)) {
    if (again) {
#pragma unroll
      for (int t = 0; t < C::DT; ++t) dQa[t] = zero16();
      const int first = max(0, pos - s.window + 1), ns = min(s.sinks, first);
      const int count = pos < 0 ? 0 : ns + pos + 1 - first;
      for (int t = 0; t < count; ++t) {
        const int key = t < ns ? t : first + t - ns;
        const uint16_t* kr = (const uint16_t*)(Kg + (size_t)key * krs);
        const uint16_t* vr = (const uint16_t*)(Vg + (size_t)key * vrs);
        float x = 0.0f, y = 0.0f;
#pragma unroll
        for (int c = 0; c < C::KC; ++c) {
          pin(Qr[c]);  // (or the unpacked values are kept over the loop)
          pin(Gr[c]);
          x = dot8(*(const u32x4*)(kr + 16 * c + 8 * h), Qr[c], x);
          y = dot8(*(const u32x4*)(vr + 16 * c + 8 * h), Gr[c], y);
        }
        x = sum_halves(x);
        y = sum_halves(y);
        const float d = round_bf16(exp2_hw(fmaf(x, sl, -l2)) * (y - dl));
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const u32x2 kk = *(const u32x2*)(kr + 32 * dt + 8 * g + 4 * h);
            dQa[dt][4 * g] = fmaf(d, bf_lo(kk[0]), dQa[dt][4 * g]);
            dQa[dt][4 * g + 1] = fmaf(d, bf_hi(kk[0]), dQa[dt][4 * g + 1]);
            dQa[dt][4 * g + 2] = fmaf(d, bf_lo(kk[1]), dQa[dt][4 * g + 2]);
            dQa[dt][4 * g + 3] = fmaf(d, bf_hi(kk[1]), dQa[dt][4 * g + 3]);
          }
      }
    }
  }
  // (every wave is past its last tile)
  const int rows = i1 - i0 - 32 * wave;
  store_rows<D>(smem_a + wave * kRowsOut<D>, lane, dQa, s.scale, dQg, s.q_row, [&](int r) { return r <= rows; });
}

// ---- dK, dV: key owner ----

// The part of a wave: 32 keys of a key head, their K and V rows as B operands, dK^T and dV^T in fp32 (chain
// n < DT: dV of d tile n, else dK of d tile n - DT), and a step over 64 query rows staged in LDS.
template <int D>
struct WinKeyWave {
  using C = WbCfg<D>;
  static constexpr int NS = 4 * C::KC + 8 * C::DT;  // slots of a step
  static constexpr bool PRIME = D == 128;           // a step's last slots read the next one's first operands
  static constexpr int RING = PRIME ? 8 : 5;
  static_assert(!PRIME || NS % RING == 0, "an operand keeps its place in the ring");
  int h;
  float sl;
  uint32_t row_rd, tr_rd, st_rd;
  u32x4 ring[RING];  // operands, RING - 1 slots ahead
  f32x16 first;      // -Dl of rows 0-31 of the next step
  u32x4 Kr[C::KC], Vr[C::KC];
  f32x16 st[2 * C::DT];

  __device__ __forceinline__ void init(int lane, float scale) {
    h = lane >> 5;
    sl = scale * kLog2e;
    const int l32 = lane & 31, g16 = lane >> 4, s16 = lane & 15;
    row_rd = 2 * (l32 * C::P + 8 * h);
    tr_rd = 2 * ((4 * h + (s16 >> 2)) * C::P + 16 * (g16 & 1) + 4 * (s16 & 3));
    st_rd = 16 * h;
#pragma unroll
    for (int n = 0; n < 2 * C::DT; ++n) st[n] = zero16();
  }

  // S and dP operand i of the rows staged at stage_a (+ row_rd)
  __device__ __forceinline__ u32x4 row_operand(uint32_t row_a, int i) const {
    const int t = i / (2 * C::KC), c = (i % (2 * C::KC)) >> 1;
    return lds_b128_w(row_a + ((i & 1) ? C::TBYTES : 0) + 2 * (32 * t * C::P + 16 * c));
  }
  // -Dl of rows 32t .. 32t + 31 where the accumulators of dP have them
  __device__ __forceinline__ void minus_dl(f32x16& y, uint32_t stat_a, int t) const {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v = lds_f4_w(stat_a + 256 + 4 * (32 * t + 8 * g));
#pragma unroll
      for (int r = 0; r < 4; ++r) y[4 * g + r] = v[r];
    }
  }
  __device__ __forceinline__ void prime(uint32_t stage_a) {
#pragma unroll
    for (int k = 0; k < RING - 1; ++k) ring[k] = row_operand(stage_a + row_rd, k);
    minus_dl(first, stage_a + C::STAT + st_rd, 0);
  }

  // Query rows staged at LDS byte address stage_a; MASK: row r of the tile (position p0 + r) sees the lane's
  // key where (uint)(p0 + r - key) < lim; d0 = p0 + 4h - key. Slots (one product each):
  //   [0, 2KC) S and dP of rows 0-31 in turn, [2KC, 4KC) of rows 32-63, then dV and dK, 16 rows at a time over
  //   the d tiles: two products that follow each other never add to the same sum, since the second would
  //   wait for the first to leave the matrix core
  // Beside them p, then dS, of rows 0-31 from slot 2KC, of rows 32-63 from slot 4KC.
  // part(0 .. NPART): copies of the next rows, issued among the products.
  // FINE: with what rounding has left of dS, after the other products.
  template <bool MASK, bool FINE, int NPART, class Part>
  __device__ __forceinline__ void step(uint32_t stage_a, uint32_t next_a, int d0, uint32_t lim, Part part) {
    constexpr int PPS = 8 / C::KC;
    uint32_t row_a = stage_a + row_rd, tr_a = stage_a + tr_rd, stat_a = stage_a + C::STAT + st_rd;
    uint32_t next_row_a = next_a + row_rd, next_stat_a = next_a + C::STAT + st_rd;
    pin(row_a);
    pin(tr_a);
    pin(stat_a);
    if (PRIME) {
      pin(next_row_a);
      pin(next_stat_a);
    }
    if (MASK) asm volatile("" : "+v"(d0));
    if (!PRIME) prime(stage_a);
    f32x16 x0 = zero16(), x1 = zero16(), y0 = first, y1;  // y: dP - Dl
    uint32_t Pp[16], dS[16], low[16];
    auto operand = [&](int i) -> u32x4 {
      if (i >= NS) return row_operand(next_row_a, i - NS);
      if (i < 4 * C::KC) return row_operand(row_a, i);
      const int k = i - 4 * C::KC, j = k / C::DT % 4, dt = k % C::DT;
      const uint32_t src = tr_a + (k >= 4 * C::DT ? 0 : C::TBYTES) + 2 * (16 * j * C::P + 32 * dt);
      const u32x2 lo = lds_tr_w(src), hi = lds_tr_w(src + 2 * 8 * C::P);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    // vector work in slot i: kind 1 = p, 2 = dS of pairs u0 .. of half t; PPS pairs to a slot
    struct Work {
      int kind, t, u0, cnt;
    };
    auto work = [&](int i) -> Work {
      if (i < 2 * C::KC || i >= 6 * C::KC) return {0, 0, 0, 0};
      const int t = i >= 4 * C::KC, n = (i - (t ? 4 : 2) * C::KC) * PPS;
      return n < 8 ? Work{1, t, n, PPS} : Work{2, t, n - 8, PPS};
    };
    static_assert(C::KC == 2 * C::DT, "slots of a half's vector work");
    // l log2(e) of pairs u and u + 1 (u even) of half t
    auto stats = [&](int t, int u) { return lds_f4_w(stat_a + 4 * (32 * t + 4 * u)); };
    auto seen = [&](int t, int r) { return (uint32_t)(d0 + 32 * t + 8 * (r >> 2) + (r & 3)) < lim; };
    auto p_pair = [&](f32x16& x, int t, int u, float l0, float l1) {
      const int r = 2 * u;
      float p0 = x[r], p1 = x[r + 1];
      if (MASK) {  // p = 0
        p0 = seen(t, r) ? p0 : -INFINITY;
        p1 = seen(t, r + 1) ? p1 : -INFINITY;
      }
      p0 = exp2_hw(fmaf(p0, sl, -l0));
      p1 = exp2_hw(fmaf(p1, sl, -l1));
      pin(p0, p1);
      x[r] = p0;
      x[r + 1] = p1;
      uint32_t pk = pack_bf16(p0, p1);
      pin(pk);
      Pp[8 * t + u] = pk;
    };
    auto ds_pair = [&](const f32x16& x, const f32x16& y, int t, int u) {
      const int r = 2 * u;
      const float d0 = x[r] * y[r], d1 = x[r + 1] * y[r + 1];
      uint32_t pk = pack_bf16(d0, d1);
      pin(pk);
      dS[8 * t + u] = pk;
      if (FINE) low[8 * t + u] = pack_bf16(rest_bf16(d0), rest_bf16(d1));
    };
    constexpr int SA = 3;
    f32x4 sring[4];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if ((i & 1) && i / 2 < NPART) part(i / 2);
      if (PRIME || i + RING - 1 < NS) ring[(i + RING - 1) % RING] = operand(i + RING - 1);
      if (const Work w = work(i + SA); w.kind == 1 && w.u0 % 2 == 0) sring[w.u0 / 2] = stats(w.t, w.u0);
      if (i == C::KC) minus_dl(y1, stat_a, 1);
      if (PRIME && i == NS - RING) minus_dl(first, next_stat_a, 0);
      const u32x4& op = ring[i % RING];
      if (i < 4 * C::KC) {
        const int t = i / (2 * C::KC), c = (i % (2 * C::KC)) >> 1;
        if (i & 1) {
          if (t) y1 = mfma(op, Vr[c], y1);
          else y0 = mfma(op, Vr[c], y0);
        } else {
          if (t) x1 = mfma(op, Kr[c], x1);
          else x0 = mfma(op, Kr[c], x0);
        }
      } else {
        const int k = i - 4 * C::KC, j = k / C::DT % 4, n = k % C::DT + (k >= 4 * C::DT ? C::DT : 0);
        const uint32_t* src = n >= C::DT ? dS : Pp;
        st[n] = mfma(op, u32x4{src[4 * j], src[4 * j + 1], src[4 * j + 2], src[4 * j + 3]}, st[n]);
      }
      const Work w = work(i);
      if (w.cnt) {
#pragma unroll
        for (int u = w.u0; u < w.u0 + w.cnt; ++u) {
          if (w.kind == 1)
            p_pair(w.t ? x1 : x0, w.t, u, sring[u / 2][2 * (u % 2)], sring[u / 2][2 * (u % 2) + 1]);
          else
            ds_pair(w.t ? x1 : x0, w.t ? y1 : y0, w.t, u);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (FINE)
#pragma unroll
      for (int k = 0; k < 4 * C::DT; ++k) {
        const int j = k / C::DT, n = C::DT + k % C::DT;
        st[n] = mfma(operand(4 * C::KC + 4 * C::DT + k), u32x4{low[4 * j], low[4 * j + 1], low[4 * j + 2], low[4 * j + 3]},
                     st[n]);
      }
  }
};

template <int D, bool FINE>
__global__ void __launch_bounds__(256, D == 64 && !FINE ? 2 : 1) win_dkdv_kernel(WinBwdArgs a) {
  using C = WbCfg<D>;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * C::STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  const WinShape& s = a.s;
  const bool narrow = a.narrow;  // blocks of 32 keys
  const int BN = narrow ? 32 : kBwdBlockN;
  const int nkb = (s.TK + BN - 1) / BN;
  // the key blocks first, then (far) the parts of the rows that see block 0's sinks alone
  const int groups = s.B * s.NKV, near = groups * nkb;
  const bool far = (int)blockIdx.x >= near;
  int group, blk;
  if (far)
    decode_workgroup(blockIdx.x - near, groups, a.splits, false, kBwdDispatchRound, group, blk);
  else
    decode_workgroup(blockIdx.x, groups, nkb, false, kBwdDispatchRound, group, blk);
  const int b = group / s.NKV, kvh = group - b * s.NKV;
  const int kb = far ? 0 : blk;
  const WinSeq sq = win_seq(s, b);
  const int k0 = kb * BN;
  const bool split = kb == 0 && a.splits > 0;  // sink keys go through the workspace
  if (k0 >= sq.lk) return;                     // (the sink kernel reads nothing of such a sequence either)
  const int k1 = min(k0 + BN, sq.lk) - 1;

  // query rows [ilo, ihi] of each head, tiles [tlo, tlo + nt), and the items [f0, f1) of head * nt + tile
  int ilo = max(0, k0 - sq.off);
  int ihi = min(sq.lq - 1, min(k1 + s.window - 1, sq.lk - 1) - sq.off);
  int tlo = 0, nt = 0;
  if (narrow && k0 < s.sinks) ihi = sq.lq - 1;
  if (ilo <= ihi) {
    tlo = ilo / kTile;
    nt = ihi / kTile - tlo + 1;
  }
  if (split) {
    const int tn = ihi >= ilo ? tlo + nt : 0;  // the first tile that only sink keys are seen from
    if (far) {
      ilo = tn * kTile;
      ihi = sq.lq - 1;
      tlo = tn;
      nt = max(0, (sq.lq + kTile - 1) / kTile - tn);
    } else if (nt) {
      ihi = min(sq.lq - 1, tn * kTile - 1);  // the rest of the last tile sees the sinks
    }
  }
  const int items = s.G * nt;
  const int f0 = far ? (int)((int64_t)items * blk / a.splits) : 0;
  const int f1 = far ? (int)((int64_t)items * (blk + 1) / a.splits) : items;

  // alone: a wave takes every fs-th item by itself, for 32 sinks (far) or the block's 32 keys (narrow)
  const bool alone = far || narrow;
  const int halves = far ? (s.sinks + 31) / 32 : 1, fs = alone ? 4 / halves : 1, fw = alone ? f0 + wave / halves : f0;
  const int kw0 = far ? 32 * (wave % halves) : narrow ? k0 : k0 + 32 * wave, kw1 = min(kw0 + 31, k1);
  const int key = kw0 + l32;
  const bool sink_key = key < s.sinks;
  const int most = sq.lk - key;  // rows of the sequence that stand at the key or behind it
  const uint32_t lim = (uint32_t)max(0, sink_key ? most : far ? 0 : min(s.window, most));
  const bool wave_on = kw0 <= k1;

  const char* Qg = (const char*)(a.q + b * s.q_seq + kvh * s.G * D);
  const char* Gg = (const char*)(a.dO + b * s.o_seq + kvh * s.G * D);
  const size_t stat0 = ((size_t)b * s.NH + kvh * s.G) * s.TQ, stats = (size_t)s.B * s.NH * s.TQ;
  const uint32_t qrs = 2 * s.q_row, grs = 2 * s.o_row;

  WinKeyWave<D> wv;
  wv.init(lane, s.scale);
  {
    const int kc = min(key, k1);  // rows past the end are read in bounds, never stored
    const uint16_t* kr = a.k + b * s.k_seq + (size_t)kc * s.k_row + kvh * D + 8 * h;
    const uint16_t* vr = a.v + b * s.v_seq + (size_t)kc * s.v_row + kvh * D + 8 * h;
#pragma unroll
    for (int c = 0; c < C::KC; ++c) {
      wv.Kr[c] = *(const u32x4*)(kr + 16 * c);
      wv.Vr[c] = *(const u32x4*)(vr + 16 * c);
    }
  }
  // How the tiles of a head see the wave's 32 keys: those of tv0 .. tv1 - 1 at all, of tw0 .. tw1 - 1 whole
  // (every row every key)
  const int tend = tlo + nt;
  const bool sinks = kw0 < s.sinks;
  int tv0 = max(tlo, (kw0 - sq.off) >> 6), tv1 = sinks ? tend : min(tend, ((kw0 + 30 + s.window - sq.off) >> 6) + 1);
  int tw0 = max(tv0, (kw1 - sq.off + kTile - 1) >> 6);
  int tw1 = min(((kw0 + s.window - kTile - sq.off) >> 6) + 1, sq.lq / kTile);
  if (!wave_on) tv1 = tv0;
  tw1 = min(tw1, tv1);
  if (tw0 >= tw1) tw0 = tw1 = tv1;

  if (alone) {
    const uint32_t st = lds_at(smem) + wave * C::STAGE;
    for (int f = fw; f < f1; f += fs) {
      const int g = f / nt, t = tlo + f - g * nt;
      const int lo = max(ilo - t * kTile, 0), hi = min(ihi - t * kTile, kTile - 1);
      const char* qs = Qg + (size_t)t * kTile * qrs + 2 * g * D;
      const char* gs = Gg + (size_t)t * kTile * grs + 2 * g * D;
      const float* sp = a.Dsum + stat0 + (size_t)g * s.TQ + t * kTile + clamp_row(lane, lo, hi);
#pragma unroll 1
      for (int w = 0; w < 4; ++w) {
        const typename C::Slots cp(w, lane);
#pragma unroll
        for (int n = 0; n < C::LPW; ++n) cp.copy(n, lo, hi, qs, qrs, gs, grs, st);
      }
      dma4_v(sp + stats, st + C::STAT);
      dma4_v(sp, st + C::STAT + 256);
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
      if (wv.PRIME) wv.prime(st);
      wv.template step<true, FINE, 0>(st, st, sq.off + t * kTile + 4 * h - key, lim, [](int) {});
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
    }
  } else if (f0 < f1) {
    const typename C::Slots cp(wave, lane);
    int f = f0, g = f0 / nt, t = tlo + f0 - g * nt;  // item f: query tile t of head g
    // the item to copy: its first rows, and the statistics of tile 0 of its head
    int fc = f, tc = t;
    const char* qs = Qg + (size_t)t * kTile * qrs + 2 * g * D;
    const char* gs = Gg + (size_t)t * kTile * grs + 2 * g * D;
    const float* sp = a.Dsum + stat0 + (size_t)g * s.TQ;
    // stages of item f, of those behind it, and of the item to copy
    constexpr int AHEAD = wv.PRIME ? 2 : 1;
    uint32_t st = lds_at(smem), next = st + C::STAGE, dst = st;
    auto part = [&](int n) __attribute__((always_inline)) {
      const int lo = max(ilo - tc * kTile, 0), hi = min(ihi - tc * kTile, kTile - 1);
      if (n < C::LPW) {
        cp.copy(n, lo, hi, qs, qrs, gs, grs, dst);
      } else if (wave == 0) {
        const float* p = sp + tc * kTile + clamp_row(lane, lo, hi);
        dma4_v(p + stats, dst + C::STAT);
        dma4_v(p, dst + C::STAT + 256);
      }
    };
    constexpr int PARTS = C::LPW + 1;
    // (the last item again, to where nothing reads, when there is no other)
    auto aim = [&](uint32_t to) __attribute__((always_inline)) {
      if (fc + 1 < f1) {
        ++fc;
        ++tc;
        qs += (int64_t)kTile * qrs;
        gs += (int64_t)kTile * grs;
        if (tc == tend) {
          tc = tlo;
          qs += 2 * D - (int64_t)nt * kTile * qrs;
          gs += 2 * D - (int64_t)nt * kTile * grs;
          sp += s.TQ;
        }
      }
      dst = to;
    };
    // the wave's copies have arrived, then everyone's (operands that a step has read ahead are not waited for)
    auto arrive = [] {
      __builtin_amdgcn_s_waitcnt(0x0f70);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    for (int n = 0; n < PARTS; ++n) part(n);
    if (AHEAD == 2) {
      aim(next);
      for (int n = 0; n < PARTS; ++n) part(n);
    }
    arrive();
    if (AHEAD == 2) wv.prime(st);
    // item f + AHEAD is copied while `step` runs on item f
    auto item = [&](auto step) __attribute__((always_inline)) {
      const uint32_t free_a = AHEAD == 2 ? 3 * lds_at(smem) + 3 * C::STAGE - st - next : next;
      aim(free_a);
      step(st, next);
      arrive();
      const uint32_t was = st;
      st = next;
      next = AHEAD == 2 ? free_a : was;
      ++f;
      ++t;
    };
    auto idle = [&](uint32_t, uint32_t ahead) {
      for (int n = 0; n < PARTS; ++n) part(n);
      if (AHEAD == 2) wv.prime(ahead);
    };
    // loops of one form of the step each (a choice inside one loop costs a copy of the sums per tile); every
    // wave passes every item's barrier
    while (f < f1) {
      const int te = min(tend, t + f1 - f);  // this head's
      while (t < te) {
        while (t < te && (t < tv0 || t >= tv1)) item(idle);
        while (t < min(te, tv1) && (t < tw0 || t >= tw1))
          item([&](uint32_t at, uint32_t ahead) {
            wv.template step<true, FINE, PARTS>(at, ahead, sq.off + t * kTile + 4 * h - key, lim, part);
          });
        while (t < min(te, tw1) && t >= tw0)
          item([&](uint32_t at, uint32_t ahead) { wv.template step<false, FINE, PARTS>(at, ahead, 0, 0, part); });
      }
      t = tlo;
    }
  }

  if (!wave_on && !alone) return;
  // A row that does not see a key but shares its tile adds 0 * NaN to it where q or dO is not finite: such
  // keys are summed again over the rows that see them.
  float bad = 0.0f;
#pragma unroll
  for (int n = 0; n < 2 * C::DT; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad = fmaf(wv.st[n][r], 0.0f, bad);
  const bool again = key <= k1 && (!far || sink_key) && sum_halves(bad) != 0.0f;
  if (__any(again)) {
    if (again) {
#pragma unroll
      for (int n = 0; n < 2 * C::DT; ++n) wv.st[n] = zero16();
      bool lost = false;  // p is not a number: then no sum of the key is
      for (int f = fw; f < f1 && !lost; f += fs) {
        const int g = f / nt, t = tlo + f - g * nt;
        const int ra = max(ilo, t * kTile), rb = min(ihi, t * kTile + kTile - 1);
        for (int i = ra; i <= rb && !lost; ++i) {
          if ((uint32_t)(sq.off + i - key) >= lim) continue;
          const uint16_t* qr = (const uint16_t*)(Qg + (size_t)i * qrs) + g * D;
          const uint16_t* gr = (const uint16_t*)(Gg + (size_t)i * grs) + g * D;
          float x = 0.0f, y = 0.0f;
#pragma unroll
          for (int c = 0; c < C::KC; ++c) {
            pin(wv.Kr[c]);
            pin(wv.Vr[c]);
            x = dot8(*(const u32x4*)(qr + 16 * c + 8 * h), wv.Kr[c], x);
            y = dot8(*(const u32x4*)(gr + 16 * c + 8 * h), wv.Vr[c], y);
          }
          x = sum_halves(x);
          y = sum_halves(y);
          const float* sp = a.Dsum + stat0 + (size_t)g * s.TQ + i;
          const float p = exp2_hw(fmaf(x, wv.sl, -sp[stats]));
          lost = p != p;
          const float d = round_bf16(p * (y + sp[0])), pr = round_bf16(p);
#pragma unroll
          for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const u32x2 qq = *(const u32x2*)(qr + 32 * dt + 8 * u + 4 * h);
              const u32x2 gg = *(const u32x2*)(gr + 32 * dt + 8 * u + 4 * h);
              f32x16& v = wv.st[dt];
              f32x16& k = wv.st[C::DT + dt];
              v[4 * u] = fmaf(pr, bf_lo(gg[0]), v[4 * u]);
              v[4 * u + 1] = fmaf(pr, bf_hi(gg[0]), v[4 * u + 1]);
              v[4 * u + 2] = fmaf(pr, bf_lo(gg[1]), v[4 * u + 2]);
              v[4 * u + 3] = fmaf(pr, bf_hi(gg[1]), v[4 * u + 3]);
              k[4 * u] = fmaf(d, bf_lo(qq[0]), k[4 * u]);
              k[4 * u + 1] = fmaf(d, bf_hi(qq[0]), k[4 * u + 1]);
              k[4 * u + 2] = fmaf(d, bf_lo(qq[1]), k[4 * u + 2]);
              k[4 * u + 3] = fmaf(d, bf_hi(qq[1]), k[4 * u + 3]);
            }
        }
      }
    }
  }
  const uint32_t lds = lds_at(smem) + wave * kRowsOut<D>;  // (every wave is past its last item)
  if (!alone) {
    auto live = [&](int r) { return kw0 + r <= k1 && !(split && kw0 + r < s.sinks); };
    store_rows<D>(lds, lane, wv.st + C::DT, s.scale, a.dK + b * s.k_seq + (size_t)kw0 * s.k_row + kvh * D, s.k_row, live);
    store_rows<D>(lds, lane, wv.st, 1.0f, a.dV + b * s.v_seq + (size_t)kw0 * s.v_row + kvh * D, s.v_row, live);
  }
  if (!split && !narrow) return;
  // sums of the sinks, fp32 [dK, dV][sink][D]: part 0 the block's own rows, then the far parts; waves that took
  // items alone join their sums in LDS
  float* out = a.part + ((size_t)group * (a.splits + 1) + (far ? blk + 1 : 0)) * 2 * s.sinks * D;
  float* own = (float*)(smem + wave * C::STAGE);
  float *ko = alone ? own + l32 * 2 * D : out + key * D, *vo = alone ? ko + D : ko + s.sinks * D;
  static_assert(32 * 2 * D * 4 <= C::STAGE, "a wave's sums in its stage");
  if ((sink_key || narrow) && key <= k1)
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x16& v = wv.st[dt];
        const f32x16& k = wv.st[C::DT + dt];
        const int d0 = 32 * dt + 8 * u + 4 * h;
        *(f32x4*)(ko + d0) = f32x4{k[4 * u], k[4 * u + 1], k[4 * u + 2], k[4 * u + 3]};
        *(f32x4*)(vo + d0) = f32x4{v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]};
      }
  if (!alone) return;
  __syncthreads();
  for (int n = tid; n < (narrow ? k1 - k0 + 1 : min(s.sinks, sq.lk)) * (D / 2); n += 256) {
    const int j = n / (D / 2), c = 4 * (n % (D / 2));
    f32x4 sum = {0, 0, 0, 0};
    for (int w = j / 32; w < 4; w += halves) sum += *(const f32x4*)(smem + w * C::STAGE + 4 * ((j & 31) * 2 * D + c));
    if (!narrow) {
      *(f32x4*)(out + (c < D ? j * D + c : (s.sinks + j) * D + c - D)) = sum;
      continue;
    }
    if (c < D) sum *= s.scale;
    uint16_t* o = c < D ? a.dK + b * s.k_seq + (size_t)(k0 + j) * s.k_row + c
                        : a.dV + b * s.v_seq + (size_t)(k0 + j) * s.v_row + c - D;
    *(u32x2*)(o + kvh * D) = u32x2{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
  }
}

// dK, dV of the sink keys: a workgroup per (sequence, key head) and key; 8 threads to four columns, each with
// every 8th part, joined in order.
template <int D>
__global__ void __launch_bounds__(D * 4) win_sink_kernel(WinBwdArgs a) {
  __shared__ f32x4 sums[8][D / 2];
  const WinShape& s = a.s;
  const int group = blockIdx.x / s.sinks, key = blockIdx.x - group * s.sinks;
  const int b = group / s.NKV, kvh = group - b * s.NKV;
  if (key >= win_seq(s, b).lk) return;
  const int t = threadIdx.x % (D / 2), w = threadIdx.x / (D / 2), isv = t / (D / 4), c = 4 * (t % (D / 4));
  const size_t step = (size_t)2 * s.sinks * D;
  const float* in = a.part + (size_t)group * (a.splits + 1) * step + (size_t)isv * s.sinks * D + key * D + c;
  f32x4 sum = {0, 0, 0, 0};
#pragma unroll 4
  for (int v = w; v <= a.splits; v += 8) sum += *(const f32x4*)(in + v * step);
  sums[w][t] = sum;
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int v = 1; v < 8; ++v) sum += sums[v][t];
  if (!isv) sum *= s.scale;
  uint16_t* o = isv ? a.dV + b * s.v_seq + (size_t)key * s.v_row : a.dK + b * s.k_seq + (size_t)key * s.k_row;
  *(u32x2*)(o + kvh * D + c) = u32x2{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
}

template <int D, bool FINE>
hipError_t launch(const WinBwdArgs& a, hipStream_t s) {
  const WinShape& p = a.s;
  const unsigned groups = (unsigned)(p.B * p.NKV);
  const unsigned nq = groups * p.G * ((p.TQ + kDqBlockM - 1) / kDqBlockM);
  const unsigned nk = a.narrow ? groups * ((p.TK + 31) / 32) : groups * ((p.TK + kBwdBlockN - 1) / kBwdBlockN + a.splits);
  hipLaunchKernelGGL((win_dq_kernel<D, FINE>), dim3(nq), dim3(256), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((win_dkdv_kernel<D, FINE>), dim3(nk), dim3(256), 0, s, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.splits == 0) return e;
  hipLaunchKernelGGL(win_sink_kernel<D>, dim3(groups * p.sinks), dim3(D * 4), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_window_backward(const WinBwdArgs& a, int D, hipStream_t s) {
  const WinShape& p = a.s;
  const bool fine = (int64_t)p.B * p.NH * p.TQ <= kFineRows && p.G * ((p.TQ + kTile - 1) / kTile) <= kFineItems;
  if (D == 64) return fine ? launch<64, true>(a, s) : launch<64, false>(a, s);
  return fine ? launch<128, true>(a, s) : launch<128, false>(a, s);
}

}  // namespace mla
