// attn_window_fwd.hip -- windowAttentionForward on gfx950 for many query rows.
//
// Per (sequence, head, query row): s = q.k (fp32), running max m and sum l of exp2((s - m) c) with
// c = log2(e)/sqrt(D) over the visible keys, O = sum bf16(p) v in fp32; out = bf16(O/l),
// l_out = m/sqrt(D) + ln(l). The scores and the sums stay in fp32. p is rounded to bf16 because the
// matrix cores take bf16 operands: half a step of 2^-8 per weight, the size of out's own rounding.
//
// Work split: 4 waves x 32 query rows of one head per workgroup, three workgroups per CU at D = 64, two at
// D = 128 (what their registers leave). A wave computes
// S^T (keys x queries), so that a lane holds one query's scores: row statistics need one exchange between
// lane halves, and the packed p of a tile are the B operand of O^T += V^T.P^T as they lie. K and V tiles
// of 64 keys go global -> LDS by direct copies, two stages deep. Step j of the pipeline runs the softmax of
// tile j on the vector ALU between the matrix products of S of tile j + 1 and P.V of tile j - 1.
//
// Masks: a wave skips the tiles that none of its rows sees, and masks those that its rows see in part, before
// the step: a compare per score with the causal border or the window's end, and where a tile has both one
// unsigned compare, (uint)(pos - key) < window. The sinks add a compare in tile 0, which holds all of them
// and comes first.
//
// The reference point m moves only when a tile's max exceeds it by 2^8 in the exponent's base (l and O
// are fp32 and p keeps its relative precision under any reference point), so O is rarely rescaled.
//
// Keys that no row of the workgroup sees are never read (their rows are replaced by a visible one and
// masked). A hidden key whose value row is not finite would still add 0 * NaN to the rows that do not see
// it but share its tile: rows that end up not finite are summed again one visible key at a time.
//
// Bound: vector instructions. At D = 64 a wave issues about 240 of them to a tile, 32 exponentials among them, some
// 1400 cycles beside the 512 of its matrix products, and takes 1640 with two others on its SIMD; at D = 128 it is
// both, and with a full chip the power: VALU busy 48%, matrix cores 45%. Measured: (B, T, NH, D) = (2, 8192, 16,
// 128), window 2048: 278 us, 865 TFLOP/s of visible scores; (8, 2048, 12, 64), window 512: 58 us, 390 TFLOP/s. All
// keys visible: (4, 4096, 16, 128) 285 us, 965 TFLOP/s; (8, 2048, 12, 64) 81 us.
// Tried without gain: a third stage of LDS (spills at D = 64).
#include <type_traits>

#include "attn_common.hpp"
#include "attn_window.hpp"

namespace mla {

template <int D>
struct WfCfg {
  static constexpr int BM = kFwdBlockM;
  static constexpr int BN = kTile;
  static constexpr int KP = D + 8;       // K row pitch (elements): 16-byte row reads are conflict-free
  static constexpr int KSLOTS = KP / 8;  // 16-byte slots of a padded K row
  static constexpr int VSLOTS = D / 8;   // V rows are unpadded and XOR-swizzled
  static constexpr int KBYTES = BN * KP * 2;
  static constexpr int VBYTES = BN * D * 2;
  static constexpr int STAGE = KBYTES + VBYTES;
  static constexpr int KPW = (KSLOTS + 3) / 4;  // copy instructions of 1 KB per wave (max)
  static constexpr int VPW = (VSLOTS + 3) / 4;
  static constexpr int KC = D / 16;
  static constexpr int DT = D / 32;
};

// What a pipeline step does: S of the next tile, P.V of the previous one, the softmax of this one.
template <bool S_, bool PV_, bool SM_>
struct WfStep {
  static constexpr bool S = S_, PV = PV_, SM = SM_;
};

template <int D>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2) win_fwd_kernel(WinFwdArgs a) {
  using C = WfCfg<D>;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * C::STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  const WinShape& s = a.s;
  const int nqb = (s.TQ + C::BM - 1) / C::BM;
  // the blocks of all heads that share a key head follow each other on one XCD
  int group, blk;
  decode_workgroup(blockIdx.x, s.B * s.NKV, nqb * s.G, true, kFwdDispatchRound, group, blk);
  const int b = group / s.NKV, kvh = group - b * s.NKV;
  const int qb = blk / s.G, head = kvh * s.G + (blk - qb * s.G);
  const WinSeq sq = win_seq(s, b);
  const int i0 = qb * C::BM;
  if (i0 >= sq.lq) return;
  const int i1 = min(i0 + C::BM, sq.lq) - 1;
  const WinTiles wt = win_tiles(s, sq, i0, i1);
  const int i = i0 + 32 * wave + l32;  // this lane's query row
  const bool row_ok = i <= i1;
  const int pos = sq.off + i;
  uint16_t* Og = a.out + b * s.o_seq + (size_t)(i0 + 32 * wave) * s.o_row + head * D;  // the wave's rows
  float* lg = a.l ? a.l + ((size_t)b * s.NH + head) * s.TQ : nullptr;

  if (wt.n == 0) {  // every row stands before the first key
    if (row_ok) {
#pragma unroll
      for (int c = 0; c < D / 16; ++c) *(u32x4*)(Og + (size_t)l32 * s.o_row + 16 * c + 8 * h) = u32x4{0, 0, 0, 0};
      if (lg && h == 0) lg[i] = -INFINITY;
    }
    return;
  }

  const char* Kg = (const char*)(a.k + b * s.k_seq + kvh * D);
  const char* Vg = (const char*)(a.v + b * s.v_seq + kvh * D);
  const uint32_t krs = 2 * s.k_row, vrs = 2 * s.v_row;

  // Q^T as B operands: lane holds row i, d = 16c + 8h .. +7
  u32x4 Qr[C::KC];
  const uint16_t* Qg = a.q + b * s.q_seq + (size_t)min(i, i1) * s.q_row + head * D;
#pragma unroll
  for (int c = 0; c < C::KC; ++c) Qr[c] = *(const u32x4*)(Qg + 16 * c + 8 * h);

  // Copies: 1 KB instruction n of the wave covers 16-byte slots 64 (wave + 4n) .. + 63 of a tile; slot t is (row
  // t / SLOTS, chunk t % SLOTS); pad chunks repeat the row's last one. Rows are held in [lo, hi], the keys
  // that some row of the workgroup sees. Step j copies V(j) and K(j + 2), in parts that it issues among its
  // products: issued together before them, addresses and copies took a third of a step.
  int krow[C::KPW], vrow[C::VPW];
  uint32_t kchunk[C::KPW], vchunk[C::VPW];
  auto vx = [](int r) { return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); };
#pragma unroll
  for (int n = 0; n < C::KPW; ++n) {
    const int t = 64 * (wave + 4 * n) + lane;
    krow[n] = t / C::KSLOTS;
    kchunk[n] = 16 * min(t % C::KSLOTS, D / 8 - 1);
  }
#pragma unroll
  for (int n = 0; n < C::VPW; ++n) {
    const int t = 64 * (wave + 4 * n) + lane;
    vrow[n] = t / C::VSLOTS;
    vchunk[n] = 16 * ((t % C::VSLOTS) ^ vx(vrow[n]));
  }
  const uint32_t smem_a = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)smem;
  struct Aim {  // a tile to copy: its first row, the rows to read, the LDS stage
    const char* src;
    int lo, hi;
    uint32_t dst;
  };
  auto aim = [&](Aim& x, int j, uint32_t rs, uint32_t dst) {
    const int kt = wt.tile(j);
    if (j > 0) x.src += (int64_t)C::BN * (kt - wt.tile(j - 1)) * rs;
    x.lo = j < wt.sink ? 0 : max(wt.lo - kt * C::BN, 0);
    x.hi = j < wt.sink ? s.sinks - 1 : min(wt.hi - kt * C::BN, C::BN - 1);
    x.dst = dst;
  };
  Aim ka{Kg + (size_t)wt.tile(0) * C::BN * krs, 0, 0, 0}, va{Vg + (size_t)wt.tile(0) * C::BN * vrs, 0, 0, 0};
  auto copy_k = [&](int n) __attribute__((always_inline)) {
    if (wave + 4 * n < C::KSLOTS)
      dma16(__umul24(clamp_row(krow[n], ka.lo, ka.hi), krs) + kchunk[n], ka.src, ka.dst + 1024 * (wave + 4 * n));
  };
  auto copy_v = [&](int n) __attribute__((always_inline)) {
    if (wave + 4 * n < C::VSLOTS)
      dma16(__umul24(clamp_row(vrow[n], va.lo, va.hi), vrs) + vchunk[n], va.src, va.dst + 1024 * (wave + 4 * n));
  };
  constexpr int PARTS = C::KPW + C::VPW;
  auto part = [&](int n) __attribute__((always_inline)) {
    if (n < C::VPW) copy_v(n);
    else copy_k(n - C::VPW);
  };
  auto no_part = [](int) {};

  // LDS operand bases (elements inside a stage). K rows: A operand of S^T, lane = key row. V^T by
  // transposing reads: group lane/16 covers 16 d of a 32-d tile, source lane t = lane%16 points at key row
  // 4h + t/4 (+8 for the second read), in the key order {8g + 4h + i} in which lane half h holds P.
  const int k_rd = l32 * C::KP + 8 * h;
  const int g16 = lane >> 4, s16 = lane & 15;
  int v_rd[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt) {
    const int r = 4 * h + (s16 >> 2), ch = 4 * dt + 2 * (g16 & 1) + ((s16 & 3) >> 1);
    v_rd[dt] = r * D + 8 * (ch ^ vx(r)) + 4 * (s16 & 1);
  }

  const float c1 = s.scale * kLog2e;
  const float slack = 8.0f / c1;
  f32x16 O[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt) O[dt] = zero16();
  float m_run = -INFINITY, l_run = 0.0f, alpha = 1.0f;
  bool rescale = false;

  // One step: the products in a fixed order, one per slot (P.V first, then S), each slot with the operand
  // reads of a later one and a slice of the softmax that does not depend on it. Scheduling fences keep the
  // order. Xc = S^T of tile j (in), Xn = S^T of tile j + 1 (out), Pin = P of tile j - 1, Pout = P of tile j.
  // Softmax: slots [0, BSLOT) max of the score pairs, BSLOT the reference point, then exponent,
  // exp2, and sum and packed P in three stages per pair.
  auto wstep = [&](auto flags, int rd, const f32x16& Xc0, const f32x16& Xc1, f32x16& Xn0, f32x16& Xn1,
                   const uint32_t(&Pin)[16], uint32_t(&Pout)[16], auto part) __attribute__((always_inline)) {
    using F = decltype(flags);
    if (F::PV && rescale) {
      asm volatile("" ::: "memory");  // keeps the rescale behind its branch
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] *= alpha;
    }
    const uint16_t* kb = (const uint16_t*)(smem + rd * C::STAGE) + k_rd;
    const uint16_t* vb = (const uint16_t*)(smem + rd * C::STAGE + C::KBYTES);
    constexpr int NSM = F::S ? 2 * C::KC : 0;
    constexpr int NPV = F::PV ? 4 * C::DT : 0;
    constexpr int NM = NSM + NPV;
    constexpr int APS = D == 64 ? 2 : 1;  // score pairs entering per slot
    constexpr int BSLOT = 16 / APS;
    constexpr int CPS = D == 64 ? 4 : 2;
    constexpr int LAST = BSLOT + 1 + 15 / CPS + 2;
    constexpr int NV = NM > LAST + 1 ? NM : LAST + 1;
    auto operand = [&](int n) -> u32x4 {
      if (n < NPV) {
        const int c = n / C::DT, dt = n % C::DT;
        const u32x2 lo = lds_tr(vb + v_rd[dt] + 16 * c * D);
        const u32x2 hi = lds_tr(vb + v_rd[dt] + (16 * c + 8) * D);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
      const int t = n - NPV;
      return lds_read16(kb + (t & 1) * 32 * C::KP + 16 * (t >> 1));
    };
    constexpr int RING = D == 64 ? 3 : 6;
    u32x4 ring[RING];
#pragma unroll
    for (int n = 0; n < RING - 1; ++n)
      if (n < NM) ring[n] = operand(n);
    float mxa = -INFINITY, mxb = -INFINITY, ls0 = 0.0f, ls1 = 0.0f, mb = 0.0f;
    float t0[16], t1[16], e0[16], e1[16];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if (n < PARTS) part(n);
      if (n < NM) {
        if (n + RING - 1 < NM) ring[(n + RING - 1) % RING] = operand(n + RING - 1);
        const u32x4& op = ring[n % RING];
        if (n < NPV) {
          const int c = n / C::DT, dt = n % C::DT;
          O[dt] = mfma(op, u32x4{Pin[4 * c], Pin[4 * c + 1], Pin[4 * c + 2], Pin[4 * c + 3]}, O[dt]);
        } else {
          const int t = n - NPV;
          if (t & 1)
            Xn1 = mfma(op, Qr[t >> 1], (t >> 1) ? Xn1 : zero16());
          else
            Xn0 = mfma(op, Qr[t >> 1], (t >> 1) ? Xn0 : zero16());
        }
      }
      if (F::SM) {
#pragma unroll
        for (int p = 0; p < 16; ++p)
          if (n == p / APS) {
            const f32x16& Xs = p < 8 ? Xc0 : Xc1;
            const float a0 = Xs[(2 * p) & 15], a1 = Xs[(2 * p + 1) & 15];
            if (p & 1)
              mxb = max3f(mxb, a0, a1);
            else
              mxa = max3f(mxa, a0, a1);
            pin(mxa, mxb);
          }
        if (n == BSLOT) {
          const float mt = max_halves(fmaxf(mxa, mxb));
          const bool need = mt > m_run + slack;  // the first visible key's tile: m_run is -inf
          rescale = __any(need);
          const float m_new = need ? mt : m_run;
          // a row that has seen no key yet keeps -inf; its exponents are taken against 0
          mb = m_new == -INFINITY ? 0.0f : m_new * c1;
          alpha = need ? exp2_hw((m_run - m_new) * c1) : 1.0f;
          l_run *= alpha;
          m_run = m_new;
        }
#pragma unroll
        for (int p = 0; p < 16; ++p) {
          const int st = n - (BSLOT + 1 + p / CPS);
          const f32x16& Xs = p < 8 ? Xc0 : Xc1;
          if (st == 0) {
            t0[p] = fmaf(Xs[(2 * p) & 15], c1, -mb);
            t1[p] = fmaf(Xs[(2 * p + 1) & 15], c1, -mb);
            pin(t0[p], t1[p]);
          } else if (st == 1) {
            e0[p] = exp2_hw(t0[p]);
            e1[p] = exp2_hw(t1[p]);
            pin(e0[p], e1[p]);
          } else if (st == 2) {
            ls0 = p ? ls0 + e0[p] : e0[p];
            ls1 = p ? ls1 + e1[p] : e1[p];
            pin(ls0, ls1);
            uint32_t pk = pack_bf16(e0[p], e1[p]);
            pin(pk);
            Pout[p] = pk;
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (F::SM) l_run += ls0 + ls1;
  };

  f32x16 Sc0 = zero16(), Sc1 = zero16(), Sn0 = zero16(), Sn1 = zero16();
  uint32_t Pc[16], Pp[16];
#pragma unroll
  for (int t = 0; t < 16; ++t) Pc[t] = Pp[t] = 0u;
  auto sync = [&]() {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };
  // Step j: every wave copies K(j + 2) and V(j) into stage j & 1, which the steps before have finished
  // reading, runs its part, then all wait for the copies. Every wave passes every step's barrier.
  const int n = wt.n;
  auto aim_both = [&](int j) __attribute__((always_inline)) {
    if (j + 2 < n) {
      aim(ka, j + 2, krs, smem_a + (j & 1) * C::STAGE);
    } else {  // the last tile again, to where nothing reads: the parts need no branch
      ka.dst = smem_a + (j & 1) * C::STAGE;
    }
    aim(va, j, vrs, smem_a + (j & 1) * C::STAGE + C::KBYTES);
  };
  auto copy = [&](int j) __attribute__((always_inline)) {
    aim_both(j);
#pragma unroll
    for (int t = 0; t < PARTS; ++t) part(t);
  };
  auto scores = [&](int j) __attribute__((always_inline)) {  // S of tile j into Sc
    const uint16_t* kb = (const uint16_t*)(smem + (j & 1) * C::STAGE) + k_rd;
    Sc0 = zero16();
    Sc1 = zero16();
#pragma unroll
    for (int c = 0; c < C::KC; ++c) {
      Sc0 = mfma(lds_read16(kb + 16 * c), Qr[c], Sc0);
      Sc1 = mfma(lds_read16(kb + 32 * C::KP + 16 * c), Qr[c], Sc1);
    }
  };
  // This wave's rows [pw0, pw1] (positions) see tiles of the steps jw0 .. jw1 (and, behind the sink tile,
  // up to two that only its neighbours see: masked whole).
  const int pw0 = sq.off + i0 + 32 * wave, pw1 = min(pw0 + 31, sq.off + i1);
  const int j_of = wt.sink - wt.t0;  // step of window tile kt: kt + j_of
  const bool active = i0 + 32 * wave <= i1 && pw1 >= 0;
  const int jw0 = !active ? n + 1 : s.sinks > 0 ? 0 : max(0, pw0 - s.window + 1) / C::BN + j_of;
  const int jw1 = active ? pw1 / C::BN + j_of : -1;
  auto hide = [&](f32x16& X0, f32x16& X1, auto seen) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      f32x16& X = e < 16 ? X0 : X1;
      X[e & 15] = seen(32 * (e >> 4) + 8 * ((e & 15) >> 2) + (e & 3)) ? X[e & 15] : -INFINITY;
    }
  };
  auto mask = [&](auto first, int j, f32x16& X0, f32x16& X1) __attribute__((always_inline)) {
    const int ka = wt.tile(j) * C::BN;
    const bool all_before = ka + C::BN - 1 <= pw0, all_inside = pw0 + 31 - ka < s.window;
    if (all_before && all_inside) return;
    int dq = pos - ka - 4 * h;  // score e is of key ka + 4h + off
    asm volatile("" : "+v"(dq));  // (opaque: 32 loop-invariant bounds would be kept instead)
    const uint32_t window = s.window;
    if (decltype(first)::value) {
      // keys ka + 4h + off < sinks: the sinks are in tile 0, and that is the wave's first one then
      const int few = min(s.sinks - ka - 4 * h, dq + 1);
      hide(X0, X1, [&](int off) { return (uint32_t)(dq - off) < window || off < few; });
    } else if (all_inside) {  // the border alone
      hide(X0, X1, [&](int off) { return off <= dq; });
    } else if (all_before) {  // the window's end alone
      const int end = dq - s.window;
      hide(X0, X1, [&](int off) { return off > end; });
    } else {
      hide(X0, X1, [&](int off) { return (uint32_t)(dq - off) < window; });
    }
  };
  int j = 0;
  auto run = [&](auto flags) __attribute__((always_inline)) {
    using F = decltype(flags);
    if (F::SM) {
      aim_both(j);
      mask(std::bool_constant<!F::PV>(), j, Sc0, Sc1);
      wstep(flags, (j + 1) & 1, Sc0, Sc1, Sn0, Sn1, Pp, Pc, part);
    } else {
      if (j < n) copy(j);
      wstep(flags, (j + 1) & 1, Sc0, Sc1, Sn0, Sn1, Pp, Pc, no_part);
    }
    if (F::S) {
      Sc0 = Sn0;
      Sc1 = Sn1;
    }
    if (F::SM) {
#pragma unroll
      for (int t = 0; t < 16; ++t) Pp[t] = Pc[t];
    }
    if (j < n) sync();
    ++j;
  };

  aim(ka, 0, krs, smem_a);
#pragma unroll
  for (int t = 0; t < C::KPW; ++t) copy_k(t);
  if (n > 1) {
    aim(ka, 1, krs, smem_a + C::STAGE);
#pragma unroll
    for (int t = 0; t < C::KPW; ++t) copy_k(t);
  }
  sync();
  if (jw0 == 0) scores(0);
  __syncthreads();
  while (j < min(jw0 - 1, n)) {
    copy(j);
    sync();
    ++j;
  }
  if (active) {
    if (jw0 > 0) {  // step jw0 - 1
      copy(j);
      scores(jw0);
      sync();
      ++j;
    }
    run(WfStep<true, false, true>());  // (behind the wave's last tile S is of no use, and unused)
    if (j < jw1 && ((jw1 - j) & 1)) run(WfStep<true, true, true>());
    while (j < jw1) {  // two steps in turn on swapped buffers
      aim_both(j);
      mask(std::false_type(), j, Sc0, Sc1);
      wstep(WfStep<true, true, true>(), (j + 1) & 1, Sc0, Sc1, Sn0, Sn1, Pp, Pc, part);
      sync();
      aim_both(j + 1);
      mask(std::false_type(), j + 1, Sn0, Sn1);
      wstep(WfStep<true, true, true>(), j & 1, Sn0, Sn1, Sc0, Sc1, Pc, Pp, part);
      sync();
      j += 2;
    }
    if (j == jw1) run(WfStep<false, true, true>());
    run(WfStep<false, true, false>());
  }
  while (j < n) {
    copy(j);
    sync();
    ++j;
  }

  // ---- out = bf16(O / l), l = m/sqrt(D) + ln(sum) ----
  const float lt = sum_halves(l_run);
  // rows whose sum is finite and whose output is not: summed again over their visible keys alone
  float bad = 0.0f;
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad = fmaf(O[dt][r], 0.0f, bad);
  const bool again = row_ok && pos >= 0 && lt - lt == 0.0f && sum_halves(bad) != 0.0f;
  if (__any(again)) {
    if (again) {
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt) O[dt] = zero16();
      const float mb = m_run * c1;
      const int first = max(0, pos - s.window + 1);
      const int ns = min(s.sinks, first);
      for (int t = 0; t < ns + pos + 1 - first; ++t) {
        const int key = t < ns ? t : first + t - ns;
        const uint16_t* kr = (const uint16_t*)(Kg + (size_t)key * krs);
        const uint16_t* vr = (const uint16_t*)(Vg + (size_t)key * vrs);
        float x = 0.0f;
#pragma unroll
        for (int c = 0; c < C::KC; ++c) {
          asm volatile("" : "+v"(Qr[c]));  // (or the unpacked values are kept over the loop)
          const u32x4 kk = *(const u32x4*)(kr + 16 * c + 8 * h);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            x = fmaf(bf_lo(kk[w]), bf_lo(Qr[c][w]), x);
            x = fmaf(bf_hi(kk[w]), bf_hi(Qr[c][w]), x);
          }
        }
        const float p = round_bf16(exp2_hw(fmaf(sum_halves(x), c1, -mb)));
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const u32x2 vv = *(const u32x2*)(vr + 32 * dt + 8 * g + 4 * h);
            O[dt][4 * g] = fmaf(p, bf_lo(vv[0]), O[dt][4 * g]);
            O[dt][4 * g + 1] = fmaf(p, bf_hi(vv[0]), O[dt][4 * g + 1]);
            O[dt][4 * g + 2] = fmaf(p, bf_lo(vv[1]), O[dt][4 * g + 2]);
            O[dt][4 * g + 3] = fmaf(p, bf_hi(vv[1]), O[dt][4 * g + 3]);
          }
      }
    }
  }
  const bool empty = pos < 0;
  const float inv = 1.0f / lt;
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[dt][r] = empty ? 0.0f : O[dt][r] * inv;
  if (lg && h == 0 && row_ok) lg[i] = empty ? -INFINITY : m_run * s.scale + logf(lt);
  __syncthreads();  // every wave is past its last P.V
  const int rows = i1 - i0 - 32 * wave;
  store_rows<D>(smem_a + wave * kRowsOut<D>, lane, O, 1.0f, Og, s.o_row, [&](int r) { return r <= rows; });
}

hipError_t launch_window_forward(const WinFwdArgs& a, int D, hipStream_t s) {
  const int nqb = (a.s.TQ + kFwdBlockM - 1) / kFwdBlockM;
  const dim3 grid((unsigned)(a.s.B * a.s.NH * nqb));
  if (D == 64)
    hipLaunchKernelGGL(win_fwd_kernel<64>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(win_fwd_kernel<128>, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace mla
