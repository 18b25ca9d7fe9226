// Gradients of causal softmax attention: dq, and each row's delta (see gdn_attn_bwd.hip).
#include "gdn_attn.h"

namespace omx {
namespace {

constexpr int kBM = 128, kBN = 32, kNW = 4, kNT = 64 * kNW;
constexpr int kRing = 4;  // blocks of 32 keys in LDS

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// A workgroup's 128 rows, 32 a wavefront with their q and do in registers, against the keys they
// see, 32 at a time.  A block goes through three phases, laid out group by group, one product to
// each with the loads and arithmetic that run beside it:
//   A: dP^T = V dO^T            | P = exp(S - lse)          | reads of v, then of the next k
//   B: the next block's S^T     | dS = P (dP - delta)       | reads of k, then of k transposed
//   C: dQ^T += K^T dS^T         |                           | reads of k transposed, then of the next v
// Bound by the MFMAs, three products a block: B=4 T=4,096 of 32/8 heads of 128 760 to 820 us (the
// compiler's own order, tiles of 64 keys: 805 to 860); with few tiles by the longest and the loads
// before it: 3,001 tokens in 5 sequences of 16/2 heads of 256 56 us (73).
// WIN: as for the forward, the blocks being the sinks' and those from the first row's window on; window 1,024
// and 16 sinks at B=4 T=4,096 of 32/8 heads of 128 403 us.
template <int DP, bool WIN>
__global__ __launch_bounds__(kNT) __attribute__((amdgpu_waves_per_eu(DP == 256 ? 1 : 2)))
void attn_dq_kernel(AttnParams p, int ranks) {
  constexpr int KS = DP / 16, DB = DP / 32, EG = 16 / KS, PF = 4;
  constexpr int NJ = kBN * DP / 8 / 64 / kNW, kLoads = 2 * NJ;  // a wavefront's loads of k (of both), a block
  constexpr int kVal = kBN * DP, kSlot = 2 * kVal;              // of a slot: k, then v
  __shared__ __align__(16) bf16_t ring[kRing * kSlot];

  const int tid = threadIdx.x, l = tid & 63, h = l >> 5, c = l & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AttnLane lane = attn_lane<DP>();
  const int G = p.G, D = p.D, Hkv = p.Hkv, Hq = Hkv * G, per = kBM / G;

  int unit, rank;
  attn_place((int)blockIdx.x, (p.cu ? 1 : p.N) * Hkv, ranks, unit, rank);
  if (rank >= ranks) return;
  const int hk = unit % Hkv;
  AttnTile it;
  if (!attn_tile(p, unit / Hkv, rank, per, it)) return;
  const int t0 = it.tile * per, nt = it.len - t0 < per ? it.len - t0 : per;

  const int row = 32 * w + c, rt = row / G, rg = row - rt * G;
  const bool live = rt < nt;
  const long long tok = it.start + t0 + rt, at = tok * Hq + hk * G + rg;
  const int pos = t0 + rt, w_lo = t0 + (32 * w) / G, w_hi = t0 + (32 * w + 31) / G;

  // fetches block kb's keys (and values) into its slot; blocks past the last have an empty range
  // (with a window these are the sinks' and from the first row's window on, `shift` keys later: block kb
  // begins at key0(kb))
  int nb = (t0 + nt + kBN - 1) / kBN, sink_blocks = 0, shift = 0;
  if constexpr (WIN) {
    const int lo = t0 - p.window + 1;
    sink_blocks = (p.sinks + kBN - 1) / kBN;
    shift = lo > sink_blocks * kBN ? lo - sink_blocks * kBN : 0;
    nb = (t0 + nt - shift + kBN - 1) / kBN;
  }
  auto key0 = [&](int kb) { return kb * kBN + (WIN && kb >= sink_blocks ? shift : 0); };
  constexpr int kStep = 64 / (DP / 8) * kNW, NO = kStep % 16 ? 2 : 1;
  static_assert(NO * kStep % 16 == 0 && NO <= NJ, "rows whose swizzle repeats");
  const unsigned kld2 = (unsigned)(p.k_ld * 2), vld2 = (unsigned)(p.v_ld * 2);
  unsigned koff[NJ], voff[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int r = stage_row<DP, kNW>(w, j), seg = stage_seg<DP>(r);
    koff[j] = 8 * seg < D ? (unsigned)r * kld2 + 16u * (unsigned)seg : kDropOffset;
    voff[j] = 8 * seg < D ? (unsigned)r * vld2 + 16u * (unsigned)seg : kDropOffset;
  }
  const unsigned lds0 = lds_address(ring) + 1024u * (unsigned)w;
  auto fetch = [&](int kb, const void* rows, long long ld, unsigned ld2, const unsigned (&off)[NJ], unsigned part) {
    int left = it.len - key0(kb);  // rows past the sequence read as zeros
    left = left < kBN ? left : kBN;
    loads_to_lds16(rsrc_words((const bf16_t*)rows + (it.start + key0(kb)) * ld + hk * D,
                              kb < nb ? (unsigned)(left - 1) * ld2 + 2u * D : 0),
                   lds0 + 2u * (kSlot * (unsigned)(kb & (kRing - 1)) + part), off);
  };
  auto fetch_k = [&](int kb) { fetch(kb, p.k, p.k_ld, kld2, koff, 0); };
  auto fetch_v = [&](int kb) { fetch(kb, p.v, p.v_ld, vld2, voff, kVal); };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) {
    fetch_k(i);
    fetch_v(i);
  }

  u32x4 q[KS], dout[KS];
  float delta = 0.f, lse2;
  {
    u32x4 o[KS], rest[KS];
    const long long rl = live ? tok : it.start + t0, al = rl * Hq + hk * G + (live ? rg : 0);
    lse2 = p.lse[al] * kLog2e;
    load_row(dout, (const bf16_t*)p.dout + al * D, D, h);
    load_row(o, (const bf16_t*)p.o + al * D, D, h);
    load_row(rest, (const bf16_t*)(p.o_rest ? p.o_rest : p.o) + al * D, D, h);
    load_row(q, (const bf16_t*)p.q + rl * p.q_ld + (long long)(hk * G + (live ? rg : 0)) * D, D, h);
    clear_past(dout, D, h);
    clear_past(o, D, h);
    clear_past(rest, D, h);
    clear_past(q, D, h);
#pragma unroll
    for (int s = 0; s < KS; ++s) delta = dot8(dout[s], o[s], delta);
    if (p.o_rest)
#pragma unroll
      for (int s = 0; s < KS; ++s) delta = dot8(dout[s], rest[s], delta);
  }
  delta = sum_halves(delta);
  lse2 = live ? lse2 : INFINITY;  // idle rows: weights of 0
  if (live && h == 0) {
    float* st = p.stats + 2 * (tok * Hq + hk * G) + rg;
    st[0] = lse2;
    st[G] = -delta;
  }
  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = zero16();
  const float cs = p.scale * kLog2e;

  u32x4 f[PF], ds[2];
  auto slot = [&](int kb) { return ring + (kb & (kRing - 1)) * kSlot; };
  auto tr = [&](const bf16_t* sk, AttnLane ln, int t) { return attn_frag_tr<DP>(sk, ln, 16 * (t / DB), t % DB); };
  auto mask = [&](int kb, f32x16& s) {
    if constexpr (WIN) {
      const unsigned see = (unsigned)window_bits(p, pos, key0(kb)) >> 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!((see >> (8 * (i / 4) + i % 4)) & 1)) s[i] = -INFINITY;
      return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (kb * kBN + 8 * (i / 4) + 4 * h + i % 4 > pos) s[i] = -INFINITY;
  };
  // block kb, whose scores are s and whose first fragments of v are in f; leaves the next one's
  auto turn = [&](auto more, int kb, f32x16& s, f32x16& sn) {
    constexpr bool kMore = decltype(more)::value;
    wait_loads<kLoads>();  // all but block kb + 2: block kb + 1 is there
    lds_barrier();         // everyone's; and block kb - 1's slot is free
    const bf16_t *st = slot(kb), *st1 = slot(kb + 1);
    const int k0 = key0(kb);
    if (k0 + kBN - 1 > w_lo || (WIN && k0 <= w_hi - p.window && k0 + kBN > p.sinks)) mask(kb, s);
    const AttnLane ln = fresh(lane);
    f32x16 dp = zero16();
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      dp = mma32(f[t % PF], dout[t], dp);
      if (t + PF < KS)
        f[t % PF] = attn_frag<DP>(st + kVal, ln, 0, t + PF);
      else
        f[t % PF] = kMore ? attn_frag<DP>(st1, ln, 0, t + PF - KS) : tr(st, ln, t + PF - KS);
#pragma unroll
      for (int e = EG * t; e < EG * (t + 1); ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], cs, -lse2));
      __builtin_amdgcn_sched_barrier(0);
    }
    sn = zero16();
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      if constexpr (kMore) {
        sn = mma32(f[t % PF], q[t], sn);
        f[t % PF] = t + PF < KS ? attn_frag<DP>(st1, ln, 0, t + PF) : tr(st, ln, t + PF - KS);
      }
#pragma unroll
      for (int e = EG * t; e < EG * (t + 1); ++e) {
        s[e] *= dp[e] - delta;
        if (e & 1) ds[e / 8][e / 2 % 4] = pack_bf16(s[e - 1], s[e]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      dq[t % DB] = mma32(f[t % PF], ds[t / DB], dq[t % DB]);
      if (t + PF < KS)
        f[t % PF] = tr(st, ln, t + PF);
      else if (kMore)
        f[t % PF] = attn_frag<DP>(st1 + kVal, ln, 0, t + PF - KS);
      if (t == 0) fetch_k(kb + kRing - 1);
      if (t == KS / 2) fetch_v(kb + kRing - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  wait_loads<2 * kLoads>();  // block 0 (and what was loaded behind the blocks, which is in use)
  lds_barrier();
  f32x16 s0 = zero16(), s1;
#pragma unroll
  for (int t = 0; t < KS; ++t) s0 = mma32(attn_frag<DP>(slot(0), lane, 0, t), q[t], s0);
#pragma unroll
  for (int t = 0; t < PF; ++t) f[t] = attn_frag<DP>(slot(0) + kVal, lane, 0, t);
  // the wavefront's own last block: rows of it see no keys of later ones
  const int w_kb = (w_hi - shift) / kBN, last = w_kb < nb - 1 ? w_kb : nb - 1;
  int kb = 0;
  while (kb + 1 < last) {
    turn(Yes(), kb++, s0, s1);
    turn(Yes(), kb++, s1, s0);
  }
  if (kb < last) {
    turn(Yes(), kb++, s0, s1);
    s0 = s1;
  }
  turn(No(), kb++, s0, s1);
  for (; kb < nb; ++kb) {  // other wavefronts' blocks: its part of the loads
    wait_loads<kLoads>();
    lds_barrier();
    fetch_k(kb + kRing - 1);
    fetch_v(kb + kRing - 1);
  }
  wait_loads<0>();
  if (live) store_rows<DB>((bf16_t*)p.dq + at * D, dq, p.scale, D, h);
}

}  // namespace

hipError_t launch_attn_dq(const AttnParams& p, hipStream_t stream) {
  const long long ranks = attn_ranks(p, kBM / p.G), units = (long long)(p.cu ? 1 : p.N) * p.Hkv;
  const unsigned grid = (unsigned)attn_grid(units, ranks);
  const int r = (int)ranks;
  switch (p.D <= 64 ? 64 : (p.D <= 128 ? 128 : 256)) {
#define OMX_DQ(DP)                                                   \
  case DP:                                                           \
    if (p.window > 0)                                                \
      attn_dq_kernel<DP, true><<<grid, kNT, 0, stream>>>(p, r);      \
    else                                                             \
      attn_dq_kernel<DP, false><<<grid, kNT, 0, stream>>>(p, r);     \
    break;
    OMX_DQ(64)
    OMX_DQ(128)
    OMX_DQ(256)
#undef OMX_DQ
  }
  return hipGetLastError();
}

}  // namespace omx
