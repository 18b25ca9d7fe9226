// Gradients of causal softmax attention: dk and dv, for heads of up to 128 (see gdn_attn_bwd.hip).
#include <type_traits>

#include "gdn_attn.h"

namespace omx {
namespace {

constexpr int kNW = 4, kNT = 64 * kNW;

// ------------------------------------------------------------------------------------ dk, dv
// A workgroup's 128 keys, 32 a wavefront with their k and v in registers, against the rows that
// see them, 32 a stage:
//   S = Q K^T, dP = dO V^T - delta (rows x keys), P = exp(S - lse), dS = P dP,
//   dV^T += dO^T P, dK^T += Q^T dS
// One wavefront a SIMD (its registers hold k, v, dk, dv), so nothing but its own instructions can
// fill the time between dependent ones.  They are laid out as a pipeline of two phases a stage,
// each a sequence of groups of one product with the loads and arithmetic that run beside it:
//   1: S and dP of the next stage | P and dS of this one | reads of its transposed fragments
//   2: dV and dK of this stage    | reads of the next but one's fragments, and the next's lse, delta
// The order is pinned group by group; left to itself the compiler put all products of a phase
// behind all loads, two reads ahead (B=4 T=4,096 of 32/8 heads of 128: 1,690 us, now 1,020 to 1,150; the
// MFMAs are busy for 56% of it, the clock falls to 1.9 GHz under them).  Stages lie in
// a ring of six LDS buffers, filled from memory directly.
// WIN: a tile's rows are those whose window reaches its keys; the first tiles' keys, which all rows see as
// sinks, are summed in shares of their own (attn_dkv_window_plan).  Window 1,024 and 16 sinks at the same size:
// 605 us, an eighth of it products of rows at both ends of the band that see none of a wavefront's keys.
constexpr int kRows = 32;        // rows of a stage
constexpr int kRing = 6;

template <int I>
struct Slot {
  static constexpr int i = I;
};

// WIN: a row sees its last p.window keys and the first p.sinks.
template <int DP, bool WIN>
__global__ __launch_bounds__(kNT) __attribute__((amdgpu_waves_per_eu(1, 1)))
void attn_dkv_kernel(AttnParams p, int ranks) {
  constexpr int KS = DP / 16, DB = DP / 32, NG = 2 * KS, EG = 16 / NG;
  constexpr int NJ = kRows * DP / 8 / 64 / kNW, kLoads = 2 * NJ + 1;  // a wavefront's, a stage

  // the ring: of each stage its rows of q, of do, their lse / ln 2 and -delta
  constexpr int kDo = kRows * DP, kStats = 2 * kRows * DP, kSlot = kStats + 4 * kRows;
  __shared__ __align__(16) bf16_t ring[kRing * kSlot];

  const int tid = threadIdx.x, l = tid & 63, h = l >> 5, c = l & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AttnLane lane = attn_lane<DP>();
  const int G = p.G, D = p.D, Hkv = p.Hkv, Hq = Hkv * G, per = kRows / G;

  int unit, rank;
  attn_place((int)blockIdx.x, (p.cu ? 1 : p.N) * Hkv, ranks, unit, rank);
  if (rank >= ranks) return;
  const int hk = unit % Hkv;
  std::conditional_t<WIN, WindowShare, DkvShare> it;
  if constexpr (WIN) {
    if (!dkv_window_share(p, unit / Hkv, rank, per, it)) return;
  } else {
    if (!dkv_share(p, unit / Hkv, rank, per, it)) return;
  }
  const int kw = it.k0 + 32 * w, key = kw + c;
  // stages from the last to the first: a unit's workgroups, which start together and see different
  // numbers of rows, then read the same rows at the same time, and its XCD's L2 serves most of them
  const int n = (it.tb - it.ta + per - 1) / per, t_last = it.ta + (n - 1) * per;
  // of these the wavefront's keys are seen by the first na
  int na = t_last + per - kw <= 0 ? 0 : (t_last + per - kw + per - 1) / per;
  na = na < n ? na : n;

  u32x4 kf[KS], vf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = 16 * s + 8 * h;
    kf[s] = vf[s] = u32x4{0, 0, 0, 0};
    if (key < it.len && d < D) {
      kf[s] = *(const u32x4*)((const bf16_t*)p.k + (it.start + key) * p.k_ld + hk * D + d);
      vf[s] = *(const u32x4*)((const bf16_t*)p.v + (it.start + key) * p.v_ld + hk * D + d);
    }
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
  const float cs = p.scale * kLog2e;

  const unsigned qld2 = (unsigned)(p.q_ld * 2), old2 = (unsigned)(Hq * D * 2);
  unsigned qoff[NJ], ooff[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int r = stage_row<DP, kNW>(w, j), seg = stage_seg<DP>(r), t = r / G, g = r - t * G;
    const bool in = t < per && 8 * seg < D;
    const unsigned x = (unsigned)g * 2u * D + 16u * (unsigned)seg;
    qoff[j] = in ? (unsigned)t * qld2 + x : kDropOffset;
    ooff[j] = in ? (unsigned)t * old2 + x : kDropOffset;
  }
  const int sr = l % kRows;  // lanes 0-31 fetch the rows' lse, 32-63 their -delta
  const unsigned soff = sr / G < per ? (unsigned)(sr / G) * 8u * Hq + 4u * (unsigned)(sr % G + (l / kRows) * G) : kDropOffset;
  // The next stage to fetch, from the last tokens on.  Rows past the sequence read as zeros: they
  // add nothing.  Past the last stage the ranges are empty, so that every turn counts the same
  // loads; all four wavefronts fetch the same lse and -delta for the same reason.
  const bf16_t* q_at = (const bf16_t*)p.q + (it.start + t_last) * p.q_ld + (long long)hk * G * D;
  const bf16_t* o_at = (const bf16_t*)p.dout + ((it.start + t_last) * Hq + hk * G) * D;
  const float* s_at = p.stats + 2 * ((it.start + t_last) * Hq + hk * G);
  const int m0 = it.len - t_last < per ? it.len - t_last : per;
  const unsigned q_all = (unsigned)(per - 1) * qld2 + 2u * D * G, o_all = (unsigned)(per - 1) * old2 + 2u * D * G;
  const unsigned s_all = (unsigned)(per - 1) * 8u * Hq + 8u * G;
  unsigned q_range = n > 0 ? (unsigned)(m0 - 1) * qld2 + 2u * D * G : 0;
  unsigned o_range = n > 0 ? (unsigned)(m0 - 1) * old2 + 2u * D * G : 0;
  unsigned s_range = n > 0 ? (unsigned)(m0 - 1) * 8u * Hq + 8u * G : 0;
  const unsigned lds0 = lds_address(ring);
  auto stage_q = [&](int slot) {
    loads_to_lds16(rsrc_words(q_at, q_range), lds0 + 2u * kSlot * (unsigned)slot + 1024u * (unsigned)w, qoff);
  };
  auto stage_o = [&](int slot) {
    loads_to_lds16(rsrc_words(o_at, o_range), lds0 + 2u * (kSlot * (unsigned)slot + kDo) + 1024u * (unsigned)w, ooff);
  };
  auto stage_s = [&](int slot) { load_to_lds4(rsrc_words(s_at, s_range), lds0 + 2u * (kSlot * (unsigned)slot + kStats), soff); };
  auto stage_next = [&](bool more) {
    q_at -= per * p.q_ld;
    o_at -= (long long)per * Hq * D;
    s_at -= 2 * (long long)per * Hq;
    q_range = more ? q_all : 0;
    o_range = more ? o_all : 0;
    s_range = more ? s_all : 0;
  };
  auto stage = [&](bool more, int slot) {
    stage_q(slot);
    stage_o(slot);
    stage_s(slot);
    stage_next(more);
  };

  u32x4 fq[KS], fo[KS];  // fragments of the stage whose S and dP come next
  f32x4 lse[4];          // of the stage whose P and dS come next
  u32x4 tf[NG];          // transposed fragments, and
  u32x4 pb[2], db[2];    //   P and dS, of the stage whose dV and dK come next

  // a stage's fragment that group g of phase 2 multiplies: dO^T and Q^T in turn
  auto tr = [&](const bf16_t* st, int g) {
    return attn_frag_tr<DP>(g & 1 ? st : st + kDo, lane, 16 * (g / (2 * DB)), (g / 2) % DB);
  };
  auto row_lse = [&](const bf16_t* st, int j) { lse[j] = *((const f32x4*)(st + kStats) + 2 * j + h); };
  auto row_delta = [&](f32x16& dp, const bf16_t* st, int j) {  // what the sums of a stage's dP start from
    const f32x4 x = *((const f32x4*)(st + kStats) + kRows / 4 + 2 * j + h);
#pragma unroll
    for (int i = 0; i < 4; ++i) dp[4 * j + i] = x[i];
  };
  auto grad = [&](f32x16& s, f32x16& dp, int e) {
    dp[e] *= s[e];
    if (e & 1) {
      pb[e / 8][(e / 2) % 4] = pack_bf16(s[e - 1], s[e]);
      db[e / 8][(e / 2) % 4] = pack_bf16(dp[e - 1], dp[e]);
    }
  };
  auto phase1 = [&](f32x16& s, f32x16& dp, f32x16& sn, f32x16& dpn, const bf16_t* st) {
    sn = zero16();
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (g & 1)
        dpn = mma32(fo[g / 2], vf[g / 2], dpn);
      else
        sn = mma32(fq[g / 2], kf[g / 2], sn);
      tf[g] = tr(st, g);
#pragma unroll
      for (int e = EG * g; e < EG * (g + 1); ++e) {  // P of these rows, dS of those before
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], cs, -lse[e / 4][e % 4]));
        if (e >= EG) grad(s, dp, e - EG);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int e = 16 - EG; e < 16; ++e) grad(s, dp, e);
  };
  auto phase2 = [&](f32x16& dp, const bf16_t* st1, const bf16_t* st2, bool more, int fetch) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int d = (g / 2) % DB, k = g / (2 * DB);
      if (g & 1)
        dk[d] = mma32(tf[g], db[k], dk[d]);
      else
        dv[d] = mma32(tf[g], pb[k], dv[d]);
      if (g & 1)
        fo[g / 2] = attn_frag<DP>(st2 + kDo, lane, 0, g / 2);
      else
        fq[g / 2] = attn_frag<DP>(st2, lane, 0, g / 2);
      if (g % (NG / 4) == 0) row_lse(st1, g / (NG / 4));
      if (g % (NG / 4) == 1) row_delta(dp, st2, g / (NG / 4));
      if (g == 0) stage_q(fetch);
      if (g == 3) stage_o(fetch);
      if (g == 6) stage_s(fetch);
      if (g == 7) stage_next(more);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // row r of a stage is token t + r / G: before the key if r < (key - t) G
  auto mask = [&](f32x16& s, int t) {
    if constexpr (WIN) {
      const RowMask m = row_mask(p, key, t);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 8 * (i / 4) + 4 * h + i % 4;
        if (r < m.first || r >= m.past) s[i] = -INFINITY;
      }
      return;
    }
    const int first = (key - t) * G;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (8 * (i / 4) + 4 * h + i % 4 < first) s[i] = -INFINITY;
  };

  // Stage i, in buffer i % kRing.  At its barrier stage i + 2 is there.  Behind it stage i +
  // kRing - 1 is fetched into the buffer of i - 1, whose last reads were used before the barrier:
  // so the barrier need not wait for the reads of this stage.
  auto turn = [&](int i, auto slot, f32x16& s, f32x16& dp, f32x16& sn, f32x16& dpn) {
    constexpr int I = decltype(slot)::i;
    if (i < na) {
      const int t = t_last - i * per;
      if (t < kw + 31 || (WIN && past_window(p, kw, t, per))) mask(s, t);
      phase1(s, dp, sn, dpn, ring + I * kSlot);
    }
    wait_loads<(kRing - 4) * kLoads>();
    asm volatile("s_barrier" ::: "memory");
    const bool more = i + kRing < n;
    if (i < na)
      phase2(dp, ring + (I + 1) % kRing * kSlot, ring + (I + 2) % kRing * kSlot, more, (I + kRing - 1) % kRing);
    else  // rows that see none of this wavefront's keys: its share of the loads
      stage(more, (I + kRing - 1) % kRing);
  };
  if (n > 0) {
    static_assert(kRing == 6, "the turns below");
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) stage(i + 1 < n, i);
    wait_loads<3 * kLoads>();  // stages 0 and 1
    asm volatile("s_barrier" ::: "memory");
    const bf16_t *st0 = ring, *st1 = ring + kSlot;
    f32x16 s0 = zero16(), dp0, s1, dp1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      row_delta(dp0, st0, j);
      row_delta(dp1, st1, j);
      row_lse(st0, j);
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      s0 = mma32(attn_frag<DP>(st0, lane, 0, k), kf[k], s0);
      dp0 = mma32(attn_frag<DP>(st0 + kDo, lane, 0, k), vf[k], dp0);
      fq[k] = attn_frag<DP>(st1, lane, 0, k);
      fo[k] = attn_frag<DP>(st1 + kDo, lane, 0, k);
    }
    for (int i = 0;; i += kRing) {
      turn(i, Slot<0>(), s0, dp0, s1, dp1);
      if (i + 1 >= n) break;
      turn(i + 1, Slot<1>(), s1, dp1, s0, dp0);
      if (i + 2 >= n) break;
      turn(i + 2, Slot<2>(), s0, dp0, s1, dp1);
      if (i + 3 >= n) break;
      turn(i + 3, Slot<3>(), s1, dp1, s0, dp0);
      if (i + 4 >= n) break;
      turn(i + 4, Slot<4>(), s0, dp0, s1, dp1);
      if (i + 5 >= n) break;
      turn(i + 5, Slot<5>(), s1, dp1, s0, dp0);
      if (i + 6 >= n) break;
    }
  }
  wait_loads<0>();
  if (key >= it.len) return;
  const long long at = ((it.start + key) * Hkv + hk) * D;
  if constexpr (WIN) {
    if (p.splits > 1 && it.share == 0 && h == 0) p.shares[at / D] = it.sink ? 1 : it.shares;
  } else {
    if (p.splits > 1 && it.share == 0 && h == 0) p.shares[at / D] = it.shares;
  }
  if (it.shares > 1) {
    float *pk, *pv;
    const long long ps = dkv_part(p, it, at, pk, pv);
    store_part<DB>(pk + ps, dk, p.scale, D, h);
    store_part<DB>(pv + ps, dv, 1.f, D, h);
  } else {
    store_rows<DB>((bf16_t*)p.dk + at, dk, p.scale, D, h);
    store_rows<DB>((bf16_t*)p.dv + at, dv, 1.f, D, h);
  }
}

}  // namespace

void launch_attn_dkv_narrow(const AttnParams& p, unsigned grid, int ranks, hipStream_t stream) {
  if (p.D <= 64 && p.window > 0)
    attn_dkv_kernel<64, true><<<grid, kNT, 0, stream>>>(p, ranks);
  else if (p.D <= 64)
    attn_dkv_kernel<64, false><<<grid, kNT, 0, stream>>>(p, ranks);
  else if (p.window > 0)
    attn_dkv_kernel<128, true><<<grid, kNT, 0, stream>>>(p, ranks);
  else
    attn_dkv_kernel<128, false><<<grid, kNT, 0, stream>>>(p, ranks);
}

}  // namespace omx
