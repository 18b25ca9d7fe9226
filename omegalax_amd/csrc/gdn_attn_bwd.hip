// Gradients of causal softmax attention over packed prompts, from the forward's output and the
// logarithm of each row's sum:
//
//   p_ij = exp(s_ij - lse_i),  dv_j = sum_i p_ij do_i,  delta_i = do_i . o_i,
//   ds_ij = p_ij (do_i . v_j - delta_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// Two kernels, each of which owns what it sums, so no sum depends on the order of atomics: one
// passes over the keys for a tile of rows (dq, and delta for the other), one over the rows for a
// tile of keys (dk, dv).  The scores and do . v are formed in both, 7 products in place of 5.
#include "gdn_attn.h"

namespace omx {
namespace {

constexpr int kNW = 4, kNT = 64 * kNW;
constexpr int kRows = 32, kRing = 4;  // a stage's rows, stages in LDS

// dk and dv for heads of more than 128.  A wavefront's 32 keys, of the workgroup's 128, stay with
// their sums in registers (k and v 128, dk and dv 256 of a lane's 512, so one wavefront a SIMD);
// stages of 32 rows go past them through a ring in LDS.  A stage is four phases, one product after
// the other with the loads and arithmetic that run beside it:
//   S = Q K^T | dP = dO V^T, P = exp(S - lse) | dV^T += dO^T P, dS = P (dP - delta) | dK^T += Q^T dS
// 3,001 tokens in 5 sequences of 16/2 heads of 256: 74 us (125 with stages of 64 rows twice buffered,
// the compiler's order and whole tiles in four shares each).  A stage takes 1.5 times its MFMAs; the
// rest is what comes before the first stage and the partial sums behind the last, about 14 us.
template <int DP>
__global__ __launch_bounds__(kNT) __attribute__((amdgpu_waves_per_eu(1)))
void attn_dkv_wide_kernel(AttnParams p, int ranks) {
  constexpr int KS = DP / 16, DB = DP / 32, PF = 4;
  constexpr int NJ = kRows * DP / 8 / 64 / kNW, kLoads = 2 * NJ + 1;  // a wavefront's loads, a stage
  constexpr int kSlot = 2 * kRows * DP;                               // of a slot: q, then do
  static_assert(KS == 16, "one element of the scores beside each product");
  __shared__ __align__(16) bf16_t ring[kRing * kSlot];
  __shared__ __align__(16) float stats[kRing * 128];  // a stage's lse, its delta from 64 on
  __shared__ __align__(16) u32x4 offs[2][kNT];
  __shared__ unsigned soffs[kNT];

  const int tid = threadIdx.x, l = tid & 63, h = l >> 5, c = l & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AttnLane lane = attn_lane<DP>();
  const int G = p.G, D = p.D, Hkv = p.Hkv, Hq = Hkv * G, per = kRows / G;

  int unit, rank;
  attn_place((int)blockIdx.x, (p.cu ? 1 : p.N) * Hkv, ranks, unit, rank);
  if (rank >= ranks) return;
  const int hk = unit % Hkv;
  DkvShare it;
  if (!dkv_share(p, unit / Hkv, rank, per, it)) return;
  const int kw = it.k0 + 32 * w, key = kw + c;  // the wavefront's first key, the lane's

  // stages from the last to the first: a unit's workgroups, which start together and see different
  // numbers of rows, then read the same rows at the same time, and its XCD's L2 serves most of them
  const int n = (it.tb - it.ta + per - 1) / per, t_last = it.ta + (n - 1) * per;
  // of these the wavefront's keys are seen by the first na
  int na = t_last + per - kw <= 0 ? 0 : (t_last + per - kw + per - 1) / per;
  na = na < n ? na : n;

  const unsigned qld2 = (unsigned)(p.q_ld * 2), old2 = (unsigned)(Hq * D * 2);
  const unsigned lds0 = lds_address(ring) + 1024u * (unsigned)w;
  const unsigned lds1 = lds_address(stats) + 256u * (unsigned)(w & 1);
  // The offsets of a thread's loads are the same each stage, and kept in LDS: registers are full.
  static_assert(NJ == 4, "four loads a thread");
  {
    u32x4 x, y;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int r = stage_row<DP, kNW>(w, j), seg = stage_seg<DP>(r), t = r / G, g = r - t * G;
      const bool in = t < per && 8 * seg < D;
      const unsigned z = (unsigned)g * 2u * D + 16u * (unsigned)seg;
      x[j] = in ? (unsigned)t * qld2 + z : kDropOffset;
      y[j] = in ? (unsigned)t * old2 + z : kDropOffset;
    }
    offs[0][tid] = x;
    offs[1][tid] = y;
    soffs[tid] = l / G < per ? (unsigned)(l / G) * 8u * Hq + 4u * (unsigned)(l % G) : kDropOffset;
  }
  // Fetches stage i's rows of q (of do) into its slot; stages past the last have an empty range, and
  // so have rows past the sequence, which read as zeros and add nothing.
  auto fetch = [&](int i, u32x4 x, const bf16_t* rows, long long ld, unsigned ld2, unsigned part) {
    const int t = t_last - i * per, left = it.len - t, m = left < per ? left : per;
    const unsigned off[NJ] = {x[0], x[1], x[2], x[3]};
    loads_to_lds16(rsrc_words(rows + (it.start + t) * ld + (long long)hk * G * D,
                              i < n ? (unsigned)(m - 1) * ld2 + 2u * D * G : 0),
                   lds0 + 2u * (kSlot * (unsigned)(i & (kRing - 1)) + part), off);
  };
  auto fetch_q = [&](int i, u32x4 off) { fetch(i, off, (const bf16_t*)p.q, p.q_ld, qld2, 0); };
  auto fetch_do = [&](int i, u32x4 off) {
    fetch(i, off, (const bf16_t*)p.dout, (long long)Hq * D, old2, kRows * DP);
  };
  auto fetch_stats = [&](int i, unsigned off) {  // lse (even wavefronts) or delta (odd ones)
    const int t = t_last - i * per, left = it.len - t, m = left < per ? left : per;
    load_to_lds4(rsrc_words(p.stats + 2 * ((it.start + t) * Hq + hk * G) + (w & 1) * G,
                            i < n ? (unsigned)(m - 1) * 8u * Hq + 4u * G : 0),
                 lds1 + 512u * (unsigned)(i & (kRing - 1)), off);
  };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) {
    fetch_q(i, offs[0][tid]);
    fetch_do(i, offs[1][tid]);
    fetch_stats(i, soffs[tid]);
  }

  u32x4 kf[KS], vf[KS];
  {
    const long long tok = it.start + (key < it.len ? key : it.len - 1);
    load_row(kf, (const bf16_t*)p.k + tok * p.k_ld + hk * D, D, h);
    load_row(vf, (const bf16_t*)p.v + tok * p.v_ld + hk * D, D, h);
    clear_past(kf, D, h);
    clear_past(vf, D, h);
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
  const float cs = p.scale * kLog2e;

  wait_loads<0>();  // k and v too: no wait for them remains for the loop
  lds_barrier();
  u32x4 f[PF];
#pragma unroll
  for (int i = 0; i < PF; ++i) f[i] = attn_frag<DP>(ring, lane, 0, i);
  int i0 = 0;
  for (; i0 < na; ++i0) {
    wait_loads<kLoads>();  // all but stage i0 + 2: the next is there
    lds_barrier();         // everyone's; and the last one's slot is free
    const bf16_t* sq = ring + (i0 & (kRing - 1)) * kSlot;
    const bf16_t* so = sq + kRows * DP;
    const bf16_t* sn = ring + ((i0 + 1) & (kRing - 1)) * kSlot;
    const float* ss = stats + 128 * (i0 & (kRing - 1));
    const AttnLane ln = fresh(lane);
    auto tr = [&](const bf16_t* x, int i) { return attn_frag_tr<DP>(x, ln, 16 * (i / DB), i % DB); };
    auto stat = [&](int i) { return *(const f32x4*)(ss + 8 * i + 4 * h); };
    f32x16 s = zero16(), dp = zero16();
    f32x4 st;  // lse, then delta, of four rows
    u32x4 pw[2], ds[2], off;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      s = mma32(f[i % PF], kf[i], s);
      f[i % PF] = i + PF < KS ? attn_frag<DP>(sq, ln, 0, i + PF) : attn_frag<DP>(so, ln, 0, i + PF - KS);
      if (i == KS - PF) st = stat(0);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int t = t_last - i0 * per;
    if (t < kw + 31) {  // row r is token t + r / G: before the key if r < (key - t) G
      int first = lane_id() & 31;
      asm volatile("" : "+v"(first));
      first = (kw + first - t) * G;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i / 4) + 4 * h + i % 4 < first) s[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      dp = mma32(f[i % PF], vf[i], dp);
      f[i % PF] = i + PF < KS ? attn_frag<DP>(so, ln, 0, i + PF) : tr(so, i + PF - KS);
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], cs, -st[i % 4]));
      if (i % 4 == 3) st = stat(i < 15 ? i / 4 + 1 : 8);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) pw[k] = pack8_of(s, k);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      dv[i % DB] = mma32(f[i % PF], pw[i / DB], dv[i % DB]);
      f[i % PF] = i + PF < KS ? tr(so, i + PF) : tr(sq, i + PF - KS);
      s[i] *= dp[i] + st[i % 4];
      if (i % 4 == 3 && i < 15) st = stat(8 + i / 4 + 1);
      if (i == KS - PF) off = offs[0][tid];
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) ds[k] = pack8_of(s, k);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      dk[i % DB] = mma32(f[i % PF], ds[i / DB], dk[i % DB]);
      f[i % PF] = i + PF < KS ? tr(sq, i + PF) : attn_frag<DP>(sn, ln, 0, i + PF - KS);
      if (i == 1) {
        fetch_q(i0 + kRing - 1, off);
        off = offs[1][tid];
      }
      if (i == 6) {
        fetch_do(i0 + kRing - 1, off);
        off[0] = soffs[tid];
      }
      if (i == 10) fetch_stats(i0 + kRing - 1, off[0]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  for (; i0 < n; ++i0) {  // rows before every key of the wavefront: its part of the loads
    wait_loads<kLoads>();
    lds_barrier();
    fetch_q(i0 + kRing - 1, offs[0][tid]);
    fetch_do(i0 + kRing - 1, offs[1][tid]);
    fetch_stats(i0 + kRing - 1, soffs[tid]);
  }
  wait_loads<0>();
  if (key >= it.len) return;
  const long long at = ((it.start + key) * Hkv + hk) * D;
  if (p.splits > 1 && it.share == 0 && h == 0) p.shares[at / D] = it.shares;
  if (it.shares > 1) {
    const long long ps = (long long)it.share * p.tokens * Hkv * D + at;
    store_part<DB>(p.part_k + ps, dk, p.scale, D, h);
    store_part<DB>(p.part_v + ps, dv, 1.f, D, h);
  } else {
    store_rows<DB>((bf16_t*)p.dk + at, dk, p.scale, D, h);
    store_rows<DB>((bf16_t*)p.dv + at, dv, 1.f, D, h);
  }
}

// The shares' sums, 8 elements a thread, of tiles with more than one.  Bound by its bytes: 4 a share
// and 2 out.
__global__ __launch_bounds__(256) void attn_dkv_sum_kernel(AttnParams p, long long n) {
  const long long i = 8 * ((long long)blockIdx.x * 256 + threadIdx.x);
  if (i >= n) return;
  const int shares = p.shares[i / p.D];
  if (shares < 2) return;
  const float* src = blockIdx.y ? p.part_v : p.part_k;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < shares; ++s)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4 y = *(const f32x4*)(src + s * n + i + 4 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * j + e] += y[e];
    }
  *(u32x4*)((bf16_t*)(blockIdx.y ? p.dv : p.dk) + i) =
      u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
}

}  // namespace

int attn_dkv_tile_tokens() { return kDkvKeys; }

// How tiles of keys are shared.  The time is estimated, in stages, for sequences of equal length and
// each number m of tiles' rows (4 g stages each) in a share: workgroups, one a compute unit, make
// a round; shares that fill one or two end with the longest, more of them even out up to half a share,
// and whole tiles, which go longest first, altogether; around a workgroup's stages pass
// 16 more, and its partial sums take a twentieth.  Of 1 to 16 shares that takes the best within 1%
// in 20 of 21 layouts and lengths (heads of 64, 128 and 256, one sequence of 700 to 16,000 tokens and
// five of 3,001), within 5% in all; they are 1.0 to 4.2 times as fast as whole tiles: 4,000 tokens of
// 16/2 heads of 256, both passes, 1,704 us whole, 496 in 7 shares, 620 in 8.  Partial sums take 512 MiB
// at most.
DkvPlan attn_dkv_plan(long long units, long long T, long long N, int G, long long row_bytes) {
  DkvPlan plan{1, 0};
  if (N > 64 || T == 0 || units == 0) return plan;  // shares are found by lanes that hold a sequence each
  const long long seqs = N > 0 ? N : 1, nt = (T / seqs + kDkvKeys - 1) / kDkvKeys;
  const long long longest = (T + kDkvKeys - 1) / kDkvKeys;  // of sequences of any lengths
  long long room = (512ll << 20) / row_bytes;
  room = room < 16 ? room : 16;
  units *= seqs;
  const double tile = 4. * G, even = (double)(units * nt) * nt * tile / (2 * kComputeUnits);
  double best = 0;
  for (long long s = 1; s <= room && s <= nt; ++s) {
    const long long m = (nt + s - 1) / s;
    long long shares = 0, parts = 0;
    for (long long q = 0; q * m < nt; ++q) {
      const long long n = (q + 1) * (nt - q * m < m ? nt - q * m : m);
      shares += n;
      parts += q > 0 ? n : 0;
    }
    const long long rounds = (units * shares + kComputeUnits - 1) / kComputeUnits;
    const double each = m * tile;
    const double ends = s == 1 ? even : (rounds <= 2 ? rounds * each : even + each / 2);
    const double cost = (ends > each ? ends : each) + 16. * rounds + units * parts / 20.;
    if (s == 1 || cost < best) {
      best = cost;
      const long long most = (longest + m - 1) / m;
      plan.splits = s == 1 ? 1 : (int)(most < room ? most : room);
      plan.tiles = (int)m;
    }
  }
  return plan;
}

hipError_t launch_attn_dkv(const AttnParams& p, hipStream_t stream) {
  const long long ranks = attn_ranks(p, kDkvKeys) * p.splits, units = (long long)(p.cu ? 1 : p.N) * p.Hkv;
  const unsigned grid = (unsigned)attn_grid(units, ranks);
  if (p.D <= 128)
    launch_attn_dkv_narrow(p, grid, (int)ranks, stream);
  else
    attn_dkv_wide_kernel<256><<<grid, kNT, 0, stream>>>(p, (int)ranks);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const long long n = p.tokens * p.Hkv * p.D;
  attn_dkv_sum_kernel<<<dim3((unsigned)((n + 2047) / 2048), 2), 256, 0, stream>>>(p, n);
  return hipGetLastError();
}

}  // namespace omx
