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

constexpr int kNW = 4, kNT = 64 * kNW, kBM = 128, kBN = 64;

// the same column in fp32, as one of the shares of a sum
template <int DB>
__device__ __forceinline__ void store_part(float* row, const f32x16 (&x)[DB], float f, int D, int h) {
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * d + 8 * g + 4 * h;
      if (col < D) *(f32x4*)(row + col) = f32x4{x[d][4 * g] * f, x[d][4 * g + 1] * f, x[d][4 * g + 2] * f, x[d][4 * g + 3] * f};
    }
}

// sum of the products of two rows' 8 bf16 elements
__device__ __forceinline__ float dot8(u32x4 a, u32x4 b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, (uint32_t)a[i]),
                                        __builtin_bit_cast(bf16x2_t, (uint32_t)b[i]), s, false);
  return s;
}

// ------------------------------------------------------------------------------------ dq
template <int DP>
__global__ __launch_bounds__(kNT) __attribute__((amdgpu_waves_per_eu(DP == 256 ? 1 : 2)))
void attn_dq_kernel(AttnParams p, int ranks) {
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int NJ = kBN * DP / 8 / 64 / kNW;
  __shared__ __align__(16) bf16_t sK0[kBN * DP], sK1[kBN * DP], sV0[kBN * DP], sV1[kBN * DP];

  const int tid = threadIdx.x, l = tid & 63, h = l >> 5, c = l & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
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

  u32x4 q[KS], dout[KS];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = 16 * s + 8 * h;
    q[s] = dout[s] = u32x4{0, 0, 0, 0};
    if (live && d < D) {
      q[s] = *(const u32x4*)((const bf16_t*)p.q + tok * p.q_ld + (long long)(hk * G + rg) * D + d);
      dout[s] = *(const u32x4*)((const bf16_t*)p.dout + at * D + d);
      delta += dot8(dout[s], *(const u32x4*)((const bf16_t*)p.o + at * D + d));
      if (p.o_rest) delta += dot8(dout[s], *(const u32x4*)((const bf16_t*)p.o_rest + at * D + d));
    }
  }
  delta = sum_halves(delta);
  const float lse2 = live ? p.lse[at] * kLog2e : INFINITY;  // idle rows: weights of 0
  if (live && h == 0) p.delta[at] = delta;

  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = zero16();
  const float cs = p.scale * kLog2e;
  const int nkt = (t0 + nt + kBN - 1) / kBN;

  int srow[NJ], sseg[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    srow[j] = stage_row<DP, kNW>(w, j);
    sseg[j] = stage_seg<DP>(srow[j]);
  }
  const unsigned kld2 = (unsigned)(p.k_ld * 2), vld2 = (unsigned)(p.v_ld * 2);
  auto stage = [&](int kt, bf16_t* sk, bf16_t* sv) {
    const int left = it.len - kt * kBN, n = left < kBN ? left : kBN;  // rows past the sequence
    const long long a = it.start + (long long)kt * kBN;               //   read as zeros
    const auto kr = buf_rsrc((const bf16_t*)p.k + a * p.k_ld + hk * D, (unsigned)(n - 1) * kld2 + 2u * D);
    const auto vr = buf_rsrc((const bf16_t*)p.v + a * p.v_ld + hk * D, (unsigned)(n - 1) * vld2 + 2u * D);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int i = w + kNW * j;
      const bool in = 8 * sseg[j] < D;
      const unsigned so = 16u * (unsigned)sseg[j];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void*)(sk + 512 * i), 16,
                                               in ? (unsigned)srow[j] * kld2 + so : kDropOffset, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void*)(sv + 512 * i), 16,
                                               in ? (unsigned)srow[j] * vld2 + so : kDropOffset, 0, 0, 0);
    }
  };
  auto compute = [&](int kt, const bf16_t* sk, const bf16_t* sv) {
    const int key0 = kt * kBN;
    if (key0 > w_hi) return;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int k = 0; k < KS; ++k) s = mma32(attn_frag<DP>(sk, 32 * b, k), q[k], s);
#pragma unroll
      for (int k = 0; k < KS; ++k) dp = mma32(attn_frag<DP>(sv, 32 * b, k), dout[k], dp);
      if (key0 + 32 * b + 31 > w_lo) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 32 * b + 8 * (i / 4) + 4 * h + i % 4 > pos) s[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[i], cs, -lse2));
        s[i] = x * (dp[i] - delta);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const u32x4 ds = pack8_of(s, k);
#pragma unroll
        for (int d = 0; d < DB; ++d) dq[d] = mma32(attn_frag_tr<DP>(sk, 32 * b + 16 * k, d), ds, dq[d]);
      }
    }
  };
  stage(0, sK0, sV0);
  for (int kt = 0; kt < nkt; kt += 2) {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    lds_barrier();
    if (kt + 1 < nkt) stage(kt + 1, sK1, sV1);
    compute(kt, sK0, sV0);
    if (kt + 1 >= nkt) break;
    __builtin_amdgcn_s_waitcnt(0x0F70);
    lds_barrier();
    if (kt + 2 < nkt) stage(kt + 2, sK0, sV0);
    compute(kt + 1, sK1, sV1);
  }
  if (live) store_rows<DB>((bf16_t*)p.dq + at * D, dq, p.scale, D, h);
}

// ------------------------------------------------------------------------------------ dk, dv
constexpr int kKeys = 32 * kNW;  // keys of a workgroup's tile
constexpr int kRows = 64;        // rows of a stage

template <int DP, bool DK, bool DV>
__global__ __launch_bounds__(kNT) __attribute__((amdgpu_waves_per_eu(DP == 256 || (DK && DV) ? 1 : 2)))
void attn_dkv_kernel(AttnParams p, int ranks) {
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int NJ = kRows * DP / 8 / 64 / kNW;
  __shared__ __align__(16) bf16_t sQ0[kRows * DP], sQ1[kRows * DP], sO0[kRows * DP], sO1[kRows * DP];
  __shared__ __align__(16) float sS0[2 * kRows], sS1[2 * kRows];  // lse and delta of a stage's rows

  const int tid = threadIdx.x, l = tid & 63, h = l >> 5, c = l & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.G, D = p.D, Hkv = p.Hkv, Hq = Hkv * G, per = kRows / G;

  int unit, rank;
  attn_place((int)blockIdx.x, (p.cu ? 1 : p.N) * Hkv, ranks, unit, rank);
  if (rank >= ranks) return;
  const int hk = unit % Hkv;
  AttnTile it;
  if (!attn_tile(p, unit / Hkv, rank, kKeys, it)) return;
  // the first tiles' keys are seen by most rows: those first
  const int k0 = (it.tiles - 1 - it.tile) * kKeys;
  // this share's rows: tokens [ta, tb) in whole stages
  int ta = k0, tb = it.len;
  if (p.splits > 1) {
    const int n = (it.len - k0 + per - 1) / per, each = (n + p.splits - 1) / p.splits;
    const int first = (int)blockIdx.y * each;
    ta = first < n ? k0 + first * per : it.len;
    tb = first + each < n ? ta + each * per : it.len;
  }
  const int key = k0 + 32 * w + c;
  const bool live = key < it.len;
  const long long tok = it.start + key;

  u32x4 kf[KS], vf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = 16 * s + 8 * h;
    kf[s] = vf[s] = u32x4{0, 0, 0, 0};
    if (live && d < D) {
      kf[s] = *(const u32x4*)((const bf16_t*)p.k + tok * p.k_ld + hk * D + d);
      if constexpr (DK) vf[s] = *(const u32x4*)((const bf16_t*)p.v + tok * p.v_ld + hk * D + d);
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
  const unsigned soff = l / G < per ? (unsigned)(l / G) * 4u * Hq + 4u * (unsigned)(l % G) : kDropOffset;
  auto stage = [&](int t, bf16_t* sq, bf16_t* so, float* ss) {
    const int left = it.len - t, n = left < per ? left : per;  // rows past the sequence read as
    const long long a = it.start + t;                          //   zeros: they add nothing
    const auto qr = buf_rsrc((const bf16_t*)p.q + a * p.q_ld + (long long)hk * G * D,
                             (unsigned)(n - 1) * qld2 + 2u * D * G);
    const auto dr = buf_rsrc((const bf16_t*)p.dout + (a * Hq + hk * G) * D, (unsigned)(n - 1) * old2 + 2u * D * G);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int i = w + kNW * j;
      const unsigned x = qoff[j], y = ooff[j];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(qr, (lds_void*)(sq + 512 * i), 16, x, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(dr, (lds_void*)(so + 512 * i), 16, y, 0, 0, 0);
    }
    if (w < 2) {
      const auto sr = buf_rsrc((w ? p.delta : p.lse) + a * Hq + hk * G, (unsigned)(n - 1) * 4u * Hq + 4u * G);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sr, (lds_void*)(ss + kRows * w), 4, soff, 0, 0, 0);
    }
  };
  auto compute = [&](int t, const bf16_t* sq, const bf16_t* so, const float* ss) {
    const int kw = k0 + 32 * w;
    if (t + per <= kw) return;  // every row is before every key of the wavefront
#pragma unroll
    for (int rb = 0; rb < kRows / 32; ++rb) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int k = 0; k < KS; ++k) s = mma32(attn_frag<DP>(sq, 32 * rb, k), kf[k], s);
#pragma unroll
      for (int k = 0; k < KS; ++k)
        if constexpr (DK) dp = mma32(attn_frag<DP>(so, 32 * rb, k), vf[k], dp);
      if (t < kw + 31) {  // row r is token t + r / G: before the key if r < (key - t) G
        const int first = (key - t) * G;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * rb + 8 * (i / 4) + 4 * h + i % 4 < first) s[i] = -INFINITY;
      }
      f32x16 ds;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 lse = *(const f32x4*)(ss + 32 * rb + 8 * j + 4 * h);
        const f32x4 del = *(const f32x4*)(ss + kRows + 32 * rb + 8 * j + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[4 * j + i] = __builtin_amdgcn_exp2f(fmaf(s[4 * j + i], cs, -lse[i] * kLog2e));
          ds[4 * j + i] = s[4 * j + i] * (dp[4 * j + i] - del[i]);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const u32x4 pb = pack8_of(s, k), db = pack8_of(ds, k);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          if constexpr (DV) dv[d] = mma32(attn_frag_tr<DP>(so, 32 * rb + 16 * k, d), pb, dv[d]);
          if constexpr (DK) dk[d] = mma32(attn_frag_tr<DP>(sq, 32 * rb + 16 * k, d), db, dk[d]);
        }
      }
    }
  };
  // from the last stage to the first: a unit's workgroups, which start together and see different
  // numbers of rows, then read the same rows at the same time, and its XCD's L2 serves most of them
  if (ta < tb) {
    int t = ta + (tb - ta - 1) / per * per;
    stage(t, sQ0, sO0, sS0);
    for (; t >= ta; t -= 2 * per) {
      __builtin_amdgcn_s_waitcnt(0x0F70);
      lds_barrier();
      if (t - per >= ta) stage(t - per, sQ1, sO1, sS1);
      compute(t, sQ0, sO0, sS0);
      if (t - per < ta) break;
      __builtin_amdgcn_s_waitcnt(0x0F70);
      lds_barrier();
      if (t - 2 * per >= ta) stage(t - 2 * per, sQ0, sO0, sS0);
      compute(t - per, sQ1, sO1, sS1);
    }
  }
  if (!live) return;
  const long long at = (tok * Hkv + hk) * D;
  if (p.splits > 1) {
    const long long ps = (long long)blockIdx.y * p.tokens * Hkv * D + at;
    if constexpr (DK) store_part<DB>(p.part_k + ps, dk, p.scale, D, h);
    if constexpr (DV) store_part<DB>(p.part_v + ps, dv, 1.f, D, h);
  } else {
    if constexpr (DK) store_rows<DB>((bf16_t*)p.dk + at, dk, p.scale, D, h);
    if constexpr (DV) store_rows<DB>((bf16_t*)p.dv + at, dv, 1.f, D, h);
  }
}

// The shares' sums, 8 elements a thread.  Bound by its bytes: 4 a share and 2 out.
__global__ __launch_bounds__(256) void attn_dkv_sum_kernel(const float* pk, const float* pv, bf16_t* dk,
                                                           bf16_t* dv, int splits, long long n) {
  const long long i = 8 * ((long long)blockIdx.x * 256 + threadIdx.x);
  if (i >= n) return;
  const float* src = blockIdx.y ? pv : pk;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4 y = *(const f32x4*)(src + s * n + i + 4 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * j + e] += y[e];
    }
  *(u32x4*)((blockIdx.y ? dv : dk) + i) =
      u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
}

template <int DP>
void dkv(const AttnParams& p, int ranks, dim3 grid, hipStream_t stream) {
  attn_dkv_kernel<DP, false, true><<<grid, kNT, 0, stream>>>(p, ranks);
  attn_dkv_kernel<DP, true, false><<<grid, kNT, 0, stream>>>(p, ranks);
}

}  // namespace

int attn_dkv_tile_tokens() { return kKeys; }

hipError_t launch_attn_dq(const AttnParams& p, hipStream_t stream) {
  const long long ranks = attn_ranks(p, kBM / p.G), units = (long long)(p.cu ? 1 : p.N) * p.Hkv;
  const unsigned grid = (unsigned)attn_grid(units, ranks);
  if (p.D <= 64) attn_dq_kernel<64><<<grid, kNT, 0, stream>>>(p, (int)ranks);
  else if (p.D <= 128) attn_dq_kernel<128><<<grid, kNT, 0, stream>>>(p, (int)ranks);
  else attn_dq_kernel<256><<<grid, kNT, 0, stream>>>(p, (int)ranks);
  return hipGetLastError();
}

int attn_dkv_splits(long long units, long long T, long long N, int G) {
  // two workgroups for each compute unit, and no share below eight stages of rows on average
  const long long tiles = units * ((T + kKeys - 1) / kKeys + (N > 0 ? N - 1 : 0));
  const long long most = T / (N > 0 ? N : 1) * G / (8 * kRows);
  long long s = 512 / (tiles > 0 ? tiles : 1);
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 8 ? 8 : s));
}

hipError_t launch_attn_dkv(const AttnParams& p, hipStream_t stream) {
  const long long ranks = attn_ranks(p, kKeys), units = (long long)(p.cu ? 1 : p.N) * p.Hkv;
  const dim3 grid((unsigned)attn_grid(units, ranks), (unsigned)p.splits);
  if (p.D <= 64) dkv<64>(p, (int)ranks, grid, stream);
  else if (p.D <= 128) dkv<128>(p, (int)ranks, grid, stream);
  else dkv<256>(p, (int)ranks, grid, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const long long n = p.tokens * p.Hkv * p.D;
  attn_dkv_sum_kernel<<<dim3((unsigned)((n + 2047) / 2048), 2), 256, 0, stream>>>(
      p.part_k, p.part_v, (bf16_t*)p.dk, (bf16_t*)p.dv, p.splits, n);
  return hipGetLastError();
}

}  // namespace omx
