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

#ifndef FRESH
#define FRESH fresh
#endif
namespace omx {
namespace {

constexpr int kNW = 4, kNT = 64 * kNW, kBM = 128, kBN = 64;

// The same for heads of 256, ...
constexpr int kWideRows = 64;
template <int DP, int KB, bool DK, bool DV>
__global__ __launch_bounds__(kNT) __attribute__((amdgpu_waves_per_eu(DP == 256 || (DK && DV) || KB > 1 ? 1 : 2)))
void attn_dkv_wide_kernel(AttnParams p, int ranks) {
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int NJ = kWideRows * DP / 8 / 64 / kNW;
  __shared__ __align__(16) bf16_t sQ0[kWideRows * DP], sQ1[kWideRows * DP], sO0[kWideRows * DP], sO1[kWideRows * DP];
  __shared__ __align__(16) float sS0[2 * kWideRows], sS1[2 * kWideRows];  // lse and delta of a stage's rows

  const int tid = threadIdx.x, l = tid & 63, h = l >> 5, c = l & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AttnLane lane = attn_lane<DP>();
  const int G = p.G, D = p.D, Hkv = p.Hkv, Hq = Hkv * G, per = kWideRows / G;

  int unit, rank;
  attn_place((int)blockIdx.x, (p.cu ? 1 : p.N) * Hkv, ranks, unit, rank);
  if (rank >= ranks) return;
  const int hk = unit % Hkv;
  constexpr int kKeys = kDkvKeys;
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
  const int kw = k0 + 32 * KB * w;  // the wavefront's first key

  // with two blocks of keys a wavefront, v stays in LDS: its fragments would not fit beside the
  // sums, and two blocks a read of q and do leave the LDS time for them
  constexpr bool VL = KB == 2 && DP == 128;
  __shared__ __align__(16) bf16_t sV[VL ? kKeys * DP : 8];
  u32x4 kf[KB][KS], vf[KB][KS];
  f32x16 dk[KB][DB], dv[KB][DB];
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    const int key = kw + 32 * b + c;
    const long long tok = it.start + key;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * h;
      kf[b][s] = vf[b][s] = u32x4{0, 0, 0, 0};
      if (key < it.len && d < D) {
        kf[b][s] = *(const u32x4*)((const bf16_t*)p.k + tok * p.k_ld + hk * D + d);
        if constexpr (DK) vf[b][s] = *(const u32x4*)((const bf16_t*)p.v + tok * p.v_ld + hk * D + d);
      }
      if constexpr (VL)  // read back by this wavefront alone
        *(u32x4*)(sV + (32 * (KB * w + b) + c) * DP + (((2 * s + h) ^ attn_swz<DP>(c)) << 3)) = vf[b][s];
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[b][d] = dv[b][d] = zero16();
  }
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
  const unsigned soff = l / G < per ? (unsigned)(l / G) * 8u * Hq + 4u * (unsigned)(l % G) : kDropOffset;
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
      const auto sr = buf_rsrc(p.stats + 2 * (a * Hq + hk * G) + w * G, (unsigned)(n - 1) * 8u * Hq + 4u * G);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sr, (lds_void*)(ss + kWideRows * w), 4, soff, 0, 0, 0);
    }
  };
  auto compute = [&](int t, const bf16_t* sq, const bf16_t* so, const float* ss) {
    if (t + per <= kw) return;  // every row is before every key of the wavefront
#ifdef U1
#pragma unroll 1
#else
#pragma unroll
#endif
    for (int rb = 0; rb < kWideRows / 32; ++rb) {
      const AttnLane ln = FRESH(lane);
      f32x16 s[KB], dp[KB];
#pragma unroll
      for (int b = 0; b < KB; ++b) s[b] = dp[b] = zero16();
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 a = attn_frag<DP>(sq, ln, 32 * rb, k);
#pragma unroll
        for (int b = 0; b < KB; ++b) s[b] = mma32(a, kf[b][k], s[b]);
      }
      if constexpr (DK) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const u32x4 a = attn_frag<DP>(so, ln, 32 * rb, k);
#pragma unroll
          for (int b = 0; b < KB; ++b)
            dp[b] = mma32(a, VL ? attn_frag<DP>(sV, ln, 32 * (KB * w + b), k) : vf[b][k], dp[b]);
        }
      }
      if (t < kw + 32 * KB - 1) {  // row r is token t + r / G: before the key if r < (key - t) G
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const int first = (kw + 32 * b + c - t) * G;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * rb + 8 * (i / 4) + 4 * h + i % 4 < first) s[b][i] = -INFINITY;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 lse = *(const f32x4*)(ss + 32 * rb + 8 * j + 4 * h);
        const f32x4 del = *(const f32x4*)(ss + kWideRows + 32 * rb + 8 * j + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float l2 = lse[i];
#pragma unroll
          for (int b = 0; b < KB; ++b) {
            s[b][4 * j + i] = __builtin_amdgcn_exp2f(fmaf(s[b][4 * j + i], cs, -l2));
            if constexpr (DK) dp[b][4 * j + i] = s[b][4 * j + i] * (dp[b][4 * j + i] + del[i]);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        u32x4 pb[KB], db[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          if constexpr (DV) pb[b] = pack8_of(s[b], k);
          if constexpr (DK) db[b] = pack8_of(dp[b], k);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          if constexpr (DV) {
            const u32x4 a = attn_frag_tr<DP>(so, ln, 32 * rb + 16 * k, d);
#pragma unroll
            for (int b = 0; b < KB; ++b) dv[b][d] = mma32(a, pb[b], dv[b][d]);
          }
          if constexpr (DK) {
            const u32x4 a = attn_frag_tr<DP>(sq, ln, 32 * rb + 16 * k, d);
#pragma unroll
            for (int b = 0; b < KB; ++b) dk[b][d] = mma32(a, db[b], dk[b][d]);
          }
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
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    const int key = kw + 32 * b + c;
    if (key >= it.len) continue;
    const long long at = ((it.start + key) * Hkv + hk) * D;
    if (p.splits > 1) {
      const long long ps = (long long)blockIdx.y * p.tokens * Hkv * D + at;
      if constexpr (DK) store_part<DB>(p.part_k + ps, dk[b], p.scale, D, h);
      if constexpr (DV) store_part<DB>(p.part_v + ps, dv[b], 1.f, D, h);
    } else {
      if constexpr (DK) store_rows<DB>((bf16_t*)p.dk + at, dk[b], p.scale, D, h);
      if constexpr (DV) store_rows<DB>((bf16_t*)p.dv + at, dv[b], 1.f, D, h);
    }
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

}  // namespace

int attn_dkv_tile_tokens() { return kDkvKeys; }

int attn_dkv_splits(long long units, long long T, long long N, int G) {
  // a workgroup for each compute unit, and no share below eight stages of rows on average
  const long long tiles = units * ((T + kDkvKeys - 1) / kDkvKeys + (N > 0 ? N - 1 : 0));
  const long long most = T / (N > 0 ? N : 1) * G / (8 * kWideRows);
  long long s = 256 / (tiles > 0 ? tiles : 1);
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 8 ? 8 : s));
}

hipError_t launch_attn_dkv(const AttnParams& p, hipStream_t stream) {
  const long long ranks = attn_ranks(p, kDkvKeys), units = (long long)(p.cu ? 1 : p.N) * p.Hkv;
  const dim3 grid((unsigned)attn_grid(units, ranks), (unsigned)p.splits);
  if (p.D <= 128)
    launch_attn_dkv_narrow(p, grid, (int)ranks, stream);
  else
    attn_dkv_wide_kernel<256, 1, true, true><<<grid, kNT, 0, stream>>>(p, (int)ranks);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const long long n = p.tokens * p.Hkv * p.D;
  attn_dkv_sum_kernel<<<dim3((unsigned)((n + 2047) / 2048), 2), 256, 0, stream>>>(
      p.part_k, p.part_v, (bf16_t*)p.dk, (bf16_t*)p.dv, p.splits, n);
  return hipGetLastError();
}

}  // namespace omx
