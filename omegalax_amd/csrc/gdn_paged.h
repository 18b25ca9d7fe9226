// The decode step over a paged cache: what its kernels for bf16 and for 8 bits share.
#pragma once

#include <climits>

#include "gdn_attn.h"

namespace omx {

typedef const __attribute__((address_space(4))) int32_t const_i32;

// C += A(16x16) B(16x16), contraction of 16 keys
__device__ __forceinline__ f32x4 mma_pv(u32x2 a, u32x2 b, f32x4 c) { return mma16k16(a, b, c); }

constexpr int kDecNW = 4;
template <int DP> constexpr int kStageKeys = 4096 / DP;  // 64, 32, 16 keys

// A sequence's keys that its next token sees, in stages of `sk`: those it holds and the new one's, at
// position `held`.  With a window the stages are counted without the `skip` ones between the last of the
// sinks' and the window's first.
struct Seen {
  int keys, lo, sink_stages, skip, stages;  // lo: the window's first key; one stage at least: it writes the output
  __device__ __forceinline__ int at(int st) const { return st < sink_stages ? st : st + skip; }
};
template <bool WIN>
__device__ __forceinline__ Seen seen_of(const AttnParams& p, int held, int cap, int sk) {
  Seen x;
  x.keys = held < 0 ? 0 : (held < cap ? held + 1 : cap);
  x.lo = 0, x.sink_stages = 0, x.skip = 0;
  if constexpr (WIN) {
    const int pos = held < cap ? held : cap;
    x.lo = pos - p.window + 1;
    x.sink_stages = (int)((p.sinks + (long long)sk - 1) / sk);
    x.skip = x.lo / sk > x.sink_stages ? x.lo / sk - x.sink_stages : 0;
  }
  const int n = (x.keys + sk - 1) / sk - x.skip;
  x.stages = n < 1 ? 1 : n;
  return x;
}
template <bool WIN>
__device__ __forceinline__ int stages_of(const AttnParams& p, int held, int cap, int sk) {
  return seen_of<WIN>(p, held, cap, sk).stages;
}

// Stages of each range: equal shares, but no less than eight, two for each wavefront over a cache of bf16 and one
// for each of the eight in 8 bits.  (There two cost up to a fifth more: 8,000 keys of 8/8 heads of 64 16.7 us, with
// 16 stages a range 20.3; 4 x 4,000 keys of 16/4 heads of 128 19.4 and 21.6.)
__device__ __forceinline__ int range_stages(int all, int splits) {
  const int per = (all + splits - 1) / splits;
  return per > 2 * kDecNW ? per : 2 * kDecNW;
}

// The range of workgroup wg, of p.splits: stages [x, x1) of all sequences', from stage st0 of sequence b
// on; false past the last.
template <bool WIN>
__device__ __forceinline__ bool decode_range(const AttnParams& p, int wg, int cap, int sk, int& b, int& st0, int& x,
                                             int& x1) {
  const int l = lane_id();
  // lane n holds the stages of sequence n, n + 64, ..: the first 64 are read once
  const int v0 = l < p.N ? stages_of<WIN>(p, p.held[l], cap, sk) : 0;
  int v = v0;
  for (int n = l + 64; n < p.N; n += 64) v += stages_of<WIN>(p, p.held[n], cap, sk);
  const int all = wave_total(v), per = range_stages(all, p.splits);
  if ((long long)wg * per >= all) return false;
  x = wg * per;
  x1 = x + per < all ? x + per : all;
  v = v0;
  for (int n0 = 0, base = 0;;) {  // x < all: some 64 sequences hold it
    const int upto = base + wave_scan(v);
    const unsigned long long past = __ballot(upto > x);
    if (past) {
      const int s = __ffsll(past) - 1;
      b = n0 + s;
      st0 = x - __builtin_amdgcn_readlane(upto - v, s);
      return true;
    }
    base = __builtin_amdgcn_readlane(upto, 63);
    n0 += 64;
    v = n0 + l < p.N ? stages_of<WIN>(p, p.held[n0 + l], cap, sk) : 0;
  }
}

namespace {
// Joins a row's segments, with W of a workgroup's four wavefronts on one row.
template <int DP, int W, bool WIN, int SK>
__global__ __launch_bounds__(256) void decode_join_kernel(AttnParams p) {
  constexpr int E = DP / 64;
  typedef float fE __attribute__((ext_vector_type(E)));
  __shared__ float sAcc[4][DP];
  const int l = lane_id(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = w % W;
  const int Hq = p.Hkv * p.G;
  const int rows = p.N * Hq, row = (int)blockIdx.x * (4 / W) + w / W;
  const bool live = row < rows;
  const int b = live ? row / Hq : 0, head = live ? row % Hq : 0;
  const int cap = p.table_w * p.page, nst = stages_of<WIN>(p, p.held[b], cap, SK);
  int v = 0, y = 0;
  for (int n = l; n < p.N; n += 64) {
    const int x = stages_of<WIN>(p, p.held[n], cap, SK);
    v += x;
    if (n < b) y += x;
  }
  const int before = wave_total(y), per = range_stages(wave_total(v), p.splits);
  const int w0 = before / per, segs = live ? (before + nst - 1) / per - w0 + 1 : 1;
  if (segs == 1 && W == 1) return;  // written already (with W > 1 a whole workgroup agrees on it below)
  float M = -3e38f, den = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (segs > 1) {
    for (int s = l; s < segs; s += 64) M = fmaxf(M, p.part_ml[2 * ((long long)(w0 + s + b) * Hq + head)]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    for (int s0 = 0; s0 < segs; s0 += 64) {  // weights a lane, then the sums, eight reads in flight
      const int n = segs - s0 < 64 ? segs - s0 : 64;
      float a = 0.f;
      if (l < n) {
        const long long at = (long long)(w0 + s0 + l + b) * Hq + head;
        const float ls = p.part_ml[2 * at + 1];
        a = ls == 0.f ? 0.f : __builtin_amdgcn_exp2f(p.part_ml[2 * at] - M);
        den += a * ls;
      }
      for (int s = part; s < n; s += 8 * W) {
        fE v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int su = s + W * u < n ? s + W * u : n - 1;
          v[u] = *(const fE*)(p.part_o + ((long long)(w0 + s0 + su + b) * Hq + head) * DP + E * l);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float as = __shfl(a, (s + W * u) & 63, 64);
          const float f = s + W * u < n ? as : 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += f * v[u][e];
        }
      }
    }
    den = wave_sum(den);
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) sAcc[w][E * l + e] = acc[e];
    __syncthreads();
    if (part != 0 || segs == 1) return;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int u = 1; u < W; ++u) acc[e] += sAcc[w + u][E * l + e];
  }
  const float inv = den > 0.f ? 1.f / den : (den == 0.f ? 0.f : den);
  bf16_t* op = (bf16_t*)p.o + (long long)row * DP + E * l;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = f2bf(acc[e] * inv);
}

template <int DP, bool WIN, int SK>
void launch_decode_join(const AttnParams& p, hipStream_t stream) {
  // a row has at most as many segments as its key head has workgroups; four wavefronts share a row
  // where there are few rows
  const unsigned rows = (unsigned)(p.N * p.Hkv * p.G);
  if (rows <= 512)
    decode_join_kernel<DP, 4, WIN, SK><<<rows, 256, 0, stream>>>(p);
  else
    decode_join_kernel<DP, 1, WIN, SK><<<(rows + 3) / 4, 256, 0, stream>>>(p);
}
}  // namespace

}  // namespace omx
