// The paged key-value cache: the append of new tokens and the decode step of one token a sequence.
#include <climits>

#include "gdn_attn.h"

namespace omx {
namespace {

typedef const __attribute__((address_space(4))) int32_t const_i32;

// C += A(16x16) B(16x16), contraction of 16 keys
__device__ __forceinline__ f32x4 mma_pv(u32x2 a, u32x2 b, f32x4 c) { return mma16k16(a, b, c); }

// ------------------------------------------------------------------------------------ append
// Token i of sequence n goes to position held[n] + i: page table[n, position / page], row
// position % page.  Both sides of a token's copy are rows of Hkv * D contiguous elements, so a
// wavefront copies whole tokens, 16 bytes a lane.  Bound by the bytes: each read and written once.
constexpr int kWriteTokens = 4;  // tokens per wavefront

__global__ __launch_bounds__(256) void kv_write_kernel(AttnParams p) {
  const int l = lane_id();
  const long long t0 = ((long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kWriteTokens;
  if (t0 >= p.tokens) return;
  const int segs = p.Hkv * p.D / 8;  // 16-byte segments of a token's row
  int end = 0;
  const bool lanes = p.cu && !p.plan;  // lane n holds sequence n's end
  if (lanes) {
    end = l + 1 < p.N ? p.cu[l + 1] : p.T;
    end = end < 0 ? 0 : (end > p.T ? p.T : end);
    end = wave_scan_max(end);
  }
#pragma unroll 1
  for (int i = 0; i < kWriteTokens; ++i) {
    const long long t = t0 + i;
    if (t >= p.tokens) return;
    int seq, at;
    if (lanes) {
      seq = __popcll(__ballot(l < p.N && end <= (int)t));
      at = (int)t - (seq > 0 ? __builtin_amdgcn_readlane(end, seq - 1) : 0);
    } else if (p.plan) {
      int lo = 0, hi = p.N;  // cu_plan[lo] <= t < cu_plan[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.cu_plan[mid] <= (int)t) lo = mid; else hi = mid;
      }
      seq = lo;
      at = (int)t - p.cu_plan[lo];
    } else {
      seq = (int)(t / p.T);
      at = (int)(t - (long long)seq * p.T);
    }
    const int held = p.held[seq];
    if (held < 0) continue;
    const long long pos = (long long)held + at;
    const long long slot = pos / p.page;
    if (slot >= p.table_w) continue;
    const int id = p.table[(long long)seq * p.table_w + slot];
    if (id < 0 || id >= p.n_pages) continue;
    const long long dst = ((long long)id * p.page + (pos - slot * p.page)) * p.Hkv * p.D;
    const u32x4* ks = (const u32x4*)((const bf16_t*)p.k + t * p.k_ld);
    const u32x4* vs = (const u32x4*)((const bf16_t*)p.v + t * p.v_ld);
    u32x4* kd = (u32x4*)((bf16_t*)p.k_pages + dst);
    u32x4* vd = (u32x4*)((bf16_t*)p.v_pages + dst);
    for (int s = l; s < segs; s += 64) {
      kd[s] = ks[s];
      vd[s] = vs[s];
    }
  }
}

// ------------------------------------------------------------------------------------ decode
// A workgroup's four wavefronts take turns at stages of a sequence's keys, each with its own LDS
// buffers and no barrier between stages.  Keys and values go from memory to LDS without passing
// registers, two stages deep (128 KiB in flight a compute unit), and are read once for all query
// heads of a key head, which are the columns of 16x16 products: S^T = K Q^T, O^T += V^T P^T.
// Bound by reading the cache.
//
// With `splits` = 1 a workgroup takes one sequence's key head.  Otherwise each key head has `splits`
// workgroups, and the sequences' stages, laid end to end, are cut into as many equal ranges: lengths
// may differ as they like, and all workgroups still end together.  A range's part of one sequence
// is a segment; workgroup w's of sequence b is kept at w + b (a staircase: each next segment has
// the next w or the next b), and the join adds up a sequence's.  A sequence in one segment needs none.
constexpr int kDecNW = 4;
template <int DP> constexpr int kStageKeys = 4096 / DP;  // 64, 32, 16 keys: 8 KiB of each of K, V

// stages of a sequence, one at least: it writes the output
__device__ __forceinline__ int stages_of(int held, int cap, int sk) {
  const int keys = held < 0 ? 0 : (held < cap ? held + 1 : cap);
  const int n = (keys + sk - 1) / sk;
  return n < 1 ? 1 : n;
}

// stages of each range: equal shares, but no less than two stages a wavefront
__device__ __forceinline__ int range_stages(int all, int splits) {
  const int per = (all + splits - 1) / splits;
  return per > 2 * kDecNW ? per : 2 * kDecNW;
}

template <int DP, int NQ>
__global__ __launch_bounds__(64 * kDecNW) __attribute__((amdgpu_waves_per_eu(1)))
void attn_decode_kernel(AttnParams p) {
  constexpr int SK = kStageKeys<DP>, NG = SK / 16;  // keys of a stage, its groups of 16
  constexpr int KS = DP / 32, DB = DP / 16;
  constexpr int NJ = 8;                             // staging instructions of K (and of V)
  constexpr int RPI = 512 / DP;                     // rows per instruction
  __shared__ __align__(16) bf16_t sK0[kDecNW][SK * DP], sK1[kDecNW][SK * DP];
  __shared__ __align__(16) bf16_t sV0[kDecNW][SK * DP], sV1[kDecNW][SK * DP];
  __shared__ float sM[kDecNW][16 * NQ], sL[kDecNW][16 * NQ];

  const int tid = threadIdx.x, l = tid & 63, g4 = l >> 4, r = l & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.G, Hkv = p.Hkv, Hq = Hkv * G;
  const int hk = (int)blockIdx.x % Hkv, wg = (int)blockIdx.x / Hkv;
  const int cap = p.table_w * p.page;

  // the range: stages [x, x1) of all sequences', from stage st0 of sequence b on
  int b = wg, st0 = 0, x = 0, x1 = INT_MAX;
  if (p.splits > 1) {
    // lane n holds the stages of sequence n, n + 64, ..: the first 64 are read once
    const int v0 = l < p.N ? stages_of(p.held[l], cap, SK) : 0;
    int v = v0;
    for (int n = l + 64; n < p.N; n += 64) v += stages_of(p.held[n], cap, SK);
    const int all = wave_total(v), per = range_stages(all, p.splits);
    if ((long long)wg * per >= all) return;
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
        break;
      }
      base = __builtin_amdgcn_readlane(upto, 63);
      n0 += 64;
      v = n0 + l < p.N ? stages_of(p.held[n0 + l], cap, SK) : 0;
    }
  }

  for (;;) {  // a segment a turn
  const_i32* table = (const_i32*)(p.table + (long long)b * p.table_w);
  const int held = ((const_i32*)p.held)[b];
  // keys: those held and the new one, at position `held`; past the table there is no room for it
  const int keys = held < 0 ? 0 : (held < cap ? held + 1 : cap);
  const int nst = stages_of(held, cap, SK);
  const int st1 = nst - st0 < x1 - x ? nst : st0 + (x1 - x);
  const bool alone = st0 == 0 && st1 == nst;

  u32x4 q[NQ][KS];
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      q[n][s] = u32x4{0, 0, 0, 0};
      if (16 * n + r < G)
        q[n][s] = *(const u32x4*)((const bf16_t*)p.q + b * p.q_ld + (long long)(hk * G + 16 * n + r) * DP + 32 * s + 8 * g4);
    }

  f32x4 o[NQ][DB];
  float m[NQ], ls[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = -1e30f;
    ls[n] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[n][d] = zero4();
  }
  const float cs = p.scale * kLog2e;
  const unsigned ld2 = (unsigned)(Hkv * DP * 2);

  // pages of a stage's groups of 16 keys, -1 where there is none
  struct Ids { int id[NG], off[NG]; };
  auto look = [&](int st) {
    Ids x;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int key = st * SK + 16 * g;
      const int slot = key / p.page;
      int id = key < keys ? table[slot] : -1;  // key < keys <= cap: the slot is in the table
      x.id[g] = id >= 0 && id < p.n_pages ? id : -1;
      x.off[g] = key - slot * p.page;
    }
    return x;
  };
  // returns the groups that hold keys
  auto stage = [&](const Ids& x, bf16_t* sk, bf16_t* sv) -> unsigned {
    unsigned have = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (x.id[g] < 0) continue;
      have |= 1u << g;
      const long long at = ((long long)x.id[g] * p.page + x.off[g]) * Hkv * DP + hk * DP;
#pragma unroll
      for (int j = 0; j < NJ / NG; ++j) {
        const int i = g * (NJ / NG) + j;
        const int row = RPI * i + l / (DP / 8);
        const unsigned lo = (unsigned)(row & 15) * ld2 + 16u * (unsigned)stage_seg<DP>(row);
        __builtin_amdgcn_global_load_lds((glob_void*)((const char*)((const bf16_t*)p.k_pages + at) + lo),
                                         (lds_void*)(sk + 512 * i), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((glob_void*)((const char*)((const bf16_t*)p.v_pages + at) + lo),
                                         (lds_void*)(sv + 512 * i), 16, 0, 0);
      }
    }
    return have;
  };

  auto compute = [&](int st, bf16_t* sk, bf16_t* sv, unsigned have) {
    const int key0 = st * SK;
    constexpr unsigned kAll = (1u << NG) - 1;
    const bool whole = have == kAll && key0 + SK < keys;  // every row a held key
    if (!whole) {
      // rows without a key are cleared (a weight of zero does not clear a NaN), and the new
      // token's row comes from the arguments: its page has no copy of it yet
      for (int i = l; i < SK * DP / 8; i += 64) {
        const int row = i / (DP / 8);
        if (key0 + row >= keys || !((have >> (row / 16)) & 1)) *(u32x4*)(sv + 8 * i) = u32x4{0, 0, 0, 0};
      }
      const int row = held - key0;
      if (row >= 0 && row < SK && held < cap && ((have >> (row / 16)) & 1)) {
        const int slot = held / p.page;
        const long long at = ((long long)table[slot] * p.page + (held - slot * p.page)) * Hkv * DP + hk * DP;
        if (l < DP / 8) {
          const u32x4 kx = *(const u32x4*)((const bf16_t*)p.k + b * p.k_ld + hk * DP + 8 * l);
          const u32x4 vx = *(const u32x4*)((const bf16_t*)p.v + b * p.v_ld + hk * DP + 8 * l);
          const int sl = row * DP + ((l ^ attn_swz<DP>(row)) << 3);
          *(u32x4*)(sk + sl) = kx;
          *(u32x4*)(sv + sl) = vx;
          *(u32x4*)((bf16_t*)p.k_pages + at + 8 * l) = kx;
          *(u32x4*)((bf16_t*)p.v_pages + at + 8 * l) = vx;
        }
      }
      wave_lds_fence();
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      f32x4 s[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        s[g] = zero4();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const u32x4 a = *(const u32x4*)(sk + (16 * g + r) * DP + (((4 * k + g4) ^ attn_swz<DP>(r)) << 3));
          s[g] = mma16(a, q[n][k], s[g]);
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!whole && (key0 + 16 * g + 4 * g4 + i >= keys || !((have >> g) & 1))) s[g][i] = -INFINITY;
          mx = fmaxf(mx, s[g][i]);
        }
      if (__any((mx - m[n]) * cs > 8.f)) {
        // the row's maximum over the four lanes that share it
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m[n], mx);
        const float a = __builtin_amdgcn_exp2f((m[n] - mn) * cs);
        m[n] = mn;
        ls[n] *= a;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][d][i] *= a;
      }
      const float mc = m[n] * cs;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[g][i] = __builtin_amdgcn_exp2f(fmaf(s[g][i], cs, -mc));
          ls[n] += s[g][i];
        }
        // the weights as two bf16 terms (off by at most 2^-16 together): a step is bound by its bytes, and
        // one term's rounding was half of its error (2.5e-3 against 64 bits, 1.7e-3 the output's own)
        const u32x2 pb = u32x2{pack_bf16(s[g][0], s[g][1]), pack_bf16(s[g][2], s[g][3])};
        const u32x2 pr = u32x2{pack_bf16(lo_part(s[g][0]), lo_part(s[g][1])), pack_bf16(lo_part(s[g][2]), lo_part(s[g][3]))};
        const int vr = 16 * g + 4 * g4 + (r >> 2);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const int col = 16 * d + 4 * (r & 3);
          const u32x2 a = ds_read_tr(sv + vr * DP + (((col >> 3) ^ attn_swz<DP>(vr)) << 3) + (col & 7));
          o[n][d] = mma_pv(a, pb, o[n][d]);
          o[n][d] = mma_pv(a, pr, o[n][d]);
        }
      }
    }
    // the buffers are free for the next stage once these reads are done
    __builtin_amdgcn_s_waitcnt(0xc07f);
  };

  // this wavefront's stages: st0 + w, then every fourth
  {
    constexpr unsigned kAll = (1u << NG) - 1;
    int st = st0 + w;
    unsigned have0 = 0, have1 = 0;
    Ids next;
    if (st < st1) have0 = stage(look(st), sK0[w], sV0[w]);
    if (st + kDecNW < st1) have1 = stage(look(st + kDecNW), sK1[w], sV1[w]);
    next = look(st + 2 * kDecNW);
    // a whole stage in flight behind the awaited one is 2 NJ instructions
    for (; st < st1; st += 2 * kDecNW) {
      if (st + kDecNW < st1 && have1 == kAll)
        __builtin_amdgcn_s_waitcnt(0x0F70 | (2 * NJ & 15) | ((2 * NJ >> 4) << 14));
      else
        __builtin_amdgcn_s_waitcnt(0x0F70);
      __builtin_amdgcn_wave_barrier();
      compute(st, sK0[w], sV0[w], have0);
      if (st + 2 * kDecNW < st1) {
        have0 = stage(next, sK0[w], sV0[w]);
        next = look(st + 3 * kDecNW);
      }
      if (st + kDecNW >= st1) break;
      if (st + 2 * kDecNW < st1 && have0 == kAll)
        __builtin_amdgcn_s_waitcnt(0x0F70 | (2 * NJ & 15) | ((2 * NJ >> 4) << 14));
      else
        __builtin_amdgcn_s_waitcnt(0x0F70);
      __builtin_amdgcn_wave_barrier();
      compute(st + kDecNW, sK1[w], sV1[w], have1);
      if (st + 3 * kDecNW < st1) {
        have1 = stage(next, sK1[w], sV1[w]);
        next = look(st + 4 * kDecNW);
      }
    }
  }

  // ---------------------------------------------------------------- the four wavefronts' sums
  // buffers 0 of K and V, 16 KiB a wavefront together, hold 16 rows of DP fp32 (NQ = 1)
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    ls[n] += __shfl_xor(ls[n], 16, 64);
    ls[n] += __shfl_xor(ls[n], 32, 64);
    if (g4 == 0) {
      sM[w][16 * n + r] = m[n] * cs;
      sL[w][16 * n + r] = ls[n];
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    // rows of DP fp32: row r in the first half of the columns in K's buffer, the rest in V's
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      float* dst = (float*)(d < DB / 2 ? sK0[w] : sV0[w]);
      *(f32x4*)(dst + r * (DP / 2) + 16 * (d % (DB / 2)) + 4 * g4) = o[n][d];
    }
    __syncthreads();
    const int rows = G - 16 * n < 16 ? G - 16 * n : 16;
    for (int i = tid; i < rows * DP / 4; i += 64 * kDecNW) {
      const int row = i / (DP / 4), col = 4 * (i % (DP / 4));
      float M = sM[0][16 * n + row];
#pragma unroll
      for (int x = 1; x < kDecNW; ++x) M = fmaxf(M, sM[x][16 * n + row]);
      f32x4 acc = zero4();
      float den = 0.f;
#pragma unroll
      for (int x = 0; x < kDecNW; ++x) {
        const float lx = sL[x][16 * n + row];
        const float a = lx == 0.f ? 0.f : __builtin_amdgcn_exp2f(sM[x][16 * n + row] - M);
        den += a * lx;
        const float* src = (const float*)(col < DP / 2 ? sK0[x] : sV0[x]);
        acc += a * *(const f32x4*)(src + row * (DP / 2) + (col % (DP / 2)));
      }
      const long long at = (long long)b * Hq + hk * G + 16 * n + row;
      if (!alone) {
        const long long ps = (long long)(wg + b) * Hq + hk * G + 16 * n + row;
        *(f32x4*)(p.part_o + ps * DP + col) = acc;
        if (col == 0) {
          p.part_ml[2 * ps] = M;
          p.part_ml[2 * ps + 1] = den;
        }
      } else {
        const float inv = den > 0.f ? 1.f / den : (den == 0.f ? 0.f : den);
        *(u32x2*)((bf16_t*)p.o + at * DP + col) =
            u32x2{pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
      }
    }
    __syncthreads();
  }
  x += st1 - st0;
  if (p.splits == 1 || x >= x1) return;
  st0 = 0;
  ++b;
  }
}

// Joins a row's segments, with W of a workgroup's four wavefronts on one row.
template <int DP, int W>
__global__ __launch_bounds__(256) void decode_join_kernel(AttnParams p) {
  constexpr int E = DP / 64, SK = kStageKeys<DP>;
  typedef float fE __attribute__((ext_vector_type(E)));
  __shared__ float sAcc[4][DP];
  const int l = lane_id(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = w % W;
  const int Hq = p.Hkv * p.G;
  const int rows = p.N * Hq, row = (int)blockIdx.x * (4 / W) + w / W;
  const bool live = row < rows;
  const int b = live ? row / Hq : 0, head = live ? row % Hq : 0;
  const int cap = p.table_w * p.page, nst = stages_of(p.held[b], cap, SK);
  int v = 0, y = 0;
  for (int n = l; n < p.N; n += 64) {
    const int x = stages_of(p.held[n], cap, SK);
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

template <int DP>
void decode_dp(const AttnParams& p, hipStream_t stream) {
  const unsigned grid = (unsigned)((p.splits > 1 ? p.splits : p.N) * p.Hkv);
  if (p.G <= 16)
    attn_decode_kernel<DP, 1><<<grid, 64 * kDecNW, 0, stream>>>(p);
  else
    attn_decode_kernel<DP, 2><<<grid, 64 * kDecNW, 0, stream>>>(p);
  if (p.splits == 1) return;
  // a row has at most as many segments as its key head has workgroups; four wavefronts share a row
  // where there are few rows
  const unsigned rows = (unsigned)(p.N * p.Hkv * p.G);
  if (rows <= 512)
    decode_join_kernel<DP, 4><<<rows, 256, 0, stream>>>(p);
  else
    decode_join_kernel<DP, 1><<<(rows + 3) / 4, 256, 0, stream>>>(p);
}

}  // namespace

bool paged_dims_supported(int D) { return D == 64 || D == 128 || D == 256; }

int kv_write_tokens() { return 4 * kWriteTokens; }

hipError_t launch_kv_write(const AttnParams& p, hipStream_t stream) {
  const long long per = kv_write_tokens();
  kv_write_kernel<<<(unsigned)((p.tokens + per - 1) / per), 256, 0, stream>>>(p);
  return hipGetLastError();
}

int decode_splits(long long N, long long Hkv, long long D, long long capacity) {
  // One workgroup a sequence and key head where a sequence is so short that the join costs more than
  // it saves (B=1, 4 key heads of 128, calls one after the other: 611 keys 14.4 us in one launch, 18.5 in
  // two, 1,500 keys 21.8 and 18.0), and for more than 1,024 sequences, where each row's join sums up all
  // their lengths.  Otherwise one for each compute unit: their buffers allow no second.  Equal ranges
  // against a workgroup each, 32/8 heads of 128: 64 sequences of 4,000 keys 190 us (187), between 1,000
  // and 7,000 207 (230), 63 of 1,000 and one of 30,000 84 (380); 1,024 of 100 199 (196), with one of
  // 30,000 244 (532).  16/2 heads of 256, sequences of 75 to 525 keys: 512 98 (81), 1,024 182 (156),
  // 4,096 723 (579).
  if (N > 1024 || capacity * D <= (1 << 17)) return 1;
  // stages are counted in 32 bits, and a range's end lies up to a range past the last
  if (N * (capacity / 16 + 1) > INT_MAX / 2) return 1;
  const long long s = kComputeUnits / Hkv;
  return (int)(s < 2 ? 1 : s);
}

hipError_t launch_attn_decode(const AttnParams& p, hipStream_t stream) {
  if (p.D == 64) decode_dp<64>(p, stream);
  else if (p.D == 128) decode_dp<128>(p, stream);
  else decode_dp<256>(p, stream);
  return hipGetLastError();
}

}  // namespace omx
