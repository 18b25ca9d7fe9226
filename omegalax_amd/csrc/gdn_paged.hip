// The paged key-value cache: the append of new tokens and the decode step of one token a sequence.
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
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(end, o, 64);
      if (l >= o && x > end) end = x;
    }
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
// One workgroup takes a sequence's key head, or a share of its keys (`splits` of them); its four
// wavefronts take turns at stages of 8192 / DP keys... each with its own LDS buffers and no
// barrier between stages.  Keys and values go from memory to LDS without passing registers, two
// stages deep (128 KiB in flight a compute unit), and are read once for all query heads, which
// are the columns of 16x16 products: S^T = K Q^T, O^T += V^T P^T.
constexpr int kDecNW = 4;
template <int DP> constexpr int kStageKeys = 4096 / DP;  // 64, 32, 16 keys: 8 KiB of each of K, V

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
  const int b = (int)blockIdx.x / Hkv, hk = (int)blockIdx.x % Hkv, split = (int)blockIdx.y;
  const int cap = p.table_w * p.page;
  const_i32* table = (const_i32*)(p.table + (long long)b * p.table_w);
  const int held = ((const_i32*)p.held)[b];
  // keys: those held and the new one, at position `held`; past the table there is no room for it
  const int keys = held < 0 ? 0 : (held < cap ? held + 1 : cap);
  const int nst = (keys + SK - 1) / SK, each = (nst + p.splits - 1) / p.splits;
  const int st0 = split * each < nst ? split * each : nst;
  const int st1 = st0 + each < nst ? st0 + each : nst;

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
        const u32x2 pb = u32x2{pack_bf16(s[g][0], s[g][1]), pack_bf16(s[g][2], s[g][3])};
        const int vr = 16 * g + 4 * g4 + (r >> 2);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const int col = 16 * d + 4 * (r & 3);
          const u32x2 a = ds_read_tr(sv + vr * DP + (((col >> 3) ^ attn_swz<DP>(vr)) << 3) + (col & 7));
          o[n][d] = mma_pv(a, pb, o[n][d]);
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
      if (p.splits > 1) {
        const long long ps = (long long)split * p.tokens * Hq + at;
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
    if (n + 1 < NQ) __syncthreads();
  }
}

template <int DP>
void decode_dp(const AttnParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)(p.N * p.Hkv), (unsigned)p.splits);
  if (p.G <= 16)
    attn_decode_kernel<DP, 1><<<grid, 64 * kDecNW, 0, stream>>>(p);
  else
    attn_decode_kernel<DP, 2><<<grid, 64 * kDecNW, 0, stream>>>(p);
}

}  // namespace

bool paged_dims_supported(int D) { return D == 64 || D == 128 || D == 256; }

hipError_t launch_kv_write(const AttnParams& p, hipStream_t stream) {
  const long long per = 4 * kWriteTokens;
  kv_write_kernel<<<(unsigned)((p.tokens + per - 1) / per), 256, 0, stream>>>(p);
  return hipGetLastError();
}

int decode_splits(long long units, long long capacity) {
  // two workgroups' worth of keys for each compute unit, none below 256 keys
  long long s = (512 + units - 1) / units;
  const long long most = (capacity + 255) / 256;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 256 ? 256 : s));
}

hipError_t launch_attn_decode(const AttnParams& p, hipStream_t stream) {
  if (p.D == 64) decode_dp<64>(p, stream);
  else if (p.D == 128) decode_dp<128>(p, stream);
  else decode_dp<256>(p, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  return launch_attn_join(p, stream);
}

}  // namespace omx
