// The paged key-value cache: the append of new tokens and the decode step of one token a sequence.
#include "gdn_paged.h"

namespace omx {
namespace {

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
template <int DP, int NQ, bool WIN>
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
  if (p.splits > 1 && !decode_range<WIN>(p, wg, cap, SK, b, st0, x, x1)) return;

  for (;;) {  // a segment a turn
  const_i32* table = (const_i32*)(p.table + (long long)b * p.table_w);
  const int held = ((const_i32*)p.held)[b];
  // keys: those held and the new one, at position `held`; past the table there is no room for it
  const Seen seen = seen_of<WIN>(p, held, cap, SK);
  const int keys = seen.keys, nst = seen.stages;
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
      const int key = (WIN ? seen.at(st) : st) * SK + 16 * g;
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
    const int key0 = (WIN ? seen.at(st) : st) * SK;
    constexpr unsigned kAll = (1u << NG) - 1;
    const bool whole = have == kAll && key0 + SK < keys &&  // every row a held key, and seen
                       !(WIN && key0 < seen.lo && key0 + SK > p.sinks);
    if (!whole) {
      // rows without a key, or not seen, are cleared (a weight of zero does not clear a NaN), and the new
      // token's row comes from the arguments: its page has no copy of it yet
      for (int i = l; i < SK * DP / 8; i += 64) {
        const int row = i / (DP / 8);
        const int key = key0 + row;
        if (key >= keys || !((have >> (row / 16)) & 1) || (WIN && key < seen.lo && key >= p.sinks)) *(u32x4*)(sv + 8 * i) = u32x4{0, 0, 0, 0};
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
          const int key = key0 + 16 * g + 4 * g4 + i;
          // (selects: of the three joined by || the compiler may make branches, and lost a write so in gdn_cache8.hip)
          const bool no = (key >= keys) | !((have >> g) & 1) | (WIN & (key < seen.lo) & (key >= p.sinks));
          s[g][i] = (!whole & no) ? -INFINITY : s[g][i];
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

template <int DP, bool WIN>
void decode_dp(const AttnParams& p, hipStream_t stream) {
  const unsigned grid = (unsigned)((p.splits > 1 ? p.splits : p.N) * p.Hkv);
  if (p.G <= 16)
    attn_decode_kernel<DP, 1, WIN><<<grid, 64 * kDecNW, 0, stream>>>(p);
  else
    attn_decode_kernel<DP, 2, WIN><<<grid, 64 * kDecNW, 0, stream>>>(p);
  if (p.splits > 1) launch_decode_join<DP, WIN, kStageKeys<DP>>(p, stream);
}
template <int DP>
void decode_dp(const AttnParams& p, hipStream_t stream) {
  if (p.window > 0) decode_dp<DP, true>(p, stream);
  else decode_dp<DP, false>(p, stream);
}

}  // namespace

bool paged_dims_supported(int D) { return D == 64 || D == 128 || D == 256; }

int kv_write_tokens() { return 4 * kWriteTokens; }

hipError_t launch_kv_write(const AttnParams& p, hipStream_t stream) {
  const long long per = kv_write_tokens();
  kv_write_kernel<<<(unsigned)((p.tokens + per - 1) / per), 256, 0, stream>>>(p);
  return hipGetLastError();
}

int decode_splits(long long N, long long Hkv, long long D, long long capacity, long long seen, bool eight) {
  // One workgroup a sequence and key head where a sequence is so short that the join costs more than
  // it saves (B=1, 4 key heads of 128, calls one after the other: 611 keys 14.4 us in one launch, 18.5 in
  // two, 1,500 keys 21.8 and 18.0), and for more than 1,024 sequences, where each row's join sums up all
  // their lengths.  Otherwise one for each compute unit: their buffers allow no second.  Equal ranges
  // against a workgroup each, 32/8 heads of 128: 64 sequences of 4,000 keys 190 us (187), between 1,000
  // and 7,000 207 (230), 63 of 1,000 and one of 30,000 84 (380); 1,024 of 100 199 (196), with one of
  // 30,000 244 (532).  16/2 heads of 256, sequences of 75 to 525 keys: 512 98 (81), 1,024 182 (156),
  // 4,096 723 (579).
  // Of a cache in 8 bits, whose wavefronts pass twice the keys in a turn, twice the keys are short (1,200
  // keys of 128: one sequence of 4 heads 14 us, shared 18, 64 of 2 heads 19 and 27; 4,800: 29 and 18, 56 and 44).
  // With a window sequences are taken for alike, as all that pass it are (lengths are not known here), and
  // sharing only evens out the last round of workgroups, for some 11 us (the join, and a second sequence's start
  // in most ranges): a key's bytes take a workgroup 19 ps each, or its part of 6.2 TB/s.  64 sequences of 8 heads
  // of 128, two whole rounds, 1,024 keys: 63 us (70), in 8 bits 39 (49); 40 of 8, 3,000 keys: 115 us (102), 71
  // (66); one of 4, 2,048 keys: 28 us (17), 18 (17).
  // Where few sequences pass a long window theirs are the last workgroups: 63 of 1,000 to 1,400 tokens and one of
  // 30,000, 32/8 heads of 128, window 1,024 62 us, 8,000 148, 20,000 293, and 94 without a window.
  const int bytes = eight ? 1 : 2;
  if (N > 1024) return 1;
  if (seen < capacity) {
    const long long groups = N * Hkv, rounds = (groups + kComputeUnits - 1) / kComputeUnits;
    const double fill = (double)groups / (kComputeUnits * rounds), each = 2. * D * bytes * seen;
    if (rounds * each * (fill < 0.46 ? 1.9e-5 : fill * 4.1e-5) * (1 - fill) < 11.) return 1;
  } else if (capacity * D * bytes <= (1 << 18)) {
    return 1;
  }
  // stages are counted in 32 bits, and a range's end lies up to a range past the last
  if (N * (seen / 16 + 1) > INT_MAX / 2) return 1;
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
