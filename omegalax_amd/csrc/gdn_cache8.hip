// A paged key-value cache in 8 bits: the append of new tokens and the decode step.
//
//   x ~ c 2^e,  c an e4m3 number, e the exponent of the token's block: 16 tokens of a head (a page holds
//   whole blocks), e = max over the block's tokens of ceil(log2(max |x| / 448)), within [-100, 120]
//
// A power of two costs no accuracy against any other scale, as e4m3 numbers are as exact at every size,
// and has the block's older tokens, which a larger new one pushes down, divided exactly, but for
// the smallest: c' = round(c 2^(e - e')).  Number times power is a bf16 value (gdn_attn.h).
#include "gdn_paged.h"

namespace omx {
namespace {

constexpr int kLeastExp = -100, kMostExp = 120;
// Larger values are clamped: what they are rounded to has to stay within bf16.
constexpr float kLargest8 = 1.875f * 0x1p127f;

// the exponent that a largest value asks for: of its bits, one more if the fraction is above that of 448
__device__ __forceinline__ int asked_exp(float most) {
  const int e = (int)((__float_as_uint(most) + 0x1fffffu) >> 23) - 127 - 8;
  return e < kLeastExp ? kLeastExp : (e > kMostExp ? kMostExp : e);
}
// the size of a value in its block's largest: values that are not finite do not count
__device__ __forceinline__ float size8(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? fminf(a, kLargest8) : 0.f;
}
// two bf16 as codes, for a block's 2^-e; a value that is not finite becomes a NaN
__device__ __forceinline__ uint32_t code2(uint32_t x, float down, uint32_t old, bool hi) {
  float a = bf2f((bf16_t)(x & 0xffffu)), b = bf2f((bf16_t)(x >> 16));
  if (fabsf(a) < INFINITY) a = fminf(fmaxf(a, -kLargest8), kLargest8);
  if (fabsf(b) < INFINITY) b = fminf(fmaxf(b, -kLargest8), kLargest8);
  return hi ? __builtin_amdgcn_cvt_pk_fp8_f32(a * down, b * down, old, true)
            : __builtin_amdgcn_cvt_pk_fp8_f32(a * down, b * down, old, false);
}
// 16 bf16 as 16 codes
__device__ __forceinline__ u32x4 code16(u32x4 a, u32x4 b, float down) {
  u32x4 c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c[i] = code2(a[2 * i + 1], down, code2(a[2 * i], down, 0, false), true);
    c[2 + i] = code2(b[2 * i + 1], down, code2(b[2 * i], down, 0, false), true);
  }
  return c;
}
// 16 codes for a block whose exponent grew: each times 2^(old - new), rounded again
__device__ __forceinline__ u32x4 again16(u32x4 c, float shift) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32x2 x = widen4(c[i], 1.f);
    r[i] = code2(x[1], shift, code2(x[0], shift, 0, false), true);
  }
  return r;
}
__device__ __forceinline__ float most16(u32x4 a, u32x4 b) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t x = k ? b[i] : a[i];
      m = fmaxf(m, fmaxf(size8(bf2f((bf16_t)(x & 0xffffu))), size8(bf2f((bf16_t)(x >> 16)))));
    }
  return m;
}
// 2^(a - b) of exponents a <= b
__device__ __forceinline__ float exp_shift(int a, int b) { return a - b < -126 ? 0.f : exp_scale(a - b); }

// ------------------------------------------------------------------------------------ append
// Token i of sequence n goes to position held[n] + i, as in the cache of bf16.  A wavefront takes the
// blocks that begin with one of its kSpan tokens (a block of a sequence's first new token among them),
// whole and for one head: a lane has 16 columns of every DP / 64-th group of rows.  The largest values
// are found over the wavefront, and the block's older tokens read only if its exponent grows.
constexpr int kSpan = 16;

template <int DP>
__global__ __launch_bounds__(256) void kv_write8_kernel(AttnParams p, int span) {
  constexpr int NR = DP / 64, LR = DP / 16, RJ = 64 / LR;  // rows: NR loads of RJ, LR lanes each
  const int l = lane_id(), hk = (int)blockIdx.y, seg = l % LR;
  const long long t0 = ((long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * span;
  const long long t1 = t0 + span < p.tokens ? t0 + span : p.tokens;
  const bool lanes = p.cu && !p.plan;  // lane n holds sequence n's end
  int end = 0;
  if (lanes) {
    end = l + 1 < p.N ? p.cu[l + 1] : p.T;
    end = end < 0 ? 0 : (end > p.T ? p.T : end);
    end = wave_scan_max(end);
  }
  for (long long t = t0; t < t1;) {
    int seq;
    long long start, stop;  // of the sequence's new tokens
    if (lanes) {
      seq = __popcll(__ballot(l < p.N && end <= (int)t));
      start = seq > 0 ? __builtin_amdgcn_readlane(end, seq - 1) : 0;
      stop = __builtin_amdgcn_readlane(end, seq);
    } else if (p.plan) {
      int lo = 0, hi = p.N;  // cu_plan[lo] <= t < cu_plan[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.cu_plan[mid] <= (int)t) lo = mid; else hi = mid;
      }
      seq = lo;
      start = p.cu_plan[lo];
      stop = p.cu_plan[lo + 1];
    } else {
      seq = (int)(t / p.T);
      start = (long long)seq * p.T;
      stop = start + p.T;
    }
    const int held = p.held[seq];
    if (held < 0) {
      t = stop;
      continue;
    }
    long long pos = held + (t - start);
    if (t > start && pos % 16 != 0) {  // a block that another wavefront began, or this one
      t += 16 - pos % 16;
      if (t > stop) t = stop;
      continue;
    }
    const int r0 = (int)(pos % 16);
    const int m = stop - t < 16 - r0 ? (int)(stop - t) : 16 - r0;
    const long long slot = pos / p.page;
    const int id = slot < p.table_w ? p.table[(long long)seq * p.table_w + slot] : -1;
    if (id >= 0 && id < p.n_pages) {
      const int row = (int)(pos - slot * p.page) - r0;  // the block's first, of the page
      const long long at = (((long long)id * p.page + row) * p.Hkv + hk) * DP + 16 * seg;
      const long long block = ((long long)id * (p.page / 16) + row / 16) * p.Hkv + hk;
      u32x4 x[2][NR][2];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          const int r = RJ * j + l / LR - r0;
          x[kv][j][0] = x[kv][j][1] = u32x4{0, 0, 0, 0};
          if (r >= 0 && r < m) {
            const bf16_t* src = kv ? (const bf16_t*)p.v + (t + r) * p.v_ld : (const bf16_t*)p.k + (t + r) * p.k_ld;
            x[kv][j][0] = *(const u32x4*)(src + hk * DP + 16 * seg);
            x[kv][j][1] = *(const u32x4*)(src + hk * DP + 16 * seg + 8);
          }
        }
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        int8_t* exps = kv ? p.v_exps : p.k_exps;
        uint8_t* pool = (uint8_t*)(kv ? p.v_pages : p.k_pages) + at;
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < NR; ++j) most = fmaxf(most, most16(x[kv][j][0], x[kv][j][1]));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
        int e = asked_exp(most);
        if (r0 > 0) {
          const int before = exps[block];
          if (before < e) {
            const float shift = exp_shift(before, e);
#pragma unroll
            for (int j = 0; j < NR; ++j) {
              const int r = RJ * j + l / LR;
              u32x4* c = (u32x4*)(pool + (long long)r * p.Hkv * DP);
              if (r < r0) *c = again16(*c, shift);
            }
          }
          e = e > before ? e : before;
        }
        const float down = exp_scale(-e);
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          const int r = RJ * j + l / LR;
          if (r >= r0 && r < r0 + m) *(u32x4*)(pool + (long long)r * p.Hkv * DP) = code16(x[kv][j][0], x[kv][j][1], down);
        }
        if (l == 0) exps[block] = (int8_t)e;
      }
    }
    t += m;
  }
}

// ------------------------------------------------------------------------------------ decode
// As for the cache of bf16 (gdn_paged.hip), whose products these are; a stage goes through registers, two
// stages ahead, and is put into LDS as bf16.  The wavefront whose stage holds the new token's block writes it.
template <int DP, int NQ, bool WIN>
__global__ __launch_bounds__(64 * kDecNW) __attribute__((amdgpu_waves_per_eu(1)))
void attn_decode8_kernel(AttnParams p) {
  constexpr int SK = kStageKeys<DP>, NG = SK / 16;  // keys of a stage, its blocks
  constexpr int KS = DP / 32, DB = DP / 16;
  constexpr int NR = 4, RJ = 1024 / DP, LR = DP / 16;  // loads of K (and of V), their rows, a row's lanes
  __shared__ __align__(16) bf16_t sK[kDecNW][SK * DP], sV[kDecNW][SK * DP];
  __shared__ float sM[kDecNW][16 * NQ], sL[kDecNW][16 * NQ];

  const int tid = threadIdx.x, l = tid & 63, g4 = l >> 4, r = l & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.G, Hkv = p.Hkv, Hq = Hkv * G;
  const int hk = (int)blockIdx.x % Hkv, wg = (int)blockIdx.x / Hkv;
  const int cap = p.table_w * p.page;
  const int lrow = l / LR, seg = l % LR;
  bf16_t *sk = sK[w], *sv = sV[w];
  const unsigned zero = lane_zero();

  int b = wg, st0 = 0, x = 0, x1 = INT_MAX;
  if (p.splits > 1 && !decode_range<WIN>(p, wg, cap, SK, b, st0, x, x1)) return;

  for (;;) {  // a segment a turn
  const_i32* table = (const_i32*)(p.table + (long long)b * p.table_w);
  const int held = ((const_i32*)p.held)[b];
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

  // a stage's codes and exponents, and which of its blocks are there
  struct Raw {
    u32x4 k[NR], v[NR];
    int ke[NG], ve[NG];
    unsigned have;
  };
  auto load = [&](int st) {
    Raw y;
    y.have = 0;
    const unsigned ld = (unsigned)(Hkv * DP);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int key = seen.at(st) * SK + 16 * g;
      const int slot = key / p.page, off = key - slot * p.page;
      int id = st < st1 && key < keys ? table[slot] : -1;  // key < keys <= cap: the slot is in the table
      const bool there = id >= 0 && id < p.n_pages;
      y.have |= there ? 1u << g : 0u;
      id = there ? id : 0;
      const long long at = (((long long)id * p.page + off) * Hkv + hk) * DP;
      const long long block = ((long long)id * (p.page / 16) + off / 16) * Hkv + hk;
      const auto kr = uniform_rsrc((const char*)p.k_pages + at, there ? 15u * ld + DP : 0u);
      const auto vr = uniform_rsrc((const char*)p.v_pages + at, there ? 15u * ld + DP : 0u);
#pragma unroll
      for (int j = g * (NR / NG); j < (g + 1) * (NR / NG); ++j) {
        const unsigned off = (unsigned)((RJ * j + lrow) & 15) * ld + 16u * (unsigned)seg;
        y.k[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, off, 0, 0));
        y.v[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, off, 0, 0));
      }
      y.ke[g] = (int8_t)__builtin_amdgcn_raw_buffer_load_b8(uniform_rsrc(p.k_exps + block, there ? 1u : 0u), zero, 0, 0);
      y.ve[g] = (int8_t)__builtin_amdgcn_raw_buffer_load_b8(uniform_rsrc(p.v_exps + block, there ? 1u : 0u), zero, 0, 0);
    }
    return y;
  };
  // the new token's codes into the stage that holds its block, and into the cache
  auto amend = [&](int key0, u32x4 (&c)[NR], int (&e)[NG], const bf16_t* src, void* pages, int8_t* exps) {
    const u32x4 a = *(const u32x4*)(src + hk * DP + 16 * seg), a2 = *(const u32x4*)(src + hk * DP + 16 * seg + 8);
    float most = most16(a, a2);
#pragma unroll
    for (int i = 1; i < LR; i <<= 1) most = fmaxf(most, __shfl_xor(most, i, 64));
    const int gb = (held - key0) / 16, r0 = held % 16;
    const int slot = held / p.page, off = held - slot * p.page - r0;
    const long long at = (((long long)table[slot] * p.page + off) * Hkv + hk) * DP;
    const long long block = ((long long)table[slot] * (p.page / 16) + off / 16) * Hkv + hk;
    int before = kLeastExp;
#pragma unroll
    for (int g = 0; g < NG; ++g)
      if (g == gb && r0 > 0) before = e[g];
    const int ask = asked_exp(most), now = ask > before ? ask : before;
    const float shift = exp_shift(before, now);
    const u32x4 mine = code16(a, a2, exp_scale(-now));
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const int row = RJ * j + lrow, r1 = row & 15;
      if (row / 16 != gb || r1 > r0) continue;
      if (r1 == r0) c[j] = mine;
      else if (now > before) c[j] = again16(c[j], shift);
      if (r1 == r0 || now > before) *(u32x4*)((uint8_t*)pages + at + (long long)r1 * Hkv * DP + 16 * seg) = c[j];
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
      if (g == gb) e[g] = now;
    if (l == 0) exps[block] = (int8_t)now;
  };
  auto compute = [&](int st, Raw& y) {
    const int key0 = seen.at(st) * SK;
    constexpr unsigned kAll = (1u << NG) - 1;
    const unsigned have = y.have;
    const bool whole = have == kAll && key0 + SK < keys &&  // every row a held key, and seen
                       !(WIN && key0 < seen.lo && key0 + SK > p.sinks);
    if (!whole) {
      const int row = held - key0;
      if (row >= 0 && row < SK && held < cap && ((have >> (row / 16)) & 1)) {
        amend(key0, y.k, y.ke, (const bf16_t*)p.k + b * p.k_ld, p.k_pages, p.k_exps);
        amend(key0, y.v, y.ve, (const bf16_t*)p.v + b * p.v_ld, p.v_pages, p.v_exps);
      }
    }
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const int row = RJ * j + lrow, g = RJ * j / 16;
      const float ks = exp_scale(y.ke[g]), vs = exp_scale(y.ve[g]);
      const int key = key0 + row;
      // rows without a key, or not seen, are cleared: a weight of zero does not clear a NaN
      const bool no = !whole && (key >= keys || !((have >> g) & 1) || (WIN && key < seen.lo && key >= p.sinks));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int to = row * DP + (((2 * seg + i) ^ attn_swz<DP>(row)) << 3);
        *(u32x4*)(sk + to) = widen8(y.k[j][2 * i], y.k[j][2 * i + 1], ks);
        *(u32x4*)(sv + to) = no ? u32x4{0, 0, 0, 0} : widen8(y.v[j][2 * i], y.v[j][2 * i + 1], vs);
      }
    }
    wave_lds_fence();
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
          if (!whole && (key >= keys || !((have >> g) & 1) || (WIN && key < seen.lo && key >= p.sinks))) s[g][i] = -INFINITY;
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
        // the weights as two bf16 terms (off by at most 2^-16 together)
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
    __builtin_amdgcn_wave_barrier();
  };

  {
    int st = st0 + w;  // this wavefront's stages: st0 + w, then every fourth
    Raw y0 = load(st), y1 = load(st + kDecNW);
    for (; st < st1; st += 2 * kDecNW) {
      compute(st, y0);
      y0 = load(st + 2 * kDecNW);
      if (st + kDecNW >= st1) break;
      compute(st + kDecNW, y1);
      y1 = load(st + 3 * kDecNW);
    }
  }

  // ---------------------------------------------------------------- the four wavefronts' sums
  // buffers of K and V, 16 KiB a wavefront together, hold 16 rows of DP fp32
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
      float* dst = (float*)(d < DB / 2 ? sk : sv);
      *(f32x4*)(dst + r * (DP / 2) + 16 * (d % (DB / 2)) + 4 * g4) = o[n][d];
    }
    __syncthreads();
    const int rows = G - 16 * n < 16 ? G - 16 * n : 16;
    for (int i = tid; i < rows * DP / 4; i += 64 * kDecNW) {
      const int row = i / (DP / 4), col = 4 * (i % (DP / 4));
      float M = sM[0][16 * n + row];
#pragma unroll
      for (int u = 1; u < kDecNW; ++u) M = fmaxf(M, sM[u][16 * n + row]);
      f32x4 acc = zero4();
      float den = 0.f;
#pragma unroll
      for (int u = 0; u < kDecNW; ++u) {
        const float lx = sL[u][16 * n + row];
        const float a = lx == 0.f ? 0.f : __builtin_amdgcn_exp2f(sM[u][16 * n + row] - M);
        den += a * lx;
        const float* src = (const float*)(col < DP / 2 ? sK[u] : sV[u]);
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
void decode8_dp(const AttnParams& p, hipStream_t stream) {
  const unsigned grid = (unsigned)((p.splits > 1 ? p.splits : p.N) * p.Hkv);
  if (p.G <= 16)
    attn_decode8_kernel<DP, 1, WIN><<<grid, 64 * kDecNW, 0, stream>>>(p);
  else
    attn_decode8_kernel<DP, 2, WIN><<<grid, 64 * kDecNW, 0, stream>>>(p);
  if (p.splits > 1) launch_decode_join<DP, WIN>(p, stream);
}
template <int DP>
void decode8_dp(const AttnParams& p, hipStream_t stream) {
  if (p.window > 0) decode8_dp<DP, true>(p, stream);
  else decode8_dp<DP, false>(p, stream);
}

}  // namespace

int kv_write8_tokens() { return 4 * kSpan; }

hipError_t launch_kv_write8(const AttnParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.tokens + 4 * kSpan - 1) / (4 * kSpan)), (unsigned)p.Hkv);
  if (p.D == 64) kv_write8_kernel<64><<<grid, 256, 0, stream>>>(p, kSpan);
  else if (p.D == 128) kv_write8_kernel<128><<<grid, 256, 0, stream>>>(p, kSpan);
  else kv_write8_kernel<256><<<grid, 256, 0, stream>>>(p, kSpan);
  return hipGetLastError();
}

hipError_t launch_attn_decode8(const AttnParams& p, hipStream_t stream) {
  if (p.D == 64) decode8_dp<64>(p, stream);
  else if (p.D == 128) decode8_dp<128>(p, stream);
  else decode8_dp<256>(p, stream);
  return hipGetLastError();
}

}  // namespace omx
