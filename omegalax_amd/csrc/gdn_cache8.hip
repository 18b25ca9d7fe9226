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
// Transposed read of 8-bit elements: lanes 2i and 2i + 1 of 16 give the addresses of the two halves of row
// i's 16 columns, and lane j gets column j of the 8 rows (verified on MI355X).
__device__ __forceinline__ u32x2 ds_read_tr8(const uint8_t* p) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      (__attribute__((address_space(3))) i32x2*)(unsigned long long)(const __attribute__((address_space(3))) uint8_t*)p));
}
// 2^(a - b) of exponents a <= b
__device__ __forceinline__ float exp_shift(int a, int b) { return a - b < -126 ? 0.f : exp_scale(a - b); }

// ------------------------------------------------------------------------------------ append
// Token i of sequence n goes to position held[n] + i, as in the cache of bf16.  A wavefront takes the
// blocks that begin with one of its kSpan tokens (a block of a sequence's first new token among them),
// whole and for one head's keys or values: a lane has 16 columns of every DP / 64-th group of rows.  The largest values
// are found over the wavefront; the block's older tokens are written only if its exponent grows.  Rows from
// the last offset on are no tokens: taken for the last sequence's they would raise the exponents of those it has.
// Bound by the bytes where there are many: 32,000 tokens of 8 heads of 128 36 us, 4.0 TB/s; 77 tokens 5.
// (4,200 tokens 14, with keys and values by one wavefront, one after the other, 17.)
constexpr int kSpan = 16;

template <int DP>
__global__ __launch_bounds__(256) void kv_write8_kernel(AttnParams p) {
  constexpr int NR = DP / 64, LR = DP / 16, RJ = 64 / LR;  // rows: NR loads of RJ, LR lanes each
  const int l = lane_id(), hk = (int)blockIdx.y >> 1, seg = l % LR;
  const bool value = blockIdx.y & 1;
  const bf16_t* src = (const bf16_t*)(value ? p.v : p.k) + hk * DP + 16 * seg;
  const long long src_ld = value ? p.v_ld : p.k_ld;
  uint8_t* pool = (uint8_t*)(value ? p.v_pages : p.k_pages);
  int8_t* exps = value ? p.v_exps : p.k_exps;
  const long long t0 = ((long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kSpan;
  const bool lanes = p.cu && !p.plan;  // lane n holds sequence n's end
  int end = 0;
  long long t1 = t0 + kSpan < p.tokens ? t0 + kSpan : p.tokens;
  if (p.cu) {
    const int n = lanes ? l : p.N - 1;
    end = n < p.N ? p.cu[n + 1] : 0;
    end = end < 0 ? 0 : (end > p.T ? p.T : end);
    if (lanes) end = wave_scan_max(end);
    else end = end > p.cu_plan[n] ? end : p.cu_plan[n];
    const int last = __builtin_amdgcn_readlane(end, 63);
    t1 = last < t1 ? last : t1;
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
      stop = lo + 1 < p.N ? p.cu_plan[lo + 1] : end;
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
    // the rows are on their way before the table is read
    u32x4 x[NR][2];
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const int r = RJ * j + l / LR - r0;
      x[j][0] = x[j][1] = u32x4{0, 0, 0, 0};
      if (r >= 0 && r < m) {
        x[j][0] = *(const u32x4*)(src + (t + r) * src_ld);
        x[j][1] = *(const u32x4*)(src + (t + r) * src_ld + 8);
      }
    }
    const long long slot = pos / p.page;
    const int id = slot < p.table_w ? p.table[(long long)seq * p.table_w + slot] : -1;
    if (id >= 0 && id < p.n_pages) {
      const int row = (int)(pos - slot * p.page) - r0;  // the block's first, of the page
      uint8_t* to = pool + (((long long)id * p.page + row) * p.Hkv + hk) * DP + 16 * seg;
      int8_t* at = exps + ((long long)id * (p.page / 16) + row / 16) * p.Hkv + hk;
      int before = kLeastExp;
      u32x4 old[NR];  // the block's older tokens, read beside their exponent
      if (r0 > 0) {
        before = *at;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          const int r = RJ * j + l / LR;
          old[j] = *(const u32x4*)(to + (long long)(r < r0 ? r : 0) * p.Hkv * DP);
        }
      }
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < NR; ++j) most = fmaxf(most, most16(x[j][0], x[j][1]));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
      const int ask = asked_exp(most), e = ask > before ? ask : before;
      if (r0 > 0 && e > before) {
        const float shift = exp_shift(before, e);
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          const int r = RJ * j + l / LR;
          if (r < r0) *(u32x4*)(to + (long long)r * p.Hkv * DP) = again16(old[j], shift);
        }
      }
      const float down = exp_scale(-e);
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        const int r = RJ * j + l / LR;
        if (r >= r0 && r < r0 + m) *(u32x4*)(to + (long long)r * p.Hkv * DP) = code16(x[j][0], x[j][1], down);
      }
      if (l == 0) *at = (int8_t)e;
    }
    t += m;
  }
}

// ------------------------------------------------------------------------------------ decode
// As for the cache of bf16 (gdn_paged.hip): equal ranges of all sequences' stages, a wavefront's stages in
// turns, read once for all query heads of a key head.  A stage's numbers go from memory to LDS as they
// are, into a wavefront's one slot, whose keys and values are refilled by turns: the next stage's keys once
// this one's scores are formed, its values once these are added up (128 KiB a compute unit with eight
// wavefronts, 64 with the four of more than 16 query heads a key head).  They become bf16 on the way from there into a
// product, each once: keys by rows of 8, values by transposed reads of 8 keys, the 8 that a lane's weights
// of two blocks stand for.  The wavefront whose stage holds the new token's block puts the token into it,
// there and in the cache; it rounds it while its first stage is on its way (after it: 69 us where now 64).
// Half the bytes of the cache of bf16, and bound less by them: 64 sequences of 4,000 keys of 16/2 heads of 256
// 64 us with the join, 4.4 TB/s in the kernel (in bf16 102); 611 keys of 16/4 heads of 128 10.7 us (11.8).
template <int DP> constexpr int kStage8 = 8192 / DP;  // keys: 8 KiB of K, 8 of V

// Place of 16-byte segment s of row r: s ^ swz8(r).  Reads of 16 rows' 8 bytes at one column, and transposed
// ones of 8 rows at two neighbouring, rows 4a .. and 16 + 4a .., then fall into different banks.
template <int DP>
__device__ __forceinline__ int swz8(int r) {
  if constexpr (DP == 256) return (r ^ (((r >> 4) & 1) << 2)) & 15;
  if constexpr (DP == 128) return ((r >> 1) & 7) ^ (((r >> 4) & 1) << 1);
  return ((r >> 2) & 3) ^ ((r >> 4) & 1);
}

// wavefronts of a workgroup: two a SIMD where their registers allow it
template <int NQ> constexpr int kDec8NW = NQ == 1 ? 8 : 4;

template <int DP, int NQ, bool WIN>
__global__ __launch_bounds__(64 * kDec8NW<NQ>) __attribute__((amdgpu_waves_per_eu(kDec8NW<NQ> / 4)))
void attn_decode8_kernel(AttnParams p) {
  constexpr int SK = kStage8<DP>, NG = SK / 16, NC = SK / 32;  // keys of a stage, its blocks, pairs of them
  constexpr int KS = DP / 32, DB = DP / 16;
  constexpr int NI = DP / 64, RI = 1024 / DP, LR = DP / 16;     // loads of a block, their rows, a row's lanes
  constexpr int kV = SK * DP, kE = 2 * kV, kNew = kE + 512;     // a slot: K, V, their exponents (4 bytes each)
  constexpr int kSlot = kNew + 2560;                            // and the new token's k, v and old exponents
  constexpr int kSum = DP + 16;                                 // a row of sums: four rows fill the banks
  static_assert(16 * kSum * 4 <= kSlot, "a slot holds 16 rows of sums");
  constexpr int kLoads = NG * NI + 1;                           // of K, and of V
  constexpr int NW = kDec8NW<NQ>;
  __shared__ __align__(16) uint8_t slots[NW][kSlot];
  __shared__ float sM[NW][16 * NQ], sL[NW][16 * NQ];

  const int tid = threadIdx.x, l = tid & 63, g4 = l >> 4, r = l & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.G, Hkv = p.Hkv, Hq = Hkv * G;
  const int hk = (int)blockIdx.x % Hkv, wg = (int)blockIdx.x / Hkv;
  const int cap = p.table_w * p.page;
  const int lrow = l / LR, seg = l % LR;
  const unsigned ld = (unsigned)(Hkv * DP);
  // a lane's offsets in a block's loads; the swizzle tells even blocks from odd ones
  unsigned off[2][NI];
#pragma unroll
  for (int i = 0; i < 2 * NI; ++i) {
    const int row = RI * (i % NI) + lrow;
    off[i / NI][i % NI] = (unsigned)row * ld + 16u * (unsigned)(seg ^ swz8<DP>(16 * (i / NI) + row));
  }

  int b = wg, st0 = 0, x = 0, x1 = INT_MAX;
  if (p.splits > 1 && !decode_range<WIN>(p, wg, cap, SK, b, st0, x, x1)) return;

  for (;;) {  // a segment a turn
  const_i32* table = (const_i32*)(p.table + (long long)b * p.table_w);
  const int held = ((const_i32*)p.held)[b];
  const Seen seen = seen_of<WIN>(p, held, cap, SK);
  const int keys = seen.keys, nst = seen.stages;
  const int st1 = nst - st0 < x1 - x ? nst : st0 + (x1 - x);
  const bool alone = st0 == 0 && st1 == nst;

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

  // blocks of a stage: their number in the cache, none from st1 on
  struct Ids { unsigned at[NG], have; };
  auto look = [&](int st) __attribute__((always_inline)) {
    Ids y;
    y.have = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int key = (WIN ? seen.at(st) : st) * SK + 16 * g;
      const int slot = (int)(__umulhi((unsigned)key, p.page_mul) >> p.page_shift), off = key - slot * p.page;
      const int id = st < st1 && key < keys ? table[slot] : -1;  // key < keys <= cap: the slot is in the table
      const bool there = id >= 0 && id < p.n_pages;
      y.have |= there ? 1u << g : 0u;
      y.at[g] = there ? (unsigned)id * (unsigned)(p.page / 16) + (unsigned)(off / 16) : 0u;
    }
    return y;
  };
  // Fetches a stage's keys (or values); a block that is not there has an empty range and reads as zeros, so
  // that every stage counts the same loads.
  uint8_t* const slot = slots[w];
  const unsigned lds = lds_address(slot);
  auto stage = [&](const Ids& y, const void* pages, const int8_t* exps, unsigned to,
                   unsigned to_exps) __attribute__((always_inline)) {
    unsigned eo = kDropOffset;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const bool there = (y.have >> g) & 1;
      const long long at = ((long long)y.at[g] * 16 * Hkv + hk) * DP;
      loads_to_lds16_on(rsrc_words((const char*)pages + at, there ? 15u * ld + DP : 0u), lds + to + 1024u * NI * g, off[g & 1]);
      if (there && l == g) eo = y.at[g] * (unsigned)Hkv + (unsigned)hk;
    }
    load_to_lds1(rsrc_words(exps, kDropOffset), lds + to_exps, eo);
  };
  auto stage_k = [&](const Ids& y) __attribute__((always_inline)) { stage(y, p.k_pages, p.k_exps, 0, kE); };
  auto stage_v = [&](const Ids& y) __attribute__((always_inline)) { stage(y, p.v_pages, p.v_exps, kV, kE + 256); };
  // The new token as its block will hold it: a lane's 16 codes, the block's exponent, and by what its older
  // codes are multiplied if that grew.  Formed while the first stage is on its way.
  struct New {
    u32x4 codes;
    int now;
    float shift;
    bool grew;
  };
  const int r0 = held & 15;
  auto quantise = [&](const uint8_t* row, int before) __attribute__((always_inline)) {
    const u32x4 a = *(const u32x4*)(row + 32 * seg), a2 = *(const u32x4*)(row + 32 * seg + 16);
    float most = most16(a, a2);
#pragma unroll
    for (int i = 1; i < LR; i <<= 1) most = fmaxf(most, __shfl_xor(most, i, 64));
    const int ask = asked_exp(most);
    New y;
    before = r0 > 0 ? before : kLeastExp;
    y.now = ask > before ? ask : before;
    y.grew = ask > before;
    y.shift = exp_shift(before, y.now);
    y.codes = code16(a, a2, exp_scale(-y.now));
    return y;
  };
  // puts it into the stage that holds its block, number `at`, and into the cache
  auto amend = [&](const New& y, int gb, unsigned at, uint8_t* codes, uint8_t* ex, void* pages,
                   int8_t* exps) __attribute__((always_inline)) {
    uint8_t* to = (uint8_t*)pages + ((long long)at * 16 * Hkv + hk) * DP + 16 * seg;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int row = RI * j + lrow;
      if (row > r0 || (row < r0 && !y.grew)) continue;
      u32x4* c = (u32x4*)(codes + (16 * gb + row) * DP + ((seg ^ swz8<DP>(16 * gb + row)) << 4));
      const u32x4 x = row == r0 ? y.codes : again16(*c, y.shift);
      *c = x;
      *(u32x4*)(to + (long long)row * Hkv * DP) = x;
    }
    if (l == 0) {
      exps[(long long)at * Hkv + hk] = (int8_t)y.now;
      ex[4 * gb] = (uint8_t)y.now;
    }
  };
  uint8_t *const sk = slot, *const sv = slot + kV;
  // lane 2i + j of 16 reads 8 of the 16 columns of row 4 g4 + i (16 more from i = 4 on)
  const int vrow = 4 * g4 + ((r >> 1) & 3) + 16 * (r >> 3);
  // A wavefront's stages, st0 + w and then every NW-th.  The next one's keys are fetched once this one's
  // scores are formed, its values once theirs are added up.
  {
    int st = st0 + w;
    Ids y = look(st), next;
    // whose stage holds the new token's block, of number `into`
    const bool room = held >= 0 && held < cap;
    const int at_new = room ? held : 0, st_new = at_new / SK - seen.skip;  // (in the window's part, or nothing is skipped)
    const int new_slot = (int)(__umulhi((unsigned)at_new, p.page_mul) >> p.page_shift);
    const int new_id = room && st_new >= st && st_new < st1 && (st_new - st) % NW == 0 ? table[new_slot] : -1;
    const bool ours = new_id >= 0 && new_id < p.n_pages;
    const unsigned into = (unsigned)new_id * (unsigned)(p.page / 16) + (unsigned)((at_new - new_slot * p.page) / 16);
    New nk{}, nv{};
    if (ours) {
      const unsigned to = l < DP / 8 ? 16u * (unsigned)l : kDropOffset;
      const unsigned eo = l == 0 ? into * (unsigned)Hkv + (unsigned)hk : kDropOffset;
      load_to_lds16(rsrc_words((const bf16_t*)p.k + b * p.k_ld + hk * DP, 2u * DP), lds + kNew, to);
      load_to_lds16(rsrc_words((const bf16_t*)p.v + b * p.v_ld + hk * DP, 2u * DP), lds + kNew + 1024u, to);
      load_to_lds1(rsrc_words(p.k_exps, kDropOffset), lds + kNew + 2048u, eo);
      load_to_lds1(rsrc_words(p.v_exps, kDropOffset), lds + kNew + 2304u, eo);
    }
    if (st < st1) {
      stage_k(y);
      stage_v(y);
    }
    if (ours) {
      asm volatile("s_waitcnt vmcnt(%0)" :: "n"(2 * kLoads) : "memory");  // all but the stage
      nk = quantise(slot + kNew, (int)(int8_t)slot[kNew + 2048]);
      nv = quantise(slot + kNew + 1024, (int)(int8_t)slot[kNew + 2304]);
    }
    // (behind the loads into LDS, which the compiler does not count: it waits for all of them with these)
    u32x4 q[NQ][KS];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        q[n][s] = u32x4{0, 0, 0, 0};
        if (16 * n + r < G)
          q[n][s] = *(const u32x4*)((const bf16_t*)p.q + b * p.q_ld + (long long)(hk * G + 16 * n + r) * DP + 32 * s + 8 * g4);
      }
    for (; st < st1; st += NW, y = next) {
      const bool more = st + NW < st1;
      if (more) next = look(st + NW);
      const unsigned have = y.have;
      const int key0 = (WIN ? seen.at(st) : st) * SK;
      constexpr unsigned kAll = (1u << NG) - 1;
      const bool whole = have == kAll && key0 + SK < keys &&  // every row a held key, and seen
                         !(WIN && key0 < seen.lo && key0 + SK > p.sinks);
      const bool mine = ours && st == st_new;
      const int gb = (held - key0) / 16;  // the new token's block

      asm volatile("s_waitcnt vmcnt(%0)" :: "n"(kLoads) : "memory");  // the keys: all but the values
      if (mine) {
        amend(nk, gb, into, sk, slot + kE, p.k_pages, p.k_exps);
        wave_lds_fence();
      }
      const int ke = (int)(int8_t)slot[kE + 4 * (l & (NG - 1))];
      f32x4 s[NQ][NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float scale = exp_scale(__builtin_amdgcn_readlane(ke, g));
        const uint8_t* row = sk + (16 * g + r) * DP;
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][g] = zero4();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const u32x2 c = *(const u32x2*)(row + (((2 * k + (g4 >> 1)) ^ swz8<DP>(16 * (g & 1) + r)) << 4) + 8 * (g4 & 1));
          const u32x4 a = widen8(c[0], c[1], scale);
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][g] = mma16(a, q[n][k], s[n][g]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads are done
      if (more) stage_k(next);

      u32x4 pb[NQ][NC], pr[NQ][NC];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        if (!whole) {
          // (selects of whole conditions: of the three joined by || the compiler makes a branch of the last, and
          // loses one element's write on it, which its assembly shows as an exec mask set and reset around nothing)
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + 16 * g + 4 * g4 + i;
              const bool no = (key >= keys) | !((have >> g) & 1) | (WIN & (key < seen.lo) & (key >= p.sinks));
              s[n][g][i] = no ? -INFINITY : s[n][g][i];
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[n][g][i]);
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
            s[n][g][i] = __builtin_amdgcn_exp2f(fmaf(s[n][g][i], cs, -mc));
            ls[n] += s[n][g][i];
          }
          // the weights as two bf16 terms (off by at most 2^-16 together)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float u = s[n][g][2 * i], v = s[n][g][2 * i + 1];
            pb[n][g / 2][2 * (g & 1) + i] = pack_bf16(u, v);
            pr[n][g / 2][2 * (g & 1) + i] = pack_bf16(lo_part(u), lo_part(v));
          }
        }
      }

      if (more)
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"(kLoads) : "memory");  // the values: all but the next keys
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (!whole) {
        if (mine) amend(nv, gb, into, sv, slot + kE + 256, p.v_pages, p.v_exps);
        // rows without a key, or not seen, are cleared: a weight of zero does not clear a NaN
        for (int i = l; i < SK * LR; i += 64) {
          const int row = i / LR, key = key0 + row;
          if (key >= keys || !((have >> (row / 16)) & 1) || (WIN && key < seen.lo && key >= p.sinks))
            *(u32x4*)(sv + 16 * i) = u32x4{0, 0, 0, 0};
        }
        wave_lds_fence();
      }
      const int ve = (int)(int8_t)slot[kE + 256 + 4 * (l & (NG - 1))];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float s0 = exp_scale(__builtin_amdgcn_readlane(ve, 2 * c)), s1 = exp_scale(__builtin_amdgcn_readlane(ve, 2 * c + 1));
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const u32x2 v = ds_read_tr8(sv + (32 * c + vrow) * DP + ((d ^ swz8<DP>(vrow)) << 4) + 8 * (r & 1));
          const u32x2 lo = widen4(v[0], s0), hi = widen4(v[1], s1);
          const u32x4 a = u32x4{lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            o[n][d] = mma16(a, pb[n][c], o[n][d]);
            o[n][d] = mma16(a, pr[n][c], o[n][d]);
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads are done
      if (more) stage_v(next);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is on its way into LDS
  }

  // ---------------------------------------------------------------- the wavefronts' sums
  // a wavefront's slot holds 16 rows of kSum fp32
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    ls[n] += __shfl_xor(ls[n], 16, 64);
    ls[n] += __shfl_xor(ls[n], 32, 64);
    if (g4 == 0) {
      sM[w][16 * n + r] = m[n] * cs;
      sL[w][16 * n + r] = ls[n];
    }
  }
  lds_barrier();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
      if (16 * n + r < G) *(f32x4*)((float*)slot + r * kSum + 16 * d + 4 * g4) = o[n][d];
    lds_barrier();
    const int rows = G - 16 * n < 16 ? G - 16 * n : 16;
    for (int i = tid; i < rows * DP / 4; i += 64 * NW) {
      const int row = i / (DP / 4), col = 4 * (i % (DP / 4));
      float M = sM[0][16 * n + row];
#pragma unroll
      for (int u = 1; u < NW; ++u) M = fmaxf(M, sM[u][16 * n + row]);
      f32x4 acc = zero4();
      float den = 0.f;
#pragma unroll
      for (int u = 0; u < NW; ++u) {
        const float lx = sL[u][16 * n + row];
        const float a = lx == 0.f ? 0.f : __builtin_amdgcn_exp2f(sM[u][16 * n + row] - M);
        den += a * lx;
        acc += a * *(const f32x4*)((const float*)slots[u] + row * kSum + col);
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
    lds_barrier();
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
    attn_decode8_kernel<DP, 1, WIN><<<grid, 64 * kDec8NW<1>, 0, stream>>>(p);
  else
    attn_decode8_kernel<DP, 2, WIN><<<grid, 64 * kDec8NW<2>, 0, stream>>>(p);
  if (p.splits > 1) launch_decode_join<DP, WIN, kStage8<DP>>(p, stream);
}
template <int DP>
void decode8_dp(const AttnParams& p, hipStream_t stream) {
  if (p.window > 0) decode8_dp<DP, true>(p, stream);
  else decode8_dp<DP, false>(p, stream);
}

}  // namespace

int kv_write8_tokens() { return 4 * kSpan; }

hipError_t launch_kv_write8(const AttnParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.tokens + 4 * kSpan - 1) / (4 * kSpan)), 2u * (unsigned)p.Hkv);
  if (p.D == 64) kv_write8_kernel<64><<<grid, 256, 0, stream>>>(p);
  else if (p.D == 128) kv_write8_kernel<128><<<grid, 256, 0, stream>>>(p);
  else kv_write8_kernel<256><<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

hipError_t launch_attn_decode8(const AttnParams& p, hipStream_t stream) {
  if (p.D == 64) decode8_dp<64>(p, stream);
  else if (p.D == 128) decode8_dp<128>(p, stream);
  else decode8_dp<256>(p, stream);
  return hipGetLastError();
}

}  // namespace omx
