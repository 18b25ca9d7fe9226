// Causal softmax attention of whole prompts and of new tokens over a paged cache.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  s_ij = scale q_i . k_j,  j <= i
//
// One workgroup takes a tile of 128 rows (token, query head of one key head) and passes over the
// keys once, 64 at a time, with the running maximum and sum of each row's softmax.  The keys' and
// values' tiles go from memory to LDS without passing through registers, one tile ahead.  A
// wavefront owns 32 rows and forms S^T = K Q^T, whose fragment holds one row per lane: maximum
// and sum are sums within a lane and one exchange of halves, and P^T is the B operand of
// O^T += V^T P^T as it stands.  Scores, statistics and sums are fp32; the weights are rounded to
// bf16 (off by at most 2^-8 of each) for the second product, and their sum is that of the unrounded ones.
//
// Two wavefronts a SIMD for heads up to 128, one (two tiles of k and v fill the LDS) for 256.  The
// MFMAs bound it where there are many tiles: B=4 T=4,096 of 32/8 heads of 128 525 to 547 us, 1,010 to
// 1,050 TFLOP/s at about 1.9 GHz (a library product of 8,192 cubed reaches 1,204 to 1,254).  With fewer tiles than the
// chip has places the longest one does: T=1,900 of 16/2 heads of 256, 238 tiles, 53 to 58 us, of which
// the last tile's 30 tiles of keys take 47.  Sharing its keys between two workgroups cost as much
// in partial sums and the join as it saved there (59 us and 12), at 1,000 tokens too (36 and 36).
//
// With a window a tile passes over the sinks and the keys from its first row's window on, 17 tiles of 64 for a
// window of 1,024 and 4 sinks, however long the prompt: 12,000 tokens of 16/2 heads of 256 240 to 250 us (all
// keys 1,090), B=4 T=4,096 of 32/8 heads of 128 290 to 310.  Which keys a row sees is one word of bits a tile
// (window_bits): compared key by key, the rows' limits took 5,000 spilled registers.
//
// Of a cache in 8 bits a tile's codes come a tile ahead into registers, and go to LDS as bf16 beside the
// products of the values.  Instructions bound it, 11 to 12 an MFMA: 700 new on 7,000 tokens each of 6 sequences,
// 32/8 heads of 128 498 us (from a cache of bf16 489), 16/4 of 64 183 (179), 16/2 of 256 533 (484).
#include "gdn_attn.h"

namespace omx {
namespace {

constexpr int kBM = 128, kBN = 64;

// m starts here: below any score, and finite, so that rows which have seen no key stay at 0
constexpr float kLow = -1e30f;

constexpr int kNW = 4, kNT = 64 * kNW;

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// WIN: a row sees its last p.window keys and the first p.sinks.
// CACHE: the keys and values are those of prompts (0), of pages in bf16 (1) or in 8 bits (2).
template <int DP, int CACHE, bool WIN>
__global__ __launch_bounds__(kNT) __attribute__((amdgpu_waves_per_eu(DP == 256 ? 1 : 2)))
void attn_fwd_kernel(AttnParams p, int ranks) {
  constexpr bool PAGED = CACHE != 0, EIGHT = CACHE == 2;
  constexpr int KS = DP / 16, DB = DP / 32;      // steps of a score, blocks of an output row
  constexpr int NG = 2 * KS, EG = 32 / NG;       // products of a tile's scores (and of its values)
  constexpr int PF = 4;                          // fragments read ahead of their products
  constexpr int NJ = kBN * DP / 8 / 64 / kNW;    // staging instructions per wavefront and tile
  constexpr int kTile = kBN * DP;
  __shared__ __align__(16) bf16_t sK[2 * kTile], sV[2 * kTile];  // two tiles each, by their parity
  __shared__ float sRow[kNW][DP];  // of a row that is summed again

  const int tid = threadIdx.x, l = tid & 63, h = l >> 5, c = l & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AttnLane lane = attn_lane<DP>();
  const int G = p.G, D = p.D, Hkv = p.Hkv, per = kBM / G;

  int unit, rank;
  const int units = (p.cu ? 1 : p.N) * Hkv;
  attn_place((int)blockIdx.x, units, ranks, unit, rank);
  if (rank >= ranks) return;
  const int split = (int)blockIdx.y;
  const int hk = unit % Hkv;
  AttnTile it;
  if (!attn_tile(p, unit / Hkv, rank, per, it)) return;
  const int t0 = it.tile * per;                                   // first token of the tile
  const int nt = it.len - t0 < per ? it.len - t0 : per;           // its tokens
  int held = 0;
  bool idle = false;
  if constexpr (PAGED) {
    held = __builtin_amdgcn_readfirstlane(p.held[it.seq]);
    idle = held < 0;  // a sequence that takes no part: zeros
    held = held < 0 ? 0 : (held > p.table_w * p.page ? p.table_w * p.page : held);
  }

  // this lane's row
  const int row = 32 * w + c, rt = row / G, rg = row - rt * G;
  const bool live = rt < nt;
  const long long tok = it.start + t0 + rt;
  const int pos = held + t0 + rt;                                 // its last key
  const int w_lo = held + t0 + (32 * w) / G;                      // the wavefront's first row's
  const int w_hi = held + t0 + (32 * w + 31) / G;                 //   and last row's last key

  u32x4 q[KS];
  auto load_q = [&]() __attribute__((always_inline)) {
    const bf16_t* qp = (const bf16_t*)p.q + tok * p.q_ld + (long long)(hk * G + rg) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * h;
      q[s] = u32x4{0, 0, 0, 0};
      if (live && d < D) q[s] = *(const u32x4*)(qp + d);
    }
  };
  if constexpr (!PAGED) load_q();

  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = zero16();
  float m = kLow, lsum = 0.f;
  const float cs = p.scale * kLog2e;

  // the tile's keys: 0 .. last, in tiles of kBN, of which this split takes [kt0, kt1)
  const int keys = held + t0 + nt;
  int kt0 = 0, kt1 = (keys + kBN - 1) / kBN;
  // With a window the tiles are of a list: the sinks (in a cache whole groups of 16; more than a tile of a
  // prompt's in whole tiles), then the keys from the first row's window on; `shift` keys between are left out.
  // Tile `cut` holds the last of the sinks and the first of the window.
  int sink_keys = 0, shift = 0, lo = 0, cut = -1;
  if constexpr (WIN) {
    lo = held + t0 - p.window + 1;
    sink_keys = PAGED ? (p.sinks + 15) & ~15 : (p.sinks <= kBN ? p.sinks : (p.sinks + kBN - 1) / kBN * kBN);
    const int from = PAGED ? lo & ~15 : lo;
    shift = from > sink_keys ? from - sink_keys : 0;
    if (shift > 0 && sink_keys % kBN != 0) cut = sink_keys / kBN;
    kt1 = (keys - shift + kBN - 1) / kBN;
  }
  auto place = [&](int x) { return x + (WIN && x >= sink_keys ? shift : 0); };  // the key at x
  auto key0 = [&](int kt) { return place(kt * kBN); };
  if (PAGED && p.splits > 1) {
    const int each = (kt1 + p.splits - 1) / p.splits;
    kt0 = split * each < kt1 ? split * each : kt1;
    kt1 = kt0 + each < kt1 ? kt0 + each : kt1;
  }
  if (idle) kt1 = kt0;

  // ---------------------------------------------------------------- staging
  // a lane's place in a wavefront's instructions: kStep rows lie between them, and after NO of them
  // (16 rows, or a multiple) the swizzle repeats
  constexpr int kStep = 64 / (DP / 8) * kNW, NO = kStep % 16 ? 2 : 1;
  static_assert(NO * kStep % 16 == 0, "rows whose swizzle repeats");
  const unsigned kld2 = PAGED ? (unsigned)(Hkv * D * 2) : (unsigned)(p.k_ld * 2);
  const unsigned vld2 = PAGED ? (unsigned)(Hkv * D * 2) : (unsigned)(p.v_ld * 2);
  unsigned koff[NO], voff[NO];
#pragma unroll
  for (int n = 0; n < NO; ++n) {
    const int row = stage_row<DP, kNW>(w, n), seg = stage_seg<DP>(row), r = PAGED ? row & 15 : row;
    koff[n] = 8 * seg < D ? (unsigned)r * kld2 + 16u * (unsigned)seg : kDropOffset;
    voff[n] = 8 * seg < D ? (unsigned)r * vld2 + 16u * (unsigned)seg : kDropOffset;
  }
  // The cache: a tile's pages, one for each of its four groups of 16 keys (a page is a multiple of 16
  // tokens).  Lane n asks for that of group n % 4 of the n / 4-th tile, of four, a tile before the answers are
  // needed (the first ones for three tiles at once): with a scalar load for
  // each group, each waited for, a turn took 3 (32/8 heads of 128) to 18% more (16/4 of 64).
  typedef const __attribute__((address_space(4))) int32_t const_i32;
  const_i32* table = PAGED ? (const_i32*)(p.table + (long long)it.seq * p.table_w) : nullptr;
  const int row_bytes = EIGHT ? Hkv * D : Hkv * D * 2;
  const unsigned blk_bytes = 16u * (unsigned)row_bytes;  // a group's, of a pool
  struct Asked { int id, of; };                          // a page, and which of its blocks (-1: no key)
  auto ask = [&](int kt) {
    const int tile = kt + (l >> 2 & 3), key = place(tile * kBN + 16 * (l & 3)), slot = (int)(__umulhi((unsigned)key, p.page_mul) >> p.page_shift);
    const bool in = (tile < kt1) & (key < keys) & (slot < p.table_w);
    return Asked{(int)__builtin_amdgcn_raw_buffer_load_b32(uniform_rsrc((const void*)table, 4u * (unsigned)p.table_w),
                                                           in ? 4u * (unsigned)slot : kDropOffset, 0, 0),
                 in ? (key - slot * p.page) >> 4 : -1};
  };
  // Of each group whether there is a page, and of those that this wavefront stages the block's offset in a pool (of
  // bf16) or its number (of 8 bits).
  constexpr int NP = !PAGED ? 1 : (EIGHT ? DP / 64 : (DP == 64 ? 2 : 4));
  struct Pages { long long at[EIGHT ? 1 : NP]; unsigned blk[EIGHT ? NP : 1], have; };
  auto group = [&](int n) {  // of the wavefront's n-th
    if constexpr (EIGHT) return DP == 256 ? n : (DP == 128 ? 2 * n + w / 2 : w);
    return DP == 64 ? 2 * n + w / 2 : n;
  };
  auto told = [&](const Asked& y, int of_tile) {
    Pages x;
    const bool there = (y.of >= 0) & (y.id >= 0) & (y.id < p.n_pages);
    const unsigned blk = there ? (unsigned)y.id * (unsigned)(p.page / 16) + (unsigned)y.of : 0u;
    x.have = (unsigned)__ballot(there) >> 4 * of_tile & 15u;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const unsigned b = (unsigned)__builtin_amdgcn_readlane((int)blk, 4 * of_tile + group(n));
      if constexpr (EIGHT) x.blk[n] = b;
      else x.at[n] = (long long)((unsigned long long)b * blk_bytes) + 2 * hk * D;
    }
    return x;
  };
  // Fetches a share of a tile of keys (or values) into LDS: NL instructions from the j0-th on.  They
  // are spread over a tile's products (all at once they hold a wavefront up for as long as its
  // memory path takes them in: 1,000 of 4,000 cycles a tile of heads of 256).  Tiles past the last
  // one have an empty range.
  constexpr int NL = 2, NF = NJ / NL;
  auto fetch = [&](int kt, const Pages& x, const void* pool, const void* rows, long long ld, unsigned ld2,
                   const unsigned (&lane_off)[NO], const bf16_t* dst, int j0) {
    const unsigned lds = lds_address(dst + (kt & 1) * kTile) + 1024u * (unsigned)w;
    if constexpr (PAGED) {
      // (of heads of 256 both instructions are of one group)
      constexpr int NS = DP == 256 ? NL : 1;
#pragma unroll
      for (int j = j0; j < j0 + NL; j += NS) {
        const int n = DP == 64 ? j : kStep * j / 16;  // the wavefront's group of the instruction's rows
        unsigned at[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) at[i] = lane_off[(j + i) % NO];
        loads_to_lds16(rsrc_words((const char*)pool + x.at[n], (x.have >> group(n)) & 1 ? 16u * ld2 : 0),
                       lds + 1024u * kNW * j, at);
      }
    } else {
      int left = it.len - key0(kt);  // rows past the sequence read as zeros
      left = left < kBN ? left : kBN;
      unsigned at[NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) at[j] = lane_off[(j0 + j) % NO] + (unsigned)((j0 + j) / NO * NO * kStep) * ld2;
      loads_to_lds16(rsrc_words((const bf16_t*)rows + (it.start + key0(kt)) * ld + hk * D,
                                kt < kt1 ? (unsigned)(left - 1) * ld2 + 2u * D : 0),
                     lds + 1024u * kNW * j0, at);
    }
  };
  // the tile of a prompt that holds the sinks and the window's first: lanes with a row of each
  auto fetch_cut = [&](const void* rows, long long ld, unsigned ld2, const unsigned (&lane_off)[NO], const bf16_t* dst) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int on = j / NO * NO * kStep, row = stage_row<DP, kNW>(w, j % NO) + on;
      const unsigned lds = lds_address(dst) + 1024u * (unsigned)w + 1024u * kNW * (unsigned)j;
      const bf16_t* at = (const bf16_t*)rows + it.start * ld + hk * D;
      const int left = it.len - shift < kBN ? it.len - shift : kBN;
      if (row < sink_keys)
        load_to_lds16(rsrc_words(at, (unsigned)(sink_keys - 1) * ld2 + 2u * D), lds, lane_off[j % NO] + (unsigned)on * ld2);
      else
        load_to_lds16(rsrc_words(at + shift * ld, (unsigned)(left - 1) * ld2 + 2u * D), lds, lane_off[j % NO] + (unsigned)on * ld2);
    }
  };
  // Of a cache in 8 bits a thread loads NR segments of 16 numbers and their exponents into registers, two
  // tiles ahead of the values' products and three of the keys', and a tile later puts them into LDS as
  // bf16, a half segment beside every other product of the values.
  constexpr int NR = DP / 64, kRows8 = 4096 / DP;  // rows of the workgroup's j-th load: kRows8 j ..
  struct Raw { u32x4 x[NR]; unsigned char e[NR]; };
  // A lane's row of the first load and its segment.  Eight lanes' writes of a half of theirs fill the banks if
  // four are of a row whose swizzle differs in its lowest bit, four further (with rows in order every write
  // took twice its time).
  int row8, seg8;
  {
    const int l = tid & 63, low = 4 * (l >> 2 & 1);
    if constexpr (DP == 64) row8 = 16 * w + low + ((l >> 3 & 3) | (l >> 5) << 3);
    else if constexpr (DP == 128) row8 = 8 * w + low + (l >> 4);
    else row8 = 8 * (w >> 1) + 2 * (w & 1) + low + (l >> 5);
    seg8 = (l & 3) + (DP == 64 ? 0 : 4 * (l >> 3 & (DP == 128 ? 1 : 3)));
  }
  const unsigned zero8 = lane_zero();
  // (a block's offset in a pool is one product; exponents lie within 32 bits of their pool's first)
  const unsigned off8 = (unsigned)(row8 & 15) * (unsigned)row_bytes + 16u * (unsigned)seg8;
  auto load8 = [&](const Pages& x, const void* pool, const int8_t* exps) {
    Raw r;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const bool there = (x.have >> group(j)) & 1;
      const unsigned blk = x.blk[j];
      r.x[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
          uniform_rsrc((const char*)pool + hk * DP + (unsigned long long)blk * blk_bytes, there ? 15u * row_bytes + DP : 0u),
          off8, 0, 0));
      r.e[j] = __builtin_amdgcn_raw_buffer_load_b8(
          uniform_rsrc(exps, kDropOffset), zero8 + (there ? blk * (unsigned)Hkv + (unsigned)hk : kDropOffset), 0, 0);
    }
    return r;
  };
  auto store8 = [&](const Raw& r, bf16_t* dst, int n) {  // the n-th of 2 NR halves
    const int row = kRows8 * (n / 2) + row8;
    *(u32x4*)(dst + row * DP + (((2 * seg8 + n % 2) ^ attn_swz<DP>(row)) << 3)) =
        widen8(r.x[n / 2][2 * (n % 2)], r.x[n / 2][2 * (n % 2) + 1], exp_scale((int8_t)r.e[n / 2]));
  };
  auto store8_all = [&](const Raw& r, bf16_t* dst) {
#pragma unroll
    for (int n = 0; n < 2 * NR; ++n) store8(r, dst, n);
  };
  Raw rv, rk;  // values of the next tile, keys of the one after
  auto fetch_k = [&](int kt, const Pages& x, int j) { fetch(kt, x, p.k_pages, p.k, p.k_ld, kld2, koff, sK, NL * j); };
  auto fetch_v = [&](int kt, const Pages& x, int j) { fetch(kt, x, p.v_pages, p.v, p.v_ld, vld2, voff, sV, NL * j); };

  // ---------------------------------------------------------------- one tile of keys
  // A wavefront's tiles go through two phases, in which its instructions are laid out group by
  // group, one product to each with the loads and arithmetic that run beside it:
  //   1: scores of the next tile  | weights and their sum of this one | reads of k, then of v
  //   2: weighted values of this  | maximum of the next one's scores  | reads of v
  Pages pn, pk;  // of the tile whose values come next, and of the one after, whose keys do
  Pages pl;      // of the third, in 8 bits
  Asked pa;      // and of the next but these
  u32x4 f[PF], pb[4];
  float mx = 0.f;
  auto kfrag = [&](const bf16_t* sk, AttnLane ln, int t) { return attn_frag<DP>(sk, ln, 32 * (t & 1), t / 2); };
  auto vfrag = [&](const bf16_t* sv, AttnLane ln, int t) { return attn_frag_tr<DP>(sv, ln, 16 * (t / DB), t % DB); };
  auto first = [&](const bf16_t* sk, f32x16 (&s)[2]) {
    const AttnLane ln = fresh(lane);
    s[0] = s[1] = zero16();
#pragma unroll
    for (int t = 0; t < NG; ++t) s[t & 1] = mma32(kfrag(sk, ln, t), q[t / 2], s[t & 1]);
    mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 32; ++e) mx = fmaxf(mx, s[e / 16][e % 16]);
  };
  auto mask = [&](int kt, f32x16 (&s)[2], unsigned have) {
    mx = -INFINITY;
    if constexpr (WIN) {
      unsigned long long see = window_bits(p, pos, key0(kt));
      if (kt == cut) {
        const unsigned long long sinks = keys_below(sink_keys - kt * kBN);
        see = (sinks & keys_below(p.sinks - kt * kBN)) | (~sinks & window_bits(p, pos, kt * kBN + shift));
      }
      if constexpr (PAGED)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (!((have >> g) & 1)) see &= ~(0xffffull << 16 * g);
      see >>= 4 * h;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        if (!((see >> (32 * (e / 16) + 8 * (e % 16 / 4) + e % 4)) & 1)) s[e / 16][e % 16] = -INFINITY;
        mx = fmaxf(mx, s[e / 16][e % 16]);
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const int key = key0(kt) + 32 * (e / 16) + 8 * (e % 16 / 4) + 4 * h + e % 4;
      if (key > pos || (PAGED && !((have >> (e / 8)) & 1))) s[e / 16][e % 16] = -INFINITY;
      mx = fmaxf(mx, s[e / 16][e % 16]);
    }
  };
  auto phase1 = [&](auto more, f32x16 (&s)[2], f32x16 (&sn)[2], const bf16_t* sk, const bf16_t* sv, int kt) {
    constexpr bool kMore = decltype(more)::value;
    const AttnLane ln = fresh(lane);
    if constexpr (kMore) {
#pragma unroll
      for (int t = 0; t < PF; ++t) f[t] = kfrag(sk, ln, t);
      sn[0] = sn[1] = zero16();
    }
    mx = max_halves(mx);
    // the maximum is only raised, and what is summed so far scaled down, when some row's grew
    // by more than 2^8: the weights stay below that, far inside bf16 and fp32
    if (__any((mx - m) * cs > 8.f)) {
      const float mn = fmaxf(m, mx);
      const float a = __builtin_amdgcn_exp2f((m - mn) * cs);
      m = mn;
      lsum *= a;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= a;
    }
    const float mc = m * cs;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NG; ++t) {
      if constexpr (kMore) sn[t & 1] = mma32(f[t % PF], q[t / 2], sn[t & 1]);
      if (kMore && t + PF < NG) f[t % PF] = kfrag(sk, ln, t + PF);
      if (t + PF >= NG) f[t % PF] = vfrag(sv, ln, t + PF - NG);
#pragma unroll
      for (int e = EG * t; e < EG * (t + 1); ++e) {
        const int b = e / 16, i = e % 16;
        s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], cs, -mc));
        sum[e & 3] += s[b][i];
        if (e & 1) pb[e / 8][e / 2 % 4] = pack_bf16(s[b][i - 1], s[b][i]);
      }
      // (here: left to itself the compiler puts the sums behind the last product, where nothing runs beside
      // them.  B=4 T=4,096 of 16/4 heads of 64 170 us, now 162; heads of 128 and 256, with more products to run
      // beside and fewer registers, lose up to 1.5% by it, but for 128 in 8 bits, which then spills none.)
      if constexpr (DP == 64 || (EIGHT && DP == 128))
        asm volatile("" : "+v"(sum[0]), "+v"(sum[1]), "+v"(sum[2]), "+v"(sum[3]));
      if (!EIGHT && t % (NG / NF) == 0) fetch_v(kt + 1, pn, t / (NG / NF));
      __builtin_amdgcn_sched_barrier(0);
    }
    lsum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };
  auto phase2 = [&](auto more, f32x16 (&sn)[2], const bf16_t* sv, int kt) {
    const AttnLane ln = fresh(lane);
    mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < NG; ++t) {
      o[t % DB] = mma32(f[t % PF], pb[t / DB], o[t % DB]);
      if (t + PF < NG) f[t % PF] = vfrag(sv, ln, t + PF);
      if constexpr (decltype(more)::value) {
#pragma unroll
        for (int e = EG * t; e < EG * (t + 1); ++e) mx = fmaxf(mx, sn[e / 16][e % 16]);
        if constexpr (DP == 64) asm volatile("" : "+v"(mx));
      }
      if constexpr (EIGHT) {
        static_assert(8 * NR <= NG, "halves of values, then of keys, beside every other product");
        if (t % 2 == 0 && t / 2 < 2 * NR) store8(rv, sV + ((kt + 1) & 1) * kTile, t / 2);
        if (t % 2 == 0 && t / 2 >= 2 * NR && t / 2 < 4 * NR) store8(rk, sK + (kt & 1) * kTile, t / 2 - 2 * NR);
        if (t == 4 * NR) rv = load8(pk, p.v_pages, p.v_exps);
        if (t == 8 * NR - 1) rk = load8(pl, p.k_pages, p.k_exps);
      } else if (t % (NG / 2 / NF) == 0 && t < NG / 2) {
        fetch_k(kt + 2, pk, t / (NG / 2 / NF));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // rows of a staged tile that hold no key, or none that a row sees, are cleared: a weight of zero does
  // not clear them of a NaN
  auto clear = [&](int kt, bf16_t* sv, unsigned have) {
    for (int i = tid; i < kBN * DP / 8; i += kNT) {
      const int r = i / (DP / 8);
      const int key = place(kt * kBN + r);
      if (key >= keys || !((have >> (r / 16)) & 1) || (WIN && key < lo && key >= p.sinks)) *(u32x4*)(sv + 8 * i) = u32x4{0, 0, 0, 0};
    }
  };
  unsigned have = 15;
  // tile kt's values and the next one's keys are there
  auto enter = [&](int kt) {
    if constexpr (!EIGHT) wait_loads<0>();  // this wavefront's part of the tiles
    lds_barrier();    // everyone's; and the other buffers are free
    if constexpr (PAGED) {
      const int k0 = key0(kt);
      if (have != 15 || k0 + kBN > keys || (WIN && k0 < lo && k0 + kBN > p.sinks)) {  // uniform in the workgroup
        clear(kt, sV + (kt & 1) * kTile, have);
        lds_barrier();
      }
    }
  };
  auto leave = [&](int kt) {
    if constexpr (PAGED) {
      have = pn.have;
      pn = pk;
      if constexpr (EIGHT) {
        pk = pl;
        pl = told(pa, 0);
        pa = ask(kt + 5);
      } else {
        pk = told(pa, 0);
        pa = ask(kt + 4);
      }
    }
  };
  if (kt0 < kt1) {
    Pages p0;
    p0.have = pn.have = pk.have = 15;
    if constexpr (PAGED) {
      const Asked all = ask(kt0);
      pa = ask(kt0 + (EIGHT ? 4 : 3));
      load_q();  // (behind the pages, whose answers would wait for them)
      p0 = told(all, 0);
      pn = told(all, 1);
      pk = told(all, 2);
      if constexpr (EIGHT) pl = told(all, 3);
      have = p0.have;
    }
    if constexpr (EIGHT) {
      const Raw k0 = load8(p0, p.k_pages, p.k_exps), v0 = load8(p0, p.v_pages, p.v_exps);
      const Raw k1 = load8(pn, p.k_pages, p.k_exps);
      rv = load8(pn, p.v_pages, p.v_exps);
      rk = load8(pk, p.k_pages, p.k_exps);
      store8_all(k0, sK + (kt0 & 1) * kTile);
      store8_all(v0, sV + (kt0 & 1) * kTile);
      store8_all(k1, sK + ((kt0 + 1) & 1) * kTile);
    } else {
      const bool both = WIN && !PAGED && cut == 0;
      if (both) {
        fetch_cut(p.k, p.k_ld, kld2, koff, sK);
        fetch_cut(p.v, p.v_ld, vld2, voff, sV);
      }
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        if (!both) {
          fetch_k(kt0, p0, j);
          fetch_v(kt0, p0, j);
        }
        fetch_k(kt0 + 1, pn, j);
      }
      wait_loads<0>();
    }
    lds_barrier();
    // the wavefront's own last tile: rows of it see no keys of later ones
    const int w_kt = (w_hi - shift) / kBN, last_kt = w_kt < kt1 - 1 ? w_kt : kt1 - 1;
    int kt = kt0;
    if (kt <= last_kt) {
      f32x16 s0[2], s1[2];
      auto turn = [&](auto more, f32x16 (&s)[2], f32x16 (&sn)[2]) {
        enter(kt);
        const int k0 = key0(kt);
        if (k0 + kBN - 1 > w_lo || have != 15 || (WIN && k0 <= w_hi - p.window && k0 + kBN > p.sinks)) mask(kt, s, have);
        phase1(more, s, sn, sK + ((kt + 1) & 1) * kTile, sV + (kt & 1) * kTile, kt);
        phase2(more, sn, sV + (kt & 1) * kTile, kt);
        leave(kt);
        ++kt;
      };
      first(sK + (kt & 1) * kTile, s0);
      while (kt + 1 < last_kt) {
        turn(Yes(), s0, s1);
        turn(Yes(), s1, s0);
      }
      if (kt < last_kt) {
        turn(Yes(), s0, s1);
        s0[0] = s1[0];
        s0[1] = s1[1];
      }
      turn(No(), s0, s1);
    }
    for (; kt < kt1; ++kt) {  // other wavefronts' tiles: its part of the loads
      enter(kt);
      if constexpr (EIGHT) {
        store8_all(rv, sV + ((kt + 1) & 1) * kTile);
        store8_all(rk, sK + (kt & 1) * kTile);
        rv = load8(pk, p.v_pages, p.v_exps);
        rk = load8(pl, p.k_pages, p.k_exps);
      } else {
#pragma unroll
        for (int j = 0; j < NF; ++j) {
          fetch_v(kt + 1, pn, j);
          fetch_k(kt + 2, pk, j);
        }
      }
      leave(kt);
    }
  }
  wait_loads<0>();

  // A weight of zero does not keep a NaN or an infinity among a tile's values from the rows that do
  // not see it.  Rows whose sums are not finite though their weights are, are summed again over
  // the keys that they see, one row at a time: slow, and only for values that are not finite.
  {
    float z = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) z = fmaf(o[d][i], 0.f, z);
    unsigned long long bad = __ballot(live && z != 0.f && sum_halves(lsum) < INFINITY);
    bad = (bad | bad >> 32) & 0xffffffffu;
    while (bad) {
      const int r = __ffsll(bad) - 1;
      bad &= bad - 1;
      const int row1 = 32 * w + r, pos1 = held + t0 + row1 / G;
      const bf16_t* q1 = (const bf16_t*)p.q + (it.start + t0 + row1 / G) * p.q_ld + (long long)(hk * G + row1 % G) * D;
      const float m1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), r)) * cs;
      float acc[DP / 64];
#pragma unroll
      for (int e = 0; e < DP / 64; ++e) acc[e] = 0.f;
      static_assert(kBN == 64, "a key a lane");
      for (int kt = kt0; kt < kt1 && key0(kt) <= pos1; ++kt) {
        const int key = place(kt * kBN + l);
        bool see = key <= pos1 && (!WIN || key > pos1 - p.window || key < p.sinks);
        long long at = (it.start + key) * p.k_ld + hk * D, av = (it.start + key) * p.v_ld + hk * D;
        if constexpr (PAGED) {
          const int sl = key / p.page;
          const int id = see && sl < p.table_w ? table[sl] : -1;
          see = id >= 0 && id < p.n_pages;
          at = av = ((long long)id * p.page + (key - sl * p.page)) * Hkv * D + hk * D;
        }
        float s1 = 0.f, vs = 0.f;
        if constexpr (EIGHT) {
          if (see) {
            const long long block = at / D / (16 * Hkv) * Hkv + hk;
            const float ks = exp_scale(p.k_exps[block]);
            vs = exp_scale(p.v_exps[block]);
            for (int d = 0; d < D; d += 8) {
              const u32x2 x = *(const u32x2*)((const char*)p.k_pages + at + d);
              s1 = dot8(*(const u32x4*)(q1 + d), widen8(x[0], x[1], ks), s1);
            }
          }
        } else if (see) {
          for (int d = 0; d < D; d += 8)
            s1 = dot8(*(const u32x4*)(q1 + d), *(const u32x4*)((const bf16_t*)(PAGED ? p.k_pages : p.k) + at + d), s1);
        }
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s1, cs, -m1));
        unsigned long long seen = __ballot(see);
        while (seen) {
          const int j = __ffsll(seen) - 1;
          seen &= seen - 1;
          const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p1), j));
          const long long aj = __shfl(av, j, 64);
          const float vsj = EIGHT ? __shfl(vs, j, 64) : 0.f;
#pragma unroll
          for (int e = 0; e < DP / 64; ++e) {
            if (64 * e + l >= D) continue;
            float x;
            if constexpr (EIGHT)
              x = bf2f((bf16_t)(widen4(((const uint8_t*)p.v_pages)[aj + 64 * e + l], vsj)[0] & 0xffffu));
            else
              x = bf2f(((const bf16_t*)(PAGED ? p.v_pages : p.v))[aj + 64 * e + l]);
            acc[e] = fmaf(pj, x, acc[e]);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < DP / 64; ++e) sRow[w][64 * e + l] = acc[e];
      wave_lds_fence();
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = sRow[w][32 * d + 8 * (i / 4) + 4 * h + i % 4];
          o[d][i] = c == r ? x : o[d][i];
        }
      wave_lds_fence();
    }
  }

  // ---------------------------------------------------------------- output
  lsum = sum_halves(lsum);
  if (!live) return;
  const int Hq = Hkv * G, head = hk * G + rg;
  if (PAGED && p.splits > 1) {
    const long long at = ((long long)split * p.tokens + tok) * Hq + head;
    float* po = p.part_o + at * DP;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4*)(po + 32 * d + 8 * g + 4 * h) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (h == 0) {
      p.part_ml[2 * at] = m * cs;
      p.part_ml[2 * at + 1] = lsum;
    }
    return;
  }
  const float inv = lsum > 0.f ? 1.f / lsum : (lsum == 0.f ? 0.f : lsum);  // a NaN stays
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] *= inv;
  store_rows<DB>((bf16_t*)p.o + (tok * Hq + head) * D, o, 1.f, D, h);
  if (p.o_rest) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = lo_part(o[d][i]);
    store_rows<DB>((bf16_t*)p.o_rest + (tok * Hq + head) * D, o, 1.f, D, h);
  }
  if (p.lse && h == 0) p.lse[tok * Hq + head] = lsum > 0.f ? m * p.scale + __logf(lsum) : (lsum == 0.f ? -INFINITY : lsum);
}

// Joins the shares of a row: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, with W of a
// workgroup's four wavefronts on one row, each lane E columns.  The weights are formed once, a
// share a lane.  Bound by its reads, 4 (DP + 2) bytes a share and row, and for few rows by the
// latency of a wavefront's chain of reads, which the four cut short.
template <int DP, int W>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnParams p) {
  constexpr int E = DP / 64;
  typedef float fE __attribute__((ext_vector_type(E)));
  __shared__ float sAcc[4][DP];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, part = w % W;
  const long long rows = p.tokens * p.Hkv * p.G, row = (long long)blockIdx.x * (4 / W) + w / W;
  const bool live = row < rows;
  float acc[E], den = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (live) {
    static_assert(kAttnMaxSplits <= 64, "a share a lane");
    float a = kLow * kLog2e, ls = 0.f;
    if (l < p.splits) {
      a = p.part_ml[2 * (l * rows + row)];
      ls = p.part_ml[2 * (l * rows + row) + 1];
    }
    float M = a;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    a = ls == 0.f ? 0.f : __builtin_amdgcn_exp2f(a - M);
    den = wave_sum(a * ls);
    for (int s = part; s < p.splits; s += 8 * W) {  // eight reads in flight
      fE x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int su = s + W * u < p.splits ? s + W * u : p.splits - 1;
        x[u] = *(const fE*)(p.part_o + (su * rows + row) * DP + E * l);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float as = __shfl(a, s + W * u, 64);
        const float f = s + W * u < p.splits ? as : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += f * x[u][e];
      }
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) sAcc[w][E * l + e] = acc[e];
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int x = 1; x < W; ++x) acc[e] += sAcc[w + x][E * l + e];
  }
  if (!live) return;
  const float inv = den > 0.f ? 1.f / den : (den == 0.f ? 0.f : den);
  bf16_t* op = (bf16_t*)p.o + row * DP + E * l;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = f2bf(acc[e] * inv);
}

// The tile list of more than 64 packed sequences, and their repaired offsets: one workgroup.
// plan: [count, 0, (sequence, tile) by rank], tiles with most keys first.  Tiles are counted by
// place in kBuckets buckets of equal width, then placed bucket by bucket from the last; within a
// bucket the order is of no consequence.
constexpr int kPlanNT = 1024, kBuckets = 2048;
__global__ __launch_bounds__(kPlanNT) void attn_plan_kernel(const int32_t* cu, const int32_t* held, int cap,
                                                            int32_t* plan, int32_t* out, int N, int T, int per) {
  __shared__ int sScan[kPlanNT], sCount[kBuckets];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  int shift = 0;
  while (((T + per - 1) / per + (held ? cap / per : 0)) >> shift >= kBuckets) ++shift;
  for (int i = tid; i < kBuckets; i += kPlanNT) sCount[i] = 0;
  // the ordered repair: a running maximum of the clamped offsets
  int carry = 0;
  for (int n0 = 0; n0 < N; n0 += kPlanNT) {
    const int n = n0 + tid;
    int e = n + 1 < N ? cu[n + 1] : T;
    e = e < 0 ? 0 : (e > T ? T : e);
    sScan[tid] = e > carry ? e : carry;
    __syncthreads();
    for (int o = 1; o < kPlanNT; o <<= 1) {
      const int x = tid >= o ? sScan[tid - o] : 0;
      __syncthreads();
      if (x > sScan[tid]) sScan[tid] = x;
      __syncthreads();
    }
    if (n < N) out[n + 1] = sScan[tid];
    carry = sScan[kPlanNT - 1];
    __syncthreads();
  }
  if (tid == 0) out[0] = 0;
  __syncthreads();  // out is read below by other threads of this workgroup
  for (int n = w; n < N; n += kPlanNT / 64) {
    const int nt = (out[n + 1] - out[n] + per - 1) / per, first = tiles_held(held, n, cap, per);
    for (int j = l; j < nt; j += 64) atomicAdd(&sCount[(first + j) >> shift], 1);
  }
  __syncthreads();
  // where each bucket starts: the tiles of later buckets come first
  if (tid == 0) {
    int at = 0;
    for (int b = kBuckets - 1; b >= 0; --b) {
      const int x = sCount[b];
      sCount[b] = at;
      at += x;
    }
    plan[0] = at;
    plan[1] = 0;
  }
  __syncthreads();
  for (int n = w; n < N; n += kPlanNT / 64) {
    const int nt = (out[n + 1] - out[n] + per - 1) / per, first = tiles_held(held, n, cap, per);
    for (int j = l; j < nt; j += 64) {
      const int at = atomicAdd(&sCount[(first + j) >> shift], 1);
      plan[2 + 2 * (long long)at] = n;
      plan[3 + 2 * (long long)at] = j;
    }
  }
}

int padded_dim(int D) { return D <= 64 ? 64 : (D <= 128 ? 128 : 256); }

template <int DP>
void join(const AttnParams& p, hipStream_t stream) {
  const long long rows = p.tokens * p.Hkv * p.G;
  if (p.splits > 8)
    attn_join_kernel<DP, 4><<<(unsigned)rows, 256, 0, stream>>>(p);
  else
    attn_join_kernel<DP, 1><<<(unsigned)((rows + 3) / 4), 256, 0, stream>>>(p);
}

hipError_t launch_attn_join(const AttnParams& p, hipStream_t stream) {
  switch (padded_dim(p.D)) {
    case 64: join<64>(p, stream); break;
    case 128: join<128>(p, stream); break;
    default: join<256>(p, stream); break;
  }
  return hipGetLastError();
}

}  // namespace

int attn_tile_tokens(int G) { return kBM / G; }

long long attn_ranks(const AttnParams& p, int per) {
  const long long tiles = ((long long)p.T + per - 1) / per;
  if (!p.cu) return tiles;
  const long long most = tiles + p.N;  // a sequence adds at most one partial tile
  return most < p.T ? most : p.T;
}

size_t attn_plan_words(long long T, long long N, int per) {
  if (N <= 64) return 0;
  return (size_t)(2 + 2 * ((T + per - 1) / per + N));
}

hipError_t launch_attn_plan(const AttnParams& p, int per, hipStream_t stream) {
  attn_plan_kernel<<<1, kPlanNT, 0, stream>>>(p.cu, p.held, p.table_w * p.page, p.plan, p.cu_plan, p.N,
                                                    p.T, per);
  return hipGetLastError();
}

hipError_t launch_attn_fwd(const AttnParams& p, hipStream_t stream) {
  const int per = attn_tile_tokens(p.G);
  const long long ranks = attn_ranks(p, per), units = (long long)(p.cu ? 1 : p.N) * p.Hkv;
  const bool paged = p.k_pages != nullptr;
  const dim3 grid((unsigned)attn_grid(units, ranks), paged ? (unsigned)p.splits : 1u);
  const bool win = p.window > 0;
  switch (padded_dim(p.D)) {
#define OMX_FWD1(DP, CACHE)                                                      \
  if (win)                                                                       \
    attn_fwd_kernel<DP, CACHE, true><<<grid, kNT, 0, stream>>>(p, (int)ranks);   \
  else                                                                           \
    attn_fwd_kernel<DP, CACHE, false><<<grid, kNT, 0, stream>>>(p, (int)ranks);
#define OMX_FWD(DP)                                                              \
  case DP:                                                                       \
    if (paged && p.k_exps) {                                                     \
      OMX_FWD1(DP, 2)                                                            \
    } else if (paged) {                                                          \
      OMX_FWD1(DP, 1)                                                            \
    } else {                                                                     \
      OMX_FWD1(DP, 0)                                                            \
    }                                                                            \
    break;
    OMX_FWD(64)
    OMX_FWD(128)
    OMX_FWD(256)
#undef OMX_FWD
#undef OMX_FWD1
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !paged || p.splits == 1) return e;
  return launch_attn_join(p, stream);
}

}  // namespace omx
