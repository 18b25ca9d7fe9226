// Softmax attention: what its kernels share.
//
// Rows.  A key head's g = Hq / Hkv query heads see the same keys, so their queries are one
// matrix: row r of a tile that starts at token t0 is token t0 + r / g, head r % g.  A tile of R
// rows takes the whole tokens that fit, R / g, and leaves the rest of its rows idle.  A tile
// then reads its keys once for all g heads, and the gradients of a key head sum over its query
// heads inside one product.
//
// Fragments.  All products are v_mfma_f32_32x32x16_bf16 with, for l the lane, h = l / 32 and
// c = l % 32 (verified on MI355X by products of small integers):
//   A[c][8h .. 8h+7],  B[8h .. 8h+7][c],  C[8 (i / 4) + 4h + i % 4][c], i = 0..15
// A product that leaves its result C[key][row] feeds the next one, whose contraction runs over
// the keys, without exchanging lanes: elements 8s .. 8s+7 of a lane's C are the keys 16s + 4h +
// {0..3, 8..11}, and taking them as the B operand of step s only asks that the A operand lists
// its keys in the same order, which two transposed LDS reads of 4 keys each do.
#pragma once

#include "gdn_common.h"
#include "gdn_kernels.h"
#include "gdn_mfma.h"

namespace omx {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) void glob_void;

// C += A(32x16) B(16x32)
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// elements 8s .. 8s+7 of a C fragment as a B operand (see the top of this file)
__device__ __forceinline__ u32x4 pack8_of(const f32x16& c, int s) {
  return u32x4{pack_bf16(c[8 * s], c[8 * s + 1]), pack_bf16(c[8 * s + 2], c[8 * s + 3]),
               pack_bf16(c[8 * s + 4], c[8 * s + 5]), pack_bf16(c[8 * s + 6], c[8 * s + 7])};
}

// value of the lane 32 away combined with the lane's own
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// four-element pieces of a C fragment's column, scaled, rounded and exchanged between the halves
// of the wavefront so that each lane stores 8 neighbours of its row
template <int DB>
__device__ __forceinline__ void store_rows(bf16_t* row, const f32x16 (&x)[DB], float f, int D, int h) {
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      const auto a = __builtin_amdgcn_permlane32_swap(pack_bf16(x[d][4 * g] * f, x[d][4 * g + 1] * f),
                                                      pack_bf16(x[d][4 * g + 4] * f, x[d][4 * g + 5] * f), false, false);
      const auto b = __builtin_amdgcn_permlane32_swap(pack_bf16(x[d][4 * g + 2] * f, x[d][4 * g + 3] * f),
                                                      pack_bf16(x[d][4 * g + 6] * f, x[d][4 * g + 7] * f), false, false);
      const int col = 32 * d + 8 * g + 8 * h;
      if (col < D) *(u32x4*)(row + col) = u32x4{a[0], b[0], a[1], b[1]};
    }
}

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

// A cache in 8 bits: e4m3 numbers, with a power of two for each 16 tokens of a head, kept as its
// exponent.  Number times power is a bf16 value as it stands (the conversion applies both; verified on
// MI355X for every code), so whoever reads it goes on as with a cache of bf16.
__device__ __forceinline__ float exp_scale(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }
__device__ __forceinline__ u32x2 widen4(uint32_t c, float scale) {
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, true))};
}
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi, float scale) {
  const u32x2 a = widen4(lo, scale), b = widen4(hi, scale);
  return u32x4{a[0], a[1], b[0], b[1]};
}

// s + the products of two rows' 8 bf16 elements
__device__ __forceinline__ float dot8(u32x4 a, u32x4 b, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, (uint32_t)a[i]),
                                        __builtin_bit_cast(bf16x2_t, (uint32_t)b[i]), s, false);
  return s;
}

// Rows of DP bf16 in LDS without padding, in 16-byte segments: segment s of row r lies at
// s ^ swz(r).  One pass of a 16-byte read serves lanes {0-3, 12-15, 20-27} (and the rest of
// each half), whose rows' images must differ in the 16 segments that the 64 banks hold; one
// pass of a transposed 8-byte read serves four neighbouring rows' four neighbouring segments,
// which must lie in different quarters.  The row's low bits go to the segment's high ones and
// the other way round, which gives both.  Rows of 64 elements fill the banks two by two.
template <int DP>
__device__ __forceinline__ int attn_swz(int r) {
  return DP == 64 ? ((((r >> 1) & 1) << 2) | ((r >> 2) & 3)) : (((r & 3) << 2) | ((r >> 2) & 3));
}

// A lane's byte offsets in such a tile, for the two kinds of fragments: step and column block
// only flip bits of the segment.
struct AttnLane {
  unsigned f, t;
};
template <int DP>
__device__ __forceinline__ AttnLane attn_lane() {
  const int l = lane_id(), h = l >> 5, c = l & 31, s = l & 15, r = 4 * h + (s >> 2);
  return {(unsigned)(c * DP * 2 + ((h ^ attn_swz<DP>(c)) << 4)),
          (unsigned)(r * DP * 2 + (((2 * ((l >> 4) & 1) + ((s >> 1) & 1)) ^ attn_swz<DP>(r)) << 4) + 8 * (s & 1))};
}
// the same, recomputed from here on: keeps the compiler from holding every offset in a register
__device__ __forceinline__ AttnLane fresh(AttnLane ln) {
  asm volatile("" : "+v"(ln.f), "+v"(ln.t));
  return ln;
}

// A operand (32 rows row0 .. +31, elements 16 step .. +15) of a [row][DP] LDS tile
template <int DP>
__device__ __forceinline__ u32x4 attn_frag(const bf16_t* base, AttnLane ln, int row0, int step) {
  return *(const u32x4*)((const char*)(base + row0 * DP) + (ln.f ^ (unsigned)(step << 5)));
}

// A operand whose rows are the tile's columns 32 cb .. +31 and whose contraction runs over its
// rows row0 + {4h .. +3, 8 + 4h .. +3}: the order of pack8_of (row0 a multiple of 16; eight rows
// on, the swizzle differs in bit 1)
template <int DP>
__device__ __forceinline__ u32x4 attn_frag_tr(const bf16_t* base, AttnLane ln, int row0, int cb) {
  const unsigned at = ln.t ^ (unsigned)(cb << 6);
  const u32x2 a = ds_read_tr((const bf16_t*)((const char*)(base + row0 * DP) + at));
  const u32x2 b = ds_read_tr((const bf16_t*)((const char*)(base + (row0 + 8) * DP) + (at ^ 32u)));
  return u32x4{a[0], a[1], b[0], b[1]};
}

// Loads of 16 (or 4) bytes a lane into LDS at `lds` + 16 (4) lane, past the compiler's book of
// outstanding loads: with the builtin it put a wait for all of them before reads of buffers that
// they do not touch.  Whoever reads the bytes waits for them with wait_loads.
// (The resource's words are uniform; readfirstlane also puts one there that the compiler keeps in
// a vector register, and five wait states then lie between that write and the load.  m0, which
// holds the LDS address, is named as overwritten: the compiler sets it before each use of its own,
// and must not count on an earlier value.  It warns that it would not save a reserved register's.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ u32x4 rsrc_words(const void* p, unsigned bytes) {
  const unsigned long long a = (unsigned long long)p;
  return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((unsigned)a),
               (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffffu),
               (unsigned)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}
// the same for the builtin loads: of a resource that the compiler does not know to be uniform they become
// a loop over its values
__device__ __forceinline__ __amdgpu_buffer_rsrc_t uniform_rsrc(const void* p, unsigned bytes) {
  const unsigned long long a = (unsigned long long)p;
  const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((unsigned)a);
  const unsigned hi = (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
  return buf_rsrc((const void*)((unsigned long long)hi << 32 | lo), (unsigned)__builtin_amdgcn_readfirstlane(bytes));
}
// zero, as a lane's offset that the compiler takes for one of its own: a value that it knows to be the same for
// all lanes goes to a scalar register, and is waited for, as soon as it is loaded
__device__ __forceinline__ unsigned lane_zero() {
  unsigned z = 0;
  asm("" : "+v"(z));
  return z;
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(unsigned long long)(const __attribute__((address_space(3))) char*)p;
}
__device__ __forceinline__ void load_to_lds16(u32x4 rsrc, unsigned lds, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(rsrc) : "memory", "m0");
}
// several of them, each 4 KiB further in LDS: a workgroup of four wavefronts takes turns
__device__ __forceinline__ void loads_to_lds16(u32x4 rsrc, unsigned lds, const unsigned (&off)[4]) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
               "s_add_u32 m0, m0, 4096\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
               "s_add_u32 m0, m0, 4096\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
               "s_add_u32 m0, m0, 4096\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %5, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]),
                  "s"(rsrc) : "memory", "m0", "scc");
}
__device__ __forceinline__ void loads_to_lds16(u32x4 rsrc, unsigned lds, const unsigned (&off)[2]) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
               "s_add_u32 m0, m0, 4096\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off[0]), "v"(off[1]), "s"(rsrc) : "memory", "m0", "scc");
}
__device__ __forceinline__ void loads_to_lds16(u32x4 rsrc, unsigned lds, const unsigned (&off)[1]) {
  load_to_lds16(rsrc, lds, off[0]);
}
// N of them, each 1 KiB further in LDS: one wavefront
__device__ __forceinline__ void loads_to_lds16_on(u32x4 rsrc, unsigned lds, const unsigned (&off)[4]) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
               "s_add_u32 m0, m0, 1024\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
               "s_add_u32 m0, m0, 1024\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
               "s_add_u32 m0, m0, 1024\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %5, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]),
                  "s"(rsrc) : "memory", "m0", "scc");
}
__device__ __forceinline__ void loads_to_lds16_on(u32x4 rsrc, unsigned lds, const unsigned (&off)[2]) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
               "s_add_u32 m0, m0, 1024\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off[0]), "v"(off[1]), "s"(rsrc) : "memory", "m0", "scc");
}
__device__ __forceinline__ void loads_to_lds16_on(u32x4 rsrc, unsigned lds, const unsigned (&off)[1]) {
  load_to_lds16(rsrc, lds, off[0]);
}
// a byte a lane, into the low byte of 4 at `lds` + 4 lane
__device__ __forceinline__ void load_to_lds1(u32x4 rsrc, unsigned lds, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_ubyte %1, %2, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(rsrc) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds4(u32x4 rsrc, unsigned lds, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop

// waits until at most N of the wavefront's vector memory operations are outstanding
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "the counter's range");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// A lane's fragments (elements 8h .. of each 16) of a row of D elements, D a multiple of 8.  No load
// is behind a branch, where each would be waited for before the next; what lies past D is cleared
// once all are issued.
template <int KS>
__device__ __forceinline__ void load_row(u32x4 (&x)[KS], const void* row, int D, int h) {
#pragma unroll
  for (int s = 0; s < KS; ++s) x[s] = *(const u32x4*)((const bf16_t*)row + (16 * s + 8 * h < D ? 16 * s + 8 * h : 0));
}
template <int KS>
__device__ __forceinline__ void clear_past(u32x4 (&x)[KS], int D, int h) {
  if (D == 16 * KS) return;
#pragma unroll
  for (int s = 0; s < KS; ++s)
    if (16 * s + 8 * h >= D) x[s] = u32x4{0, 0, 0, 0};
}

// One staging instruction writes 1 KiB of LDS, 64 / (DP / 8) rows.  Of a tile's instructions a
// wavefront takes w, w + NW, ...: row of lane l in its j-th, and the segment it fetches.
template <int DP, int NW>
__device__ __forceinline__ int stage_row(int w, int j) {
  constexpr int CH = DP / 8;
  return (64 / CH) * (w + NW * j) + lane_id() / CH;
}
template <int DP>
__device__ __forceinline__ int stage_seg(int row) {
  return (lane_id() % (DP / 8)) ^ attn_swz<DP>(row);
}

// Inclusive sum and maximum over the lanes of non-negative integers, by lane shifts within rows of
// 16 and two broadcasts of a row's last lane (a few cycles each, where an exchange through LDS
// takes a hundred), and the total.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_i<0x111, 0xf>(v);
  v += dpp_i<0x112, 0xf>(v);
  v += dpp_i<0x114, 0xf>(v);
  v += dpp_i<0x118, 0xf>(v);
  v += dpp_i<0x142, 0xa>(v);
  v += dpp_i<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ int wave_scan_max(int v) {
  auto up = [&](int x) { v = x > v ? x : v; };
  up(dpp_i<0x111, 0xf>(v));
  up(dpp_i<0x112, 0xf>(v));
  up(dpp_i<0x114, 0xf>(v));
  up(dpp_i<0x118, 0xf>(v));
  up(dpp_i<0x142, 0xa>(v));
  up(dpp_i<0x143, 0xc>(v));
  return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// Which tile a workgroup takes: sequence `seq` of tokens start .. start + len, tile `tile` of
// `tiles`.
struct AttnTile {
  int seq, len, tile, tiles;
  long long start;
};

// Tokens a sequence has before its first tile's, in tiles: its tiles' places in the order of work.
__device__ __forceinline__ int tiles_held(const int32_t* held, int n, int cap, int per) {
  if (!held) return 0;
  const int x = held[n];
  return (x < 0 ? 0 : (x < cap ? x : cap)) / per;
}

// Tokens of sequence n of at most 64 in lane n; the offsets are read as their ordered repair.
__device__ __forceinline__ void packed_span(const int32_t* cu, int N, int T, int& start, int& len) {
  const int n = lane_id();
  int end = n + 1 < N ? cu[n + 1] : T;
  end = end < 0 ? 0 : (end > T ? T : end);
  end = wave_scan_max(end);
  const int prev = __shfl_up(end, 1, 64);
  start = n == 0 ? 0 : prev;
  len = n < N ? end - start : 0;
}

// Tile of rank `rank` of sequences packed by cu, those with most keys first (a tile's work grows
// with its index, from what a cache held on), found by every wavefront for itself when there are
// at most 64 sequences: lane n holds sequence n.
__device__ __forceinline__ bool packed_tile(const int32_t* cu, const int32_t* held, int cap, int N, int T, int per,
                                            int rank, AttnTile& it) {
  const int n = lane_id();
  int start, len;
  packed_span(cu, N, T, start, len);
  const int nt = (len + per - 1) / per;
  const int first = n < N ? tiles_held(held, n, cap, per) : 0;
  // at(j): tiles of place j and more
  auto at = [&](int j) {
    int v = first + nt - j;
    return wave_total(v < 0 ? 0 : (v > nt ? nt : v));
  };
  if (rank >= at(0)) return false;
  int lo = 0, hi = (T + per - 1) / per + (held ? cap / per : 0);  // at(lo) > rank >= at(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at(mid) > rank) lo = mid; else hi = mid;
  }
  const int k = rank - at(lo + 1);  // the k-th of the sequences that have a tile at place lo
  const bool has = first <= lo && lo < first + nt;
  const unsigned long long have = __ballot(has);
  const unsigned long long below = have & ((1ull << n) - 1);
  const unsigned long long mine = __ballot(has && __popcll(below) == k);
  const int s = __ffsll(mine) - 1;
  it.seq = __builtin_amdgcn_readfirstlane(s);
  it.start = __builtin_amdgcn_readlane(start, it.seq);
  it.len = __builtin_amdgcn_readlane(len, it.seq);
  it.tile = lo - __builtin_amdgcn_readlane(first, it.seq);
  it.tiles = __builtin_amdgcn_readlane(nt, it.seq);
  return true;
}

// Tile of rank `rank` of sequence or packed row `row`; false past the last one.
__device__ __forceinline__ bool attn_tile(const AttnParams& p, int row, int rank, int per,
                                          AttnTile& it) {
  if (!p.cu) {
    it.seq = row;
    it.len = p.T;
    it.start = (long long)row * p.T;
    it.tiles = (p.T + per - 1) / per;
    it.tile = it.tiles - 1 - rank;
    return it.tile >= 0;
  }
  if (!p.plan) return packed_tile(p.cu, p.held, p.table_w * p.page, p.N, p.T, per, rank, it);
  // more than 64 sequences: the plan kernel's list (count, then sequence and tile per rank)
  const int32_t* plan = p.plan;
  if (rank >= __builtin_amdgcn_readfirstlane(plan[0])) return false;
  it.seq = __builtin_amdgcn_readfirstlane(plan[2 + 2 * (long long)rank]);
  it.tile = __builtin_amdgcn_readfirstlane(plan[3 + 2 * (long long)rank]);
  const int start = __builtin_amdgcn_readfirstlane(p.cu_plan[it.seq]);
  it.start = start;
  it.len = __builtin_amdgcn_readfirstlane(p.cu_plan[it.seq + 1]) - start;
  it.tiles = (it.len + per - 1) / per;
  return true;
}

// Order of the workgroups: (unit, rank) of workgroup `bid`, with units (a sequence's or packed
// row's key head) kept on few of the 8 XCDs, whose L2s then hold that head's keys and values.
// Consecutive workgroups go to consecutive XCDs.  The grid is attn_grid() workgroups; ranks
// past a unit's last tile have nothing to do.
__device__ __forceinline__ void attn_place(int bid, int units, int ranks, int& unit, int& rank) {
  if (units % 8 == 0) {
    const int x = bid & 7, j = bid >> 3, each = units / 8;
    unit = x + 8 * (j % each);
    rank = j / each;
  } else if (8 % units == 0) {
    const int x = bid & 7, j = bid >> 3, r = 8 / units;
    unit = x / r;
    rank = j * r + x % r;
  } else {
    unit = bid % units;
    rank = bid / units;
  }
}
inline long long attn_grid(long long units, long long ranks) {
  if (units % 8 != 0 && 8 % units == 0) {
    const long long r = 8 / units;
    return 8 * ((ranks + r - 1) / r);
  }
  return units * ranks;
}

// keys of a workgroup's tile of the kernels that sum dk and dv
constexpr int kDkvKeys = 128;

// Work of a workgroup of the kernels that sum dk and dv: rows of tokens [ta, tb), whole stages of
// `per` and at least one, for the 128 keys from k0 on.  When there are few tiles, workgroups share a
// tile's rows.  Those grow with the tile's place j, counted from its sequence's end: it has
// ceil((j + 1) / m) shares, so that shares are alike, with m = p.share_tiles unless the longest tile
// would have more than `splits` then.
struct DkvShare {
  int len, k0, ta, tb, share, shares;
  long long start;
};

// That of rank `rank` of sequence or packed row `row`, of at most 64 sequences if there are shares;
// false past the last.  Tiles that most rows see come first (of each sequence, when shared).
__device__ __forceinline__ bool dkv_share(const AttnParams& p, int row, int rank, int per, DkvShare& it) {
  int len, tiles, tile, share = 0, shares = 1;
  long long start;
  if (p.splits == 1) {
    AttnTile t;
    if (!attn_tile(p, row, rank, kDkvKeys, t)) return false;
    len = t.len, tiles = t.tiles, tile = t.tile, start = t.start;
  } else {
    int first = 0, n = lane_id() == 0 ? p.T : 0;  // lane i: sequence i
    if (p.cu) packed_span(p.cu, p.N, p.T, first, n);
    const int nt = (n + kDkvKeys - 1) / kDkvKeys;
    const int least = (__builtin_amdgcn_readlane(wave_scan_max(nt), 63) + p.splits - 1) / p.splits;
    const int m = p.share_tiles > least ? p.share_tiles : least;
    int mine = 0;  // nt tiles' shares, m tiles a time
    for (int q = 0; q < p.splits; ++q) {
      const int left = nt - q * m;
      mine += (q + 1) * (left < 0 ? 0 : (left < m ? left : m));
    }
    const int end = wave_scan(mine);
    const unsigned long long past = __ballot(end > rank);
    if (!past) return false;
    const int s = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
    int x = __builtin_amdgcn_readlane(end, s) - 1 - rank, q = 0;  // from the sequence's last tile on
    while (q + 1 < p.splits && x >= (q + 1) * m) x -= ++q * m;
    start = (p.cu ? 0 : (long long)row * p.T) + __builtin_amdgcn_readlane(first, s);
    len = __builtin_amdgcn_readlane(n, s);
    tiles = __builtin_amdgcn_readlane(nt, s);
    shares = q + 1;
    tile = q * m + x / shares;
    share = x % shares;
  }
  const int k0 = (tiles - 1 - tile) * kDkvKeys;
  int ta = k0, tb = len;
  if (shares > 1) {  // j >= shares - 1 tiles lie behind this one, of at least four stages but for the last
    const int n = (len - k0 + per - 1) / per;
    ta = k0 + n * share / shares * per;
    if (share + 1 < shares) tb = k0 + n * (share + 1) / shares * per;
  }
  it.len = len, it.k0 = k0, it.ta = ta, it.tb = tb, it.share = share, it.shares = shares, it.start = start;
  return true;
}

// The same with a window.  A tile of keys is seen by the rows up to window - 1 behind its last key; one
// that holds sinks (its first ceil(sinks / 128) of them) by all rows behind it.  Those come first, with up
// to p.sink_splits shares each, the others as without a window, with up to p.splits, all of p.share_tiles
// tiles' rows or so.
__device__ __forceinline__ int window_shares(int tiles, int per, int most) {
  const int n = (tiles + per - 1) / per;
  return n < 1 ? 1 : (n < most ? n : most);
}
// shares of the last n tiles of a sequence: of the x-th from its end min(x / m, splits - 1) + 1
__device__ __forceinline__ int tail_shares(int n, int m, int splits) {
  int sum = 0;
  for (int q = 0; q < splits; ++q) {
    const int left = n - q * m;
    sum += (q + 1) * (left < 0 ? 0 : (left < m || q + 1 == splits ? left : m));
  }
  return sum;
}

struct WindowShare : DkvShare {
  int seq;
  bool sink;
};
__device__ __forceinline__ bool dkv_window_share(const AttnParams& p, int row, int rank, int per, WindowShare& it) {
  const int sinks = (int)((p.sinks + kDkvKeys - 1ll) / kDkvKeys);
  int len, tile, share = 0, shares = 1;
  long long start;
  if (p.splits == 1 && p.sink_splits == 1) {
    AttnTile t;
    if (!attn_tile(p, row, rank, kDkvKeys, t)) return false;
    len = t.len, tile = t.tiles - 1 - t.tile, start = t.start, it.seq = t.seq;
  } else {
    int first = 0, n = lane_id() == 0 ? p.T : 0;  // lane i: sequence i
    if (p.cu) packed_span(p.cu, p.N, p.T, first, n);
    const int nt = (n + kDkvKeys - 1) / kDkvKeys, ns = nt < sinks ? nt : sinks;
    const int a = window_shares(nt, p.share_tiles, p.sink_splits);
    const int end = wave_scan(ns * a + tail_shares(nt - ns, p.share_tiles, p.splits));
    const unsigned long long past = __ballot(end > rank);
    if (!past) return false;
    const int s = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
    const int nsinks = __builtin_amdgcn_readlane(ns, s), na = __builtin_amdgcn_readlane(a, s);
    int x = rank - (s > 0 ? __builtin_amdgcn_readlane(end, s - 1) : 0);
    if (x < nsinks * na) {
      tile = x / na, share = x % na, shares = na;
    } else {
      x = __builtin_amdgcn_readlane(end, s) - 1 - rank;  // from the sequence's last tile on
      int q = 0;
      while (q + 1 < p.splits && x >= (q + 1) * p.share_tiles) x -= ++q * p.share_tiles;
      shares = q + 1;
      tile = __builtin_amdgcn_readlane(nt, s) - 1 - (q * p.share_tiles + x / shares);
      share = x % shares;
    }
    start = (p.cu ? 0 : (long long)row * p.T) + __builtin_amdgcn_readlane(first, s);
    len = __builtin_amdgcn_readlane(n, s);
    it.seq = p.cu ? s : row;
  }
  const int k0 = tile * kDkvKeys;
  it.sink = tile < sinks;
  int ta = k0, tb = len;
  if (!it.sink && len - k0 > kDkvKeys - 1 + p.window) tb = k0 + kDkvKeys - 1 + p.window;
  if (shares > 1) {  // whole stages
    const long long n = (tb - k0 + per - 1) / per;
    ta = k0 + (int)(n * share / shares) * per;
    if (share + 1 < shares) tb = k0 + (int)(n * (share + 1) / shares) * per;
  }
  it.len = len, it.k0 = k0, it.ta = ta, it.tb = tb, it.share = share, it.shares = shares, it.start = start;
  return true;
}

// Where a workgroup's partial sums of a key go: element `at` of the tokens' keys, `slot` of the sinks'.
__device__ __forceinline__ long long dkv_part(const AttnParams& p, const DkvShare& it, long long at, float*& k, float*& v) {
  k = p.part_k, v = p.part_v;
  return (long long)it.share * p.tokens * p.Hkv * p.D + at;
}
__device__ __forceinline__ long long dkv_part(const AttnParams& p, const WindowShare& it, long long at, float*& k, float*& v) {
  if (!it.sink) return dkv_part(p, (const DkvShare&)it, at, k, v);
  k = p.sink_k, v = p.sink_v;
  const long long keys = (p.sinks + kDkvKeys - 1ll) / kDkvKeys * kDkvKeys, row = (long long)p.Hkv * p.D;
  return (((long long)it.share * p.N + it.seq) * keys) * row + (at - it.start * row);
}

// Which of the 64 keys from k0 on a row at `pos` sees, a bit a key.  (Compared key by key, the bounds took 32
// registers more, and with those of a cache thousands were spilled.)
__device__ __forceinline__ unsigned long long keys_below(int n) {
  return n <= 0 ? 0ull : (n < 64 ? (1ull << n) - 1 : ~0ull);
}
__device__ __forceinline__ unsigned long long window_bits(const AttnParams& p, int pos, int k0) {
  const int upto = pos + 1 - k0;
  return keys_below(upto) & (~keys_below(upto - p.window) | keys_below(p.sinks - k0));
}

// Rows r of a stage that starts at token t which do not see key `key`: those before it, r < first, and with
// a window r >= past.
struct RowMask {
  int first, past;
};
__device__ __forceinline__ RowMask row_mask(const AttnParams& p, int key, int t) {
  const int back = key > t ? key - t : 0, on = p.window - (t - key);
  return {back * p.G, key < p.sinks ? 1 << 30 : (on < 0 ? 0 : (on < 64 ? on * p.G : 1 << 30))};
}
// whether some row of a stage of `per` tokens is past the window of some of 32 keys
__device__ __forceinline__ bool past_window(const AttnParams& p, int kw, int t, int per) {
  return t + (per - 1) - kw >= p.window && kw + 32 > p.sinks;
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace omx
