// Pages of a paged cache, dealt and returned on the GPU: no length leaves it.
//
// Free pages lie on a stack: free[0 .. count).  Of the entries that new tokens need and that name no page
// yet, in order of sequence and slot, the k-th takes free[count - 1 - k]; of those that are returned, n in
// all, the k-th goes to free[count + n - 1 - k], so that what is dealt and returned leaves the stack as it was.
// Every place is a prefix sum, so the order of execution changes nothing.  Bound by latency: a few
// dependent reads, and for many tokens the 12 bytes written for each.  One workgroup deals a whole batch, its
// entries 16 a thread to one sum: 64 sequences of a token each 8.1 us, and 8.3 to return none; 512 prompts
// of 300 on pages of 16 14.0, 4.2 for their tokens' slots and 11.8 to return them.  (With a sum for every turn's
// entry of a thread the calls took 37 and 50 us.)
#include <climits>

#include "gdn_attn.h"

namespace omx {
namespace {

constexpr int kNT = 1024;

// Inclusive sum over the workgroup, and its total; `s` holds a word a wavefront.
template <int NT, class I>
__device__ __forceinline__ I block_scan(I v, I* s, I& total) {
  const int l = lane_id(), w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const I x = __shfl_up(v, o, 64);
    if (l >= o) v += x;
  }
  __syncthreads();
  if (l == 63) s[w] = v;
  __syncthreads();
  I before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i < w) before += s[i];
    total += s[i];
  }
  return before + v;
}

__device__ __forceinline__ bool a_page(int id, int n_pages) { return id >= 0 && id < n_pages; }
__device__ __forceinline__ int on_stack(const PagesParams& p) {
  const int c = *p.count;
  return c < 0 ? 0 : (c < p.n_pages ? c : p.n_pages);
}

// the last n in [0, N) with start[n] <= x, for start[0] <= x; S: of any memory
template <class S>
__device__ __forceinline__ int last_upto(const S* start, int N, int x) {
  int lo = 0, hi = N;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// positions and slots of packed tokens t
template <class S>
__device__ __forceinline__ void map_token(const PagesParams& p, const S* cu, int used, int t) {
  int pos = -1;
  long long slot = -1;
  if (t < used) {
    const int n = last_upto(cu, p.N, t);
    const unsigned at = (unsigned)p.lengths[n] + (unsigned)(t - cu[n]), i = at / (unsigned)p.page;
    pos = at < INT_MAX ? (int)at : INT_MAX;
    const int id = i < (unsigned)p.table_w ? p.table[(long long)n * p.table_w + i] : -1;
    if (a_page(id, p.n_pages)) slot = (long long)id * p.page + (at - i * (unsigned)p.page);
  }
  p.positions[t] = pos;
  p.slots[t] = slot;
}

// Four counts of up to 16 bits each in one word: a turn of the loops below takes 4 kNT neighbouring entries of
// a table four times over, four a thread each time, and finds all their places by one sum.
__device__ __forceinline__ int field(unsigned long long x, int j) { return (int)(x >> 16 * j & 0xffff); }

// One workgroup: the sequences' offsets, then their entries, flat, and (map) their tokens.
// `first`: [N + 1] entries before each sequence's, in LDS (kLdsSeqs of them at most) or memory.
constexpr int kLdsSeqs = 4096;

template <bool LDS>
__global__ __launch_bounds__(kNT) void pages_assign_kernel(PagesParams p, int map) {
  __shared__ int sFirst[LDS ? kLdsSeqs + 1 : 1], sCu[LDS ? kLdsSeqs + 1 : 1], sSlot[LDS ? kLdsSeqs : 1];
  __shared__ long long sWave[kNT / 64];
  const int tid = threadIdx.x;
  const int count = on_stack(p);
  int* first = LDS ? sFirst : p.first;
  int* cu = LDS ? sCu : p.cu;
  // tokens and entries of the sequences before, in one sum: no more than 2^31 tokens and 2^31 entries
  long long tokens = 0, entries = 0;
  for (int n0 = 0; n0 < p.N; n0 += kNT) {
    const int n = n0 + tid;
    const int held = n < p.N ? p.lengths[n] : -1, more = n < p.N ? p.new_tokens[n] : 0;
    long long m = held >= 0 && more > 0 ? (more < p.T ? more : p.T) : 0, total;
    const long long end = tokens + block_scan<kNT>(m, sWave, total);
    // tokens past T have no place
    const long long a = end - m < p.T ? end - m : p.T, b = end < p.T ? end : p.T;
    m = b - a;
    tokens += total;
    long long slots = 0;
    if (m > 0) {
      const long long i0 = held / p.page, i1 = (held + m - 1) / p.page + 1;
      slots = (i1 < p.table_w ? i1 : p.table_w) - i0;
      slots = slots > 0 ? slots : 0;
    }
    const long long upto = entries + block_scan<kNT>(slots, sWave, total);
    entries += total;
    if (n < p.N) {
      first[n] = (int)(upto - slots);
      cu[n] = (int)a;
      if (LDS) {
        p.cu[n] = (int)a;
        sSlot[n] = held / p.page;
      }
    }
  }
  const int used = (int)(tokens < p.T ? tokens : p.T), all = (int)entries;
  if (tid == 0) {
    first[p.N] = all;
    cu[p.N] = p.cu[p.N] = used;
  }
  __syncthreads();
  int needed = 0;
  for (int f0 = 0; f0 < all; f0 += 16 * kNT) {
    int* at[16];
    int id[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // all reads before the sum
      const int f = f0 + 4 * (j * kNT + tid);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        id[4 * j + i] = 0;
        at[4 * j + i] = nullptr;
      }
      if (f0 + 4 * j * kNT >= all) continue;  // uniform
      int n = f < all ? last_upto(first, p.N, f) : 0, upto = f < all ? first[n + 1] : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (f + i >= all) continue;
        while (f + i >= upto) upto = first[++n + 1];  // (entries of a sequence that follows)
        const int slot = LDS ? sSlot[n] : p.lengths[n] / p.page;
        at[4 * j + i] = p.table + (long long)n * p.table_w + slot + (f + i - first[n]);
        id[4 * j + i] = *at[4 * j + i];
      }
    }
    unsigned long long mine = 0, total;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (at[e] && !a_page(id[e], p.n_pages)) mine += 1ull << 16 * (e / 4);
    const unsigned long long upto = block_scan<kNT>(mine, (unsigned long long*)sWave, total) - mine;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (f0 + 4 * j * kNT >= all) continue;
      int k = needed + field(upto, j);
#pragma unroll
      for (int e = 4 * j; e < 4 * j + 4; ++e) {
        if (!at[e] || a_page(id[e], p.n_pages)) continue;
        if (k < count) *at[e] = p.free[count - 1 - k];
        ++k;
      }
      needed += field(total, j);
    }
  }
  if (tid == 0) {
    *p.count = needed < count ? count - needed : 0;
    *p.missing = needed < count ? 0 : needed - count;
  }
  if (!map) return;
  __syncthreads();
  for (int t = tid; t < p.T; t += kNT) map_token(p, cu, used, t);
}

__global__ __launch_bounds__(256) void pages_map_kernel(PagesParams p) {
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  if (t < p.T) map_token(p, p.cu, p.cu[p.N], (int)t);
}

// Whether entry i of a row that keeps `keep` tokens goes back: past those, or with a window behind what the
// next token sees, but for the sinks'.  (A table's positions fit 31 bits.)
__device__ __forceinline__ bool goes_back(const PagesParams& p, int id, int keep, int i) {
  const int from = i * p.page;
  const bool past = from >= keep, behind = (p.window > 0) & (from >= p.sinks) & (from + p.page - 1 <= keep - p.window);
  return a_page(id, p.n_pages) & (keep >= 0) & (past | behind);
}

// Entries of the tables, flat, kPer a workgroup of kBackNT threads, four neighbours a thread and turn.
constexpr int kBackNT = 256, kPer = 4096;

// which of four neighbours go back
__device__ __forceinline__ int back_of(const PagesParams& p, long long f, int (&id)[4]) {
  const long long all = (long long)p.N * p.table_w;
  int n = f < all ? (int)(f / p.table_w) : 0, slot[4], kept[4], mask = 0;
  slot[0] = (int)(f - (long long)n * p.table_w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // reads first
    id[i] = f + i < all ? p.table[f + i] : -1;
    kept[i] = f + i < all ? p.lengths[n] : -1;
    if (i == 3) break;
    slot[i + 1] = slot[i] + 1;
    if (slot[i + 1] == p.table_w) slot[i + 1] = 0, ++n;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (goes_back(p, id[i], kept[i], slot[i])) mask |= 1 << i;
  return mask;
}
__device__ __forceinline__ void give_back(const PagesParams& p, long long f, const int (&id)[4], int mask, long long top) {
  // the first of them goes to free[top], the next below it
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!((mask >> i) & 1)) continue;
    if (top < p.n_pages) p.free[top] = id[i];
    p.table[f + i] = -1;
    --top;
  }
}

// few entries, kOneRelease at most, of kLdsRows rows: one workgroup, which keeps them all in registers.  Its
// instructions bound it, so what a row returns lies in LDS as slots: those from sFrom on, and with a window
// those from its sinks' on before sBehind.
constexpr int kLdsRows = 8192;
constexpr int kTurns = 8;  // of four entries a thread
constexpr long long kOneRelease = 4 * kTurns * kNT;

template <bool WIN>
__global__ __launch_bounds__(kNT) void pages_release_one_kernel(PagesParams p) {
  typedef int i32x4u __attribute__((ext_vector_type(4), aligned(4)));
  __shared__ unsigned long long sWave[kNT / 64];
  __shared__ int sFrom[kLdsRows], sBehind[WIN ? kLdsRows : 1];
  const int all = p.N * p.table_w, sinks = (int)(((unsigned)p.sinks + p.page - 1) / p.page);
  const int count = on_stack(p);
  for (int n = threadIdx.x; n < p.N; n += kNT) {
    const int keep = p.lengths[n];
    sFrom[n] = keep < 0 ? INT_MAX : keep / p.page + (keep % p.page != 0);
    if (WIN) sBehind[n] = keep < p.window ? 0 : (keep - p.window + 1) / p.page;
  }
  int id[kTurns][4], mask[kTurns];
#pragma unroll
  for (int j = 0; j < kTurns; ++j) {
    const int f = 4 * (j * kNT + (int)threadIdx.x);
    if (f + 3 < all) {
      const i32x4u x = *(const i32x4u*)(p.table + f);
#pragma unroll
      for (int i = 0; i < 4; ++i) id[j][i] = x[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) id[j][i] = f + i < all ? p.table[f + i] : -1;
    }
  }
  __syncthreads();
  // the first entry's row and slot, from turn to turn
  const int down = 4 * kNT / p.table_w, on = 4 * kNT % p.table_w;
  int n0 = 4 * (int)threadIdx.x / p.table_w, slot0 = 4 * (int)threadIdx.x % p.table_w;
  unsigned long long mine[2] = {0, 0}, upto[2], total[2];
#pragma unroll
  for (int j = 0; j < kTurns; ++j) {
    mask[j] = 0;
    if (4 * j * kNT >= all) continue;  // uniform
    int n = n0, slot = slot0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = n < p.N ? n : p.N - 1;
      const bool behind = WIN ? (slot >= sinks) & (slot < sBehind[m]) : false;
      if (a_page(id[j][i], p.n_pages) & ((slot >= sFrom[m]) | behind)) mask[j] |= 1 << i;
      if (++slot == p.table_w) slot = 0, ++n;
    }
    mine[j / 4] += (unsigned long long)__popc(mask[j]) << 16 * (j % 4);
    n0 += down;
    slot0 += on;
    if (slot0 >= p.table_w) slot0 -= p.table_w, ++n0;
  }
  int n = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    upto[h] = block_scan<kNT>(mine[h], sWave, total[h]) - mine[h];
#pragma unroll
    for (int j = 0; j < 4; ++j) n += field(total[h], j);
  }
  int done = 0;
#pragma unroll
  for (int j = 0; j < kTurns; ++j) {
    if (4 * j * kNT >= all) continue;
    give_back(p, 4 * (j * kNT + (int)threadIdx.x), id[j], mask[j], (long long)count + n - 1 - done - field(upto[j / 4], j % 4));
    done += field(total[j / 4], j % 4);
  }
  if (threadIdx.x == 0) *p.count = count + n < p.n_pages ? count + n : p.n_pages;
}

// many: a count for each kPer entries, and the stack's count as it was
__global__ __launch_bounds__(kBackNT) void pages_count_kernel(PagesParams p) {
  __shared__ int sWave[kBackNT / 64];
  int id[4], mine = 0, total;
#pragma unroll
  for (int j = 0; j < kPer / (4 * kBackNT); ++j)
    mine += __popc(back_of(p, (long long)blockIdx.x * kPer + 4 * (j * kBackNT + (int)threadIdx.x), id));
  block_scan<kBackNT>(mine, sWave, total);
  if (threadIdx.x != 0) return;
  p.first[1 + blockIdx.x] = total;
  if (blockIdx.x == 0) p.first[0] = on_stack(p);
}

__global__ __launch_bounds__(kBackNT) void pages_release_kernel(PagesParams p) {
  __shared__ int sWave[kBackNT / 64];
  __shared__ long long sSum[kBackNT / 64];
  long long before = 0, n = 0, total;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kBackNT) {
    const int x = p.first[1 + i];
    n += x;
    if (i < (int)blockIdx.x) before += x;
  }
  block_scan<kBackNT>(before, sSum, total);
  before = total;
  block_scan<kBackNT>(n, sSum, total);
  n = total;
  const int count = p.first[0];
  for (int j = 0; j < kPer / (4 * kBackNT); ++j) {
    const long long f = (long long)blockIdx.x * kPer + 4 * (j * kBackNT + (int)threadIdx.x);
    int id[4], here;
    const int mask = back_of(p, f, id), k = __popc(mask);
    const int upto = block_scan<kBackNT>(k, sWave, here);
    give_back(p, f, id, mask, count + n - 1 - (before + upto - k));
    before += here;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.count = (int)(count + n < p.n_pages ? count + n : p.n_pages);
}

constexpr long long kOneMap = 4096;         // tokens that the assigning workgroup maps

}  // namespace

size_t pages_assign_words(long long N) { return N > kLdsSeqs ? (size_t)N + 1 : 0; }

hipError_t launch_pages_assign(const PagesParams& p, hipStream_t stream) {
  const int map = p.T <= kOneMap;
  if (p.N <= kLdsSeqs)
    pages_assign_kernel<true><<<1, kNT, 0, stream>>>(p, map);
  else
    pages_assign_kernel<false><<<1, kNT, 0, stream>>>(p, map);
  if (!map) pages_map_kernel<<<(unsigned)((p.T + 255) / 256), 256, 0, stream>>>(p);
  return hipGetLastError();
}

size_t pages_release_words(long long N, long long table_w) {
  return N * table_w > kOneRelease || N > kLdsRows ? (size_t)((N * table_w + kPer - 1) / kPer + 1) : 0;
}

hipError_t launch_pages_release(const PagesParams& p, hipStream_t stream) {
  const long long entries = (long long)p.N * p.table_w;
  if (pages_release_words(p.N, p.table_w) == 0) {
    if (p.window > 0)
      pages_release_one_kernel<true><<<1, kNT, 0, stream>>>(p);
    else
      pages_release_one_kernel<false><<<1, kNT, 0, stream>>>(p);
  } else {
    const unsigned grid = (unsigned)((entries + kPer - 1) / kPer);
    pages_count_kernel<<<grid, kBackNT, 0, stream>>>(p);
    pages_release_kernel<<<grid, kBackNT, 0, stream>>>(p);
  }
  return hipGetLastError();
}

}  // namespace omx
