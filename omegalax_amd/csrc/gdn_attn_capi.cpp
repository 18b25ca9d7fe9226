// C ABI of the softmax attention operators: argument validation, workspaces and launch, as in
// gdn_capi.cpp, whose error reporting this file shares.
#include "omx_gdn.h"

#include <hip/hip_runtime.h>

#include <climits>

#include "gdn_capi.h"
#include "gdn_kernels.h"

namespace {

using omx::aligned;
using omx::fail;
using omx::launch_status;
using omx::ok;

constexpr int64_t kMaxTokens = ((int64_t)1 << 31) - 4096;  // token and tile indexes are 32 bits

struct Shape {
  int64_t N, B, T, Hq, Hkv, D;
  bool packed;
};

int check_shape(const char* fn, const Shape& s) {
  REQUIRE(s.Hkv >= 1 && s.Hq >= 1, "%s: head counts must be positive (Hq=%lld, Hkv=%lld)", fn,
          (long long)s.Hq, (long long)s.Hkv);
  REQUIRE(s.Hq % s.Hkv == 0, "%s: query heads (%lld) must be a multiple of key heads (%lld)", fn,
          (long long)s.Hq, (long long)s.Hkv);
  REQUIRE(s.Hq <= 4096, "%s: too many query heads (%lld)", fn, (long long)s.Hq);
  REQUIRE(s.D >= 1 && s.D % 8 == 0, "%s: head dim %lld must be a positive multiple of 8", fn, (long long)s.D);
  if (s.D > omx::kAttnMaxD)
    return fail(OMX_GDN_EUNSUPPORTED, "%s: head dim %lld above %d", fn, (long long)s.D, omx::kAttnMaxD);
  if (s.Hq / s.Hkv > omx::kAttnMaxG)
    return fail(OMX_GDN_EUNSUPPORTED, "%s: %lld query heads per key head, above %d", fn,
                (long long)(s.Hq / s.Hkv), omx::kAttnMaxG);
  REQUIRE(s.B >= 0 && s.T >= 0, "%s: negative shape (B=%lld, T=%lld)", fn, (long long)s.B, (long long)s.T);
  REQUIRE(s.B <= kMaxTokens && s.T <= kMaxTokens && s.B * s.T <= kMaxTokens, "%s: too many tokens (B=%lld, T=%lld)", fn,
          (long long)s.B, (long long)s.T);
  if (s.packed) {
    REQUIRE(s.B == 1, "%s: cu_seqlens requires batch 1 (got %lld)", fn, (long long)s.B);
    REQUIRE(s.N >= 1 && s.N <= (1 << 20), "%s: sequence count %lld out of range", fn, (long long)s.N);
  } else {
    REQUIRE(s.N == s.B, "%s: without cu_seqlens N must equal B (%lld vs %lld)", fn, (long long)s.N, (long long)s.B);
  }
  return OMX_GDN_OK;
}

// a token stride: whole 16-byte segments, at least the heads it holds, within 32-bit tile offsets
int check_ld(const char* fn, const char* name, int64_t ld, int64_t least) {
  REQUIRE(ld >= least && ld % 8 == 0 && ld <= (1 << 22),
          "%s: %s must be a multiple of 8 in [%lld, %d] (got %lld)", fn, name, (long long)least, 1 << 22, (long long)ld);
  return OMX_GDN_OK;
}

int check_scale(const char* fn, float scale) {
  REQUIRE(scale > 0.f && scale <= 1048576.f, "%s: scale must be positive and at most 2^20", fn);
  return OMX_GDN_OK;
}

int check_cache(const char* fn, const void* kp, const void* vp, int64_t n_pages, int64_t page,
                const int32_t* table, int64_t table_w, const int32_t* held, int64_t D, int64_t Hkv) {
  if (!omx::paged_dims_supported((int)D))
    return fail(OMX_GDN_EUNSUPPORTED, "%s: head dim %lld of a paged cache not compiled (64/128/256)", fn, (long long)D);
  REQUIRE(page >= 16 && page % 16 == 0 && page <= 65536, "%s: page size %lld must be a multiple of 16 in [16, 65536]",
          fn, (long long)page);
  REQUIRE(n_pages >= 0 && n_pages <= INT_MAX, "%s: page count %lld out of range", fn, (long long)n_pages);
  REQUIRE(table_w >= 0 && table_w <= kMaxTokens && table_w * page <= kMaxTokens,
          "%s: block table of %lld pages of %lld tokens out of range", fn, (long long)table_w, (long long)page);
  REQUIRE(Hkv * D <= (1 << 22), "%s: %lld key heads of dim %lld out of range", fn, (long long)Hkv, (long long)D);
  REQUIRE(held && (table || table_w == 0) && ((kp && vp) || n_pages == 0), "%s: a required pointer is NULL", fn);
  REQUIRE(aligned(kp, 16) && aligned(vp, 16), "%s: k_pages and v_pages must be 16-byte aligned", fn);
  return OMX_GDN_OK;
}

// What a workspace size is told for: shapes and tables that an entry point may take.  Others have none.
bool sized(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N) {
  return B >= 0 && B <= kMaxTokens && T >= 0 && T <= kMaxTokens && B * T <= kMaxTokens && N >= 0 && N <= kMaxTokens &&
         Hkv >= 1 && Hq >= 1 && Hq <= 4096 && Hq % Hkv == 0 && Hq / Hkv <= omx::kAttnMaxG && D >= 1 && D <= omx::kAttnMaxD;
}
bool sized_table(int64_t page, int64_t table_w) {
  return page >= 1 && page <= 65536 && table_w >= 0 && table_w <= kMaxTokens && page * table_w <= kMaxTokens;
}

size_t align_up(size_t x) { return (x + 255) / 256 * 256; }

// The plan of more than 64 packed sequences for tiles of `per` tokens: tile list, offsets.
struct PlanWs {
  size_t list, cu, total;
};
PlanWs plan_ws(size_t at, int64_t T, int64_t N, int per) {
  PlanWs w{at, at, at};
  const size_t words = omx::attn_plan_words(T, N, per);
  if (words == 0) return w;
  w.cu = w.list + align_up(words * 4);
  w.total = w.cu + align_up((size_t)(N + 1) * 4);
  return w;
}
// points the kernels at a plan and makes it
hipError_t use_plan(omx::AttnParams& p, const PlanWs& w, void* workspace, int per, hipStream_t stream) {
  p.plan = p.cu_plan = nullptr;
  if (!p.cu || w.total == w.list) return hipSuccess;
  p.plan = (int32_t*)((char*)workspace + w.list);
  p.cu_plan = (int32_t*)((char*)workspace + w.cu);
  return omx::launch_attn_plan(p, per, stream);
}

// Splits of the keys of a paged prefill: few rows leave compute units idle.  Each row of a batch has
// its own tiles; packed sequences add at most one tile each to those of all their tokens.  Two
// workgroups a compute unit, shares of 128 keys at least, 32 at most: with up to 64, 16 new tokens on
// 100,000 of 8/2 heads of 128 take 67 us (85), on 6,000 19 (17); 8/1 heads of 256 on 20,000 56 (43).
int paged_splits(const Shape& x, int64_t capacity) {  // capacity: keys that a tile sees at most
  const int64_t per = omx::attn_tile_tokens((int)(x.Hq / x.Hkv)), each = (x.T + per - 1) / per;
  const int64_t tiles = (x.packed ? each + x.N - 1 : x.N * each) * x.Hkv;
  int64_t s = tiles > 0 ? 2 * omx::kComputeUnits / tiles : 1;
  const int64_t most = capacity / 128;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > omx::kAttnMaxSplits ? omx::kAttnMaxSplits : s));
}

struct SplitWs {
  size_t o, ml, total;
};
SplitWs split_ws(size_t at, int splits, int64_t rows, int64_t D) {
  SplitWs w{at, at, at};
  if (splits <= 1) return w;
  w.ml = at + align_up((size_t)splits * rows * D * 4);
  w.total = w.ml + align_up((size_t)splits * rows * 8);
  return w;
}

omx::AttnParams params(const Shape& s, float scale) {
  omx::AttnParams p{};
  p.N = (int)s.N; p.T = (int)s.T; p.Hkv = (int)s.Hkv; p.G = (int)(s.Hq / s.Hkv); p.D = (int)s.D;
  p.tokens = s.B * s.T;
  p.scale = scale;
  p.splits = 1;
  return p;
}

// A launch has less than 2^32 threads, 256 a workgroup.
constexpr int64_t kMaxGroups = (1 << 24) - 1;

// workgroups of a kernel over tiles of `per` tokens, in the worst case of every packing (of up to three
// key heads, the grid is filled up to a multiple of 8)
int check_grid(const char* fn, const Shape& s, int64_t per) {
  int64_t ranks = (s.T + per - 1) / per + (s.packed ? s.N : 0);
  ranks = ranks < s.T ? ranks : s.T;  // each tile has a token
  REQUIRE((s.packed ? 1 : s.N) * ranks * s.Hkv + 8 <= kMaxGroups, "%s: grid too large", fn);
  return OMX_GDN_OK;
}

// What a row sees: its last `window` keys, all of them for 0, and the first `sinks`.
struct Sight {
  int64_t window, sinks;
};
constexpr Sight kAllKeys{0, 0};

int check_sight(const char* fn, const Sight& x) {
  REQUIRE(x.window >= 1, "%s: window %lld must be at least 1", fn, (long long)x.window);
  REQUIRE(x.sinks >= 0, "%s: sinks %lld must not be negative", fn, (long long)x.sinks);
  return OMX_GDN_OK;
}
// that of sequences of at most `keys`: kernels for a window only where it leaves out a key
void look_at(omx::AttnParams& p, const Sight& x, int64_t keys) {
  if (x.window == 0 || x.window >= keys || x.sinks >= keys - x.window) return;
  p.window = (int)x.window;
  p.sinks = (int)x.sinks;
}
// keys of at most `keys` that `rows` queries in a row see together, in whole tiles of 64
int64_t seen_keys(const Sight& x, int64_t keys, int64_t rows) {
  if (x.window == 0 || x.window >= keys || x.sinks >= keys - x.window) return keys;
  const int64_t n = x.window + x.sinks + rows + 128;
  return n < keys ? n : keys;
}
// a key's page by a product, for keys of 31 bits: with 2^(l-1) < page <= 2^l the multiplier, rounded up, is off by
// less than 2^l in 2^(31+l), too little to carry a quotient's fraction over
void divide_by_page(omx::AttnParams& p, int64_t page) {
  int l = 0;
  while (((int64_t)1 << l) < page) ++l;
  p.page_mul = (unsigned)((((uint64_t)1 << (31 + l)) + page - 1) / page);
  p.page_shift = (unsigned)(l - 1);
}
// the exponents of a cache in 8 bits: both or neither
int check_exps(const char* fn, const int8_t* k_exps, const int8_t* v_exps) {
  REQUIRE(!k_exps == !v_exps, "%s: k_exps and v_exps go together", fn);
  return OMX_GDN_OK;
}
int check_any_sight(const char* fn, const Sight& x) {
  REQUIRE(x.window >= 0, "%s: window %lld must not be negative (0: all keys)", fn, (long long)x.window);
  REQUIRE(x.sinks >= 0 && (x.window > 0 || x.sinks == 0), "%s: sinks %lld must not be negative, and need a window", fn,
          (long long)x.sinks);
  return OMX_GDN_OK;
}

}  // namespace

extern "C" {

size_t omx_gdn_attn_fwd_workspace_size(int64_t T, int64_t Hq, int64_t Hkv, int64_t N) {
  if (!sized(1, T, Hq, Hkv, 1, N)) return 0;
  return plan_ws(0, T, N, omx::attn_tile_tokens((int)(Hq / Hkv))).total;
}

namespace {
int attn_fwd(const char* fn, const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
             const int32_t* cu_seqlens, int64_t N, void* o, float* lse, void* o_rest, int64_t B, int64_t T, int64_t Hq,
             int64_t Hkv, int64_t D, float scale, const Sight& sight, void* workspace, size_t workspace_bytes,
             void* stream) {
  const Shape s{N, B, T, Hq, Hkv, D, cu_seqlens != nullptr};
  int rc = check_shape(fn, s);
  if (!rc) rc = check_ld(fn, "q_ld", q_ld, Hq * D);
  if (!rc) rc = check_ld(fn, "k_ld", k_ld, Hkv * D);
  if (!rc) rc = check_ld(fn, "v_ld", v_ld, Hkv * D);
  if (!rc) rc = check_scale(fn, scale);
  const int per = rc ? 1 : omx::attn_tile_tokens((int)(Hq / Hkv));
  if (!rc) rc = check_grid(fn, s, per);
  if (rc) return rc;
  const PlanWs ws = plan_ws(0, T, s.packed ? N : 0, per);
  REQUIRE(workspace_bytes >= ws.total, "%s: workspace of %zu bytes is smaller than the %zu needed", fn,
          workspace_bytes, ws.total);
  if (B * T == 0) return ok();
  REQUIRE(q && k && v && o, "%s: a required pointer is NULL", fn);
  REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(o, 16) && aligned(o_rest, 16),
          "%s: q, k, v, o, o_rest must be 16-byte aligned", fn);
  REQUIRE(ws.total == 0 || (workspace && aligned(workspace, 16)), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  omx::AttnParams p = params(s, scale);
  p.q = q; p.k = k; p.v = v; p.o = o; p.o_rest = o_rest; p.lse = lse;
  p.q_ld = q_ld; p.k_ld = k_ld; p.v_ld = v_ld; p.cu = cu_seqlens;
  look_at(p, sight, T);
  hipError_t e = use_plan(p, ws, workspace, per, (hipStream_t)stream);
  if (e == hipSuccess) e = omx::launch_attn_fwd(p, (hipStream_t)stream);
  return launch_status(e, fn);
}
}  // namespace

int omx_gdn_attn_fwd(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                     const int32_t* cu_seqlens, int64_t N, void* o, float* lse, void* o_rest, int64_t B, int64_t T,
                     int64_t Hq, int64_t Hkv, int64_t D, float scale, void* workspace, size_t workspace_bytes,
                     void* stream) {
  return attn_fwd("omx_gdn_attn_fwd", q, k, v, q_ld, k_ld, v_ld, cu_seqlens, N, o, lse, o_rest, B, T, Hq, Hkv, D, scale,
                  kAllKeys, workspace, workspace_bytes, stream);
}

int omx_gdn_attn_window_fwd(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                            const int32_t* cu_seqlens, int64_t N, void* o, float* lse, void* o_rest, int64_t B,
                            int64_t T, int64_t Hq, int64_t Hkv, int64_t D, float scale, int64_t window, int64_t sinks,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const Sight sight{window, sinks};
  const int rc = check_sight("omx_gdn_attn_window_fwd", sight);
  if (rc) return rc;
  return attn_fwd("omx_gdn_attn_window_fwd", q, k, v, q_ld, k_ld, v_ld, cu_seqlens, N, o, lse, o_rest, B, T, Hq, Hkv, D,
                  scale, sight, workspace, workspace_bytes, stream);
}

namespace {
// the rows' lse and delta, the plans of the two kernels' tiles, dk and dv in shares
struct AttnBwdWs {
  size_t stats;
  PlanWs rows, keys;
  omx::DkvPlan share;
  size_t shares, part_k, part_v, sink_k, sink_v, total;
  omx::AttnParams sight;  // its window and sinks
};
AttnBwdWs attn_bwd_ws(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N, const Sight& sight) {
  AttnBwdWs w{};
  const int per = omx::attn_dkv_tile_tokens();
  w.rows = plan_ws(align_up((size_t)(B * T * Hq) * 8), T, N, omx::attn_tile_tokens((int)(Hq / Hkv)));
  w.keys = plan_ws(w.rows.total, T, N, per);
  look_at(w.sight, sight, T);
  const int window = w.sight.window, sinks = w.sight.sinks;
  w.share = window > 0 ? omx::attn_dkv_window_plan(B, T, N, (int)Hkv, (int)(Hq / Hkv), (int)D, window, sinks)
                       : omx::attn_dkv_plan(B * Hkv, T, N, (int)(Hq / Hkv), B * T * Hkv * D * 8);
  w.shares = w.part_k = w.part_v = w.total = w.keys.total;
  if (w.share.splits > 1) {
    const size_t one = align_up((size_t)w.share.splits * B * T * Hkv * D * 4);
    w.part_k = w.shares + align_up((size_t)(B * T * Hkv) * 4);
    w.part_v = w.part_k + one;
    w.total = w.part_v + one;
  }
  w.sink_k = w.sink_v = w.total;
  if (w.share.sink_splits > 1) {
    const size_t one = align_up((size_t)w.share.sink_splits * (N > 0 ? N : B) * omx::attn_sink_keys(sinks) * Hkv * D * 4);
    w.sink_v = w.sink_k + one;
    w.total = w.sink_v + one;
  }
  return w;
}

int attn_bwd(const char* fn, const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
             const int32_t* cu_seqlens, int64_t N, const void* o, const float* lse, const void* o_rest, const void* d_o,
             void* dq, void* dk, void* dv, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, float scale,
             const Sight& sight, void* workspace, size_t workspace_bytes, void* stream) {
  const Shape s{N, B, T, Hq, Hkv, D, cu_seqlens != nullptr};
  int rc = check_shape(fn, s);
  if (!rc) rc = check_ld(fn, "q_ld", q_ld, Hq * D);
  if (!rc) rc = check_ld(fn, "k_ld", k_ld, Hkv * D);
  if (!rc) rc = check_ld(fn, "v_ld", v_ld, Hkv * D);
  if (!rc) rc = check_scale(fn, scale);
  const int per = rc ? 1 : omx::attn_tile_tokens((int)(Hq / Hkv));
  if (!rc) rc = check_grid(fn, s, per);
  if (rc) return rc;
  const AttnBwdWs ws = attn_bwd_ws(B, T, Hq, Hkv, D, s.packed ? N : 0, sight);
  REQUIRE(workspace_bytes >= ws.total, "%s: workspace of %zu bytes is smaller than the %zu needed", fn,
          workspace_bytes, ws.total);
  if (B * T == 0) return ok();
  REQUIRE(q && k && v && o && lse && d_o && dq && dk && dv, "%s: a required pointer is NULL", fn);
  REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(o, 16) && aligned(o_rest, 16) && aligned(d_o, 16) && aligned(dq, 16) &&
              aligned(dk, 16) && aligned(dv, 16),
          "%s: q, k, v, o, o_rest, d_o, dq, dk, dv must be 16-byte aligned", fn);
  REQUIRE(workspace && aligned(workspace, 16), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  omx::AttnParams p = params(s, scale);
  p.q = q; p.k = k; p.v = v; p.o = const_cast<void*>(o); p.lse = const_cast<float*>(lse); p.dout = d_o;
  p.o_rest = const_cast<void*>(o_rest);
  p.q_ld = q_ld; p.k_ld = k_ld; p.v_ld = v_ld; p.cu = cu_seqlens;
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.stats = (float*)((char*)workspace + ws.stats);
  p.shares = (int32_t*)((char*)workspace + ws.shares);
  p.part_k = (float*)((char*)workspace + ws.part_k);
  p.part_v = (float*)((char*)workspace + ws.part_v);
  p.splits = ws.share.splits;
  p.share_tiles = ws.share.tiles;
  p.window = ws.sight.window;
  p.sinks = ws.sight.sinks;
  p.sink_splits = ws.share.sink_splits;
  p.sink_k = (float*)((char*)workspace + ws.sink_k);
  p.sink_v = (float*)((char*)workspace + ws.sink_v);
  if (p.window > 0)
    REQUIRE(omx::attn_dkv_groups(p) <= kMaxGroups, "%s: grid too large", fn);
  const hipStream_t st = (hipStream_t)stream;
  hipError_t e = use_plan(p, ws.rows, workspace, per, st);
  if (e == hipSuccess) e = omx::launch_attn_dq(p, st);
  if (e == hipSuccess) e = use_plan(p, ws.keys, workspace, omx::attn_dkv_tile_tokens(), st);
  if (e == hipSuccess) e = omx::launch_attn_dkv(p, st);
  return launch_status(e, fn);
}
}  // namespace

size_t omx_gdn_attn_bwd_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N) {
  if (!sized(B, T, Hq, Hkv, D, N)) return 0;
  return attn_bwd_ws(B, T, Hq, Hkv, D, N, kAllKeys).total;
}

size_t omx_gdn_attn_window_bwd_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N,
                                              int64_t window, int64_t sinks) {
  if (!sized(B, T, Hq, Hkv, D, N) || window < 1 || sinks < 0) return 0;
  return attn_bwd_ws(B, T, Hq, Hkv, D, N, Sight{window, sinks}).total;
}

int omx_gdn_attn_bwd(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                     const int32_t* cu_seqlens, int64_t N, const void* o, const float* lse, const void* o_rest, const void* d_o,
                     void* dq, void* dk, void* dv, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                     float scale, void* workspace, size_t workspace_bytes, void* stream) {
  return attn_bwd("omx_gdn_attn_bwd", q, k, v, q_ld, k_ld, v_ld, cu_seqlens, N, o, lse, o_rest, d_o, dq, dk, dv, B, T, Hq,
                  Hkv, D, scale, kAllKeys, workspace, workspace_bytes, stream);
}

int omx_gdn_attn_window_bwd(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                            const int32_t* cu_seqlens, int64_t N, const void* o, const float* lse, const void* o_rest,
                            const void* d_o, void* dq, void* dk, void* dv, int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                            int64_t D, float scale, int64_t window, int64_t sinks, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const Sight sight{window, sinks};
  const int rc = check_sight("omx_gdn_attn_window_bwd", sight);
  if (rc) return rc;
  return attn_bwd("omx_gdn_attn_window_bwd", q, k, v, q_ld, k_ld, v_ld, cu_seqlens, N, o, lse, o_rest, d_o, dq, dk, dv, B,
                  T, Hq, Hkv, D, scale, sight, workspace, workspace_bytes, stream);
}

size_t omx_gdn_kv_write_workspace_size(int64_t T, int64_t N) {
  if (!sized(1, T, 1, 1, 1, N)) return 0;
  return plan_ws(0, T, N, omx::attn_dkv_tile_tokens()).total;
}

namespace {
// (k_exps null: a cache of bf16)
int kv_write(const char* fn, const void* k, const void* v, int64_t k_ld, int64_t v_ld, const int32_t* cu_seqlens,
             int64_t N, void* k_pages, void* v_pages, int8_t* k_exps, int8_t* v_exps, int64_t n_pages,
             int64_t page_size, const int32_t* block_table, int64_t table_width, const int32_t* lengths, int64_t B,
             int64_t T, int64_t Hkv, int64_t D, void* workspace, size_t workspace_bytes, void* stream) {
  const Shape s{N, B, T, Hkv, Hkv, D, cu_seqlens != nullptr};
  int rc = check_shape(fn, s);
  if (!rc) rc = check_ld(fn, "k_ld", k_ld, Hkv * D);
  if (!rc) rc = check_ld(fn, "v_ld", v_ld, Hkv * D);
  if (rc) return rc;
  if (k_exps)
    REQUIRE((B * T / omx::kv_write8_tokens() + 1) * 2 * Hkv <= kMaxGroups, "%s: grid too large", fn);
  else
    REQUIRE(B * T <= kMaxGroups * omx::kv_write_tokens(), "%s: grid too large", fn);
  const int per = omx::attn_dkv_tile_tokens();
  const PlanWs ws = plan_ws(0, T, s.packed ? N : 0, per);
  REQUIRE(workspace_bytes >= ws.total, "%s: workspace of %zu bytes is smaller than the %zu needed", fn,
          workspace_bytes, ws.total);
  if (B * T == 0) return ok();
  rc = check_cache(fn, k_pages, v_pages, n_pages, page_size, block_table, table_width, lengths, D, Hkv);
  if (rc) return rc;
  REQUIRE(k && v, "%s: a required pointer is NULL", fn);
  REQUIRE(aligned(k, 16) && aligned(v, 16), "%s: k and v must be 16-byte aligned", fn);
  REQUIRE(ws.total == 0 || (workspace && aligned(workspace, 16)), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  omx::AttnParams p = params(s, 1.f);
  p.k = k; p.v = v; p.k_ld = k_ld; p.v_ld = v_ld; p.cu = cu_seqlens;
  p.k_pages = k_pages; p.v_pages = v_pages; p.k_exps = k_exps; p.v_exps = v_exps; p.table = block_table; p.held = lengths;
  p.table_w = (int)table_width; p.page = (int)page_size; p.n_pages = (int)n_pages;
  hipError_t e = use_plan(p, ws, workspace, per, (hipStream_t)stream);
  if (e == hipSuccess) e = k_exps ? omx::launch_kv_write8(p, (hipStream_t)stream) : omx::launch_kv_write(p, (hipStream_t)stream);
  return launch_status(e, fn);
}
}  // namespace

int omx_gdn_kv_write(const void* k, const void* v, int64_t k_ld, int64_t v_ld, const int32_t* cu_seqlens, int64_t N,
                     void* k_pages, void* v_pages, int64_t n_pages, int64_t page_size, const int32_t* block_table,
                     int64_t table_width, const int32_t* lengths, int64_t B, int64_t T, int64_t Hkv, int64_t D,
                     void* workspace, size_t workspace_bytes, void* stream) {
  return kv_write("omx_gdn_kv_write", k, v, k_ld, v_ld, cu_seqlens, N, k_pages, v_pages, nullptr, nullptr, n_pages,
                  page_size, block_table, table_width, lengths, B, T, Hkv, D, workspace, workspace_bytes, stream);
}

int omx_gdn_kv_write8(const void* k, const void* v, int64_t k_ld, int64_t v_ld, const int32_t* cu_seqlens, int64_t N,
                      void* k_pages, void* v_pages, int8_t* k_exps, int8_t* v_exps, int64_t n_pages,
                      int64_t page_size, const int32_t* block_table, int64_t table_width, const int32_t* lengths,
                      int64_t B, int64_t T, int64_t Hkv, int64_t D, void* workspace, size_t workspace_bytes,
                      void* stream) {
  REQUIRE(k_exps && v_exps, "%s: a required pointer is NULL", "omx_gdn_kv_write8");
  return kv_write("omx_gdn_kv_write8", k, v, k_ld, v_ld, cu_seqlens, N, k_pages, v_pages, k_exps, v_exps, n_pages,
                  page_size, block_table, table_width, lengths, B, T, Hkv, D, workspace, workspace_bytes, stream);
}


namespace {
struct PagedWs {
  PlanWs plan;
  SplitWs split;
  int splits;
  size_t total;
};
PagedWs paged_ws(const Shape& s, int64_t capacity, const Sight& sight) {
  PagedWs w{};
  w.plan = plan_ws(0, s.T, s.packed ? s.N : 0, omx::attn_tile_tokens((int)(s.Hq / s.Hkv)));
  w.splits = paged_splits(s, seen_keys(sight, capacity, omx::attn_tile_tokens((int)(s.Hq / s.Hkv))));
  w.split = split_ws(w.plan.total, w.splits, s.B * s.T * s.Hq, s.D);
  w.total = w.split.total;
  return w;
}
}  // namespace

size_t omx_gdn_attn_paged_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N,
                                         int packed, int64_t page_size, int64_t table_width) {
  const Shape s{N, B, T, Hq, Hkv, D, packed != 0};
  if (!sized(B, T, Hq, Hkv, D, N) || !sized_table(page_size, table_width)) return 0;
  return paged_ws(s, page_size * table_width, kAllKeys).total;
}

namespace {
int attn_paged(const char* fn, const void* q, int64_t q_ld, const int32_t* cu_seqlens, int64_t N, const void* k_pages,
               const void* v_pages, const int8_t* k_exps, const int8_t* v_exps, int64_t n_pages, int64_t page_size,
               const int32_t* block_table, int64_t table_width, const int32_t* lengths, void* o, int64_t B, int64_t T,
               int64_t Hq, int64_t Hkv, int64_t D, float scale, const Sight& sight, void* workspace,
               size_t workspace_bytes, void* stream) {
  const Shape s{N, B, T, Hq, Hkv, D, cu_seqlens != nullptr};
  int rc = check_shape(fn, s);
  if (!rc) rc = check_ld(fn, "q_ld", q_ld, Hq * D);
  if (!rc) rc = check_scale(fn, scale);
  const int per = rc ? 1 : omx::attn_tile_tokens((int)(Hq / Hkv));
  if (!rc) rc = check_grid(fn, s, per);
  if (rc) return rc;
  if (B * T == 0) return ok();
  rc = check_cache(fn, k_pages, v_pages, n_pages, page_size, block_table, table_width, lengths, D, Hkv);
  if (rc) return rc;
  REQUIRE(table_width * page_size + T <= kMaxTokens, "%s: too many tokens", fn);
  const PagedWs ws = paged_ws(s, page_size * table_width, sight);
  REQUIRE(workspace_bytes >= ws.total, "%s: workspace of %zu bytes is smaller than the %zu needed", fn,
          workspace_bytes, ws.total);
  REQUIRE(q && o, "%s: a required pointer is NULL", fn);
  REQUIRE(aligned(q, 16) && aligned(o, 16), "%s: q and o must be 16-byte aligned", fn);
  REQUIRE(ws.total == 0 || (workspace && aligned(workspace, 16)), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  omx::AttnParams p = params(s, scale);
  p.q = q; p.q_ld = q_ld; p.o = o; p.cu = cu_seqlens;
  p.k_pages = const_cast<void*>(k_pages); p.v_pages = const_cast<void*>(v_pages);
  p.k_exps = const_cast<int8_t*>(k_exps); p.v_exps = const_cast<int8_t*>(v_exps);
  look_at(p, sight, table_width * page_size + T);
  divide_by_page(p, page_size);
  p.table = block_table; p.held = lengths;
  p.table_w = (int)table_width; p.page = (int)page_size; p.n_pages = (int)n_pages;
  p.splits = ws.splits;
  p.part_o = (float*)((char*)workspace + ws.split.o);
  p.part_ml = (float*)((char*)workspace + ws.split.ml);
  hipError_t e = use_plan(p, ws.plan, workspace, per, (hipStream_t)stream);
  if (e == hipSuccess) e = omx::launch_attn_fwd(p, (hipStream_t)stream);
  return launch_status(e, fn);
}
}  // namespace

int omx_gdn_attn_paged(const void* q, int64_t q_ld, const int32_t* cu_seqlens, int64_t N, const void* k_pages,
                       const void* v_pages, int64_t n_pages, int64_t page_size, const int32_t* block_table,
                       int64_t table_width, const int32_t* lengths, void* o, int64_t B, int64_t T, int64_t Hq,
                       int64_t Hkv, int64_t D, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  return attn_paged("omx_gdn_attn_paged", q, q_ld, cu_seqlens, N, k_pages, v_pages, nullptr, nullptr, n_pages, page_size,
                    block_table, table_width, lengths, o, B, T, Hq, Hkv, D, scale, kAllKeys, workspace, workspace_bytes,
                    stream);
}

size_t omx_gdn_attn_paged_window_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N,
                                                int packed, int64_t page_size, int64_t table_width, int64_t window,
                                                int64_t sinks) {
  const Shape s{N, B, T, Hq, Hkv, D, packed != 0};
  if (!sized(B, T, Hq, Hkv, D, N) || !sized_table(page_size, table_width) || window < 0 || sinks < 0) return 0;
  return paged_ws(s, page_size * table_width, Sight{window, sinks}).total;
}

int omx_gdn_attn_paged_window(const void* q, int64_t q_ld, const int32_t* cu_seqlens, int64_t N, const void* k_pages,
                              const void* v_pages, const int8_t* k_exps, const int8_t* v_exps, int64_t n_pages,
                              int64_t page_size, const int32_t* block_table, int64_t table_width,
                              const int32_t* lengths, void* o, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                              float scale, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes,
                              void* stream) {
  const char* fn = "omx_gdn_attn_paged_window";
  const Sight sight{window, sinks};
  int rc = check_any_sight(fn, sight);
  if (!rc) rc = check_exps(fn, k_exps, v_exps);
  if (rc) return rc;
  return attn_paged(fn, q, q_ld, cu_seqlens, N, k_pages, v_pages, k_exps, v_exps, n_pages, page_size, block_table,
                    table_width, lengths, o, B, T, Hq, Hkv, D, scale, sight, workspace, workspace_bytes, stream);
}

namespace {
int decode_splits(const Sight& sight, int64_t B, int64_t Hkv, int64_t D, int64_t capacity, bool eight) {
  return omx::decode_splits(B, Hkv, D, capacity, seen_keys(sight, capacity, 1), eight);
}
SplitWs decode_ws(int splits, int64_t B, int64_t Hq, int64_t D) {
  // (one count of splits + B segments, of one row a head each)
  return splits > 1 ? split_ws(0, splits + (int)B, Hq, D) : split_ws(0, 1, 0, D);
}
}  // namespace

size_t omx_gdn_attn_decode_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page_size,
                                          int64_t table_width) {
  if (B < 1 || !sized(B, 1, Hq, Hkv, D, B) || !sized_table(page_size, table_width)) return 0;
  return decode_ws(decode_splits(kAllKeys, B, Hkv, D, page_size * table_width, false), B, Hq, D).total;
}

namespace {
int attn_decode(const char* fn, const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                void* k_pages, void* v_pages, int8_t* k_exps, int8_t* v_exps, int64_t n_pages, int64_t page_size,
                const int32_t* block_table, int64_t table_width, const int32_t* lengths, void* out, int64_t B,
                int64_t Hq, int64_t Hkv, int64_t D, float scale, const Sight& sight, void* workspace,
                size_t workspace_bytes, void* stream) {
  const Shape s{B, B, 1, Hq, Hkv, D, false};
  int rc = check_shape(fn, s);
  if (!rc) rc = check_ld(fn, "q_ld", q_ld, Hq * D);
  if (!rc) rc = check_ld(fn, "k_ld", k_ld, Hkv * D);
  if (!rc) rc = check_ld(fn, "v_ld", v_ld, Hkv * D);
  if (!rc) rc = check_scale(fn, scale);
  if (rc) return rc;
  REQUIRE(B <= 65535 * 16 && B * Hkv <= kMaxGroups && B * Hq <= INT_MAX / 4, "%s: batch %lld out of range", fn, (long long)B);
  if (B == 0) return ok();
  rc = check_cache(fn, k_pages, v_pages, n_pages, page_size, block_table, table_width, lengths, D, Hkv);
  if (rc) return rc;
  const int splits = decode_splits(sight, B, Hkv, D, page_size * table_width, k_exps != nullptr);
  const SplitWs ws = decode_ws(splits, B, Hq, D);
  REQUIRE(workspace_bytes >= ws.total, "%s: workspace of %zu bytes is smaller than the %zu needed", fn,
          workspace_bytes, ws.total);
  REQUIRE(q && k && v && out, "%s: a required pointer is NULL", fn);
  REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16), "%s: q, k, v, out must be 16-byte aligned", fn);
  REQUIRE(ws.total == 0 || (workspace && aligned(workspace, 16)), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  omx::AttnParams p = params(s, scale);
  p.q = q; p.k = k; p.v = v; p.o = out;
  p.q_ld = q_ld; p.k_ld = k_ld; p.v_ld = v_ld;
  p.k_exps = k_exps; p.v_exps = v_exps;
  look_at(p, sight, table_width * page_size + 1);
  divide_by_page(p, page_size);
  p.k_pages = k_pages; p.v_pages = v_pages; p.table = block_table; p.held = lengths;
  p.table_w = (int)table_width; p.page = (int)page_size; p.n_pages = (int)n_pages;
  p.splits = splits;
  p.part_o = (float*)((char*)workspace + ws.o);
  p.part_ml = (float*)((char*)workspace + ws.ml);
  return launch_status(k_exps ? omx::launch_attn_decode8(p, (hipStream_t)stream) : omx::launch_attn_decode(p, (hipStream_t)stream), fn);
}
}  // namespace

int omx_gdn_attn_decode_step(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                             void* k_pages, void* v_pages, int64_t n_pages, int64_t page_size,
                             const int32_t* block_table, int64_t table_width, const int32_t* lengths, void* out,
                             int64_t B, int64_t Hq, int64_t Hkv, int64_t D, float scale, void* workspace,
                             size_t workspace_bytes, void* stream) {
  return attn_decode("omx_gdn_attn_decode_step", q, k, v, q_ld, k_ld, v_ld, k_pages, v_pages, nullptr, nullptr, n_pages,
                     page_size, block_table, table_width, lengths, out, B, Hq, Hkv, D, scale, kAllKeys, workspace,
                     workspace_bytes, stream);
}

size_t omx_gdn_attn_decode_window_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page_size,
                                                 int64_t table_width, int64_t window, int64_t sinks) {
  if (B < 1 || !sized(B, 1, Hq, Hkv, D, B) || !sized_table(page_size, table_width) || window < 0 || sinks < 0) return 0;
  // (for either cache: one in 8 bits is shared later, never sooner)
  return decode_ws(decode_splits(Sight{window, sinks}, B, Hkv, D, page_size * table_width, false), B, Hq, D).total;
}

int omx_gdn_attn_decode_window(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                               void* k_pages, void* v_pages, int8_t* k_exps, int8_t* v_exps, int64_t n_pages,
                               int64_t page_size, const int32_t* block_table, int64_t table_width,
                               const int32_t* lengths, void* out, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                               float scale, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes,
                               void* stream) {
  const char* fn = "omx_gdn_attn_decode_window";
  const Sight sight{window, sinks};
  int rc = check_any_sight(fn, sight);
  if (!rc) rc = check_exps(fn, k_exps, v_exps);
  if (rc) return rc;
  return attn_decode(fn, q, k, v, q_ld, k_ld, v_ld, k_pages, v_pages, k_exps, v_exps, n_pages, page_size, block_table,
                     table_width, lengths, out, B, Hq, Hkv, D, scale, sight, workspace, workspace_bytes, stream);
}


namespace {
int check_pages(const char* fn, const int32_t* table, int64_t N, int64_t table_w, const int32_t* lengths,
                const int32_t* free_pages, const int32_t* free_count, int64_t n_pages, int64_t page) {
  REQUIRE(N >= 0 && N <= (1 << 20), "%s: sequence count %lld out of range", fn, (long long)N);
  REQUIRE(page >= 16 && page % 16 == 0 && page <= 65536, "%s: page size %lld must be a multiple of 16 in [16, 65536]",
          fn, (long long)page);
  REQUIRE(n_pages >= 0 && n_pages <= INT_MAX, "%s: page count %lld out of range", fn, (long long)n_pages);
  REQUIRE(table_w >= 0 && table_w <= kMaxTokens && table_w * page <= kMaxTokens,
          "%s: block table of %lld pages of %lld tokens out of range", fn, (long long)table_w, (long long)page);
  REQUIRE((lengths || N == 0) && (table || N * table_w == 0) && (free_pages || n_pages == 0) && free_count,
          "%s: a required pointer is NULL", fn);
  return OMX_GDN_OK;
}
omx::PagesParams pages(int32_t* table, int64_t N, int64_t table_w, const int32_t* lengths, int32_t* free_pages,
                       int32_t* free_count, int64_t n_pages, int64_t page, void* workspace) {
  omx::PagesParams p{};
  p.table = table; p.N = (int)N; p.table_w = (int)table_w; p.lengths = lengths; p.free = free_pages; p.count = free_count;
  p.n_pages = (int)n_pages; p.page = (int)page; p.first = (int32_t*)workspace;
  return p;
}
}  // namespace

size_t omx_gdn_pages_assign_workspace_size(int64_t N) {
  return N < 0 || N > (1 << 20) ? 0 : align_up(omx::pages_assign_words(N) * 4);
}

int omx_gdn_pages_assign(int32_t* block_table, int64_t N, int64_t table_width, const int32_t* lengths,
                         const int32_t* new_tokens, int32_t* free_pages, int32_t* free_count, int64_t n_pages,
                         int64_t page_size, int64_t T, int32_t* cu_seqlens, int32_t* positions, int64_t* slots,
                         int32_t* missing, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "omx_gdn_pages_assign";
  const int rc = check_pages(fn, block_table, N, table_width, lengths, free_pages, free_count, n_pages, page_size);
  if (rc) return rc;
  REQUIRE(T >= 0 && T <= kMaxTokens, "%s: too many tokens (%lld)", fn, (long long)T);
  // entries of new tokens are counted in 32 bits: those of T tokens, and two more for each sequence
  REQUIRE(T / page_size + 2 * N <= INT_MAX, "%s: too many tokens (%lld)", fn, (long long)T);
  const size_t need = omx_gdn_pages_assign_workspace_size(N);
  REQUIRE(workspace_bytes >= need, "%s: workspace of %zu bytes is smaller than the %zu needed", fn, workspace_bytes, need);
  REQUIRE(need == 0 || (workspace && aligned(workspace, 16)), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  REQUIRE((new_tokens || N == 0) && cu_seqlens && missing && ((positions && slots) || T == 0), "%s: a required pointer is NULL", fn);
  omx::PagesParams p = pages(block_table, N, table_width, lengths, free_pages, free_count, n_pages, page_size, workspace);
  p.new_tokens = new_tokens; p.T = T; p.cu = cu_seqlens; p.positions = positions; p.slots = (long long*)slots; p.missing = missing;
  return launch_status(omx::launch_pages_assign(p, (hipStream_t)stream), fn);
}

size_t omx_gdn_pages_release_workspace_size(int64_t N, int64_t table_width) {
  if (N < 0 || N > (1 << 20) || table_width < 0 || table_width > kMaxTokens) return 0;
  return align_up(omx::pages_release_words(N, table_width) * 4);
}

int omx_gdn_pages_release(int32_t* block_table, int64_t N, int64_t table_width, const int32_t* lengths,
                          int32_t* free_pages, int32_t* free_count, int64_t n_pages, int64_t page_size, int64_t window,
                          int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "omx_gdn_pages_release";
  int rc = check_pages(fn, block_table, N, table_width, lengths, free_pages, free_count, n_pages, page_size);
  if (!rc) rc = check_any_sight(fn, Sight{window, sinks});
  if (rc) return rc;
  REQUIRE(N * table_width <= kMaxGroups * 4096, "%s: grid too large", fn);
  const size_t need = omx_gdn_pages_release_workspace_size(N, table_width);
  REQUIRE(workspace_bytes >= need, "%s: workspace of %zu bytes is smaller than the %zu needed", fn, workspace_bytes, need);
  REQUIRE(need == 0 || (workspace && aligned(workspace, 16)), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  if (N * table_width == 0) return ok();
  omx::PagesParams p = pages(block_table, N, table_width, lengths, free_pages, free_count, n_pages, page_size, workspace);
  p.window = window < kMaxTokens ? (int)window : 0;  // no position is behind a window of all
  p.sinks = (int)(sinks < kMaxTokens ? sinks : kMaxTokens);
  return launch_status(omx::launch_pages_release(p, (hipStream_t)stream), fn);
}

}  // extern "C"
