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
int paged_splits(const Shape& x, int64_t capacity) {
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

}  // namespace

extern "C" {

size_t omx_gdn_attn_fwd_workspace_size(int64_t T, int64_t Hq, int64_t Hkv, int64_t N) {
  if (!sized(1, T, Hq, Hkv, 1, N)) return 0;
  return plan_ws(0, T, N, omx::attn_tile_tokens((int)(Hq / Hkv))).total;
}

int omx_gdn_attn_fwd(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                     const int32_t* cu_seqlens, int64_t N, void* o, float* lse, void* o_rest, int64_t B, int64_t T,
                     int64_t Hq, int64_t Hkv, int64_t D, float scale, void* workspace, size_t workspace_bytes,
                     void* stream) {
  const char* fn = "omx_gdn_attn_fwd";
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
  hipError_t e = use_plan(p, ws, workspace, per, (hipStream_t)stream);
  if (e == hipSuccess) e = omx::launch_attn_fwd(p, (hipStream_t)stream);
  return launch_status(e, fn);
}

namespace {
// the rows' lse and delta, the plans of the two kernels' tiles, dk and dv in shares
struct AttnBwdWs {
  size_t stats;
  PlanWs rows, keys;
  omx::DkvPlan share;
  size_t shares, part_k, part_v, total;
};
AttnBwdWs attn_bwd_ws(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N) {
  AttnBwdWs w{};
  const int per = omx::attn_dkv_tile_tokens();
  w.rows = plan_ws(align_up((size_t)(B * T * Hq) * 8), T, N, omx::attn_tile_tokens((int)(Hq / Hkv)));
  w.keys = plan_ws(w.rows.total, T, N, per);
  w.share = omx::attn_dkv_plan(B * Hkv, T, N, (int)(Hq / Hkv), B * T * Hkv * D * 8);
  w.shares = w.part_k = w.part_v = w.total = w.keys.total;
  if (w.share.splits > 1) {
    const size_t one = align_up((size_t)w.share.splits * B * T * Hkv * D * 4);
    w.part_k = w.shares + align_up((size_t)(B * T * Hkv) * 4);
    w.part_v = w.part_k + one;
    w.total = w.part_v + one;
  }
  return w;
}
}  // namespace

size_t omx_gdn_attn_bwd_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N) {
  if (!sized(B, T, Hq, Hkv, D, N)) return 0;
  return attn_bwd_ws(B, T, Hq, Hkv, D, N).total;
}

int omx_gdn_attn_bwd(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                     const int32_t* cu_seqlens, int64_t N, const void* o, const float* lse, const void* o_rest, const void* d_o,
                     void* dq, void* dk, void* dv, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                     float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "omx_gdn_attn_bwd";
  const Shape s{N, B, T, Hq, Hkv, D, cu_seqlens != nullptr};
  int rc = check_shape(fn, s);
  if (!rc) rc = check_ld(fn, "q_ld", q_ld, Hq * D);
  if (!rc) rc = check_ld(fn, "k_ld", k_ld, Hkv * D);
  if (!rc) rc = check_ld(fn, "v_ld", v_ld, Hkv * D);
  if (!rc) rc = check_scale(fn, scale);
  const int per = rc ? 1 : omx::attn_tile_tokens((int)(Hq / Hkv));
  if (!rc) rc = check_grid(fn, s, per);
  if (rc) return rc;
  const AttnBwdWs ws = attn_bwd_ws(B, T, Hq, Hkv, D, s.packed ? N : 0);
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
  const hipStream_t st = (hipStream_t)stream;
  hipError_t e = use_plan(p, ws.rows, workspace, per, st);
  if (e == hipSuccess) e = omx::launch_attn_dq(p, st);
  if (e == hipSuccess) e = use_plan(p, ws.keys, workspace, omx::attn_dkv_tile_tokens(), st);
  if (e == hipSuccess) e = omx::launch_attn_dkv(p, st);
  return launch_status(e, fn);
}

size_t omx_gdn_kv_write_workspace_size(int64_t T, int64_t N) {
  if (!sized(1, T, 1, 1, 1, N)) return 0;
  return plan_ws(0, T, N, omx::attn_dkv_tile_tokens()).total;
}

int omx_gdn_kv_write(const void* k, const void* v, int64_t k_ld, int64_t v_ld, const int32_t* cu_seqlens, int64_t N,
                     void* k_pages, void* v_pages, int64_t n_pages, int64_t page_size, const int32_t* block_table,
                     int64_t table_width, const int32_t* lengths, int64_t B, int64_t T, int64_t Hkv, int64_t D,
                     void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "omx_gdn_kv_write";
  const Shape s{N, B, T, Hkv, Hkv, D, cu_seqlens != nullptr};
  int rc = check_shape(fn, s);
  if (!rc) rc = check_ld(fn, "k_ld", k_ld, Hkv * D);
  if (!rc) rc = check_ld(fn, "v_ld", v_ld, Hkv * D);
  if (rc) return rc;
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
  p.k_pages = k_pages; p.v_pages = v_pages; p.table = block_table; p.held = lengths;
  p.table_w = (int)table_width; p.page = (int)page_size; p.n_pages = (int)n_pages;
  hipError_t e = use_plan(p, ws, workspace, per, (hipStream_t)stream);
  if (e == hipSuccess) e = omx::launch_kv_write(p, (hipStream_t)stream);
  return launch_status(e, fn);
}

namespace {
struct PagedWs {
  PlanWs plan;
  SplitWs split;
  int splits;
  size_t total;
};
PagedWs paged_ws(const Shape& s, int64_t capacity) {
  PagedWs w{};
  w.plan = plan_ws(0, s.T, s.packed ? s.N : 0, omx::attn_tile_tokens((int)(s.Hq / s.Hkv)));
  w.splits = paged_splits(s, capacity);
  w.split = split_ws(w.plan.total, w.splits, s.B * s.T * s.Hq, s.D);
  w.total = w.split.total;
  return w;
}
}  // namespace

size_t omx_gdn_attn_paged_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t N,
                                         int packed, int64_t page_size, int64_t table_width) {
  const Shape s{N, B, T, Hq, Hkv, D, packed != 0};
  if (!sized(B, T, Hq, Hkv, D, N) || !sized_table(page_size, table_width)) return 0;
  return paged_ws(s, page_size * table_width).total;
}

int omx_gdn_attn_paged(const void* q, int64_t q_ld, const int32_t* cu_seqlens, int64_t N, const void* k_pages,
                       const void* v_pages, int64_t n_pages, int64_t page_size, const int32_t* block_table,
                       int64_t table_width, const int32_t* lengths, void* o, int64_t B, int64_t T, int64_t Hq,
                       int64_t Hkv, int64_t D, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "omx_gdn_attn_paged";
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
  const PagedWs ws = paged_ws(s, page_size * table_width);
  REQUIRE(workspace_bytes >= ws.total, "%s: workspace of %zu bytes is smaller than the %zu needed", fn,
          workspace_bytes, ws.total);
  REQUIRE(q && o, "%s: a required pointer is NULL", fn);
  REQUIRE(aligned(q, 16) && aligned(o, 16), "%s: q and o must be 16-byte aligned", fn);
  REQUIRE(ws.total == 0 || (workspace && aligned(workspace, 16)), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  omx::AttnParams p = params(s, scale);
  p.q = q; p.q_ld = q_ld; p.o = o; p.cu = cu_seqlens;
  p.k_pages = const_cast<void*>(k_pages); p.v_pages = const_cast<void*>(v_pages);
  p.table = block_table; p.held = lengths;
  p.table_w = (int)table_width; p.page = (int)page_size; p.n_pages = (int)n_pages;
  p.splits = ws.splits;
  p.part_o = (float*)((char*)workspace + ws.split.o);
  p.part_ml = (float*)((char*)workspace + ws.split.ml);
  hipError_t e = use_plan(p, ws.plan, workspace, per, (hipStream_t)stream);
  if (e == hipSuccess) e = omx::launch_attn_fwd(p, (hipStream_t)stream);
  return launch_status(e, fn);
}

namespace {
SplitWs decode_ws(int splits, int64_t B, int64_t Hq, int64_t D) {
  // (one count of splits + B segments, of one row a head each)
  return splits > 1 ? split_ws(0, splits + (int)B, Hq, D) : split_ws(0, 1, 0, D);
}
}  // namespace

size_t omx_gdn_attn_decode_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t page_size,
                                          int64_t table_width) {
  if (B < 1 || !sized(B, 1, Hq, Hkv, D, B) || !sized_table(page_size, table_width)) return 0;
  return decode_ws(omx::decode_splits(B, Hkv, D, page_size * table_width), B, Hq, D).total;
}

int omx_gdn_attn_decode_step(const void* q, const void* k, const void* v, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                             void* k_pages, void* v_pages, int64_t n_pages, int64_t page_size,
                             const int32_t* block_table, int64_t table_width, const int32_t* lengths, void* out,
                             int64_t B, int64_t Hq, int64_t Hkv, int64_t D, float scale, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const char* fn = "omx_gdn_attn_decode_step";
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
  const int splits = omx::decode_splits(B, Hkv, D, page_size * table_width);
  const SplitWs ws = decode_ws(splits, B, Hq, D);
  REQUIRE(workspace_bytes >= ws.total, "%s: workspace of %zu bytes is smaller than the %zu needed", fn,
          workspace_bytes, ws.total);
  REQUIRE(q && k && v && out, "%s: a required pointer is NULL", fn);
  REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16), "%s: q, k, v, out must be 16-byte aligned", fn);
  REQUIRE(ws.total == 0 || (workspace && aligned(workspace, 16)), "%s: workspace must be non-NULL and 16-byte aligned", fn);
  omx::AttnParams p = params(s, scale);
  p.q = q; p.k = k; p.v = v; p.o = out;
  p.q_ld = q_ld; p.k_ld = k_ld; p.v_ld = v_ld;
  p.k_pages = k_pages; p.v_pages = v_pages; p.table = block_table; p.held = lengths;
  p.table_w = (int)table_width; p.page = (int)page_size; p.n_pages = (int)n_pages;
  p.splits = splits;
  p.part_o = (float*)((char*)workspace + ws.o);
  p.part_ml = (float*)((char*)workspace + ws.ml);
  return launch_status(omx::launch_attn_decode(p, (hipStream_t)stream), fn);
}

}  // extern "C"
