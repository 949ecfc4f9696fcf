// Paged key/value cache, the attention over it and the verification of drafted tokens: C entry points, argument checks and launches
// (kernels in paged_cache.h, paged_rows.h, paged_tiles.h, paged_deal.h, draft_kernels.h).
#include <string.h>

#include <algorithm>

#include "host_common.h"
#include "draft_kernels.h"
#include "paged_tiles.h"

using namespace fgrpo;

namespace {

constexpr long long kMostBetween = 1LL << 26;      // elements between tokens: 16 of them behind a 32-bit offset

int check_cache(const char* who, const fgrpo_paged_cache* c, const int32_t* table, long long table_st, int width, const int32_t* lens,
                const int32_t* cu, int B, int T) {
  if (!c || !c->k || !c->v || !lens || !cu) return fail(FGRPO_ERR_BAD_ARG, "%s: null argument", who);
  if (B <= 0 || T <= 0 || width < 0 || (width > 0 && !table)) return fail(FGRPO_ERR_BAD_ARG, "%s: B=%d T=%d width=%d", who, B, T, width);
  if (table_st < 0 || (table_st < width && B > 1)) return fail(FGRPO_ERR_BAD_ARG, "%s: rows of the block table %lld apart, %d wide", who, table_st, width);
  if (c->num_blocks <= 0 || c->heads <= 0) return fail(FGRPO_ERR_BAD_ARG, "%s: num_blocks=%d heads=%d", who, c->num_blocks, c->heads);
  if (c->block_size < 16 || c->block_size > 65536 || (c->block_size & (c->block_size - 1)))
    return fail(FGRPO_ERR_UNSUPPORTED, "%s: block size %d (a power of two from 16 to 65536)", who, c->block_size);
  if ((long long)width * c->block_size > (1LL << 31) - 65536)      // places a few steps behind the last are formed in 32 bits
    return fail(FGRPO_ERR_UNSUPPORTED, "%s: a block table of %d blocks of %d (at most 2^31 - 2^16 tokens)", who, width, c->block_size);
  if (c->head_dim != 128 && c->head_dim != 64) return fail(FGRPO_ERR_UNSUPPORTED, "%s: head dimension %d not supported (128 or 64)", who, c->head_dim);
  if (c->dtype != FGRPO_BF16 && c->dtype != FGRPO_F8E4M3) return fail(FGRPO_ERR_BAD_ARG, "%s: cache dtype=%d", who, c->dtype);
  const bool fp8 = c->dtype == FGRPO_F8E4M3;
  if (fp8 && (!c->k_scale || !c->v_scale)) return fail(FGRPO_ERR_BAD_ARG, "%s: an e4m3 cache has scales", who);
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(FGRPO_ERR_ALIGN, "%s: the cache must be 16-byte aligned", who);
  for (int i = 0; i < 3; ++i) {
    if (c->k_stride[i] < 0 || c->v_stride[i] < 0 || c->k_stride[i] % 16 || c->v_stride[i] % 16)
      return fail(FGRPO_ERR_ALIGN, "%s: strides of the cache must be multiples of 16 elements", who);
    if (fp8 && (c->k_scale_stride[i] < 0 || c->v_scale_stride[i] < 0)) return fail(FGRPO_ERR_BAD_ARG, "%s: negative stride", who);
    if (i == 1 && (c->k_stride[i] >= kMostBetween || c->v_stride[i] >= kMostBetween || (fp8 && (c->k_scale_stride[i] >= kMostBetween || c->v_scale_stride[i] >= kMostBetween))))
      return fail(FGRPO_ERR_UNSUPPORTED, "%s: tokens of the cache 2^26 elements apart or more", who);
  }
  return 0;
}

PagedView view_of(const fgrpo_paged_cache* c, const int32_t* table, long long table_st, int width, const int32_t* lens, const int32_t* cu, int B, int T) {
  PagedView v;
  memset(&v, 0, sizeof(v));
  v.k = (char*)c->k, v.v = (char*)c->v, v.k_scale = c->k_scale, v.v_scale = c->v_scale;
  for (int i = 0; i < 3; ++i)
    v.k_st[i] = c->k_stride[i], v.v_st[i] = c->v_stride[i], v.ks_st[i] = c->k_scale_stride[i], v.vs_st[i] = c->v_scale_stride[i];
  v.table = width > 0 ? table : lens, v.lens = lens, v.cu = cu, v.table_st = width > 0 ? table_st : 0, v.reach = width * c->block_size;
  v.B = B, v.T = T, v.width = width > 0 ? width : 1, v.page_log2 = __builtin_ctz(c->block_size), v.num_pages = c->num_blocks, v.Hkv = c->heads;
  return v;
}

#define PAGED_DISPATCH(kernel, c, grid, threads, st, ...)                                                              \
  do {                                                                                                                 \
    const bool fp8_ = (c)->dtype == FGRPO_F8E4M3;                                                                      \
    if ((c)->head_dim == 128 && fp8_) hipLaunchKernelGGL((kernel<128, true>), grid, dim3(threads), 0, st, __VA_ARGS__);  \
    else if ((c)->head_dim == 128) hipLaunchKernelGGL((kernel<128, false>), grid, dim3(threads), 0, st, __VA_ARGS__);    \
    else if (fp8_) hipLaunchKernelGGL((kernel<64, true>), grid, dim3(threads), 0, st, __VA_ARGS__);                      \
    else hipLaunchKernelGGL((kernel<64, false>), grid, dim3(threads), 0, st, __VA_ARGS__);                               \
    HIP_TRY(hipGetLastError());                                                                                        \
  } while (0)

// How a call is divided, from shapes alone: rows of an item (16, 32: one wavefront; 128: four) and work-groups.
// Up to 16 rows a sequence and K/V head take blocks of 16 (64 sequences of 1000 .. 4000 keys, 12 / 2 heads, bf16: 38 us, blocks of 32 42; e4m3 32.5, 36).
// Every block reads its keys, from L2 but for the first, so with many blocks tiles of 128 win, and with few their larger parts and merges cost more than that: us,
// 32 / 128, bf16, D = 128, by blocks x keys that the table has room for: 128 K 25 / 46 (4 sequences to 16000) and 21 / 28 (16 to 4000),
// 384 K 27 / 37, 512 K 38 / 62, 50 / 77, 40 / 39, 39 / 36 and 43 / 39 (from 4 sequences to 64), 768 K 47 / 38, 1 M 60 / 45, 57 / 42, 85 / 84, 2 M 100 / 51, 220 / 146;
// D = 64: 256 K 21 / 30, 512 K 26 / 24, 640 K 25 / 27, 1 M 36 / 29; e4m3 alike.  So: 512 K.  One block a sequence is never far behind (75 / 72, 43 / 39; e4m3 89 / 111).
struct PagedPlan {
  int rows, W, items;      // items: as in PagedSplit
  size_t slots() const { return 2ull * W; }
  size_t rec_bytes() const { return (size_t)W * 2 * sizeof(int4); }
  size_t part_bytes(int D) const { return slots() * rows * D * 4; }
  size_t bytes(int D) const { return rec_bytes() + part_bytes(D) + slots() * rows * sizeof(float2); }
};
PagedPlan plan_paged(const fgrpo_paged_cache* c, int width, int n_seq, int T, int G, int max_len) {
  const long long tokens = max_len > 0 ? (max_len < T ? max_len : T) : ((long long)T + n_seq - 1) / n_seq, rows = tokens * G;      // not known: the mean
  const double blocks = ((double)T * G + 31.0 * n_seq) / 32 * c->heads, keys = (double)width * c->block_size;
  PagedPlan r{rows <= 16 ? 16 : rows <= 32 || blocks * keys <= 512 * 1024 ? 32 : kPagedRows, 0, 0};
  const long long items = ((long long)T * G / r.rows + n_seq) * c->heads, steps = ((long long)width * c->block_size + 63) / 64 + 1;
  long long W = r.rows == kPagedRows ? std::min(2LL * num_cus(), 512LL) : 4LL * num_cus();      // 512: a lane of a wavefront for each of an XCD's eighth
  if (items < W && items * steps < W) W = items * steps;
  r.W = (int)round_up(W, 8);
  // Few items, many parts: merged an item's unit a work-group (one sequence of 100000 keys 54 us, else 94; 16 of 1000 .. 4000 17.2, 25.7; 48 of 128 .. 8000, 12 / 2
  // heads, 43 and 46).  At half as many work-groups an item it is behind: 128 sequences of 1000 .. 4000 with four drafts 78 us, else 73.
  if (r.rows != kPagedRows && 4 * items <= r.W) r.items = (int)items;
  return r;
}

template <int HD, bool PAIRS, int SHAPE, int RB>
int launch_merge(const PagedAttn& p, const PagedSplit& sp, hipStream_t st) {
  if (sp.items > 0)
    hipLaunchKernelGGL((paged_merge_items_kernel<HD, PAIRS, SHAPE, RB>), dim3(sp.items, RB * HD / (SHAPE == 32 ? 8 : 16)), dim3(256), 0, st, p, sp);
  else
    hipLaunchKernelGGL((paged_merge_kernel<HD, PAIRS, SHAPE, RB>), dim3(sp.W, RB), dim3(256), 0, st, p, sp);
  HIP_TRY(hipGetLastError());
  return 0;
}
template <int HD, bool FP8>
int launch_attn(const PagedPlan& plan, const PagedAttn& p, const PagedSplit& sp, hipStream_t st) {
  const dim3 grid(sp.W);
  if (plan.rows == 16) hipLaunchKernelGGL((paged_rows16_kernel<HD, FP8>), grid, dim3(64), 0, st, p, sp);
  else if (plan.rows == 32) hipLaunchKernelGGL((paged_rows_kernel<HD, FP8>), grid, dim3(64), 0, st, p, sp);
  else hipLaunchKernelGGL((paged_tiles_kernel<HD, FP8>), grid, dim3(256), 0, st, p, sp);
  HIP_TRY(hipGetLastError());
  if (plan.rows == 16) return launch_merge<HD, FP8, 16, 1>(p, sp, st);
  if (plan.rows == 32) return launch_merge<HD, FP8, 32, 1>(p, sp, st);
  return launch_merge<HD, false, 32, kPagedTileRB>(p, sp, st);
}

int verify_chunks(int V) { return (V + kVerifyChunk - 1) / kVerifyChunk; }
size_t verify_sums_bytes(int n_seq, int V) { return (size_t)n_seq * verify_chunks(V) * sizeof(double2); }

template <bool F32, bool ALIGNED>
int launch_verify(const VerifyParams& p, hipStream_t st) {
  hipLaunchKernelGGL((verify_sums_kernel<F32, ALIGNED>), dim3(p.B * p.chunks), dim3(kVerifyThreads), 0, st, p);
  HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL((verify_draw_kernel<F32, ALIGNED>), dim3(p.B), dim3(kVerifyThreads), 0, st, p);
  HIP_TRY(hipGetLastError());
  return 0;
}

}  // namespace

extern "C" {

int fgrpo_paged_cache_write(const fgrpo_paged_cache* cache, const void* k, const void* v, long long k_stride_t, long long k_stride_h,
                            long long v_stride_t, long long v_stride_h, const int32_t* block_table, long long table_stride, int width,
                            const int32_t* seqused_k, const int32_t* cu_seqlens, int n_seq, int T, void* stream) {
  const int rc = check_cache("paged_cache_write", cache, block_table, table_stride, width, seqused_k, cu_seqlens, n_seq, T);
  if (rc) return rc;
  if (!k || !v) return fail(FGRPO_ERR_BAD_ARG, "paged_cache_write: null argument");
  if (!aligned16(k) || !aligned16(v)) return fail(FGRPO_ERR_ALIGN, "paged_cache_write: k/v must be 16-byte aligned");
  const long long st[4] = {k_stride_t, k_stride_h, v_stride_t, v_stride_h};
  for (int i = 0; i < 4; ++i)
    if (st[i] < 0 || st[i] % 8) return fail(FGRPO_ERR_ALIGN, "paged_cache_write: strides must be multiples of 8 elements");
  if (width == 0) return 0;      // no sequence has a place
  PagedWrite p;
  p.c = view_of(cache, block_table, table_stride, width, seqused_k, cu_seqlens, n_seq, T);
  p.k = (const bf16_t*)k, p.v = (const bf16_t*)v, p.k_t = k_stride_t, p.k_h = k_stride_h, p.v_t = v_stride_t, p.v_h = v_stride_h;
  PAGED_DISPATCH(paged_write_kernel, cache, dim3((T + 3) / 4), 256, (hipStream_t)stream, p);
  return 0;
}

int fgrpo_paged_cache_read(const fgrpo_paged_cache* cache, const int32_t* block_table, long long table_stride, int width,
                           const int32_t* seqused_k, const int32_t* cu_seqlens_k, int n_seq, int total, void* k_out, void* v_out, void* stream) {
  const int rc = check_cache("paged_cache_read", cache, block_table, table_stride, width, seqused_k, cu_seqlens_k, n_seq, total);
  if (rc) return rc;
  if (!k_out || !v_out) return fail(FGRPO_ERR_BAD_ARG, "paged_cache_read: null argument");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(FGRPO_ERR_ALIGN, "paged_cache_read: outputs must be 16-byte aligned");
  if (width == 0) return 0;
  PagedRead p;
  p.c = view_of(cache, block_table, table_stride, width, seqused_k, cu_seqlens_k, n_seq, total);
  p.k = (bf16_t*)k_out, p.v = (bf16_t*)v_out;
  PAGED_DISPATCH(paged_read_kernel, cache, dim3((total + 3) / 4), 256, (hipStream_t)stream, p);
  return 0;
}

size_t fgrpo_paged_attn_workspace(const fgrpo_paged_cache* cache, int width, int n_seq, int T, int Hq, int max_len) {
  if (!cache || cache->heads <= 0 || Hq <= 0 || Hq % cache->heads || n_seq <= 0 || T <= 0 || width < 0 || (cache->head_dim != 128 && cache->head_dim != 64)) return 0;
  return plan_paged(cache, width, n_seq, T, Hq / cache->heads, max_len).bytes(cache->head_dim);
}

int fgrpo_paged_attn_fwd(const void* q, long long q_stride_t, long long q_stride_h, const fgrpo_paged_cache* cache, const int32_t* block_table,
                         long long table_stride, int width, const int32_t* seqused_k, const int32_t* cu_seqlens_q, int n_seq, int T, int Hq,
                         int max_len, float softmax_scale, int causal, void* out, float* lse, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_cache("paged_attn_fwd", cache, block_table, table_stride, width, seqused_k, cu_seqlens_q, n_seq, T);
  if (rc) return rc;
  if (!q || !out) return fail(FGRPO_ERR_BAD_ARG, "paged_attn_fwd: null argument");
  if (Hq <= 0 || Hq % cache->heads) return fail(FGRPO_ERR_BAD_ARG, "paged_attn_fwd: Hq=%d Hkv=%d", Hq, cache->heads);
  if (!(softmax_scale > 0.f)) return fail(FGRPO_ERR_BAD_ARG, "paged_attn_fwd: softmax scale must be positive");
  if (!aligned16(q) || !aligned16(out)) return fail(FGRPO_ERR_ALIGN, "paged_attn_fwd: q/out must be 16-byte aligned");
  if (q_stride_t < 0 || q_stride_h < 0 || q_stride_t % 8 || q_stride_h % 8)
    return fail(FGRPO_ERR_ALIGN, "paged_attn_fwd: strides must be multiples of 8 elements");
  const int G = Hq / cache->heads;
  if ((long long)T * G >= (1LL << 31) - 256) return fail(FGRPO_ERR_UNSUPPORTED, "paged_attn_fwd: T=%d rows of %d heads", T, G);
  hipStream_t st = (hipStream_t)stream;
  PagedAttn p;
  p.c = view_of(cache, block_table, table_stride, width, seqused_k, cu_seqlens_q, n_seq, T);
  p.q = (const bf16_t*)q, p.q_t = q_stride_t, p.q_h = q_stride_h, p.out = (bf16_t*)out, p.lse = lse;
  p.scale = softmax_scale, p.Hq = Hq, p.G = G, p.causal = causal != 0;
  const PagedPlan plan = plan_paged(cache, width, n_seq, T, G, max_len);
  const size_t need = plan.bytes(cache->head_dim);
  if (!ws || ws_bytes < need) return fail(FGRPO_ERR_WORKSPACE, "paged_attn_fwd: workspace %zu < %zu", ws ? ws_bytes : 0, need);
  if (!aligned16(ws)) return fail(FGRPO_ERR_ALIGN, "paged_attn_fwd: workspace must be 16-byte aligned");
  PagedSplit sp;
  sp.W = plan.W, sp.items = plan.items, sp.most_parts = plan.items > 0 ? 1024 : 128;      // what a merge reads one behind the other
  sp.rec = (int4*)ws;
  sp.part = (float*)((char*)ws + plan.rec_bytes());
  sp.ml = (float2*)((char*)sp.part + plan.part_bytes(cache->head_dim));
  if (cache->dtype == FGRPO_F8E4M3) return cache->head_dim == 128 ? launch_attn<128, true>(plan, p, sp, st) : launch_attn<64, true>(plan, p, sp, st);
  return cache->head_dim == 128 ? launch_attn<128, false>(plan, p, sp, st) : launch_attn<64, false>(plan, p, sp, st);
}

size_t fgrpo_verify_drafts_workspace(int n_seq, int V) {
  if (n_seq <= 0 || V <= 0) return 0;
  return verify_sums_bytes(n_seq, V) + (size_t)n_seq * sizeof(int);
}

int fgrpo_verify_drafts(const void* target, long long target_stride, const void* draft, long long draft_stride, int draft_rows, int dtype,
                        const int64_t* ids, const float* u, const int32_t* cu_seqlens, int n_seq, int T, int V, int32_t* accepted, int64_t* tokens,
                        void* ws, size_t ws_bytes, void* stream) {
  if (!target || !ids || !u || !cu_seqlens || !accepted || !tokens) return fail(FGRPO_ERR_BAD_ARG, "verify_drafts: null argument");
  if (n_seq <= 0 || T <= 0 || V <= 0 || target_stride < V || draft_rows < 0 || (draft && draft_stride < V))
    return fail(FGRPO_ERR_BAD_ARG, "verify_drafts: n_seq=%d T=%d V=%d, rows %lld and %lld apart", n_seq, T, V, target_stride, draft_stride);
  if (dtype != FGRPO_BF16 && dtype != FGRPO_F32) return fail(FGRPO_ERR_BAD_ARG, "verify_drafts: dtype=%d", dtype);
  if (V > 0x7fffffff - 2 * kVerifyChunk || (long long)n_seq * verify_chunks(V) >= (1LL << 31))
    return fail(FGRPO_ERR_UNSUPPORTED, "verify_drafts: %d sequences over a vocabulary of %d", n_seq, V);
  const size_t need = fgrpo_verify_drafts_workspace(n_seq, V);
  if (!ws || ws_bytes < need) return fail(FGRPO_ERR_WORKSPACE, "verify_drafts: workspace %zu < %zu", ws ? ws_bytes : 0, need);
  if (!aligned16(ws)) return fail(FGRPO_ERR_ALIGN, "verify_drafts: workspace must be 16-byte aligned");
  VerifyParams p{target, draft, (const long long*)ids, u, cu_seqlens, target_stride, draft_stride, n_seq, T, V, draft_rows, verify_chunks(V), accepted, (long long*)tokens,
                 (double2*)ws, (int*)((char*)ws + verify_sums_bytes(n_seq, V))};
  const bool f32 = dtype == FGRPO_F32;
  // rows that begin at multiples of 16 bytes are read 16 bytes at a time (64 sequences, 151936 tokens, bf16: 19.0 us, else 31.7; fp32 23.4, 34.5; 32000 tokens 12.6, 17.4)
  const long long es = f32 ? 4 : 2;
  const bool whole = aligned16(target) && target_stride * es % 16 == 0 && (!draft || (aligned16(draft) && draft_stride * es % 16 == 0));
  hipStream_t st = (hipStream_t)stream;
  if (f32) return whole ? launch_verify<true, true>(p, st) : launch_verify<true, false>(p, st);
  return whole ? launch_verify<false, true>(p, st) : launch_verify<false, false>(p, st);
}

}  // extern "C"
