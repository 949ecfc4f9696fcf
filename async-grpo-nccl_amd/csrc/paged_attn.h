// Attention of new tokens over a paged cache (paged_cache.h): token i of the q_b new ones of sequence b sees the keys
// j < k_b, and with the causal mask j <= k_b - q_b + i.  o = softmax(c q K^T) V over what it sees; nothing seen: o = 0, lse = -inf.
//
// The G query heads of a K/V head read the same keys, so a work-group's rows are (token, head of the group) pairs, row r of a
// sequence being token r / G, head r mod G: 128 of them whatever G is.  A wavefront has 32 rows and computes
// S^T = K Q^T and O^T = V^T P^T with the matrix instruction's operands as the packed attention has them (attn_kernels.h): a lane owns one
// row, and its probabilities are the next product's operand as they lie.
// An e4m3 cache: codes are exact in bf16, so the products take them as they are; a key's scale multiplies its scores (exactly as
// often as it would its D values, at a D-th of the work), and a value's scale its probability, in fp32, before that is
// rounded to bf16 for the second product.  Sums, maxima and both accumulators are fp32.
#pragma once
#include "paged_cache.h"

namespace fgrpo {

struct PagedAttn {
  PagedView c;
  const bf16_t* q;       // [T][Hq][HD], strides in elements
  long long q_t, q_h;
  bf16_t* out;           // [T][Hq][HD] contiguous
  float* lse;            // [Hq][T] or null
  float scale;
  int Hq, G, causal;
};

constexpr int kPagedRows = 128;

// 64 rows of one head, 16-byte pieces of the bf16 tile each: cache -> LDS.  Keys from k_end on are the last one again (masked).
template <int HD, bool FP8>
__device__ __forceinline__ void paged_stage(const PagedView& c, const char* base, const long long (&st)[3], int b, int head, int k0, int k_end, char* tile) {
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    const int ch = threadIdx.x + 256 * i, row = ch / (HD / 8), j = min(k0 + row, k_end - 1);
    const long long o = paged_offset(st, paged_page(c, b, j), j & ((1 << c.page_log2) - 1), head) + ch % (HD / 8) * 8;
    u32x4_t x;
    if constexpr (FP8) x = paged_restore(*(const uint2*)(base + o), 1.f);
    else x = *(const u32x4_t*)(base + 2 * o);
    *(u32x4_t*)(tile + row * (HD * 2) + (((ch % (HD / 8)) ^ attn_swz<HD>(row)) << 4)) = x;
  }
}

template <int HD, bool FP8>
static __global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedAttn p) {
  constexpr int KS = HD / 16, DB = HD / 32, TILE = kAttnBK * HD * 2;
  __shared__ __attribute__((aligned(16))) char smem[2 * TILE];
  __shared__ __attribute__((aligned(16))) float s_scale[2][kAttnBK];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const AttnLane<HD> L = attn_lane<HD>(lane);
  const int head = blockIdx.y;
  // the tile of this number: sequences one behind the other
  int tile = blockIdx.x, b = 0, q0 = 0, nq = 0;
  for (; b < p.c.B; ++b) {
    q0 = min(max(p.c.cu[b], 0), p.c.T);
    nq = min(max(p.c.cu[b + 1], q0), p.c.T) - q0;
    const int n = (int)(((long long)nq * p.G + kPagedRows - 1) / kPagedRows);
    if (tile < n) break;
    tile -= n;
  }
  if (b >= p.c.B) return;
  const int len = paged_len(p.c, b), rows = nq * p.G, r0 = tile * kPagedRows;
  const int row = r0 + 32 * wave + (lane & 31), tok = row / p.G, hq = head * p.G + row % p.G;
  const bool valid = row < rows;
  const int seen = !valid ? 0 : p.causal ? min(max(len - nq + tok + 1, 0), len) : len;
  const int last_tok = (min(r0 + kPagedRows, rows) - 1) / p.G;
  const int k_end = p.causal ? min(max(len - nq + last_tok + 1, 0), len) : len;
  bf16x8_t qf[KS];
  attn_row_operand(qf, p.q + (long long)(q0 + (valid ? tok : 0)) * p.q_t + (long long)hq * p.q_h, valid, h);
  f32x16_t acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const float c = p.scale * kLog2e;
  for (int kb = 0; kb < k_end; kb += kAttnBK) {
    __syncthreads();
    paged_stage<HD, FP8>(p.c, p.c.k, p.c.k_st, b, head, kb, k_end, smem);
    paged_stage<HD, FP8>(p.c, p.c.v, p.c.v_st, b, head, kb, k_end, smem + TILE);
    if (FP8 && threadIdx.x < 2 * kAttnBK) {
      const int i = threadIdx.x % kAttnBK, j = min(kb + i, k_end - 1), page = paged_page(p.c, b, j), place = j & ((1 << p.c.page_log2) - 1);
      if (threadIdx.x < kAttnBK) s_scale[0][i] = p.c.k_scale[paged_offset(p.c.ks_st, page, place, head)] * c;
      else s_scale[1][i] = p.c.v_scale[paged_offset(p.c.vs_st, page, place, head)];
    }
    __syncthreads();
    f32x16_t s[2];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[mb][r] = 0.f;
#pragma unroll
      for (int st = 0; st < KS; ++st) s[mb] = FGRPO_MFMA(attn_frag<HD>(smem, L, mb, st), qf[st], s[mb]);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = 32 * mb + 8 * (r >> 2) + 4 * h + (r & 3);
        const float x = s[mb][r] * (FP8 ? s_scale[0][at] : c);      // in powers of two
        s[mb][r] = kb + at < seen ? x : -INFINITY;
        mx = fmaxf(mx, s[mb][r]);
      }
    mx = fmaxf(mx, attn_swap32(mx));
    const float m_new = fmaxf(m_run, mx), m_use = m_new == -INFINITY ? 0.f : m_new, alpha = fast_exp2(m_run - m_use);
    float sum = 0.f;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = fast_exp2(s[mb][r] - m_use);
        sum += e;
        s[mb][r] = FP8 ? e * s_scale[1][32 * mb + 8 * (r >> 2) + 4 * h + (r & 3)] : e;
      }
    l_run = l_run * alpha + sum;
    m_run = m_new;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float tmp[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) tmp[j] = s[g / 2][8 * (g % 2) + j];
      const bf16x8_t pf = attn_pack8(tmp);
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] = FGRPO_MFMA(attn_frag_tr<HD>(smem + TILE, L, 16 * g, db), pf, acc[db]);
    }
  }
  const float l = l_run + attn_swap32(l_run);
  if (valid) {
    attn_store_rowmajor(acc, l > 0.f ? 1.f / l : 0.f, p.out + ((long long)(q0 + tok) * p.Hq + hq) * HD, h);
    if (p.lse && h == 0) p.lse[(long long)hq * p.c.T + q0 + tok] = l > 0.f ? (m_run + __log2f(l)) * 0.6931471805599453f : -INFINITY;
  }
}

}  // namespace fgrpo
