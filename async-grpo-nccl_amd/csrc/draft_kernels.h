// Verification of drafted tokens.  The chunk of sequence b is rows cu[b] .. cu[b+1] - 1: its last committed token, then K drafts.  Row
// cu[b] + i of `target` is the policy's distribution behind the chunk's first i + 1 tokens; `draft` has a row for each draft, in
// order (row cu[b] - c + i, c sequences that have rows in front of b): the distribution it was drawn from (no `draft`: each was
// chosen outright, 1 at it; a row past its end counts as zeros).
// Draft i, token d, stands while u_i draft_i(d) < target_i(d).  At the first that falls the token comes from max(target_i - draft_i, 0), or
// from target_i where that leaves nothing (equal rows, or rounding); behind K that stand from target_K.  Drawn by the row's own
// u: the first x whose running sum exceeds u times the sum, and the last x that counts where rounding leaves none.
// Products of two fp32 values and differences of bf16 or fp32 ones are exact in 64 bits, and the sums are held in 64: over 1.5e5
// tokens fp32 sums would move the borders between tokens by some of the tokens' own probability.  Values that are no
// probability (NaN, infinite, negative) count as zero; a row with nothing left gives token -1.
#pragma once
#include "lmhead_kernels.h"

namespace fgrpo {

struct VerifyParams {
  const void* target;    // [T][V], rows t_st apart, bf16 or fp32
  const void* draft;     // [drafts][V], rows d_st apart, or null
  const long long* ids;  // [T]
  const float* u;        // [T]
  const int* cu;         // [B + 1]
  long long t_st, d_st;
  int B, T, V, f32, drafts;
  int* accepted;         // [B]
  long long* tokens;     // [T]
};

__device__ __forceinline__ double draft_prob(const void* row, int f32, long long i) {
  const float x = f32 ? ((const float*)row)[i] : __uint_as_float((uint32_t)((const uint16_t*)row)[i] << 16);
  return x > 0.f && x < INFINITY ? (double)x : 0.0;
}
__device__ __forceinline__ const void* draft_row(const void* base, int f32, long long st, long long r) {
  return (const char*)base + r * st * (f32 ? 4 : 2);
}

// what is drawn from: `gone` null and tok < 0: p itself; gone null: p without tok; else max(p - gone, 0)
struct DraftRest {
  const void* p;
  const void* gone;
  long long tok;
  int f32;
  __device__ __forceinline__ double at(int x) const {
    const double a = draft_prob(p, f32, x);
    if (gone) return fmax(a - draft_prob(gone, f32, x), 0.0);
    return x == tok ? fmax(a - 1.0, 0.0) : a;
  }
};

// One work-group a sequence.
static __global__ __launch_bounds__(1024) void verify_drafts_kernel(VerifyParams p) {
  __shared__ double sh[17];
  __shared__ int sh_i[16];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lo = min(max(p.cu[b], 0), p.T), hi = min(max(p.cu[b + 1], lo), p.T);
  if (hi <= lo) {
    if (tid == 0) p.accepted[b] = 0;
    return;
  }
  const int K = hi - lo - 1;
  int first = lo;                // the sequence's first row of `draft`
  for (int i0 = 0; i0 < b; i0 += 64) first -= __popcll(__ballot(i0 + lane < b && p.cu[i0 + lane + 1] > p.cu[i0 + lane]));
  // the first draft that falls
  int n = K;
  for (int i0 = 0; i0 < K && n == K; i0 += 64) {
    const int i = i0 + lane;
    bool falls = false;
    if (i < K) {
      const long long d = p.ids[lo + i + 1];
      falls = true;
      if (d >= 0 && d < p.V) {
        const double a = draft_prob(draft_row(p.target, p.f32, p.t_st, lo + i), p.f32, d);
        const int r = first + i;
        const double q = !p.draft ? 1.0 : r >= 0 && r < p.drafts ? draft_prob(draft_row(p.draft, p.f32, p.d_st, r), p.f32, d) : 0.0;
        falls = !((double)p.u[lo + i] * q < a);
      }
    }
    const unsigned long long m = __ballot(falls);
    if (m) n = i0 + __ffsll(m) - 1;
  }
  const int row = lo + n;
  DraftRest rest{draft_row(p.target, p.f32, p.t_st, row), nullptr, -1, p.f32};
  if (n < K) {
    const int r = first + n;
    if (!p.draft) rest.tok = p.ids[row + 1];
    else if (r >= 0 && r < p.drafts) rest.gone = draft_row(p.draft, p.f32, p.d_st, r);
  }
  auto block_sum = [&](double x) {
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
    __syncthreads();
    if (lane == 0) sh[wave] = x;
    __syncthreads();
    double t = 0;
    for (int w = 0; w < 16; ++w) t += sh[w];
    return t;
  };
  double total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    double s = 0;
    for (int x = tid; x < p.V; x += 1024) s += rest.at(x);
    total = block_sum(s);
    if (total > 0 || (!rest.gone && rest.tok < 0)) break;
    rest.gone = nullptr, rest.tok = -1;
  }
  const double want = (double)p.u[row] * total;
  // the first x whose running sum exceeds it, 1024 at a time
  double before = 0;
  int found = -1, last = -1;
  for (int x0 = 0; x0 < p.V && found < 0; x0 += 1024) {
    const int x = x0 + tid;
    const double w = x < p.V ? rest.at(x) : 0.0;
    double upto = w;
    for (int d = 1; d < 64; d <<= 1) {
      const double y = __shfl_up(upto, d, 64);
      if (lane >= d) upto += y;
    }
    __syncthreads();
    if (lane == 63) sh[wave] = upto;
    __syncthreads();
    double base = before;
    for (int i = 0; i < wave; ++i) base += sh[i];
    const unsigned long long over = __ballot(w > 0 && base + upto > want), some = __ballot(w > 0);
    if (lane == 0) sh_i[wave] = over ? x0 + 64 * wave + __ffsll(over) - 1 : -1;
    __syncthreads();
    for (int i = 0; i < 16 && found < 0; ++i) found = sh_i[i];
    __syncthreads();
    if (lane == 0) sh_i[wave] = some ? x0 + 64 * wave + 63 - __clzll(some) : -1;
    __syncthreads();
    for (int i = 0; i < 16; ++i) last = max(last, sh_i[i]);
    for (int i = 0; i < 16; ++i) before += sh[i];
  }
  if (found < 0) found = last;
  if (tid == 0) p.accepted[b] = n;
  for (int i = tid; i <= K; i += 1024) p.tokens[lo + i] = i < n ? p.ids[lo + i + 1] : i == n ? found : -1;
}

}  // namespace fgrpo
