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

constexpr int kVerifyThreads = 256, kVerifyRun = 16, kVerifyChunk = kVerifyThreads * kVerifyRun;      // tokens of a work-group

struct VerifyParams {
  const void* target;    // [T][V], rows t_st apart, bf16 or fp32
  const void* draft;     // [drafts][V], rows d_st apart, or null
  const long long* ids;  // [T]
  const float* u;        // [T]
  const int* cu;         // [B + 1]
  long long t_st, d_st;
  int B, T, V, drafts, chunks;
  int* accepted;         // [B]
  long long* tokens;     // [T]
  double2* sums;         // [B][chunks] of what is drawn from, and of the target's row
  int* first;            // [B] the sequence's first row of `draft`
};

template <bool F32>
struct VerifyRow {
  static constexpr int ES = F32 ? 4 : 2, VEC = 16 / ES;
  const char* at;
  __device__ __forceinline__ static VerifyRow of(const void* base, long long st, long long r) { return VerifyRow{(const char*)base + r * st * ES}; }
  __device__ __forceinline__ static double prob(float x) { return x > 0.f && x < INFINITY ? (double)x : 0.0; }
  __device__ __forceinline__ double one(long long i) const {
    return prob(F32 ? ((const float*)at)[i] : __uint_as_float((uint32_t)((const uint16_t*)at)[i] << 16));
  }
  // tokens x .. x + VEC - 1 of a row of V; ALIGNED: 16 bytes at once
  template <bool ALIGNED>
  __device__ __forceinline__ void some(double (&out)[VEC], int x, int V) const {
    if (ALIGNED && x + VEC <= V) {
      const u32x4_t w = *(const u32x4_t*)(at + (long long)x * ES);
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = prob(__uint_as_float(F32 ? w[i] : i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = x + i < V ? one(x + i) : 0.0;
    }
  }
};

// what is drawn from: the target's row, less the draft's, or less 1 at one token
template <bool F32>
struct VerifyRest {
  VerifyRow<F32> p, gone;
  bool less;
  int tok;
  template <bool ALIGNED>
  __device__ __forceinline__ void some(double (&rest)[VerifyRow<F32>::VEC], double (&all)[VerifyRow<F32>::VEC], int x, int V) const {
    constexpr int VEC = VerifyRow<F32>::VEC;
    p.template some<ALIGNED>(all, x, V);
    if (less) {
      double q[VEC];
      gone.template some<ALIGNED>(q, x, V);
#pragma unroll
      for (int i = 0; i < VEC; ++i) rest[i] = fmax(all[i] - q[i], 0.0);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) rest[i] = x + i == tok ? fmax(all[i] - 1.0, 0.0) : all[i];
    }
  }
};
template <bool F32>
__device__ __forceinline__ VerifyRest<F32> verify_rest(const VerifyParams& p, int lo, int K, int n, int first) {
  VerifyRest<F32> r{VerifyRow<F32>::of(p.target, p.t_st, lo + n), {nullptr}, false, -1};
  if (n < K) {
    const int row = first + n;
    if (!p.draft) {
      const long long d = p.ids[lo + n + 1];
      r.tok = d >= 0 && d < p.V ? (int)d : -1;
    } else if (row >= 0 && row < p.drafts) {
      r.gone = VerifyRow<F32>::of(p.draft, p.d_st, row), r.less = true;
    }
  }
  return r;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}

// Which drafts stand, and the sums of a chunk of the vocabulary: work-group (sequence, chunk).  Every chunk finds the row by itself
// (a few loads that depend on each other, beside hundreds of work-groups that stream); the first leaves it for the second launch.
// Bound by its loads, two rows a sequence: 64 sequences, 151936 tokens, fp32, 78 MB in 25 us with the launch behind it; 4 of 32000 in bf16 10 us, two launches.
template <bool F32, bool ALIGNED>
static __global__ __launch_bounds__(kVerifyThreads) void verify_sums_kernel(VerifyParams p) {
  constexpr int VEC = VerifyRow<F32>::VEC;
  __shared__ double2 sh[kVerifyThreads / 64];
  const int b = blockIdx.x / p.chunks, chunk = blockIdx.x - b * p.chunks, tid = threadIdx.x, lane = tid & 63;
  const int lo = min(max(p.cu[b], 0), p.T), hi = min(max(p.cu[b + 1], lo), p.T), K = hi - lo - 1;
  if (K < 0) {
    if (chunk == 0 && tid == 0) p.accepted[b] = 0;
    return;
  }
  int first = lo;                // each sequence in front that has rows has one row less of `draft`
  if (p.draft)
    for (int i0 = 0; i0 < b; i0 += 64) first -= __popcll(__ballot(i0 + lane < b && p.cu[i0 + lane + 1] > p.cu[i0 + lane]));
  int n = K;                     // the first draft that falls
  for (int i0 = 0; i0 < K && n == K; i0 += 64) {
    const int i = i0 + lane;
    bool falls = false;
    if (i < K) {
      const long long d = p.ids[lo + i + 1];
      falls = true;
      if (d >= 0 && d < p.V) {
        const double a = VerifyRow<F32>::of(p.target, p.t_st, lo + i).one(d);
        const int r = first + i;
        const double q = !p.draft ? 1.0 : r >= 0 && r < p.drafts ? VerifyRow<F32>::of(p.draft, p.d_st, r).one(d) : 0.0;
        falls = !((double)p.u[lo + i] * q < a);
      }
    }
    const unsigned long long m = __ballot(falls);
    if (m) n = i0 + __ffsll(m) - 1;
  }
  n = __builtin_amdgcn_readfirstlane(n);
  if (chunk == 0 && tid == 0) p.accepted[b] = n, p.first[b] = first;
  const VerifyRest<F32> rest = verify_rest<F32>(p, lo, K, n, first);
  double s = 0, t = 0;
#pragma unroll
  for (int i = 0; i < kVerifyRun / VEC; ++i) {
    const int x = chunk * kVerifyChunk + (i * kVerifyThreads + tid) * VEC;
    double r[VEC], a[VEC];
    rest.template some<ALIGNED>(r, a, x, p.V);
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += r[j], t += a[j];
  }
  s = wave_sum(s), t = wave_sum(t);
  if (lane == 0) sh[tid / 64] = make_double2(s, t);
  __syncthreads();
  if (tid == 0) {
    double2 x = sh[0];
    for (int i = 1; i < kVerifyThreads / 64; ++i) x.x += sh[i].x, x.y += sh[i].y;
    p.sums[(long long)b * p.chunks + chunk] = x;
  }
}

// sum of x over the threads in front of this one; `total` over all of them
__device__ __forceinline__ double block_before(double x, double* sh, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double upto = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double y = __shfl_up(upto, d, 64);
    if (lane >= d) upto += y;
  }
  __syncthreads();
  if (lane == 63) sh[wave] = upto;
  __syncthreads();
  double before = upto - x;
  total = 0;
  for (int i = 0; i < kVerifyThreads / 64; ++i) {
    if (i < wave) before += sh[i];
    total += sh[i];
  }
  return before;
}
__device__ __forceinline__ int block_min(int x, int* sh) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = min(x, __shfl_xor(x, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  for (int i = 0; i < kVerifyThreads / 64; ++i) x = min(x, sh[i]);
  return x;
}

// The chunk that the drawn place falls into, then the token: a work-group a sequence.
template <bool F32, bool ALIGNED>
static __global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyParams p) {
  constexpr int VEC = VerifyRow<F32>::VEC, FAR = 0x7fffffff;
  __shared__ double sh[kVerifyThreads / 64];
  __shared__ int sh_i[kVerifyThreads / 64];
  __shared__ double sh_before;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int lo = min(max(p.cu[b], 0), p.T), hi = min(max(p.cu[b + 1], lo), p.T), K = hi - lo - 1;
  if (K < 0) return;
  const int n = min(max(p.accepted[b], 0), K);
  VerifyRest<F32> rest = verify_rest<F32>(p, lo, K, n, p.first[b]);
  const double2* sums = p.sums + (long long)b * p.chunks;
  double total = 0, all = 0;
  for (int c = tid; c < p.chunks; c += kVerifyThreads) total += sums[c].x, all += sums[c].y;
  block_before(total, sh, total);
  block_before(all, sh, all);
  const bool whole = !(total > 0);      // nothing is left: the target's row
  if (whole) total = all, rest.less = false, rest.tok = -1;
  const double want = (double)p.u[lo + n] * total;
  double before = 0;
  int chunk = FAR, last = FAR;          // the first that passes it; the last that holds anything (counted from the end)
  for (int c0 = 0; c0 < p.chunks; c0 += kVerifyThreads) {
    const int c = c0 + tid;
    const double x = c < p.chunks ? (whole ? sums[c].y : sums[c].x) : 0.0;
    double sum, at = before + block_before(x, sh, sum);
    const int here = block_min(x > 0 && at + x > want ? c : FAR, sh_i);
    last = min(last, block_min(x > 0 ? p.chunks - 1 - c : FAR, sh_i));
    if (here != FAR) {
      chunk = here;
      if (c == here) sh_before = at;
      break;
    }
    before += sum;
  }
  long long token = -1;
  if (chunk != FAR || last != FAR) {
    const bool passes = chunk != FAR;   // else rounding kept the running sum below: the last token that counts
    if (!passes) chunk = p.chunks - 1 - last;
    __syncthreads();
    const double start = passes ? sh_before : 0.0;
    const int x0 = chunk * kVerifyChunk + tid * kVerifyRun;
    double r[kVerifyRun], mine = 0;
#pragma unroll
    for (int i = 0; i < kVerifyRun / VEC; ++i) {
      double a[VEC], c[VEC];
      rest.template some<ALIGNED>(a, c, x0 + i * VEC, p.V);
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[i * VEC + j] = a[j], mine += a[j];
    }
    double sum, at = start + block_before(mine, sh, sum);
    int here = FAR, end = FAR;
#pragma unroll
    for (int i = 0; i < kVerifyRun; ++i) {
      at += r[i];
      if (r[i] > 0) {
        if (passes && at > want) here = min(here, x0 + i);
        end = p.V - 1 - (x0 + i);
      }
    }
    here = block_min(here, sh_i), end = block_min(end, sh_i);
    token = here != FAR ? here : end != FAR ? p.V - 1 - end : -1;
  }
  for (int i = tid; i <= K; i += kVerifyThreads) p.tokens[lo + i] = i < n ? p.ids[lo + i + 1] : i == n ? token : -1;
}

}  // namespace fgrpo
