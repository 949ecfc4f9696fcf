// Attention of new tokens over a paged cache (paged_cache.h): token i of the q_b new ones of sequence b sees the keys
// j < k_b, and with the causal mask j <= k_b - q_b + i.  o = softmax(c q K^T) V over what it sees; nothing seen: o = 0, lse = -inf.
//
// The G query heads of a K/V head read the same keys, so rows are (token, head of the group) pairs, row r of a sequence being token
// r / G, head r mod G: tiles of rows are full whatever G is.  A wavefront has 32 rows (paged_tiles.h) or 16 and 32 (paged_rows.h) and
// computes S^T = K Q^T and O^T = V^T P^T with the matrix instruction's operands as the packed attention has them (attn_kernels.h): a lane owns one
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

}  // namespace fgrpo
