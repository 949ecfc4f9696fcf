// How the attention over a paged cache is dealt to work-groups (paged_rows.h, paged_tiles.h), computed by each of them from cu and lens,
// the lanes taking a sequence each: nothing is known on the host but the shapes, nothing is waited for, and a captured call follows new
// lengths.
//
// An item is a tile of ROWS rows of a sequence and K/V head with all its keys; items are in the order (sequence, head, tile).  Its weight
// is about its keys x G.  Shares: `used` work-groups take equal stretches of the sum of the weights, cut inside items where need be.
// Parts of an item leave fp32 sums in slots, which paged_merge_kernel adds up in the order of the keys (no atomics: bit-reproducible).
#pragma once
#include "paged_attn.h"

namespace fgrpo {

constexpr int kPagedMaxParts = 128;      // of an item: what the merge reads one behind the other

struct PagedSplit {
  int W;                 // work-groups of the launch, a multiple of 8
  int odd;               // only odd slots begin items
  float* part;           // [2 W][row blocks][32 x HD] sums of a part, as attn_store_partial leaves them
  float2* ml;            // [2 W][row blocks][32] maximum (in powers of two) and sum
  int4* rec;             // [2 W] for the slot of an item's first part: {sequence + 1, tile, head, parts (negative: its slots are neighbours)}; 0: none
};
// slot of part i of an item whose first is in `slot`.  Shares: work-group w has 2 w for an item that an earlier one began and 2 w + 1 for one
// that it begins and does not end.
__device__ __forceinline__ int paged_slot(int slot, int i, bool neighbours) { return neighbours ? slot + i : i ? slot - 1 + 2 * i : slot; }

// Weight of tile t (ROWS rows) of a sequence: whole numbers in doubles, exact below 2^53.
struct PagedWeight {
  double base, slope;      // w_t = base + slope (t + 1)
  int tiles, len, nq, q0;
  __device__ __forceinline__ double of(int t) const { return base + slope * (t + 1); }
  __device__ __forceinline__ double upto(int n) const { return base * n + slope * 0.5 * n * (n + 1.0); }      // tiles 0 .. n - 1
};
template <int ROWS>
__device__ __forceinline__ PagedWeight paged_weight(const PagedAttn& p, int b) {
  PagedWeight w;
  w.q0 = min(max(p.c.cu[b], 0), p.c.T);
  w.nq = min(max(p.c.cu[b + 1], w.q0), p.c.T) - w.q0;
  w.len = paged_len(p.c, b);
  w.tiles = (int)(((long long)w.nq * p.G + ROWS - 1) / ROWS);
  w.base = (double)(p.causal ? max(w.len - w.nq, 0) : w.len) * p.G + ROWS;
  w.slope = p.causal ? ROWS : 0;
  return w;
}
__device__ __forceinline__ double uniform(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
struct PagedTotal {
  double weight, most, items;      // of all items; the heaviest; how many
};
template <int ROWS>
__device__ __forceinline__ PagedTotal paged_total(const PagedAttn& p) {
  const int lane = threadIdx.x & 63;
  PagedTotal s{0, 1, 0};
  for (int b = lane; b < p.c.B; b += 64) {
    const PagedWeight w = paged_weight<ROWS>(p, b);
    if (w.tiles > 0) s.weight += w.upto(w.tiles) * p.c.Hkv, s.most = fmax(s.most, w.of(w.tiles - 1)), s.items += (double)w.tiles * p.c.Hkv;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1)
    s.weight += __shfl_xor(s.weight, d, 64), s.most = fmax(s.most, __shfl_xor(s.most, d, 64)), s.items += __shfl_xor(s.items, d, 64);
  return PagedTotal{uniform(s.weight), uniform(s.most), uniform(s.items)};
}

struct PagedItem {
  int b, head, t;          // b >= B: behind the last
  double at, index;        // weight and number of the items in front of it
};
// The item that holds place `x` of the weights, or of the numbers.
template <int ROWS, bool NUMBERS>
__device__ __forceinline__ PagedItem paged_item(const PagedAttn& p, double x) {
  const int lane = threadIdx.x & 63;
  PagedItem s{p.c.B, 0, 0, 0, 0};
  double weight = 0, number = 0;      // in front of the 64 at hand
  for (int b0 = 0; b0 < p.c.B; b0 += 64) {
    const int b = b0 + lane;
    double m = 0, n = 0;
    if (b < p.c.B) {
      const PagedWeight w = paged_weight<ROWS>(p, b);
      m = w.upto(w.tiles) * p.c.Hkv, n = (double)w.tiles * p.c.Hkv;
    }
    double upto_m = m, upto_n = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double y = __shfl_up(upto_m, d, 64), z = __shfl_up(upto_n, d, 64);
      if (lane >= d) upto_m += y, upto_n += z;
    }
    const unsigned long long past = __ballot((NUMBERS ? number + upto_n : weight + upto_m) > x);      // the first lane past it holds the sequence
    if (past) {
      const int l = __ffsll(past) - 1;
      s.b = b0 + l;
      s.at = weight + __shfl(upto_m - m, l, 64), s.index = number + __shfl(upto_n - n, l, 64);
      break;
    }
    weight += __shfl(upto_m, 63, 64), number += __shfl(upto_n, 63, 64);
  }
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  if (s.b >= p.c.B) return PagedItem{p.c.B, 0, 0, uniform(weight), uniform(number)};
  const PagedWeight w = paged_weight<ROWS>(p, s.b);
  const double one = NUMBERS ? (double)w.tiles : w.upto(w.tiles);      // of one head
  double r = x - (NUMBERS ? s.index : s.at);
  int head = (int)fmin(floor(r / one), p.c.Hkv - 1.0), t = 0;
  if (head > 0 && one * head > r) --head;
  if (head + 1 < p.c.Hkv && one * (head + 1) <= r) ++head;
  r -= one * head;
  if (NUMBERS) {
    t = (int)fmin(r, w.tiles - 1.0);
  } else {
    for (int low = 0, high = w.tiles - 1; low <= high;) {      // the last tile that begins at r or before
      const int mid = (low + high) / 2;
      if (w.upto(mid) <= r) t = mid, low = mid + 1;
      else high = mid - 1;
    }
  }
  s.head = __builtin_amdgcn_readfirstlane(head), s.t = __builtin_amdgcn_readfirstlane(t);
  s.at = uniform(s.at + w.upto(w.tiles) * s.head + w.upto(s.t)), s.index = uniform(s.index + (double)w.tiles * s.head + s.t);
  return s;
}
template <int ROWS>
__device__ __forceinline__ void paged_next(const PagedAttn& p, PagedItem& s, const PagedWeight& w) {
  s.at = uniform(s.at + w.of(s.t));
  if (++s.t < w.tiles) return;
  s.t = 0;
  if (++s.head < p.c.Hkv) return;
  s.head = 0;
  do ++s.b; while (s.b < p.c.B && paged_weight<ROWS>(p, s.b).tiles == 0);
  s.b = __builtin_amdgcn_readfirstlane(s.b);
}

// Shares: work-group `at` of `used` has the weights [bound(at), bound(at + 1)).
struct PagedShares {
  double total, used;
  __device__ __forceinline__ double bound(int at) const { return uniform(floor(total * at / used)); }
  __device__ __forceinline__ int holding(double x) const {      // the share that holds place x
    int w = (int)floor(x * used / total);
    while (w > 0 && bound(w) > x) --w;
    while (w + 1 < used && bound(w + 1) <= x) ++w;
    return __builtin_amdgcn_readfirstlane(w);
  }
};
__device__ __forceinline__ PagedShares paged_shares(const PagedTotal& t, int W, double least) {      // least: weight that is worth a work-group
  const double used = fmin(fmin((double)W, ceil(t.weight / least)), floor(t.weight * (kPagedMaxParts - 2) / t.most));
  return PagedShares{t.weight, uniform(fmax(used, 1.0))};
}
// what a work-group walks of an item, in steps of KB keys: places x0 .. x1 of its weight
struct PagedRange {
  int k0, k1;
};
template <int KB>
__device__ __forceinline__ PagedRange paged_range(double x0, double x1, double weight, int k_end) {
  const int steps = (k_end + KB - 1) / KB;
  const int s0 = __builtin_amdgcn_readfirstlane((int)floor(x0 * steps / weight)), s1 = __builtin_amdgcn_readfirstlane((int)floor(x1 * steps / weight));
  return PagedRange{s0 * KB, min(k_end, s1 * KB)};
}
// the keys that rows r0 .. r0 + n - 1 of a sequence see at all, and those that all of them see
struct PagedSight {
  int most, least;
};
__device__ __forceinline__ PagedSight paged_sight(const PagedAttn& p, const PagedWeight& w, int r0, int n) {
  if (!p.causal) return PagedSight{w.len, w.len};
  const int rows = w.nq * p.G, last = (min(r0 + n, rows) - 1) / p.G, first = r0 / p.G;
  return PagedSight{min(max(w.len - w.nq + last + 1, 0), w.len), min(max(w.len - w.nq + first + 1, 0), w.len)};
}
__device__ __forceinline__ int paged_table_at(const PagedView& c, int b, int i) {      // by the scalar unit: b and i are the same in all lanes.  As it stands: not yet held inside the cache
  const auto* row = (const __attribute__((address_space(4))) int*)(c.table + (long long)b * c.table_st);
  return row[min(i, c.width - 1)];
}
__device__ __forceinline__ float paged_lse(float m, float l) { return l > 0.f ? (m + __log2f(l)) * 0.6931471805599453f : -INFINITY; }

// Columns that a lane's accumulator values are.  Value r of block db: column 32 db + 8 (r / 4) + 4 h + r % 4.  PAIRS (the transposing reads moved
// pairs of e4m3 codes): blocks 2 n and 2 n + 1 hold the even and the odd columns of 64, value r is column
// 64 n + 2 (8 (r / 4) + 4 h + r % 4) + (block % 2), and the values of both blocks with r / 4 = g are eight neighbours.
template <int HD, bool PAIRS>
__device__ __forceinline__ void paged_store_row(const f32x16_t (&acc)[HD / 32], float mul, bf16_t* row, int h) {
  if constexpr (!PAIRS) {
    attn_store_rowmajor(acc, mul, row, h);
  } else {
#pragma unroll
    for (int n = 0; n < HD / 64; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x4_t x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = pack_bf16x2(acc[2 * n][4 * g + i] * mul, acc[2 * n + 1][4 * g + i] * mul);
        *(u32x4_t*)(row + 64 * n + 16 * g + 8 * h) = x;
      }
  }
}

// Adds up the parts of the item whose first is in slot blockIdx.x, in the order of the keys: work-group y takes 32 rows and NC / DB of their
// columns, a thread four columns of a row at a time.  RB: blocks of 32 rows of a tile.
template <int HD, bool PAIRS, int RB, int NC>
static __global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttn p, PagedSplit sp) {
  constexpr int DB = HD / 32, ROWS = 32 * RB, WIDE = 4;
  const int first = sp.odd ? 2 * blockIdx.x + 1 : blockIdx.x, lane = threadIdx.x & 63, h = lane >> 5, g = threadIdx.x >> 6;
  const int4 head = sp.rec[first];
  if (head.x == 0) return;
  const bool neighbours = head.w < 0;
  const int np = neighbours ? -head.w : head.w;
  const int b = min(max(head.x - 1, 0), p.c.B - 1), rb = blockIdx.y / (DB / NC), db0 = blockIdx.y % (DB / NC) * NC;
  const int q0 = min(max(p.c.cu[b], 0), p.c.T), nq = min(max(p.c.cu[b + 1], q0), p.c.T) - q0;
  const int row = head.y * ROWS + 32 * rb + (lane & 31);
  if (row >= nq * p.G) return;
  const int tok = q0 + row / p.G, hq = head.z * p.G + row % p.G;
  float m = -INFINITY, l = 0.f;
  float4 o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* part = sp.part + (long long)rb * (32 * HD) + (64 * (4 * db0 + g) + lane) * 4;
  const float2* ml = sp.ml + rb * 32 + (lane & 31);
  for (int i0 = 0; i0 < np; i0 += WIDE) {
    float2 x[WIDE];
    float4 y[WIDE][NC];
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      const long long slot = (long long)RB * min(paged_slot(first, min(i0 + i, np - 1), neighbours), 2 * sp.W - 1);
      x[i] = ml[slot * 32];
#pragma unroll
      for (int c = 0; c < NC; ++c) y[i][c] = *(const float4*)(part + slot * (32 * HD) + 1024 * c);
    }
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      if (i0 + i >= np) break;
      const float m_new = fmaxf(m, x[i].x), m_use = m_new == -INFINITY ? 0.f : m_new, a = fast_exp2(m - m_use), e = fast_exp2(x[i].x - m_use);
      l = l * a + x[i].y * e;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        o[c] = make_float4(o[c].x * a + y[i][c].x * e, o[c].y * a + y[i][c].y * e, o[c].z * a + y[i][c].z * e, o[c].w * a + y[i][c].w * e);
      m = m_new;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  bf16_t* dst = p.out + ((long long)tok * p.Hq + hq) * HD;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int db = db0 + c;
    if constexpr (PAIRS) {
      const int col = 64 * (db / 2) + 2 * (8 * g + 4 * h) + db % 2;
      dst[col] = f32_to_bf16_rn(o[c].x * inv), dst[col + 2] = f32_to_bf16_rn(o[c].y * inv), dst[col + 4] = f32_to_bf16_rn(o[c].z * inv), dst[col + 6] = f32_to_bf16_rn(o[c].w * inv);
    } else {
      uint2 x;
      x.x = pack_bf16x2(o[c].x * inv, o[c].y * inv), x.y = pack_bf16x2(o[c].z * inv, o[c].w * inv);
      *(uint2*)(dst + 32 * db + 8 * g + 4 * h) = x;
    }
  }
  if (p.lse && db0 == 0 && g == 0 && h == 0) p.lse[(long long)hq * p.c.T + tok] = paged_lse(m, l);
}

}  // namespace fgrpo
