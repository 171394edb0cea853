// ascan_attend.cuh -- causal softmax attention over packed sequences: what its
// kernels share.
//
//   s[i,j] = scale q[i].k[j]  (j <= i, same sequence)     p = softmax over j
//   o[i]   = sum_j p[i,j] v[j]
//
// The softmax is taken in one pass over the keys, in units of log 2 and
// against a running reference m: l = sum 2^(s - m), o = sum 2^(s - m) v, both
// scaled down when m grows.  What the gradients need of a row is
// lse[i] = m + log2 l, so that p[i,j] = 2^(s[i,j] - lse[i]) without another
// pass, and d[i] = do[i].o[i]:
//
//   ds[i,j] = p[i,j] (do[i].v[j] - d[i])
//   dq[i] = scale sum_j ds[i,j] k[j]   dk[j] = scale sum_i ds[i,j] q[i]
//   dv[j] = sum_i p[i,j] do[i]
//
// Where p is close to 1, do.v - d is a difference of nearly equal numbers: d
// takes o with 16 bits or more (a 16-bit o and what its rounding left over),
// for with o's own 8 a sharp row's ds would be rounding alone.
//
// dq is summed by one kernel (a CTA holds query rows and walks the keys) and
// dk, dv by another (a CTA holds key rows and walks the queries of every head
// that shares them), so every sum has one owner and a fixed order, and results
// repeat bit for bit.  A single kernel would save two of seven products and
// pay with atomics.
//
// Tiles start at their sequence's start, so a tile holds tokens of one
// sequence; rows past its end belong to another and are replaced by zeros
// before they meet a product, for 0 * NaN would let one sequence's values into
// another.  A value that is not finite behind the causal mask is kept out of
// the earlier rows in the same way.
#pragma once

#include "ascan_mscan.cuh"

namespace ascan {
namespace attend {

using mscan::allow_smem;
using mscan::from_f;
using mscan::Rows;
using mscan::to_f;

constexpr float kLog2e = 1.4426950408889634f;

struct Problem {
  Rows q, k, v, d_out;  // d_out: gradients only
  const void* cu;
  int cu64, H, share, dk, dv;  // query heads; query heads of a key head
  long long N, BL;
  float scale;
  void* out;              // [BL, H, dv]; the forward's, also in the gradients
  void* rest;             // what its rounding left over (16-bit types; may be null)
  float* lse;             // [H, BL], log2; may be null in the forward
  float* d;               // [H, BL]: do.o (gradients)
  uint32_t* top;          // float16 gradients on the tensor cores: bits of the largest finite |do| and |v|, else null
  void *d_q, *d_k, *d_v;  // contiguous
  uint32_t* err;
};

__device__ __forceinline__ long long cu_at(const Problem& p, long long i) {
  const long long v = p.cu64 ? static_cast<const long long*>(p.cu)[i]
                             : static_cast<long long>(static_cast<const int*>(p.cu)[i]);
  return v < 0 ? 0 : (v > p.BL ? p.BL : v);
}

// Tiles of `rows` tokens, at most cu[n] / rows + n before sequence n's first:
// as many numbers as BL / rows + N, some without a tile.
inline long long tile_bound(const Problem& p, int rows) { return p.BL / rows + p.N; }

struct Tile {
  int start, len;  // the sequence's
  int first;       // the tile's first token in it; -1: no tile
};

// Numbers below 2^30 and tiles of 2^SHIFT rows: a search costs a load and a few
// instructions a step, in front of everything else that a CTA does.
__device__ __forceinline__ Tile tile_of(int start, int end, int sequence, int x, int shift) {
  Tile t;
  t.start = start;
  t.len = end - start;
  t.first = (x - (start >> shift) - sequence) * (1 << shift);
  if (t.first < 0 || t.first >= t.len) t.first = -1;
  return t;
}
template <int SHIFT, typename F>
__device__ __forceinline__ Tile find_tile(const Problem& p, int x, F at) {
  int lo = 0, hi = static_cast<int>(p.N) - 1;  // the last sequence whose tiles start at or before x
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((at(mid) >> SHIFT) + mid <= x) lo = mid;
    else hi = mid - 1;
  }
  return tile_of(at(lo), at(lo + 1), lo, x, SHIFT);
}
template <int SHIFT>
__device__ __forceinline__ Tile find_tile(const Problem& p, int x) {
  return find_tile<SHIFT>(p, x, [&](int i) { return static_cast<int>(cu_at(p, i)); });
}

// The same by a warp, thirty-two sequences a step: one trip to memory where a
// search by halves takes one for each doubling of their number.
template <int SHIFT>
__device__ __forceinline__ Tile find_tile_warp(const Problem& p, int x) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = static_cast<int>(p.N);
  while (n > 1) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const bool in = lane * step < n && (static_cast<int>(cu_at(p, i)) >> SHIFT) + i <= x;
    // starts do not fall, so the lanes that are in are the first ones
    const int ahead = max(__popc(__ballot_sync(0xffffffffu, in)), 1) - 1;
    lo += ahead * step;
    n = min(step, n - ahead * step);
  }
  return tile_of(static_cast<int>(cu_at(p, lo)), static_cast<int>(cu_at(p, lo + 1)), lo, x, SHIFT);
}

// Rows of no sequence come out zero; slab x of the packed axis is the x-th CTA's.
template <typename T>
__device__ __forceinline__ void zero_outside(const Problem& p, void* to, int head, int heads, int dim, long long x, int rows,
                                             int thread, int threads) {
  const long long t0 = x * rows, t1 = min(t0 + rows, p.BL);
  const long long c0 = cu_at(p, 0), c1 = cu_at(p, p.N);
  if (t0 >= c0 && t1 <= c1) return;
  for (long long t = t0; t < t1; ++t)
    if (t < c0 || t >= c1)
      for (int d = thread; d < dim; d += threads) static_cast<T*>(to)[(t * heads + head) * dim + d] = from_f<T>(0.f);
}

// The tensor-core kernels (ascan_attend_tc.cu).
bool tc_usable(const Problem& p, int dtype, bool backward);
int tc_forward(const Problem& p, int dtype, cudaStream_t s);
int tc_backward(const Problem& p, int dtype, cudaStream_t s);

}  // namespace attend
}  // namespace ascan
