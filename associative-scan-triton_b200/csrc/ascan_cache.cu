// ascan_cache.cu -- compilation unit of the scan library: a paged cache of keys
// and values in 8 bits, and the attention of single tokens that reads it.
//
// A page holds `page` tokens of every key head, [heads, page, dim] in e4m3,
// with one float32 scale for each head: x = scale * e.  Scales are powers of
// two, 2^-64 to 2^64.  e4m3 is a floating-point format, so a finer scale would
// not make its steps finer, and powers of two cost nothing where it matters:
// x / scale and scale * e are exact, so a written value is rounded once; when a
// later token is larger than the page's scale reaches, what the page holds
// moves to the larger scale without another rounding (but for values below
// 2^-6 of the scale, whose steps are fixed); and in a product the scale is an
// addition to the exponent.
#include "ascan_impl.cuh"
#include "ascan_mscan.cuh"
#include "ascan_tc.cuh"

namespace ascan {
namespace cache {

using namespace tc;

using mscan::from_f;
using mscan::Rows;
using mscan::to_f;

constexpr int kScaleBits = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct Cache {
  uint8_t *k, *v;  // [pages, heads, page, dim]
  float *ks, *vs;  // [pages, heads]
  long long pages;
  int heads, page, dk, dv;
  const int* table;  // [B, width]
  long long B, width;
};

__device__ __forceinline__ long long index_at(const void* p, int is64, long long i) {
  return is64 ? static_cast<const long long*>(p)[i] : static_cast<long long>(static_cast<const int*>(p)[i]);
}

// Sixteen rows of a page from row `row`.
__device__ __forceinline__ void tma_page(uint32_t to, const CUtensorMap* m, int row, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to),
      "l"(m), "r"(0), "r"(row), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

// All lanes; false when the copies did not come within the limit.
__device__ __noinline__ bool wait_slow(uint64_t* b, uint32_t parity, uint32_t* err) {
  const unsigned long long start = now_ns();
  while (!bar_try(b, parity))
    if (now_ns() - start > kStageTimeoutNs) {
      report(ASCAN_DEV_ERR_STAGE, (static_cast<unsigned long long>(blockIdx.x) << 32) | threadIdx.x, err);
      return false;
    }
  return true;
}
__device__ __forceinline__ bool wait_group(uint64_t* b, uint32_t parity, uint32_t* err) {
  return __all_sync(kFull, bar_try(b, parity) || wait_slow(b, parity, err));
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// ---------------------------------------------------------------------------
// new tokens into their pages
// ---------------------------------------------------------------------------

struct WriteArgs {
  Cache c;
  Rows x[2];  // keys, values
  const void *starts, *cu;
  int starts64, cu64;
  long long BL, units;
  uint32_t* err;
};

// The smallest power of two that brings `top` to at most 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_bits(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = static_cast<int>(b >> 23) - 127 - ((b & 0x7fffffu) > 0x600000u ? 7 : 8);
  return max(-kScaleBits, min(kScaleBits, e));
}

// Four values to e4m3, to nearest; NaN becomes its NaN, what lies beyond the
// scale's reach (infinities too) its largest value.
__device__ __forceinline__ uint32_t pack4(const float* y) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[1]), "f"(y[0]));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[3]), "f"(y[2]));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

__device__ __forceinline__ uint32_t half2_of(uint16_t e) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(e));
  return r;
}

__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  const uint32_t a = half2_of(static_cast<uint16_t>(w)), b = half2_of(static_cast<uint16_t>(w >> 16));
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  const float v[4] = {x.x * f, x.y * f, y.x * f, y.y * f};
  return pack4(v);
}

// Eight elements as they lie in memory, and as floats.
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];

  __device__ __forceinline__ void load(const T* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    } else {
      T* e = reinterpret_cast<T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f(reinterpret_cast<const T*>(w)[i]); }
  // The largest magnitude, infinities included, NaN not.
  __device__ __forceinline__ float largest() const {
    if (sizeof(T) == 4) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf((*this)[i]));
      return m;
    }
    const uint32_t e[4] = {w[0].x & 0x7fff7fffu, w[0].y & 0x7fff7fffu, w[0].z & 0x7fff7fffu, w[0].w & 0x7fff7fffu};
    using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    auto as = [&](int i) { return *reinterpret_cast<const Pair*>(&e[i]); };
    const Pair m = __hmax2(__hmax2(as(0), as(1)), __hmax2(as(2), as(3)));
    const float x = to_f(m.x), y = to_f(m.y);
    return fmaxf(x == x ? x : 0.f, y == y ? y : 0.f);
  }
};

// A group of G threads writes what one request adds to one page of one head:
// the largest magnitude first, which gives the scale, then the rounded values.
// Up to HOLD vectors of eight elements a thread stay in registers in between
// (16-bit: a page of 64 tokens of 128 in all); of longer pieces the rest is read
// again.  More in registers would leave room for fewer groups an SM, and it is
// their number that hides the reads in front.
// Memory and the chain of dependent reads in front of it (request, page, scale)
// bound it: 16384 tokens of 4 heads of 128 take 19.8 us (2.5 TB/s), and took 27
// with every vector read twice, one after the other; eight vectors held, at 80
// registers, 32 us.
template <typename T, int G>
__global__ void __launch_bounds__(kThreads, 5) write_kernel(const __grid_constant__ WriteArgs a, int vec_k, int vec_v) {
  constexpr int UNITS = kThreads / G;
  constexpr int HOLD = sizeof(T) == 4 ? 2 : (G == 32 ? 2 : 4);
  const Cache& c = a.c;
  const int gl = threadIdx.x % G, sub = threadIdx.x / G, lane = threadIdx.x & 31;
  if (blockIdx.x == 0) {
    if (a.cu64) validate_cu(static_cast<const int64_t*>(a.cu), c.B, a.BL, a.err);
    else validate_cu(static_cast<const int32_t*>(a.cu), c.B, a.BL, a.err);
  }
  const long long unit = static_cast<long long>(blockIdx.x) * UNITS + sub;
  if (unit >= a.units) return;  // whole groups
  const int half = static_cast<int>(unit) & 1, h = static_cast<int>(unit >> 1) % c.heads;
  const int x = static_cast<int>(unit >> 1) / c.heads;  // piece number
  auto cu_at = [&](int i) {
    const long long v = index_at(a.cu, a.cu64, i);
    return static_cast<int>(v < 0 ? 0ll : (v > a.BL ? a.BL : v));
  };
  // pieces of request b start at cu[b] / page + 2 b: no more than its tokens
  // fill and two that they begin and end in.  A warp looks at thirty-two
  // requests at once.
  int b = 0;
  for (int n = static_cast<int>(c.B); n > 1;) {
    const int step = (n + 31) / 32, i = b + lane * step;
    const bool in = lane * step < n && cu_at(i) / c.page + 2 * i <= x;
    const int ahead = max(__popc(__ballot_sync(kFull, in)), 1) - 1;
    b += ahead * step;
    n = min(step, n - ahead * step);
  }
  const int c0 = cu_at(b), len = cu_at(b + 1) - c0;
  const long long begin = index_at(a.starts, a.starts64, b);
  if (begin < 0 || len <= 0) return;  // no request, or nothing new
  int id = -1, place = 0, from = 0, to = 0;
  if (begin < 0x3fff0000) {  // what follows stays below 2^31
    const int start = static_cast<int>(begin);
    place = start / c.page + (x - c0 / c.page - 2 * b);
    from = max(start, place * c.page), to = min(start + len, (place + 1) * c.page);
    if (place < 0 || from >= to) return;
    if (place < c.width) id = c.table[b * c.width + place];
  }
  if (id < 0 || id >= c.pages) {
    if (gl == 0) report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(b), a.err);
    return;
  }
  const bool is_v = half != 0;
  const int dim = is_v ? c.dv : c.dk, first = from - place * c.page, n = to - from;
  const bool vec = is_v ? vec_v : vec_k;
  const Rows& r = a.x[is_v];
  const T* src = static_cast<const T*>(r.p) + (c0 + from - static_cast<long long>(begin)) * r.st + h * r.sh;
  uint8_t* dst = (is_v ? c.v : c.k) + ((static_cast<long long>(id) * c.heads + h) * c.page + first) * dim;
  float* scale = (is_v ? c.vs : c.ks) + static_cast<long long>(id) * c.heads + h;
  const float held = first > 0 ? *scale : 0.f;
  const int per_row = dim / 8, work = n * per_row;
  // vector gl + G k of the piece is vector `col` of row `row`
  const int step_row = G / per_row, step_col = G % per_row;
  auto advance = [&](int& row, int& col) {
    row += step_row, col += step_col;
    if (col >= per_row) col -= per_row, ++row;
  };
  const int row0 = gl / per_row, col0 = gl % per_row;
  Eight<T> kept[HOLD];
  int row = row0, col = col0;
#pragma unroll
  for (int k = 0; k < HOLD; ++k) {
    if (gl + G * k < work) kept[k].load(src + row * r.st + col * 8, vec);
    advance(row, col);
  }
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < HOLD; ++k)
    if (gl + G * k < work) top = fmaxf(top, kept[k].largest());
  for (int e = gl + G * HOLD; e < work; e += G) {
    Eight<T> v;
    v.load(src + row * r.st + col * 8, vec);
    top = fmaxf(top, v.largest());
    advance(row, col);
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  if (G > 32) {
    __shared__ float tops[G / 32];
    if (lane == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();  // everyone has read the scale too
#pragma unroll
    for (int w = 0; w < G / 32; ++w) top = fmaxf(top, tops[w]);
  } else {
    __syncwarp();
  }
  const bool infinite = top == INFINITY;
  if (infinite) {  // the largest that is not, by every warp of the group alike
    top = 0.f;
    for (int e = lane; e < work; e += 32) {
      Eight<T> v;
      v.load(src + e / per_row * r.st + e % per_row * 8, vec);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (fabsf(v[q]) < INFINITY) top = fmaxf(top, fabsf(v[q]));
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  }
  const float need = fmaxf(pow2(scale_bits(top)), held);
  if (first > 0 && need > held) {  // what the page holds moves to the larger scale
    const float f = held / need;
    uint4* old = reinterpret_cast<uint4*>(dst - first * dim);
    for (int e = gl; e < first * dim / 16; e += G) {
      uint4 w = old[e];
      w.x = rescale4(w.x, f), w.y = rescale4(w.y, f), w.z = rescale4(w.z, f), w.w = rescale4(w.w, f);
      old[e] = w;
    }
  }
  if (gl == 0 && need != held) *scale = need;
  const float inv = 1.f / need;
  auto put = [&](const Eight<T>& v, int e) {
    float y[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) y[q] = v[q] * inv;
    if (infinite) {
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] = fabsf(y[q]) < INFINITY ? y[q] : NAN;
    }
    reinterpret_cast<uint2*>(dst)[e] = make_uint2(pack4(y), pack4(y + 4));
  };
#pragma unroll
  for (int k = 0; k < HOLD; ++k)
    if (gl + G * k < work) put(kept[k], gl + G * k);
  row = row0, col = col0;
  for (int k = 0; k < HOLD; ++k) advance(row, col);
  for (int e = gl + G * HOLD; e < work; e += G) {
    Eight<T> v;
    v.load(src + row * r.st + col * 8, vec);
    put(v, e);
    advance(row, col);
  }
}

// ---------------------------------------------------------------------------
// attention of single tokens
// ---------------------------------------------------------------------------

constexpr int kStepWarps = 4;                          // that compute; a fifth loads
constexpr int kStepThreads = (kStepWarps + 1) * 32;
constexpr int kGroup = 16;                             // tokens of a warp at a time
constexpr int kStepTile = kStepWarps * kGroup;
constexpr int kCtasPerSm = 3;
constexpr int kMaxCtas = 148 * kCtasPerSm;

struct StepArgs {
  Cache c;
  Rows q;
  const void* lengths;
  int lengths64, H, share, row_tiles;  // sixteen query heads of a key head are a row tile
  float scale;
  void* out;
  float* part;        // per CTA two slots of [16] references, [16] sums, [16][dv] rows
  long long* before;  // [B + 1]: tiles of all requests before each
  uint32_t* err;
};

struct StepMaps {
  CUtensorMap k, v;
};

__device__ __forceinline__ int slot_floats(int dv) { return 32 + 16 * dv; }

// Tokens of request b; what does not fit its row of pages is left out.
__device__ __forceinline__ int length_of(const StepArgs& a, long long b) {
  const long long n = index_at(a.lengths, a.lengths64, b), room = min(a.c.width * a.c.page, static_cast<long long>(ASCAN_ATTENTION_MAX_TOKENS));
  if (n > room && blockIdx.x == 0) report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(b), a.err);
  return static_cast<int>(n < 0 ? 0 : min(n, room));
}
__device__ __forceinline__ int tiles_of_length(int n) { return (n + kStepTile - 1) / kStepTile; }

__device__ __forceinline__ void mma(float* d, const uint32_t* a, const uint32_t* b) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// An 8 x 8 matrix of 16-bit elements, a row for four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float2 float2_of(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(kFull, x, 1));
  return fmaxf(x, __shfl_xor_sync(kFull, x, 2));
}
// Over the lanes that differ in lane / 4.
__device__ __forceinline__ float column_max(float x) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) x = fmaxf(x, __shfl_xor_sync(kFull, x, o));
  return x;
}
__device__ __forceinline__ float column_sum(float x) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) x += __shfl_xor_sync(kFull, x, o);
  return x;
}

// Tiles of the requests: their total, and the request that tile `begin` of the
// list lies in, with the tiles before it; the first CTA writes the sums down
// for the launch that joins.  All threads of the block.
struct Found {
  long long total, before;
  int b;
};
__device__ __forceinline__ Found find_request(const StepArgs& a, int groups, long long (&scratch)[kStepWarps + 2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Found f{0, 0, 0};
  long long begin = 0;
  for (int pass = 0; pass < 2; ++pass) {  // the total, then the place
    long long sum = 0;
    for (long long b0 = 0; b0 < a.c.B; b0 += kStepThreads) {
      const long long b = b0 + threadIdx.x;
      const long long n = b < a.c.B ? tiles_of_length(length_of(a, b)) : 0;
      long long inc = n;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const long long x = __shfl_up_sync(kFull, inc, o);
        if (lane >= o) inc += x;
      }
      __syncthreads();
      if (lane == 31) scratch[warp] = inc;
      __syncthreads();
      long long front = sum;
      for (int w = 0; w <= kStepWarps; ++w) {
        if (w < warp) front += scratch[w];
        sum += scratch[w];
      }
      inc += front;
      if (pass == 0) {
        if (blockIdx.x == 0 && b < a.c.B) {
          if (b == 0) a.before[0] = 0;
          a.before[b + 1] = inc;
        }
      } else if (begin >= (inc - n) * groups && begin < inc * groups) {
        scratch[kStepWarps + 1] = b;  // one thread's
      }
      if (pass == 1 && begin < sum * groups) {
        __syncthreads();
        f.b = static_cast<int>(scratch[kStepWarps + 1]);
        break;
      }
    }
    if (pass == 0) {
      f.total = sum * groups;
      begin = f.total / gridDim.x * blockIdx.x + min(f.total % gridDim.x, static_cast<long long>(blockIdx.x));
      if (begin >= f.total) return f;
    }
  }
  // the tiles before it, from the lengths again
  long long n = 0;
  for (int b = threadIdx.x; b < f.b; b += kStepThreads) n += tiles_of_length(length_of(a, b));
#pragma unroll
  for (int o = 16; o > 0; o /= 2) n += __shfl_xor_sync(kFull, n, o);
  __syncthreads();
  if (lane == 0) scratch[warp] = n;
  __syncthreads();
  for (int w = 0; w <= kStepWarps; ++w) f.before += scratch[w] * groups;
  return f;
}

// A place in the list of tiles: request by request, key head and row tile by
// row tile, and what the warp has of the tile.
struct Place {
  int b, group, tile, tiles, len;
  int page, row;  // of the request's pages, and in it, where the warp's tokens begin

  __device__ __forceinline__ void enter(const StepArgs& a, int warp) {
    const int t0 = tile * kStepTile + warp * kGroup;
    page = t0 / a.c.page;
    row = t0 - page * a.c.page;
  }
  __device__ __forceinline__ void request(const StepArgs& a) {
    len = length_of(a, b);
    tiles = tiles_of_length(len);
  }
  __device__ __forceinline__ bool has(int warp) const { return tile * kStepTile + warp * kGroup < len; }
  // There is a next one.
  __device__ __forceinline__ void next(const StepArgs& a, int warp, int groups) {
    if (++tile < tiles) {
      row += kStepTile;
      while (row >= a.c.page) row -= a.c.page, ++page;
      return;
    }
    tile = 0;
    if (++group == groups) {
      group = 0;
      do {
        ++b;
        request(a);
      } while (tiles == 0);
    }
    enter(a, warp);
  }
};

__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, %0;" ::"n"(kStepWarps * 32) : "memory"); }

// Groups in flight for each warp: what three CTAs of an SM have room for.
__host__ __device__ constexpr int stages(int r) { return r == 1 ? 4 : 3; }

// The tiles of all requests, key heads and row tiles are one list; a CTA takes
// an equal run of it, wherever requests begin and end, and walks it piece by
// piece (a piece: what it has of one request, head and row tile).  Each of four
// warps takes sixteen tokens of a tile with m16n8k16 products of float16, the
// tokens and the values' elements along the 16 and queries along the 8, which
// a key head often has no more of:
//
//   S^T = K q^T [tokens, queries]     O^T += V^T P^T [elements, queries]
//
// e4m3 values are exact in float16, queries are brought to at most 2^15 by a
// power of two each, and weights lie between 0 and 2^8, so both keep 11 bits or
// more (22 where queries are float32: the rest of each goes through a second
// product).  A lane's column of S^T and of O^T is the same query, and the
// softmax's reference moves only when a score exceeds it by 2^8, so nothing is
// exchanged between lanes but P, for its transposition.
//
// Memory bounds it, so each warp has several groups of sixteen tokens in
// flight, over the ends of pieces too: 2 KB of keys and of values, each one TMA
// copy into its own slots, and their scales behind the same barrier.  A fifth
// warp asks for them, a lane for each of the four (when each warp asked for its
// own, 600 instructions went into a group, and 128 requests of 4000 tokens took
// 163 us).  From shared memory the operands come sixteen bytes a load: which
// elements and tokens stand for which index of a product is free as long as
// both operands agree, and the choice here together with the copies' swizzle
// meets no bank twice.
//
// Measured, 16 query heads on 4 of keys, 128 wide, bfloat16 queries: 128 ragged
// requests of 4000 tokens on average (525 MB) 101 to 111 us, 4.7 to 5.2 TB/s, and one
// of 131072 (134 MB) 36 us with its join, 3.7 TB/s, of which memory needs 20;
// the start, the last wait and the join of a CTA's eighteen tiles are the rest.
// Half of the issue slots are busy.
//
// U: 64-element parts of a key.  NV: bytes of a value row per lane.  R: queries
// in eights (one if no key head has more than eight).
template <typename T, int U, int NV, int R>
__global__ void __launch_bounds__(kStepThreads, sizeof(T) == 4 ? 2 : kCtasPerSm)
    step_kernel(const __grid_constant__ StepArgs a, const __grid_constant__ StepMaps maps) {
  constexpr bool FINE = sizeof(T) == 4;
  constexpr int TERMS = FINE ? 2 : 1, S = stages(R);
  constexpr int KB = kGroup * 64 * U, VB = kGroup * 8 * NV;  // bytes of a group
  extern __shared__ __align__(1024) unsigned char ring[];     // [warp][stage][keys, values]
  __shared__ uint64_t full[kStepWarps][S], empty[kStepWarps][S];
  __shared__ float scales[kStepWarps][S][2];
  __shared__ int usable[kStepWarps][S];
  __shared__ long long scratch[kStepWarps + 2];
  __shared__ float s_m[kStepWarps][8 * R], s_l[kStepWarps][8 * R];
  __shared__ float s_o[2][8 * R][NV * 8 + 4];
  const Cache& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int groups = c.heads * a.row_tiles;  // of a request

  if (smem_u32(ring) & 1023u) {  // the swizzled layouts need it
    if (threadIdx.x == 0) report(ASCAN_DEV_ERR_STAGE, 0xffffffffull, a.err);
    return;
  }
  if (threadIdx.x < kStepWarps) {
    for (int i = 0; i < S; ++i) bar_init(&full[lane][i], 2), bar_init(&empty[lane][i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Found f = find_request(a, groups, scratch);  // and all threads have met
  const long long run = f.total / gridDim.x, more = f.total % gridDim.x;
  const long long begin = run * blockIdx.x + min(more, static_cast<long long>(blockIdx.x));
  const long long end = begin + run + (blockIdx.x < more);
  // requests without tokens, dealt to all CTAs
  for (long long b = blockIdx.x; b < c.B; b += gridDim.x)
    if (length_of(a, b) == 0)
      for (int e = threadIdx.x; e < a.H * c.dv; e += kStepThreads) static_cast<T*>(a.out)[b * a.H * c.dv + e] = from_f<T>(0.f);
  if (begin >= end) return;

  const int mine = warp < kStepWarps ? warp : lane;  // the warp that computes
  Place use;
  use.b = f.b;
  use.request(a);
  use.group = static_cast<int>((begin - f.before) / use.tiles);
  use.tile = static_cast<int>((begin - f.before) % use.tiles);
  use.enter(a, mine);

  if (warp == kStepWarps) {
    // ---- loads: lane w for warp w ----
    if (lane >= kStepWarps) return;
    unsigned char* slots = ring + mine * S * (KB + VB);
    int at = 0, phase = 1;  // a first pass finds all slots empty
#pragma unroll 1
    for (long long left = end - begin; left > 0; --left) {
      if (use.has(mine)) {
        const int id = __ldg(c.table + use.b * c.width + use.page), hk = use.group / a.row_tiles;
        uint64_t* bar = &full[mine][at];
        if (!bar_try(&empty[mine][at], phase) && !wait_slow(&empty[mine][at], phase, a.err)) return;
        if (id < 0 || id >= c.pages) {
          report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(use.b), a.err);
          usable[mine][at] = 0;
          bar_arrive(bar);
          bar_arrive(bar);
        } else {
          const int page = id * c.heads + hk;
          const uint32_t to = smem_u32(slots + at * (KB + VB));
          usable[mine][at] = 1;
          bar_expect(bar, KB + VB);
          tma_page(to, &maps.k, use.row, page, bar);
          tma_page(to + KB, &maps.v, use.row, page, bar);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&scales[mine][at][0])), "l"(c.ks + page) : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&scales[mine][at][1])), "l"(c.vs + page) : "memory");
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
        }
        if (++at == S) at = 0, phase ^= 1;
      }
      if (left > 1) use.next(a, mine, groups);
    }
    return;
  }

  const float c2 = a.scale * kLog2e;
  const unsigned char* slots = ring + warp * S * (KB + VB);
  int slot = 0, stage = 0, phase = 0;
  bool alive = true;
#pragma unroll 1
  for (long long at = begin; at < end; ) {
    const int tile0 = use.tile, tile1 = static_cast<int>(min(static_cast<long long>(use.tiles), tile0 + (end - at)));
    const int hk = use.group / a.row_tiles, h0 = hk * a.share + use.group % a.row_tiles * 16;
    const int rows = min(16, (hk + 1) * a.share - h0);

    // ---- queries as operands: index 2 t4.. of product (u, w) is element
    // 16 (U t4 + u) + 4 w.. of the head; lane / 4 is the query here, and of
    // products its columns are queries 2 t4 and 2 t4 + 1
    uint32_t q[TERMS][R][U * 4][2];
    float qf[R][2];  // what a query's scores are in units of
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = g + 8 * r;
      float x[U * 16], top = 0.f;
#pragma unroll
      for (int e = 0; e < U * 16; ++e) {
        const int d = 16 * U * t4 + e;
        x[e] = row < rows && d < c.dk ? to_f(static_cast<const T*>(a.q.p)[use.b * a.q.st + (h0 + row) * a.q.sh + d]) : 0.f;
        top = fmaxf(top, fabsf(x[e]));
      }
      top = quad_max(top);
      const int e2 = max(-100, static_cast<int>(__float_as_uint(top) >> 23) - 127);
      const float up = pow2(14 - e2), unit = pow2(e2 - 14) * c2;
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[r][e] = __shfl_sync(kFull, unit, (2 * t4 + e) * 4);
#pragma unroll
      for (int u = 0; u < U * 4; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float y0 = x[u * 4 + half * 2] * up, y1 = x[u * 4 + half * 2 + 1] * up;
          const uint32_t hi = hf2(y0, y1);
          q[0][r][u][half] = hi;
          if (FINE) {
            const float2 z = float2_of(hi);
            q[TERMS - 1][r][u][half] = hf2(y0 - z.x, y1 - z.y);
          }
        }
    }

    float o[R][NV / 2][4], m[R][2], l[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r][0] = m[r][1] = -INFINITY;
      l[r][0] = l[r][1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) o[r][i][0] = o[r][i][1] = o[r][i][2] = o[r][i][3] = 0.f;
    }

#pragma unroll 1
    for (int tile = tile0; tile < tile1; ++tile) {
      const int tokens = use.len - (tile * kStepTile + warp * kGroup);  // sixteen of them at most are the warp's
      if (tokens <= 0) break;
      if (alive) alive = wait_group(&full[warp][stage], phase, a.err);
      const unsigned char* ks = slots + stage * (KB + VB);
      const unsigned char* vs = ks + KB;
      if (alive && usable[warp][stage]) {
        const float kscale = scales[warp][stage][0], vscale = scales[warp][stage][1];
        // element e of s: token g + 8 (e / 2), query 2 t4 + e % 2
        float s[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          uint32_t word[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = 8 * i + g;
            const uint4 x = *reinterpret_cast<const uint4*>(
                ks + row * 64 * U + (U == 2 ? ((2 * t4 + u) ^ (row & 7)) << 4 : (t4 ^ ((row >> 1) & 3)) << 4));
            word[i][0] = x.x, word[i][1] = x.y, word[i][2] = x.z, word[i][3] = x.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t ka[4] = {half2_of(static_cast<uint16_t>(word[0][e])), half2_of(static_cast<uint16_t>(word[1][e])),
                                    half2_of(static_cast<uint16_t>(word[0][e] >> 16)), half2_of(static_cast<uint16_t>(word[1][e] >> 16))};
#pragma unroll
            for (int z = 0; z < TERMS; ++z)
#pragma unroll
              for (int r = 0; r < R; ++r) mma(s[r], ka, q[TERMS - 1 - z][r][u * 4 + e]);
          }
        }
        // in units of log 2; a page's value scale is added to the exponent
        const float lv = static_cast<float>(static_cast<int>(__float_as_uint(vscale) >> 23) - 127);
        bool past = false;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[r][e] *= qf[r][e & 1] * kscale;
            if (g + 8 * (e >> 1) >= tokens) s[r][e] = -INFINITY;
            past |= s[r][e] + lv > m[r][e & 1] + 8.f;
          }
        // the reference moves when weights would pass 2^8
        if (__any_sync(kFull, past)) {
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float next = fmaxf(m[r][e], column_max(fmaxf(s[r][e], s[r][e + 2])) + lv);
              const float fall = next == -INFINITY ? 1.f : ex2(m[r][e] - next);
              m[r][e] = next;
              l[r][e] *= fall;
#pragma unroll
              for (int i = 0; i < NV / 2; ++i) o[r][i][e] *= fall, o[r][i][e + 2] *= fall;
            }
        }
        uint32_t pb[TERMS][R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float ref0 = m[r][0] == -INFINITY ? 0.f : m[r][0], ref1 = m[r][1] == -INFINITY ? 0.f : m[r][1];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = ex2(s[r][2 * i] - ref0), p1 = ex2(s[r][2 * i + 1] - ref1);
            l[r][0] += p0;
            l[r][1] += p1;
            const float w0 = p0 * vscale, w1 = p1 * vscale;
            const uint32_t hi = hf2(w0, w1);
            pb[0][r][i] = transpose8(hi);
            if (FINE) {
              const float2 z = float2_of(hi);
              pb[TERMS - 1][r][i] = transpose8(hf2(w0 - z.x, w1 - z.y));
            }
          }
        }
        uint32_t vr[4][NV / 4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = (j >> 1) * 8 + 2 * t4 + (j & 1);
          if (NV == 16) {
            const uint4 x = *reinterpret_cast<const uint4*>(vs + row * 128 + ((g ^ (row & 7)) << 4));
            vr[j][0] = x.x, vr[j][1] = x.y, vr[j][NV / 4 - 2] = x.z, vr[j][NV / 4 - 1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(vs + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8);
            vr[j][0] = x.x, vr[j][1] = x.y;
          }
        }
        if (tokens < kGroup) {  // what lies behind the last token may be anything
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((j >> 1) * 8 + 2 * t4 + (j & 1) >= tokens)
#pragma unroll
              for (int e = 0; e < NV / 4; ++e) vr[j][e] = 0;
        }
        // rows g and g + 8 of product i are elements NV g + 2 i and the next
#pragma unroll
        for (int e = 0; e < NV / 4; ++e)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // byte pairs of two tokens, two elements at once
            const uint32_t x = __byte_perm(vr[0][e], vr[1][e], half ? 0x7362 : 0x5140);
            const uint32_t y = __byte_perm(vr[2][e], vr[3][e], half ? 0x7362 : 0x5140);
            const uint32_t va[4] = {half2_of(static_cast<uint16_t>(x)), half2_of(static_cast<uint16_t>(x >> 16)),
                                    half2_of(static_cast<uint16_t>(y)), half2_of(static_cast<uint16_t>(y >> 16))};
#pragma unroll
            for (int z = 0; z < TERMS; ++z)
#pragma unroll
              for (int r = 0; r < R; ++r) mma(o[r][e * 2 + half], va, pb[TERMS - 1 - z][r]);
          }
      }
      __syncwarp();  // the slot has been read
      if (lane == 0) bar_arrive(&empty[warp][stage]);
      if (++stage == S) stage = 0, phase ^= 1;
    }

    // ---- the warps' parts of the piece meet: two and two, then both ----
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[r][e] = column_sum(l[r][e]);
        if (g == 0) s_m[warp][2 * t4 + e + 8 * r] = m[r][e], s_l[warp][2 * t4 + e + 8 * r] = l[r][e];
      }
    meet();
    float fall[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 2 * t4 + e + 8 * r;
        const float top = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
        fall[r][e] = ex2(m[r][e] - (top == -INFINITY ? 0.f : top));
      }
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
      if (warp >> 1 == 1 - turn) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < NV / 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float2* to = reinterpret_cast<float2*>(&s_o[warp & 1][2 * t4 + e + 8 * r][g * NV + 2 * i]);
              float2 x = make_float2(o[r][i][e] * fall[r][e], o[r][i][e + 2] * fall[r][e]);
              if (turn == 1) x.x += to->x, x.y += to->y;
              *to = x;
            }
      }
      meet();
    }
    const bool whole = tile0 == 0 && tile1 == use.tiles;
    float* part = a.part + (static_cast<long long>(blockIdx.x) * 2 + slot) * slot_floats(c.dv);
    for (int e = threadIdx.x; e < rows * c.dv; e += kStepWarps * 32) {
      const int row = e / c.dv, d = e % c.dv;
      const float top = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int z = 0; z < kStepWarps; ++z) sum = fmaf(s_l[z][row], ex2(s_m[z][row] - ref), sum);
      const float x = s_o[0][row][d] + s_o[1][row][d];
      if (whole) {
        static_cast<T*>(a.out)[(static_cast<long long>(use.b) * a.H + h0 + row) * c.dv + d] = from_f<T>(x / sum);
      } else {
        if (d == 0) part[row] = top, part[16 + row] = sum;
        part[32 + row * c.dv + d] = x;
      }
    }
    meet();  // read before the next piece's are written
    slot = 1;  // pieces after the first begin with their request's first tile
    at += tile1 - tile0;
    use.tile = tile1 - 1;
    if (at < end) use.next(a, warp, groups);
  }
}

// Joins the parts of rows that several CTAs had, in the CTAs' order: a CTA per
// query head of a request; 128 threads take the elements, and slice z of the
// CTA every Z-th part.  Launched while the step still runs, so that it costs 3.4
// us where one request is all there is.
template <typename T, int Z>
__global__ void __launch_bounds__(128 * Z) join_kernel(const __grid_constant__ StepArgs a, int ctas) {
  const Cache& c = a.c;
  __shared__ float s_m[Z], s_l[Z], s_x[Z][128];
  const long long b = blockIdx.y;
  const int h = blockIdx.x, z = threadIdx.x >> 7, d = threadIdx.x & 127;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long n = a.before[b], tiles = a.before[b + 1] - n;
  const int groups = c.heads * a.row_tiles, row = h % a.share % 16;
  const long long total = a.before[c.B] * groups;
  if (tiles == 0) return;
  const long long first = n * groups + (h / a.share * a.row_tiles + h % a.share / 16) * tiles, last = first + tiles - 1;
  // the CTA that has tile t: runs of size + 1 come first
  const long long size = total / ctas, more = total % ctas;
  auto cta_of = [&](long long t) { return t < more * (size + 1) ? t / (size + 1) : more + (t - more * (size + 1)) / size; };
  auto begin_of = [&](long long i) { return size * i + min(more, i); };
  const int i0 = static_cast<int>(cta_of(first)), i1 = static_cast<int>(cta_of(last));
  if (i0 == i1) return;  // that CTA wrote it
  float m = -INFINITY, l = 0.f, x = 0.f;
  constexpr int D = 8;  // parts in flight
  for (int i = i0 + z; i <= i1; i += Z * D) {
    float pm[D], pl[D], px[D], top = m;
#pragma unroll
    for (int e = 0; e < D; ++e) {
      pm[e] = -INFINITY, pl[e] = px[e] = 0.f;
      const int j = i + e * Z;
      if (j <= i1) {
        // a CTA's first piece is in slot 0; one that it came to later in slot 1
        const float* part = a.part + (2ll * j + (begin_of(j) < first)) * slot_floats(c.dv);
        pm[e] = part[row], pl[e] = part[16 + row];
        if (d < c.dv) px[e] = part[32 + row * c.dv + d];
      }
    }
#pragma unroll
    for (int e = 0; e < D; ++e) top = fmaxf(top, pm[e]);
    const float ref = top == -INFINITY ? 0.f : top, keep = ex2(m - ref);
    l *= keep, x *= keep, m = top;
#pragma unroll
    for (int e = 0; e < D; ++e) {
      const float f = ex2(pm[e] - ref);
      l = fmaf(pl[e], f, l);
      x = fmaf(px[e], f, x);
    }
  }
  if (Z > 1) {
    if (d == 0) s_m[z] = m, s_l[z] = l;
    s_x[z][d] = x;
    __syncthreads();
    if (z != 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < Z; ++i) top = fmaxf(top, s_m[i]);
    const float ref = top == -INFINITY ? 0.f : top;
    l = x = 0.f;
#pragma unroll
    for (int i = 0; i < Z; ++i) {
      const float f = ex2(s_m[i] - ref);
      l = fmaf(s_l[i], f, l);
      x = fmaf(s_x[i][d], f, x);
    }
  }
  if (d < c.dv) static_cast<T*>(a.out)[(b * a.H + h) * c.dv + d] = from_f<T>(x / l);
}

// Sixteen rows of a page: rows of 128 bytes or 64, zeros behind the head's last
// element.
static bool map_pages(CUtensorMap* m, const uint8_t* pool, const Cache& c, int dim) {
  const auto fn = encode_fn();
  if (!fn) return false;
  const bool wide = dim > 64;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(c.page), static_cast<cuuint64_t>(c.pages) * c.heads};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(dim) * c.page};
  const cuuint32_t box[3] = {wide ? 128u : 64u, kGroup, 1}, one[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(pool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            wide ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int U, int NV, int R>
static int launch_step(const StepArgs& a, const StepMaps& m, int ctas, cudaStream_t s) {
  static std::atomic<unsigned long long> done{};
  constexpr size_t bytes = static_cast<size_t>(kStepWarps) * stages(R) * kGroup * (64 * U + 8 * NV);
  const int rc = mscan::allow_smem(step_kernel<T, U, NV, R>, bytes, done);
  if (rc != ASCAN_OK) return rc;
  step_kernel<T, U, NV, R><<<ctas, kStepThreads, bytes, s>>>(a, m);
  return launch_status();
}

template <typename T, int R>
static int pick_step(const StepArgs& a, const StepMaps& m, int ctas, cudaStream_t s) {
  if (a.c.dk > 64) return a.c.dv > 64 ? launch_step<T, 2, 16, R>(a, m, ctas, s) : launch_step<T, 2, 8, R>(a, m, ctas, s);
  return a.c.dv > 64 ? launch_step<T, 1, 16, R>(a, m, ctas, s) : launch_step<T, 1, 8, R>(a, m, ctas, s);
}

// Launched while the step still runs: its CTAs are set up as the step's end, and
// wait for all that the step wrote.
template <typename T, int Z>
static int join(const StepArgs& a, int ctas, dim3 grid, cudaStream_t s) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(128 * Z);
  config.stream = s;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, join_kernel<T, Z>, a, ctas) == cudaSuccess ? launch_status() : ASCAN_ECUDA;
}

template <typename T>
static int step(const StepArgs& a, const StepMaps& m, cudaStream_t s) {
  const int ctas = 148 * (sizeof(T) == 4 ? 2 : kCtasPerSm);
  const int rc = a.share <= 8 ? pick_step<T, 1>(a, m, ctas, s) : pick_step<T, 2>(a, m, ctas, s);
  if (rc != ASCAN_OK) return rc;
  // a row of a few requests lies in many CTAs' parts, one of many in one or two
  const dim3 grid(a.H, static_cast<unsigned>(a.c.B));
  if (a.c.B * a.c.heads * a.row_tiles * 4 < ctas) return join<T, 8>(a, ctas, grid, s);
  return join<T, 1>(a, ctas, grid, s);
}

// A pool without pages: every row is zero, and one with tokens an error.
template <typename T>
__global__ void __launch_bounds__(kThreads) no_pages_kernel(const __grid_constant__ StepArgs a) {
  const long long n = a.c.B * a.H * a.c.dv;
  for (long long e = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; e < n; e += gridDim.x * static_cast<long long>(kThreads)) {
    static_cast<T*>(a.out)[e] = from_f<T>(0.f);
    const long long b = e / (static_cast<long long>(a.H) * a.c.dv);
    if (index_at(a.lengths, a.lengths64, b) > 0) report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(b), a.err);
  }
}

template <typename T>
static int run_step(StepArgs& a, cudaStream_t s) {
  if (a.c.pages == 0) {
    no_pages_kernel<T><<<148, kThreads, 0, s>>>(a);
    return launch_status();
  }
  // Tensor maps are made through the driver, which wants a current context
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return ASCAN_EDEVICE;
  StepMaps m;
  if (!map_pages(&m.k, a.c.k, a.c, a.c.dk) || !map_pages(&m.v, a.c.v, a.c, a.c.dv)) return ASCAN_ECUDA;
  return step<T>(a, m, s);
}

template <typename T>
static int write(const WriteArgs& a, int vec_k, int vec_v, cudaStream_t s) {
  // A single token per request is a row of 128 elements, which a warp takes;
  // longer pieces fill eight.
  if (a.BL <= 2 * a.c.B) write_kernel<T, 32><<<static_cast<unsigned>((a.units + 7) / 8), kThreads, 0, s>>>(a, vec_k, vec_v);
  else write_kernel<T, kThreads><<<static_cast<unsigned>(a.units), kThreads, 0, s>>>(a, vec_k, vec_v);
  return launch_status();
}

static bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static int fill(Cache& c, const ascan_cache* x, const int32_t* table, int64_t B, int64_t width) {
  if (!x || x->pages < 0 || x->heads <= 0 || x->heads > 65535 || x->pages > 0x7fffffffll / x->heads || x->page <= 0 || x->page > ASCAN_CACHE_MAX_PAGE ||
      x->page % 16 || x->key_dim <= 0 || x->value_dim <= 0 || x->key_dim % 16 || x->value_dim % 16 ||
      x->key_dim > ASCAN_ATTENTION_MAX_DIM || x->value_dim > ASCAN_ATTENTION_MAX_DIM)
    return ASCAN_EINVAL;
  if (B < 0 || B > 65535 || width < 0 || width > (1ll << 31)) return ASCAN_EINVAL;
  if (B == 0) return ASCAN_OK;
  if (x->pages > 0 && (!x->keys || !x->values || !x->key_scales || !x->value_scales || !aligned(x->keys) || !aligned(x->values)))
    return ASCAN_EINVAL;
  if (width > 0 && !table) return ASCAN_EINVAL;
  c = Cache{static_cast<uint8_t*>(x->keys), static_cast<uint8_t*>(x->values), x->key_scales, x->value_scales, x->pages,
            x->heads, x->page, x->key_dim, x->value_dim, table, B, width};
  return ASCAN_OK;
}

static bool rows_ok(const ascan_rows* r) {
  return r && r->data && r->heads > 0 && r->heads <= 65535 && r->stride_token >= 0 && r->stride_head >= 0;
}

}  // namespace cache
}  // namespace ascan

using namespace ascan;

extern "C" {

int ascan_cache_write(const ascan_rows* keys, const ascan_rows* values, const ascan_cache* cache, const int32_t* pages,
                      int64_t num_seq, int64_t width, const void* starts, int starts_type, const void* cu_seqlens,
                      int cu_index_type, int64_t seq_total, int dtype, void* stream) {
  cache::WriteArgs a{};
  const int rc = cache::fill(a.c, cache, pages, num_seq, width);
  if (rc != ASCAN_OK) return rc;
  if (seq_total < 0 || seq_total > ASCAN_ATTENTION_MAX_TOKENS || dtype < ASCAN_F32 || dtype > ASCAN_BF16 ||
      (starts_type != ASCAN_I32 && starts_type != ASCAN_I64) || (cu_index_type != ASCAN_I32 && cu_index_type != ASCAN_I64))
    return ASCAN_EINVAL;
  if (num_seq == 0 || seq_total == 0) return ASCAN_OK;
  if (!cache::rows_ok(keys) || !cache::rows_ok(values) || keys->heads != cache->heads || values->heads != cache->heads ||
      !starts || !cu_seqlens)
    return ASCAN_EINVAL;
  a.x[0] = mscan::Rows{keys->data, keys->stride_token, keys->stride_head, 1};
  a.x[1] = mscan::Rows{values->data, values->stride_token, values->stride_head, 1};
  a.starts = starts;
  a.starts64 = starts_type == ASCAN_I64;
  a.cu = cu_seqlens;
  a.cu64 = cu_index_type == ASCAN_I64;
  a.BL = seq_total;
  a.units = (seq_total / cache->page + 2 * num_seq) * cache->heads * 2;
  if (a.units > 0x7fffffffll) return ASCAN_EINVAL;
  a.err = g_err_host;
  const int v = dtype == ASCAN_F32 ? 4 : 8;
  int vec[2];
  for (int i = 0; i < 2; ++i) vec[i] = cache::aligned(a.x[i].p) && a.x[i].st % v == 0 && a.x[i].sh % v == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ASCAN_F32) return cache::write<float>(a, vec[0], vec[1], s);
  if (dtype == ASCAN_F16) return cache::write<__half>(a, vec[0], vec[1], s);
  return cache::write<__nv_bfloat16>(a, vec[0], vec[1], s);
}

size_t ascan_cache_step_workspace(int64_t num_seq, int value_dim) {
  if (num_seq <= 0 || value_dim <= 0) return 256;
  return 512 + sizeof(float) * 2 * cache::kMaxCtas * (32 + 16 * static_cast<size_t>(value_dim)) + sizeof(long long) * (num_seq + 1);
}

int ascan_cache_step(const ascan_rows* queries, const ascan_cache* cache, const int32_t* pages, int64_t num_seq,
                     int64_t width, const void* lengths, int lengths_type, int dtype, float scale, void* out,
                     void* workspace, size_t workspace_bytes, void* stream) {
  cache::StepArgs a{};
  const int rc = cache::fill(a.c, cache, pages, num_seq, width);
  if (rc != ASCAN_OK) return rc;
  if (dtype < ASCAN_F32 || dtype > ASCAN_BF16 || (lengths_type != ASCAN_I32 && lengths_type != ASCAN_I64)) return ASCAN_EINVAL;
  if (!(scale > 0.f) || !(scale < INFINITY)) return ASCAN_EINVAL;
  if (num_seq == 0) return ASCAN_OK;
  if (!cache::rows_ok(queries) || queries->heads % cache->heads || !lengths || !out) return ASCAN_EINVAL;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) ||
      workspace_bytes < ascan_cache_step_workspace(num_seq, cache->value_dim))
    return ASCAN_EWORKSPACE;
  a.q = mscan::Rows{queries->data, queries->stride_token, queries->stride_head, 1};
  a.lengths = lengths;
  a.lengths64 = lengths_type == ASCAN_I64;
  a.H = queries->heads;
  a.share = queries->heads / cache->heads;
  a.row_tiles = (a.share + 15) / 16;
  a.scale = scale;
  a.out = out;
  a.before = static_cast<long long*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + (sizeof(long long) * (num_seq + 1) + 255) / 256 * 256);
  a.err = g_err_host;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ASCAN_F32) return cache::run_step<float>(a, s);
  if (dtype == ASCAN_F16) return cache::run_step<__half>(a, s);
  return cache::run_step<__nv_bfloat16>(a, s);
}

}  // extern "C"

namespace ascan {
ASCAN_UNIT_ERROR_ACCESSORS(cache)
}  // namespace ascan
