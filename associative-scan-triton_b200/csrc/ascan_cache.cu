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

namespace ascan {
namespace cache {

using mscan::from_f;
using mscan::Rows;
using mscan::to_f;

constexpr int kScaleBits = 64;

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

// Four values to e4m3, to nearest; infinities and NaN become its NaN, finite
// values beyond the largest scale's reach its largest.
__device__ __forceinline__ uint32_t pack4(const float* x) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = fabsf(x[i]) < INFINITY ? x[i] : NAN;
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

// Eight elements as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float* x) {
  if (vec) {
    constexpr int N = sizeof(T) == 4 ? 4 : 8;
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + i));
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int q = 0; q < N; ++q) x[i + q] = to_f(e[q]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f(p[i]);
  }
}

// A group of G threads writes what one request adds to one page of one head:
// the largest magnitude first, which gives the scale, then the rounded values
// (read again, out of the nearest cache).
template <typename T, int G>
__global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ WriteArgs a, int vec_k, int vec_v) {
  constexpr int UNITS = kThreads / G;
  const Cache& c = a.c;
  const int gl = threadIdx.x % G, sub = threadIdx.x / G;
  if (blockIdx.x == 0) {
    if (a.cu64) validate_cu(static_cast<const int64_t*>(a.cu), c.B, a.BL, a.err);
    else validate_cu(static_cast<const int32_t*>(a.cu), c.B, a.BL, a.err);
  }
  const long long unit = static_cast<long long>(blockIdx.x) * UNITS + sub;
  if (unit >= a.units) return;  // whole groups
  const bool is_v = unit & 1;
  const int h = static_cast<int>((unit >> 1) % c.heads);
  const long long x = (unit >> 1) / c.heads;  // piece number
  auto cu_at = [&](long long i) {
    const long long v = index_at(a.cu, a.cu64, i);
    return v < 0 ? 0ll : (v > a.BL ? a.BL : v);
  };
  // pieces of request b start at cu[b] / page + 2 b: no more than its tokens
  // fill and two that they begin and end in
  long long lo = 0, hi = c.B - 1;
  while (lo < hi) {
    const long long mid = (lo + hi + 1) >> 1;
    if (cu_at(mid) / c.page + 2 * mid <= x) lo = mid;
    else hi = mid - 1;
  }
  const long long b = lo, c0 = cu_at(b), len = cu_at(b + 1) - c0, start = index_at(a.starts, a.starts64, b);
  if (start < 0 || len <= 0) return;  // no request, or nothing new
  const long long place = start / c.page + (x - c0 / c.page - 2 * b);
  const long long from = max(start, place * c.page), to = min(start + len, (place + 1) * c.page);
  if (from >= to) return;
  long long id = -1;
  if (place < c.width) id = c.table[b * c.width + place];
  if (id < 0 || id >= c.pages) {
    if (gl == 0) report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(b), a.err);
    return;
  }
  const int dim = is_v ? c.dv : c.dk, first = static_cast<int>(from - place * c.page), n = static_cast<int>(to - from);
  const bool vec = is_v ? vec_v : vec_k;
  const Rows& r = a.x[is_v];
  const T* src = static_cast<const T*>(r.p) + (c0 + from - start) * r.st + h * r.sh;
  uint8_t* dst = (is_v ? c.v : c.k) + ((id * c.heads + h) * c.page) * dim;
  float* scale = (is_v ? c.vs : c.ks) + id * c.heads + h;
  const int per_row = dim / 8, work = n * per_row;
  float top = 0.f;
  for (int e = gl; e < work; e += G) {
    float v[8];
    load8(src + (e / per_row) * r.st + (e % per_row) * 8, vec, v);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float m = fabsf(v[q]);
      if (m < INFINITY) top = fmaxf(top, m);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  const float held = first > 0 ? *scale : 0.f;
  if (G > 32) {
    __shared__ float tops[G / 32];
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();  // everyone has read the scale too
#pragma unroll
    for (int w = 0; w < G / 32; ++w) top = fmaxf(top, tops[w]);
  } else {
    __syncwarp();
  }
  const float need = fmaxf(pow2(scale_bits(top)), held);
  if (first > 0 && need > held) {  // what the page holds moves to the larger scale
    const float f = held / need;
    for (int e = gl; e < first * dim / 16; e += G) {
      uint4 w = reinterpret_cast<uint4*>(dst)[e];
      w.x = rescale4(w.x, f), w.y = rescale4(w.y, f), w.z = rescale4(w.z, f), w.w = rescale4(w.w, f);
      reinterpret_cast<uint4*>(dst)[e] = w;
    }
  }
  if (gl == 0 && need != held) *scale = need;
  const float inv = 1.f / need;
  for (int e = gl; e < work; e += G) {
    float v[8];
    load8(src + (e / per_row) * r.st + (e % per_row) * 8, vec, v);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] *= inv;
    *reinterpret_cast<uint2*>(dst + (first + e / per_row) * dim + (e % per_row) * 8) = make_uint2(pack4(v), pack4(v + 4));
  }
}

// ---------------------------------------------------------------------------
// attention of single tokens
// ---------------------------------------------------------------------------

constexpr int kStepThreads = 128;
constexpr int kStepTile = 64;  // tokens of a tile: sixteen of each warp
constexpr int kMaxCtas = 148 * 4;

struct StepArgs {
  Cache c;
  Rows q;
  const void* lengths;
  int lengths64, H, share, row_tiles;  // sixteen query heads of a key head are a row tile
  float scale;
  void* out;
  float* part;  // per CTA two slots of [16] references, [16] sums, [16][dv] rows
  uint32_t* err;
};

__device__ __forceinline__ int slot_floats(int dv) { return 32 + 16 * dv; }

// Tokens of request b; what does not fit its row of pages is left out.
__device__ __forceinline__ long long length_of(const StepArgs& a, long long b) {
  const long long n = index_at(a.lengths, a.lengths64, b), room = a.c.width * a.c.page;
  return n < 0 ? 0 : min(n, room);
}
__device__ __forceinline__ long long tiles_of(const StepArgs& a, long long b) {
  return (length_of(a, b) + kStepTile - 1) / kStepTile;
}

// Sum over the block's 128 threads, the same for all; `scratch` of 4.
__device__ __forceinline__ long long block_sum(long long x, long long* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) x += __shfl_xor_sync(kFull, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
  __syncthreads();
  return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// Tiles of all requests before `until`.
__device__ __forceinline__ long long tiles_before(const StepArgs& a, long long until, long long* scratch) {
  long long n = 0;
  for (long long b = threadIdx.x; b < until; b += kStepThreads) {
    n += tiles_of(a, b);
    if (blockIdx.x == 0 && index_at(a.lengths, a.lengths64, b) > a.c.width * a.c.page)
      report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(b), a.err);
  }
  return block_sum(n, scratch);
}

__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_from(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float2 float2_of(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(kFull, x, 1));
  return fmaxf(x, __shfl_xor_sync(kFull, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(kFull, x, 1);
  return x + __shfl_xor_sync(kFull, x, 2);
}

// The tiles of all requests, key heads and row tiles are one list; a CTA takes
// an equal run of it, wherever requests begin and end, and walks it piece by
// piece (a piece: what it has of one request, head and row tile).  Each warp
// takes sixteen tokens of a tile with m16n8k16 products of float16: e4m3
// values are exact there, queries are brought to at most 2^15 by a power of
// two per row, and weights lie between 0 and 2^8, so both keep 11 bits or more
// (22 where queries are float32: the rest of each goes through a second
// product).  Keys and values go from memory to registers as the operands want
// them, sixteen bytes a load: which dims and tokens stand for which index of a
// product is free as long as both operands agree.
//
// U: 64-element parts of a key.  NV: bytes of a value row per lane.
template <typename T, int U, int NV>
__global__ void __launch_bounds__(kStepThreads, sizeof(T) == 4 ? 2 : 3) step_kernel(const __grid_constant__ StepArgs a) {
  constexpr bool FINE = sizeof(T) == 4;
  constexpr int TERMS = FINE ? 2 : 1;
  const Cache& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  __shared__ long long scratch[4];
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ float s_o[4][16][NV * 8 + 4];

  const int groups = c.heads * a.row_tiles;  // of a request
  const long long total = tiles_before(a, c.B, scratch) * groups;
  const long long begin = total / gridDim.x * blockIdx.x + min(total % gridDim.x, static_cast<long long>(blockIdx.x));
  const long long end = begin + total / gridDim.x + (blockIdx.x < total % gridDim.x);
  // requests without tokens, dealt to all CTAs
  for (long long b = blockIdx.x; b < c.B; b += gridDim.x)
    if (tiles_of(a, b) == 0)
      for (int e = threadIdx.x; e < a.H * c.dv; e += kStepThreads) static_cast<T*>(a.out)[b * a.H * c.dv + e] = from_f<T>(0.f);
  if (begin >= end) return;

  // The request that `begin` lies in: 128 at a time, then one by one.
  long long b = 0, before = 0;  // tiles of the requests before b, times groups
  while (true) {
    const long long n = b + threadIdx.x < c.B ? tiles_of(a, b + threadIdx.x) : 0;
    const long long sum = block_sum(n, scratch) * groups;
    if (before + sum > begin) break;
    before += sum;
    b += kStepThreads;
  }
  for (long long n; before + (n = tiles_of(a, b) * groups) <= begin; ++b) before += n;

  const float c2 = a.scale * 1.4426950408889634f;
  int slot = 0;
  for (long long at = begin; at < end; ) {
    const long long tiles = tiles_of(a, b), rel = at - before;
    if (rel >= tiles * groups) {  // next request with tokens
      before += tiles * groups;
      ++b;
      continue;
    }
    const int group = static_cast<int>(rel / tiles);
    const long long tile0 = rel % tiles, tile1 = min(tiles, tile0 + (end - at));
    const int hk = group / a.row_tiles, h0 = hk * a.share + group % a.row_tiles * 16;
    const int rows = min(16, (hk + 1) * a.share - h0);
    const long long len = length_of(a, b);

    // ---- queries as operands: index 2 t4.. of product (u, w) is element
    // 64 u + 16 t4 + 4 w.. of the head
    uint32_t q[TERMS][U * 4][4];
    float qf[2];  // what a row's scores are in units of
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + 8 * r;
      float x[U * 16], top = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int d = 64 * u + 16 * t4 + e;
          x[u * 16 + e] = row < rows && d < c.dk ? to_f(static_cast<const T*>(a.q.p)[b * a.q.st + (h0 + row) * a.q.sh + d]) : 0.f;
          top = fmaxf(top, fabsf(x[u * 16 + e]));
        }
      top = quad_max(top);
      const int e2 = max(-100, static_cast<int>(__float_as_uint(top) >> 23) - 127);
      const float up = pow2(14 - e2);
      qf[r] = pow2(e2 - 14) * c2;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float y0 = x[u * 16 + w * 4 + half * 2] * up, y1 = x[u * 16 + w * 4 + half * 2 + 1] * up;
            const uint32_t hi = half2_from(y0, y1);
            q[0][u * 4 + w][half * 2 + r] = hi;
            if (FINE) {
              const float2 f = float2_of(hi);
              q[TERMS - 1][u * 4 + w][half * 2 + r] = half2_from(y0 - f.x, y1 - f.y);
            }
          }
    }

    float o[NV][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    uint4 kr[2][U];
    uint32_t vr[4][NV / 4];
    float kscale = 0.f, vscale = 1.f;
    bool ok = false;
    const int* row_of_pages = c.table + b * c.width;
    long long id = 0;
    auto page_of = [&](long long tile) {
      const long long t0 = tile * kStepTile + warp * 16;
      ok = tile < tile1 && t0 < len;
      if (!ok) return;
      id = __ldg(row_of_pages + t0 / c.page);
      if (id < 0 || id >= c.pages) {
        if (lane == 0) report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(b), a.err);
        ok = false;
      }
    };
    auto load_k = [&](long long tile) {
      if (!ok) return;
      const int in_page = static_cast<int>((tile * kStepTile + warp * 16) % c.page);
      const uint8_t* at_k = c.k + ((id * c.heads + hk) * c.page + in_page) * c.dk;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u)
          kr[i][u] = 64 * u + 16 * t4 < c.dk ? __ldcs(reinterpret_cast<const uint4*>(at_k + (8 * i + g) * c.dk + 64 * u + 16 * t4))
                                             : make_uint4(0, 0, 0, 0);
      kscale = __ldg(c.ks + id * c.heads + hk);
    };
    auto load_v = [&](long long tile) {
      if (!ok) return;
      const int in_page = static_cast<int>((tile * kStepTile + warp * 16) % c.page);
      const uint8_t* at_v = c.v + ((id * c.heads + hk) * c.page + in_page) * c.dv;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = (j >> 1) * 8 + 2 * t4 + (j & 1);
        if (NV == 16) {
          const uint4 x = g * 16 < c.dv ? __ldcs(reinterpret_cast<const uint4*>(at_v + tok * c.dv + g * 16)) : make_uint4(0, 0, 0, 0);
          vr[j][0] = x.x, vr[j][1] = x.y, vr[j][NV / 4 - 2] = x.z, vr[j][NV / 4 - 1] = x.w;
        } else {
          const uint2 x = g * 8 < c.dv ? __ldcs(reinterpret_cast<const uint2*>(at_v + tok * c.dv + g * 8)) : make_uint2(0, 0);
          vr[j][0] = x.x, vr[j][1] = x.y;
        }
      }
      vscale = __ldg(c.vs + id * c.heads + hk);
    };

    page_of(tile0);
    load_k(tile0);
    load_v(tile0);
#pragma unroll 1
    for (long long tile = tile0; tile < tile1; ++tile) {
      const bool now = ok;
      float w[2][4], vsc = vscale;
      const long long t0 = tile * kStepTile + warp * 16;
      const int left = static_cast<int>(min(16ll, len - t0));  // tokens of the sixteen
      if (now) {
        float s[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const uint32_t word[4] = {kr[i][u].x, kr[i][u].y, kr[i][u].z, kr[i][u].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t b0 = half2_of(static_cast<uint16_t>(word[e])), b1 = half2_of(static_cast<uint16_t>(word[e] >> 16));
#pragma unroll
              for (int x = 0; x < TERMS; ++x) mma(s[i], q[TERMS - 1 - x][u * 4 + e], b0, b1);
            }
          }
        }
        // in units of log 2; a page's value scale is added to the exponent
        const float lv = static_cast<float>(static_cast<int>(__float_as_uint(vsc) >> 23) - 127);
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool in = 8 * i + 2 * t4 + (e & 1) < left;
            s[i][e] = in ? s[i][e] * (qf[e >> 1] * kscale) : -INFINITY;
            top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
          }
#pragma unroll
        for (int r = 0; r < 2; ++r) top[r] = quad_max(top[r]) + lv;
        // the reference moves when weights would pass 2^8
        if (__any_sync(kFull, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {
          float f[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float next = fmaxf(m[r], top[r]);
            f[r] = next == -INFINITY ? 1.f : ex2(m[r] - next);
            m[r] = next;
            l[r] *= f[r];
          }
#pragma unroll
          for (int i = 0; i < NV; ++i) o[i][0] *= f[0], o[i][1] *= f[0], o[i][2] *= f[1], o[i][3] *= f[1];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float ref = m[e >> 1] == -INFINITY ? 0.f : m[e >> 1];
            const float p = ex2(s[i][e] - ref);
            l[e >> 1] += p;
            w[i][e] = p * vsc;
          }
      }
      page_of(tile + 1);
      load_k(tile + 1);
      if (now) {
        if (left < 16) {  // what lies behind the last token may be anything
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((j >> 1) * 8 + 2 * t4 + (j & 1) >= left)
#pragma unroll
              for (int e = 0; e < NV / 4; ++e) vr[j][e] = 0;
        }
        uint32_t pa[TERMS][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t hi = half2_from(w[i][2 * r], w[i][2 * r + 1]);
            pa[0][2 * i + r] = hi;
            if (FINE) {
              const float2 f = float2_of(hi);
              pa[TERMS - 1][2 * i + r] = half2_from(w[i][2 * r] - f.x, w[i][2 * r + 1] - f.y);
            }
          }
#pragma unroll
        for (int e = 0; e < NV / 4; ++e)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // byte pairs of two tokens, two elements at once
            const uint32_t x = __byte_perm(vr[0][e], vr[1][e], half ? 0x7362 : 0x5140);
            const uint32_t y = __byte_perm(vr[2][e], vr[3][e], half ? 0x7362 : 0x5140);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t b0 = half2_of(static_cast<uint16_t>(k ? x >> 16 : x)), b1 = half2_of(static_cast<uint16_t>(k ? y >> 16 : y));
#pragma unroll
              for (int z = 0; z < TERMS; ++z) mma(o[e * 4 + half * 2 + k], pa[TERMS - 1 - z], b0, b1);
            }
          }
      }
      load_v(tile + 1);
    }

    // ---- the warps' parts of the piece meet ----
#pragma unroll
    for (int r = 0; r < 2; ++r) l[r] = quad_sum(l[r]);
    __syncthreads();  // the piece before has been read
    if (t4 == 0)
#pragma unroll
      for (int r = 0; r < 2; ++r) s_m[warp][g + 8 * r] = m[r], s_l[warp][g + 8 * r] = l[r];
    // column n of product i is element NV n + i of the value; lane t4 has
    // columns 2 t4 and 2 t4 + 1
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s_o[warp][g + 8 * (e >> 1)][(2 * t4 + (e & 1)) * NV + i] = o[i][e];
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == tiles;
    float* part = a.part + (static_cast<long long>(blockIdx.x) * 2 + slot) * slot_floats(c.dv);
    for (int e = threadIdx.x; e < rows * c.dv; e += kStepThreads) {
      const int row = e / c.dv, d = e % c.dv;
      float top = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f, x = 0.f;
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const float f = ex2(s_m[z][row] - ref);
        sum = fmaf(s_l[z][row], f, sum);
        x = fmaf(s_o[z][row][d], f, x);
      }
      if (whole) {
        static_cast<T*>(a.out)[(b * a.H + h0 + row) * c.dv + d] = from_f<T>(x / sum);
      } else {
        if (d == 0) part[row] = top, part[16 + row] = sum;
        part[32 + row * c.dv + d] = x;
      }
    }
    slot = 1;  // pieces after the first begin with their request's first tile
    at += tile1 - tile0;
  }
}

// Joins the parts of rows that several CTAs had, in the CTAs' order: a CTA per
// query head of a request; 128 threads take the elements, and quarter z of the
// CTA every fourth part.
template <typename T>
__global__ void __launch_bounds__(512) join_kernel(const __grid_constant__ StepArgs a, int ctas) {
  const Cache& c = a.c;
  __shared__ long long scratch[16];
  __shared__ float s_m[4], s_l[4], s_x[4][128];
  const long long b = blockIdx.y;
  const int h = blockIdx.x, tid = threadIdx.x, z = tid >> 7, d = tid & 127;
  long long n = 0, all = 0;
  for (long long i = tid; i < c.B; i += 512) {
    const long long x = tiles_of(a, i);
    all += x;
    if (i < b) n += x;
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) all += __shfl_xor_sync(kFull, all, o), n += __shfl_xor_sync(kFull, n, o);
  if ((tid & 31) == 0) scratch[tid >> 5] = all;
  __syncthreads();
  all = 0;
  for (int i = 0; i < 16; ++i) all += scratch[i];
  __syncthreads();
  if ((tid & 31) == 0) scratch[tid >> 5] = n;
  __syncthreads();
  n = 0;
  for (int i = 0; i < 16; ++i) n += scratch[i];
  const int groups = c.heads * a.row_tiles, row = h % a.share % 16;
  const long long tiles = tiles_of(a, b), total = all * groups;
  if (tiles == 0) return;
  const long long first = n * groups + (h / a.share * a.row_tiles + h % a.share / 16) * tiles, last = first + tiles - 1;
  // the CTA that has tile t: runs of size + 1 come first
  const long long size = total / ctas, more = total % ctas;
  auto cta_of = [&](long long t) { return t < more * (size + 1) ? t / (size + 1) : more + (t - more * (size + 1)) / size; };
  auto begin_of = [&](long long i) { return size * i + min(more, i); };
  const long long i0 = cta_of(first), i1 = cta_of(last);
  if (i0 == i1) return;  // that CTA wrote it
  float m = -INFINITY, l = 0.f, x = 0.f;
  for (long long i = i0 + z; i <= i1; i += 4) {
    // a CTA's first piece is in slot 0; one that it came to later in slot 1
    const float* part = a.part + (2 * i + (begin_of(i) < first)) * slot_floats(c.dv);
    const float pm = part[row], pl = part[16 + row], px = d < c.dv ? part[32 + row * c.dv + d] : 0.f;
    const float next = fmaxf(m, pm), ref = next == -INFINITY ? 0.f : next;
    const float f = ex2(m - ref), e = ex2(pm - ref);
    l = fmaf(l, f, pl * e);
    x = fmaf(x, f, px * e);
    m = next;
  }
  if (d == 0) s_m[z] = m, s_l[z] = l;
  s_x[z][d] = x;
  __syncthreads();
  if (z != 0 || d >= c.dv) return;
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), ref = top == -INFINITY ? 0.f : top;
  l = x = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = ex2(s_m[i] - ref);
    l = fmaf(s_l[i], f, l);
    x = fmaf(s_x[i][d], f, x);
  }
  static_cast<T*>(a.out)[(b * a.H + h) * c.dv + d] = from_f<T>(x / l);
}

template <typename T>
static int step(const StepArgs& a, int ctas, cudaStream_t s) {
  const bool wide_k = a.c.dk > 64, wide_v = a.c.dv > 64;
  if (wide_k && wide_v) step_kernel<T, 2, 16><<<ctas, kStepThreads, 0, s>>>(a);
  else if (wide_k) step_kernel<T, 2, 8><<<ctas, kStepThreads, 0, s>>>(a);
  else if (wide_v) step_kernel<T, 1, 16><<<ctas, kStepThreads, 0, s>>>(a);
  else step_kernel<T, 1, 8><<<ctas, kStepThreads, 0, s>>>(a);
  const int rc = launch_status();
  if (rc != ASCAN_OK) return rc;
  join_kernel<T><<<dim3(a.H, static_cast<unsigned>(a.c.B)), 512, 0, s>>>(a, ctas);
  return launch_status();
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
  if (!x || x->pages < 0 || x->heads <= 0 || x->heads > 65535 || x->page <= 0 || x->page > ASCAN_CACHE_MAX_PAGE ||
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

size_t ascan_cache_step_workspace(int value_dim) {
  if (value_dim <= 0) return 256;
  return 256 + sizeof(float) * 2 * cache::kMaxCtas * (32 + 16 * static_cast<size_t>(value_dim));
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
      workspace_bytes < ascan_cache_step_workspace(cache->value_dim))
    return ASCAN_EWORKSPACE;
  a.q = mscan::Rows{queries->data, queries->stride_token, queries->stride_head, 1};
  a.lengths = lengths;
  a.lengths64 = lengths_type == ASCAN_I64;
  a.H = queries->heads;
  a.share = queries->heads / cache->heads;
  a.row_tiles = (a.share + 15) / 16;
  a.scale = scale;
  a.out = out;
  a.part = static_cast<float*>(workspace);
  a.err = g_err_host;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int ctas = 148 * 3;
  if (dtype == ASCAN_F32) return cache::step<float>(a, ctas, s);
  if (dtype == ASCAN_F16) return cache::step<__half>(a, ctas, s);
  return cache::step<__nv_bfloat16>(a, ctas, s);
}

}  // extern "C"

namespace ascan {
ASCAN_UNIT_ERROR_ACCESSORS(cache)
}  // namespace ascan
