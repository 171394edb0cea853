// ascan_attend.cu -- compilation unit of the scan library: causal softmax
// attention, its entry points and its kernels in float32 arithmetic.
//
// The kernels here serve float32 tensors, and 16-bit ones whose head sizes the
// tensor-core kernels do not take.  A CTA holds 64 rows of one side in shared
// memory as floats and walks tiles of 64 rows of the other; a thread has a
// 4 x 4 part of the scores and 4 rows of the sums, read sixteen bytes at a
// time with rows four words off a multiple of the banks.  Multiply-adds bound
// them: a tile of scores of heads of 128 is 64 of them for each 8 loads.  3001
// tokens in 5 ragged sequences, 12 heads of 64, float32: forward 157 us, dq 222, dk and
// dv 288, d = do.o 10 (10.45 GFLOP, so 15 TFLOP/s in all, of 74); single
// multiply-adds and copies through registers took 857 us instead of 677.  What
// is left over is the CTAs of the longest sequence, which end last, and four
// shared-memory loads for every sixteen pairs of multiply-adds.
#include "ascan_impl.cuh"
#include "ascan_attend.cuh"
#include "ascan_pairs.cuh"

namespace ascan {
namespace attend {

constexpr int kR = 64;  // rows of a tile, as find_tile's shift has it
constexpr int kPlainThreads = 256;
constexpr int kPs = kR + 4;    // row of a tile of scores, in floats

__device__ __forceinline__ void check_cu(const Problem& p) {
  if (p.cu64) validate_cu(static_cast<const int64_t*>(p.cu), p.N, p.BL, p.err);
  else validate_cu(static_cast<const int32_t*>(p.cu), p.N, p.BL, p.err);
}

// 64 rows of one head as floats; rows from `len` on and columns from `dim` on
// are zeros.  float32 rows at 16 bytes are copied four elements at a time, past
// the registers: `wait_tiles` comes before they are read.
template <typename T, int D>
__device__ __forceinline__ void load_tile(float* to, const Rows& r, int head, long long token, int len, int dim) {
  const T* src = static_cast<const T*>(r.p) + token * r.st + head * r.sh;
  if (sizeof(T) == 4 && dim % 4 == 0 && r.st % 4 == 0 && r.sh % 4 == 0 && (reinterpret_cast<uintptr_t>(r.p) & 15u) == 0) {
    const int d = threadIdx.x % (D / 4) * 4;
#pragma unroll
    for (int i = threadIdx.x / (D / 4); i < kR; i += kPlainThreads / (D / 4)) {
      const int bytes = i < len && d < dim ? 16 : 0;  // the rest of the sixteen is filled with zeros
      const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to + i * (D + 4) + d));
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(bytes ? src + i * r.st + d : src), "r"(bytes) : "memory");
    }
    return;
  }
  for (int e = threadIdx.x; e < kR * D; e += kPlainThreads) {
    const int i = e / D, d = e % D;
    to[i * (D + 4) + d] = i < len && d < dim ? to_f(src[i * r.st + d]) : 0.f;
  }
}
__device__ __forceinline__ void wait_tiles() {
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
}

// s[a][b] = x[row ty*4+a] . y[row tx+16b], two elements an instruction
template <int D>
__device__ __forceinline__ void dots(const float* x, const float* y, int tx, int ty, int dim, float (&s)[4][4]) {
  uint64_t acc[4][4];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = 0;
  const float* xr = x + ty * 4 * (D + 4);
  const float* yr = y + tx * (D + 4);
#pragma unroll 4
  for (int d = 0; d < dim; d += 4) {
    ulonglong2 u[4], v[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) u[a] = *reinterpret_cast<const ulonglong2*>(xr + a * (D + 4) + d);
#pragma unroll
    for (int b = 0; b < 4; ++b) v[b] = *reinterpret_cast<const ulonglong2*>(yr + 16 * b * (D + 4) + d);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[a][b] = fma2(u[a].y, v[b].y, fma2(u[a].x, v[b].x, acc[a][b]));
  }
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float2 f = unpair(acc[a][b]);
      s[a][b] = f.x + f.y;
    }
}

// acc[a][..] += sum_k w[row ty*4+a][k] y[k][..], columns tx*4 + 64 c, in pairs.
// With `causal` a row takes k up to its own only (what lies behind may be NaN).
template <int D, bool CAUSAL>
__device__ __forceinline__ void rows_times(const float* w, const float* y, int tx, int ty, uint64_t (&acc)[4][D / 32]) {
#pragma unroll 2
  for (int k = 0; k < kR; k += 4) {
    float4 p[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) p[a] = *reinterpret_cast<const float4*>(w + (ty * 4 + a) * kPs + k);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(y + (k + e) * (D + 4) + tx * 4 + 64 * c);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          if (CAUSAL && k + e > ty * 4 + a) continue;
          const float f = e == 0 ? p[a].x : (e == 1 ? p[a].y : (e == 2 ? p[a].z : p[a].w));
          const uint64_t f2 = pair(f, f);
          acc[a][2 * c] = fma2(f2, v.x, acc[a][2 * c]);
          acc[a][2 * c + 1] = fma2(f2, v.y, acc[a][2 * c + 1]);
        }
      }
  }
}

// acc[a][..] += sum_k w[k][column ty*4+a] y[k][..]; with `causal` a column
// takes k from its own on.
template <int D, bool CAUSAL>
__device__ __forceinline__ void columns_times(const float* w, const float* y, int tx, int ty, uint64_t (&acc)[4][D / 32]) {
#pragma unroll 4
  for (int k = 0; k < kR; ++k) {
    const float4 p = *reinterpret_cast<const float4*>(w + k * kPs + ty * 4);
    const uint64_t f[4] = {pair(p.x, p.x), pair(p.y, p.y), pair(p.z, p.z), pair(p.w, p.w)};
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(y + k * (D + 4) + tx * 4 + 64 * c);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        if (CAUSAL && k < ty * 4 + a) continue;
        acc[a][2 * c] = fma2(f[a], v.x, acc[a][2 * c]);
        acc[a][2 * c + 1] = fma2(f[a], v.y, acc[a][2 * c + 1]);
      }
    }
  }
}

template <typename T, int D>
__device__ __forceinline__ void store_rows(void* to, int head, int heads, long long token, int len, int dim, int tx, int ty,
                                           const uint64_t (&acc)[4][D / 32], const float (&f)[4]) {
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    if (ty * 4 + a >= len) continue;
    T* row = static_cast<T*>(to) + ((token + ty * 4 + a) * heads + head) * dim;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const float2 x = unpair(acc[a][c]);
      const int d = tx * 4 + 64 * (c / 2) + 2 * (c % 2);
      if (d < dim) row[d] = from_f<T>(x.x * f[a]);
      if (d + 1 < dim) row[d + 1] = from_f<T>(x.y * f[a]);
    }
  }
}

// Over the 16 threads of a row.
__device__ __forceinline__ float row_max(float x) {
#pragma unroll
  for (int o = 8; o > 0; o /= 2) x = fmaxf(x, __shfl_xor_sync(kFull, x, o));
  return x;
}
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = 8; o > 0; o /= 2) x += __shfl_xor_sync(kFull, x, o);
  return x;
}

template <int D>
constexpr size_t plain_smem(int tiles, int scores) {
  return sizeof(float) * (static_cast<size_t>(tiles) * kR * (D + 4) + static_cast<size_t>(scores) * kR * kPs);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPlainThreads) forward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float plain_smem_base[];
  float *qs = plain_smem_base, *ks = qs + kR * (D + 4), *vs = ks + kR * (D + 4), *ps = vs + kR * (D + 4);
  const int h = blockIdx.y, hk = h / p.share, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  if (blockIdx.x == 0 && h == 0) check_cu(p);
  zero_outside<T>(p, p.out, h, p.H, p.dv, blockIdx.x, kR, threadIdx.x, blockDim.x);
  const Tile t = find_tile<6>(p, gridDim.x - 1 - blockIdx.x);  // long rows first
  if (t.first < 0) return;
  const int len = min(kR, t.len - t.first);
  load_tile<T, D>(qs, p.q, h, t.start + t.first, len, p.dk);
  uint64_t acc[4][D / 32];
  float l[4], m[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    l[a] = 0.f, m[a] = -INFINITY;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) acc[a][c] = 0;
  }
  const float c2 = p.scale * kLog2e;
  for (int j = 0; j <= t.first; j += kR) {
    const bool own = j == t.first;
    __syncthreads();
    load_tile<T, D>(ks, p.k, hk, t.start + j, own ? len : kR, p.dk);
    load_tile<T, D>(vs, p.v, hk, t.start + j, own ? len : kR, p.dv);
    wait_tiles();
    float s[4][4];
    dots<D>(qs, ks, tx, ty, p.dk, s);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        s[a][b] = own && tx + 16 * b > ty * 4 + a ? -INFINITY : s[a][b] * c2;
        top = fmaxf(top, s[a][b]);
      }
      top = fmaxf(m[a], row_max(top));
      const float ref = top == -INFINITY ? 0.f : top;  // a row of -inf so far
      const float keep = exp2f(m[a] - ref);
      m[a] = top;
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        s[a][b] = exp2f(s[a][b] - ref);
        sum += s[a][b];
        ps[(ty * 4 + a) * kPs + tx + 16 * b] = s[a][b];
      }
      l[a] = fmaf(l[a], keep, row_sum(sum));
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[a][c] = mul2(acc[a][c], pair(keep, keep));
    }
    __syncwarp();  // a warp's rows of the scores are its own
    if (own) rows_times<D, true>(ps, vs, tx, ty, acc);
    else rows_times<D, false>(ps, vs, tx, ty, acc);
  }
  float f[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    f[a] = 1.f / l[a];
    if (p.lse && tx == 0 && ty * 4 + a < len) p.lse[h * p.BL + t.start + t.first + ty * 4 + a] = m[a] + log2f(l[a]);
  }
  store_rows<T, D>(p.out, h, p.H, t.start + t.first, len, p.dv, tx, ty, acc, f);
  if (p.rest) {
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const float2 x = unpair(acc[a][c]);
        acc[a][c] = pair(x.x * f[a] - to_f(from_f<T>(x.x * f[a])), x.y * f[a] - to_f(from_f<T>(x.y * f[a])));
      }
    const float one[4] = {1.f, 1.f, 1.f, 1.f};
    store_rows<T, D>(p.rest, h, p.H, t.start + t.first, len, p.dv, tx, ty, acc, one);
  }
}

// d = do.o.  Memory bounds it: sixteen lanes a row with sixteen bytes each where
// alignment allows (vec), eight rows in flight for a warp; else a warp per row.
template <typename T>
__global__ void __launch_bounds__(kPlainThreads) dot_kernel(const __grid_constant__ Problem p, int vec) {
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0) check_cu(p);
  const long long warp = (static_cast<long long>(blockIdx.x) * kPlainThreads + threadIdx.x) >> 5;
  const long long warps = static_cast<long long>(gridDim.x) * (kPlainThreads / 32);
  const long long units = p.BL * p.H;
  float top = 0.f, top_v = 0.f;  // the largest finite |do| and |v| of the sequences' rows, where asked for
  const long long begin = cu_at(p, 0), end = cu_at(p, p.N);
  auto note = [&](float& top, long long t, float x) {
    x = fabsf(x);
    if (x < INFINITY && t >= begin && t < end) top = fmaxf(top, x);
  };
  const T *g = static_cast<const T*>(p.d_out.p), *o = static_cast<const T*>(p.out), *r = static_cast<const T*>(p.rest);
  if (vec) {
    constexpr int V = 16 / sizeof(T), ROWS = 4;
    const int gl = lane & 15;
    const long long first = warp * 2 * ROWS, step = warps * 2 * ROWS;
    // token and head of the warp's first row, moved on without divisions
    long long t0 = first / p.H;
    int h0 = static_cast<int>(first % p.H);
    const long long step_t = step / p.H;
    const int step_h = static_cast<int>(step % p.H);
    for (long long u0 = first; u0 < units; u0 += step, t0 += step_t, h0 += step_h) {
      if (h0 >= p.H) h0 -= p.H, ++t0;
      long long t[ROWS];
      int h[ROWS];
#pragma unroll
      for (int e = 0; e < ROWS; ++e) {
        t[e] = t0, h[e] = h0 + 2 * e + (lane >> 4);
        while (h[e] >= p.H) h[e] -= p.H, ++t[e];
      }
      uint4 x[ROWS], y[ROWS], z[ROWS];
      const int parts = p.dv > 16 * V ? 2 : 1;  // a row of 128 floats is two rounds
      float sum[ROWS] = {};
      for (int part = 0; part < parts; ++part) {
        const int d = part * 16 * V + gl * V;
#pragma unroll
        for (int e = 0; e < ROWS; ++e) {
          const long long u = u0 + 2 * e + (lane >> 4);
          x[e] = y[e] = z[e] = make_uint4(0, 0, 0, 0);
          if (u < units && d < p.dv) {
            x[e] = __ldcs(reinterpret_cast<const uint4*>(g + t[e] * p.d_out.st + h[e] * p.d_out.sh + d));
            y[e] = __ldcs(reinterpret_cast<const uint4*>(o + u * p.dv + d));
            if (r) z[e] = __ldcs(reinterpret_cast<const uint4*>(r + u * p.dv + d));
          }
        }
#pragma unroll
        for (int e = 0; e < ROWS; ++e) {
          const T *a = reinterpret_cast<const T*>(&x[e]), *b = reinterpret_cast<const T*>(&y[e]), *c = reinterpret_cast<const T*>(&z[e]);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            sum[e] = fmaf(to_f(a[i]), to_f(b[i]) + to_f(c[i]), sum[e]);
            if (std::is_same<T, __half>::value) note(top, t[e], to_f(a[i]));
          }
        }
      }
#pragma unroll
      for (int e = 0; e < ROWS; ++e) {
#pragma unroll
        for (int i = 8; i > 0; i /= 2) sum[e] += __shfl_xor_sync(kFull, sum[e], i);
        const long long u = u0 + 2 * e + (lane >> 4);
        if (gl == 0 && u < units) p.d[h[e] * p.BL + t[e]] = sum[e];
      }
    }
  } else {
    for (long long u = warp; u < units; u += warps) {
      const long long t = u / p.H;
      const int h = static_cast<int>(u % p.H);
      float x = 0.f;
      for (int d = lane; d < p.dv; d += 32) {
        const float y = to_f(g[t * p.d_out.st + h * p.d_out.sh + d]);
        x = fmaf(y, to_f(o[u * p.dv + d]) + (r ? to_f(r[u * p.dv + d]) : 0.f), x);
        note(top, t, y);
      }
#pragma unroll
      for (int e = 16; e > 0; e /= 2) x += __shfl_xor_sync(kFull, x, e);
      if (lane == 0) p.d[h * p.BL + t] = x;
    }
  }
  if constexpr (std::is_same<T, __half>::value) {  // a maximum does not depend on the order
    if (!p.top) return;
    constexpr int V = 16 / sizeof(T);
    const int heads = p.H / p.share, d = (lane & 15) * V;
#pragma unroll 4
    for (long long u = warp * 2 + (lane >> 4); u < p.BL * heads; u += warps * 2) {
      if (d >= p.dv) continue;
      const long long t = u / heads;
      const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.v.p) + t * p.v.st + u % heads * p.v.sh + d);
#pragma unroll
      for (int i = 0; i < V; ++i) note(top_v, t, to_f(reinterpret_cast<const T*>(&x)[i]));
    }
    const uint32_t bits = __reduce_max_sync(kFull, __float_as_uint(top)), bits_v = __reduce_max_sync(kFull, __float_as_uint(top_v));
    if (lane == 0) atomicMax(p.top, bits), atomicMax(p.top + 1, bits_v);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kPlainThreads) dq_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float plain_smem_base[];
  constexpr int S = kR * (D + 4);
  float *qs = plain_smem_base, *gs = qs + S, *ks = gs + S, *vs = ks + S, *ps = vs + S;
  const int h = blockIdx.y, hk = h / p.share, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  zero_outside<T>(p, p.d_q, h, p.H, p.dk, blockIdx.x, kR, threadIdx.x, blockDim.x);
  const Tile t = find_tile<6>(p, gridDim.x - 1 - blockIdx.x);
  if (t.first < 0) return;
  const int len = min(kR, t.len - t.first);
  const long long at = t.start + t.first;
  load_tile<T, D>(qs, p.q, h, at, len, p.dk);
  load_tile<T, D>(gs, p.d_out, h, at, len, p.dv);
  uint64_t acc[4][D / 32];
  float lse[4], d[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const bool in = ty * 4 + a < len;
    lse[a] = in ? p.lse[h * p.BL + at + ty * 4 + a] : 0.f;
    d[a] = in ? p.d[h * p.BL + at + ty * 4 + a] : 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) acc[a][c] = 0;
  }
  const float c2 = p.scale * kLog2e;
  for (int j = 0; j <= t.first; j += kR) {
    const bool own = j == t.first;
    __syncthreads();
    load_tile<T, D>(ks, p.k, hk, t.start + j, own ? len : kR, p.dk);
    load_tile<T, D>(vs, p.v, hk, t.start + j, own ? len : kR, p.dv);
    wait_tiles();
    float s[4][4], g[4][4];
    dots<D>(qs, ks, tx, ty, p.dk, s);
    dots<D>(gs, vs, tx, ty, p.dv, g);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b)  // a sequence's first token sees one key, with p = 1: no ds, not even a rounding
        ps[(ty * 4 + a) * kPs + tx + 16 * b] =
            own && tx + 16 * b > ty * 4 + a ? 0.f : exp2f(fmaf(s[a][b], c2, -lse[a])) * (g[a][b] - d[a]) * (t.first + ty * 4 + a == 0 ? 0.f : 1.f);
    __syncwarp();
    if (own) rows_times<D, true>(ps, ks, tx, ty, acc);
    else rows_times<D, false>(ps, ks, tx, ty, acc);
  }
  const float f[4] = {p.scale, p.scale, p.scale, p.scale};
  store_rows<T, D>(p.d_q, h, p.H, at, len, p.dk, tx, ty, acc, f);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPlainThreads) dkdv_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float plain_smem_base[];
  constexpr int S = kR * (D + 4);
  float *ks = plain_smem_base, *vs = ks + S, *qs = vs + S, *gs = qs + S, *ps = gs + S, *ds = ps + kR * kPs;
  const int hk = blockIdx.y, heads = p.H / p.share, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  zero_outside<T>(p, p.d_k, hk, heads, p.dk, blockIdx.x, kR, threadIdx.x, blockDim.x);
  zero_outside<T>(p, p.d_v, hk, heads, p.dv, blockIdx.x, kR, threadIdx.x, blockDim.x);
  const Tile t = find_tile<6>(p, blockIdx.x);  // a sequence's first keys have the most queries
  if (t.first < 0) return;
  const int len = min(kR, t.len - t.first);
  const long long at = t.start + t.first;
  load_tile<T, D>(ks, p.k, hk, at, len, p.dk);
  load_tile<T, D>(vs, p.v, hk, at, len, p.dv);
  uint64_t dk[4][D / 32], dv[4][D / 32];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dk[a][c] = dv[a][c] = 0;
  const float c2 = p.scale * kLog2e;
  for (int g = 0; g < p.share; ++g) {
    const int h = hk * p.share + g;
    for (int i = t.first; i < t.len; i += kR) {
      const bool own = i == t.first;
      const int n = min(kR, t.len - i);
      __syncthreads();
      load_tile<T, D>(qs, p.q, h, t.start + i, n, p.dk);
      load_tile<T, D>(gs, p.d_out, h, t.start + i, n, p.dv);
      wait_tiles();
      float s[4][4], e[4][4];
      dots<D>(qs, ks, tx, ty, p.dk, s);
      dots<D>(gs, vs, tx, ty, p.dv, e);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int row = ty * 4 + a;
        const float lse = row < n ? p.lse[h * p.BL + t.start + i + row] : 0.f;
        const float d = row < n ? p.d[h * p.BL + t.start + i + row] : 0.f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const bool off = row >= n || (own && tx + 16 * b > row);
          const float x = off ? 0.f : exp2f(fmaf(s[a][b], c2, -lse));
          ps[row * kPs + tx + 16 * b] = x;
          ds[row * kPs + tx + 16 * b] = off ? 0.f : x * (e[a][b] - d) * (i + row == 0 ? 0.f : 1.f);
        }
      }
      __syncthreads();
      if (own) {
        columns_times<D, true>(ps, gs, tx, ty, dv);
        columns_times<D, true>(ds, qs, tx, ty, dk);
      } else {
        columns_times<D, false>(ps, gs, tx, ty, dv);
        columns_times<D, false>(ds, qs, tx, ty, dk);
      }
    }
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f}, f[4] = {p.scale, p.scale, p.scale, p.scale};
  store_rows<T, D>(p.d_v, hk, heads, at, len, p.dv, tx, ty, dv, one);
  store_rows<T, D>(p.d_k, hk, heads, at, len, p.dk, tx, ty, dk, f);
}

template <typename T, int D>
static int plain_forward(const Problem& p, cudaStream_t s) {
  static std::atomic<unsigned long long> done{};
  const size_t bytes = plain_smem<D>(3, 1);
  const int rc = allow_smem(forward_kernel<T, D>, bytes, done);
  if (rc != ASCAN_OK) return rc;
  forward_kernel<T, D><<<dim3(tile_bound(p, kR), p.H), kPlainThreads, bytes, s>>>(p);
  return launch_status();
}

template <typename T, int D>
static int plain_backward(const Problem& p, cudaStream_t s) {
  static std::atomic<unsigned long long> done[2]{};
  const size_t q_bytes = plain_smem<D>(4, 1), k_bytes = plain_smem<D>(4, 2);
  int rc = allow_smem(dq_kernel<T, D>, q_bytes, done[0]);
  if (rc == ASCAN_OK) rc = allow_smem(dkdv_kernel<T, D>, k_bytes, done[1]);
  if (rc != ASCAN_OK) return rc;
  dq_kernel<T, D><<<dim3(tile_bound(p, kR), p.H), kPlainThreads, q_bytes, s>>>(p);
  rc = launch_status();
  if (rc != ASCAN_OK) return rc;
  dkdv_kernel<T, D><<<dim3(tile_bound(p, kR), p.H / p.share), kPlainThreads, k_bytes, s>>>(p);
  return launch_status();
}

template <typename T>
static int run_forward(const Problem& p, cudaStream_t s) {
  return max(p.dk, p.dv) <= 64 ? plain_forward<T, 64>(p, s) : plain_forward<T, 128>(p, s);
}

template <typename T>
static int run_backward(const Problem& p, bool tc, int dtype, cudaStream_t s) {
  const long long ctas = (p.BL * p.H + kPlainThreads / 32 - 1) / (kPlainThreads / 32);
  constexpr int v = 16 / sizeof(T);
  auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
  const bool vec = p.dv % v == 0 && p.d_out.st % v == 0 && p.d_out.sh % v == 0 && aligned(p.d_out.p) && aligned(p.out) && aligned(p.rest);
  if (p.top && cudaMemsetAsync(p.top, 0, 2 * sizeof(uint32_t), s) != cudaSuccess) return ASCAN_ECUDA;
  dot_kernel<T><<<static_cast<unsigned>(min(ctas, 148ll * 16)), kPlainThreads, 0, s>>>(p, vec);
  const int rc = launch_status();
  if (rc != ASCAN_OK) return rc;
  if (tc) return tc_backward(p, dtype, s);
  return max(p.dk, p.dv) <= 64 ? plain_backward<T, 64>(p, s) : plain_backward<T, 128>(p, s);
}

static int fill(Problem& p, const ascan_rows* q, const ascan_rows* k, const ascan_rows* v, const void* cu, int cu_type,
                int64_t N, int64_t BL, int dk, int dv, int dtype, float scale) {
  if (N < 0 || BL < 0 || BL > ASCAN_ATTENTION_MAX_TOKENS || N > ASCAN_ATTENTION_MAX_TOKENS) return ASCAN_EINVAL;
  if (dk <= 0 || dv <= 0 || dk > ASCAN_ATTENTION_MAX_DIM || dv > ASCAN_ATTENTION_MAX_DIM) return ASCAN_EINVAL;
  if (dtype < ASCAN_F32 || dtype > ASCAN_BF16 || (cu_type != ASCAN_I32 && cu_type != ASCAN_I64)) return ASCAN_EINVAL;
  if (!(scale > 0.f) || !(scale < INFINITY)) return ASCAN_EINVAL;
  if (N == 0 || BL == 0) return ASCAN_OK;
  const ascan_rows* r[3] = {q, k, v};
  for (const ascan_rows* x : r)
    if (!x || !x->data || x->heads <= 0 || x->heads > 65535 || x->stride_token < 0 || x->stride_head < 0) return ASCAN_EINVAL;
  if (!cu || k->heads != v->heads || q->heads % k->heads) return ASCAN_EINVAL;
  p.q = Rows{q->data, q->stride_token, q->stride_head, 1};
  p.k = Rows{k->data, k->stride_token, k->stride_head, 1};
  p.v = Rows{v->data, v->stride_token, v->stride_head, 1};
  p.cu = cu;
  p.cu64 = cu_type == ASCAN_I64;
  p.H = q->heads;
  p.share = q->heads / k->heads;
  p.dk = dk;
  p.dv = dv;
  p.N = N;
  p.BL = BL;
  p.scale = scale;
  p.err = g_err_host;
  return ASCAN_OK;
}

}  // namespace attend
}  // namespace ascan

using namespace ascan;

extern "C" {

int ascan_attention_forward(const ascan_rows* queries, const ascan_rows* keys, const ascan_rows* values,
                            const void* cu_seqlens, int cu_index_type, int64_t num_seq, int64_t seq_total, int key_dim,
                            int value_dim, int dtype, float scale, void* out, void* out_rest, float* lse, void* stream) {
  attend::Problem p{};
  const int rc = attend::fill(p, queries, keys, values, cu_seqlens, cu_index_type, num_seq, seq_total, key_dim, value_dim,
                              dtype, scale);
  if (rc != ASCAN_OK || num_seq == 0 || seq_total == 0) return rc;
  if (!out || (dtype != ASCAN_F32 && !out_rest != !lse)) return ASCAN_EINVAL;
  p.out = out;
  p.rest = dtype == ASCAN_F32 ? nullptr : out_rest;
  p.lse = lse;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (attend::tc_usable(p, dtype, false)) return attend::tc_forward(p, dtype, s);
  if (dtype == ASCAN_F32) return attend::run_forward<float>(p, s);
  if (dtype == ASCAN_F16) return attend::run_forward<__half>(p, s);
  return attend::run_forward<__nv_bfloat16>(p, s);
}

size_t ascan_attention_workspace(int64_t seq_total, int query_heads) {
  if (seq_total <= 0 || query_heads <= 0) return 256;
  return 512 + sizeof(float) * static_cast<size_t>(seq_total) * query_heads;
}

int ascan_attention_backward(const ascan_rows* queries, const ascan_rows* keys, const ascan_rows* values,
                             const ascan_rows* d_out, const void* out, const void* out_rest, const float* lse,
                             const void* cu_seqlens, int cu_index_type, int64_t num_seq, int64_t seq_total, int key_dim,
                             int value_dim, int dtype, float scale, void* d_queries, void* d_keys, void* d_values,
                             void* workspace, size_t workspace_bytes, void* stream) {
  attend::Problem p{};
  const int rc = attend::fill(p, queries, keys, values, cu_seqlens, cu_index_type, num_seq, seq_total, key_dim, value_dim,
                              dtype, scale);
  if (rc != ASCAN_OK || num_seq == 0 || seq_total == 0) return rc;
  if (!d_out || !d_out->data || d_out->heads != queries->heads || d_out->stride_token < 0 || d_out->stride_head < 0 ||
      !out || !lse || !d_queries || !d_keys || !d_values)
    return ASCAN_EINVAL;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) ||
      workspace_bytes < ascan_attention_workspace(seq_total, queries->heads))
    return ASCAN_EWORKSPACE;
  p.d_out = mscan::Rows{d_out->data, d_out->stride_token, d_out->stride_head, 1};
  p.out = const_cast<void*>(out);
  p.rest = dtype == ASCAN_F32 ? nullptr : const_cast<void*>(out_rest);
  p.lse = const_cast<float*>(lse);
  p.d = static_cast<float*>(workspace) + 64;
  p.d_q = d_queries;
  p.d_k = d_keys;
  p.d_v = d_values;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool tc = attend::tc_usable(p, dtype, true);
  p.top = tc && dtype == ASCAN_F16 ? static_cast<uint32_t*>(workspace) : nullptr;
  if (dtype == ASCAN_F32) return attend::run_backward<float>(p, tc, dtype, s);
  if (dtype == ASCAN_F16) return attend::run_backward<__half>(p, tc, dtype, s);
  return attend::run_backward<__nv_bfloat16>(p, tc, dtype, s);
}

}  // extern "C"

namespace ascan {
ASCAN_UNIT_ERROR_ACCESSORS(attend)
}  // namespace ascan
