// ascan_mscan.cu -- compilation unit of the scan library: the matrix-state
// recurrence (ascan_mscan.cuh has the mathematics), its plain kernel for
// every type and head size, the carry chain, the gate gradients, the sums
// over shared heads, and the one-token step.
#include "ascan_impl.cuh"
#include "ascan_mscan.cuh"
#include "ascan_mscan_common.cuh"

namespace ascan {
namespace mscan {

constexpr int kPlainThreads = 256;
constexpr int kPlainChunk = 64;

// ---------------------------------------------------------------------------
// The plain kernel: one CTA per (segment, head, form), float32 fused
// multiply-adds, for float32, float16 and what the tensor-core kernel does not
// take.  A chunk of 64 tokens lies in shared memory, A and B with the tokens
// along the rows' unit stride, C as stored; the state stays there from chunk
// to chunk.  Every product gives a thread a tile of 4 x 4 values (8 x 4 at 128
// wide), so two (three) 16-byte reads feed 16 (32) multiply-adds.  Measured at
// 6001 tokens of 12 heads of 64 x 64, float32, forward and gradients: 668 us,
// 0.19 of the multiply-add rate (9.4 GFLOP); tiles are loaded without overlap,
// and three CTAs an SM hide it in part (two took a ninth longer, tiles of 2 x 4
// over 32 tokens twice as long).
// ---------------------------------------------------------------------------

template <int DM>
struct PlainSmem {
  static constexpr int kLt = kPlainChunk + 4, kLd = DM + 4;
  float s[DM * DM];
  float at[DM * kLt];          // [dim][token]; then the masked scores, [column token][row token]
  float bt[DM * kLt];          // [dim][token]
  float c[kPlainChunk * kLd];  // [token][dim]
  double g[kPlainChunk];
  float row[kPlainChunk], col[kPlainChunk];
  float total;
};

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }

// acc += x (a row of four values)
__device__ __forceinline__ void fma4(float* acc, float x, const float4& y) {
  acc[0] = fmaf(x, y.x, acc[0]);
  acc[1] = fmaf(x, y.y, acc[1]);
  acc[2] = fmaf(x, y.z, acc[2]);
  acc[3] = fmaf(x, y.w, acc[3]);
}

// Four elements of a row, zero beyond dim.
template <typename T>
__device__ __forceinline__ float4 row4(const T* p, int d, int dim, bool vec) {
  if (vec && d + 4 <= dim) {
    if (sizeof(T) == 4) return *reinterpret_cast<const float4*>(p + d);
    const uint2 u = *reinterpret_cast<const uint2*>(p + d);
    const T* e = reinterpret_cast<const T*>(&u);
    return make_float4(to_f(e[0]), to_f(e[1]), to_f(e[2]), to_f(e[3]));
  }
  return make_float4(d < dim ? to_f(p[d]) : 0.f, d + 1 < dim ? to_f(p[d + 1]) : 0.f, d + 2 < dim ? to_f(p[d + 2]) : 0.f,
                     d + 3 < dim ? to_f(p[d + 3]) : 0.f);
}

template <typename T>
__device__ __forceinline__ bool rows_aligned(const Rows& r) {
  return (reinterpret_cast<uintptr_t>(r.p) % (4 * sizeof(T))) == 0 && r.st % 4 == 0 && r.sh % 4 == 0;
}

// Tokens along the unit stride: a lane takes one token, so the stores spread
// over the banks.
template <typename T, int DM>
__device__ __forceinline__ void load_turned(float* dst, const Rows& r, long long t0, int len, int h, int dim) {
  constexpr int LT = PlainSmem<DM>::kLt, THREADS = kPlainThreads;
  const bool vec = rows_aligned<T>(r);
  const T* base = static_cast<const T*>(r.p) + t0 * r.st + (h / r.share) * r.sh;
#pragma unroll 4
  for (int e = threadIdx.x; e < kPlainChunk * DM / 4; e += THREADS) {
    const int t = e % kPlainChunk, d = e / kPlainChunk * 4;
    const float4 x = t < len ? row4(base + t * r.st, d, dim, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
    dst[d * LT + t] = x.x;
    dst[(d + 1) * LT + t] = x.y;
    dst[(d + 2) * LT + t] = x.z;
    dst[(d + 3) * LT + t] = x.w;
  }
}

template <typename T, int DM>
__device__ __forceinline__ void load_rows(float* dst, const Rows& r, long long t0, int len, int h, int dim) {
  constexpr int LD = PlainSmem<DM>::kLd, THREADS = kPlainThreads;
  const bool vec = rows_aligned<T>(r);
  const T* base = static_cast<const T*>(r.p) + t0 * r.st + (h / r.share) * r.sh;
#pragma unroll 4
  for (int e = threadIdx.x; e < kPlainChunk * DM / 4; e += THREADS) {
    const int t = e / (DM / 4), d = e % (DM / 4) * 4;
    *reinterpret_cast<float4*>(dst + t * LD + d) =
        t < len ? row4(base + t * r.st, d, dim, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

template <typename T, int DM>
__global__ void __launch_bounds__(kPlainThreads, DM == 64 ? 3 : 1)
    plain_kernel(const __grid_constant__ Launch L, const bool state_only) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  using Sm = PlainSmem<DM>;
  Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
  constexpr int LT = Sm::kLt, LD = Sm::kLd, THREADS = kPlainThreads;
  constexpr int TX = DM / 4;             // threads along the values, four each
  constexpr int R = TX * kPlainChunk / THREADS;  // rows per thread: 4 or 8
  const Problem& p = L.p;
  const Form& f = L.f[blockIdx.z];
  const int tid = threadIdx.x, j = blockIdx.x, h = blockIdx.y;
  const bool rev = f.rev != 0;
  const int da = f.da, dc = f.dc;
  const long long mat = static_cast<long long>(da) * dc;
  const long long t0 = j * p.seg, t1 = min(t0 + p.seg, p.BL);
  const int tx = tid % TX, ty = tid / TX, d0 = tx * 4, r0 = ty * R;

  if (!state_only) fill_outside<T>(p, f);

  const long long n_first = first_beyond(p, t0);
  const long long n_last = first_from(p, t1);  // one past the last sequence that starts before t1
  for (long long m = 0; m < n_last - n_first; ++m) {
    const long long n = rev ? n_last - 1 - m : n_first + m;
    const long long b0 = cu_at(p, n), b1 = cu_at(p, n + 1);
    const long long ps = max(b0, t0), pe = min(b1, t1);
    if (pe <= ps) continue;
    const bool from_start = rev ? pe == b1 : ps == b0;  // the state begins in this piece
    const bool to_end = rev ? ps == b0 : pe == b1;      // ... and ends in it
    if (state_only && to_end) continue;
    const float* from = from_start ? (f.init ? f.init + (n * p.H + h) * mat : nullptr)
                                   : f.carry + (static_cast<long long>(rev ? j + 1 : j - 1) * p.H + h) * mat;
    const bool zero = from == nullptr || (state_only && !from_start);
    const long long fi = from_start ? f.si : dc, fj = from_start ? f.sj : 1;
    for (int e = tid; e < DM * DM; e += THREADS) {
      const int i = e / DM, d = e % DM;
      sm.s[e] = (!zero && i < da && d < dc) ? from[i * fi + d * fj] : 0.f;
    }
    const int chunks = static_cast<int>((pe - ps + kPlainChunk - 1) / kPlainChunk);
    float decay = 1.f;
    for (int cc = 0; cc < chunks; ++cc) {
      const long long s0 = ps + static_cast<long long>(rev ? chunks - 1 - cc : cc) * kPlainChunk;
      const int len = static_cast<int>(min(static_cast<long long>(kPlainChunk), pe - s0));
      __syncthreads();
      if (f.snap && !state_only) {
        const long long at = rev ? s0 + len : s0;
        if (at > ps && at < pe && (at - ps) % p.restart == 0)
          for (int e = tid; e < mat; e += THREADS)
            f.snap[(snap_slot(p, at) * p.H + h) * mat + e] = sm.s[(e / dc) * DM + e % dc];
      }
      if (!state_only) load_turned<T, DM>(sm.at, f.a, s0, len, h, da);
      load_turned<T, DM>(sm.bt, f.b, s0, len, h, da);
      load_rows<T, DM>(sm.c, f.c, s0, len, h, dc);
      if (tid < 32) {
        const double g0 = 2 * tid < len ? static_cast<double>(load_gate(p, s0 + 2 * tid, h)) : 0.0;
        const double g1 = 2 * tid + 1 < len ? static_cast<double>(load_gate(p, s0 + 2 * tid + 1, h)) : 0.0;
        // sums in the scan's direction (backwards of all later tokens), never
        // differences of longer ones: a gate that is not finite must not reach
        // the tokens before it
        double inc = g0 + g1;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const double u = rev ? __shfl_down_sync(kFull, inc, o) : __shfl_up_sync(kFull, inc, o);
          if (rev ? tid + o < 32 : tid >= o) inc += u;
        }
        const double end = __shfl_sync(kFull, inc, rev ? 0 : 31);
        double before = rev ? __shfl_down_sync(kFull, inc, 1) : __shfl_up_sync(kFull, inc, 1);
        if (tid == (rev ? 31 : 0)) before = 0.0;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const double g = rev ? (q ? before : before + g1) : (q ? inc : before + g0);
          sm.g[2 * tid + q] = g;
          sm.row[2 * tid + q] = expf(static_cast<float>(g)) * f.sr;
          sm.col[2 * tid + q] = expf(static_cast<float>(end - g)) * f.sc;
        }
        if (tid == 31) sm.total = expf(static_cast<float>(end));
      }
      __syncthreads();
      if (!state_only) {
        // scores: 4 rows by 4 columns; blocks outside the mask are zero
        const int sr0 = (tid / 16) * 4, sc0 = (tid % 16) * 4;
        float sacc[4][4] = {};
        if (rev ? sc0 + 3 >= sr0 : sc0 <= sr0 + 3) {
#pragma unroll 4
          for (int d = 0; d < da; ++d) {
            const float4 y = ld4(&sm.bt[d * LT + sc0]);
            const float4 x = ld4(&sm.at[d * LT + sr0]);
            fma4(sacc[0], x.x, y);
            fma4(sacc[1], x.y, y);
            fma4(sacc[2], x.z, y);
            fma4(sacc[3], x.w, y);
          }
        }
        float acc[R][4] = {};
        // acc += (R values of a row of x) times (four values of y)
        auto outer = [&](const float* x, const float4& y) {
#pragma unroll
          for (int q = 0; q < R; q += 4) {
            const float4 v = ld4(x + q);
            fma4(acc[q], v.x, y), fma4(acc[q + 1], v.y, y), fma4(acc[q + 2], v.z, y), fma4(acc[q + 3], v.w, y);
          }
        };
#pragma unroll 4
        for (int i = 0; i < da; ++i) outer(&sm.at[i * LT + r0], ld4(&sm.s[i * DM + d0]));
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[r][q] *= sm.row[r0 + r];
        __syncthreads();  // A has been read: the scores take its place
        float* pt = sm.at;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = sr0 + e, at = sc0 + c;
            const bool on = (rev ? at >= r : at <= r) && at < len;
            const double dg = sm.g[r] - sm.g[at];
            v[e] = on ? sacc[e][c] * f.sp * expf(static_cast<float>(dg)) : 0.f;
          }
          *reinterpret_cast<float4*>(&pt[(sc0 + c) * LT + sr0]) = make_float4(v[0], v[1], v[2], v[3]);
        }
        __syncthreads();
        // columns before (after) the thread's rows meet all of them
        const int c_from = rev ? r0 + R : 0, c_to = rev ? len : min(r0, len);
#pragma unroll 4
        for (int c = c_from; c < c_to; ++c) outer(&pt[c * LT + r0], ld4(&sm.c[c * LD + d0]));
        // the columns of the rows themselves: masked ones are left out, not
        // multiplied by zero, so that a NaN there reaches no row; a row's own
        // comes after the dots, which leave it out
#pragma unroll
        for (int q = 0; q < R; ++q) {
          if (r0 + q >= len) continue;
          const float4 y = ld4(&sm.c[(r0 + q) * LD + d0]);
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (rev ? q > r : q < r) fma4(acc[r], pt[(r0 + q) * LT + r0 + r], y);
        }
        const bool vec = dc % 4 == 0 && (reinterpret_cast<uintptr_t>(f.out) & 15u) == 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const bool on = r0 + r < len;
          const long long t = s0 + r0 + r, at = (t * p.H + h) * dc + d0;
          float dot = 0.f;
          if (f.rowdot && on && d0 < dc) {
            const T* x = static_cast<const T*>(f.dot.p) + t * f.dot.st + (h / f.dot.share) * f.dot.sh;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (d0 + q < dc) dot = fmaf(acc[r][q], to_f(x[d0 + q]), dot);
          }
          if (on) fma4(acc[r], pt[(r0 + r) * LT + r0 + r], ld4(&sm.c[(r0 + r) * LD + d0]));
          if (on && d0 < dc) {
            if (vec && (f.out_f32 || sizeof(T) == 4)) {
              *reinterpret_cast<float4*>(static_cast<float*>(f.out) + at) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (d0 + q < dc) {
                  if (f.out_f32) static_cast<float*>(f.out)[at + q] = acc[r][q];
                  else static_cast<T*>(f.out)[at + q] = from_f<T>(acc[r][q]);
                }
            }
          }
          if (f.rowdot) {
#pragma unroll
            for (int o = TX / 2; o > 0; o /= 2) dot += __shfl_xor_sync(kFull, dot, o);
            if (on && tx == 0) f.rowdot[h * p.BL + t] = dot;
          }
        }
      }
      {  // the update: R rows a pass, four tokens a step
        const float total = sm.total;
        decay *= total;
        if (!state_only) __syncthreads();  // every thread has read the old state
        for (int i0 = ty * R; i0 < DM; i0 += kPlainChunk) {
          float st[R][4] = {};
#pragma unroll 2
          for (int c = 0; c < len; c += 4) {  // rows past the end are zero in both operands
            const float4 k = ld4(&sm.col[c]);
            float4 y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q] = ld4(&sm.c[(c + q) * LD + d0]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const float4 x = ld4(&sm.bt[(i0 + r) * LT + c]);
              fma4(st[r], x.x * k.x, y[0]);
              fma4(st[r], x.y * k.y, y[1]);
              fma4(st[r], x.z * k.z, y[2]);
              fma4(st[r], x.w * k.w, y[3]);
            }
          }
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float4* to = reinterpret_cast<float4*>(&sm.s[(i0 + r) * DM + d0]);
            const float4 o = *to;
            *to = make_float4(fmaf(total, o.x, st[r][0]), fmaf(total, o.y, st[r][1]), fmaf(total, o.z, st[r][2]),
                              fmaf(total, o.w, st[r][3]));
          }
        }
      }
    }
    __syncthreads();
    if (state_only) {
      float* to = f.carry + (static_cast<long long>(j) * p.H + h) * mat;
      for (int e = tid; e < mat; e += THREADS) to[e] = sm.s[(e / dc) * DM + e % dc];
      // a piece that holds the sequence's start takes nothing from before
      if (tid == 0) f.dec[j * p.H + h] = from_start ? -1.f : decay;
    } else if (to_end && f.fin) {
      float* to = f.fin + (n * p.H + h) * mat;
      for (int e = tid; e < mat; e += THREADS)
        to[(e / dc) * f.si + (e % dc) * f.sj] = sm.s[(e / dc) * DM + e % dc];
    }
    __syncthreads();
  }
}

// Chains the segments' own contributions in scan order: carry[j] becomes the
// state that leaves segment j.  One thread per element; a segment that no
// sequence leaves restarts the chain (its carry is never read).  The decays
// of 256 segments are looked up side by side, and four segments' elements are
// in flight at once.
__global__ void __launch_bounds__(256) chain_kernel(const __grid_constant__ Launch L) {
  const Problem& p = L.p;
  const Form& f = L.f[blockIdx.z];
  const int h = blockIdx.y, tid = threadIdx.x;
  const long long mat = static_cast<long long>(f.da) * f.dc;
  const long long e = static_cast<long long>(blockIdx.x) * 256 + tid;
  __shared__ float dec[256];  // of the segment; -1: starts anew; -2: nothing crosses
  float state = 0.f;
  const long long hop = static_cast<long long>(p.H) * mat;
  for (int m0 = 0; m0 + 1 < p.J; m0 += 256) {
    const int count = min(256, p.J - 1 - m0);
    __syncthreads();
    if (tid < count) {
      const int j = f.rev ? p.J - 1 - (m0 + tid) : m0 + tid;
      const long long edge = f.rev ? j * p.seg : min((j + 1) * p.seg, p.BL);  // token after the boundary
      const long long n = first_beyond(p, edge);
      dec[tid] = n >= p.N || cu_at(p, n) >= edge ? -2.f : f.dec[j * p.H + h];
    }
    __syncthreads();
    if (e >= mat) continue;
    const long long step = f.rev ? -hop : hop;
    float* at = f.carry + ((f.rev ? p.J - 1 - m0 : m0) * static_cast<long long>(p.H) + h) * mat + e;
    for (int m = 0; m < count; m += 4, at += 4 * step) {
      float x[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = m + q < count && dec[m + q] > -2.f ? at[q * step] : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (m + q >= count || dec[m + q] == -2.f) continue;
        // an anew segment keeps its own; else what entered it has come through
        state = dec[m + q] < 0.f ? x[q] : fmaf(dec[m + q], state, x[q]);
        if (dec[m + q] >= 0.f) at[q * step] = state;
      }
    }
  }
}

// Gate gradients of one stretch of at most p.restart (128, 256 or 1024) tokens: the product of
// the two states at its end, then the reverse sum of q.dq - k.dk over it.
// blockIdx.z takes every gridDim.z-th stretch of the segment.
__global__ void __launch_bounds__(256)
    gate_grad_kernel(const __grid_constant__ Launch L, const float* __restrict__ final_state,
                     const float* __restrict__ d_final, float* __restrict__ part, void* __restrict__ out,
                     int out_type) {
  const Problem& p = L.p;
  const Form& fq = L.f[0];
  const Form& fk = L.f[1];
  const int tid = threadIdx.x, j = blockIdx.x, h = blockIdx.y, lane = tid & 31, warp = tid >> 5;
  const long long mat = static_cast<long long>(fq.da) * fq.dc;
  const long long t0 = j * p.seg, t1 = min(t0 + p.seg, p.BL);
  __shared__ float red[8];
  auto put = [&](long long t, float x) {
    if (part) part[t * p.H + h] = x;
    else store_any(out, out_type, t * p.H + h, x);
  };
  if (blockIdx.z == 0) {
    const long long c0 = min(t1, cu_at(p, 0)), c1 = max(t0, cu_at(p, p.N));
    for (long long t = t0 + tid; t < t1; t += 256)
      if (t < c0 || t >= c1) put(t, 0.f);
  }
  int stretch = 0;
  for (long long n = first_beyond(p, t0); n < p.N && cu_at(p, n) < t1; ++n) {
    const long long b0 = cu_at(p, n), b1 = cu_at(p, n + 1);
    const long long ps = max(b0, t0), pe = min(b1, t1);
    for (long long s0 = ps; s0 < pe; s0 += p.restart, ++stretch) {
      if (stretch % gridDim.z != blockIdx.z) continue;
      const long long s1 = min(s0 + p.restart, pe);
      const float *x = nullptr, *y = nullptr;
      if (s1 < pe) {
        x = fq.snap + (snap_slot(p, s1) * p.H + h) * mat;
        y = fk.snap + (snap_slot(p, s1) * p.H + h) * mat;
      } else if (pe < b1) {
        x = fq.carry + (static_cast<long long>(j) * p.H + h) * mat;
        y = fk.carry + (static_cast<long long>(j + 1) * p.H + h) * mat;
      } else if (d_final) {
        x = final_state + (n * p.H + h) * mat;
        y = d_final + (n * p.H + h) * mat;
      }
      float dot = 0.f;
      if (x && mat % 4 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15u) == 0) {
#pragma unroll 4
        for (long long e = tid; e < mat / 4; e += 256) {
          const float4 a = __ldcs(reinterpret_cast<const float4*>(x) + e), b = __ldcs(reinterpret_cast<const float4*>(y) + e);
          dot = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, dot))));
        }
      } else if (x) {
        for (long long e = tid; e < mat; e += 256) dot = fmaf(x[e], y[e], dot);
      }
      // four tokens a thread, latest first
      float v[4], sum = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const long long t = s1 - 1 - (tid * 4 + q);
        v[q] = 0.f;
        if (t >= s0) {
          const long long at = h * p.BL + t, half = p.H * p.BL;
          const float a = fq.rowdot[at] + (fq.dot_parts > 1 ? fq.rowdot[at + half] : 0.f);
          v[q] = a - (fk.rowdot[at] + (fk.dot_parts > 1 ? fk.rowdot[at + half] : 0.f));
        }
        sum += v[q];
      }
      float inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const float up = __shfl_up_sync(kFull, inc, o);
        if (lane >= o) inc += up;
      }
#pragma unroll
      for (int o = 16; o > 0; o /= 2) dot += __shfl_xor_sync(kFull, dot, o);
      __syncthreads();
      if (lane == 0) red[warp] = dot;
      __syncthreads();
      float base = 0.f;
      for (int w = 0; w < 8; ++w) base += red[w];
      __syncthreads();
      if (lane == 31) red[warp] = inc;
      __syncthreads();
      for (int w = 0; w < warp; ++w) base += red[w];
      base += inc - sum;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const long long t = s1 - 1 - (tid * 4 + q);
        base += v[q];
        if (t < s0) continue;
        // no state before the token, or a gate that drops it: nothing passes,
        // and the sums' rounding must not stand in for that
        const bool none = (!fq.init && t == b0) || expf(load_gate(p, t, h)) == 0.f;
        put(t, none ? 0.f : base);
      }
    }
  }
}

// Sums the float32 parts of heads that share one input head, in head order.
template <typename T>
__global__ void __launch_bounds__(256)
    share_sum_kernel(const float* __restrict__ part, T* __restrict__ out, long long n, int share, int dim) {
  const long long first = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<long long>(gridDim.x) * 256;
  if (dim % 4 == 0 && (reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T))) == 0) {
    const int quads = dim / 4;
    for (long long e = first; e < n / 4; e += step) {
      const long long row = e / quads;
      const float4* at = reinterpret_cast<const float4*>(part) + row * share * quads + e % quads;
      float4 x = __ldcs(at);
#pragma unroll 4
      for (int s = 1; s < share; ++s) {
        const float4 y = __ldcs(at + static_cast<long long>(s) * quads);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
      }
      T v[4] = {from_f<T>(x.x), from_f<T>(x.y), from_f<T>(x.z), from_f<T>(x.w)};
      if (sizeof(T) == 4) reinterpret_cast<float4*>(out)[e] = x;
      else reinterpret_cast<uint2*>(out)[e] = *reinterpret_cast<const uint2*>(v);
    }
    return;
  }
  for (long long e = first; e < n; e += step) {
    const long long row = e / dim, d = e % dim;
    float x = 0.f;
    for (int s = 0; s < share; ++s) x += part[(row * share + s) * dim + d];
    out[e] = from_f<T>(x);
  }
}

// ---------------------------------------------------------------------------
// One token: out = scale * q (e^g S + k v^T), the new state written back.
// Bound by reading and writing the state; a CTA takes 128 columns of one
// (request, head), a lane four of them, and its warps share the rows, eight in
// flight each.  256 requests of 12 heads of 128 x 128: 66 us, 6.1 TB/s; one
// request (32 columns a CTA): 3.2 us.
// ---------------------------------------------------------------------------

struct StepArgs {
  Rows q, k, v, gate;
  const int* slots;
  const float* state;
  float* state_out;
  void* out;
  long long pool;
  int H, dk, dv, gate_type, vec;
  float scale;
  uint32_t* err;
};

template <typename T, int LANES>
__global__ void __launch_bounds__(256) step_kernel(const __grid_constant__ StepArgs a) {
  constexpr int RPP = 256 / LANES;  // rows per pass
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const int lane = tid % LANES, r0 = tid / LANES;
  const int d = (blockIdx.x * LANES + lane) * 4;
  const int nv = max(0, min(4, a.dv - d));
  const long long slot = a.slots ? a.slots[b] : b;
  T* out = static_cast<T*>(a.out) + (static_cast<long long>(b) * a.H + h) * a.dv;
  if (slot < 0 || slot >= a.pool) {
    // negative: a row without a request; too large: reported, nothing touched
    if (slot >= a.pool && tid == 0 && h == 0 && blockIdx.x == 0) report(ASCAN_DEV_ERR_INDEX, slot, a.err);
    if (r0 == 0)
      for (int q = 0; q < nv; ++q) out[d + q] = from_f<T>(0.f);
    return;
  }
  const T* q = static_cast<const T*>(a.q.p) + b * a.q.st + (h / a.q.share) * a.q.sh;
  const T* k = static_cast<const T*>(a.k.p) + b * a.k.st + (h / a.k.share) * a.k.sh;
  const T* v = static_cast<const T*>(a.v.p) + b * a.v.st + (h / a.v.share) * a.v.sh;
  const float decay = expf(load_any(a.gate.p, a.gate_type, b * a.gate.st + (h / a.gate.share) * a.gate.sh));
  const long long base = (slot * a.H + h) * a.dk * static_cast<long long>(a.dv);
  const float* src = a.state + base;
  float* dst = a.state_out + base;
  float vv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int x = 0; x < 4; ++x) vv[x] = x < nv ? to_f(v[d + x]) : 0.f;
  if (a.vec && nv == 4) {
    constexpr int U = LANES == 32 ? 8 : 4;  // rows in flight per thread
    for (int i0 = r0; i0 < a.dk; i0 += RPP * U) {
      float4 s[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * RPP < a.dk)
          s[u] = __ldcs(reinterpret_cast<const float4*>(src + static_cast<long long>(i0 + u * RPP) * a.dv + d));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * RPP;
        if (i < a.dk) {
          const float ki = to_f(k[i]), qi = to_f(q[i]);
          s[u].x = fmaf(ki, vv[0], decay * s[u].x);
          s[u].y = fmaf(ki, vv[1], decay * s[u].y);
          s[u].z = fmaf(ki, vv[2], decay * s[u].z);
          s[u].w = fmaf(ki, vv[3], decay * s[u].w);
          __stcs(reinterpret_cast<float4*>(dst + static_cast<long long>(i) * a.dv + d), s[u]);
          acc[0] = fmaf(qi, s[u].x, acc[0]);
          acc[1] = fmaf(qi, s[u].y, acc[1]);
          acc[2] = fmaf(qi, s[u].z, acc[2]);
          acc[3] = fmaf(qi, s[u].w, acc[3]);
        }
      }
    }
  } else {
    for (int i = r0; i < a.dk; i += RPP) {
      const float ki = to_f(k[i]), qi = to_f(q[i]);
      for (int x = 0; x < nv; ++x) {
        const long long at = static_cast<long long>(i) * a.dv + d + x;
        const float s = fmaf(ki, vv[x], decay * src[at]);
        dst[at] = s;
        acc[x] = fmaf(qi, s, acc[x]);
      }
    }
  }
  __shared__ float4 part[256];
  part[tid] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (r0 == 0) {
    for (int r = 1; r < RPP; ++r) {
      const float4 o = part[r * LANES + lane];
      acc[0] += o.x, acc[1] += o.y, acc[2] += o.z, acc[3] += o.w;
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (x < nv) out[d + x] = from_f<T>(acc[x] * a.scale);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

constexpr long long kSms = 148;

// What runs at once, and of how many tokens segments are multiples: a chunk of
// the tensor-core kernel costs about 5 us however few of its tokens are there,
// and a carry pass comes on top (128 instead of 256: 257 tokens took 53 us, not
// 34, 16 ragged prompts of 16384 tokens 183 us, not 166); the plain one's
// granules may be shorter (128: float32 training 690 us, 256: 766 us).
struct Fit {
  long long room;
  int granule;
};

// Segments: the launch should fill the SMs, and a split that a sequence
// crosses costs a second pass over two of the operands, about half of the
// main pass's time.  Over all counts the cheapest estimate of
// waves * segment length (* 1.5 when there are more segments than sequences)
// is taken; equal sequences split at their own ends.  `room`: CTAs that run
// at once.
static long long pick_segments(long long BL, long long N, long long lanes, int granule, long long room) {
  const long long most = min(min((BL + granule - 1) / granule, 4096ll), 65535ll);
  const double inf = 1e30;
  long long best = 1;
  double best_cost = inf;
  for (long long J = 1; J <= most; J = J < 64 ? J + 1 : J + 8) {
    const long long seg = ((BL + J - 1) / J + granule - 1) / granule * granule;
    const long long waves = (J * lanes + room - 1) / room;
    const double cost = static_cast<double>(waves) * (seg + 2.0 * granule) * (J > N ? 1.5 : 1.0);
    if (cost < best_cost * 0.97) best = J, best_cost = cost;
    if (J * lanes > 16 * room) break;
  }
  return best;
}

template <typename T, int DM>
static int plain_launch(const Launch& l, int roles, bool state_only, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  const int rc = allow_smem(plain_kernel<T, DM>, sizeof(PlainSmem<DM>), done);
  if (rc != ASCAN_OK) return rc;
  plain_kernel<T, DM><<<dim3(l.p.J, l.p.H, roles), kPlainThreads, sizeof(PlainSmem<DM>), s>>>(l, state_only);
  return launch_status();
}

static int plain_run(const Launch& l, int roles, bool state_only, int dtype, cudaStream_t s) {
  int dm = 64;
  for (int r = 0; r < roles; ++r) dm = max(dm, max(l.f[r].da, l.f[r].dc) > 64 ? 128 : 64);
#define MSCAN_PLAIN(T) (dm == 64 ? plain_launch<T, 64>(l, roles, state_only, s) : plain_launch<T, 128>(l, roles, state_only, s))
  if (dtype == ASCAN_F32) return MSCAN_PLAIN(float);
  if (dtype == ASCAN_F16) return MSCAN_PLAIN(__half);
  return MSCAN_PLAIN(__nv_bfloat16);
#undef MSCAN_PLAIN
}

static int run_forms(Launch& l, int roles, int dtype, cudaStream_t s) {
  int rc = ASCAN_OK;
  const bool tc = tc_usable(l, roles, dtype);
  l.p.restart = restart_of(tc, l.p.gate_type);
  for (int r = 0; r < roles; ++r) l.f[r].dot_parts = tc ? tc_dot_parts(l.f[r]) : 1;
  if (l.p.J > 1) {
    rc = tc ? tc_run(l, roles, true, s) : plain_run(l, roles, true, dtype, s);
    if (rc != ASCAN_OK) return rc;
    long long mat = 0;
    for (int r = 0; r < roles; ++r) mat = max(mat, static_cast<long long>(l.f[r].da) * l.f[r].dc);
    chain_kernel<<<dim3(static_cast<unsigned>((mat + 255) / 256), l.p.H, roles), 256, 0, s>>>(l);
    rc = launch_status();
    if (rc != ASCAN_OK) return rc;
  }
  return tc ? tc_run(l, roles, false, s) : plain_run(l, roles, false, dtype, s);
}

struct Plan {
  long long J, seg, slots;
  size_t carry, snap, part_q, part_k, part_v, part_g, rowdot, total;
};

static size_t up(size_t x) { return (x + 255) / 256 * 256; }

// The plain kernel's CTAs fit three to an SM up to 64 wide.
static Fit fit_for(int dtype, int dk, int dv) {
  if (dtype == ASCAN_BF16) return {kSms, 256};
  return {max(dk, dv) <= 64 ? 3 * kSms : kSms, 128};
}

// Layout of the workspace; the same arithmetic serves the size query.  Of
// bfloat16 rows it is not known yet whether the tensor cores take them: room
// for their stretches, the shorter ones.
static Plan make_plan(long long BL, long long N, int H, int hq, int hk, int hv, int hg, int dk, int dv, int dtype,
                      int gate_type, bool backward) {
  const Fit fit = fit_for(dtype, dk, dv);
  Plan w{};
  w.J = pick_segments(BL, N, static_cast<long long>(H) * (backward ? 3 : 1), fit.granule, fit.room);
  w.seg = ((BL + w.J - 1) / w.J + fit.granule - 1) / fit.granule * fit.granule;
  w.J = (BL + w.seg - 1) / w.seg;
  const size_t mat = static_cast<size_t>(dk) * dv * H * 4;
  w.carry = w.J > 1 ? up(w.J * mat) + up(static_cast<size_t>(w.J) * H * 4) : 0;
  w.slots = BL / restart_of(dtype == ASCAN_BF16, gate_type) + 1;
  const size_t rows = static_cast<size_t>(BL) * H * 4;
  w.total = w.carry * (backward ? 3 : 1);
  if (backward) {
    w.snap = up(w.slots * mat);
    w.rowdot = up(2 * rows);
    w.part_q = hq < H ? up(rows * dk) : 0;
    w.part_k = hk < H ? up(rows * dk) : 0;
    w.part_v = hv < H ? up(rows * dv) : 0;
    w.part_g = hg < H ? up(rows) : 0;
    w.total += 2 * w.snap + 2 * w.rowdot + w.part_q + w.part_k + w.part_v + w.part_g;
  }
  w.total += 256;
  return w;
}

static bool rows_ok(const ascan_rows* r, int H) {
  return r && r->data && r->heads > 0 && r->heads <= H && H % r->heads == 0 && r->stride_token >= 0 &&
         r->stride_head >= 0;
}

static Rows rows_of(const ascan_rows* r, int H) {
  return Rows{r->data, r->stride_token, r->stride_head, H / r->heads};
}

static int check(const ascan_rows* q, const ascan_rows* k, const ascan_rows* v, const ascan_rows* g, int gate_dtype,
                 const void* cu, int cu_type, int64_t N, int64_t BL, int H, int dk, int dv, int dtype) {
  if (!cu || N < 0 || BL < 0 || H <= 0 || H > 65535 || dk <= 0 || dv <= 0) return ASCAN_EINVAL;
  if (dk > ASCAN_MATRIX_SCAN_MAX_DIM || dv > ASCAN_MATRIX_SCAN_MAX_DIM) return ASCAN_EINVAL;
  if (cu_type != ASCAN_I32 && cu_type != ASCAN_I64) return ASCAN_EINVAL;
  if (dtype < ASCAN_F32 || dtype > ASCAN_BF16 || gate_dtype < ASCAN_F32 || gate_dtype > ASCAN_BF16) return ASCAN_EINVAL;
  if (BL > (1ll << 40)) return ASCAN_EINVAL;
  if (BL == 0 || N == 0) return ASCAN_OK;
  if (!rows_ok(q, H) || !rows_ok(k, H) || !rows_ok(v, H) || !rows_ok(g, H)) return ASCAN_EINVAL;
  return ASCAN_OK;
}

static Problem problem_of(const Plan& w, const ascan_rows* g, int gate_dtype, const void* cu, int cu_type, int64_t N,
                          int64_t BL, int H) {
  Problem p{};
  p.cu = cu;
  p.cu64 = cu_type == ASCAN_I64;
  p.J = static_cast<int>(w.J);
  p.H = H;
  p.gate_type = gate_dtype;
  p.N = N;
  p.BL = BL;
  p.seg = w.seg;
  p.gate = rows_of(g, H);
  p.err = g_err_host;
  return p;
}

}  // namespace mscan
}  // namespace ascan

using namespace ascan;
using namespace ascan::mscan;

extern "C" {

size_t ascan_matrix_scan_workspace(int64_t seq_total, int64_t num_seq, int num_heads, int query_heads, int key_heads,
                                   int value_heads, int gate_heads, int key_dim, int value_dim, int backward) {
  if (seq_total <= 0 || num_seq <= 0 || num_heads <= 0 || key_dim <= 0 || value_dim <= 0) return 256;
  size_t need = 0;
  for (int dtype : {ASCAN_F32, ASCAN_F16, ASCAN_BF16})
    for (int gate_dtype : {ASCAN_F32, ASCAN_F16, ASCAN_BF16})
      need = max(need, ascan_matrix_scan_workspace_of(seq_total, num_seq, num_heads, query_heads, key_heads, value_heads,
                                                      gate_heads, key_dim, value_dim, dtype, gate_dtype, backward));
  return need;
}

size_t ascan_matrix_scan_workspace_of(int64_t seq_total, int64_t num_seq, int num_heads, int query_heads,
                                      int key_heads, int value_heads, int gate_heads, int key_dim, int value_dim,
                                      int dtype, int gate_dtype, int backward) {
  if (seq_total <= 0 || num_seq <= 0 || num_heads <= 0 || key_dim <= 0 || value_dim <= 0) return 256;
  return make_plan(seq_total, num_seq, num_heads, query_heads, key_heads, value_heads, gate_heads, key_dim, value_dim,
                   dtype, gate_dtype, backward != 0)
      .total;
}

int ascan_matrix_scan_forward(const ascan_rows* queries, const ascan_rows* keys, const ascan_rows* values,
                              const ascan_rows* log_gates, int gate_dtype, const void* cu_seqlens, int cu_index_type,
                              int64_t num_seq, int64_t seq_total, int num_heads, int key_dim, int value_dim, int dtype,
                              float scale, const float* initial_state, void* out, float* final_state, void* workspace,
                              size_t workspace_bytes, void* stream) {
  int rc = check(queries, keys, values, log_gates, gate_dtype, cu_seqlens, cu_index_type, num_seq, seq_total, num_heads,
                 key_dim, value_dim, dtype);
  if (rc != ASCAN_OK) return rc;
  if (seq_total == 0 || num_seq == 0) return ASCAN_OK;
  if (!out) return ASCAN_EINVAL;
  const Plan w = make_plan(seq_total, num_seq, num_heads, queries->heads, keys->heads, values->heads, log_gates->heads,
                           key_dim, value_dim, dtype, gate_dtype, false);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < w.total) return ASCAN_EWORKSPACE;
  Launch l{};
  l.p = problem_of(w, log_gates, gate_dtype, cu_seqlens, cu_index_type, num_seq, seq_total, num_heads);
  char* at = static_cast<char*>(workspace);
  Form& f = l.f[0];
  f.a = rows_of(queries, num_heads);
  f.b = rows_of(keys, num_heads);
  f.c = rows_of(values, num_heads);
  f.da = key_dim;
  f.dc = value_dim;
  f.sp = f.sr = scale;
  f.sc = 1.f;
  f.out = out;
  f.init = initial_state;
  f.fin = final_state;
  f.fine = final_state != nullptr;
  f.si = value_dim;
  f.sj = 1;
  f.carry = reinterpret_cast<float*>(at);
  f.dec = reinterpret_cast<float*>(at + up(static_cast<size_t>(w.J) * key_dim * value_dim * num_heads * 4));
  f.out_f32 = dtype == ASCAN_F32;
  return run_forms(l, 1, dtype, static_cast<cudaStream_t>(stream));
}

int ascan_matrix_scan_backward(const ascan_rows* queries, const ascan_rows* keys, const ascan_rows* values,
                               const ascan_rows* log_gates, int gate_dtype, const ascan_rows* d_out,
                               const float* initial_state, const float* final_state, const float* d_final_state,
                               const void* cu_seqlens, int cu_index_type, int64_t num_seq, int64_t seq_total,
                               int num_heads, int key_dim, int value_dim, int dtype, float scale, void* d_queries,
                               void* d_keys, void* d_values, void* d_log_gates, float* d_initial_state,
                               void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(queries, keys, values, log_gates, gate_dtype, cu_seqlens, cu_index_type, num_seq, seq_total, num_heads,
                 key_dim, value_dim, dtype);
  if (rc != ASCAN_OK) return rc;
  if (seq_total == 0 || num_seq == 0) return ASCAN_OK;
  if (!d_queries || !d_keys || !d_values || !d_log_gates || !rows_ok(d_out, num_heads) || d_out->heads != num_heads)
    return ASCAN_EINVAL;
  if (d_final_state && !final_state) return ASCAN_EINVAL;
  const int H = num_heads, dk = key_dim, dv = value_dim;
  const Plan w = make_plan(seq_total, num_seq, H, queries->heads, keys->heads, values->heads, log_gates->heads, dk, dv, dtype,
                           gate_dtype, true);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < w.total) return ASCAN_EWORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Launch l{};
  l.p = problem_of(w, log_gates, gate_dtype, cu_seqlens, cu_index_type, num_seq, seq_total, H);
  char* at = static_cast<char*>(workspace);
  auto take = [&](size_t n) {
    char* p = n ? at : nullptr;
    at += n;
    return reinterpret_cast<float*>(p);
  };
  const Rows q = rows_of(queries, H), k = rows_of(keys, H), v = rows_of(values, H), o = rows_of(d_out, H);
  const size_t mat = up(static_cast<size_t>(w.J) * dk * dv * H * 4);
  for (int r = 0; r < 3; ++r) {
    Form& f = l.f[r];
    f.carry = take(w.carry);
    f.dec = w.carry ? reinterpret_cast<float*>(reinterpret_cast<char*>(f.carry) + mat) : nullptr;
    f.rev = r != 0;
    f.fine = r == 2 ? d_initial_state != nullptr : gate_dtype == ASCAN_F32;
    f.sp = scale;
    f.sr = r == 0 ? scale : 1.f;
    f.sc = r == 0 ? 1.f : scale;
    f.da = r == 2 ? dk : dv;
    f.dc = r == 2 ? dv : dk;
    f.si = r == 2 ? dv : 1;  // the user's states are [dk, dv]; dq and dk hold theirs transposed
    f.sj = r == 2 ? 1 : dv;
    f.a = r == 0 ? o : (r == 1 ? v : k);
    f.b = r == 0 ? v : (r == 1 ? o : q);
    f.c = r == 0 ? k : (r == 1 ? q : o);
    f.init = r == 0 ? initial_state : d_final_state;
    f.out_f32 = dtype == ASCAN_F32;
  }
  l.f[2].fin = d_initial_state;
  l.f[0].snap = take(w.snap);
  l.f[1].snap = take(w.snap);
  l.f[0].rowdot = take(w.rowdot);
  l.f[1].rowdot = take(w.rowdot);
  l.f[0].dot = q;
  l.f[1].dot = k;
  float* parts[3] = {take(w.part_q), take(w.part_k), take(w.part_v)};
  float* part_g = take(w.part_g);
  void* outs[3] = {d_queries, d_keys, d_values};
  const int heads[3] = {queries->heads, keys->heads, values->heads};
  for (int r = 0; r < 3; ++r) {
    l.f[r].out = parts[r] ? parts[r] : outs[r];
    if (parts[r]) l.f[r].out_f32 = 1;
  }
  rc = run_forms(l, 3, dtype, s);
  if (rc != ASCAN_OK) return rc;
  gate_grad_kernel<<<dim3(l.p.J, H, static_cast<unsigned>(min(8ll, (w.seg + l.p.restart - 1) / l.p.restart))), 256, 0, s>>>(
      l, final_state, d_final_state, part_g, d_log_gates, gate_dtype);
  rc = launch_status();
  auto sum = [&](const float* part, void* out, int heads_x, int dim, int type) {
    if (!part || rc != ASCAN_OK) return;
    const long long n = seq_total * heads_x * dim;
    const unsigned grid = static_cast<unsigned>(min((n + 255) / 256, kSms * 16));
    if (type == ASCAN_F32)
      share_sum_kernel<float><<<grid, 256, 0, s>>>(part, static_cast<float*>(out), n, H / heads_x, dim);
    else if (type == ASCAN_F16)
      share_sum_kernel<__half><<<grid, 256, 0, s>>>(part, static_cast<__half*>(out), n, H / heads_x, dim);
    else
      share_sum_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(part, static_cast<__nv_bfloat16*>(out), n, H / heads_x, dim);
    rc = launch_status();
  };
  for (int r = 0; r < 3; ++r) sum(parts[r], outs[r], heads[r], r == 2 ? dv : dk, dtype);
  sum(part_g, d_log_gates, log_gates->heads, 1, gate_dtype);
  return rc;
}

int ascan_matrix_scan_step(const ascan_rows* queries, const ascan_rows* keys, const ascan_rows* values,
                           const ascan_rows* log_gates, int gate_dtype, const int32_t* slots, int64_t num_rows,
                           int64_t pool_size, int num_heads, int key_dim, int value_dim, int dtype, float scale,
                           const float* state, float* state_out, void* out, void* stream) {
  if (num_rows < 0 || num_rows > 65535 || pool_size < 0 || num_heads <= 0 || num_heads > 65535 || key_dim <= 0 ||
      value_dim <= 0 || value_dim > (1 << 20))
    return ASCAN_EINVAL;
  if (dtype < ASCAN_F32 || dtype > ASCAN_BF16 || gate_dtype < ASCAN_F32 || gate_dtype > ASCAN_BF16) return ASCAN_EINVAL;
  if (num_rows == 0) return ASCAN_OK;
  if (!rows_ok(queries, num_heads) || !rows_ok(keys, num_heads) || !rows_ok(values, num_heads) ||
      !rows_ok(log_gates, num_heads) || !state || !state_out || !out)
    return ASCAN_EINVAL;
  if (!slots && num_rows > pool_size) return ASCAN_EINVAL;
  StepArgs a{};
  a.q = rows_of(queries, num_heads);
  a.k = rows_of(keys, num_heads);
  a.v = rows_of(values, num_heads);
  a.gate = rows_of(log_gates, num_heads);
  a.slots = slots;
  a.state = state;
  a.state_out = state_out;
  a.out = out;
  a.pool = pool_size;
  a.H = num_heads;
  a.dk = key_dim;
  a.dv = value_dim;
  a.gate_type = gate_dtype;
  a.vec = value_dim % 4 == 0 && ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(state_out)) & 15u) == 0;
  a.scale = scale;
  a.err = g_err_host;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Few (request, head) pairs: 32 columns a CTA instead of 128, four times
  // the CTAs for the same bytes.
  const bool narrow = num_rows * num_heads < kSms;
  const unsigned cols = narrow ? 32 : 128;
  const dim3 grid((value_dim + cols - 1) / cols, num_heads, static_cast<unsigned>(num_rows));
#define MSCAN_STEP(T) (narrow ? (void)(step_kernel<T, 8><<<grid, 256, 0, s>>>(a)) : (void)(step_kernel<T, 32><<<grid, 256, 0, s>>>(a)))
  if (dtype == ASCAN_F32) MSCAN_STEP(float);
  else if (dtype == ASCAN_F16) MSCAN_STEP(__half);
  else MSCAN_STEP(__nv_bfloat16);
#undef MSCAN_STEP
  return launch_status();
}

}  // extern "C"

namespace ascan {
ASCAN_UNIT_ERROR_ACCESSORS(mscan)
}  // namespace ascan
