// ascan_rotate.cu -- compilation unit of the scan library: RMS norm of every
// query and key head, weight, and rotation by position, with its gradients.
//
//   xh = x * rsqrt(mean(x^2) + eps),  n = xh * w,  y = R(pos) n
//   dz = R(pos)^T dy,  dx = r (w dz - xh mean(w dz xh)),  dw = sum dz xh
//
// Every head is read once and written once, so device memory bounds large
// calls and launch latency small ones.  A group of lanes holds one head as
// one 16-byte vector per lane; the rotation's partner comes by a shuffle (or
// sits in the same vector when pairs are adjacent), and the sums go over the
// group by shuffles.  Where the whole head turns, a lane holds 8 bytes of each
// half instead and has both sides of its pairs.  A group walks the heads of
// consecutive tokens with several heads' loads in flight and a token's angles
// read once for all of them.  Queries and keys share a launch: the first CTAs
// take the query heads, the rest the key heads.  The weights' gradients stay
// in registers over all of a group's heads, meet in shared memory, and a
// second launch adds the CTAs' rows in a fixed order, so results repeat bit
// for bit.
//
// Measured, bfloat16 heads of 128: 16384 tokens of 24 heads 38 us forward (5.3
// TB/s), 66 + 2 us gradients (4.6 TB/s); 65536 tokens of 20 heads 138 us (5.1
// TB/s); 16 tokens 2.9 us.  Six or eight loads in flight: no faster or slower;
// three CTAs an SM for the gradients: 76 us.
#include "ascan_impl.cuh"
#include "ascan_mscan.cuh"
#include "ascan_pairs.cuh"

namespace ascan {
namespace rotate {

using mscan::from_f;
using mscan::load_any;
using mscan::store_any;
using mscan::to_f;

constexpr int kRotThreads = 256;

struct Side {  // queries or keys
  const void* x;
  long long st, sh;
  const void* dy;  // gradients only
  long long dst, dsh;
  const void* w;
  void* out;     // y, or dx
  float* part;   // [CTAs, dim]: rows of the weight gradient
  void* dw;
  int heads, ctas;
  int slices, heads_per;  // vector kernel: groups per token, heads of each
  long long span;         // tokens in a row per group
};

struct Args {
  Side side[2];
  const float *cos_table, *sin_table;
  const void *positions, *cu;
  long long rows, N, tokens;
  int index64, half, interleaved, dim, wtype;
  float eps;
  uint32_t* err;
};

__device__ __forceinline__ long long index_at(const void* p, int is64, long long i) {
  return is64 ? static_cast<const long long*>(p)[i] : static_cast<long long>(static_cast<const int*>(p)[i]);
}

// Table row of token t; -1: zero row.
__device__ __forceinline__ long long table_row(const Args& a, long long t) {
  long long pos;
  if (a.positions) {
    pos = index_at(a.positions, a.index64, t);
  } else {
    long long lo = 0, hi = a.N;  // first sequence that ends beyond t
    while (lo < hi) {
      const long long mid = (lo + hi) >> 1;
      if (index_at(a.cu, a.index64, mid + 1) > t) hi = mid;
      else lo = mid + 1;
    }
    if (lo >= a.N) return -1;
    pos = t - index_at(a.cu, a.index64, lo);
    if (pos < 0) return -1;
  }
  if (pos < 0 || pos >= a.rows) {
    report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(t), a.err);
    return -1;
  }
  return pos;
}

__device__ __forceinline__ void check_cu(const Args& a) {
  if (!a.cu || blockIdx.x != 0) return;
  if (a.index64) validate_cu(static_cast<const int64_t*>(a.cu), a.N, a.tokens, a.err);
  else validate_cu(static_cast<const int32_t*>(a.cu), a.N, a.tokens, a.err);
}

template <typename T>
struct Vec {
  static constexpr int V = 16 / sizeof(T);
};

// A lane's 16 bytes as register pairs of floats and back.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, uint64_t* x);
template <>
__device__ __forceinline__ void unpack<float>(const uint4& u, uint64_t* x) {
  x[0] = pair(__uint_as_float(u.x), __uint_as_float(u.y));
  x[1] = pair(__uint_as_float(u.z), __uint_as_float(u.w));
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& u, uint64_t* x) {
  const uint32_t e[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pair(__uint_as_float(e[i] << 16), __uint_as_float(e[i] & 0xffff0000u));
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint4& u, uint64_t* x) {
  const uint32_t e[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&e[i]));
    x[i] = pair(f.x, f.y);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const uint64_t* x);
template <>
__device__ __forceinline__ uint4 pack<float>(const uint64_t* x) {
  const float2 a = unpair(x[0]), b = unpair(x[1]);
  return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
}
template <>
__device__ __forceinline__ uint4 pack<__nv_bfloat16>(const uint64_t* x) {
  uint32_t e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = unpair(x[i]);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(e[i]) : "f"(a.y), "f"(a.x));
  }
  return make_uint4(e[0], e[1], e[2], e[3]);
}
template <>
__device__ __forceinline__ uint4 pack<__half>(const uint64_t* x) {
  uint32_t e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = unpair(x[i]);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(e[i]) : "f"(a.y), "f"(a.x));
  }
  return make_uint4(e[0], e[1], e[2], e[3]);
}

template <int G>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = G / 2; o > 0; o /= 2) x += __shfl_xor_sync(kFull, x, o);
  return x;
}

// Sequence lookups of tokens that come in order: the last one found serves
// until the token leaves it.
struct Place {
  long long start = 0, end = -1;
};

// Table row of token t in order; -1: zero row.
__device__ __forceinline__ long long next_row(const Args& a, long long t, Place& at) {
  if (a.positions || t >= at.end || t < at.start) {
    const long long row = table_row(a, t);
    if (!a.positions && row >= 0) {
      at.start = t - row;
      at.end = at.start;
      long long lo = 0, hi = a.N;
      while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (index_at(a.cu, a.index64, mid + 1) > t) hi = mid;
        else lo = mid + 1;
      }
      at.end = index_at(a.cu, a.index64, lo + 1);
    }
    return row;
  }
  const long long row = t - at.start;
  if (row >= a.rows) {
    report(ASCAN_DEV_ERR_INDEX, static_cast<unsigned long long>(t), a.err);
    return -1;
  }
  return row;
}

// Where a lane's 16 bytes of a head lie.
//   kSplit: the whole head turns in halves; a lane has 8 bytes of each, so both
//           sides of its pairs
//   kAdjacent: pairs are neighbours
//   kPart: part of the head turns in halves; 16 bytes in a row, the partner's
//          come by shuffles
enum Pairing { kSplit, kAdjacent, kPart };

// How the lane's elements of a token turn: y = x p + x' q with x' the partner,
// for the forward with the weights in p and q (w cos, +-w' sin), for the
// gradients of the transposed turn without them (cos, -+sin).
template <typename T, Pairing P, bool BWD>
struct Turn {
  static constexpr int V = Vec<T>::V;
  uint64_t p[V / 2], q[V / 2];

  // Element of the head that the lane's i-th is.
  static __device__ __forceinline__ int element(const Args& a, int gl, int i) {
    if (P == kSplit) return i < V / 2 ? gl * (V / 2) + i : a.half + gl * (V / 2) + i - V / 2;
    return gl * V + i;
  }

  // `w`: the side's weights as floats, in shared memory.
  __device__ __forceinline__ void load(const Args& a, const float* w, long long row, int gl) {
    constexpr int A = P == kPart ? V : V / 2;  // angles of the lane
    float c[A], s[A];
#pragma unroll
    for (int i = 0; i < A; ++i) c[i] = 1.f, s[i] = 0.f;
    // kPart: lanes of the second half have the same angles as their partners
    const int hv = a.half / V, first = P == kPart ? (gl < hv ? gl : gl - hv) * V : gl * (V / 2);
    const bool turns = row >= 0 && first < a.half;
    if (turns) {
      const float* ct = a.cos_table + row * a.half + first;
      const float* st = a.sin_table + row * a.half + first;
      if (A == 2) {
        const float2 x = __ldg(reinterpret_cast<const float2*>(ct)), y = __ldg(reinterpret_cast<const float2*>(st));
        c[0] = x.x, c[1] = x.y, s[0] = y.x, s[1] = y.y;
      } else {
#pragma unroll
        for (int i = 0; i < A; i += 4) {
          const float4 x = __ldg(reinterpret_cast<const float4*>(ct + i)), y = __ldg(reinterpret_cast<const float4*>(st + i));
          c[i] = x.x, c[i + 1] = x.y, c[i + 2] = x.z, c[i + 3] = x.w;
          s[i] = y.x, s[i + 1] = y.y, s[i + 2] = y.z, s[i + 3] = y.w;
        }
      }
    }
    float pv[V], qv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int d = element(a, gl, i), at = P == kSplit ? i % A : (P == kAdjacent ? i / 2 : i);
      const bool low = P == kSplit ? i < A : (P == kAdjacent ? i % 2 == 0 : gl < hv);
      pv[i] = c[at];
      qv[i] = low == BWD ? s[at] : -s[at];
      if (!BWD) {
        const int other = P == kAdjacent ? d ^ 1 : (low ? d + a.half : d - a.half);
        pv[i] *= d < a.dim ? w[d] : 0.f;
        qv[i] *= turns ? w[other] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = pair(pv[2 * i], pv[2 * i + 1]), q[i] = pair(qv[2 * i], qv[2 * i + 1]);
  }

  // Every lane of the warp takes part.
  template <int G>
  __device__ __forceinline__ void apply(const uint4& raw, int partner, const uint64_t* x, uint64_t* y) const {
    uint64_t o[V / 2];
    if (P == kSplit) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) o[i] = x[(i + V / 4) % (V / 2)];
    } else if (P == kAdjacent) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 e = unpair(x[i]);
        o[i] = pair(e.y, e.x);
      }
    } else {
      uint4 r;
      r.x = __shfl_sync(kFull, raw.x, partner, G);
      r.y = __shfl_sync(kFull, raw.y, partner, G);
      r.z = __shfl_sync(kFull, raw.z, partner, G);
      r.w = __shfl_sync(kFull, raw.w, partner, G);
      unpack<T>(r, o);
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) y[i] = fma2(o[i], q[i], mul2(x[i], p[i]));
  }
};

// A lane's 16 bytes of a head: in one piece, or 8 bytes of each half.
template <Pairing P>
__device__ __forceinline__ uint4 get(const char* at, long long half_bytes) {
  if (P != kSplit) return __ldcs(reinterpret_cast<const uint4*>(at));
  const uint2 a = __ldcs(reinterpret_cast<const uint2*>(at)), b = __ldcs(reinterpret_cast<const uint2*>(at + half_bytes));
  return make_uint4(a.x, a.y, b.x, b.y);
}
template <Pairing P>
__device__ __forceinline__ void put(char* at, long long half_bytes, const uint4& v) {
  if (P != kSplit) {
    __stcs(reinterpret_cast<uint4*>(at), v);
  } else {
    __stcs(reinterpret_cast<uint2*>(at), make_uint2(v.x, v.y));
    __stcs(reinterpret_cast<uint2*>(at + half_bytes), make_uint2(v.z, v.w));
  }
}

// A group walks `span` tokens in order and, for each, heads [h0, h0 + heads_per)
// of its side.  DEPTH heads' loads are always in flight, over token boundaries
// too.  The arithmetic runs on register pairs: with single floats this kernel
// was bound by instructions, not memory.
template <typename T, int G, int DEPTH, Pairing P, bool BWD>
__global__ void __launch_bounds__(kRotThreads, BWD ? 2 : 3) vec_kernel(const __grid_constant__ Args a) {
  constexpr int V = Vec<T>::V, H = V / 2;
  constexpr int GROUPS = kRotThreads / G;
  const bool is_key = static_cast<int>(blockIdx.x) >= a.side[0].ctas;
  const Side& sd = a.side[is_key];
  const int cta = is_key ? blockIdx.x - a.side[0].ctas : blockIdx.x;
  const int gl = threadIdx.x % G, group = threadIdx.x / G;
  const bool on = gl * V < a.dim;
  const int hv = a.half / V;
  const int partner = gl < hv ? gl + hv : (gl < 2 * hv ? gl - hv : gl);  // kPart
  check_cu(a);
  const long long g = static_cast<long long>(cta) * GROUPS + group;
  const int h0 = static_cast<int>(g % sd.slices) * sd.heads_per, heads = min(sd.heads_per, sd.heads - h0);
  const long long first = g / sd.slices * sd.span;
  const int tokens = static_cast<int>(max(0ll, min(sd.span, a.tokens - first)));
  // every group of a warp runs the same number of rounds: the shuffles need them
  const int items = static_cast<int>(sd.span) * sd.heads_per;
  const float inv = 1.f / static_cast<float>(a.dim);
  constexpr int E = sizeof(T);
  const long long half_bytes = static_cast<long long>(a.half) * E;
  const int lane_bytes = gl * (P == kSplit ? 8 : 16);
  // running addresses: next head, and from the last head to the next token
  const char* src = static_cast<const char*>(sd.x) + (first * sd.st + h0 * sd.sh) * E + lane_bytes;
  const char* dsrc = BWD ? static_cast<const char*>(sd.dy) + (first * sd.dst + h0 * sd.dsh) * E + lane_bytes : nullptr;
  const long long hop = sd.sh * E, wrap = (sd.st - (sd.heads_per - 1) * sd.sh) * E;
  const long long dhop = sd.dsh * E, dwrap = (sd.dst - (sd.heads_per - 1) * sd.dsh) * E;
  char* dst = static_cast<char*>(sd.out) + (first * sd.heads + h0) * a.dim * E + lane_bytes;
  const int out_hop = a.dim * E, out_wrap = (sd.heads - sd.heads_per + 1) * a.dim * E;
  uint4 raw[DEPTH], draw[BWD ? DEPTH : 1];
  int lt = 0, lh = 0;  // the next load
  auto load = [&](int q) {
    raw[q] = make_uint4(0, 0, 0, 0);
    if (BWD) draw[q] = make_uint4(0, 0, 0, 0);
    if (on && lt < tokens && lh < heads) {
      raw[q] = get<P>(src, half_bytes);
      if (BWD) draw[q] = get<P>(dsrc, half_bytes);
    }
    const bool end = ++lh == sd.heads_per;
    src += end ? wrap : hop;
    if (BWD) dsrc += end ? dwrap : dhop;
    if (end) lh = 0, ++lt;
  };
#pragma unroll
  for (int q = 0; q < DEPTH; ++q) load(q);
  Turn<T, P, BWD> turn;
  Place place;
  long long row = tokens > 0 ? next_row(a, first, place) : -1;
  __shared__ float weights[G * V];
  for (int d = threadIdx.x; d < a.dim; d += kRotThreads) weights[d] = load_any(sd.w, a.wtype, d);
  __syncthreads();
  uint64_t w[BWD ? H : 1], dw[BWD ? H : 1];
  if (BWD) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const int d = Turn<T, P, BWD>::element(a, gl, 2 * i);
      w[i] = on ? pair(weights[d], weights[d + 1]) : 0;
      dw[i] = 0;
    }
  }
  int ct = 0, ch = 0;  // the next head to finish
  for (int r = 0; r < items; r += DEPTH) {
#pragma unroll
    for (int q = 0; q < DEPTH; ++q) {
      if (r + q >= items) break;
      if (ch == 0) {
        if (ct > 0) row = ct < tokens ? next_row(a, first + ct, place) : -1;
        turn.load(a, weights, row, gl);
      }
      const bool live = ct < tokens && ch < heads;
      uint64_t x[H], y[H], acc;
      unpack<T>(raw[q], x);
      acc = mul2(x[0], x[0]);
#pragma unroll
      for (int i = 1; i < H; ++i) acc = fma2(x[i], x[i], acc);
      float2 s2 = unpair(acc);
      const float rs = rsqrtf(fmaf(group_sum<G>(s2.x + s2.y), inv, a.eps));
      const uint64_t rs2 = pair(rs, rs);
      if (!BWD) {
        turn.template apply<G>(raw[q], partner, x, y);
#pragma unroll
        for (int i = 0; i < H; ++i) y[i] = mul2(y[i], rs2);
      } else {
        uint64_t dy[H], dz[H];
        unpack<T>(draw[q], dy);
        turn.template apply<G>(draw[q], partner, dy, dz);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          x[i] = mul2(x[i], rs2);  // xh
          const uint64_t gw = mul2(dz[i], x[i]);
          if (live && row >= 0) dw[i] = add2(dw[i], gw);
          acc = i == 0 ? mul2(gw, w[i]) : fma2(gw, w[i], acc);
        }
        s2 = unpair(acc);
        const float mean = -group_sum<G>(s2.x + s2.y) * inv;
        const uint64_t mean2 = pair(mean, mean);
#pragma unroll
        for (int i = 0; i < H; ++i) y[i] = mul2(rs2, fma2(x[i], mean2, mul2(w[i], dz[i])));
      }
      load(q);
      if (live && on) put<P>(dst, half_bytes, row >= 0 ? pack<T>(y) : make_uint4(0, 0, 0, 0));
      const bool end = ++ch == sd.heads_per;
      dst += end ? out_wrap : out_hop;
      if (end) ch = 0, ++ct;
    }
  }
  if (BWD) {
    __shared__ float red[GROUPS][G * V];
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float2 e = unpair(dw[i]);
      const int d = Turn<T, P, BWD>::element(a, gl, 2 * i);
      if (on) red[group][d] = e.x, red[group][d + 1] = e.y;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.dim; d += kRotThreads) {
      float x = 0.f;
      for (int e = 0; e < GROUPS; ++e) x += red[e][d];
      sd.part[static_cast<long long>(cta) * a.dim + d] = x;
    }
  }
}

// Any head size, stride and alignment: a warp per head, the partner's element
// read again (it is in the same lines).  The weight gradient of element
// lane + 32 k stays in register k, eight of them per pass over the elements.
template <typename T, bool BWD>
__global__ void __launch_bounds__(kRotThreads) any_kernel(const __grid_constant__ Args a) {
  constexpr int K = 8;
  const bool is_key = static_cast<int>(blockIdx.x) >= a.side[0].ctas;
  const Side& sd = a.side[is_key];
  const int cta = is_key ? blockIdx.x - a.side[0].ctas : blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  check_cu(a);
  const long long units = a.tokens * sd.heads;
  const float inv = 1.f / static_cast<float>(a.dim);
  __shared__ float red[kRotThreads / 32][32 * K];
  for (int e0 = 0; e0 < a.dim; e0 += 32 * K) {
    float dw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k] = 0.f;
    for (long long unit = static_cast<long long>(cta) * 8 + warp; unit < units; unit += static_cast<long long>(sd.ctas) * 8) {
      const long long t = unit / sd.heads;
      const int h = static_cast<int>(unit % sd.heads);
      const long long row = table_row(a, t);
      const T* x = static_cast<const T*>(sd.x) + t * sd.st + h * sd.sh;
      const T* dy = BWD ? static_cast<const T*>(sd.dy) + t * sd.dst + h * sd.dsh : nullptr;
      // partner of element d, its cosine and its signed sine (in R)
      auto turn = [&](int d, float& c, float& s) {
        c = 1.f, s = 0.f;
        if (row < 0 || d >= 2 * a.half) return d;
        const bool low = a.interleaved ? d % 2 == 0 : d < a.half;
        const int at = a.interleaved ? d / 2 : (low ? d : d - a.half);
        c = a.cos_table[row * a.half + at];
        s = a.sin_table[row * a.half + at] * (low ? -1.f : 1.f);
        return a.interleaved ? (low ? d + 1 : d - 1) : (low ? d + a.half : d - a.half);
      };
      float sq = 0.f;
      for (int d = lane; d < a.dim; d += 32) {
        const float v = to_f(x[d]);
        sq = fmaf(v, v, sq);
      }
      const float rs = rsqrtf(fmaf(group_sum<32>(sq), inv, a.eps));
      auto grad = [&](int d) {  // dz of element d
        float c, s;
        const int o = turn(d, c, s);
        return o == d ? to_f(dy[d]) : fmaf(-s, to_f(dy[o]), c * to_f(dy[d]));
      };
      float mean = 0.f;
      if (BWD) {
        for (int d = lane; d < a.dim; d += 32)
          mean = fmaf(grad(d) * to_f(x[d]) * rs, load_any(sd.w, a.wtype, d), mean);
        mean = group_sum<32>(mean) * inv;
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int d = e0 + 32 * k + lane;
        if (d >= a.dim) continue;
        const float w = load_any(sd.w, a.wtype, d), xv = to_f(x[d]) * rs;
        float y;
        if (!BWD) {
          float c, s;
          const int o = turn(d, c, s);
          y = o == d ? xv * w : fmaf(s, to_f(x[o]) * rs * load_any(sd.w, a.wtype, o), c * xv * w);
        } else {
          const float dz = grad(d);
          if (row >= 0) dw[k] = fmaf(dz, xv, dw[k]);
          // a head of one element: 1 - xh^2 is eps / (x^2 + eps), which the
          // difference of the general form would lose
          y = a.dim == 1 ? w * dz * a.eps * rs * rs * rs : rs * fmaf(-xv, mean, w * dz);
        }
        static_cast<T*>(sd.out)[(t * sd.heads + h) * a.dim + d] = from_f<T>(row < 0 ? 0.f : y);
      }
    }
    if (BWD) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) red[warp][32 * k + lane] = dw[k];
      __syncthreads();
      const int d = e0 + threadIdx.x;
      if (d < a.dim) {
        float s = 0.f;
        for (int g = 0; g < kRotThreads / 32; ++g) s += red[g][threadIdx.x];
        sd.part[static_cast<long long>(cta) * a.dim + d] = s;
      }
    }
  }
}

// Adds the CTAs' rows: 32 columns and 32 slices of the rows per CTA, the
// slices joined in order.
__global__ void __launch_bounds__(1024) weight_kernel(const __grid_constant__ Args a) {
  const Side& sd = a.side[blockIdx.y];
  const int d = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  __shared__ float red[32][32];
  float x = 0.f;
  if (d < a.dim) {
#pragma unroll 4
    for (int c = slice; c < sd.ctas; c += 32) x += sd.part[static_cast<long long>(c) * a.dim + d];
  }
  red[slice][threadIdx.x & 31] = x;
  __syncthreads();
  if (slice == 0 && d < a.dim) {
    for (int s = 1; s < 32; ++s) x += red[s][threadIdx.x];
    store_any(sd.dw, a.wtype, d, x);
  }
}

constexpr long long kMaxCtas = 148 * 6;

// CTAs of the plain form for one side: its share of the heads, at most what
// its work fills.
static void split(Args& a, long long per_cta) {
  const long long total = a.side[0].heads + a.side[1].heads;
  for (int s = 0; s < 2; ++s) {
    const long long fill = (a.tokens * a.side[s].heads + per_cta - 1) / per_cta;
    const long long share = max(1ll, kMaxCtas * a.side[s].heads / total);
    a.side[s].ctas = static_cast<int>(min(fill, share));
  }
}

// Groups of the vector kernel.  Each side gets its share (by heads) of the
// groups that are resident at once.  With fewer tokens than groups a token's
// heads are dealt to several groups, for the shortest chain; with more, a
// group takes whole tokens, several in a row, and reads their angles once.
static void split_groups(Args& a, int groups_per_cta, int ctas_per_sm) {
  const long long total = a.side[0].heads + a.side[1].heads, room = 148ll * ctas_per_sm;
  for (int s = 0; s < 2; ++s) {
    Side& sd = a.side[s];
    const long long groups = max(1ll, room * sd.heads / total) * groups_per_cta;
    const long long slices = max(1ll, min(static_cast<long long>(sd.heads), groups / max(1ll, a.tokens)));
    sd.heads_per = static_cast<int>((sd.heads + slices - 1) / slices);
    sd.slices = (sd.heads + sd.heads_per - 1) / sd.heads_per;
    sd.span = (a.tokens * sd.slices + groups - 1) / groups;
    const long long used = (a.tokens + sd.span - 1) / sd.span * sd.slices;
    sd.ctas = static_cast<int>((used + groups_per_cta - 1) / groups_per_cta);
  }
}

template <typename T, bool BWD>
static int run(Args& a, bool vec, cudaStream_t s) {
  if (vec) {
    const int lanes = a.dim / Vec<T>::V;
    const int g = lanes <= 8 ? 8 : (lanes <= 16 ? 16 : 32);
    split_groups(a, kRotThreads / g, BWD ? 2 : 3);
    const unsigned grid = a.side[0].ctas + a.side[1].ctas;
    const Pairing pairing = a.interleaved ? kAdjacent : (2 * a.half == a.dim ? kSplit : kPart);
    constexpr int D = BWD ? 2 : 4;
#define ROT_LAUNCH(GG, PP) vec_kernel<T, GG, D, PP, BWD><<<grid, kRotThreads, 0, s>>>(a)
#define ROT_CASE(GG)                                \
  if (pairing == kSplit) ROT_LAUNCH(GG, kSplit);    \
  else if (pairing == kAdjacent) ROT_LAUNCH(GG, kAdjacent); \
  else ROT_LAUNCH(GG, kPart)
    if (g == 8) { ROT_CASE(8); }
    else if (g == 16) { ROT_CASE(16); }
    else { ROT_CASE(32); }
#undef ROT_CASE
#undef ROT_LAUNCH
  } else {
    split(a, kRotThreads / 32);
    any_kernel<T, BWD><<<a.side[0].ctas + a.side[1].ctas, kRotThreads, 0, s>>>(a);
  }
  int rc = launch_status();
  if (BWD && rc == ASCAN_OK) {
    weight_kernel<<<dim3((a.dim + 31) / 32, 2), 1024, 0, s>>>(a);
    rc = launch_status();
  }
  return rc;
}

static bool side_ok(const ascan_rows* r) {
  return r && r->data && r->heads > 0 && r->heads <= 65535 && r->stride_token >= 0 && r->stride_head >= 0;
}

static bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static bool rows_vec(const ascan_rows* r, int v) {
  return aligned(r->data) && r->stride_token % v == 0 && r->stride_head % v == 0;
}

static int fill(Args& a, const ascan_rows* q, const ascan_rows* k, const void* wq, const void* wk, int wtype,
                const float* ct, const float* st, int64_t rows, int half, int interleaved, const void* positions,
                const void* cu, int itype, int64_t N, int64_t tokens, int dim, int dtype, float eps, void* oq, void* ok) {
  if (tokens < 0 || tokens > (1ll << 40) || dim <= 0 || dim > (1 << 20) || half < 0 || 2 * half > dim || rows < 0 || N < 0)
    return ASCAN_EINVAL;
  if (dtype < ASCAN_F32 || dtype > ASCAN_BF16 || wtype < ASCAN_F32 || wtype > ASCAN_BF16) return ASCAN_EINVAL;
  if (itype != ASCAN_I32 && itype != ASCAN_I64) return ASCAN_EINVAL;
  if (!positions == !cu) return ASCAN_EINVAL;
  if (tokens == 0) return ASCAN_OK;
  if (!side_ok(q) || !side_ok(k) || !wq || !wk || !oq || !ok || (half > 0 && (!ct || !st))) return ASCAN_EINVAL;
  const ascan_rows* r[2] = {q, k};
  const void* w[2] = {wq, wk};
  void* o[2] = {oq, ok};
  for (int s = 0; s < 2; ++s) {
    a.side[s].x = r[s]->data;
    a.side[s].st = r[s]->stride_token;
    a.side[s].sh = r[s]->stride_head;
    a.side[s].w = w[s];
    a.side[s].out = o[s];
    a.side[s].heads = r[s]->heads;
  }
  a.cos_table = ct;
  a.sin_table = st;
  a.positions = positions;
  a.cu = cu;
  a.rows = rows;
  a.N = N;
  a.tokens = tokens;
  a.index64 = itype == ASCAN_I64;
  a.half = half;
  a.interleaved = interleaved != 0;
  a.dim = dim;
  a.wtype = wtype;
  a.eps = eps;
  a.err = g_err_host;
  return ASCAN_OK;
}

static bool vec_ok(const Args& a, const ascan_rows* q, const ascan_rows* k, const ascan_rows* dq, const ascan_rows* dk,
                   int dtype) {
  const int v = dtype == ASCAN_F32 ? 4 : 8;
  if (a.dim % v || a.dim / v > 32 || a.half % v) return false;
  if (!rows_vec(q, v) || !rows_vec(k, v) || !aligned(a.side[0].out) || !aligned(a.side[1].out)) return false;
  if (dq && (!rows_vec(dq, v) || !rows_vec(dk, v))) return false;
  return a.half == 0 || (aligned(a.cos_table) && aligned(a.sin_table));
}

}  // namespace rotate
}  // namespace ascan

using namespace ascan;

extern "C" {

int ascan_qk_norm_rotate(const ascan_rows* queries, const ascan_rows* keys, const void* query_weight,
                         const void* key_weight, int weight_dtype, const float* cos_table, const float* sin_table,
                         int64_t table_rows, int half, int interleaved, const void* positions, const void* cu_seqlens,
                         int index_type, int64_t num_seq, int64_t tokens, int dim, int dtype, float eps,
                         void* out_queries, void* out_keys, void* stream) {
  rotate::Args a{};
  const int rc = rotate::fill(a, queries, keys, query_weight, key_weight, weight_dtype, cos_table, sin_table, table_rows,
                              half, interleaved, positions, cu_seqlens, index_type, num_seq, tokens, dim, dtype, eps,
                              out_queries, out_keys);
  if (rc != ASCAN_OK || tokens == 0) return rc;
  const bool vec = rotate::vec_ok(a, queries, keys, nullptr, nullptr, dtype);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ASCAN_F32) return rotate::run<float, false>(a, vec, s);
  if (dtype == ASCAN_F16) return rotate::run<__half, false>(a, vec, s);
  return rotate::run<__nv_bfloat16, false>(a, vec, s);
}

size_t ascan_qk_norm_rotate_workspace(int64_t tokens, int query_heads, int key_heads, int dim) {
  (void)query_heads;
  (void)key_heads;
  if (tokens <= 0 || dim <= 0) return 256;
  return 256 + static_cast<size_t>(rotate::kMaxCtas + 2) * dim * sizeof(float);
}

int ascan_qk_norm_rotate_backward(const ascan_rows* queries, const ascan_rows* keys, const void* query_weight,
                                  const void* key_weight, int weight_dtype, const float* cos_table,
                                  const float* sin_table, int64_t table_rows, int half, int interleaved,
                                  const void* positions, const void* cu_seqlens, int index_type, int64_t num_seq,
                                  int64_t tokens, int dim, int dtype, float eps, const ascan_rows* d_out_queries,
                                  const ascan_rows* d_out_keys, void* d_queries, void* d_keys, void* d_query_weight,
                                  void* d_key_weight, void* workspace, size_t workspace_bytes, void* stream) {
  rotate::Args a{};
  const int rc = rotate::fill(a, queries, keys, query_weight, key_weight, weight_dtype, cos_table, sin_table, table_rows,
                              half, interleaved, positions, cu_seqlens, index_type, num_seq, tokens, dim, dtype, eps,
                              d_queries, d_keys);
  if (rc != ASCAN_OK || tokens == 0) return rc;
  if (!rotate::side_ok(d_out_queries) || !rotate::side_ok(d_out_keys) || d_out_queries->heads != queries->heads ||
      d_out_keys->heads != keys->heads || !d_query_weight || !d_key_weight)
    return ASCAN_EINVAL;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) ||
      workspace_bytes < ascan_qk_norm_rotate_workspace(tokens, queries->heads, keys->heads, dim))
    return ASCAN_EWORKSPACE;
  const ascan_rows* dy[2] = {d_out_queries, d_out_keys};
  void* dw[2] = {d_query_weight, d_key_weight};
  for (int s = 0; s < 2; ++s) {
    a.side[s].dy = dy[s]->data;
    a.side[s].dst = dy[s]->stride_token;
    a.side[s].dsh = dy[s]->stride_head;
    a.side[s].dw = dw[s];
  }
  // the query CTAs' rows come first; split() keeps each side within its share
  const long long total = queries->heads + keys->heads;
  a.side[0].part = static_cast<float*>(workspace);
  a.side[1].part = a.side[0].part + max(1ll, rotate::kMaxCtas * queries->heads / total) * dim;
  const bool vec = rotate::vec_ok(a, queries, keys, d_out_queries, d_out_keys, dtype);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ASCAN_F32) return rotate::run<float, true>(a, vec, s);
  if (dtype == ASCAN_F16) return rotate::run<__half, true>(a, vec, s);
  return rotate::run<__nv_bfloat16, true>(a, vec, s);
}

}  // extern "C"

namespace ascan {
ASCAN_UNIT_ERROR_ACCESSORS(rotate)
}  // namespace ascan
