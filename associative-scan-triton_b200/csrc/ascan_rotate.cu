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
// group by shuffles.  A group walks the heads of consecutive tokens with
// several heads' loads in flight and a token's angles read once for all of
// them.  Queries and keys share a launch: the first CTAs take the query heads,
// the rest the key heads.  The weights' gradients stay in registers over all
// of a group's heads, meet in shared memory, and a second launch adds the
// CTAs' rows in a fixed order, so results repeat bit for bit.
#include "ascan_impl.cuh"
#include "ascan_mscan.cuh"

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

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float* x) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < Vec<T>::V; ++i) x[i] = to_f(e[i]);
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float* x) {
  uint4 u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < Vec<T>::V; ++i) e[i] = from_f<T>(x[i]);
  return u;
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

// How the lane's elements of a token turn: y[i] = x[i] p[i] + x'[i] q[i] with x'
// the partner, for the forward with the weights in p and q (w[i] cos, +-w' sin),
// for the gradients of the transposed turn without them (cos, -+sin).
template <typename T, bool BWD>
struct Turn {
  static constexpr int V = Vec<T>::V;
  float p[V], q[V];

  __device__ __forceinline__ void load(const Args& a, const Side& sd, long long row, int gl, int partner) {
    float c[V], s[V];
    const int hv = a.half / V;
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = 1.f, s[i] = 0.f;
    if (row >= 0 && gl < 2 * hv) {
      const float* ct = a.cos_table + row * a.half;
      const float* st = a.sin_table + row * a.half;
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const int at = (gl * V + i) / 2;
          c[i] = c[i + 1] = __ldg(ct + at);
          const float v = __ldg(st + at);
          s[i] = -v, s[i + 1] = v;
        }
      } else {
        const int at = (gl < hv ? gl : gl - hv) * V;
        const float sign = gl < hv ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const float4 cv = __ldg(reinterpret_cast<const float4*>(ct + at + i));
          const float4 sv = __ldg(reinterpret_cast<const float4*>(st + at + i));
          c[i] = cv.x, c[i + 1] = cv.y, c[i + 2] = cv.z, c[i + 3] = cv.w;
          s[i] = sign * sv.x, s[i + 1] = sign * sv.y, s[i + 2] = sign * sv.z, s[i + 3] = sign * sv.w;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (BWD) {
        p[i] = c[i], q[i] = -s[i];
      } else {
        const int mine = gl * V + i, other = a.interleaved ? mine ^ 1 : partner * V + i;
        p[i] = mine < a.dim ? c[i] * load_any(sd.w, a.wtype, mine) : 0.f;
        q[i] = s[i] != 0.f ? s[i] * load_any(sd.w, a.wtype, other) : 0.f;
      }
    }
  }

  // Every lane of the warp takes part.
  template <int G>
  __device__ __forceinline__ void apply(const Args& a, const uint4& raw, int partner, const float* x, float* y) const {
    float o[V];
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = x[i ^ 1];
    } else {
      uint4 r;
      r.x = __shfl_sync(kFull, raw.x, partner, G);
      r.y = __shfl_sync(kFull, raw.y, partner, G);
      r.z = __shfl_sync(kFull, raw.z, partner, G);
      r.w = __shfl_sync(kFull, raw.w, partner, G);
      unpack<T>(r, o);
    }
    // an element that does not turn has q = 0; select, so that an infinity in
    // its place of the pair does not become 0 * inf
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = q[i] == 0.f ? x[i] * p[i] : fmaf(o[i], q[i], x[i] * p[i]);
  }
};

// A group walks `span` tokens in order and, for each, heads [h0, h1) of its
// side.  DEPTH heads' loads are always in flight, over token boundaries too.
template <typename T, int G, int DEPTH, bool BWD>
__global__ void __launch_bounds__(kRotThreads, BWD ? 2 : 3) vec_kernel(const __grid_constant__ Args a) {
  constexpr int V = Vec<T>::V;
  constexpr int GROUPS = kRotThreads / G;
  const bool is_key = static_cast<int>(blockIdx.x) >= a.side[0].ctas;
  const Side& sd = a.side[is_key];
  const int cta = is_key ? blockIdx.x - a.side[0].ctas : blockIdx.x;
  const int gl = threadIdx.x % G, group = threadIdx.x / G;
  const bool on = gl * V < a.dim;
  const int hv = a.half / V;
  const int partner = gl < hv ? gl + hv : (gl < 2 * hv ? gl - hv : gl);
  check_cu(a);
  const long long g = static_cast<long long>(cta) * GROUPS + group;
  const int slice = static_cast<int>(g % sd.slices);
  const int h0 = slice * sd.heads_per, h1 = min(h0 + sd.heads_per, sd.heads);
  const long long first = g / sd.slices * sd.span;
  const long long tokens = max(0ll, min(static_cast<long long>(sd.span), a.tokens - first));
  // every group of a warp runs the same number of rounds: the shuffles need them
  const int items = static_cast<int>(sd.span) * sd.heads_per;
  float w[V], dw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = BWD && on ? load_any(sd.w, a.wtype, gl * V + i) : 0.f;
    dw[i] = 0.f;
  }
  const float inv = 1.f / static_cast<float>(a.dim);
  const T* src = static_cast<const T*>(sd.x) + gl * V;
  const T* dsrc = BWD ? static_cast<const T*>(sd.dy) + gl * V : nullptr;
  uint4 raw[DEPTH], draw[BWD ? DEPTH : 1];
  int lt = 0, lh = h0;  // the next load
  auto load = [&](int q) {
    const bool ok = on && lt < tokens && lh < h1;
    raw[q] = ok ? __ldcs(reinterpret_cast<const uint4*>(src + (first + lt) * sd.st + lh * sd.sh)) : make_uint4(0, 0, 0, 0);
    if (BWD) draw[q] = ok ? __ldcs(reinterpret_cast<const uint4*>(dsrc + (first + lt) * sd.dst + lh * sd.dsh)) : make_uint4(0, 0, 0, 0);
    if (++lh >= h0 + sd.heads_per) lh = h0, ++lt;
  };
#pragma unroll
  for (int q = 0; q < DEPTH; ++q) load(q);
  Turn<T, BWD> turn;
  Place place;
  long long row = -1;
  int ct = 0, ch = h0;  // the next head to finish
  for (int r = 0; r < items; r += DEPTH) {
#pragma unroll
    for (int q = 0; q < DEPTH; ++q) {
      const long long t = first + ct;
      const bool live = ct < tokens && ch < h1;
      if (ch == h0) {
        row = ct < tokens ? next_row(a, t, place) : -1;
        turn.load(a, sd, row, gl, partner);
      }
      float x[V], y[V], sq = 0.f;
      unpack<T>(raw[q], x);
#pragma unroll
      for (int i = 0; i < V; ++i) sq = fmaf(x[i], x[i], sq);
      const float rs = rsqrtf(fmaf(group_sum<G>(sq), inv, a.eps));
      if (!BWD) {
        turn.template apply<G>(a, raw[q], partner, x, y);
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = row >= 0 ? y[i] * rs : 0.f;
      } else {
        float dy[V], dz[V], sum = 0.f;
        unpack<T>(draw[q], dy);
        turn.template apply<G>(a, draw[q], partner, dy, dz);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[i] *= rs;  // xh
          const float gw = dz[i] * x[i];
          if (live && row >= 0) dw[i] += gw;
          sum = fmaf(gw, w[i], sum);
        }
        const float mean = group_sum<G>(sum) * inv;
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = row >= 0 ? rs * fmaf(-x[i], mean, w[i] * dz[i]) : 0.f;
      }
      load(q);
      if (live && on)
        __stcs(reinterpret_cast<uint4*>(static_cast<T*>(sd.out) + (t * sd.heads + ch) * a.dim + gl * V), pack<T>(y));
      if (++ch >= h0 + sd.heads_per) ch = h0, ++ct;
    }
  }
  if (BWD) {
    __shared__ float red[GROUPS][G * V];
#pragma unroll
    for (int i = 0; i < V; ++i) red[group][gl * V + i] = dw[i];
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
    constexpr int D = BWD ? 2 : 4;
    if (g == 8) vec_kernel<T, 8, D, BWD><<<grid, kRotThreads, 0, s>>>(a);
    else if (g == 16) vec_kernel<T, 16, D, BWD><<<grid, kRotThreads, 0, s>>>(a);
    else vec_kernel<T, 32, D, BWD><<<grid, kRotThreads, 0, s>>>(a);
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
