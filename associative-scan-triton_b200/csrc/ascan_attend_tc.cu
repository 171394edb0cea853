// ascan_attend_tc.cu -- compilation unit of the scan library: causal softmax
// attention on the fifth-generation tensor cores (bfloat16 and float16).
//
// Tiles are 128 tokens by 128; TMA brings them into shared memory (128-byte
// swizzle), accumulators and the operands that are computed on the way live in
// tensor memory, one thread of the row per lane.  One CTA per SM, by warp:
//
//   0-7  softmax: scores -> probabilities (or their derivatives), rounded to
//        the inputs' type as operands of the next product
//   8    TMA loads
//   9    issues the products
//   10   gradients of keys and values: the rows' statistics
//
// forward: two tiles of queries share the keys and values that pass; while one
//   tile's scores are on the tensor cores the other's softmax runs.  Per tile
//   S = Q K^T, then P in place, O += P V.  The reference of a row's softmax
//   moves only when a score exceeds it by 2^8: until then nothing in O has to
//   be touched, and P stays in range (float16's 2^16 included).
// dq: one tile of queries walks the keys: S = Q K^T and dP = dO V^T, dS in
//   S's place, dQ += dS K.  Two S take turns, so that the next one is computed
//   while the warps are at this one.
// dk, dv: one tile of keys walks the queries of all heads that share it, with
//   everything transposed: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO with P^T in
//   S^T's place, dK += dS^T Q with dS^T in dP^T's.  The next S^T follows dV's
//   product, so that its softmax runs while dK's and the next dP^T's do.
//
// Rounding P and dS to the inputs' type adds an error of the size of the
// result's own rounding: each is off by at most half a step of itself, and
// independently, so a sum of them is off by that of its root of squares.
// Scores, sums, and what is subtracted from dP are float32.  Before gradients O
// is divided by the sum of the rounded P, so that it is a mean of values
// whatever the roundings are: what all values share stays exact in do.o, whose
// difference from dP is all that is left of a gradient where values are alike.
// The gradients' own P comes from the exact sum.  (The second sum takes the
// forward of 8 x 2048 tokens of 12 heads from 142 to 166 us; without gradients
// O's own rounding is larger than what it would mend.)
//
// A value that is not finite may stand behind the mask in the tile that the
// diagonal crosses, and rows behind a sequence's end belong to another one;
// 0 * NaN would carry them into other rows.  So rows behind the end are zeroed
// in shared memory before they meet a product as its inner side, and in the
// diagonal's tile what is not finite is too; where the mask lets it through it
// is added to the finished rows (forward), makes a row NaN (dv), or has done so
// through the scores already (dq, dk).
//
// Measured, bfloat16, heads of 128 (half of all products count, as the mask has
// it): forward of 32768 tokens of 16 heads 3383 us, 1300 TFLOP/s; of 16 x 1024
// 121 us and of 64 x 256 73 us, where the blocks at a tile's start and on the
// diagonal, whose two halves have nothing to overlap with, are most of the
// work.  With gradients, 8 x 2048 tokens of 12 heads: forward 171 us (603
// TFLOP/s), dq 176 (three products, 878 TFLOP/s), dk and dv 228 (four, 904
// TFLOP/s), do.o 36.  On long sequences the
// power limit and the exponentials bound the forward: the tensor cores take 1024
// cycles for a block's two products and the special-function units as many for
// its exponentials at sixteen a cycle, so three of eight are polynomials on the
// multiply-add pipe.  The gradients are bound by what one CTA does in a row:
// about 7 us before the first product and after the last, and the way scores ->
// derivative -> next product for each block in between.
//
// Every wait is bounded: one that runs out sets the device error word and an
// abort flag, every role then leaves its loop, loads and products in flight
// are waited for, and tensor memory is freed.
#include "ascan_impl.cuh"
#include "ascan_attend.cuh"
#include "ascan_pairs.cuh"
#include "ascan_tc.cuh"

namespace ascan {
namespace attend {

using namespace tc;

constexpr int kC = 128;  // rows and columns of a tile
constexpr int kTcWarps = 12, kTcThreads = kTcWarps * 32;
constexpr int kBlock = 16384;  // 128 rows of 64 elements
constexpr int kMaxSlots = 6;

struct Maps {
  CUtensorMap q, k, v, d_out;
};

// A slot for tiles of keys and of values.
__host__ __device__ inline int slot_bytes(int dk, int dv) { return dk > 64 || dv > 64 ? 2 * kBlock : kBlock; }

struct Common {
  uint64_t drain;
  int abort;
  uint32_t tmem;
};

__device__ __noinline__ bool wait_slow(uint64_t* b, uint32_t parity, Common* t, uint32_t* err) {
  const unsigned long long start = now_ns();
  volatile int* ab = &t->abort;
  while (true) {
    for (int i = 0; i < 16; ++i)
      if (bar_try(b, parity)) return true;
    if (*ab) return false;
    if (now_ns() - start > kStageTimeoutNs) {
      *ab = 1;
      report(ASCAN_DEV_ERR_STAGE, (static_cast<unsigned long long>(blockIdx.x) << 32) | threadIdx.x, err);
      return false;
    }
  }
}

struct Ctl {
  Common* t;
  uint32_t* err;
  __device__ __forceinline__ bool wait(uint64_t* b, uint32_t parity) const {
    return bar_try(b, parity) || wait_slow(b, parity, t, err);
  }
  // All lanes of a role wait; false once the CTA gives up.
  __device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity) const { return __all_sync(kFull, wait(b, parity)); }
  // After a give-up: what is in flight must land before the CTA leaves.
  __device__ __forceinline__ void land(uint64_t* b, uint32_t parity) const {
    const unsigned long long start = now_ns();
    while (!bar_try(b, parity) && now_ns() - start < kStageTimeoutNs) {
    }
  }
};

__device__ __forceinline__ void warp_arrive(uint64_t* b) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) bar_arrive(b);
}

// Loads a tile of `dim` columns; `on` has received its bytes before.
__device__ __forceinline__ void load_tile(unsigned char* to, const CUtensorMap* m, int dim, int head, long long token, uint64_t* on) {
  for (int b = 0; b * 64 < dim; ++b) tma_rows(smem_u32(to) + b * kBlock, m, b * 64, head, static_cast<int>(token), on);
}
__device__ __forceinline__ uint32_t tile_bytes(int dim) { return dim > 64 ? 2 * kBlock : kBlock; }

// A B^T over `dim` columns of two tiles in shared memory.
__device__ __forceinline__ void scores(uint32_t to, uint64_t a, uint64_t b, uint32_t id, int dim) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (k * 16 >= dim) break;
    const uint32_t o = (k >> 2) * (kBlock >> 4) + (k & 3) * 2;
    mma_smem(to, a + o, b + o, id, k > 0);
  }
}

// The wait for a load, tied to its registers: the next load may be in flight
// while these are worked on.
__device__ __forceinline__ void wait_ld16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(uint64_t x);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(uint64_t x) {
  const float2 f = unpair(x);
  return bf2(f.x, f.y);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(uint64_t x) {
  const float2 f = unpair(x);
  return hf2(f.x, f.y);
}
template <typename T>
__device__ __forceinline__ uint64_t unpack2(uint32_t x);
template <>
__device__ __forceinline__ uint64_t unpack2<__nv_bfloat16>(uint32_t x) { return pair(lo_f(x), hi_f(x)); }
template <>
__device__ __forceinline__ uint64_t unpack2<__half>(uint32_t x) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
  return pair(f.x, f.y);
}
__device__ __forceinline__ uint64_t pair_of(const uint32_t* x) { return pair(__uint_as_float(x[0]), __uint_as_float(x[1])); }
__device__ __forceinline__ uint64_t ex2_2(uint64_t x) {
  const float2 f = unpair(x);
  return pair(ex2(f.x), ex2(f.y));
}
// Of eight pairs of scores so many take the polynomial.
constexpr int kPoly = 3;

// 2^x of a pair by a polynomial of degree 4 on [-1/2, 1/2] (fitted to the
// smallest relative error, 2.6e-6) and the exponent's bits; below 2^-126 what is
// left is as small, and NaN comes out infinite, which makes a row NaN as well.
// The special function unit has four lanes for the
// scheduler's thirty-two.
__device__ __forceinline__ uint64_t poly_ex2_2(uint64_t x) {
  float2 f = unpair(x);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(f.x) : "f"(-126.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(f.y) : "f"(-126.f));
  const uint64_t y = pair(f.x, f.y), magic = pair(12582912.f, 12582912.f);
  const uint64_t n = add2(y, magic);  // the nearest whole number, in the low bits
  const uint64_t r = fma2(add2(n, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), y);
  uint64_t q = fma2(pair(0.009570100344717503f, 0.009570100344717503f), r, pair(0.05591785907745361f, 0.05591785907745361f));
  q = fma2(q, r, pair(0.240247443318367f, 0.240247443318367f));
  q = fma2(q, r, pair(0.6931217908859253f, 0.6931217908859253f));
  q = fma2(q, r, pair(0.9999992847442627f, 0.9999992847442627f));
  const float2 a = unpair(n), b = unpair(q);
  return pair(__uint_as_float((__float_as_uint(a.x) << 23) + __float_as_uint(b.x)),
              __uint_as_float((__float_as_uint(a.y) << 23) + __float_as_uint(b.y)));
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

template <typename T>
__device__ __forceinline__ bool f16() { return false; }
template <>
__device__ __forceinline__ bool f16<__half>() { return true; }

// sum + 0 * x for both elements of a word: NaN if one is not finite.
template <typename T>
__device__ __forceinline__ uint32_t zero_times(uint32_t x, uint32_t sum) {
  if (f16<T>()) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0));
  else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0));
  return sum;
}

// Row `row` of a tile with `blocks` of 64 columns from block `b`: zeros if it is
// not `live`, else without what is not finite.  True if there was any.
template <typename T>
__device__ __forceinline__ bool clean_row(unsigned char* tile, int row, int b, int blocks, bool live) {
  auto place = [&](int c) { return reinterpret_cast<uint4*>(tile + (b + (c >> 3)) * kBlock + row * 128 + (((c & 7) ^ (row & 7)) << 4)); };
  uint32_t sum[2] = {0, 0};
#pragma unroll 8
  for (int c = 0; c < 8 * blocks; ++c) {
    if (!live) {
      *place(c) = make_uint4(0, 0, 0, 0);
      continue;
    }
    const uint4 x = *place(c);
    sum[0] = zero_times<T>(x.x, sum[0]);
    sum[1] = zero_times<T>(x.y, sum[1]);
    sum[0] = zero_times<T>(x.z, sum[0]);
    sum[1] = zero_times<T>(x.w, sum[1]);
  }
  if (!(((sum[0] | sum[1]) & 0x7fff7fffu) != 0)) return false;
  const uint32_t ones = f16<T>() ? 0x7c00u : 0x7f80u;
#pragma unroll 1
  for (int c = 0; c < 64 * blocks; ++c) {
    uint16_t* at = reinterpret_cast<uint16_t*>(place(c >> 3)) + (c & 7);
    if ((*at & ones) == ones) *at = 0;
  }
  return true;
}

// 64 columns of a warp's 32 rows from registers (32 packed words a lane) to
// memory in whole lines; `stage`: 4 KB of the warp's own.
__device__ __forceinline__ void store_block(unsigned char* stage, const uint32_t* x, unsigned char* to, long long stride, int rows,
                                            int cols) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
  __syncwarp();
  const int c = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3);
    if (r < rows && c * 8 < cols)
      *reinterpret_cast<uint4*>(to + r * stride + c * 16) = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
  }
  __syncwarp();
}

// 64 columns of the warp's lanes, times f, packed.
template <typename T>
__device__ __forceinline__ void fetch_block(uint32_t tm, float f, uint32_t* out) {
  const uint64_t f2 = pair(f, f);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t x[32];
    tmem_ld32(tm + 32 * half, x);
    wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) out[16 * half + i] = pack2<T>(mul2(pair_of(x + 2 * i), f2));
  }
}

// dS of a sequence's first token, in the low half: it sees one key, with p = 1,
// so there is none, not even a rounding, unless something is not finite.
template <typename T>
__device__ __forceinline__ uint32_t only_key(uint32_t w) {
  const float x = unpair(unpack2<T>(w)).x;
  return x - x == 0.f ? 0u : 0x7fffu;
}

// float16's steps end at 2^-24, where a P or dS of a long row soon would be.  So
// P is taken in units of 2^-15 there (for dv), and dS in units that bring the
// most it can be to 2^15 or less: |dS| = p |dP - sum p dP| <= max |dP| / 2, and
// |dP| <= dv max |do| max |v|, whose exponents are rounded up here.
template <typename T>
__device__ __forceinline__ float p_bits() { return f16<T>() ? 15.f : 0.f; }
template <typename T>
__device__ __forceinline__ float ds_unit(const Problem& p) {
  if (!f16<T>()) return 1.f;
  const int g = static_cast<int>(__ldg(p.top) >> 23), v = static_cast<int>(__ldg(p.top + 1) >> 23);
  if (g == 0 || v == 0) return 1.f;  // nothing but zeros
  const int log_dv = 32 - __clz(p.dv - 1);
  return __uint_as_float(static_cast<uint32_t>(g - 126 + v - 126 + log_dv - 1 - 15 + 127) << 23);
}

__device__ __forceinline__ bool misplaced(const unsigned char* smem, uint32_t* err) {
  if (!(smem_u32(smem) & 1023u)) return false;  // the swizzled layouts need it
  if (threadIdx.x == 0) report(ASCAN_DEV_ERR_STAGE, 0xffffffffull, err);
  return true;
}

// A place in the ring and the parity of its turn.
struct Cursor {
  int at = 0;
  uint32_t turn = 0;
  __device__ __forceinline__ void next(int ns) {
    if (++at == ns) at = 0, turn ^= 1;
  }
};

// A value that all lanes have: behind a shuffle the compiler knows it, and keeps
// what a product is issued with in uniform registers.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(kFull, x, 0); }

// All 512 columns of tensor memory, by one warp; the barriers are ready behind it.
__device__ __forceinline__ uint32_t open_tmem(Common* t, int warp = 9) {
  if (threadIdx.x >> 5 == warp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&t->tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    fence_before();
  }
  __syncthreads();
  fence_after();
  return uniform(t->tmem);
}
__device__ __forceinline__ void close_tmem(uint32_t tm, int warp = 9) {
  __syncwarp();
  fence_before();
  __syncthreads();
  if (threadIdx.x >> 5 == warp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm));
  }
}
__device__ __forceinline__ void bars_done() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  fence_async();
}

// cu_seqlens as the scans check it, by `threads` threads.
__device__ __forceinline__ void check_cu(const Problem& p, int thread, int threads) {
  uint32_t bits = 0;
  auto at = [&](long long i) {
    return p.cu64 ? static_cast<const long long*>(p.cu)[i] : static_cast<long long>(static_cast<const int*>(p.cu)[i]);
  };
  for (long long i = thread; i <= p.N; i += threads) {
    const long long v = at(i);
    if (v < 0 || v > p.BL || (i < p.N && at(i + 1) < v)) bits |= ASCAN_DEV_ERR_CU_ORDER;
    if (i == p.N && v != p.BL) bits |= ASCAN_DEV_ERR_CU_END;
  }
  if (bits) report(bits, 0ull, p.err);
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

constexpr int kFwdSoftmax = 8, kFwdThreads = (kFwdSoftmax + 2) * 32;

// The forward's ring: a slot less than the gradients', for rows on their way out.
__host__ __device__ inline int forward_slots(int dk, int dv) { return dk > 64 || dv > 64 ? 4 : kMaxSlots; }
constexpr int kStage = 4096;  // of a warp: 32 rows of 64 elements

// An item's place is searched for in shared memory, eight times as fast as
// through what the slots leave of the first cache.
constexpr int kEnds = 512;
constexpr int kItems = 4;  // that the loads may be ahead

// A work item: two tiles of queries of one head; `key` blocks of keys of each.
struct Item {
  int start, token, left;  // the sequence's first token, the item's, and the sequence's from there on
  int h, n_a, n_b, n;      // n 0: no tokens
};
struct ForwardTail {
  Common c;
  uint64_t q_full, q_empty, full[kMaxSlots], empty[kMaxSlots], s_full[2], p_ready[2], o_done[2], item_full[kItems], item_empty[kItems], next_full;
  alignas(16) uint32_t next[4];  // the scheduler's answer
  Item items[kItems];           // n 0: no more
  uint32_t bad[4][2][4];  // by work item: tokens of the tiles' own blocks with values that are not finite
  int ends[kEnds];        // cu_seqlens, if it is no longer
};

// Takes over the work of a CTA that has not been launched yet: the answer, its
// number or none, comes to `to`.
__device__ __forceinline__ void ask_work(uint32_t* to, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(to)),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ int read_work(const uint32_t* from) {  // -1: none is left
  uint32_t got, x;
  asm volatile(
      "{\n .reg .b128 r;\n .reg .pred p;\n .reg .b32 y, z, w;\n .reg .b64 lo, hi;\n"
      " ld.shared.v2.b64 {lo, hi}, [%2];\n mov.b128 r, {lo, hi};\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, r;\n}\n"
      : "=r"(got), "=r"(x)
      : "r"(smem_u32(from))
      : "memory");
  return got ? static_cast<int>(x) : -1;
}

__device__ __forceinline__ Item find_item(const Problem& p, const int* ends, int x, int h) {
  Item i;
  i.h = h;
  const Tile t = p.N < kEnds ? find_tile<8>(p, x, [&](int n) { return ends[n]; }) : find_tile<8>(p, x);
  const int own = t.first / kC;  // the first tile's own block of keys
  i.start = t.start;
  i.token = t.start + t.first;
  i.left = t.len - t.first;
  i.n_a = t.first < 0 ? 0 : own + 1;
  i.n_b = t.first >= 0 && i.left > kC ? own + 2 : 0;
  i.n = max(i.n_a, i.n_b);
  return i;
}

// To the warps that compute: the count-th item with tokens, or that there is
// none any more.
__device__ __forceinline__ bool hand_out(const Ctl& ctl, ForwardTail& s, uint32_t count, const Item& it) {
  const uint32_t u = count % kItems;
  if (count >= kItems && !ctl.wait(&s.item_empty[u], (count / kItems - 1) & 1)) return false;
  s.items[u] = it;
  bar_arrive(&s.item_full[u]);
  return true;
}

// What a row has added up: its exponentials, the same rounded as P, and the
// reference that they are taken against.
struct RowState {
  uint64_t l[2], z[2];
  float m;
};

// P of a block whose scores exceed the row's reference by more than 2^8 (the
// first block is one), or that the diagonal crosses (columns up to `last`): the
// maximum first, then O and the sums to the new reference (o32: O's columns in
// blocks of 32).  Out of line, so that the loop that runs nearly always keeps
// everything in registers: with 227 KB of shared memory in use a spilled one
// costs more than it saves.
template <typename T, bool TRAIN>
__device__ __noinline__ RowState move_reference(uint32_t ts, uint32_t to, int last, int o32, float c2, RowState r) {
  const int blocks = __reduce_max_sync(kFull, last) / 32;  // of 32 columns, up to the last that a row of the warp sees
  float high = -INFINITY;
#pragma unroll 1
  for (int i = 0; i <= blocks; ++i) {
    uint32_t sc[32];
    tmem_ld32(ts + 32 * i, sc);
    wait_ld();
#pragma unroll
    for (int e = 0; e < 32; e += 2)
      high = max3(high, 32 * i + e > last ? -INFINITY : __uint_as_float(sc[e]),
                  32 * i + e + 1 > last ? -INFINITY : __uint_as_float(sc[e + 1]));
  }
  const float next = (high - r.m) * c2 > 8.f ? high : r.m;
  if (o32 > 0 && __any_sync(kFull, next != r.m)) {
    const float f = next == -INFINITY ? 1.f : ex2((r.m - next) * c2);
    const uint64_t f2 = pair(f, f);
    r.l[0] = mul2(r.l[0], f2), r.l[1] = mul2(r.l[1], f2);
    if (TRAIN) r.z[0] = mul2(r.z[0], f2), r.z[1] = mul2(r.z[1], f2);
#pragma unroll 1
    for (int i = 0; i < o32; ++i) {
      uint32_t o[32];
      tmem_ld32(to + 32 * i, o);
      wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
      tmem_st32(to + 32 * i, o);
    }
  }
  r.m = next;
  const float ref = r.m == -INFINITY ? 0.f : -r.m * c2;  // a row of -inf so far
  const uint64_t ref2 = pair(ref, ref), c22 = pair(c2, c2);
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = 0;
    if (i <= blocks) {
      uint32_t sc[32];
      tmem_ld32(ts + 32 * i, sc);
      wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (32 * i + e > last) sc[e] = 0xff800000u;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint64_t y = ex2_2(fma2(pair_of(sc + 2 * e), c22, ref2));
        w[e] = pack2<T>(y);
        r.l[e & 1] = add2(r.l[e & 1], y);
        if (TRAIN) r.z[e & 1] = add2(r.z[e & 1], unpack2<T>(w[e]));
      }
    }
    tmem_st16(ts + 16 * i, w);
  }
  return r;
}

// TRAIN: a gradient will follow.  A CTA works through items: its own, and then
// those of CTAs that were not launched yet, so that loads and products of the
// next item run while the rows of this one are finished.
template <typename T, bool TRAIN>
__global__ void __launch_bounds__(kFwdThreads, 1) tc_forward_kernel(const __grid_constant__ Problem p, const __grid_constant__ Maps maps) {
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (misplaced(smem, p.err)) return;
  const int slot = slot_bytes(p.dk, p.dv), ns = forward_slots(p.dk, p.dv), q_bytes = tile_bytes(p.dk);
  unsigned char *ring = smem + 2 * q_bytes, *stages = ring + ns * slot;
  ForwardTail& s = *reinterpret_cast<ForwardTail*>(stages + kFwdSoftmax * kStage);
  const Ctl ctl{&s.c, p.err};
  if (tid == 0) {
    bar_init(&s.q_full, 1);
    bar_init(&s.q_empty, 1);
    for (int i = 0; i < ns; ++i) bar_init(&s.full[i], 1), bar_init(&s.empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(&s.s_full[i], 1);
      bar_init(&s.p_ready[i], 4);
      bar_init(&s.o_done[i], 1);
    }
    for (int i = 0; i < kItems; ++i) bar_init(&s.item_full[i], 1), bar_init(&s.item_empty[i], kFwdSoftmax + 1);
    bar_init(&s.next_full, 1);
    bar_init(&s.c.drain, 1);
    s.c.abort = 0;
    bars_done();
  }
  if (p.N < kEnds)
    for (int i = tid; i <= p.N; i += kFwdThreads) s.ends[i] = static_cast<int>(cu_at(p, i));
  const uint32_t tm = open_tmem(&s.c, kFwdSoftmax + 1);
  bool ok = true;
  uint32_t base = 0;  // of the item's loads in the ring: K0, then (K[j+1], V[j]) for every j

  if (warp < kFwdSoftmax) {
    const int x = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad) << 21, ts = tm + lanes + x * kC, to = tm + lanes + 256 + x * kC;
    const float c2 = p.scale * kLog2e;
    const uint64_t c22 = pair(c2, c2);
    const int n32 = (p.dv + 31) / 32;
    uint32_t sp = 0, op = 0;  // phases: scores seen, rows finished
    for (uint32_t count = 0; ok; ++count) {
      const uint32_t u = count % kItems;
      if (!(ok = ctl.warp_wait(&s.item_full[u], (count / kItems) & 1))) break;
      const Item it = s.items[u];
      warp_arrive(&s.item_empty[u]);
      if (it.n == 0) break;
      const int mine = x ? it.n_b : it.n_a, left = it.left - x * kC;  // of the sequence from this tile on
      uint32_t* bad = &s.bad[count & 3][x][quad];
      if (lane == 0) *bad = 0;
      __syncwarp();
      RowState r{{0, 0}, {0, 0}, -INFINITY};
      for (int j = 0; j < mine; ++j, sp ^= 1) {
        const bool diagonal = j == mine - 1;
        if (diagonal) {  // its values may only come from this sequence, and only finite
          const uint32_t v = base + (j < it.n - 1 ? 2 * j + 2 : 2 * it.n - 1);  // of the ring's loads
          if (!(ok = ctl.warp_wait(&s.full[v % ns], (v / ns) & 1))) break;
          if (clean_row<T>(ring + v % ns * slot, row, 0, p.dv > 64 ? 2 : 1, row < left)) atomicOr(bad, 1u << lane);
          fence_async();
        }
        if (!(ok = ctl.warp_wait(&s.s_full[x], sp))) break;
        fence_after();
        // Nearly every block leaves the reference where it was: P is computed
        // with it while the maximum is looked for, and again if it has to move.
        uint32_t w[64];
        bool again = true;
        if (j > 0 && !diagonal) {
          float high = -INFINITY;
          uint64_t a[2] = {0, 0};
          const uint64_t ref2 = pair(-r.m * c2, -r.m * c2);
          uint32_t sc[2][16];
          tmem_ld16(ts, sc[0]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t* x16 = sc[i & 1];
            wait_ld16(x16);
            if (i < 7) tmem_ld16(ts + 16 * (i + 1), sc[(i + 1) & 1]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint64_t z = fma2(pair_of(x16 + 2 * e), c22, ref2);
              const uint64_t y = e >= 8 - kPoly ? poly_ex2_2(z) : ex2_2(z);
              high = max3(high, __uint_as_float(x16[2 * e]), __uint_as_float(x16[2 * e + 1]));
              w[8 * i + e] = pack2<T>(y);
              a[e & 1] = add2(a[e & 1], y);
            }
          }
          again = __any_sync(kFull, !((high - r.m) * c2 <= 8.f));
          if (!again) r.l[0] = add2(r.l[0], a[0]), r.l[1] = add2(r.l[1], a[1]);
        }
        if (again) {
          r = move_reference<T, TRAIN>(ts, to, diagonal ? row : kC - 1, j > 0 ? n32 : 0, c2, r);
        } else {
          if (TRAIN) {
#pragma unroll
            for (int e = 0; e < 64; ++e) r.z[e & 1] = add2(r.z[e & 1], unpack2<T>(w[e]));
          }
          tmem_st32(ts, w);
          tmem_st32(ts + 32, w + 32);
        }
        wait_st();
        fence_before();
        warp_arrive(&s.p_ready[x]);
      }
      if (!ok) break;
      if (mine > 0) {
        if (!(ok = ctl.warp_wait(&s.o_done[x], op))) break;
        op ^= 1;
        fence_after();
        const float2 a = unpair(add2(r.l[0], r.l[1])), b2 = unpair(add2(r.z[0], r.z[1]));
        const float l = a.x + a.y, inv = 1.f / (TRAIN ? b2.x + b2.y : l);
        const long long token = static_cast<long long>(it.token) + x * kC + row;
        if (TRAIN && row < left) p.lse[it.h * p.BL + token] = r.m * c2 + log2f(l);
        bool any = false;
        for (int i = 0; i < 4; ++i) any |= s.bad[count & 3][0][i] != 0 || (x == 1 && s.bad[count & 3][1][i] != 0);
        // whole lines: a lane's own row would be 32 of them for every store
        const long long stride = static_cast<long long>(p.H) * p.dv * 2, first = ((token - lane) * p.H + it.h) * p.dv * 2;
        const int rows = left - quad * 32;
#pragma unroll 1
        for (int b = 0; b * 64 < p.dv; ++b) {
          uint32_t u[32], v[TRAIN ? 32 : 1];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int d0 = 64 * b + 32 * half;
            uint32_t o[32];
            tmem_ld32(to + d0, o);
            wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
            if (any) {  // what was taken out of the values goes where the mask lets it
              for (int y = 0; y <= x; ++y)
                for (int i = 0; i < kC; ++i) {
                  if (!(s.bad[count & 3][y][i >> 5] >> (i & 31) & 1) || (y == x && i > row)) continue;
                  const T* from = static_cast<const T*>(p.v.p) + (static_cast<long long>(it.token) + y * kC + i) * p.v.st + it.h / p.share * p.v.sh;
#pragma unroll
                  for (int e = 0; e < 32; ++e)
                    if (d0 + e < p.dv) {
                      const float q = to_f(from[d0 + e]);
                      if (!(fabsf(q) < INFINITY)) o[e] = __float_as_uint(__uint_as_float(o[e]) + q);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              u[16 * half + e] = pack2<T>(pair_of(o + 2 * e));
              if (TRAIN) v[16 * half + e] = pack2<T>(fma2(unpack2<T>(u[16 * half + e]), pair(-1.f, -1.f), pair_of(o + 2 * e)));
            }
          }
          store_block(stages + warp * kStage, u, static_cast<unsigned char*>(p.out) + first + b * 128, stride, rows, p.dv - 64 * b);
          if (TRAIN) store_block(stages + warp * kStage, v, static_cast<unsigned char*>(p.rest) + first + b * 128, stride, rows, p.dv - 64 * b);
        }
      }
      base += 2 * it.n;
    }
  } else if (warp == kFwdSoftmax) {
    uint32_t q_loads = 0, loads = 0;
    Cursor to;
    int work = blockIdx.x;
    for (uint32_t asked = 0; ok; ++asked) {
      if (lane == 0) {  // the next number comes while this one's tiles are loaded
        bar_expect(&s.next_full, 16);
        ask_work(s.next, &s.next_full);
      }
      const int x = static_cast<int>(gridDim.x) / p.H - 1 - work / p.H, h = work % p.H;  // long rows first, a tile's heads together
      const Item it = find_item(p, s.ends, x, h);
      if (x == 0 && h == 0) check_cu(p, lane, 32);
      zero_outside<T>(p, p.out, h, p.H, p.dv, x, 2 * kC, lane, 32);
      if (it.n > 0 && lane == 0) {
        ok = hand_out(ctl, s, q_loads, it);
        if (ok && q_loads > 0) ok = ctl.wait(&s.q_empty, (q_loads - 1) & 1);
        if (ok) {
          bar_expect(&s.q_full, q_bytes * (it.n_b ? 2 : 1));
          load_tile(smem, &maps.q, p.dk, it.h, it.token, &s.q_full);
          if (it.n_b) load_tile(smem + q_bytes, &maps.q, p.dk, it.h, it.token + kC, &s.q_full);
          ++q_loads;
        }
        const int hk = it.h / p.share;
        auto load = [&](bool is_v, int j) {
          // a first pass finds all slots empty
          if (ok) ok = ctl.wait(&s.empty[to.at], to.turn ^ 1);
          if (!ok) return;
          bar_expect(&s.full[to.at], tile_bytes(is_v ? p.dv : p.dk));
          load_tile(ring + to.at * slot, is_v ? &maps.v : &maps.k, is_v ? p.dv : p.dk, hk, it.start + j * kC, &s.full[to.at]);
          to.next(ns);
          ++loads;
        };
        load(false, 0);
        for (int j = 0; ok && j < it.n; ++j) {
          if (j + 1 < it.n) load(false, j + 1);
          load(true, j);
        }
      }
      ok = __shfl_sync(kFull, ok, 0) && ctl.warp_wait(&s.next_full, asked & 1);
      if (!ok) break;
      work = read_work(s.next);
      __syncwarp();
      if (work < 0) {
        Item none{};
        if (lane == 0) hand_out(ctl, s, q_loads, none);
        break;
      }
    }
    if (lane == 0 && *reinterpret_cast<volatile int*>(&s.c.abort)) {  // what is in flight must land
      if (q_loads > 0) ctl.land(&s.q_full, (q_loads - 1) & 1);
      for (uint32_t e = loads > static_cast<uint32_t>(ns) ? loads - ns : 0; e < loads; ++e) ctl.land(&s.full[e % ns], (e / ns) & 1);
    }
  } else {
    // One thread: a vote of the warp at every wait would cost a tenth of the time.
    if (elect_one()) {
      const uint32_t id_s = idesc(kC, false, f16<T>()), id_o = idesc((p.dv + 15) / 16 * 16, true, f16<T>());
      const uint64_t q[2] = {desc(smem_u32(smem), 16), desc(smem_u32(smem) + q_bytes, 16)};
      const uint64_t k0 = desc(smem_u32(ring), 16), v0 = desc(smem_u32(ring), kBlock);
      uint32_t pp[2] = {0, 0}, qp = 0;  // phases of p_ready and q_full
      Cursor c;
      for (uint32_t count = 0; ok; ++count) {
        const uint32_t u = count % kItems;
        if (!(ok = ctl.wait(&s.item_full[u], (count / kItems) & 1))) break;
        const Item it = s.items[u];
        bar_arrive(&s.item_empty[u]);
        if (it.n == 0) break;
        {
          const int n = it.n;
          if (!(ok = ctl.wait(&s.q_full, qp) && ctl.wait(&s.full[c.at], c.turn))) break;
          qp ^= 1;
          const uint64_t k1 = k0 + c.at * (slot >> 4);
          scores(tm, q[0], k1, id_s, p.dk);
          commit(&s.s_full[0]);
          if (it.n_b) {
            scores(tm + kC, q[1], k1, id_s, p.dk);
            commit(&s.s_full[1]);
          }
          commit(&s.empty[c.at]);
          if (n == 1) commit(&s.q_empty);
          c.next(ns);
          for (int j = 0; ok && j < n; ++j) {
            const bool more = j + 1 < n;
            const int ik = c.at;
            if (more) {
              if (!(ok = ctl.wait(&s.full[c.at], c.turn))) break;
              c.next(ns);
            }
            const int iv = c.at;
            if (!(ok = ctl.wait(&s.full[c.at], c.turn))) break;
            c.next(ns);
            const uint64_t k = k0 + ik * (slot >> 4), v = v0 + iv * (slot >> 4);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int mine = x ? it.n_b : it.n_a;
              if (j >= mine) continue;
              if (!(ok = ctl.wait(&s.p_ready[x], pp[x]))) break;
              pp[x] ^= 1;
              fence_after();
#pragma unroll
              for (int e = 0; e < kC / 16; ++e)
                mma_tmem(tm + 256 + x * kC, tm + x * kC + e * 8, v + e * 128, id_o, j + e > 0);
              if (x == 1 || !it.n_b) commit(&s.empty[iv]);
              if (j + 1 < mine) {
                scores(tm + x * kC, q[x], k, id_s, p.dk);
                commit(&s.s_full[x]);
              } else {
                commit(&s.o_done[x]);
              }
              if (more && (x == 1 || !it.n_b)) {
                commit(&s.empty[ik]);
                if (j + 2 == n) commit(&s.q_empty);  // these were the last scores
              }
            }
          }
        }
      }
      commit(&s.c.drain);  // nothing of this CTA's is in flight after it
      ctl.land(&s.c.drain, 0);
    }
  }
  close_tmem(tm, kFwdSoftmax + 1);
}

// ---------------------------------------------------------------------------
// gradients of the queries
// ---------------------------------------------------------------------------

// A tile of keys is held until dq's product, one of values only until dP's.  In
// one ring of five the values' next slot came free with the keys before last,
// a thousand cycles too late for every tile.
constexpr int kKeySlots = 3, kValueSlots = 2;

struct DqTail {
  Common c;
  uint64_t q_full, k_full[kKeySlots], k_empty[kKeySlots], v_full[kValueSlots], v_empty[kValueSlots];
  uint64_t dp_full, dp_free, ds_ready, o_done, mean_ready, sums_ready;
  alignas(16) float mean[2][kC];  // halves of the sum of the sequence's first keys
  float sums[2][kC];  // of a row's dS as rounded, by half of the columns
};

// A row's dS add up to nothing, so its dq does not depend on what all keys have
// in common; rounded dS do not, quite.  With c near the keys' mean (of the
// sequence's first block),
//
//   dq = scale (sum_j dS[j] k[j] - (sum_j dS[j]) c)
//
// is the same without roundings, and with them what the keys share stays out of
// their error: where it was half of the keys' spread, dq's distance from 64 bits
// was 1.53 times that of one rounding, and two independent ones make 1.41.
template <typename T>
__global__ void __launch_bounds__(kTcThreads, 1) tc_dq_kernel(const __grid_constant__ Problem p, const __grid_constant__ Maps maps) {
  extern __shared__ __align__(1024) unsigned char smem[];
  const int h = blockIdx.y, hk = h / p.share, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Tile t = find_tile_warp<7>(p, gridDim.x - 1 - blockIdx.x);
  if (t.first < 0) zero_outside<T>(p, p.d_q, h, p.H, p.dk, blockIdx.x, kC, tid, kTcThreads);
  if (t.first < 0 || misplaced(smem, p.err)) return;
  const int q_bytes = tile_bytes(p.dk), g_bytes = tile_bytes(p.dv);
  unsigned char *k_ring = smem + q_bytes + g_bytes, *v_ring = k_ring + kKeySlots * q_bytes;
  DqTail& s = *reinterpret_cast<DqTail*>(v_ring + kValueSlots * g_bytes);
  const Ctl ctl{&s.c, p.err};
  const int n = t.first / kC + 1, len = min(kC, t.len - t.first);
  const long long at = t.start + t.first;
  if (tid == 8 * 32) {  // the loading warp's, which need not wait for the others
    bar_init(&s.q_full, 1);
    for (int i = 0; i < kKeySlots; ++i) bar_init(&s.k_full[i], 1), bar_init(&s.k_empty[i], 1);
    for (int i = 0; i < kValueSlots; ++i) bar_init(&s.v_full[i], 1), bar_init(&s.v_empty[i], 1);
    bar_init(&s.dp_full, 1);
    bar_init(&s.dp_free, 8);
    bar_init(&s.ds_ready, 8);
    bar_init(&s.o_done, 1);
    bar_init(&s.mean_ready, 2);
    bar_init(&s.sums_ready, 8);
    bar_init(&s.c.drain, 1);
    s.c.abort = 0;
    bars_done();
    bar_expect(&s.q_full, q_bytes + g_bytes);
    load_tile(smem, &maps.q, p.dk, h, at, &s.q_full);
    load_tile(smem + q_bytes, &maps.d_out, p.dv, h, at, &s.q_full);
  }
  const uint32_t tm = open_tmem(&s.c);
  constexpr uint32_t kDp = 256, kDq = 384;  // two places of S, then dP and dQ

  if (warp < 8) {
    const int side = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad) << 21;
    const float lse = row < len ? p.lse[h * p.BL + at + row] : 0.f, d = row < len ? p.d[h * p.BL + at + row] : 0.f;
    const float c2 = p.scale * kLog2e;
    const float unit = ds_unit<T>(p), per = 1.f / unit;
    const uint64_t c22 = pair(c2, c2), lse2 = pair(-lse, -lse), d2 = pair(-d * per, -d * per), per2 = pair(per, per);
    uint64_t sum[2] = {0, 0};
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!(ok = ctl.warp_wait(&s.dp_full, j & 1))) break;  // S was issued before dP
      fence_after();
      const uint32_t ts = tm + lanes + (j & 1) * kC + 64 * side;
      uint32_t sc[64], g[64];
      tmem_ld32(tm + lanes + kDp + 64 * side, g);
      tmem_ld32(tm + lanes + kDp + 64 * side + 32, g + 32);
      tmem_ld32(ts, sc);
      tmem_ld32(ts + 32, sc + 32);
      wait_ld();
      fence_before();
      warp_arrive(&s.dp_free);
      const bool diagonal = j == n - 1;
      uint32_t w[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const uint64_t z = fma2(pair_of(sc + 2 * e), c22, lse2), y = (e & 7) >= 8 - kPoly ? poly_ex2_2(z) : ex2_2(z);
        w[e] = pack2<T>(mul2(y, f16<T>() ? fma2(pair_of(g + 2 * e), per2, d2) : add2(pair_of(g + 2 * e), d2)));
      }
      if (diagonal) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int c = 64 * side + 2 * e;
          w[e] &= (c <= row ? 0xffffu : 0u) | (c + 1 <= row ? 0xffff0000u : 0u);
        }
        if (side == 0 && t.first + row == 0) w[0] = only_key<T>(w[0]);
        // keys of the rows behind the mask, and of other sequences
        if (64 * side < p.dk) clean_row<T>(k_ring + j % kKeySlots * q_bytes, row, side, 1, row < len);
        fence_async();
      }
      tmem_st32(ts, w);
      wait_st();
      fence_before();
      warp_arrive(&s.ds_ready);
#pragma unroll
      for (int e = 0; e < 32; ++e) sum[e & 1] = add2(sum[e & 1], unpack2<T>(w[e]));
    }
    const float2 both = unpair(add2(sum[0], sum[1]));
    s.sums[side][row] = both.x + both.y;
    warp_arrive(&s.sums_ready);
    if (ok && 64 * side < p.dk && ctl.warp_wait(&s.sums_ready, 0) && ctl.warp_wait(&s.mean_ready, 0) && ctl.warp_wait(&s.o_done, 0)) {
      fence_after();
      const float f = -p.scale * unit * (s.sums[0][row] + s.sums[1][row]) / static_cast<float>(min(kC, t.len));
      const uint64_t f2 = pair(f, f), scale2 = pair(p.scale * unit, p.scale * unit);
      uint32_t w[32];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t x[32];
        tmem_ld32(tm + lanes + kDq + 64 * side + 32 * half, x);
        wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 a = *reinterpret_cast<const float2*>(&s.mean[0][64 * side + 32 * half + 2 * e]);
          const float2 b = *reinterpret_cast<const float2*>(&s.mean[1][64 * side + 32 * half + 2 * e]);
          w[16 * half + e] = pack2<T>(fma2(add2(pair(a.x, a.y), pair(b.x, b.y)), f2, mul2(pair_of(x + 2 * e), scale2)));
        }
      }
      store_block(smem + side * kBlock + quad * 4096, w,
                  static_cast<unsigned char*>(p.d_q) + ((at + quad * 32) * p.H + h) * p.dk * 2 + side * 128,
                  static_cast<long long>(p.H) * p.dk * 2, len - quad * 32, p.dk - 64 * side);
    }
  } else if (warp == 8) {
    if (lane == 0) {
      Cursor k, v;
      int loads = 0;  // tiles of both
      for (; loads < n; ++loads) {
        // a first pass finds all slots empty
        if (!ctl.wait(&s.k_empty[k.at], k.turn ^ 1)) break;
        bar_expect(&s.k_full[k.at], q_bytes);
        load_tile(k_ring + k.at * q_bytes, &maps.k, p.dk, hk, t.start + loads * kC, &s.k_full[k.at]);
        if (!ctl.wait(&s.v_empty[v.at], v.turn ^ 1)) {
          ctl.land(&s.k_full[k.at], k.turn);
          break;
        }
        bar_expect(&s.v_full[v.at], g_bytes);
        load_tile(v_ring + v.at * g_bytes, &maps.v, p.dv, hk, t.start + loads * kC, &s.v_full[v.at]);
        k.next(kKeySlots);
        v.next(kValueSlots);
      }
      if (loads < n) {
        ctl.land(&s.q_full, 0);
        for (int e = max(0, loads - kKeySlots); e < loads; ++e) ctl.land(&s.k_full[e % kKeySlots], (e / kKeySlots) & 1);
        for (int e = max(0, loads - kValueSlots); e < loads; ++e) ctl.land(&s.v_full[e % kValueSlots], (e / kValueSlots) & 1);
      }
    }
  } else if (warp == 9) {
    if (elect_one()) {  // one thread, without votes
      const uint32_t id_s = idesc(kC, false, f16<T>()), id_o = idesc((p.dk + 15) / 16 * 16, true, f16<T>());
      const uint64_t q = desc(smem_u32(smem), 16), g = desc(smem_u32(smem) + q_bytes, 16);
      const uint64_t k0 = desc(smem_u32(k_ring), 16), o0 = desc(smem_u32(k_ring), kBlock), v0 = desc(smem_u32(v_ring), 16);
      Cursor kc, vc;
      int held[2] = {0, 0};  // slots of the keys that a product still has to come for
      bool ok = ctl.wait(&s.q_full, 0);
      for (int j = -1; ok && j < n; ++j) {
        if (j + 1 < n) {  // the next tile's scores, while the warps are at this one's
          if (!(ok = ctl.wait(&s.k_full[kc.at], kc.turn))) break;
          scores(tm + ((j + 1) & 1) * kC, q, k0 + kc.at * (q_bytes >> 4), id_s, p.dk);
          held[(j + 1) & 1] = kc.at;
          kc.next(kKeySlots);
          if (!(ok = ctl.wait(&s.v_full[vc.at], vc.turn) && (j < 0 || ctl.wait(&s.dp_free, j & 1)))) break;
          fence_after();
          scores(tm + kDp, g, v0 + vc.at * (g_bytes >> 4), id_s, p.dv);
          commit(&s.dp_full);
          commit(&s.v_empty[vc.at]);
          vc.next(kValueSlots);
        }
        if (j < 0) continue;
        if (!(ok = ctl.wait(&s.ds_ready, j & 1))) break;
        fence_after();
        const int at_k = held[j & 1];
        // the warps' halves of dS lie 64 columns apart
#pragma unroll
        for (int k = 0; k < kC / 16; ++k)
          mma_tmem(tm + kDq, tm + (j & 1) * kC + (k >> 2) * 64 + (k & 3) * 8, o0 + at_k * (q_bytes >> 4) + k * 128, id_o, j + k > 0);
        commit(&s.k_empty[at_k]);
        if (j == n - 1) commit(&s.o_done);
      }
      commit(&s.c.drain);
      ctl.land(&s.c.drain, 0);
    }
  } else {
    // sums over the first keys, without what is not finite, four elements a lane
    const int half = warp - 10, rows = min(kC, t.len);
    const T* k = static_cast<const T*>(p.k.p) + static_cast<long long>(t.start) * p.k.st + hk * p.k.sh + 4 * lane;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (4 * lane < p.dk) {
#pragma unroll 8
      for (int i = half; i < rows; i += 2) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(k + i * p.k.st));
        const float2 a = unpair(unpack2<T>(w.x)), b = unpair(unpack2<T>(w.y));
        const float v[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += fabsf(v[e]) < INFINITY ? v[e] : 0.f;
      }
    }
    *reinterpret_cast<float4*>(&s.mean[half][4 * lane]) = make_float4(x[0], x[1], x[2], x[3]);
    warp_arrive(&s.mean_ready);
    if (half == 0) zero_outside<T>(p, p.d_q, h, p.H, p.dk, blockIdx.x, kC, lane, 32);
  }
  close_tmem(tm);
}

// ---------------------------------------------------------------------------
// gradients of the keys and values
// ---------------------------------------------------------------------------

// Queries are held from their scores to dK's product, the last one of a tile.
constexpr int kQuerySlots = 3;

struct DkvTail {
  Common c;
  uint64_t kv_full, q_full[kQuerySlots], q_empty[kQuerySlots], g_full[2], g_empty[2], stat_full[2], stat_empty[2];
  uint64_t s_full, p_ready, dp_full, ds_ready, o_done;
  alignas(16) float lse[2][kC], d[2][kC];  // negated, of the queries that pass
  int bad;                     // 1 + the last query of the diagonal's tile whose dO is not finite
};

template <typename T>
__global__ void __launch_bounds__(kTcThreads, 1) tc_dkdv_kernel(const __grid_constant__ Problem p, const __grid_constant__ Maps maps) {
  extern __shared__ __align__(1024) unsigned char smem[];
  const int hk = blockIdx.y, heads = p.H / p.share, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Tile t = find_tile_warp<7>(p, blockIdx.x);  // a sequence's first keys have the most queries
  if (t.first < 0) {
    zero_outside<T>(p, p.d_k, hk, heads, p.dk, blockIdx.x, kC, tid, kTcThreads);
    zero_outside<T>(p, p.d_v, hk, heads, p.dv, blockIdx.x, kC, tid, kTcThreads);
  }
  if (t.first < 0 || misplaced(smem, p.err)) return;
  const int k_bytes = tile_bytes(p.dk), v_bytes = tile_bytes(p.dv);
  unsigned char *q_ring = smem + k_bytes + v_bytes, *g_ring = q_ring + kQuerySlots * k_bytes;
  DkvTail& s = *reinterpret_cast<DkvTail*>(g_ring + 2 * v_bytes);
  const Ctl ctl{&s.c, p.err};
  const int blocks = (t.len - t.first + kC - 1) / kC, len = min(kC, t.len - t.first);
  const int total = blocks * p.share;  // tiles of queries, head by head
  const long long at = t.start + t.first;
  if (tid == 8 * 32) {  // the loading warp's, which need not wait for the others
    bar_init(&s.kv_full, 1);
    for (int i = 0; i < kQuerySlots; ++i) bar_init(&s.q_full[i], 1), bar_init(&s.q_empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(&s.g_full[i], 1);
      bar_init(&s.g_empty[i], 1);
      bar_init(&s.stat_full[i], 1);
      bar_init(&s.stat_empty[i], 8);
    }
    bar_init(&s.s_full, 1);
    bar_init(&s.p_ready, 8);
    bar_init(&s.dp_full, 1);
    bar_init(&s.ds_ready, 8);
    bar_init(&s.o_done, 1);
    bar_init(&s.c.drain, 1);
    s.c.abort = 0;
    s.bad = 0;
    bars_done();
    bar_expect(&s.kv_full, k_bytes + v_bytes);
    load_tile(smem, &maps.k, p.dk, hk, at, &s.kv_full);
    load_tile(smem + k_bytes, &maps.v, p.dv, hk, at, &s.kv_full);
  }
  const uint32_t tm = open_tmem(&s.c);
  constexpr uint32_t kDp = 128, kDv = 256, kDk = 384;

  if (warp < 8) {
    const int side = warp >> 2, quad = warp & 3, row = quad * 32 + lane;  // of the keys; columns are queries
    const uint32_t lanes = static_cast<uint32_t>(quad) << 21, ts = tm + lanes + 64 * side, td = tm + lanes + kDp + 64 * side;
    const float c2 = p.scale * kLog2e, unit = ds_unit<T>(p), per = exp2f(-p_bits<T>()) / unit;
    const uint64_t c22 = pair(c2, c2), per2 = pair(per, per);
    bool ok = true;
    for (int i = 0, b = 0; i < total; ++i, b = b + 1 < blocks ? b + 1 : 0) {
      const int u = i & 1;
      const bool diagonal = b == 0;
      const int n = min(kC, t.len - t.first - b * kC);
      const bool edge = diagonal || n < kC;
      if (!(ok = ctl.warp_wait(&s.stat_full[u], (i >> 1) & 1) && ctl.warp_wait(&s.s_full, i & 1))) break;
      fence_after();
      uint64_t x[32];
      uint32_t w[32];
      {
        uint32_t sc[64];
        tmem_ld32(ts, sc);
        tmem_ld32(ts + 32, sc + 32);
        wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float4 l = *reinterpret_cast<const float4*>(&s.lse[u][64 * side + 2 * e]);
          const uint64_t z0 = fma2(pair_of(sc + 2 * e), c22, pair(l.x, l.y)), z1 = fma2(pair_of(sc + 2 * e + 2), c22, pair(l.z, l.w));
          x[e] = (e & 7) >= 8 - kPoly ? poly_ex2_2(z0) : ex2_2(z0);
          x[e + 1] = (e & 7) + 1 >= 8 - kPoly ? poly_ex2_2(z1) : ex2_2(z1);
        }
      }
      if (edge) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float2 f = unpair(x[e]);
          const int c = 64 * side + 2 * e;
          if ((diagonal && c < row) || c >= n) f.x = 0.f;
          if ((diagonal && c + 1 < row) || c + 1 >= n) f.y = 0.f;
          x[e] = pair(f.x, f.y);
        }
      }
#pragma unroll
      for (int e = 0; e < 32; ++e) w[e] = pack2<T>(x[e]);
      tmem_st32(ts, w);
      if (edge) {
        // queries and upstream gradients of rows behind the mask, and of other
        // sequences, once both score products have read them
        if (!(ok = ctl.warp_wait(&s.dp_full, i & 1))) break;
        if (64 * side < p.dk) clean_row<T>(q_ring + i % kQuerySlots * k_bytes, row, side, 1, row < n);
        if (64 * side < p.dv && clean_row<T>(g_ring + u * v_bytes, row, side, 1, row < n) && diagonal) atomicMax(&s.bad, row + 1);
        fence_async();
      }
      wait_st();
      fence_before();
      warp_arrive(&s.p_ready);
      if (!(ok = ctl.warp_wait(&s.dp_full, i & 1))) break;
      fence_after();
      {
        uint32_t g[64];
        tmem_ld32(td, g);
        tmem_ld32(td + 32, g + 32);
        wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float4 d = *reinterpret_cast<const float4*>(&s.d[u][64 * side + 2 * e]);
          uint64_t y0 = add2(pair_of(g + 2 * e), pair(d.x, d.y)), y1 = add2(pair_of(g + 2 * e + 2), pair(d.z, d.w));
          if (f16<T>()) y0 = mul2(y0, per2), y1 = mul2(y1, per2);
          w[e] = pack2<T>(mul2(x[e], y0));
          w[e + 1] = pack2<T>(mul2(x[e + 1], y1));
        }
      }
      if (edge) {  // 0 * NaN again
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int c = 64 * side + 2 * e;
          w[e] &= ((diagonal && c < row) || c >= n ? 0u : 0xffffu) | ((diagonal && c + 1 < row) || c + 1 >= n ? 0u : 0xffff0000u);
        }
        if (diagonal && side == 0 && t.first + row == 0) w[0] = (w[0] & 0xffff0000u) | only_key<T>(w[0]);
      }
      tmem_st32(td, w);
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) {
        bar_arrive(&s.ds_ready);
        bar_arrive(&s.stat_empty[u]);
      }
    }
    if (ok && ctl.warp_wait(&s.o_done, 0)) {
      fence_after();
      // behind the last product, whose inputs were ready after every clean_row
      const bool bad = row < *reinterpret_cast<volatile int*>(&s.bad);
      unsigned char* stage = smem + warp * 4096;
      uint32_t w[32];
      if (64 * side < p.dv) {
        fetch_block<T>(tm + lanes + kDv + 64 * side, bad ? NAN : exp2f(-p_bits<T>()), w);
        store_block(stage, w, static_cast<unsigned char*>(p.d_v) + ((at + quad * 32) * heads + hk) * p.dv * 2 + side * 128,
                    static_cast<long long>(heads) * p.dv * 2, len - quad * 32, p.dv - 64 * side);
      }
      if (64 * side < p.dk) {
        fetch_block<T>(tm + lanes + kDk + 64 * side, p.scale * unit, w);
        store_block(stage, w, static_cast<unsigned char*>(p.d_k) + ((at + quad * 32) * heads + hk) * p.dk * 2 + side * 128,
                    static_cast<long long>(heads) * p.dk * 2, len - quad * 32, p.dk - 64 * side);
      }
    }
  } else if (warp == 8) {
    if (lane == 0) {
      int q_loads = 0, g_loads = 0;
      Cursor q, g;
      for (int i = 0, b = 0, h = hk * p.share; i < total; ++i) {
        const int token = static_cast<int>(at) + b * kC;
        // a first pass finds all slots empty
        if (!ctl.wait(&s.q_empty[q.at], q.turn ^ 1)) break;
        bar_expect(&s.q_full[q.at], k_bytes);
        load_tile(q_ring + q.at * k_bytes, &maps.q, p.dk, h, token, &s.q_full[q.at]);
        q.next(kQuerySlots);
        ++q_loads;
        if (!ctl.wait(&s.g_empty[g.at], g.turn ^ 1)) break;
        bar_expect(&s.g_full[g.at], v_bytes);
        load_tile(g_ring + g.at * v_bytes, &maps.d_out, p.dv, h, token, &s.g_full[g.at]);
        g.next(2);
        ++g_loads;
        if (++b == blocks) b = 0, ++h;
      }
      if (g_loads < total) {
        ctl.land(&s.kv_full, 0);
        for (int i = max(0, q_loads - kQuerySlots); i < q_loads; ++i) ctl.land(&s.q_full[i % kQuerySlots], (i / kQuerySlots) & 1);
        for (int i = max(0, g_loads - 2); i < g_loads; ++i) ctl.land(&s.g_full[i & 1], (i >> 1) & 1);
      }
    }
  } else if (warp == 9) {
    if (elect_one()) {  // one thread, without votes
      const uint32_t id_s = idesc(kC, false, f16<T>()), id_k = idesc((p.dk + 15) / 16 * 16, true, f16<T>()),
                     id_v = idesc((p.dv + 15) / 16 * 16, true, f16<T>());
      const uint64_t k = desc(smem_u32(smem), 16), v = desc(smem_u32(smem) + k_bytes, 16);
      const uint64_t q0 = desc(smem_u32(q_ring), 16), g0 = desc(smem_u32(g_ring), 16);          // for scores
      const uint64_t q1 = desc(smem_u32(q_ring), kBlock), g1 = desc(smem_u32(g_ring), kBlock);  // as values
      Cursor c, held;  // queries: the next tile's scores, and its product with dS
      bool ok = ctl.wait(&s.kv_full, 0);
      for (int i = -1; ok && i < total; ++i) {
        const bool more = i + 1 < total;
        const int u = i & 1, nu = (i + 1) & 1;
        if (i >= 0) {
          if (!(ok = ctl.wait(&s.p_ready, i & 1))) break;
          fence_after();
          // the warps' halves of P lie 64 columns apart
#pragma unroll
          for (int e = 0; e < kC / 16; ++e)
            mma_tmem(tm + kDv, tm + (e >> 2) * 64 + (e & 3) * 8, g1 + u * (v_bytes >> 4) + e * 128, id_v, i + e > 0);
          commit(&s.g_empty[u]);
        }
        if (more) {  // in P's place, which that product has read
          if (!(ok = ctl.wait(&s.q_full[c.at], c.turn))) break;
          scores(tm, k, q0 + c.at * (k_bytes >> 4), id_s, p.dk);
          commit(&s.s_full);
          c.next(kQuerySlots);
        }
        if (i >= 0) {
          if (!(ok = ctl.wait(&s.ds_ready, i & 1))) break;
          fence_after();
#pragma unroll
          for (int e = 0; e < kC / 16; ++e)
            mma_tmem(tm + kDk, tm + kDp + (e >> 2) * 64 + (e & 3) * 8, q1 + held.at * (k_bytes >> 4) + e * 128, id_k, i + e > 0);
          commit(&s.q_empty[held.at]);
          held.next(kQuerySlots);
          if (!more) commit(&s.o_done);
        }
        if (more) {
          if (!(ok = ctl.wait(&s.g_full[nu], ((i + 1) >> 1) & 1))) break;
          scores(tm + kDp, v, g0 + nu * (v_bytes >> 4), id_s, p.dv);
          commit(&s.dp_full);
        }
      }
      commit(&s.c.drain);
      ctl.land(&s.c.drain, 0);
    }
  } else if (warp == 10) {
    for (int i = 0, b = 0, h = hk * p.share; i < total; ++i) {
      const int u = i & 1;
      const long long token = at + static_cast<long long>(b) * kC, n = t.len - t.first - static_cast<long long>(b) * kC;
      float l[4], d[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = e * 32 + lane;
        l[e] = c < n ? p_bits<T>() - p.lse[h * p.BL + token + c] : 0.f;
        d[e] = c < n ? -p.d[h * p.BL + token + c] : 0.f;
      }
      if (i > 1 && !ctl.warp_wait(&s.stat_empty[u], (i / 2 - 1) & 1)) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) s.lse[u][e * 32 + lane] = l[e], s.d[u][e * 32 + lane] = d[e];
      warp_arrive(&s.stat_full[u]);
      if (++b == blocks) b = 0, ++h;
    }
  } else {
    zero_outside<T>(p, p.d_k, hk, heads, p.dk, blockIdx.x, kC, lane, 32);
    zero_outside<T>(p, p.d_v, hk, heads, p.dv, blockIdx.x, kC, lane, 32);
  }
  close_tmem(tm);
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

static bool map_rows(CUtensorMap* m, const Rows& r, int dim, int heads, long long BL, int dtype) {
  const auto fn = encode_fn();
  if (!fn) return false;
  const long long sh = heads > 1 ? r.sh : dim;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(BL)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(r.st) * 2};
  const cuuint32_t box[3] = {64, 1, kC}, one[3] = {1, 1, 1};
  return fn(m, dtype == ASCAN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void*>(r.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows that a tensor map can describe: 16-byte bases and strides, head sizes in
// whole 16-byte pieces, heads that do not overlap.
static bool rows_usable(const Rows& r, int dim, int heads) {
  if ((reinterpret_cast<uintptr_t>(r.p) & 15u) || dim % 8 || r.st % 8 || r.st < dim || r.st >= (1ll << 38)) return false;
  return heads == 1 || (r.sh % 8 == 0 && r.sh >= dim && r.sh < (1ll << 38));
}
static bool aligned(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; }

bool tc_usable(const Problem& p, int dtype, bool backward) {
  if (dtype == ASCAN_F32 || tile_bound(p, 2 * kC) * p.H > 0x7fffffffll) return false;
  const int heads = p.H / p.share;
  if (!rows_usable(p.q, p.dk, p.H) || !rows_usable(p.k, p.dk, heads) || !rows_usable(p.v, p.dv, heads)) return false;
  if (!aligned(p.out) || !aligned(p.rest)) return false;
  if (backward && (!rows_usable(p.d_out, p.dv, p.H) || !aligned(p.d_q) || !aligned(p.d_k) || !aligned(p.d_v))) return false;
  return encode_fn() != nullptr;
}

// Tensor maps are made through the driver, which wants a current context; a
// thread whose first CUDA call this is has none until the runtime is told its
// device.
static int make_maps(Maps& m, const Problem& p, int dtype, bool backward) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return ASCAN_EDEVICE;
  memset(&m, 0, sizeof(m));
  const int heads = p.H / p.share;
  if (!map_rows(&m.q, p.q, p.dk, p.H, p.BL, dtype) || !map_rows(&m.k, p.k, p.dk, heads, p.BL, dtype) ||
      !map_rows(&m.v, p.v, p.dv, heads, p.BL, dtype) || (backward && !map_rows(&m.d_out, p.d_out, p.dv, p.H, p.BL, dtype)))
    return ASCAN_ECUDA;
  return ASCAN_OK;
}

static int bytes_of(int dim) { return dim > 64 ? 2 * kBlock : kBlock; }

template <typename T, bool TRAIN>
static int forward(const Problem& p, const Maps& m, cudaStream_t s) {
  static std::atomic<unsigned long long> done{};
  const int rc = allow_smem(tc_forward_kernel<T, TRAIN>, kSmemLimit, done);
  if (rc != ASCAN_OK) return rc;
  const size_t smem = 2 * bytes_of(p.dk) + forward_slots(p.dk, p.dv) * slot_bytes(p.dk, p.dv) + kFwdSoftmax * kStage + sizeof(ForwardTail);
  tc_forward_kernel<T, TRAIN><<<static_cast<unsigned>(tile_bound(p, 2 * kC) * p.H), kFwdThreads, smem, s>>>(p, m);
  return launch_status();
}

template <typename T>
static int backward(const Problem& p, const Maps& m, cudaStream_t s) {
  static std::atomic<unsigned long long> done[2]{};
  int rc = allow_smem(tc_dq_kernel<T>, kSmemLimit, done[0]);
  if (rc == ASCAN_OK) rc = allow_smem(tc_dkdv_kernel<T>, kSmemLimit, done[1]);
  if (rc != ASCAN_OK) return rc;
  const size_t k = bytes_of(p.dk), v = bytes_of(p.dv);
  // one CTA an SM in any case: each takes all of tensor memory
  const size_t q_smem = max(k + v + kKeySlots * k + kValueSlots * v + sizeof(DqTail), static_cast<size_t>(120 << 10));
  const size_t kv_smem = max(k + v + kQuerySlots * k + 2 * v + sizeof(DkvTail), static_cast<size_t>(120 << 10));
  tc_dq_kernel<T><<<dim3(tile_bound(p, kC), p.H), kTcThreads, q_smem, s>>>(p, m);
  rc = launch_status();
  if (rc != ASCAN_OK) return rc;
  tc_dkdv_kernel<T><<<dim3(tile_bound(p, kC), p.H / p.share), kTcThreads, kv_smem, s>>>(p, m);
  return launch_status();
}
static_assert(14 * kBlock + sizeof(DkvTail) <= kSmemLimit &&
              14 * kBlock + sizeof(ForwardTail) <= kSmemLimit && 14 * kBlock + sizeof(DqTail) <= kSmemLimit,
              "heads of 128 leave no more for the barriers and statistics");

int tc_forward(const Problem& p, int dtype, cudaStream_t s) {
  Maps m;
  const int rc = make_maps(m, p, dtype, false);
  if (rc != ASCAN_OK) return rc;
  if (p.lse && p.rest) return dtype == ASCAN_BF16 ? forward<__nv_bfloat16, true>(p, m, s) : forward<__half, true>(p, m, s);
  return dtype == ASCAN_BF16 ? forward<__nv_bfloat16, false>(p, m, s) : forward<__half, false>(p, m, s);
}

int tc_backward(const Problem& p, int dtype, cudaStream_t s) {
  Maps m;
  const int rc = make_maps(m, p, dtype, true);
  if (rc != ASCAN_OK) return rc;
  return dtype == ASCAN_BF16 ? backward<__nv_bfloat16>(p, m, s) : backward<__half>(p, m, s);
}

}  // namespace attend

ASCAN_UNIT_ERROR_ACCESSORS(attend_tc)

}  // namespace ascan
