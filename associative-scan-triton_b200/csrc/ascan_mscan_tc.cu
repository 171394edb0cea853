// ascan_mscan_tc.cu -- compilation unit of the scan library: the matrix-state
// recurrence on the fifth-generation tensor cores (bfloat16).
//
// One CTA per (segment, head, form) walks its chunks of 128 tokens.  Per chunk
//
//   scores = A B^T            A, B from shared memory            [128, 128]
//   O      = A S              S the state entering the chunk     [128, dc]
//   U     += (col . B)^T C    what the chunk adds to the state   [da, dc]
//   O      = row . O + P C    P = masked, decayed scores
//
// with float32 accumulators in tensor memory.  What is computed on the way to
// an operand would lose digits as one bfloat16: col.B, P and S are each split
// into two (16 bits together), so that a result keeps its own rounding only,
// 2^-16 of its size before it; and col.B into three (24 bits) where a float32
// result depends on the state.  A and C come as stored, so they are exact.
//
// Roles, by warp (one CTA per SM; every hand-over is an mbarrier):
//   0-7    row warps, two for each 32 tokens: scores -> P in place in tensor
//          memory, scale O by the row factors, store the finished rows (each
//          takes one half of the columns; P is the longest part of a chunk)
//   8-11   state warps: the decayed operand S and U make the next operand S
//          in shared memory and, of what its first term leaves over, the next U
//   12-15  column warps: (col . B)^T transposed into tensor memory; tails and
//          values that are not finite in C
//   16     TMA loads of the A, B, C tiles into shared-memory slots
//   17     issues the products
//   18     the chunk's gate sums, row and column factors
//
// Tensor memory (512 columns of 128 lanes): scores/P 128, O 128, U 128,
// (col.B)^T 128: two terms of all tokens, or three of half of them at a time.
// Lanes are tokens for scores and O, state rows for U.
//
// A token whose value is not finite would reach earlier rows of its chunk
// through 0 * NaN; the column warps replace such values by zero and note the
// first token of each column, and the row and state warps put NaN where the
// mask lets the value through.
//
// What bounds it: the instructions of its roles.  At 16384 tokens of 12 heads
// of 128 x 128 the forward reads what it must (161 MB) at 27% of the memory
// rate with the tensor pipe 29% busy; a scheduler issues 0.45 instructions a
// cycle, and its warps wait for other roles, fixed latencies and instructions.
// Hence one body per form, loop bodies of sixteen columns, and rare work out
// of line (a hundred instructions more in the state warps' loop made the rows
// a sixth slower).  65536 tokens: 237 us for the rows (3.4 TB/s of operands
// and results) after 111 us of carries, at four products of which the causal
// half of two is wasted.
//
// Every wait is bounded: one that runs out sets the device error word and an
// abort flag, every role then leaves its loop, loads and products in flight
// are waited for, and tensor memory is freed.
#include "ascan_impl.cuh"
#include "ascan_mscan.cuh"
#include "ascan_mscan_common.cuh"
#include "ascan_pairs.cuh"

namespace ascan {
namespace mscan {

constexpr int kC = 128;             // tokens of a chunk
constexpr int kTcWarps = 19;
constexpr int kTcThreads = kTcWarps * 32;
constexpr uint32_t kColSc = 0, kColO = 128, kColU = 256, kColK = 384;
constexpr unsigned long long kStageTimeoutNs = 2000000000ull;
constexpr size_t kSmemLimit = 232448;

struct TcMaps {
  CUtensorMap m[3][5];  // per form: A, B, C, the rows to take dots with, the output
};

// Shared memory after the tile slots and the S operand.
struct TcTail {
  // Negated gate sums in units of log 2, up to and with the token (backwards:
  // of all after it), two tokens an entry: floats of both, then what the
  // floats leave over
  float4 lg[kC / 2];
  // col[s]: the decay between token s and the edge of its 32 tokens (their
  // last, or backwards the token before their first); far[b]: from there to
  // the end (start) of the chunk.  The column factor is the product of both.
  float col[kC];
  float far[4];
  // per value column, the chunk's first token that is not finite: chunk number
  // + 1 in the high bits, and below them its rank from the far end, so that
  // a maximum finds it and nothing has to be cleared
  uint32_t bad[2][kC];
  uint64_t full[6], empty[6];  // slots of A: 0, 1; of C: 2, 3; of B: 4 and, if there is room, 5
  uint64_t tab_full, tab_empty, sc_full, in_full, p_ready, kt_ready[4], kt_free[2], u_full[2], s_ready, o_full, o_free, d_full, drain;
  uint64_t added[2];     // without rows: the chunk's accumulator has been added to the sum
  uint64_t own_read[4];  // by 32 tokens: the second row warp has its rows' own scores
  float total;
  int bad_chunk[2];  // chunk number + 1 when bad[] holds something
  int abort;
  uint32_t tmem;
};

// A slot waits for its rows to leave the chip and C's for the last product, so
// both are double; B is done with early, and a second slot of it is a bonus.
struct TcGeom {
  int slot_bytes, s_bytes;  // bytes of a slot and of one term of S
  int b_slots;
  __host__ __device__ int bytes() const { return (4 + b_slots) * slot_bytes + 2 * s_bytes; }
};

__host__ __device__ inline TcGeom tc_geom(int da, int dc) {
  TcGeom g;
  g.slot_bytes = (da > 64 || dc > 64) ? 32768 : 16384;
  g.s_bytes = (da > 64 ? 128 : 64) * 128 * (dc > 64 ? 2 : 1);
  g.b_slots = 2;
  if (g.bytes() + sizeof(TcTail) > kSmemLimit) g.b_slots = 1;
  return g;
}

// ---- instructions ----------------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// 128 tokens by 64 elements of one head, from column x (a multiple of 64).
__device__ __forceinline__ void tma_rows(uint32_t to, const CUtensorMap* m, int x, int head, int token, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to),
      "l"(m), "r"(x), "r"(head), "r"(token), "r"(smem_u32(bar))
      : "memory");
}
// One lane of the warp, by the instruction that the compiler knows to pick
// one: behind it operands stay in uniform registers, and a product takes 50
// cycles to issue instead of 90 (it runs for 64).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc))
      : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc))
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define TC_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define TC_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])

// 32 columns of the warp's 32 lanes; volatile, and the wait follows before use.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : TC_R8(r, 0), TC_R8(r, 8), TC_R8(r, 16), TC_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : TC_R8(r, 0), TC_R8(r, 8)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : TC_R8(r, 0) : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), TC_I8(r, 0)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      TC_I8(r, 0), TC_I8(r, 8)
      : "memory");
}

// 16 lanes by 8 columns; a pair of registers holds 4 columns: lane l of the
// warp has column l % 4 of row l / 4, then of row l / 4 + 8.
__device__ __forceinline__ void tmem_st16x128(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two floats to packed bfloat16 (a low, b high)
__device__ __forceinline__ uint32_t bf2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// The n lowest of 32 bits (none below 0, all above 31).
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); }

// The pair as packed bfloat16, and what that leaves over as another.
__device__ __forceinline__ uint32_t round2(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  return bf2(a, b);
}
__device__ __forceinline__ uint64_t left2(uint64_t x, uint32_t hi) {
  return fma2(pair(lo_f(hi), hi_f(hi)), pair(-1.f, -1.f), x);
}
__device__ __forceinline__ uint32_t rest2(uint64_t x, uint32_t hi) { return round2(left2(x, hi)); }

// x = total * hi + v, eight columns.
__device__ __forceinline__ void add_state(const uint4& hi, uint64_t total2, const float* v, uint64_t* x) {
  const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = fma2(total2, pair(lo_f(h[e]), hi_f(h[e])), pair(v[2 * e], v[2 * e + 1]));
}

// Shared-memory operand descriptors, 128-byte swizzle.  Along the unit-stride
// side a row is 64 elements; `lbo` is the distance of the next 64 (used when
// that side is not the products' inner one), rows of 8 are 1024 bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// float32 accumulators, bfloat16 operands, M = 128; b_mn: B's unit stride is
// along N.
__device__ __forceinline__ uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

// Element i of N (a power of two), without indexing registers.
template <int N>
__device__ __forceinline__ uint32_t pick(const uint32_t* x, int i) {
  uint32_t y[N / 2];
#pragma unroll
  for (int c = 0; c < N / 2; ++c) y[c] = i & (N / 2) ? x[c + N / 2] : x[c];
#pragma unroll
  for (int half = N / 4; half > 0; half /= 2)
#pragma unroll
    for (int c = 0; c < half; ++c) y[c] = i & half ? y[c + half] : y[c];
  return y[0];
}

// Token of a bad[] entry if it is chunk `it`'s, else -1.
__device__ __forceinline__ int first_bad(uint32_t key, uint32_t it, bool rev) {
  if (key >> 8 != it + 1) return -1;
  const int rank = static_cast<int>(key & 255u);
  return rev ? rank : kC - 1 - rank;
}

// The long way of a wait, out of line: three warps of different roles share a
// scheduler's instruction cache, and what is rare must not take room in it.
__device__ __noinline__ bool wait_slow(uint64_t* b, uint32_t parity, TcTail* t, uint32_t* err) {
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
  TcTail* t;
  uint32_t* err;
  // All lanes of a role wait; false once the CTA gives up.
  __device__ __forceinline__ bool wait(uint64_t* b, uint32_t parity) const {
    return bar_try(b, parity) || wait_slow(b, parity, t, err);
  }
  __device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity) const {
    return __all_sync(kFull, wait(b, parity));
  }
};

// The part of one sequence that lies in the CTA's segment.
struct Piece {
  long long n, ps, pe;
  int m;  // how far the search came; -1: none left
  bool from_start, to_end;
};

__device__ __noinline__ Piece next_piece(const Problem* pp, bool rev, bool state_only, int m) {
  const Problem& p = *pp;
  const long long t0 = static_cast<long long>(blockIdx.x) * p.seg, t1 = min(t0 + p.seg, p.BL);
  const long long n0 = first_beyond(p, t0), n1 = first_from(p, t1);
  Piece x;
  while (m < n1 - n0) {
    x.n = rev ? n1 - 1 - m : n0 + m;
    ++m;
    const long long b0 = cu_at(p, x.n), b1 = cu_at(p, x.n + 1);
    x.ps = max(b0, t0);
    x.pe = min(b1, t1);
    x.from_start = rev ? x.pe == b1 : x.ps == b0;
    x.to_end = rev ? x.ps == b0 : x.pe == b1;
    x.m = m;
    if (x.pe > x.ps && !(state_only && x.to_end)) return x;
  }
  x.m = -1;
  return x;
}

// The CTA's chunks in scan order.
template <bool rev, bool state_only>
struct Walk {
  const Problem& p;
  Piece x;
  long long s0;         // chunk start
  int chunks, cc, len;  // of the piece; chunk; its tokens

  __device__ __forceinline__ explicit Walk(const Problem& p_) : p(p_), chunks(0), cc(-1) {
    x.m = 0;
  }
  __device__ __forceinline__ bool next() {
    if (++cc >= chunks) {
      const Piece y = next_piece(&p, rev, state_only, x.m);
      if (y.m < 0) return false;
      x = y;
      cc = 0;
      chunks = static_cast<int>((x.pe - x.ps + kC - 1) / kC);
    }
    // without rows against the scan: see the gates
    s0 = x.ps + static_cast<long long>(rev != state_only ? chunks - 1 - cc : cc) * kC;
    len = static_cast<int>(min(static_cast<long long>(kC), x.pe - s0));
    return true;
  }
  __device__ __forceinline__ bool last() const { return cc == chunks - 1; }
};

// A sequence's last state to global memory, eight columns at a time: `total`
// times the first term of the operand S that its last chunk began with
// (`base`: the lane's row; blocks of 64 columns are `block` bytes apart), and
// what tensor memory holds.  `on` is false for lanes without a row.
__device__ __noinline__ void put_final(uint32_t tm, const unsigned char* base, int block, int row, float total, float* to,
                                       long long sj, int dc, bool on) {
  const uint64_t total2 = pair(total, total);
#pragma unroll 1
  for (int d = 0; d < dc; d += 8) {
    uint32_t u[8];
    tmem_ld8(tm + d, u);
    wait_ld();
    if (!on) continue;
    const unsigned char* at = base + (d >> 6) * block + ((((d >> 3) ^ row) & 7) << 4);
    uint64_t x[4];
    const float* v = reinterpret_cast<const float*>(u);
    add_state(*reinterpret_cast<const uint4*>(at), total2, v, x);
    float y[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) unpair(x[q], y[2 * q], y[2 * q + 1]);
    if (sj == 1) {
      *reinterpret_cast<float4*>(to + d) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(to + d + 4) = make_float4(y[4], y[5], y[6], y[7]);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) to[(d + q) * sj] = y[q];
    }
  }
}

// `from` null: zeros.  Columns up to the next 16 are written too.
__device__ __noinline__ void get_state(uint32_t tm, const float* from, long long sj, int dc, bool on) {
  // sixteen columns' loads in flight
#pragma unroll 1
  for (int d = 0; d < dc; d += 16) {
    uint32_t v[16];
    if (from && on && sj == 1) {
#pragma unroll
      for (int q = 0; q < 16; q += 4) {
        const uint4 x = d + q < dc ? __ldg(reinterpret_cast<const uint4*>(from + d + q)) : make_uint4(0, 0, 0, 0);
        v[q] = x.x, v[q + 1] = x.y, v[q + 2] = x.z, v[q + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 16; ++q) v[q] = from && on && d + q < dc ? __float_as_uint(__ldg(from + (d + q) * sj)) : 0u;
    }
    tmem_st16(tm + d, v);
  }
  wait_st();
}

// NaN for what a value that is not finite reaches: rows from its token on
// (row < 0: all of the lanes, the state).
__device__ __noinline__ void spread_bad(uint32_t tm, const uint32_t* bad, uint32_t it, bool rev, int row, int d0, int d1) {
#pragma unroll 1
  for (int d = d0; d < d1; ++d) {
    const int first = first_bad(bad[d], it, rev);
    if (first < 0) continue;
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(tm + d));
    wait_ld();
    if (row < 0 || (rev ? row <= first : row >= first)) v = 0x7fffffffu;
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(tm + d), "r"(v) : "memory");
  }
  wait_st();
}

// One form over the CTA's segment.  What differs between the forms is fixed
// at compile time: the code that a CTA runs has to fit the instruction caches
// (with all variants in one body the row warps waited longer for instructions
// than for anything else).
template <bool REV, bool DOTS, bool STATE, bool FINE>
__device__ __forceinline__ void body(const Problem& p, const Form& f, const CUtensorMap* map) {
  extern __shared__ __align__(1024) unsigned char smem[];
  constexpr bool rev = REV, state_only = STATE;
  const int da = f.da, dc = f.dc, h = blockIdx.y;
  const TcGeom geo = tc_geom(da, dc);
  unsigned char* s_op = smem + (4 + geo.b_slots) * geo.slot_bytes;
  TcTail& t = *reinterpret_cast<TcTail*>(s_op + 2 * geo.s_bytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Ctl ctl{&t, p.err};

  if (smem_u32(smem) & 1023u) {  // the swizzled layouts need it
    if (tid == 0) report(ASCAN_DEV_ERR_STAGE, 0xffffffffull, p.err);
    return;
  }
  if (!state_only) fill_outside<__nv_bfloat16>(p, f);
  if (tid == 0) {
    for (int i = 0; i < 6; ++i) {
      bar_init(&t.full[i], 1);
      bar_init(&t.empty[i], i < 2 ? (state_only ? 8 : 9) : (i < 4 ? (DOTS ? 9 : 1) : 5));  // the products, and the row or column warps
    }
    bar_init(&t.tab_full, 1);
    bar_init(&t.tab_empty, state_only ? 12 : 16);
    bar_init(&t.sc_full, 1);
    bar_init(&t.in_full, 1);
    bar_init(&t.p_ready, 8);
    for (int i = 0; i < 4; ++i) bar_init(&t.kt_ready[i], 4);
    for (int i = 0; i < 2; ++i) bar_init(&t.kt_free[i], 1);
    bar_init(&t.u_full[0], 1);
    bar_init(&t.u_full[1], 1);
    bar_init(&t.s_ready, 4);
    bar_init(&t.o_full, 1);
    bar_init(&t.o_free, 8);
    bar_init(&t.d_full, 1);
    bar_init(&t.drain, 1);
    for (int i = 0; i < 2; ++i) bar_init(&t.added[i], 4);
    for (int i = 0; i < 4; ++i) bar_init(&t.own_read[i], 1);
    t.abort = 0;
    t.bad_chunk[0] = t.bad_chunk[1] = 0;
    static_assert(sizeof(TcTail) <= 3072, "the ring of 128-wide tiles leaves no more");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async();
  }
  for (int i = tid; i < 2 * kC; i += kTcThreads) t.bad[i / kC][i % kC] = 0;
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&t.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    fence_before();
  }
  __syncthreads();
  fence_after();
  const uint32_t tm = t.tmem;
  const int n16 = (dc + 15) / 16;  // 16-column pieces of the values
  const int blocks_a = da > 64 ? 2 : 1, blocks_c = dc > 64 ? 2 : 1;
  const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // the warp's quarter of tensor memory
  auto slot_at = [&](int x) { return smem + x * geo.slot_bytes; };
  // without rows B has A's slots
  auto slot_of_b = [&](uint32_t it) { return state_only ? static_cast<int>(it & 1) : (geo.b_slots == 2 ? 4 + static_cast<int>(it & 1) : 4); };
  auto phase_of_b = [&](uint32_t it) { return state_only || geo.b_slots == 2 ? (it >> 1) & 1 : it & 1; };
  Walk<REV, STATE> w(p);
  // (col . B)^T in two bfloat16 terms, or three where a float32 result depends
  // on the state, by halves of the chunk's tokens.  A term of a half takes 32
  // columns.  With rows there are four such places: of three terms, the second
  // half's take turns with the first's.  Without rows each half has four of its
  // own (kColK's, or the scores'): two terms of two chunks, or three of one.
  constexpr int terms = FINE ? 3 : 2;
  auto kt_at = [&](int half, int term, uint32_t ph) {
    if (state_only) return tm + (half ? kColK : kColSc) + 32 * (term + (FINE ? 0 : 2 * ph));
    return tm + kColK + 32 * ((terms * half + term) & 3);
  };

  // A half's terms are ready.  Without rows the columns may be two chunks ahead
  // of the products, so its barrier alternates with the chunks: one's parity
  // would be back where it was.
  auto kt_bar = [&](int half, uint32_t it) { return &t.kt_ready[state_only ? half + 2 * (it & 1) : half]; };
  auto kt_parity = [&](uint32_t it) { return (state_only ? it >> 1 : it) & 1; };

  // The column role.  Without rows the first four row warps take it too, and
  // each four build one half of the chunk's operand.
  auto columns = [&](int part) {
    const int i = (warp & 3) * 32 + lane;
    const bool work = i < blocks_a * 64;
    // The warp's 32 rows of (col.B)^T: matrix m of a load has rows 8 m.. and 8
    // tokens; lane r of it points at token r's 16 bytes.
    const int lead = (i >> 6) * 16384 + (lane & 7) * 128 + ((((i & 32) >> 3) + (lane >> 3) ^ (lane & 7)) << 4);
    for (uint32_t it = 0; w.next(); ++it) {
      const uint32_t ph = it & 1;
      const int slot_b = slot_of_b(it), slot_c = 2 + ph;
      const unsigned char* bt = slot_at(slot_b);
      unsigned char* ct = slot_at(slot_c);
      // The update before is done: its operand may be overwritten, and the row
      // and state warps have read what bad[ph] held two chunks ago.
      if (!state_only && it > 0) {
        if (!ctl.warp_wait(&t.u_full[ph ^ 1], ((it - 1) >> 1) & 1)) break;
        fence_after();
      }
      if (!state_only || w.len < kC)
        if (!ctl.warp_wait(&t.full[slot_c], (it >> 1) & 1)) break;
      if (state_only) {
        if (i >= w.len && part == 0)  // another sequence's token, or past the end
          for (int q = 0; q < 8 * blocks_c; ++q) *reinterpret_cast<uint4*>(ct + (q >> 3) * 16384 + i * 128 + ((q & 7) << 4)) = make_uint4(0, 0, 0, 0);
      } else {  // one token row of C per thread
        const bool live = i < w.len;
        const __nv_bfloat162 none = __float2bfloat162_rn(0.f);
        __nv_bfloat162 sum = none;  // sum of 0 * x: NaN if any x is not finite
#pragma unroll 2
        for (int q = 0; q < 8 * blocks_c; ++q) {
          uint4* at = reinterpret_cast<uint4*>(ct + (q >> 3) * 16384 + i * 128 + (((q & 7) ^ (i & 7)) << 4));
          if (live) {
            const uint4 x = *at;
            sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x.x), none, sum);
            sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x.y), none, sum);
            sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x.z), none, sum);
            sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x.w), none, sum);
          } else {
            *at = make_uint4(0, 0, 0, 0);  // another sequence's token, or past the end
          }
        }
        const bool bad = !(__low2float(sum) == 0.f && __high2float(sum) == 0.f);
        if (bad) {  // note and clear
          for (int d = 0; d < blocks_c * 64; ++d) {
            uint16_t* at = reinterpret_cast<uint16_t*>(ct + (d >> 6) * 16384 + i * 128 + ((((d & 63) >> 3) ^ (i & 7)) << 4) + (d & 7) * 2);
            if ((*at & 0x7f80u) == 0x7f80u) {
              *at = 0;
              atomicMax(&t.bad[ph][d], ((it + 1) << 8) | static_cast<uint32_t>(rev ? i : kC - 1 - i));
            }
          }
          t.bad_chunk[ph] = static_cast<int>(it) + 1;
        }
      }
      fence_async();
      if (!ctl.warp_wait(&t.tab_full, ph)) break;
      if (!ctl.warp_wait(&t.full[slot_b], phase_of_b(it))) break;
      const uint32_t src = smem_u32(bt) + lead;
      const bool tail = w.len < kC;
      bool ok = true;
#pragma unroll 1
      for (int half = state_only ? part : 0; half < (state_only ? part + 1 : 2); ++half) {
        // the places are free when the update that last used them is done
        if (state_only && !FINE) {
          if (it > 1) ok = ctl.warp_wait(&t.u_full[ph], ((it >> 1) & 1) ^ 1);
        } else if (state_only) {
          if (it > 0) ok = ctl.warp_wait(&t.kt_free[half], ph ^ 1);
        } else if (FINE && half == 1) {
          ok = ctl.warp_wait(&t.kt_free[0], ph);
        }
        if (!ok) break;
        if (FINE || state_only) fence_after();
        if (work) {
          const uint32_t k0 = kt_at(half, 0, ph) + lanes, k1 = kt_at(half, 1, ph) + lanes, k2 = kt_at(half, 2, ph) + lanes;
#pragma unroll 1
          for (int s1 = 0; s1 < kC / 2; s1 += 16) {
            const int s0 = half * (kC / 2) + s1;
            uint32_t hi[8], lo[8], least[8];  // [half of the rows][8 tokens][rows 0-7, 8-15]
            const float fb = t.far[s0 >> 5];
            const uint64_t fb2 = pair(fb, fb);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              uint32_t r[4];
              asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                           : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                           : "r"(src + (s0 + 8 * g) * 128)
                           : "memory");
              const int s = s0 + 8 * g + 2 * (lane & 3);
              const float2 cf = *reinterpret_cast<const float2*>(&t.col[s]);
              if (tail) {  // select, not multiply: the rows there are another sequence's
                const uint32_t keep = (s < w.len ? 0xffffu : 0u) | (s + 1 < w.len ? 0xffff0000u : 0u);
#pragma unroll
                for (int m = 0; m < 4; ++m) r[m] &= keep;
              }
              const uint64_t cf2 = mul2(pair(cf.x, cf.y), fb2);
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                uint64_t x = mul2(pair(lo_f(r[m]), hi_f(r[m])), cf2);
                const int at = (m >> 1) * 4 + g * 2 + (m & 1);
                hi[at] = round2(x);
                x = left2(x, hi[at]);
                lo[at] = round2(x);
                if (FINE) least[at] = rest2(x, lo[at]);
              }
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const uint32_t to = (static_cast<uint32_t>(m) << 20) + s1 / 2;
              tmem_st16x128(k0 + to, hi + 4 * m);
              tmem_st16x128(k1 + to, lo + 4 * m);
              if (FINE) tmem_st16x128(k2 + to, least + 4 * m);
            }
          }
          wait_st();
        }
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(kt_bar(half, it));
      }
      if (!ok) break;
      if (lane == 0) {
        bar_arrive(&t.tab_empty);
        bar_arrive(&t.empty[slot_b]);
      }
    }
  };

  if (warp < 8) {
    // ---- row warps ----
    const int quad = warp & 3, side = warp >> 2, row = quad * 32 + lane;
    const uint64_t sp2 = pair(f.sp, f.sp);
    // The side's columns: half of the whole.  At 64 columns and fewer the two
    // sides share a stage block, each a half of its rows.
    const bool wide = dc > 64;
    const int c16 = side * (wide ? 4 : 2), c16_end = min(c16 + (wide ? 4 : 2), n16);
    const int block = wide ? side : 0;
    constexpr bool dots = DOTS;  // the forms whose rows the gate's gradient needs
    uint32_t dot_loads = 0;
    uint32_t park[8] = {};
    int held = -1;  // slot that the last rows leave from
    auto release = [&] {
      if (held >= 0 && lane == 0) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        bar_arrive(&t.empty[held]);
      }
      held = -1;
    };
    if (state_only && warp < 4) columns(0);
    for (uint32_t it = 0; !state_only && w.next(); ++it) {
      const uint32_t ph = it & 1;
      const int slot_a = ph;
      unsigned char* stage = slot_at(slot_a);
      if (!ctl.warp_wait(&t.tab_full, ph)) break;
      const float4 l4 = t.lg[row >> 1];
      const float lx = (row & 1) ? -l4.y : -l4.x, ly = (row & 1) ? -l4.w : -l4.z;
      const uint64_t lx2 = pair(lx, lx), ly2 = pair(ly, ly);
      const float rf = ex2(lx) * f.sr;
      if (!ctl.warp_wait(&t.sc_full, ph)) break;
      fence_after();
      // A token's own term does not depend on any gate, and with it the dots
      // would lose the digits of what does: P leaves it out, and it is added
      // after the dots.  Both warps of the 32 tokens need it; the one whose
      // columns these are not reads its rows' own scores before P takes their
      // place.
      float own = 0.f;
      if (dots && side != quad >> 1) {
        uint32_t s[32];
        tmem_ld32(tm + lanes + kColSc + 32 * quad, s);
        wait_ld();
        own = __uint_as_float(pick<32>(s, lane));
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&t.own_read[quad]);
      }
      // Sixteen columns at a time, those that the mask leaves something of.
      // Where a block of 32 lies wholly inside, the decay is that of the row
      // to the block's edge times col[], two products an element; in the
      // row's own block every decay is computed by itself, and masked scores
      // are cleared as bits (a product with zero would keep a NaN).  (Longer loop bodies would run once or
      // twice a chunk and wait for their instructions.)
      const int b0 = 2 * max(2 * side, rev ? quad : 0), b1 = 2 * min(2 * side + 2, rev ? 4 : quad + 1);
      // The row's own block comes last.
      bool ok = true;
#pragma unroll 1
      for (int i = b0; i < b1; ++i) {
        const int b = rev ? b0 + b1 - 2 - i + 2 * (i & 1) : i;
        const uint32_t col = tm + lanes + kColSc + 32 * (b >> 1);
        uint32_t s[16], hi[8];
        tmem_ld16(col + 16 * (b & 1), s);
        uint64_t pv[8];
        if (b >> 1 != quad) {
          const float4 e4 = t.lg[rev ? 16 * (b >> 1) - 1 : 16 * (b >> 1) + 15];
          const float rd = ex2((lx + e4.y) + (ly + e4.w)) * f.sp;
          const uint64_t rd2 = pair(rd, rd);
#pragma unroll
          for (int c = 0; c < 8; c += 2) {
            const float4 m = *reinterpret_cast<const float4*>(&t.col[16 * b + 2 * c]);
            pv[c] = mul2(pair(m.x, m.y), rd2);
            pv[c + 1] = mul2(pair(m.z, m.w), rd2);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float4 m = t.lg[8 * b + c];
            float x0, x1;
            unpair(add2(add2(lx2, pair(m.x, m.y)), add2(ly2, pair(m.z, m.w))), x0, x1);
            pv[c] = mul2(sp2, pair(ex2(x0), ex2(x1)));
          }
        }
        wait_ld();
        if (dots && b >> 1 == quad) {
          const float x = __uint_as_float(pick<16>(s, lane & 15));
          if (b & 1) {
            own = lane & 16 ? x : own;
          } else {
            own = x;
            ok = ctl.warp_wait(&t.own_read[quad], ph);
            if (!ok) break;
            fence_after();
          }
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) pv[c] = mul2(pair(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), pv[c]);
        // P's place is the block's own: first terms in its lower half, second
        // in its upper.  The upper half's scores must be read before, so the
        // first step of a block parks its second terms in registers.
#pragma unroll
        for (int c = 0; c < 8; ++c) hi[c] = round2(pv[c]);
        uint32_t lo[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) lo[c] = rest2(pv[c], hi[c]);
        if (b >> 1 == quad || (rev && 16 * b + 16 > w.len)) {
          // the columns that count, as the bits of the packed pairs
          const int from = (rev ? row + dots : 0) - 16 * b, to = (rev ? w.len : row + 1 - dots) - 16 * b;
          const uint32_t keep = below(to) & ~below(from);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t bits = (keep & (1u << (2 * c)) ? 0xffffu : 0u) | (keep & (2u << (2 * c)) ? 0xffff0000u : 0u);
            hi[c] &= bits;
            lo[c] &= bits;
          }
        }
        tmem_st8(col + 8 * (b & 1), hi);
        if (b & 1) {
          tmem_st8(col + 16, park);
          tmem_st8(col + 24, lo);
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) park[c] = lo[c];
        }
      }
      if (!ok) break;
      own *= f.sp;
      const uint64_t own2 = pair(own, own);
#pragma unroll 1
      for (int b = max(2 * side, rev ? 0 : quad + 1); b < min(2 * side + 2, rev ? quad : 4); ++b) {  // outside the mask
        uint32_t none[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) none[c] = 0u;
        tmem_st16(tm + lanes + kColSc + 32 * b, none);
        tmem_st16(tm + lanes + kColSc + 32 * b + 16, none);
      }
      __syncwarp();
      if (lane == 0) bar_arrive(&t.tab_empty);
      release();
      if (!ctl.warp_wait(&t.in_full, ph)) break;
      fence_after();
      // The products have read A: its slot holds first the rows to take dots
      // with, then the finished rows on their way to whole-line stores.
      if (dots && tid == 0) {
        bar_expect(&t.d_full, blocks_c * 16384);
        for (int b = 0; b < blocks_c; ++b)
          tma_rows(smem_u32(stage + b * 16384), &map[3], b * 64, h / f.dot.share, static_cast<int>(w.s0), &t.d_full);
        ++dot_loads;
      }
      const uint64_t rf2 = pair(rf, rf);
#pragma unroll 1
      for (int b = c16; b < c16_end; ++b) {
        uint32_t v[16];
        tmem_ld16(tm + lanes + kColO + 16 * b, v);
        wait_ld();
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          float x, y;
          unpair(mul2(pair(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), rf2), x, y);
          v[c] = __float_as_uint(x), v[c + 1] = __float_as_uint(y);
        }
        tmem_st16(tm + lanes + kColO + 16 * b, v);
      }
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&t.p_ready);

      if (dots && !ctl.warp_wait(&t.d_full, ph)) break;
      if (dots && !ctl.warp_wait(&t.full[2 + ph], (it >> 1) & 1)) break;
      if (!ctl.warp_wait(&t.o_full, ph)) break;
      fence_after();
      if (t.bad_chunk[ph] == static_cast<int>(it) + 1) spread_bad(tm + lanes + kColO, t.bad[ph], it, rev, row, 16 * c16, min(dc, 16 * c16_end));
      unsigned char* mine = stage + block * 16384 + row * 128;
      const unsigned char* values = slot_at(2 + ph) + block * 16384 + row * 128;
      // the own term of eight columns
      auto add_own = [&](uint64_t* x, int piece) {
        const uint4 y = *reinterpret_cast<const uint4*>(values + ((piece ^ (row & 7)) << 4));
        x[0] = fma2(own2, pair(lo_f(y.x), hi_f(y.x)), x[0]);
        x[1] = fma2(own2, pair(lo_f(y.y), hi_f(y.y)), x[1]);
        x[2] = fma2(own2, pair(lo_f(y.z), hi_f(y.z)), x[2]);
        x[3] = fma2(own2, pair(lo_f(y.w), hi_f(y.w)), x[3]);
      };
      uint64_t dot2 = 0;
#pragma unroll 1
      for (int b = c16; b < c16_end; ++b) {
        uint32_t v[16];
        tmem_ld16(tm + lanes + kColO + 16 * b, v);
        wait_ld();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint4* piece = reinterpret_cast<uint4*>(mine + ((((b & 3) * 2 + q) ^ (row & 7)) << 4));
          uint64_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = pair(__uint_as_float(v[8 * q + 2 * e]), __uint_as_float(v[8 * q + 2 * e + 1]));
          if (dots) {
            const uint4 y = *piece;
            dot2 = fma2(x[0], pair(lo_f(y.x), hi_f(y.x)), dot2);
            dot2 = fma2(x[1], pair(lo_f(y.y), hi_f(y.y)), dot2);
            dot2 = fma2(x[2], pair(lo_f(y.z), hi_f(y.z)), dot2);
            dot2 = fma2(x[3], pair(lo_f(y.w), hi_f(y.w)), dot2);
            if (!f.out_f32) add_own(x, (b & 3) * 2 + q);
          }
          if (!f.out_f32) *piece = make_uint4(round2(x[0]), round2(x[1]), round2(x[2]), round2(x[3]));
        }
      }
      if (f.out_f32) {
        // 16 columns of float32 fill half a row of the stage
#pragma unroll 1
        for (int b = c16; b < c16_end; ++b) {
          uint32_t v[16];
          tmem_ld16(tm + lanes + kColO + 16 * b, v);
          wait_ld();
          const int half = (wide ? b & 1 : side) * 4, q = lane & 3, r0 = quad * 32 + (lane >> 2);
          if (dots) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint64_t x[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) x[c] = pair(__uint_as_float(v[8 * e + 2 * c]), __uint_as_float(v[8 * e + 2 * c + 1]));
              add_own(x, (b & 3) * 2 + e);
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                float lo, hi;
                unpair(x[c], lo, hi);
                v[8 * e + 2 * c] = __float_as_uint(lo), v[8 * e + 2 * c + 1] = __float_as_uint(hi);
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(mine + (((half + c) ^ (row & 7)) << 4)) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
          __syncwarp();
          if (16 * b + q * 4 < dc)
#pragma unroll 2
            for (int r = r0; r < min(quad * 32 + 32, w.len); r += 8)
              *reinterpret_cast<uint4*>(static_cast<float*>(f.out) + ((w.s0 + r) * p.H + h) * dc + 16 * b + q * 4) =
                  *reinterpret_cast<const uint4*>(stage + block * 16384 + r * 128 + (((half + q) ^ (r & 7)) << 4));
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) {
        bar_arrive(&t.o_free);
        if (dots) bar_arrive(&t.empty[2 + ph]);
      }
      // The warp's 32 rows to memory: whole ones by bulk copies that the slot
      // waits for one chunk later, those at a piece's end by the lanes.
      fence_async();
      __syncwarp();
      if (!f.out_f32) {
        if (wide && quad * 32 + 32 <= w.len) {
          if (lane == 0)
            asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(&map[4]),
                         "r"(side * 64), "r"(h), "r"(static_cast<int>(w.s0) + quad * 32),
                         "r"(smem_u32(stage + side * 16384 + quad * 4096))
                         : "memory");
        } else {
          const int bits = wide ? 3 : 2, q = (lane & ((1 << bits) - 1)) + (wide ? 0 : side * 4);
#pragma unroll 1
          for (int r = quad * 32 + (lane >> bits); r < min(quad * 32 + 32, w.len); r += 32 >> bits)
            if (64 * block + 8 * q < dc)
              *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(f.out) + ((w.s0 + r) * p.H + h) * dc + 64 * block + 8 * q) =
                  *reinterpret_cast<const uint4*>(stage + block * 16384 + r * 128 + ((q ^ (r & 7)) << 4));
          __syncwarp();
        }
      }
      if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      held = slot_a;
      if (dots && row < w.len && c16 < c16_end) {
        float x, y;
        unpair(dot2, x, y);
        f.rowdot[(static_cast<long long>(side) * p.H + h) * p.BL + w.s0 + row] = x + y;
      }
    }
    if (!state_only && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (dot_loads && !state_only) {  // in flight only after a give-up
      const unsigned long long start = now_ns();
      while (!bar_try(&t.d_full, (dot_loads - 1) & 1) && now_ns() - start < kStageTimeoutNs) {
      }
    }
  } else if (warp < 12) {
    // ---- state warps ----
    const int i = tid - 256;
    const int rows = (da + 15) / 16 * 16;  // the product with S runs over whole sixteens
    const bool work = (warp - 8) * 32 < rows;
    const long long mat = static_cast<long long>(da) * dc;
    const uint32_t ut = tm + lanes + kColU;
    if (state_only) {
      // One piece: every chunk's contribution comes from a fresh accumulator
      // (U's place or O's) and is added here, where the operand S is otherwise,
      // [4 columns][row]; at the end what came in, decayed, on top.
      const int cap = blocks_a * 64, n32 = (dc + 31) / 32;  // columns beyond dc have places of their own
      float4* sum = reinterpret_cast<float4*>(s_op) + i;
      uint32_t it = 0;
      float decay = 0.f;
      bool ok = true;
      for (; ok && w.next(); ++it) {
        ok = ctl.warp_wait(&t.tab_full, it & 1);
        if (!ok) break;
        decay = t.total;
        __syncwarp();
        if (lane == 0) bar_arrive(&t.tab_empty);
        ok = ctl.warp_wait(&t.u_full[it & 1], (it >> 1) & 1);
        if (!ok) break;
        fence_after();
        if (work) {
#pragma unroll 1
          for (int b = 0; b < n32; ++b) {
            float v[32];
            tmem_ld32((it & 1 ? tm + lanes + kColO : ut) + 32 * b, reinterpret_cast<uint32_t*>(v));
            wait_ld();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              float4* at = sum + (8 * b + q) * cap;
              const float4 old = it > 0 ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
              *at = make_float4(old.x + v[4 * q], old.y + v[4 * q + 1], old.z + v[4 * q + 2], old.w + v[4 * q + 3]);
            }
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&t.added[it & 1]);
      }
      if (ok && it > 0) {
        if (work && i < da) {
          const bool begins = w.x.from_start && f.init;
          const float* from = f.init + (w.x.n * p.H + h) * mat + i * f.si;
          float* to = f.carry + (static_cast<long long>(blockIdx.x) * p.H + h) * mat + static_cast<long long>(i) * dc;
#pragma unroll 1
          for (int d = 0; d < dc; d += 4) {
            float4 v = sum[d / 4 * cap];
            if (begins) {
              v.x = fmaf(decay, __ldg(from + d * f.sj), v.x);
              v.y = fmaf(decay, __ldg(from + (d + 1) * f.sj), v.y);
              v.z = fmaf(decay, __ldg(from + (d + 2) * f.sj), v.z);
              v.w = fmaf(decay, __ldg(from + (d + 3) * f.sj), v.w);
            }
            *reinterpret_cast<float4*>(to + d) = v;
          }
        }
        // a piece that holds the sequence's start takes nothing from before
        if (i == 0) f.dec[blockIdx.x * p.H + h] = w.x.from_start ? -1.f : decay;
      }
    }
    // The state lives in two places: 8 bits of it as the first term of the
    // operand S, and the rest, below 2^-8 of it, as what the chunk's update
    // starts from in tensor memory.  So the products add to values of one
    // chunk's size: they truncate, and over the many chunks of a long sequence
    // the whole state would lose 6e-5 of its norm to that (65536 tokens, gates
    // of 0), where now float32 rounds once a chunk.
    const int block_bytes = geo.s_bytes / blocks_c;
    uint64_t before2 = 0;  // the decay over the chunk before
    for (uint32_t it = 0; !state_only && w.next(); ++it) {
      const uint32_t ph = it & 1;
      const bool first = w.cc == 0;
      if (!ctl.warp_wait(&t.tab_full, ph)) break;
      const float total = t.total;
      __syncwarp();
      if (lane == 0) bar_arrive(&t.tab_empty);
      if (it > 0) {  // the update before this chunk; it also follows the last use of S
        if (!ctl.warp_wait(&t.u_full[ph ^ 1], ((it - 1) >> 1) & 1)) break;
        fence_after();
      }
      if (first) {
        const float* from = nullptr;
        long long sj = 1;
        if (!w.x.from_start)
          from = f.carry + ((static_cast<long long>(blockIdx.x) + (rev ? 1 : -1)) * p.H + h) * mat + static_cast<long long>(i) * dc;
        else if (f.init)
          from = f.init + (w.x.n * p.H + h) * mat + i * f.si, sj = f.sj;
        if (work) get_state(ut, from, sj, dc, i < da);
      } else if (work && t.bad_chunk[ph ^ 1] == static_cast<int>(it)) {
        spread_bad(ut, t.bad[ph ^ 1], it - 1, rev, -1, 0, dc);
      }
      float* snap = nullptr;
      if (DOTS && f.snap && i < da) {
        const long long edge = rev ? w.s0 + w.len : w.s0;
        if (edge > w.x.ps && edge < w.x.pe && (edge - w.x.ps) % p.restart == 0)
          // both forms' stored states only meet each other, so they may lie as
          // the lanes hold them: whole lines a store
          snap = f.snap + (snap_slot(p, edge) * p.H + h) * mat + i * 8;
      }
      const uint64_t total2 = pair(total, total);
      const uint32_t keep = first ? 0u : ~0u;
      if (first) before2 = 0;
      if (work) {
#pragma unroll 1
        for (int b = 0; b < n16; ++b) {
          float v[16];
          tmem_ld16(ut + 16 * b, reinterpret_cast<uint32_t*>(v));
          wait_ld();
          if (i < rows) {
            // S: row i of 64 columns is 128 bytes; two 16-byte pieces per 16 columns
            unsigned char* base = s_op + (b >> 2) * block_bytes + i * 128;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint4* at = reinterpret_cast<uint4*>(base + ((((b & 3) * 2 + q) ^ (i & 7)) << 4));
              uint4* at_lo = reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(at) + geo.s_bytes);
              uint64_t x[4];
              uint4 old = *at;
              old.x &= keep, old.y &= keep, old.z &= keep, old.w &= keep;
              add_state(old, before2, v + 8 * q, x);
              if (DOTS && snap && 16 * b + 8 * q < dc) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) unpair(x[e], y[2 * e], y[2 * e + 1]);
                float4* to = reinterpret_cast<float4*>(snap + (2 * b + q) * 8 * da);
                to[0] = make_float4(y[0], y[1], y[2], y[3]);
                to[1] = make_float4(y[4], y[5], y[6], y[7]);
              }
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                hi[e] = round2(x[e]);
                x[e] = left2(x[e], hi[e]);
                lo[e] = round2(x[e]);
                unpair(mul2(x[e], total2), v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
              }
              *at = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              *at_lo = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
          }
          tmem_st16(ut + 16 * b, reinterpret_cast<const uint32_t*>(v));
        }
        wait_st();
      }
      before2 = total2;
      fence_async();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&t.s_ready);
      if (w.last() && w.x.to_end && f.fin) {
        if (!ctl.warp_wait(&t.u_full[ph], (it >> 1) & 1)) break;
        fence_after();
        if (work) {
          if (t.bad_chunk[ph] == static_cast<int>(it) + 1) spread_bad(ut, t.bad[ph], it, rev, -1, 0, dc);
          put_final(ut, s_op + i * 128, block_bytes, i, total, f.fin + (w.x.n * p.H + h) * mat + i * f.si, f.sj, dc, i < da);
        }
      }
    }
  } else if (warp < 16) {
    columns(state_only ? 1 : 0);
  } else if (warp == 16) {
    // ---- loads: what comes free first is asked for first ----
    if (lane == 0) {
      uint32_t count = 0;  // chunks
      bool ok = true;
      auto load = [&](int slot, uint32_t use, int which, int blocks, const Rows& r) {
        if (use > 0 && !ctl.wait(&t.empty[slot], (use - 1) & 1)) return false;
        bar_expect(&t.full[slot], blocks * 16384);
#pragma unroll 1
        for (int b = 0; b < blocks; ++b)
          tma_rows(smem_u32(slot_at(slot) + b * 16384), &map[which], b * 64, h / r.share, static_cast<int>(w.s0), &t.full[slot]);
        return true;
      };
      uint32_t a_loads = 0, b_loads = 0, c_loads = 0;
      while (ok && w.next()) {
        ok = load(2 + (count & 1), count >> 1, 2, blocks_c, f.c);
        c_loads += ok;
        if (ok) {
          ok = load(slot_of_b(count), state_only || geo.b_slots == 2 ? count >> 1 : count, 1, blocks_a, f.b);
          b_loads += ok;
        }
        if (ok && !state_only) {
          ok = load(count & 1, count >> 1, 0, blocks_a, f.a);
          a_loads += ok;
        }
        ++count;
      }
      // a load in flight must land before the CTA leaves (only after a give-up)
      auto land = [&](int slot, uint32_t uses) {
        const unsigned long long start = now_ns();
        while (uses > 0 && !bar_try(&t.full[slot], (uses - 1) & 1) && now_ns() - start < kStageTimeoutNs) {
        }
      };
      for (int x = 0; x < 2; ++x) {
        land(x, ((state_only ? b_loads : a_loads) + 1 - x) >> 1);
        land(2 + x, (c_loads + 1 - x) >> 1);
        if (state_only) continue;
        if (geo.b_slots == 2) land(4 + x, (b_loads + 1 - x) >> 1);
        else if (x == 0) land(4, b_loads);
      }
    }
  } else if (warp == 17) {
    // ---- products ----
    const uint32_t id_sc = idesc(kC, false), id_v = idesc((dc + 15) / 16 * 16, true);
    const int ka = (da + 15) / 16;
    const uint64_t ds = desc(smem_u32(s_op), geo.s_bytes / blocks_c);
    // U += (col . B)^T C over 64 tokens, small terms first: the fewer products
    // truncate at full size
    auto update = [&](int half, uint32_t ph, uint64_t c) {
      if (elect_one()) {
#pragma unroll 1
        for (int term = terms - 1; term >= 0; --term) {
          const uint32_t kt = kt_at(half, term, ph);
#pragma unroll 1
          for (int k = 0; k < kC / 32; ++k)
            mma_tmem(tm + (state_only && ph ? kColO : kColU), kt + k * 8, c + (half * 4 + k) * 128, id_v,
                     !state_only || half + k > 0 || term < terms - 1);
        }
        commit(&t.kt_free[half]);
      }
    };
    for (uint32_t it = 0; w.next(); ++it) {
      const uint32_t ph = it & 1;
      const int sa = ph, sb = slot_of_b(it), sc = 2 + ph;
      const uint64_t c = desc(smem_u32(slot_at(sc)), 16384);
      if (!ctl.warp_wait(&t.full[sb], phase_of_b(it))) break;
      if (!state_only) {
        if (!ctl.warp_wait(&t.full[sa], (it >> 1) & 1)) break;
        // the scores go where the previous chunk's P lies until its product is done
        if (it > 0 && !ctl.warp_wait(&t.o_full, ph ^ 1)) break;
        fence_after();
        const uint64_t a = desc(smem_u32(slot_at(sa)), 16), b = desc(smem_u32(slot_at(sb)), 16);
        if (elect_one()) {
#pragma unroll 1
          for (int k = 0; k < ka; ++k) {
            const uint32_t o = (k >> 2) * 1024 + (k & 3) * 2;  // in 16 bytes: the next 64 columns, 16 of them
            mma_smem(tm + kColSc, a + o, b + o, id_sc, k > 0);
          }
          commit(&t.sc_full);
          commit(&t.empty[sb]);
        }
        if (!ctl.warp_wait(&t.s_ready, ph)) break;
        // the update's first half only waits for the state to have been read
        if (!ctl.warp_wait(kt_bar(0, it), kt_parity(it))) break;
        if (!ctl.warp_wait(&t.full[sc], (it >> 1) & 1)) break;
        fence_after();
        update(0, ph, c);
        if (it > 0 && !ctl.warp_wait(&t.o_free, ph ^ 1)) break;
        fence_after();
        if (elect_one()) {
#pragma unroll 1
          for (int term = 0; term < 2; ++term)
#pragma unroll 1
            for (int k = 0; k < ka; ++k)
              mma_smem(tm + kColO, a + (k >> 2) * 1024 + (k & 3) * 2, ds + term * (geo.s_bytes >> 4) + k * 128, id_v, term + k > 0);
          commit(&t.in_full);
          commit(&t.empty[sa]);
        }
      } else {
        if (it > 1 && !ctl.warp_wait(&t.added[ph], ((it >> 1) & 1) ^ 1)) break;  // accumulators take turns
        if (!ctl.warp_wait(&t.full[sc], (it >> 1) & 1)) break;
        if (!ctl.warp_wait(kt_bar(0, it), kt_parity(it))) break;
        fence_after();
        update(0, ph, c);
      }
      if (!ctl.warp_wait(kt_bar(1, it), kt_parity(it))) break;
      fence_after();
      update(1, ph, c);
      if (elect_one()) {
        commit(&t.u_full[ph]);
        if (state_only) commit(&t.empty[sc]);
      }
      if (!state_only) {
        if (!ctl.warp_wait(&t.p_ready, ph)) break;
        fence_after();
        if (elect_one()) {
#pragma unroll 1
          for (int term = 0; term < 2; ++term)
#pragma unroll 1
            for (int k = 0; k < kC / 16; ++k)
              mma_tmem(tm + kColO, tm + kColSc + (k >> 1) * 32 + (k & 1) * 8 + term * 16, c + k * 128, id_v, true);
          commit(&t.o_full);
          commit(&t.empty[sc]);
        }
      }
    }
    if (elect_one()) commit(&t.drain);  // nothing of this CTA's is in flight after it
    const unsigned long long start = now_ns();
    while (!bar_try(&t.drain, 0) && now_ns() - start < kStageTimeoutNs) {
    }
  } else {
    // ---- gates: four tokens a lane ----
    // Without rows the chunks come against the scan's order, and the column
    // factors reach to the far end of the piece: what the chunks before this
    // one (after it in the scan) decay by is in `passed`.  The chunks' updates
    // then add up with nothing to scale between them.
    double passed = 0.0;
    for (uint32_t it = 0; w.next(); ++it) {
      double g[4], sum = 0.0;
      float raw[4] = {0.f, 0.f, 0.f, 0.f};
      const long long at = w.s0 * p.gate.st + (h / p.gate.share) * p.gate.sh;
      if (p.gate_type == ASCAN_F32) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (lane * 4 + q < w.len) raw[q] = __ldg(static_cast<const float*>(p.gate.p) + at + (lane * 4 + q) * p.gate.st);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (lane * 4 + q < w.len)
            raw[q] = __uint_as_float(static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(p.gate.p) + at + (lane * 4 + q) * p.gate.st)) << 16);
      }
      // Sums run in the scan's direction and are never differences of longer
      // ones: a gate that is not finite must not reach the tokens before it.
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int q = rev ? 3 - e : e;
        if (rev) g[q] = sum;
        sum += static_cast<double>(raw[q] < kGateFloor ? kGateFloor : raw[q]);
        if (!rev) g[q] = sum;
      }
      double inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const double u = rev ? __shfl_down_sync(kFull, inc, o) : __shfl_up_sync(kFull, inc, o);
        if (rev ? lane + o < 32 : lane >= o) inc += u;
      }
      const double end = __shfl_sync(kFull, inc, rev ? 0 : 31);
      double before = rev ? __shfl_down_sync(kFull, inc, 1) : __shfl_up_sync(kFull, inc, 1);
      if (lane == (rev ? 31 : 0)) before = 0.0;
      float lx[4], ly[4], col[4];
      float2 whole;
      const double y = end * -1.4426950408889634;
      whole.x = static_cast<float>(y);
      whole.y = static_cast<float>(y - static_cast<double>(whole.x));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const double x = (before + g[q]) * -1.4426950408889634;
        lx[q] = static_cast<float>(x);
        ly[q] = static_cast<float>(x - static_cast<double>(lx[q]));
      }
      // the edge of the lane's 32 tokens: their last, or the one before them
      float ex = __shfl_sync(kFull, lx[3], rev ? (lane & 24) - 1 : lane | 7);
      float ey = __shfl_sync(kFull, ly[3], rev ? (lane & 24) - 1 : lane | 7);
      if (rev && lane < 8) ex = whole.x, ey = whole.y;  // before the chunk's first token
#pragma unroll
      for (int q = 0; q < 4; ++q) col[q] = ex2((lx[q] - ex) + (ly[q] - ey));
      float far = ex2((ex - whole.x) + (ey - whole.y)) * f.sc;
      float all = ex2(-whole.x);
      if (state_only) {
        far *= ex2(static_cast<float>(passed * 1.4426950408889634));
        passed += end;
        all = ex2(static_cast<float>(passed * 1.4426950408889634));
      }
      if (it > 0 && !ctl.warp_wait(&t.tab_empty, (it & 1) ^ 1)) break;
      t.lg[lane * 2] = make_float4(lx[0], lx[1], ly[0], ly[1]);
      t.lg[lane * 2 + 1] = make_float4(lx[2], lx[3], ly[2], ly[3]);
      *reinterpret_cast<float4*>(&t.col[lane * 4]) = make_float4(col[0], col[1], col[2], col[3]);
      if ((lane & 7) == 0) t.far[lane >> 3] = far;
      if (lane == 0) t.total = all;
      __syncwarp();
      if (lane == 0) bar_arrive(&t.tab_full);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == 17) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm));
  }
}

template <bool STATE, bool FINE>
__device__ __forceinline__ void dispatch(const Problem& p, const Form& f, const CUtensorMap* map) {
  if (!STATE && f.rowdot) {
    if (f.rev) body<true, true, false, FINE>(p, f, map);
    else body<false, true, false, FINE>(p, f, map);
  } else {
    if (f.rev) body<true, false, STATE, FINE>(p, f, map);
    else body<false, false, STATE, FINE>(p, f, map);
  }
}

template <bool STATE>
__global__ void __launch_bounds__(kTcThreads, 1)
    tc_kernel(const __grid_constant__ Launch L, const __grid_constant__ TcMaps maps) {
  const Form& f = L.f[blockIdx.z];
  const CUtensorMap* map = maps.m[blockIdx.z];
  if (f.fine) dispatch<STATE, true>(L.p, f, map);
  else dispatch<STATE, false>(L.p, f, map);
}

static bool map_rows(CUtensorMap* m, const Rows& r, int dim, long long BL, int H, int tokens = kC) {
  const auto fn = encode_fn();
  if (!fn) return false;
  const int heads = H / r.share;
  const long long sh = heads > 1 ? r.sh : (dim + 7) / 8 * 8;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(BL)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(r.st) * 2};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(tokens)}, one[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(r.p), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// bfloat16 rows that a tensor map can describe: 16-byte bases and strides,
// head sizes in whole 16-byte pieces, heads that do not overlap.
static bool rows_usable(const Rows& r, int dim, int H) {
  if (!r.p) return true;
  if ((reinterpret_cast<uintptr_t>(r.p) & 15u) || dim % 8 || r.st % 8 || r.st < dim || r.st >= (1ll << 38)) return false;
  return H / r.share == 1 || (r.sh % 8 == 0 && r.sh >= dim && r.sh < (1ll << 38));
}

int tc_dot_parts(const Form& f) { return f.dc > 32 ? 2 : 1; }

bool tc_usable(const Launch& l, int roles, int dtype) {
  if (dtype != ASCAN_BF16 || l.p.gate_type == ASCAN_F16 || l.p.BL > 0x7fffff00ll) return false;
  for (int r = 0; r < roles; ++r) {
    const Form& f = l.f[r];
    if (!rows_usable(f.a, f.da, l.p.H) || !rows_usable(f.b, f.da, l.p.H) || !rows_usable(f.c, f.dc, l.p.H) ||
        !rows_usable(f.dot, f.dc, l.p.H) || (reinterpret_cast<uintptr_t>(f.out) & 15u) ||
        (reinterpret_cast<uintptr_t>(f.init) & 15u) || (reinterpret_cast<uintptr_t>(f.fin) & 15u))
      return false;
  }
  return encode_fn() != nullptr;
}

int tc_run(const Launch& l, int roles, bool state_only, cudaStream_t s) {
  // Tensor maps are made through the driver, which wants a current context;
  // a thread whose first CUDA call this is (autograd's, with every buffer out
  // of torch's cache) has none until the runtime is told its device.
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return ASCAN_EDEVICE;
  TcMaps maps;
  memset(&maps, 0, sizeof(maps));
  size_t smem = 0;
  for (int r = 0; r < roles; ++r) {
    const Form& f = l.f[r];
    if (!map_rows(&maps.m[r][0], f.a, f.da, l.p.BL, l.p.H) || !map_rows(&maps.m[r][1], f.b, f.da, l.p.BL, l.p.H) ||
        !map_rows(&maps.m[r][2], f.c, f.dc, l.p.BL, l.p.H) ||
        (f.rowdot && !map_rows(&maps.m[r][3], f.dot, f.dc, l.p.BL, l.p.H)) ||
        (!f.out_f32 && !map_rows(&maps.m[r][4], Rows{f.out, static_cast<long long>(l.p.H) * f.dc, f.dc, 1}, f.dc, l.p.BL, l.p.H, 32)))
      return ASCAN_ECUDA;
    const TcGeom g = tc_geom(f.da, f.dc);
    const size_t need = g.bytes() + sizeof(TcTail);
    if (need > smem) smem = need;
  }
  static std::atomic<unsigned long long> done[2]{};
  const int rc = state_only ? allow_smem(tc_kernel<true>, kSmemLimit, done[1]) : allow_smem(tc_kernel<false>, kSmemLimit, done[0]);
  if (rc != ASCAN_OK) return rc;
  const dim3 grid(l.p.J, l.p.H, roles);
  if (state_only) tc_kernel<true><<<grid, kTcThreads, smem, s>>>(l, maps);
  else tc_kernel<false><<<grid, kTcThreads, smem, s>>>(l, maps);
  return launch_status();
}

}  // namespace mscan

ASCAN_UNIT_ERROR_ACCESSORS(mscan_tc)

}  // namespace ascan
