// ascan_mscan.cuh -- the matrix-state recurrence: what its kernels share.
//
//   S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T        o[t] = scale * q[t] S[t]
//
// per head, S a [Dk, Dv] matrix in float32.  Over a chunk of tokens with
// G[t] the inclusive sum of g inside the chunk this is
//
//   o[t]  = scale * (e^{G[t]} q[t] S_in + sum_{s<=t} e^{G[t]-G[s]} (q[t].k[s]) v[s])
//   S_out = e^{G[C]} S_in + sum_s e^{G[C]-G[s]} k[s] v[s]^T
//
// i.e. two masked products and two products with the state.  The gradients
// are the same form with the operands in other places:
//
//   dq: rows do, columns v, values k, forwards      (state: sum v k^T)
//   dk: rows v, columns do, values q, backwards     (state: sum do q^T)
//   dv: rows k, columns q, values do, backwards     (state: sum q do^T)
//
// where "backwards" masks s >= t, swaps the row factor e^{G[t]} with the
// column factor e^{G[C]-G[s]} and walks the chunks from the last.  So one
// kernel per data type serves the forward and all three gradients (`Form`).
// The gate's gradient follows from the rows of two of them: with
// a[t] = q[t].dq[t] and b[t] = k[t].dk[t],
//
//   dg[t] = sum_{u=t..e} (a[u] - b[u]) + <S[e], dS[e]>
//
// for any later token e of the sequence.  Taking e at most `restart` tokens
// away (both state matrices are stored there) keeps the differences short;
// one sum over a long sequence would lose the digits that the many terms
// share.  Both dots leave out the token's own term (s = t), which is the same
// in a and b: it does not depend on any gate, while all the rest shrinks with
// e^g, so at g = -8 a float32 a - b with it would keep two or three digits.
//
// Work is split over heads and over segments of `seg` tokens of the packed
// axis.  A segment that a sequence crosses needs the state that enters it: a
// first launch computes each segment's own contribution (state_only), a
// second one chains them, and the main launch starts every segment from its
// carry.  Chunks never span two sequences, so no value of one sequence, not
// even a NaN, meets another's.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/ascan.h"

namespace ascan {
namespace mscan {

// Tokens between stored states.  A float32 gate gradient carries the rounding
// of every row dot between them.  On the tensor cores (P and S in 16 bits) one
// chunk's stretch leaves 2.6e-6 of its norm at the median of 700 sizes, 5.0e-6
// at the 99th percentile and 6.0e-6 at most; 256 tokens 2.6e-6, 6.2e-6 and
// 9.8e-6, for 358 us instead of 385 at 8 x 2048 tokens x 12 heads of 128 x 128.
// Float32 arithmetic takes 256 tokens.  A 16-bit gradient needs no more than
// the longest stretch, whose stores of up to 64 KB a head weigh less.
constexpr int kRestart16 = 1024, kRestartPlain = 256, kRestartTc = 128;
inline int restart_of(bool tensor_cores, int gate_type) {
  return gate_type != ASCAN_F32 ? kRestart16 : (tensor_cores ? kRestartTc : kRestartPlain);
}
constexpr float kGateFloor = -200.f;  // e^-200 is 0 in float32; keeps -inf out of differences

struct Rows {  // [tokens, heads, dim] with unit stride along dim
  const void* p;
  long long st, sh;  // strides in elements
  int share;         // problem heads per head of this tensor
};

struct Form {
  Rows a, b, c;  // row, column and value operands
  Rows dot;      // optional: row dots of the output, without each token's own term, with this tensor
  int da, dc, rev;
  int fine;          // tensor cores: a float32 result depends on the state, so keep all bits of what enters it
  float sp, sr, sc;  // factors of the scores, of the rows and of the columns
  void* out;         // [BL, H, dc]
  int out_f32;
  float* rowdot;      // [2, H, BL]: sums over halves of the columns
  int dot_parts;      // how many of them the kernel wrote (set before the launch)
  const float* init;  // per sequence and head, element (i, j) at i*si + j*sj; may be null
  float* fin;
  long long si, sj;
  float* carry;  // [J, H, da*dc]: the state that leaves a segment
  float* dec;    // [J, H]: the decay over the segment's crossing piece
  float* snap;   // [slots, H, da*dc] or null
};

struct Problem {
  const void* cu;
  int cu64, J, H, gate_type;
  int restart;  // tokens between stored states, set before the launch
  long long N, BL, seg;
  Rows gate;  // [BL, heads, 1]
  uint32_t* err;
};

struct Launch {
  Problem p;
  Form f[3];
};

__device__ __forceinline__ long long cu_at(const Problem& p, long long i) {
  const long long v = p.cu64 ? static_cast<const long long*>(p.cu)[i]
                             : static_cast<long long>(static_cast<const int*>(p.cu)[i]);
  return v < 0 ? 0 : (v > p.BL ? p.BL : v);
}

// The first sequence whose end lies beyond token t (N if none does).
__device__ __forceinline__ long long first_beyond(const Problem& p, long long t) {
  long long lo = 0, hi = p.N;
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (cu_at(p, mid + 1) > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// The first sequence that starts at or after token t (N if none does).
__device__ __forceinline__ long long first_from(const Problem& p, long long t) {
  long long lo = 0, hi = p.N;
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (cu_at(p, mid) >= t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float load_any(const void* p, int type, long long i) {
  if (type == ASCAN_F32) return static_cast<const float*>(p)[i];
  if (type == ASCAN_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_any(void* p, int type, long long i, float x) {
  if (type == ASCAN_F32) static_cast<float*>(p)[i] = x;
  else if (type == ASCAN_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

// A log gate; -inf (the state is dropped) and all that is 0 after exp in
// float32 become one finite value, NaN stays NaN.
__device__ __forceinline__ float load_gate(const Problem& p, long long t, int h) {
  const float g = load_any(p.gate.p, p.gate_type, t * p.gate.st + (h / p.gate.share) * p.gate.sh);
  return g < kGateFloor ? kGateFloor : g;
}

// Slot of the state stored at token `at`: stored positions of one sequence
// are `restart` apart and at least as far from those of the next, so the
// quotient is unique.
__device__ __forceinline__ long long snap_slot(const Problem& p, long long at) { return at / p.restart; }

// A kernel's dynamic shared memory beyond 48 KB has to be allowed once on
// every device that runs it; `done` holds a bit for each.
template <typename K>
inline int allow_smem(K kernel, size_t bytes, std::atomic<unsigned long long>& done) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return ASCAN_EDEVICE;
  const unsigned long long bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return ASCAN_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != cudaSuccess)
    return ASCAN_ECUDA;
  done.fetch_or(bit, std::memory_order_release);
  return ASCAN_OK;
}

// The tensor-core kernel (ascan_mscan_tc.cu).
bool tc_usable(const Launch& l, int roles, int dtype);
int tc_dot_parts(const Form& f);
int tc_run(const Launch& l, int roles, bool state_only, cudaStream_t s);

}  // namespace mscan
}  // namespace ascan
