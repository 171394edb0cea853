// ascan_mscan_common.cuh -- device parts that both matrix-scan kernels use;
// included after ascan_impl.cuh (each unit has its own error word).
#pragma once

#include "ascan_mscan.cuh"

namespace ascan {
namespace mscan {

// cu_seqlens as the scans check it; every other read of it is clamped.
__device__ __forceinline__ void check_cu(const Problem& p) {
  if (p.cu64) validate_cu(static_cast<const int64_t*>(p.cu), p.N, p.BL, p.err);
  else validate_cu(static_cast<const int32_t*>(p.cu), p.N, p.BL, p.err);
}

// What belongs to no chunk: rows outside all sequences come out zero, and
// empty sequences hand their state through.
template <typename T>
__device__ __forceinline__ void fill_outside(const Problem& p, const Form& f) {
  const int j = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, step = blockDim.x;
  const long long t0 = j * p.seg, t1 = min(t0 + p.seg, p.BL);
  if (j == 0 && h == 0 && blockIdx.z == 0) check_cu(p);
  const long long c0 = min(t1, cu_at(p, 0)), c1 = max(t0, cu_at(p, p.N));
  for (long long t = t0; t < t1; ++t) {
    if (t >= c0 && t < c1) {
      t = c1 - 1;
      continue;
    }
    for (int d = tid; d < f.dc; d += step) {
      const long long at = (t * p.H + h) * f.dc + d;
      if (f.out_f32) static_cast<float*>(f.out)[at] = 0.f;
      else static_cast<T*>(f.out)[at] = from_f<T>(0.f);
    }
  }
  if (f.fin && j == 0) {
    const long long mat = static_cast<long long>(f.da) * f.dc;
    bool empty = false;
    for (long long n = tid; n < p.N; n += step) empty |= cu_at(p, n + 1) <= cu_at(p, n);
    if (__syncthreads_or(empty))
      for (long long n = 0; n < p.N; ++n)
        if (cu_at(p, n + 1) <= cu_at(p, n))
          for (long long e = tid; e < mat; e += step)
            f.fin[(n * p.H + h) * mat + e] = f.init ? f.init[(n * p.H + h) * mat + e] : 0.f;
  }
}

}  // namespace mscan
}  // namespace ascan
