// What the attention kernels share: the reference of a row's exponentials, probabilities as matrix-core operands, and the
// parts that slices of a row's keys leave for the last of them.
#pragma once
#include <math.h>

#include "miq_common.h"

namespace miq {

// The reference of the exponentials is raised only when a score passes it by more than 2^4 (a probability, 2^11 at the
// reference, then stays below 2^15), so that the output is seldom rescaled (131000 positions 50 -> 47 us a replay); each
// row by its own scores alone, so that a token's bits do not depend on its neighbours' queries. The unit is as high as
// that and fp16's range allow: two fp16 numbers hold it to 2^-25, so that of 100000 keys that share 0.1 % beside one the sum
// is right to 4e-7 (5e-6 at 2^7; a slack of 2^8 takes the same time).
constexpr float kA4UnitLog2 = 11.f, kA4Slack = 4.f;

// the maximum over the four lanes c, c + 16, c + 32, c + 48
__device__ __forceinline__ float rows_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// 2^n of a row: q 2^n has its largest magnitude in [2^13, 2^14) (less below fp32's normal range); 1 for non-finite rows
__device__ __forceinline__ int row_shift(float mx) {
  const int e = (int)((__float_as_uint(mx) >> 23) & 255);
  return e == 255 ? 0 : 13 + 127 - max(e, 1);
}

// A row's reference: a score s (the matrix cores' sum) has the probability 2^((s - shift) back + neg), a fused product
// and sum. Scores below kA4Far units of log 2 have shift 0 and a whole reference, neg = kA4UnitLog2 - rint(the highest),
// which is exact, so that rescaling is by powers of two. Past it no fp32 number lies near enough to all scores: the
// highest is taken off in the matrix cores' units first, where it leaves an exact 0 for its own key. (A reference
// rounded in units of log 2 is off by its last place, 2^7 at 2^30, and takes the exponentials of every key to 0 or
// to infinity.)
constexpr float kA4Far = 4194304.f, kA4NoKey = 3.402823466e38f;  // 2^22; neg of a row that has met no key
struct Ref {
  float shift, neg;
};
// the exponent that the row's highest score (-inf: none) has now
__device__ __forceinline__ float ref_exponent(const Ref& r, float mx, float back) { return fmaf(mx - r.shift, back, r.neg); }
// Takes mx as the reference where the exponent is past the slack; returns what the row's sums are rescaled by.
__device__ __forceinline__ float ref_raise(Ref& r, float mx, float back) {
  if (!(ref_exponent(r, mx, back) > kA4UnitLog2 + kA4Slack)) return 1.f;
  const float top = mx * back;  // past fp32's range: NaN, as the difference of two such scores is
  const Ref n = fabsf(top) < kA4Far ? Ref{0.f, kA4UnitLog2 - rintf(top)} : Ref{mx, kA4UnitLog2 + (top - top)};
  const float f = __builtin_amdgcn_exp2f(fmaf(r.shift - n.shift, back, n.neg - r.neg));
  r = n;
  return f;
}
// the reference in units of log 2, -inf for none
__device__ __forceinline__ float ref_log2(const Ref& r, float back) {
  return r.neg == kA4NoKey ? -INFINITY : fmaf(r.shift, back, kA4UnitLog2 - r.neg);
}

// Parts of slices pass through the device-scope coherence point: stores and loads past the XCD's own L2.
__device__ __forceinline__ void put2(float* p, float a, float b) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get2(const float* p) {
  return __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the last of the `slices` that stored their parts (the counter is left zero).
__device__ __forceinline__ bool last_slice(int* ctr, int slices, int* last) {
  parts_stored();
  __syncthreads();
  if (threadIdx.x == 0) {
    *last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == slices - 1;
    if (*last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *last;
}
// 8 probabilities as matrix-core operands: the nearest fp16 number, and the one nearest to what that leaves (to 2^-25 at
// the least). Both to the nearest: towards zero, all small probabilities shrink alike beside a large one (of 16000 keys that
// share 1 % by a part in 6000). The sum of probabilities is taken of the operands, by the matrix cores.
__device__ __forceinline__ void split_p(const float* p, half8v* ph) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  const float minus = __uint_as_float(opaque(0xBF800000u));  // -1: a difference would take a conversion of hi of its own
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const half2v hi = __builtin_convertvector((float2v){p[2 * x], p[2 * x + 1]}, half2v);
    ph[0][2 * x] = hi.x;
    ph[0][2 * x + 1] = hi.y;
    ph[1][2 * x] = (_Float16)fmaf((float)hi.x, minus, p[2 * x]);
    ph[1][2 * x + 1] = (_Float16)fmaf((float)hi.y, minus, p[2 * x + 1]);
  }
}
__device__ __forceinline__ half8v ones() { return (half8v){1, 1, 1, 1, 1, 1, 1, 1}; }

}  // namespace miq
