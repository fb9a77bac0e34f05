// What the kernels of packed-sequence attention and of the bucketed relative position bias share.
#pragma once
#include "i2r_common.h"
#include "../../include/i2r_hip.h"
#include <float.h>
#include <algorithm>

#define PA_LOG2E 1.4426950408889634f
#define PA_MAX_BUCKETS 64
#define PA_MAX_DISTANCE 1024

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// position difference key - query without wrapping (positions are any int32): v_sub_i32 with the clamp bit
__device__ __forceinline__ int pa_apart(int pos_k, int pos_q) { return __builtin_elementwise_sub_sat(pos_k, pos_q); }

// entry of the (2 * max_distance + 1) distance tables that a position difference falls on
__device__ __forceinline__ int pa_entry(int apart, int max_distance) {
  return min(max(apart, -max_distance), max_distance) + max_distance;
}

// table value in log2 units.  A finite entry stays finite (the type's lowest value times log2(e) would be -inf, which
// hides a key); infinities and NaN pass.
__device__ __forceinline__ float pa_log2_units(float t) {
  float b = t * PA_LOG2E;
  return fabsf(t) <= FLT_MAX ? fminf(fmaxf(b, -FLT_MAX), FLT_MAX) : b;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
  for (int c = 0; c < (int)(sizeof(T) / 2); ++c) {
    vec w = *(const vec*)(p + c * (16 / sizeof(T)));
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) x[c * (16 / sizeof(T)) + i] = (float)w[i];
  }
}

// fp16 holds no probability below 6e-8 and few digits below 6e-5: there p and ds carry 2^12 in the backward, taken out at the
// end, and p 2^7 in the forward, where it may be 2^8 before the reference exponent moves (2^15 of the type's 2^16).  Each is
// then rounded by at most 2^-25 / 2^7 = 2^-32, and what many small ones are together is not lost.  (A ds of 16 and more leaves
// the type with its 2^12: those rows are done again pair by pair, in fp32, and off the matrix cores.)
template <typename T>
struct Lift {
  static constexpr float LOG2 = sizeof(T) == 2 && __is_same(T, f16_t) ? 12.0f : 0.0f;
  static constexpr float DOWN = LOG2 > 0.0f ? 1.0f / 4096.0f : 1.0f;
  static constexpr float FWD_LOG2 = __is_same(T, f16_t) ? 7.0f : 0.0f;
};
