// What the token operators (token_norm.hip, matmul_fp8.hip, cross_attn.hip) share: their value types, rows read and written in chunks of
// eight, and the step into 8 bits (OCP e4m3, largest value 448).
#pragma once
#include "rtp_common.h"

typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;

#define RTP_FP8_MAX 448.0f
// a launch counts its threads in 32 bits
static inline bool rtp_launchable(long blocks, long threads) { return blocks * threads < (1L << 32); }

#define RTP_FP8_AMAX_FLOOR 0x1p-100f   // keeps 448 / amax finite; a block of zeros gets the floor's scale

// Eight consecutive values at any address (rows of odd length or odd stride start anywhere): one unaligned 16- or 32-byte access,
// which global memory takes at every alignment of the element; element by element only where the row ends inside the chunk.
template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, int n) {
  typedef T tv8 __attribute__((ext_vector_type(8)));
  if (n >= 8) {
    tv8 r;
    __builtin_memcpy(&r, p, sizeof(r));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.f;
  }
}
// as load8, marked to leave the caches first
template <typename T>
__device__ __forceinline__ void load8_once(float (&v)[8], const T* p, int n) {
  typedef T tv8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  if (n >= 8) {
    const tv8 r = __builtin_nontemporal_load((const tv8*)p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
  } else {
    load8(v, p, n);
  }
}
// load8 or load8_once, by a condition that all lanes share
template <typename T>
__device__ __forceinline__ void load8_if(bool once, float (&v)[8], const T* p, int n) {
  if (once) load8_once(v, p, n);
  else load8(v, p, n);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n) {
  typedef T tv8 __attribute__((ext_vector_type(8)));
  if (n >= 8) {
    tv8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)v[j];
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)v[j];
  }
}

// Outputs of more than the last-level cache drive each other out of it before the next pass reads them: they are stored past it.
#define RTP_FAR_BYTES (256L << 20)
// as store8, marked to leave the caches first
template <typename T>
__device__ __forceinline__ void store8_far(T* p, const float (&v)[8], int n) {
  typedef T tv8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  if (n >= 8) {
    tv8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)v[j];
    __builtin_nontemporal_store(r, (tv8*)p);
  } else {
    store8(p, v, n);
  }
}

// eight values times `up` -> eight e4m3 bytes, round to nearest even (|v * up| <= 448 up to one fp32 rounding: never out of range)
__device__ __forceinline__ i32x2 to_fp8x8(const float (&v)[8], float up) {
  i32x2 r = {0, 0};
  r[0] = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * up, v[1] * up, r[0], false);
  r[0] = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * up, v[3] * up, r[0], true);
  r[1] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * up, v[5] * up, r[1], false);
  r[1] = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * up, v[7] * up, r[1], true);
  return r;
}

// largest magnitude of eight values; a NaN does not count (it stays where it is)
__device__ __forceinline__ float amax8(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
  return m;
}
