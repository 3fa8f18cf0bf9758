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

// Eight consecutive values at any address (rows of odd length or odd stride start anywhere): one unaligned 16- or 32-byte access, which global memory
// takes at every alignment of the element.
template <typename T> using vec8 = T __attribute__((ext_vector_type(8), aligned(sizeof(T))));
template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p) {
  const vec8<T> r = *(const vec8<T>*)p;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
}
// Rows in chunks of eight columns, by what their length n allows: a multiple of 8, any from 8 on, fewer.
enum RowKind { ROW_WHOLE, ROW_RAGGED, ROW_SHORT };
// Columns c .. c + 7, zeros behind the row's end, in two steps: all loads of a row first, then their values.  A ragged row's last chunk is read as the
// row's last eight columns and moved into place in registers: element by element it is another trip to memory for the whole wave (bf16, 20480 x 1023:
// norm 47 us, so 31, its gradients 72 and 40; 8192 x 4094 quantised in blocks of 128 x 128: 41 and 21).  `once`: marked to leave the caches first.
template <RowKind KIND, typename T>
__device__ __forceinline__ vec8<T> fetch8(const T* row, int c, int n, bool once = false) {
  vec8<T> r;
  if constexpr (KIND == ROW_SHORT) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = c + j < n ? row[c + j] : (T)0.f;
  } else {
    const vec8<T>* p = (const vec8<T>*)(row + (c + 8 > n ? n - 8 : c));
    r = once ? __builtin_nontemporal_load(p) : *p;
  }
  return r;
}
template <RowKind KIND, typename T>
__device__ __forceinline__ void settle8(float (&v)[8], const vec8<T>& r, int c, int n) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
  if constexpr (KIND != ROW_SHORT) {
    const int over = c + 8 > n ? c + 8 - n : 0;
    if (KIND == ROW_RAGGED && __any(over)) {
#pragma unroll
      for (int s = 1; s < 8; s *= 2)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = over & s ? (j + s < 8 ? v[j + s] : 0.f) : v[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = over > 7 ? 0.f : v[j];
  }
}
// eight values, or the first n of them
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n) {
  if (n >= 8) {
    vec8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)v[j];
    *(vec8<T>*)p = r;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)v[j];
  }
}
// Outputs of more than the last-level cache drive each other out of it before the next pass reads them: they are stored past it.
#define RTP_FAR_BYTES (256L << 20)
// eight values, `far`: marked to leave the caches first
template <typename T>
__device__ __forceinline__ void put8(T* p, const float (&v)[8], bool far) {
  vec8<T> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)v[j];
  if (far) __builtin_nontemporal_store(r, (vec8<T>*)p);
  else *(vec8<T>*)p = r;
}
// columns c .. c + 7 of a row of n
template <RowKind KIND, typename T>
__device__ __forceinline__ void put_row8(T* row, const float (&v)[8], int c, int n, bool far = false) {
  if (KIND != ROW_SHORT && c + 8 <= n) {
    put8(row + c, v, far);
  } else if constexpr (KIND != ROW_WHOLE) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < n) row[c + j] = (T)v[j];
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
