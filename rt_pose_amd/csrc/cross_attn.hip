// Cross attention to an encoder's states of another length: o = softmax(scale * q k^T over the keys that count) v, with grouped heads, its
// gradients, and its form for a few query rows (single tokens).
//
//   forward     s = scale q k^T;  p = exp(s - max);  o = p v / sum p          row statistic kept: L = max + log2(sum) (base 2)
//   backward    p = exp2(s - L);  dp = do v^T;  ds = p (dp - delta), delta = sum_d do o;  dq = scale ds k;  dk = scale ds^T q;  dv = p^T do
//
// Keys are masked for a whole batch entry (its length, or one truth value per key), as an encoder's padding is; so a masked key is neither
// read nor multiplied: it is staged as zeros, whatever stands in memory, and its gradients are zeros.  A row without keys gives zeros.
//
// All heads of a group read the same k and v: the kernels work on ROWS r = token * group + head-in-group of one (batch, kv head), R = sq * group.
//
// Products are v_mfma_f32_32x32x16 on tiles of 32 rows x 32 keys.  The forward pass forms s^T = k q^T: a lane then holds 16 keys of ONE row,
// the row's maximum and sum are its own registers plus the other half wave's, and p^T is already laid out as the second operand of
// o^T = v^T p^T once the keys of a step are taken in the order the accumulator holds them -- v is read from LDS transposed
// (ds_read_b64_tr_b16) in that same order.  p never leaves the registers.  dq works the same way; dk / dv with rows and keys exchanged.
// Operands of 16 bits, everything else fp32: p and ds are rounded once to 16 bits for their second product (2^-9 of each, averaged over the
// keys), the sums they enter are fp32.
#include <type_traits>

#include "rtp_prof.h"
#include "token_common.h"

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4_xa;
typedef __attribute__((address_space(3))) void lds_void_xa;
typedef __attribute__((address_space(1))) void glb_void_xa;

__device__ __attribute__((aligned(16))) bf16_t g_zero_line_xa[8];   // what masked rows and columns behind the head's width are staged from

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <typename T> struct Vec8;
template <> struct Vec8<bf16_t> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };

struct XaParams {
  const void *q, *k, *v, *d_o;
  long q_bs, q_ss, q_hs, k_bs, k_ss, k_hs, v_bs, v_ss, v_hs, o_bs, o_ss, o_hs;   // o_*: of d_o
  const unsigned* bits;      // [b][words]: one bit per key, from key_mask and key_lens; null: key_lens alone
  const int* lens;           // [b] or null
  int b, sq, sk, hq, hkv, d, grp, rows;
  unsigned grp_magic;        // ceil(2^32 / grp): r / grp = mulhi(r, magic) for r * grp < 2^32
  int words;
  int tiles, units, nsplit;  // workgroups = tiles x units (batch x kv head x split)
  float scale, scale_log2;
  void *o, *o_lo, *dq, *dk, *dv;
  float *lse, *delta, *part, *part_lse;
  const float* lse_in;
};

// Workgroup -> (tile, unit): all tiles of a unit run on one XCD (workgroups go round the 8 XCDs), so that a unit's k and v stay in one L2.
__device__ __forceinline__ bool xa_place(const XaParams& p, int& tile, int& bh, int& split) {
  const unsigned j = blockIdx.x >> 3, unit = (j / (unsigned)p.tiles) * 8 + (blockIdx.x & 7);
  tile = j % (unsigned)p.tiles;
  if (unit >= (unsigned)p.units) return false;
  bh = unit / (unsigned)p.nsplit;
  split = unit % (unsigned)p.nsplit;
  return true;
}

__device__ __forceinline__ int xa_len(const XaParams& p, int b) {
  if (!p.lens) return p.sk;
  const int n = p.lens[b];
  return n < 0 ? 0 : n > p.sk ? p.sk : n;
}
// bits of the 32 keys from key0 on
__device__ __forceinline__ unsigned xa_word(const XaParams& p, int b, int len, int key0) {
  if (p.bits) return p.bits[(long)b * p.words + (key0 >> 5)];
  const int n = len - key0;
  return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}
__device__ __forceinline__ long xa_row_off(const XaParams& p, int r, long ss, long hs) {
  const unsigned s = p.grp == 1 ? (unsigned)r : __umulhi((unsigned)r, p.grp_magic);
  return (long)s * ss + (long)(r - (int)s * p.grp) * hs;
}

// ---- LDS images: rows of CH 16-byte chunks, chunk c of row r at slot c ^ swz(r), so that rows read at one chunk lie in different banks
template <int DT> struct XaImg {
  static constexpr int CH = DT == 1 ? 4 : DT == 2 ? 8 : 16, PITCH = CH * 16;   // bytes per row
  __device__ static __forceinline__ int swz(int r) { return CH == 4 ? (r >> 2) & 3 : CH == 8 ? (r >> 1) & 7 : r & 15; }
};
// Per-lane byte offsets inside an image; rows + 16 and + 32 are plain additions (swz has period 16).
template <int DT> struct XaAddr {
  int row[2 * DT];        // 32 rows as instruction rows, 16 columns of the step: row l % 32, chunk 2 step + l / 32
  int tr[DT][2];          // transposed: columns 32 dt + l % 32, rows 4 (l / 32) + {0..3} and + 8
  __device__ __forceinline__ XaAddr(int lane) {
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int s = 0; s < 2 * DT; ++s) row[s] = r * XaImg<DT>::PITCH + (((2 * s + h) ^ XaImg<DT>::swz(r)) << 4);
    const int a = (lane & 15) >> 2, pp = lane & 3, ds = (lane >> 4) & 1;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = 4 * h + a + 8 * e, c = 4 * t + 2 * ds + (pp >> 1);
        tr[t][e] = k * XaImg<DT>::PITCH + ((c ^ XaImg<DT>::swz(k)) << 4) + (pp & 1) * 8;
      }
  }
};
template <typename V>
__device__ __forceinline__ V xa_frag(const uint8_t* img, int off) { return *(const V*)(img + off); }
template <typename V>
__device__ __forceinline__ V xa_frag_tr(const uint8_t* img, int lo, int hi) {
  const s16x4 l = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_xa*)(img + lo));
  const s16x4 h = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_xa*)(img + hi));
  const s16x8 r = {l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
  return __builtin_bit_cast(V, r);
}

// Stage ROWS rows of `src` (row r at src + off(r), valid where ok(r)) by LDS-DMA: 256 threads, 16 B each and step, no registers for the data.
template <int DT, int ROWS, typename T, typename Off, typename Ok>
__device__ __forceinline__ void xa_stage(uint8_t* img, const T* src, int d, Off off, Ok ok) {
  constexpr int CH = XaImg<DT>::CH, STEPS = ROWS * CH / 256;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int item = i * 256 + threadIdx.x, r = item / CH, c = (item % CH) ^ XaImg<DT>::swz(r);
    const void* a = ok(r) && c * 8 < d ? (const void*)(src + off(r) + c * 8) : (const void*)g_zero_line_xa;
    __builtin_amdgcn_global_load_lds((const glb_void_xa*)a, (lds_void_xa*)(img + i * 4096 + wave * 1024), 16, 0, 0);
  }
}

__device__ __forceinline__ float xa_halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xa_halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// a row operand held in registers: columns 16 s + 8 h .. + 7 of one row; zeros behind the head's width and for rows that are none
template <int DT, typename T>
__device__ __forceinline__ void xa_load_row(typename Vec8<T>::type (&f)[2 * DT], const T* row, bool ok, int d, int h) {
#pragma unroll
  for (int s = 0; s < 2 * DT; ++s) {
    const int c = 16 * s + 8 * h;
    const T* a = ok && c < d ? row + c : (const T*)g_zero_line_xa;
    f[s] = *(const typename Vec8<T>::type*)a;
  }
}

#define XA_M0 (-3.402823466e38f)
#define XA_SLACK 8.0f   // the running maximum moves only when it is exceeded by 2^8: p stays below 2^8, and most tiles rescale nothing

// ------------------------------------------------------------------------------------------------ forward
// Four waves: 4 / KW groups of 32 rows, and KW waves that share rows and split each tile of keys (few rows: the keys are the work).
// Tiles of BK keys go through two LDS buffers, the next one on its way while this one is used: one barrier a tile.
template <int KW> struct XaKeys { static constexpr int BK = KW == 4 ? 128 : 64, SUB = BK / 32 / KW; };

template <typename T, int DT, int KW>
__global__ __launch_bounds__(256, 2) void xattn_fwd_kernel(XaParams p) {
  typedef typename Vec8<T>::type V;
  constexpr int BK = XaKeys<KW>::BK, SUB = XaKeys<KW>::SUB, IMG = BK * XaImg<DT>::PITCH;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int tile, bh, split;
  if (!xa_place(p, tile, bh, split)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = bh / p.hkv, hk = bh % p.hkv, h = lane >> 5;
  const int kw = wave % KW, r0 = tile * (128 / KW) + (wave / KW) * 32, r = r0 + (lane & 31);
  const int len = xa_len(p, b), nt = (len + BK - 1) / BK;
  const int t0 = (int)((long)nt * split / p.nsplit), t1 = (int)((long)nt * (split + 1) / p.nsplit);
  const T* kp = (const T*)p.k + (long)b * p.k_bs + (long)hk * p.k_hs;
  const T* vp = (const T*)p.v + (long)b * p.v_bs + (long)hk * p.v_hs;
  const XaAddr<DT> ad(lane);

  V qf[2 * DT];
  xa_load_row<DT, T>(qf, (const T*)p.q + (long)b * p.q_bs + (long)(hk * p.grp) * p.q_hs + (r < p.rows ? xa_row_off(p, r, p.q_ss, p.q_hs) : 0), r < p.rows, p.d, h);
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = XA_M0, l = 0.f;

  auto stage = [&](int t, int buf) {
    unsigned w[BK / 32];
#pragma unroll
    for (int i = 0; i < BK / 32; ++i) w[i] = xa_word(p, b, len, t * BK + i * 32);
    auto ok = [&](int row) {
      unsigned x = w[0];
#pragma unroll
      for (int i = 1; i < BK / 32; ++i) x = (row >> 5) == i ? w[i] : x;
      return ((x >> (row & 31)) & 1u) != 0;
    };
    xa_stage<DT, BK>(lds + buf * 2 * IMG, kp + (long)t * BK * p.k_ss, p.d, [&](int row) { return (long)row * p.k_ss; }, ok);
    xa_stage<DT, BK>(lds + buf * 2 * IMG + IMG, vp + (long)t * BK * p.v_ss, p.d, [&](int row) { return (long)row * p.v_ss; }, ok);
  };
  auto compute = [&](int t, int buf) {
    const uint8_t *ki = lds + buf * 2 * IMG, *vi = ki + IMG;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const int sub = kw * SUB + u;
      const unsigned w = xa_word(p, b, len, t * BK + sub * 32);
      if (w == 0) continue;
      f32x16 s;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
      for (int st = 0; st < 2 * DT; ++st) s = mfma32(xa_frag<V>(ki + sub * 32 * XaImg<DT>::PITCH, ad.row[st]), qf[st], s);
      if (w != ~0u) {
        const unsigned wl = w >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = (wl >> (8 * (i / 4) + i % 4)) & 1u ? s[i] : -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      mx = xa_halves_max(mx) * p.scale_log2;
      if (__any(mx > m + XA_SLACK)) {
        const float mn = fmaxf(m, mx), a = exp2f(m - mn);
        m = mn;
        l *= a;
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[t2][i] *= a;
      }
      V pb[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[i] * p.scale_log2 - m);
        l += e;
        pb[i >> 3][i & 7] = (T)e;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2)
          o[t2] = mfma32(xa_frag_tr<V>(vi + (sub * 32 + c * 16) * XaImg<DT>::PITCH, ad.tr[t2][0], ad.tr[t2][1]), pb[c], o[t2]);
    }
  };
  if (t0 < t1) {
    stage(t0, 0);
    for (int t = t0; t < t1; ++t) {
      __syncthreads();
      if (t + 1 < t1) stage(t + 1, (t + 1 - t0) & 1);
      if (r0 < p.rows) compute(t, (t - t0) & 1);
    }
  }
  l = xa_halves_sum(l);
  if constexpr (KW > 1) {       // waves of one row group meet in LDS, added in wave order
    __syncthreads();
    float* x = (float*)lds;
    constexpr int SLOT = (DT * 16 + 2) * 64;
    if (kw > 0) {
      float* y = x + ((wave / KW) * (KW - 1) + kw - 1) * SLOT + lane;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) y[(t * 16 + i) * 64] = o[t][i];
      y[DT * 16 * 64] = m;
      y[(DT * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int k = 1; k < KW; ++k) {
      const float* y = x + ((wave / KW) * (KW - 1) + k - 1) * SLOT + lane;
      const float m2 = y[DT * 16 * 64], l2 = y[(DT * 16 + 1) * 64], mn = fmaxf(m, m2), a = exp2f(m - mn), a2 = exp2f(m2 - mn);
      m = mn;
      l = l * a + l2 * a2;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = o[t][i] * a + y[(t * 16 + i) * 64] * a2;
    }
  }
  if (r >= p.rows) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float L = l == 0.f ? -INFINITY : m + log2f(l);
  const long row = (long)bh * p.rows + r;
  if (p.nsplit > 1) {
    const long prow = (long)split * p.b * p.hkv * p.rows + row;
    if (h == 0) p.part_lse[prow] = L;
    float* po = p.part + prow * p.d;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int c = 32 * t + 2 * i + 4 * h;
        if (c < p.d) *(f32x4*)(po + c) = f32x4{o[t][i] * inv, o[t][i + 1] * inv, o[t][i + 2] * inv, o[t][i + 3] * inv};
      }
  } else {
    if (p.lse && h == 0) p.lse[row] = l == 0.f ? INFINITY : L;
    const int s = r / p.grp, g = r % p.grp;
    const long oo = (((long)b * p.sq + s) * p.hq + hk * p.grp + g) * p.d;
    typedef T tv4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int c = 32 * t + 2 * i + 4 * h;
        if (c < p.d) {
          tv4 hi, lo;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = o[t][i + j] * inv;
            hi[j] = (T)x;
            lo[j] = (T)(x - (float)hi[j]);
          }
          *(tv4*)((T*)p.o + oo + c) = hi;
          if (p.o_lo) *(tv4*)((T*)p.o_lo + oo + c) = lo;
        }
      }
  }
}

// o of a row = sum over splits of 2^(L_split - L) o_split.  16 lanes a row, 8 columns each.
template <typename T>
__global__ __launch_bounds__(256) void xattn_join_kernel(XaParams p) {
  const long rows = (long)p.b * p.hkv * p.rows, row = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int c = (threadIdx.x & 15) * 8;
  if (row >= rows) return;
  float mx = -INFINITY;
  for (int s = 0; s < p.nsplit; ++s) {
    const float x = p.part_lse[s * rows + row];
    mx = x > mx || x != x ? x : mx;      // a NaN stays
  }
  float sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (mx > -INFINITY || mx != mx)
    for (int s = 0; s < p.nsplit; ++s) {
      const float w = exp2f(p.part_lse[s * rows + row] - mx);
      sum += w;
      if (c < p.d) {
        float v[8];
        load8(v, p.part + (s * rows + row) * p.d + c, 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += v[j] * w;
      }
    }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (p.lse && (threadIdx.x & 15) == 0) p.lse[row] = sum == 0.f ? INFINITY : mx + log2f(sum);
  if (c >= p.d) return;
  const int bh = (int)(row / p.rows), r = (int)(row % p.rows), s = r / p.grp, g = r % p.grp;
  const long oo = (((long)(bh / p.hkv) * p.sq + s) * p.hq + (bh % p.hkv) * p.grp + g) * p.d + c;
  float lo[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    acc[j] *= inv;
    lo[j] = acc[j] - (float)(T)acc[j];
  }
  store8((T*)p.o + oo, acc, 8);
  if (p.o_lo) store8((T*)p.o_lo + oo, lo, 8);
}

// ------------------------------------------------------------------------------------------------ masks
// one bit per key: 64 keys a wave (two words)
__global__ __launch_bounds__(256) void xattn_bits_kernel(const uint8_t* mask, long m_bs, long m_ss, const int* lens, unsigned* bits, int sk, int words) {
  const unsigned per = ((unsigned)words + 7) / 8;
  const int key = (blockIdx.x % per) * 256 + threadIdx.x, b = blockIdx.x / per;
  const int len = lens ? lens[b] : sk;
  const bool on = key < sk && key < len && mask[(long)b * m_bs + (long)key * m_ss] != 0;
  const unsigned long long w = __ballot(on);
  const int at = key >> 5;
  if ((threadIdx.x & 31) == 0 && at < words) bits[(long)b * words + at] = (threadIdx.x & 32) ? (unsigned)(w >> 32) : (unsigned)w;
}

// ------------------------------------------------------------------------------------------------ backward: delta
// delta of a row = sum_d do * o, from o as it was before its rounding (o + what the rounding left over): with few keys the difference
// dp - delta cancels, and o's rounding alone would be most of it.  16 lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void xattn_delta_kernel(XaParams p) {
  const long rows = (long)p.b * p.hkv * p.rows, row = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int c = (threadIdx.x & 15) * 8;
  float t = 0.f;
  if (row < rows && c < p.d) {
    const int bh = (int)(row / p.rows), r = (int)(row % p.rows), s = r / p.grp, g = r % p.grp, b = bh / p.hkv, hq = (bh % p.hkv) * p.grp + g;
    const long oo = (((long)b * p.sq + s) * p.hq + hq) * p.d + c;
    float hi[8], lo[8], d[8];
    load8(hi, (const T*)p.o + oo, 8);
    load8(lo, (const T*)p.o_lo + oo, 8);
    load8(d, (const T*)p.d_o + (long)b * p.o_bs + (long)s * p.o_ss + (long)hq * p.o_hs + c, 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) t += (hi[j] + lo[j]) * d[j];
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if (row < rows && (threadIdx.x & 15) == 0) p.delta[row] = t;
}

// ------------------------------------------------------------------------------------------------ backward: dq
// the forward kernel's shape: s^T and dp^T with a lane per row, dq^T = k^T ds^T, k read from LDS both ways
template <typename T, int DT, int KW>
__global__ __launch_bounds__(256, (DT > 2 ? 1 : 2)) void xattn_dq_kernel(XaParams p) {
  typedef typename Vec8<T>::type V;
  constexpr int BK = XaKeys<KW>::BK, SUB = XaKeys<KW>::SUB, IMG = BK * XaImg<DT>::PITCH;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int tile, bh, split;
  if (!xa_place(p, tile, bh, split)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = bh / p.hkv, hk = bh % p.hkv, h = lane >> 5;
  const int kw = wave % KW, r0 = tile * (128 / KW) + (wave / KW) * 32, r = r0 + (lane & 31);
  const bool rok = r < p.rows;
  const int len = xa_len(p, b), nt = (len + BK - 1) / BK;
  const int t0 = (int)((long)nt * split / p.nsplit), t1 = (int)((long)nt * (split + 1) / p.nsplit);
  const T* kp = (const T*)p.k + (long)b * p.k_bs + (long)hk * p.k_hs;
  const T* vp = (const T*)p.v + (long)b * p.v_bs + (long)hk * p.v_hs;
  const XaAddr<DT> ad(lane);
  const long row = (long)bh * p.rows + r;
  V qf[2 * DT], df[2 * DT];
  xa_load_row<DT, T>(qf, (const T*)p.q + (long)b * p.q_bs + (long)(hk * p.grp) * p.q_hs + (rok ? xa_row_off(p, r, p.q_ss, p.q_hs) : 0), rok, p.d, h);
  xa_load_row<DT, T>(df, (const T*)p.d_o + (long)b * p.o_bs + (long)(hk * p.grp) * p.o_hs + (rok ? xa_row_off(p, r, p.o_ss, p.o_hs) : 0), rok, p.d, h);
  const float L = rok ? p.lse_in[row] : INFINITY, delta = rok ? p.delta[row] : 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;

  auto stage = [&](int t, int buf) {
    unsigned w[BK / 32];
#pragma unroll
    for (int i = 0; i < BK / 32; ++i) w[i] = xa_word(p, b, len, t * BK + i * 32);
    auto ok = [&](int row) {
      unsigned x = w[0];
#pragma unroll
      for (int i = 1; i < BK / 32; ++i) x = (row >> 5) == i ? w[i] : x;
      return ((x >> (row & 31)) & 1u) != 0;
    };
    xa_stage<DT, BK>(lds + buf * 2 * IMG, kp + (long)t * BK * p.k_ss, p.d, [&](int row) { return (long)row * p.k_ss; }, ok);
    xa_stage<DT, BK>(lds + buf * 2 * IMG + IMG, vp + (long)t * BK * p.v_ss, p.d, [&](int row) { return (long)row * p.v_ss; }, ok);
  };
  auto compute = [&](int t, int buf) {
    const uint8_t *ki = lds + buf * 2 * IMG, *vi = ki + IMG;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const int sub = kw * SUB + u;
      const unsigned w = xa_word(p, b, len, t * BK + sub * 32);
      if (w == 0) continue;
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
#pragma unroll
      for (int st = 0; st < 2 * DT; ++st) {
        s = mfma32(xa_frag<V>(ki + sub * 32 * XaImg<DT>::PITCH, ad.row[st]), qf[st], s);
        dp = mfma32(xa_frag<V>(vi + sub * 32 * XaImg<DT>::PITCH, ad.row[st]), df[st], dp);
      }
      if (w != ~0u) {
        const unsigned wl = w >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = (wl >> (8 * (i / 4) + i % 4)) & 1u ? s[i] : -INFINITY;
      }
      V ds[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i >> 3][i & 7] = (T)(__builtin_amdgcn_exp2f(s[i] * p.scale_log2 - L) * (dp[i] - delta));
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2)
          acc[t2] = mfma32(xa_frag_tr<V>(ki + (sub * 32 + c * 16) * XaImg<DT>::PITCH, ad.tr[t2][0], ad.tr[t2][1]), ds[c], acc[t2]);
    }
  };
  if (t0 < t1) {
    stage(t0, 0);
    for (int t = t0; t < t1; ++t) {
      __syncthreads();
      if (t + 1 < t1) stage(t + 1, (t + 1 - t0) & 1);
      if (r0 < p.rows) compute(t, (t - t0) & 1);
    }
  }
  if constexpr (KW > 1) {
    __syncthreads();
    float* x = (float*)lds;
    constexpr int SLOT = DT * 16 * 64;
    if (kw > 0) {
      float* y = x + ((wave / KW) * (KW - 1) + kw - 1) * SLOT + lane;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) y[(t * 16 + i) * 64] = acc[t][i];
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int k = 1; k < KW; ++k) {
      const float* y = x + ((wave / KW) * (KW - 1) + k - 1) * SLOT + lane;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] += y[(t * 16 + i) * 64];
    }
  }
  if (!rok) return;
  typedef T tv4 __attribute__((ext_vector_type(4)));
  const int s = r / p.grp, g = r % p.grp;
  const long oo = (((long)b * p.sq + s) * p.hq + hk * p.grp + g) * p.d;
  float* po = p.part + ((long)split * p.b * p.hkv * p.rows + row) * p.d;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int c = 32 * t + 2 * i + 4 * h;
      if (c < p.d) {
        const f32x4 v = {acc[t][i] * p.scale, acc[t][i + 1] * p.scale, acc[t][i + 2] * p.scale, acc[t][i + 3] * p.scale};
        if (p.nsplit > 1) {
          *(f32x4*)(po + c) = v;
        } else {
          const tv4 z = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
          *(tv4*)((T*)p.dq + oo + c) = z;
        }
      }
    }
}

// dq of a row = sum over splits, in their order
template <typename T>
__global__ __launch_bounds__(256) void xattn_dq_join_kernel(XaParams p) {
  const long rows = (long)p.b * p.hkv * p.rows, row = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int c = (threadIdx.x & 15) * 8;
  if (row >= rows || c >= p.d) return;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8];
  for (int s = 0; s < p.nsplit; ++s) {
    load8(v, p.part + (s * rows + row) * p.d + c, 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += v[j];
  }
  const int bh = (int)(row / p.rows), r = (int)(row % p.rows), s = r / p.grp, g = r % p.grp;
  store8((T*)p.dq + (((long)(bh / p.hkv) * p.sq + s) * p.hq + (bh % p.hkv) * p.grp + g) * p.d + c, acc, 8);
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv
// Each wave keeps 32 keys (k, v as second operands in registers, dk^T and dv^T as accumulators) and walks the rows: s = q k^T and
// dp = do v^T with a lane per key, then dv^T += do^T p and dk^T += q^T ds with q and do read from LDS both ways.  A lane's key touches its own
// column of the products alone, so a masked key needs nothing inside the loop: zeros are written for it at the end.
template <typename T, int DT>
__global__ __launch_bounds__(256, (DT > 2 ? 1 : 2)) void xattn_dkv_kernel(XaParams p) {
  typedef typename Vec8<T>::type V;
  constexpr int BR = 64, IMG = BR * XaImg<DT>::PITCH, BUF = 2 * IMG + 2 * BR * 4;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int tile, bh, split;
  if (!xa_place(p, tile, bh, split)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = bh / p.hkv, hk = bh % p.hkv, h = lane >> 5;
  const int key0 = tile * 128 + wave * 32, key = key0 + (lane & 31);
  const int len = xa_len(p, b), nt = (p.rows + BR - 1) / BR;
  unsigned any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= tile * 128 + i * 32 < p.sk ? xa_word(p, b, len, tile * 128 + i * 32) : 0u;
  const unsigned w = key0 < p.sk ? xa_word(p, b, len, key0) : 0u;
  const bool kok = (w >> (lane & 31)) & 1u;
  const int t0 = (int)((long)nt * split / p.nsplit), t1 = any ? (int)((long)nt * (split + 1) / p.nsplit) : t0;
  const XaAddr<DT> ad(lane);
  V kf[2 * DT], vf[2 * DT];
  xa_load_row<DT, T>(kf, (const T*)p.k + (long)b * p.k_bs + (long)hk * p.k_hs + (kok ? (long)key * p.k_ss : 0), kok, p.d, h);
  xa_load_row<DT, T>(vf, (const T*)p.v + (long)b * p.v_bs + (long)hk * p.v_hs + (kok ? (long)key * p.v_ss : 0), kok, p.d, h);
  const T* qp = (const T*)p.q + (long)b * p.q_bs + (long)(hk * p.grp) * p.q_hs;
  const T* dp_ = (const T*)p.d_o + (long)b * p.o_bs + (long)(hk * p.grp) * p.o_hs;
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[t][i] = dv[t][i] = 0.f;

  auto stage = [&](int t, int buf) {
    uint8_t* at = lds + buf * BUF;
    auto ok = [&](int row) { return t * BR + row < p.rows; };
    xa_stage<DT, BR>(at, qp, p.d, [&](int row) { return xa_row_off(p, t * BR + row, p.q_ss, p.q_hs); }, ok);
    xa_stage<DT, BR>(at + IMG, dp_, p.d, [&](int row) { return xa_row_off(p, t * BR + row, p.o_ss, p.o_hs); }, ok);
    if (threadIdx.x < 2 * BR) {      // L and delta of the rows; rows that are none get p = 0
      const int row = t * BR + (threadIdx.x & (BR - 1));
      const bool first = threadIdx.x < BR;
      float x = first ? INFINITY : 0.f;
      if (row < p.rows) x = (first ? p.lse_in : p.delta)[(long)bh * p.rows + row];
      ((float*)(at + 2 * IMG))[threadIdx.x] = x;
    }
  };
  auto compute = [&](int t, int buf) {
    const uint8_t *qi = lds + buf * BUF, *di = qi + IMG;
    const float* st = (const float*)(qi + 2 * IMG);
#pragma unroll
    for (int u = 0; u < BR / 32; ++u) {
      if (t * BR + u * 32 >= p.rows) continue;
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
#pragma unroll
      for (int e = 0; e < 2 * DT; ++e) {
        s = mfma32(xa_frag<V>(qi + u * 32 * XaImg<DT>::PITCH, ad.row[e]), kf[e], s);
        dp = mfma32(xa_frag<V>(di + u * 32 * XaImg<DT>::PITCH, ad.row[e]), vf[e], dp);
      }
      V pb[2], sb[2];
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 L = *(const f32x4*)(st + u * 32 + 2 * i + 4 * h), dl = *(const f32x4*)(st + BR + u * 32 + 2 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = __builtin_amdgcn_exp2f(s[i + j] * p.scale_log2 - L[j]);
          pb[(i + j) >> 3][(i + j) & 7] = (T)e;
          sb[(i + j) >> 3][(i + j) & 7] = (T)(e * (dp[i + j] - dl[j]));
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
          const int off = (u * 32 + c * 16) * XaImg<DT>::PITCH;
          dv[t2] = mfma32(xa_frag_tr<V>(di + off, ad.tr[t2][0], ad.tr[t2][1]), pb[c], dv[t2]);
          dk[t2] = mfma32(xa_frag_tr<V>(qi + off, ad.tr[t2][0], ad.tr[t2][1]), sb[c], dk[t2]);
        }
    }
  };
  if (t0 < t1) {
    stage(t0, 0);
    for (int t = t0; t < t1; ++t) {
      __syncthreads();
      if (t + 1 < t1) stage(t + 1, (t + 1 - t0) & 1);
      if (w) compute(t, (t - t0) & 1);
    }
  }
  if (key >= p.sk) return;
  typedef T tv4 __attribute__((ext_vector_type(4)));
  const long oo = (((long)b * p.sk + key) * p.hkv + hk) * p.d;
  const long all = (long)p.b * p.sk * p.hkv * p.d;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int c = 32 * t + 2 * i + 4 * h;
      if (c < p.d) {
        f32x4 x, y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = kok ? dk[t][i + j] * p.scale : 0.f;
          y[j] = kok ? dv[t][i + j] : 0.f;
        }
        if (p.nsplit > 1) {
          *(f32x4*)(p.part + (2L * split) * all + oo + c) = x;
          *(f32x4*)(p.part + (2L * split + 1) * all + oo + c) = y;
        } else {
          const tv4 zx = {(T)x[0], (T)x[1], (T)x[2], (T)x[3]}, zy = {(T)y[0], (T)y[1], (T)y[2], (T)y[3]};
          *(tv4*)((T*)p.dk + oo + c) = zx;
          *(tv4*)((T*)p.dv + oo + c) = zy;
        }
      }
    }
}

// dk and dv = sums over the splits of the rows, in their order; the splits lie 2 * all floats apart, dk and dv in turn
template <typename T>
__global__ __launch_bounds__(256) void xattn_dkv_join_kernel(XaParams p, long all) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= 2 * all) return;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8];
  for (int s = 0; s < p.nsplit; ++s) {
    load8(v, p.part + 2L * s * all + i, 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += v[j];
  }
  store8(i < all ? (T*)p.dk + i : (T*)p.dv + (i - all), acc, 8);
}

// ------------------------------------------------------------------------------------------------ launches
// How the work is cut, from sizes alone, so that the workspace query and the launch agree.
struct XaPlan {
  int kw, tiles, nsplit;       // forward and dq
  int ktiles, ksplit;          // dk, dv
};
static int xa_clamp(long v, long lo, long hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }
static XaPlan xa_plan(const RtpXattn* a) {
  XaPlan pl;
  const long rows = (long)a->sq * (a->hq / a->hkv), bh = (long)a->b * a->hkv;
  // up to 32 rows the four waves of a workgroup split the keys, up to 64 two and two: with few rows the keys are the work
  pl.kw = rows <= 32 ? 4 : rows <= 64 ? 2 : 1;
  pl.tiles = rtp_div_up(rows, 128 / pl.kw);
  const long wgs = pl.tiles * bh, bk = pl.kw == 4 ? 128 : 64, nt = rtp_div_up(a->sk, bk);
  // two workgroups for each CU; a split has at least four tiles, or its partial results cost as much as they save
  pl.nsplit = xa_clamp(512 / (wgs > 0 ? wgs : 1), 1, nt / 4 > 1 ? nt / 4 : 1);
  pl.ktiles = rtp_div_up(a->sk, 128);
  const long kwgs = pl.ktiles * bh, rt = rtp_div_up(rows, 64);
  pl.ksplit = xa_clamp(512 / (kwgs > 0 ? kwgs : 1), 1, rt / 4 > 1 ? rt / 4 : 1);
  return pl;
}
static int xa_words(int sk) { return rtp_div_up(sk, 128) * 4; }
static long xa_round(long bytes) { return (bytes + 255) & ~255L; }

static int xa_check(const RtpXattn* a) {
  if (!a || a->b < 0 || a->sq < 0 || a->sk < 0 || a->hkv < 1 || a->hq < 1 || a->d < 1 || a->hq % a->hkv) return RTP_ERR_SHAPE;
  if (a->dtype != RTP_DT_F16 && a->dtype != RTP_DT_BF16) return RTP_ERR_UNSUPPORTED;
  if (a->d % 8 || a->d > 128) return RTP_ERR_UNSUPPORTED;
  const long grp = a->hq / a->hkv, rows = a->sq * grp;
  if (rows * grp >= (1L << 31) || a->sk > (1 << 30)) return RTP_ERR_SHAPE;
  const XaPlan pl = xa_plan(a);
  const long units = (long)a->b * a->hkv * (pl.nsplit > pl.ksplit ? pl.nsplit : pl.ksplit);
  const long tiles = pl.tiles > pl.ktiles ? pl.tiles : pl.ktiles;
  if ((units + 8) * tiles >= (1L << 31) || (long)a->b * xa_words(a->sk) >= (1L << 31) || (long)a->b * a->hkv * rows >= (1L << 34)) return RTP_ERR_SHAPE;
  if (!(a->scale > 0.f) || a->scale > 3e38f) return RTP_ERR_SHAPE;
  return RTP_OK;
}
static bool xa_aligned(const void* p, long bs, long ss, long hs) { return !((size_t)p & 15) && !(bs & 7) && !(ss & 7) && !(hs & 7); }

static XaParams xa_params(const RtpXattn* a) {
  XaParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v;
  p.q_bs = a->q_bs; p.q_ss = a->q_ss; p.q_hs = a->q_hs;
  p.k_bs = a->k_bs; p.k_ss = a->k_ss; p.k_hs = a->k_hs;
  p.v_bs = a->v_bs; p.v_ss = a->v_ss; p.v_hs = a->v_hs;
  p.lens = a->key_lens;
  p.b = a->b; p.sq = a->sq; p.sk = a->sk; p.hq = a->hq; p.hkv = a->hkv; p.d = a->d;
  p.grp = a->hq / a->hkv;
  p.rows = a->sq * p.grp;
  p.grp_magic = p.grp > 1 ? (unsigned)(((1UL << 32) + p.grp - 1) / p.grp) : 0u;
  p.words = xa_words(a->sk);
  p.scale = a->scale;
  p.scale_log2 = a->scale * 1.44269504088896340736f;
  return p;
}
static int xa_grid(XaParams& p, int tiles, int nsplit) {
  p.tiles = tiles;
  p.nsplit = nsplit;
  p.units = p.b * p.hkv * nsplit;
  return (p.units + 7) / 8 * 8 * tiles;
}

extern "C" long rtp_xattn_workspace_bytes(const RtpXattn* a, int backward) {
  if (xa_check(a) != RTP_OK) return -1;
  const XaPlan pl = xa_plan(a);
  const long rows = (long)a->b * a->sq * a->hq;
  long n = a->key_mask ? xa_round((long)a->b * xa_words(a->sk) * 4) : 0;
  if (!backward) return n + (pl.nsplit > 1 ? xa_round(rows * pl.nsplit * a->d * 4) + xa_round(rows * pl.nsplit * 4) : 0);
  const long q = pl.nsplit > 1 ? rows * pl.nsplit * a->d * 4 : 0;
  const long kv = pl.ksplit > 1 ? 2L * pl.ksplit * a->b * a->sk * a->hkv * a->d * 4 : 0;
  return n + xa_round(rows * 4) + xa_round(q > kv ? q : kv);   // dq and dk / dv run one after the other
}

static int xa_bits(const RtpXattn* a, XaParams& p, uint8_t*& ws, hipStream_t st) {
  if (!a->key_mask) return RTP_OK;
  p.bits = (unsigned*)ws;
  ws += xa_round((long)a->b * p.words * 4);
  hipLaunchKernelGGL(xattn_bits_kernel, dim3((unsigned)rtp_div_up(p.words, 8) * a->b), dim3(256), 0, st, (const uint8_t*)a->key_mask, a->m_bs, a->m_ss, a->key_lens,
                     (unsigned*)p.bits, a->sk, p.words);
  RTP_CHECK_LAUNCH();
  return RTP_OK;
}

// f(type, width in 32-column steps) for the call's head width
template <typename F>
static int xa_types(const RtpXattn* a, F f) {
  auto width = [&](auto t) {
    if (a->d <= 32) return f(t, std::integral_constant<int, 1>{});
    if (a->d <= 64) return f(t, std::integral_constant<int, 2>{});
    if (a->d <= 96) return f(t, std::integral_constant<int, 3>{});
    return f(t, std::integral_constant<int, 4>{});
  };
  return a->dtype == RTP_DT_BF16 ? width(bf16_t{}) : width(_Float16{});
}
template <typename K>
static int xa_launch(K kernel, int grid, int bytes, bool* once, hipStream_t st, const XaParams& p) {
  if (bytes > 65536 && rtp_once_per_device(once) &&
      hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return RTP_ERR_LAUNCH;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), bytes, st, p);
  RTP_CHECK_LAUNCH();
  return RTP_OK;
}
template <int DT, int KW> constexpr int xa_bytes() { return 4 * XaKeys<KW>::BK * XaImg<DT>::PITCH; }

template <typename T, int DT, int KW>
static int xa_fwd(int grid, hipStream_t st, const XaParams& p) {
  static bool once[RTP_MAX_DEVICES];
  return xa_launch(xattn_fwd_kernel<T, DT, KW>, grid, xa_bytes<DT, KW>(), once, st, p);
}
template <typename T, int DT, int KW>
static int xa_dq(int grid, hipStream_t st, const XaParams& p) {
  static bool once[RTP_MAX_DEVICES];
  return xa_launch(xattn_dq_kernel<T, DT, KW>, grid, xa_bytes<DT, KW>(), once, st, p);
}
template <typename T, int DT>
static int xa_dkv(int grid, hipStream_t st, const XaParams& p) {
  static bool once[RTP_MAX_DEVICES];
  return xa_launch(xattn_dkv_kernel<T, DT>, grid, 2 * (2 * 64 * XaImg<DT>::PITCH + 2 * 64 * 4), once, st, p);
}

extern "C" int rtp_xattn_forward(const RtpXattn* a, void* o, void* o_lo, float* lse, void* ws, long ws_bytes, void* stream) {
  const int rc = xa_check(a);
  if (rc != RTP_OK) return rc;
  if (a->b == 0 || a->sq == 0) return RTP_OK;
  if (!a->q || !o || (a->sk > 0 && (!a->k || !a->v)) || (!o_lo) != (!lse)) return RTP_ERR_SHAPE;
  if (!xa_aligned(a->q, a->q_bs, a->q_ss, a->q_hs) || !xa_aligned(a->k, a->k_bs, a->k_ss, a->k_hs) || !xa_aligned(a->v, a->v_bs, a->v_ss, a->v_hs) ||
      ((size_t)o & 15) || ((size_t)o_lo & 15) || ((size_t)ws & 255))
    return RTP_ERR_ALIGN;
  const long need = rtp_xattn_workspace_bytes(a, 0);
  if (ws_bytes < need || (need > 0 && !ws)) return RTP_ERR_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  RtpProfScope prof(RTP_FAM_POINTWISE, st);
  XaParams p = xa_params(a);
  uint8_t* at = (uint8_t*)ws;
  const int rb = xa_bits(a, p, at, st);
  if (rb != RTP_OK) return rb;
  p.o = o; p.o_lo = o_lo; p.lse = lse;
  const XaPlan pl = xa_plan(a);
  const int grid = xa_grid(p, pl.tiles, pl.nsplit);
  const long rows = (long)a->b * a->sq * a->hq;
  if (pl.nsplit > 1) {
    p.part = (float*)at;
    p.part_lse = (float*)(at + xa_round(rows * pl.nsplit * a->d * 4));
  }
  return xa_types(a, [&](auto t, auto dt) {
    typedef decltype(t) T;
    constexpr int DT = decltype(dt)::value;
    const int r = pl.kw == 4 ? xa_fwd<T, DT, 4>(grid, st, p) : pl.kw == 2 ? xa_fwd<T, DT, 2>(grid, st, p) : xa_fwd<T, DT, 1>(grid, st, p);
    if (r != RTP_OK || pl.nsplit == 1) return r;
    hipLaunchKernelGGL((xattn_join_kernel<T>), dim3(rtp_div_up(rows, 16)), dim3(256), 0, st, p);
    RTP_CHECK_LAUNCH();
    return RTP_OK;
  });
}

extern "C" int rtp_xattn_backward(const RtpXattn* a, const void* o, const void* o_lo, const float* lse, const void* d_o, long o_bs, long o_ss, long o_hs,
                                  void* dq, void* dk, void* dv, void* ws, long ws_bytes, void* stream) {
  const int rc = xa_check(a);
  if (rc != RTP_OK) return rc;
  if (a->b == 0 || a->sq == 0 || a->sk == 0) return RTP_ERR_SHAPE;   // nothing to compute: the caller fills the gradients with zeros
  if (!a->q || !a->k || !a->v || !o || !o_lo || !lse || !d_o || !ws || (!dk) != (!dv)) return RTP_ERR_SHAPE;
  if (!xa_aligned(a->q, a->q_bs, a->q_ss, a->q_hs) || !xa_aligned(a->k, a->k_bs, a->k_ss, a->k_hs) || !xa_aligned(a->v, a->v_bs, a->v_ss, a->v_hs) ||
      !xa_aligned(d_o, o_bs, o_ss, o_hs) || (((size_t)o | (size_t)o_lo | (size_t)dq | (size_t)dk | (size_t)dv) & 15) || ((size_t)ws & 255))
    return RTP_ERR_ALIGN;
  if (ws_bytes < rtp_xattn_workspace_bytes(a, 1)) return RTP_ERR_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  RtpProfScope prof(RTP_FAM_POINTWISE, st);
  XaParams p = xa_params(a);
  uint8_t* at = (uint8_t*)ws;
  const int rb = xa_bits(a, p, at, st);
  if (rb != RTP_OK) return rb;
  const long rows = (long)a->b * a->sq * a->hq;
  p.d_o = d_o; p.o_bs = o_bs; p.o_ss = o_ss; p.o_hs = o_hs;
  p.o = (void*)o; p.o_lo = (void*)o_lo; p.lse_in = lse;
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.delta = (float*)at;
  p.part = (float*)(at + xa_round(rows * 4));
  const XaPlan pl = xa_plan(a);
  return xa_types(a, [&](auto t, auto dt) {
    typedef decltype(t) T;
    constexpr int DT = decltype(dt)::value;
    hipLaunchKernelGGL((xattn_delta_kernel<T>), dim3(rtp_div_up(rows, 16)), dim3(256), 0, st, p);
    RTP_CHECK_LAUNCH();
    if (dq) {
      const int grid = xa_grid(p, pl.tiles, pl.nsplit);
      const int r = pl.kw == 4 ? xa_dq<T, DT, 4>(grid, st, p) : pl.kw == 2 ? xa_dq<T, DT, 2>(grid, st, p) : xa_dq<T, DT, 1>(grid, st, p);
      if (r != RTP_OK) return r;
      if (pl.nsplit > 1) {
        hipLaunchKernelGGL((xattn_dq_join_kernel<T>), dim3(rtp_div_up(rows, 16)), dim3(256), 0, st, p);
        RTP_CHECK_LAUNCH();
      }
    }
    if (!dk) return RTP_OK;
    const int grid = xa_grid(p, pl.ktiles, pl.ksplit), r = xa_dkv<T, DT>(grid, st, p);
    if (r != RTP_OK) return r;
    if (pl.ksplit > 1) {
      const long all = (long)a->b * a->sk * a->hkv * a->d;
      hipLaunchKernelGGL((xattn_dkv_join_kernel<T>), dim3(rtp_div_up(2 * all, 2048)), dim3(256), 0, st, p, all);
      RTP_CHECK_LAUNCH();
    }
    return RTP_OK;
  });
}
