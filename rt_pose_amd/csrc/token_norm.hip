// Root-mean-square norm of token rows with the residual's addition, in values or in 8 bits with scales, its backward pass, and the
// step into 8 bits by itself.
//
//   s = round(x + r)        y = s * rho * w        rho = 1 / sqrt(mean(s^2) + eps)
//   backward, g = dy * w, xhat = s * rho:   dx = dr = rho * (g - xhat * mean(g * xhat)) + ds        dw = sum over rows of dy * xhat
//   8 bits: each 128 columns of a row share a = max(max|y|, 2^-100); q = e4m3(y * (448 / a)), scale = a / 448
//
// All of it is bound by HBM: 4 streams forward (x, r in; y, s out), 4 backward (dy, ds, s in; dx out), 16-64 operations per chunk of
// eight.  A row is read ONCE: a group of LPR lanes holds it in registers (NV chunks of eight per lane) between the sum of squares and
// the output, and the backward pass forms both of its row sums (s^2 and g * s) from one reading, so nothing but s is kept for it.
// Sums are fp32, in an order that depends on the row's length alone.
#include <type_traits>

#include "rtp_prof.h"
#include "token_common.h"

// sum over the LPR lanes of a row; every lane gets it.  `red` holds one float per wave of the workgroup and is used twice in a row by
// callers: the closing barrier keeps the second use off the first one's reads.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (LPR > 64) {
    constexpr int NW = LPR / 64;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += red[i];
    __syncthreads();
  }
  return v;
}

struct NormParams {
  const void *x, *res, *w;
  void *y, *s;
  uint8_t* q;
  float* scale;
  long x_rs, res_rs, q_rs, rows;
  int h;
  bool far;                  // s and y are larger than the last-level cache
  bool once;                 // x and res are far larger than the L2s
  float eps;
};

// Bound by HBM: 20480 x 1024 bf16 with the residual 32 us for 168 MB, 5.2 TB/s; 16384 x 8192 to 8 bits 163 us for 944 MB, 5.8 TB/s (a large copy
// moves 4.96).  8 x 4096, a token's rows: 4.3 us, one trip to memory and the launch.
template <typename T, typename W, int LPR, int NV, bool OUT8, RowKind KIND>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void rmsnorm_fwd_kernel(NormParams p) {
  constexpr int THREADS = LPR > 256 ? LPR : 256;
  __shared__ float red[THREADS / 64];
  const int lane = threadIdx.x % LPR;
  const long row = (long)blockIdx.x * (THREADS / LPR) + threadIdx.x / LPR;
  if (LPR <= 64 && row >= p.rows) return;   // wider groups: one row per workgroup, the grid is exact
  const T* x = (const T*)p.x + row * p.x_rs;
  const T* r = p.res ? (const T*)p.res + row * p.res_rs : nullptr;
  T* so = p.s ? (T*)p.s + row * p.h : nullptr;
  float v[NV][8], wv[NV][8];
  float sq = 0.f;
  vec8<T> xr[NV];
  vec8<W> wr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) xr[i] = fetch8<KIND>(x, (lane + i * LPR) * 8, p.h, p.once);
  if (r) {
    vec8<T> rr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) rr[i] = fetch8<KIND>(r, (lane + i * LPR) * 8, p.h, p.once);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float rv[8];
      settle8<KIND, T>(v[i], xr[i], (lane + i * LPR) * 8, p.h);
      settle8<KIND, T>(rv, rr[i], (lane + i * LPR) * 8, p.h);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (float)(T)(v[i][j] + rv[j]);   // the stream as it is written is what is normed
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) settle8<KIND, T>(v[i], xr[i], (lane + i * LPR) * 8, p.h);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) wr[i] = fetch8<KIND>((const W*)p.w, (lane + i * LPR) * 8, p.h);
#pragma unroll
  for (int i = 0; i < NV; ++i) settle8<KIND, W>(wv[i], wr[i], (lane + i * LPR) * 8, p.h);
  if (so) {
#pragma unroll
    for (int i = 0; i < NV; ++i) put_row8<KIND>(so, v[i], (lane + i * LPR) * 8, p.h, p.far);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) sq += v[i][j] * v[i][j];
  const float rho = 1.f / sqrtf(row_sum<LPR>(sq, red) / (float)p.h + p.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + i * LPR) * 8, n = p.h - c;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * rho * wv[i][j];
    if constexpr (!OUT8) {
      put_row8<KIND>((T*)p.y + row * p.h, v[i], c, p.h, p.far);
    } else {
      // a block of 128 columns = 16 neighbouring lanes; columns behind the row's end are zeros and change nothing
      float a = amax8(v[i]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
      a = fmaxf(a, RTP_FP8_AMAX_FLOOR);
      if (n > 0) {
        *(i32x2*)(p.q + row * p.q_rs + c) = to_fp8x8(v[i], RTP_FP8_MAX / a);   // up to the row's end rounded up to 8: inside its padding
        if ((lane & 15) == 0) p.scale[row * ((p.h + 127) >> 7) + (c >> 7)] = a / RTP_FP8_MAX;
      }
    }
  }
}

struct NormBwdParams {
  const void *s, *w, *dy, *ds;
  void* dx;
  float* part;   // [gridDim.x][h], or null: dw is not wanted
  long s_rs, dy_rs, ds_rs, rows;
  int h;
  float eps;
};

// Workgroups walk the rows with a stride; each lane keeps its columns' share of dw in registers over all its rows, a workgroup leaves one
// partial row, and rmsnorm_dw_kernel adds those in fixed order: no atomics.  20480 x 1024 bf16: 34.5 us for 168 MB, 4.9 TB/s, and 4 for dw.
template <typename T, typename W, int LPR, int NV, RowKind KIND>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void rmsnorm_bwd_kernel(NormBwdParams p) {
  constexpr int THREADS = LPR > 256 ? LPR : 256, GROUPS = THREADS / LPR;
  __shared__ float red[THREADS / 64];
  __shared__ float comb[GROUPS > 1 ? GROUPS * LPR * NV * 8 : 1];
  const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  float wv[NV][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    settle8<KIND, W>(wv[i], fetch8<KIND>((const W*)p.w, (lane + i * LPR) * 8, p.h), (lane + i * LPR) * 8, p.h);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
  }
  for (long row = (long)blockIdx.x * GROUPS + grp; row < p.rows; row += (long)gridDim.x * GROUPS) {
    float s[NV][8], g[NV][8], d[NV][8];      // all of a row's loads at once: one trip to memory for it
    float sq = 0.f, gs = 0.f;
    vec8<T> sr[NV], gr[NV], dr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      sr[i] = fetch8<KIND>((const T*)p.s + row * p.s_rs, (lane + i * LPR) * 8, p.h);
      gr[i] = fetch8<KIND>((const T*)p.dy + row * p.dy_rs, (lane + i * LPR) * 8, p.h);
    }
    if (p.ds) {
#pragma unroll
      for (int i = 0; i < NV; ++i) dr[i] = fetch8<KIND>((const T*)p.ds + row * p.ds_rs, (lane + i * LPR) * 8, p.h);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      settle8<KIND, T>(s[i], sr[i], (lane + i * LPR) * 8, p.h);
      settle8<KIND, T>(g[i], gr[i], (lane + i * LPR) * 8, p.h);
    }
    if (p.ds) {
#pragma unroll
      for (int i = 0; i < NV; ++i) settle8<KIND, T>(d[i], dr[i], (lane + i * LPR) * 8, p.h);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) d[i][j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sq += s[i][j] * s[i][j];
        gs += g[i][j] * wv[i][j] * s[i][j];
      }
    const float rho = 1.f / sqrtf(row_sum<LPR>(sq, red) / (float)p.h + p.eps);
    const float back = row_sum<LPR>(gs, red) / (float)p.h * rho * rho;   // mean(g * xhat) * rho: xhat * mean = s * back
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * LPR) * 8, n = p.h - c;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw[i][j] += g[i][j] * s[i][j] * rho;
        d[i][j] += rho * (g[i][j] * wv[i][j] - s[i][j] * back);
      }
      put_row8<KIND>((T*)p.dx + row * p.h, d[i], c, p.h);
    }
  }
  if (!p.part) return;
  if constexpr (GROUPS > 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) comb[grp * (LPR * NV * 8) + (lane + i * LPR) * 8 + j] = dw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < p.h; c += THREADS) {
      float t = 0.f;
      for (int k = 0; k < GROUPS; ++k) t += comb[k * (LPR * NV * 8) + c];
      p.part[(long)blockIdx.x * p.h + c] = t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * LPR) * 8;
      put_row8<KIND>(p.part + (long)blockIdx.x * p.h, dw[i], c, p.h);
    }
  }
}

// dw[c] = sum of the partial rows: 16 columns (one 64-byte line) x 64 row slots per workgroup, so that few columns still make enough loads,
// eight of a thread's at once (1024 rows of 1024: 4.1 us, one after the other 6.4)
template <typename W>
__global__ __launch_bounds__(1024) void rmsnorm_dw_kernel(const float* part, int slots, int h, W* dw) {
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, k = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float t = 0.f;
  if (c < h) {
#pragma unroll 8
    for (int i = k; i < slots; i += 64) t += part[(long)i * h + c];
  }
  red[k][cl] = t;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (k < o) red[k][cl] += red[k + o][cl];
    __syncthreads();
  }
  if (k == 0 && c < h) dw[c] = (W)red[0][cl];
}

// ------------------------------------------------------------------------------------------------ launches
// lanes per row and chunks per lane by the row's length: 16 lanes up to 128 columns (four rows a wave), a wave up to 2048, a workgroup of
// 256 up to 8192, of 512 up to 16384, where its registers end (2500 x 16384 bf16: gradients 78 us, with 1024 threads of half as many registers 119;
// ragged widths keep 108 bytes a lane in scratch, fp32 172, and read them back in the loop over rows: 2500 x 16383 108 us, in fp32 174 and 164 whole)
#define NORM_MAX_H 16384

template <typename F>
static int norm_lanes(int h, F f) {
  if (h <= 128) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  if (h <= 512) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  if (h <= 1024) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  if (h <= 2048) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
  if (h <= 4096) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  if (h <= 8192) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
  return f(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
}

// f(lanes, chunks, kind of rows)
template <typename F>
static int norm_shape(int h, F f) {
  if (h < 8) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{}, std::integral_constant<RowKind, ROW_SHORT>{});
  return norm_lanes(h, [&](auto lpr, auto nv) {
    return h % 8 ? f(lpr, nv, std::integral_constant<RowKind, ROW_RAGGED>{}) : f(lpr, nv, std::integral_constant<RowKind, ROW_WHOLE>{});
  });
}

// value type x weight type (fp32 weights beside half values, or the values' own type)
template <typename F>
static int norm_types(int dtype, int w_dtype, F f) {
  if (dtype == RTP_DT_F32 && w_dtype == RTP_DT_F32) return f(float{}, float{});
  if (dtype == RTP_DT_F16 && w_dtype == RTP_DT_F16) return f(_Float16{}, _Float16{});
  if (dtype == RTP_DT_F16 && w_dtype == RTP_DT_F32) return f(_Float16{}, float{});
  if (dtype == RTP_DT_BF16 && w_dtype == RTP_DT_BF16) return f(bf16_t{}, bf16_t{});
  if (dtype == RTP_DT_BF16 && w_dtype == RTP_DT_F32) return f(bf16_t{}, float{});
  return RTP_ERR_UNSUPPORTED;
}

template <bool OUT8>
static int norm_forward(NormParams p, int dtype, int w_dtype, hipStream_t st) {
  if (p.rows < 0 || p.h < 1 || p.rows >= (1L << 31)) return RTP_ERR_SHAPE;
  if (p.h > NORM_MAX_H) return RTP_ERR_UNSUPPORTED;
  if (p.rows == 0) return RTP_OK;
  if (!p.x || !p.w || (p.res && !p.s)) return RTP_ERR_SHAPE;
  RtpProfScope prof(RTP_FAM_NORM, st);
  // 16384 x 8192 to 8 bits (s of 268 MB) 174 us, 187 without; 40960 x 2048 ten times in a row, each on the last one's outputs (2 x 168 MB), 118
  // against 124; but 20480 x 1024 (2 x 42 MB), done always, 31.4 against 27.9.
  const long size = dtype == RTP_DT_F32 ? 4 : 2;
  // Rows of x and res that are read and done with, past the caches too: 8192 x 8192 91 us, 106 without; 2500 x 16384 (78 MB) 57 and 64; but 16384 x 1024
  // (32 MB) 27 and 23.  (The backward pass gains nothing by either.)
  p.once = p.rows * p.h * size > (64L << 20);
  p.far = p.rows * p.h * ((p.s ? size : 0) + (OUT8 ? 1 : size)) > RTP_FAR_BYTES;
  return norm_types(dtype, w_dtype, [&](auto t, auto w) {
    return norm_shape(p.h, [&](auto lpr, auto nv, auto kind) {
      constexpr int LPR = decltype(lpr)::value, NV = decltype(nv)::value, THREADS = LPR > 256 ? LPR : 256;
      if (!rtp_launchable(rtp_div_up(p.rows, THREADS / LPR), THREADS)) return RTP_ERR_SHAPE;
      hipLaunchKernelGGL((rmsnorm_fwd_kernel<decltype(t), decltype(w), LPR, NV, OUT8, decltype(kind)::value>), dim3(rtp_div_up(p.rows, THREADS / LPR)), dim3(THREADS), 0,
                         st, p);
      RTP_CHECK_LAUNCH();
      return RTP_OK;
    });
  });
}

extern "C" int rtp_rmsnorm_forward(const void* x, long x_rs, const void* res, long res_rs, const void* w, int w_dtype, void* y, void* s,
                                   long rows, int h, int dtype, float eps, void* stream) {
  if (rows > 0 && !y) return RTP_ERR_SHAPE;
  NormParams p{x, res, w, y, s, nullptr, nullptr, x_rs, res_rs, 0, rows, h, false, false, eps};
  return norm_forward<false>(p, dtype, w_dtype, (hipStream_t)stream);
}

extern "C" int rtp_rmsnorm_fp8_forward(const void* x, long x_rs, const void* res, long res_rs, const void* w, int w_dtype, void* q, long q_rs,
                                       float* scale, void* s, long rows, int h, int dtype, float eps, void* stream) {
  if (rows > 0 && (!q || !scale)) return RTP_ERR_SHAPE;
  if (q_rs < ((h + 15) & ~15)) return RTP_ERR_SHAPE;
  if (((size_t)q & 15) || (q_rs & 15)) return RTP_ERR_ALIGN;
  NormParams p{x, res, w, nullptr, s, (uint8_t*)q, scale, x_rs, res_rs, q_rs, rows, h, false, false, eps};
  return norm_forward<true>(p, dtype, w_dtype, (hipStream_t)stream);
}

// partial rows of dw: four workgroups per CU walk the rows where a wave takes one (20480 x 1024: 34.5 us, with two 39.4), two where a workgroup of 256
// does (their partial rows are longer: 2048 x 8192 34 us, with four 45, with one 38), one of 512 (as many fit: 2500 x 16384 80 us, with two 88), fewer
// where there are fewer rows
extern "C" int rtp_rmsnorm_backward_slots(long rows, int h) {
  if (rows < 1 || h < 1 || h > NORM_MAX_H) return 0;
  const int groups = h <= 128 ? 16 : h <= 2048 ? 4 : 1;
  const long need = (rows + groups - 1) / groups;
  const long most = h <= 2048 ? 1024 : h <= 8192 ? 512 : 256;
  return (int)(need < most ? need : most);
}

extern "C" int rtp_rmsnorm_backward(const void* s, long s_rs, const void* w, int w_dtype, const void* dy, long dy_rs, const void* ds, long ds_rs,
                                    void* dx, void* dw, float* part, long rows, int h, int dtype, float eps, void* stream) {
  if (rows < 1 || h < 1 || rows >= (1L << 31)) return RTP_ERR_SHAPE;
  if (h > NORM_MAX_H) return RTP_ERR_UNSUPPORTED;
  if (!s || !w || !dy || !dx || (dw && !part)) return RTP_ERR_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  RtpProfScope prof(RTP_FAM_NORM, st);
  NormBwdParams p{s, w, dy, ds, dx, dw ? part : nullptr, s_rs, dy_rs, ds_rs, rows, h, eps};
  const int slots = rtp_rmsnorm_backward_slots(rows, h);
  return norm_types(dtype, w_dtype, [&](auto t, auto wt) {
    return norm_shape(h, [&](auto lpr, auto nv, auto kind) {
      constexpr int LPR = decltype(lpr)::value, NV = decltype(nv)::value, THREADS = LPR > 256 ? LPR : 256;
      typedef decltype(wt) W;
      hipLaunchKernelGGL((rmsnorm_bwd_kernel<decltype(t), W, LPR, NV, decltype(kind)::value>), dim3(slots), dim3(THREADS), 0, st, p);
      RTP_CHECK_LAUNCH();
      if (!dw) return RTP_OK;
      hipLaunchKernelGGL((rmsnorm_dw_kernel<W>), dim3(rtp_div_up(h, 16)), dim3(1024), 0, st, part, slots, h, (W*)dw);
      RTP_CHECK_LAUNCH();
      return RTP_OK;
    });
  });
}

// ------------------------------------------------------------------------------------------------ quantising by itself
struct QuantParams {
  const void* x;
  uint8_t* q;
  float* scale;
  long x_rs, q_rs, rows;
  int cols, kb;
};

// blocks of 1 x 128, rows in memory order: 16 lanes a block, four rows a lane so that four loads are in flight
#define QUANT_ROWS 4
template <typename T, RowKind KIND>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantParams p) {
  const unsigned g = blockIdx.x * 16u + (threadIdx.x >> 4);
  const int lane = threadIdx.x & 15;
  const long row0 = (long)(g / (unsigned)p.kb) * QUANT_ROWS;
  const int b = (int)(g % (unsigned)p.kb), c = b * 128 + lane * 8, n = p.cols - c;
  float v[QUANT_ROWS][8];
  vec8<T> r[QUANT_ROWS];
#pragma unroll
  for (int u = 0; u < QUANT_ROWS; ++u) r[u] = fetch8<KIND>((const T*)p.x + (row0 + u < p.rows ? row0 + u : p.rows - 1) * p.x_rs, c, p.cols);
#pragma unroll
  for (int u = 0; u < QUANT_ROWS; ++u) settle8<KIND, T>(v[u], r[u], c, p.cols);
#pragma unroll
  for (int u = 0; u < QUANT_ROWS; ++u) {
    float a = amax8(v[u]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
    a = fmaxf(a, RTP_FP8_AMAX_FLOOR);
    if (row0 + u < p.rows && n > 0) {
      *(i32x2*)(p.q + (row0 + u) * p.q_rs + c) = to_fp8x8(v[u], RTP_FP8_MAX / a);
      if (lane == 0) p.scale[(row0 + u) * p.kb + b] = a / RTP_FP8_MAX;
    }
  }
}

// blocks of 128 x 128, rows in memory order: one workgroup a block, held in registers between its maximum and the output.  8192 x 4096 bf16: 17 us for
// 101 MB, 6.0 TB/s.
template <typename T, RowKind KIND>
__global__ __launch_bounds__(256) void quant_square_kernel(QuantParams p) {
  __shared__ float red[4];
  const int lane = threadIdx.x & 15, b = blockIdx.x % (unsigned)p.kb;
  const long row0 = (long)(blockIdx.x / (unsigned)p.kb) * 128 + (threadIdx.x >> 4);
  const int c = b * 128 + lane * 8, n = p.cols - c;
  float v[8][8];
  vec8<T> r[8];
  float a = 0.f;
#pragma unroll
  for (int u = 0; u < 8; ++u) r[u] = fetch8<KIND>((const T*)p.x + (row0 + u * 16 < p.rows ? row0 + u * 16 : p.rows - 1) * p.x_rs, c, p.cols);
#pragma unroll
  for (int u = 0; u < 8; ++u) settle8<KIND, T>(v[u], r[u], c, p.cols);     // a row behind the last one repeats it: the block's maximum stays
#pragma unroll
  for (int u = 0; u < 8; ++u) a = fmaxf(a, amax8(v[u]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), RTP_FP8_AMAX_FLOOR);
  const float up = RTP_FP8_MAX / a;
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (row0 + u * 16 < p.rows && n > 0) *(i32x2*)(p.q + (row0 + u * 16) * p.q_rs + c) = to_fp8x8(v[u], up);
  if (threadIdx.x == 0) p.scale[blockIdx.x] = a / RTP_FP8_MAX;
}

// Either block, x given by columns (a transpose's view: x[r][c] at c * x_rs + r).  A tile of 128 rows x 128 columns goes through LDS twice: read
// along the columns' memory order, taken by each thread as 32 columns of two neighbouring rows (one LDS word a column for 16-bit types, held in
// registers from the maximum to the output), and the bytes once more so that they leave as whole rows.  1000 x 20481 bf16: 14 us for 62 MB, 4.4 TB/s
// (a chunk's loads one after the other: 17).
template <typename T, bool SQUARE, RowKind KIND>
__global__ __launch_bounds__(256) void quant_turned_kernel(QuantParams p) {
  constexpr int PITCH = 128 + 16 / sizeof(T), QPITCH = 144;     // keep 16-byte accesses aligned and rows apart
  typedef T tv2 __attribute__((ext_vector_type(2)));
  __shared__ __attribute__((aligned(16))) T tile[128 * PITCH];
  __shared__ float red[4][128];
  // workgroups go round the 8 XCDs: tiles of neighbouring rows, which share the lines at their border, follow each other on one of them
  const unsigned rt = (unsigned)((p.rows + 127) >> 7), at = blockIdx.x >> 3;
  const int b = (int)(at / rt) * 8 + (blockIdx.x & 7), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long row0 = (long)(at % rt) * 128;
  if (b >= p.kb) return;
  {
    const int ch = (threadIdx.x & 15) * 8;
    vec8<T> r[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int c = b * 128 + (threadIdx.x >> 4) + u * 16;
      r[u] = fetch8<KIND>((const T*)p.x + (long)(c < p.cols ? c : p.cols - 1) * p.x_rs, (int)row0 + ch, (int)p.rows);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      float v[8];
      settle8<KIND, T>(v, r[u], (int)row0 + ch, (int)p.rows);
      if (b * 128 + (threadIdx.x >> 4) + u * 16 >= p.cols) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
      }
      store8(tile + ((threadIdx.x >> 4) + u * 16) * PITCH + ch, v, 8);
    }
  }
  __syncthreads();
  float v[2][32], a[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const tv2 x = *(const tv2*)(tile + (wave * 32 + c) * PITCH + 2 * lane);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      v[e][c] = (float)x[e];
      a[e] = fmaxf(a[e], fabsf(v[e][c]));
    }
  }
  float up[2], top[2];
  if constexpr (SQUARE) {
    float m = fmaxf(a[0], a[1]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    top[0] = top[1] = fmaxf(fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])), RTP_FP8_AMAX_FLOOR);
    if (threadIdx.x == 0) p.scale[(row0 >> 7) * p.kb + b] = top[0] / RTP_FP8_MAX;
  } else {
    red[wave][2 * lane] = a[0];
    red[wave][2 * lane + 1] = a[1];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * lane + e;
      top[e] = fmaxf(fmaxf(fmaxf(red[0][r], red[1][r]), fmaxf(red[2][r], red[3][r])), RTP_FP8_AMAX_FLOOR);
      if (wave == 0 && row0 + r < p.rows) p.scale[(row0 + r) * p.kb + b] = top[e] / RTP_FP8_MAX;
    }
  }
  // every thread has read the tile (the barrier above): the bytes take its place
  uint8_t* bytes = (uint8_t*)tile;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    up[e] = RTP_FP8_MAX / top[e];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float lo[8], hi[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = v[e][16 * k + j];
        hi[j] = v[e][16 * k + 8 + j];
      }
      const i32x2 l = to_fp8x8(lo, up[e]), h = to_fp8x8(hi, up[e]);
      *(i32x4*)(bytes + (2 * lane + e) * QPITCH + wave * 32 + k * 16) = i32x4{l[0], l[1], h[0], h[1]};
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = (threadIdx.x >> 3) + u * 32, c = (threadIdx.x & 7) * 16;
    if (row0 + r < p.rows && b * 128 + c < p.cols)
      *(i32x4*)(p.q + (row0 + r) * p.q_rs + b * 128 + c) = *(const i32x4*)(bytes + r * QPITCH + c);
  }
}

extern "C" int rtp_quantize_fp8(const void* x, long x_rs, int turned, void* q, long q_rs, float* scale, long rows, int cols, int square, int dtype,
                                void* stream) {
  if (rows < 0 || rows >= (1L << 31) || cols < 1 || cols > (1 << 30) || q_rs < ((cols + 15) & ~15)) return RTP_ERR_SHAPE;
  if (rows == 0) return RTP_OK;
  if (!x || !q || !scale) return RTP_ERR_SHAPE;
  if (((size_t)q & 15) || (q_rs & 15)) return RTP_ERR_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  RtpProfScope prof(RTP_FAM_NORM, st);
  const int kb = (cols + 127) >> 7;
  QuantParams p{x, (uint8_t*)q, scale, x_rs, q_rs, rows, cols, kb};
  const long tiles = ((rows + 127) >> 7) * kb, turned_tiles = ((rows + 127) >> 7) * ((kb + 7) & ~7), groups = ((rows + QUANT_ROWS - 1) / QUANT_ROWS) * kb;
  if (!rtp_launchable(turned ? turned_tiles : square ? tiles : (groups + 15) / 16, 256)) return RTP_ERR_SHAPE;
  auto go = [&](auto t) {
    typedef decltype(t) T;
    if (turned && square)
      hipLaunchKernelGGL((rows < 8   ? quant_turned_kernel<T, true, ROW_SHORT>
                          : rows % 8 ? quant_turned_kernel<T, true, ROW_RAGGED>
                                     : quant_turned_kernel<T, true, ROW_WHOLE>),
                         dim3((unsigned)turned_tiles), dim3(256), 0, st, p);
    else if (turned)
      hipLaunchKernelGGL((rows < 8   ? quant_turned_kernel<T, false, ROW_SHORT>
                          : rows % 8 ? quant_turned_kernel<T, false, ROW_RAGGED>
                                     : quant_turned_kernel<T, false, ROW_WHOLE>),
                         dim3((unsigned)turned_tiles), dim3(256), 0, st, p);
    else if (square)
      hipLaunchKernelGGL((cols < 8 ? quant_square_kernel<T, ROW_SHORT> : cols % 8 ? quant_square_kernel<T, ROW_RAGGED> : quant_square_kernel<T, ROW_WHOLE>),
                         dim3((unsigned)tiles), dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((cols < 8 ? quant_rows_kernel<T, ROW_SHORT> : cols % 8 ? quant_rows_kernel<T, ROW_RAGGED> : quant_rows_kernel<T, ROW_WHOLE>),
                         dim3(rtp_div_up(groups, 16)), dim3(256), 0, st, p);
    RTP_CHECK_LAUNCH();
    return RTP_OK;
  };
  if (dtype == RTP_DT_F32) return go(float{});
  if (dtype == RTP_DT_F16) return go(_Float16{});
  if (dtype == RTP_DT_BF16) return go(bf16_t{});
  return RTP_ERR_UNSUPPORTED;
}
