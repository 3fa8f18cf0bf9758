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
typedef __attribute__((address_space(3))) uint8_t lds_u8_xa;
typedef __attribute__((address_space(4))) unsigned cst_u32_xa;   // read-only for the whole launch: uniform addresses become scalar loads

__device__ __attribute__((aligned(16))) bf16_t g_zero_line_xa[8];   // what masked rows and columns behind the head's width are staged from

__device__ float g_inf_xa = INFINITY;

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <typename T> struct Vec8;
template <> struct Vec8<bf16_t> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };

// sixteen fp32 values of a lane as the second operands of two products; with LO what their rounding left over follows in two more.  Where few rows
// leave the matrix unit idle (KW = 4) p and ds go in as both halves: nothing of them is lost then.
template <typename T, bool LO> struct XaSecond {
  typename Vec8<T>::type v[LO ? 4 : 2];
  __device__ __forceinline__ void set(int i, float x) {
    v[i >> 3][i & 7] = (T)x;
    if constexpr (LO) v[2 + (i >> 3)][i & 7] = (T)(x - (float)(T)x);
  }
};

struct XaParams {
  const void *q, *k, *v, *d_o;
  long q_bs, q_ss, q_hs, k_bs, k_ss, k_hs, v_bs, v_ss, v_hs, o_bs, o_ss, o_hs;   // o_*: of d_o
  const unsigned* bits;      // [b][words]: one bit per key, from key_mask and key_lens; null: key_lens alone
  const int* lens;           // [b] or null
  int b, sq, sk, hq, hkv, d, grp, rows;
  unsigned grp_magic;        // ceil(2^32 / grp): r / grp = mulhi(r, magic) for r * grp < 2^32
  int words;
  int tiles, units, nsplit;  // workgroups = tiles x units (batch x kv head x split)
  int near;                  // kv heads whose rows share a 128-byte line
  int pairs;                 // forward: pairs of a batch entry and a run of its tiles of keys, or 0: units are batch x kv head
  bool ragged;               // pairs follow the entries' lengths
  float scale, scale_log2;
  void *o, *o_lo, *dq, *dk, *dv;
  float *lse, *delta, *part, *part_lse;
  const float* lse_in;
};

// workgroup -> tile of rows, group of `near` units, which of them.  Heads whose rows share a line follow each other on one XCD: with one of them on
// each XCD every line goes to several L2s (15 rows x 20480 keys, 8 x 8 heads of 32: forward 55.7 us, so 40.4; backward 95.8, so 79.5).
__device__ __forceinline__ bool xa_group(const XaParams& p, int& tile, unsigned& group, unsigned& member) {
  const unsigned j = blockIdx.x >> 3, y = j / (unsigned)p.tiles;
  tile = j % (unsigned)p.tiles;
  group = y / (unsigned)p.near * 8 + (blockIdx.x & 7);
  member = y % (unsigned)p.near;
  return group * p.near < (unsigned)p.units;
}
// Workgroup -> (tile, unit): all tiles of a unit run on one XCD (workgroups go round the 8 XCDs), so that a unit's k and v stay in one L2.
// Batch entries with more keys come first (up to 64 entries: each lane ranks one): the last workgroups to start are then the short ones.
__device__ __forceinline__ bool xa_place(const XaParams& p, int& tile, int& b, int& hk, int& split) {
  unsigned group, member;
  if (!xa_group(p, tile, group, member)) return false;
  const unsigned some = p.hkv / p.near, bg = group / (unsigned)p.nsplit;
  split = group % (unsigned)p.nsplit;
  b = bg / some;
  hk = (bg % some) * p.near + member;
  if (p.lens && p.b > 1 && p.b <= 64) {
    const int lane = threadIdx.x & 63, mine = lane < p.b ? p.lens[lane] : 0;
    int rank = 0;
    for (int i = 0; i < p.b; ++i) {
      const int other = __builtin_amdgcn_readlane(mine, i);
      rank += other > mine || (other == mine && i < lane);
    }
    b = __builtin_ctzll(__ballot(lane < p.b && rank == b));
  }
  return true;
}

// The forward pass in runs of tiles of keys, `pairs` of them at most.  Where entries have lengths (p.ragged, 2 to 64 entries, a lane each) one
// length of run does for all: the shortest (long ones: up to a sixteenth) that leaves no more runs than pairs, so that every workgroup has the same
// to do, whatever the lengths are (one row, 8 entries of 0 to 5120 keys x 8 heads of 128: 20.1 us; every entry in as many runs 26.6).  Entry i has runs
// first .. first + n - 1.  A run has two tiles at least: 8 x 8 heads, 256 keys, in two runs of one tile 7.4 us and 3.7 for the join, uncut 8.9.
struct XaShares { int tiles, run, first, n; };      // tiles, first and n: of the lane's entry
#define XA_RUN 2
__device__ __forceinline__ XaShares xa_shares(const XaParams& p, int bk) {
  const int lane = threadIdx.x & 63;
  XaShares s;
  const int len = lane < p.b ? p.lens[lane] : 0;
  s.tiles = ((len < 0 ? 0 : len > p.sk ? p.sk : len) + bk - 1) / bk;
  auto sum = [&](int v) {
    for (int o = 1; o < p.b; o <<= 1) v += __shfl_xor(v, o, 64);
    return __builtin_amdgcn_readfirstlane(v);
  };
  const unsigned even = ((unsigned)sum(s.tiles) + p.pairs - 1) / (unsigned)p.pairs;
  s.run = even > XA_RUN ? even : XA_RUN;
  while (true) {                 // ends: one run for each entry is fewer than pairs
    s.n = (unsigned)(s.tiles + s.run - 1) / (unsigned)s.run;
    if (sum(s.n) <= p.pairs) break;
    s.run += 1 + s.run / 16;
  }
  s.first = s.n;
  for (int o = 1; o < p.b; o <<= 1) {
    const int v = __shfl_up(s.first, o, 64);
    s.first += lane >= o ? v : 0;
  }
  s.first -= s.n;
  return s;
}

__device__ __forceinline__ int xa_len(const XaParams& p, int b) {
  if (!p.lens) return p.sk;
  const int n = (int)((const cst_u32_xa*)p.lens)[b];
  return n < 0 ? 0 : n > p.sk ? p.sk : n;
}
// this workgroup's tile of rows, batch entry, kv head, pair and run of tiles of keys
__device__ __forceinline__ bool xa_place_run(const XaParams& p, int bk, int& tile, int& b, int& hk, int& pair, int& t0, int& t1) {
  if (p.pairs == 0) {
    if (!xa_place(p, tile, b, hk, pair)) return false;
    t0 = 0;
    t1 = (xa_len(p, b) + bk - 1) / bk;
    return true;
  }
  unsigned group, member;
  if (!xa_group(p, tile, group, member)) return false;
  const unsigned some = p.hkv / p.near;
  pair = group / some;
  hk = (group % some) * p.near + member;
  if (!p.ragged) {
    b = pair / p.nsplit;
    const int split = pair % p.nsplit, nt = (xa_len(p, b) + bk - 1) / bk;
    t0 = (int)((long)nt * split / p.nsplit);
    t1 = (int)((long)nt * (split + 1) / p.nsplit);
    return true;
  }
  const XaShares s = xa_shares(p, bk);
  const unsigned long mine = __ballot(pair >= s.first && pair < s.first + s.n);
  if (mine == 0) return false;
  b = __builtin_ctzll(mine);
  t0 = (pair - __builtin_amdgcn_readlane(s.first, b)) * s.run;
  t1 = __builtin_amdgcn_readlane(s.tiles, b);
  if (t0 + s.run < t1) t1 = t0 + s.run;
  return true;
}
// bits of the 32 keys from key0 on
__device__ __forceinline__ unsigned xa_word(const XaParams& p, int b, int len, int key0) {
  if (p.bits) return ((const cst_u32_xa*)p.bits)[(long)b * p.words + (key0 >> 5)];
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

// Staging by LDS-DMA: 256 threads, 16 B each and step, no registers for the data.  Step i brings rows i * 256 / CH + thread / CH.
template <int DT>
__device__ __forceinline__ int xa_chunk() {      // this thread's column chunk: the same in every step (swz has period 16, steps are 16 rows or more)
  constexpr int CH = XaImg<DT>::CH;
  return (int)(threadIdx.x % CH) ^ XaImg<DT>::swz(threadIdx.x / CH);
}
// The transfers are written out: from the builtin the compiler knows that LDS is written, and waits for ALL of them in front of every
// transposing read.  Nothing is returned to registers; xa_landed() is what orders them.
__device__ __forceinline__ unsigned xa_m0(const uint8_t* img, int bytes) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  return __builtin_amdgcn_readfirstlane((unsigned)(size_t)(lds_u8_xa*)img + bytes + wave * 1024);
}
__device__ __forceinline__ void xa_dma(uint8_t* img, int step, const void* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(xa_m0(img, step * 4096)), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void xa_dma(uint8_t* img, int step, const void* base, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(xa_m0(img, step * 4096)), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void xa_dma4(uint8_t* lds, const void* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane((unsigned)(size_t)(lds_u8_xa*)lds)), "v"(src)
               : "memory", "m0");
}
// Which rows of an image a thread brings, and their byte offsets from the first one.  Where every row and column of a tile counts (most tiles)
// an access is a uniform address and one 32-bit offset a lane; otherwise each lane picks its row or the line of zeros.
template <int DT, typename T>
struct XaLoader {
  static constexpr int CH = XaImg<DT>::CH, ROWS = 256 / CH;
  int r, c;
  bool col;
  __device__ __forceinline__ XaLoader(int d) : r(threadIdx.x / CH), c(xa_chunk<DT>() * 8), col(c < d) {}
  // keys: bit of w for each
  template <int BK>
  __device__ __forceinline__ void keys(uint8_t* img, const T* src, long ss, unsigned off, bool whole, const unsigned (&w)[BK / 32]) const {
#pragma unroll
    for (int i = 0; i < BK / ROWS; ++i) {
      const char* at = (const char*)(src + (long)(i * ROWS) * ss);
      if (whole) {
        xa_dma(img, i, at, off);
      } else {
        const unsigned word = CH == 4 ? (threadIdx.x < 128 ? w[2 * i] : w[2 * i + 1]) : w[i * ROWS / 32];
        xa_dma(img, i, col && ((word >> ((i * ROWS + r) & 31)) & 1u) ? at + off : (const char*)g_zero_line_xa);
      }
    }
  }
  // query rows r0 .. r0 + BR - 1; `even`: the group divides a step's rows, so that a step is a whole number of tokens.  Widths between the images' take
  // the road that is not `whole` for every tile; with two steps of columns dk / dv's kernel keeps its addresses in scratch there (20 to 28 bytes a
  // lane): heads of 40, 48 and 56 take 145, 143 and 143 us where heads of 64 take 136.
  template <int BR>
  __device__ __forceinline__ void rows(uint8_t* img, const XaParams& p, const T* src, long ss, long hs, unsigned off, bool even, bool whole, int r0) const {
#pragma unroll
    for (int i = 0; i < BR / ROWS; ++i) {
      const int first = r0 + i * ROWS;
      const char* at = (const char*)(src + (even ? (long)(first / p.grp) * ss : 0L));
      if (whole) {
        xa_dma(img, i, at, off);
      } else {
        const char* mine = even ? at + off : (const char*)(src + xa_row_off(p, first + r, ss, hs) + c);
        xa_dma(img, i, col && first + r < p.rows ? mine : (const char*)g_zero_line_xa);
      }
    }
  }
};

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

// Eight accumulators of a lane -- columns 16 q + 8 (i / 4) + 4 h + i % 4 of one row, i < 8 -- rounded and stored: the half waves swap four columns
// each, and a lane then holds eight neighbouring ones.
template <typename T>
__device__ __forceinline__ void xa_store8(T* row, const float (&x)[8], int q, int h, int d, bool ok) {
  typedef T tv2 __attribute__((ext_vector_type(2)));
  unsigned a[2], b[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const tv2 lo = {(T)x[2 * e], (T)x[2 * e + 1]}, hi = {(T)x[4 + 2 * e], (T)x[5 + 2 * e]};
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi), false, false);
    a[e] = r[0];
    b[e] = r[1];
  }
  const int c = 16 * q + 8 * h;
  if (ok && c < d) *(i32x4*)(row + c) = i32x4{(int)a[0], (int)a[1], (int)b[0], (int)b[1]};
}
// the same for partial results, which stay fp32
__device__ __forceinline__ void xa_store8(float* row, const float (&x)[8], int q, int h, int d) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int c = 16 * q + 8 * e + 4 * h;
    if (c < d) *(f32x4*)(row + c) = f32x4{x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]};
  }
}
// a whole accumulator: columns 32 t .. 32 t + 31
template <typename T>
__device__ __forceinline__ void xa_store(T* row, const f32x16& x, int t, int h, int d, bool ok) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float y[8] = {x[8 * j], x[8 * j + 1], x[8 * j + 2], x[8 * j + 3], x[8 * j + 4], x[8 * j + 5], x[8 * j + 6], x[8 * j + 7]};
    xa_store8<T>(row, y, 2 * t + j, h, d, ok);
  }
}

// The accumulators of the KW waves that share rows, added with the given weights in wave order.  Every wave leaves its own in LDS and gathers every
// KW-th sixteen columns of all of them: f(q, values) for its q, columns 16 q + ...  Waves that share nothing (KW = 1) keep theirs.
template <int DT, int KW> struct XaMeet { static constexpr int SLOT = DT * 16 * 64 * 4, BYTES = KW > 1 ? 4 * SLOT : 0; };
template <int DT, int KW, typename F>
__device__ __forceinline__ void xa_gather(const f32x16 (&acc)[DT], const float (&weight)[KW], uint8_t* lds, int wave, F f) {
  const int lane = threadIdx.x & 63, kw = wave % KW;
  if constexpr (KW == 1) {
#pragma unroll
    for (int q = 0; q < 2 * DT; ++q) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = acc[q / 2][8 * (q & 1) + i] * weight[0];
      f(q, v);
    }
  } else {
    constexpr int SLOT = XaMeet<DT, KW>::SLOT / 4;
    __syncthreads();             // the weights have been read from the same place
    float* mine = (float*)lds + wave * SLOT + lane;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[(t * 16 + i) * 64] = acc[t][i];
    __syncthreads();
    const float* all = (const float*)lds + (wave / KW) * KW * SLOT + lane;
#pragma unroll
    for (int u = 0; u < (2 * DT + KW - 1) / KW; ++u) {
      const int q = kw + u * KW;
      if (q >= 2 * DT) break;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KW; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += all[k * SLOT + (q * 8 + i) * 64] * weight[k];
      f(q, v);
    }
  }
}

#define XA_M0 (-3.402823466e38f)
#define XA_SLACK 8.0f   // the running maximum moves only when it is exceeded by 2^8: p stays below 2^8, and most tiles rescale nothing

// fp16 has 2^-14 .. 65504 at full precision, and p (1 / keys on the average) and ds lie at its lower end.  So p is taken times 2^7 forward (with the
// slack at most 2^15) and times 2^14 backward (p <= 1); ds starts at 2^14 too, and a row or key whose |ds| would pass 2^15 lowers its own
// factor and what it has summed so far.  bf16 has fp32's range: no factors.
template <typename T> struct XaRange { static constexpr bool NARROW = false; static constexpr float FWD = 0.f, BWD = 0.f; };
template <> struct XaRange<_Float16> { static constexpr bool NARROW = true; static constexpr float FWD = 7.f, BWD = 14.f; };
// this lane's sixteen ds (times 2^ex) and the other half wave's of the same row or key; acc: the DT accumulators of that row or key
template <int DT>
__device__ __forceinline__ bool xa_narrow(f32x16& x, f32x16 (&acc)[DT], float& ex) {
  float mx = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 16; ++i) mx = fmaxf(mx, fabsf(x[i]));
  mx = xa_halves_max(mx);
  if (!__any(mx > 32768.f)) return false;
  const float drop = mx > 32768.f ? fminf(ceilf(log2f(mx)) - 8.f, 100.f) : 0.f, f = exp2f(-drop);
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] *= f;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] *= f;
  ex -= drop;
  return true;
}

// ------------------------------------------------------------------------------------------------ the loop over keys
// Four waves: 4 / KW groups of 32 rows, and KW waves that share rows and split each tile of keys (few rows: the keys are the work).
// Tiles of BK keys go round NBUF LDS buffers: while one is used, the next NBUF - 1 are on their way, and the barrier in front of a tile waits
// for that tile's transfers alone (they complete in order, PER of them a wave and tile).  Two buffers leave room for more workgroups on a CU,
// which hide more than a third one (heads of 64: forward 89 us with three, 81 with two); heads up to 32 columns have small tiles and three.  In the
// backward pass of few rows the third hides nothing: its stores of dk and dv count among the newest accesses, so that the wait takes in the tile behind.
// The mask's words are scalar loads, one tile further ahead, so that nothing else counts as a vector access.
// (Forming the next tile's scores beside this one's exponentials in one wave takes half as many registers again: 81 -> 103 us.)
template <int DT, int KW> struct XaKeys {
  static constexpr int BK = KW == 4 ? 128 : 64, SUB = BK / 32 / KW, NW = BK / 32, IMG = BK * XaImg<DT>::PITCH;
  static constexpr int NBUF = DT == 1 ? 3 : 2, RING = NBUF * 2 * IMG;
  static constexpr int BYTES = RING > XaMeet<DT, KW>::BYTES ? RING : XaMeet<DT, KW>::BYTES;     // the waves meet where the tiles were
};
// The compiler does not know of the transfers: whatever it loaded before the loop has to have arrived before the loop, or it would wait for it
// inside, and with it for all transfers.
__device__ __forceinline__ void xa_settle() { __builtin_amdgcn_s_waitcnt(0x0F70); }   // vmcnt(0)
// everything but the newest N vector accesses of this wave is done, and its LDS reads; then all waves
template <int N>
__device__ __forceinline__ void xa_landed() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// f(tile, images of k and v, words) for the tiles t0 .. t1 - 1
template <typename T, int DT, int KW, typename F>
__device__ __forceinline__ void xa_over_keys(const XaParams& p, uint8_t* lds, int b, int hk, int t0, int t1, bool busy, F compute) {
  typedef XaKeys<DT, KW> K;
  constexpr int BK = K::BK, NW = K::NW, NBUF = K::NBUF, IMG = K::IMG, PER = 2 * BK / XaLoader<DT, T>::ROWS;
  if (t0 >= t1) return;
  const int len = xa_len(p, b);
  const T* kp = (const T*)p.k + (long)b * p.k_bs + (long)hk * p.k_hs;
  const T* vp = (const T*)p.v + (long)b * p.v_bs + (long)hk * p.v_hs;
  const XaLoader<DT, T> ld(p.d);
  const unsigned k_off = (unsigned)(ld.r * (int)p.k_ss + ld.c) * 2u, v_off = (unsigned)(ld.r * (int)p.v_ss + ld.c) * 2u;
  const bool full = p.d == XaImg<DT>::CH * 8;
  unsigned w[NBUF + 1][NW];           // of the tiles t, t + 1, ...
  auto words = [&](int t, unsigned (&x)[NW]) {
#pragma unroll
    for (int i = 0; i < NW; ++i) x[i] = t < t1 ? xa_word(p, b, len, t * BK + i * 32) : 0u;
  };
  auto stage = [&](int t, uint8_t* at, const unsigned (&x)[NW]) {
    unsigned all = full ? ~0u : 0u;
#pragma unroll
    for (int i = 0; i < NW; ++i) all &= x[i];
    if (all == ~0u) {
      ld.template keys<BK>(at, kp + (long)t * BK * p.k_ss, p.k_ss, k_off, true, x);
      ld.template keys<BK>(at + IMG, vp + (long)t * BK * p.v_ss, p.v_ss, v_off, true, x);
    } else {
      ld.template keys<BK>(at, kp + (long)t * BK * p.k_ss, p.k_ss, k_off, false, x);
      ld.template keys<BK>(at + IMG, vp + (long)t * BK * p.v_ss, p.v_ss, v_off, false, x);
    }
  };
#pragma unroll
  for (int i = 0; i <= NBUF; ++i) words(t0 + i, w[i]);
#pragma unroll
  for (int i = 0; i < NBUF - 1; ++i)
    if (t0 + i < t1) stage(t0 + i, lds + i * 2 * IMG, w[i]);
  xa_settle();
  int use = 0, fill = (NBUF - 1) * 2 * IMG;
  for (int t = t0; t < t1; ++t) {
    if (NBUF == 3 && t + 1 < t1) xa_landed<PER>();
    else xa_landed<0>();
    if (t + NBUF - 1 < t1) stage(t + NBUF - 1, lds + fill, w[NBUF - 1]);
    if (busy) compute(t, lds + use, lds + use + IMG, w[0]);
    use = use + 2 * IMG == K::RING ? 0 : use + 2 * IMG;
    fill = fill + 2 * IMG == K::RING ? 0 : fill + 2 * IMG;
#pragma unroll
    for (int j = 0; j < NBUF; ++j)
#pragma unroll
      for (int i = 0; i < NW; ++i) w[j][i] = w[j + 1][i];
    words(t + NBUF + 1, w[NBUF]);
  }
}
// scores of keys that do not count: minus infinity
__device__ __forceinline__ void xa_mask(f32x16& s, unsigned w, int h) {
  const unsigned wl = w >> (4 * h);
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = (wl >> (8 * (i / 4) + i % 4)) & 1u ? s[i] : -INFINITY;
}
// this wave's words of a tile
template <int KW, int NW>
__device__ __forceinline__ void xa_mine(const unsigned (&w)[NW], int kw, unsigned (&m)[NW / KW]) {
#pragma unroll
  for (int u = 0; u < NW / KW; ++u) {
    m[u] = w[u];
#pragma unroll
    for (int k = 1; k < KW; ++k) m[u] = kw == k ? w[k * (NW / KW) + u] : m[u];
  }
}

// ------------------------------------------------------------------------------------------------ forward
// Many rows are bound by the matrix and vector units together: 32 x 32 scores of a head of 64 are 8 matrix instructions (256 cycles) and a dozen vector
// instructions a score, the exponential at a quarter of the others' rate.  8 x 8 heads of 64, 2048 x 2048: 84 us, 0.82 PFLOP/s; left out one at a time,
// staging, exponentials, masks or either product give about a tenth each.  4 x 8 heads of 64, 2560 rows x 0 to 5120 keys: 91 us, 0.59 PFLOP/s, and 85
// with as many keys in entries of equal length: 640 workgroups of two and two waves, of which all with keys are resident at once.
// Few rows are bound by memory and latency: one row, 8 entries of 0 to 2560 keys x 8 heads of 128: 15 us and 4.5 for the join (42 MB, 8.5 us at a large
// copy's rate); one tile of keys alone takes 7.4 us, further ones 2.1 each.
// Waves for each SIMD that LDS allows and the registers are shared by (backward of few rows, 8 x 8 heads x 20480 keys x 64 with three: 81 us, with two,
// which LDS allows, and no spills: 69.5; heads of 128: two 129, one 72.5; dk and
// dv of 4 x 8 heads of 128, 2560 rows x 5120 keys: two with spills 640, one 572)
template <int DT> struct XaWaves {
  static constexpr int FWD = DT == 1 ? 4 : DT == 2 ? 3 : 2, BWD = DT > 2 ? 2 : 3, FEW = DT == 1 ? 3 : DT == 2 ? 2 : 1, DKV = DT == 4 ? 1 : BWD;
};

template <typename T, int DT, int KW>
__global__ __launch_bounds__(256, XaWaves<DT>::FWD) void xattn_fwd_kernel(XaParams p) {
  typedef typename Vec8<T>::type V;
  constexpr int SUB = XaKeys<DT, KW>::SUB, NW = XaKeys<DT, KW>::NW, PITCH = XaImg<DT>::PITCH;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int tile, b, hk, pair, t0, t1;
  if (!xa_place_run(p, XaKeys<DT, KW>::BK, tile, b, hk, pair, t0, t1)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = b * p.hkv + hk, h = lane >> 5;
  const int kw = wave % KW, r0 = tile * (128 / KW) + (wave / KW) * 32, r = r0 + (lane & 31);
  const XaAddr<DT> ad(lane);

  V qf[2 * DT];
  xa_load_row<DT, T>(qf, (const T*)p.q + (long)b * p.q_bs + (long)(hk * p.grp) * p.q_hs + (r < p.rows ? xa_row_off(p, r, p.q_ss, p.q_hs) : 0), r < p.rows, p.d, h);
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = XA_M0, l = 0.f;

  xa_over_keys<T, DT, KW>(p, lds, b, hk, t0, t1, r0 < p.rows, [&](int, const uint8_t* ki, const uint8_t* vi, const unsigned (&words)[NW]) {
    unsigned w[SUB], any = 0, all = ~0u;
    xa_mine<KW, NW>(words, kw, w);
#pragma unroll
    for (int u = 0; u < SUB; ++u) any |= w[u], all &= w[u];
    if (any == 0) return;
    ki += kw * SUB * 32 * PITCH;
    vi += kw * SUB * 32 * PITCH;
    f32x16 s[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
    for (int st = 0; st < 2 * DT; ++st)
#pragma unroll
      for (int u = 0; u < SUB; ++u) s[u] = mfma32(xa_frag<V>(ki + u * 32 * PITCH, ad.row[st]), qf[st], s[u]);
    if (all != ~0u) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) xa_mask(s[u], w[u], h);
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
    mx = xa_halves_max(mx) * p.scale_log2 - XaRange<T>::FWD;
    if (__any(mx > m + XA_SLACK)) {
      const float mn = fmaxf(m, mx), a = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= a;
#pragma unroll
      for (int t2 = 0; t2 < DT; ++t2)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t2][i] *= a;
    }
    XaSecond<T, KW == 4> pb[SUB];
    float part[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      part[u] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[u][i] * p.scale_log2 - m);
        part[u] += e;
        pb[u].set(i, e);
      }
      l += part[u];
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
          const V f = xa_frag_tr<V>(vi + (u * 32 + c * 16) * PITCH, ad.tr[t2][0], ad.tr[t2][1]);
          if constexpr (KW == 4) o[t2] = mfma32(f, pb[u].v[2 + c], o[t2]);
          o[t2] = mfma32(f, pb[u].v[c], o[t2]);
        }
  });
  l = xa_halves_sum(l);
  float weight[KW];              // of the waves that share these rows
  if constexpr (KW > 1) {
    __syncthreads();             // nobody reads the tiles any more
    float* st = (float*)lds;
    st[wave * 128 + lane] = m;
    st[wave * 128 + 64 + lane] = l;
    __syncthreads();
    const float* all = st + (wave / KW) * KW * 128 + lane;
    m = XA_M0;
#pragma unroll
    for (int k = 0; k < KW; ++k) m = fmaxf(m, all[k * 128]);
    l = 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      weight[k] = __builtin_amdgcn_exp2f(all[k * 128] - m);
      l += all[k * 128 + 64] * weight[k];
    }
  } else {
    weight[0] = 1.f;
  }
  const bool rok = r < p.rows, none = l == 0.f;
  const float inv = none ? 0.f : 1.f / l, L = m + log2f(l);
#pragma unroll
  for (int k = 0; k < KW; ++k) weight[k] *= inv;
  const long row = (long)bh * p.rows + r, prow = ((long)pair * p.hkv + hk) * p.rows + r;
  if (rok && h == 0 && kw == 0) {
    if (p.pairs) p.part_lse[prow] = none ? -INFINITY : L;
    else if (p.lse) p.lse[row] = none ? INFINITY : L;
  }
  const int tok = rok ? r / p.grp : 0, g = rok ? r % p.grp : 0;
  const long oo = (((long)b * p.sq + tok) * p.hq + hk * p.grp + g) * p.d;
  xa_gather<DT, KW>(o, weight, lds, wave, [&](int q, float (&v)[8]) {
    if (p.pairs) {
      if (rok && !none) xa_store8(p.part + prow * p.d, v, q, h, p.d);      // a run without keys leaves nothing: nobody reads it
      return;
    }
    xa_store8<T>((T*)p.o + oo, v, q, h, p.d, rok);
    if (p.o_lo) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] -= (float)(T)v[i];
      xa_store8<T>((T*)p.o_lo + oo, v, q, h, p.d, rok);
    }
  });
}

// Partial results, joined by one wave per row: groups of L lanes (8 columns each) take turns, so that the loads of a row are under way together, and
// the groups are added in a fixed order.
template <int DT> struct XaJoin { static constexpr int L = DT == 1 ? 4 : DT == 2 ? 8 : 16; };
template <int L>
__device__ __forceinline__ float xa_groups_sum(float v) {
#pragma unroll
  for (int o = L; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// o of a row = sum over runs of 2^(L_run - L) o_run.  bk: keys of a tile
template <typename T, int DT>
__global__ __launch_bounds__(256) void xattn_join_kernel(XaParams p, int bk) {
  const long rows = (long)p.b * p.hkv * p.rows, row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  constexpr int L = XaJoin<DT>::L;
  const int lane = threadIdx.x & 63, c = lane % L * 8;
  if (row >= rows) return;
  const int bh = (int)(row / p.rows), b = bh / p.hkv, hk = bh % p.hkv, r = (int)(row % p.rows);
  int first = b * p.nsplit, n = p.nsplit;
  if (p.ragged) {
    const XaShares s = xa_shares(p, bk);
    first = __builtin_amdgcn_readlane(s.first, __builtin_amdgcn_readfirstlane(b));
    n = __builtin_amdgcn_readlane(s.n, __builtin_amdgcn_readfirstlane(b));
  }
  const long at = ((long)first * p.hkv + hk) * p.rows + r, step = (long)p.hkv * p.rows;     // this row of the runs
  float mx = -INFINITY;
  for (int s = lane; s < n; s += 64) {
    const float x = p.part_lse[at + s * step];
    mx = x > mx || x != x ? x : mx;      // a NaN stays
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float x = __shfl_xor(mx, o, 64);
    mx = x > mx || x != x ? x : mx;
  }
  float sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (mx != -INFINITY) {
#pragma unroll 4
    for (int s = lane / L; s < n; s += 64 / L) {
      const float lse = p.part_lse[at + s * step], w = exp2f(lse - mx);
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (c < p.d) load8(v, p.part + (at + s * step) * p.d + c);
      sum += w;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += lse == -INFINITY ? 0.f : v[j] * w;      // a run without keys has left nothing
    }
    sum = xa_groups_sum<L>(sum);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = xa_groups_sum<L>(acc[j]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? INFINITY : mx + log2f(sum);
  if (c >= p.d || lane >= L) return;
  const int s = r / p.grp, g = r % p.grp;
  const long oo = (((long)b * p.sq + s) * p.hq + hk * p.grp + g) * p.d + c;
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
// delta of a row by itself, for a pass without the gradient of q (whose kernel forms it otherwise).  16 lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void xattn_delta_kernel(XaParams p) {
  const long rows = (long)p.b * p.hkv * p.rows, row = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int c = (threadIdx.x & 15) * 8;
  float t = 0.f;
  if (row < rows && c < p.d) {
    const int bh = (int)(row / p.rows), r = (int)(row % p.rows), s = r / p.grp, g = r % p.grp, b = bh / p.hkv, hq = (bh % p.hkv) * p.grp + g;
    const long oo = (((long)b * p.sq + s) * p.hq + hq) * p.d + c;
    float hi[8], lo[8], d[8];
    load8(hi, (const T*)p.o + oo);
    load8(lo, (const T*)p.o_lo + oo);
    load8(d, (const T*)p.d_o + (long)b * p.o_bs + (long)s * p.o_ss + (long)hq * p.o_hs + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) t += (hi[j] + lo[j]) * d[j];
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if (row < rows && (threadIdx.x & 15) == 0) p.delta[row] = t;
}

// delta = sum_d do o of this lane's row (do in df), from o as it was before its rounding (o + what the rounding left over): with few keys the
// difference dp - delta cancels, and o's rounding alone would be most of it
template <typename T, int DT>
__device__ __forceinline__ float xa_delta(const XaParams& p, const typename Vec8<T>::type (&df)[2 * DT], int b, int hk, int r, bool rok, int h) {
  const int tok = rok ? r / p.grp : 0, g = rok ? r % p.grp : 0;
  const long oo = (((long)b * p.sq + tok) * p.hq + hk * p.grp + g) * p.d;
  typename Vec8<T>::type oh[2 * DT], ol[2 * DT];
  xa_load_row<DT, T>(oh, (const T*)p.o + oo, rok, p.d, h);
  xa_load_row<DT, T>(ol, (const T*)p.o_lo + oo, rok, p.d, h);
  float delta = 0.f;
#pragma unroll
  for (int st = 0; st < 2 * DT; ++st)
#pragma unroll
    for (int j = 0; j < 8; ++j) delta += ((float)oh[st][j] + (float)ol[st][j]) * (float)df[st][j];
  return xa_halves_sum(delta);
}

// the gradient of row r of q (acc times `out`, summed over the KW waves that share it), or this split's part of it
template <typename T, int DT, int KW>
__device__ __forceinline__ void xa_store_dq(const XaParams& p, const f32x16 (&acc)[DT], float out, uint8_t* lds, int wave, int b, int hk, int split, int r, int h) {
  const bool rok = r < p.rows;
  const long prow = ((long)split * p.b * p.hkv + (long)b * p.hkv + hk) * p.rows + r;
  const int tok = rok ? r / p.grp : 0, g = rok ? r % p.grp : 0;
  const long oo = (((long)b * p.sq + tok) * p.hq + hk * p.grp + g) * p.d;
  float weight[KW];
  if constexpr (KW > 1) {        // fp16: each wave has a factor of its own
    __syncthreads();
    float* st = (float*)lds;
    st[wave * 64 + (threadIdx.x & 63)] = out;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KW; ++k) weight[k] = st[((wave / KW) * KW + k) * 64 + (threadIdx.x & 63)];
  } else {
    weight[0] = out;
  }
  xa_gather<DT, KW>(acc, weight, lds, wave, [&](int q, float (&v)[8]) {
    if (p.nsplit == 1) xa_store8<T>((T*)p.dq + oo, v, q, h, p.d, rok);
    else if (rok) xa_store8(p.part + prow * p.d, v, q, h, p.d);
  });
}

// ------------------------------------------------------------------------------------------------ backward: dq
// the forward kernel's shape: s^T and dp^T with a lane per row, dq^T = k^T ds^T, k read from LDS both ways.  Three products for the forward pass's two:
// 4 x 8 heads of 64, 2560 rows x 0 to 5120 keys 108 us, 0.75 PFLOP/s (entries of equal length 103).  As in the forward pass every fragment that is read
// from LDS feeds one matrix instruction: by count the two are as busy as each other.
template <typename T, int DT, int KW>
__global__ __launch_bounds__(256, XaWaves<DT>::BWD) void xattn_dq_kernel(XaParams p) {
  typedef typename Vec8<T>::type V;
  constexpr int SUB = XaKeys<DT, KW>::SUB, NW = XaKeys<DT, KW>::NW, PITCH = XaImg<DT>::PITCH;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int tile, b, hk, split;
  if (!xa_place(p, tile, b, hk, split)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = b * p.hkv + hk, h = lane >> 5;
  const int kw = wave % KW, r0 = tile * (128 / KW) + (wave / KW) * 32, r = r0 + (lane & 31);
  const bool rok = r < p.rows;
  const XaAddr<DT> ad(lane);
  const long row = (long)bh * p.rows + r;
  V qf[2 * DT], df[2 * DT];
  xa_load_row<DT, T>(qf, (const T*)p.q + (long)b * p.q_bs + (long)(hk * p.grp) * p.q_hs + (rok ? xa_row_off(p, r, p.q_ss, p.q_hs) : 0), rok, p.d, h);
  xa_load_row<DT, T>(df, (const T*)p.d_o + (long)b * p.o_bs + (long)(hk * p.grp) * p.o_hs + (rok ? xa_row_off(p, r, p.o_ss, p.o_hs) : 0), rok, p.d, h);
  float ex = XaRange<T>::BWD, L = (rok ? p.lse_in[row] : INFINITY) - ex;     // p times 2^ex
  const float delta = xa_delta<T, DT>(p, df, b, hk, r, rok, h);      // left for the gradients of k and v too (every split the same value)
  if (rok && h == 0 && kw == 0) p.delta[row] = delta;
  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;

  const int nt = (xa_len(p, b) + XaKeys<DT, KW>::BK - 1) / XaKeys<DT, KW>::BK;
  const int t0 = (int)((long)nt * split / p.nsplit), t1 = (int)((long)nt * (split + 1) / p.nsplit);
  xa_over_keys<T, DT, KW>(p, lds, b, hk, t0, t1, r0 < p.rows, [&](int, const uint8_t* ki, const uint8_t* vi, const unsigned (&words)[NW]) {
    unsigned w[SUB], any = 0;
    xa_mine<KW, NW>(words, kw, w);
#pragma unroll
    for (int u = 0; u < SUB; ++u) any |= w[u];
    if (any == 0) return;
    ki += kw * SUB * 32 * PITCH;
    vi += kw * SUB * 32 * PITCH;
    f32x16 s[SUB], dp[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = dp[u][i] = 0.f;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int st = 0; st < 2 * DT; ++st) {
        s[u] = mfma32(xa_frag<V>(ki + u * 32 * PITCH, ad.row[st]), qf[st], s[u]);
        dp[u] = mfma32(xa_frag<V>(vi + u * 32 * PITCH, ad.row[st]), df[st], dp[u]);
      }
    XaSecond<T, false> ds[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      if (w[u] != ~0u) xa_mask(s[u], w[u], h);
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[u][i] = __builtin_amdgcn_exp2f(s[u][i] * p.scale_log2 - L) * (dp[u][i] - delta);
    }
    if constexpr (XaRange<T>::NARROW) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const float before = ex;
        if (xa_narrow<DT>(dp[u], acc, ex)) {
          L += before - ex;
          const float f = exp2f(ex - before);
#pragma unroll
          for (int k = 0; k < SUB; ++k)
            if (k != u) dp[k] *= f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[u].set(i, dp[u][i]);
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
          const V f = xa_frag_tr<V>(ki + (u * 32 + c * 16) * PITCH, ad.tr[t2][0], ad.tr[t2][1]);
          acc[t2] = mfma32(f, ds[u].v[c], acc[t2]);
        }
  });
  xa_store_dq<T, DT, KW>(p, acc, p.scale * exp2f(-ex), lds, wave, b, hk, split, r, h);
}

// dq of a row = sum over splits
template <typename T, int DT>
__global__ __launch_bounds__(256) void xattn_dq_join_kernel(XaParams p) {
  const long rows = (long)p.b * p.hkv * p.rows, row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  constexpr int L = XaJoin<DT>::L;
  const int lane = threadIdx.x & 63, c = lane % L * 8;
  if (row >= rows) return;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = lane / L; s < p.nsplit; s += 64 / L) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < p.d) load8(v, p.part + (s * rows + row) * p.d + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += v[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = xa_groups_sum<L>(acc[j]);
  if (c >= p.d || lane >= L) return;
  const int bh = (int)(row / p.rows), r = (int)(row % p.rows), s = r / p.grp, g = r % p.grp;
  store8((T*)p.dq + (((long)(bh / p.hkv) * p.sq + s) * p.hq + (bh % p.hkv) * p.grp + g) * p.d + c, acc, 8);
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv
// Each wave keeps 32 keys (k, v as second operands in registers, dk^T and dv^T as accumulators) and walks the rows: s = q k^T and
// dp = do v^T with a lane per key, then dv^T += do^T p and dk^T += q^T ds with q and do read from LDS both ways.  A lane's key touches its own
// column of the products alone, so a masked key needs nothing inside the loop: zeros are written for it at the end.  Four products: at the same sizes
// 136 us, 0.79 PFLOP/s; 640 workgroups with keys, of one length, two or three to a CU.  Bound by LDS, by count: a step of 32 x 32 of 64 columns is 16
// matrix instructions (512 cycles) beside 16 reads of 16 bytes a lane, half of them for L and delta, and 16 transposing ones of 8: 96 KB for the four
// SIMDs, 768 cycles at 128 bytes a cycle.
template <int DT> struct XaRows {      // tiles of rows: 64, one for each lane of the wave that brings their L or delta; two buffers
  static constexpr int BR = 64, IMG = BR * XaImg<DT>::PITCH, BUF = 2 * IMG + 2 * BR * 4, BYTES = 2 * BUF;
};
template <typename T, int DT>
__global__ __launch_bounds__(256, XaWaves<DT>::DKV) void xattn_dkv_kernel(XaParams p) {
  typedef typename Vec8<T>::type V;
  typedef XaRows<DT> R;
  constexpr int BR = R::BR, IMG = R::IMG, BUF = R::BUF;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int tile, b, hk, split;
  if (!xa_place(p, tile, b, hk, split)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = b * p.hkv + hk, h = lane >> 5;
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
  float ex = XaRange<T>::BWD, less = 1.f;      // ds times 2^ex, in p's factor times `less`

  const XaLoader<DT, T> ld(p.d);
  const bool even = XaLoader<DT, T>::ROWS % p.grp == 0, full = p.d == XaImg<DT>::CH * 8;
  const int lr = ld.r / p.grp, lg = ld.r % p.grp;
  const unsigned q_off = (unsigned)(lr * (int)p.q_ss + lg * (int)p.q_hs + ld.c) * 2u, o_off = (unsigned)(lr * (int)p.o_ss + lg * (int)p.o_hs + ld.c) * 2u;
  auto stage = [&](int t, uint8_t* at) {
    if (full && even && (t + 1) * BR <= p.rows) {
      ld.template rows<BR>(at, p, qp, p.q_ss, p.q_hs, q_off, true, true, t * BR);
      ld.template rows<BR>(at + IMG, p, dp_, p.o_ss, p.o_hs, o_off, true, true, t * BR);
    } else {
      ld.template rows<BR>(at, p, qp, p.q_ss, p.q_hs, q_off, even, false, t * BR);
      ld.template rows<BR>(at + IMG, p, dp_, p.o_ss, p.o_hs, o_off, even, false, t * BR);
    }
    if (wave < 2) {      // L and delta of the rows, by DMA too; rows that are none get L = infinity and so p = 0
      const int row = t * BR + lane;
      const float* src = wave ? (const float*)g_zero_line_xa : &g_inf_xa;
      if (row < p.rows) src = (wave ? p.delta : p.lse_in) + (long)bh * p.rows + row;
      xa_dma4(at + 2 * IMG + wave * (BR * 4), src);
    }
  };
  auto compute = [&](int t, const uint8_t* qi) {
    const uint8_t* di = qi + IMG;
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
      XaSecond<T, false> pb, sb;
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 L = *(const f32x4*)(st + u * 32 + 2 * i + 4 * h), dl = *(const f32x4*)(st + BR + u * 32 + 2 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = __builtin_amdgcn_exp2f(s[i + j] * p.scale_log2 - (XaRange<T>::NARROW ? L[j] - XaRange<T>::BWD : L[j]));
          pb.set(i + j, e);
          dp[i + j] = e * (dp[i + j] - dl[j]);
          if constexpr (XaRange<T>::NARROW) dp[i + j] *= less;
        }
      }
      if constexpr (XaRange<T>::NARROW) {
        if (xa_narrow<DT>(dp, dk, ex)) less = exp2f(ex - XaRange<T>::BWD);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) sb.set(i, dp[i]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
          const int off = (u * 32 + c * 16) * XaImg<DT>::PITCH;
          const V df = xa_frag_tr<V>(di + off, ad.tr[t2][0], ad.tr[t2][1]), qf = xa_frag_tr<V>(qi + off, ad.tr[t2][0], ad.tr[t2][1]);
          dv[t2] = mfma32(df, pb.v[c], dv[t2]);
          dk[t2] = mfma32(qf, sb.v[c], dk[t2]);
        }
    }
  };
  if (t0 < t1) stage(t0, lds);
  xa_settle();
  for (int t = t0; t < t1; ++t) {
    xa_landed<0>();
    if (t + 1 < t1) stage(t + 1, lds + ((t + 1 - t0) & 1) * BUF);
    if (w) compute(t, lds + ((t - t0) & 1) * BUF);
  }
  if (key >= p.sk) return;
  const float k_out = p.scale * exp2f(-ex), v_out = exp2f(-XaRange<T>::BWD);
  const long oo = (((long)b * p.sk + key) * p.hkv + hk) * p.d;
  const long all = (long)p.b * p.sk * p.hkv * p.d;
#pragma unroll
  for (int t = 0; t < DT; ++t) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {     // a key that does not count: zeros, whatever the products made of its column
      dk[t][i] = kok ? dk[t][i] * k_out : 0.f;
      dv[t][i] = kok ? dv[t][i] * v_out : 0.f;
    }
    if (p.nsplit > 1) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int c = 32 * t + 2 * i + 4 * h;
        if (c < p.d) {
          *(f32x4*)(p.part + (2L * split) * all + oo + c) = f32x4{dk[t][i], dk[t][i + 1], dk[t][i + 2], dk[t][i + 3]};
          *(f32x4*)(p.part + (2L * split + 1) * all + oo + c) = f32x4{dv[t][i], dv[t][i + 1], dv[t][i + 2], dv[t][i + 3]};
        }
      }
    } else {
      xa_store<T>((T*)p.dk + oo, dk[t], t, h, p.d, true);
      xa_store<T>((T*)p.dv + oo, dv[t], t, h, p.d, true);
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward, up to 32 rows
// All rows are one tile, so a tile of keys is done with once read: its dk and dv are complete, and dq is summed on.  One pass over k and v, which
// are the work (8 x 8 heads of 32, 15 rows x 0 to 20480 keys: dq and dk / dv one after the other 105 us, here 67: 252 MB with the zeros of keys that
// do not count, 3.8 TB/s; a large copy's rate would be 51 us for forward and backward together).  Each wave takes 32 keys of a tile both
// ways round from the same fragments, operands exchanged: a lane per row for ds^T and dq, a lane per key for p, ds and dk / dv.
template <int DT> struct XaFew {       // key tiles, then the images of do and q, then L and delta of the rows
  static constexpr int ROWS_IMG = 32 * XaImg<DT>::PITCH, AT = XaKeys<DT, 4>::BYTES, BYTES = AT + 2 * ROWS_IMG + 2 * 32 * 4;
};
template <typename T, int DT>
__global__ __launch_bounds__(256, XaWaves<DT>::FEW) void xattn_bwd_few_kernel(XaParams p) {
  typedef typename Vec8<T>::type V;
  constexpr int NW = XaKeys<DT, 4>::NW, PITCH = XaImg<DT>::PITCH;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int tile, b, hk, split;
  if (!xa_place(p, tile, b, hk, split)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = b * p.hkv + hk, h = lane >> 5, r = lane & 31;
  const bool rok = r < p.rows;
  const XaAddr<DT> ad(lane);
  const long row = (long)bh * p.rows + r;
  V qf[2 * DT], df[2 * DT];
  xa_load_row<DT, T>(qf, (const T*)p.q + (long)b * p.q_bs + (long)(hk * p.grp) * p.q_hs + (rok ? xa_row_off(p, r, p.q_ss, p.q_hs) : 0), rok, p.d, h);
  xa_load_row<DT, T>(df, (const T*)p.d_o + (long)b * p.o_bs + (long)(hk * p.grp) * p.o_hs + (rok ? xa_row_off(p, r, p.o_ss, p.o_hs) : 0), rok, p.d, h);
  const float delta = xa_delta<T, DT>(p, df, b, hk, r, rok, h), L0 = rok ? p.lse_in[row] : INFINITY;
  float ex = XaRange<T>::BWD, L = L0 - ex;
  uint8_t *di = lds + XaFew<DT>::AT, *qi = di + XaFew<DT>::ROWS_IMG;
  float* st = (float*)(qi + XaFew<DT>::ROWS_IMG);
  if (wave == 0) {       // the rows once more as images, and their statistics, for the other way round
#pragma unroll
    for (int e = 0; e < 2 * DT; ++e) {
      *(V*)(di + ad.row[e]) = df[e];
      *(V*)(qi + ad.row[e]) = qf[e];
    }
    if (h == 0) {
      st[r] = L0 - XaRange<T>::BWD;
      st[32 + r] = delta;
    }
  }
  __syncthreads();
  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;

  const int nt = (p.sk + XaKeys<DT, 4>::BK - 1) / XaKeys<DT, 4>::BK;       // tiles without a key that counts too: every key gets its gradient
  const int t0 = (int)((long)nt * split / p.nsplit), t1 = (int)((long)nt * (split + 1) / p.nsplit);
  xa_over_keys<T, DT, 4>(p, lds, b, hk, t0, t1, true, [&](int t, const uint8_t* ki, const uint8_t* vi, const unsigned (&words)[NW]) {
    unsigned w[1];
    xa_mine<4, NW>(words, wave, w);
    const int key = t * 128 + wave * 32 + r;
    const long oo = (((long)b * p.sk + key) * p.hkv + hk) * p.d;
    const bool in = key < p.sk, kok = (w[0] >> r) & 1u;
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int t2 = 0; t2 < DT; ++t2)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[t2][i] = dv[t2][i] = 0.f;
    if (w[0] != 0) {
      ki += wave * 32 * PITCH;
      vi += wave * 32 * PITCH;
      f32x16 s, dp, s2, d2;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = s2[i] = d2[i] = 0.f;
#pragma unroll
      for (int e = 0; e < 2 * DT; ++e) {
        const V kf = xa_frag<V>(ki, ad.row[e]), vf = xa_frag<V>(vi, ad.row[e]);
        s = mfma32(kf, qf[e], s);
        dp = mfma32(vf, df[e], dp);
        s2 = mfma32(qf[e], kf, s2);
        d2 = mfma32(df[e], vf, d2);
      }
      // a lane per row: dq
      if (w[0] != ~0u) xa_mask(s, w[0], h);
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = __builtin_amdgcn_exp2f(s[i] * p.scale_log2 - L) * (dp[i] - delta);
      if constexpr (XaRange<T>::NARROW) {
        const float before = ex;
        if (xa_narrow<DT>(dp, acc, ex)) L += before - ex;
      }
      XaSecond<T, true> ds, pb, sb;
#pragma unroll
      for (int i = 0; i < 16; ++i) ds.set(i, dp[i]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
          const V f = xa_frag_tr<V>(ki + c * 16 * PITCH, ad.tr[t2][0], ad.tr[t2][1]);
          acc[t2] = mfma32(f, ds.v[2 + c], acc[t2]);
          acc[t2] = mfma32(f, ds.v[c], acc[t2]);
        }
      // a lane per key: dk, dv
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 Lr = *(const f32x4*)(st + 2 * i + 4 * h), dl = *(const f32x4*)(st + 32 + 2 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = __builtin_amdgcn_exp2f(s2[i + j] * p.scale_log2 - Lr[j]);
          pb.set(i + j, e);
          d2[i + j] = e * (d2[i + j] - dl[j]);
        }
      }
      float k_out = p.scale;
      if constexpr (XaRange<T>::NARROW) {
        float kx = XaRange<T>::BWD;
        xa_narrow<DT>(d2, dk, kx);
        k_out *= exp2f(-kx);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) sb.set(i, d2[i]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t2 = 0; t2 < DT; ++t2) {
          const V f = xa_frag_tr<V>(di + c * 16 * PITCH, ad.tr[t2][0], ad.tr[t2][1]), g = xa_frag_tr<V>(qi + c * 16 * PITCH, ad.tr[t2][0], ad.tr[t2][1]);
          dv[t2] = mfma32(f, pb.v[2 + c], dv[t2]);
          dv[t2] = mfma32(f, pb.v[c], dv[t2]);
          dk[t2] = mfma32(g, sb.v[2 + c], dk[t2]);
          dk[t2] = mfma32(g, sb.v[c], dk[t2]);
        }
      const float v_out = exp2f(-XaRange<T>::BWD);
#pragma unroll
      for (int t2 = 0; t2 < DT; ++t2)
#pragma unroll
        for (int i = 0; i < 16; ++i) {     // a key that does not count: zeros, whatever the products made of its column
          dk[t2][i] = kok ? dk[t2][i] * k_out : 0.f;
          dv[t2][i] = kok ? dv[t2][i] * v_out : 0.f;
        }
    }
    if (p.dk) {
#pragma unroll
      for (int t2 = 0; t2 < DT; ++t2) {
        xa_store<T>((T*)p.dk + oo, dk[t2], t2, h, p.d, in);
        xa_store<T>((T*)p.dv + oo, dv[t2], t2, h, p.d, in);
      }
    }
  });
  if (!p.dq) return;
  xa_store_dq<T, DT, 4>(p, acc, p.scale * exp2f(-ex), lds, wave, b, hk, split, r, h);
}

// dk and dv = sums over the splits of the rows, in their order; the splits lie 2 * all floats apart, dk and dv in turn
template <typename T>
__global__ __launch_bounds__(256) void xattn_dkv_join_kernel(XaParams p, long all) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= 2 * all) return;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8];
  for (int s = 0; s < p.nsplit; ++s) {
    load8(v, p.part + 2L * s * all + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += v[j];
  }
  store8(i < all ? (T*)p.dk + i : (T*)p.dv + (i - all), acc, 8);
}

// ------------------------------------------------------------------------------------------------ launches
// How the work is cut, from sizes alone, so that the workspace query and the launch agree.
struct XaPlan {
  int kw, tiles, bk;           // forward and dq
  int fsplit, pairs;           // forward: runs of an entry (without lengths), of all entries (0: not cut)
  bool ragged;
  int nsplit;                  // dq
  int ktiles, ksplit;          // dk, dv
};
static int xa_clamp(long v, long lo, long hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }
static XaPlan xa_plan(const RtpXattn* a) {
  XaPlan pl;
  const long rows = (long)a->sq * (a->hq / a->hkv), bh = (long)a->b * a->hkv;
  // Up to 32 rows the four waves of a workgroup split the keys: with few rows the keys are the work.  Two and two up to 64 rows, and where four
  // groups of rows would leave fewer than four workgroups to a CU (4 x 2560 rows x 8 heads, 640 workgroups: forward 99 us, two and two 84).
  const long wide = rtp_div_up(rows, 128) * bh;
  pl.kw = rows <= 32 ? 4 : rows <= 64 || wide < 1024 ? 2 : 1;
  pl.tiles = rtp_div_up(rows, 128 / pl.kw);
  const long wgs = pl.tiles * bh, nt = rtp_div_up(a->sk, pl.kw == 4 ? 128 : 64);
  pl.bk = pl.kw == 4 ? 128 : 64;
  // as many workgroups as run at once (LDS: two for each CU, one with four waves on keys of over 64 columns, three below 32); a split of dq has at
  // least four tiles, or its partial results cost as much as they save
  const long slots = pl.kw < 4 ? 512 : a->d > 64 ? 256 : a->d > 32 ? 512 : 768;
  pl.nsplit = xa_clamp(slots / (wgs > 0 ? wgs : 1), 1, nt / 4 > 1 ? nt / 4 : 1);
  pl.fsplit = xa_clamp(slots / (wgs > 0 ? wgs : 1), 1, nt / XA_RUN > 1 ? nt / XA_RUN : 1);
  pl.ragged = pl.fsplit > 1 && a->key_lens && a->b > 1 && a->b <= 64;
  const long most = pl.fsplit > 1 ? slots / ((long)pl.tiles * a->hkv) : 0;       // at least two for each entry
  pl.pairs = pl.fsplit == 1 ? 0 : !pl.ragged ? a->b * pl.fsplit : xa_clamp(most, 1, a->b * ((nt + XA_RUN - 1) / XA_RUN));
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
  const long bh = (long)a->b * a->hkv;
  if (bh >= (1L << 28) || !rtp_launchable((bh * pl.nsplit + 64) * pl.tiles, 256) || !rtp_launchable((bh * pl.ksplit + 64) * pl.ktiles, 256) ||
      !rtp_launchable(bh * rows, 16) || !rtp_launchable((long)a->b * xa_words(a->sk), 32))
    return RTP_ERR_SHAPE;
  if (!(a->scale > 0.f) || a->scale > 2e38f) return RTP_ERR_SHAPE;       // times log2(e) still finite
  return RTP_OK;
}
static bool xa_aligned(const void* p, long bs, long ss, long hs) { return !((size_t)p & 15) && !(bs & 7) && !(ss & 7) && !(hs & 7); }
// offsets inside a staged step are 32 bits: up to 64 tokens and the heads of a group
static bool xa_near(const RtpXattn* a, long ss, long hs) {
  const long grp = a->hq / a->hkv;
  return ss >= 0 && hs >= 0 && ss <= (1L << 23) && hs * grp <= (1L << 28);
}

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
static int xa_blocks(XaParams& p) {
  // `near` heads together, where one tile has all rows and eight groups or more are left for each XCD
  p.near = 1;
  while (p.tiles == 1 && p.near * 2 * p.d <= 64 && p.hkv % (p.near * 2) == 0 && p.units / (p.near * 2) >= 64) p.near *= 2;
  return (p.units / p.near + 7) / 8 * 8 * p.near * p.tiles;
}
static int xa_grid(XaParams& p, int tiles, int nsplit) {
  p.tiles = tiles;
  p.nsplit = nsplit;
  p.units = p.b * p.hkv * nsplit;
  return xa_blocks(p);
}

extern "C" long rtp_xattn_workspace_bytes(const RtpXattn* a, int backward) {
  if (xa_check(a) != RTP_OK) return -1;
  const XaPlan pl = xa_plan(a);
  const long rows = (long)a->b * a->sq * a->hq;
  const long n = a->key_mask && !backward ? xa_round((long)a->b * xa_words(a->sk) * 4) : 0;
  const long parts = (long)pl.pairs * a->sq * a->hq;
  if (!backward) return n + xa_round(parts * a->d * 4) + xa_round(parts * 4);
  const long q = pl.nsplit > 1 ? rows * pl.nsplit * a->d * 4 : 0;
  const long kv = pl.ksplit > 1 ? 2L * pl.ksplit * a->b * a->sk * a->hkv * a->d * 4 : 0;
  return xa_round(rows * 4) + xa_round(q > kv ? q : kv);   // dq and dk / dv run one after the other
}

extern "C" int rtp_xattn_row_waves(const RtpXattn* a) { return xa_check(a) == RTP_OK ? xa_plan(a).kw : -1; }

// where the masks' bits stand behind lse, for the backward pass
static unsigned* xa_kept(const RtpXattn* a, const float* lse) { return (unsigned*)lse + (((long)a->b * a->sq * a->hq + 63) & ~63L); }

static int xa_bits(const RtpXattn* a, XaParams& p, float* lse, uint8_t*& ws, hipStream_t st) {
  if (!a->key_mask || a->sk == 0) return RTP_OK;      // no keys: a launch of no workgroups would be an error
  p.bits = lse ? xa_kept(a, lse) : (unsigned*)ws;
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
static int xa_launch(K kernel, int grid, int bytes, std::atomic<bool>* once, hipStream_t st, const XaParams& p) {
  if (bytes > 65536 &&
      !rtp_once_per_device(once, [&] { return hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess; }))
    return RTP_ERR_LAUNCH;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), bytes, st, p);
  RTP_CHECK_LAUNCH();
  return RTP_OK;
}

template <typename T, int DT, int KW>
static int xa_fwd(int grid, hipStream_t st, const XaParams& p) {
  static std::atomic<bool> once[RTP_MAX_DEVICES];
  return xa_launch(xattn_fwd_kernel<T, DT, KW>, grid, XaKeys<DT, KW>::BYTES, once, st, p);
}
template <typename T, int DT, int KW>
static int xa_dq(int grid, hipStream_t st, const XaParams& p) {
  static std::atomic<bool> once[RTP_MAX_DEVICES];
  return xa_launch(xattn_dq_kernel<T, DT, KW>, grid, XaKeys<DT, KW>::BYTES, once, st, p);
}
template <typename T, int DT>
static int xa_dkv(int grid, hipStream_t st, const XaParams& p) {
  static std::atomic<bool> once[RTP_MAX_DEVICES];
  return xa_launch(xattn_dkv_kernel<T, DT>, grid, XaRows<DT>::BYTES, once, st, p);
}
template <typename T, int DT>
static int xa_bwd_few(int grid, hipStream_t st, const XaParams& p) {
  static std::atomic<bool> once[RTP_MAX_DEVICES];
  return xa_launch(xattn_bwd_few_kernel<T, DT>, grid, XaFew<DT>::BYTES, once, st, p);
}

extern "C" int rtp_xattn_forward(const RtpXattn* a, void* o, void* o_lo, float* lse, void* ws, long ws_bytes, void* stream) {
  const int rc = xa_check(a);
  if (rc != RTP_OK) return rc;
  if (a->b == 0 || a->sq == 0) return RTP_OK;
  if (!a->q || !o || (a->sk > 0 && (!a->k || !a->v)) || (!o_lo) != (!lse)) return RTP_ERR_SHAPE;
  if (!xa_aligned(a->q, a->q_bs, a->q_ss, a->q_hs) || !xa_aligned(a->k, a->k_bs, a->k_ss, a->k_hs) || !xa_aligned(a->v, a->v_bs, a->v_ss, a->v_hs) ||
      ((size_t)o & 15) || ((size_t)o_lo & 15) || ((size_t)ws & 255))
    return RTP_ERR_ALIGN;
  if (!xa_near(a, a->q_ss, a->q_hs) || !xa_near(a, a->k_ss, 0) || !xa_near(a, a->v_ss, 0)) return RTP_ERR_SHAPE;
  const long need = rtp_xattn_workspace_bytes(a, 0);
  if (ws_bytes < need || (need > 0 && !ws)) return RTP_ERR_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  RtpProfScope prof(RTP_FAM_POINTWISE, st);
  XaParams p = xa_params(a);
  uint8_t* at = (uint8_t*)ws;
  const int rb = xa_bits(a, p, lse, at, st);
  if (rb != RTP_OK) return rb;
  p.o = o; p.o_lo = o_lo; p.lse = lse;
  const XaPlan pl = xa_plan(a);
  int grid = xa_grid(p, pl.tiles, pl.fsplit);
  if (pl.pairs) {
    p.pairs = pl.pairs;
    p.ragged = pl.ragged;
    p.units = pl.pairs * a->hkv;
    grid = xa_blocks(p);
    p.part = (float*)at;
    p.part_lse = (float*)(at + xa_round((long)pl.pairs * a->sq * a->hq * a->d * 4));
  }
  return xa_types(a, [&](auto t, auto dt) {
    typedef decltype(t) T;
    constexpr int DT = decltype(dt)::value;
    const int r = pl.kw == 4 ? xa_fwd<T, DT, 4>(grid, st, p) : pl.kw == 2 ? xa_fwd<T, DT, 2>(grid, st, p) : xa_fwd<T, DT, 1>(grid, st, p);
    if (r != RTP_OK || !pl.pairs) return r;
    hipLaunchKernelGGL((xattn_join_kernel<T, DT>), dim3(rtp_div_up((long)a->b * a->sq * a->hq, 4)), dim3(256), 0, st, p, pl.bk);
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
  if (!xa_near(a, a->q_ss, a->q_hs) || !xa_near(a, a->k_ss, 0) || !xa_near(a, a->v_ss, 0) || !xa_near(a, o_ss, o_hs)) return RTP_ERR_SHAPE;
  if (ws_bytes < rtp_xattn_workspace_bytes(a, 1)) return RTP_ERR_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  RtpProfScope prof(RTP_FAM_POINTWISE, st);
  XaParams p = xa_params(a);
  uint8_t* at = (uint8_t*)ws;
  if (a->key_mask) p.bits = xa_kept(a, lse);
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
    auto join_dq = [&]() {
      if (pl.nsplit > 1) hipLaunchKernelGGL((xattn_dq_join_kernel<T, DT>), dim3(rtp_div_up(rows, 4)), dim3(256), 0, st, p);
      RTP_CHECK_LAUNCH();
      return RTP_OK;
    };
    if (pl.kw == 4) {
      const int grid = xa_grid(p, pl.tiles, pl.nsplit), r = xa_bwd_few<T, DT>(grid, st, p);
      return r != RTP_OK || !dq ? r : join_dq();
    }
    if (!dq) {
      hipLaunchKernelGGL((xattn_delta_kernel<T>), dim3(rtp_div_up(rows, 16)), dim3(256), 0, st, p);
      RTP_CHECK_LAUNCH();
    } else {
      const int grid = xa_grid(p, pl.tiles, pl.nsplit);
      int r = pl.kw == 2 ? xa_dq<T, DT, 2>(grid, st, p) : xa_dq<T, DT, 1>(grid, st, p);
      if (r == RTP_OK) r = join_dq();
      if (r != RTP_OK) return r;
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
