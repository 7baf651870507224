// Rows of class values: what the kernels over two models' class distributions share (toplogits.hip, distill.hip,
// verify.hip).  A row is one voxel's or one token's K class values; row r = (n, v) starts at n*sN + v*sV and its
// classes are sK apart, so one kernel takes channels-last voxels, channels-first volumes (sK = V) and vocabulary rows.
#pragma once
#include "common.h"

namespace devis {

constexpr int64_t MAX_CLASSES = (int64_t)1 << 30;      // class numbers, and a step past them, stay below 2^31

struct RowShape { int64_t sN, sV, sK, N, V; int K; };

__device__ __forceinline__ int64_t row_offset(const RowShape& s, int64_t r) {
  if (s.V == 1) return r * s.sN;
  const int64_t n = r / s.V;
  return n * s.sN + (r - n * s.V) * s.sV;
}

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }

// log2 of a positive sum to about 2^-25 absolute at the price of a fp32 logarithm: the exponent is taken off, so that the
// hardware logarithm's result is at most 1/2, and what rounding the sum to fp32 left over is added in first order.
__device__ __forceinline__ double log2_split(double x) {
  const float f = (float)x;
  float mant = __builtin_amdgcn_frexp_mantf(f);
  int e = __builtin_amdgcn_frexp_expf(f);
  const bool low = mant < 0.70710678f;
  mant = low ? 2.f * mant : mant;
  e -= low ? 1 : 0;
  const float left = (float)(x - (double)f) * __builtin_amdgcn_rcpf(f) * 1.4426950408889634f;
  return (double)e + ((double)__builtin_amdgcn_logf(mant) + (double)left);
}

// 2^y to about 1e-11 relative: 2^(y - n) by the exponential's series, nine terms of it at |y - n| ln 2 <= 0.35.  A dozen fp64
// operations, no more than a fp32 exponential with its argument split.
__device__ __forceinline__ double exp2_series(double y) {
  const double n = rint(fmin(fmax(y, -1050.), 1020.)), f = (y - n) * 0.6931471805599453;
  double e = 1. / 362880.;
  e = fma(e, f, 1. / 40320.);
  e = fma(e, f, 1. / 5040.);
  e = fma(e, f, 1. / 720.);
  e = fma(e, f, 1. / 120.);
  e = fma(e, f, 1. / 24.);
  e = fma(e, f, 1. / 6.);
  e = fma(e, f, 0.5);
  e = fma(e, f, 1.);
  e = fma(e, f, 1.);
  return y < -1050. ? 0. : ldexp(e, (int)n);
}
// log2 of a positive sum as exactly: one Newton step from log2_split
__device__ __forceinline__ double log2_newton(double x) {
  const double l = log2_split(x);
  return fma(x * exp2_series(-l) - 1., 1.4426950408889634, l);
}

// 16 bytes of consecutive classes.  A row of an odd vocabulary starts at any multiple of the element size: the copies
// below compile to one 16-byte access that the hardware takes at any address.
template <typename T> constexpr int vec_of() { return 16 / (int)sizeof(T); }

struct Raw16 { uint32_t w[4]; };

template <typename T> __device__ __forceinline__ Raw16 load16(const T* p) {
  Raw16 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
__device__ __forceinline__ void unpack(const Raw16& r, float (&x)[8]) {      // bf16
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __builtin_bit_cast(float, r.w[i] << 16);
    x[2 * i + 1] = __builtin_bit_cast(float, r.w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const Raw16& r, float (&x)[4]) {      // fp32
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __builtin_bit_cast(float, r.w[i]);
}
// PAST: write past the caches (an array that does not fit them, read by nobody before it has left them)
typedef __attribute__((ext_vector_type(4))) uint32_t devis_u32x4;
typedef devis_u32x4 devis_u32x4_any __attribute__((aligned(2)));
template <bool PAST> __device__ __forceinline__ void store16(void* p, devis_u32x4 v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, (devis_u32x4_any*)p);
  else *(devis_u32x4_any*)p = v;
}
template <bool PAST> __device__ __forceinline__ void store_vec(bf16* p, const float (&x)[8]) {
  devis_u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  store16<PAST>(p, v);
}
template <bool PAST> __device__ __forceinline__ void store_vec(float* p, const float (&x)[4]) {
  devis_u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(uint32_t, x[i]);
  store16<PAST>(p, v);
}
template <bool PAST, typename T> __device__ __forceinline__ void store_vec(T* p, const float (&x)[1]) { *p = (T)x[0]; }

// The thread's number, opaque to the optimiser where it is asked for: what is computed from it (offsets of a tile, of a
// path that is rarely taken) is computed there and not kept in registers from the start.
__device__ __forceinline__ uint32_t lane_id() {
  uint32_t lane = threadIdx.x;
  asm volatile("" : "+v"(lane));
  return lane;
}
// f(x, c): x = the values of classes c, c + 1, .. (VEC of them, or one at a time behind the last whole vector), over
// the classes [lo, hi) of one row, dealt to the BS threads of a block vector by vector.  UNIT: the classes are
// adjacent in memory (sK = 1) and travel 16 bytes at a time, U loads in flight; otherwise one by one.
template <typename T, bool UNIT, int BS, int U = 4, typename F>
__device__ __forceinline__ void each_class(int tid, const T* __restrict__ p, int64_t sK, int lo, int hi, F f) {
  if constexpr (UNIT) {
    constexpr int VEC = vec_of<T>();
    const int full = (hi - lo) / VEC;
    const T* q = p + lo;
    int v = tid;
    if constexpr (U > 1) {
      for (; v + (U - 1) * BS < full; v += U * BS) {
        Raw16 r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = load16(q + (int64_t)(v + u * BS) * VEC);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float x[VEC];
          unpack(r[u], x);
          f(x, lo + (v + u * BS) * VEC);
        }
      }
    }
    for (; v < full; v += BS) {
      float x[VEC];
      unpack(load16(q + (int64_t)v * VEC), x);
      f(x, lo + v * VEC);
    }
    const int c = lo + full * VEC + tid;
    if (c < hi) {
      float x[1] = {(float)p[c]};
      f(x, c);
    }
  } else {
    for (int c = lo + tid; c < hi; c += BS) {
      float x[1] = {(float)p[(int64_t)c * sK]};
      f(x, c);
    }
  }
}

template <int N> __device__ __forceinline__ float max_of(const float (&x)[N]) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
  return m;
}
template <int N> __device__ __forceinline__ float sum_of(const float (&x)[N]) {
  if constexpr (N == 1) return x[0];
  else {
    float y[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) y[i] = x[2 * i] + x[2 * i + 1];
    return sum_of(y);
  }
}

template <int N> __device__ __forceinline__ double sum_of(const double (&x)[N]) {
  if constexpr (N == 1) return x[0];
  else {
    double y[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) y[i] = x[2 * i] + x[2 * i + 1];
    return sum_of(y);
  }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// block-wide reductions, the result in every thread; `s` holds BS/64 entries and is free again on return
template <int BS> __device__ __forceinline__ float block_max(float v, float* s) {
  v = wave_max(v);
  if constexpr (BS > 64) {
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int i = 1; i < BS / 64; ++i) v = fmaxf(v, s[i]);
    __syncthreads();
  }
  return v;
}
template <int BS> __device__ __forceinline__ double block_sum(double v, double* s) {
  v = wave_sum(v);
  if constexpr (BS > 64) {
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int i = 1; i < BS / 64; ++i) v += s[i];
    __syncthreads();
  }
  return v;
}

// ---- few classes: a thread takes a whole row into registers.  KT = 2, 4, 8 or 16 bounds K; FULL: K = KT adjacent
// classes, one load of the whole row.
// (Distillation of 500000 rows, forward + backward, against a lane a row that streams its classes, below: 4 classes 17 and
// 38 us, 8 24 and 48, 16 31 and 70; top logits 16 classes 12 and 12.)
constexpr int FEW_CLASSES = 16;

template <typename T, int KT, bool FULL>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int64_t sK, int K, float (&x)[KT]) {
  if constexpr (FULL) {
    T raw[KT];
    __builtin_memcpy(raw, p, sizeof raw);
#pragma unroll
    for (int c = 0; c < KT; ++c) x[c] = (float)raw[c];
  } else {
#pragma unroll
    for (int c = 0; c < KT; ++c) x[c] = c < K ? (float)p[(int64_t)c * sK] : neg_inf();
  }
}
// A lane's element `lane` of an array whose place the whole block shares: a scalar address and one 32-bit offset a lane,
// where 64-bit addresses of every class and slot would take most of the registers.  `lane` stays below 256 * FEW_STRIDE.
constexpr int64_t FEW_STRIDE = (int64_t)1 << 20;
// The block's tiles of 256 rows: readfirstlane keeps the tile number scalar and the loop's addresses from becoming
// running 64-bit pointers a lane, one for every class and slot.
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
template <typename T> __device__ __forceinline__ T lane_load(const T* __restrict__ shared, uint32_t lane) {
  T v;
  __builtin_memcpy(&v, (const char*)shared + lane * (uint32_t)sizeof(T), sizeof(T));
  return v;
}
template <typename T, int KT, bool FULL>
__device__ __forceinline__ void lane_load_row(const T* __restrict__ shared, uint32_t lane, int64_t sK, int K, float (&x)[KT]) {
  if constexpr (FULL) {
    T raw[KT];
    __builtin_memcpy(raw, (const char*)shared + lane * (uint32_t)sizeof(T), sizeof raw);
#pragma unroll
    for (int c = 0; c < KT; ++c) x[c] = (float)raw[c];
  } else {
#pragma unroll
    for (int c = 0; c < KT; ++c) x[c] = c < K ? (float)lane_load(shared + c * sK, lane) : neg_inf();
  }
}
template <typename T, int KT, bool FULL>
__device__ __forceinline__ void store_row(T* __restrict__ p, int64_t sK, int K, const float (&x)[KT]) {
  if constexpr (FULL) {
    T raw[KT];
#pragma unroll
    for (int c = 0; c < KT; ++c) raw[c] = (T)x[c];
    __builtin_memcpy(p, raw, sizeof raw);
  } else {
#pragma unroll
    for (int c = 0; c < KT; ++c) if (c < K) p[(int64_t)c * sK] = (T)x[c];
  }
}

// rows of several shapes walked together as (n, v): one long v where every shape allows it
inline bool one_stride(const RowShape& s) { return s.N == 1 || s.V == 1 || s.sN == s.V * s.sV; }
inline void merge_rows(RowShape& s) {
  s.sV = s.V == 1 ? s.sN : s.sV;
  s.V *= s.N;
  s.N = 1;
  s.sN = 0;
}
// The kernels of few classes take 256 rows v at a time, for each n: rows that do not come as one long v, few of them side by side
// (small images, channels first), would leave most lanes idle and go the way of more classes instead.  us, top logits +
// distillation forward + backward, 4 fp32 classes channels first, 256 v at a time and any row a lane: 10^6 x 2 2633, 144;
// 10^5 x 16 299, 113; 30000 x 64 106, 127; 8000 x 200 59, 116.
constexpr int64_t FEW_V = 32;
inline bool side_by_side(const RowShape& a, const RowShape& b) { return a.V >= FEW_V || (one_stride(a) && one_stride(b)); }
inline dim3 few_grid(int64_t N, int64_t V, int most) {
  int64_t bx = cdiv(V, 256), by = N;
  if (bx > most) bx = most;
  const int64_t room = most / bx;
  if (by > room) by = room;
  return dim3((unsigned)bx, (unsigned)by);
}

#define DEVIS_DISPATCH_FEW(K, unit, LAUNCH)                                                 do {                                                                                        if ((K) <= 2) { if ((unit) && (K) == 2) LAUNCH(2, true); else LAUNCH(2, false); }         else if ((K) <= 4) { if ((unit) && (K) == 4) LAUNCH(4, true); else LAUNCH(4, false); }     else if ((K) <= 8) { if ((unit) && (K) == 8) LAUNCH(8, true); else LAUNCH(8, false); }     else { if ((unit) && (K) == 16) LAUNCH(16, true); else LAUNCH(16, false); }             } while (0)

// ---- a few dozen classes and many rows: one thread a row, the classes streamed in chunks of 8.  A wave a row would leave
// most of its lanes without work at the end of each row.  Classes first, the lanes' rows are adjacent and every load is
// whole lines; classes last, each lane walks its own row 16 bytes at a time, and a wave's load is 64 lines.
// A lane's time is that of its row until the rows fill the card, a wave's grows with the rows: which is less depends on the
// classes, and on the slots, every pair of which the lane looks at.  Microseconds a lane a row and a wave a row, bf16 classes
// last, distillation forward + backward / top logits:
//   64 classes, 4 slots    8192 rows  36, 34 / 11, 16    32768 rows  33, 98         500000 rows  231, 1379 / 94, 722
//   64 classes, 16 slots   8192 rows 116, 36             32768 rows 118, 105        500000 rows  963, 1511 / 105, 898
//   256 classes, 4 slots   8192 rows  66, 34 / 34, 16    32768 rows  67, 103        200000 rows  285,  563 / 78, 301
//   256 classes, 16 slots 32768 rows 165, 112            200000 rows 524, 616 / 197, 334
constexpr int LANE_CLASSES = 256;             // classes at most: the slots' bits of 256 rows fill 9 KB of LDS
constexpr int LANE_SLOTS = 16;                // slots at most: the list of the largest stays in registers
constexpr int64_t LANE_ROWS = 8192;           // rows at least (17 classes, 4 slots, 2048 rows: 24 us a lane a row, 18 a wave a row)
inline bool lane_rows(int64_t rows, int64_t K, int64_t k) {
  const int64_t least = 96 * K * (k > 4 ? 4 : 1);
  return K <= LANE_CLASSES && k <= LANE_SLOTS && rows >= (least > LANE_ROWS ? least : LANE_ROWS);
}

// running maximum and sum of exponentials against it (fp64: one lane adds up the whole row)
struct LaneSum {
  float m;
  double s;
  __device__ __forceinline__ void add(const float (&x)[8], float scale) {
    const float mx = max_of(x);
    if (mx > m) { s *= (double)exp2_f((m - mx) * scale); m = mx; }
    const float ref = m == neg_inf() ? 0.f : m;
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = exp2_f((x[i] - ref) * scale);
    s += (double)sum_of(e);
  }
  __device__ __forceinline__ void add_one(float x, float scale) {
    if (x > m) { s *= (double)exp2_f((m - x) * scale); m = x; }
    s += (double)exp2_f((x - (m == neg_inf() ? 0.f : m)) * scale);
  }
};

// eight classes c.. of one row, -inf behind the last
template <typename T, bool UNIT>
__device__ __forceinline__ void load8(const T* __restrict__ p, int64_t sK, int c, int K, float (&x)[8]) {
  if (UNIT && c + 8 <= K) {
    if constexpr (sizeof(T) == 2) unpack(load16(p + c), x);
    else {
      unpack(load16(p + c), *(float(*)[4])x);
      unpack(load16(p + c + 4), *(float(*)[4])(x + 4));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c + i < K ? (float)p[(int64_t)(c + i) * (UNIT ? 1 : sK)] : neg_inf();
  }
}

// one block a row: rows over a 2-D grid (a dimension holds less than 2^32 threads)
inline dim3 row_grid(int64_t rows) {
  const int64_t x = rows < (1 << 20) ? rows : (1 << 20);
  return dim3((unsigned)x, (unsigned)cdiv(rows, x));
}
constexpr int64_t MAX_ROWS = (int64_t)65535 << 20;
__device__ __forceinline__ int64_t grid_row() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

inline bool rows_ok(int64_t sN, int64_t sV, int64_t sK, int64_t N, int64_t V, int64_t K) {
  return N > 0 && V > 0 && K > 0 && K <= MAX_CLASSES && sN >= 0 && sV >= 0 && sK > 0 && N <= MAX_ROWS / V;
}

}  // namespace devis
