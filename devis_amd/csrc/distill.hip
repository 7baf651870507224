// Distillation from a teacher's top logits (toplogits.hip makes them), loss and gradient.
//
//   teacher: k slots (t_j, class i_j), t_j = -inf for an empty one, and optionally rest = log sum of exp(t / T) over
//   every other class;  p = softmax over {t_j / T} and rest,  q = softmax(z / T) of the student's row,
//   q_rest = the sum of q over the classes in no slot
//   L      = T^2 [ sum_j p_j (log p_j - log q_{i_j}) + p_rest (log p_rest - log q_rest) ]
//   dL/dz_c = T [ q_c - sum_{j: i_j = c} p_j ],  and T [ q_c - p_rest q_c / q_rest ] for a class in no slot.
//
// Without rest, p_rest = 0 and the top is renormalised.  Both passes are bound by memory: the forward reads the row
// once with a running maximum and sum per thread, keeping the classes in no slot apart (a bit per class in LDS tells
// them); the backward reads it once more and writes the gradient: for a class in no slot it is one exponential times a
// factor of the row, W = 1/s - p_rest/s_rest; the k listed classes are put right afterwards.  4096 x 131072 bf16, 64 slots
// and rest: forward 196 us (5.5 TB/s), backward 402 us (5.3 TB/s; a copy moves 5.0), together 614.
#include "rows.h"

#include <type_traits>

namespace devis {

constexpr int DIS_MAX_K = DEVIS_TOP_MAX_K;
// classes whose slot bits are in LDS at a time (16 KB; 512 bytes for a wave's row, all it has)
template <int BS> constexpr int dis_seg() { return BS == 64 ? 4096 : 131072; }
// Rows that a wave takes, many to a block; longer ones take a block each.  Many rows are better off with waves up to 8 KB.
// Forward + backward, us, a wave and a block a row, 20 slots (16 of the lesser counts):
//   20000 rows of 1000 bf16   85, 131     1100  95, 135     2000  109, 136     3000  121, 145     4000  158, 181    fp32 4000  245, 230
//    6000 rows of 1100        36,  49     2000  42,  52     4000   54,  60     2000 rows of 600  20, 21    1100  22, 22    4000  29, 27
constexpr int DIS_SHORT = 1024;               // classes of any number of rows
constexpr int64_t DIS_SHORT_BYTES = 8192, DIS_SHORT_ROWS = 4096;
// A gradient as large as the 256 MB Infinity Cache cannot stay there for its reader: written past the caches it leaves the
// logits in them, which the backward reads from the last row on.  Loss and gradient of 4096 x 131072 bf16 rows: 658 us with
// ordinary stores, 613 past the caches; 2048 x 65536 (256 MB) 198 and 175; below, the gradient is better kept.
constexpr double DIS_PAST_BYTES = 256. * 1024 * 1024;
constexpr int DIS_MAX_BLOCKS = 2048;          // 8 blocks of 256 threads on each of 256 CUs
constexpr int DIS_MAX_WAVES = 8192;           // or as many blocks of a wave

// what the backward needs of a row
struct RowStats { float ref, w, m, inv_s; };  // gradient of a class in no slot: exp((z - ref)/T) w;  q = exp((z - m)/T) inv_s

// The ends of a row: fp64 for long rows.  Of the short ones of a wave each there are many, and the library's fp64 functions
// would cost more than the row: logarithms by a Newton step, exponentials and quotients in fp32.
template <bool LONG> __device__ __forceinline__ double end_log2(double x) { return LONG || !(x > 0.) ? log2(x) : log2_newton(x); }
template <bool LONG> __device__ __forceinline__ double end_exp2(double x) { return LONG ? exp2(x) : (double)exp2_f((float)x); }
template <bool LONG> __device__ __forceinline__ double end_div(double a, double b) { return LONG ? a / b : a * (double)(1.f / (float)b); }

// What a class adds to a row's divergence, from the logarithms (base 2) of its shares p and q:  p (r - 1 - log r),  r = q / p.
// The listed classes and the rest have shares that sum to one on both sides, so these add up to sum p log(p / q); but they are
// never negative, nothing cancels among them, and an error e that every log q of the row has in common - its sum of fp32
// exponentials, whose constant log2(e) / T rounds the same way in every row - changes the total by sum (q - p) e = 0 and
// e^2 / 2 instead of e.  The series is for |log r| <= 1/2; what it leaves out is 2e-9 of it.
__device__ __forceinline__ double kl_part(double log2_p, double log2_q) {
  const double p = exp2_series(log2_p), l = (log2_q - log2_p) * 0.6931471805599453;
  if (p != 0. && fabs(l) <= 0.5) {
    double s = 1. / 3628800.;
    s = fma(s, l, 1. / 362880.);
    s = fma(s, l, 1. / 40320.);
    s = fma(s, l, 1. / 5040.);
    s = fma(s, l, 1. / 720.);
    s = fma(s, l, 1. / 120.);
    s = fma(s, l, 1. / 24.);
    s = fma(s, l, 1. / 6.);
    s = fma(s, l, 0.5);
    return p * (l * l * s);
  }
  const double q = exp2_series(log2_q);
  return p == 0. ? q : q - fma(p, l, p);
}

struct Teacher {
  const void* values; const void* indices; const float* rest; const uint8_t* mask;
  RowShape o;                                 // strides of values / indices, K = number of slots
  int value_kind, index_kind;
};

__device__ __forceinline__ int class_at(const void* idx, int kind, int64_t at) {
  if (kind == DEVIS_LABEL_U8) return ((const uint8_t*)idx)[at];
  if (kind == DEVIS_LABEL_I32) return ((const int32_t*)idx)[at];
  const int64_t c = ((const int64_t*)idx)[at];
  return c < 0 || c > 0x7ffffffe ? -1 : (int)c;
}

__device__ __forceinline__ float slot_value(const Teacher& t, int64_t i) {
  return t.value_kind == DEVIS_F32 ? ((const float*)t.values)[i] : (float)((const bf16*)t.values)[i];
}

// rest - hi / T.  Of a masked row both are near the type's lowest value and their difference is what counts: the quotient is
// rounded correctly (by its remainder; hi times a rounded 1 / T would be off by 1e22), and what it is taken off from is exact.
__device__ __forceinline__ double rest_gap(float rest, float hi, double inv_t, float temperature) {
  const double q = (double)hi * inv_t;
  return (double)rest - fma(fma(-q, (double)temperature, (double)hi), inv_t, q);
}

// a row that takes no part; no counted row has this reference with a factor of zero
__device__ __forceinline__ RowStats not_counted() { return RowStats{__builtin_inff(), 0.f, 0.f, 0.f}; }

struct SlotShared {
  double logp[DIS_MAX_K];      // logarithm (base 2) of each slot's share
  float p[DIS_MAX_K];          // its share
  int c[DIS_MAX_K];            // its class, -1 for an empty slot
  double p_rest, log_p_rest;
  int state;                   // 0 row not counted (masked, or every slot empty), 1 counted, 2 a slot names no class
};

// The teacher's softmax of one row, by the first wave (lane l: slots l and l + 64), in
// fp64 and the shares rounded once: the loss is the difference of near-equal logarithms once the student is near the
// teacher (104 rows of 1231 classes at temperature 4: fp32 exponentials here cost 1.4e-6 of it, 3e-7 in the student's sums).
template <bool LONG>
__device__ __forceinline__ void teacher_row(const Teacher& t, int64_t r, int K, double inv_t, float temperature, int lane, SlotShared& sh) {
  const int k = t.o.K;
  const int64_t at = row_offset(t.o, r);
  float v[2];
  int cls[2];
  bool bad = false, any = false;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = lane + 64 * u;
    v[u] = neg_inf();
    cls[u] = 0;
    if (j < k) {
      const int64_t i = at + j * t.o.sK;
      v[u] = slot_value(t, i);
      if (v[u] != neg_inf()) {
        any = true;
        cls[u] = class_at(t.indices, t.index_kind, i);
        if (cls[u] < 0 || cls[u] >= K) { bad = true; cls[u] = 0; }
      }
    }
  }
  const int state = !__any(any) ? 0 : __any(bad) ? 2 : 1;
  // The largest value is taken off before anything is scaled: of a teacher whose values are all the type's lowest the small
  // differences stay.
  const float hi = wave_max(fmaxf(v[0], v[1]));
  const double yr = t.rest ? rest_gap(t.rest[r], hi, inv_t, temperature) : -__builtin_inf(), shift = fmax(yr, 0.);
  double y[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) y[u] = v[u] == neg_inf() ? -__builtin_inf() : ((double)v[u] - (double)hi) * inv_t;
  y[0] = (y[0] - shift) * 1.4426950408889634;
  y[1] = (y[1] - shift) * 1.4426950408889634;
  const double e0 = exp2_series(y[0]), e1 = exp2_series(y[1]), y_rest = (yr - shift) * 1.4426950408889634, er = exp2_series(y_rest);
  const double sum = wave_sum(e0 + e1) + er;
  const double ls = end_log2<LONG>(sum);
  const double inv = end_div<LONG>(1., sum);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = lane + 64 * u;
    if (j < k) {
      sh.p[j] = (float)((u ? e1 : e0) * inv);
      sh.logp[j] = y[u] - ls;
      // an empty slot takes part in nothing
      sh.c[j] = y[u] == -__builtin_inf() ? -1 : cls[u];
    }
  }
  if (lane == 0) {
    sh.p_rest = er * inv;
    sh.log_p_rest = y_rest - ls;
    sh.state = state;
  }
}

// the class of slot j, -1 for an empty one
__device__ __forceinline__ int slot_class(const Teacher& t, int64_t at, int j, int K) {
  const int64_t i = at + j * t.o.sK;
  const int c = class_at(t.indices, t.index_kind, i);
  return slot_value(t, i) == neg_inf() || c >= K ? -1 : c;
}

__device__ __forceinline__ bool row_masked(const Teacher& t, int64_t r) { return t.mask && t.mask[r] == 0; }

// (without rest its share of the teacher is zero, and the student's share of those classes is summed apart all the same)
template <typename T, bool UNIT, int BS>
__global__ void __launch_bounds__(BS, BS == 256 ? 8 : BS == 1024 ? 4 : 1)
k_distill_fwd(const T* __restrict__ z, RowShape s, Teacher t, float scale, double inv_t, float temperature, RowStats* __restrict__ stats,
              float* __restrict__ per_row, double* __restrict__ partial) {
  constexpr bool LONG = BS > 64;
  __shared__ SlotShared sh;
  constexpr int SEG = dis_seg<BS>();
  __shared__ uint32_t s_bits[SEG / 32];
  __shared__ double s_red[BS / 64];
  __shared__ float s_max[BS / 64];
  const int K = s.K;
  const int64_t NV = s.N * s.V;
  double loss_sum = 0.;
  int count = 0;
  const int64_t first_row = grid_row();
  if (first_row >= NV) return;
  for (int64_t r = first_row; r < NV; r += gridDim.x) {
    const int tid = lane_id();
    const T* p = z + row_offset(s, r);
    // the slots' classes, wanted first of all for their bits, and the mask come in together
    constexpr int OWN = BS < DIS_MAX_K ? DIS_MAX_K / BS : 1;
    const int64_t slots = row_offset(t.o, r);
    int own[OWN];
#pragma unroll
    for (int u = 0; u < OWN; ++u) own[u] = tid + u * BS < t.o.K ? slot_class(t, slots, tid + u * BS, K) : -1;
    if (row_masked(t, r)) {
      if (tid == 0) {
        if (per_row) per_row[r] = 0.f;
        if (stats) stats[r] = not_counted();
      }
      if (LONG) break;
      continue;
    }
    if (tid < 64) teacher_row<LONG>(t, r, K, inv_t, temperature, tid, sh);
    // running maximum and sum of the classes in no slot: fp32, in which a thread adds trees of 16 or 32 classes in turn; what that
    // and the exponentials leave over is in every logarithm of the row and drops out of its loss (kl_part)
    float m = neg_inf(), acc = 0.f;
    const auto absorb = [&](auto& x) {
      constexpr int N = sizeof(x) / sizeof(float);
      const float mx = max_of(x);
      if (mx > m) { acc *= exp2_f((m - mx) * scale); m = mx; }
      const float ref = m == neg_inf() ? 0.f : m;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = exp2_f((x[i] - ref) * scale);
      acc += sum_of(x);
    };
    for (int lo = 0; lo < K; lo += SEG) {
      const int hi = K - lo < SEG ? K : lo + SEG;
      for (int i = tid; i < (hi - lo + 31) / 32; i += BS) s_bits[i] = 0;
      __syncthreads();
#pragma unroll
      for (int u = 0; u < OWN; ++u)
        if (own[u] >= lo && own[u] < hi) atomicOr(&s_bits[(own[u] - lo) >> 5], 1u << ((own[u] - lo) & 31));
      __syncthreads();
      if constexpr (UNIT) {
        constexpr int VEC = vec_of<T>();
        const T* q = p + lo;
        const int full = (hi - lo) / VEC;
        // the slot bits of vector v: a byte, or half of one
        const auto bits = [&](int v) -> uint32_t {
          if constexpr (VEC == 8) return ((const uint8_t*)s_bits)[v];
          else return (((const uint8_t*)s_bits)[v >> 1] >> ((v & 1) * 4)) & 15u;
        };
        int v = tid;
        for (; v + 3 * BS < full; v += 4 * BS) {
          Raw16 raw[4];
          float x[4 * VEC];
          uint32_t b = 0;
#pragma unroll
          for (int u = 0; u < 4; ++u) raw[u] = load16(q + (int64_t)(v + u * BS) * VEC);
#pragma unroll
          for (int u = 0; u < 4; ++u) b |= bits(v + u * BS) << (u * VEC);
#pragma unroll
          for (int u = 0; u < 4; ++u) unpack(raw[u], *(float(*)[VEC])(x + u * VEC));
          if (b) {
#pragma unroll
            for (int i = 0; i < 4 * VEC; ++i) x[i] = (b >> i) & 1u ? neg_inf() : +x[i];
          }
          absorb(x);
        }
        for (; v < full; v += BS) {
          float x[VEC];
          unpack(load16(q + (int64_t)v * VEC), x);
          const uint32_t b = bits(v);
          if (b) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = (b >> i) & 1u ? neg_inf() : +x[i];
          }
          absorb(x);
        }
        const int c = full * VEC + tid;
        if (c < hi - lo && !((s_bits[c >> 5] >> (c & 31)) & 1u)) {
          float x[1] = {(float)q[c]};
          absorb(x);
        }
      } else {
        for (int c = lo + tid; c < hi; c += BS) {
          float x[1] = {(float)p[(int64_t)c * s.sK]};
          if ((s_bits[(c - lo) >> 5] >> ((c - lo) & 31)) & 1u) continue;
          absorb(x);
        }
      }
      __syncthreads();
    }
    const float m_rest = block_max<BS>(m, s_max);              // (its barrier also ends the wait for the teacher's shares)
    const float ref = m_rest == neg_inf() ? 0.f : m_rest;
    const double sum_rest = block_sum<BS>(m == neg_inf() ? (double)acc : (double)acc * (double)exp2_f((m - ref) * scale), s_red);
    if (threadIdx.x < 64) {
      const int tid = lane_id();
      // the listed classes' logits; a class in two slots counts once in the student's sum (its first slot)
      float x[2];
      bool first[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = tid + 64 * u;
        x[u] = neg_inf();
        first[u] = false;
        if (j < t.o.K && sh.c[j] >= 0) {
          x[u] = (float)p[(int64_t)sh.c[j] * s.sK];
          bool again = false;
#pragma unroll 8
          for (int i = 0; i < j; ++i) again |= sh.c[i] == sh.c[j];
          first[u] = !again;
        }
      }
      const float m_all = fmaxf(m_rest, wave_max(fmaxf(x[0], x[1])));
      const double m_d = m_all == neg_inf() ? 0. : (double)m_all;
      double mine = 0.;
#pragma unroll
      for (int u = 0; u < 2; ++u) if (first[u]) mine += (double)exp2_f((x[u] - (float)m_d) * scale);
      const double to_m = m_rest == neg_inf() ? 0. : end_exp2<LONG>(((double)m_rest - m_d) * inv_t * 1.4426950408889634);
      const double sum = wave_sum(mine) + (m_rest == neg_inf() ? sum_rest : sum_rest * to_m);
      const double ls = end_log2<LONG>(sum);  // log q = (x - m)/T - ls: the large part cancels first
      double kl = 0.;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = tid + 64 * u;
        if (j < t.o.K && sh.c[j] >= 0) {
          const double logq = x[u] == neg_inf() ? -__builtin_inf() : ((double)x[u] - m_d) * inv_t * 1.4426950408889634 - ls;
          kl += kl_part(sh.logp[j], logq);
          if (!first[u]) kl -= exp2_series(logq);              // the q of a class in two slots counts once
        }
      }
      kl = wave_sum(kl);
      if (tid == 0 && sh.state != 1) {
        const float v = sh.state == 2 ? __builtin_nanf("") : 0.f;
        if (per_row) per_row[r] = v;
        if (stats) stats[r] = sh.state == 2 ? RowStats{0.f, v, 0.f, v} : not_counted();
        if (sh.state == 2) { loss_sum += (double)v; ++count; }
      } else if (tid == 0) {
        const double log_q_rest = sum_rest == 0. ? -__builtin_inf() : ((double)ref - m_d) * inv_t * 1.4426950408889634 + end_log2<LONG>(sum_rest) - ls;
        kl += kl_part(sh.log_p_rest, log_q_rest);
        const double inv = sum > 0. ? end_div<LONG>(1., sum) : sum == 0. ? 0. : sum;
        // q = exp((z - m_rest)/T) * w before the teacher's share of the rest is taken off
        const double w = m_rest == neg_inf() ? 0. : inv * to_m - end_div<LONG>(sh.p_rest, sum_rest);
        const double loss = (double)temperature * (double)temperature * kl;
        if (per_row) per_row[r] = (float)loss;
        if (stats) stats[r] = RowStats{ref, (float)w, (float)m_d, (float)inv};
        loss_sum += loss;
        ++count;
      }
    }
    if (LONG) break;                           // one row a block: nothing of the row's end is kept in registers from the start
    __syncthreads();
  }
  if (partial && threadIdx.x == 0) {
    partial[2 * first_row] = loss_sum;
    partial[2 * first_row + 1] = (double)count;
  }
}

// The sum or mean of the counted rows' losses; scal = what a row's gradient is multiplied by, and the rows counted.  More
// partials than DIS_FINAL are first added up by DIS_STAGE blocks, in fixed order.
constexpr int64_t DIS_FINAL = 16384;
constexpr int DIS_STAGE = 512;

__global__ void __launch_bounds__(256)
k_distill_stage(const double* __restrict__ partial, int64_t n, double* __restrict__ out) {
  __shared__ double s_red[4];
  const int64_t each = (n + DIS_STAGE - 1) / DIS_STAGE, lo = blockIdx.x * each, hi = lo + each < n ? lo + each : n;
  double loss = 0., count = 0.;
  for (int64_t i = lo + threadIdx.x; i < hi; i += 256) { loss += partial[2 * i]; count += partial[2 * i + 1]; }
  loss = block_sum<256>(loss, s_red);
  count = block_sum<256>(count, s_red);
  if (threadIdx.x == 0) { out[2 * blockIdx.x] = loss; out[2 * blockIdx.x + 1] = count; }
}

__global__ void __launch_bounds__(1024)
k_distill_finalize(const double* __restrict__ partial, int n, int mean, float* __restrict__ out, float* __restrict__ scal) {
  __shared__ double s_red[16];
  double loss = 0., count = 0.;
  for (int i = threadIdx.x; i < n; i += 1024) { loss += partial[2 * i]; count += partial[2 * i + 1]; }
  loss = block_sum<1024>(loss, s_red);
  count = block_sum<1024>(count, s_red);
  if (threadIdx.x == 0) {
    const double f = mean ? 1. / (count > 0. ? count : 1.) : 1.;
    out[0] = (float)(loss * f);
    scal[0] = (float)f;
    scal[1] = (float)count;
  }
}

template <typename T, bool UNIT, bool PAST, int BS>
__global__ void __launch_bounds__(BS, BS == 256 ? 8 : BS == 1024 ? 4 : 1)
k_distill_bwd(const T* __restrict__ z, RowShape s, Teacher t, float scale, double inv_t, float temperature,
              const RowStats* __restrict__ stats, const float* __restrict__ scal, const float* __restrict__ grad, int grad_rows,
              T* __restrict__ dz, RowShape d) {
  __shared__ SlotShared sh;
  constexpr bool LONG = BS > 64;
  const int K = s.K;
  const int64_t NV = s.N * s.V;
  for (int64_t i = grid_row(); i < NV; i += gridDim.x) {
    const int64_t r = NV - 1 - i;              // what the forward read last is still in the caches: it is read first
    const int tid = lane_id();
    const T* p = z + row_offset(s, r);
    T* q = dz + row_offset(d, r);
    RowStats st = not_counted();
    if (!row_masked(t, r)) st = stats[r];
    const bool live = !(st.ref == __builtin_inff() && st.w == 0.f);
    if (live && tid < 64) teacher_row<LONG>(t, r, K, inv_t, temperature, tid, sh);       // for the listed classes, at the end
    const float g = grad_rows ? grad[r] : grad[0] * scal[0];
    const float f = g * temperature;
    const float w = f * st.w;
    if (!live) {
      for (int c = tid; c < K; c += BS) q[(int64_t)c * d.sK] = (T)0.f;
    } else {
      each_class<T, UNIT, BS>(tid, p, s.sK, 0, K, [&](auto& x, int c) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = exp2_f((x[i] - st.ref) * scale) * w;
        store_vec<PAST>(q + (int64_t)c * (UNIT ? 1 : d.sK), x);
      });
      // the listed classes are written again, by other threads: after these stores have been taken
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      for (int j = tid; j < t.o.K; j += BS) {
        const int c = sh.c[j];
        if (c < 0 || sh.state == 2) continue;
        float share = 0.f;
#pragma unroll 8
        for (int i = 0; i < t.o.K; ++i) share += sh.c[i] == c ? sh.p[i] : 0.f;
        const float x = (float)p[(int64_t)c * s.sK];
        const float qc = x == neg_inf() ? 0.f : exp2_f((x - st.m) * scale) * st.inv_s;
        q[(int64_t)c * d.sK] = (T)(f * (qc - share));
      }
    }
    if (LONG) break;
    __syncthreads();
  }
}

// ---- few classes: one thread a row, everything in registers, nothing kept for the backward.  For a mean and for
// the gradient exponentials and logarithms are fp32 (FEW_ROW_LOSS below: fp64).  Sums over rows are fp64.  2 x 128^3 x 4
// bf16, two slots and rest: 37 us forward, 32 backward (75 and 109 MB; VALU issue is 91 and 83 % busy: 265 and 199 instructions
// a row); 70 us for the loss of every row.
__device__ __forceinline__ float log2_f(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float rcp_f(float x) { return __builtin_amdgcn_rcpf(x); }

// a sum of shares of numbers in range stays in range where rounding alone would carry it past the largest (a student's mask
// of the type's lowest value on a listed class); NaN stays
__device__ __forceinline__ float in_range(float x) { return x > 3.4028235e38f ? 3.4028235e38f : x; }

// x[c], and ec = e[c]; -inf and 0 of an empty slot
template <int KT, typename S>
__device__ __forceinline__ float pick_class(const float (&x)[KT], int c, const S (&e)[KT], S& ec) {
  float v = neg_inf();
  ec = 0;
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    const float xi = x[i];
    const S ei = e[i];
    if (c == i) { v = xi; ec = ei; }
  }
  return v;
}

// p (r - 1 - log r) times T, of a finite l = -log r and pd = p T l: by its series where q and p are near (what is left out is 4e-8
// of it), otherwise as it stands
__device__ __forceinline__ float kl_part(float p, float q, float l, float pd, float temperature) {
  float s = -1.f / 362880.f;
  s = fmaf(s, l, 1.f / 40320.f);
  s = fmaf(s, l, -1.f / 5040.f);
  s = fmaf(s, l, 1.f / 720.f);
  s = fmaf(s, l, -1.f / 120.f);
  s = fmaf(s, l, 1.f / 24.f);
  s = fmaf(s, l, -1.f / 6.f);
  s = fmaf(s, l, 0.5f);
  return fabsf(l) <= 0.5f ? pd * (l * s) : fmaf(temperature, q - p, pd);
}

// What few_row works out.  A row's own loss is what is left when logarithms cancel (a student near its teacher at a high
// temperature: 0.02 of numbers near 1), so for it everything is fp64.  Of many rows that would be half of the step, and fp32
// differences of logarithms would not do: what rounds alike in every row - a constant, a sum - is a bias of their mean (9
// classes, temperature 4, losses of 2e-5: 4e-3 of it).  A mean is fp32 and adds up, for each of the row's classes (the
// rest is one),
//   p (r - 1 - log r),  r = q / p,   instead of   -p log r :
// the same total, because the p and the q each sum to one, of terms that are never negative and do not cancel; and an error e
// that all log r of a row share, as that of a logarithm of a sum, changes the total by sum p (r - 1) e = 0 and e^2 / 2.
// (A share below 2^-126 of a class that is open to the student counts as zero in a mean: what it adds is less than 1e-38 of the
// logits' distance.)
enum { FEW_GRADIENT, FEW_MEAN_LOSS, FEW_ROW_LOSS };

// KS bounds the slots as KT bounds the classes; S is the type of shares and sums.
template <int KT, int KS, typename S> struct FewRow {
  float x[KT], a[KS];          // logits; slots: logit below the largest
  S e[KT], p[KS];              // exponentials, of a class in a slot against the row's maximum, else against m_rest; shares
  int c[KS];
  unsigned listed;
  int state;                   // as SlotShared::state
  float m;                     // student: maximum, sum of exponentials against it, 1 / sum
  S sum, inv;
  S sum_rest, to_m;            // classes in no slot: sum against m_rest, exp((m_rest - m)/T)
  S p_rest;
  S off;                       // with a loss: log2(S_student / S_teacher), both against their own maxima
  double off_rest;             // with a loss: log2(p_rest / q_rest)
  unsigned twice;              // classes in two slots
  bool alive[KS], rest_alive;  // a slot, the rest has a share, be it too small for S
};

// exponents (base 2) from which on a share is none, here as in exp2_series
constexpr float NO_SHARE = -1050.f;

__device__ __forceinline__ float few_exp(float x, float ref, float scale, double) { return exp2_f((x - ref) * scale); }
__device__ __forceinline__ double few_exp(double x, double ref, float, double scale) { return exp2_series((x - ref) * scale); }
__device__ __forceinline__ float few_log(float x) { return log2_f(x); }
__device__ __forceinline__ double few_log(double x) { return log2_newton(x); }
__device__ __forceinline__ float few_rcp(float x) { return rcp_f(x); }       // within 2^-23: a share's own exponential is no better
__device__ __forceinline__ double few_rcp(double x) { return 1. / x; }

// Row (n, v0 + lane) with n and v0 the block's.  Straight-line: a row that is not counted is worked out all the same and
// dropped at the end.
template <typename T, int KT, int KS, bool FULL, bool REST, int WANT, typename S>
__device__ __forceinline__ void few_row(const T* __restrict__ z, const RowShape& s, const Teacher& t, int64_t n, int64_t v0,
                                        uint32_t lane, float scale, double inv_t, float temperature, FewRow<KT, KS, S>& w) {
  const int K = s.K, k = t.o.K;
  const double scale_d = inv_t * 1.4426950408889634;
  const int64_t r0 = n * s.V + v0, at = n * t.o.sN + v0 * t.o.sV;
  const uint32_t slot = lane * (uint32_t)t.o.sV;
  // every load first, raw: nothing is looked at before all of them are on their way.  Slots behind the last read the last.
  lane_load_row<T, KT, FULL>(z + n * s.sN + v0 * s.sV, lane * (uint32_t)s.sV, s.sK, K, w.x);
  const float rest = REST && t.rest ? lane_load(t.rest + r0, lane) : neg_inf();
  const unsigned keep = t.mask ? lane_load(t.mask + r0, lane) : 1u;
  const bool wide = t.value_kind == DEVIS_F32;
  uint32_t raw[KS];
  int64_t of[KS];
#pragma unroll
  for (int j = 0; j < KS; ++j) of[j] = at + (j < k ? j : k - 1) * t.o.sK;
  if (wide) {
#pragma unroll
    for (int j = 0; j < KS; ++j) raw[j] = lane_load((const uint32_t*)t.values + of[j], slot);
  } else {
#pragma unroll
    for (int j = 0; j < KS; ++j) raw[j] = lane_load((const uint16_t*)t.values + of[j], slot);
  }
  if (t.index_kind == DEVIS_LABEL_U8) {
#pragma unroll
    for (int j = 0; j < KS; ++j) w.c[j] = lane_load((const uint8_t*)t.indices + of[j], slot);
  } else if (t.index_kind == DEVIS_LABEL_I32) {
#pragma unroll
    for (int j = 0; j < KS; ++j) w.c[j] = lane_load((const int32_t*)t.indices + of[j], slot);
  } else {
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const int64_t c = lane_load((const int64_t*)t.indices + of[j], slot);
      w.c[j] = c < 0 || c >= K ? -1 : (int)c;
    }
  }
  float hi = neg_inf();
  bool bad = false;
  w.listed = w.twice = 0;
#pragma unroll
  for (int j = 0; j < KS; ++j) {
    w.a[j] = __builtin_bit_cast(float, raw[j] << (wide ? 0 : 16));
    w.a[j] = j < k ? +w.a[j] : neg_inf();
    const bool filled = w.a[j] != neg_inf();
    bad = bad || (filled && (unsigned)w.c[j] >= (unsigned)K);
    w.c[j] = filled ? w.c[j] & (FEW_CLASSES - 1) : FEW_CLASSES;
    if constexpr (WANT == FEW_MEAN_LOSS) w.twice |= w.listed & (1u << w.c[j]);
    w.listed |= 1u << w.c[j];
    hi = fmaxf(hi, w.a[j]);
  }
  w.listed &= (1u << FEW_CLASSES) - 1;
  w.twice &= (1u << FEW_CLASSES) - 1;
  w.state = w.listed == 0 || keep == 0 ? 0 : bad ? 2 : 1;
  // teacher, in base 2 against its largest logarithm
  double a_rest = -__builtin_inf();
  S shift = 0;
  if constexpr (REST) {
    a_rest = rest_gap(rest, hi, inv_t, temperature) * 1.4426950408889634;
    // from here on the rest is all of the teacher, and a number that S holds as it is cancels where it has to
    a_rest = a_rest > 4096. && a_rest < __builtin_inf() ? 4096. : a_rest;
    shift = (S)fmax(a_rest, 0.);
  }
  w.rest_alive = REST && !(a_rest - (double)shift < NO_SHARE);
  w.p_rest = REST ? few_exp((S)a_rest, shift, 1.f, 1.) : (S)0;
  S sum_t = w.p_rest;
#pragma unroll
  for (int j = 0; j < KS; ++j) {
    w.a[j] -= hi;
    w.p[j] = REST ? few_exp((S)w.a[j] * (S)scale_d, shift, 1.f, 1.) : few_exp((S)w.a[j], (S)0, scale, scale_d);
    if constexpr (WANT == FEW_MEAN_LOSS) w.alive[j] = !(w.a[j] * scale - shift < NO_SHARE);      // (an empty slot's is -inf)
    w.p[j] = w.c[j] == FEW_CLASSES ? (S)0 : +w.p[j];
    sum_t += w.p[j];
  }
  const S inv_sum_t = few_rcp(sum_t);
#pragma unroll
  for (int j = 0; j < KS; ++j) w.p[j] *= inv_sum_t;
  w.p_rest *= inv_sum_t;
  // student
  w.m = max_of(w.x);
  w.m = w.m == neg_inf() ? 0.f : +w.m;
  float m_rest = neg_inf();
  w.sum = w.sum_rest = w.to_m = 0;
  if constexpr (REST) {
#pragma unroll
    for (int c = 0; c < KT; ++c) m_rest = fmaxf(m_rest, (w.listed >> c) & 1u ? neg_inf() : +w.x[c]);
    m_rest = m_rest == neg_inf() ? +w.m : m_rest;
    w.to_m = few_exp((S)m_rest, (S)w.m, scale, scale_d);
#pragma unroll
    for (int c = 0; c < KT; ++c) {
      const bool l = (w.listed >> c) & 1u;
      w.e[c] = few_exp((S)w.x[c], (S)(l ? +w.m : m_rest), scale, scale_d);
      w.sum += l ? +w.e[c] : (S)0;
      w.sum_rest += l ? (S)0 : +w.e[c];
    }
    w.sum += w.sum_rest * w.to_m;
  } else {
#pragma unroll
    for (int c = 0; c < KT; ++c) w.e[c] = few_exp((S)w.x[c], (S)w.m, scale, scale_d);
    w.sum = sum_of(w.e);
  }
  if constexpr (WANT == FEW_GRADIENT) {
    w.inv = w.sum == (S)0 ? (S)0 : few_rcp(w.sum);
  } else {
    if constexpr (WANT == FEW_ROW_LOSS) w.off = few_log(w.sum) - few_log(sum_t) - shift;
    else w.off = few_log(w.sum * inv_sum_t) - shift;
    if constexpr (REST) w.off_rest = (a_rest - ((double)m_rest - (double)w.m) * scale_d) + (double)(w.off - few_log(w.sum_rest));
  }
}

// (without rest its share of the teacher is zero, and what the student gives those classes still counts)
template <typename T, int KT, int KS, bool FULL, bool ROWS>
__global__ void __launch_bounds__(256)
k_distill_few_fwd(const T* __restrict__ z, RowShape s, Teacher t, float scale, double inv_t, float temperature,
                  float* __restrict__ per_row, double* __restrict__ partial) {
  typedef typename std::conditional<ROWS, double, float>::type S;
  __shared__ double s_red[4];
  const S unit = (S)((double)temperature * 0.6931471805599453);      // of the logarithms to base 2
  double loss_sum = 0.;
  int count = 0;
  const int64_t tiles = (s.V + 255) / 256;
  for (int64_t n = blockIdx.y; n < s.N; n += gridDim.y) {
    for (int64_t i = blockIdx.x; i < tiles; i += gridDim.x) {
      const int64_t v0 = (int64_t)scalar((int)i) * 256;
      const uint32_t lane = lane_id();
      if (v0 + lane >= s.V) continue;
      FewRow<KT, KS, S> w;
      few_row<T, KT, KS, FULL, true, ROWS ? FEW_ROW_LOSS : FEW_MEAN_LOSS>(z, s, t, n, v0, lane, scale, inv_t, temperature, w);
      S sum = 0;
      bool barred = false;                     // a listed class has probability zero
      if constexpr (ROWS) {
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          S e;
          const float x = pick_class(w.x, w.c[j], w.e, e);
          const S d = x == neg_inf() ? (S)__builtin_inff() : w.off * unit + ((S)w.a[j] - ((S)x - (S)w.m));
          barred = barred || (d == (S)__builtin_inff() && w.p[j] != (S)0);
          sum += w.p[j] == (S)0 ? (S)0 : w.p[j] * d;
        }
        const S d = w.sum_rest == (S)0 ? (S)__builtin_inff() : w.off_rest * unit;
        sum += w.p_rest == (S)0 ? (S)0 : w.p_rest * d;
      } else {
        const float inv = w.sum == 0.f ? 0.f : rcp_f(w.sum);
        // slot j; the q of a class that an earlier slot names counts there
        const auto part_of = [&](int j, bool again) {
          float e;
          const float x = pick_class(w.x, w.c[j], w.e, e);
          const bool none = x == neg_inf();
          barred |= none & w.alive[j];
          const float d = none ? 0.f : fmaf(w.off, unit, w.a[j] - (x - w.m)), pd = w.p[j] * d;       // d = T log(p / q)
          return again ? fmaf(-temperature, w.p[j], pd) : kl_part(w.p[j], e * inv, d * (float)inv_t, pd, temperature);
        };
#pragma unroll
        for (int j = 0; j < KS; ++j) sum += part_of(j, false);
        if (w.twice) {                         // rarely: once more
          sum = 0;
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            bool again = false;
#pragma unroll
            for (int i = 0; i < j; ++i) again |= w.c[i] == w.c[j];
            sum += part_of(j, again);
          }
        }
        sum = barred ? sum + __builtin_inff() : in_range(sum);
        const float q = w.sum_rest * w.to_m * inv;
        // (a small share of a student's lowest values is a number where their distance is past the largest one)
        const double l = w.off_rest * 0.6931471805599453;
        const float part = kl_part(w.p_rest, q, (float)l, (float)((double)w.p_rest * (l * (double)temperature)), temperature);
        sum += w.sum_rest == 0.f && w.rest_alive ? __builtin_inff() : w.p_rest == 0.f ? temperature * q : part;
      }
      float loss = (float)(sum * (S)temperature);              // the terms are T (log p - log q)
      loss = w.state == 1 ? loss : w.state ? __builtin_nanf("") : 0.f;
      if (ROWS) per_row[n * s.V + v0 + lane] = loss;
      loss_sum += (double)loss;
      count += w.state ? 1 : 0;
    }
  }
  if (partial) {
    loss_sum = block_sum<256>(loss_sum, s_red);
    const double counted = block_sum<256>((double)count, s_red);
    if (threadIdx.x == 0) {
      const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
      partial[2 * b] = loss_sum;
      partial[2 * b + 1] = counted;
    }
  }
}

template <typename T, int KT, int KS, bool FULL, bool REST>
__global__ void __launch_bounds__(256)
k_distill_few_bwd(const T* __restrict__ z, RowShape s, Teacher t, float scale, double inv_t, float temperature,
                  const float* __restrict__ scal, const float* __restrict__ grad, int grad_rows, T* __restrict__ dz, RowShape d) {
  const float g_all = grad_rows ? 0.f : grad[0] * scal[0];
  const int64_t tiles = (s.V + 255) / 256;
  for (int64_t n = blockIdx.y; n < s.N; n += gridDim.y) {
    for (int64_t i = blockIdx.x; i < tiles; i += gridDim.x) {
      const int64_t v0 = (int64_t)scalar((int)i) * 256;
      const uint32_t lane = lane_id();
      if (v0 + lane >= s.V) continue;
      const float f = temperature * (grad_rows ? lane_load(grad + n * s.V + v0, lane) : g_all);
      FewRow<KT, KS, float> w;
      few_row<T, KT, KS, FULL, REST, FEW_GRADIENT>(z, s, t, n, v0, lane, scale, inv_t, temperature, w);
      const float w_rest = REST && w.sum_rest != 0.f ? w.to_m * w.inv - w.p_rest * rcp_f(w.sum_rest) : 0.f;
      const float fill = w.state ? __builtin_nanf("") : 0.f;
      float out[KT];
#pragma unroll
      for (int c = 0; c < KT; ++c) {
        float share = 0.f;
#pragma unroll
        for (int j = 0; j < KS; ++j) share += w.c[j] == c ? +w.p[j] : 0.f;
        const bool l = !REST || ((w.listed >> c) & 1u);
        out[c] = f * (l ? fmaf(w.e[c], w.inv, -share) : w.e[c] * w_rest);
        out[c] = w.state == 1 ? +out[c] : fill;
      }
      store_row<T, KT, FULL>(dz + n * d.sN + (v0 + lane) * d.sV, d.sK, s.K, out);
    }
  }
}

// ---- a few dozen classes and many rows: one thread a row (rows.h), with the arithmetic of the few.
// the teacher of one lane's row: largest value, whether a slot is filled, whether one names no class; f(j, value, class)
template <typename F>
__device__ __forceinline__ void each_slot(const Teacher& t, int64_t at, int K, F f) {
  for (int j = 0; j < t.o.K; ++j) {
    const int64_t i = at + j * t.o.sK;
    const float v = slot_value(t, i);
    const int c = class_at(t.indices, t.index_kind, i);
    if (v != neg_inf()) f(j, v, c);
  }
}

template <typename T, bool UNIT>
__global__ void __launch_bounds__(256)
k_distill_lane_fwd(const T* __restrict__ z, RowShape s, Teacher t, float scale, double inv_t, float temperature,
                   RowStats* __restrict__ stats, float* __restrict__ per_row, double* __restrict__ partial) {
  __shared__ uint32_t s_bits[256 * (LANE_CLASSES / 32 + 1)];       // a row's words, one apart from the next lane's
  __shared__ double s_red[4];
  const double scale_d = inv_t * 1.4426950408889634;
  const int K = s.K, words = (K + 31) / 32;
  uint32_t* const bits = s_bits + threadIdx.x * (LANE_CLASSES / 32 + 1);
  const int64_t NV = s.N * s.V;
  double loss_sum = 0.;
  int count = 0;
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < NV; r += (int64_t)gridDim.x * 256) {
    const T* p = z + row_offset(s, r);
    const int64_t at = row_offset(t.o, r);
    float hi = neg_inf();
    bool any = false, bad = false, twice = false;
    for (int i = 0; i < words; ++i) bits[i] = 0;
    if (!row_masked(t, r)) {
      each_slot(t, at, K, [&](int, float v, int c) {
        any = true;
        hi = fmaxf(hi, v);
        if (c < 0 || c >= K) bad = true;
        else {
          twice = twice || ((bits[c >> 5] >> (c & 31)) & 1u);
          bits[c >> 5] |= 1u << (c & 31);
        }
      });
    }
    float loss = 0.f;
    RowStats st = not_counted();
    if (any && bad) {
      loss = __builtin_nanf("");
      st = RowStats{0.f, loss, 0.f, loss};
    } else if (any) {
      LaneSum in = {neg_inf(), 0.}, left = {neg_inf(), 0.};                // listed classes, and all others
      for (int c = 0; c < K; c += 8) {
        float x[8];
        load8<T, UNIT>(p, s.sK, c, K, x);
        const uint32_t b = (bits[c >> 5] >> (c & 31)) & 255u;
        if (b) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if ((b >> i) & 1u) {
              const float xi = x[i];
              in.add_one(xi, scale);
              x[i] = neg_inf();
            }
          }
        }
        left.add(x, scale);
      }
      const float m_all = fmaxf(in.m, left.m), m = m_all == neg_inf() ? 0.f : m_all;
      const float ref = left.m == neg_inf() ? 0.f : left.m;
      const double d_rest = left.m == neg_inf() ? 0. : ((double)left.m - (double)m) * scale_d, to_m = exp2_series(d_rest);
      const double sum = left.s * to_m + (in.m == neg_inf() ? in.s : in.s * exp2_series(((double)in.m - (double)m) * scale_d));
      const double a_rest = t.rest ? rest_gap(t.rest[r], hi, inv_t, temperature) * 1.4426950408889634 : -__builtin_inf();
      const double shift = fmax(a_rest, 0.), e_rest = exp2_series(a_rest - shift);
      double sum_t = e_rest;
      each_slot(t, at, K, [&](int, float v, int) { sum_t += exp2_series(fma((double)v - (double)hi, scale_d, -shift)); });
      const double ls_t = log2_newton(sum_t) + shift, ls = log2_newton(sum), p_rest = e_rest / sum_t;
      double kl = kl_part(a_rest - ls_t, left.s == 0. ? -__builtin_inf() : d_rest + log2_newton(left.s) - ls);
      each_slot(t, at, K, [&](int j, float v, int c) {
        const float x = (float)p[(int64_t)c * s.sK];
        const double logq = x == neg_inf() ? -__builtin_inf() : fma((double)x - (double)m, scale_d, -ls);
        kl += kl_part(fma((double)v - (double)hi, scale_d, -ls_t), logq);
        if (twice) {                           // the q of a class in two slots counts once
          bool again = false;
          each_slot(t, at, K, [&](int j2, float, int c2) { again = again || (j2 < j && c2 == c); });
          if (again) kl -= exp2_series(logq);
        }
      });
      loss = (float)(kl * (double)temperature * (double)temperature);
      const float inv = sum == 0. ? 0.f : rcp_f((float)sum);
      st = RowStats{ref, left.s == 0. ? 0.f : (float)to_m * inv - (float)p_rest * rcp_f((float)left.s), m, inv};
    }
    if (per_row) per_row[r] = loss;
    if (stats) stats[r] = st;
    loss_sum += (double)loss;
    count += any ? 1 : 0;
  }
  if (partial) {
    loss_sum = block_sum<256>(loss_sum, s_red);
    const double counted = block_sum<256>((double)count, s_red);
    if (threadIdx.x == 0) {
      partial[2 * blockIdx.x] = loss_sum;
      partial[2 * blockIdx.x + 1] = counted;
    }
  }
}

template <typename T, bool UNIT>
__global__ void __launch_bounds__(256)
k_distill_lane_bwd(const T* __restrict__ z, RowShape s, Teacher t, float scale, double inv_t, float temperature,
                   const RowStats* __restrict__ stats, const float* __restrict__ scal, const float* __restrict__ grad, int grad_rows,
                   T* __restrict__ dz, RowShape d) {
  const int K = s.K;
  const int64_t NV = s.N * s.V;
  const float g_all = grad_rows ? 0.f : grad[0] * scal[0];
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < NV; r += (int64_t)gridDim.x * 256) {
    const T* p = z + row_offset(s, r);
    T* q = dz + row_offset(d, r);
    RowStats st = not_counted();
    if (!row_masked(t, r)) st = stats[r];
    const bool live = !(st.ref == __builtin_inff() && st.w == 0.f);
    const float f = temperature * (grad_rows ? grad[r] : g_all), w = f * st.w;
    for (int c = 0; c < K; c += 8) {
      float x[8];
      load8<T, UNIT>(p, s.sK, c, K, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = live ? exp2_f((x[i] - st.ref) * scale) * w : 0.f;
      if (UNIT && c + 8 <= K) {
        if constexpr (sizeof(T) == 2) store_vec<false>(q + c, x);
        else {
          store_vec<false>(q + c, *(const float(*)[4])x);
          store_vec<false>(q + c + 4, *(const float(*)[4])(x + 4));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (c + i < K) q[(int64_t)(c + i) * d.sK] = (T)x[i];
      }
    }
    if (live && !(st.w != st.w && st.inv_s != st.inv_s)) {           // a NaN row is NaN as it stands
      // (shares in fp32 with the hardware's reciprocal: the class's own exponential, from which they are taken off, is no better)
      const int64_t at = row_offset(t.o, r);
      float hi = neg_inf(), shift = 0.f, sum = 0.f;
      each_slot(t, at, K, [&](int, float v, int) { hi = fmaxf(hi, v); });
      if (t.rest) {
        const float a_rest = (float)(rest_gap(t.rest[r], hi, inv_t, temperature) * 1.4426950408889634);
        shift = fmaxf(a_rest, 0.f);
        sum = exp2_f(a_rest - shift);
      }
      each_slot(t, at, K, [&](int, float v, int) { sum += exp2_f(fmaf(v - hi, scale, -shift)); });
      const float inv_sum = rcp_f(sum);
      each_slot(t, at, K, [&](int, float, int c) {
        if (c < 0 || c >= K) return;           // the forward would have seen it: the slots have been rewritten since
        float share = 0.f;
        each_slot(t, at, K, [&](int, float v, int c2) { share += c2 == c ? exp2_f(fmaf(v - hi, scale, -shift)) : 0.f; });
        const float x = (float)p[(int64_t)c * s.sK];
        const float qc = x == neg_inf() ? 0.f : exp2_f((x - st.m) * scale) * st.inv_s;
        q[(int64_t)c * d.sK] = (T)(f * (qc - share * inv_sum));
      });
    }
  }
}

static RowShape student_rows(const devis_distill_params* a) { return {a->sN, a->sV, a->sK, a->N, a->V, (int)a->K}; }
static RowShape slot_rows(const devis_distill_params* a) { return {a->oN, a->oV, a->oK, a->N, a->V, (int)a->k}; }
// few classes, and rows that a 32-bit offset reaches from the block's first
static bool few_classes(const devis_distill_params* a) {
  return a->K <= FEW_CLASSES && (a->V == 1 ? a->sN : a->sV) <= FEW_STRIDE && (a->V == 1 ? a->oN : a->oV) <= FEW_STRIDE &&
         side_by_side(student_rows(a), slot_rows(a));
}

// one block a row, or for short rows as many blocks as run at once
static bool long_rows(const devis_distill_params* a) {
  return a->K > DIS_SHORT && !(a->N * a->V >= DIS_SHORT_ROWS && a->K * (a->dtype == DEVIS_F32 ? 4 : 2) <= DIS_SHORT_BYTES);
}
// fewer rows than CUs: a block four times as large takes each (forward + backward, us, 1024 and 256 threads: 16 fp32 rows of
// 8192 17, 17, of 16384 18, 19, of 32768 19, 22; 200 rows of 32768 25, 29, of 131072 bf16 41, 47; 300 rows of 32768 36, 34)
static bool few_rows(const devis_distill_params* a) { return a->K >= 16384 && a->N * a->V < 256; }
static dim3 distill_grid(const devis_distill_params* a) {
  const int64_t NV = a->N * a->V;
  return long_rows(a) ? row_grid(NV) : dim3((unsigned)(NV < DIS_MAX_WAVES ? NV : DIS_MAX_WAVES));
}
static int64_t distill_partials(const devis_distill_params* a) { return long_rows(a) ? a->N * a->V : DIS_MAX_WAVES; }

static bool distill_args_ok(const devis_distill_params* a, const void* logits) {
  if (!a || !logits || !a->values || !a->indices) return false;
  if (!rows_ok(a->sN, a->sV, a->sK, a->N, a->V, a->K) || !rows_ok(a->oN, a->oV, a->oK, a->N, a->V, a->K)) return false;
  if (a->k < 1 || a->k > a->K || a->k > DIS_MAX_K || a->index_dtype < 0 || a->index_dtype > 2) return false;
  if (!(a->temperature > 0x1p-100f) || !(a->temperature < 0x1p100f)) return false;
  if (a->values_dtype != DEVIS_F32 && a->values_dtype != DEVIS_BF16) return false;
  return a->dtype == DEVIS_F32 || a->dtype == DEVIS_BF16;
}

}  // namespace devis

using namespace devis;

// KERNEL(KT, KS, FULL, FLAG); the slots are bounded at 2, 4 or the classes, because they are half of the work of a row
#define DISTILL_FEW_FULL(KERNEL, KT, KS, FLAG) do { if (unit && a->K == KT) KERNEL(KT, KS, true, FLAG); else KERNEL(KT, KS, false, FLAG); } while (0)
#define DISTILL_FEW_KS(KERNEL, KT, FLAG) do { if (a->k <= 2) DISTILL_FEW_FULL(KERNEL, KT, 2, FLAG); else if (a->k <= 4) DISTILL_FEW_FULL(KERNEL, KT, 4, FLAG); else DISTILL_FEW_FULL(KERNEL, KT, KT, FLAG); } while (0)
#define DISTILL_FEW_KT(KERNEL, FLAG)                                                                              \
  do {                                                                                                            \
    if (a->K <= 2) DISTILL_FEW_FULL(KERNEL, 2, 2, FLAG);                                                          \
    else if (a->K <= 4) DISTILL_FEW_KS(KERNEL, 4, FLAG);                                                          \
    else if (a->K <= 8) DISTILL_FEW_KS(KERNEL, 8, FLAG);                                                          \
    else DISTILL_FEW_KS(KERNEL, 16, FLAG);                                                                        \
  } while (0)

#define DISTILL_DISPATCH(KERNEL)                                                                                  \
  DEVIS_DISPATCH_DTYPE(a->dtype, {                                                                                \
    if (!long_rows(a)) { if (unit) KERNEL(true, 64); else KERNEL(false, 64); }                                    \
    else if (unit && few_rows(a)) KERNEL(true, 1024);                                                             \
    else if (unit) KERNEL(true, 256);                                                                             \
    else KERNEL(false, 256);                                                                                      \
  })

extern "C" {

size_t devis_distill_workspace_bytes(const devis_distill_params* a) {
  return a && a->N > 0 && a->V > 0 ? (size_t)(distill_partials(a) + DIS_STAGE) * 2 * sizeof(double) : 0;
}

size_t devis_distill_stats_bytes(const devis_distill_params* a) {
  return a && a->N > 0 && a->V > 0 && !few_classes(a) ? (size_t)a->N * (size_t)a->V * sizeof(RowStats) : 0;
}

int devis_distill_fwd(const devis_distill_params* a, const void* logits, float* per_row, float* loss, float* scal, void* stats,
                      void* ws, size_t ws_bytes, void* stream) {
  if (!distill_args_ok(a, logits) || (!per_row && !loss) || (loss && (!ws || !scal))) return DEVIS_ERR_BAD_ARG;
  if (loss && ws_bytes < devis_distill_workspace_bytes(a)) return DEVIS_ERR_WORKSPACE;
  RowShape s = student_rows(a);
  Teacher t = {a->values, a->indices, a->rest, a->row_mask, slot_rows(a), a->values_dtype, a->index_dtype};
  const double inv_t = 1.0 / (double)a->temperature;
  const float scale = (float)(1.4426950408889634 * inv_t);
  const bool unit = a->sK == 1;
  const dim3 rows = distill_grid(a);
  int64_t parts = long_rows(a) ? a->N * a->V : rows.x;
  double* part = loss ? (double*)ws : nullptr;
  if (few_classes(a)) {
    if (one_stride(s) && one_stride(t.o)) { merge_rows(s); merge_rows(t.o); }
    const dim3 grid = few_grid(s.N, s.V, DIS_MAX_BLOCKS);
    parts = (int64_t)grid.x * grid.y;
#define LAUNCH_FEW_R(KT, KS, FULL, ROWS) hipLaunchKernelGGL((k_distill_few_fwd<T, KT, KS, FULL, ROWS>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)logits, s, t, scale, inv_t, a->temperature, per_row, part)
    DEVIS_DISPATCH_DTYPE(a->dtype, { if (per_row) DISTILL_FEW_KT(LAUNCH_FEW_R, true); else DISTILL_FEW_KT(LAUNCH_FEW_R, false); });
#undef LAUNCH_FEW_R
  } else if (lane_rows(a->N * a->V, a->K, a->k)) {
    const int64_t blocks = cdiv(a->N * a->V, 256);
    parts = blocks < DIS_MAX_BLOCKS ? blocks : DIS_MAX_BLOCKS;
#define LAUNCH_LANE(UNIT) hipLaunchKernelGGL((k_distill_lane_fwd<T, UNIT>), dim3((unsigned)parts), dim3(256), 0, (hipStream_t)stream, (const T*)logits, s, t, scale, inv_t, a->temperature, (RowStats*)stats, per_row, part)
    DEVIS_DISPATCH_DTYPE(a->dtype, { if (unit) LAUNCH_LANE(true); else LAUNCH_LANE(false); });
#undef LAUNCH_LANE
  } else {
#define LAUNCH_DISTILL_FWD(UNIT, BS) hipLaunchKernelGGL((k_distill_fwd<T, UNIT, BS>), rows, dim3(BS), 0, (hipStream_t)stream, (const T*)logits, s, t, scale, inv_t, a->temperature, (RowStats*)stats, per_row, part)
    DISTILL_DISPATCH(LAUNCH_DISTILL_FWD);
  }
#undef LAUNCH_DISTILL_FWD
  const int rc = launch_status();
  if (rc || !loss) return rc;
  if (parts > DIS_FINAL) {
    hipLaunchKernelGGL(k_distill_stage, dim3(DIS_STAGE), dim3(256), 0, (hipStream_t)stream, (const double*)part, parts, part + 2 * parts);
    part += 2 * parts;
    parts = DIS_STAGE;
  }
  hipLaunchKernelGGL(k_distill_finalize, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const double*)part, (int)parts, a->mean, loss, scal);
  return launch_status();
}

int devis_distill_bwd(const devis_distill_params* a, const void* logits, const void* stats, const float* scal, const float* grad,
                      int grad_rows, void* dlogits, int64_t dN, int64_t dV, int64_t dK, void* stream) {
  if (!distill_args_ok(a, logits) || (!stats && !few_classes(a)) || !grad || !dlogits || (!grad_rows && !scal)) return DEVIS_ERR_BAD_ARG;
  if (!rows_ok(dN, dV, dK, a->N, a->V, a->K)) return DEVIS_ERR_BAD_ARG;
  RowShape s = student_rows(a), d = {dN, dV, dK, a->N, a->V, (int)a->K};
  Teacher t = {a->values, a->indices, a->rest, a->row_mask, slot_rows(a), a->values_dtype, a->index_dtype};
  const double inv_t = 1.0 / (double)a->temperature;
  const float scale = (float)(1.4426950408889634 * inv_t);
  const bool unit = a->sK == 1 && dK == 1;
  if (few_classes(a)) {
    if (one_stride(s) && one_stride(t.o) && one_stride(d)) { merge_rows(s); merge_rows(t.o); merge_rows(d); }
    const dim3 grid = few_grid(s.N, s.V, 8192);
#define LAUNCH_FEW(KT, KS, FULL, REST) hipLaunchKernelGGL((k_distill_few_bwd<T, KT, KS, FULL, REST>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)logits, s, t, scale, inv_t, a->temperature, scal, grad, grad_rows, (T*)dlogits, d)
    DEVIS_DISPATCH_DTYPE(a->dtype, { if (a->rest) DISTILL_FEW_KT(LAUNCH_FEW, true); else DISTILL_FEW_KT(LAUNCH_FEW, false); });
#undef LAUNCH_FEW
    return launch_status();
  }
  const dim3 rows = distill_grid(a);
  if (lane_rows(a->N * a->V, a->K, a->k)) {
    const int64_t blocks = cdiv(a->N * a->V, 256);
    const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
#define LAUNCH_LANE(UNIT) hipLaunchKernelGGL((k_distill_lane_bwd<T, UNIT>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)logits, s, t, scale, inv_t, a->temperature, (const RowStats*)stats, scal, grad, grad_rows, (T*)dlogits, d)
    DEVIS_DISPATCH_DTYPE(a->dtype, { if (unit) LAUNCH_LANE(true); else LAUNCH_LANE(false); });
#undef LAUNCH_LANE
    return launch_status();
  }
  const bool past = (double)(a->N * a->V) * (double)a->K * (a->dtype == DEVIS_F32 ? 4 : 2) >= DIS_PAST_BYTES;
#define LAUNCH_DISTILL_BWD(UNIT, PAST, BS) hipLaunchKernelGGL((k_distill_bwd<T, UNIT, PAST, BS>), rows, dim3(BS), 0, (hipStream_t)stream, (const T*)logits, s, t, scale, inv_t, a->temperature, (const RowStats*)stats, scal, grad, grad_rows, (T*)dlogits, d)
  DEVIS_DISPATCH_DTYPE(a->dtype, {
    if (!long_rows(a)) { if (unit) LAUNCH_DISTILL_BWD(true, false, 64); else LAUNCH_DISTILL_BWD(false, false, 64); }
    else if (!unit) LAUNCH_DISTILL_BWD(false, false, 256);
    else if (few_rows(a)) LAUNCH_DISTILL_BWD(true, false, 1024);
    else if (past) LAUNCH_DISTILL_BWD(true, true, 256);
    else LAUNCH_DISTILL_BWD(true, false, 256);
  });
#undef LAUNCH_DISTILL_BWD
  return launch_status();
}

}  // extern "C"
