// Verification of drafted classes against a target's probabilities, with the random numbers given.
//
//   a sequence of n drafted classes d_0..d_{n-1}:  d_t is accepted while  u_t q_t[d_t] < p_t[d_t]  (u_t < p_t[d_t]
//   without the drafter's probabilities q);  a = the number accepted before the first that is not.
//   One class is then drawn: weights w = max(p_a - q_a, 0) if a < n (without q: p_a with d_a taken out; p_a itself if
//   nothing is left of it), w = p_n if all were accepted and the target has a row n;  the drawn class is the first c
//   with  sum_{c' <= c} w  >  r sum w.
//
// What is accepted and drawn is then distributed as the target's own draws.  Products and sums are fp64: the class
// drawn next to a border depends on them (fp32 would move the border by up to 1e-5 of the mass at 10^5 classes).
// A weight that is not above zero (NaN among them) counts as zero; r that is not below 1 draws the last class with
// weight.
#include "rows.h"

namespace devis {

struct VerifyArgs {
  const void* tokens; const float* accept_u; const float* sample_u; const void* lengths;
  void* out_tokens; void* out_accepted;
  int64_t B; int T, Tp, K;
  int64_t pB, pT, pK, qB, qT, qK;
  int token_kind;                             // DEVIS_LABEL_I64 or _I32: tokens, lengths and both outputs
};

__device__ __forceinline__ int64_t int_at(const void* p, int kind, int64_t i) {
  return kind == DEVIS_LABEL_I32 ? (int64_t)((const int32_t*)p)[i] : ((const int64_t*)p)[i];
}
__device__ __forceinline__ void put_int(void* p, int kind, int64_t i, int64_t v) {
  if (kind == DEVIS_LABEL_I32) ((int32_t*)p)[i] = (int32_t)v;
  else ((int64_t*)p)[i] = v;
}
__device__ __forceinline__ int draft_length(const VerifyArgs& a, int64_t b) {
  if (!a.lengths) return a.T;
  const int64_t n = int_at(a.lengths, a.token_kind, b);
  return n < 0 ? 0 : n > a.T ? a.T : (int)n;
}

// is draft t of sequence b accepted?  A class outside [0, K) has probability zero.
template <typename T>
__device__ __forceinline__ bool draft_ok(const VerifyArgs& a, const T* p, const T* q, int64_t b, int t) {
  const int64_t d = int_at(a.tokens, a.token_kind, b * a.T + t);
  if (d < 0 || d >= a.K) return false;
  const double pd = (double)(float)p[b * a.pB + t * a.pT + d * a.pK];
  double u = (double)a.accept_u[b * a.T + t];
  if (q) u *= (double)(float)q[b * a.qB + t * a.qT + d * a.qK];
  return u < pd;
}

// what one sequence's class is drawn from
template <typename T> struct Draw {
  const T* p; const T* q;                     // q null: the target's row alone
  int64_t pK, qK;
  int skip;                                   // class taken out, -1 none
};
__device__ __forceinline__ double weight_of(float x, float y, bool keep) {
  const double w = (double)x - (double)y;
  return w > 0. && keep ? w : 0.;
}

// f(w, c): the weights of classes c, c + 1, .. of [lo, hi), dealt vector by vector to `stride` threads of which this is
// number `me`; four vectors of each model in flight.
template <typename T, bool UNIT, bool DRAFTER, typename F>
__device__ __forceinline__ void each_weight(const Draw<T>& d, int lo, int hi, int me, int stride, F f) {
  const auto one = [&](int c) {
    double w[1] = {weight_of((float)d.p[(int64_t)c * (UNIT ? 1 : d.pK)], DRAFTER && d.q ? (float)d.q[(int64_t)c * (UNIT ? 1 : d.qK)] : 0.f, c != d.skip)};
    f(w, c);
  };
  if constexpr (UNIT) {
    constexpr int VEC = vec_of<T>();
    const int full = (hi - lo) / VEC;
    const bool two = DRAFTER && d.q;
    const auto vec = [&](const Raw16& rp, const Raw16& rq, int c) {
      float x[VEC], y[VEC];
      unpack(rp, x);
      unpack(rq, y);
      double w[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = weight_of(x[i], y[i], c + i != d.skip);
      f(w, c);
    };
    int v = me;
    for (; v + 3 * stride < full; v += 4 * stride) {
      Raw16 rp[4], rq[4] = {};
#pragma unroll
      for (int u = 0; u < 4; ++u) rp[u] = load16(d.p + lo + (int64_t)(v + u * stride) * VEC);
      if (two) {
#pragma unroll
        for (int u = 0; u < 4; ++u) rq[u] = load16(d.q + lo + (int64_t)(v + u * stride) * VEC);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) vec(rp[u], rq[u], lo + (v + u * stride) * VEC);
    }
    for (; v < full; v += stride) {
      Raw16 rq = {};
      if (two) rq = load16(d.q + lo + (int64_t)v * VEC);
      vec(load16(d.p + lo + (int64_t)v * VEC), rq, lo + v * VEC);
    }
    const int c = lo + full * VEC + me;
    if (c < hi) one(c);
  } else {
    for (int c = lo + me; c < hi; c += stride) one(c);
  }
}

// One block a sequence, of 64, 256 or 1024 threads (verify_threads).  Each wave sums the weights of one stretch of the row; the
// stretch in which the goal lies is read once more, a vector a thread, and the class found by a prefix sum over the block.
// 200 sequences of 7 drafts over 131072 bf16 classes: 22 us, 105 MB; one sequence of 4 over 32768 fp32: 8.3 us.
template <typename T, bool UNIT, bool DRAFTER, int BS>
__global__ void __launch_bounds__(BS)
k_verify(const T* __restrict__ p, const T* __restrict__ q, VerifyArgs a) {
  constexpr int WAVES = BS / 64, VEC = UNIT ? vec_of<T>() : 1;
  __shared__ double s_sum[WAVES], s_scan[WAVES];
  __shared__ int s_n, s_pick, s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x) {
    const int len = draft_length(a, b);
    if (tid < 64) {
      int n = len;
      for (int t0 = 0; t0 < len; t0 += 64) {
        const int t = t0 + lane;
        const bool ok = t >= len || draft_ok(a, p, q, b, t);
        const unsigned long long bad = __ballot(!ok);
        if (bad) { n = t0 + __ffsll(bad) - 1; break; }
      }
      if (lane == 0) { s_n = n; s_pick = 0x7fffffff; s_last = -1; }
    }
    __syncthreads();
    const int n = s_n;
    int drawn = -1;
    if (n < a.Tp) {                            // else all are accepted and there is no row behind them
      Draw<T> d = {p + b * a.pB + n * a.pT, nullptr, a.pK, a.qK, -1};
      if (n < len) {
        if (DRAFTER) d.q = q + b * a.qB + n * a.qT;
        else {
          const int64_t c = int_at(a.tokens, a.token_kind, b * a.T + n);
          d.skip = c < 0 || c >= a.K ? -1 : (int)c;
        }
      }
      const int stretch = ((a.K + WAVES - 1) / WAVES + 64 * VEC - 1) / (64 * VEC) * (64 * VEC);
      double total = 0.;
      for (int round = 0; round < 2; ++round) {
        const int64_t lo = (int64_t)wave * stretch;
        double sum = 0.;
        if (lo < a.K) {
          const int hi = lo + stretch < a.K ? (int)(lo + stretch) : a.K;
          each_weight<T, UNIT, DRAFTER>(d, (int)lo, hi, lane, 64, [&](auto& w, int) { sum += sum_of(w); });
        }
        sum = wave_sum(sum);
        if (lane == 0) s_sum[wave] = sum;
        __syncthreads();
        total = 0.;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) total += s_sum[i];
        if (total > 0. || (!d.q && d.skip < 0)) break;
        d.q = nullptr;                         // nothing is left over: the target's row itself
        d.skip = -1;
        __syncthreads();
      }
      if (total > 0.) {
        const double goal = (double)a.sample_u[b] * total;
        // the stretch in which the running sum passes the goal, or the last that holds weight
        int pick = 0;
        double before = 0., run = 0.;
        bool open = true;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
          if (open && s_sum[i] > 0.) {
            pick = i;
            before = run;
            open = !(run + s_sum[i] > goal);
          }
          run += s_sum[i];
        }
        const int lo = pick * stretch, hi = lo + (int64_t)stretch < a.K ? lo + stretch : a.K;
        run = before;
        for (int c0 = lo; c0 < hi; c0 += BS * VEC) {
          // this thread's VEC classes
          const int64_t c = (int64_t)c0 + tid * VEC;
          double w[VEC];
          if (UNIT && c + VEC <= hi) {
            float x[VEC], y[VEC] = {};
            if constexpr (UNIT) {
              unpack(load16(d.p + c), x);
              if (DRAFTER && d.q) unpack(load16(d.q + c), y);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[i] = weight_of(x[i], y[i], c + i != d.skip);
          } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              w[i] = c + i < hi ? weight_of((float)d.p[(c + i) * a.pK], DRAFTER && d.q ? (float)d.q[(c + i) * a.qK] : 0.f, c + i != d.skip) : 0.;
          }
          double mine = 0.;
#pragma unroll
          for (int i = 0; i < VEC; ++i) mine += w[i];
          double scan = mine;
#pragma unroll
          for (int o = 1; o < 64; o <<= 1) {
            const double up = __shfl_up(scan, o, 64);
            if (lane >= o) scan += up;
          }
          if (lane == 63) s_scan[wave] = scan;
          __syncthreads();
          double at = run + (scan - mine);
#pragma unroll
          for (int i = 0; i < WAVES; ++i) {
            if (i < wave) at += s_scan[i];
            run += s_scan[i];
          }
          int here = -1, last = -1;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            at += w[i];
            if (w[i] > 0.) {
              last = (int)c + i;
              if (here < 0 && at > goal) here = last;
            }
          }
          // lanes are in class order: the first lane that passes, the last that holds weight
          const unsigned long long passes = __ballot(here >= 0), holds = __ballot(last >= 0);
          if (passes && lane == __ffsll(passes) - 1) atomicMin(&s_pick, here);
          if (holds && lane == 63 - __clzll((long long)holds)) atomicMax(&s_last, last);
          __syncthreads();
          if (s_pick != 0x7fffffff) break;
        }
        drawn = s_pick != 0x7fffffff ? s_pick : s_last;
      }
    }
    for (int t = tid; t < a.Tp; t += BS)
      put_int(a.out_tokens, a.token_kind, b * a.Tp + t, t < n ? int_at(a.tokens, a.token_kind, b * a.T + t) : t == n ? drawn : -1);
    if (tid == 0) put_int(a.out_accepted, a.token_kind, b, n);
    __syncthreads();
  }
}

// few classes: one thread a sequence (128^3 voxels of 4 fp32 classes in 25 us, 134 MB; a block a sequence: 5.5 ms).  The rows of each place are loaded whole (they share the cache line that the drafted
// class's own probability is in), so a refused draft is drawn again from registers.
template <typename T, int KT, bool FULL, bool DRAFTER>
__global__ void __launch_bounds__(256)
k_verify_few(const T* __restrict__ p, const T* __restrict__ q, VerifyArgs a) {
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < a.B; b += (int64_t)gridDim.x * 256) {
    const int len = draft_length(a, b);
    int n = 0, drawn = -1;
    for (;; ++n) {
      if (n >= a.Tp) break;                    // all accepted and no row behind them
      float x[KT], y[KT] = {};
      load_row<T, KT, FULL>(p + b * a.pB + n * a.pT, a.pK, a.K, x);
      const bool drafted = n < len;
      int64_t tok = -1;
      if (drafted) {
        tok = int_at(a.tokens, a.token_kind, b * a.T + n);
        double u = (double)a.accept_u[b * a.T + n];
        float pd = 0.f, qd = 0.f;
        if (DRAFTER) load_row<T, KT, FULL>(q + b * a.qB + n * a.qT, a.qK, a.K, y);
#pragma unroll
        for (int c = 0; c < KT; ++c) {
          pd = tok == c ? x[c] : pd;
          if (DRAFTER) qd = tok == c ? y[c] : qd;
        }
        if (DRAFTER) u *= (double)qd;
        if (tok >= 0 && tok < a.K && u < (double)pd) {
          put_int(a.out_tokens, a.token_kind, b * a.Tp + n, tok);
          continue;
        }
      }
      double w[KT], total = 0.;
#pragma unroll
      for (int c = 0; c < KT; ++c) {
        double v = (double)x[c];
        if (DRAFTER) v = drafted ? v - (double)y[c] : v;
        else v = drafted && tok == c ? 0. : v;
        w[c] = (FULL || c < a.K) && v > 0. ? v : 0.;
        total += w[c];
      }
      if (!(total > 0.)) {
        total = 0.;
#pragma unroll
        for (int c = 0; c < KT; ++c) {
          w[c] = (FULL || c < a.K) && x[c] > 0.f ? (double)x[c] : 0.;
          total += w[c];
        }
      }
      const double goal = (double)a.sample_u[b] * total;
      double run = 0.;
      bool open = true;
#pragma unroll
      for (int c = 0; c < KT; ++c) {
        run += w[c];
        drawn = open && w[c] > 0. ? c : drawn;               // the last with weight so far
        open = open && !(w[c] > 0. && run > goal);
      }
      break;
    }
    for (int t = n; t < a.Tp; ++t) put_int(a.out_tokens, a.token_kind, b * a.Tp + t, t == n ? drawn : -1);
    put_int(a.out_accepted, a.token_kind, b, n);
  }
}

// dozens of classes and many sequences (rows.h): one thread a sequence, the weights added up and then walked, 8 at a time
template <typename T, bool UNIT, bool DRAFTER>
__global__ void __launch_bounds__(256)
k_verify_lane(const T* __restrict__ p, const T* __restrict__ q, VerifyArgs a) {
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < a.B; b += (int64_t)gridDim.x * 256) {
    const int len = draft_length(a, b);
    int n = 0, drawn = -1;
    while (n < len && draft_ok(a, p, q, b, n)) {
      put_int(a.out_tokens, a.token_kind, b * a.Tp + n, int_at(a.tokens, a.token_kind, b * a.T + n));
      ++n;
    }
    if (n < a.Tp) {
      Draw<T> d = {p + b * a.pB + n * a.pT, nullptr, a.pK, a.qK, -1};
      if (n < len) {
        if (DRAFTER) d.q = q + b * a.qB + n * a.qT;
        else {
          const int64_t c = int_at(a.tokens, a.token_kind, b * a.T + n);
          d.skip = c < 0 || c >= a.K ? -1 : (int)c;
        }
      }
      const auto weights = [&](int c, double (&w)[8]) {
        float x[8], y[8] = {};
        load8<T, UNIT>(d.p, a.pK, c, a.K, x);                  // -inf behind the last class: no weight
        if (DRAFTER && d.q) load8<T, UNIT>(d.q, a.qK, c, a.K, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = c + i < a.K ? weight_of(x[i], y[i], c + i != d.skip) : 0.;
      };
      double w[8], total = 0.;
      for (int c = 0; c < a.K; c += 8) { weights(c, w); total += sum_of(w); }
      if (!(total > 0.) && (d.q || d.skip >= 0)) {             // nothing is left over: the target's row itself
        d.q = nullptr;
        d.skip = -1;
        total = 0.;
        for (int c = 0; c < a.K; c += 8) { weights(c, w); total += sum_of(w); }
      }
      if (total > 0.) {
        const double goal = (double)a.sample_u[b] * total;
        double run = 0.;
        bool open = true;
        for (int c = 0; c < a.K && open; c += 8) {
          weights(c, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            run += w[i];
            drawn = open && w[i] > 0. ? c + i : drawn;         // the last with weight so far
            open = open && !(w[i] > 0. && run > goal);
          }
        }
      }
    }
    for (int t = n; t < a.Tp; ++t) put_int(a.out_tokens, a.token_kind, b * a.Tp + t, t == n ? drawn : -1);
    put_int(a.out_accepted, a.token_kind, b, n);
  }
}

// Few sequences want a row's read as short as one CU can make it, many the fewest threads that wait for each other.  us, bf16, 5
// drafts, 64 / 256 threads: 4000 sequences of 1000 classes 10, 21; 2000 of 2000 11, 12; 200 of 2000 9, 6; 2000 of 4000 18, 15.
// 256 / 1024 threads: 200 sequences of 4000 6, 8; 200 of 16000 9, 10; 200 of 32000 12, 11; 200 of 64000 22, 15; 64 of 64000 18, 12;
// 500 of 16000 12, 18; 500 of 32000 18, 23; 500 of 64000 31, 31; 1000 of 64000 52, 58; 2000 of 16000 30, 66; 500 of 131072 61, 52.
static int verify_threads(int64_t B, int64_t K) {
  return K <= 1024 ? 64 : K <= 16384 || (K <= 65536 && B >= 256) ? 256 : 1024;
}

}  // namespace devis

using namespace devis;

extern "C" int devis_verify_drafts(const devis_verify_params* v, const void* target, const void* draft, void* out_tokens,
                                   void* out_accepted, void* stream) {
  if (!v || !target || !out_tokens || !out_accepted || !v->sample_u) return DEVIS_ERR_BAD_ARG;
  if (v->B <= 0 || v->T < 0 || v->T > MAX_CLASSES || (v->Tp != v->T && v->Tp != v->T + 1) || v->Tp < 1) return DEVIS_ERR_BAD_ARG;
  if (v->K < 1 || v->K > MAX_CLASSES || (v->T > 0 && (!v->tokens || !v->accept_u))) return DEVIS_ERR_BAD_ARG;
  if (v->token_dtype != DEVIS_LABEL_I64 && v->token_dtype != DEVIS_LABEL_I32) return DEVIS_ERR_BAD_ARG;
  const VerifyArgs a = {v->tokens, v->accept_u, v->sample_u, v->lengths, out_tokens, out_accepted, v->B, (int)v->T, (int)v->Tp,
                        (int)v->K, v->pB, v->pT, v->pK, v->qB, v->qT, v->qK, v->token_dtype};
  if (v->K <= FEW_CLASSES) {
    const dim3 grid = few_grid(1, v->B, 8192);
    const bool unit = v->pK == 1 && (!draft || v->qK == 1);
#define LAUNCH_FEW(DRAFTER, KT, FULL) hipLaunchKernelGGL((k_verify_few<T, KT, FULL, DRAFTER>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)target, (const T*)draft, a)
#define LAUNCH_FEW_DRAFTER(KT, FULL) LAUNCH_FEW(true, KT, FULL)
#define LAUNCH_FEW_ALONE(KT, FULL) LAUNCH_FEW(false, KT, FULL)
    DEVIS_DISPATCH_DTYPE(v->dtype, {
      if (draft) DEVIS_DISPATCH_FEW(v->K, unit, LAUNCH_FEW_DRAFTER);
      else DEVIS_DISPATCH_FEW(v->K, unit, LAUNCH_FEW_ALONE);
    });
#undef LAUNCH_FEW_ALONE
#undef LAUNCH_FEW_DRAFTER
#undef LAUNCH_FEW
    return launch_status();
  }
  // the row is walked two or three times, as if for many slots (3 drafts of 64 classes, 8192 sequences: 15.7 us a lane a sequence,
  // 11.5 a block; 256 classes, 32768: 53 and 36; 1 draft, 500000 of 64: 95 and 334, 200000 of 256: 84 and 139)
  if (lane_rows(v->B, v->K, LANE_SLOTS)) {
    const dim3 grid = few_grid(1, v->B, 8192);
    const bool unit = v->pK == 1 && (!draft || v->qK == 1);
#define LAUNCH_LANE(UNIT, DRAFTER) hipLaunchKernelGGL((k_verify_lane<T, UNIT, DRAFTER>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)target, (const T*)draft, a)
    DEVIS_DISPATCH_DTYPE(v->dtype, {
      if (draft) { if (unit) LAUNCH_LANE(true, true); else LAUNCH_LANE(false, true); }
      else { if (unit) LAUNCH_LANE(true, false); else LAUNCH_LANE(false, false); }
    });
#undef LAUNCH_LANE
    return launch_status();
  }
  const int threads = verify_threads(v->B, v->K);
  const unsigned blocks = (unsigned)(v->B < (1 << 20) ? v->B : (1 << 20));
  const bool unit = v->pK == 1 && (!draft || v->qK == 1);
#define LAUNCH_VERIFY(UNIT, DRAFTER, BS) hipLaunchKernelGGL((k_verify<T, UNIT, DRAFTER, BS>), dim3(blocks), dim3(BS), 0, (hipStream_t)stream, (const T*)target, (const T*)draft, a)
#define LAUNCH_VERIFY_U(DRAFTER, BS) do { if (unit) LAUNCH_VERIFY(true, DRAFTER, BS); else LAUNCH_VERIFY(false, DRAFTER, BS); } while (0)
#define LAUNCH_VERIFY_B(DRAFTER) do { if (threads == 64) LAUNCH_VERIFY_U(DRAFTER, 64); else if (threads == 256) LAUNCH_VERIFY_U(DRAFTER, 256); else LAUNCH_VERIFY_U(DRAFTER, 1024); } while (0)
  DEVIS_DISPATCH_DTYPE(v->dtype, { if (draft) LAUNCH_VERIFY_B(true); else LAUNCH_VERIFY_B(false); });
#undef LAUNCH_VERIFY_B
#undef LAUNCH_VERIFY_U
#undef LAUNCH_VERIFY
  return launch_status();
}
