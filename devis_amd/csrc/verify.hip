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

constexpr int VER_SEGS = 64;                  // segments of a row whose weights are summed apart

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

// the weights of one sequence's draw
template <typename T> struct Draw {
  const T* p; const T* q;                     // q null: the target's row alone
  int64_t pK, qK;
  int skip;                                   // class taken out, -1 none
  __device__ __forceinline__ double whole(int c) const {
    const double x = (double)(float)p[(int64_t)c * pK];
    return x > 0. ? x : 0.;
  }
  __device__ __forceinline__ double weight(int c) const {
    double x = (double)(float)p[(int64_t)c * pK];
    if (q) x -= (double)(float)q[(int64_t)c * qK];
    return x > 0. && c != skip ? x : 0.;
  }
};

template <typename T>
__global__ void __launch_bounds__(256)
k_verify(const T* __restrict__ p, const T* __restrict__ q, VerifyArgs a) {
  __shared__ double s_w[VER_SEGS], s_p[VER_SEGS], s_run[256];
  __shared__ int s_n, s_seg, s_pick, s_last;
  __shared__ bool s_all;
  __shared__ double s_goal;
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
      if (lane == 0) s_n = n;
    }
    __syncthreads();
    const int n = s_n;
    const bool draws = n < a.Tp;
    int drawn = -1;
    if (draws) {
      Draw<T> d = {p + b * a.pB + n * a.pT, nullptr, a.pK, a.qK, -1};
      if (n < len) {
        if (q) d.q = q + b * a.qB + n * a.qT;
        else {
          const int64_t c = int_at(a.tokens, a.token_kind, b * a.T + n);
          d.skip = c < 0 || c >= a.K ? -1 : (int)c;
        }
      }
      const int seg = ((a.K + VER_SEGS - 1) / VER_SEGS + 63) / 64 * 64;       // classes of a segment
      for (int i = 0; i < VER_SEGS / 4; ++i) {
        const int g = wave * (VER_SEGS / 4) + i;
        const int64_t lo = (int64_t)g * seg;
        const int hi = lo + seg < a.K ? (int)(lo + seg) : a.K;
        double w = 0., v = 0.;
        for (int64_t c = lo + lane; c < hi; c += 64) { w += d.weight((int)c); v += d.whole((int)c); }
        w = wave_sum(w);
        v = wave_sum(v);
        if (lane == 0) { s_w[g] = w; s_p[g] = v; }
      }
      __syncthreads();
      if (tid == 0) {
        double total = 0., whole = 0.;
        for (int g = 0; g < VER_SEGS; ++g) { total += s_w[g]; whole += s_p[g]; }
        const bool all = !(total > 0.);
        double* const sum = all ? s_p : s_w;
        const double goal = (double)a.sample_u[b] * (all ? whole : total);
        double run = 0.;
        int pick = -1;
        double before = 0.;
        for (int g = 0; g < VER_SEGS; ++g) {
          if (sum[g] > 0.) {
            pick = g;                          // the last with weight, if the goal is never passed
            before = run;
            if (run + sum[g] > goal) break;
          }
          run += sum[g];
        }
        s_seg = pick;
        s_all = all;
        s_goal = goal - before;
        s_pick = 0x7fffffff;
        s_last = -1;
      }
      __syncthreads();
      const bool all = s_all;
      const int g = s_seg;
      if (g >= 0) {                            // -1: no class has weight
        const int64_t lo = (int64_t)g * seg;
        const int hi = lo + seg < a.K ? (int)(lo + seg) : a.K;
        const int each = (seg + 255) / 256;
        const int64_t c0 = lo + (int64_t)tid * each;
        const int c1 = c0 + each < hi ? (int)(c0 + each) : hi;
        double mine = 0.;
        for (int64_t c = c0; c < c1; ++c) mine += all ? d.whole((int)c) : d.weight((int)c);
        s_run[tid] = mine;
        __syncthreads();
        double run = 0.;
        for (int i = 0; i < tid; ++i) run += s_run[i];
        const double goal = s_goal;
        if (mine > 0.) {
          int last = -1, pick = -1;
          for (int64_t c = c0; c < c1 && pick < 0; ++c) {
            const double w = all ? d.whole((int)c) : d.weight((int)c);
            if (w > 0.) {
              last = (int)c;
              run += w;
              if (run > goal) pick = (int)c;
            }
          }
          if (pick >= 0) atomicMin(&s_pick, pick);
          atomicMax(&s_last, last);
        }
        __syncthreads();
        drawn = s_pick != 0x7fffffff ? s_pick : s_last;
      }
    }
    for (int t = tid; t < a.Tp; t += 256)
      put_int(a.out_tokens, a.token_kind, b * a.Tp + t, t < n ? int_at(a.tokens, a.token_kind, b * a.T + t) : t == n ? drawn : -1);
    if (tid == 0) put_int(a.out_accepted, a.token_kind, b, n);
    __syncthreads();
  }
}

// few classes: one thread a sequence.  The rows of each place are loaded whole (they share the cache line that the drafted
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

}  // namespace devis

using namespace devis;

extern "C" int devis_verify_drafts(const devis_verify_params* v, const void* target, const void* draft, void* out_tokens,
                                   void* out_accepted, void* stream) {
  if (!v || !target || !out_tokens || !out_accepted || !v->sample_u) return DEVIS_ERR_BAD_ARG;
  if (v->B <= 0 || v->T < 0 || v->T > 0x7ffffffe || (v->Tp != v->T && v->Tp != v->T + 1) || v->Tp < 1) return DEVIS_ERR_BAD_ARG;
  if (v->K < 1 || v->K >= 0x7fffffff || (v->T > 0 && (!v->tokens || !v->accept_u))) return DEVIS_ERR_BAD_ARG;
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
  const unsigned blocks = (unsigned)(v->B < (1 << 20) ? v->B : (1 << 20));
  DEVIS_DISPATCH_DTYPE(v->dtype, hipLaunchKernelGGL(k_verify<T>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, (const T*)target, (const T*)draft, a));
  return launch_status();
}
