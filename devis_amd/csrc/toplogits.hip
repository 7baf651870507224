// The k largest logits of every row and the log-sum-exp of what is left: a teacher's row reduced to what
// distillation (distill.hip) learns from.
//
//   order the classes by (value descending, class ascending); values / indices = the first k;
//   rest = log sum over the classes not among them of exp(z_c / T).
//
// A class is its 64-bit key (value as an ordered integer, class counted downwards), so keys differ and every tie falls to
// the lowest class.  Bound by memory: one read of the row.  Long rows (k_top_wide): 2048 x 131072 bf16, 64 kept, in 112 us =
// 4.8 TB/s (two reads of the row, as k_top_rows does it: 196 us).  Few classes (k_top_few): 2 x 128^3 x 4 fp32 in 22 us,
// 126 MB.  Dozens of classes (k_top_lane): 2 x 64^3 x 104 bf16, 5 kept, in 157 us, classes first 174.
#include "rows.h"

namespace devis {

constexpr int TOP_MAX_K = DEVIS_TOP_MAX_K;
constexpr int TOP_CAP = 1024;                 // list entries; >= 8 * TOP_MAX_K, see the refinement below

__device__ __forceinline__ float nan_high(float x) { return x != x ? __builtin_inff() : x; }

__device__ __forceinline__ uint64_t top_key(float x, int c) {
  uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);        // -0 orders as 0
  b ^= (uint32_t)((int32_t)b >> 31) | 0x80000000u;
  return ((uint64_t)b << 32) | (uint32_t)~c;
}
__device__ __forceinline__ int key_class(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float key_value(uint64_t key) {
  uint32_t b = (uint32_t)(key >> 32);
  b ^= (b >> 31) ? 0x80000000u : 0xffffffffu;
  return __builtin_bit_cast(float, b);
}

// Fewer rows than CUs: 1024 threads each, where the reading is longer than bringing four times as many threads together (us, 256
// and 1024 threads: one bf16 row of 32768 8.5, 10.8, of 65536 11.1, 12.5, of 131072 16.6, 15.8, of 262144 26.5, 22.4; 64 rows of
// 65536 15.6, 15.0, of 131072 21.1, 18.3; 200 rows of 32768 9.6, 12.3, of 65536 16.5, 15.5; 300 rows of 131072 29, 38).  Rows of up
// to TOP_CAP classes take a wave each (20000 rows of 1000: 49, and 73 with 256 threads).
constexpr int TOP_WIDE_K = 65536;
constexpr int64_t TOP_WIDE_ROWS = 256;
template <int BS> constexpr int top_groups() { return BS == 256 ? 8 : BS == 1024 ? 4 : 0; }     // k_top_wide: groups a thread
template <int BS> struct TopShared {
  union {
    uint64_t group[BS];                      // general: the threads' largest keys
    uint32_t thread_max[BS];                 // wide: their values as ordered integers
  };
  union {
    struct { float max[top_groups<BS>() * BS + 1], sum[top_groups<BS>() * BS + 1]; } groups;       // wide, until the list is begun
    struct { uint64_t list[TOP_CAP], left[BS > 64 ? TOP_CAP : 1]; };          // left: what the first k leave of it, by rank
  };
  uint64_t tau, kth;
  double red[BS / 64];
  float max[BS / 64];
  int wave_items[BS / 64], n;
};

// what becomes of the list: its first k are the answer, the others join the rest (`sum`, against `base`)
template <typename T, typename I, bool UNIT, int BS>
__device__ __forceinline__ void top_finish(const T* __restrict__ p, const RowShape& s, int64_t r, int k, float scale, double inv_t,
                                           T* __restrict__ values, I* __restrict__ indices, const RowShape& o,
                                           float* __restrict__ rest, TopShared<BS>& sh, int n, double sum, float base) {
  const int tid = threadIdx.x, K = s.K;
  // Rank the list; what does not make the first k joins the rest, in the order of its ranks: the list's own order is that in
  // which the waves came, and sums that followed it would differ from call to call (one wave comes in one order only).
  const auto to_rest = [&](uint64_t key) {
    // far above `base` where large classes lie side by side and one thread held them all: past what fp32 holds
    sum += exp2_series(((double)key_value(key) - (double)base) * inv_t * 1.4426950408889634);
  };
  for (int i = tid; i < n; i += BS) {
    const uint64_t key = sh.list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.list[j] > key ? 1 : 0;
    if (rank < k) {
      const int64_t at_o = row_offset(o, r) + rank * o.sK;
      const int c = key_class(key);
      values[at_o] = p[(int64_t)c * s.sK];
      indices[at_o] = (I)c;
      if (rank == k - 1) sh.kth = key;
    } else if (BS > 64) {
      sh.left[rank] = key;
    } else {
      to_rest(key);
    }
  }
  if (BS > 64 && rest && n > k) {
    __syncthreads();
    for (int i = k + tid; i < n; i += BS) to_rest(sh.left[i]);
  }
  if (rest) {
    sum = block_sum<BS>(sum, sh.red);
    __syncthreads();
    const int tid = lane_id();
    float ref = base;
    // the rest lies far below `base` or too far above it, or is infinite: take its own largest value as reference
    if (!(sum > 0x1p-60) || !(sum < 0x1p900) || !(ref < __builtin_inff())) {
      const uint64_t kth = sh.kth;
      float m = neg_inf();
      each_class<T, UNIT, BS, 1>(tid, p, s.sK, 0, K, [&](auto& x, int c) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = nan_high(x[i]);
          if (top_key(y, c + i) < kth) m = fmaxf(m, y);
        }
      });
      ref = block_max<BS>(m, sh.max);
      float acc = 0.f;
      each_class<T, UNIT, BS, 1>(tid, p, s.sK, 0, K, [&](auto& x, int c) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = nan_high(x[i]);
          if (top_key(y, c + i) < kth && y > neg_inf()) acc += exp2_f((y - ref) * scale);
        }
      });
      sum = block_sum<BS>((double)acc, sh.red);
    }
    if (tid == 0) {
      const bool unbounded = !(fabsf(ref) < __builtin_inff());       // nothing is left (-inf), or infinities are
      rest[r] = unbounded ? ref : (float)((double)ref * inv_t + log(sum));
    }
  }
}

// One row, any strides and any contents, by one block, in two passes.  Pass 1: each thread's largest key; the k-th largest
// of these BS keys, tau, has at least k keys at or above it, and rarely many more (73 expected for k = 64 of 256 threads).
// Pass 2: keys >= tau go to a list in LDS, everything else into the sum of exponentials; the list is ranked by counting.
template <typename T, typename I, bool UNIT, int BS, int U>
__device__ __forceinline__ void top_row_general(const T* __restrict__ p, const RowShape& s, int64_t r, int k, float scale, double inv_t,
                                T* __restrict__ values, I* __restrict__ indices, const RowShape& o, float* __restrict__ rest,
                                TopShared<BS>& sh) {
  const int tid = lane_id(), K = s.K;
  // pass 1: this thread's largest key (the vector first, then the class within it)
  float best = neg_inf();
  int at = -1;
  each_class<T, UNIT, BS, U>(tid, p, s.sK, 0, K, [&](auto& x, int c) {
    constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = nan_high(x[i]);
    const float m = max_of(x);
    if (m > best || at < 0) { best = m; at = c; }
  });
  uint64_t mine = 0;
  if (at >= 0) {
    int c = at;
    while (nan_high((float)p[(int64_t)c * s.sK]) != best) ++c;       // ends inside the vector that gave `best`
    mine = top_key(best, c);
  }
  sh.group[tid] = mine;
  if (tid == 0) { sh.tau = 0; sh.n = 0; }
  __syncthreads();
  {
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < BS; ++j) above += sh.group[j] > mine ? 1 : 0;
    if (mine != 0 && above == k - 1) sh.tau = mine;       // fewer than k threads hold a class: tau stays 0, all are listed
  }
  __syncthreads();
  uint64_t tau = sh.tau;
  float floor_v, base;
  double sum;
  int n;
  uint64_t below = ~0ull;                                // some key no class reaches
  for (;;) {
    floor_v = tau ? key_value(tau) : neg_inf();
    base = floor_v == neg_inf() ? 0.f : floor_v;
    float acc = 0.f;
    each_class<T, UNIT, BS, U>(tid, p, s.sK, 0, K, [&](auto& x, int c) {
      constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = nan_high(x[i]);
      if (max_of(x) >= floor_v) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint64_t key = top_key(x[i], c + i);
          if (key >= tau) {
            const int at_n = atomicAdd(&sh.n, 1);
            if (at_n < TOP_CAP) sh.list[at_n] = key;
            x[i] = neg_inf();
          }
        }
      }
      float e[N];
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = exp2_f((x[i] - base) * scale);
      acc += sum_of(e);
    });
    __syncthreads();
    n = sh.n;
    sum = (double)acc;
    if (n <= TOP_CAP) break;
    // More keys than the list holds (many large classes dealt to few threads).  Halve the interval [tau, below) until
    // between k and TOP_CAP keys are left: keys differ, so the count takes every value in between.
    __syncthreads();
    for (;;) {
      const uint64_t mid = tau + (below - tau) / 2;
      int cnt = 0;
      each_class<T, UNIT, BS, U>(tid, p, s.sK, 0, K, [&](auto& x, int c) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) cnt += top_key(nan_high(x[i]), c + i) >= mid ? 1 : 0;
      });
      const int total = (int)block_sum<BS>((double)cnt, sh.red);
      if (total < k) below = mid;
      else tau = mid;
      if (total >= k && total <= TOP_CAP) break;
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
  }
  top_finish<T, I, UNIT, BS>(p, s, r, k, scale, inv_t, values, indices, o, rest, sh, n, sum, base);
}

template <typename T, typename I, bool UNIT, int BS>
__global__ void __launch_bounds__(BS)
k_top_rows(const T* __restrict__ z, RowShape s, int k, float scale, double inv_t, T* __restrict__ values,
           I* __restrict__ indices, RowShape o, float* __restrict__ rest) {
  __shared__ TopShared<BS> sh;
  const int64_t r = grid_row();
  if (r < s.N * s.V)
    top_row_general<T, I, UNIT, BS, 4>(z + row_offset(s, r), s, r, k, scale, inv_t, values, indices, o, rest, sh);
}

// Long rows of adjacent classes, read once.  The classes are summed in groups of 8 vectors of one thread, each group's
// maximum and sum of exponentials against it kept in LDS (16 KB a block: eight blocks of 256 threads stay on a CU).  The
// k-th largest of the threads' maxima, found bit by bit by one wave, is a floor under the first k; only the groups that
// reach it (about k of them) are read again, vector by vector over the whole block, and every other group's sum goes
// into the rest as it is.  (Groups and threads add in fp32, the block in fp64; rest is one fp32 number, which the sum's few 2^-24
// move by no more than its own rounding does.)  Rows on which this stalls - most groups reach the floor, because classes are equal or masked -
// go the general way.
constexpr int TOP_GROUP = 8;                  // vectors of a group
constexpr int TOP_ITEMS = 440;                // groups read again (with the rest of the LDS: 1/8 of a CU)

template <typename T, typename I, int BS>
__global__ void __launch_bounds__(BS, BS == 256 ? 8 : 4)
k_top_wide(const T* __restrict__ z, RowShape s, int k, float scale, double inv_t, T* __restrict__ values,
           I* __restrict__ indices, RowShape o, float* __restrict__ rest) {
  constexpr int VEC = vec_of<T>(), GROUPS = top_groups<BS>();
  __shared__ TopShared<BS> sh;
  __shared__ int s_item[TOP_ITEMS];
  const int tid = threadIdx.x, K = s.K;
  const int64_t r = grid_row();
  if (r >= s.N * s.V) return;
  const int full = K / VEC;                                    // whole vectors
  const int groups = (full + TOP_GROUP * BS - 1) / (TOP_GROUP * BS);
  const int each = (groups + GROUPS - 1) / GROUPS;             // longer rows: `each` times as many vectors a group
  const T* p = z + row_offset(s, r);
  float best = neg_inf();
  bool holds = false;
  for (int g = 0; g * each < groups; ++g) {
    float gm = neg_inf(), gs = 0.f;
    for (int h = 0; h < 2 * each; ++h) {
      const int v0 = (g * each * TOP_GROUP + h * 4) * BS + tid;
      Raw16 raw[4];
      float x[4][VEC], m = neg_inf(), e[4];
      if (v0 - tid + 4 * BS <= full) {
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = load16(p + (int64_t)(v0 + u * BS) * VEC);
#pragma unroll
        for (int u = 0; u < 4; ++u) unpack(raw[u], x[u]);
      } else {
        if (v0 >= full) continue;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (v0 + u * BS < full) unpack(load16(p + (int64_t)(v0 + u * BS) * VEC), x[u]);
          else
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[u][i] = neg_inf();
        }
      }
      holds = true;
#pragma unroll
      for (int u = 0; u < 4; ++u) m = fmaxf(m, max_of(x[u]));
      const float ref = m == neg_inf() ? 0.f : m;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[u][i] = exp2_f((x[u][i] - ref) * scale);
        e[u] = sum_of(x[u]);
      }
      const float sum = sum_of(e);
      if (m > gm) { gs *= exp2_f((gm - m) * scale); gm = m; gs += sum; }
      else gs += m == neg_inf() ? sum : sum * exp2_f((m - gm) * scale);
    }
    if (gs != gs) gm = __builtin_inff();                     // a NaN, which orders as +inf, or an infinity
    sh.groups.max[g * BS + tid] = gm;
    sh.groups.sum[g * BS + tid] = gs;
    best = fmaxf(best, gm);
  }
  const int c_tail = full * VEC + tid;
  const bool tail = c_tail < K;
  const float x_tail = tail ? nan_high((float)p[c_tail]) : neg_inf();
  best = fmaxf(best, x_tail);
  sh.thread_max[tid] = holds || tail ? (uint32_t)(top_key(best, 0) >> 32) : 0;
  if (tid == 0) sh.n = 0;
  __syncthreads();
  if (tid < 64) {
    // the largest value that at least k threads reach; a bf16 value is in the upper half of its key
    constexpr int BITS = 8 * sizeof(T);
    uint32_t key[BS / 64], floor_key = 0;
#pragma unroll
    for (int i = 0; i < BS / 64; ++i) key[i] = sh.thread_max[i * 64 + tid] >> (32 - BITS);
    for (int bit = BITS - 1; bit >= 0; --bit) {
      const uint32_t probe = floor_key | (1u << bit);
      int reach = 0;
#pragma unroll
      for (int i = 0; i < BS / 64; ++i) reach += __popcll(__ballot(key[i] >= probe));
      if (reach >= k) floor_key = probe;
    }
    if (tid == 0) {
      uint32_t b = floor_key << (32 - BITS);
      if (BITS == 16 && !(b >> 31) && floor_key) b |= 0xffffu;       // negative values are stored inverted
      sh.tau = (uint64_t)b << 32;
    }
  }
  __syncthreads();
  const uint64_t tau = sh.tau;
  const float floor_v = tau ? key_value(tau) : neg_inf();
  float base = floor_v == neg_inf() ? 0.f : floor_v;
  float acc = 0.f;
  uint32_t hit = 0;                                            // this thread's groups that are read again
  for (int g = 0; g * each < groups; ++g) {
    const float gm = sh.groups.max[g * BS + tid];
    if (gm >= floor_v) hit |= 1u << g;
    else acc += sh.groups.sum[g * BS + tid] * exp2_f((gm - base) * scale);
  }
  // their list in the order of the threads: which thread reads which group, and so every sum, is the same in every call
  int at = 0, in_wave = 0, items = 0;
  for (int g = 0; g * each < groups; ++g) {
    const unsigned long long reach = __ballot((hit >> g) & 1u);
    at += __popcll(reach & ((1ull << (tid & 63)) - 1));
    in_wave += __popcll(reach);
  }
  if ((tid & 63) == 0) sh.wave_items[tid >> 6] = in_wave;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < BS / 64; ++i) {
    at += i < (tid >> 6) ? sh.wave_items[i] : 0;
    items += sh.wave_items[i];
  }
  for (; hit; hit &= hit - 1, ++at) if (at < TOP_ITEMS) s_item[at] = (__ffs(hit) - 1) * BS + tid;
  __syncthreads();
  bool stalled = items > TOP_ITEMS || !tau;
  if (!stalled) {
    const auto take = [&](float x, int c) {
      if (x >= floor_v) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < TOP_CAP) sh.list[at] = top_key(x, c);
      } else {
        acc += exp2_f((x - base) * scale);
      }
    };
    for (int q = tid; q < items * TOP_GROUP; q += BS) {
      const int item = s_item[q / TOP_GROUP], g = item / BS, t = item % BS;
      for (int h = 0; h < each; ++h) {
        const int v = ((g * each + h) * TOP_GROUP + q % TOP_GROUP) * BS + t;
        if (v < full) {
          float x[VEC];
          unpack(load16(p + (int64_t)v * VEC), x);
#pragma unroll
          for (int i = 0; i < VEC; ++i) take(nan_high(x[i]), v * VEC + i);
        }
      }
    }
    if (tail) take(x_tail, c_tail);
    __syncthreads();
    stalled = sh.n > TOP_CAP;
  }
  if (stalled) {
    __syncthreads();
    top_row_general<T, I, true, BS, 1>(p, s, r, k, scale, inv_t, values, indices, o, rest, sh);
  } else {
    top_finish<T, I, true, BS>(p, s, r, k, scale, inv_t, values, indices, o, rest, sh, sh.n, (double)acc, base);
  }
}

// the largest value over T and the logarithm may cancel: in fp64, rounded once
__device__ __forceinline__ float log_rest(float m, double sum, double inv_t) {
  return (float)fma((double)m, inv_t, 0.6931471805599453 * log2_split(sum));
}

// few classes: one thread a row.  Slot by slot the largest value left, the lowest class first (strict comparison).
template <typename T, typename I, int KT, bool FULL>
__global__ void __launch_bounds__(256)
k_top_few(const T* __restrict__ z, RowShape s, int k, float scale, double inv_t, T* __restrict__ values, I* __restrict__ indices,
          RowShape o, float* __restrict__ rest) {
  for (int64_t n = blockIdx.y; n < s.N; n += gridDim.y) {
    for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < s.V; v += (int64_t)gridDim.x * 256) {
      float x[KT];
      load_row<T, KT, FULL>(z + n * s.sN + v * s.sV, s.sK, s.K, x);
      uint32_t key[KT];                      // ordered integer of the value; 0: taken, or no class
#pragma unroll
      for (int c = 0; c < KT; ++c) key[c] = FULL || c < s.K ? (uint32_t)(top_key(nan_high(x[c]), 0) >> 32) : 0;
      const int64_t at = n * o.sN + v * o.sV;
      for (int j = 0; j < k; ++j) {
        uint32_t best = 0;
        int bc = 0;
        float bx = 0.f;
#pragma unroll
        for (int c = 0; c < KT; ++c) {
          const bool more = key[c] > best;
          best = more ? key[c] : best;
          bc = more ? c : bc;
          bx = more ? x[c] : bx;
        }
#pragma unroll
        for (int c = 0; c < KT; ++c) key[c] = c == bc ? 0 : key[c];
        values[at + j * o.sK] = (T)bx;
        indices[at + j * o.sK] = (I)bc;
      }
      if (rest) {
        float m = neg_inf();
#pragma unroll
        for (int c = 0; c < KT; ++c) {
          x[c] = key[c] ? nan_high(x[c]) : neg_inf();
          m = fmaxf(m, x[c]);
        }
        const float ref = fabsf(m) < __builtin_inff() ? m : 0.f;
        float e[KT];
#pragma unroll
        for (int c = 0; c < KT; ++c) e[c] = exp2_f((x[c] - ref) * scale);
        // m is -inf (nothing left) or +inf: it is the answer
        rest[n * s.V + v] = ref == m ? log_rest(m, (double)sum_of(e), inv_t) : m;
      }
    }
  }
}

// A few dozen classes and many rows (rows.h): a thread a row, the KS >= k largest keys so far in registers, in order.  Each
// class that comes leaves one loser, itself or the last of the list, for the rest.
template <typename T, typename I, bool UNIT, int KS>
__global__ void __launch_bounds__(256)
k_top_lane(const T* __restrict__ z, RowShape s, int k, float scale, double inv_t, T* __restrict__ values, I* __restrict__ indices,
           RowShape o, float* __restrict__ rest) {
  const int K = s.K;
  const int64_t NV = s.N * s.V;
  const auto value = [](uint32_t key) { return key ? key_value((uint64_t)key << 32) : neg_inf(); };
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < NV; r += (int64_t)gridDim.x * 256) {
    const T* p = z + row_offset(s, r);
    uint32_t top[KS];                          // ordered integers of the values, 0: none yet
    int at[KS];
#pragma unroll
    for (int j = 0; j < KS; ++j) top[j] = at[j] = 0;
    LaneSum left = {neg_inf(), 0.};
    for (int c0 = 0; c0 < K; c0 += 8) {
      float x[8];
      load8<T, UNIT>(p, s.sK, c0, K, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t key = c0 + i < K ? (uint32_t)(top_key(nan_high(x[i]), 0) >> 32) : 0;
        uint32_t loser = key;
        if (key > top[KS - 1]) {
          loser = top[KS - 1];
#pragma unroll
          for (int j = KS - 1; j > 0; --j) {
            const bool past = key > top[j - 1], here = key > top[j];         // strict: the lower class stays in front
            at[j] = past ? +at[j - 1] : here ? c0 + i : +at[j];
            top[j] = past ? +top[j - 1] : here ? key : +top[j];
          }
          at[0] = key > top[0] ? c0 + i : +at[0];
          top[0] = key > top[0] ? key : +top[0];
        }
        x[i] = value(loser);
      }
      left.add(x, scale);
    }
    const int64_t out = row_offset(o, r);
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      if (j < k) {
        values[out + j * o.sK] = p[(int64_t)at[j] * s.sK];
        indices[out + j * o.sK] = (I)at[j];
      } else if (top[j]) {
        left.add_one(value(top[j]), scale);
      }
    }
    // nothing left (-inf), or infinities are: the maximum is the answer
    if (rest) rest[r] = fabsf(left.m) < __builtin_inff() ? log_rest(left.m, left.s, inv_t) : left.m;
  }
}

}  // namespace devis

using namespace devis;

extern "C" int devis_top_logits(const void* logits, int64_t sN, int64_t sV, int64_t sK, int dtype, int64_t N, int64_t V,
                                int64_t K, int64_t k, float temperature, void* values, void* indices, int index_dtype,
                                int64_t oN, int64_t oV, int64_t oK, float* rest, void* stream) {
  if (!logits || !values || !indices || !rows_ok(sN, sV, sK, N, V, K) || !rows_ok(oN, oV, oK, N, V, K)) return DEVIS_ERR_BAD_ARG;
  if (k < 1 || k > K || k > TOP_MAX_K || !(temperature > 0x1p-100f) || !(temperature < 0x1p100f)) return DEVIS_ERR_BAD_ARG;
  if (index_dtype != DEVIS_LABEL_I32 && !(index_dtype == DEVIS_LABEL_U8 && K <= 256)) return DEVIS_ERR_BAD_ARG;
  RowShape s = {sN, sV, sK, N, V, (int)K}, o = {oN, oV, oK, N, V, (int)k};
  const int64_t NV = N * V;
  const double inv_t = 1.0 / (double)temperature;
  const float scale = (float)(1.4426950408889634 * inv_t);
  const hipStream_t st = (hipStream_t)stream;
  if (K <= FEW_CLASSES && side_by_side(s, o)) {
    if (one_stride(s) && one_stride(o)) { merge_rows(s); merge_rows(o); }
    const dim3 grid = few_grid(s.N, s.V, 8192);
#define LAUNCH_FEW(KT, FULL) hipLaunchKernelGGL((k_top_few<T, I, KT, FULL>), grid, dim3(256), 0, st, (const T*)logits, s, (int)k, scale, inv_t, (T*)values, (I*)indices, o, rest)
    DEVIS_DISPATCH_DTYPE(dtype, {
      if (index_dtype == DEVIS_LABEL_U8) { typedef uint8_t I; DEVIS_DISPATCH_FEW(K, sK == 1, LAUNCH_FEW); }
      else { typedef int32_t I; DEVIS_DISPATCH_FEW(K, sK == 1, LAUNCH_FEW); }
    });
#undef LAUNCH_FEW
    return launch_status();
  }
  if (lane_rows(NV, K, k)) {
    const int64_t tiles = cdiv(NV, 256);
    const dim3 grid((unsigned)(tiles < 8192 ? tiles : 8192));
#define LAUNCH_LANE(UNIT, KS) hipLaunchKernelGGL((k_top_lane<T, I, UNIT, KS>), grid, dim3(256), 0, st, (const T*)logits, s, (int)k, scale, inv_t, (T*)values, (I*)indices, o, rest)
#define LAUNCH_LANE_U(KS) do { if (sK == 1) LAUNCH_LANE(true, KS); else LAUNCH_LANE(false, KS); } while (0)
    DEVIS_DISPATCH_DTYPE(dtype, {
      if (index_dtype == DEVIS_LABEL_U8) { typedef uint8_t I; if (k <= 4) LAUNCH_LANE_U(4); else LAUNCH_LANE_U(16); }
      else { typedef int32_t I; if (k <= 4) LAUNCH_LANE_U(4); else LAUNCH_LANE_U(16); }
    });
#undef LAUNCH_LANE_U
#undef LAUNCH_LANE
    return launch_status();
  }
#define LAUNCH_TOP(I, UNIT, BS) hipLaunchKernelGGL((k_top_rows<T, I, UNIT, BS>), row_grid(NV), dim3(BS), 0, st, (const T*)logits, s, (int)k, scale, inv_t, (T*)values, (I*)indices, o, rest)
#define LAUNCH_TOP_U(I, BS) do { if (sK == 1) LAUNCH_TOP(I, true, BS); else LAUNCH_TOP(I, false, BS); } while (0)
#define LAUNCH_WIDE(I, BS) hipLaunchKernelGGL((k_top_wide<T, I, BS>), row_grid(NV), dim3(BS), 0, st, (const T*)logits, s, (int)k, scale, inv_t, (T*)values, (I*)indices, o, rest)
#define LAUNCH_TOP_B(I)                                                                                           \
  do {                                                                                                            \
    if (K <= TOP_CAP) LAUNCH_TOP_U(I, 64);                                                                        \
    else if (sK != 1) LAUNCH_TOP(I, false, 256);                                                                  \
    else if (K >= TOP_WIDE_K && NV < TOP_WIDE_ROWS) LAUNCH_WIDE(I, 1024);                                         \
    else LAUNCH_WIDE(I, 256);                                                                                     \
  } while (0)
  DEVIS_DISPATCH_DTYPE(dtype, { if (index_dtype == DEVIS_LABEL_U8) LAUNCH_TOP_B(uint8_t); else LAUNCH_TOP_B(int32_t); });
#undef LAUNCH_TOP_B
#undef LAUNCH_WIDE
#undef LAUNCH_TOP_U
#undef LAUNCH_TOP
  return launch_status();
}
