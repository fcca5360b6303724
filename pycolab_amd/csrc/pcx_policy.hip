// pcx_policy.hip -- what a policy's logits become: sampled actions, and the log-probability of actions taken and the
// policy's entropy with the gradient of both with respect to the logits.
//
// Definitions, for one row of logits x over the actions, `allowed` where the action is legal, x is no NaN and x > -inf:
//   w_j = exp((x_j - max x) / T) for the allowed actions (an action that equals the maximum weighs 1, infinite or not).
//   sample: order the allowed actions by (x descending, index ascending).  Keep the first top_k of them; of those, each
//   whose predecessors weigh less than top_p of the kept ones' total; of those, each with w_j >= min_p; the first always.
//   What is kept is a prefix of that order, so it is described by the last kept value and how many of the actions with
//   that very value are kept (the lowest indices).  The action is the first j in index order whose running sum of kept
//   weights exceeds u times their total; T <= 0 takes the first of the order.  No allowed action: PCX_ACTION_NONE.
//   log_prob: with d_j = (x_j - max x) / T and s = sum exp d_j:  log p_a = d_a - log s,
//   H = log s - (sum d_j exp d_j) / s;  d(log p_a) = (1[j = a] - p_j) / T,  dH = -p_j (log p_j + H) / T.
//
// Sampling decides by where one number falls between two sums, so its weights and sums are 64-bit: a float32 sum would
// pick another action once in some million rows.  MI355X multiplies and adds 64-bit floats at the rate of 32-bit ones,
// which puts exp at about 25 instructions.  Sums that atomics build are whole numbers: their order does not matter.
#include "pcx_internal.h"

#include <cmath>

using pcx::set_error;

namespace {

constexpr int NONE = PCX_ACTION_NONE;

template <int DT> struct Logit;
template <> struct Logit<PCX_F32> {
  typedef float T;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Logit<PCX_F16> {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};
template <> struct Logit<PCX_BF16> {
  typedef __bf16 T;
  static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};

struct Rows {
  int64_t n, row_stride, legal_stride;
  int32_t actions;
  const void* logits;
  const uint8_t* legal;  // or null
};

template <typename T, int N> struct Pack { T v[N]; };

// A logit as an unsigned number of the same order, with the bits its type has (a 16-bit search takes half the steps of a
// 32-bit one); 0 stands for "not allowed".  (+0 and -0 are one value.)
template <int DT> constexpr int KEY_SHIFT = DT == PCX_BF16 ? 16 : DT == PCX_F16 ? 13 : 0;
template <int DT>
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u)) >> KEY_SHIFT<DT>;
}
template <int DT>
__device__ __forceinline__ float value_of(uint32_t key) {
  const uint32_t k = key << KEY_SHIFT<DT>;
  return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~(k | ((1u << KEY_SHIFT<DT>) - 1u)));
}
__device__ __forceinline__ bool allowed(float x, bool legal) { return legal && x > -INFINITY; }  // (a NaN compares false)

// N neighbouring logits of a row from j on, -infinity where they are not allowed or not there (j may lie behind the end).
template <int DT, int N>
__device__ __forceinline__ void load_logits(const typename Logit<DT>::T* x_row, const uint8_t* l_row, int j, int end, float* x) {
  typedef typename Logit<DT>::T T;
  constexpr int W = N % (16 / (int)sizeof(T)) == 0 ? 16 / (int)sizeof(T) : N % 4 == 0 ? 4 : 2 - N % 2;  // elements per load
#pragma unroll
  for (int i = 0; i < N; i += W) {
    Pack<T, W> q = {};
    Pack<uint8_t, W> ok;
#pragma unroll
    for (int c = 0; c < W; ++c) ok.v[c] = 1;
    if (j + i + W <= end) {
      __builtin_memcpy(&q, x_row + j + i, sizeof q);
      if (l_row) __builtin_memcpy(&ok, l_row + j + i, sizeof ok);
    } else {
#pragma unroll
      for (int c = 0; c < W; ++c) {
        ok.v[c] = 0;
        if (j + i + c < end) {
          q.v[c] = x_row[j + i + c];
          ok.v[c] = l_row ? l_row[j + i + c] : 1;
        }
      }
    }
#pragma unroll
    for (int c = 0; c < W; ++c) {
      const float v = Logit<DT>::get(q.v[c]);
      x[i + c] = allowed(v, ok.v[c] != 0) ? v : -INFINITY;
    }
  }
}
template <int DT, int N>
__device__ __forceinline__ void load_keys(const Rows& rows, int64_t row, int j, int end, uint32_t* key) {
  float x[N];
  load_logits<DT, N>(reinterpret_cast<const typename Logit<DT>::T*>(rows.logits) + row * rows.row_stride,
                     rows.legal ? rows.legal + row * rows.legal_stride : nullptr, j, end, x);
#pragma unroll
  for (int i = 0; i < N; ++i) key[i] = x[i] > -INFINITY ? order_of<DT>(x[i]) : 0u;
}

// exp(d) for d <= 0 in 64 bits, to about a unit in the last place: d = n ln 2 + r with ln 2 in two parts, the upper one short
// enough that n times it is exact (the reduction of Cody and Waite), the Taylor series
// of exp(r), |r| <= ln(2) / 2, to r^13 / 13! (the next term is 4e-18), and n in the exponent.
// Four at a time: a chain of twenty dependent instructions leaves the unit idle, four side by side do not (8 x 2^20
// logits without rules: 41 -> 36 us, all launches included); and the coefficients are held in scalar registers, which the
// four share -- left to itself the compiler copies each into vector registers for every element.
__device__ __forceinline__ double scalar(double c) { asm("" : "+s"(c)); return c; }
template <int N>
__device__ __forceinline__ void exp64(double* d) {
  double n[N], p[N];
#pragma unroll
  for (int i = 0; i < N; ++i) d[i] = fmax(d[i], -800.0);
  const double log2e = scalar(1.4426950408889634), ln2_hi = scalar(-0.6931471803691238), ln2_lo = scalar(-1.9082149292705877e-10);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    n[i] = rint(d[i] * log2e);
    d[i] = fma(n[i], ln2_hi, d[i]);
    d[i] = fma(n[i], ln2_lo, d[i]);
    p[i] = 1.0 / 6227020800.0;
  }
  constexpr double C[13] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                            1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
  for (int k = 0; k < 13; ++k) {
    const double c = scalar(C[k]);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = fma(p[i], d[i], c);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) d[i] = ldexp(p[i], (int)n[i]);
}
// exp((x - best) * rate); 0 for -infinity, 1 where x is the best, infinite or not.
template <int N>
__device__ __forceinline__ void weights(const float* x, float best, double rate, double* w) {
  constexpr int AT_ONCE = N % 4 == 0 ? 4 : N % 3 == 0 ? 3 : N % 2 == 0 ? 2 : 1;
#pragma unroll
  for (int i = 0; i < N; i += AT_ONCE) {
    double d[AT_ONCE];
#pragma unroll
    for (int c = 0; c < AT_ONCE; ++c) {
      const double v = ((double)x[i + c] - (double)best) * rate;
      d[c] = x[i + c] == best ? 0.0 : v;
    }
    exp64<AT_ONCE>(d);
#pragma unroll
    for (int c = 0; c < AT_ONCE; ++c) w[i + c] = d[c];
  }
}
__device__ __forceinline__ double weight_of(float x, float best, double rate) {
  double w;
  weights<1>(&x, best, rate, &w);
  return w;
}

// ---------------------------------------------------------------- reductions over a group of THREADS (one wave, or a workgroup)

// v from the lane that a data-parallel primitive names, 0 where it names none.
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V moved(V v) {
  if constexpr (sizeof(V) == 8) {
    uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, true);
    return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
  } else {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, true));
  }
}
template <typename V>
__device__ __forceinline__ V from_lane(V v, int lane) {
  if constexpr (sizeof(V) == 8) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
  } else {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  }
}
// Prefix within a wave: each lane with those below it (f's neutral element is 0): steps of 1, 2, 4, 8 within rows of 16
// lanes, then row to row.
template <typename V, typename F>
__device__ __forceinline__ V wave_prefix(V v, F f) {
  v = f(v, moved<0x111, 0xF>(v));
  v = f(v, moved<0x112, 0xF>(v));
  v = f(v, moved<0x114, 0xF>(v));
  v = f(v, moved<0x118, 0xF>(v));
  v = f(v, moved<0x142, 0xA>(v));  // the last lane of rows 0 and 2 to rows 1 and 3
  v = f(v, moved<0x143, 0xC>(v));  // lane 31 to the upper half
  return v;
}

template <int THREADS>
struct Group {
  static constexpr int WAVES = THREADS / 64;
  struct Scratch { uint64_t slot[2][WAVES]; };
  Scratch* s;
  int t;      // thread within the group
  int phase;  // which half of the slots the next exchange uses: its readers are through before that half is written again
  // one number per wave (the same in all its lanes), joined in the waves' order
  template <typename V, typename F>
  __device__ __forceinline__ V join(V v, F f) {
    if constexpr (WAVES == 1) return v;
    V* const slot = reinterpret_cast<V*>(s->slot[phase]);
    phase ^= 1;
    if ((t & 63) == 0) slot[t >> 6] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) v = f(v, slot[i]);
    return v;
  }
  __device__ __forceinline__ double sum(double v) {
    auto add = [](double a, double b) { return a + b; };
    return join(from_lane(wave_prefix(v, add), 63), add);
  }
  __device__ __forceinline__ float sum(float v) {
    auto add = [](float a, float b) { return a + b; };
    return join(from_lane(wave_prefix(v, add), 63), add);
  }
  __device__ __forceinline__ uint32_t max(uint32_t v) {
    auto most = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    return join(from_lane(wave_prefix(v, most), 63), most);
  }
  __device__ __forceinline__ uint32_t min(uint32_t v) { return ~max(~v); }
  // `mine` counted per wave already (of ballots)
  __device__ __forceinline__ uint32_t count(uint32_t mine) {
    return join(mine, [](uint32_t a, uint32_t b) { return a + b; });
  }
  // the sum of the threads before this one, and of all
  template <typename V>
  __device__ __forceinline__ V scan(V v, V* total) {
    auto add = [](V a, V b) { return a + b; };
    const V in = wave_prefix(v, add);
    V before = moved<0x138, 0xF>(in);  // one lane up across the whole wave
    V all = from_lane(in, 63);
    if constexpr (WAVES > 1) {
      V* const slot = reinterpret_cast<V*>(s->slot[phase]);
      phase ^= 1;
      if ((t & 63) == 63) slot[t >> 6] = in;
      __syncthreads();
      all = V(0);
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        if (i == (t >> 6)) before = all + before;
        all += slot[i];
      }
    }
    *total = all;
    return before;
  }
};
__device__ __forceinline__ uint32_t ballots(bool b) { return (uint32_t)__popcll(__ballot(b)); }

// ---------------------------------------------------------------- sampling

struct Rules {
  float temperature, top_p, min_p;
  int32_t top_k;
  const float* temperature_row;
  const int32_t* top_k_row;
  const float* top_p_row;
  const float* min_p_row;
};
struct RowRules { float temperature, top_p, min_p; int32_t top_k; };
__device__ __forceinline__ RowRules rules_of(const Rules& r, int64_t row) {
  RowRules o;
  o.temperature = r.temperature_row ? r.temperature_row[row] : r.temperature;
  o.top_k = r.top_k_row ? r.top_k_row[row] : r.top_k;
  o.top_p = r.top_p_row ? r.top_p_row[row] : r.top_p;
  const float m = r.min_p_row ? r.min_p_row[row] : r.min_p;
  o.min_p = m < 1.0f ? m : (m >= 1.0f ? 1.0f : 0.0f);  // (a NaN asks for nothing)
  return o;
}

struct SampleArgs {
  Rows rows;
  Rules rules;
  const float* uniforms;
  int32_t* out;
};

// The weights of N keys (0: none).
template <int DT, int N>
__device__ __forceinline__ void key_weights(const uint32_t* key, float best, double rate, double* w) {
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = key[i] ? value_of<DT>(key[i]) : -INFINITY;
  weights<N>(x, best, rate, w);
}

// A thread holds a whole row: few actions, many rows.  Bound by the 64-bit exponentials of CAP actions, those that do not exist
// too: 2^20 rows of 5 float32 logits and legal flags 13.5 us with CAP = 6, 2.5 TB/s, 15.4 with 8.
template <int DT, int CAP>
__global__ __launch_bounds__(256) void pcx_sample_rows(SampleArgs a) {
  typedef typename Logit<DT>::T T;
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows.n) return;
  const T* const x_row = reinterpret_cast<const T*>(a.rows.logits) + row * a.rows.row_stride;
  const uint8_t* const l_row = a.rows.legal ? a.rows.legal + row * a.rows.legal_stride : nullptr;
  const RowRules r = rules_of(a.rules, row);
  const int A = a.rows.actions;
  float x[CAP];
  load_logits<DT, CAP>(x_row, l_row, 0, A, x);
  float best = -INFINITY;
  int first = NONE;
#pragma unroll
  for (int j = 0; j < CAP; ++j)
    if (x[j] > best) { best = x[j]; first = j; }
  if (first == NONE || !(r.temperature > 0.0f)) { a.out[row] = first; return; }
  const double rate = 1.0 / (double)r.temperature;
  double w[CAP];
  weights<CAP>(x, best, rate, w);
  if (r.top_k > 0 && r.top_k < A) {
#pragma unroll
    for (int j = 0; j < CAP; ++j) {
      int rank = 0;
#pragma unroll
      for (int i = 0; i < CAP; ++i) rank += i < j ? x[i] >= x[j] : x[i] > x[j];
      if (rank >= r.top_k) w[j] = -w[j];  // (dropped: its sign, while the others are still being ranked)
    }
#pragma unroll
    for (int j = 0; j < CAP; ++j)
      if (!(w[j] > 0.0)) w[j] = 0.0;
  }
  if (r.top_p < 1.0f) {
    double total = 0.0;
#pragma unroll
    for (int j = 0; j < CAP; ++j) total += w[j];
    const double target = (double)r.top_p * total;
    uint32_t keep = 0;
#pragma unroll
    for (int j = 0; j < CAP; ++j) {
      double ahead = 0.0;
#pragma unroll
      for (int i = 0; i < CAP; ++i) ahead += (i < j ? x[i] >= x[j] : x[i] > x[j]) ? w[i] : 0.0;
      if (j == first || ahead < target) keep |= 1u << j;
    }
#pragma unroll
    for (int j = 0; j < CAP; ++j)
      if (!((keep >> j) & 1u)) w[j] = 0.0;
  }
  double total = 0.0;
#pragma unroll
  for (int j = 0; j < CAP; ++j) {
    if (w[j] < (double)r.min_p) w[j] = 0.0;
    total += w[j];
  }
  const double target = (double)a.uniforms[row] * total;
  double run = 0.0;
  int pick = NONE, last = NONE;
#pragma unroll
  for (int j = 0; j < CAP; ++j) {
    run += w[j];
    if (w[j] > 0.0) last = j;
    if (pick == NONE && w[j] > 0.0 && run > target) pick = j;
  }
  a.out[row] = pick == NONE ? last : pick;
}

// Of the elements whose key is `value`, those from the `keep`-th on (in index order) are let go.
template <int THREADS, int EP>
__device__ __forceinline__ void drop_ties(Group<THREADS>& g, uint32_t value, uint32_t keep, uint32_t* key, double* w) {
  uint32_t mine = 0, total;
#pragma unroll
  for (int i = 0; i < EP; ++i) mine += key[i] == value;
  uint32_t at = g.scan(mine, &total);
  if (total <= keep) return;
#pragma unroll
  for (int i = 0; i < EP; ++i)
    if (key[i] == value && at++ >= keep) { key[i] = 0; w[i] = 0.0; }
}

// Where among the group's elements (EP neighbouring ones a thread) the running sum of weights passes the target: `part` of
// their total, or absolutely with what lies before them.
template <int THREADS, int EP>
__device__ __forceinline__ int draw_action(Group<THREADS>& g, const double* w, double part, double offset, bool absolute) {
  double mine = 0.0, total;
#pragma unroll
  for (int i = 0; i < EP; ++i) mine += w[i];
  const double before = g.scan(mine, &total);
  const double target = absolute ? part : part * total;
  uint32_t pick = 0xFFFFFFFFu, last = 0;
  double run = offset + before;
#pragma unroll
  for (int i = 0; i < EP; ++i) {
    run += w[i];
    if (w[i] > 0.0) {
      last = (uint32_t)(g.t * EP + i) + 1;
      if (run > target && pick == 0xFFFFFFFFu) pick = (uint32_t)(g.t * EP + i);
    }
  }
  pick = g.min(pick);
  if (pick != 0xFFFFFFFFu) return (int)pick;
  return (int)g.max(last) - 1;  // (u is one or more, or no number: the last one kept)
}

// The largest key t in [lo, hi] with at least k keys >= t; k keys or more are >= lo.
template <int THREADS, int EP>
__device__ __forceinline__ uint32_t find_rank(Group<THREADS>& g, const uint32_t* key, uint32_t k, uint32_t lo, uint32_t hi) {
  while (lo < hi) {
    const uint32_t mid = hi - (hi - lo) / 2;
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < EP; ++i) c += ballots(key[i] >= mid);
    if (g.count(c) >= k) lo = mid; else hi = mid - 1;
  }
  return lo;
}
// The largest key t whose elements >= t weigh at least `target`, and what those above it weigh.
template <int THREADS, int EP>
__device__ __forceinline__ uint32_t find_mass(Group<THREADS>& g, const uint32_t* key, const double* w, double target, uint32_t lo, uint32_t hi, double* above) {
  double over = 0.0;
  while (lo < hi) {
    const uint32_t mid = hi - (hi - lo) / 2;
    double m = 0.0;
#pragma unroll
    for (int i = 0; i < EP; ++i) m += key[i] >= mid ? w[i] : 0.0;
    m = g.sum(m);
    if (m >= target) lo = mid;
    else { hi = mid - 1; over = m; }
  }
  *above = over;
  return lo;
}

// The rules on a group's elements, EP neighbouring ones a thread in index order, of which best_key is the largest key (not
// 0) and `low` no more than the smallest but 0; `of` says how many actions the row has.  Which element is drawn.
template <int DT, int THREADS, int EP>
__device__ __forceinline__ int choose(Group<THREADS>& g, uint32_t* key, uint32_t low, uint32_t best_key, const RowRules& r, int of, double u) {
  if (r.top_k > 0 && r.top_k < of) {
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < EP; ++i) c += ballots(key[i] != 0);
    if (g.count(c) > (uint32_t)r.top_k) {
      const uint32_t edge = find_rank<THREADS, EP>(g, key, (uint32_t)r.top_k, low, best_key);
      low = edge;
      uint32_t above = 0, equal = 0;
#pragma unroll
      for (int i = 0; i < EP; ++i) {
        above += ballots(key[i] > edge);
        equal += key[i] == edge;
        if (key[i] < edge) key[i] = 0;
      }
      const uint32_t keep = (uint32_t)r.top_k - g.count(above);
      uint32_t total;
      uint32_t at = g.scan(equal, &total);
      if (total > keep) {
#pragma unroll
        for (int i = 0; i < EP; ++i)
          if (key[i] == edge && at++ >= keep) key[i] = 0;
      }
    }
  }
  const float best = value_of<DT>(best_key);
  const double rate = 1.0 / (double)r.temperature;
  double w[EP];
  key_weights<DT, EP>(key, best, rate, w);
  if (r.top_p < 1.0f) {
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < EP; ++i) total += w[i];
    total = g.sum(total);
    const double target = (double)r.top_p * total;
    // What lies below the edge weighs at most (1 - top_p) of the total: an action of that much / (2 * all) cannot be the edge.
    uint32_t lo = low;
    const float floor_x = best + (float)(log((total - target) / (2.0 * of)) * (double)r.temperature);
    if (floor_x > -3e38f && floor_x < best) {
      const uint32_t floor_key = order_of<DT>(floor_x);
      lo = floor_key > low ? floor_key : low;
    }
    double above;
    const uint32_t edge = find_mass<THREADS, EP>(g, key, w, target, lo, best_key, &above);
#pragma unroll
    for (int i = 0; i < EP; ++i)
      if (key[i] < edge) { key[i] = 0; w[i] = 0.0; }
    const double need = ceil((target - above) / weight_of(value_of<DT>(edge), best, rate));
    drop_ties<THREADS, EP>(g, edge, need >= 1.0 ? (need < 4e9 ? (uint32_t)need : 0xFFFFFFFFu) : 1u, key, w);
  }
#pragma unroll
  for (int i = 0; i < EP; ++i)
    if (w[i] < (double)r.min_p) w[i] = 0.0;
  return draw_action<THREADS, EP>(g, w, u, 0.0, false);
}

// A wave or a workgroup holds a row in registers, EP neighbouring actions a thread.  Where top_k keeps few of a workgroup's
// row, it first cuts at the k-th largest of the threads' largest keys -- at least k elements reach that, and seldom many
// more -- and one wave chooses among those alone: no 64-bit exponentials and no workgroup-wide searches for the rest.
// Bound by the chain of one row's steps, at five rows a CU: 4,096 rows of 4,096 bfloat16 logits with every rule 25 us, 1.3
// TB/s of the 5.2 that a copy reaches (146 without the cut; 36 with a barrier in every step of the search for it, 30 with the
// searches from the lowest key there is and not from the lowest that can be meant).
template <int DT, int THREADS, int EP>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS, EP <= 8 ? 5 : EP == 16 ? 4 : 2) void pcx_sample_group(SampleArgs a) {
  constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1;
  constexpr int FEW = 512;  // elements a wave chooses among
  __shared__ typename Group<THREADS>::Scratch scratch[ROWS];
  Group<THREADS> g{&scratch[threadIdx.x / THREADS], (int)(threadIdx.x % THREADS), 0};
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
  if (row >= a.rows.n) return;  // (a whole group)
  const RowRules r = rules_of(a.rules, row);
  const int A = a.rows.actions, j0 = g.t * EP;
  uint32_t key[EP];
  load_keys<DT, EP>(a.rows, row, j0, A, key);
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < EP; ++i) most = key[i] > most ? key[i] : most;
  // A workgroup's waves each look at all threads' largest keys, by themselves: one barrier, not one a step of the search.
  constexpr int TOPS = THREADS < 256 ? 1 : THREADS / 64;
  uint32_t tops[TOPS] = {most}, best_key;
  Group<64> one{nullptr, (int)(threadIdx.x & 63), 0};
  if constexpr (THREADS >= 256) {
    __shared__ uint32_t all_tops[THREADS];
    all_tops[threadIdx.x] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TOPS; ++i) {
      tops[i] = all_tops[i * 64 + one.t];
      most = tops[i] > most ? tops[i] : most;
    }
    best_key = one.max(most);
  } else {
    best_key = g.max(most);
  }
  if (best_key == 0 || !(r.temperature > 0.0f)) {
    uint32_t first = 0xFFFFFFFFu;
#pragma unroll
    for (int i = EP - 1; i >= 0; --i)
      if (key[i] == best_key) first = (uint32_t)(j0 + i);
    first = g.min(first);
    if (g.t == 0) a.out[row] = best_key ? (int)first : NONE;
    return;
  }
  const double u = (double)a.uniforms[row];
  if constexpr (THREADS >= 256) {
    __shared__ uint32_t few_key[FEW];
    __shared__ uint16_t few_at[FEW];
    if (r.top_k > 0 && r.top_k <= THREADS / 2 && r.top_k < A) {
      uint32_t least = tops[0];
#pragma unroll
      for (int i = 1; i < TOPS; ++i) least = tops[i] < least ? tops[i] : least;
      least = one.min(least);
      const uint32_t cut = find_rank<64, TOPS>(one, tops, (uint32_t)r.top_k, least ? least : 1u, best_key);
      uint32_t c = 0, total;
#pragma unroll
      for (int i = 0; i < EP; ++i) c += key[i] >= cut;
      uint32_t at = g.scan(c, &total);
      if (total <= FEW) {
#pragma unroll
        for (int i = 0; i < EP; ++i)
          if (key[i] >= cut) {
            few_key[at] = key[i];
            few_at[at++] = (uint16_t)(j0 + i);
          }
        __syncthreads();
        if (g.t >= 64) return;
        int pick;
        if (total <= 128) {
          uint32_t k[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) k[i] = (uint32_t)(g.t * 2 + i) < total ? few_key[g.t * 2 + i] : 0;
          pick = choose<DT, 64, 2>(one, k, cut, best_key, r, A, u);
        } else {
          uint32_t k[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) k[i] = (uint32_t)(g.t * 8 + i) < total ? few_key[g.t * 8 + i] : 0;
          pick = choose<DT, 64, 8>(one, k, cut, best_key, r, A, u);
        }
        if (g.t == 0) a.out[row] = few_at[pick];
        return;
      }
    }
  }
  const int pick = choose<DT, THREADS, EP>(g, key, 1u, best_key, r, A, u);
  if (g.t == 0) a.out[row] = pick;
}

// ---- rows that no workgroup holds, of which top_k keeps few (or the temperature only the best) --------------------------
//
// A workgroup reads its row twice: once for every thread's largest key, whose k-th largest is the cut, once for the elements
// that reach it, which go to one wave as in pcx_sample_group.  Where more than FEW do -- many equal logits -- the k-th largest
// key of the row is searched for with a pass a step, and exactly the k elements that the rule keeps are taken.
// Bound by the passes' loads, 16 neighbouring logits a thread in flight (32: 26 -> 30 us): 269 rows of 33,380 float16 logits with
// top_k 40 and top_p take 26 us where the divided rows' launches below take 136, one row of 131,072 float32 ones 44 (65), of
// 262,144 82 (65), 64 rows of those 94 (156); with top_k 256 ten more; the best alone
// of 262,144 36, where divided rows of 300,000 take 16.  So the limit weighs 20 us of a few long rows against 60 of
// many: how many there are cannot decide, since the two ways round their sums in different places and a row's answer must
// not depend on the others.
constexpr int TOP_THREADS = 512, TOP_EP = 16;
// Is this such a row?  By the row's own rules, however they were given, so that a row's answer does not depend on the others.
__host__ __device__ __forceinline__ bool keeps_few(float temperature, int32_t top_k) {
  return !(temperature > 0.0f) || (top_k > 0 && top_k <= TOP_THREADS / 2);
}
template <int DT>
__global__ __launch_bounds__(TOP_THREADS, 4) void pcx_sample_top(SampleArgs a) {
  constexpr int FEW = 512, WAVES = TOP_THREADS / 64, TURN = TOP_THREADS * TOP_EP;
  __shared__ Group<TOP_THREADS>::Scratch scratch;
  __shared__ uint32_t all_tops[TOP_THREADS], few_key[FEW], few_at[FEW], sorted_key[FEW], sorted_at[FEW], found;
  Group<TOP_THREADS> g{&scratch, (int)threadIdx.x, 0};
  Group<64> one{nullptr, (int)(threadIdx.x & 63), 0};
  const int64_t row = blockIdx.x;
  const RowRules r = rules_of(a.rules, row);
  if (!keeps_few(r.temperature, r.top_k)) return;
  const int A = a.rows.actions;
  uint32_t key[TOP_EP];
  // key[] of every turn of neighbouring elements, in index order
  auto each = [&](auto f) {
#pragma unroll 1
    for (int64_t lo = 0; lo < A; lo += TURN) {
      const int j = (int)lo + g.t * TOP_EP;  // (A is at most 2^24)
      load_keys<DT, TOP_EP>(a.rows, row, j, A, key);
      f(j);
    }
  };
  uint32_t most = 0, first = 0;
  each([&](int j) {
#pragma unroll
    for (int i = 0; i < TOP_EP; ++i)
      if (key[i] > most) { most = key[i]; first = (uint32_t)(j + i); }
  });
  all_tops[g.t] = most;
  if (g.t == 0) found = 0;
  __syncthreads();
  uint32_t tops[WAVES], best_key = 0, least = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    tops[i] = all_tops[i * 64 + one.t];
    best_key = tops[i] > best_key ? tops[i] : best_key;
    least = tops[i] < least ? tops[i] : least;
  }
  best_key = one.max(best_key);
  if (best_key == 0 || !(r.temperature > 0.0f)) {
    first = g.min(most == best_key ? first : 0xFFFFFFFFu);
    if (g.t == 0) a.out[row] = best_key ? (int)first : NONE;
    return;
  }
  least = one.min(least);
  const uint32_t k = (uint32_t)r.top_k;
  uint32_t cut = find_rank<64, WAVES>(one, tops, k, least ? least : 1u, best_key);
  auto take = [&](bool yes, uint32_t what, uint32_t where) {
    if (!yes) return;
    const uint32_t at = atomicAdd(&found, 1u);
    if (at < FEW) { few_key[at] = what; few_at[at] = where; }
  };
  each([&](int j) {
#pragma unroll
    for (int i = 0; i < TOP_EP; ++i) take(key[i] >= cut, key[i], (uint32_t)(j + i));
  });
  __syncthreads();
  uint32_t total = found;
  if (total > FEW) {
    uint32_t lo = cut, hi = best_key;
    while (lo < hi) {
      const uint32_t mid = hi - (hi - lo) / 2;
      uint32_t c = 0;
      each([&](int) {
#pragma unroll
        for (int i = 0; i < TOP_EP; ++i) c += ballots(key[i] >= mid);
      });
      if (g.count(c) >= k) lo = mid; else hi = mid - 1;
    }
    uint32_t above = 0;
    each([&](int) {
#pragma unroll
      for (int i = 0; i < TOP_EP; ++i) above += ballots(key[i] > lo);
    });
    uint32_t ties = k - g.count(above);  // how many of the row's elements with that very key are still kept, the first ones
    if (g.t == 0) found = 0;
    __syncthreads();
    each([&](int j) {
      uint32_t equal = 0, all;
#pragma unroll
      for (int i = 0; i < TOP_EP; ++i) equal += key[i] == lo;
      uint32_t before = g.scan(equal, &all);
#pragma unroll
      for (int i = 0; i < TOP_EP; ++i) take(key[i] > lo || (key[i] == lo && before++ < ties), key[i], (uint32_t)(j + i));
      ties = all < ties ? ties - all : 0u;
    });
    cut = lo;
    __syncthreads();
    total = found;
  }
  // in index order: an element's place is how many have a lower index
  if ((uint32_t)g.t < total) {
    const uint32_t at = few_at[g.t];
    uint32_t place = 0;
    for (uint32_t i = 0; i < total; ++i) place += few_at[i] < at;
    sorted_key[place] = few_key[g.t];
    sorted_at[place] = at;
  }
  __syncthreads();
  if (g.t >= 64) return;
  const double u = (double)a.uniforms[row];
  int pick;
  if (total <= 128) {
    uint32_t some[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) some[i] = (uint32_t)(g.t * 2 + i) < total ? sorted_key[g.t * 2 + i] : 0;
    pick = choose<DT, 64, 2>(one, some, cut, best_key, r, A, u);
  } else {
    uint32_t some[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) some[i] = (uint32_t)(g.t * 8 + i) < total ? sorted_key[g.t * 8 + i] : 0;
    pick = choose<DT, 64, 8>(one, some, cut, best_key, r, A, u);
  }
  if (g.t == 0) a.out[row] = (int)sorted_at[pick];
}

// ---- rows that no workgroup holds: divided among workgroups, one launch per question ------------------------------------
//
// The best logit; the edges of top_k and of top_p, a digit of the order key at a time; what each slice keeps; the slice and
// the action that the number falls to.  8 x 2^20 float32 logits with top_p take 101 us in ten launches, of which one pass
// over them, the floor, is 6.5: four more passes read them again (from the 256 MB cache: 7 us each if that were all), and the
// chain of launches alone is 65 us, the time of a single row.

constexpr int SLICE = 8192;    // actions per workgroup
constexpr int WEP = 32;        // ... per thread of 256, all of them in flight before the first is looked at
constexpr int BINS = 2048;     // of a digit of the order key: at most 11 bits
struct RowState {
  uint64_t best;               // (order key, ~index) of the best action
  double total, target, above; // weights: of what top_k leaves, top_p of it, ahead of the current digit's bin
  uint64_t count_above;        // actions ahead of the current digit's bin
  uint32_t prefix;             // the digits found so far
  uint32_t edge, ties;         // kept: keys above `edge`, and `ties` (lowest indices) that equal it
  uint32_t active;             // bit 0: the row samples; 1: top_k cuts; 2: top_p cuts
};
struct Slot { double weight; uint64_t ties; };

// Sums that atomics build are sums of whole numbers, so that their order does not matter; a word has 64 bits, and a tail of
// many small weights must not vanish beside a large one.  So there are two words a bin: in LDS, of a slice's 2^13 weights, those
// from 2^-12 of the best one's on in units of 2^-50, the smaller ones of 2^-62 (off by 2^-39 of themselves, and by 2^-39 of the
// total, which is at least 1, if they are 2^24); in memory, a slice's bin below 2^-9 in units of 2^-62, exactly, and one from
// there on in units of 2^-(63 - log2 A), off by A 2^-55 of itself.  A 64-bit float's sum of A numbers is known to A 2^-53.
constexpr double SMALL = 1.0 / 4096.0;
constexpr uint64_t LOW = 1ull << 53;  // (2^11 slices of less)
// large 2^12 + small, in units of 2^-62: a word for memory, and which
__device__ __forceinline__ uint64_t slice_sum(uint64_t large, uint64_t small, int scale, bool* is_low) {
  *is_low = large < (LOW >> 12) && (large << 12) + small < LOW;  // (small is at most 2^63)
  if (*is_low) return (large << 12) + small;
  return (uint64_t)(ldexp((double)large, scale - 50) + ldexp((double)small, scale - 62) + 0.5);
}
__device__ __forceinline__ double weight_of(uint64_t high, uint64_t low, int scale) { return ldexp((double)high, -scale) + ldexp((double)low, -62); }
struct WideArgs {
  SampleArgs a;
  int64_t row0;                // first row of this batch of launches
  int32_t slices, scale;       // high words' unit: 2^-scale
  RowState* state;             // [rows]
  uint64_t* high;              // [2][rows][BINS]: the first digit's, the later digits'
  uint64_t* low;
  uint32_t* count;
  Slot* slots;                 // [rows][slices]
  int32_t batch;
  int32_t others;              // rows that keep few are pcx_sample_top's
};
// The digits of a key, from the top: 11, 11 and 10 bits of 32; 11 and 5 of bfloat16's 16, 11 and 8 of float16's 19.
template <int DT> constexpr int LEVELS = DT == PCX_F32 ? 3 : 2;
template <int DT>
__host__ __device__ __forceinline__ int digit_shift(int level) {
  constexpr int BITS = 32 - KEY_SHIFT<DT>;
  return level == 0 ? BITS - 11 : level == 1 && BITS > 22 ? BITS - 22 : 0;
}
template <int DT>
__device__ __forceinline__ uint32_t digit_of(uint32_t key, int level) {
  const uint32_t bits = level == 0 ? 11u : (uint32_t)(digit_shift<DT>(level - 1) - digit_shift<DT>(level));
  return (key >> digit_shift<DT>(level)) & ((1u << bits) - 1u);
}
template <int DT>
__device__ __forceinline__ bool same_prefix(uint32_t key, uint32_t prefix, int level) {
  return level == 0 || key >> digit_shift<DT>(level - 1) == prefix >> digit_shift<DT>(level - 1);
}

__global__ __launch_bounds__(256) void pcx_sample_clear(WideArgs w) {
  const int row = blockIdx.x;
  for (int i = threadIdx.x; i < 2 * BINS; i += 256) {
    const int64_t at = ((int64_t)(i / BINS) * w.batch + row) * BINS + i % BINS;
    w.high[at] = w.low[at] = 0;
    w.count[at] = 0;
  }
  if (threadIdx.x == 0) w.state[row] = RowState{};
}
// The keys of this thread in a slice: SLICE / 256, in packs that lie 256 packs apart.
template <int DT>
__device__ __forceinline__ void load_slice(const WideArgs& w, int row, int lo, uint32_t* key) {
  constexpr int W = 16 / (int)sizeof(typename Logit<DT>::T);
  const int end = w.a.rows.actions - lo < SLICE ? w.a.rows.actions : lo + SLICE;
#pragma unroll
  for (int i = 0; i < WEP / W; ++i) load_keys<DT, W>(w.a.rows, w.row0 + row, lo + (i * 256 + (int)threadIdx.x) * W, end, key + i * W);
}
template <int DT>
__device__ __forceinline__ int slice_index(int lo, int i) {
  constexpr int W = 16 / (int)sizeof(typename Logit<DT>::T);
  return lo + ((i / W) * 256 + (int)threadIdx.x) * W + i % W;
}
template <int DT>
__global__ __launch_bounds__(256) void pcx_sample_best(WideArgs w) {
  __shared__ Group<256>::Scratch scratch;
  Group<256> g{&scratch, (int)threadIdx.x, 0};
  const int row = blockIdx.y, lo = blockIdx.x * SLICE;
  if (w.others) {
    const RowRules r = rules_of(w.a.rules, w.row0 + row);
    if (keeps_few(r.temperature, r.top_k)) return;  // (no best: the next launches pass the row over)
  }
  uint32_t key[WEP];
  load_slice<DT>(w, row, lo, key);
  uint32_t top = 0, at = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < WEP; ++i) top = key[i] > top ? key[i] : top;
  top = g.max(top);
#pragma unroll
  for (int i = 0; i < WEP; ++i)
    if (key[i] == top && (uint32_t)slice_index<DT>(lo, i) < at) at = (uint32_t)slice_index<DT>(lo, i);
  at = g.min(at);
  if (threadIdx.x == 0 && top) atomicMax(reinterpret_cast<unsigned long long*>(&w.state[row].best), (unsigned long long)top << 32 | (uint32_t)~at);
}
// Weights (and counts, where top_k asks for them) per value of one digit, of the keys that agree with the digits found so
// far: one pass over the logits, bound by the first digit's exponentials and LDS atomics (8 x 2^20 float32: 23 us; the second
// digit 15, the third 11; a bin's two words of every slice added to memory: 34 and 22).  A slice a workgroup: with half the workgroups, two slices each, 4 us more.
enum { FIRST = 0, BY_COUNT = 2, BY_MASS = 4 };  // the first digit; a later one of top_k's edge, of top_p's (a row's active bit)
template <int DT, int KIND>
__global__ __launch_bounds__(256) void pcx_sample_digit(WideArgs w, int level, int counts) {
  // (40 KB at most: four workgroups a CU; three, with counts of 32 bits, 115 us where this takes 101: top_k = 5,000 of 8 x 2^20)
  constexpr int PILE = 256, FULL = PILE - 64;
  __shared__ unsigned long long mass[2 * BINS];
  __shared__ uint32_t count[KIND == BY_MASS ? 1 : BINS / 2], piles[KIND == FIRST ? 1 : 4][KIND == FIRST ? 1 : PILE];  // (two counts a word)
  const int row = blockIdx.y, lo = blockIdx.x * SLICE;
  const RowState st = w.state[row];
  if (KIND != FIRST && !(st.active & KIND)) return;
  const RowRules r = rules_of(w.a.rules, w.row0 + row);
  const uint32_t best_key = (uint32_t)(st.best >> 32);
  if (!best_key || !(r.temperature > 0.0f)) return;
  uint32_t key[WEP];
  load_slice<DT>(w, row, lo, key);
  const float best = value_of<DT>(best_key);
  const double rate = 1.0 / (double)r.temperature;
  for (int i = threadIdx.x; i < BINS; i += 256) {
    mass[i] = 0;
    mass[BINS + i] = 0;
    if constexpr (KIND != BY_MASS) count[i / 2] = 0;
  }
  __syncthreads();
  auto add = [&](const uint32_t* four) {
    double v[4];
    key_weights<DT, 4>(four, best, rate, v);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (four[c]) {
        const uint32_t d = digit_of<DT>(four[c], level);
        if constexpr (KIND != BY_MASS)
          if (counts) atomicAdd(&count[d / 2], d & 1 ? 65536u : 1u);
        const bool small = v[c] < SMALL;
        atomicAdd(&mass[small ? BINS + d : d], (unsigned long long)(ldexp(v[c], small ? 62 : 50) + 0.5));
      }
  };
  if constexpr (KIND == FIRST) {
#pragma unroll 1
    for (int i = 0; i < WEP; i += 4) {
      add(key);
#pragma unroll
      for (int c = 0; c < WEP - 4; ++c) key[c] = key[c + 4];
    }
  } else {
    // Later digits concern some of the keys: a wave piles those up and weighs them four a lane (weighed where they lie, with
    // most lanes idle, the second digit of 8 x 2^20 float32 logits took 20 us, this way 15).
    uint32_t* const pile = piles[threadIdx.x >> 6];
    const uint32_t lane = threadIdx.x & 63;
    uint32_t high = 0;
    auto weigh = [&]() {
      uint32_t four[4];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int c = 0; c < 4; ++c) four[c] = c * 64 + lane < high ? pile[c * 64 + lane] : 0u;
      __builtin_amdgcn_wave_barrier();
      high = 0;
      add(four);
    };
#pragma unroll 1
    for (int i = 0; i < WEP; i += 4) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool mine = key[c] && same_prefix<DT>(key[c], st.prefix, level);
        const uint64_t who = __ballot(mine);
        if (mine) pile[high + __popcll(who & ((1ull << lane) - 1))] = key[c];
        high += (uint32_t)__popcll(who);
        if (high > FULL) weigh();
      }
#pragma unroll
      for (int c = 0; c < WEP - 4; ++c) key[c] = key[c + 4];
    }
    if (high) weigh();
  }
  __syncthreads();
  const int64_t at = ((int64_t)(KIND != FIRST) * w.batch + row) * BINS;
  for (int i = threadIdx.x; i < BINS; i += 256) {
    if constexpr (KIND != BY_MASS)
      if (const uint32_t n = (count[i / 2] >> (16 * (i & 1))) & 0xFFFFu) atomicAdd(&w.count[at + i], n);
    if (mass[i] | mass[BINS + i]) {
      bool is_low;
      const uint64_t sum = slice_sum(mass[i], mass[BINS + i], w.scale, &is_low);
      atomicAdd(reinterpret_cast<unsigned long long*>((is_low ? w.low : w.high) + at + i), (unsigned long long)sum);
    }
  }
}
// Which bin of the digit the edge lies in.  by_mass: top_p's edge, else top_k's.
template <int DT>
__global__ __launch_bounds__(256) void pcx_sample_edge(WideArgs w, int level, int by_mass) {
  __shared__ Group<256>::Scratch scratch;
  __shared__ RowState next;
  Group<256> g{&scratch, (int)threadIdx.x, 0};
  const int row = blockIdx.x;
  RowState st = w.state[row];
  const RowRules r = rules_of(w.a.rules, w.row0 + row);
  const uint32_t best_key = (uint32_t)(st.best >> 32);
  if (!best_key || !(r.temperature > 0.0f)) return;
  if (level > 0 && !(st.active & (by_mass ? 4u : 2u))) return;
  const int64_t at = ((int64_t)(level != 0) * w.batch + row) * BINS;
  // thread 0 has the highest bins: eight a thread
  uint64_t counts[8], c_mine = 0, c_all;
  double masses[8], m_mine = 0.0, m_all;
  const int64_t mine_at = at + BINS - 8 * ((int)threadIdx.x + 1);
  const Pack<uint64_t, 8> high = *reinterpret_cast<const Pack<uint64_t, 8>*>(w.high + mine_at), low = *reinterpret_cast<const Pack<uint64_t, 8>*>(w.low + mine_at);
  const Pack<uint32_t, 8> n = *reinterpret_cast<const Pack<uint32_t, 8>*>(w.count + mine_at);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    counts[i] = n.v[7 - i];
    masses[i] = weight_of(high.v[7 - i], low.v[7 - i], w.scale);
    c_mine += counts[i];
    m_mine += masses[i];
  }
  if (level != 0) {  // for the next digit
    *reinterpret_cast<Pack<uint64_t, 8>*>(w.high + mine_at) = Pack<uint64_t, 8>{};
    *reinterpret_cast<Pack<uint64_t, 8>*>(w.low + mine_at) = Pack<uint64_t, 8>{};
    *reinterpret_cast<Pack<uint32_t, 8>*>(w.count + mine_at) = Pack<uint32_t, 8>{};
  }
  const uint64_t c = g.scan(c_mine, &c_all);
  const double m = g.scan(m_mine, &m_all);
  if (level == 0) {
    st.above = 0.0;
    st.count_above = 0;
    if (by_mass) {
      if (!(st.active & 2u)) st.total = m_all;
      st.target = (double)r.top_p * st.total;
      if (r.top_p < 1.0f) st.active |= 4u;
    } else if (r.top_k > 0 && c_all > (uint64_t)r.top_k) {
      st.active |= 2u;
    }
  }
  const bool cuts = (st.active & (by_mass ? 4u : 2u)) != 0;
  if (threadIdx.x == 0) next = st;
  __syncthreads();
  if (cuts) {
    // the first bin, from the top, at which the edge is reached
    uint32_t found = 0xFFFFFFFFu;
    uint64_t c_run = c, c_at = 0;
    double m_run = m, m_at = 0.0;  // ahead of the bin taken
    int bin_at = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(by_mass ? masses[i] > 0.0 : counts[i] > 0) || found != 0xFFFFFFFFu) continue;
      c_at = c_run;
      m_at = m_run;
      bin_at = BINS - 1 - ((int)threadIdx.x * 8 + i);
      c_run += counts[i];
      m_run += masses[i];
      const bool reached = by_mass ? st.above + m_run >= st.target : st.count_above + c_run >= (uint64_t)r.top_k;
      if (reached) found = threadIdx.x;
    }
    uint32_t who = g.min(found);
    // (sums over parts can miss the target by their rounding: then the lowest bin that holds anything)
    const uint32_t lowest = g.max(bin_at >= 0 ? threadIdx.x : 0u);
    if (who == 0xFFFFFFFFu) who = lowest;
    const bool mine = who == threadIdx.x && bin_at >= 0;
    if (mine) {
      next.count_above = st.count_above + c_at;
      next.above = st.above + m_at;
      next.prefix = (level == 0 ? 0u : st.prefix) | ((uint32_t)bin_at << digit_shift<DT>(level));
      if (level == LEVELS<DT> - 1) {
        const double tie = weight_of(value_of<DT>(next.prefix), value_of<DT>(best_key), 1.0 / (double)r.temperature);
        next.edge = next.prefix;
        if (by_mass) {
          const double need = ceil((st.target - next.above) / tie);
          const uint32_t limit = (st.active & 2u) && next.edge == st.edge ? st.ties : 0xFFFFFFFFu;  // (what top_k left of them)
          next.ties = need >= 1.0 ? (need < 4e9 ? (uint32_t)need : 0xFFFFFFFFu) : 1u;
          if (next.ties > limit) next.ties = limit;
        } else {
          next.ties = (uint32_t)((uint64_t)r.top_k - next.count_above);
          next.total = next.above + (double)next.ties * tie;
        }
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) w.state[row] = next;
}
// What of a slice is kept: weight above the edge, and how many equal it.
template <int DT>
__global__ __launch_bounds__(256) void pcx_sample_weigh(WideArgs w) {
  __shared__ Group<256>::Scratch scratch;
  Group<256> g{&scratch, (int)threadIdx.x, 0};
  const int row = blockIdx.y, lo = blockIdx.x * SLICE;
  const RowState st = w.state[row];
  const RowRules r = rules_of(w.a.rules, w.row0 + row);
  const uint32_t best_key = (uint32_t)(st.best >> 32);
  if (!best_key || !(r.temperature > 0.0f)) return;
  uint32_t key[WEP];
  load_slice<DT>(w, row, lo, key);
  const float best = value_of<DT>(best_key);
  const double rate = 1.0 / (double)r.temperature;
  double mine = 0.0;
  uint32_t ties = 0;
#pragma unroll
  for (int i = 0; i < WEP; i += 4) {
    double v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      ties += ballots(st.edge && key[i + c] == st.edge);
      if (key[i + c] <= st.edge) key[i + c] = 0;
    }
    key_weights<DT, 4>(key + i, best, rate, v);
#pragma unroll
    for (int c = 0; c < 4; ++c) mine += v[c] >= (double)r.min_p ? v[c] : 0.0;
  }
  mine = g.sum(mine);
  ties = g.count(ties);
  if (threadIdx.x == 0) w.slots[(int64_t)row * w.slices + blockIdx.x] = Slot{mine, ties};
}
// The slice that the number falls into, then the action within it.
template <int DT>
__global__ __launch_bounds__(256) void pcx_sample_pick(WideArgs w) {
  __shared__ Group<256>::Scratch scratch;
  __shared__ double offset;
  __shared__ uint32_t ties_left;
  Group<256> g{&scratch, (int)threadIdx.x, 0};
  const int row = blockIdx.x;
  const int64_t at = w.row0 + row;
  const RowState st = w.state[row];
  const RowRules r = rules_of(w.a.rules, at);
  const uint32_t best_key = (uint32_t)(st.best >> 32);
  if (w.others && keeps_few(r.temperature, r.top_k)) return;
  if (!best_key || !(r.temperature > 0.0f)) {
    if (threadIdx.x == 0) w.a.out[at] = best_key ? (int)~(uint32_t)st.best : NONE;
    return;
  }
  const float best = value_of<DT>(best_key);
  const double rate = 1.0 / (double)r.temperature;
  double tie = st.edge ? weight_of(value_of<DT>(st.edge), best, rate) : 0.0;
  if (tie < (double)r.min_p) tie = 0.0;
  // neighbouring slices a thread: (2^24 actions are 2048 slices, eight a thread)
  const Slot* const slots = w.slots + (int64_t)row * w.slices;
  const int per = (w.slices + 255) / 256, s0 = (int)threadIdx.x * per;
  uint64_t ties = 0, ties_all;
  for (int i = s0; i < s0 + per && i < w.slices; ++i) ties += slots[i].ties;
  const uint64_t ties_before = g.scan(ties, &ties_all);
  uint64_t left = ties_before < st.ties ? st.ties - ties_before : 0;
  const uint64_t left0 = left;
  double mine = 0.0, total;
  for (int i = s0; i < s0 + per && i < w.slices; ++i) {
    const uint64_t kept = slots[i].ties < left ? slots[i].ties : left;
    left -= kept;
    mine += slots[i].weight + (double)kept * tie;
  }
  const double before = g.scan(mine, &total);
  const double goal = (double)w.a.uniforms[at] * total;
  uint32_t chosen = 0xFFFFFFFFu, last = 0;
  double run = before, run_at = 0.0, run_last = 0.0;
  uint64_t left_at = 0, left_last = 0;
  left = left0;
  for (int i = s0; i < s0 + per && i < w.slices; ++i) {
    const uint64_t kept = slots[i].ties < left ? slots[i].ties : left;
    const double weight = slots[i].weight + (double)kept * tie;
    if (weight > 0.0) {
      last = (uint32_t)i + 1;
      run_last = run;
      left_last = left;
      if (run + weight > goal && chosen == 0xFFFFFFFFu) { chosen = (uint32_t)i; run_at = run; left_at = left; }
    }
    run += weight;
    left -= kept;
  }
  uint32_t slice = g.min(chosen);
  if (slice == 0xFFFFFFFFu) {  // (u asks for more than there is: the last slice that holds anything)
    slice = g.max(last) - 1;
    chosen = last - 1;
    run_at = run_last;
    left_at = left_last;
  }
  if (chosen == slice) { offset = run_at; ties_left = (uint32_t)(left_at < 0xFFFFFFFFull ? left_at : 0xFFFFFFFFull); }
  __syncthreads();
  const int lo = (int)slice * SLICE, j0 = lo + (int)threadIdx.x * WEP;
  const int end = w.a.rows.actions - lo < SLICE ? w.a.rows.actions : lo + SLICE;
  uint32_t key[WEP];
  double v[WEP];
  load_keys<DT, WEP>(w.a.rows, at, j0, end, key);
#pragma unroll
  for (int i = 0; i < WEP; ++i)
    if (key[i] < st.edge) key[i] = 0;
  key_weights<DT, WEP>(key, best, rate, v);
#pragma unroll
  for (int i = 0; i < WEP; ++i)
    if (v[i] < (double)r.min_p) v[i] = 0.0;
  if (st.edge) drop_ties<256, WEP>(g, st.edge, ties_left, key, v);
  const int pick = draw_action<256, WEP>(g, v, goal, offset, true);
  if (threadIdx.x == 0) w.a.out[at] = lo + pick;
}

// ---------------------------------------------------------------- log-probability, entropy and their gradient

struct LogProbArgs {
  Rows rows;
  float rate;                 // 1 / temperature
  const int32_t* taken;
  float* log_prob;            // [n]
  float* entropy;             // [n]
  float2* stats;              // [n]: the largest logit, sum exp((x - largest) / T); 0 where nothing is allowed
  const float* grad_log_prob; // backward, or null
  const float* grad_entropy;  // backward, or null
  void* grad;                 // [n][actions]
  float4* partial;            // [n][slices], when a row is divided
  int32_t slices;
};

// exp(d) for d <= 0, d = x log2(e) carried in two parts: good to about 2^-23 however large x is.
__device__ __forceinline__ float exp_of(float d) {
  const float hi = d * 1.44269502f;
  const float lo = fmaf(d, 1.44269502f, -hi) + d * 1.925963033e-8f;
  const float e = __builtin_amdgcn_exp2f(hi);
  return d > -200.0f ? fmaf(e, lo * 0.693147181f, e) : 0.0f;
}

// Running (largest x, sum of exp, sum of d exp) of a part of a row, relative to the largest so far.
struct Soft {
  float m, s, t;
  __device__ __forceinline__ void join(float m2, float s2, float t2, float rate) {
    if (!(m2 > -INFINITY)) return;
    if (!(m > -INFINITY)) { m = m2; s = s2; t = t2; return; }
    const float big = fmaxf(m, m2);
    const float d1 = m == big ? 0.0f : (m - big) * rate, d2 = m2 == big ? 0.0f : (m2 - big) * rate;
    const float e1 = exp_of(d1), e2 = exp_of(d2);
    t = (e1 > 0.0f ? e1 * fmaf(d1, s, t) : 0.0f) + (e2 > 0.0f ? e2 * fmaf(d2, s2, t2) : 0.0f);
    s = e1 * s + e2 * s2;
    m = big;
  }
};
template <int DT>
__device__ __forceinline__ void finish_row(const LogProbArgs& a, int64_t row, const Soft& v) {
  typedef typename Logit<DT>::T T;
  const bool some = v.m > -INFINITY;
  const float ls = some ? logf(v.s) : 0.0f;
  a.entropy[row] = some ? ls - v.t / v.s : 0.0f;
  a.stats[row] = some ? make_float2(v.m, v.s) : make_float2(0.0f, 0.0f);
  const int taken = a.taken[row];
  float lp = 0.0f;
  if (taken != NONE && (taken < 0 || taken >= a.rows.actions)) lp = NAN;  // (no such action: not passed over in silence)
  else if (taken != NONE && some) {
    const float x = Logit<DT>::get(reinterpret_cast<const T*>(a.rows.logits)[row * a.rows.row_stride + taken]);
    const bool ok = allowed(x, a.rows.legal ? a.rows.legal[row * a.rows.legal_stride + taken] != 0 : true);
    lp = ok ? (x == v.m ? 0.0f : (x - v.m) * a.rate) - ls : -INFINITY;
  }
  a.log_prob[row] = lp;
}

// sum of exp and of d exp of N logits relative to `big` (> -infinity); -infinity adds nothing
template <int N>
__device__ __forceinline__ void soft_sums(const float* x, float big, float rate, float* s, float* t) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = x[i] == big ? 0.0f : fmaxf((x[i] - big) * rate, -1e4f), e = exp_of(d);  // (d e is 0 long before -1e4)
    *s += e;
    *t = fmaf(d, e, *t);
  }
}
// A wave (few actions) or a workgroup takes a row, 16 neighbouring logits a thread and turn: read once, the largest logit and
// the sums relative to it kept per thread and joined at the end.  4,096 rows of 4,096 bfloat16 logits: 17 us, 1.9 TB/s of the
// 5.2 that a copy reaches (25 with an exponential in every step of the join); half of it is the exponentials, two rounds of
// workgroups wait for their first bytes, and asking for the action's logit ahead of the row gained nothing.
template <int DT, int THREADS>
__global__ __launch_bounds__(256) void pcx_log_prob_forward(LogProbArgs a) {
  typedef typename Logit<DT>::T T;
  constexpr int ROWS = 256 / THREADS, EP = THREADS == 64 ? 8 : 16;
  __shared__ typename Group<THREADS>::Scratch scratch[ROWS];
  const int t = threadIdx.x % THREADS;
  Group<THREADS> g{&scratch[threadIdx.x / THREADS], t, 0};
  const int64_t unit = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
  if (unit >= a.rows.n * a.slices) return;
  const int64_t row = unit / a.slices;
  const int slice = (int)(unit - row * a.slices);
  const int lo = a.slices > 1 ? slice * SLICE : 0;
  const int end = a.slices > 1 && a.rows.actions - lo > SLICE ? lo + SLICE : a.rows.actions;
  const T* const x_row = reinterpret_cast<const T*>(a.rows.logits) + row * a.rows.row_stride;
  const uint8_t* const l_row = a.rows.legal ? a.rows.legal + row * a.rows.legal_stride : nullptr;
  Soft v{-INFINITY, 0.0f, 0.0f};
  for (int j = lo + t * EP; j < end; j += THREADS * EP) {
    float x[EP];
    load_logits<DT, EP>(x_row, l_row, j, end, x);
    float big = x[0];
#pragma unroll
    for (int i = 1; i < EP; ++i) big = fmaxf(big, x[i]);
    if (!(big > -INFINITY)) continue;
    float s = 0.0f, tt = 0.0f;
    soft_sums<EP>(x, big, a.rate, &s, &tt);
    v.join(big, s, tt, a.rate);
  }
  // the threads' parts relative to the row's largest logit, then plain sums
  const uint32_t top = g.max(v.m > -INFINITY ? order_of<PCX_F32>(v.m) : 0u);
  if (top) {
    const float big = value_of<PCX_F32>(top), d = v.m == big ? 0.0f : (v.m - big) * a.rate, e = v.m > -INFINITY ? exp_of(d) : 0.0f;
    v.t = g.sum(e > 0.0f ? e * fmaf(d, v.s, v.t) : 0.0f);
    v.s = g.sum(e > 0.0f ? e * v.s : 0.0f);
    v.m = big;
  }
  if (t != 0) return;
  if (a.slices > 1) a.partial[unit] = make_float4(v.m, v.s, v.t, 0.0f);
  else finish_row<DT>(a, row, v);
}
template <int DT>
__global__ __launch_bounds__(64) void pcx_log_prob_join(LogProbArgs a) {
  const int64_t row = blockIdx.x;
  Soft v{-INFINITY, 0.0f, 0.0f};
  for (int i = threadIdx.x; i < a.slices; i += 64) {
    const float4 p = a.partial[row * a.slices + i];
    v.join(p.x, p.y, p.z, a.rate);
  }
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) {
    const float m2 = __shfl_xor(v.m, k), s2 = __shfl_xor(v.s, k), t2 = __shfl_xor(v.t, k);
    v.join(m2, s2, t2, a.rate);
  }
  if (threadIdx.x) return;
  finish_row<DT>(a, row, v);
}

// One row's numbers for the gradient of its elements.
struct RowGrad { float m, inv, ls, h, gl, ge; int taken; bool some; };
__device__ __forceinline__ RowGrad row_grad(const LogProbArgs& a, int64_t row) {
  RowGrad g;
  const float2 st = a.stats[row];
  g.some = st.y > 0.0f;
  g.m = st.x;
  g.inv = 1.0f / st.y;
  g.ls = logf(st.y);
  g.h = a.entropy[row];
  g.taken = a.taken[row];
  g.gl = a.grad_log_prob && g.taken != NONE ? a.grad_log_prob[row] : 0.0f;
  if (g.taken != NONE && (g.taken < 0 || g.taken >= a.rows.actions)) g.gl = NAN;
  g.ge = a.grad_entropy ? a.grad_entropy[row] : 0.0f;
  return g;
}
__device__ __forceinline__ float element_grad(const RowGrad& g, float x, int j, float rate) {
  const float d = x == g.m ? 0.0f : fmaxf((x - g.m) * rate, -1e4f);
  const float p = exp_of(d) * g.inv;
  const float v = ((j == g.taken ? g.gl : 0.0f) - p * (g.gl + g.ge * (d - g.ls + g.h))) * rate;
  return x > -INFINITY ? v : 0.0f;
}
// Read once, written once: the same rows 23 us, 2.9 TB/s.
template <int DT, int THREADS>
__global__ __launch_bounds__(256) void pcx_log_prob_backward_kernel(LogProbArgs a) {
  typedef typename Logit<DT>::T T;
  constexpr int ROWS = 256 / THREADS, W = 16 / (int)sizeof(T);
  const int t = threadIdx.x % THREADS;
  const int64_t unit = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
  if (unit >= a.rows.n * a.slices) return;
  const int64_t row = unit / a.slices;
  const int slice = (int)(unit - row * a.slices);
  const int lo = a.slices > 1 ? slice * SLICE : 0;
  const int end = a.slices > 1 && a.rows.actions - lo > SLICE ? lo + SLICE : a.rows.actions;
  const T* const x_row = reinterpret_cast<const T*>(a.rows.logits) + row * a.rows.row_stride;
  const uint8_t* const l_row = a.rows.legal ? a.rows.legal + row * a.rows.legal_stride : nullptr;
  const RowGrad g = row_grad(a, row);
  T* const out = reinterpret_cast<T*>(a.grad) + row * a.rows.actions;
#pragma unroll 2
  for (int j = lo + t * W; j < end; j += THREADS * W) {
    float x[W];
    load_logits<DT, W>(x_row, l_row, j, end, x);
    Pack<T, W> q;
#pragma unroll
    for (int i = 0; i < W; ++i) q.v[i] = Logit<DT>::put(element_grad(g, x[i], j + i, a.rate));
    if (j + W <= end) __builtin_memcpy(out + j, &q, sizeof q);
    else
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (j + i < end) out[j + i] = q.v[i];
  }
}
// Few actions: a thread holds a row (2^20 rows of 5 float32 logits and legal flags: 12 us forward, 17 with its gradient's
// write, 3 TB/s; the flags come byte by byte).
template <int DT, int CAP>
__global__ __launch_bounds__(256) void pcx_log_prob_rows(LogProbArgs a) {
  typedef typename Logit<DT>::T T;
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows.n) return;
  float x[CAP];
  load_logits<DT, CAP>(reinterpret_cast<const T*>(a.rows.logits) + row * a.rows.row_stride, a.rows.legal ? a.rows.legal + row * a.rows.legal_stride : nullptr,
                       0, a.rows.actions, x);
  Soft v{x[0], 0.0f, 0.0f};
#pragma unroll
  for (int i = 1; i < CAP; ++i) v.m = fmaxf(v.m, x[i]);
  if (v.m > -INFINITY) soft_sums<CAP>(x, v.m, a.rate, &v.s, &v.t);
  finish_row<DT>(a, row, v);
}
template <int DT, int CAP>
__global__ __launch_bounds__(256) void pcx_log_prob_rows_backward(LogProbArgs a) {
  typedef typename Logit<DT>::T T;
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows.n) return;
  float x[CAP];
  load_logits<DT, CAP>(reinterpret_cast<const T*>(a.rows.logits) + row * a.rows.row_stride, a.rows.legal ? a.rows.legal + row * a.rows.legal_stride : nullptr,
                       0, a.rows.actions, x);
  const RowGrad g = row_grad(a, row);
  T* const out = reinterpret_cast<T*>(a.grad) + row * a.rows.actions;
#pragma unroll
  for (int i = 0; i < CAP; ++i)
    if (i < a.rows.actions) out[i] = Logit<DT>::put(element_grad(g, x[i], i, a.rate));
}

// ---------------------------------------------------------------- plans and entry points

constexpr int ROW_IN_GROUP = 16384;  // actions a workgroup holds in registers
constexpr int ROW_ALONE = 1 << 18;   // ... one goes through alone where top_k keeps few (pcx_sample_top has both sides' times)
constexpr int WIDE_BATCH = 1024;     // rows per batch of launches beyond that
constexpr int64_t CHUNK = 1 << 22;   // rows per launch otherwise (a grid has fewer than 2^32 threads)

int check_rows(const pcx_logits_desc* d, Rows* r, const char* who) {
  if (!d) return set_error(PCX_E_INVALID, "%s: null description", who);
  if (d->dtype != PCX_F32 && d->dtype != PCX_F16 && d->dtype != PCX_BF16)
    return set_error(PCX_E_INVALID, "%s: logits are float32, float16 or bfloat16", who);
  if (d->n < 0 || d->n > (int64_t)1 << 31) return set_error(PCX_E_INVALID, "%s: %lld rows", who, (long long)d->n);
  if (d->actions < 1 || d->actions > 1 << 24) return set_error(PCX_E_INVALID, "%s: %d actions", who, d->actions);
  if (d->row_stride < 0 || d->legal_stride < 0) return set_error(PCX_E_INVALID, "%s: negative stride", who);
  r->n = d->n; r->row_stride = d->row_stride; r->legal_stride = d->legal_stride; r->actions = d->actions;
  return 0;
}
bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }
int elem_size(int dtype) { return dtype == PCX_F32 ? 4 : 2; }

// The rows of one launch, from row0 on.
Rows rows_from(const Rows& all, int64_t row0, int es) {
  Rows r = all;
  r.n = all.n - row0 < CHUNK ? all.n - row0 : CHUNK;
  r.logits = reinterpret_cast<const uint8_t*>(all.logits) + row0 * all.row_stride * es;
  if (all.legal) r.legal = all.legal + row0 * all.legal_stride;
  return r;
}

int wide_slices(int actions) { return (actions + SLICE - 1) / SLICE; }
uint64_t wide_bytes(int64_t n, int actions) {
  if (actions <= ROW_IN_GROUP) return 0;
  const uint64_t rows = (uint64_t)(n < WIDE_BATCH ? n : WIDE_BATCH);
  return rows * (sizeof(RowState) + 2ull * BINS * 20 + (uint64_t)wide_slices(actions) * sizeof(Slot)) + 1024;
}
// A row of logits is divided among workgroups where there are too few rows to fill the chip.
int log_prob_slices(int64_t n, int actions) { return actions > 2 * SLICE && n < 2048 ? wide_slices(actions) : 1; }

template <int DT>
int sample_wide(const SampleArgs& a, bool others, void* workspace, hipStream_t st) {
  const int slices = wide_slices(a.rows.actions);
  int log2a = 0;
  while ((1 << log2a) < a.rows.actions) ++log2a;
  for (int64_t row0 = 0; row0 < a.rows.n; row0 += WIDE_BATCH) {
    WideArgs w{a};
    w.row0 = row0;
    w.batch = (int32_t)(a.rows.n - row0 < WIDE_BATCH ? a.rows.n - row0 : WIDE_BATCH);
    w.slices = slices;
    w.scale = 63 - log2a;
    w.others = others;
    uint8_t* p = reinterpret_cast<uint8_t*>(workspace);
    w.high = reinterpret_cast<uint64_t*>(p); p += (size_t)w.batch * 2 * BINS * 8;
    w.low = reinterpret_cast<uint64_t*>(p); p += (size_t)w.batch * 2 * BINS * 8;
    w.state = reinterpret_cast<RowState*>(p); p += (size_t)w.batch * sizeof(RowState);
    w.slots = reinterpret_cast<Slot*>(p); p += (size_t)w.batch * slices * sizeof(Slot);
    w.count = reinterpret_cast<uint32_t*>(p);
    const dim3 rows((unsigned)w.batch), grid((unsigned)slices, (unsigned)w.batch), block(256);
    hipLaunchKernelGGL(pcx_sample_clear, rows, block, 0, st, w);
    hipLaunchKernelGGL((pcx_sample_best<DT>), grid, block, 0, st, w);
    const bool k = a.rules.top_k_row || (a.rules.top_k > 0 && a.rules.top_k < a.rows.actions);
    const bool p_ = a.rules.top_p_row || a.rules.top_p < 1.0f;
    if (k || p_) {
      hipLaunchKernelGGL((pcx_sample_digit<DT, FIRST>), grid, block, 0, st, w, 0, k);
      for (int by_mass = k ? 0 : 1; by_mass <= (p_ ? 1 : 0); ++by_mass)
        for (int level = 0; level < LEVELS<DT>; ++level) {
          if (level && by_mass) hipLaunchKernelGGL((pcx_sample_digit<DT, BY_MASS>), grid, block, 0, st, w, level, 0);
          else if (level) hipLaunchKernelGGL((pcx_sample_digit<DT, BY_COUNT>), grid, block, 0, st, w, level, 1);
          hipLaunchKernelGGL((pcx_sample_edge<DT>), rows, block, 0, st, w, level, by_mass);
        }
    }
    hipLaunchKernelGGL((pcx_sample_weigh<DT>), grid, block, 0, st, w);
    hipLaunchKernelGGL((pcx_sample_pick<DT>), rows, block, 0, st, w);
  }
  return 0;
}
template <int DT>
int sample_type(const SampleArgs& all, void* workspace, hipStream_t st) {
  const int A = all.rows.actions;
  // (Which way a row goes, its actions and its own rules say, not how many rows there are: its answer must not depend on them.)
  bool top = false;
  if (A > ROW_IN_GROUP) {
    const Rules& r = all.rules;
    const bool every = keeps_few(r.temperature_row ? 1.0f : r.temperature, r.top_k_row ? 0 : r.top_k);  // whatever the rows' own rules say
    top = A <= ROW_ALONE && (every || r.temperature_row || r.top_k_row);
    if (!top || !every)
      if (int rc = sample_wide<DT>(all, top, workspace, st)) return rc;
    if (!top) return 0;
  }
  for (int64_t row0 = 0; row0 < all.rows.n; row0 += CHUNK) {
    SampleArgs a = all;
    a.rows = rows_from(all.rows, row0, elem_size(DT));
    a.uniforms += row0;
    a.out += row0;
    if (a.rules.temperature_row) a.rules.temperature_row += row0;
    if (a.rules.top_k_row) a.rules.top_k_row += row0;
    if (a.rules.top_p_row) a.rules.top_p_row += row0;
    if (a.rules.min_p_row) a.rules.min_p_row += row0;
    const dim3 block(256), per_thread((unsigned)((a.rows.n + 255) / 256)), per_wave((unsigned)((a.rows.n + 3) / 4)), per_group((unsigned)a.rows.n);
    if (top) hipLaunchKernelGGL((pcx_sample_top<DT>), per_group, dim3(TOP_THREADS), 0, st, a);
    else if (A <= 6) hipLaunchKernelGGL((pcx_sample_rows<DT, 6>), per_thread, block, 0, st, a);
    else if (A <= 8) hipLaunchKernelGGL((pcx_sample_rows<DT, 8>), per_thread, block, 0, st, a);
    else if (A <= 16) hipLaunchKernelGGL((pcx_sample_rows<DT, 16>), per_thread, block, 0, st, a);
    else if (A <= 128) hipLaunchKernelGGL((pcx_sample_group<DT, 64, 2>), per_wave, block, 0, st, a);
    else if (A <= 256) hipLaunchKernelGGL((pcx_sample_group<DT, 64, 4>), per_wave, block, 0, st, a);
    else if (A <= 512) hipLaunchKernelGGL((pcx_sample_group<DT, 64, 8>), per_wave, block, 0, st, a);
    else if (A <= 1024) hipLaunchKernelGGL((pcx_sample_group<DT, 64, 16>), per_wave, block, 0, st, a);
    else if (A <= 4096) hipLaunchKernelGGL((pcx_sample_group<DT, 256, 16>), per_group, block, 0, st, a);
    else hipLaunchKernelGGL((pcx_sample_group<DT, 512, 32>), per_group, dim3(512), 0, st, a);
  }
  return 0;
}
template <int DT>
int log_prob_type(const LogProbArgs& all, bool backward, hipStream_t st) {
  const int A = all.rows.actions;
  for (int64_t row0 = 0; row0 < all.rows.n; row0 += CHUNK) {
    LogProbArgs a = all;
    a.rows = rows_from(all.rows, row0, elem_size(DT));
    a.taken += row0;
    a.entropy += row0;
    a.stats += row0;
    if (a.log_prob) a.log_prob += row0;
    if (a.grad_log_prob) a.grad_log_prob += row0;
    if (a.grad_entropy) a.grad_entropy += row0;
    if (a.grad) a.grad = reinterpret_cast<uint8_t*>(a.grad) + row0 * A * elem_size(DT);
    const int64_t units = a.rows.n * a.slices;  // (slices > 1: few rows, one chunk)
    const dim3 block(256), per_thread((unsigned)((a.rows.n + 255) / 256)), per_wave((unsigned)((units + 3) / 4)), per_group((unsigned)units);
    if (!backward) {
      if (A <= 8) hipLaunchKernelGGL((pcx_log_prob_rows<DT, 8>), per_thread, block, 0, st, a);
      else if (A <= 32) hipLaunchKernelGGL((pcx_log_prob_rows<DT, 32>), per_thread, block, 0, st, a);
      else if (A <= 2048) hipLaunchKernelGGL((pcx_log_prob_forward<DT, 64>), per_wave, block, 0, st, a);
      else hipLaunchKernelGGL((pcx_log_prob_forward<DT, 256>), per_group, block, 0, st, a);
      if (a.slices > 1) hipLaunchKernelGGL((pcx_log_prob_join<DT>), dim3((unsigned)a.rows.n), dim3(64), 0, st, a);
    } else {
      if (A <= 8) hipLaunchKernelGGL((pcx_log_prob_rows_backward<DT, 8>), per_thread, block, 0, st, a);
      else if (A <= 32) hipLaunchKernelGGL((pcx_log_prob_rows_backward<DT, 32>), per_thread, block, 0, st, a);
      else if (A <= 2048) hipLaunchKernelGGL((pcx_log_prob_backward_kernel<DT, 64>), per_wave, block, 0, st, a);
      else hipLaunchKernelGGL((pcx_log_prob_backward_kernel<DT, 256>), per_group, block, 0, st, a);
    }
  }
  return 0;
}

}  // namespace

extern "C" {

int pcx_sample_size(const pcx_logits_desc* d, uint64_t* bytes) {
  Rows r;
  if (int rc = check_rows(d, &r, "pcx_sample_size")) return rc;
  if (!bytes) return set_error(PCX_E_INVALID, "pcx_sample_size: null");
  *bytes = wide_bytes(r.n, r.actions);
  return 0;
}

int pcx_sample_actions(const pcx_logits_desc* d, const pcx_sampling* rules, const void* logits, const uint8_t* legal,
                       const float* uniforms, int32_t* actions_out, void* workspace, uint64_t workspace_bytes, void* stream) {
  SampleArgs a{};
  if (int rc = check_rows(d, &a.rows, "pcx_sample_actions")) return rc;
  if (!rules) return set_error(PCX_E_INVALID, "pcx_sample_actions: no rules");
  if (!rules->temperature_row && !(rules->temperature >= 0.0f)) return set_error(PCX_E_INVALID, "pcx_sample_actions: the temperature must be 0 or more");
  if (!rules->top_k_row && rules->top_k < 0) return set_error(PCX_E_INVALID, "pcx_sample_actions: top_k must be 0 (all) or more");
  if (!rules->top_p_row && !(rules->top_p >= 0.0f)) return set_error(PCX_E_INVALID, "pcx_sample_actions: top_p must be 0 or more");
  if (!rules->min_p_row && !(rules->min_p >= 0.0f && rules->min_p <= 1.0f)) return set_error(PCX_E_INVALID, "pcx_sample_actions: min_p must lie in [0, 1]");
  if (!a.rows.n) return 0;
  if (!logits || !uniforms || !actions_out || misaligned(logits, elem_size(d->dtype)) || misaligned(uniforms, 4) || misaligned(actions_out, 4) ||
      misaligned(rules->temperature_row, 4) || misaligned(rules->top_k_row, 4) || misaligned(rules->top_p_row, 4) || misaligned(rules->min_p_row, 4))
    return set_error(PCX_E_INVALID, "pcx_sample_actions: null or misaligned pointer");
  const uint64_t need = wide_bytes(a.rows.n, a.rows.actions);
  if (need && (!workspace || workspace_bytes < need || misaligned(workspace, 16)))
    return set_error(PCX_E_INVALID, "pcx_sample_actions: the workspace needs %llu bytes, 16-byte aligned", (unsigned long long)need);
  a.rows.logits = logits;
  a.rows.legal = legal;
  a.rules = Rules{rules->temperature, rules->top_p, rules->min_p, rules->top_k, rules->temperature_row, rules->top_k_row, rules->top_p_row, rules->min_p_row};
  a.uniforms = uniforms;
  a.out = actions_out;
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (d->dtype == PCX_F32) rc = sample_type<PCX_F32>(a, workspace, st);
  else if (d->dtype == PCX_F16) rc = sample_type<PCX_F16>(a, workspace, st);
  else rc = sample_type<PCX_BF16>(a, workspace, st);
  if (rc) return rc;
  PCX_HIP(hipGetLastError());
  return 0;
}

int pcx_log_prob_size(const pcx_logits_desc* d, uint64_t* bytes) {
  Rows r;
  if (int rc = check_rows(d, &r, "pcx_log_prob_size")) return rc;
  if (!bytes) return set_error(PCX_E_INVALID, "pcx_log_prob_size: null");
  const int slices = log_prob_slices(r.n, r.actions);
  *bytes = slices > 1 ? (uint64_t)r.n * slices * sizeof(float4) : 0;
  return 0;
}

static int log_prob_call(const pcx_logits_desc* d, float temperature, LogProbArgs* a, bool backward, void* stream, const char* who) {
  if (!(temperature > 0.0f) || !(1.0f / temperature > 0.0f) || !(1.0f / temperature < INFINITY))
    return set_error(PCX_E_INVALID, "%s: the temperature must be a positive number", who);
  if (misaligned(a->rows.logits, elem_size(d->dtype)) || misaligned(a->taken, 4) || misaligned(a->log_prob, 4) || misaligned(a->entropy, 4) ||
      misaligned(a->stats, 8) || misaligned(a->grad_log_prob, 4) || misaligned(a->grad_entropy, 4) || misaligned(a->grad, elem_size(d->dtype)))
    return set_error(PCX_E_INVALID, "%s: misaligned pointer", who);
  a->rate = 1.0f / temperature;
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (d->dtype == PCX_F32) rc = log_prob_type<PCX_F32>(*a, backward, st);
  else if (d->dtype == PCX_F16) rc = log_prob_type<PCX_F16>(*a, backward, st);
  else rc = log_prob_type<PCX_BF16>(*a, backward, st);
  if (rc) return rc;
  PCX_HIP(hipGetLastError());
  return 0;
}

int pcx_log_prob(const pcx_logits_desc* d, float temperature, const void* logits, const uint8_t* legal, const int32_t* actions,
                 float* log_prob, float* entropy, float* stats, void* workspace, uint64_t workspace_bytes, void* stream) {
  LogProbArgs a{};
  if (int rc = check_rows(d, &a.rows, "pcx_log_prob")) return rc;
  if (!a.rows.n) return 0;
  if (!logits || !actions || !log_prob || !entropy || !stats) return set_error(PCX_E_INVALID, "pcx_log_prob: null pointer");
  a.slices = log_prob_slices(a.rows.n, a.rows.actions);
  const uint64_t need = a.slices > 1 ? (uint64_t)a.rows.n * a.slices * sizeof(float4) : 0;
  if (need && (!workspace || workspace_bytes < need || misaligned(workspace, 16)))
    return set_error(PCX_E_INVALID, "pcx_log_prob: the workspace needs %llu bytes, 16-byte aligned", (unsigned long long)need);
  a.rows.logits = logits;
  a.rows.legal = legal;
  a.taken = actions;
  a.log_prob = log_prob;
  a.entropy = entropy;
  a.stats = reinterpret_cast<float2*>(stats);
  a.partial = reinterpret_cast<float4*>(workspace);
  return log_prob_call(d, temperature, &a, false, stream, "pcx_log_prob");
}

int pcx_log_prob_backward(const pcx_logits_desc* d, float temperature, const void* logits, const uint8_t* legal, const int32_t* actions,
                          const float* entropy, const float* stats, const float* grad_log_prob, const float* grad_entropy,
                          void* grad_logits, void* stream) {
  LogProbArgs a{};
  if (int rc = check_rows(d, &a.rows, "pcx_log_prob_backward")) return rc;
  if (!a.rows.n) return 0;
  if (!logits || !actions || !entropy || !stats || !grad_logits) return set_error(PCX_E_INVALID, "pcx_log_prob_backward: null pointer");
  a.slices = log_prob_slices(a.rows.n, a.rows.actions);
  a.rows.logits = logits;
  a.rows.legal = legal;
  a.taken = actions;
  a.entropy = const_cast<float*>(entropy);
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.grad_log_prob = grad_log_prob;
  a.grad_entropy = grad_entropy;
  a.grad = grad_logits;
  return log_prob_call(d, temperature, &a, true, stream, "pcx_log_prob_backward");
}

}  // extern "C"
