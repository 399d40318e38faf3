// r3_logprob.hip -- log probabilities of given labels, with the entropy and the best alternatives of every row, and their
// gradient: what a softmax classification loss is made of.
//
// For a row x of `classes` logits, with m = max x:
//   S = sum_j e^(x_j - m),   T = sum_j e^(x_j - m) (x_j - m)
//   log p_j = (x_j - m) - log S,   H = -sum_j p_j log p_j = log S - T / S
//   d x_j = dl [j = label] + sum_k dtop_k [j = top_k] - p_j (dl + sum_k dtop_k + dH (log p_j + H))
// One pass over the logits forward and one backward: (m, S, T) of two parts join as
//   m = max(m1, m2),  S = sum_i S_i e^(m_i - m),  T = sum_i e^(m_i - m) (T_i + S_i (m_i - m)),
// so a lane keeps a running triple and lanes, wavefronts and workgroups join theirs.  Both directions are bound by HBM.
//
// All of it in 32 bits.  A difference is held above -150 where it is a FACTOR (e^-150 is 0 in fp32): 0 * -inf would make the
// entropy NaN for every masked class.  The exponential itself sees the plain difference, so NaN and +inf reach S and T.
#include <hip/hip_runtime.h>

#include "../r3_kernels.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int TOP_MAX = 64;  // a wavefront holds the list of its best, one a lane

template <typename T, int N>
struct Pack {
  T v[N];
};
// 16 bytes from an address that is aligned to one element only (the row of an odd number of classes): global accesses need
// no more, and the compiler makes one wide load of it
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}

// an order of the floats as unsigned numbers; no float is 0 (the key of "nothing"); -0 is +0; every NaN is above +inf
__device__ __forceinline__ unsigned ord(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unord(unsigned u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
// greater = better: by value, then the lowest index
__device__ __forceinline__ unsigned long long make_key(float x, unsigned index) {
  return ((unsigned long long)ord(x) << 32) | (unsigned)~index;
}

__device__ __forceinline__ unsigned long long offered(float x, unsigned index) {
  return x == -__builtin_inff() ? 0ull : make_key(x, index);
}

struct Stat {  // of the values seen so far
  float m = -3.402823466e38f, s = 0.f, t = 0.f;
  __device__ __forceinline__ void raise(float to) {  // the reference point moves up to `to`
    const float d = m - to;
    const float r = __builtin_amdgcn_exp2f(d * LOG2E);
    t = r * (t + fmaxf(d, -150.f) * s);
    s *= r;
    m = to;
  }
  __device__ __forceinline__ void add(float x) {  // (x <= m)
    const float d = x - m;
    const float e = __builtin_amdgcn_exp2f(d * LOG2E);
    s += e;
    t = fmaf(e, fmaxf(d, -150.f), t);
  }
  __device__ __forceinline__ void join(float m2, float s2, float t2) {
    Stat o;
    o.m = m2, o.s = s2, o.t = t2;
    const float top = fmaxf(m, m2);
    raise(top);
    o.raise(top);
    s += o.s;
    t += o.t;
  }
};
template <int LANES>
__device__ __forceinline__ void join_lanes(Stat& a) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) a.join(__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.t, o));
}

struct Out {
  const int64_t* labels;
  int64_t ignore;
  int has_ignore;
  int k;
  float* log_prob;
  float* entropy;
  float* top_lp;
  int64_t* top_ix;
  float* stats;  // (rows, 2): m, log S
  Out from(int64_t row) const {  // of the rows from this one on
    Out o = *this;
    if (labels) o.labels += row;
    if (log_prob) o.log_prob += row;
    if (entropy) o.entropy += row;
    if (top_lp) o.top_lp += row * k;
    if (top_ix) o.top_ix += row * k;
    if (stats) o.stats += 2 * row;
    return o;
  }
};

// One thread per row: what the row's triple says.  S = 0 only where every class is -inf: log p is -inf there and the
// entropy 0 (nothing is left to be uncertain about); the backward pass knows such a row by its log S = -inf.
template <typename T>
__device__ __forceinline__ void finish_row(const Stat& a, int64_t row, const T* x, int64_t classes, const Out& o, float& m,
                                           float& ls) {
  m = a.m;
  ls = logf(a.s);
  if (o.stats) {
    o.stats[2 * row] = m;
    o.stats[2 * row + 1] = ls;
  }
  if (o.entropy) o.entropy[row] = a.s == 0.f ? 0.f : ls - a.t / a.s;
  if (o.labels) {
    const int64_t y = o.labels[row];
    float lp;
    if (o.has_ignore && y == o.ignore) lp = 0.f;
    else if (y < 0 || y >= classes) lp = __uint_as_float(0x7fc00000u);  // (a label that is none: NaN, and no read)
    else lp = a.s == 0.f ? -__builtin_inff() : ((float)x[y] - m) - ls;
    o.log_prob[row] = lp;
  }
}
__device__ __forceinline__ float top_value(float x, float m, float ls) {
  return ls == -__builtin_inff() ? -__builtin_inff() : (x - m) - ls;
}

// ---------------------------------------------------------------------------------------------- few classes
// LANES neighbouring lanes hold a row in registers, E values a lane.  VEC: 16-byte loads (aligned rows of whole packs).
// Few lanes a row exchange less and keep its best alternatives cheap; many read and write whole lines together, which the
// gradient needs most.  Values a lane, 4 / 8 / 16, us: forward 785664 x 16 fp32 17.6 / 14.4 / 16.8, 100000 x 32 7.8 / 7.0 /
// 7.5, 100000 x 64 with the best four 21.7 / 16.1 / 15.0; gradient 392832 x 16 12.5 / 12.7 / 15.6, 200000 x 15 10.5 / 14.5 /
// 22.4, 50000 x 81 10.8 / 9.6 / 11.2.
template <typename T, int LANES, int E, bool VEC>
__device__ __forceinline__ void load_row(const T* x, int lane, int64_t classes, float (&v)[E], int (&at)[E]) {
  constexpr int W = VEC ? (E * (int)sizeof(T) < 16 ? E : 16 / (int)sizeof(T)) : 1;
#pragma unroll
  for (int c = 0; c < E / W; ++c) {
    const int i = (c * LANES + lane) * W;
    if constexpr (VEC) {
      if (i < classes) {
        const Pack<T, W> p = load_pack<T, W>(x + i);
#pragma unroll
        for (int j = 0; j < W; ++j) v[c * W + j] = (float)p.v[j];
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) v[c * W + j] = 0.f;
      }
    } else {
      v[c] = i < classes ? (float)x[i] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < W; ++j) at[c * W + j] = i + j;
  }
}

template <typename T, int LANES, int E, bool VEC, bool TOP>
__global__ __launch_bounds__(256) void logprob_small_kernel(const T* __restrict__ logits, int64_t rows, int classes,
                                                            int64_t stride, Out o) {
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = g / LANES;
  const int lane = (int)(g % LANES);
  if (row >= rows) return;  // (whole groups: the exchanges below stay inside a group)
  const T* x = logits + row * stride;
  float v[E];
  int at[E];
  load_row<T, LANES, E, VEC>(x, lane, classes, v, at);
  float top = -3.402823466e38f;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (at[e] < classes) top = fmaxf(top, v[e]);
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  Stat a;
  a.m = top;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (at[e] < classes) a.add(v[e]);
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) {  // (one reference point for the group: plain sums)
    a.s += __shfl_xor(a.s, d);
    a.t += __shfl_xor(a.t, d);
  }
  float m = 0.f, ls = 0.f;
  if (lane == 0) finish_row(a, row, x, classes, o, m, ls);
  if constexpr (TOP) {
    unsigned u[E];
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] = at[e] < classes ? ord(v[e]) : 0u;
    for (int k = 0; k < o.k; ++k) {
      unsigned best = 0u;
      int which = 0x7fffffff;
#pragma unroll
      for (int e = 0; e < E; ++e)  // (a lane's places rise with e: the first of equals is the lowest)
        if (u[e] > best) best = u[e], which = at[e];
#pragma unroll
      for (int d = 1; d < LANES; d <<= 1) {
        const unsigned b2 = __shfl_xor(best, d);
        const int w2 = __shfl_xor(which, d);
        if (b2 > best || (b2 == best && w2 < which)) best = b2, which = w2;
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at[e] == which) u[e] = 0u;
      if (lane == 0) {
        o.top_lp[row * o.k + k] = top_value(unord(best), m, ls);
        o.top_ix[row * o.k + k] = which;
      }
    }
  }
}

template <typename T, int LANES, int E, bool VEC>
__global__ __launch_bounds__(256) void logprob_small_backward_kernel(const T* __restrict__ logits, int64_t rows, int classes,
                                                                     int64_t stride, Out o, const float* __restrict__ d_lp,
                                                                     const float* __restrict__ d_h,
                                                                     const float* __restrict__ d_top, T* __restrict__ dx) {
  constexpr int W = VEC ? (E * (int)sizeof(T) < 16 ? E : 16 / (int)sizeof(T)) : 1;
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = g / LANES;
  const int lane = (int)(g % LANES);
  if (row >= rows) return;
  float v[E];
  int at[E];
  load_row<T, LANES, E, VEC>(logits + row * stride, lane, classes, v, at);
  const float m = o.stats[2 * row], ls = o.stats[2 * row + 1];
  const bool empty = ls == -__builtin_inff();
  int64_t y = -1;
  float dl = 0.f, sum = 0.f, dh = 0.f, h = 0.f;
  if (d_lp) {
    y = o.labels[row];
    dl = d_lp[row];
    if (o.has_ignore && y == o.ignore) y = -1, dl = 0.f;
    else if (y < 0 || y >= classes) y = -1, dl = __uint_as_float(0x7fc00000u);
    sum = dl;
  }
  if (d_h) dh = d_h[row], h = o.entropy[row];
  if (d_top)
    for (int k = 0; k < o.k; ++k) sum += d_top[row * o.k + k];
  float r[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float lp = (v[e] - m) - ls, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    r[e] = (at[e] == y ? dl : 0.f) - p * (sum + dh * (fmaxf(lp, -150.f) + h));
  }
  if (d_top)
    for (int k = 0; k < o.k; ++k) {
      const int64_t ix = o.top_ix[row * o.k + k];
      const float d = d_top[row * o.k + k];
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at[e] == ix) r[e] += d;
    }
  T* out = dx + row * (int64_t)classes;
#pragma unroll
  for (int c = 0; c < E / W; ++c) {
    if (at[c * W] < classes) {
      Pack<T, W> p;
#pragma unroll
      for (int j = 0; j < W; ++j) p.v[j] = (T)(empty ? 0.f : r[c * W + j]);
      __builtin_memcpy(out + at[c * W], &p, sizeof(p));
    }
  }
}

// ---------------------------------------------------------------------------------------------- many classes
// The best keys a wavefront has seen, sorted, one a lane.
struct Best {
  unsigned long long key = 0;
  unsigned long long bound = 0;  // what k keys are known to pass, the list's or not (uniform)
  unsigned long long least = 0;  // what a key has to pass: the k-th best, or `bound`
  float floor = -__builtin_inff();  // its value
  // A value by the upper 16 bits of its place in the order (0: a masked class, which is no key).  They stay numbers from here
  // on: widened to a float's 32 bits again, those of an infinity would be a NaN's, and those of a tiny negative number's -0's.
  static __device__ __forceinline__ unsigned upper(float x) { return x != -__builtin_inff() ? ord(x) >> 16 : 0u; }
  // The j-th greatest of the lanes' (0: fewer have any).
  static __device__ __forceinline__ unsigned of_lanes(unsigned mine, int j) {
    unsigned t = 0;
#pragma unroll
    for (int b = 15; b >= 0; --b) {
      const unsigned more = t | 1u << b;
      if (__popcll(__ballot(mine >= more)) >= j) t = more;
    }
    return t;
  }
  __device__ __forceinline__ void seed(unsigned t) {  // k elements are known to reach these upper 16 bits
    bound = t ? ((unsigned long long)(t << 16) << 32) - 1 : 0ull;
    least = bound;
    floor = t ? unord(t << 16) : -__builtin_inff();
  }
  __device__ __forceinline__ void insert(unsigned long long in, int k) {  // `in` uniform
    const unsigned lo = (unsigned)key, hi = (unsigned)(key >> 32);
    // lane i takes lane i - 1's (wave_shr:1); lane 0 keeps its own, which the comparison below sees as "not better"
    const unsigned plo = __builtin_amdgcn_update_dpp(0xffffffffu, lo, 0x138, 0xf, 0xf, false);
    const unsigned phi = __builtin_amdgcn_update_dpp(0xffffffffu, hi, 0x138, 0xf, 0xf, false);
    const unsigned long long prev = ((unsigned long long)phi << 32) | plo;
    key = key > in ? key : (prev > in ? in : prev);
    lo_hi(k);
  }
  __device__ __forceinline__ void lo_hi(int k) {
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)key, k - 1);
    const unsigned hi = __builtin_amdgcn_readlane((unsigned)(key >> 32), k - 1);
    const unsigned long long kth = ((unsigned long long)hi << 32) | lo;
    if (kth > bound) {
      least = kth;
      floor = unord(hi);
    }
  }
  // every lane offers one key (0: none); all lanes of the wavefront call
  __device__ __forceinline__ void offer(unsigned long long in, int k) {
    unsigned long long who = __ballot(in > least);
    while (who) {
      const int l = __builtin_ctzll(who);
      const unsigned lo = __builtin_amdgcn_readlane((unsigned)in, l), hi = __builtin_amdgcn_readlane((unsigned)(in >> 32), l);
      insert(((unsigned long long)hi << 32) | lo, k);
      if ((int)__lane_id() == l) in = 0;
      who = __ballot(in > least);
    }
  }
};

// The wavefronts' lists in shared memory: each key that is among the k best goes to its rank (keys differ: each holds its
// place in the row).  k <= 64 and at most 16 lists: at most 1024 comparisons a thread, all reading one address.
template <int THREADS, typename F>
__device__ __forceinline__ void write_best(const unsigned long long* lists, int n, int k, const F& write) {
  for (int q = threadIdx.x; q < n; q += THREADS) {
    const unsigned long long mine = lists[q];
    if (mine == 0) continue;
    int rank = 0;
    for (int r = 0; r < n; ++r) rank += lists[r] > mine;
    if (rank < k) write(rank, mine);
  }
}

// A masked class (-inf) is no key: a row with fewer than k others has its lowest masked classes behind them, which one
// wavefront looks for from the row's beginning -- at most 2 k elements on.
template <typename T, typename F>
__device__ __forceinline__ void fill_masked(const T* x, int64_t classes, int have, int k, const F& write) {
  const int lane = threadIdx.x & 63;
  for (int64_t b = 0; have < k && b < classes; b += 64) {
    const bool in = b + lane < classes && (float)x[b + lane] == -__builtin_inff();
    const unsigned long long who = __ballot(in);
    const int rank = have + __popcll(who & ((1ull << lane) - 1));
    if (in && rank < k) write(rank, make_key(-__builtin_inff(), (unsigned)(b + lane)));
    have += __popcll(who);
  }
}

constexpr int FEW = 1024;  // keys that are ranked as they are
constexpr int UNROLL = 4;  // packs of a lane in flight

// WAVES wavefronts walk [from, to) of a row together (WAVES = 1: four rows a workgroup, a wavefront each).
// split > 1: a row is walked by `split` workgroups, whose triples and keys go to `part` for logprob_join_kernel.
template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void logprob_row_kernel(const T* __restrict__ logits, int64_t rows,
                                                                                    int64_t classes, int64_t stride, int split,
                                                                                    int64_t span, float* __restrict__ part,
                                                                                    unsigned long long* __restrict__ part_keys,
                                                                                    Out o) {
  constexpr int W = 16 / (int)sizeof(T);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int64_t row;
  int s = 0;
  if constexpr (WAVES == 1) {
    row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= rows) return;
  } else {
    row = blockIdx.x / (unsigned)split;
    s = (int)(blockIdx.x % (unsigned)split);
  }
  const int64_t from = s * span, to = from + span < classes ? from + span : classes;
  const T* x = logits + row * stride;
  const int64_t packs = (to - from) / W;
  const int first = WAVES == 1 ? 0 : wave * 64;
  Stat a;
  Best best;
  __shared__ unsigned reached[64];
  for (int64_t c0 = 0; c0 < packs; c0 += (int64_t)WAVES * 64 * UNROLL) {
    const int64_t c = c0 + first;
    Pack<T, W> p[UNROLL];
    float top = a.m;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t i = c + (int64_t)u * WAVES * 64 + lane;
      if (i < packs) p[u] = load_pack<T, W>(x + from + i * W);
      else
#pragma unroll
        for (int j = 0; j < W; ++j) p[u].v[j] = (T)-__builtin_inff();
    }
    float high[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      high[u] = (float)p[u].v[0];
#pragma unroll
      for (int j = 1; j < W; ++j) high[u] = __builtin_elementwise_maximum(high[u], (float)p[u].v[j]);  // (NaN stays)
      top = fmaxf(top, high[u]);
    }
    a.raise(top);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int j = 0; j < W; ++j) a.add((float)p[u].v[j]);
    if constexpr (TOP) {
      if (c0 == 0) {
        // A bound from the first block, which k elements reach: the k-th greatest of every wavefront's greatest few lanes.
        // Of a block of 16384 some 25 reach it then, where each wavefront alone would collect 98 of its 1024 for a list
        // of 20, and each costs what reading 150 cost (one row of 50001, the best 20: 11.8 us, 18.2 us without; 67 rows
        // of 131072: 16.3 + 4.1 us, 28 + 6 us without).
        float most = high[0];
#pragma unroll
        for (int u = 1; u < UNROLL; ++u) most = __builtin_elementwise_maximum(most, high[u]);  // (packs that are not there are -inf)
        if constexpr (WAVES == 1) {
          best.seed(Best::of_lanes(Best::upper(most), o.k));
        } else {
          constexpr int EACH = 64 / WAVES;
          const int whole = packs / 64 < WAVES ? (int)(packs / 64) : WAVES;  // wavefronts with a pack for every lane
          if (whole * EACH >= o.k) {
            const unsigned mine = Best::upper(most), t = Best::of_lanes(mine, EACH);
            const unsigned long long in = __ballot(mine >= t);
            const int rank = __popcll(in & ((1ull << lane) - 1));
            if (mine >= t && rank < EACH) reached[wave * EACH + rank] = mine;  // (t = 0: zeros among them)
            __syncthreads();
            best.seed(Best::of_lanes(lane < whole * EACH ? reached[lane] : 0u, o.k));
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int64_t i = c + (int64_t)u * WAVES * 64 + lane;
        if (__ballot(i < packs && !(high[u] < best.floor) && high[u] != -__builtin_inff())) {  // (equal: a lower place may come in)
#pragma unroll
          for (int j = 0; j < W; ++j)
            best.offer(i < packs ? offered((float)p[u].v[j], (unsigned)(from + i * W + j)) : 0ull, o.k);
        }
      }
    }
  }
  {  // the elements behind the last whole pack: the first wavefront's
    const int64_t i = from + packs * W + lane;
    if (first == 0) {
      const bool in = lane < W && i < to;
      const float v = in ? (float)x[i] : 0.f;
      if (in) {
        a.raise(fmaxf(a.m, v));
        a.add(v);
      }
      if constexpr (TOP) best.offer(in ? offered(v, (unsigned)i) : 0ull, o.k);
    }
  }
  join_lanes<64>(a);
  if constexpr (WAVES == 1) {
    float m = 0.f, ls = 0.f;
    if (lane == 0) finish_row(a, row, x, classes, o, m, ls);
    if constexpr (TOP) {
      m = __shfl(m, 0);
      ls = __shfl(ls, 0);
      const auto write = [&](int rank, unsigned long long mine) {
        o.top_lp[row * o.k + rank] = top_value(unord((unsigned)(mine >> 32)), m, ls);
        o.top_ix[row * o.k + rank] = (int64_t)(unsigned)~(unsigned)mine;
      };
      if (lane < o.k && best.key != 0) write(lane, best.key);
      fill_masked(x, classes, __popcll(__ballot(lane < o.k && best.key != 0)), o.k, write);
    }
  } else {
    __shared__ float sh[WAVES][3];
    __shared__ float done[2];
    __shared__ unsigned long long keys[TOP ? WAVES * TOP_MAX : 1];
    __shared__ int lists[WAVES];
    if (lane == 0) sh[wave][0] = a.m, sh[wave][1] = a.s, sh[wave][2] = a.t;
    const unsigned long long kept = TOP ? __ballot(lane < o.k && best.key != 0) : 0;  // (the first of the lanes)
    if (TOP && lane == 0) lists[wave] = __popcll(kept);
    __syncthreads();
    int many = 0;
    if constexpr (TOP) {
      int before = 0;
      for (int w = 0; w < WAVES; ++w) {
        before += w < wave ? lists[w] : 0;
        many += lists[w];
      }
      if (kept >> lane & 1) keys[before + lane] = best.key;
    }
    if (threadIdx.x == 0) {
      for (int w = 1; w < WAVES; ++w) a.join(sh[w][0], sh[w][1], sh[w][2]);
      if (split > 1) {
        float* q = part + 3 * (row * split + s);
        q[0] = a.m, q[1] = a.s, q[2] = a.t;
      } else {
        float m, ls;
        finish_row(a, row, x, classes, o, m, ls);
        done[0] = m, done[1] = ls;
      }
    }
    if constexpr (TOP) {
      __syncthreads();
      const auto write = [&](int rank, unsigned long long mine) {
        if (split > 1) part_keys[(row * split + s) * o.k + rank] = mine;
        else {
          o.top_lp[row * o.k + rank] = top_value(unord((unsigned)(mine >> 32)), done[0], done[1]);
          o.top_ix[row * o.k + rank] = (int64_t)(unsigned)~(unsigned)mine;
        }
      };
      write_best<WAVES * 64>(keys, many, o.k, write);
      if (split > 1) {
        if ((int)threadIdx.x < o.k && (int)threadIdx.x >= many) write(threadIdx.x, 0ull);
      } else if (wave == 0) {
        fill_masked(x, classes, many, o.k, write);
      }
    }
  }
}

// The parts of one row a workgroup: the triples in a fixed order; the keys by rank.  A key of 0: none.
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void logprob_join_kernel(const T* __restrict__ logits, int64_t rows, int64_t classes,
                                                           int64_t stride, int split, const float* __restrict__ part,
                                                           const unsigned long long* __restrict__ part_keys, Out o) {
  __shared__ float done[2];
  const int64_t row = blockIdx.x;
  if (threadIdx.x < 64) {
    Stat a;
    for (int s = threadIdx.x; s < split; s += 64) {
      const float* q = part + 3 * (row * split + s);
      a.join(q[0], q[1], q[2]);
    }
    join_lanes<64>(a);
    if (threadIdx.x == 0) {
      float m, ls;
      finish_row(a, row, logits + row * stride, classes, o, m, ls);
      done[0] = m, done[1] = ls;
    }
  }
  if constexpr (TOP) {
    __shared__ unsigned long long lists[FEW];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = split * o.k;
    const unsigned long long* keys = part_keys + row * n;
    int many = n;
    if (n <= FEW) {
      for (int q = threadIdx.x; q < n; q += 256) lists[q] = keys[q];
    } else {  // through four wavefronts' lists
      Best best;
      for (int q = wave * 64; q < n; q += 256) best.offer(q + lane < n ? keys[q + lane] : 0ull, o.k);
      if (lane < o.k) lists[wave * o.k + lane] = best.key;
      many = 4 * o.k;
    }
    __syncthreads();
    const auto write = [&](int rank, unsigned long long mine) {
      o.top_lp[row * o.k + rank] = top_value(unord((unsigned)(mine >> 32)), done[0], done[1]);
      o.top_ix[row * o.k + rank] = (int64_t)(unsigned)~(unsigned)mine;
    };
    write_best<256>(lists, many, o.k, write);
    if (wave == 0) {  // (every list is sorted, its empty places behind)
      int have = 0;
      for (int q = lane; q < many; q += 64) have += lists[q] != 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) have += __shfl_xor(have, d);
      fill_masked(logits + row * stride, classes, have, o.k, write);
    }
  }
}

// LANES lanes walk a row's segment; the gradient's own pack holds what a lane read, so a row is read once and written once.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void logprob_row_backward_kernel(const T* __restrict__ logits, int64_t rows, int64_t classes,
                                                                   int64_t stride, int split, int64_t span, Out o,
                                                                   const float* __restrict__ d_lp,
                                                                   const float* __restrict__ d_h,
                                                                   const float* __restrict__ d_top, T* __restrict__ dx) {
  constexpr int W = 16 / (int)sizeof(T), ROWS = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t row = (int64_t)(blockIdx.x / (unsigned)split) * ROWS + threadIdx.x / LANES;
  const int s = (int)(blockIdx.x % (unsigned)split);
  if (row >= rows) return;
  const int64_t from = s * span, to = from + span < classes ? from + span : classes;
  const T* x = logits + row * stride;
  T* out = dx + row * classes;
  const float m = o.stats[2 * row], ls = o.stats[2 * row + 1];
  const bool empty = ls == -__builtin_inff();
  int64_t y = -1;
  float dl = 0.f, sum = 0.f, dh = 0.f, h = 0.f;
  if (d_lp) {
    y = o.labels[row];
    dl = d_lp[row];
    if (o.has_ignore && y == o.ignore) y = -1, dl = 0.f;
    else if (y < 0 || y >= classes) y = -1, dl = __uint_as_float(0x7fc00000u);
    sum = dl;
  }
  if (d_h) dh = d_h[row], h = o.entropy[row];
  if (d_top)
    for (int k = 0; k < o.k; ++k) sum += d_top[row * o.k + k];
  const auto one = [&](float v, int64_t at, float more) {
    const float lp = (v - m) - ls, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    const float r = (at == y ? dl : 0.f) - p * (sum + dh * (fmaxf(lp, -150.f) + h)) + more;
    return (T)(empty ? 0.f : r);
  };
  const int64_t packs = (to - from) / W;
  for (int64_t c = lane; c < packs; c += LANES * UNROLL) {
    Pack<T, W> p[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (c + u * LANES < packs) p[u] = load_pack<T, W>(x + from + (c + u * LANES) * W);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (c + u * LANES < packs) {
        const int64_t at = from + (c + u * LANES) * W;
#pragma unroll
        for (int j = 0; j < W; ++j) p[u].v[j] = one((float)p[u].v[j], at + j, 0.f);
        __builtin_memcpy(out + at, &p[u], sizeof(p[u]));
      }
  }
  const int64_t i = from + packs * W + lane;
  if (i < to) out[i] = one((float)x[i], i, 0.f);  // (LANES >= W: one round)
  if (d_top) {  // the best alternatives' own, written again behind the others (4096 x 65536, 8 of them: 1160 us looked for at
                // every element, 394 so, 384 without any)
    if constexpr (LANES == 256) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    for (int k = lane; k < o.k; k += LANES) {
      const int64_t at = o.top_ix[row * o.k + k];
      if (at >= from && at < to) out[at] = one((float)x[at], at, d_top[row * o.k + k]);
    }
  }
}

// ---------------------------------------------------------------------------------------------- launches
// Rows of up to SMALL_MAX classes stay in registers (50000 x 128: 9.6 us, 29.6 if a wavefront walks each); up to WAVE_MAX a
// wavefront walks one (300 x 4000 with the best eight: 13.8 us so, 9.1 by four or sixteen; 8000 x 1000: 17); longer ones
// four wavefronts, or sixteen where those are a workgroup a compute unit at most (67 x 131072 with the best twenty: 34 and
// 22 us; 8000 x 16000: 100 and 151).  A row is split where rows are fewer than compute units, into parts of PART at least
// (one row of 1000000 with the best eight: 93 us whole, 19 so, 66 in parts of 8192, whose lists are many).
constexpr int SMALL_MAX = 128, WAVE_MAX = 1024;
constexpr int64_t PART = 32768;

int row_split(int64_t rows, int64_t classes) {
  if (classes <= WAVE_MAX) return 1;
  int64_t s = r3_cu_count() / rows;
  if (s > classes / PART) s = classes / PART;
  return s < 1 ? 1 : (s > 256 ? 256 : (int)s);
}
int64_t row_span(int64_t classes, int split) {  // (whole packs of 8)
  return ((classes + split - 1) / split + 7) / 8 * 8;
}

template <typename T, int LANES, int E>
int small_forward(const T* x, int64_t rows, int classes, int64_t stride, const Out& o, hipStream_t st) {
  const int64_t blocks = (rows * LANES + 255) / 256;
  if (blocks > 0x7fffffff) return -1;
  const int w = E * (int)sizeof(T) < 16 ? E : 16 / (int)sizeof(T);
  const bool vec = classes % w == 0;
  const dim3 g((unsigned)blocks), b(256);
  if (vec) {
    if (o.k) hipLaunchKernelGGL((logprob_small_kernel<T, LANES, E, true, true>), g, b, 0, st, x, rows, classes, stride, o);
    else hipLaunchKernelGGL((logprob_small_kernel<T, LANES, E, true, false>), g, b, 0, st, x, rows, classes, stride, o);
  } else {
    if (o.k) hipLaunchKernelGGL((logprob_small_kernel<T, LANES, E, false, true>), g, b, 0, st, x, rows, classes, stride, o);
    else hipLaunchKernelGGL((logprob_small_kernel<T, LANES, E, false, false>), g, b, 0, st, x, rows, classes, stride, o);
  }
  return hipGetLastError() == hipSuccess ? 0 : -2;
}
template <typename T, int LANES, int E>
int small_backward(const T* x, int64_t rows, int classes, int64_t stride, const Out& o, const float* d_lp, const float* d_h,
                   const float* d_top, T* dx, hipStream_t st) {
  const int64_t blocks = (rows * LANES + 255) / 256;
  if (blocks > 0x7fffffff) return -1;
  const int w = E * (int)sizeof(T) < 16 ? E : 16 / (int)sizeof(T);
  const dim3 g((unsigned)blocks), b(256);
  if (classes % w == 0)
    hipLaunchKernelGGL((logprob_small_backward_kernel<T, LANES, E, true>), g, b, 0, st, x, rows, classes, stride, o, d_lp, d_h,
                       d_top, dx);
  else
    hipLaunchKernelGGL((logprob_small_backward_kernel<T, LANES, E, false>), g, b, 0, st, x, rows, classes, stride, o, d_lp, d_h,
                       d_top, dx);
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

template <typename T, int WAVES>
int row_forward(const T* x, int64_t rows, int64_t classes, int64_t stride, int split, float* part, unsigned long long* keys,
                const Out& o, hipStream_t st) {
  const int64_t blocks = WAVES == 1 ? (rows + 3) / 4 : rows * split;
  if (blocks > 0x7fffffff) return -1;
  const dim3 g((unsigned)blocks), b(WAVES == 1 ? 256 : WAVES * 64);
  const int64_t span = row_span(classes, split);
  if (o.k)
    hipLaunchKernelGGL((logprob_row_kernel<T, WAVES, true>), g, b, 0, st, x, rows, classes, stride, split, span, part, keys, o);
  else
    hipLaunchKernelGGL((logprob_row_kernel<T, WAVES, false>), g, b, 0, st, x, rows, classes, stride, split, span, part, keys, o);
  if (hipGetLastError() != hipSuccess) return -2;
  if (split > 1) {
    if (o.k)
      hipLaunchKernelGGL((logprob_join_kernel<T, true>), dim3((unsigned)rows), dim3(256), 0, st, x, rows, classes, stride,
                         split, part, keys, o);
    else
      hipLaunchKernelGGL((logprob_join_kernel<T, false>), dim3((unsigned)rows), dim3(256), 0, st, x, rows, classes, stride,
                         split, part, keys, o);
    if (hipGetLastError() != hipSuccess) return -2;
  }
  return 0;
}

// A launch has fewer than 2^32 threads, and one of more is cut short without an error: of many rows so many are taken at a time
// (at 256 threads a row 2^30; the gradient's split rows take 256 more for every 16384 classes, which memory bounds).
constexpr int64_t ROWS = 1 << 22;

template <typename T>
int forward(const T* x, int64_t rows, int64_t classes, int64_t stride, int split, const Out& o, void* ws, hipStream_t st) {
  const int c = (int)classes;
  if (c <= 4) return small_forward<T, 1, 4>(x, rows, c, stride, o, st);
  if (c <= 16) return small_forward<T, 2, 8>(x, rows, c, stride, o, st);
  if (c <= 32) return small_forward<T, 4, 8>(x, rows, c, stride, o, st);
  if (c <= 64) return small_forward<T, 4, 16>(x, rows, c, stride, o, st);
  if (c <= SMALL_MAX) return small_forward<T, 8, 16>(x, rows, c, stride, o, st);
  if (c <= WAVE_MAX) return row_forward<T, 1>(x, rows, classes, stride, 1, nullptr, nullptr, o, st);
  unsigned long long* keys = static_cast<unsigned long long*>(ws);
  float* part = reinterpret_cast<float*>(keys + (size_t)rows * split * o.k);
  if (rows * split <= r3_cu_count()) return row_forward<T, 16>(x, rows, classes, stride, split, part, keys, o, st);
  return row_forward<T, 4>(x, rows, classes, stride, split, part, keys, o, st);
}

template <typename T>
int backward(const T* x, int64_t rows, int64_t classes, int64_t stride, const Out& o, const float* d_lp, const float* d_h,
             const float* d_top, T* dx, hipStream_t st) {
  const int c = (int)classes;
  if (c <= 4) return small_backward<T, 1, 4>(x, rows, c, stride, o, d_lp, d_h, d_top, dx, st);
  if (c <= 16) return small_backward<T, 4, 4>(x, rows, c, stride, o, d_lp, d_h, d_top, dx, st);
  if (c <= 32) return small_backward<T, 8, 4>(x, rows, c, stride, o, d_lp, d_h, d_top, dx, st);
  if (c <= 64) return small_backward<T, 8, 8>(x, rows, c, stride, o, d_lp, d_h, d_top, dx, st);
  if (c <= SMALL_MAX) return small_backward<T, 16, 8>(x, rows, c, stride, o, d_lp, d_h, d_top, dx, st);
  if (c <= WAVE_MAX) {
    const int64_t blocks = (rows + 3) / 4;
    if (blocks > 0x7fffffff) return -1;
    hipLaunchKernelGGL((logprob_row_backward_kernel<T, 64>), dim3((unsigned)blocks), dim3(256), 0, st, x, rows, classes, stride,
                       1, classes, o, d_lp, d_h, d_top, dx);
  } else {
    int64_t split = (classes + 16383) / 16384;
    if (rows * split > 0x7fffffff) split = 1;
    if (rows > 0x7fffffff) return -1;
    hipLaunchKernelGGL((logprob_row_backward_kernel<T, 256>), dim3((unsigned)(rows * split)), dim3(256), 0, st, x, rows,
                       classes, stride, (int)split, row_span(classes, (int)split), o, d_lp, d_h, d_top, dx);
  }
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

}  // namespace

size_t r3k_logprob_workspace_bytes(int64_t rows, int64_t classes, int k) {
  if (rows <= 0 || classes <= WAVE_MAX) return 0;
  const int split = row_split(rows, classes);
  return split == 1 ? 0 : (size_t)rows * split * (3 * sizeof(float) + k * sizeof(unsigned long long));
}

int r3k_logprob(const void* x, int dtype, int64_t rows, int64_t classes, int64_t stride, const int64_t* labels, int64_t ignore,
                int has_ignore, int k, float* log_prob, float* entropy, float* top_lp, int64_t* top_ix, float* stats, void* ws,
                size_t ws_bytes, hipStream_t st) {
  if (rows < 0 || classes < 1 || classes > 0x7fffffff || k < 0 || k > TOP_MAX || k > classes || dtype < 0 || dtype > 2) return -1;
  if (rows == 0) return 0;
  if (rows > (1ll << 40) || !x || stride < 0 || (labels && !log_prob) || (k && (!top_lp || !top_ix))) return -1;
  const size_t need = r3k_logprob_workspace_bytes(rows, classes, k);
  if (need && (!ws || ws_bytes < need)) return -3;
  if (need && (reinterpret_cast<uintptr_t>(ws) & 7)) return -1;
  const int split = row_split(rows, classes);  // (of the whole call: the last few rows of many have no workspace)
  const Out all{labels, ignore, has_ignore, k, log_prob, entropy, top_lp, top_ix, stats};
  for (int64_t at = 0; at < rows; at += ROWS) {
    const int64_t n = rows - at < ROWS ? rows - at : ROWS;
    const Out o = all.from(at);
    const auto run = [&](auto type) { return forward(static_cast<const decltype(type)*>(x) + at * stride, n, classes, stride, split, o, ws, st); };
    const int rc = dtype == 0 ? run(0.f) : dtype == 1 ? run((_Float16)0) : run((__bf16)0);
    if (rc != 0) return rc;
  }
  return 0;
}

int r3k_logprob_backward(const void* x, int dtype, int64_t rows, int64_t classes, int64_t stride, const int64_t* labels,
                         int64_t ignore, int has_ignore, int k, const float* stats, const float* entropy,
                         const int64_t* top_ix, const float* d_lp, const float* d_h, const float* d_top, void* dx,
                         hipStream_t st) {
  if (rows < 0 || classes < 1 || classes > 0x7fffffff || k < 0 || k > TOP_MAX || k > classes || dtype < 0 || dtype > 2) return -1;
  if (rows == 0) return 0;
  if (rows > (1ll << 40) || !x || stride < 0 || !stats || !dx || (d_lp && !labels) || (d_h && !entropy) || (d_top && (!k || !top_ix)))
    return -1;
  const Out all{labels, ignore, has_ignore, k, nullptr, const_cast<float*>(entropy), nullptr, const_cast<int64_t*>(top_ix),
                const_cast<float*>(stats)};
  for (int64_t at = 0; at < rows; at += ROWS) {
    const int64_t n = rows - at < ROWS ? rows - at : ROWS;
    const Out o = all.from(at);
    const float *lp = d_lp ? d_lp + at : nullptr, *h = d_h ? d_h + at : nullptr, *top = d_top ? d_top + at * k : nullptr;
    const auto run = [&](auto type) {
      typedef decltype(type) T;
      return backward(static_cast<const T*>(x) + at * stride, n, classes, stride, o, lp, h, top, static_cast<T*>(dx) + at * classes, st);
    };
    const int rc = dtype == 0 ? run(0.f) : dtype == 1 ? run((_Float16)0) : run((__bf16)0);
    if (rc != 0) return rc;
  }
  return 0;
}
