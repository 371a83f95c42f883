// Expert selection with a balancing bias and expert groups, forward and backward.
//
//   s_e = softmax(x)_e or sigmoid(x_e),   c_e = s_e + bias_e   (the bias takes part in the choice only)
//   a group's value is the sum of its two largest c; the best `top_groups` groups stay
//   the top_k largest c of those groups are chosen, w_i = scale * s_i / ||s_chosen||_p  (p = 0: not divided)
//   scores_e = s_e / sum_e s_e   (for the softmax that is s_e itself)
//
// One warp owns a token and holds its experts in registers, PL consecutive ones a lane, fetched V at a time.
// A lane with up to eight sorts them once, as keys whose last three bits are the place, and a round of the
// choice is one reduction of the lanes' heads (1678 instructions a token with the places compared anew in every
// round).  FULL: the experts fill all places of all lanes.
//
// The order of the experts is exact: equal values go to the lowest id, and values that 32 bits cannot tell
// apart are ordered by their 64-bit ones.  Without a bias the scores have the order of the logits, which are
// compared as they are.  Each comparison that decides (neighbours in the chosen order, the last chosen one
// and the next, the last group that stays and the next) is checked against a bound of the arithmetic's error; in a
// token with a closer pair, a few in a thousand, what is in question is ordered in 64 bits.  That path is kept
// short, as the last token's latency is the launch's: with all of the choice redone a launch of 37 us ended 13 us
// later for five tokens with close groups.
//
// 32768 x 256 bf16 in 8 groups, sigmoid and bias: 39 us (36 MB, 0.14 of the copy bandwidth), bound by
// instructions, 900 a token, of which 0.84 a cycle and scheduler are issued.  Backward from the weights alone 12 us:
// the chosen logits' sectors, ids, gradients and the rows written are 28 MB, 0.37 of the copy bandwidth; its loads
// wait for the ids (11 of 17 cycles between a warp's instructions).
#include "common.cuh"

namespace mb {

namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Unsigned key in the order of the floats; NaN counts as +infinity, -0 as 0.  0 is below every key.
__device__ __forceinline__ unsigned ordered(float v) {
  unsigned u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) u = 0x7f800000u;
  if (u == 0x80000000u) u = 0u;
  return u ^ (unsigned(int(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// The value of a key that has lost its last bits: without them that of -infinity, 0x007fffff, is a NaN's.
__device__ __forceinline__ float value_of(unsigned key) { return from_ordered(max(key, 0x007fffffu)); }

// Experts of a lane: PL consecutive ones, so that a lower lane has lower ids.
template <int PL>
__device__ __forceinline__ int expert_of(int j, int lane) {
  return lane * PL + j;
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Slots {
  T v[V];
};

template <typename T, int PL, int V, bool FULL>
__device__ __forceinline__ void load_slots(const T* row, int lane, int experts, float fill, float (&x)[PL]) {
#pragma unroll
  for (int j = 0; j < PL; j += V) {
    const int e = expert_of<PL>(j, lane);
    if (FULL || e < experts) {  // experts % V == 0
      const Slots<T, V> p = *reinterpret_cast<const Slots<T, V>*>(row + e);
#pragma unroll
      for (int k = 0; k < V; ++k) x[j + k] = to_float(p.v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) x[j + k] = fill;
    }
  }
}

template <typename T, int PL, int V, bool FULL>
__device__ __forceinline__ void store_slots(T* row, int lane, int experts, const float (&x)[PL]) {
#pragma unroll
  for (int j = 0; j < PL; j += V) {
    const int e = expert_of<PL>(j, lane);
    if (FULL || e < experts) {
      Slots<T, V> p;
#pragma unroll
      for (int k = 0; k < V; ++k) p.v[k] = from_float<T>(x[j + k]);
      *reinterpret_cast<Slots<T, V>*>(row + e) = p;
    }
  }
}

__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(float x) { return reciprocal(1.f + __expf(-x)); }

// Scores of a lane's slots; returns what a single score needs to be taken again (maximum and inverse sum
// of the softmax) and the sum of all scores.
struct RowStat {
  float top, inv, total;
};

template <int PL, bool FULL>
__device__ __forceinline__ RowStat scores_of(const float (&x)[PL], int lane, int experts, bool use_sigmoid,
                                             float (&s)[PL]) {
  RowStat r{0.f, 1.f, 0.f};
  float sum = 0.f;
  if (use_sigmoid) {
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      s[j] = sigmoid(x[j]);
      if (!FULL && expert_of<PL>(j, lane) >= experts) s[j] = 0.f;
      sum += s[j];
    }
    r.total = warp_sum_f(sum);
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < PL; ++j) top = fmaxf(top, x[j]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    r.top = top == -INFINITY ? 0.f : top;         // nothing but -inf: every score is zero
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      s[j] = __expf(x[j] - r.top);
      if (!FULL && expert_of<PL>(j, lane) >= experts) s[j] = 0.f;
      sum += s[j];
    }
    sum = warp_sum_f(sum);
    r.inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < PL; ++j) s[j] *= r.inv;
    r.total = sum == 0.f ? 0.f : 1.f;
  }
  return r;
}

__device__ __forceinline__ float score_at(float x, const RowStat& r, bool use_sigmoid) {
  return use_sigmoid ? sigmoid(x) : __expf(x - r.top) * r.inv;
}

// ---- the choice in 64 bits: lane i returns the i-th expert ---------------------------------------------
__device__ __forceinline__ double key64(double v) { return v != v ? INFINITY : v; }

// What a choice goes by, in 64 bits, into c.
template <typename T>
__device__ __forceinline__ void choice_wide(const T* row, const SelectArgs& a, double* c, int lane) {
  const int E = a.experts;
  double top = -INFINITY, sum = 0.;
  if (!a.use_sigmoid) {
    for (int e = lane; e < E; e += 32) top = fmax(top, double(to_float(row[e])));
    for (int d = 16; d > 0; d >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (top == -INFINITY) top = 0.;
  }
#pragma unroll 4
  for (int e = lane; e < E; e += 32) {
    const double x = to_float(row[e]);
    c[e] = a.use_sigmoid ? 1. / (1. + exp(-x)) : exp(x - top);
    sum += c[e];
  }
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  for (int e = lane; e < E; e += 32) {
    const double s = a.use_sigmoid ? c[e] : (sum == 0. ? 0. : c[e] / sum);
    c[e] = key64(a.bias != nullptr ? s + double(a.bias[e]) : s);
  }
  __syncwarp();
}

// The groups that stay, as choose_groups returns them.
template <typename T>
__device__ __noinline__ unsigned groups_wide(const T* row, const SelectArgs& a, double* c, int shift, int lane) {
  choice_wide(row, a, c, lane);
  const int g = lane >> shift, size = a.group_size;
  double b1 = -INFINITY, b2 = -INFINITY;
  if (g < a.groups) {
    for (int i = lane & ((1 << shift) - 1); i < size; i += 1 << shift) {
      const double v = c[g * size + i];
      b2 = fmax(b2, fmin(b1, v));
      b1 = fmax(b1, v);
    }
  }
  for (int d = 1 << shift >> 1; d > 0; d >>= 1) {
    const double o1 = __shfl_xor_sync(0xffffffffu, b1, d), o2 = __shfl_xor_sync(0xffffffffu, b2, d);
    b2 = fmax(fmin(b1, o1), fmax(b2, o2));
    b1 = fmax(b1, o1);
  }
  const double value = key64(size > 1 ? b1 + b2 : b1);
  int rank = 0;
  for (int h = 0; h < a.groups; ++h) {
    const double o = __shfl_sync(0xffffffffu, value, h << shift);
    rank += o > value || (o == value && h < g);
  }
  return __ballot_sync(0xffffffffu, g < a.groups && rank < a.top_groups);
}

template <typename T>
__device__ __noinline__ int choose_wide(const T* row, const SelectArgs& a, double* c, int lane) {
  const int E = a.experts;
  choice_wide(row, a, c, lane);
  unsigned kept = 0xffffffffu;
  const int size = a.group_size;
  if (a.top_groups < a.groups) {
    double value = -INFINITY;
    if (lane < a.groups) {
      double b1 = -INFINITY, b2 = -INFINITY;
      for (int i = 0; i < size; ++i) {
        const double v = c[lane * size + i];
        if (v > b1) { b2 = b1; b1 = v; } else if (v > b2) { b2 = v; }
      }
      value = key64(size > 1 ? b1 + b2 : b1);
    }
    int rank = 0;
    for (int h = 0; h < a.groups; ++h) {
      const double o = __shfl_sync(0xffffffffu, value, h);
      rank += o > value || (o == value && h < lane);
    }
    kept = __ballot_sync(0xffffffffu, lane < a.groups && rank < a.top_groups);
    __syncwarp();
  }
  // Lane's experts are lane, lane + 32, ...: at most 32 of them, the taken ones a bit each.
  unsigned gone = 0u;
  int mine = 0;
  for (int i = 0; i < a.top_k; ++i) {
    double best = -INFINITY;
    int at = 0x7fffffff;
    for (int e = lane, n = 0; e < E; e += 32, ++n) {
      if ((gone >> n & 1u) || !(kept >> (e / size) & 1u)) continue;
      const double v = a.bias != nullptr ? c[e] : key64(double(to_float(row[e])));
      if (at == 0x7fffffff || v > best) { best = v; at = e; }
    }
    for (int d = 16; d > 0; d >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, best, d);
      const int oe = __shfl_xor_sync(0xffffffffu, at, d);
      if (oe != 0x7fffffff && (at == 0x7fffffff || ov > best || (ov == best && oe < at))) { best = ov; at = oe; }
    }
    if ((at & 31) == lane) gone |= 1u << (at >> 5);
    if (lane == i) mine = at;
  }
  return mine;
}

// The order in 64 bits of the n experts that lanes hold, no others being in question: lane i returns the i-th.  Takes
// a tenth of the time of the choice from all, which at the end of a launch every SM waits for.
template <typename T>
__device__ __noinline__ int order_wide(const T* row, const SelectArgs& a, float top, int mine, int n, int lane) {
  double sum = 0.;
  if (a.bias != nullptr && !a.use_sigmoid) {
    for (int e = lane; e < a.experts; e += 32) sum += exp(double(to_float(row[e])) - double(top));
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  }
  double c = -INFINITY;
  if (lane < n) {
    c = to_float(row[mine]);
    if (a.bias != nullptr) {
      if (a.use_sigmoid) c = 1. / (1. + exp(-c));
      else c = sum == 0. ? 0. : exp(c - double(top)) / sum;
      c += double(a.bias[mine]);
    }
    c = key64(c);
  }
  int rank = 0, sorted = 0;
  for (int i = 0; i < n; ++i) {
    const double o = __shfl_sync(0xffffffffu, c, i);
    const int e = __shfl_sync(0xffffffffu, mine, i);
    rank += o > c || (o == c && e < mine);
  }
  for (int i = 0; i < n; ++i) {
    const int at = __shfl_sync(0xffffffffu, rank, i), e = __shfl_sync(0xffffffffu, mine, i);
    if (at == lane) sorted = e;
  }
  return sorted;
}

__host__ __device__ constexpr int padded_slot(int e) { return e + (e >> 5) * 4; }

// Descending sort by a fixed network (Batcher's odd-even merge).
template <int N>
__device__ __forceinline__ void sort_down(unsigned (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const unsigned hi = max(k[i + j], k[i + j + q]), lo = min(k[i + j], k[i + j + q]);
            k[i + j] = hi;
            k[i + j + q] = lo;
          }
}

// The two largest of a group that spans 2^shift lanes, in all of them.
__device__ __forceinline__ void join_best(float& b1, float& b2, int shift) {
  for (int d = 1 << shift >> 1; d > 0; d >>= 1) {
    const float o1 = __shfl_xor_sync(0xffffffffu, b1, d), o2 = __shfl_xor_sync(0xffffffffu, b2, d);
    b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
    b1 = fmaxf(b1, o1);
  }
}

// Whether groups stay, as lane bits: bit g << shift.  `b1`, `b2`: the largest values of group lane >> shift.  The
// lanes of a group share its comparisons.  Sets `doubt` when the last group that stays and the next are closer
// than the arithmetic tells apart: the errors of two scores each, and of what makes up a sum, whose parts may be
// larger than the sum, 1.13 x 2^-19 of the largest (2^-20 x 0.88 for the keys' bits, 2^-24 for each rounding).
__device__ __forceinline__ unsigned choose_groups(float b1, float b2, int shift, const SelectArgs& a, int lane,
                                                  float margin, bool& doubt) {
  const int g = lane >> shift;
  const bool there = g < a.groups;
  const unsigned value = there ? ordered(a.group_size > 1 ? b1 + b2 : b1) : 0u;
  int rank = 0;
  for (int h = 0; h < a.groups; h += 1 << shift) {
    const int other = h + (lane & ((1 << shift) - 1));                // of another group's number
    const unsigned o = __shfl_sync(0xffffffffu, value, other << shift);
    rank += other < a.groups && (o > value || (o == value && other < g));
  }
  for (int d = 1 << shift >> 1; d > 0; d >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, d);
  const bool stays = there && rank < a.top_groups;
  const float last = from_ordered(__reduce_min_sync(0xffffffffu, stays ? value : 0xffffffffu));
  const float next = from_ordered(__reduce_max_sync(0xffffffffu, stays ? 0u : value));
  const float part = fmaxf(fabsf(b1) < INFINITY ? fabsf(b1) : 0.f, fabsf(b2) < INFINITY ? fabsf(b2) : 0.f);
  const float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, there ? __float_as_uint(part) : 0u));
  const float gap = last - next;
  doubt = !(gap > 2.f * margin + 0x1p-18f * largest || gap == INFINITY);
  return __ballot_sync(0xffffffffu, stays);
}

template <typename T, int PL, int V, bool FULL>
__global__ void __launch_bounds__(kWarps * 32)
select_fwd_kernel(const T* __restrict__ logits, const SelectArgs a, T* __restrict__ scores, T* __restrict__ weights,
                  int64_t* __restrict__ ids) {
  constexpr bool kSorted = PL <= 8;
  constexpr unsigned kPlace = kSorted ? 7u : 0u;          // key bits that hold 7 - place instead of value
  extern __shared__ double shared[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.experts;
  const int64_t t = int64_t(blockIdx.x) * kWarps + warp;
  if (t >= a.tokens) return;
  const T* row = logits + t * E;
  float x[PL], s[PL];
  load_slots<T, PL, V, FULL>(row, lane, E, -INFINITY, x);
  const RowStat r = scores_of<PL, FULL>(x, lane, E, a.use_sigmoid, s);
  {
    const float inv_total = a.use_sigmoid && r.total != 0.f ? reciprocal(r.total) : 1.f;
    float out[PL];
#pragma unroll
    for (int j = 0; j < PL; ++j) out[j] = s[j] * inv_total;
    store_slots<T, PL, V, FULL>(scores + t * E, lane, E, out);
  }

  // Twice the error of a score: exponent's rounding and unit, division, sum (1.6 x 2^-22 for the sigmoid,
  // 1.6 x 2^-20 of the largest for the softmax).  Where two values are compared, the rounding of the sum with the
  // bias and the bits that a key gives to the place come on top: 2^-20 of the values.
  const float margin = a.use_sigmoid ? 0x1p-20f : 0x1p-18f * r.inv;
  const bool biased = a.bias != nullptr;
  float* const mine_shared = reinterpret_cast<float*>(shared + warp * E);
  const bool grouped = a.top_groups < a.groups;
  bool doubt = false;
  unsigned key[PL];
  if (biased) {
    float add[PL];
    // 16-byte bias vectors; the launcher sees to the alignment where V > 1.
    load_slots<float, PL, (V > 4 ? 4 : V), FULL>(a.bias, lane, E, 0.f, add);
#pragma unroll
    for (int j = 0; j < PL; ++j) s[j] += add[j];
  }
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    const int e = expert_of<PL>(j, lane);
    const bool there = FULL || e < E;
    if (grouped && a.aligned_shift < 0 && there) mine_shared[padded_slot(e)] = s[j] != s[j] ? INFINITY : s[j];
    const unsigned k = (ordered(biased ? s[j] : x[j]) & ~kPlace) | (kPlace - (unsigned(j) & kPlace));
    key[j] = there ? k : 0u;
  }
  if constexpr (kSorted) sort_down(key);
  if (grouped) {
    float b1 = -INFINITY, b2 = -INFINITY;
    if (a.aligned_shift >= 0) {                           // groups of whole lanes, a power of two of them
      if (kSorted && biased) {                            // the places' bits are within what `doubt` allows
        b1 = value_of(key[0] & ~kPlace);
        if (PL > 1) b2 = value_of(key[PL > 1 ? 1 : 0] & ~kPlace);
      } else {
#pragma unroll
        for (int j = 0; j < PL; ++j) {
          const float v = FULL || expert_of<PL>(j, lane) < E ? (s[j] != s[j] ? INFINITY : s[j]) : -INFINITY;
          b2 = fmaxf(b2, fminf(b1, v));
          b1 = fmaxf(b1, v);
        }
      }
      join_best(b1, b2, a.aligned_shift);
      unsigned stays = choose_groups(b1, b2, a.aligned_shift, a, lane, margin, doubt);
      if (doubt) stays = groups_wide<T>(row, a, shared + warp * E, a.aligned_shift, lane);
      if (!(stays >> (lane >> a.aligned_shift << a.aligned_shift) & 1u)) {
#pragma unroll
        for (int j = 0; j < PL; ++j) key[j] = 0u;
      }
    } else {
      __syncwarp();
      const int shift = a.group_shift, g = lane >> shift;
      if (g < a.groups) {
        for (int i = lane & ((1 << shift) - 1); i < a.group_size; i += 1 << shift) {
          const float v = mine_shared[padded_slot(g * a.group_size + i)];
          b2 = fmaxf(b2, fminf(b1, v));
          b1 = fmaxf(b1, v);
        }
      }
      join_best(b1, b2, shift);
      unsigned stays = choose_groups(b1, b2, shift, a, lane, margin, doubt);
      if (doubt) {
        __syncwarp();                                     // the values in 32 bits have been read
        stays = groups_wide<T>(row, a, shared + warp * E, shift, lane);
      }
      const float inv_size = 1.f / float(a.group_size);
#pragma unroll
      for (int j = 0; j < PL; ++j) {
        const int place = kSorted ? int(kPlace - (key[j] & kPlace)) : j;
        const int g2 = int((lane * PL + place + 0.5f) * inv_size);           // exact: at most 1024 experts
        if (!(stays >> (g2 << shift & 31) & 1u)) key[j] = 0u;
      }
      if constexpr (kSorted) sort_down(key);
    }
  }

  // With values that a key does not hold exactly one expert more than is chosen: the last has to be told from
  // the next.
  const bool inexact = biased || (kSorted && sizeof(T) == 4);
  const int rounds = a.top_k + (inexact ? 1 : 0);
  int mine = 0;                        // lane i: the i-th choice and its key
  unsigned mine_key = 0u, next_key = 0u;                  // the last key taken
  auto take = [&](int i) {
    unsigned head;
    int at;
    if constexpr (kSorted) {
      head = key[0] & ~kPlace;
      at = lane * PL + int(kPlace - (key[0] & kPlace));
    } else {
      head = 0u;
      at = 0;
#pragma unroll
      for (int j = 0; j < PL; ++j)
        if (key[j] > head) { head = key[j]; at = expert_of<PL>(j, lane); }
    }
    const unsigned best = __reduce_max_sync(0xffffffffu, head);
    const int from = __ffs(__ballot_sync(0xffffffffu, head == best)) - 1;     // the lowest lane has the lowest id
    const int e = __shfl_sync(0xffffffffu, at, from);
    if (lane == i) { mine = e; mine_key = best; }
    next_key = best;
    if (lane == from) {
      if constexpr (kSorted) {
#pragma unroll
        for (int j = 0; j + 1 < PL; ++j) key[j] = key[j + 1];
        key[PL - 1] = 0u;
      } else {
#pragma unroll
        for (int j = 0; j < PL; ++j)
          if (expert_of<PL>(j, lane) == e) key[j] = 0u;
      }
    }
  };
  for (int i = 0; i < rounds; ++i) take(i);
  bool crowd = false;                                     // more than 31 experts come into question
  if (inexact) {                                          // all neighbours at once; a key of 0: no expert was left
    auto close_keys = [&](unsigned k, unsigned next) {
      if (!biased) return k == next;
      const float c = value_of(k), d = value_of(next), gap = c - d;
      return !(gap > margin + 0x1p-20f * fmaxf(fabsf(c), fabsf(d)) || gap == INFINITY);
    };
    const bool last = lane == a.top_k - 1;
    const unsigned down = __shfl_down_sync(0xffffffffu, mine_key, 1), next = last ? next_key : down;
    bool close = lane < a.top_k && next != 0u && close_keys(mine_key, next);
    if (__any_sync(0xffffffffu, close)) {
      // Experts that are alike in logit and bias are equal.  Not so behind the last choice, where others that are
      // as close may follow.
      const int other = __shfl_down_sync(0xffffffffu, mine, 1);
      if (close && !last)
        close = !(ordered(to_float(row[mine])) == ordered(to_float(row[other])) &&
                  (!biased || a.bias[mine] == a.bias[other]));
      if (__any_sync(0xffffffffu, close)) {
        // Those behind the last choice that are as close to it come into question too; others do not, as they
        // are further from all choices.
        const unsigned end = __shfl_sync(0xffffffffu, mine_key, a.top_k - 1);
        int n = a.top_k;
        while (n < 32 && next_key != 0u && close_keys(end, next_key)) take(++n);
        if (n < 32) mine = order_wide<T>(row, a, r.top, mine, n, lane);
        else crowd = true;
      }
    }
  }
  if (crowd) {
    __syncwarp();
    mine = choose_wide<T>(row, a, shared + warp * E, lane);
  }

  const bool live = lane < a.top_k;
  const float w = live ? score_at(to_float(row[mine]), r, a.use_sigmoid) : 0.f;
  float factor = a.scale;
  if (a.norm_p != 0) {
    const float acc = warp_sum_f(a.norm_p == 1 ? w : w * w);
    // Chosen scores that are all zero have zero weights.
    factor = acc == 0.f ? 0.f : a.scale / (a.norm_p == 1 ? acc : sqrtf(acc));
  }
  if (live) {
    weights[t * a.top_k + lane] = from_float<T>(w * factor);
    ids[t * a.top_k + lane] = mine;
  }
}

// dlogits from the gradients of the weights and (optionally) of the scores.  The scores are taken again
// from the logits, which costs the bytes that stored scores would and keeps their 32 bits.
template <typename T, int PL, int V, bool FULL>
__global__ void __launch_bounds__(kWarps * 32)
select_bwd_kernel(const T* __restrict__ logits, const SelectArgs a, const int64_t* __restrict__ ids,
                  const T* __restrict__ dscores, int64_t dscores_stride, const T* __restrict__ dweights,
                  T* __restrict__ dlogits) {
  const int lane = threadIdx.x & 31, E = a.experts;
  const int64_t t = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = logits + t * E;
  const bool live = lane < a.top_k;
  const int mine = live ? int(ids[t * a.top_k + lane]) : 0;
  const float dw = live && dweights != nullptr ? to_float(dweights[t * a.top_k + lane]) * a.scale : 0.f;
  const float mine_x = to_float(row[mine]);
  float x[PL], s[PL];
  RowStat r{0.f, 1.f, 0.f};
  const bool whole = !a.use_sigmoid || dscores != nullptr;      // more than the chosen experts' own logits
  if (whole) {
    load_slots<T, PL, V, FULL>(row, lane, E, -INFINITY, x);
    r = scores_of<PL, FULL>(x, lane, E, a.use_sigmoid, s);
  }
  const float w = live ? score_at(mine_x, r, a.use_sigmoid) : 0.f;
  float dsel = dw;
  if (a.norm_p != 0) {
    const float acc = warp_sum_f(a.norm_p == 1 ? w : w * w);
    const float dot = warp_sum_f(dw * w);
    const float inv = acc == 0.f ? 0.f : 1.f / (a.norm_p == 1 ? acc : sqrtf(acc));
    dsel = (dw - dot * inv * (a.norm_p == 1 ? 1.f : w * inv)) * inv;
  }
  if (!live) dsel = 0.f;
  float g[PL];
  float inner = 0.f, inv_total = 1.f;
  if (dscores != nullptr) {
    load_slots<T, PL, V, FULL>(dscores + t * dscores_stride, lane, E, 0.f, g);
#pragma unroll
    for (int j = 0; j < PL; ++j) inner += g[j] * s[j];
    if (a.use_sigmoid && r.total != 0.f) inv_total = 1.f / r.total;
  }
  // softmax: inner = <ds, s> with both gradients; sigmoid: <g, scores> of the scores' gradient alone.
  inner = a.use_sigmoid ? (dscores != nullptr ? warp_sum_f(inner) * inv_total : 0.f) : warp_sum_f(inner + dsel * w);
  T* out = dlogits + t * E;
  {
    float d[PL];
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      d[j] = 0.f;
      if (whole) {
        const float gs = dscores != nullptr ? g[j] : 0.f;
        d[j] = a.use_sigmoid ? (gs - inner) * inv_total * s[j] * sigmoid(-x[j]) : s[j] * (gs - inner);
      }
    }
    store_slots<T, PL, V, FULL>(out, lane, E, d);
  }
  __syncwarp();               // the chosen experts' values over the ones just stored
  if (live) {
    const float gs = dscores != nullptr ? to_float(dscores[t * dscores_stride + mine]) : 0.f;
    float d;
    if (a.use_sigmoid) d = ((dscores != nullptr ? (gs - inner) * inv_total : 0.f) + dsel) * w * sigmoid(-mine_x);
    else d = w * (gs + dsel - inner);
    out[mine] = from_float<T>(d);
  }
}

template <typename T, int V>
bool row_vectors(int experts, const void* p) {
  return experts % V == 0 && reinterpret_cast<uintptr_t>(p) % (V * sizeof(T)) == 0;
}

// PL slots a lane, fetched up to 16 bytes at a time where the rows allow it, else one by one.
#define MB_SELECT_ONE(PL, V, aligned, CALL)                               \
  if (!aligned(V)) { CALL(PL, 1, false); }                                \
  else if (a.experts == 32 * PL) { CALL(PL, V, true); }                   \
  else { CALL(PL, V, false); }
#define MB_SELECT_SWITCH(T, aligned, CALL)                                \
  constexpr int W = 16 / sizeof(T);                                       \
  if (a.experts <= 32) { CALL(1, 1, false); }                             \
  else if (a.experts <= 64) { MB_SELECT_ONE(2, 2, aligned, CALL) }        \
  else if (a.experts <= 128) { MB_SELECT_ONE(4, 4, aligned, CALL) }       \
  else if (a.experts <= 256) { MB_SELECT_ONE(8, W, aligned, CALL) }       \
  else if (a.experts <= 512) { MB_SELECT_ONE(16, W, aligned, CALL) }      \
  else { MB_SELECT_ONE(32, W, aligned, CALL) }

int ceil_log2(int n) {
  int bits = 0;
  while (1 << bits < n) ++bits;
  return bits;
}

bool complete(SelectArgs& a) {
  if (a.experts < 1 || a.experts > kRouterMaxExperts || a.top_k < 1 || a.top_k > kSelectMaxTopK) return false;
  if (a.groups < 1 || a.groups > kSelectMaxGroups || a.experts % a.groups != 0 || a.top_groups < 1 ||
      a.top_groups > a.groups || a.top_k > a.top_groups * (a.experts / a.groups) || a.norm_p < 0 || a.norm_p > 2)
    return false;
  a.group_size = a.experts / a.groups;
  a.group_shift = 0;
  while (2 << a.group_shift << ceil_log2(a.groups) <= 32) ++a.group_shift;
  // Lanes of a group where it takes whole ones, a power of two of them.
  const int per_lane = 1 << ceil_log2((a.experts + 31) / 32);
  const int span = a.group_size % per_lane == 0 ? a.group_size / per_lane : 0;
  a.aligned_shift = span > 0 && (span & (span - 1)) == 0 && span * a.groups <= 32 ? ceil_log2(span) : -1;
  return true;
}

}  // namespace

cudaError_t select_experts_fwd(DType type, const void* logits, SelectArgs a, void* scores, void* weights,
                               int64_t* ids, cudaStream_t stream) {
  if (!complete(a)) return cudaErrorInvalidValue;
  if (a.tokens == 0) return cudaSuccess;
  const size_t shared = size_t(a.experts) * kWarps * sizeof(double);       // at most 32 KB
  MB_SWITCH_FLOAT(type, T, {
#define MB_SELECT_ALIGNED(v)                                                                                     \
  (row_vectors<T, v>(a.experts, logits) && row_vectors<T, v>(a.experts, scores) &&                                \
   row_vectors<float, (v > 4 ? 4 : v)>(a.experts, a.bias))
#define MB_SELECT_FWD(PL, V, FULL)                                                                               \
  select_fwd_kernel<T, PL, V, FULL><<<ceil_div(a.tokens, kWarps), kWarps * 32, shared, stream>>>(                      \
      static_cast<const T*>(logits), a, static_cast<T*>(scores), static_cast<T*>(weights), ids)
    MB_SELECT_SWITCH(T, MB_SELECT_ALIGNED, MB_SELECT_FWD)
  })
#undef MB_SELECT_FWD
#undef MB_SELECT_ALIGNED
  return cudaGetLastError();
}

cudaError_t select_experts_bwd(DType type, const void* logits, SelectArgs a, const int64_t* ids, const void* dscores,
                               int64_t dscores_stride, const void* dweights, void* dlogits, cudaStream_t stream) {
  if (!complete(a)) return cudaErrorInvalidValue;
  if (a.tokens == 0) return cudaSuccess;
  MB_SWITCH_FLOAT(type, T, {
#define MB_SELECT_ALIGNED(v)                                                              \
  (row_vectors<T, v>(a.experts, logits) && row_vectors<T, v>(a.experts, dlogits) &&        \
   (dscores == nullptr || row_vectors<T, v>(a.experts, dscores)))
#define MB_SELECT_BWD(PL, V, FULL)                                                                               \
  select_bwd_kernel<T, PL, V, FULL><<<ceil_div(a.tokens, kWarps), kWarps * 32, 0, stream>>>(                           \
      static_cast<const T*>(logits), a, ids, static_cast<const T*>(dscores), dscores_stride,                     \
      static_cast<const T*>(dweights), static_cast<T*>(dlogits))
    MB_SELECT_SWITCH(T, MB_SELECT_ALIGNED, MB_SELECT_BWD)
  })
#undef MB_SELECT_BWD
#undef MB_SELECT_ALIGNED
  return cudaGetLastError();
}

}  // namespace mb
