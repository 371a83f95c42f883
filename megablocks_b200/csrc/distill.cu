// Distillation from a teacher's top logits, loss and gradient:
//
//   p = softmax(teacher values / T) over a row's used slots,  q = softmax(z / T) over the vocabulary
//   loss = T^2 sum_i p_i (log p_i - log q_{id_i}) + hard * (logsumexp(z) - z_target)
//   dloss / dz_j = T (q_j - sum_{i: id_i = j} p_i) + hard * (softmax(z)_j - [j = target])
//
// Bound by memory: a logit is read once and its gradient written once.  Where a row fits shared memory, CTAs
// stay and walk the rows.  A row is fetched by bulk copies, in chunks, and worked on in three passes over shared
// memory (maximum, as the chunks arrive; sums; gradient, stored straight to memory); the last pass hands its chunks
// back, and a warp of its own fetches the next row's into them and prepares the next row's teacher.  Two CTAs share
// an SM where two rows fit, so that one takes exponentials, of which there are two a logit, while the other waits for a
// sum or a copy.  Maximum and sums in one pass, with a maximum per thread, took 20 % longer.  Longer rows, and passes
// without a gradient, stream the row from memory with a running maximum; a gradient then reads it again, from
// L2.  The few columns that the teacher or the target names are written again, with their whole value and one
// rounding, after the row.
//
// 8192 rows of 51200 bf16 logits, 64 of the teacher: 333 us at 1965 MHz (1.68 GB, 0.77 of the copy bandwidth); pass
// after pass, at the 1880 MHz that the power limit leaves, 343, and 351 with the mean and the backward pass's factor.
// Neither the exponential unit (0.56 of its rate) nor the issue slots (0.51) nor memory is full: the barriers
// between a row's passes leave each of them idle in turn.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace mb {

namespace {

constexpr int kChunks = 4;                        // most chunks of a row in shared memory; with 8: 357 us of kernel
constexpr int kMaxThreads = 256;
constexpr int kRowThreads = 768;                  // of an SM that work on rows; 640: 363 us, 512: 368, 896: 416
constexpr int kSharedBytes = 226 * 1024;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kMost = 0x1p30f;                  // of an offset: its rounding, 2^6 at most, is an exponent

// 16 bytes of logits as pairs of fp32 values, on which the arithmetic runs two to an instruction.
template <typename T>
constexpr int kPairs = 8 / sizeof(T);

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float2 (&x)[kPairs<T>]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (std::is_same<T, float>::value) {
    x[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
    x[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      else
        x[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float2 (&x)[kPairs<T>]) {
  uint32_t w[4];
  if constexpr (std::is_same<T, float>::value) {
    w[0] = __float_as_uint(x[0].x), w[1] = __float_as_uint(x[0].y);
    w[2] = __float_as_uint(x[1].x), w[3] = __float_as_uint(x[1].y);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 q = __floats2bfloat162_rn(x[i].x, x[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&q);
      } else {
        const __half2 q = __floats2half2_rn(x[i].x, x[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&q);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 load_shared(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ float2 splat2(float v) { return make_float2(v, v); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 exp2_pair(float2 x) { return make_float2(exp2_approx(x.x), exp2_approx(x.y)); }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__device__ __forceinline__ float load_value(const void* p, DType type, int64_t i) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  if (type == kF16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// A row cut at 16-byte boundaries: `head` elements, `packs` of 16 bytes, `tail` elements.
template <typename T>
struct Cut {
  int head, packs, tail;
  __device__ __forceinline__ Cut(const T* row, int n) {
    constexpr int VEC = 16 / sizeof(T);
    const int phase = int(reinterpret_cast<uintptr_t>(row) % 16) / int(sizeof(T));
    head = min(n, (VEC - phase) % VEC);
    packs = (n - head) / VEC;
    tail = n - head - packs * VEC;
  }
};

// e^(x / T) and e^x, relative to the row's maximum.  At a temperature of 2 or 4 the second is a power of
// the first, which spares the exponential unit: two passes over both would keep it busier than memory.
struct Powers {
  float k;                     // log2(e) / T
  int squares;                 // e^x = (e^(x / T))^(2^squares); 3: take it by itself
  __device__ __forceinline__ float second(float first, float x_minus_max) const {
    if (squares == 3) return exp2_approx(x_minus_max * kLog2e);
    if (squares >= 1) first *= first;
    if (squares == 2) first *= first;
    return first;
  }
  __device__ __forceinline__ float2 second(float2 first, float2 x_minus_max) const {
    if (squares == 3) return exp2_pair(__fmul2_rn(x_minus_max, splat2(kLog2e)));
    if (squares >= 1) first = __fmul2_rn(first, first);
    if (squares == 2) first = __fmul2_rn(first, first);
    return first;
  }
};

// Running maximum and sums.  Differences are taken before they are scaled, so that logits far from zero
// lose nothing.
struct Online {
  float m = -INFINITY, soft = 0.f, hard = 0.f;
  __device__ __forceinline__ void raise(float top, const Powers& w, bool two) {
    if (top > m) {
      const float f = exp2_approx((m - top) * w.k);
      if (two) hard *= w.second(f, m - top);
      soft *= f;
      m = top;
    }
  }
  __device__ __forceinline__ void add(float x, const Powers& w, bool two) {
    raise(x, w, two);
    const float d = x - (m == -INFINITY ? 0.f : m), e = exp2_approx(d * w.k);
    soft += e;
    if (two) hard += w.second(e, d);
  }
  template <int N>
  __device__ __forceinline__ void add(const float2 (&x)[N], const Powers& w, bool two) {
    float2 top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = make_float2(fmaxf(top.x, x[i].x), fmaxf(top.y, x[i].y));
    raise(fmaxf(top.x, top.y), w, two);
    const float2 minus = splat2(m == -INFINITY ? 0.f : -m), k2 = splat2(w.k);
    float2 s = splat2(0.f), h = s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 d = __fadd2_rn(x[i], minus), e = exp2_pair(__fmul2_rn(d, k2));
      s = __fadd2_rn(s, e);
      if (two) h = __fadd2_rn(h, w.second(e, d));
    }
    soft += s.x + s.y;
    hard += h.x + h.y;
  }
};

// Maximum and sums of the row; `red` holds 3 floats a warp.  Ends with a barrier behind its reads.
__device__ __forceinline__ Online block_sums(Online o, const Powers& w, bool two, float* red) {
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto join = [&](Online part) {
    const float top = warp_max(part.m);
    if (part.m != -INFINITY) {                    // a NaN sum of a lane without a maximum stays
      const float f = exp2_approx((part.m - top) * w.k);
      part.soft *= f;
      if (two) part.hard *= w.second(f, part.m - top);
    }
    part.soft = warp_sum(part.soft);
    if (two) part.hard = warp_sum(part.hard);
    part.m = top;
    return part;
  };
  o = join(o);
  if (lane == 0) { red[3 * warp] = o.m; red[3 * warp + 1] = o.soft; red[3 * warp + 2] = o.hard; }
  __syncthreads();
  Online part;
  if (lane < warps) { part.m = red[3 * lane]; part.soft = red[3 * lane + 1]; part.hard = red[3 * lane + 2]; }
  part = join(part);
  __syncthreads();
  if (!two) part.hard = part.soft;
  return part;
}

// The teacher's row in shared memory: `slots` values each of p (0 in unused slots), column (-1 there) and z, the
// named columns' logits, which the row's threads fill in.
__host__ __device__ constexpr int padded_slots(int top) { return (top + 3) / 4 * 4; }
struct Teacher {
  float* p;
  int* column;
  float* z;
  __device__ __forceinline__ Teacher(void* place, int top)
      : p(static_cast<float*>(place)), column(reinterpret_cast<int*>(p + padded_slots(top))),
        z(p + 2 * padded_slots(top)) {}
};

// What a row's threads have to know about it.
struct TeacherFacts {
  float entropy;               // sum p log p
  int live;                    // any slot is used
  int twice;                   // a column is named by more than one slot
  int target_named;            // the target is a named column
};

// Slots that name column c, other than slot i.
__device__ __forceinline__ bool named_elsewhere(const Teacher& t, int top, int c, int i) {
  int found = 0;
  for (int k = 0; k < padded_slots(top); k += 4) {
    const int4 q = *reinterpret_cast<const int4*>(t.column + k);
    found |= int(q.x == c && k != i) | int(q.y == c && k + 1 != i) | int(q.z == c && k + 2 != i) |
             int(q.w == c && k + 3 != i);
  }
  return found != 0;
}

// Fills it, with one warp.  `named`: the facts about columns are wanted.
__device__ __forceinline__ TeacherFacts teacher_row(const DistillArgs& a, int64_t row, const Teacher& t, int target,
                                                    bool named) {
  const int lane = threadIdx.x & 31;
  const float inv_t = 1.f / a.temperature;
  float top = -INFINITY;
  bool any = false;            // NaN is a value too, and shows in the loss
  for (int i0 = lane; i0 < padded_slots(a.top); i0 += 128) {      // 128 slots in flight
    int64_t id[4];
    float value[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 32 * u;
      const int64_t at = row * a.top + i;
      id[u] = -1;
      value[u] = -INFINITY;
      if (i < a.top) {
        id[u] = a.ids64 ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int*>(a.ids)[at];
        value[u] = load_value(a.values, a.value_type, at);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 32 * u;
      if (i >= padded_slots(a.top)) break;
      const bool used = id[u] >= 0 && id[u] < a.vocab;
      t.column[i] = used ? int(id[u]) : -1;
      t.p[i] = used ? value[u] : -INFINITY;
      top = fmaxf(top, t.p[i]);
      any |= t.p[i] != -INFINITY;
    }
  }
  top = warp_max(top);
  const bool live = __any_sync(0xffffffffu, any);
  float sum = 0.f;
  // Differences first: the ends of the type, divided by a small temperature, would be infinite.
  for (int i = lane; i < a.top; i += 32) sum += live ? exp2_approx((t.p[i] - top) * inv_t * kLog2e) : 0.f;
  sum = warp_sum(sum);
  const float log_sum = kLn2 * __log2f(sum), inv = 1.f / sum;
  float ent = 0.f;
  for (int i = lane; i < a.top; i += 32) {
    const float x = (t.p[i] - top) * inv_t;
    const float w = live ? exp2_approx(x * kLog2e) * inv : 0.f;
    if (w != 0.f) ent += w * (x - log_sum);
    t.p[i] = w;
    if (w == 0.f) t.column[i] = -1;
  }
  TeacherFacts f{warp_sum(ent), live, 0, 0};
  __syncwarp();
  if (named) {
    for (int i = lane; i < a.top; i += 32) {
      const int c = t.column[i];
      if (c >= 0) f.twice |= named_elsewhere(t, a.top, c, i);
      f.target_named |= target >= 0 && c == target;
    }
    f.twice = __any_sync(0xffffffffu, f.twice);
    f.target_named = __any_sync(0xffffffffu, f.target_named);
  }
  return f;
}

__device__ __forceinline__ int target_of(const DistillArgs& a, int64_t row) {
  const int64_t wanted = a.targets != nullptr ? a.targets[row] : -1;
  return wanted >= 0 && wanted < a.vocab ? int(wanted) : -1;
}

// Coefficients of a row's gradient, probabilities' sums included.
struct RowGrad {
  float soft, hard;            // 0: that part is absent
  float offset;                // 2^(z k - offset) is e^((z - max) / T) up to a factor that `soft` makes good
  float max;
  Powers w;
};

enum Parts { kNothing, kOne, kBoth };                // to learn from a row; whatever its logits where nothing
__device__ __forceinline__ Parts parts_of(const RowGrad& g) {
  if (g.soft == 0.f && g.hard == 0.f) return kNothing;
  return g.hard == 0.f && fabsf(g.offset) <= kMost ? kOne : kBoth;
}

template <Parts P, int N>
__device__ __forceinline__ void gradient(const RowGrad& g, float2 (&x)[N]) {
  if constexpr (P == kNothing) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = splat2(0.f);
  } else if constexpr (P == kOne) {
    const float2 k2 = splat2(g.w.k), minus = splat2(-g.offset), soft = splat2(g.soft);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __fmul2_rn(soft, exp2_pair(__ffma2_rn(x[i], k2, minus)));
  } else {
    const float2 k2 = splat2(g.w.k), minus = splat2(-g.max), soft = splat2(g.soft), hard = splat2(g.hard);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 d = __fadd2_rn(x[i], minus), e = exp2_pair(__fmul2_rn(d, k2));
      x[i] = __ffma2_rn(hard, g.w.second(e, d), __fmul2_rn(soft, e));
    }
  }
}
__device__ __forceinline__ float gradient(const RowGrad& g, float z) {
  float2 x[1] = {make_float2(z, z)};
  const Parts parts = parts_of(g);
  if (parts == kNothing) return 0.f;
  if (parts == kOne) gradient<kOne>(g, x);
  else gradient<kBoth>(g, x);
  return x[0].x;
}
// Calls body(parts as a constant).
template <typename F>
__device__ __forceinline__ void with_parts(const RowGrad& g, F&& body) {
  const Parts parts = parts_of(g);
  if (parts == kNothing) body(std::integral_constant<Parts, kNothing>{});
  else if (parts == kOne) body(std::integral_constant<Parts, kOne>{});
  else body(std::integral_constant<Parts, kBoth>{});
}

__device__ __forceinline__ RowGrad row_grad(const DistillArgs& a, const TeacherFacts& f, bool has_target, float scale,
                                            float max, float sum_soft, float sum_hard, const Powers& w) {
  RowGrad g;
  g.w = w;
  g.max = max;
  g.soft = f.live ? a.temperature * scale / sum_soft : 0.f;
  if (f.entropy != f.entropy) g.soft = NAN;       // the teacher's probabilities are NaN, and so is their sum
  g.hard = has_target ? a.hard_weight * scale / sum_hard : 0.f;
  if (w.squares == 0) {                           // one probability serves both parts
    g.soft += g.hard;
    g.hard = 0.f;
  }
  g.offset = max * w.k;
  if (parts_of(g) == kOne) g.soft *= exp2_approx(-fmaf(max, w.k, -g.offset));
  return g;
}

// Writes a row's gradient over a row in memory (`grad` itself, possibly).
template <typename T>
__device__ __forceinline__ void write_gradient(const T* src, const Cut<T>& cut, T* grad, int vocab, const RowGrad& g) {
  auto one = [&](int i) { grad[i] = from_float<T>(gradient(g, to_float(src[i]))); };
  if (reinterpret_cast<uintptr_t>(grad + cut.head) % 16 == 0) {
    if (int(threadIdx.x) < cut.head) one(threadIdx.x);
    if (int(threadIdx.x) < cut.tail) one(vocab - cut.tail + threadIdx.x);
    const uint4* from = reinterpret_cast<const uint4*>(src + cut.head);
    uint4* to = reinterpret_cast<uint4*>(grad + cut.head);
    with_parts(g, [&](auto parts) {
      constexpr int kAhead = 4;        // packs of a thread in flight
      for (int i = threadIdx.x; i < cut.packs; i += kAhead * blockDim.x) {
        uint4 v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (i + u * int(blockDim.x) < cut.packs) v[u] = from[i + u * blockDim.x];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (i + u * int(blockDim.x) >= cut.packs) break;
          float2 x[kPairs<T>];
          unpack<T>(v[u], x);
          gradient<decltype(parts)::value>(g, x);
          to[i + u * blockDim.x] = pack<T>(x);
        }
      }
    });
  } else {
    for (int i = threadIdx.x; i < vocab; i += blockDim.x) one(i);
  }
}

// The columns that the teacher or the target names, with their logits `z` and `z_target` from before the
// row was written.  A column named more than once is written by its first slot, with all its shares.
template <typename T>
__device__ __forceinline__ void write_named(const DistillArgs& a, T* grad, const RowGrad& g, float soft_scale,
                                            float hard_scale, const Teacher& t, const TeacherFacts& f, int target,
                                            float z_target, int threads) {
  for (int i = threadIdx.x; i < a.top; i += threads) {
    const int c = t.column[i];
    if (c < 0) continue;
    float share = t.p[i];
    if (f.twice) {
      share = 0.f;
      bool first = true;
      for (int k = 0; k < a.top; ++k) {
        if (t.column[k] != c) continue;
        first &= k >= i;
        share += t.p[k];
      }
      if (!first) continue;
    }
    grad[c] = from_float<T>(gradient(g, t.z[i]) - soft_scale * share - (c == target ? hard_scale : 0.f));
  }
  if (int(threadIdx.x) == threads - 1 && target >= 0 && !f.target_named)
    grad[target] = from_float<T>(gradient(g, z_target) - hard_scale);
}

__device__ __forceinline__ Powers powers(const DistillArgs& a) {
  const float t = a.temperature;
  return {kLog2e / t, t == 1.f ? 0 : (t == 2.f ? 1 : (t == 4.f ? 2 : 3))};
}

// Maximum of 16 bytes; of 16-bit types in their own arithmetic, which is exact.
template <typename T>
__device__ __forceinline__ float pack_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    using P2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    const P2* q = reinterpret_cast<const P2*>(&v);
    const P2 m = __hmax2(__hmax2(q[0], q[1]), __hmax2(q[2], q[3]));
    return fmaxf(to_float(m.x), to_float(m.y));
  }
}

// Rows in shared memory.  All warps but the last work on a row; the last fetches the next one and prepares its
// teacher.  Shared memory holds the 16-byte blocks of memory that a row touches, `chunk` blocks to a chunk.
template <typename T>
__global__ void __launch_bounds__(kRowThreads + 32)
distill_rows_kernel(const DistillArgs a, int row_bytes, int chunk, float* __restrict__ stats, T* grad) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ float red[4][kRowThreads / 32];
  __shared__ alignas(8) uint64_t full[kChunks], empty[kChunks];
  __shared__ int abort_flag;
  __shared__ TeacherFacts facts[3];
  const int threads = blockDim.x - 32, warps = threads >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slots = padded_slots(a.top);
  float* teachers = reinterpret_cast<float*>(shared + row_bytes);          // [3]
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int c = 0; c < kChunks; ++c) {
      ptx::mbar_init(ptx::smem_u32(&full[c]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty[c]), warps);
    }
    ptx::fence_barrier_init();
  }
  __syncthreads();
  auto row_of = [&](int64_t row) { return static_cast<const T*>(a.logits) + row * a.vocab; };
  const uint32_t blocks = ptx::smem_u32(shared);

  if (warp == warps) {
    // The teacher has three places: the named columns of the row before are still being written.
    int set = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto prepare = [&](int64_t row, bool again) {
      if (row < a.rows) {
        const TeacherFacts f = teacher_row(a, row, Teacher(teachers + set * 3 * slots, a.top), target_of(a, row), true);
        if (lane == 0) facts[set] = f;
        const T* in = row_of(row);
        const Cut<T> cut(in, a.vocab);
        const int first = cut.head > 0 ? 1 : 0, last = first + cut.packs;  // blocks that are whole
        const T* block0 = in + cut.head - first * VEC;
        for (int c = 0; c < kChunks && c * chunk * 16 < row_bytes; ++c) {
          if (again)
            ok = ok && ptx::mbar_wait(ptx::smem_u32(&empty[c]), phase, &abort_flag, a.status, kDistillTimeout, kWaitNs);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) {
            const uint32_t bar = ptx::smem_u32(&full[c]);
            const int from = max(first, c * chunk), to = min(last, (c + 1) * chunk);
            ptx::mbar_arrive_expect_tx(bar, uint32_t(max(0, to - from)) * 16);
            if (from < to) ptx::bulk_load(blocks + from * 16, block0 + from * VEC, uint32_t(to - from) * 16, bar);
          }
          __syncwarp();
        }
        if (again) phase ^= 1u;
      }
      set = set == 2 ? 0 : set + 1;
    };
    prepare(blockIdx.x, false);
    __syncthreads();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
      prepare(row + gridDim.x, true);
      __syncthreads();
    }
    if (*static_cast<volatile int*>(&abort_flag) != 0) {           // a wait ran out: let the copies in flight end
      const uint64_t t0 = ptx::globaltimer_ns();
      while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
    return;
  }

  const Powers w = powers(a);
  auto group_sync = [&] { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); };
  __syncthreads();
  int set = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* in = row_of(row);
    const Cut<T> cut(in, a.vocab);
    const int first = cut.head > 0 ? 1 : 0, last = first + cut.packs;
    const T* copy = reinterpret_cast<const T*>(shared) + first * VEC - cut.head;         // where element 0 would lie
    const Teacher t(teachers + set * 3 * slots, a.top);
    const int target = target_of(a, row);
    const bool two = target >= 0 && w.squares != 0;
    // The elements before the first and behind the last 16-byte boundary stay in memory: one thread's each.
    const int tail0 = a.vocab - cut.tail;
    const int mine = int(threadIdx.x) < cut.head ? int(threadIdx.x)
                     : int(threadIdx.x) - cut.head < cut.tail ? tail0 + int(threadIdx.x) - cut.head : -1;
    const float edge = mine >= 0 ? to_float(in[mine]) : -INFINITY;
    auto value_at = [&](int c) { return to_float(c < cut.head || c >= tail0 ? in[c] : copy[c]); };
    // The row's whole blocks, a thread's share of them.
    auto each = [&](auto&& body) {
#pragma unroll 4
      for (int i = first + threadIdx.x; i < last; i += threads) body(i);
    };

    // The maximum, chunk by chunk as they arrive.
    float top = edge;
    for (int c = 0; c < kChunks && c * chunk * 16 < row_bytes; ++c) {
      if (!ptx::mbar_wait(ptx::smem_u32(&full[c]), phase, &abort_flag, a.status, kDistillTimeout, kWaitNs)) break;
      const int to = min(last, (c + 1) * chunk);
#pragma unroll 4
      for (int i = max(first, c * chunk) + int(threadIdx.x); i < to; i += threads)
        top = fmaxf(top, pack_max<T>(load_shared(blocks + i * 16)));
    }
    const TeacherFacts f = facts[set];
    top = warp_max(top);
    if (lane == 0) red[0][warp] = top;
    group_sync();
    top = warp_max(lane < warps ? red[0][lane] : -INFINITY);
    const bool ok = *static_cast<volatile int*>(&abort_flag) == 0;
    const float base = top == -INFINITY ? 0.f : top;

    // 2^(z k - offset) is e^((z - max) / T) up to the rounding of the offset, which all of the row share.  Where that
    // is too large (a row of the type's lowest value), or the hard part wants them, differences come first.
    const float offset = base * w.k;
    const bool differ = two || !(fabsf(offset) <= kMost);
    float2 soft = splat2(0.f), hard = soft;
    float cross = 0.f;
    for (int i = threadIdx.x; i < a.top; i += threads) {
      if (t.column[i] < 0) continue;
      t.z[i] = value_at(t.column[i]);  // before the row may be overwritten
      cross += t.p[i] * (t.z[i] - base);
    }
    const float z_target = target >= 0 ? value_at(target) : 0.f;
    if (mine >= 0) {
      soft.x = differ ? exp2_approx((edge - base) * w.k) : exp2_approx(fmaf(edge, w.k, -offset));
      if (two) hard.x = w.second(soft.x, edge - base);
    }
    const float2 minus = splat2(differ ? -base : -offset), k2 = splat2(w.k);
    auto add = [&](auto with_hard) {
      each([&](int i) {
        float2 x[kPairs<T>];
        unpack<T>(load_shared(blocks + i * 16), x);
#pragma unroll
        for (int k = 0; k < kPairs<T>; ++k) {
          if constexpr (decltype(with_hard)::value) {
            const float2 d = __fadd2_rn(x[k], minus), e = exp2_pair(__fmul2_rn(d, k2));
            soft = __fadd2_rn(soft, e);
            hard = __fadd2_rn(hard, w.second(e, d));
          } else {
            soft = __fadd2_rn(soft, exp2_pair(__ffma2_rn(x[k], k2, minus)));
          }
        }
      });
    };
    if (ok) {
      if (differ) add(std::true_type{});
      else add(std::false_type{});
    }
    {
      const float s = warp_sum(soft.x + soft.y), h = two ? warp_sum(hard.x + hard.y) : 0.f, c = warp_sum(cross);
      if (lane == 0) { red[1][warp] = s; red[2][warp] = h; red[3][warp] = c; }
    }
    group_sync();
    float sum_soft = warp_sum(lane < warps ? red[1][lane] : 0.f);
    const float all_cross = warp_sum(lane < warps ? red[3][lane] : 0.f);
    if (!differ) sum_soft *= exp2_approx(-fmaf(base, w.k, -offset));
    const float sum_hard = two ? warp_sum(lane < warps ? red[2][lane] : 0.f) : sum_soft;
    if (threadIdx.x == 32 % threads) {
      float l = 0.f;
      if (f.live) l = a.temperature * a.temperature * (f.entropy - kLn2 * (all_cross * w.k - __log2f(sum_soft)));
      if (target >= 0) l += a.hard_weight * (kLn2 * __log2f(sum_hard) + (top - z_target));
      *reinterpret_cast<float4*>(stats + 4 * row) = make_float4(ok ? l : NAN, top, sum_soft, sum_hard);
    }
    const RowGrad g = row_grad(a, f, target >= 0, a.scale, top, sum_soft, sum_hard, w);
    T* out = grad + row * a.vocab;
    if (mine >= 0) out[mine] = from_float<T>(gradient(g, edge));
    T* block0 = out + cut.head - first * VEC;      // where block 0 would lie
    const bool aligned = reinterpret_cast<uintptr_t>(block0) % 16 == 0;
    with_parts(g, [&](auto parts) {
      uint4* to16 = reinterpret_cast<uint4*>(block0);
      for (int c = 0; c < kChunks && c * chunk * 16 < row_bytes; ++c) {
        const int to = ok ? min(last, (c + 1) * chunk) : 0, from = max(first, c * chunk) + int(threadIdx.x);
        auto value = [&](int i) {
          float2 x[kPairs<T>];
          unpack<T>(load_shared(blocks + i * 16), x);
          gradient<decltype(parts)::value>(g, x);
          return pack<T>(x);
        };
        if (aligned) {
#pragma unroll 4
          for (int i = from; i < to; i += threads) to16[i] = value(i);
        } else {
          for (int i = from; i < to; i += threads) {
            const uint4 v = value(i);
            const T* one = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int k = 0; k < VEC; ++k) block0[i * VEC + k] = one[k];
          }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&empty[c]));
      }
    });
    __syncthreads();
    write_named(a, out, g, a.temperature * a.scale, a.hard_weight * a.scale, t, f, target, z_target, threads);
    phase ^= 1u;
    set = set == 2 ? 0 : set + 1;
  }
}

// Rows streamed from memory, one a CTA.
template <typename T>
__global__ void __launch_bounds__(kMaxThreads)
distill_fwd_kernel(const DistillArgs a, float* __restrict__ stats, T* grad) {
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ float red[3 * kMaxThreads / 32];
  __shared__ TeacherFacts facts;
  const int64_t row = blockIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.vocab;
  const Cut<T> cut(in, a.vocab);
  const Teacher t(shared, a.top);
  const int target = target_of(a, row);
  const Powers w = powers(a);
  const bool two = target >= 0 && w.squares != 0;               // a second sum, at temperature one
  Online sums;
  {
    auto one = [&](int i) { sums.add(to_float(in[i]), w, two); };
    if (int(threadIdx.x) < cut.head) one(threadIdx.x);
    if (int(threadIdx.x) < cut.tail) one(a.vocab - cut.tail + threadIdx.x);
  }
  const uint4* body = reinterpret_cast<const uint4*>(in + cut.head);
  constexpr int kAhead = 4;            // packs of a thread in flight
  for (int i = threadIdx.x; i < cut.packs; i += kAhead * blockDim.x) {
    uint4 v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i + u * int(blockDim.x) < cut.packs) v[u] = body[i + u * blockDim.x];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u * int(blockDim.x) >= cut.packs) break;
      float2 x[kPairs<T>];
      unpack<T>(v[u], x);
      sums.add(x, w, two);
    }
  }
  if (threadIdx.x < 32) {
    const TeacherFacts f = teacher_row(a, row, t, target, grad != nullptr);
    if (threadIdx.x == 0) facts = f;
  }
  sums = block_sums(sums, w, two, red);
  const TeacherFacts f = facts;
  const bool live = f.live != 0;
  const float log_soft = __log2f(sums.soft);

  // Loss, and the named columns' logits before the row may be overwritten.
  const float z_target = target >= 0 ? to_float(in[target]) : 0.f;
  float cross = 0.f;
  for (int i = threadIdx.x; i < a.top; i += blockDim.x) {
    const int c = t.column[i];
    if (c < 0) continue;
    t.z[i] = to_float(in[c]);
    cross += t.p[i] * fmaf(t.z[i] - sums.m, w.k, -log_soft);
  }
  cross = warp_sum(cross);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = cross;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = 0.f;
    for (int k = 0; k < int(blockDim.x >> 5); ++k) sum += red[k];
    float l = live ? a.temperature * a.temperature * (f.entropy - kLn2 * sum) : 0.f;
    if (target >= 0) l += a.hard_weight * (kLn2 * __log2f(sums.hard) + (sums.m - z_target));
    *reinterpret_cast<float4*>(stats + 4 * row) = make_float4(l, sums.m, sums.soft, sums.hard);
  }
  if (grad == nullptr) return;
  T* out = grad + row * a.vocab;
  const RowGrad g = row_grad(a, f, target >= 0, a.scale, sums.m, sums.soft, sums.hard, w);
  write_gradient(in, cut, out, a.vocab, g);
  __syncthreads();
  write_named(a, out, g, a.temperature * a.scale, a.hard_weight * a.scale, t, f, target, z_target, blockDim.x);
}

template <typename T>
__global__ void __launch_bounds__(kMaxThreads)
distill_bwd_kernel(const DistillArgs a, const float* __restrict__ stats, const float* __restrict__ grad_out,
                   T* __restrict__ grad) {
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ TeacherFacts facts;
  const int64_t row = blockIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.vocab;
  const Cut<T> cut(in, a.vocab);
  const Teacher t(shared, a.top);
  const int target = target_of(a, row);
  if (threadIdx.x < 32) {
    const TeacherFacts f = teacher_row(a, row, t, target, true);
    if (threadIdx.x == 0) facts = f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.top; i += blockDim.x)
    if (t.column[i] >= 0) t.z[i] = to_float(in[t.column[i]]);
  const float z_target = target >= 0 ? to_float(in[target]) : 0.f;
  const float scale = a.scale * *grad_out;
  const float4 st = *reinterpret_cast<const float4*>(stats + 4 * row);
  const RowGrad g = row_grad(a, facts, target >= 0, scale, st.y, st.z, st.w, powers(a));
  T* out = grad + row * a.vocab;
  write_gradient(in, cut, out, a.vocab, g);
  __syncthreads();
  write_named(a, out, g, a.temperature * scale, a.hard_weight * scale, t, facts, target, z_target, blockDim.x);
}

__global__ void __launch_bounds__(1024)
distill_mean_kernel(const float* __restrict__ stats, int64_t rows, float* __restrict__ mean) {
  __shared__ float red[32];
  float sum = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) sum += stats[4 * r];
  sum = warp_sum(sum);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = warp_sum(red[threadIdx.x]);
    if (threadIdx.x == 0) *mean = sum / float(rows);
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
scale_unless_one_kernel(T* __restrict__ x, int64_t numel, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.f) return;
  constexpr int VEC = 16 / sizeof(T);
  const int64_t step = int64_t(gridDim.x) * 256, start = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int64_t packs = numel / VEC;
  for (int64_t i = start; i < packs; i += step) {
    float2 v[kPairs<T>];
    unpack<T>(reinterpret_cast<const uint4*>(x)[i], v);
#pragma unroll
    for (int k = 0; k < kPairs<T>; ++k) v[k] = __fmul2_rn(v[k], splat2(f));
    reinterpret_cast<uint4*>(x)[i] = pack<T>(v);
  }
  for (int64_t i = packs * VEC + start; i < numel; i += step) x[i] = from_float<T>(to_float(x[i]) * f);
}

// Threads a row: four packs each at least, so that short rows do not pay for idle warps.
int row_threads(int64_t bytes) {
  int threads = 32;
  while (threads < kMaxThreads && threads * 64 < bytes) threads *= 2;
  return threads;
}

bool valid(const DistillArgs& a) {
  return a.vocab >= 1 && a.top >= 1 && a.top <= kDistillMaxTop && a.rows >= 0 && a.rows <= 0x7fffffffll &&
         a.temperature > 0.f;
}

}  // namespace

cudaError_t distill_fwd(DType type, const DistillArgs& a, float* stats, void* grad, int sms, cudaStream_t stream) {
  if (!valid(a)) return cudaErrorInvalidValue;
  if (a.rows == 0) return cudaSuccess;
  const size_t slots = 3 * size_t(padded_slots(a.top)) * 4;
  MB_SWITCH_FLOAT(type, T, {
    const int64_t bytes = int64_t(a.vocab) * sizeof(T);
    const int64_t row_bytes = (bytes + 15) / 16 * 16 + 16, shared = row_bytes + 3 * int64_t(slots);
    if (grad != nullptr && shared <= kSharedBytes) {
      auto kernel = distill_rows_kernel<T>;
      // The most that any row takes, once: the limit is the kernel's, and another thread may set and launch too.
      static std::atomic<bool> allowed[64];
      const cudaError_t rc = allow_shared(kernel, kSharedBytes, allowed);
      if (rc != cudaSuccess) return rc;
      // As many CTAs as fit an SM, 24 warps between them, but no more than leave each thread four blocks.
      const int resident = max(1, int(min(int64_t(16), kSharedBytes / (shared + 1024))));
      const int threads = max(32, min(kRowThreads / resident, int((bytes + 63) / 64)) / 32 * 32);
      const int64_t grid = min(a.rows, int64_t(sms) * resident);
      // Chunks of whole rounds of the threads.
      const int chunk = int((row_bytes / 16 + kChunks * threads - 1) / (kChunks * threads)) * threads;
      kernel<<<unsigned(grid), threads + 32, shared, stream>>>(a, int(row_bytes), chunk, stats, static_cast<T*>(grad));
    } else {
      distill_fwd_kernel<T><<<unsigned(a.rows), row_threads(bytes), slots, stream>>>(a, stats, static_cast<T*>(grad));
    }
  })
  return cudaGetLastError();
}

cudaError_t distill_mean(const float* stats, int64_t rows, float* mean, cudaStream_t stream) {
  distill_mean_kernel<<<1, 1024, 0, stream>>>(stats, rows, mean);
  return cudaGetLastError();
}

cudaError_t distill_bwd(DType type, const DistillArgs& a, const float* stats, const float* grad_out, void* grad,
                        cudaStream_t stream) {
  if (!valid(a)) return cudaErrorInvalidValue;
  if (a.rows == 0) return cudaSuccess;
  const size_t slots = 3 * size_t(padded_slots(a.top)) * 4;
  MB_SWITCH_FLOAT(type, T, {
    distill_bwd_kernel<T><<<unsigned(a.rows), row_threads(int64_t(a.vocab) * sizeof(T)), slots, stream>>>(
        a, stats, grad_out, static_cast<T*>(grad));
  })
  return cudaGetLastError();
}

cudaError_t scale_unless_one(DType type, void* x, int64_t numel, const float* factor, int sms, cudaStream_t stream) {
  if (numel == 0) return cudaSuccess;
  MB_SWITCH_FLOAT(type, T, {
    const int64_t want = (numel / (16 / sizeof(T)) + 255) / 256;
    const int grid = int(want < 1 ? 1 : (want > int64_t(sms) * 8 ? int64_t(sms) * 8 : want));
    scale_unless_one_kernel<T><<<grid, 256, 0, stream>>>(static_cast<T*>(x), numel, factor);
  })
  return cudaGetLastError();
}

}  // namespace mb
