// Distillation from a teacher's top logits, loss and gradient:
//
//   p = softmax(teacher values / T) over a row's used slots,  q = softmax(z / T) over the vocabulary
//   loss = T^2 sum_i p_i (log p_i - log q_{id_i}) + hard * (logsumexp(z) - z_target)
//   dloss / dz_j = T (q_j - sum_{i: id_i = j} p_i) + hard * (softmax(z)_j - [j = target])
//
// Bound by memory: a logit is read once and its gradient written once.  A CTA takes a row.  Where the row
// fits shared memory it is fetched there by bulk copies, all of them in flight from the start, and both
// passes (the running maximum and sum; the gradient) run on that copy; longer rows take the second pass
// from L2.  The few columns that the teacher or the target names are written again, with their whole
// value and one rounding, after the row.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace mb {

namespace {

constexpr int kChunks = 8;                        // bulk copies of a row, each with a barrier of its own
constexpr int kMaxThreads = 512;
constexpr int kSharedRow = 200 * 1024;            // longest row, in bytes, that is kept in shared memory
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

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
};

// Running maximum and sums.  Differences are taken before they are scaled, so that logits far from zero
// lose nothing.
struct Online {
  float m = -INFINITY, soft = 0.f, hard = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], const Powers& w, bool two) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    if (top > m) {
      const float f = exp2_approx((m - top) * w.k);
      if (two) hard *= w.second(f, m - top);
      soft *= f;
      m = top;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = exp2_approx((x[i] - base) * w.k);
      soft += e;
      if (two) hard += w.second(e, x[i] - base);
    }
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

// The teacher's row in shared memory: p (0 in unused slots) and column (-1 there).  One warp; returns
// whether any slot is used, and sum p log p.
__device__ __forceinline__ bool teacher_row(const DistillArgs& a, int64_t row, float* p, int* column, float* entropy) {
  const int lane = threadIdx.x & 31;
  const float inv_t = 1.f / a.temperature;
  float top = -INFINITY;
  for (int i = lane; i < a.top; i += 32) {
    const int64_t at = row * a.top + i;
    const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int*>(a.ids)[at];
    const bool used = id >= 0 && id < a.vocab;
    column[i] = used ? int(id) : -1;
    p[i] = used ? load_value(a.values, a.value_type, at) * inv_t : -INFINITY;
    top = fmaxf(top, p[i]);
  }
  top = warp_max(top);
  const bool live = top > -INFINITY;
  float sum = 0.f;
  for (int i = lane; i < a.top; i += 32) sum += live ? exp2_approx((p[i] - top) * kLog2e) : 0.f;
  sum = warp_sum(sum);
  const float log_sum = kLn2 * __log2f(sum), inv = 1.f / sum;
  float ent = 0.f;
  for (int i = lane; i < a.top; i += 32) {
    const float x = p[i] - top;
    const float w = live ? exp2_approx(x * kLog2e) * inv : 0.f;
    if (w != 0.f) ent += w * (x - log_sum);
    p[i] = w;
    if (w == 0.f) column[i] = -1;
  }
  *entropy = warp_sum(ent);
  __syncwarp();
  return live;
}

// Coefficients of a row's gradient, probabilities' sums included.
struct RowGrad {
  float soft, hard;            // 0: that part is absent
  float offset;                // 2^(z k - offset) is e^((z - max) / T) up to a factor that `soft` makes good
  float max;
  Powers w;
};

template <int N>
__device__ __forceinline__ void gradient(const RowGrad& g, float (&x)[N]) {
  if (g.soft == 0.f && g.hard == 0.f) {           // nothing to learn from this row, whatever its logits
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
  } else if (g.hard == 0.f) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = g.soft * exp2_approx(fmaf(x[i], g.w.k, -g.offset));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = exp2_approx((x[i] - g.max) * g.w.k);
      x[i] = fmaf(g.hard, g.w.second(e, x[i] - g.max), g.soft * e);
    }
  }
}

__device__ __forceinline__ RowGrad row_grad(const DistillArgs& a, bool live, bool has_target, float scale, float max,
                                            float sum_soft, float sum_hard, const Powers& w) {
  RowGrad g;
  g.w = w;
  g.max = max;
  g.soft = live ? a.temperature * scale / sum_soft : 0.f;
  g.hard = has_target ? a.hard_weight * scale / sum_hard : 0.f;
  if (w.squares == 0) {                           // one probability serves both parts
    g.soft += g.hard;
    g.hard = 0.f;
  }
  g.offset = max * w.k;
  if (g.hard == 0.f && g.soft != 0.f) g.soft *= exp2_approx(-fmaf(max, w.k, -g.offset));
  return g;
}

// Writes a row's gradient; `src` is the row in shared or global memory (`grad` itself, possibly).
template <typename T>
__device__ __forceinline__ void write_gradient(const T* src, const Cut<T>& cut, T* grad, int vocab, const RowGrad& g) {
  constexpr int VEC = 16 / sizeof(T);
  const bool vector = reinterpret_cast<uintptr_t>(src + cut.head) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(grad + cut.head) % 16 == 0;
  auto one = [&](int i) {
    float x[1] = {to_float(src[i])};
    gradient(g, x);
    grad[i] = from_float<T>(x[0]);
  };
  if (vector) {
    if (int(threadIdx.x) < cut.head) one(threadIdx.x);
    if (int(threadIdx.x) < cut.tail) one(vocab - cut.tail + threadIdx.x);
    for (int p = threadIdx.x; p < cut.packs; p += blockDim.x) {
      Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(src + cut.head + p * VEC);
      float x[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = to_float(v.v[k]);
      gradient(g, x);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v.v[k] = from_float<T>(x[k]);
      *reinterpret_cast<Pack<T, VEC>*>(grad + cut.head + p * VEC) = v;
    }
  } else {
    for (int i = threadIdx.x; i < vocab; i += blockDim.x) one(i);
  }
}

// The columns that the teacher or the target names, with their logits `z` and `z_target` from before the
// row was written.  A column named more than once is written by its first slot, with all its shares.
template <typename T>
__device__ __forceinline__ void write_named(const DistillArgs& a, T* grad, const RowGrad& g, float soft_scale,
                                            float hard_scale, const float* p, const int* column, const float* z,
                                            int target, float z_target) {
  for (int i = threadIdx.x; i < a.top; i += blockDim.x) {
    const int c = column[i];
    if (c < 0) continue;
    float share = 0.f;
    bool first = true;
    for (int k = 0; k < a.top; ++k) {
      if (column[k] != c) continue;
      if (k < i) { first = false; break; }
      share += p[k];
    }
    if (!first) continue;
    float x[1] = {z[i]};
    gradient(g, x);
    grad[c] = from_float<T>(x[0] - soft_scale * share - (c == target ? hard_scale : 0.f));
  }
  if (threadIdx.x == 0 && target >= 0) {
    bool named = false;
    for (int k = 0; k < a.top; ++k) named |= column[k] == target;
    if (!named) {
      float x[1] = {z_target};
      gradient(g, x);
      grad[target] = from_float<T>(x[0] - hard_scale);
    }
  }
}

__device__ __forceinline__ Powers powers(const DistillArgs& a) {
  const float t = a.temperature;
  return {kLog2e / t, t == 1.f ? 0 : (t == 2.f ? 1 : (t == 4.f ? 2 : 3))};
}

template <typename T, bool CACHED>
__global__ void __launch_bounds__(kMaxThreads)
distill_fwd_kernel(const DistillArgs a, float* __restrict__ stats, T* grad) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ float red[3 * kMaxThreads / 32];
  __shared__ alignas(8) uint64_t bars[kChunks];
  __shared__ int abort_flag;
  __shared__ float entropy_s;
  __shared__ int live_s;
  const int64_t row = blockIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.vocab;
  const Cut<T> cut(in, a.vocab);
  float* p = reinterpret_cast<float*>(shared);
  int* column = reinterpret_cast<int*>(p + a.top);
  float* z = reinterpret_cast<float*>(column + a.top);
  T* copy = nullptr;
  int chunk_packs = 1;
  if constexpr (CACHED) {
    unsigned char* base = shared + (3 * size_t(a.top) * 4 + 15) / 16 * 16;
    copy = reinterpret_cast<T*>(base + reinterpret_cast<uintptr_t>(in) % 16);
    const int all = kChunks * int(blockDim.x);          // whole rounds of the block in every chunk
    chunk_packs = max(1, (cut.packs + all - 1) / all) * int(blockDim.x);
    if (threadIdx.x == 0) {
      abort_flag = 0;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) ptx::mbar_init(ptx::smem_u32(&bars[c]), 1);
      ptx::fence_barrier_init();
      ptx::fence_proxy_async_smem();
      for (int c = 0; c * chunk_packs < cut.packs; ++c) {
        const int n = min(chunk_packs, cut.packs - c * chunk_packs);
        const uint32_t bar = ptx::smem_u32(&bars[c]);
        ptx::mbar_arrive_expect_tx(bar, uint32_t(n) * 16);
        ptx::bulk_load(ptx::smem_u32(copy + cut.head + c * chunk_packs * VEC), in + cut.head + c * chunk_packs * VEC,
                       uint32_t(n) * 16, bar);
      }
    }
    if (int(threadIdx.x) < cut.head) copy[threadIdx.x] = in[threadIdx.x];
    if (int(threadIdx.x) < cut.tail) copy[a.vocab - cut.tail + threadIdx.x] = in[a.vocab - cut.tail + threadIdx.x];
  }
  const int64_t wanted = a.targets != nullptr ? a.targets[row] : -1;
  const int target = wanted >= 0 && wanted < a.vocab ? int(wanted) : -1;
  if (threadIdx.x < 32) {
    float entropy;
    const bool live = teacher_row(a, row, p, column, &entropy);
    if (threadIdx.x == 0) { entropy_s = entropy; live_s = live; }
  }
  __syncthreads();
  const bool live = live_s != 0;
  const T* src = CACHED ? copy : in;

  const Powers w = powers(a);
  const bool two = target >= 0 && w.squares != 0;               // a second sum, at temperature one
  Online sums;
  {
    auto one = [&](int i) {
      const float x[1] = {to_float(src[i])};
      sums.add(x, w, two);
    };
    if (int(threadIdx.x) < cut.head) one(threadIdx.x);
    if (int(threadIdx.x) < cut.tail) one(a.vocab - cut.tail + threadIdx.x);
  }
  for (int c = 0; c * chunk_packs < cut.packs; ++c) {
    int first = c * chunk_packs + threadIdx.x, last = min(cut.packs, (c + 1) * chunk_packs);
    if constexpr (CACHED) {
      const uint32_t bar = ptx::smem_u32(&bars[c]);
      if (!ptx::mbar_wait(bar, 0, &abort_flag, a.status, kDistillTimeout, kWaitNs)) {
        // The row never came: no result, and no way out before the copies have ended or the limit is reached.
        if (threadIdx.x == 0) stats[4 * row] = NAN;
        for (; c * chunk_packs < cut.packs; ++c) {
          const uint64_t t0 = ptx::globaltimer_ns();
          while (!ptx::mbar_try_wait(ptx::smem_u32(&bars[c]), 0) && ptx::globaltimer_ns() - t0 < kWaitNs) {}
        }
        return;
      }
    } else {
      last = cut.packs;
    }
    for (int i = first; i < last; i += blockDim.x) {
      const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(src + cut.head + i * VEC);
      float x[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = to_float(v.v[k]);
      sums.add(x, w, two);
    }
    if constexpr (!CACHED) break;
  }
  sums = block_sums(sums, w, two, red);
  const float log_soft = __log2f(sums.soft);

  // Loss, and the named columns' logits before the row may be overwritten.
  const float z_target = target >= 0 ? to_float(src[target]) : 0.f;
  float cross = 0.f;
  for (int i = threadIdx.x; i < a.top; i += blockDim.x) {
    const int c = column[i];
    if (c < 0) continue;
    z[i] = to_float(src[c]);
    cross += p[i] * fmaf(z[i] - sums.m, w.k, -log_soft);
  }
  cross = warp_sum(cross);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = cross;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = 0.f;
    for (int w = 0; w < int(blockDim.x >> 5); ++w) sum += red[w];
    float l = live ? a.temperature * a.temperature * (entropy_s - kLn2 * sum) : 0.f;
    if (target >= 0) l += a.hard_weight * (kLn2 * __log2f(sums.hard) + (sums.m - z_target));
    *reinterpret_cast<float4*>(stats + 4 * row) = make_float4(l, sums.m, sums.soft, sums.hard);
  }
  if (grad == nullptr) return;
  T* out = grad + row * a.vocab;
  const RowGrad g = row_grad(a, live, target >= 0, a.scale, sums.m, sums.soft, sums.hard, w);
  write_gradient(src, cut, out, a.vocab, g);
  __syncthreads();
  write_named(a, out, g, a.temperature * a.scale, a.hard_weight * a.scale, p, column, z, target, z_target);
}

template <typename T>
__global__ void __launch_bounds__(kMaxThreads)
distill_bwd_kernel(const DistillArgs a, const float* __restrict__ stats, const float* __restrict__ grad_out,
                   T* __restrict__ grad) {
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ int live_s;
  const int64_t row = blockIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.vocab;
  const Cut<T> cut(in, a.vocab);
  float* p = reinterpret_cast<float*>(shared);
  int* column = reinterpret_cast<int*>(p + a.top);
  float* z = reinterpret_cast<float*>(column + a.top);
  const int64_t wanted = a.targets != nullptr ? a.targets[row] : -1;
  const int target = wanted >= 0 && wanted < a.vocab ? int(wanted) : -1;
  if (threadIdx.x < 32) {
    float entropy;
    const bool live = teacher_row(a, row, p, column, &entropy);
    if (threadIdx.x == 0) live_s = live;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.top; i += blockDim.x)
    if (column[i] >= 0) z[i] = to_float(in[column[i]]);
  const float z_target = target >= 0 ? to_float(in[target]) : 0.f;
  const float scale = a.scale * *grad_out;
  const float4 st = *reinterpret_cast<const float4*>(stats + 4 * row);
  const RowGrad g = row_grad(a, live_s != 0, target >= 0, scale, st.y, st.z, st.w, powers(a));
  T* out = grad + row * a.vocab;
  write_gradient(in, cut, out, a.vocab, g);
  __syncthreads();
  write_named(a, out, g, a.temperature * scale, a.hard_weight * scale, p, column, z, target, z_target);
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
    Pack<T, VEC> v = reinterpret_cast<Pack<T, VEC>*>(x)[i];
#pragma unroll
    for (int k = 0; k < VEC; ++k) v.v[k] = from_float<T>(to_float(v.v[k]) * f);
    reinterpret_cast<Pack<T, VEC>*>(x)[i] = v;
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

cudaError_t distill_fwd(DType type, const DistillArgs& a, float* stats, void* grad, cudaStream_t stream) {
  if (!valid(a)) return cudaErrorInvalidValue;
  if (a.rows == 0) return cudaSuccess;
  MB_SWITCH_FLOAT(type, T, {
    const int64_t bytes = int64_t(a.vocab) * sizeof(T);
    const int threads = row_threads(bytes);
    const size_t slots = (3 * size_t(a.top) * 4 + 15) / 16 * 16;
    if (grad != nullptr && bytes <= kSharedRow) {
      const size_t shared = slots + size_t(bytes) + 32;
      if (shared > 48 * 1024) {
        const cudaError_t rc = cudaFuncSetAttribute(distill_fwd_kernel<T, true>,
                                                    cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared));
        if (rc != cudaSuccess) return rc;
      }
      distill_fwd_kernel<T, true><<<unsigned(a.rows), threads, shared, stream>>>(a, stats, static_cast<T*>(grad));
    } else {
      distill_fwd_kernel<T, false><<<unsigned(a.rows), threads, slots, stream>>>(a, stats, static_cast<T*>(grad));
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
  const size_t slots = (3 * size_t(a.top) * 4 + 15) / 16 * 16;
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
