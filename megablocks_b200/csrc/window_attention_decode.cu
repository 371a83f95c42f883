// Windowed attention of one new token per sequence over a key-value cache.
//
//   out = softmax(scale q K^T) V   over the first `sinks` and the last `window` of the valid keys
//
// Bound by the bytes of the visible keys and values.  The keys of a (sequence, key head) are split over a
// cluster of CTAs, each CTA's over its four warps; a warp streams 16 keys at a time through a ring of its own
// (asynchronous copies, no block barrier), takes all query heads that share the key head as the rows of one
// 16-row matrix product, and keeps its own running maximum, sum and output.  Warps are joined in shared
// memory and CTAs over the cluster's shared memory, in a fixed order: one launch, no workspace.  The products
// run on warp-level MMAs: 16 rows would leave the 128-row tensor-memory ones seven eighths empty, and the
// memory sets the pace.
//
// 64 sequences of up to 8192 keys, 32 over 8 heads of 128, window 4096: 170 us, 5.4 TB/s of visible keys and values, 0.82
// of the copy bandwidth; sequences of different lengths end at different times.  One sequence: 12.4 us for 16.8 MB, of
// which the launch of a cluster and the join are 6 and the rest a chain of 16-key steps.
#include <cstdint>

#include "window_attention.cuh"

namespace mb {
namespace attn {

namespace {

constexpr int kStages = 3;             // steps of a warp's ring
constexpr int kKeys = 16;              // keys of a warp's step
constexpr int kRows = 16;              // query heads of a CTA
constexpr int kMaxSplits = 8;          // CTAs of a cluster; 16 of them start 2 us later

// A step of 16 keys takes a warp a microsecond, most of it latency, and eight warps' rings fill an SM: two CTAs
// of four, or one of eight for few sequences, whose CTAs do not fill the SMs.
template <int D, int kWarps>
struct DecodeLayout {
  static constexpr int kPitch = D * 2 + 16;                        // bytes; keeps matrix loads off one another's banks
  static constexpr int kStageBytes = 2 * kKeys * kPitch;           // K, V
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kJoinBytes = kRows * D * 4 + 2 * kRows * 4; // output, maximum, sum of the CTA
  static constexpr int kBytes = kRingBytes + kJoinBytes;
  static_assert(kWarps * (kRows * D * 4 + 2 * kRows * 4) <= kRingBytes && 2 * kMaxSplits * kRows * 4 <= kRingBytes,
                "the warps' results, and later the parts' weights, fit the ring");
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kIsBf16<T>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float remote_float(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(smem_u32(p), rank)));
  return v;
}

// Weight of a part whose maximum is m beside the joint one; parts without a key have m = -inf.
__device__ __forceinline__ float join_weight(float m, float top) { return m == -INFINITY ? 0.f : exp2_approx(m - top); }

template <typename T, int D, int kWarps>
__global__ void __launch_bounds__(kWarps * 32)
window_decode_kernel(const DecodeParams p) {
  using L = DecodeLayout<D, kWarps>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = gridDim.x, split = blockIdx.x;               // a cluster spans x
  const int ratio = p.heads / p.kv_heads, blocks = (ratio + kRows - 1) / kRows;
  const int kv_head = blockIdx.y / blocks, row0 = blockIdx.y % blocks * kRows, b = blockIdx.z;
  const int rows = min(kRows, ratio - row0), head0 = kv_head * ratio + row0;

  const int len = max(0, min(p.capacity, p.lengths[b]));
  const int lo = max(0, len - p.window), first = min(p.sinks, lo);
  const int visible = first + len - lo;
  // This CTA's keys, counted over the visible ones: whole steps of the four warps.
  const int steps = (visible + kWarps * kKeys - 1) / (kWarps * kKeys);
  const int begin = int(int64_t(steps) * split / splits), end = int(int64_t(steps) * (split + 1) / splits);

  const T* kbase = static_cast<const T*>(p.k) + b * p.k_batch + kv_head * p.k_head;
  const T* vbase = static_cast<const T*>(p.v) + b * p.v_batch + kv_head * p.v_head;
  uint8_t* ring = smem + warp * (kStages * L::kStageBytes);
  constexpr int kChunks = D / 8, kAbreast = 32 / kChunks;         // 16-byte pieces of a key; keys a warp copies at once
  const int piece = lane % kChunks, key0 = lane / kChunks;
  const bool inside = piece * 8 < p.dim;
  // Where this lane's piece of visible key 0 would lie, if it were among the last keys.
  const T* kwin = kbase + int64_t(lo - first) * p.k_row + (inside ? piece * 8 : 0);
  const T* vwin = vbase + int64_t(lo - first) * p.v_row + (inside ? piece * 8 : 0);
  auto load = [&](int step) {
    if (step < end) {
      const int base = (step * kWarps + warp) * kKeys;
      const uint32_t dst = smem_u32(ring + (step - begin) % kStages * L::kStageBytes) + key0 * L::kPitch + piece * 16;
      if (base >= first && base + kKeys <= visible) {             // 16 keys in a row, but for few steps
        const T* ks = kwin + int64_t(base + key0) * p.k_row;
        const T* vs = vwin + int64_t(base + key0) * p.v_row;
        const int bytes = inside ? 16 : 0;
#pragma unroll
        for (int i = 0; i < kKeys / kAbreast; ++i) {
          copy16(dst + i * kAbreast * L::kPitch, ks, bytes);
          copy16(dst + (kKeys + i * kAbreast) * L::kPitch, vs, bytes);
          ks += kAbreast * p.k_row;
          vs += kAbreast * p.v_row;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kKeys / kAbreast; ++i) {
          const int at = base + key0 + i * kAbreast;
          const bool there = at < visible && inside;
          const int64_t row = there ? at + (at < first ? first - lo : 0) : first - lo;       // else zeros, nothing is read
          copy16(dst + i * kAbreast * L::kPitch, kwin + row * p.k_row, there ? 16 : 0);
          copy16(dst + (kKeys + i * kAbreast) * L::kPitch, vwin + row * p.v_row, there ? 16 : 0);
        }
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load(begin + s);

  // Queries as A fragments: rows lane / 4 and + 8, columns 2 (lane % 4) and + 8 of each 16.
  uint32_t qf[D / 16][4];
  {
    const T* q = static_cast<const T*>(p.q) + (int64_t(b) * p.heads + head0) * p.dim;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = lane / 4 + (u & 1) * 8, col = i * 16 + (lane % 4) * 2 + (u >> 1) * 8;
        qf[i][u] = row < rows && col < p.dim ? *reinterpret_cast<const uint32_t*>(q + row * p.dim + col) : 0u;
      }
  }
  const float scale = p.scale * kLog2e;
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int u = 0; u < 4; ++u) o[i][u] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

  for (int step = begin; step < end; ++step) {
    load(step + kStages - 1);
    copy_wait<kStages - 1>();
    __syncwarp();
    const uint32_t stage = smem_u32(ring + (step - begin) % kStages * L::kStageBytes);
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      // Two 8-key tiles: matrices (keys 0-7 | 8-15) x (dim 0-7 | 8-15) of the 16.
      const uint4 f = ldmatrix_x4(stage + (lane % 8 + lane / 16 * 8) * L::kPitch + i * 32 + (lane / 8 % 2) * 16);
      mma16816<T>(s[0], qf[i], f.x, f.y);
      mma16816<T>(s[1], qf[i], f.z, f.w);
    }
    const int at = (step * kWarps + warp) * kKeys + (lane % 4) * 2;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        s[n][u] = at + n * 8 + (u & 1) < visible ? s[n][u] * scale : -INFINITY;
        top[u >> 1] = fmaxf(top[u >> 1], s[n][u]);
      }
    float factor[2], base[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      const float now = fmaxf(m[h], top[h]);
      factor[h] = now == m[h] ? 1.f : exp2_approx(m[h] - now);
      m[h] = now;
      base[h] = now == -INFINITY ? 0.f : now;
      sum[h] *= factor[h];
    }
    if (__any_sync(0xffffffffu, factor[0] != 1.f || factor[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) o[i][u] *= factor[u >> 1];
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        s[n][u] = exp2_approx(s[n][u] - base[u >> 1]);
        sum[u >> 1] += s[n][u];
      }
    // Probabilities of 16 keys as one A fragment, rounded to the values' type for the product.
    const uint32_t pf[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]),
                            pack2<T>(s[1][2], s[1][3])};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint4 f = ldmatrix_x4_trans(stage + (kKeys + lane % 16) * L::kPitch + i * 32 + lane / 16 * 16);
      mma16816<T>(o[2 * i], pf, f.x, f.y);
      mma16816<T>(o[2 * i + 1], pf, f.z, f.w);
    }
    __syncwarp();                      // the stage is loaded again by the next step
  }
  copy_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
  }

  // Join the warps, then the CTAs of the cluster.
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);                    // [warp][rows][D], then [warp][2][rows]
  float* part_m = part + kWarps * kRows * D;
  float* joint = reinterpret_cast<float*>(smem + L::kRingBytes);   // [rows][D], maximum[rows], sum[rows]
  float* joint_m = joint + kRows * D;
  float* joint_sum = joint_m + kRows;
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<float2*>(part + (warp * kRows + lane / 4 + h * 8) * D + i * 8 + (lane % 4) * 2) =
          make_float2(o[i][2 * h], o[i][2 * h + 1]);
  if (lane % 4 == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      part_m[(warp * 2) * kRows + lane / 4 + h * 8] = m[h];
      part_m[(warp * 2 + 1) * kRows + lane / 4 + h * 8] = sum[h];
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < rows * D; x += kWarps * 32) {
    const int r = x / D, d = x % D;
    float top = -INFINITY, total = 0.f, value = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_m[w * 2 * kRows + r]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float weight = join_weight(part_m[w * 2 * kRows + r], top);
      total += weight * part_m[(w * 2 + 1) * kRows + r];
      value += weight * part[(w * kRows + r) * D + d];
    }
    joint[x] = value;
    if (d == 0) { joint_m[r] = top; joint_sum[r] = total; }
  }
  cluster_sync_all();
  // Every CTA reads all parts' maxima and sums at once (a remote read takes as long as a few keys), then its share
  // of the outputs.
  float* weight = reinterpret_cast<float*>(smem);                  // [split][rows]; the warps' parts have been read
  float* sums = weight + kMaxSplits * kRows;
  for (int x = threadIdx.x; x < splits * rows; x += kWarps * 32) {
    const int s = x / rows, r = x % rows;
    weight[s * kRows + r] = remote_float(joint_m + r, s);
    sums[s * kRows + r] = remote_float(joint_sum + r, s);
  }
  __syncthreads();
  if (int(threadIdx.x) < rows) {
    const int r = threadIdx.x;
    float top = -INFINITY, total = 0.f;
    for (int s = 0; s < splits; ++s) top = fmaxf(top, weight[s * kRows + r]);
    for (int s = 0; s < splits; ++s) total += join_weight(weight[s * kRows + r], top) * sums[s * kRows + r];
    const float inv = total == 0.f ? 0.f : 1.f / total;            // an idle slot: zeros
    for (int s = 0; s < splits; ++s) weight[s * kRows + r] = join_weight(weight[s * kRows + r], top) * inv;
  }
  __syncthreads();
  T* out = static_cast<T*>(p.out) + (int64_t(b) * p.heads + head0) * p.dim;
  for (int x = split * (kWarps * 32) + threadIdx.x; x < rows * D; x += splits * (kWarps * 32)) {
    const int r = x / D, d = x % D;
    if (d >= p.dim) continue;
    float value = 0.f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) value = fmaf(weight[s * kRows + r], remote_float(joint + x, s), value);
    out[r * p.dim + d] = from_float<T>(value);
  }
  cluster_sync_all();                  // no CTA leaves while another reads its shared memory
}

template <typename T, int D, int kWarps>
cudaError_t launch_decode(const DecodeParams& p, dim3 grid, cudaStream_t stream) {
  auto kernel = window_decode_kernel<T, D, kWarps>;
  constexpr int bytes = DecodeLayout<D, kWarps>::kBytes;
  static std::atomic<bool> allowed[64];
  const cudaError_t rc = allow_shared(kernel, bytes, allowed);
  if (rc != cudaSuccess) return rc;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(kWarps * 32);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = grid.x;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, p);
}

template <typename T>
cudaError_t launch_decode(const DecodeParams& p, int sms, cudaStream_t stream) {
  const int ratio = p.heads / p.kv_heads, blocks = (ratio + kRows - 1) / kRows;
  const int64_t units = int64_t(p.batch) * p.kv_heads * blocks;
  // The split that ends first: waves of CTAs, each as long as its keys and a start and end that take about as
  // long as 192 keys; no CTA with less than a step of four warps.
  const int64_t keys = int64_t(p.window < p.capacity ? p.window : p.capacity) + p.sinks;
  int splits = 1;
  int64_t best = INT64_MAX;
  for (int s = 1; s <= kMaxSplits && (s == 1 || keys > (s / 2) * 4 * kKeys); s *= 2) {
    const int64_t cost = (units * s + 2 * sms - 1) / (2 * sms) * (keys / s + 192);
    if (cost < best) { best = cost; splits = s; }
  }
  const dim3 grid(splits, p.kv_heads * blocks, p.batch);
  const bool few = units * splits <= sms && keys > splits * 4 * kKeys;
  if (p.dim <= 64) return few ? launch_decode<T, 64, 8>(p, grid, stream) : launch_decode<T, 64, 4>(p, grid, stream);
  return few ? launch_decode<T, 128, 8>(p, grid, stream) : launch_decode<T, 128, 4>(p, grid, stream);
}

}  // namespace

cudaError_t decode(bool bf16, const DecodeParams& p, int sms, cudaStream_t stream) {
  if (p.batch == 0) return cudaSuccess;
  return bf16 ? launch_decode<__nv_bfloat16>(p, sms, stream) : launch_decode<__half>(p, sms, stream);
}

}  // namespace attn
}  // namespace mb
