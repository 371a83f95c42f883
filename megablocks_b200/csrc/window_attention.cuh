// Pieces that the windowed-attention kernels share.
#pragma once

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace mb {
namespace attn {

using namespace ptx;

constexpr uint64_t kWaitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 splat2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 pair_of(uint32_t lo, uint32_t hi) {
  return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ float2 exp2_pair(float2 x) { return make_float2(exp2_approx(x.x), exp2_approx(x.y)); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

template <typename T>
constexpr bool kIsBf16 = std::is_same<T, __nv_bfloat16>::value;

// Valid tokens of a sequence.
__device__ __forceinline__ int length_of(const Params& p, int b) {
  return p.lengths == nullptr ? p.seq : max(0, min(p.seq, p.lengths[b]));
}

// A value that all lanes have, in a uniform register: what an MMA's descriptors are made of.  From ordinary
// registers each descriptor is moved there again, which took longer than the MMA itself.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// Tiles are stored as D / 64 boxes of [rows][64] 16-bit values with 128-byte swizzle: one layout that
// serves as a K-major operand (contraction along dim) and as an MN-major one (contraction along the rows).
template <int ROWS>
__device__ __forceinline__ uint64_t desc_along_dim(uint32_t tile, int k) {      // k-th 16 of dim
  return smem_desc_sw128(tile, 16, 1024) + (((k >> 2) * (ROWS * 128) + (k & 3) * 32) >> 4);
}
template <int ROWS>
__device__ __forceinline__ uint64_t desc_along_rows(uint32_t tile, int k) {     // k-th 16 of the rows
  return smem_desc_sw128(tile, ROWS * 128, 1024) + ((k * 2048) >> 4);
}

// Rows [first, ROWS) of a tile set to zero by one warp, visible to the tensor cores afterwards: what lies
// behind a sequence's end meets probabilities of zero, and must not be infinite or NaN there.
template <int ROWS, int D>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int first, int lane) {
  for (int i = first * 8 + lane; i < ROWS * 8; i += 32)
#pragma unroll
    for (int box = 0; box < D / 64; ++box)
      *reinterpret_cast<uint4*>(tile + box * (ROWS * 128) + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// Columns 32 c to 32 c + 31 of an array of 32-bit registers.
template <int N>
__device__ __forceinline__ uint32_t (&chunk_of(uint32_t (&r)[N], int c))[32] {
  return *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]);
}

// 32 columns of a thread's row, scaled and rounded, into a staged tile of 128 rows.
template <typename T>
__device__ __forceinline__ void stage_row(uint8_t* tile, int row, int chunk, const uint32_t (&r)[32], float scale) {
  uint8_t* box = tile + (chunk >> 1) * (kTile * 128) + row * 128;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    uint4 q;
    q.x = pack2<T>(__uint_as_float(r[v * 8 + 0]) * scale, __uint_as_float(r[v * 8 + 1]) * scale);
    q.y = pack2<T>(__uint_as_float(r[v * 8 + 2]) * scale, __uint_as_float(r[v * 8 + 3]) * scale);
    q.z = pack2<T>(__uint_as_float(r[v * 8 + 4]) * scale, __uint_as_float(r[v * 8 + 5]) * scale);
    q.w = pack2<T>(__uint_as_float(r[v * 8 + 6]) * scale, __uint_as_float(r[v * 8 + 7]) * scale);
    *reinterpret_cast<uint4*>(box + ((((chunk & 1) * 4 + v) ^ (row & 7)) * 16)) = q;
  }
}

__device__ __forceinline__ void group_barrier(int id) {        // the 128 threads of a row group
  asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory");
}

// Waits of the warp that issues MMAs.  A wait that runs out is recorded; from then on none waits, the loops run
// to their end on whatever is there, in bounds, and the result is not valid.
struct IssueWait {
  volatile int* abort_flag;
  int* status;
  bool dead;
  __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity) {
    if (!dead && !mbar_try_wait(bar, parity))
      dead = !mbar_wait(bar, parity, abort_flag, status, kErrMma, kWaitNs);
    tcgen05_fence_after();
  }
};

// How much of the 32 keys from `k0` on the 32 queries from `i0` on see.
enum Sight { kNone, kSome, kAll };
__device__ __forceinline__ Sight sight(int i0, int k0, int window, int sinks) {
  if (k0 > i0 + 31 || (k0 + 31 <= i0 - window && k0 >= sinks)) return kNone;
  return k0 + 31 <= i0 && (k0 > i0 + 31 - window || k0 + 31 < sinks) ? kAll : kSome;
}

// The keys (bits) of 32 that a row sees: [from, to], and those below `keep` up to `to`.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
__device__ __forceinline__ uint32_t seen_bits(int from, int to, int keep) {
  return bits_below(to + 1) & (~bits_below(from) | bits_below(keep));
}

// A wait that ran out leaves copies and MMAs in flight: give them time before tensor memory is freed.
__device__ __forceinline__ void settle(const volatile int* abort_flag) {
  if (*abort_flag == 0) return;
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
}

}  // namespace attn
}  // namespace mb
