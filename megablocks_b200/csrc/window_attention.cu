// Windowed causal attention, forward, on the 5th-generation tensor cores.
//
//   o_i = sum_j softmax_j(scale q_i k_j) v_j   over   j <= i  and  (i - j < window  or  j < sinks)
//
// A CTA owns 256 queries of one head as two tiles of 128.  S = Q K^T of a tile of 128 keys lands in tensor
// memory, where a group of 128 threads, one a query, turns it into probabilities in place (16 bits, two to a
// column); they are the A operand of O += P V, whose sum stays in tensor memory for the whole row.  The two
// groups alternate, so that one takes exponentials while the tensor cores work for the other.  One warp
// loads by TMA, one issues the MMAs.  The running maximum follows a row lazily: O is scaled again only when
// the maximum has grown by 2^8, which leaves probabilities at most 256 times their value and sums in 32 bits.
// Tiles that no query of a group sees are not loaded, and only tiles on the window's edges are masked.
#include "window_attention.cuh"

namespace mb {
namespace attn {

namespace {

constexpr int kThreads = 384;          // warp 0 loads, warp 1 issues MMAs, warps 4-7 and 8-11 own the rows
constexpr float kLazy = 8.f;

template <int D>
struct Layout {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kBytes = (2 + kStages) * kTileBytes + 1024 + 256;
};

// The key tiles of a CTA: first the sinks' tiles before the window, then the window's.
struct Tiles {
  int sink_tiles;                      // tiles that hold a first token
  int lo[2], hi[2];                    // window's tiles of each group; hi < lo: the group has no rows
  int head;                            // sinks' tiles before lo[0]
  int count;
  __device__ __forceinline__ Tiles(const Params& p, int q0, int len) {
    sink_tiles = (p.sinks + kTile - 1) / kTile;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int first = q0 + g * kTile;
      lo[g] = max(0, first - p.window + 1) / kTile;
      hi[g] = first < len ? min(first + kTile, len) - 1 : -1;
      hi[g] = hi[g] < 0 ? -1 : hi[g] / kTile;
    }
    head = min(sink_tiles, lo[0]);
    count = head + max(hi[0], hi[1]) - lo[0] + 1;
  }
  __device__ __forceinline__ int at(int t) const { return t < head ? t : lo[0] + t - head; }
  __device__ __forceinline__ bool wanted(int g, int j) const { return j <= hi[g] && (j >= lo[g] || j < sink_tiles); }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
window_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
                  const __grid_constant__ CUtensorMap map_low, const __grid_constant__ Params p) {
  using L = Layout<D>;
  constexpr int kTileBytes = L::kTileBytes, kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tile_q = smem;
  uint8_t* ring = smem + 2 * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kStages * kTileBytes);
  uint64_t* full = bars;
  uint64_t* empty = bars + kStages;
  uint64_t* q_full = bars + 2 * kStages;           // [2]
  uint64_t* s_full = q_full + 2;                   // [2] scores of a group are in tensor memory
  uint64_t* p_full = s_full + 2;                   // [2] its probabilities are
  uint64_t* o_full = p_full + 2;                   // [2] its sum is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q0 = blockIdx.x * 2 * kTile, head = blockIdx.y, b = blockIdx.z;
  const int kv_head = head / (p.heads / p.kv_heads);
  const int len = length_of(p, b);
  const Tiles tiles(p, q0, len);

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(smem_u32(&q_full[g]), 1);
      mbar_init(smem_u32(&s_full[g]), 1);
      mbar_init(smem_u32(&p_full[g]), 4);
      mbar_init(smem_u32(&o_full[g]), 1);
    }
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), 512);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_s = tmem, tmem_o = tmem + 2 * kTile;        // S of group g at g * 128, O at 256 + g * D

  if (warp == 0) {
    // ---- loader ----------------------------------------------------------------------------------
    if (lane == 0) {
      for (int g = 0; g < 2; ++g) {
        if (tiles.hi[g] < 0) continue;
        const uint32_t bar = smem_u32(&q_full[g]);
        mbar_arrive_expect_tx(bar, kTileBytes);
        for (int box = 0; box < D / 64; ++box)
          tma_load_4d(smem_u32(tile_q + g * kTileBytes + box * (kTile * 128)), &map_q, bar, box * 64, q0 + g * kTile,
                      head, b);
      }
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = 0; t < 2 * tiles.count && ok; ++t) {             // K and V of a tile take turns
        ok = mbar_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.status, kErrLoad, kWaitNs);
        if (!ok) break;
        const uint32_t bar = smem_u32(&full[stage]);
        mbar_arrive_expect_tx(bar, kTileBytes);
        for (int box = 0; box < D / 64; ++box)
          tma_load_4d(smem_u32(ring + stage * kTileBytes + box * (kTile * 128)), (t & 1) ? &map_v : &map_k, bar,
                      box * 64, tiles.at(t >> 1) * kTile, kv_head, b);
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issuer ------------------------------------------------------------------------------
    constexpr uint32_t idesc_s = instr_desc_f16(kIsBf16<T>, false, false, kTile, kTile);
    constexpr uint32_t idesc_o = instr_desc_f16(kIsBf16<T>, false, true, kTile, D);
    int stage = 0;
    uint32_t phase = 0, p_phase[2] = {0, 0};
    bool started[2] = {false, false}, ok = true;
    auto next = [&] {
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && mbar_wait(smem_u32(bar), parity, abort_flag, p.status, kErrMma, kWaitNs);
      ok = __all_sync(0xffffffffu, ok);
      tcgen05_fence_after();
    };
    auto scores = [&](int g) {         // S_g = Q_g K^T with K in the current stage
      if (lane == 0) {
        const uint32_t q = smem_u32(tile_q + g * kTileBytes), k = smem_u32(ring + stage * kTileBytes);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          umma_f16(tmem_s + g * kTile, desc_along_dim<kTile>(q, i), desc_along_dim<kTile>(k, i), idesc_s, i != 0);
        umma_commit(smem_u32(&s_full[g]));
      }
      __syncwarp();
    };
    if (tiles.count > 0) {
      wait(&full[stage], phase);
      for (int g = 0; g < 2 && ok; ++g) {
        if (!tiles.wanted(g, tiles.at(0))) continue;
        wait(&q_full[g], 0);
        if (ok) scores(g);
      }
      if (lane == 0 && ok) umma_commit(smem_u32(&empty[stage]));
      next();
    }
    for (int t = 0; t < tiles.count && ok; ++t) {
      const int j = tiles.at(t);
      const int v_stage = stage;
      wait(&full[v_stage], phase);
      if (!ok) break;
      if ((j + 1) * kTile > len)
        zero_rows<kTile, D>(ring + v_stage * kTileBytes, len - j * kTile, lane);
      next();
      const bool more = t + 1 < tiles.count;
      if (more) wait(&full[stage], phase);
      for (int g = 0; g < 2 && ok; ++g) {
        if (tiles.wanted(g, j)) {
          wait(&p_full[g], p_phase[g]);
          p_phase[g] ^= 1u;
          if (!ok) break;
          if (lane == 0) {
            const uint32_t v = smem_u32(ring + v_stage * kTileBytes);
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
              umma_f16_ta(tmem_o + g * D, tmem_s + g * kTile + i * 8, desc_along_rows<kTile>(v, i), idesc_o,
                          started[g] || i != 0);
            if (j == tiles.hi[g]) umma_commit(smem_u32(&o_full[g]));
          }
          __syncwarp();
          started[g] = true;
        }
        if (more && tiles.wanted(g, tiles.at(t + 1))) {
          if (!started[g]) wait(&q_full[g], 0);
          if (ok) scores(g);
        }
      }
      if (lane == 0 && ok) {
        umma_commit(smem_u32(&empty[v_stage]));
        if (more) umma_commit(smem_u32(&empty[stage]));
      }
      __syncwarp();
      if (more) next();
    }
  } else if (warp >= 4) {
    // ---- rows ------------------------------------------------------------------------------------
    const int g = (warp - 4) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane, i = q0 + g * kTile + r;    // this thread's query
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t ts = tmem_s + g * kTile + lanes, to = tmem_o + g * D + lanes;
    const float scale = p.scale * kLog2e;
    float m = -INFINITY, sum = 0.f;    // reference of the exponent (scaled), sum of the probabilities
    uint32_t s_phase = 0;
    bool ok = true, first = true;
    const bool rows = tiles.hi[g] >= 0;
    if (rows) {
      for (int t = 0; t < tiles.count && ok; ++t) {
        const int j = tiles.at(t);
        if (!tiles.wanted(g, j)) continue;
        ok = mbar_wait(smem_u32(&s_full[g]), s_phase, abort_flag, p.status, kErrRows, kWaitNs);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        s_phase ^= 1u;
        tcgen05_fence_after();
        const int k0 = j * kTile, g0 = q0 + g * kTile;
        // Visible keys of this row in the tile: [from, to) of the window, and the first tokens.
        const bool edge = k0 + kTile - 1 > g0 || g0 + kTile - 1 - k0 >= p.window;
        const int upto = i - k0, from = i - p.window + 1 - k0, keep = p.sinks - k0;
        uint32_t raw[32];
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          tmem_ld_32x32(ts + c * 32, raw);
          tmem_ld_wait();
          if (edge) {
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              const int k = c * 32 + x;
              if (k <= upto && (k >= from || k < keep)) top = fmaxf(top, __uint_as_float(raw[x]));
            }
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) top = fmaxf(top, __uint_as_float(raw[x]));
          }
        }
        top *= scale;
        // The sum of the tile before is complete: its MMAs precede the ones that made these scores.
        const bool grow = top > m + kLazy;
        const float factor = grow ? exp2_approx(m - top) : 1.f;
        if (grow) { m = top; sum *= factor; }
        if (!first && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            tmem_ld_32x32(to + c * 32, raw);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; ++x) raw[x] = __float_as_uint(__uint_as_float(raw[x]) * factor);
            tmem_st_32x32(to + c * 32, raw);
          }
        }
        first = false;
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          tmem_ld_32x32(ts + c * 32, raw);
          tmem_ld_wait();
          uint32_t packed[16];
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            float e0 = exp2_approx(fmaf(__uint_as_float(raw[x]), scale, -base));
            float e1 = exp2_approx(fmaf(__uint_as_float(raw[x + 1]), scale, -base));
            if (edge) {
              const int k = c * 32 + x;
              if (!(k <= upto && (k >= from || k < keep))) e0 = 0.f;
              if (!(k + 1 <= upto && (k + 1 >= from || k + 1 < keep))) e1 = 0.f;
            }
            sum += e0 + e1;
            packed[x / 2] = pack2<T>(e0, e1);
          }
          tmem_st_32x16(ts + c * 16, packed);         // over scores that this thread has read
        }
        tmem_st_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[g]));
      }
      if (ok) {
        ok = mbar_wait(smem_u32(&o_full[g]), 0, abort_flag, p.status, kErrRows, kWaitNs);
        ok = __all_sync(0xffffffffu, ok);
        tcgen05_fence_after();
      }
    }
    const bool live = rows && i < len && ok;
    const float inv = live ? 1.f / sum : 0.f;
    if (p.lse != nullptr)
      p.lse[(int64_t(b) * p.heads + head) * p.seq_pad + i] = live ? m + __log2f(sum) : INFINITY;
    // The result, and for a backward pass what its rounding left (the row sums delta want it), one after the
    // other through the queries' tile, which has been used.
    uint8_t* staged = tile_q + g * kTileBytes;
    for (int part = 0; part < (p.out_low != nullptr ? 2 : 1); ++part) {
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t raw[32];
        if (rows && ok) {
          tmem_ld_32x32(to + c * 32, raw);
          tmem_ld_wait();
        }
#pragma unroll
        for (int x = 0; x < 32; ++x) {                // zeros behind the end, whatever was computed there
          float o = live ? __uint_as_float(raw[x]) * inv : 0.f;
          if (part == 1) o -= to_float(from_float<T>(o));
          raw[x] = __float_as_uint(o);
        }
        stage_row<T>(staged, r, c, raw, 1.f);
      }
      fence_proxy_async_smem();
      group_barrier(1 + g);
      if (quarter == 0 && lane == 0 && q0 + g * kTile < p.seq) {
        for (int box = 0; box < D / 64; ++box)
          if (box * 64 < p.dim)
            tma_store_4d(part == 0 ? &map_o : &map_low, smem_u32(staged + box * (kTile * 128)), box * 64,
                         q0 + g * kTile, head, b);
        bulk_commit_group();
        bulk_wait_read_all();
      }
      group_barrier(1 + g);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    settle(abort_flag);
    tcgen05_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D>
cudaError_t launch_forward(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& out,
                           const CUtensorMap& low, const Params& p, cudaStream_t stream) {
  auto kernel = window_fwd_kernel<T, D>;
  const cudaError_t rc = allow_shared(kernel, Layout<D>::kBytes);
  if (rc != cudaSuccess) return rc;
  const dim3 grid((p.seq + 2 * kTile - 1) / (2 * kTile), p.heads, p.batch);
  kernel<<<grid, kThreads, Layout<D>::kBytes, stream>>>(q, k, v, out, low, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t forward(bool bf16, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                    const CUtensorMap& out, const CUtensorMap& low, const Params& p, cudaStream_t stream) {
  if (p.dim <= 64)
    return bf16 ? launch_forward<__nv_bfloat16, 64>(q, k, v, out, low, p, stream)
                : launch_forward<__half, 64>(q, k, v, out, low, p, stream);
  return bf16 ? launch_forward<__nv_bfloat16, 128>(q, k, v, out, low, p, stream)
              : launch_forward<__half, 128>(q, k, v, out, low, p, stream);
}

}  // namespace attn
}  // namespace mb
