// Windowed causal attention, forward, on the 5th-generation tensor cores.
//
//   o_i = sum_j softmax_j(scale q_i k_j) v_j   over   j <= i  and  (i - j < window  or  j < sinks)
//
// A CTA owns one or two tiles of 128 queries of a head.  S = Q K^T of a tile of 128 keys lands in tensor
// memory, where a group of 128 threads, one a query, turns it into probabilities in place (16 bits, two to a
// column); they are the A operand of O += P V, whose sum stays in tensor memory for the whole row.  One warp
// loads by TMA, one issues the MMAs.  Two groups share an SM, so that one takes exponentials while the tensor
// cores work for the other: for heads of up to 64 as two CTAs, whose prologues and epilogues overlap as well;
// for larger ones, whose keys and values are twice as many bytes a product, as one CTA that loads them once
// for both.  The running maximum follows a row lazily: O is scaled again only when
// the maximum has grown by 2^8, which leaves probabilities at most 256 times their value and sums in 32 bits.
// Tiles that no query of a group sees are not loaded, and only tiles on the window's edges are masked.
#include "window_attention.cuh"

namespace mb {
namespace attn {

namespace {

constexpr float kLazy = 8.f;

template <int D>
struct Layout {
  static constexpr int kGroups = D == 128 ? 2 : 1;                 // query tiles of a CTA
  static constexpr int kThreads = 64 + kGroups * 128;              // warp 0 loads, warp 1 issues MMAs, the others own rows
  static constexpr int kResident = D == 128 ? 1 : 2;               // CTAs of an SM
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStages = 5;
  static constexpr int kColumns = kGroups * (kTile + D) > 256 ? 512 : 256;
  static constexpr int kBytes = (kGroups + kStages) * kTileBytes + 1024 + 256;
};

// The key tiles of a CTA: first the sinks' tiles before the window, then the window's.
template <int G>
struct Tiles {
  int sink_tiles;                      // tiles that hold a first token
  int lo[G], hi[G];                    // window's tiles of each group; hi < lo: the group has no rows
  int head;                            // sinks' tiles before lo[0]
  int count;
  __device__ __forceinline__ Tiles(const Params& p, int q0, int len) {
    sink_tiles = (p.sinks + kTile - 1) / kTile;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int first = q0 + g * kTile;
      lo[g] = max(0, first - p.window + 1) / kTile;
      hi[g] = first < len ? min(first + kTile, len) - 1 : -1;
      hi[g] = hi[g] < 0 ? -1 : hi[g] / kTile;
    }
    head = min(sink_tiles, lo[0]);
    count = head + max(hi[0], hi[G - 1]) - lo[0] + 1;
  }
  __device__ __forceinline__ int at(int t) const { return t < head ? t : lo[0] + t - head; }
  __device__ __forceinline__ bool wanted(int g, int j) const { return j <= hi[g] && (j >= lo[g] || j < sink_tiles); }
};

// Scores of a row's tile into probabilities, in place.  `m` is the reference of the exponent, `sum` the sum of
// the probabilities; `to` the row's sum in tensor memory, which is scaled when the reference moves.
template <typename T, int D, bool EDGE>
__device__ __forceinline__ void row_tile(uint32_t ts, uint32_t to, float scale, int from, int upto, int keep, bool first,
                                         float& m, float& sum) {
  uint32_t s[kTile];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld_32x32(ts + c * 32, chunk_of(s, c));
  tmem_ld_wait();
  if constexpr (EDGE) {
#pragma unroll
    for (int k = 0; k < kTile; ++k)
      if (!(k <= upto && (k >= from || k < keep))) s[k] = 0xff800000u;        // -infinity
  }
  float top4[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) top4[c] = __uint_as_float(s[c]);
#pragma unroll
  for (int k = 4; k < kTile; k += 4)
#pragma unroll
    for (int c = 0; c < 4; ++c) top4[c] = fmaxf(top4[c], __uint_as_float(s[k + c]));
  const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * scale;
  // The sum of the tile before is complete: its MMAs precede the ones that made these scores.
  const bool grow = top > m + kLazy;
  const float factor = grow ? exp2_approx(m - top) : 1.f;
  if (grow) { m = top; sum *= factor; }
  if (!first && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
    for (int c = 0; c < D / 16; ++c) {
      uint32_t raw[16];
      tmem_ld_32x16(to + c * 16, raw);
      tmem_ld_wait();
#pragma unroll
      for (int x = 0; x < 16; ++x) raw[x] = __float_as_uint(__uint_as_float(raw[x]) * factor);
      tmem_st_32x16(to + c * 16, raw);
    }
  }
  const float2 scale2 = splat2(scale), base2 = splat2(m == -INFINITY ? 0.f : -m);
  float2 part[2] = {splat2(0.f), splat2(0.f)};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t packed[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const float2 e = exp2_pair(__ffma2_rn(pair_of(s[c * 32 + 2 * x], s[c * 32 + 2 * x + 1]), scale2, base2));
      part[x & 1] = __fadd2_rn(part[x & 1], e);
      packed[x] = pack2<T>(e.x, e.y);  // 8 or 11 bits for the product; the sum takes them whole
    }
    tmem_st_32x16(ts + c * 16, packed);                // over scores that this thread has read
  }
  part[0] = __fadd2_rn(part[0], part[1]);
  sum += part[0].x + part[0].y;
  tmem_st_wait();
}

template <typename T, int D>
__global__ void __launch_bounds__(Layout<D>::kThreads, Layout<D>::kResident)
window_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
                  const __grid_constant__ CUtensorMap map_low, const __grid_constant__ Params p) {
  using L = Layout<D>;
  constexpr int kTileBytes = L::kTileBytes, kStages = L::kStages, G = L::kGroups;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tile_q = smem;
  uint8_t* ring = smem + G * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kStages * kTileBytes);
  uint64_t* full = bars;
  uint64_t* empty = bars + kStages;
  uint64_t* q_full = bars + 2 * kStages;           // [G]
  uint64_t* s_full = q_full + G;                   // [G] scores of a group are in tensor memory
  uint64_t* p_full = s_full + G;                   // [G] its probabilities are
  uint64_t* o_full = p_full + G;                   // [G] its sum is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + G);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q0 = blockIdx.x * G * kTile, head = blockIdx.y, b = blockIdx.z;
  const int kv_head = head / (p.heads / p.kv_heads);
  const int len = length_of(p, b);
  const Tiles<G> tiles(p, q0, len);

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int g = 0; g < G; ++g) {
      mbar_init(smem_u32(&q_full[g]), 1);
      mbar_init(smem_u32(&s_full[g]), 1);
      mbar_init(smem_u32(&p_full[g]), 4);
      mbar_init(smem_u32(&o_full[g]), 1);
    }
    fence_barrier_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), L::kColumns);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_s = tmem, tmem_o = tmem + G * kTile;        // S of group g at g * 128, O behind them at g * D

  if (warp == 0) {
    // ---- loader ----------------------------------------------------------------------------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      auto load_q = [&](int g) {
        const uint32_t bar = smem_u32(&q_full[g]);
        mbar_arrive_expect_tx(bar, kTileBytes);
        for (int box = 0; box < D / 64; ++box)
          tma_load_4d(smem_u32(tile_q + g * kTileBytes + box * (kTile * 128)), &map_q, bar, box * 64, q0 + g * kTile,
                      head, b);
      };
      if (tiles.hi[0] >= 0) load_q(0);
      for (int t = 0; t < 2 * tiles.count; ++t) {                   // K and V of a tile take turns
        if (!mbar_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.status, kErrLoad, kWaitNs)) break;
        const uint32_t bar = smem_u32(&full[stage]);
        mbar_arrive_expect_tx(bar, kTileBytes);
        for (int box = 0; box < D / 64; ++box)
          tma_load_4d(smem_u32(ring + stage * kTileBytes + box * (kTile * 128)), (t & 1) ? &map_v : &map_k, bar,
                      box * 64, tiles.at(t >> 1) * kTile, kv_head, b);
        if (t == 0 && G > 1 && tiles.hi[G - 1] >= 0) load_q(G - 1);
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issuer ------------------------------------------------------------------------------
    constexpr uint32_t idesc_s = instr_desc_f16(kIsBf16<T>, false, false, kTile, kTile);
    constexpr uint32_t idesc_o = instr_desc_f16(kIsBf16<T>, false, true, kTile, D);
    const uint32_t q_base = uniform(smem_u32(tile_q)), ring_base = uniform(smem_u32(ring)), ts = uniform(tmem_s),
                   to = uniform(tmem_o);
    int stage = 0;
    uint32_t phase = 0, p_phase[G] = {};
    bool started[G] = {}, ok = true;
    auto next = [&] {
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && mbar_wait(smem_u32(bar), parity, abort_flag, p.status, kErrMma, kWaitNs);
      ok = __all_sync(0xffffffffu, ok);
      tcgen05_fence_after();
    };
    auto scores = [&](int g) {         // S_g = Q_g K^T with K in the current stage
      if (elect_one()) {
        const uint32_t q = q_base + g * kTileBytes, k = ring_base + stage * kTileBytes;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          umma_f16(ts + g * kTile, desc_along_dim<kTile>(q, i), desc_along_dim<kTile>(k, i), idesc_s, i != 0);
        umma_commit(smem_u32(&s_full[g]));
      }
      __syncwarp();
    };
    if (tiles.count > 0) {
      wait(&full[stage], phase);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (!ok || !tiles.wanted(g, tiles.at(0))) continue;
        wait(&q_full[g], 0);
        if (ok) scores(g);
      }
      if (ok && elect_one()) umma_commit(smem_u32(&empty[stage]));
      __syncwarp();
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
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (ok && tiles.wanted(g, j)) {
          wait(&p_full[g], p_phase[g]);
          p_phase[g] ^= 1u;
          if (ok && elect_one()) {
            const uint32_t v = ring_base + v_stage * kTileBytes;
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
              umma_f16_ta(to + g * D, ts + g * kTile + i * 8, desc_along_rows<kTile>(v, i), idesc_o,
                          started[g] || i != 0);
            if (j == tiles.hi[g]) umma_commit(smem_u32(&o_full[g]));
          }
          __syncwarp();
          started[g] = true;
        }
        if (ok && more && tiles.wanted(g, tiles.at(t + 1))) {
          if (!started[g]) wait(&q_full[g], 0);
          if (ok) scores(g);
        }
      }
      if (ok && elect_one()) {
        umma_commit(smem_u32(&empty[v_stage]));
        if (more) umma_commit(smem_u32(&empty[stage]));
      }
      __syncwarp();
      if (more) next();
    }
  } else {
    // ---- rows ------------------------------------------------------------------------------------
    const int g = (warp - 2) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane, g0 = q0 + g * kTile, i = g0 + r;       // this thread's query
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t ts = tmem_s + g * kTile + lanes, to = tmem_o + g * D + lanes;
    const float scale = p.scale * kLog2e;
    float m = -INFINITY, sum = 0.f;    // reference of the exponent (scaled), sum of the probabilities
    uint32_t s_phase = 0;
    bool ok = true, first = true;
    const int lo = G > 1 && g > 0 ? tiles.lo[G - 1] : tiles.lo[0], hi = G > 1 && g > 0 ? tiles.hi[G - 1] : tiles.hi[0];
    const bool rows = hi >= 0;
    for (int t = 0; t < tiles.count && ok; ++t) {
      const int j = tiles.at(t);
      if (!(j <= hi && (j >= lo || j < tiles.sink_tiles))) continue;
      ok = mbar_wait(smem_u32(&s_full[g]), s_phase, abort_flag, p.status, kErrRows, kWaitNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      s_phase ^= 1u;
      tcgen05_fence_after();
      // Visible keys of this row in the tile: from the window's first to its own, and the first tokens.
      const int k0 = j * kTile, upto = i - k0, from = upto - p.window + 1, keep = p.sinks - k0;
      if (k0 + kTile - 1 > g0 || g0 + kTile - 1 - k0 >= p.window)
        row_tile<T, D, true>(ts, to, scale, from, upto, keep, first, m, sum);
      else
        row_tile<T, D, false>(ts, to, scale, from, upto, keep, first, m, sum);
      first = false;
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&p_full[g]));
    }
    if (rows && ok) {
      ok = mbar_wait(smem_u32(&o_full[g]), 0, abort_flag, p.status, kErrRows, kWaitNs);
      ok = __all_sync(0xffffffffu, ok);
      tcgen05_fence_after();
    }
    const bool live = rows && i < len && ok;
    const float inv = live ? 1.f / sum : 0.f;
    if (p.neg_lse != nullptr && i < p.seq_pad)
      p.neg_lse[(int64_t(b) * p.heads + head) * p.seq_pad + i] = live ? -(m + __log2f(sum)) : -INFINITY;
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
      if (quarter == 0 && lane == 0 && g0 < p.seq) {
        for (int box = 0; box < D / 64; ++box)
          if (box * 64 < p.dim)
            tma_store_4d(part == 0 ? &map_o : &map_low, smem_u32(staged + box * (kTile * 128)), box * 64, g0, head, b);
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
    tmem_dealloc(tmem, L::kColumns);
  }
}

template <typename T, int D>
cudaError_t launch_forward(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& out,
                           const CUtensorMap& low, const Params& p, cudaStream_t stream) {
  auto kernel = window_fwd_kernel<T, D>;
  const cudaError_t rc = allow_shared(kernel, Layout<D>::kBytes);
  if (rc != cudaSuccess) return rc;
  constexpr int rows = Layout<D>::kGroups * kTile;
  const dim3 grid((p.seq + rows - 1) / rows, p.heads, p.batch);
  kernel<<<grid, Layout<D>::kThreads, Layout<D>::kBytes, stream>>>(q, k, v, out, low, p);
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
