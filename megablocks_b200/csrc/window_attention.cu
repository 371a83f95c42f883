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
// Tiles that no query of a group sees are not loaded.  Within a tile a warp takes 32 keys at a time: those that
// none of its queries sees cost it nothing, and only those on an edge are masked.  The product with V starts
// on the first half of a tile's probabilities while the second half is taken.
//
// Time, and rate of the visible pairs' products (4 dim operations each):
//   1 x 16384 tokens, 32 query heads over 8 key heads of 128, window 4096: 0.97 ms at 1965 MHz, 990 TFLOP/s, 0.61 of
//     cuBLAS's burst (pass after pass 0.99 ms, at the 1665 MHz that the power limit leaves); tensor cores busy 0.51 of the
//     time, exponential unit 0.53: the products' operands from shared memory take about as long
//   1 x 8191, the same heads, window 1024: 208 us, 620 TFLOP/s; prologue and epilogue are a quarter of a CTA
//   6 x up to 1999, 16 over 4 heads of 96, window 512: 94 us
//   8 x 1024, 12 heads of 64, window 256: 37 us, 155 TFLOP/s, 1.7 TB/s; three or four tiles a CTA, half of them
//     edges, so that prologue, epilogue and hidden pairs are most of it (tensor cores busy 0.16 of the time)
// CTAs that start in the order of their lengths ended 8 % sooner than in the order of memory on the last three.
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

// Running reference of a row's exponent (scaled) and sum of its probabilities.  The sum in tensor memory, `to`,
// is scaled when the reference moves; it is complete, its MMAs precede the ones that made the scores at hand.
struct RowState {
  float m = -INFINITY, sum = 0.f;
  template <int D>
  __device__ __forceinline__ void follow(float top, uint32_t to, bool first) {
    const bool grow = top > m + kLazy;
    const bool scale = grow && m != -INFINITY;         // without a key so far the sums are zero
    const float factor = scale ? exp2_approx(m - top) : 1.f;
    if (grow) m = top;
    sum *= factor;
    if (first || !__any_sync(0xffffffffu, scale)) return;
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
};

__device__ __forceinline__ float chunk_max(const uint32_t (&s)[32]) {
  float top[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) top[x] = __uint_as_float(s[x]);
#pragma unroll
  for (int k = 4; k < 32; k += 4)
#pragma unroll
    for (int x = 0; x < 4; ++x) top[x] = fmaxf(top[x], __uint_as_float(s[k + x]));
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// Probabilities of 32 scores, rounded over them to 8 or 11 bits for the product; the sum takes them whole.
template <typename T>
__device__ __forceinline__ void chunk_exp(const uint32_t (&s)[32], uint32_t out, float2 scale2, float2 base2,
                                          float2 (&part)[2]) {
  uint32_t packed[16];
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const float2 e = exp2_pair(__ffma2_rn(pair_of(s[2 * x], s[2 * x + 1]), scale2, base2));
    part[x & 1] = __fadd2_rn(part[x & 1], e);
    packed[x] = pack2<T>(e.x, e.y);
  }
  tmem_st_32x16(out, packed);
}

__device__ __forceinline__ void arrive_stored(uint32_t bar, int lane) {
  tmem_st_wait();
  tcgen05_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// Scores of a row's tile into probabilities, in place; `half_done` and `done` get the warp's arrivals.
template <typename T, int D>
__device__ __forceinline__ void row_tile(uint32_t ts, uint32_t to, float scale, int lane, bool first, RowState& row,
                                         uint32_t half_done, uint32_t done) {
  uint32_t s[kTile];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld_32x32(ts + c * 32, chunk_of(s, c));
  tmem_ld_wait();
  const float top = fmaxf(fmaxf(chunk_max(chunk_of(s, 0)), chunk_max(chunk_of(s, 1))),
                          fmaxf(chunk_max(chunk_of(s, 2)), chunk_max(chunk_of(s, 3))));
  row.follow<D>(top * scale, to, first);
  const float2 scale2 = splat2(scale), base2 = splat2(row.m == -INFINITY ? 0.f : -row.m);
  float2 part[2] = {splat2(0.f), splat2(0.f)};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    chunk_exp<T>(chunk_of(s, c), ts + c * 16, scale2, base2, part);
    if (c & 1) arrive_stored(c == 1 ? half_done : done, lane);
  }
  part[0] = __fadd2_rn(part[0], part[1]);
  row.sum += part[0].x + part[0].y;
}

// The same for a tile on an edge: 32 keys at a time, those left out that none of the warp's queries (`i0` and 31
// more) sees of the keys from `k0` on.  The scores are read twice instead of being kept.
template <typename T, int D>
__device__ __forceinline__ void row_edge_tile(uint32_t ts, uint32_t to, float scale, int i0, int k0, const Params& p,
                                              int lane, bool first, RowState& row, uint32_t half_done, uint32_t done) {
  const int upto = i0 + lane - k0, from = upto - p.window + 1, keep = p.sinks - k0;
  uint32_t s[32];
  auto load = [&](int c, Sight seen) {
    tmem_ld_32x32(ts + c * 32, s);
    tmem_ld_wait();
    if (seen == kAll) return;
    const uint32_t bits = seen_bits(from - c * 32, upto - c * 32, keep - c * 32);
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (!(bits & (1u << k))) s[k] = 0xff800000u;    // -infinity
  };
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const Sight seen = sight(i0, k0 + c * 32, p.window, p.sinks);
    if (seen == kNone) continue;
    load(c, seen);
    top = fmaxf(top, chunk_max(s));
  }
  row.follow<D>(top * scale, to, first);
  const float2 scale2 = splat2(scale), base2 = splat2(row.m == -INFINITY ? 0.f : -row.m);
  float2 part[2] = {splat2(0.f), splat2(0.f)};
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const Sight seen = sight(i0, k0 + c * 32, p.window, p.sinks);
    if (seen == kNone) {
      const uint32_t zeros[16] = {};
      tmem_st_32x16(ts + c * 16, zeros);
    } else {
      load(c, seen);
      chunk_exp<T>(s, ts + c * 16, scale2, base2, part);
    }
    if (c & 1) arrive_stored(c == 1 ? half_done : done, lane);
  }
  part[0] = __fadd2_rn(part[0], part[1]);
  row.sum += part[0].x + part[0].y;
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
  uint64_t* p_half = s_full + G;                   // [G] half its probabilities are
  uint64_t* p_full = p_half + G;                   // [G] all are
  uint64_t* o_full = p_full + G;                   // [G] its sum is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + G);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Heads fastest and the last queries, which see the most keys, first, so that short CTAs end the launch.
  const int head = blockIdx.x % p.heads, b = blockIdx.x / p.heads;
  const int q0 = int(gridDim.y - 1 - blockIdx.y) * G * kTile;
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
      mbar_init(smem_u32(&p_half[g]), 4);
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
    const uint32_t bar0 = uniform(smem_u32(bars));                          // full[], empty[], then the groups'
    auto bar_of = [&](const uint64_t* bar) { return bar0 + uint32_t(bar - bars) * 8; };
    IssueWait wait{abort_flag, p.status, false};
    int stage = 0;
    uint32_t phase = 0, p_phase = 0;                                        // p_phase: a bit a group
    bool started[G] = {};
    auto next = [&] {
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    };
    auto scores = [&](int g) {         // S_g = Q_g K^T with K in the current stage
      if (elect_one()) {
        const uint32_t q = q_base + g * kTileBytes, k = ring_base + stage * kTileBytes;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          umma_f16(ts + g * kTile, desc_along_dim<kTile>(q, i), desc_along_dim<kTile>(k, i), idesc_s, i != 0);
        umma_commit(bar_of(&s_full[g]));
      }
      __syncwarp();
    };
    if (tiles.count > 0) {
      wait(bar_of(&full[stage]), phase);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (!tiles.wanted(g, tiles.at(0))) continue;
        wait(bar_of(&q_full[g]), 0);
        scores(g);
      }
      if (elect_one()) umma_commit(bar_of(&empty[stage]));
      __syncwarp();
      next();
    }
    for (int t = 0; t < tiles.count; ++t) {
      const int j = tiles.at(t), j_next = tiles.at(t + 1);
      const int v_stage = stage;
      const bool more = t + 1 < tiles.count;
      wait(bar_of(&full[v_stage]), phase);
      if ((j + 1) * kTile > len)
        zero_rows<kTile, D>(ring + v_stage * kTileBytes, len - j * kTile, lane);
      next();
      const uint32_t v = ring_base + v_stage * kTileBytes;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (tiles.wanted(g, j)) {
          auto product = [&](int from) {
#pragma unroll
            for (int i = from; i < from + kTile / 32; ++i)
              umma_f16_ta(to + g * D, ts + g * kTile + i * 8, desc_along_rows<kTile>(v, i), idesc_o, started[g] || i != 0);
          };
          wait(bar_of(&p_half[g]), (p_phase >> g) & 1u);
          if (elect_one()) product(0);
          __syncwarp();
          wait(bar_of(&p_full[g]), (p_phase >> g) & 1u);
          if (elect_one()) {
            product(kTile / 32);
            if (j == tiles.hi[g]) umma_commit(bar_of(&o_full[g]));
          }
          __syncwarp();
          p_phase ^= 1u << g;
          started[g] = true;
        }
        if (more && tiles.wanted(g, j_next)) {
          if (!started[g]) wait(bar_of(&q_full[g]), 0);
          wait(bar_of(&full[stage]), phase);           // passes at once for the second group
          scores(g);
        }
      }
      if (elect_one()) {
        umma_commit(bar_of(&empty[v_stage]));
        if (more) umma_commit(bar_of(&empty[stage]));
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
    RowState row;
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
      const int i0 = g0 + quarter * 32, k0 = j * kTile;
      const uint32_t half_done = smem_u32(&p_half[g]), done = smem_u32(&p_full[g]);
      if (k0 + kTile - 1 <= i0 && k0 > i0 + 31 - p.window)         // the whole tile in the window
        row_tile<T, D>(ts, to, scale, lane, first, row, half_done, done);
      else
        row_edge_tile<T, D>(ts, to, scale, i0, k0, p, lane, first, row, half_done, done);
      first = false;
    }
    if (rows && ok) {
      ok = mbar_wait(smem_u32(&o_full[g]), 0, abort_flag, p.status, kErrRows, kWaitNs);
      ok = __all_sync(0xffffffffu, ok);
      tcgen05_fence_after();
    }
    const bool live = rows && i < len && ok;
    const float inv = live ? 1.f / row.sum : 0.f;
    if (p.neg_lse != nullptr && i < p.seq_pad)
      p.neg_lse[(int64_t(b) * p.heads + head) * p.seq_pad + i] = live ? -(row.m + __log2f(row.sum)) : -INFINITY;
    // The result goes out through the queries' tile, which has been used.  What its rounding left, which the
    // backward pass wants for its row sums, goes through the ring where it is free (one group has no other to
    // wait for), else through the same tile afterwards.
    uint8_t* staged = tile_q + g * kTileBytes;
    const bool low = p.out_low != nullptr;
    constexpr int kPasses = G == 1 ? 1 : 2;
    for (int pass = 0; pass < (low ? kPasses : 1); ++pass) {
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t raw[32], rest[32];
        if (rows && ok) {
          tmem_ld_32x32(to + c * 32, raw);
          tmem_ld_wait();
        }
#pragma unroll
        for (int x = 0; x < 32; ++x) {                // zeros behind the end, whatever was computed there
          const float o = live ? __uint_as_float(raw[x]) * inv : 0.f;
          raw[x] = __float_as_uint(o);
          rest[x] = __float_as_uint(o - to_float(from_float<T>(o)));
        }
        if (pass == 0) stage_row<T>(staged, r, c, raw, 1.f);
        if (low && pass == kPasses - 1) stage_row<T>(G == 1 ? ring : staged, r, c, rest, 1.f);
      }
      fence_proxy_async_smem();
      group_barrier(1 + g);
      if (quarter == 0 && lane == 0 && g0 < p.seq) {
        for (int box = 0; box < D / 64; ++box) {
          if (box * 64 >= p.dim) continue;
          if (pass == 0) tma_store_4d(&map_o, smem_u32(staged + box * (kTile * 128)), box * 64, g0, head, b);
          if (low && pass == kPasses - 1)
            tma_store_4d(&map_low, smem_u32((G == 1 ? ring : staged) + box * (kTile * 128)), box * 64, g0, head, b);
        }
        bulk_commit_group();
        bulk_wait_read_all();
      }
      if (G > 1) group_barrier(1 + g);
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
  static std::atomic<bool> allowed[64];
  const cudaError_t rc = allow_shared(kernel, Layout<D>::kBytes, allowed);
  if (rc != cudaSuccess) return rc;
  constexpr int rows = Layout<D>::kGroups * kTile;
  const dim3 grid(p.heads * p.batch, (p.seq + rows - 1) / rows);
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
