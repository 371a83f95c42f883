// Windowed causal attention, backward, on the 5th-generation tensor cores.
//
//   P_ij  = exp(scale q_i k_j - lse_i)             dS_ij = P_ij (dO_i v_j - delta_i),  delta_i = dO_i O_i
//   dV_j  = sum_i P_ij dO_i     dK_j = scale sum_i dS_ij q_i     dQ_i = scale sum_j dS_ij k_j
//
// Two kernels of one shape.  A CTA holds two resident tiles of 128 rows and streams pairs of tiles past them:
// the keys' kernel holds K and V and streams Q and dO of every query head that shares them (so the heads'
// gradients are summed where they are made, in a fixed order), the queries' kernel holds Q and dO and streams
// K and V.  Each pair gives two products in tensor memory (scores and dO V^T, with the resident rows on the
// lanes), which the row threads, 64 columns of a row each, turn into P and dS in place; those are A operands
// of the sums, which stay in tensor memory.  Nothing is transposed and nothing is added atomically: the scores
// are computed once for either kernel, 7 products of a tile where one pass with atomic sums for dQ would take
// 5, and gradients come out the same in every run.
//
// The two products are handled one after the other, so that the tensor cores always have the other half to
// do: while the rows take exponentials of scores t, the sum with dS t - 1 and product t of dO V^T run; while they
// make dS t, the sum with P t and scores t + 1.  Heads of up to 64 leave room for two CTAs on an SM with
// streamed tiles of 64 rows; larger ones fill tensor memory with one, whose streamed tiles have 128 rows:
// with 64, reading the resident operand from shared memory again for half the columns set the pace.
//
// Time of the keys' and the queries' kernel, and rate of the visible pairs' products (8 and 6 dim operations each):
//   1 x 16384 tokens, 32 query heads over 8 key heads of 128, window 4096: 1.69 and 1.32 ms at 1965 MHz, 1140 and 1100
//     TFLOP/s, 0.70 and 0.67 of cuBLAS's burst (pass after pass 1.72 and 1.34 ms, at the 1665 MHz that the power limit
//     leaves); tensor cores busy 0.59 and 0.56 of the time, the MMAs and their operands; row sums 68 us (5.9 TB/s)
//   6 x up to 1999, 16 over 4 heads of 96, window 512: 98 and 96 us, row sums 18
//   8 x 1024, 12 heads of 64, window 256: 44 and 30 us, row sums 7.5, far queries' sums 2.8; short streams
// Row sums taken by the queries' kernel, while its first tiles arrive, cost it more than theirs does (97 -> 143 us in
// the second case): nothing hides the loads at the start of a CTA.
#include "window_attention.cuh"

namespace mb {
namespace attn {

namespace {

template <int D>
struct Layout {
  static constexpr int kRows = D == 128 ? 128 : 64;                // rows of a streamed tile
  static constexpr int kThreads = 64 + kRows * 2;                  // warp 0 loads, warp 1 issues MMAs, the others own rows
  static constexpr int kResident = D == 128 ? 1 : 2;               // CTAs of an SM
  static constexpr int kColumns = D == 128 ? 512 : 256;            // scores, other product, two sums
  static constexpr int kResidentBytes = kTile * D * 2;
  static constexpr int kStreamBytes = kRows * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kStatBytes = 2 * kRows * 4;                 // lse and delta of a streamed tile's rows
  static constexpr int kBytes = 2 * kResidentBytes + kStages * (2 * kStreamBytes + kStatBytes) + 1024 + 256;
};

// The streamed tiles of a CTA.  Keys' kernel: query tiles [lo, lo + per_head) of each of `heads` heads;
// queries' kernel: key tiles, the first tokens' before the window's.
struct Stream {
  int count, per_head, lo, head_tiles;
  __device__ __forceinline__ int tile(int t, bool keys) const {
    if (keys) return lo + t % per_head;
    return t < head_tiles ? t : lo + t - head_tiles;
  }
};

// Visible pairs of a row's 64, as bits.
struct Seen {
  uint32_t half[2];
  __device__ __forceinline__ bool at(int k) const { return half[k >> 5] >> (k & 31) & 1u; }
};

// What the rounding of a pair left, as a pair.
template <typename T>
__device__ __forceinline__ uint32_t pack_rest(float2 v, uint32_t rounded) {
  const T* r = reinterpret_cast<const T*>(&rounded);
  return pack2<T>(v.x - to_float(r[0]), v.y - to_float(r[1]));
}

// Exponentials of a row's 64 scores; in the keys' kernel also rounded over the scores.  The statistics are the
// columns' in the keys' kernel (in shared memory), the row's in the queries'.
template <typename T, bool KEYS, bool EDGE, bool SPLIT>
__device__ __forceinline__ void row_exp(const uint32_t (&s)[64], uint32_t ts, float scale, const float* col, float row,
                                        const Seen& seen, float2 (&pr)[32]) {
  const float2 scale2 = splat2(scale);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t packed[16], rest[16];
#pragma unroll
    for (int x = 0; x < 16; x += 2) {
      float2 l[2] = {splat2(row), splat2(row)};
      if constexpr (KEYS) {
        const float4 l4 = *reinterpret_cast<const float4*>(col + c * 32 + 2 * x);
        l[0] = make_float2(l4.x, l4.y), l[1] = make_float2(l4.z, l4.w);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = c * 32 + 2 * (x + u);
        float2 e = exp2_pair(__ffma2_rn(pair_of(s[k], s[k + 1]), scale2, l[u]));
        if constexpr (EDGE) {
          if (!seen.at(k)) e.x = 0.f;
          if (!seen.at(k + 1)) e.y = 0.f;
        }
        pr[c * 16 + x + u] = e;
        if constexpr (KEYS) packed[x + u] = pack2<T>(e.x, e.y);
        if constexpr (KEYS && SPLIT) rest[x + u] = pack_rest<T>(e, packed[x + u]);
      }
    }
    if constexpr (KEYS) tmem_st_32x16(ts + c * 16, packed);
    if constexpr (KEYS && SPLIT) tmem_st_32x16(ts + 32 + c * 16, rest);
  }
}

// dS over the other product.  P = 0 does not do for hidden pairs, whose product may be infinite or NaN.
template <typename T, bool KEYS, bool EDGE, bool SPLIT>
__device__ __forceinline__ void row_ds(uint32_t td, const float* col, float row, const Seen& seen,
                                       const float2 (&pr)[32]) {
  uint32_t d[64];
#pragma unroll
  for (int c = 0; c < 2; ++c) tmem_ld_32x32(td + c * 32, chunk_of(d, c));
  tmem_ld_wait();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t packed[16], rest[16];
#pragma unroll
    for (int x = 0; x < 16; x += 2) {
      float2 l[2] = {splat2(row), splat2(row)};
      if constexpr (KEYS) {
        const float4 l4 = *reinterpret_cast<const float4*>(col + c * 32 + 2 * x);
        l[0] = make_float2(l4.x, l4.y), l[1] = make_float2(l4.z, l4.w);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = c * 32 + 2 * (x + u);
        float2 ds = __fmul2_rn(pr[c * 16 + x + u], __fadd2_rn(pair_of(d[k], d[k + 1]), l[u]));
        if constexpr (EDGE) {
          if (!seen.at(k)) ds.x = 0.f;
          if (!seen.at(k + 1)) ds.y = 0.f;
        }
        packed[x + u] = pack2<T>(ds.x, ds.y);
        if constexpr (SPLIT) rest[x + u] = pack_rest<T>(ds, packed[x + u]);
      }
    }
    tmem_st_32x16(td + c * 16, packed);
    if constexpr (SPLIT) tmem_st_32x16(td + 32 + c * 16, rest);
  }
}

template <typename T, int D, bool KEYS, bool SPLIT>
__global__ void __launch_bounds__(Layout<D>::kThreads, Layout<D>::kResident)
window_bwd_kernel(const __grid_constant__ CUtensorMap map_x0, const __grid_constant__ CUtensorMap map_x1,
                  const __grid_constant__ CUtensorMap map_y0, const __grid_constant__ CUtensorMap map_y1,
                  const __grid_constant__ CUtensorMap map_out0, const __grid_constant__ CUtensorMap map_out1,
                  const __grid_constant__ Params p) {
  using L = Layout<D>;
  constexpr int kStages = L::kStages, kStream = L::kStreamBytes, kResident = L::kResidentBytes, R = L::kRows;
  constexpr int kRowWarps = R / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tile_x = smem;                                          // x0, x1
  uint8_t* ring = smem + 2 * kResident;                            // [stage]: y0, y1
  float* stats = reinterpret_cast<float*>(ring + kStages * 2 * kStream);       // [stage]: lse, delta of the R rows
  uint64_t* bars = reinterpret_cast<uint64_t*>(stats + kStages * 2 * R);
  uint64_t* full = bars;
  uint64_t* empty = bars + kStages;
  uint64_t* x_full = bars + 2 * kStages;
  uint64_t* s_full = x_full + 1;                   // scores are in tensor memory
  uint64_t* d_full = s_full + 1;                   // the other product is
  uint64_t* p_done = d_full + 1;                   // P is there (queries' kernel: the scores have been read)
  uint64_t* ds_done = p_done + 1;                  // dS is there
  uint64_t* acc_full = ds_done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Heads fastest, tiles in the order of their streams' lengths, so that short CTAs end the launch: the first keys
  // first, which most queries see, or the last queries, which see the most keys.  `part` > 0: queries far from the first tokens.
  const int ratio = p.heads / p.kv_heads;
  const int heads_here = KEYS ? p.kv_heads : p.heads;
  const int own_head = blockIdx.x % heads_here, b = blockIdx.x / heads_here;
  const int far_blocks = KEYS ? p.far_splits * ((p.sinks + kTile - 1) / kTile) : 0;
  const int part = KEYS && int(blockIdx.y) < far_blocks ? 1 + int(blockIdx.y) % p.far_splits : 0;
  const int y = int(blockIdx.y);
  const int x_tile = part > 0 ? y / p.far_splits : KEYS ? y - far_blocks : int(gridDim.y) - 1 - y;
  const int x_row = x_tile * kTile;
  const int len = length_of(p, b);

  Stream st{0, 1, 0, 0};
  if (x_row < len) {
    const int tiles = (len + R - 1) / R;
    if constexpr (KEYS) {
      // Queries from the tile's own on; up to a window behind its last key, or all for first tokens.
      st.lo = x_row / R;
      int hi = min(tiles, near_tiles(x_row, p.window, R));
      if (x_row < p.sinks) {
        if (p.far_splits == 0) hi = tiles;
        if (part > 0) {
          st.lo = p.far_first + (part - 1) * p.far_tiles;
          hi = min(tiles, st.lo + p.far_tiles);
        }
      }
      st.per_head = max(0, hi - st.lo);
      st.count = st.per_head * ratio;
    } else {
      st.lo = max(0, x_row - p.window + 1) / R;
      st.head_tiles = min((p.sinks + R - 1) / R, st.lo);
      st.count = st.head_tiles + (min(x_row + kTile, len) - 1) / R - st.lo + 1;
    }
  }
  auto stream_head = [&](int t) { return KEYS ? own_head * ratio + t / st.per_head : own_head / ratio; };

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(x_full), 1);
    mbar_init(smem_u32(s_full), 1);
    mbar_init(smem_u32(d_full), 1);
    mbar_init(smem_u32(p_done), kRowWarps);
    mbar_init(smem_u32(ds_done), kRowWarps);
    mbar_init(smem_u32(acc_full), 1);
    fence_barrier_init();
    prefetch_tensormap(&map_x0);
    prefetch_tensormap(&map_x1);
    prefetch_tensormap(&map_y0);
    prefetch_tensormap(&map_y1);
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), L::kColumns);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Scores, the other product, and the sums: dV (or dQ), dK.
  const uint32_t tmem_d = tmem + R, tmem_acc = tmem + 2 * R;

  if (warp == 0) {
    // ---- loader ----------------------------------------------------------------------------------
    if (lane == 0 && st.count > 0) {
      const uint32_t x_bar = smem_u32(x_full);
      mbar_arrive_expect_tx(x_bar, 2 * kResident);
      for (int box = 0; box < D / 64; ++box) {
        tma_load_4d(smem_u32(tile_x + box * (kTile * 128)), &map_x0, x_bar, box * 64, x_row, own_head, b);
        tma_load_4d(smem_u32(tile_x + kResident + box * (kTile * 128)), &map_x1, x_bar, box * 64, x_row, own_head, b);
      }
      int stage = 0;
      uint32_t phase = 0;
      for (int t = 0; t < st.count; ++t) {
        if (!mbar_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.status, kErrLoad, kWaitNs)) break;
        const uint32_t bar = smem_u32(&full[stage]);
        const int row = st.tile(t, KEYS) * R, h = stream_head(t);
        uint8_t* y = ring + stage * 2 * kStream;
        mbar_arrive_expect_tx(bar, 2 * kStream + (KEYS ? L::kStatBytes : 0));
        for (int box = 0; box < D / 64; ++box)
          tma_load_4d(smem_u32(y + box * (R * 128)), &map_y0, bar, box * 64, row, h, b);
        for (int box = 0; box < D / 64; ++box)
          tma_load_4d(smem_u32(y + kStream + box * (R * 128)), &map_y1, bar, box * 64, row, h, b);
        if constexpr (KEYS) {
          const int64_t at = (int64_t(b) * p.heads + h) * p.seq_pad + row;
          float* s = stats + stage * 2 * R;
          bulk_load(smem_u32(s), p.neg_lse + at, R * 4, bar);
          bulk_load(smem_u32(s + R), p.neg_delta + at, R * 4, bar);
        }
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issuer ------------------------------------------------------------------------------
    constexpr uint32_t idesc_s = instr_desc_f16(kIsBf16<T>, false, false, kTile, R);
    constexpr uint32_t idesc_a = instr_desc_f16(kIsBf16<T>, false, true, kTile, D);
    const uint32_t x0 = uniform(smem_u32(tile_x)), x1 = x0 + kResident, y_base = uniform(smem_u32(ring));
    const uint32_t ts = uniform(tmem), td = ts + R, ta = ts + 2 * R;
    // P and dS of 64 columns take the first 32 of the columns that their products took.
    auto at = [](int i) { return (i / 4) * 64 + (i % 4) * 8; };
    const uint32_t bar0 = uniform(smem_u32(bars));
    auto bar_of = [&](const uint64_t* bar) { return bar0 + uint32_t(bar - bars) * 8; };
    IssueWait wait{abort_flag, p.status, false};
    int stage = 0, next = 0;           // stages of pair t and of pair t + 1
    uint32_t next_phase = 0;
    // Products of the resident tiles with the streamed ones of stage `next`.
    auto scores = [&](int t) {
      wait(bar_of(&full[next]), next_phase);
      const int left = len - st.tile(t, KEYS) * R;
      if (left < R) {
        uint8_t* y = ring + next * 2 * kStream;
        zero_rows<R, D>(y, left, lane);
        zero_rows<R, D>(y + kStream, left, lane);
      }
      if (elect_one()) {
        const uint32_t y0 = y_base + next * 2 * kStream;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          umma_f16(ts, desc_along_dim<kTile>(x0, i), desc_along_dim<R>(y0, i), idesc_s, i != 0);
        umma_commit(bar_of(s_full));
      }
      __syncwarp();
    };
    auto other = [&] {
      if (elect_one()) {
        const uint32_t y1 = y_base + next * 2 * kStream + kStream;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          umma_f16(td, desc_along_dim<kTile>(x1, i), desc_along_dim<R>(y1, i), idesc_s, i != 0);
        umma_commit(bar_of(d_full));
      }
      __syncwarp();
    };
    if (st.count > 0) {
      wait(bar_of(x_full), 0);
      scores(0);
      other();
    }
    for (int t = 0; t < st.count; ++t) {
      const bool more = t + 1 < st.count;
      if (more && ++next == kStages) { next = 0; next_phase ^= 1u; }
      const uint32_t y0 = y_base + stage * 2 * kStream, y1 = y0 + kStream;
      wait(bar_of(p_done), t & 1);
      if constexpr (KEYS) {
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < R / 16; ++i)
            umma_f16_ta(ta, ts + at(i), desc_along_rows<R>(y1, i), idesc_a, t > 0 || i != 0);
          if constexpr (SPLIT) {
#pragma unroll
            for (int i = 0; i < R / 16; ++i) umma_f16_ta(ta, ts + 32 + at(i), desc_along_rows<R>(y1, i), idesc_a, 1);
          }
        }
        __syncwarp();
      }
      if (more) scores(t + 1);
      wait(bar_of(ds_done), t & 1);
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < R / 16; ++i)
          umma_f16_ta(ta + (KEYS ? D : 0), td + at(i), desc_along_rows<R>(y0, i), idesc_a, t > 0 || i != 0);
        if constexpr (SPLIT) {
#pragma unroll
          for (int i = 0; i < R / 16; ++i)
            umma_f16_ta(ta + (KEYS ? D : 0), td + 32 + at(i), desc_along_rows<R>(y0, i), idesc_a, 1);
        }
        umma_commit(bar_of(&empty[stage]));
        if (!more) umma_commit(bar_of(acc_full));
      }
      __syncwarp();
      if (more) other();
      stage = next;
    }
  } else {
    // ---- rows ------------------------------------------------------------------------------------
    const int half = (warp - 2) >> 2, quarter = warp & 3;         // columns 64 half to 64 half + 63 of the products
    const int r = quarter * 32 + lane, mine = x_row + r;          // this thread's key (or query)
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const uint32_t ts = tmem + lanes + half * 64, td = tmem_d + lanes + half * 64;
    const float scale = p.scale * kLog2e;
    const bool one_key = p.window == 1 && p.sinks == 0;           // for every query
    float row_lse = 0.f, row_delta = 0.f;
    if constexpr (!KEYS) {
      const int64_t at = (int64_t(b) * p.heads + own_head) * p.seq_pad + mine;
      row_lse = p.neg_lse[at];
      row_delta = p.neg_delta[at];
    }
    bool ok = true;
    int stage = 0;
    for (int t = 0; t < st.count && ok; ++t) {
      const int y_tile = st.tile(t, KEYS) * R, y_row = y_tile + half * 64;
      // Keys' kernel: queries i = y_row + column see this key when key <= i < key + window, or from the key on
      // for a first token; behind the end none does.  Queries' kernel: keys of the window, and first tokens.
      int from, to, keep = 0;          // [from, to], and [0, keep) where it is not above `to`
      bool edge;
      if constexpr (KEYS) {
        from = mine - y_row;
        to = mine < p.sinks ? 63 : int(min(int64_t(63), int64_t(mine) + p.window - 1 - y_row));
        to = min(to, len - 1 - y_row);
        edge = x_row + kTile - 1 > y_tile || (y_tile + R - 1) - x_row >= p.window || y_tile + R > len;
      } else {
        from = mine - p.window + 1 - y_row;
        to = mine - y_row;
        keep = p.sinks - y_row;
        edge = y_tile + R - 1 > x_row || (x_row + kTile - 1) - y_tile >= p.window;
      }
      Seen seen{{seen_bits(from, to, keep), seen_bits(from - 32, to - 32, keep - 32)}};
      const float* col = stats + stage * 2 * R + half * 64;
      ok = mbar_wait(smem_u32(s_full), t & 1, abort_flag, p.status, kErrRows, kWaitNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after();
      float2 pr[32];
      {
        uint32_t s[64];
        tmem_ld_32x32(ts, chunk_of(s, 0));
        tmem_ld_32x32(ts + 32, chunk_of(s, 1));
        tmem_ld_wait();
        if constexpr (!KEYS) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(p_done));
        }
        if (edge) row_exp<T, KEYS, true, SPLIT>(s, ts, scale, col, row_lse, seen, pr);
        else row_exp<T, KEYS, false, SPLIT>(s, ts, scale, col, row_lse, seen, pr);
      }
      if constexpr (KEYS) {
        tmem_st_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(p_done));
      }
      ok = mbar_wait(smem_u32(d_full), t & 1, abort_flag, p.status, kErrRows, kWaitNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after();
      // A query that sees one key has P = 1 and dS = 0 whatever the inputs are; computed, dP - delta would be what
      // its two orders of summation leave.  Such queries lie in edge tiles.
      if (one_key || (!KEYS && mine == 0)) seen.half[0] = seen.half[1] = 0u;
      else if (KEYS && y_row == 0) seen.half[0] &= ~1u;
      if (edge) row_ds<T, KEYS, true, SPLIT>(td, col + R, row_delta, seen, pr);
      else row_ds<T, KEYS, false, SPLIT>(td, col + R, row_delta, seen, pr);
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(ds_done));
      if (++stage == kStages) stage = 0;
    }
    if (st.count > 0 && ok) {
      ok = mbar_wait(smem_u32(acc_full), 0, abort_flag, p.status, kErrRows, kWaitNs);
      ok = __all_sync(0xffffffffu, ok);
      tcgen05_fence_after();
    }
    // The keys' kernel has two results, dV and dK: one for either half of the row threads where there are two.
    // The queries' kernel has dQ, whose columns they share.
    constexpr int G = R / 64;
    const int g = half;
    const bool some = st.count > 0 && ok;
    const bool live = some && mine < len;
    // A first token whose far queries are other CTAs': this CTA's share goes to the workspace.
    const bool shared_sum = KEYS && p.far_splits > 0 && mine < p.sinks && mine < p.seq;
    constexpr int kChunks = KEYS ? D / 32 : D / 32 / G;
#pragma unroll 1
    for (int which = KEYS ? g : 0; which < (KEYS ? 2 : 1); which += KEYS ? G : 1) {          // 0: dV (dQ), 1: dK
      const uint32_t acc = tmem_acc + lanes + (KEYS ? which * D : g * (D / G));
      const float factor = KEYS && which == 0 ? 1.f : p.scale;
      uint8_t* staged = tile_x + (KEYS ? which * kResident : 0);     // all products have been taken
      float* far = nullptr;
      if (shared_sum)
        far = p.far + ((((int64_t(part) * p.batch + b) * p.kv_heads + own_head) * 2 + (1 - which)) * p.sinks + mine) * p.dim;
#pragma unroll 1
      for (int c = 0; c < kChunks; ++c) {
        uint32_t raw[32];
        if (some) {
          tmem_ld_32x32(acc + c * 32, raw);
          tmem_ld_wait();
        }
        if (!live) {
#pragma unroll
          for (int x = 0; x < 32; ++x) raw[x] = 0u;
        }
        if (far != nullptr) {
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            if (c * 32 + x < p.dim)
              *reinterpret_cast<float4*>(far + c * 32 + x) =
                  make_float4(__uint_as_float(raw[x]) * factor, __uint_as_float(raw[x + 1]) * factor,
                              __uint_as_float(raw[x + 2]) * factor, __uint_as_float(raw[x + 3]) * factor);
        }
        if (part == 0) stage_row<T>(staged, r, KEYS ? c : g * kChunks + c, raw, factor);
      }
      fence_proxy_async_smem();
      if (KEYS || G == 1) group_barrier(1 + g);
      else asm volatile("bar.sync 1, 256;" ::: "memory");
      if (part == 0 && (KEYS || g == 0) && quarter == 0 && lane == 0 && x_row < p.seq) {
        for (int box = 0; box < D / 64; ++box)
          if (box * 64 < p.dim)
            tma_store_4d(KEYS && which == 0 ? &map_out1 : &map_out0, smem_u32(staged + box * (kTile * 128)), box * 64,
                         x_row, own_head, b);
        bulk_commit_group();
      }
    }
    if (quarter == 0 && lane == 0) bulk_wait_read_all();
    __syncwarp();
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    settle(abort_flag);
    tcgen05_fence_after();
    tmem_dealloc(tmem, L::kColumns);
  }
}

// delta_i = dO_i O_i with O as it was before its rounding (P (dP - delta) cancels where few keys are visible:
// with the rounded O the gradients of q and k were off by half as much again), LANES lanes of 16 bytes a row of one
// head; zero behind a sequence's end, whatever lies there.
template <typename T, int LANES>
__global__ void __launch_bounds__(256)
row_sums_kernel(const T* __restrict__ out, const T* __restrict__ low, const T* __restrict__ dout,
                const Params p) {
  // Rows in the order of memory: all heads of a token, then the next token.
  const int lane = threadIdx.x % LANES, b = blockIdx.y;
  const int64_t n = int64_t(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  const int i = int(n / p.heads), h = int(n - int64_t(i) * p.heads);
  float sum = 0.f;
  if (i < length_of(p, b) && lane * 8 < p.dim) {
    const int64_t at = (int64_t(b) * p.seq * p.heads + n) * p.dim + lane * 8;
    const uint4 x = *reinterpret_cast<const uint4*>(out + at), y = *reinterpret_cast<const uint4*>(dout + at);
    const uint4 z = *reinterpret_cast<const uint4*>(low + at);
    const T* xs = reinterpret_cast<const T*>(&x);
    const T* ys = reinterpret_cast<const T*>(&y);
    const T* zs = reinterpret_cast<const T*>(&z);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = fmaf(to_float(xs[k]) + to_float(zs[k]), to_float(ys[k]), sum);
  }
#pragma unroll
  for (int d = LANES / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) p.neg_delta[(int64_t(b) * p.heads + h) * p.seq_pad + i] = -sum;
}

// One warp a first token of a key head: its parts in order, rounded once.
template <typename T>
__global__ void __launch_bounds__(128)
sum_far_kernel(T* __restrict__ dk, T* __restrict__ dv, const Params p) {
  const int64_t n = int64_t(p.batch) * p.kv_heads * p.sinks * p.dim;
  const int64_t x = int64_t(blockIdx.x) * 128 + threadIdx.x;
  if (x >= 2 * n) return;
  // x runs over [batch][kv_heads][2][sinks][dim], the layout of a part.
  const int d = int(x % p.dim);
  int64_t rest = x / p.dim;
  const int row = int(rest % p.sinks);
  rest /= p.sinks;
  const int which = int(rest % 2);
  rest /= 2;
  const int h = int(rest % p.kv_heads), b = int(rest / p.kv_heads);
  if (row >= p.seq) return;
  float sum = 0.f;
  for (int s = 0; s <= p.far_splits; ++s) sum += p.far[s * 2 * n + x];
  T* out = which == 0 ? dk : dv;
  out[((int64_t(b) * p.seq + row) * p.kv_heads + h) * p.dim + d] = from_float<T>(sum);
}

template <typename T, int D, bool KEYS, bool SPLIT>
cudaError_t launch_backward(const CUtensorMap& x0, const CUtensorMap& x1, const CUtensorMap& y0, const CUtensorMap& y1,
                            const CUtensorMap& o0, const CUtensorMap& o1, const Params& p, cudaStream_t stream) {
  auto kernel = window_bwd_kernel<T, D, KEYS, SPLIT>;
  static std::atomic<bool> allowed[64];
  const cudaError_t rc = allow_shared(kernel, Layout<D>::kBytes, allowed);
  if (rc != cudaSuccess) return rc;
  const int far = KEYS ? p.far_splits * ((p.sinks + kTile - 1) / kTile) : 0;
  const dim3 grid((KEYS ? p.kv_heads : p.heads) * p.batch, far + (p.seq + kTile - 1) / kTile);
  kernel<<<grid, Layout<D>::kThreads, Layout<D>::kBytes, stream>>>(x0, x1, y0, y1, o0, o1, p);
  return cudaGetLastError();
}

template <bool KEYS>
cudaError_t backward(bool bf16, const CUtensorMap& x0, const CUtensorMap& x1, const CUtensorMap& y0,
                     const CUtensorMap& y1, const CUtensorMap& o0, const CUtensorMap& o1, const Params& p,
                     cudaStream_t stream) {
  auto typed = [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    if (p.dim <= 64)
      return p.split ? launch_backward<T, 64, KEYS, true>(x0, x1, y0, y1, o0, o1, p, stream)
                     : launch_backward<T, 64, KEYS, false>(x0, x1, y0, y1, o0, o1, p, stream);
    return p.split ? launch_backward<T, 128, KEYS, true>(x0, x1, y0, y1, o0, o1, p, stream)
                   : launch_backward<T, 128, KEYS, false>(x0, x1, y0, y1, o0, o1, p, stream);
  };
  return bf16 ? typed(static_cast<__nv_bfloat16*>(nullptr)) : typed(static_cast<__half*>(nullptr));
}

}  // namespace

cudaError_t row_sums(bool bf16, const void* out, const void* dout, const Params& p, cudaStream_t stream) {
  auto launch = [&](auto* x, auto lanes) {
    using T = std::remove_pointer_t<decltype(x)>;
    constexpr int kLanes = decltype(lanes)::value;
    const dim3 grid(p.seq_pad / (256 / kLanes) * p.heads, p.batch);              // seq_pad is a multiple of 256
    row_sums_kernel<T, kLanes><<<grid, 256, 0, stream>>>(static_cast<const T*>(out), static_cast<const T*>(p.out_low),
                                                         static_cast<const T*>(dout), p);
  };
  auto typed = [&](auto* x) {
    if (p.dim <= 64) launch(x, std::integral_constant<int, 8>{});
    else launch(x, std::integral_constant<int, 16>{});
  };
  if (bf16) typed(static_cast<__nv_bfloat16*>(nullptr));
  else typed(static_cast<__half*>(nullptr));
  return cudaGetLastError();
}

cudaError_t backward_keys(bool bf16, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q_stream,
                          const CUtensorMap& dout_stream, const CUtensorMap& dk, const CUtensorMap& dv, const Params& p,
                          cudaStream_t stream) {
  return backward<true>(bf16, k, v, q_stream, dout_stream, dk, dv, p, stream);
}

cudaError_t backward_queries(bool bf16, const CUtensorMap& q, const CUtensorMap& dout, const CUtensorMap& k_stream,
                             const CUtensorMap& v_stream, const CUtensorMap& dq, const Params& p, cudaStream_t stream) {
  return backward<false>(bf16, q, dout, k_stream, v_stream, dq, dq, p, stream);
}

cudaError_t sum_far(bool bf16, void* dk, void* dv, const Params& p, cudaStream_t stream) {
  const int64_t n = int64_t(2) * p.batch * p.kv_heads * p.sinks * p.dim;
  const unsigned grid = static_cast<unsigned>((n + 127) / 128);
  if (bf16)
    sum_far_kernel<<<grid, 128, 0, stream>>>(static_cast<__nv_bfloat16*>(dk), static_cast<__nv_bfloat16*>(dv), p);
  else
    sum_far_kernel<<<grid, 128, 0, stream>>>(static_cast<__half*>(dk), static_cast<__half*>(dv), p);
  return cudaGetLastError();
}

}  // namespace attn
}  // namespace mb
