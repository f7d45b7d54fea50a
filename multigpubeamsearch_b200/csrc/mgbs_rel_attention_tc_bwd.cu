// Backward of long attention with a relative bias on tcgen05, one kernel in two forms.  A block owns 128 rows and walks
// over tiles of 64 of the other side:
//
//   dq form:      rows are queries, tiles keys:     S = Q K^T,    dP = dO V^T;    acc1 += P K,      acc2 += dS K
//   dk, dv form:  rows are keys, tiles queries:     S = K Q^T,    dP = V dO^T;    acc1 += P dO,     acc2 += dS Q
//   with P = 2^(s - max - log2 sum) from the forward's statistics and dS = P (dP - delta)
//
// S, dP and the accumulators lie in tensor memory, 64 columns each.  A softmax thread owns a row: it reads S and dP and
// leaves P and dS in their places as 16-bit pairs, from where they are the A operands of the second products.  A tile's
// steps follow one another; the second block of the multiprocessor (256 of the 512 columns each) fills the waits.
//
// delta = sum_j P_ij dP_ij.  A first delta is dout . out from the 16-bit output.  A row of dS has to sum to 0, so the sum r
// of the rows made with it is the error of that delta: at the end dq loses r P k, and the other form gets delta + r.
//
// The table's gradient is summed in the dk, dv form, from the corrected delta: where values have a common mean, the first
// delta's error (the output's rounding) is large beside what is left of a row's dS over many keys, 23 u of the table's
// 2-norm for v of mean 4 and spread 1 at 1001 tokens.  Tiles beyond the reach are summed in registers, nearer ones by
// diagonals of 16 x 16 through shared memory into the warp's own sums by offset, in a fixed order.  The query heads that
// share a key head are spread over the blocks of a cluster, whose dk and dv are added through distributed shared memory.
// Rows past a length are zeroed in shared memory where they are B operands of the second products; elsewhere they only
// reach scores that are hidden and rows that are not written.
// Every wait is bounded: a block that gives up writes NaN and the error word.
//
// At 6 x 1501 causal padded tokens, 8 heads of 64 over 2: 40 us for dq, 77 us for dk, dv and the table, against 88 us and
// 134 us on the warp-level instruction (8 us of exponentials each).  What bounds them: the chain of a tile (products 800
// to 1000 clocks with their hand-overs, the row's arithmetic 1250), since the scores of the next tile are issued only
// when this one's second products are done, and the blocks' beginnings and ends; the table's diagonals take 20 us of the 77.
// (Summed in the dq form, with the first delta, the two were 57 and 56 us.)

#include <math.h>

#include <type_traits>

#include "mgbs_rel_attention_tc.cuh"

namespace mgbs {

constexpr int TB_DP_COL = 64, TB_ACC1_COL = 128, TB_ACC2_COL = 192;  // S at 0; P and dS in the places of S and dP
constexpr int TB_RIM = 192;  // a tile that is not beyond the reach has offsets below reach + TC_Q + TC_K
// A warp's 32 rows of 16 columns of dS: pairs of a row in one store, 16 rows over all banks, the other 16 half of them apart.
constexpr int TB_COLS = 16, TB_DS_PITCH = TB_COLS + 2, TB_DS_HALF = 16 * TB_DS_PITCH + 16, TB_DS = 2 * TB_DS_HALF;
template <bool KV> __host__ __device__ constexpr int tb_stages() { return KV ? 3 : 2; }
__host__ __device__ inline int tb_bias_floats(int reach) { return 2 * (reach + TB_RIM) + 1; }
template <int D, bool KV> __host__ __device__ constexpr int tb_operands() { return (2 * TC_Q + tb_stages<KV>() * 2 * TC_K) * D * 2; }
template <int D, bool KV> inline int tb_smem(int reach, int buckets) {
  const int table = KV ? 5 * tb_bias_floats(reach) + 1 + 4 * TB_DS + 2 * reach + 1 + buckets + 1 : tb_bias_floats(reach);
  const int all = 1024 + tb_operands<D, KV>() + table * 4;
  return all < 78 * 1024 ? 78 * 1024 : all;  // never more than two blocks on an SM: a third would wait for tensor memory
}

__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the four softmax warps

template <typename T, int D, bool KV>
__global__ void __launch_bounds__(TC_THREADS, 2) k_rel_tc_bwd(const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_a2,
                                                              const __grid_constant__ CUtensorMap map_b1, const __grid_constant__ CUtensorMap map_b2,
                                                              const __grid_constant__ RelArgs g, int tiles, int ranks) {
  constexpr int A_BYTES = TC_Q * D * 2, B_BYTES = TC_K * D * 2, STAGES = tb_stages<KV>();
  extern __shared__ __align__(1024) uint8_t tc_smem[];
  __shared__ __align__(8) uint64_t bars[4 * STAGES + 6];
  __shared__ __align__(16) float stat[KV ? STAGES : 1][3][TC_K];  // a stage's queries: -maximum, -log2 of the sum, -delta
  __shared__ float row_delta[KV ? 1 : TC_Q], far_sum[2][4], far_all[2];  // the second and third: dk, dv form
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const int rank = (int)(blockIdx.x % ranks);
  Where w = rel_where(blockIdx.x / ranks, tiles, KV ? g.heads_kv : g.heads, g.batch);
  if (!KV) w.tile = tiles - 1 - w.tile;  // the longest first
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int len = rel_length(g, w.b), a0 = w.tile * TC_Q;
  const int share = KV ? g.heads / g.heads_kv / ranks : 1;  // query heads of this block: rank, rank + ranks, ...
  auto head_of = [&](int n) { return KV ? (w.head * share + n) * ranks + rank : w.head; };
  auto row_of = [&](void* base, int row) {
    return row < g.tokens ? static_cast<T*>(base) + (((int64_t)w.b * g.tokens + row) * (KV ? g.heads_kv : g.heads) + w.head) * D : nullptr;
  };
  auto partial_of = [&](int head) { return g.partial + ((int64_t)head * g.batch * tiles + (int64_t)w.b * tiles + w.tile) * g.buckets; };
  if (a0 >= len) {  // the whole cluster
    if (rank == 0)
      for (int c = threadIdx.x; c < TC_Q * (D / 8); c += TC_THREADS) {
        const int row = a0 + c / (D / 8), part = c % (D / 8) * 8;
        if (row >= g.tokens) break;
        *reinterpret_cast<uint4*>(row_of(KV ? g.dk : g.dq, row) + part) = make_uint4(0u, 0u, 0u, 0u);
        if (KV) *reinterpret_cast<uint4*>(row_of(g.dv, row) + part) = make_uint4(0u, 0u, 0u, 0u);
      }
    if (KV)
      for (int i = threadIdx.x; i < share * g.buckets; i += TC_THREADS) partial_of(head_of(i / g.buckets))[i % g.buckets] = 0.f;
    return;  // the other form walks over queries below the length only: delta is not read here
  }
  const uint32_t a_at = (smem_u32(tc_smem) + 1023u) & ~1023u, b_at = a_at + 2 * A_BYTES;
  uint8_t* operands = tc_smem + (a_at - smem_u32(tc_smem));
  float* bt = reinterpret_cast<float*>(operands + tb_operands<D, KV>());
  const int side = g.reach + TB_RIM, span = 2 * side + 1;
  float* dacc = bt + span;        // dk, dv form: dS by offset, for each softmax warp's rows,
  float* ds = dacc + 4 * span + 1;  // 16 columns of it for each of them,
  int* order = reinterpret_cast<int*>(ds + 4 * TB_DS);  // the offsets by bucket and where a bucket begins
  int* begin = order + 2 * g.reach + 1;
  const uint32_t bar = smem_u32(bars);
  const uint32_t full = bar, free_ = bar + 8 * STAGES, stat_full = bar + 16 * STAGES, fixed = bar + 24 * STAGES;
  const uint32_t a_full = bar + 32 * STAGES, s_full = a_full + 8, p_full = a_full + 16, done = a_full + 24, drained = a_full + 32, a_ready = a_full + 40;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4 * STAGES + 6; ++i) mbar_init(bar + i * 8, bar + i * 8 == p_full ? 4 : 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(256u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  auto wait = [&](uint32_t b, uint32_t parity, int code) {
    if (mbar_try_wait(b, parity)) return true;
    return tc_wait_slow(b, parity, &gave_up, g.error, code);
  };
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // the tiles: rows `first` to `last` of the other side, for each of the block's query heads
  const int first = KV && g.causal ? a0 : 0, last = !KV && g.causal ? min(len, a0 + TC_Q) : len;
  const int n_tiles = (last - first + TC_K - 1) / TC_K, steps = n_tiles * share;
  // rows between the length and the tensor's end are padding that the last tile holds: zeroed before it is used
  const bool fix = len < g.tokens && first + n_tiles * TC_K > len;
  bool ok = true;

  if (warp == 5) {
    const int a_head = w.head, b_kv = KV ? 0 : w.head / (g.heads / g.heads_kv);
    if (lane == 0) {
      mbar_expect_tx(a_full, 2 * A_BYTES);
      tma_load_4d(a_at, &map_a1, a0, a_head, w.b, a_full);
      tma_load_4d(a_at + A_BYTES, &map_a2, a0, a_head, w.b, a_full);
    }
    if (!KV && len < g.tokens && a0 + TC_Q > len) {  // queries past the length must not leave a NaN in dS
      ok = wait(a_full, 0, ERR_TC_LOAD);
      if (__all_sync(0xffffffffu, ok)) {
        uint4* rows = reinterpret_cast<uint4*>(operands);
        for (int c = (len - a0) * (D / 8) + lane; c < TC_Q * (D / 8); c += 32) rows[c] = rows[TC_Q * (D / 8) + c] = make_uint4(0u, 0u, 0u, 0u);
        async_fence();
        __syncwarp();
      }
    }
    if (lane == 0) mbar_arrive(a_ready);
    int n = 0;
    for (; n < steps; ++n) {
      const int s = n % STAGES, turn = n / STAGES, tile = n % n_tiles, row = first + tile * TC_K, head = KV ? head_of(n / n_tiles) : b_kv;
      const uint32_t to = b_at + s * 2 * B_BYTES;
      if (turn > 0) ok = wait(free_ + s * 8, (turn - 1) & 1, ERR_TC_FREE);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      if (lane == 0) {
        mbar_expect_tx(full + s * 8, 2 * B_BYTES);
        tma_load_4d(to, &map_b1, row, head, w.b, full + s * 8);
        tma_load_4d(to + B_BYTES, &map_b2, row, head, w.b, full + s * 8);
      }
      if (KV) {
        const int64_t at = ((int64_t)w.b * g.heads + head) * g.tokens;
#pragma unroll
        for (int c = lane; c < TC_K; c += 32) {
          const bool in = row + c < len;
          const float2 st = in ? __ldg(g.stats + at + row + c) : make_float2(0.f, INFINITY);
          stat[s][0][c] = -st.x;
          stat[s][1][c] = -st.y;
          stat[s][2][c] = in ? -__ldg(g.delta + at + row + c) : 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(stat_full + s * 8);
      }
      if (fix) {
        if (tile == n_tiles - 1) {
          ok = wait(full + s * 8, turn & 1, ERR_TC_LOAD);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; ++n; break; }
          uint4* rows = reinterpret_cast<uint4*>(operands + 2 * A_BYTES + s * 2 * B_BYTES);
          for (int c = (len - row) * (D / 8) + lane; c < TC_K * (D / 8); c += 32) rows[c] = rows[TC_K * (D / 8) + c] = make_uint4(0u, 0u, 0u, 0u);
          async_fence();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(fixed + s * 8);
      }
    }
    if (!ok) {  // what has been asked for comes before the block ends
      tc_settle(a_full, 0);
      for (int i = n > STAGES ? n - STAGES : 0; i < n; ++i) tc_settle(full + i % STAGES * 8, (i / STAGES) & 1);
    }
  } else if (warp == 4) {
    // the whole warp walks and waits, one elected lane issues
    constexpr uint32_t id_s = tc_idesc<T>(TC_K, false), id_o = tc_idesc<T>(D, true);
    const uint64_t a1 = tc_desc<D>(a_at), a2 = tc_desc<D>(a_at + A_BYTES);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    ok = __all_sync(0xffffffffu, wait(a_full, 0, ERR_TC_LOAD) && wait(a_ready, 0, ERR_TC_LOAD));
    for (int n = 0; ok && n < steps; ++n) {
      const int s = n % STAGES;
      ok = wait(full + s * 8, (n / STAGES) & 1, ERR_TC_LOAD);
      if (fix) ok = ok && wait(fixed + s * 8, (n / STAGES) & 1, ERR_TC_LOAD);
      if (n > 0) ok = ok && wait(done, (n - 1) & 1, ERR_TC_O);  // P and dS have been used
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint64_t b1 = tc_desc<D>(b_at + s * 2 * B_BYTES), b2 = tc_desc<D>(b_at + s * 2 * B_BYTES + B_BYTES);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) tc_mma_f16(tm, a1 + kk * 2, b1 + kk * 2, id_s, kk > 0);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) tc_mma_f16(tm + TB_DP_COL, a2 + kk * 2, b2 + kk * 2, id_s, kk > 0);
        tc_commit(s_full);
      }
      __syncwarp();
      ok = __all_sync(0xffffffffu, wait(p_full, n & 1, ERR_TC_P));
      if (!ok) break;
      tc_fence_after();
      const uint64_t o1 = KV ? b2 : b1;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < TC_K / 16; ++kk) tc_mma_ts(tm + TB_ACC1_COL, tm + kk * 8, o1 + kk * (16 * D * 2 >> 4), id_o, n > 0 || kk > 0);
#pragma unroll
        for (int kk = 0; kk < TC_K / 16; ++kk) tc_mma_ts(tm + TB_ACC2_COL, tm + TB_DP_COL + kk * 8, b1 + kk * (16 * D * 2 >> 4), id_o, n > 0 || kk > 0);
        tc_commit(free_ + s * 8);
        tc_commit(done);
      }
      __syncwarp();
    }
    if (!ok) {  // products on their way end before the tensor memory is given back
      if (elect_one()) tc_commit(drained);
      __syncwarp();
      tc_settle(drained, 0);
    }
  } else {
    const int row = a0 + threadIdx.x;
    const bool in = row < len;
    const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
    const Pair sl2 = pair(g.sl2, g.sl2);
    float d = 0.f, r = 0.f, before = 0.f, after = 0.f;
    Pair nm{}, nl{}, nd{};
    if (!KV) {
      // D / 8 lanes have a row of dout and out; rows past the length repeat the last one.  On their way while the
      // tables are laid out.
      const T* y = static_cast<const T*>(g.out) + ((int64_t)w.b * g.tokens * g.heads + w.head) * D + lane % (D / 8) * 8;
      const T* z = static_cast<const T*>(g.dout) + w.b * g.ds[0] + w.head * g.ds[2] + lane % (D / 8) * 8;
      constexpr int ROWS = 128 / (D / 8), TURNS = TC_Q / ROWS;
      uint4 raw_y[TURNS], raw_z[TURNS];
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int64_t from = min(a0 + i * ROWS + (int)threadIdx.x / (D / 8), len - 1);
        raw_y[i] = __ldg(reinterpret_cast<const uint4*>(y + from * g.heads * D));
        raw_z[i] = __ldg(reinterpret_cast<const uint4*>(z + from * g.ds[1]));
      }
      const float2 st = in ? g.stats[((int64_t)w.b * g.heads + w.head) * g.tokens + row] : make_float2(0.f, INFINITY);
      fill_bias<T>(g, w.head, bt, side, threadIdx.x, 128);
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        float a[8], b[8], dot = 0.f;
        Vec16<T>::up(raw_y[i], a);
        Vec16<T>::up(raw_z[i], b);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(a[e], b[e], dot);
#pragma unroll
        for (int m = D / 16; m > 0; m >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, m);
        if (lane % (D / 8) == 0) row_delta[i * ROWS + threadIdx.x / (D / 8)] = dot;
      }
      softmax_sync();
      d = row_delta[threadIdx.x];
      nm = pair(-st.x, -st.x);
      nl = pair(-st.y, -st.y);
      nd = pair(-d, -d);
    } else {
      for (int i = threadIdx.x; i < 4 * span; i += 128) dacc[i] = 0.f;
#pragma unroll 4
      for (int i = threadIdx.x; i < 2 * g.reach + 1; i += 128) order[i] = min(max(__ldg(g.order + i), 0), 2 * g.reach);
      for (int i = threadIdx.x; i <= g.buckets; i += 128) begin[i] = min(max(__ldg(g.start + i), 0), 2 * g.reach + 1);
    }
    // The table's partial sums of one query head, from what its tiles have left by offset.
    auto finish_table = [&](int head) {
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, m);
        after += __shfl_xor_sync(0xffffffffu, after, m);
      }
      if (lane == 0) { far_sum[0][warp] = before; far_sum[1][warp] = after; }
      before = after = 0.f;
      softmax_sync();
      auto by_offset_sum = [&](int i) { return (dacc[i] + dacc[span + i]) + (dacc[2 * span + i] + dacc[3 * span + i]); };
      if (warp < 2) {  // offsets past the reach join its ends
        float rim = 0.f;
        for (int i = lane; i < TB_RIM; i += 32) rim += by_offset_sum(warp ? span - 1 - i : i);
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) rim += __shfl_xor_sync(0xffffffffu, rim, m);
        if (lane == 0) far_all[warp] = rim + (far_sum[warp][0] + far_sum[warp][1]) + (far_sum[warp][2] + far_sum[warp][3]);
      }
      softmax_sync();
      float* sorted = ds;  // the sums in the order of their buckets
      static_assert(4 * TB_DS >= 2 * 1024 + 1, "the largest reach fits");
      for (int n = threadIdx.x; n < 2 * g.reach + 1; n += 128) {
        const int i = order[n];
        sorted[n] = by_offset_sum(i + TB_RIM) + (i == 0 ? far_all[0] : i == 2 * g.reach ? far_all[1] : 0.f);
      }
      softmax_sync();
      float* partial = partial_of(head);
      for (int base = 0; base < g.buckets; base += 32) {  // four lanes per bucket
        const int b = base + threadIdx.x / 4;
        float all = 0.f;
        if (b < g.buckets)
#pragma unroll 4
          for (int n = begin[b] + (lane & 3); n < begin[b + 1]; n += 4) all += sorted[n];
        all += __shfl_xor_sync(0xffffffffu, all, 1);
        all += __shfl_xor_sync(0xffffffffu, all, 2);
        if (b < g.buckets && (lane & 3) == 0) partial[b] = ok ? all : NAN;
      }
      for (int i = threadIdx.x; i < 4 * span; i += 128) dacc[i] = 0.f;  // for the next head, which begins with a barrier
    };
    // A softmax thread's row in ds, and its lane's way down the diagonals of its half of the warp's rows.
    float* ds_row = ds + warp * TB_DS + (lane >> 4) * TB_DS_HALF + (lane & 15) * TB_DS_PITCH;
    const float* ds_walk = ds + warp * TB_DS + (lane >> 4) * TB_DS_HALF + (lane & 15);
    for (int n = 0; n < steps; ++n) {
      const int tile = n % n_tiles, b0 = first + tile * TC_K, s = n % STAGES;
      if (KV && tile == 0) {
        softmax_sync();  // the head before has read its biases
        fill_bias<T>(g, head_of(n / n_tiles), bt, side, threadIdx.x, 128);
        softmax_sync();
      }
      // key minus query: at least the reach for the whole tile, or at most minus the reach
      const int low = KV ? a0 - (b0 + TC_K - 1) : b0 - (a0 + TC_Q - 1), high = KV ? a0 + TC_Q - 1 - b0 : b0 + TC_K - 1 - a0;
      const int far = low >= g.reach ? 1 : -high >= g.reach ? -1 : 0;
      const bool edge = b0 + TC_K > len || (g.causal && high > 0) || (KV && a0 + TC_Q > len);
      // of the tile's columns the row has those from `lo` on, `held` of them; keys past the length have none (the table)
      const int lo = KV && g.causal ? max(0, row - b0) : 0, held = KV && !in ? 0 : (!KV && g.causal ? min(len, row + 1) : len) - b0 - lo;
      const float one = far > 0 ? bt[2 * side] : bt[0];
      const float* by_offset = KV ? bt + row - b0 + side : bt + b0 - row + side;
      const float *s_m = stat[KV ? s : 0][0], *s_l = stat[KV ? s : 0][1], *s_d = stat[KV ? s : 0][2];
      // after a wait that gave up the walk goes on over what is there, so that the warps meet at their barriers
      if (KV) ok = ok && wait(stat_full + s * 8, (n / STAGES) & 1, ERR_TC_LOAD);
      ok = ok && wait(s_full, n & 1, ERR_TC_S);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      Pair sum = pair(0.f, 0.f);
      // MODE 0: one bias; 1: by offset; 2: either, some pairs hidden
      auto walk = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        const Pair fixed_bias = pair(one, one);
        uint32_t sc[2][16], dp[2][16];
        tc_ld16(mine, sc[0]);
        tc_ld16(mine + TB_DP_COL, dp[0]);
#pragma unroll
        for (int i = 0; i < TC_K / 16; ++i) {
          const int c = i * 16;
          tc_wait_ld();
          if (i + 1 < TC_K / 16) {  // the next columns come while these are worked on
            tc_ld16(mine + c + 16, sc[(i + 1) & 1]);
            tc_ld16(mine + TB_DP_COL + c + 16, dp[(i + 1) & 1]);
          }
          uint32_t p[8], z[8];
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            Pair m[2], l[2], e[2];
            if (KV) {
              const float4 fm = *reinterpret_cast<const float4*>(s_m + c + j), fl = *reinterpret_cast<const float4*>(s_l + c + j), fd = *reinterpret_cast<const float4*>(s_d + c + j);
              m[0] = pair(fm.x, fm.y); m[1] = pair(fm.z, fm.w);
              l[0] = pair(fl.x, fl.y); l[1] = pair(fl.z, fl.w);
              e[0] = pair(fd.x, fd.y); e[1] = pair(fd.z, fd.w);
            } else {
              m[0] = m[1] = nm; l[0] = l[1] = nl; e[0] = e[1] = nd;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int k = j + 2 * h, at = c + k;
              const bool same = MODE == 0 || (MODE == 2 && far);
              const Pair bias = same ? fixed_bias : KV ? pair(by_offset[-at], by_offset[-at - 1]) : pair(by_offset[at], by_offset[at + 1]);
              const Pair score = fma2(pair(__uint_as_float(sc[i & 1][k]), __uint_as_float(sc[i & 1][k + 1])), sl2, bias);
              Pair prob = exp2_2(add2(add2(score, m[h]), l[h]));
              Pair grad = mul2(prob, add2(pair(__uint_as_float(dp[i & 1][k]), __uint_as_float(dp[i & 1][k + 1])), e[h]));
              if (MODE == 2) {
                float2 fp = both(prob), fg = both(grad);
                if (at < lo || at - lo >= held) fp.x = fg.x = 0.f;
                if (at + 1 < lo || at + 1 - lo >= held) fp.y = fg.y = 0.f;
                prob = pair(fp.x, fp.y);
                grad = pair(fg.x, fg.y);
              }
              const float2 fp = both(prob), fg = both(grad);
              p[k / 2] = pack2<T>(fp.x, fp.y);
              z[k / 2] = pack2<T>(fg.x, fg.y);
              if (!KV || MODE != 1) sum = add2(sum, grad);
              if (KV && (MODE == 1 || (MODE == 2 && !far))) *reinterpret_cast<float2*>(ds_row + k) = fg;
            }
          }
          tc_st8(mine + c / 2, p);  // over columns that have been read
          tc_st8(mine + TB_DP_COL + c / 2, z);
          if (KV && (MODE == 1 || (MODE == 2 && !far))) {
            // 16 x 16 of dS by diagonals, one for each half of the warp: lane l walks down the rows from column l on, modulo
            // 16, and so over two diagonals that are 16 apart.
            __syncwarp();
            float ahead = 0.f, wrapped = 0.f;
#pragma unroll
            for (int k = 0; k < TB_COLS; ++k) {
              const bool past = k + (lane & 15) >= TB_COLS;
              const float v = ds_walk[k * (TB_DS_PITCH + 1) - (past ? TB_COLS : 0)];
              ahead += past ? 0.f : v;
              wrapped += past ? v : 0.f;
            }
            float* to = dacc + warp * span + (a0 + warp * 32 + (lane & 16)) - (b0 + c) + side - (lane & 15);
            to[0] += ahead;
            __syncwarp();  // the other half's offsets are 16 further on
            to[TB_COLS] += wrapped;
            __syncwarp();
          }
        }
      };
      if (edge) walk(std::integral_constant<int, 2>());
      else if (far) walk(std::integral_constant<int, 0>());
      else walk(std::integral_constant<int, 1>());
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      const float2 f = both(sum);
      if (!KV) r += f.x + f.y;
      else {
        if (far > 0) after += f.x + f.y;
        else if (far < 0) before += f.x + f.y;
        if (tile == n_tiles - 1) finish_table(head_of(n / n_tiles));
      }
    }
    ok = ok && wait(done, (steps - 1) & 1, ERR_TC_O);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    if (!KV) {
      T* to = row_of(g.dq, row);
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t pk[32], dk[32];
        tc_ld32(mine + TB_ACC1_COL + c, pk);
        tc_ld32(mine + TB_ACC2_COL + c, dk);
        tc_wait_ld();
        if (to) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = !ok ? NAN : in ? (__uint_as_float(dk[j + e]) - r * __uint_as_float(pk[j + e])) * g.scale : 0.f;
            *reinterpret_cast<uint4*>(to + c + j) = Vec16<T>::down(v);
          }
        }
      }
      if (in) g.delta[((int64_t)w.b * g.heads + w.head) * g.tokens + row] = ok ? d + r : NAN;
    } else {
      constexpr int SP = D + 4;
      static_assert(2 * TC_Q * SP * 4 <= tb_operands<D, true>(), "the sums fit the operands");
      float* sums = reinterpret_cast<float*>(operands);  // [dv, dk][TC_Q][SP]
#pragma unroll 1
      for (int c = 0; c < 2 * D; c += 32) {
        uint32_t raw[32];
        const int which = c / D, col = c % D;
        tc_ld32(mine + (which ? TB_ACC2_COL : TB_ACC1_COL) + col, raw);
        tc_wait_ld();
        const float f = which ? g.scale : 1.f;
        if (ranks == 1) {
          T* to = row_of(which ? g.dk : g.dv, row);
          if (to) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = !ok ? NAN : in ? __uint_as_float(raw[j + e]) * f : 0.f;
              *reinterpret_cast<uint4*>(to + col + j) = Vec16<T>::down(v);
            }
          }
        } else {
          float4* to = reinterpret_cast<float4*>(sums + (which * TC_Q + threadIdx.x) * SP + col);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = !ok ? NAN : in ? __uint_as_float(raw[j + e]) * f : 0.f;
            to[j / 4] = make_float4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
  }
  if (KV && ranks > 1) {
    constexpr int SP = D + 4;
    float* sums = reinterpret_cast<float*>(operands);
    if (gave_up)
      for (int i = threadIdx.x; i < 2 * TC_Q * SP; i += TC_THREADS) sums[i] = NAN;
    rel_cluster_sync();
    for (int c = rank * TC_THREADS + threadIdx.x; c < 2 * TC_Q * (D / 8); c += ranks * TC_THREADS) {
      const int which = c / (TC_Q * (D / 8)), row = c / (D / 8) % TC_Q, part = c % (D / 8) * 8;
      T* to = row_of(which ? g.dk : g.dv, a0 + row);
      if (!to) continue;
      const float* from = sums + (which * TC_Q + row) * SP + part;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < ranks; ++i) {
        const float4 a = get_remote(from, i), b = get_remote(from + 4, i);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
      }
      *reinterpret_cast<uint4*>(to + part) = Vec16<T>::down(v);
    }
    rel_cluster_sync();  // a block's sums stay until all have been read
  }
}

namespace {

template <typename T, int D, bool KV> int run_form(const RelArgs& g, const CUtensorMap (&maps)[4], cudaStream_t st) {
  static std::atomic<uint64_t> raised{0};
  int rc = raise_smem(k_rel_tc_bwd<T, D, KV>, tb_smem<D, KV>(1024, 512), raised);
  if (rc) return rc;
  const int ranks = KV ? rel_ranks(g) : 1, tiles = (g.tokens + TC_Q - 1) / TC_Q;
  const int64_t blocks = (int64_t)tiles * g.batch * (KV ? g.heads_kv : g.heads) * ranks;
  if (blocks > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(TC_THREADS);
  cfg.dynamicSmemBytes = tb_smem<D, KV>(g.reach, g.buckets);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, k_rel_tc_bwd<T, D, KV>, maps[0], maps[1], maps[2], maps[3], g, tiles, ranks);
}

template <typename T, int D> int run_tc_bwd(const RelArgs& g, cudaStream_t st) {
  constexpr bool BF = TcType<T>::FORMAT == 1;
  for (const bool kv : {false, true}) {
    const int rows_q = kv ? TC_K : TC_Q, rows_k = kv ? TC_Q : TC_K;
    CUtensorMap q, k, v, d;
    int rc = tc_map(&q, g.q, g.qs, g, g.heads, D, rows_q, BF);
    if (!rc) rc = tc_map(&d, g.dout, g.ds, g, g.heads, D, rows_q, BF);
    if (!rc) rc = tc_map(&k, g.k, g.ks, g, g.heads_kv, D, rows_k, BF);
    if (!rc) rc = tc_map(&v, g.v, g.vs, g, g.heads_kv, D, rows_k, BF);
    if (!rc) rc = kv ? run_form<T, D, true>(g, {k, v, q, d}, st) : run_form<T, D, false>(g, {q, d, k, v}, st);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace

int rel_attention_tc_backward(const RelArgs& g, int dtype, int head_dim, cudaStream_t st) {
  if (dtype == MGBS_DT_BF16) return head_dim == 32 ? run_tc_bwd<__nv_bfloat16, 32>(g, st) : run_tc_bwd<__nv_bfloat16, 64>(g, st);
  return head_dim == 32 ? run_tc_bwd<__half, 32>(g, st) : run_tc_bwd<__half, 64>(g, st);
}

}  // namespace mgbs
