// Forward attention with a relative bias over tiles of 128 queries x 64 keys on tcgen05.  Per block (128 queries of one
// head): four softmax warps (a thread owns a query row), one warp that issues the products, one that loads by TMA.
//
//   S(t) = Q K(t)^T into tensor memory (two buffers of 64 columns); the softmax warps read it and write
//   P(t) = 2^(s - m) as 16-bit pairs into tensor memory (two buffers of 32 columns), from where it is the A operand of
//   O += P(t) V(t).  With two buffers of each, the scores of the next tile are there when a tile's softmax ends.
//
// The reference m of a row is its maximum over the first tile.  It follows only when a later tile's sum of P exceeds 2^14
// (up to there P fits both 16-bit types, and float32 sums lose nothing): then the tile is done again from its true
// maximum and the accumulator O, in tensor memory too, is rescaled.  So a tile takes no maximum as a rule.
// 256 of the 512 columns and 84 KB: two blocks per SM, one's exponentials over the other's products and waits.  What
// bounds it: the exponentials, 128 x 64 of them per tile at 16 a clock against 256 clocks of products, and the blocks'
// number (512 over 296 places): 110 us at 2 x 4096 tokens, 8 heads of 64, of which the exponentials alone are 60 and with
// a quarter of them on the multiply-add pipe 45.
//
// Rows of 128 bytes (64 for heads of 32) in the swizzled layout of that width: K-major for Q and K, MN-major for V.
// Padding past a length is zeroed in V's last tile (P = 0 must not meet a NaN there); elsewhere it only reaches scores
// that are hidden.  Every wait is bounded: a block that gives up writes NaN and the error word.

#include <math.h>

#include "mgbs_rel_attention_tc.cuh"

namespace mgbs {

constexpr int TC_STAGES = 4;                        // tiles of K and of V in shared memory
constexpr float TC_GROWTH = 16384.f;                // how far a row's sum over a tile may grow before its reference follows
constexpr int TC_P_COL = 128, TC_O_COL = 192;       // columns: S at 0 and 64, P at 128 and 160, O at 192

constexpr int TC_EVERY = 4;  // one pair of exponentials in so many goes to the multiply-add pipe (none 124 us,
                             // 3: 118, 5: 118, 4: 117 at 2 x 4096 tokens) where one bias serves a tile

// A tile as a softmax thread sees it.
struct TcTile {
  int far;  // 1 / -1: all keys beyond the reach after / before the queries, so that one bias serves
  bool edge;
  int j0, row, len, causal;
  float fixed;
  const float* by_offset;  // bias of key j0 + j at [j]
};

// Two scores of the tile, hidden ones at -inf.
__device__ __forceinline__ Pair tc_hide(const TcTile& w, int at, Pair s) {
  const int key = w.j0 + at;
  float2 f = both(s);
  if (key >= w.len || (w.causal && key > w.row)) f.x = -INFINITY;
  if (key + 1 >= w.len || (w.causal && key + 1 > w.row)) f.y = -INFINITY;
  return pair(f.x, f.y);
}

// A row's exact maximum over the tile.
static __device__ __noinline__ float tc_maximum(uint32_t scores, TcTile w, Pair sl2) {
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < TC_K / 32; ++c) {
    uint32_t raw[32];
    tc_ld32(scores + c * 32, raw);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const int at = c * 32 + j;
      const Pair b = w.far ? pair(w.fixed, w.fixed) : pair(w.by_offset[at], w.by_offset[at + 1]);
      const float2 f = both(tc_hide(w, at, fma2(pair(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), sl2, b)));
      top = fmaxf(top, fmaxf(f.x, f.y));
    }
  }
  return top;
}

__device__ __forceinline__ float clamp_above(float x) {  // NaN stays
  asm("min.NaN.f32 %0, %0, 0f42FE0000;" : "+f"(x));  // 127
  return x;
}
__device__ __forceinline__ float scaled(float y, float t, float x) {  // y 2^n, n in the low bits of t; whatever comes of an x below -125
  return x < -125.f ? 0.f : __int_as_float(__float_as_int(y) + (__float_as_int(t) << 23));
}
// 2^x on the multiply-add pipe: x = n + f with |f| <= 1/2, 2^f by the polynomial of degree 4 with the least largest relative
// error (2^-18.5, by exchange of its extreme points), n added to the exponent.  Below -125 the result is 0, as what weighs
// nothing must not be multiplied by a value near the type's largest; from 127 up, and for a NaN, it is far above the
// growth that makes the tile anew.
__device__ __forceinline__ Pair exp2_fma(Pair x) {
  float2 f = both(x);
  f = make_float2(clamp_above(f.x), clamp_above(f.y));
  x = pair(f.x, f.y);
  const Pair round = pair(12582912.f, 12582912.f);  // 1.5 * 2^23: the sum's low bits are n
  const Pair t = add2(x, round), n = add2(t, pair(-12582912.f, -12582912.f));
  const Pair r = fma2(n, pair(-1.f, -1.f), x);
  Pair y = fma2(r, pair(9.57010186330317e-3f, 9.57010186330317e-3f), pair(5.591786034055708e-2f, 5.591786034055708e-2f));
  y = fma2(r, y, pair(0.2402474483148465f, 0.2402474483148465f));
  y = fma2(r, y, pair(0.693121814743091f, 0.693121814743091f));
  y = fma2(r, y, pair(0.9999992614416005f, 0.9999992614416005f));
  const float2 v = both(y), e = both(t);
  return pair(scaled(v.x, e.x, f.x), scaled(v.y, e.y, f.y));
}

// P of the tile relative to `base` into tensor memory; returns the row's sum.
template <typename T, int MODE> __device__ __forceinline__ float tc_write_p(uint32_t scores, uint32_t to, const TcTile& w, Pair sl2, float base) {
  const Pair minus = pair(-base, -base), one = pair(w.fixed, w.fixed);
  Pair sum = pair(0.f, 0.f);
  auto two = [&](int at, uint32_t lo, uint32_t hi) {  // P of columns at and at + 1
    const bool fix = MODE == 0 || (MODE == 2 && w.far);
    Pair s = fma2(pair(__uint_as_float(lo), __uint_as_float(hi)), sl2, fix ? one : pair(w.by_offset[at], w.by_offset[at + 1]));
    if (MODE == 2) s = tc_hide(w, at, s);
    const Pair x = add2(s, minus), e = MODE == 0 && at / 2 % TC_EVERY == TC_EVERY - 1 ? exp2_fma(x) : exp2_2(x);
    sum = add2(sum, e);
    const float2 f = both(e);
    return pack2<T>(f.x, f.y);
  };
  if (MODE == 0) {  // the next 16 columns come while these are worked on
    uint32_t raw[2][16];
    tc_ld16(scores, raw[0]);
#pragma unroll
    for (int i = 0; i < TC_K / 16; ++i) {
      tc_wait_ld();
      if (i + 1 < TC_K / 16) tc_ld16(scores + (i + 1) * 16, raw[(i + 1) & 1]);
      uint32_t p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = two(i * 16 + 2 * j, raw[i & 1][2 * j], raw[i & 1][2 * j + 1]);
      tc_st8(to + i * 8, p);
    }
  } else {  // with biases to load as well, all at once is the faster: 8 heads of 64, 442368 tokens in sequences
           // of 512: 1158 us against 1204 us
    uint32_t raw[2][32];
    tc_ld32(scores, raw[0]);
    tc_ld32(scores + 32, raw[1]);
    tc_wait_ld();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t p[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) p[j] = two(c * 32 + 2 * j, raw[c][2 * j], raw[c][2 * j + 1]);
      tc_st16(to + c * 16, p);
    }
  }
  const float2 f = both(sum);
  return f.x + f.y;
}

// The same out of line, for a row's first tile and for new references.
template <typename T> static __device__ __noinline__ float tc_write_p_again(uint32_t scores, uint32_t to, TcTile w, Pair sl2, float base) {
  return tc_write_p<T, 2>(scores, to, w, sl2, base);
}

template <typename T, int D>
__global__ void __launch_bounds__(TC_THREADS, 2) k_rel_tc(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ RelArgs g, int tiles) {
  constexpr int Q_BYTES = TC_Q * D * 2, K_BYTES = TC_K * D * 2;
  extern __shared__ __align__(1024) uint8_t tc_smem[];
  __shared__ __align__(8) uint64_t bars[4 * TC_STAGES + 9];
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const Where w0 = rel_where(blockIdx.x, tiles, g.heads, g.batch);
  const int tile = tiles - 1 - w0.tile, head = w0.head, batch = w0.b;  // under a causal mask the longest rows start first
  if (batch >= rel_batch(g)) return;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int len = rel_length(g, batch), i0 = tile * TC_Q;
  T* out = static_cast<T*>(g.out) + ((int64_t)batch * g.tokens * g.heads + head) * D;
  float2* stats = g.stats ? g.stats + ((int64_t)batch * g.heads + head) * g.tokens : nullptr;
  if (i0 >= len) {
    for (int r = threadIdx.x; r < TC_Q && i0 + r < g.tokens; r += TC_THREADS) {
      uint4* to = reinterpret_cast<uint4*>(out + (int64_t)(i0 + r) * g.heads * D);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) to[c] = make_uint4(0u, 0u, 0u, 0u);
      if (stats) stats[i0 + r] = make_float2(0.f, INFINITY);
    }
    return;
  }
  const uint32_t q_at = (smem_u32(tc_smem) + 1023u) & ~1023u, k_at = q_at + Q_BYTES, v_at = k_at + TC_STAGES * K_BYTES;
  uint8_t* v_ptr = tc_smem + (v_at - smem_u32(tc_smem));
  float* bt = reinterpret_cast<float*>(v_ptr + TC_STAGES * K_BYTES);
  const uint32_t bar = smem_u32(bars);
  const uint32_t k_full = bar, v_full = bar + 8 * TC_STAGES, k_free = bar + 16 * TC_STAGES, v_free = bar + 24 * TC_STAGES;
  const uint32_t s_full = bar + 32 * TC_STAGES, p_full = s_full + 16, o_done = s_full + 32, q_full = s_full + 48, v_fixed = s_full + 56, drained = s_full + 64;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4 * TC_STAGES; ++i) mbar_init(bar + i * 8, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i * 8, 1);
      mbar_init(p_full + i * 8, 4);
      mbar_init(o_done + i * 8, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(v_fixed, 1);
    mbar_init(drained, 1);
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
  const int side = g.reach + TC_RIM;
  if (warp < 4) fill_bias<T>(g, head, bt, side, threadIdx.x, 128);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int last = g.causal ? min(len, i0 + TC_Q) : len, n_tiles = (last + TC_K - 1) / TC_K;
  // rows between the length and the tensor's end are padding that the last tile of V holds: zeroed before it is used
  const bool fix_v = len < g.tokens && n_tiles * TC_K > len;

  if (warp == 5) {
    const int head_kv = head / (g.heads / g.heads_kv);
    bool ok = true;
    if (lane == 0) {
      mbar_expect_tx(q_full, Q_BYTES);
      tma_load_4d(q_at, &map_q, i0, head, batch, q_full);
      int keys = 0, values = 0;  // tiles asked for
      while (values < n_tiles) {
        const int t = values, s = t % TC_STAGES, turn = t / TC_STAGES;
        if (turn > 0 && !(ok = wait(k_free + s * 8, (turn - 1) & 1, ERR_TC_FREE))) break;
        mbar_expect_tx(k_full + s * 8, K_BYTES);
        tma_load_4d(k_at + s * K_BYTES, &map_k, t * TC_K, head_kv, batch, k_full + s * 8);
        ++keys;
        if (turn > 0 && !(ok = wait(v_free + s * 8, (turn - 1) & 1, ERR_TC_FREE))) break;
        mbar_expect_tx(v_full + s * 8, K_BYTES);
        tma_load_4d(v_at + s * K_BYTES, &map_v, t * TC_K, head_kv, batch, v_full + s * 8);
        ++values;
      }
      if (!ok) {  // what has been asked for comes before the block ends
        tc_settle(q_full, 0);
        for (int t = max(0, keys - TC_STAGES); t < keys; ++t) tc_settle(k_full + t % TC_STAGES * 8, (t / TC_STAGES) & 1);
        for (int t = max(0, values - TC_STAGES); t < values; ++t) tc_settle(v_full + t % TC_STAGES * 8, (t / TC_STAGES) & 1);
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    if (fix_v && ok) {
      const int t = n_tiles - 1, s = t % TC_STAGES;
      ok = wait(v_full + s * 8, (t / TC_STAGES) & 1, ERR_TC_LOAD);
      if (__all_sync(0xffffffffu, ok)) {
        for (int c = (len - t * TC_K) * (D / 8) + lane; c < TC_K * (D / 8); c += 32) reinterpret_cast<uint4*>(v_ptr + s * K_BYTES)[c] = make_uint4(0u, 0u, 0u, 0u);
        async_fence();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_fixed);
      }
    }
  } else if (warp == 4) {
    // The whole warp walks and waits, one elected lane issues: descriptors then stay in uniform registers.  (With one lane
    // doing all of it, four products and a commit took 400 to 600 cycles.)
    constexpr uint32_t id_s = tc_idesc<T>(TC_K, false), id_o = tc_idesc<T>(D, true);
    const uint64_t q_desc = tc_desc<D>(q_at);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    auto score = [&](int t) {
      const int s = t % TC_STAGES;
      if (!__all_sync(0xffffffffu, wait(k_full + s * 8, (t / TC_STAGES) & 1, ERR_TC_LOAD))) return false;
      tc_fence_after();
      const uint64_t k_desc = tc_desc<D>(k_at + s * K_BYTES);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) tc_mma_f16(tm + (t & 1) * TC_K, q_desc + kk * 2, k_desc + kk * 2, id_s, kk > 0);
        tc_commit(k_free + s * 8);
        tc_commit(s_full + (t & 1) * 8);
      }
      return true;
    };
    bool ok = __all_sync(0xffffffffu, wait(q_full, 0, ERR_TC_LOAD)) && score(0) && (n_tiles < 2 || score(1));
    for (int t = 0; ok && t < n_tiles; ++t) {
      const int s = t % TC_STAGES;
      ok = wait(v_full + s * 8, (t / TC_STAGES) & 1, ERR_TC_LOAD) && (!fix_v || t + 1 < n_tiles || wait(v_fixed, 0, ERR_TC_LOAD)) &&
           wait(p_full + (t & 1) * 8, (t / 2) & 1, ERR_TC_P);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint64_t v_desc = tc_desc<D>(v_at + s * K_BYTES);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < TC_K / 16; ++kk)
          tc_mma_ts(tm + TC_O_COL, tm + TC_P_COL + (t & 1) * 32 + kk * 8, v_desc + kk * (16 * D * 2 >> 4), id_o, t > 0 || kk > 0);
        tc_commit(v_free + s * 8);
        tc_commit(o_done + (t & 1) * 8);
      }
      if (t + 2 < n_tiles) ok = score(t + 2);  // into the buffer that this tile's softmax has left
    }
    if (!ok) {  // products on their way end before the tensor memory is given back
      if (elect_one()) tc_commit(drained);
      __syncwarp();
      tc_settle(drained, 0);
    }
    __syncwarp();
  } else {
    const int row = i0 + threadIdx.x;
    const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
    float m = -INFINITY, l = 0.f;
    const Pair sl2 = pair(g.sl2, g.sl2);
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const int j0 = t * TC_K;
      const int far = j0 - (i0 + TC_Q - 1) >= g.reach ? 1 : i0 - (j0 + TC_K - 1) >= g.reach ? -1 : 0;
      const bool edge = j0 + TC_K > len || (g.causal && j0 + TC_K > i0 + 1);
      const TcTile where{far, edge, j0, row, len, g.causal, far > 0 ? bt[2 * side] : bt[0], bt + j0 - row + side};
      const uint32_t scores = mine + (t & 1) * TC_K, to = mine + TC_P_COL + (t & 1) * 32;
      // S(t) was issued behind O += P(t - 2) V(t - 2), so that P's buffer is free too
      ok = __all_sync(0xffffffffu, wait(s_full + (t & 1) * 8, (t / 2) & 1, ERR_TC_S));
      if (!ok) break;
      tc_fence_after();
      float sum = 0.f;
      bool again = t == 0;
      if (!again) {
        const float base = m == -INFINITY ? 0.f : m;  // no key yet: all terms 0
        sum = edge ? tc_write_p<T, 2>(scores, to, where, sl2, base)
              : far ? tc_write_p<T, 0>(scores, to, where, sl2, base) : tc_write_p<T, 1>(scores, to, where, sl2, base);
        // sums within 2^14 (P then fits both 16-bit types) need no new reference
        again = __any_sync(0xffffffffu, row < len && (!(sum <= TC_GROWTH) || m == -INFINITY));
      }
      if (again) {
        tc_wait_st();
        const float top = fmaxf(m, tc_maximum(scores, where, sl2));
        if (t > 0) {
          ok = __all_sync(0xffffffffu, wait(o_done + ((t - 1) & 1) * 8, ((t - 1) / 2) & 1, ERR_TC_O));  // O is still
          if (!ok) break;
          tc_fence_after();
          const float f = top == -INFINITY ? 1.f : fast_exp2(m - top);
          l *= f;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t raw[32];
            tc_ld32(mine + TC_O_COL + c * 32, raw);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) raw[j] = __float_as_uint(__uint_as_float(raw[j]) * f);
            tc_st32(mine + TC_O_COL + c * 32, raw);
          }
        }
        m = top;
        sum = tc_write_p_again<T>(scores, to, where, sl2, m == -INFINITY ? 0.f : m);
      }
      l += sum;
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + (t & 1) * 8);
    }
    if (ok) ok = __all_sync(0xffffffffu, wait(o_done + ((n_tiles - 1) & 1) * 8, ((n_tiles - 1) / 2) & 1, ERR_TC_O));
    tc_fence_after();
    const bool some = row < len && l != 0.f;
    const float inv = some ? 1.f / l : 0.f;
    T* to = out + (int64_t)row * g.heads * D;
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t raw[32];
      tc_ld32(mine + TC_O_COL + c * 32, raw);
      tc_wait_ld();
      if (row < g.tokens) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = !ok ? NAN : some ? __uint_as_float(raw[j * 8 + e]) * inv : 0.f;
          *reinterpret_cast<uint4*>(to + c * 32 + j * 8) = Vec16<T>::down(v);
        }
      }
    }
    if (stats && row < g.tokens) stats[row] = some ? make_float2(m, log2f(l)) : make_float2(0.f, INFINITY);
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
  }
}

namespace {

template <typename T, int D> int run_tc(const RelArgs& g, cudaStream_t st) {
  static std::atomic<uint64_t> raised{0};
  int rc = raise_smem(k_rel_tc<T, D>, 113 * 1024, raised);
  if (rc) return rc;
  const int tiles = (g.tokens + TC_Q - 1) / TC_Q;
  const int64_t blocks = (int64_t)tiles * g.heads * g.batch;
  if (blocks > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  constexpr bool BF = TcType<T>::FORMAT == 1;
  CUtensorMap q, k, v;
  rc = tc_map(&q, g.q, g.qs, g, g.heads, D, TC_Q, BF);
  if (!rc) rc = tc_map(&k, g.k, g.ks, g, g.heads_kv, D, TC_K, BF);
  if (!rc) rc = tc_map(&v, g.v, g.vs, g, g.heads_kv, D, TC_K, BF);
  if (rc) return rc;
  // never more than two blocks on an SM: a third would wait for tensor memory
  int smem = 1024 + (TC_Q + 2 * TC_STAGES * TC_K) * D * 2 + (2 * (g.reach + TC_RIM) + 1) * 4;
  if (smem < 78 * 1024) smem = 78 * 1024;
  k_rel_tc<T, D><<<(unsigned)blocks, TC_THREADS, smem, st>>>(q, k, v, g, tiles);
  return (int)cudaGetLastError();
}

}  // namespace

bool rel_attention_tc_fits(const RelArgs& g) { return tc_stride_fits(g.qs, g, g.heads) && tc_stride_fits(g.ks, g, g.heads_kv) && tc_stride_fits(g.vs, g, g.heads_kv); }
bool rel_attention_tc_backward_fits(const RelArgs& g) { return rel_attention_tc_fits(g) && tc_stride_fits(g.ds, g, g.heads); }

int rel_attention_tc(const RelArgs& g, int dtype, int head_dim, cudaStream_t st) {
  if (dtype == MGBS_DT_BF16) return head_dim == 32 ? run_tc<__nv_bfloat16, 32>(g, st) : run_tc<__nv_bfloat16, 64>(g, st);
  return head_dim == 32 ? run_tc<__half, 32>(g, st) : run_tc<__half, 64>(g, st);
}

}  // namespace mgbs
