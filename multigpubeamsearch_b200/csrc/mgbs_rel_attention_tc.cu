// Forward attention with a relative bias over tiles of 128 queries x 128 keys on tcgen05.  Per block (128 queries of one
// head): four softmax warps (a thread owns a query row), four loading warps, one warp that issues the products.
//
//   S(t) = Q K(t)^T into tensor memory (128 columns); the softmax warps read it, take the row maximum, write
//   P(t) = 2^(s - m) as 16-bit pairs into tensor memory (64 columns), from where it is the A operand of O += P(t) V(t).
//   S(t + 1) is issued before O += P(t) V(t), so that the exponentials of the next tile do not wait for it.
//
// The reference m of a row follows its maximum only when that has grown by more than 2^8 (P then stays within both
// 16-bit types), so that the accumulator O, which sits in tensor memory too, is rarely rescaled.  256 of the 512 columns
// and 80 KB: two blocks per SM, one's exponentials over the other's products and waits.  What bounds it: the
// exponentials, 128 x 128 of them per tile at 16 a clock against 512 clocks of products.
//
// Operands lie in shared memory in the layout without swizzle, 16-byte pieces of 8 rows side by side (128 bytes): the
// same bytes are K-major rows for Q and K and MN-major rows for V, copied asynchronously with zeros for what lies past
// the length (padding is never read, and P = 0 must not meet a NaN).  Every wait is bounded: a block that gives up
// writes NaN and the error word.

#include <math.h>

#include "mgbs_rel_attention.cuh"
#include "mgbs_tc.cuh"

namespace mgbs {

constexpr int TC_TILE = 128;
constexpr int TC_THREADS = 288;
constexpr int TC_RIM = 2 * TC_TILE;
constexpr int TC_GROUP = 128;                       // bytes of 8 rows x 16 bytes
constexpr int TC_CHUNK = TC_TILE / 8 * TC_GROUP;    // bytes between a row's 16-byte pieces
constexpr float TC_GROWTH = 8.f;                    // log2 of how far P may exceed 1
constexpr int ERR_TC_LOAD = 21, ERR_TC_FREE = 22, ERR_TC_S = 23, ERR_TC_P = 24, ERR_TC_O = 25;

template <int D> struct TcShape {
  static constexpr int MAT = D / 8 * TC_CHUNK;  // bytes of one 128-row operand
  static constexpr int P_COL = 128, O_COL = 192;
};

// Matrix descriptor without swizzle: start, leading and stride byte offsets in 16-byte units, version 1.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) | (1ull << 46);
}
// kind::f16 instruction descriptor: float32 accumulators; operand type (f16 0, bf16 1); B MN-major; N; M = 128
template <typename T> __device__ __forceinline__ constexpr uint32_t tc_idesc(int n, bool b_mn) {
  return (1u << 4) | ((sizeof(T) == 2 && !__is_same(T, __half) ? 1u : 0u) << 7) | ((!__is_same(T, __half) ? 1u : 0u) << 10) |
         ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TC_TILE >> 4) << 24);
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
        "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]),
        "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A wait that ends after a second at most, or as soon as another of the block has given up.
static __device__ __noinline__ bool tc_wait_slow(uint32_t bar, uint32_t parity, int* gave_up, int* error, int code) {
  uint64_t start, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (*reinterpret_cast<volatile int*>(gave_up)) return false;
    if (now - start > 1000000000ull) break;
  }
  if (atomicExch(gave_up, 1) == 0 && error) atomicCAS(error, 0, code);
  return false;
}

// 128 rows from `row` on into the operand layout, by four warps; rows from `len` on become zeros.  A warp's instruction
// takes 8 rows x 4 pieces: whole 64-byte runs of global memory, and 128-byte runs of shared memory.
template <typename T, int D> __device__ __forceinline__ void tc_stage(uint32_t dst, const T* head, int64_t token_stride, int row, int len, int warp, int lane) {
  const int in_group = lane & 7, piece = lane >> 3;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int group = warp * 4 + g, t = row + group * 8 + in_group;
    const bool in = t < len;
    const T* src = head + (in ? t * token_stride : 0) + piece * 8;
    const uint32_t to = dst + group * TC_GROUP + in_group * 16 + piece * TC_CHUNK;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) copy16(to + c * 4 * TC_CHUNK, src + c * 32, in ? 16u : 0u);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(TC_THREADS, 2) k_rel_tc(const __grid_constant__ RelArgs g, int tiles) {
  using Shape = TcShape<D>;
  extern __shared__ __align__(128) uint8_t tc_smem[];
  __shared__ __align__(8) uint64_t bars[7];
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const Where w0 = rel_where(tiles, g.heads);
  const int tile = tiles - 1 - w0.tile, head = w0.head, batch = w0.b;  // under a causal mask the longest rows start first
  if (batch >= rel_batch(g)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = rel_length(g, batch), i0 = tile * TC_TILE;
  T* out = static_cast<T*>(g.out) + ((int64_t)batch * g.tokens * g.heads + head) * D;
  float2* stats = g.stats ? g.stats + ((int64_t)batch * g.heads + head) * g.tokens : nullptr;
  if (i0 >= len) {
    for (int r = threadIdx.x; r < TC_TILE && i0 + r < g.tokens; r += TC_THREADS) {
      uint4* to = reinterpret_cast<uint4*>(out + (int64_t)(i0 + r) * g.heads * D);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) to[c] = make_uint4(0u, 0u, 0u, 0u);
      if (stats) stats[i0 + r] = make_float2(0.f, INFINITY);
    }
    return;
  }
  const uint32_t q_at = smem_u32(tc_smem), kv_at = q_at + Shape::MAT;
  float* bt = reinterpret_cast<float*>(tc_smem + 5 * Shape::MAT);
  const uint32_t bar = smem_u32(bars);
  const uint32_t full = bar, empty = bar + 16, s_full = bar + 32, p_full = bar + 40, o_done = bar + 48;
  if (threadIdx.x == 0) {
    mbar_init(full, 128); mbar_init(full + 8, 128);
    mbar_init(empty, 1); mbar_init(empty + 8, 1);
    mbar_init(s_full, 1); mbar_init(p_full, 128); mbar_init(o_done, 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
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
  const int last = g.causal ? min(len, i0 + TC_TILE) : len, n_tiles = (last + TC_TILE - 1) / TC_TILE;

  if (warp >= 4 && warp < 8) {
    const int head_kv = head / (g.heads / g.heads_kv);
    const T* q = static_cast<const T*>(g.q) + batch * g.qs[0] + head * g.qs[2];
    const T* k = static_cast<const T*>(g.k) + batch * g.ks[0] + head_kv * g.ks[2];
    const T* v = static_cast<const T*>(g.v) + batch * g.vs[0] + head_kv * g.vs[2];
    tc_stage<T, D>(q_at, q, g.qs[1], i0, len, warp - 4, lane);
    auto load = [&](int t) {
      const uint32_t to = kv_at + (t & 1) * 2 * Shape::MAT;
      tc_stage<T, D>(to, k, g.ks[1], t * TC_TILE, len, warp - 4, lane);
      tc_stage<T, D>(to + Shape::MAT, v, g.vs[1], t * TC_TILE, len, warp - 4, lane);
      copy_commit();
    };
    load(0);
    if (n_tiles > 1) load(1);
    for (int t = 0; t < n_tiles; ++t) {
      if (t == 0 && n_tiles > 1) copy_wait<1>();
      else copy_wait<0>();
      async_fence();
      mbar_arrive(full + (t & 1) * 8);
      // tile t has to be announced before tile t - 1 is waited for: its scores go before the product that frees t - 1
      if (t > 0 && t + 1 < n_tiles) {
        if (!wait(empty + ((t - 1) & 1) * 8, ((t - 1) / 2) & 1, ERR_TC_FREE)) break;
        load(t + 1);
      }
    }
    copy_wait<0>();
  } else if (warp == 8) {
    if (lane == 0) {
      constexpr uint32_t id_s = tc_idesc<T>(TC_TILE, false), id_o = tc_idesc<T>(D, true);
      const uint64_t q_desc = tc_desc(q_at, TC_CHUNK, TC_GROUP);
      auto score = [&](int t) {
        const uint64_t k_desc = tc_desc(kv_at + (t & 1) * 2 * Shape::MAT, TC_CHUNK, TC_GROUP);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc_mma_f16(tmem, q_desc + kk * (2 * TC_CHUNK >> 4), k_desc + kk * (2 * TC_CHUNK >> 4), id_s, kk > 0);
        tc_commit(s_full);
      };
      bool ok = wait(full, 0, ERR_TC_LOAD);
      if (ok) {
        tc_fence_after();
        score(0);
      }
      for (int t = 0; ok && t < n_tiles; ++t) {
        if (t + 1 < n_tiles) ok = wait(full + ((t + 1) & 1) * 8, ((t + 1) / 2) & 1, ERR_TC_LOAD);
        ok = ok && wait(p_full, t & 1, ERR_TC_P);
        if (!ok) break;
        tc_fence_after();
        if (t + 1 < n_tiles) score(t + 1);
        // V: 8 keys of 16 bytes per group, groups of keys TC_GROUP apart, pieces of the head TC_CHUNK apart
        const uint64_t v_desc = tc_desc(kv_at + (t & 1) * 2 * Shape::MAT + Shape::MAT, TC_GROUP, TC_CHUNK);
#pragma unroll
        for (int kk = 0; kk < TC_TILE / 16; ++kk)
          tc_mma_ts(tmem + Shape::O_COL, tmem + Shape::P_COL + kk * 8, v_desc + kk * (2 * TC_GROUP >> 4), id_o, t > 0 || kk > 0);
        tc_commit(empty + (t & 1) * 8);
        tc_commit(o_done);
      }
    }
    __syncwarp();
  } else {
    const int row = i0 + threadIdx.x;
    const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
    float m = -INFINITY, l = 0.f;
    const Pair sl2 = pair(g.sl2, g.sl2);
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      ok = wait(s_full, t & 1, ERR_TC_S);
      if (!ok) break;
      tc_fence_after();
      const int j0 = t * TC_TILE;
      const int far = j0 - (i0 + TC_TILE - 1) >= g.reach ? 1 : i0 - (j0 + TC_TILE - 1) >= g.reach ? -1 : 0;
      const bool edge = j0 + TC_TILE > len || i0 + TC_TILE > len || (g.causal && j0 + TC_TILE > i0 + 1);
      const float fixed = far > 0 ? bt[2 * side] : bt[0];
      const float* by_offset = bt + j0 - row + side;
      // scores of 32 keys, scaled and biased, hidden ones at -inf
      auto scores = [&](int c, float (&s)[32]) {
        uint32_t raw[32];
        tc_ld32(mine + c * 32, raw);
        tc_wait_ld();
        if (far) {
          const Pair b2 = pair(fixed, fixed);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 f = both(fma2(pair(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), sl2, b2));
            s[j] = f.x; s[j + 1] = f.y;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 f = both(fma2(pair(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), sl2, pair(by_offset[c * 32 + j], by_offset[c * 32 + j + 1])));
            s[j] = f.x; s[j + 1] = f.y;
          }
        }
        if (edge) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const int key = j0 + c * 32 + j;
            if (key >= len || row >= len || (g.causal && key > row)) s[j] = -INFINITY;
          }
        }
      };
      float top = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float s[32];
        scores(c, s);
#pragma unroll
        for (int j = 0; j < 32; ++j) top = fmaxf(top, s[j]);
      }
      if (t > 0) {
        ok = wait(o_done, (t - 1) & 1, ERR_TC_O);
        if (!ok) break;
        tc_fence_after();
      }
      if (t == 0) m = top;
      else if (__any_sync(0xffffffffu, top > m + TC_GROWTH)) {
        const float to = top > m + TC_GROWTH ? top : m;
        const float f = to == -INFINITY ? 1.f : fast_exp2(m - to);
        m = to;
        l *= f;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t raw[32];
          tc_ld32(mine + Shape::O_COL + c * 32, raw);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) raw[j] = __float_as_uint(__uint_as_float(raw[j]) * f);
          tc_st32(mine + Shape::O_COL + c * 32, raw);
        }
      }
      const float base = m == -INFINITY ? 0.f : m;  // no key yet: all terms 0
      const Pair minus = pair(-base, -base);
      Pair sum = pair(0.f, 0.f);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float s[32];
        scores(c, s);
        uint32_t p[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const Pair e = exp2_2(add2(pair(s[j], s[j + 1]), minus));
          sum = add2(sum, e);
          const float2 f = both(e);
          p[j / 2] = pack2<T>(f.x, f.y);
        }
        tc_st16(mine + Shape::P_COL + c * 16, p);
      }
      const float2 both_sums = both(sum);
      l += both_sums.x + both_sums.y;
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(p_full);
    }
    if (ok) ok = wait(o_done, (n_tiles - 1) & 1, ERR_TC_O);
    tc_fence_after();
    const bool some = row < len && l != 0.f;
    const float inv = ok ? (some ? 1.f / l : 0.f) : NAN;
    T* to = out + (int64_t)row * g.heads * D;
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t raw[32];
      tc_ld32(mine + Shape::O_COL + c * 32, raw);
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
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
  }
}

namespace {

template <typename T, int D> int run_tc(const RelArgs& g, cudaStream_t st) {
  static std::atomic<uint64_t> raised{0};
  const int most = 113 * 1024;
  const int rc = raise_smem(k_rel_tc<T, D>, most, raised);
  if (rc) return rc;
  const int tiles = (g.tokens + TC_TILE - 1) / TC_TILE;
  const int64_t blocks = (int64_t)tiles * g.heads * g.batch;
  if (blocks > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  // never more than two blocks on an SM: a third would wait for tensor memory
  int smem = 5 * TcShape<D>::MAT + (2 * (g.reach + TC_RIM) + 1) * 4;
  if (smem < 78 * 1024) smem = 78 * 1024;
  k_rel_tc<T, D><<<(unsigned)blocks, TC_THREADS, smem, st>>>(g, tiles);
  return (int)cudaGetLastError();
}

}  // namespace

int rel_attention_tc(const RelArgs& g, int dtype, int head_dim, cudaStream_t st) {
  if (dtype == MGBS_DT_BF16) return head_dim == 32 ? run_tc<__nv_bfloat16, 32>(g, st) : run_tc<__nv_bfloat16, 64>(g, st);
  return head_dim == 32 ? run_tc<__half, 32>(g, st) : run_tc<__half, 64>(g, st);
}

}  // namespace mgbs
