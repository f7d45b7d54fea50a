// Softmax attention with a learned bias per head and distance bucket, forward and backward:
//   s_ij = scale q_i . k_j + table[bucket(j - i), h],  P = softmax_j(s),  o_i = sum_j P_ij v_j
//   delta_i = sum_j P_ij (do_i . v_j),  dS_ij = P_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij do_i
//   dtable[b, h] = sum over sequences and pairs with bucket(j - i) = b of dS_ij
//
// Long sequences are in the files of the tcgen05 forms; the rest is here, on the warp-level matrix instruction (m16n8k16,
// 16-bit operands, float32 accumulators): short sequences, and strides that TMA cannot describe.  The scorer's 54 tokens
// take 749 us at 32768 sequences, 8 heads of 32, against 560 us for their bytes; what bounds them is the fixed latency of a
// warp's chain of products and exponentials with 16 warps on a multiprocessor (memory is busy for half of the time), so
// the time follows the clock: 880 us where it drops under load.  Scores, softmax statistics, delta and all sums stay in
// float32; P and dS are rounded to the operands' 16 bits as inputs of the next product, because that product takes 16
// bits (1.7e-3 -> 2.0e-3 of the output's norm in bfloat16, 2.1e-4 -> 2.9e-4 in float16 against products in 32 bits).
//
// Sequences of up to 64 tokens are one tile: a warp owns 16 query rows of one (sequence, head), a group of warps walks
// over the sequences of ONE head, so that the head's biases live in registers as the products' initial accumulators,
// and the backward pass sums dS over its sequences in registers (one add per score) and bins it by bucket once at its
// end.  Longer sequences go in tiles of 64 x 64 with a running maximum and sum.  Every sum is in a fixed order: no atomics.

#include <math.h>

#include "mgbs_operators.cuh"
#include "mgbs_counted.cuh"
#include "mgbs_rel_attention.cuh"

namespace mgbs {

constexpr int REL_THREADS = 128;
// Blocks per multiprocessor that a kernel's registers are held to, each the fastest of those tried:
constexpr int REL_FWD_BLOCKS = 4;  // 3: 806 us against 749 us at 32768 x 54 tokens, 8 heads of 32
constexpr int REL_BWD_BLOCKS = 3;  // 2: 546 us against 538 us at 8192 x 54 tokens
constexpr int REL_Q_BLOCKS = 2;    // 3: 93 us, 4: 121 us against 88 us at 6 x 1501 causal padded tokens, 8 heads of 64 over 2
constexpr int REL_KV_BLOCKS = 3;   // 2: 164 us, 4: 152 us against 134 us there
// rows of the short form's matrices are padded by 16 bytes: eight rows then start in distinct banks
template <int D> struct RelTile { static constexpr int PITCH = D + 8; };

// lane addresses inside a 16 x 16 block for ldmatrix (elements)
template <int PITCH> __device__ __forceinline__ int frag_a(int lane) { return ((lane & 7) + ((lane >> 3) & 1) * 8) * PITCH + (lane >> 4) * 8; }
template <int PITCH> __device__ __forceinline__ int frag_b(int lane) { return ((lane & 7) + (lane >> 4) * 8) * PITCH + ((lane >> 3) & 1) * 8; }

// s[2 per 16 columns] += A (16 x D, fragments a) times rows [16 jj, +16) of a row-major matrix, transposed: s = A M^T
template <typename T, int D> __device__ __forceinline__ void rows_product(float (&s0)[4], float (&s1)[4], const uint32_t (&a)[D / 16][4], uint32_t m) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    uint32_t b[4];
    ldsm4(b, m + kk * 32);
    mma16816<T>(s0, a[kk], b[0], b[1]);
    mma16816<T>(s1, a[kk], b[2], b[3]);
  }
}
// The same from initial values c0, c1.
template <typename T, int D>
__device__ __forceinline__ void rows_product_from(float (&s0)[4], float (&s1)[4], const float (&c0)[4], const float (&c1)[4], const uint32_t (&a)[D / 16][4], uint32_t m) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    uint32_t b[4];
    ldsm4(b, m + kk * 32);
    if (kk == 0) {
      mma16816_from<T>(s0, c0, a[kk], b[0], b[1]);
      mma16816_from<T>(s1, c1, a[kk], b[2], b[3]);
    } else {
      mma16816<T>(s0, a[kk], b[0], b[1]);
      mma16816<T>(s1, a[kk], b[2], b[3]);
    }
  }
}
// o (16 x D) += a (16 x 16) times 16 rows of a row-major matrix
template <typename T, int D> __device__ __forceinline__ void cols_product(float (&o)[D / 8][4], const uint32_t (&a)[4], uint32_t m) {
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    uint32_t b[4];
    ldsm4_t(b, m + n * 32);
    mma16816<T>(o[2 * n], a, b[0], b[1]);
    mma16816<T>(o[2 * n + 1], a, b[2], b[3]);
  }
}

// Rows r0 and r0 + 8 of a 16 x D accumulator, times f0 / f1, to global memory in 16-byte stores (row pointers p0, p1;
// null: not stored).  Lanes of a quad exchange their 4-byte pieces first.
template <typename T, int D> __device__ __forceinline__ void store_rows(const float (&o)[D / 8][4], float f0, float f1, T* p0, T* p1) {
  const int tig = threadIdx.x & 3;
#pragma unroll
  for (int g = 0; g < D / 32; ++g) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<T>(o[4 * g + i][0] * f0, o[4 * g + i][1] * f0);
    quad_transpose(r);
    if (p0) *reinterpret_cast<uint4*>(p0 + (4 * g + tig) * 8) = make_uint4(r[0], r[1], r[2], r[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<T>(o[4 * g + i][2] * f1, o[4 * g + i][3] * f1);
    quad_transpose(r);
    if (p1) *reinterpret_cast<uint4*>(p1 + (4 * g + tig) * 8) = make_uint4(r[0], r[1], r[2], r[3]);
  }
}
template <typename T, int D> __device__ __forceinline__ void store_zero_rows(T* p0, T* p1) {
  const int tig = threadIdx.x & 3;
#pragma unroll
  for (int g = 0; g < D / 32; ++g) {
    if (p0) *reinterpret_cast<uint4*>(p0 + (4 * g + tig) * 8) = make_uint4(0u, 0u, 0u, 0u);
    if (p1) *reinterpret_cast<uint4*>(p1 + (4 * g + tig) * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// A warp's 16 x D accumulators, rows times f0 / f1, to `rows` rows of global memory (pitch row_size) through a strip of
// shared memory of its own (16 rows of PITCH), so that every lane stores 16 bytes.
template <typename T, int D> __device__ __forceinline__ void store_strip(const float (&o)[D / 8][4], float f0, float f1, T* strip, T* out, int64_t row_size, int rows) {
  constexpr int PITCH = RelTile<D>::PITCH, PARTS = D / 8;
  const int lane = threadIdx.x & 31;
  __syncwarp();  // what the strip held has been read
  const uint32_t at = smem_addr(strip) + frag_a<PITCH>(lane) * 2;
#pragma unroll
  for (int n = 0; n < D / 16; ++n)
    stsm4(at + n * 32, pack2<T>(o[2 * n][0] * f0, o[2 * n][1] * f0), pack2<T>(o[2 * n][2] * f1, o[2 * n][3] * f1),
          pack2<T>(o[2 * n + 1][0] * f0, o[2 * n + 1][1] * f0), pack2<T>(o[2 * n + 1][2] * f1, o[2 * n + 1][3] * f1));
  __syncwarp();
  const int row = lane / PARTS, part = lane % PARTS * 8;
#pragma unroll
  for (int i = 0; i < PARTS / 2; ++i) {
    const int r = row + i * (32 / PARTS);
    if (r < rows) *reinterpret_cast<uint4*>(out + r * row_size + part) = *reinterpret_cast<const uint4*>(strip + r * PITCH + part);
  }
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// ------------------------------------------------------------------------------------------------------------------
// Up to 64 tokens
// ------------------------------------------------------------------------------------------------------------------

// Groups of a block: four warps are cut into groups of one, two or four; a group of three is a block of three.
template <int STRIPS> struct Groups { static constexpr int N = STRIPS == 1 ? 4 : STRIPS == 2 ? 2 : 1, THREADS = N * STRIPS * 32; };

template <int STRIPS> __device__ __forceinline__ void group_sync(int group) {
  if (STRIPS == 1) __syncwarp();
  else if (STRIPS > 2) __syncthreads();  // the group is the block
  else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(STRIPS * 32) : "memory");
}

// A group of STRIPS warps and the sequences it walks over: stream s serves head s % heads, sequences s / heads + i n.
template <int STRIPS> struct Stream {
  int group, strip, lane, first, step, head, id;
  bool live;
  __device__ __forceinline__ explicit Stream(const RelArgs& g) {
    const int warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    group = warp / STRIPS;
    strip = warp % STRIPS;
    id = blockIdx.x * Groups<STRIPS>::N + group;
    step = gridDim.x * Groups<STRIPS>::N / g.heads;
    live = id < step * g.heads;
    head = id % g.heads;
    first = id / g.heads;
  }
};

// A thread's part in copying one head's rows into shared memory, sequence after sequence of a stream: 16 bytes of every
// (STRIPS * 32 / parts)-th row.  Rows from `len` on become zeros; rows past `tokens` are not touched.
template <typename T, int D, int STRIPS> struct RowCopy {
  static constexpr int PITCH = RelTile<D>::PITCH, PARTS = D / 8, ROW_STEP = STRIPS * 32 / PARTS, TURNS = 16 * STRIPS / ROW_STEP;
  const T* src;
  int64_t next;  // elements to the stream's next sequence
  __device__ __forceinline__ RowCopy(const void* base, const int64_t (&s)[3], int head, int first, int step, int thread) {
    src = static_cast<const T*>(base) + first * s[0] + head * s[2] + (thread / PARTS) * s[1] + thread % PARTS * 8;
    next = step * s[0];
  }
  static __device__ __forceinline__ uint32_t place(int thread) { return (uint32_t)((thread / PARTS * PITCH + thread % PARTS * 8) * 2); }
  __device__ __forceinline__ void go(uint32_t dst, int64_t token_stride, int row, int tokens, int len) {
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int t = row + i * ROW_STEP;
      if (t < tokens) copy16(dst + i * ROW_STEP * PITCH * 2, src + i * ROW_STEP * token_stride, t < len ? 16u : 0u);
    }
    src += next;
  }
};

// Scores of a warp's 16 rows against 16 * STRIPS keys, as initial accumulators `bias` (bias / scale) + products, with
// what the masks hide at -inf.  All blocks of keys, also the empty ones: branches would keep the products from overlapping.
template <typename T, int D, int STRIPS>
__device__ __forceinline__ void short_scores(float (&s)[2 * STRIPS][4], const float (&bias)[2 * STRIPS][4], const uint32_t (&qa)[D / 16][4],
                                             uint32_t k_addr, bool masked, int len, int causal, int row0) {
  constexpr int PITCH = RelTile<D>::PITCH;
  const int tig = threadIdx.x & 3;
#pragma unroll
  for (int jj = 0; jj < STRIPS; ++jj) {
    rows_product_from<T, D>(s[2 * jj], s[2 * jj + 1], bias[2 * jj], bias[2 * jj + 1], qa, k_addr + jj * 16 * PITCH * 2);
  }
  if (masked) {
#pragma unroll
    for (int nb = 0; nb < 2 * STRIPS; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = nb * 8 + 2 * tig + (e & 1), i = row0 + (e >> 1) * 8;
        if (j >= len || i >= len || (causal && j > i)) s[nb][e] = -INFINITY;
      }
  }
}

// bias / scale of a warp's rows; keys from `tokens` on at -inf, rows from there on 0.
template <typename T, int STRIPS> __device__ __forceinline__ void short_bias(const RelArgs& g, int head, int row0, float (&bias)[2 * STRIPS][4]) {
  const int tig = threadIdx.x & 3;
  const float most = REL_BIG / fmaxf(1.f, g.sl2);
#pragma unroll
  for (int nb = 0; nb < 2 * STRIPS; ++nb)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = nb * 8 + 2 * tig + (e & 1), i = row0 + (e >> 1) * 8;
      bias[nb][e] = j >= g.tokens ? -INFINITY : i >= g.tokens ? 0.f : scaled_bias(rel_bias<T>(g, j - i, head), 1.f / g.scale, most);
    }
}

// In place: s -> 2^((s - max) sl2) (unnormalised).
template <int STRIPS> __device__ __forceinline__ void short_softmax(float (&s)[2 * STRIPS][4], float sl2) {
  float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
  for (int nb = 0; nb < 2 * STRIPS; ++nb) {
    m0 = fmaxf(m0, fmaxf(s[nb][0], s[nb][1]));
    m1 = fmaxf(m1, fmaxf(s[nb][2], s[nb][3]));
  }
  m0 = quad_max(m0);
  m1 = quad_max(m1);
  m0 = m0 == -INFINITY ? 0.f : m0;  // a row without keys: all terms 0
  m1 = m1 == -INFINITY ? 0.f : m1;
  // One fused step per term: the rounding of max * sl2 is a common factor of a row.  Where a row holds nothing but huge
  // masks that factor would overflow, so there the difference comes first.
  float top0 = m0 * sl2, top1 = m1 * sl2;
  if (__any_sync(0xffffffffu, fmaxf(fabsf(top0), fabsf(top1)) > 0x1p20f)) {
#pragma unroll
    for (int nb = 0; nb < 2 * STRIPS; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) { s[nb][e] -= m0; s[nb][2 + e] -= m1; }
    top0 = top1 = 0.f;
  }
#pragma unroll
  for (int nb = 0; nb < 2 * STRIPS; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      s[nb][e] = fast_exp2(fmaf(s[nb][e], sl2, -top0));
      s[nb][2 + e] = fast_exp2(fmaf(s[nb][2 + e], sl2, -top1));
    }
}

template <typename T> __device__ __forceinline__ void pack_a(uint32_t (&a)[4], const float (&x)[4], const float (&y)[4]) {
  a[0] = pack2<T>(x[0], x[1]);
  a[1] = pack2<T>(x[2], x[3]);
  a[2] = pack2<T>(y[0], y[1]);
  a[3] = pack2<T>(y[2], y[3]);
}

template <typename T, int D, int STRIPS> constexpr int short_fwd_smem() { return Groups<STRIPS>::N * 2 * 3 * 16 * STRIPS * RelTile<D>::PITCH * 2; }

template <typename T, int D, int STRIPS>
__global__ void __launch_bounds__(Groups<STRIPS>::THREADS, REL_FWD_BLOCKS) k_rel_short(const __grid_constant__ RelArgs g) {
  constexpr int PITCH = RelTile<D>::PITCH, ROWS = 16 * STRIPS, MAT = ROWS * PITCH;
  extern __shared__ __align__(16) uint8_t rel_smem[];
  const Stream<STRIPS> st(g);
  if (!st.live) return;  // whole groups; no barrier below spans groups
  const int batch = rel_batch(g);
  T* mine = reinterpret_cast<T*>(rel_smem) + st.group * 2 * 3 * MAT;
  const uint32_t base = smem_addr(mine);
  const int thread = st.strip * 32 + st.lane, gid = st.lane >> 2;
  const int head_kv = st.head / (g.heads / g.heads_kv);
  const int row0 = st.strip * 16 + gid;
  using Copy = RowCopy<T, D, STRIPS>;
  Copy q(g.q, g.qs, st.head, st.first, st.step, thread), k(g.k, g.ks, head_kv, st.first, st.step, thread), v(g.v, g.vs, head_kv, st.first, st.step, thread);
  const uint32_t place = base + Copy::place(thread);
  const int copy_row = thread / Copy::PARTS;
  auto load = [&](int b, int stage) {
    const int len = rel_length(g, b);
    const uint32_t to = place + stage * 3 * MAT * 2;
    q.go(to, g.qs[1], copy_row, g.tokens, len);
    k.go(to + MAT * 2, g.ks[1], copy_row, g.tokens, len);
    v.go(to + 2 * MAT * 2, g.vs[1], copy_row, g.tokens, len);
  };
  if (st.first < batch) load(st.first, 0);
  copy_commit();
  // rows past the last token stay zero in both stages: the copies never reach them
  for (int c = thread; c < (ROWS - g.tokens) * (D / 8); c += STRIPS * 32)
#pragma unroll
    for (int m = 0; m < 6; ++m)
      *reinterpret_cast<uint4*>(mine + m * MAT + (g.tokens + c / (D / 8)) * PITCH + c % (D / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
  float bias[2 * STRIPS][4];
  short_bias<T, STRIPS>(g, st.head, row0, bias);
  const int64_t row_size = (int64_t)g.heads * D;
  T* out = static_cast<T*>(g.out) + ((int64_t)st.first * g.tokens + st.strip * 16) * row_size + st.head * D;
  const int64_t next = (int64_t)st.step * g.tokens * row_size;
  const uint32_t ones = pack2<T>(1.f, 1.f);
  int stage = 0;
  for (int b = st.first; b < batch; b += st.step, stage ^= 1, out += next) {
    copy_wait<0>();
    group_sync<STRIPS>(st.group);  // this stage has arrived, and every warp has left the other one
    if (b + st.step < batch) load(b + st.step, stage ^ 1);
    copy_commit();
    const int len = rel_length(g, b);
    const uint32_t at = base + stage * 3 * MAT * 2;
    uint32_t qa[D / 16][4];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) ldsm4(qa[kk], at + (st.strip * 16 * PITCH + frag_a<PITCH>(st.lane)) * 2 + kk * 32);
    float s[2 * STRIPS][4];
    short_scores<T, D, STRIPS>(s, bias, qa, at + (MAT + frag_b<PITCH>(st.lane)) * 2, g.causal || len < g.tokens, len, g.causal, row0);
    short_softmax<STRIPS>(s, g.sl2);
    // The row sums come out of the product too, as one more column of ones: float32 sums of the same rounded terms that
    // multiply v, so that a row's weights still sum to one.
    float o[D / 8][4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
    for (int jj = 0; jj < STRIPS; ++jj) {
      uint32_t pa[4];
      pack_a<T>(pa, s[2 * jj], s[2 * jj + 1]);
      mma16816<T>(sum, pa, ones, ones);
      cols_product<T, D>(o, pa, at + (2 * MAT + jj * 16 * PITCH + frag_a<PITCH>(st.lane)) * 2);
    }
    // rows from the length on have no term: their sums are 0, and so are they
    store_strip<T, D>(o, sum[0] != 0.f ? 1.f / sum[0] : 0.f, sum[2] != 0.f ? 1.f / sum[2] : 0.f,
                      mine + stage * 3 * MAT + st.strip * 16 * PITCH, out, row_size, g.tokens - st.strip * 16);
  }
}

template <typename T, int D, int STRIPS> __host__ __device__ constexpr int short_bwd_group() {  // bytes of one group
  return ((2 * 4 + 1) * 16 * STRIPS * RelTile<D>::PITCH + 2 * 16 * STRIPS * (16 * STRIPS + 8)) * 2;
}

// Softmax and delta are computed anew from q, k, v, dout: neither the output nor statistics are read.
template <typename T, int D, int STRIPS>
__global__ void __launch_bounds__(Groups<STRIPS>::THREADS, REL_BWD_BLOCKS) k_rel_short_bwd(const __grid_constant__ RelArgs g) {
  constexpr int PITCH = RelTile<D>::PITCH, ROWS = 16 * STRIPS, MAT = ROWS * PITCH, PP = ROWS + 8;
  extern __shared__ __align__(16) uint8_t rel_smem[];
  const Stream<STRIPS> st(g);
  if (!st.live) return;
  uint8_t* raw = rel_smem + st.group * short_bwd_group<T, D, STRIPS>();
  T* mine = reinterpret_cast<T*>(raw);
  T* ps = mine + 8 * MAT;      // P, then dS: [query][key]
  T* dss = ps + ROWS * PP;
  T* out_strip = dss + ROWS * PP + st.strip * 16 * PITCH;  // of this warp alone
  const uint32_t base = smem_addr(mine), ps_at = smem_addr(ps), dss_at = smem_addr(dss);
  const int thread = st.strip * 32 + st.lane, gid = st.lane >> 2, tig = st.lane & 3;
  const int row0 = st.strip * 16 + gid;
  using Copy = RowCopy<T, D, STRIPS>;
  Copy q(g.q, g.qs, st.head, st.first, st.step, thread), k(g.k, g.ks, st.head, st.first, st.step, thread);
  Copy v(g.v, g.vs, st.head, st.first, st.step, thread), dout(g.dout, g.ds, st.head, st.first, st.step, thread);
  const uint32_t place = base + Copy::place(thread);
  const int copy_row = thread / Copy::PARTS;
  auto load = [&](int b, int stage) {
    const int len = rel_length(g, b);
    const uint32_t to = place + stage * 4 * MAT * 2;
    q.go(to, g.qs[1], copy_row, g.tokens, len);
    k.go(to + MAT * 2, g.ks[1], copy_row, g.tokens, len);
    v.go(to + 2 * MAT * 2, g.vs[1], copy_row, g.tokens, len);
    dout.go(to + 3 * MAT * 2, g.ds[1], copy_row, g.tokens, len);
  };
  if (st.first < g.batch) load(st.first, 0);
  copy_commit();
  for (int c = thread; c < (ROWS - g.tokens) * (D / 8); c += STRIPS * 32)
#pragma unroll
    for (int m = 0; m < 8; ++m)
      *reinterpret_cast<uint4*>(mine + m * MAT + (g.tokens + c / (D / 8)) * PITCH + c % (D / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
  float bias[2 * STRIPS][4], dbias[2 * STRIPS][4];
  short_bias<T, STRIPS>(g, st.head, row0, bias);
#pragma unroll
  for (int nb = 0; nb < 2 * STRIPS; ++nb) dbias[nb][0] = dbias[nb][1] = dbias[nb][2] = dbias[nb][3] = 0.f;
  const int64_t row_size = (int64_t)g.heads * D;
  int64_t out_at = ((int64_t)st.first * g.tokens + st.strip * 16) * row_size + st.head * D;
  const int64_t next = (int64_t)st.step * g.tokens * row_size;
  const int rows = g.tokens - st.strip * 16;
  const uint32_t strip_p = ps_at + (st.strip * 16 * PP + frag_a<PP>(st.lane)) * 2, strip_ds = dss_at + (st.strip * 16 * PP + frag_a<PP>(st.lane)) * 2;
  const uint32_t turned = (uint32_t)(((st.lane & 7) + (st.lane >> 4) * 8) * PP + st.strip * 16 + ((st.lane >> 3) & 1) * 8) * 2;
  int stage = 0;
  for (int b = st.first; b < g.batch; b += st.step, stage ^= 1, out_at += next) {
    copy_wait<0>();
    group_sync<STRIPS>(st.group);
    if (b + st.step < g.batch) load(b + st.step, stage ^ 1);
    copy_commit();
    const int len = rel_length(g, b);
    const uint32_t at = base + stage * 4 * MAT * 2;
    uint32_t fa[D / 16][4];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) ldsm4(fa[kk], at + (st.strip * 16 * PITCH + frag_a<PITCH>(st.lane)) * 2 + kk * 32);
    float s[2 * STRIPS][4], dp[2 * STRIPS][4], sum0 = 0.f, sum1 = 0.f;
    short_scores<T, D, STRIPS>(s, bias, fa, at + (MAT + frag_b<PITCH>(st.lane)) * 2, g.causal || len < g.tokens, len, g.causal, row0);
    short_softmax<STRIPS>(s, g.sl2);
#pragma unroll
    for (int n = 0; n < 2 * STRIPS; ++n) { sum0 += s[n][0] + s[n][1]; sum1 += s[n][2] + s[n][3]; }
    sum0 = quad_sum(sum0);
    sum1 = quad_sum(sum1);
    const float inv0 = sum0 != 0.f ? 1.f / sum0 : 0.f, inv1 = sum1 != 0.f ? 1.f / sum1 : 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) ldsm4(fa[kk], at + (3 * MAT + st.strip * 16 * PITCH + frag_a<PITCH>(st.lane)) * 2 + kk * 32);
    float d0 = 0.f, d1 = 0.f;
#pragma unroll
    for (int jj = 0; jj < STRIPS; ++jj) {
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[2 * jj][e] = dp[2 * jj + 1][e] = 0.f;
      rows_product<T, D>(dp[2 * jj], dp[2 * jj + 1], fa, at + (2 * MAT + jj * 16 * PITCH + frag_b<PITCH>(st.lane)) * 2);
#pragma unroll
      for (int n = 2 * jj; n < 2 * jj + 2; ++n) {
        s[n][0] *= inv0; s[n][1] *= inv0; s[n][2] *= inv1; s[n][3] *= inv1;
        d0 += s[n][0] * dp[n][0] + s[n][1] * dp[n][1];
        d1 += s[n][2] * dp[n][2] + s[n][3] * dp[n][3];
      }
    }
    d0 = quad_sum(d0);
    d1 = quad_sum(d1);
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
    for (int jj = 0; jj < STRIPS; ++jj) {
      uint32_t a[4];
      pack_a<T>(a, s[2 * jj], s[2 * jj + 1]);
      stsm4(strip_p + jj * 32, a[0], a[1], a[2], a[3]);
#pragma unroll
      for (int n = 2 * jj; n < 2 * jj + 2; ++n) {
        s[n][0] *= dp[n][0] - d0; s[n][1] *= dp[n][1] - d0;
        s[n][2] *= dp[n][2] - d1; s[n][3] *= dp[n][3] - d1;
#pragma unroll
        for (int e = 0; e < 4; ++e) dbias[n][e] += s[n][e];
      }
      pack_a<T>(a, s[2 * jj], s[2 * jj + 1]);
      stsm4(strip_ds + jj * 32, a[0], a[1], a[2], a[3]);
      cols_product<T, D>(o, a, at + (MAT + jj * 16 * PITCH + frag_a<PITCH>(st.lane)) * 2);
    }
    // rows from the length on have P = dS = 0, as queries and as keys
    store_strip<T, D>(o, g.scale, g.scale, out_strip, static_cast<T*>(g.dq) + out_at, row_size, rows);
    group_sync<STRIPS>(st.group);  // P and dS of all query strips are there
    // this warp's 16 keys: dv = P^T dout, dk = dS^T q, over the query strips
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
    for (int ii = 0; ii < STRIPS; ++ii) {
      uint32_t a[4];
      ldsm4_t(a, ps_at + ii * 16 * PP * 2 + turned);
      cols_product<T, D>(o, a, at + (3 * MAT + ii * 16 * PITCH + frag_a<PITCH>(st.lane)) * 2);
    }
    store_strip<T, D>(o, 1.f, 1.f, out_strip, static_cast<T*>(g.dv) + out_at, row_size, rows);
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
    for (int ii = 0; ii < STRIPS; ++ii) {
      uint32_t a[4];
      ldsm4_t(a, dss_at + ii * 16 * PP * 2 + turned);
      cols_product<T, D>(o, a, at + (ii * 16 * PITCH + frag_a<PITCH>(st.lane)) * 2);
    }
    store_strip<T, D>(o, g.scale, g.scale, out_strip, static_cast<T*>(g.dk) + out_at, row_size, rows);
  }
  // dS summed over this stream's sequences -> diagonals -> buckets
  copy_wait<0>();
  group_sync<STRIPS>(st.group);
  float* full = reinterpret_cast<float*>(raw);        // [ROWS][ROWS + 1]
  float* diag = full + ROWS * (ROWS + 1);             // [2 ROWS - 1]
  static_assert((16 * STRIPS * (16 * STRIPS + 1) + 32 * STRIPS) * 4 <= short_bwd_group<T, D, STRIPS>(), "the sums fit the stages");
#pragma unroll
  for (int n = 0; n < 2 * STRIPS; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) full[(row0 + (e >> 1) * 8) * (ROWS + 1) + n * 8 + 2 * tig + (e & 1)] = dbias[n][e];
  group_sync<STRIPS>(st.group);
  for (int d = thread; d < 2 * ROWS - 1; d += STRIPS * 32) {
    const int off = d - (ROWS - 1);
    float sum = 0.f;
    for (int i = max(0, -off); i < min(ROWS, ROWS - off); ++i) sum += full[i * (ROWS + 1) + i + off];
    diag[d] = sum;
  }
  group_sync<STRIPS>(st.group);
  const int side = ROWS - 1;
  for (int k = thread; k < g.buckets; k += STRIPS * 32) {
    float sum = 0.f;
    const int n0 = min(max(__ldg(g.start + k), 0), 2 * g.reach + 1), n1 = min(__ldg(g.start + k + 1), 2 * g.reach + 1);
    for (int n = n0; n < n1; ++n) {
      const int at = __ldg(g.order + n), off = at - g.reach;
      if (off >= -side && off <= side) sum += diag[off + side];
      // distances past the reach share its ends' buckets
      if (at == 0) for (int o = -side; o < -g.reach; ++o) sum += diag[o + side];
      if (at == 2 * g.reach) for (int o = g.reach + 1; o <= side; ++o) sum += diag[o + side];
    }
    g.partial[(int64_t)st.id * g.buckets + k] = sum;
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Longer sequences: tiles of 64 queries x 64 keys
// ------------------------------------------------------------------------------------------------------------------

constexpr int TILE = 64;
constexpr int REL_RIM = 2 * TILE;
inline int rel_bias_floats(int reach) { return 2 * (reach + REL_RIM) + 1; }
template <int D> __host__ __device__ constexpr int tile_bytes() { return TILE * RelTile<D>::PITCH * 2; }
// 64 rows from `row` on of one head; rows from `len` on become zeros
template <typename T, int D> __device__ __forceinline__ void stage_tile(uint32_t dst, const T* head, int64_t token_stride, int row, int len) {
  constexpr int PITCH = RelTile<D>::PITCH, PARTS = D / 8;
#pragma unroll
  for (int c = threadIdx.x; c < TILE * PARTS; c += REL_THREADS) {
    const int t = c / PARTS, part = c % PARTS;
    const bool in = row + t < len;
    copy16(dst + (t * PITCH + part * 8) * 2, head + (in ? (row + t) * token_stride + part * 8 : 0), in ? 16u : 0u);
  }
}

// Keys of tile j0 against rows of tile i0: 1 = all at least `reach` after, -1 = all at least `reach` before, else 0.
__device__ __forceinline__ int rel_side(int i0, int j0, int reach) {
  return j0 - (i0 + TILE - 1) >= reach ? 1 : i0 - (j0 + TILE - 1) >= reach ? -1 : 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(REL_THREADS) k_rel_tiles(const __grid_constant__ RelArgs g, int tiles) {
  constexpr int PITCH = RelTile<D>::PITCH, MAT = TILE * PITCH;
  extern __shared__ __align__(16) uint8_t rel_smem[];
  T* qs = reinterpret_cast<T*>(rel_smem);
  float* bt = reinterpret_cast<float*>(rel_smem + 5 * tile_bytes<D>());
  Where w = rel_where(blockIdx.x, tiles, g.heads, g.batch);
  w.tile = tiles - 1 - w.tile;  // under a causal mask the longest rows start first
  if (w.b >= rel_batch(g)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int len = rel_length(g, w.b), i0 = w.tile * TILE, row0 = i0 + warp * 16 + gid;
  T* out = static_cast<T*>(g.out) + ((int64_t)w.b * g.tokens * g.heads + w.head) * D;
  T* p0 = row0 < g.tokens ? out + (int64_t)row0 * g.heads * D : nullptr;
  T* p1 = row0 + 8 < g.tokens ? out + (int64_t)(row0 + 8) * g.heads * D : nullptr;
  float2* stats = g.stats ? g.stats + ((int64_t)w.b * g.heads + w.head) * g.tokens : nullptr;
  if (i0 >= len) {
    store_zero_rows<T, D>(p0, p1);
    if (stats && tig == 0) {
      if (p0) stats[row0] = make_float2(0.f, INFINITY);
      if (p1) stats[row0 + 8] = make_float2(0.f, INFINITY);
    }
    return;
  }
  const int head_kv = w.head / (g.heads / g.heads_kv);
  const T* q = static_cast<const T*>(g.q) + w.b * g.qs[0] + w.head * g.qs[2];
  const T* k = static_cast<const T*>(g.k) + w.b * g.ks[0] + head_kv * g.ks[2];
  const T* v = static_cast<const T*>(g.v) + w.b * g.vs[0] + head_kv * g.vs[2];
  const uint32_t q_at = smem_addr(qs), kv_at = q_at + MAT * 2;
  const int last = g.causal ? min(len, i0 + TILE) : len, n_tiles = (last + TILE - 1) / TILE;
  auto load = [&](int t) {
    const uint32_t to = kv_at + (t & 1) * 2 * MAT * 2;
    stage_tile<T, D>(to, k, g.ks[1], t * TILE, len);
    stage_tile<T, D>(to + MAT * 2, v, g.vs[1], t * TILE, len);
  };
  stage_tile<T, D>(q_at, q, g.qs[1], i0, len);
  load(0);
  copy_commit();
  fill_bias<T>(g, w.head, bt, g.reach + REL_RIM, threadIdx.x, REL_THREADS);
  const int side = g.reach + REL_RIM;
  uint32_t qa[D / 16][4];
  float o[D / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  for (int t = 0; t < n_tiles; ++t) {
    copy_wait<0>();
    __syncthreads();
    if (t + 1 < n_tiles) load(t + 1);
    copy_commit();
    if (t == 0) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) ldsm4(qa[kk], q_at + (warp * 16 * PITCH + frag_a<PITCH>(lane)) * 2 + kk * 32);
    }
    const uint32_t at = kv_at + (t & 1) * 2 * MAT * 2;
    const int j0 = t * TILE;
    float s[8][4];
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[2 * jj][e] = s[2 * jj + 1][e] = 0.f;
      rows_product<T, D>(s[2 * jj], s[2 * jj + 1], qa, at + (jj * 16 * PITCH + frag_b<PITCH>(lane)) * 2);
    }
    const int far = rel_side(i0, j0, g.reach);
    if (far) {
      const float c = far > 0 ? bt[2 * side] : bt[0];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e], g.sl2, c);
    } else {
      const float* b0 = bt + j0 + 2 * tig - row0 + side;
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e], g.sl2, b0[n * 8 + (e & 1) - (e >> 1) * 8]);
    }
    if (j0 + TILE > len || (g.causal && j0 + TILE > i0 + 1)) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + n * 8 + 2 * tig + (e & 1), i = row0 + (e >> 1) * 8;
          if (j >= len || (g.causal && j > i)) s[n][e] = -INFINITY;
        }
    }
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      t0 = fmaxf(t0, fmaxf(s[n][0], s[n][1]));
      t1 = fmaxf(t1, fmaxf(s[n][2], s[n][3]));
    }
    t0 = fmaxf(m0, quad_max(t0));
    t1 = fmaxf(m1, quad_max(t1));
    const float u0 = t0 == -INFINITY ? 0.f : t0, u1 = t1 == -INFINITY ? 0.f : t1;  // no key yet: all terms 0
    const float c0 = fast_exp2(m0 - u0), c1 = fast_exp2(m1 - u1);
    m0 = t0;
    m1 = t1;
    l0 *= c0;
    l1 *= c1;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) { o[n][0] *= c0; o[n][1] *= c0; o[n][2] *= c1; o[n][3] *= c1; }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[n][e] = fast_exp2(s[n][e] - u0);
        s[n][2 + e] = fast_exp2(s[n][2 + e] - u1);
        l0 += s[n][e];
        l1 += s[n][2 + e];
      }
    }
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      uint32_t pa[4];
      pack_a<T>(pa, s[2 * jj], s[2 * jj + 1]);
      cols_product<T, D>(o, pa, at + (MAT + jj * 16 * PITCH + frag_a<PITCH>(lane)) * 2);
    }
  }
  l0 = quad_sum(l0);
  l1 = quad_sum(l1);
  const bool in0 = row0 < len && l0 != 0.f, in1 = row0 + 8 < len && l1 != 0.f;
  store_rows<T, D>(o, in0 ? 1.f / l0 : 0.f, in1 ? 1.f / l1 : 0.f, p0, p1);
  if (stats && tig == 0) {
    // apart, because a maximum at the type's lowest value would swallow the sum; a row without keys: P = 0
    if (p0) stats[row0] = in0 ? make_float2(m0, log2f(l0)) : make_float2(0.f, INFINITY);
    if (p1) stats[row0 + 8] = in1 ? make_float2(m1, log2f(l1)) : make_float2(0.f, INFINITY);
  }
}

// dq and delta: a block owns 64 queries and walks over the keys.  Bound by the latency of a warp's chain of products and
// exponentials, with 8 warps on a multiprocessor: 88 us at 6 x 1501 causal padded tokens, 8 heads of 64 over 2 (40 us in
// the tcgen05 form).
template <typename T, int D>
__global__ void __launch_bounds__(REL_THREADS, REL_Q_BLOCKS) k_rel_tiles_dq(const __grid_constant__ RelArgs g, int tiles) {
  constexpr int PITCH = RelTile<D>::PITCH, MAT = TILE * PITCH;
  extern __shared__ __align__(16) uint8_t rel_smem[];
  float* bt = reinterpret_cast<float*>(rel_smem + 6 * tile_bytes<D>());
  const int side = g.reach + REL_RIM;
  Where w = rel_where(blockIdx.x, tiles, g.heads, g.batch);
  w.tile = tiles - 1 - w.tile;  // the longest first
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int len = rel_length(g, w.b), i0 = w.tile * TILE, row0 = i0 + warp * 16 + gid;
  const int64_t head_at = ((int64_t)w.b * g.tokens * g.heads + w.head) * D;
  const int64_t off0 = head_at + (int64_t)row0 * g.heads * D, off1 = off0 + (int64_t)8 * g.heads * D;
  T* p0 = row0 < g.tokens ? static_cast<T*>(g.dq) + off0 : nullptr;
  T* p1 = row0 + 8 < g.tokens ? static_cast<T*>(g.dq) + off1 : nullptr;
  if (i0 >= len) {
    store_zero_rows<T, D>(p0, p1);
    return;  // dk and dv walk over queries below the length only: delta is not read here
  }
  const int head_kv = w.head / (g.heads / g.heads_kv);
  const T* q = static_cast<const T*>(g.q) + w.b * g.qs[0] + w.head * g.qs[2];
  const T* k = static_cast<const T*>(g.k) + w.b * g.ks[0] + head_kv * g.ks[2];
  const T* v = static_cast<const T*>(g.v) + w.b * g.vs[0] + head_kv * g.vs[2];
  const T* dout = static_cast<const T*>(g.dout) + w.b * g.ds[0] + w.head * g.ds[2];
  const uint32_t q_at = smem_addr(rel_smem), do_at = q_at + MAT * 2, kv_at = q_at + 2 * MAT * 2;
  const int last = g.causal ? min(len, i0 + TILE) : len, n_tiles = (last + TILE - 1) / TILE;
  auto load = [&](int t) {
    const uint32_t to = kv_at + (t & 1) * 2 * MAT * 2;
    stage_tile<T, D>(to, k, g.ks[1], t * TILE, len);
    stage_tile<T, D>(to + MAT * 2, v, g.vs[1], t * TILE, len);
  };
  stage_tile<T, D>(q_at, q, g.qs[1], i0, len);
  stage_tile<T, D>(do_at, dout, g.ds[1], i0, len);
  load(0);
  copy_commit();
  fill_bias<T>(g, w.head, bt, g.reach + REL_RIM, threadIdx.x, REL_THREADS);
  const bool in0 = row0 < len, in1 = row0 + 8 < len;
  const float2* stats = g.stats + ((int64_t)w.b * g.heads + w.head) * g.tokens;
  const float2 none = make_float2(0.f, INFINITY), st0 = in0 ? stats[row0] : none, st1 = in1 ? stats[row0 + 8] : none;
  uint32_t qa[D / 16][4], da[D / 16][4];
  float o[D / 8][4], pk[D / 8][4], d0 = 0.f, d1 = 0.f, r0 = 0.f, r1 = 0.f;
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = pk[n][e] = 0.f;
  for (int t = 0; t < n_tiles; ++t) {
    copy_wait<0>();
    __syncthreads();
    if (t + 1 < n_tiles) load(t + 1);
    copy_commit();
    if (t == 0) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        ldsm4(qa[kk], q_at + (warp * 16 * PITCH + frag_a<PITCH>(lane)) * 2 + kk * 32);
        ldsm4(da[kk], do_at + (warp * 16 * PITCH + frag_a<PITCH>(lane)) * 2 + kk * 32);
      }
      // A first delta = dout . out from the 16-bit output.  A row of dS has to sum to 0, so the sum r of the rows made
      // with it is the error of that delta: at the end dq loses r P k, and dk's pass gets delta + r.
      const T* y0 = static_cast<const T*>(g.out) + off0 + 2 * tig;
      const T* y1 = static_cast<const T*>(g.out) + off1 + 2 * tig;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (in0) {
            const float2 a = unpack2<T>(da[kk][2 * half]), b = unpack2<T>(*reinterpret_cast<const uint32_t*>(y0 + kk * 16 + half * 8));
            d0 += a.x * b.x + a.y * b.y;
          }
          if (in1) {
            const float2 a = unpack2<T>(da[kk][2 * half + 1]), b = unpack2<T>(*reinterpret_cast<const uint32_t*>(y1 + kk * 16 + half * 8));
            d1 += a.x * b.x + a.y * b.y;
          }
        }
      d0 = quad_sum(d0);
      d1 = quad_sum(d1);
    }
    const uint32_t at = kv_at + (t & 1) * 2 * MAT * 2;
    const int j0 = t * TILE;
    const int far = rel_side(i0, j0, g.reach);
    const bool edge = j0 + TILE > len || i0 + TILE > len || (g.causal && j0 + TILE > i0 + 1);
    const float fixed = far > 0 ? bt[2 * side] : bt[0];
    const float* b0 = bt + j0 + 2 * tig - row0 + side;
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      float s[2][4], dp[2][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[0][e] = s[1][e] = dp[0][e] = dp[1][e] = 0.f;
      rows_product<T, D>(s[0], s[1], qa, at + (jj * 16 * PITCH + frag_b<PITCH>(lane)) * 2);
      rows_product<T, D>(dp[0], dp[1], da, at + (MAT + jj * 16 * PITCH + frag_b<PITCH>(lane)) * 2);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = (2 * jj + n) * 8 + (e & 1);
          const float bias = far ? fixed : b0[c - (e >> 1) * 8];
          float p = fast_exp2((fmaf(s[n][e], g.sl2, bias) - (e >> 1 ? st1.x : st0.x)) - (e >> 1 ? st1.y : st0.y));
          if (edge) {
            const int j = j0 + c + 2 * tig, i = row0 + (e >> 1) * 8;
            if (j >= len || i >= len || (g.causal && j > i)) p = 0.f;
          }
          s[n][e] = p;
          dp[n][e] = p * (dp[n][e] - (e >> 1 ? d1 : d0));
          if (e >> 1) r1 += dp[n][e]; else r0 += dp[n][e];
        }
      uint32_t a[4], b[4];
      pack_a<T>(a, dp[0], dp[1]);
      pack_a<T>(b, s[0], s[1]);
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t m[4];
        ldsm4_t(m, at + (jj * 16 * PITCH + frag_a<PITCH>(lane)) * 2 + n * 32);
        mma16816<T>(o[2 * n], a, m[0], m[1]);
        mma16816<T>(o[2 * n + 1], a, m[2], m[3]);
        mma16816<T>(pk[2 * n], b, m[0], m[1]);
        mma16816<T>(pk[2 * n + 1], b, m[2], m[3]);
      }
    }
  }
  r0 = quad_sum(r0);
  r1 = quad_sum(r1);
#pragma unroll
  for (int n = 0; n < D / 8; ++n) {
    o[n][0] -= r0 * pk[n][0]; o[n][1] -= r0 * pk[n][1];
    o[n][2] -= r1 * pk[n][2]; o[n][3] -= r1 * pk[n][3];
  }
  store_rows<T, D>(o, in0 ? g.scale : 0.f, in1 ? g.scale : 0.f, p0, p1);
  if (tig == 0) {
    float* delta = g.delta + ((int64_t)w.b * g.heads + w.head) * g.tokens;
    if (in0) delta[row0] = d0 + r0;
    if (in1) delta[row0 + 8] = d1 + r1;
  }
}

// dk, dv and the table's gradient: a block owns 64 keys and walks over queries, in transposed products (keys as rows), so that
// P^T and dS^T come out of the accumulators as operands of the next product.  The query heads that share the keys are spread
// over the `ranks` blocks of a cluster, whose sums are added through distributed shared memory at the end, in a fixed order:
// one block for all heads left most of the device idle (210 us against 119 us at 6 x 1501 causal tokens, 8 heads over 2).
// The table is summed here, from the corrected delta: by diagonals of a tile of dS in shared memory, whole tiles beyond the
// reach in registers.  134 us at 6 x 1501 causal padded tokens, 8 heads of 64 over 2 (77 us in the tcgen05 form).
constexpr int DS_PITCH = TILE + 1;
template <int D> __host__ __device__ constexpr int dkv_front() {  // k and v, whose place a tile of dS takes
  return 2 * tile_bytes<D>() > TILE * DS_PITCH * 4 ? 2 * tile_bytes<D>() : TILE * DS_PITCH * 4;
}
template <typename T, int D>
__global__ void __launch_bounds__(REL_THREADS, REL_KV_BLOCKS) k_rel_tiles_dkv(const __grid_constant__ RelArgs g, int tiles, int ranks) {
  constexpr int PITCH = RelTile<D>::PITCH, MAT = TILE * PITCH;
  extern __shared__ __align__(16) uint8_t rel_smem[];
  __shared__ __align__(16) float2 row_stat[2][TILE];  // a stage's queries: maximum and log2 of the sum
  __shared__ __align__(16) float row_delta[2][TILE];
  __shared__ float far_sum[2][4];
  float* ds = reinterpret_cast<float*>(rel_smem);  // one tile of dS, keys as rows, once k and v are in registers
  float* bt = reinterpret_cast<float*>(rel_smem + dkv_front<D>() + 4 * tile_bytes<D>());
  const int side = g.reach + REL_RIM, span = 2 * side + 1;
  float* dacc = bt + span;                         // dS by offset
  const int rank = (int)(blockIdx.x % ranks);
  const Where w = rel_where(blockIdx.x / ranks, tiles, g.heads_kv, g.batch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int len = rel_length(g, w.b), j0 = w.tile * TILE, row0 = j0 + warp * 16 + gid;
  auto row_of = [&](void* base, int row) { return row < g.tokens ? static_cast<T*>(base) + (((int64_t)w.b * g.tokens + row) * g.heads_kv + w.head) * D : nullptr; };
  const int share = g.heads / g.heads_kv / ranks;  // heads of this block: rank, rank + ranks, ...
  auto head_of = [&](int n) { return (w.head * share + n) * ranks + rank; };
  auto partial_of = [&](int head) { return g.partial + ((int64_t)head * g.batch * tiles + (int64_t)w.b * tiles + w.tile) * g.buckets; };
  if (j0 >= len) {  // the whole cluster
    for (int k = threadIdx.x; k < share * g.buckets; k += REL_THREADS) partial_of(head_of(k / g.buckets))[k % g.buckets] = 0.f;
    if (rank == 0) {
      store_zero_rows<T, D>(row_of(g.dk, row0), row_of(g.dk, row0 + 8));
      store_zero_rows<T, D>(row_of(g.dv, row0), row_of(g.dv, row0 + 8));
    }
    return;
  }
  const uint32_t k_at = smem_addr(rel_smem), v_at = k_at + MAT * 2, qd_at = k_at + dkv_front<D>();
  const int first = g.causal ? w.tile : 0, n_tiles = (len + TILE - 1) / TILE - first, steps = n_tiles * share;
  auto load = [&](int n) {
    const int h = head_of(n / n_tiles), row = (first + n % n_tiles) * TILE;
    const uint32_t to = qd_at + (n & 1) * 2 * MAT * 2;
    stage_tile<T, D>(to, static_cast<const T*>(g.q) + w.b * g.qs[0] + h * g.qs[2], g.qs[1], row, len);
    stage_tile<T, D>(to + MAT * 2, static_cast<const T*>(g.dout) + w.b * g.ds[0] + h * g.ds[2], g.ds[1], row, len);
    if (threadIdx.x < TILE) {  // rows past the length: zeros, and hidden below
      const int i = row + threadIdx.x;
      const int64_t at = ((int64_t)w.b * g.heads + h) * g.tokens + (i < len ? i : 0);
      copy_small<8>(smem_addr(&row_stat[n & 1][threadIdx.x]), g.stats + at, i < len);
      copy_small<4>(smem_addr(&row_delta[n & 1][threadIdx.x]), g.delta + at, i < len);
    }
  };
  stage_tile<T, D>(k_at, static_cast<const T*>(g.k) + w.b * g.ks[0] + w.head * g.ks[2], g.ks[1], j0, len);
  stage_tile<T, D>(v_at, static_cast<const T*>(g.v) + w.b * g.vs[0] + w.head * g.vs[2], g.vs[1], j0, len);
  load(0);
  copy_commit();
  uint32_t ka[D / 16][4], va[D / 16][4];
  float ok[D / 8][4], ov[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) ok[n][e] = ov[n][e] = 0.f;
  float before = 0.f, after = 0.f;  // sums of dS in tiles beyond the reach
  // The table's partial sums of one query head, from what its tiles have left by offset.
  auto finish_table = [&](int head) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, m);
      after += __shfl_xor_sync(0xffffffffu, after, m);
    }
    if (lane == 0) { far_sum[0][warp] = before; far_sum[1][warp] = after; }
    before = after = 0.f;
    __syncthreads();
    // offsets past the reach join its ends
    if (warp < 2) {
      float sum = 0.f;
      for (int i = lane; i < REL_RIM; i += 32) sum += warp ? dacc[span - 1 - i] : dacc[i];
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      if (lane == 0) dacc[warp ? span - 1 - REL_RIM : REL_RIM] += sum + (far_sum[warp][0] + far_sum[warp][1]) + (far_sum[warp][2] + far_sum[warp][3]);
    }
    __syncthreads();
    float* partial = partial_of(head);
    for (int b = threadIdx.x; b < g.buckets; b += REL_THREADS) {
      float sum = 0.f;
      const int n0 = min(max(__ldg(g.start + b), 0), 2 * g.reach + 1), n1 = min(__ldg(g.start + b + 1), 2 * g.reach + 1);
      for (int n = n0; n < n1; ++n) sum += dacc[min(max(__ldg(g.order + n), 0), 2 * g.reach) + REL_RIM];
      partial[b] = sum;
    }
  };
  for (int n = 0; n < steps; ++n) {
    const int i0 = (first + n % n_tiles) * TILE;
    if (n % n_tiles == 0) {
      __syncthreads();  // the head before has read its biases and sums
      fill_bias<T>(g, head_of(n / n_tiles), bt, side, threadIdx.x, REL_THREADS);
      for (int i = threadIdx.x; i < span; i += REL_THREADS) dacc[i] = 0.f;
    }
    copy_wait<0>();
    __syncthreads();
    if (n + 1 < steps) load(n + 1);
    copy_commit();
    if (n == 0) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        ldsm4(ka[kk], k_at + (warp * 16 * PITCH + frag_a<PITCH>(lane)) * 2 + kk * 32);
        ldsm4(va[kk], v_at + (warp * 16 * PITCH + frag_a<PITCH>(lane)) * 2 + kk * 32);
      }
      __syncthreads();  // k and v make room
    }
    const uint32_t at = qd_at + (n & 1) * 2 * MAT * 2;
    const int far = rel_side(i0, j0, g.reach);
    const float fixed = far > 0 ? bt[2 * side] : bt[0];
    const float* b0 = bt + row0 - i0 - 2 * tig + side;  // offset of key row0 from query i0 + 2 tig
    const bool edge = i0 + TILE > len || j0 + TILE > len || (g.causal && j0 + TILE > i0 + 1);
    float tile_sum = 0.f;
#pragma unroll
    for (int ii = 0; ii < 4; ++ii) {  // 16 queries each
      float s[2][4], dp[2][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[0][e] = s[1][e] = dp[0][e] = dp[1][e] = 0.f;
      rows_product<T, D>(s[0], s[1], ka, at + (ii * 16 * PITCH + frag_b<PITCH>(lane)) * 2);
      rows_product<T, D>(dp[0], dp[1], va, at + (MAT + ii * 16 * PITCH + frag_b<PITCH>(lane)) * 2);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float4 st = *reinterpret_cast<const float4*>(&row_stat[n & 1][(2 * ii + m) * 8 + 2 * tig]);
        const float2 dl = *reinterpret_cast<const float2*>(&row_delta[n & 1][(2 * ii + m) * 8 + 2 * tig]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = (2 * ii + m) * 8 + (e & 1);
          const float bias = far ? fixed : b0[(e >> 1) * 8 - c];
          float p = fast_exp2((fmaf(s[m][e], g.sl2, bias) - (e & 1 ? st.z : st.x)) - (e & 1 ? st.w : st.y));
          if (edge) {
            const int i = i0 + c + 2 * tig, j = row0 + (e >> 1) * 8;
            if (i >= len || j >= len || (g.causal && j > i)) p = 0.f;
          }
          s[m][e] = p;
          dp[m][e] = p * (dp[m][e] - (e & 1 ? dl.y : dl.x));
          tile_sum += dp[m][e];
          if (!far) ds[(warp * 16 + gid + (e >> 1) * 8) * DS_PITCH + c + 2 * tig] = dp[m][e];
        }
      }
      uint32_t a[4];
      pack_a<T>(a, s[0], s[1]);
      cols_product<T, D>(ov, a, at + (MAT + ii * 16 * PITCH + frag_a<PITCH>(lane)) * 2);
      pack_a<T>(a, dp[0], dp[1]);
      cols_product<T, D>(ok, a, at + (ii * 16 * PITCH + frag_a<PITCH>(lane)) * 2);
    }
    if (far > 0) after += tile_sum;
    else if (far < 0) before += tile_sum;
    else {
      __syncthreads();
      const int off = (int)threadIdx.x - (TILE - 1);  // key minus query of this thread's diagonal, within the tile
      if (off < TILE) {
        float sum = 0.f;
        for (int i = max(0, -off); i < min(TILE, TILE - off); ++i) sum += ds[(i + off) * DS_PITCH + i];
        dacc[j0 - i0 + off + side] += sum;
      }
      // the next tile's sums come after two barriers, its scores after one
    }
    if (n % n_tiles == n_tiles - 1) {
      __syncthreads();
      finish_table(head_of(n / n_tiles));
    }
  }
  const float in0 = row0 < len ? 1.f : 0.f, in1 = row0 + 8 < len ? 1.f : 0.f;
  if (ranks == 1) {
    store_rows<T, D>(ov, in0, in1, row_of(g.dv, row0), row_of(g.dv, row0 + 8));
    store_rows<T, D>(ok, in0 * g.scale, in1 * g.scale, row_of(g.dk, row0), row_of(g.dk, row0 + 8));
    return;
  }
  constexpr int SP = D + 4;
  float* sums = reinterpret_cast<float*>(rel_smem);  // [dv, dk][TILE][SP]
  static_assert(2 * TILE * SP * 4 <= dkv_front<D>() + 4 * tile_bytes<D>(), "the sums fit the stages");
  __syncthreads();
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = (warp * 16 + gid + (e >> 1) * 8) * SP + n * 8 + 2 * tig + (e & 1);
      sums[at] = ov[n][e];
      sums[TILE * SP + at] = ok[n][e];
    }
  rel_cluster_sync();
  for (int c = rank * REL_THREADS + threadIdx.x; c < 2 * TILE * (D / 8); c += ranks * REL_THREADS) {
    const int which = c / (TILE * (D / 8)), row = c / (D / 8) % TILE, part = c % (D / 8) * 8;
    if (j0 + row >= g.tokens) continue;
    const float* from = sums + (which * TILE + row) * SP + part;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < ranks; ++r) {
      const float4 a = get_remote(from, r), b = get_remote(from + 4, r);
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
    const float f = j0 + row < len ? (which ? g.scale : 1.f) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= f;
    *reinterpret_cast<uint4*>(row_of(which ? g.dk : g.dv, j0 + row) + part) = Vec16<T>::down(v);
  }
  rel_cluster_sync();  // a block's sums stay until all have been read
}

// ------------------------------------------------------------------------------------------------------------------
// Sums of the table's gradient
// ------------------------------------------------------------------------------------------------------------------

// Block (h, c): rows c * chunk .. of head h, row i at (h * head_step + i * row_step) * buckets.  O float: sums to
// out[(h * gridDim.y + c) * buckets + b]; else the table's type, to out[b * heads + h] (one chunk).
template <typename O>
__global__ void __launch_bounds__(256) k_rel_table_sum(const float* __restrict__ in, int64_t rows, int64_t chunk, int64_t head_step,
                                                       int64_t row_step, int buckets, O* __restrict__ out, bool final) {
  __shared__ float part[256];
  const int h = blockIdx.x;
  const int64_t r0 = blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
  for (int base = 0; base < buckets; base += 256) {
    const int width = min(256, buckets - base), groups = 256 / width;
    const int b = threadIdx.x % width, group = threadIdx.x / width;
    float sum = 0.f;
    if (group < groups)
      for (int64_t r = r0 + group; r < r1; r += groups) sum += in[(h * head_step + r * row_step) * buckets + base + b];
    part[threadIdx.x] = sum;
    __syncthreads();
    if (group == 0) {
      for (int i = 1; i < groups; ++i) sum += part[i * width + b];
      if (final) out[(int64_t)(base + b) * gridDim.x + h] = Elem<O>::down(sum);
      else out[((int64_t)h * gridDim.y + blockIdx.y) * buckets + base + b] = Elem<O>::down(sum);
    }
    __syncthreads();
  }
}

namespace {

constexpr int REL_SHORT = 64;
constexpr int REL_CHUNKS = 32;

int short_strips(int tokens) { return (tokens + 15) / 16; }

// Blocks of the short kernels: as many as the device holds at a time (`per_sm`), at least one stream per head, and
// no more than sequences x heads need.
int short_blocks(int64_t batch, int heads, int groups, int per_sm) {
  int64_t streams = (int64_t)device_sms() * per_sm * groups;
  if (streams < heads) streams = heads;
  if (streams > batch * heads) streams = batch * heads;
  return (int)((streams + groups - 1) / groups);
}

bool short_backward(const MgbsRelAttentionArgs* a) { return a->tokens <= REL_SHORT && a->heads == a->heads_kv; }

template <typename K> int resident(K kernel, int threads, int smem) {
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) n = 1;
  return n;
}

template <typename T, int D, int STRIPS> int run_short(const RelArgs& g, cudaStream_t st) {
  constexpr int smem = short_fwd_smem<T, D, STRIPS>();
  static std::atomic<uint64_t> raised{0};
  static std::atomic<int> per_sm{0};
  const int rc = raise_smem(k_rel_short<T, D, STRIPS>, smem, raised);
  if (rc) return rc;
  int n = per_sm.load(std::memory_order_relaxed);
  if (!n) per_sm.store(n = resident(k_rel_short<T, D, STRIPS>, Groups<STRIPS>::THREADS, smem), std::memory_order_relaxed);
  k_rel_short<T, D, STRIPS><<<short_blocks(g.batch, g.heads, Groups<STRIPS>::N, n), Groups<STRIPS>::THREADS, smem, st>>>(g);
  return (int)cudaGetLastError();
}

template <typename T> int finish_table(const RelArgs& g, const float* in, int64_t rows, int64_t head_step, int64_t row_step, void* dtable, cudaStream_t st) {
  k_rel_table_sum<T><<<dim3(g.heads, 1), 256, 0, st>>>(in, rows, rows, head_step, row_step, g.buckets, static_cast<T*>(dtable), true);
  return (int)cudaGetLastError();
}

// Streams of the short backward: bounded independently of the device, because the workspace holds a row for each.
constexpr int REL_BWD_STREAMS = 4096;
template <typename T, int D, int STRIPS> int run_short_bwd(const RelArgs& g, void* dtable, cudaStream_t st) {
  constexpr int smem = Groups<STRIPS>::N * short_bwd_group<T, D, STRIPS>();
  static std::atomic<uint64_t> raised{0};
  static std::atomic<int> per_sm{0};
  const int rc = raise_smem(k_rel_short_bwd<T, D, STRIPS>, smem, raised);
  if (rc) return rc;
  int n = per_sm.load(std::memory_order_relaxed);
  if (!n) per_sm.store(n = resident(k_rel_short_bwd<T, D, STRIPS>, Groups<STRIPS>::THREADS, smem), std::memory_order_relaxed);
  int blocks = short_blocks(g.batch, g.heads, Groups<STRIPS>::N, n);
  const int most = REL_BWD_STREAMS / Groups<STRIPS>::N;
  if (blocks > most) blocks = most;
  const int step = blocks * Groups<STRIPS>::N / g.heads;
  if (step < 1) return MGBS_ERR_TOO_LARGE;
  k_rel_short_bwd<T, D, STRIPS><<<blocks, Groups<STRIPS>::THREADS, smem, st>>>(g);
  const int e = (int)cudaGetLastError();
  return e ? e : finish_table<T>(g, g.partial, step, 1, g.heads, dtable, st);
}

template <typename T, int D> int run_tiles(const RelArgs& g, cudaStream_t st) {
  static std::atomic<uint64_t> raised{0};
  const int most = 5 * tile_bytes<D>() + rel_bias_floats(1024) * 4;
  const int rc = raise_smem(k_rel_tiles<T, D>, most, raised);
  if (rc) return rc;
  const int tiles = (g.tokens + TILE - 1) / TILE;
  const int64_t blocks = (int64_t)tiles * g.heads * g.batch;
  if (blocks > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  k_rel_tiles<T, D><<<(unsigned)blocks, REL_THREADS, 5 * tile_bytes<D>() + rel_bias_floats(g.reach) * 4, st>>>(g, tiles);
  return (int)cudaGetLastError();
}

template <typename T, int D> int run_tiles_bwd(const RelArgs& g, cudaStream_t st) {
  static std::atomic<uint64_t> raised_q{0}, raised_kv{0};
  const int fixed_q = 6 * tile_bytes<D>(), fixed_kv = dkv_front<D>() + 4 * tile_bytes<D>();
  int rc = raise_smem(k_rel_tiles_dq<T, D>, fixed_q + rel_bias_floats(1024) * 4, raised_q);
  if (!rc) rc = raise_smem(k_rel_tiles_dkv<T, D>, fixed_kv + 2 * rel_bias_floats(1024) * 4, raised_kv);
  if (rc) return rc;
  const int tiles = (g.tokens + TILE - 1) / TILE;
  const int64_t rows = (int64_t)g.batch * tiles, blocks = rows * g.heads;
  if (blocks > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  k_rel_tiles_dq<T, D><<<(unsigned)blocks, REL_THREADS, fixed_q + rel_bias_floats(g.reach) * 4, st>>>(g, tiles);
  rc = (int)cudaGetLastError();
  if (rc) return rc;
  const int ranks = rel_ranks(g);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * g.heads_kv * ranks));
  cfg.blockDim = dim3(REL_THREADS);
  cfg.dynamicSmemBytes = fixed_kv + 2 * rel_bias_floats(g.reach) * 4;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, k_rel_tiles_dkv<T, D>, g, tiles, ranks);
}

// The table's gradient from a row of sums per head, sequence and tile of keys.
template <typename T> int sum_table(const RelArgs& g, int tile, void* dtable, float* sums, cudaStream_t st) {
  const int64_t rows = (int64_t)g.batch * ((g.tokens + tile - 1) / tile);
  if (rows <= 256) return finish_table<T>(g, g.partial, rows, rows, 1, dtable, st);
  const int64_t chunk = (rows + REL_CHUNKS - 1) / REL_CHUNKS;
  k_rel_table_sum<float><<<dim3(g.heads, REL_CHUNKS), 256, 0, st>>>(g.partial, rows, chunk, rows, 1, g.buckets, sums, false);
  const int rc = (int)cudaGetLastError();
  return rc ? rc : finish_table<T>(g, sums, REL_CHUNKS, REL_CHUNKS, 1, dtable, st);
}

// Sequences from here on go forward on tcgen05: 442368 tokens, 8 heads, in sequences of T
//   heads of 64:  T = 65: 1419 us against 1580 us, 256: 868 against 1267, 512: 1158 against 2220
//   heads of 32:  T = 65: 1355 against 947, 256: 785 against 712, 384: 932 against 972, 512: 1056 against 1233 (half the
//                 products per exponential, so that a block's fixed costs weigh more)
// The rule asks for the number of tokens alone, while tiles are padded to 128 rows on one side and 64 on the other: just
// past a tile's end the other form is ahead by a little, 2 % at 129 tokens (64) and at 448 (32).
template <int D> constexpr int rel_tc_tokens() { return D == 64 ? 65 : 321; }
// The backward is on tcgen05 from 65 tokens on for every head size: 221184 tokens, 8 heads of 64 in sequences of T = 65:
// 1776 us against 3447 us, 129: 2250 against 3418, 192: 1526 against 2182, 1000: 3397 against 8488; heads of 32: 65: 1569
// against 2604, 129: 1998 against 2539, 192: 1343 against 1522.  Below, where only shared key heads come here, the other
// form is ahead: 33 tokens, 8 heads of 64 over 2: 3216 against 2963, 64 tokens: 1836 against 1661.
constexpr int REL_TC_BACKWARD_TOKENS = 65;
template <typename T> struct Type;
template <> struct Type<__nv_bfloat16> { static constexpr int DT = MGBS_DT_BF16; };
template <> struct Type<__half> { static constexpr int DT = MGBS_DT_F16; };
template <typename T, int D> int forward_as(const RelArgs& g, cudaStream_t st) {
  // with statistics asked for, the form whose backward reads them
  if (g.tokens > REL_SHORT || (g.stats && g.heads != g.heads_kv)) {
    if (g.tokens >= rel_tc_tokens<D>() && rel_attention_tc_fits(g)) return rel_attention_tc(g, Type<T>::DT, D, st);
    return run_tiles<T, D>(g, st);
  }
  const int strips = short_strips(g.tokens);
  return strips == 1 ? run_short<T, D, 1>(g, st) : strips == 2 ? run_short<T, D, 2>(g, st) : strips == 3 ? run_short<T, D, 3>(g, st) : run_short<T, D, 4>(g, st);
}
template <typename T, int D> int backward_as(const RelArgs& g, bool is_short, void* dtable, float* sums, cudaStream_t st) {
  if (!is_short) {
    const bool tc = g.tokens >= REL_TC_BACKWARD_TOKENS && rel_attention_tc_backward_fits(g);
    const int rc = tc ? rel_attention_tc_backward(g, Type<T>::DT, D, st) : run_tiles_bwd<T, D>(g, st);
    return rc ? rc : sum_table<T>(g, tc ? REL_TC_ROWS : TILE, dtable, sums, st);
  }
  const int strips = short_strips(g.tokens);
  return strips == 1 ? run_short_bwd<T, D, 1>(g, dtable, st) : strips == 2 ? run_short_bwd<T, D, 2>(g, dtable, st)
         : strips == 3 ? run_short_bwd<T, D, 3>(g, dtable, st) : run_short_bwd<T, D, 4>(g, dtable, st);
}

bool fits16(const void* p, const int64_t (&s)[3]) {
  return !(reinterpret_cast<uintptr_t>(p) & 15) && !(s[0] % 8) && !(s[1] % 8) && !(s[2] % 8);
}

int rel_shape(const MgbsRelAttentionArgs* a) {
  if (!a) return MGBS_ERR_ARG;
  if ((a->dtype != MGBS_DT_BF16 && a->dtype != MGBS_DT_F16) || (a->head_dim != 32 && a->head_dim != 64)) return MGBS_ERR_UNSUPPORTED;
  if (a->heads < 1 || a->heads_kv < 1 || a->heads % a->heads_kv || a->batch < 0 || a->tokens < 0) return MGBS_ERR_ARG;
  if (a->heads > 1024 || a->tokens > (1 << 20) || a->batch > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  if (a->num_buckets < 1 || a->num_buckets > 512 || a->max_distance < 1 || a->max_distance > 1024) return MGBS_ERR_ARG;
  if (!(a->scale > 0.f) || isinf(a->scale)) return MGBS_ERR_ARG;
  return 0;
}

int rel_prepare(const MgbsRelAttentionArgs* a, RelArgs* g) {
  const int rc = rel_shape(a);
  if (rc) return rc;
  if (!a->table || !a->bucket_map || !a->bucket_order || !a->bucket_start) return MGBS_ERR_ARG;
  *g = RelArgs();
  if (a->batch > 0 && a->tokens > 0) {
    if (!a->q || !a->k || !a->v || !a->out) return MGBS_ERR_ARG;
    if (!fits16(a->q, a->q_stride) || !fits16(a->k, a->k_stride) || !fits16(a->v, a->v_stride) || ((reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(a->stats)) & 15))
      return MGBS_ERR_UNSUPPORTED;
  }
  g->q = a->q; g->k = a->k; g->v = a->v; g->table = a->table; g->out = a->out; g->stats = reinterpret_cast<float2*>(a->stats);
  g->map = a->bucket_map; g->order = a->bucket_order; g->start = a->bucket_start; g->lengths = a->lengths;
  for (int i = 0; i < 3; ++i) { g->qs[i] = a->q_stride[i]; g->ks[i] = a->k_stride[i]; g->vs[i] = a->v_stride[i]; }
  g->batch = (int32_t)a->batch; g->tokens = (int32_t)a->tokens; g->heads = a->heads; g->heads_kv = a->heads_kv;
  g->buckets = a->num_buckets; g->reach = a->max_distance; g->causal = a->causal != 0;
  g->error = a->error;
  g->scale = a->scale;
  g->sl2 = a->scale * kLog2e;
  return 0;
}

struct RelWork { int64_t delta, partial, sums, total; };  // byte offsets
RelWork rel_work(const MgbsRelAttentionArgs* a) {
  RelWork w{};
  auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
  if (short_backward(a)) {
    w.total = up((int64_t)REL_BWD_STREAMS * a->num_buckets * 4);
    return w;
  }
  const int64_t tiles = (a->tokens + TILE - 1) / TILE;
  w.partial = up(a->batch * a->heads * a->tokens * 4);
  w.sums = w.partial + up(a->batch * a->heads * tiles * a->num_buckets * 4);
  w.total = w.sums + up((int64_t)a->heads * REL_CHUNKS * a->num_buckets * 4);
  return w;
}

}  // namespace

int rel_attention_counted(const MgbsRelAttentionArgs* a, const uint32_t* count_dev, int64_t count_offset, void* stream) {
  RelArgs g;
  const int rc = rel_prepare(a, &g);
  if (rc) return rc;
  if (a->batch == 0 || a->tokens == 0) return 0;
  g.count_dev = count_dev;
  g.count_offset = count_offset;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == MGBS_DT_BF16) return a->head_dim == 32 ? forward_as<__nv_bfloat16, 32>(g, st) : forward_as<__nv_bfloat16, 64>(g, st);
  return a->head_dim == 32 ? forward_as<__half, 32>(g, st) : forward_as<__half, 64>(g, st);
}

}  // namespace mgbs

extern "C" {

int mgbs_sizeof_rel_attention_args(void) { return (int)sizeof(MgbsRelAttentionArgs); }

int mgbs_rel_attention(const MgbsRelAttentionArgs* a, void* stream) { return mgbs::rel_attention_counted(a, nullptr, 0, stream); }

int64_t mgbs_rel_attention_backward_workspace(const MgbsRelAttentionArgs* a) { return mgbs::rel_shape(a) ? 0 : mgbs::rel_work(a).total; }

int mgbs_rel_attention_backward(const MgbsRelAttentionArgs* a, void* stream) {
  using namespace mgbs;
  RelArgs g;
  const int rc = rel_prepare(a, &g);
  if (rc) return rc;
  if (!a->dtable) return MGBS_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->batch == 0 || a->tokens == 0) return (int)cudaMemsetAsync(a->dtable, 0, (size_t)a->num_buckets * a->heads * 2, st);
  if (!a->dout || !a->dq || !a->dk || !a->dv || !a->workspace) return MGBS_ERR_ARG;
  if (!fits16(a->dout, a->dout_stride) || ((reinterpret_cast<uintptr_t>(a->dq) | reinterpret_cast<uintptr_t>(a->dk) | reinterpret_cast<uintptr_t>(a->dv) |
                                             reinterpret_cast<uintptr_t>(a->workspace)) & 15))
    return MGBS_ERR_UNSUPPORTED;
  const bool is_short = short_backward(a);
  if (!is_short && !a->stats) return MGBS_ERR_ARG;
  const RelWork w = rel_work(a);
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  g.dout = a->dout; g.dq = a->dq; g.dk = a->dk; g.dv = a->dv;
  for (int i = 0; i < 3; ++i) g.ds[i] = a->dout_stride[i];
  g.delta = reinterpret_cast<float*>(ws + w.delta);
  g.partial = reinterpret_cast<float*>(ws + w.partial);
  float* sums = reinterpret_cast<float*>(ws + w.sums);
  if (a->dtype == MGBS_DT_BF16)
    return a->head_dim == 32 ? backward_as<__nv_bfloat16, 32>(g, is_short, a->dtable, sums, st) : backward_as<__nv_bfloat16, 64>(g, is_short, a->dtable, sums, st);
  return a->head_dim == 32 ? backward_as<__half, 32>(g, is_short, a->dtable, sums, st) : backward_as<__half, 64>(g, is_short, a->dtable, sums, st);
}

}  // extern "C"
