// RMS norm of every query and key head with a learned gain, and the rotation by position, in one pass:
//   n = x / sqrt(mean(x^2) + eps),  y_i = R(position) (g n)_i,
// where R turns the pair (a, b) = (y_i, y_i+D/2) or (y_2i, y_2i+1) by the angle position * freq_i.
// Backward, with u = R^T dy:  dgain = sum u n,  w = g u,  dx = (w - n mean(w n)) / sqrt(mean(x^2) + eps).
//
// What bounds it: bytes (x read, y written; backward x, dy read, dx written).  A group of lanes owns one head vector,
// each lane eight pairs, so that both members of a pair are in one lane, loads and stores are 16 bytes wide and the
// only exchange is the sum of squares.  Sines and cosines are shared by all heads of a token: the block computes them
// once per token into shared memory while the loads of the vectors are in flight.
//
// Angles: position * freq / (2 pi) is taken modulo one turn as a 64-bit integer product (freq comes as 2^64 times
// its turns per position), exact for any 64-bit position: no table, no range limit, no loss at far positions.

#include <math.h>

#include "mgbs_counted.cuh"
#include "mgbs_operators.cuh"

namespace mgbs {

struct QkTensor {
  const void* x;
  void* y;         // forward: output; backward: dx
  const void* dy;  // backward
  const float* gain;
  int64_t xs[3], ys[3], ds[3];  // strides of x, y (dx) and dy in elements: batch, token, head
  int32_t heads;
  int32_t flat;  // every tensor's batch stride is tokens * token stride
};
struct QkArgs {
  QkTensor t[2];  // queries, keys
  const uint64_t* phase;
  const void* positions;
  int64_t pos_sb, pos_st;
  const uint32_t* count_dev;  // optional: batch entries to do (device value), from count_offset on
  int64_t count_offset;
  int32_t pos_bits;  // 0 = token index, 32 or 64 = element size of positions
  int32_t batch, tokens, head_dim, lanes;  // lanes: per head vector, a power of two
  int32_t tile;                            // tokens per block iteration
  float eps;
  float* partial;  // backward: [2][gridDim.x][head_dim] sums of the gain gradients
};

constexpr int QK_THREADS = 256;
constexpr int QK_ITEMS = 2;  // vectors parts in flight per thread

// The 16 elements of a lane (8 pairs): a[i], b[i].
template <typename T, bool INTER, bool VEC> struct PairIo {
  static constexpr int R = (int)sizeof(T);  // 16-byte registers of a lane: 16 * sizeof(T) / 16
  uint4 raw[R];
  __device__ __forceinline__ void load(const T* p, int chunk, int half) {
    if (VEC) {
      const uint4* lo = reinterpret_cast<const uint4*>(p + (INTER ? 16 * chunk : 8 * chunk));
      const uint4* hi = INTER ? lo + R / 2 : reinterpret_cast<const uint4*>(p + half + 8 * chunk);
#pragma unroll
      for (int i = 0; i < R / 2; ++i) { raw[i] = lo[i]; raw[R / 2 + i] = hi[i]; }
    } else {
      T* e = reinterpret_cast<T*>(raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = 8 * chunk + i;
        const bool in = c < half;
        e[INTER ? 2 * i : i] = in ? p[INTER ? 2 * c : c] : Elem<T>::down(0.f);
        e[INTER ? 2 * i + 1 : 8 + i] = in ? p[INTER ? 2 * c + 1 : half + c] : Elem<T>::down(0.f);
      }
    }
  }
  __device__ __forceinline__ void get(float (&a)[8], float (&b)[8]) const {
    float v[16];
#pragma unroll
    for (int i = 0; i < R; ++i) Vec16<T>::up(raw[i], v + i * Vec16<T>::N);
#pragma unroll
    for (int i = 0; i < 8; ++i) { a[i] = v[INTER ? 2 * i : i]; b[i] = v[INTER ? 2 * i + 1 : 8 + i]; }
  }
  static __device__ __forceinline__ void store(T* p, int chunk, int half, const float (&a)[8], const float (&b)[8]) {
    if (VEC) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) { v[INTER ? 2 * i : i] = a[i]; v[INTER ? 2 * i + 1 : 8 + i] = b[i]; }
      uint4* lo = reinterpret_cast<uint4*>(p + (INTER ? 16 * chunk : 8 * chunk));
      uint4* hi = INTER ? lo + R / 2 : reinterpret_cast<uint4*>(p + half + 8 * chunk);
#pragma unroll
      for (int i = 0; i < R / 2; ++i) {
        lo[i] = Vec16<T>::down(v + i * Vec16<T>::N);
        hi[i] = Vec16<T>::down(v + 8 + i * Vec16<T>::N);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = 8 * chunk + i;
        if (c < half) {
          p[INTER ? 2 * c : c] = Elem<T>::down(a[i]);
          p[INTER ? 2 * c + 1 : half + c] = Elem<T>::down(b[i]);
        }
      }
    }
  }
};

__device__ __forceinline__ int64_t qk_batch(const QkArgs& g) {
  if (!g.count_dev) return g.batch;
  const int64_t left = (int64_t)*g.count_dev - g.count_offset;
  return left < 0 ? 0 : (left < g.batch ? left : g.batch);
}

// (cos, sin) of the tile's tokens: cs[token][pair].
__device__ __forceinline__ void qk_angles(const QkArgs& g, uint32_t first, uint32_t count, float2* cs) {
  const uint32_t half = g.head_dim / 2;
  for (uint32_t i = threadIdx.x; i < count * half; i += QK_THREADS) {
    const uint32_t tok = i / half, pair = i - tok * half;
    const uint32_t n = first + tok, b = n / (uint32_t)g.tokens, t = n - b * (uint32_t)g.tokens;
    const int64_t at = (int64_t)b * g.pos_sb + (int64_t)t * g.pos_st;
    const int64_t pos = g.pos_bits == 64 ? static_cast<const int64_t*>(g.positions)[at]
                        : g.pos_bits == 32 ? (int64_t) static_cast<const int32_t*>(g.positions)[at] : (int64_t)t;
    const uint64_t turns = (uint64_t)pos * g.phase[pair];  // modulo one turn = 2^64
    float s, c;
    sincospif((float)(int32_t)(turns >> 32) * 4.656612873077393e-10f, &s, &c);  // 2^-31: signed half turns
    cs[i] = make_float2(c, s);
  }
}

__device__ __forceinline__ const float4* qk_cs(const float2* cs, uint32_t tok, int half, int chunk) {
  return reinterpret_cast<const float4*>(cs + tok * half + chunk * 8);
}

// Rotation coefficients of a lane's eight pairs; pairs past `half` read nothing.
template <bool VEC> __device__ __forceinline__ void qk_read_cs(const float2* cs, uint32_t tok, int half, int chunk, float (&c)[8], float (&s)[8]) {
  if (VEC) {
    const float4* p = qk_cs(cs, tok, half, chunk);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float4 f = p[i]; c[2 * i] = f.x; s[2 * i] = f.y; c[2 * i + 1] = f.z; s[2 * i + 1] = f.w; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = 8 * chunk + i < half;
      const float2 f = in ? cs[tok * half + chunk * 8 + i] : make_float2(0.f, 0.f);
      c[i] = f.x; s[i] = f.y;
    }
  }
}

template <bool INTER> __device__ __forceinline__ void qk_gains(const float* gain, int chunk, int half, float (&ga)[8], float (&gb)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = 8 * chunk + i;
    ga[i] = c < half ? __ldg(gain + (INTER ? 2 * c : c)) : 0.f;
    gb[i] = c < half ? __ldg(gain + (INTER ? 2 * c + 1 : half + c)) : 0.f;
  }
}

__device__ __forceinline__ int64_t qk_offset(const QkArgs& g, int flat, const int64_t (&s)[3], uint32_t n, int head) {
  if (flat) return (int64_t)n * s[1] + head * s[2];
  const uint32_t b = n / (uint32_t)g.tokens;
  return (int64_t)b * s[0] + (int64_t)(n - b * (uint32_t)g.tokens) * s[1] + head * s[2];
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Queries and keys of a token are one run of heads, so both share the token's angles.
template <typename T, bool INTER, bool VEC>
__global__ void __launch_bounds__(QK_THREADS) k_qk_norm_rope(const __grid_constant__ QkArgs g) {
  extern __shared__ __align__(16) float2 cs[];
  const uint32_t total = (uint32_t)(qk_batch(g) * g.tokens);
  const int half = g.head_dim / 2, lanes = g.lanes;
  const int chunk = threadIdx.x & (lanes - 1);
  const bool busy = chunk * 8 < half;
  const uint32_t row = (uint32_t)(g.t[0].heads + g.t[1].heads) * lanes;  // lanes of one token
  const float inv_d = 1.f / (float)g.head_dim;
  for (uint64_t first = (uint64_t)blockIdx.x * g.tile; first < total; first += (uint64_t)gridDim.x * g.tile) {
    const uint32_t count = min((uint32_t)g.tile, total - (uint32_t)first);
    const uint32_t items = count * row;
    for (uint32_t base = 0; base < items; base += QK_THREADS * QK_ITEMS) {
      PairIo<T, INTER, VEC> io[QK_ITEMS];
      uint32_t tok[QK_ITEMS];
      int head[QK_ITEMS];
#pragma unroll
      for (int u = 0; u < QK_ITEMS; ++u) {
        const uint32_t i = base + u * QK_THREADS + threadIdx.x;
        tok[u] = i / row;
        head[u] = (int)((i - tok[u] * row) / lanes);
        const int which = head[u] >= g.t[0].heads;
        head[u] = i < items && busy ? head[u] : -1;
        if (head[u] >= 0) {
          const QkTensor& t = g.t[which];
          io[u].load(static_cast<const T*>(t.x) + qk_offset(g, t.flat, t.xs, (uint32_t)first + tok[u], head[u] - (which ? g.t[0].heads : 0)), chunk, half);
        } else {
#pragma unroll
          for (int r = 0; r < PairIo<T, INTER, VEC>::R; ++r) io[u].raw[r] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      if (base == 0) {
        __syncthreads();  // the tile before has been read
        qk_angles(g, (uint32_t)first, count, cs);
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < QK_ITEMS; ++u) {
        float a[8], b[8], ss = 0.f;
        io[u].get(a, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
        ss = group_sum(ss, lanes);
        if (head[u] < 0) continue;
        const float r = rsqrtf(ss * inv_d + g.eps);
        const int which = head[u] >= g.t[0].heads;
        const QkTensor& t = g.t[which];
        float ga[8], gb[8], c[8], s[8];
        qk_gains<INTER>(t.gain, chunk, half, ga, gb);
        qk_read_cs<VEC>(cs, tok[u], half, chunk, c, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = a[i] * r * ga[i], q = b[i] * r * gb[i];
          a[i] = p * c[i] - q * s[i];
          b[i] = q * c[i] + p * s[i];
        }
        PairIo<T, INTER, VEC>::store(static_cast<T*>(t.y) + qk_offset(g, t.flat, t.ys, (uint32_t)first + tok[u], head[u] - (which ? g.t[0].heads : 0)), chunk, half, a, b);
      }
    }
  }
}

// blockIdx.y picks queries or keys, so that a lane's sums of the gain's gradient belong to one tensor; the sums of
// all blocks are added in a fixed order by k_qk_gain_sum (no atomics: equal calls give equal gradients).
template <typename T, bool INTER, bool VEC>
__global__ void __launch_bounds__(QK_THREADS) k_qk_norm_rope_bwd(const __grid_constant__ QkArgs g) {
  extern __shared__ __align__(16) float2 cs[];
  __shared__ float warp_sum[QK_THREADS / 32][256];
  const QkTensor& t = g.t[blockIdx.y];
  const uint32_t total = (uint32_t)(qk_batch(g) * g.tokens);
  const int half = g.head_dim / 2, lanes = g.lanes;
  const int chunk = threadIdx.x & (lanes - 1);
  const bool busy = chunk * 8 < half;
  const uint32_t row = (uint32_t)t.heads * lanes;
  const float inv_d = 1.f / (float)g.head_dim;
  float ga[8], gb[8], da[8], db[8];
  qk_gains<INTER>(t.gain, chunk, half, ga, gb);
#pragma unroll
  for (int i = 0; i < 8; ++i) da[i] = db[i] = 0.f;
  for (uint64_t first = (uint64_t)blockIdx.x * g.tile; first < total; first += (uint64_t)gridDim.x * g.tile) {
    const uint32_t count = min((uint32_t)g.tile, total - (uint32_t)first);
    const uint32_t items = count * row;
    for (uint32_t base = 0; base < items; base += QK_THREADS * QK_ITEMS) {
      PairIo<T, INTER, VEC> x[QK_ITEMS], dy[QK_ITEMS];
      uint32_t tok[QK_ITEMS];
      int head[QK_ITEMS];
#pragma unroll
      for (int u = 0; u < QK_ITEMS; ++u) {
        const uint32_t i = base + u * QK_THREADS + threadIdx.x;
        tok[u] = i / row;
        head[u] = i < items && busy ? (int)((i - tok[u] * row) / lanes) : -1;
        if (head[u] >= 0) {
          x[u].load(static_cast<const T*>(t.x) + qk_offset(g, t.flat, t.xs, (uint32_t)first + tok[u], head[u]), chunk, half);
          dy[u].load(static_cast<const T*>(t.dy) + qk_offset(g, t.flat, t.ds, (uint32_t)first + tok[u], head[u]), chunk, half);
        } else {
#pragma unroll
          for (int r = 0; r < PairIo<T, INTER, VEC>::R; ++r) x[u].raw[r] = dy[u].raw[r] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      if (base == 0) {
        __syncthreads();
        qk_angles(g, (uint32_t)first, count, cs);
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < QK_ITEMS; ++u) {
        float a[8], b[8], ua[8], ub[8], ss = 0.f, dot = 0.f;
        x[u].get(a, b);
        dy[u].get(ua, ub);
        if (head[u] >= 0) {
          float c[8], s[8];
          qk_read_cs<VEC>(cs, tok[u], half, chunk, c, s);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p = ua[i], q = ub[i];
            ua[i] = p * c[i] + q * s[i];
            ub[i] = q * c[i] - p * s[i];
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss += a[i] * a[i] + b[i] * b[i];
          dot += ua[i] * ga[i] * a[i] + ub[i] * gb[i] * b[i];
        }
        ss = group_sum(ss, lanes);
        dot = group_sum(dot, lanes);
        if (head[u] < 0) continue;
        const float r = rsqrtf(ss * inv_d + g.eps);
        const float m = dot * r * inv_d;  // mean(w n)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float na = a[i] * r, nb = b[i] * r;
          da[i] += ua[i] * na;
          db[i] += ub[i] * nb;
          a[i] = r * (ua[i] * ga[i] - na * m);
          b[i] = r * (ub[i] * gb[i] - nb * m);
        }
        PairIo<T, INTER, VEC>::store(static_cast<T*>(t.y) + qk_offset(g, t.flat, t.ys, (uint32_t)first + tok[u], head[u]), chunk, half, a, b);
      }
    }
  }
  // lanes with the same chunk, then the block's warps, then (next kernel) the blocks
#pragma unroll
  for (int i = 0; i < 8; ++i)
    for (int o = 16; o >= lanes; o >>= 1) {
      da[i] += __shfl_xor_sync(0xffffffffu, da[i], o);
      db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
    }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane < lanes) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = 8 * chunk + i;
      if (c < half) {
        warp_sum[warp][INTER ? 2 * c : c] = da[i];
        warp_sum[warp][INTER ? 2 * c + 1 : half + c] = db[i];
      }
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < g.head_dim; d += QK_THREADS) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < QK_THREADS / 32; ++w) s += warp_sum[w][d];
    g.partial[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * g.head_dim + d] = s;
  }
}

__global__ void __launch_bounds__(1024) k_qk_gain_sum(const float* __restrict__ partial, int blocks, int head_dim, float* dq_gain, float* dk_gain) {
  __shared__ float part[1024];
  const int rows = 1024 / head_dim;  // head_dim <= 256
  const int d = threadIdx.x % head_dim, r = threadIdx.x / head_dim;
  float s = 0.f;
  if (r < rows)
    for (int b = r; b < blocks; b += rows) s += partial[((int64_t)blockIdx.x * blocks + b) * head_dim + d];
  part[threadIdx.x] = s;
  __syncthreads();
  if (r == 0) {
    for (int i = 1; i < rows; ++i) s += part[i * head_dim + d];
    (blockIdx.x ? dk_gain : dq_gain)[d] = s;
  }
}

namespace {

bool aligned16(const void* p, const int64_t (&s)[3], int elem) {
  if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  for (int i = 0; i < 3; ++i)
    if ((s[i] * elem) & 15) return false;
  return true;
}

// Checks the arguments and fills the kernels' block; `vec` = 16-byte accesses fit every tensor.
int qk_prepare(const MgbsQkNormArgs* a, bool bwd, QkArgs* g, bool* vec, int* elem) {
  if (!a) return MGBS_ERR_ARG;
  if (a->dtype < MGBS_DT_BF16 || a->dtype > MGBS_DT_F32) return MGBS_ERR_UNSUPPORTED;
  if (a->head_dim < 2 || a->head_dim > 256 || a->head_dim % 2) return MGBS_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->tokens < 0 || a->heads_q < 1 || a->heads_k < 1 || a->heads_q > 4096 || a->heads_k > 4096) return MGBS_ERR_ARG;
  if (a->batch > 0 && a->tokens > 0x7fffffffll / a->batch) return MGBS_ERR_TOO_LARGE;
  if (!(a->eps >= 0.f) || isinf(a->eps)) return MGBS_ERR_ARG;
  if (a->batch == 0 || a->tokens == 0) { g->batch = g->tokens = 0; }
  else if (!a->q || !a->k || !a->q_out || !a->k_out || (bwd && (!a->dq_out || !a->dk_out))) return MGBS_ERR_ARG;
  if (!a->q_gain || !a->k_gain || !a->phase) return MGBS_ERR_ARG;
  if (a->position_bits != 0 && a->position_bits != 32 && a->position_bits != 64) return MGBS_ERR_ARG;
  if (a->position_bits != 0 && !a->positions) return MGBS_ERR_ARG;
  *elem = a->dtype == MGBS_DT_F32 ? 4 : 2;
  *vec = a->head_dim % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    QkTensor& t = g->t[i];
    t.x = i ? a->k : a->q;
    t.y = i ? a->k_out : a->q_out;
    t.dy = bwd ? (i ? a->dk_out : a->dq_out) : nullptr;
    t.gain = i ? a->k_gain : a->q_gain;
    t.heads = i ? a->heads_k : a->heads_q;
    const int64_t *xs = i ? a->k_stride : a->q_stride, *ys = i ? a->k_out_stride : a->q_out_stride, *ds = i ? a->dk_out_stride : a->dq_out_stride;
    for (int j = 0; j < 3; ++j) { t.xs[j] = xs[j]; t.ys[j] = ys[j]; t.ds[j] = bwd ? ds[j] : 0; }
    t.flat = t.xs[0] == a->tokens * t.xs[1] && t.ys[0] == a->tokens * t.ys[1] && (!bwd || t.ds[0] == a->tokens * t.ds[1]);
    *vec = *vec && aligned16(t.x, t.xs, *elem) && aligned16(t.y, t.ys, *elem) && (!bwd || aligned16(t.dy, t.ds, *elem));
  }
  g->phase = a->phase;
  g->positions = a->positions;
  g->pos_sb = a->position_stride[0];
  g->pos_st = a->position_stride[1];
  g->pos_bits = a->position_bits;
  g->count_dev = nullptr;
  g->count_offset = 0;
  g->batch = (int32_t)a->batch;
  g->tokens = (int32_t)a->tokens;
  g->head_dim = a->head_dim;
  int lanes = 1;
  while (lanes * 16 < a->head_dim) lanes *= 2;
  g->lanes = lanes;
  g->eps = a->eps;
  return 0;
}

// Tokens per block iteration: about one round of the block's items, and no more than shared memory holds.
int qk_tile(int heads, int lanes) {
  const int t = QK_THREADS * QK_ITEMS / (heads * lanes);
  return t < 1 ? 1 : t;
}

template <typename T, bool INTER, bool VEC> int qk_launch(QkArgs& g, bool bwd, int blocks, cudaStream_t st) {
  const size_t smem = (size_t)g.tile * (g.head_dim / 2) * sizeof(float2);
  if (bwd) k_qk_norm_rope_bwd<T, INTER, VEC><<<dim3(blocks, 2), QK_THREADS, smem, st>>>(g);
  else k_qk_norm_rope<T, INTER, VEC><<<blocks, QK_THREADS, smem, st>>>(g);
  return (int)cudaGetLastError();
}
template <typename T> int qk_pick(QkArgs& g, bool inter, bool vec, bool bwd, int blocks, cudaStream_t st) {
  if (inter) return vec ? qk_launch<T, true, true>(g, bwd, blocks, st) : qk_launch<T, true, false>(g, bwd, blocks, st);
  return vec ? qk_launch<T, false, true>(g, bwd, blocks, st) : qk_launch<T, false, false>(g, bwd, blocks, st);
}
int qk_dispatch(int dtype, QkArgs& g, bool inter, bool vec, bool bwd, int blocks, cudaStream_t st) {
  if (dtype == MGBS_DT_BF16) return qk_pick<__nv_bfloat16>(g, inter, vec, bwd, blocks, st);
  if (dtype == MGBS_DT_F16) return qk_pick<__half>(g, inter, vec, bwd, blocks, st);
  return qk_pick<float>(g, inter, vec, bwd, blocks, st);
}

constexpr int QK_BWD_BLOCKS = 592;  // four per SM: also the number of partial sums of the gain's gradient

}  // namespace

int qk_norm_rope_counted(const MgbsQkNormArgs* a, const uint32_t* count_dev, int64_t count_offset, void* stream) {
  QkArgs g;
  bool vec;
  int elem;
  const int rc = qk_prepare(a, false, &g, &vec, &elem);
  if (rc) return rc;
  if (g.batch == 0 || g.tokens == 0) return 0;
  g.count_dev = count_dev;
  g.count_offset = count_offset;
  g.tile = qk_tile(a->heads_q + a->heads_k, g.lanes);
  const int64_t tiles = ((int64_t)g.batch * g.tokens + g.tile - 1) / g.tile;
  const int64_t most = (int64_t)device_sms() * 8;
  return qk_dispatch(a->dtype, g, a->interleaved != 0, vec, false, (int)(tiles < most ? tiles : most), (cudaStream_t)stream);
}

}  // namespace mgbs

extern "C" {

int mgbs_sizeof_qk_norm_args(void) { return (int)sizeof(MgbsQkNormArgs); }

int mgbs_qk_norm_rope(const MgbsQkNormArgs* a, void* stream) { return mgbs::qk_norm_rope_counted(a, nullptr, 0, stream); }

int64_t mgbs_qk_norm_rope_backward_workspace(int32_t head_dim) {
  return head_dim < 2 || head_dim > 256 ? 0 : (int64_t)2 * mgbs::QK_BWD_BLOCKS * head_dim * 4;
}

int mgbs_qk_norm_rope_backward(const MgbsQkNormArgs* a, void* stream) {
  using namespace mgbs;
  QkArgs g;
  bool vec;
  int elem;
  const int rc = qk_prepare(a, true, &g, &vec, &elem);
  if (rc) return rc;
  if (!a->workspace || !a->dq_gain || !a->dk_gain) return MGBS_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  g.partial = a->workspace;
  int blocks = 0;
  if (g.batch > 0 && g.tokens > 0) {
    g.tile = qk_tile(a->heads_q > a->heads_k ? a->heads_q : a->heads_k, g.lanes);
    const int64_t tiles = ((int64_t)g.batch * g.tokens + g.tile - 1) / g.tile;
    blocks = (int)(tiles < QK_BWD_BLOCKS ? tiles : QK_BWD_BLOCKS);
    const int e = qk_dispatch(a->dtype, g, a->interleaved != 0, vec, true, blocks, st);
    if (e) return e;
  }
  k_qk_gain_sum<<<2, 1024, 0, st>>>(a->workspace, blocks, a->head_dim, a->dq_gain, a->dk_gain);
  return (int)cudaGetLastError();
}

}  // extern "C"
