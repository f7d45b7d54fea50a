// RMS norm of every query and key head with a learned gain, and the rotation by position, in one pass:
//   n = x / sqrt(mean(x^2) + eps),  y_i = R(position) (g n)_i,
// where R turns the pair (a, b) = (y_i, y_i+D/2) or (y_2i, y_2i+1) by the angle position * freq_i.
// Backward, with u = R^T dy:  dgain = sum u n,  w = g u,  dx = (w - n mean(w n)) / sqrt(mean(x^2) + eps).
//
// What bounds it: bytes (x read, y written; backward x, dy read, dx written).  A group of lanes owns one head vector,
// each lane eight pairs, so that both members of a pair are in one lane, loads and stores are 16 bytes wide and the
// only exchange is the sum of squares.  The lanes of a token's query and key heads are the columns of a block: a thread
// stays in its column and walks over tokens, several in flight at a time, so that its gains stay in registers and
// nothing is divided per vector.  Sines and cosines are shared by all heads of a token through shared memory: once per
// block where positions do not depend on the sequence and fit, else once per step.
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
  int32_t cols;      // columns (lanes of a token's heads) per block, blockIdx.y picks which
  int32_t step;      // tokens side by side in a block
  int32_t step_b, step_t;  // step = step_b * tokens + step_t
  int32_t span;      // tokens per block and turn of its loop: step, or step times the tokens in flight per thread
  float eps;
  float* partial;    // backward: [blocks][2][head_dim] sums of the gains' gradients
};

constexpr int QK_THREADS = 256;

// The 16 elements of a lane (8 pairs): a[i], b[i].
template <typename T, bool INTER, bool VEC> struct PairIo {
  static constexpr int R = (int)sizeof(T);  // 16-byte registers of a lane: 16 * sizeof(T) / 16
  uint4 raw[R];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < R; ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
  }
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

// A thread's pairs of a run of tokens: i = thread, thread + threads, ...; only the first is divided.
struct QkPairs {
  uint32_t tok, pair, add_tok, add_pair, half;
  __device__ __forceinline__ explicit QkPairs(uint32_t half_) : half(half_) {
    tok = threadIdx.x / half;
    pair = threadIdx.x - tok * half;
    add_tok = blockDim.x / half;
    add_pair = blockDim.x - add_tok * half;
  }
};

// (cos, sin) of `count` tokens from token `first` of all sequences on: cs[token][pair].  For 16-bit results the fast sine
// and cosine (absolute error 2^-21 on one turn) are far below their rounding.
template <bool FAST> __device__ __forceinline__ void qk_angles(const QkArgs& g, QkPairs p, uint32_t first, uint32_t count, float2* cs) {
  while (p.tok < count) {
    const uint32_t n = first + p.tok, b = n / (uint32_t)g.tokens, t = n - b * (uint32_t)g.tokens;
    const int64_t at = (int64_t)b * g.pos_sb + (int64_t)t * g.pos_st;
    const int64_t pos = g.pos_bits == 64 ? static_cast<const int64_t*>(g.positions)[at]
                        : g.pos_bits == 32 ? (int64_t) static_cast<const int32_t*>(g.positions)[at] : (int64_t)t;
    const float turns = (float)(int32_t)(((uint64_t)pos * __ldg(g.phase + p.pair)) >> 32);  // modulo one turn: signed, 2^-32 each
    float s, c;
    if (FAST) __sincosf(turns * 1.4629180792671596e-9f, &s, &c);  // 2 pi / 2^32
    else sincospif(turns * 4.656612873077393e-10f, &s, &c);       // 2^-31: half turns
    cs[p.tok * p.half + p.pair] = make_float2(c, s);
    p.tok += p.add_tok;
    p.pair += p.add_pair;
    if (p.pair >= p.half) { p.pair -= p.half; ++p.tok; }
  }
}

// Rotation coefficients of a lane's eight pairs; the first of them is below `half`, others past it read nothing.
template <bool VEC> __device__ __forceinline__ void qk_read_cs(const float2* cs, int chunk, int half, float (&c)[8], float (&s)[8]) {
  if (VEC) {
    const float4* p = reinterpret_cast<const float4*>(cs + chunk * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float4 f = p[i]; c[2 * i] = f.x; s[2 * i] = f.y; c[2 * i + 1] = f.z; s[2 * i + 1] = f.w; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = 8 * chunk + i < half ? cs[chunk * 8 + i] : make_float2(0.f, 0.f);
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

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// BWD 0: y from x.  BWD 1: dx from x and dy, and the block's sums of the gains' gradients.  U tokens in flight per thread.
// SHARED: the angles of all `tokens` positions are kept for the whole block.
template <typename T, bool INTER, bool VEC, int U, bool BWD, bool SHARED>
__global__ void __launch_bounds__(QK_THREADS, BWD ? 2 : 3) k_qk_norm_rope(const __grid_constant__ QkArgs g) {
  extern __shared__ __align__(16) float2 angles[];
  float2* cs = angles;
  int odd = 0;
  using Io = PairIo<T, INTER, VEC>;
  const uint32_t total = (uint32_t)(qk_batch(g) * g.tokens);
  const int half = g.head_dim / 2, lanes = g.lanes;
  const int tok = threadIdx.x / g.cols, col = blockIdx.y * g.cols + threadIdx.x % g.cols;
  const int chunk = threadIdx.x & (lanes - 1);  // columns are whole groups of lanes
  const int head_any = col / lanes, which = head_any >= g.t[0].heads;
  const bool busy = tok < g.step && head_any < g.t[0].heads + g.t[1].heads && chunk * 8 < half;
  const QkTensor& t = g.t[which];
  const int head = busy ? head_any - (which ? g.t[0].heads : 0) : 0;
  const T* x0 = static_cast<const T*>(t.x) + head * t.xs[2];
  const T* d0 = BWD ? static_cast<const T*>(t.dy) + head * t.ds[2] : nullptr;
  T* y0 = static_cast<T*>(t.y) + head * t.ys[2];
  const float inv_d = 1.f / (float)g.head_dim;
  float ga[8], gb[8], da[8], db[8];
  qk_gains<INTER>(t.gain, chunk, half, ga, gb);
#pragma unroll
  for (int i = 0; i < 8; ++i) da[i] = db[i] = 0.f;
  const QkPairs pairs(half);
  if (SHARED) {
    qk_angles<sizeof(T) == 2>(g, pairs, 0, g.tokens, cs);
    __syncthreads();
  }
  for (uint64_t first = (uint64_t)blockIdx.x * g.span; first < total; first += (uint64_t)gridDim.x * g.span) {
    const uint32_t stop = (uint32_t)min((uint64_t)total, first + g.span);
    Io x[U], dy[BWD ? U : 1];
    int b[U], at[U];
    uint32_t n = (uint32_t)first + tok;
    b[0] = n / (uint32_t)g.tokens;
    at[0] = n - b[0] * g.tokens;
#pragma unroll
    for (int u = 0; u < U; ++u, n += g.step) {
      if (u > 0) {
        b[u] = b[u - 1] + g.step_b;
        at[u] = at[u - 1] + g.step_t;
        if (at[u] >= g.tokens) { at[u] -= g.tokens; ++b[u]; }
      }
      if (busy && n < stop) {
        x[u].load(x0 + b[u] * t.xs[0] + at[u] * t.xs[1], chunk, half);
        if (BWD) dy[u].load(d0 + b[u] * t.ds[0] + at[u] * t.ds[1], chunk, half);
      } else {
        x[u].clear();
        if (BWD) dy[u].clear();
      }
    }
    if (!SHARED) {
      cs = angles + (odd ? g.span * half : 0);  // two buffers: a step's readers are past the barrier of the next one
      odd ^= 1;
      qk_angles<sizeof(T) == 2>(g, pairs, (uint32_t)first, stop - (uint32_t)first, cs);
      __syncthreads();
    }
    n = (uint32_t)first + tok;
#pragma unroll
    for (int u = 0; u < U; ++u, n += g.step) {
      const bool live = busy && n < stop;
      float a[8], bb[8], c[8], s[8], ss = 0.f;
      x[u].get(a, bb);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + bb[i] * bb[i];
      ss = group_sum(ss, lanes);
      // lanes without a vector hold zeros, which an infinite factor (eps of 0) would make NaN in the gains' gradients
      const float r = live ? rsqrtf(ss * inv_d + g.eps) : 0.f;
      // lanes past the head's pairs take part in its sums: with zeros, which only finite coefficients keep
      qk_read_cs<VEC>(cs + (live ? SHARED ? at[u] : u * g.step + tok : 0) * half, chunk * 8 < half ? chunk : 0, half, c, s);
      if (!BWD) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = a[i] * r * ga[i], q = bb[i] * r * gb[i];
          a[i] = p * c[i] - q * s[i];
          bb[i] = q * c[i] + p * s[i];
        }
      } else {
        float ua[8], ub[8], dot = 0.f;
        dy[u].get(ua, ub);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = ua[i], q = ub[i];
          ua[i] = p * c[i] + q * s[i];
          ub[i] = q * c[i] - p * s[i];
          a[i] *= r;
          bb[i] *= r;
          da[i] += ua[i] * a[i];
          db[i] += ub[i] * bb[i];
          ua[i] *= ga[i];
          ub[i] *= gb[i];
          dot += ua[i] * a[i] + ub[i] * bb[i];
        }
        const float m = group_sum(dot, lanes) * inv_d;  // mean(w n)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a[i] = r * (ua[i] - a[i] * m);
          bb[i] = r * (ub[i] - bb[i] * m);
        }
      }
      if (live) Io::store(y0 + b[u] * t.ys[0] + at[u] * t.ys[1], chunk, half, a, bb);
    }
  }
  if (BWD) {
    // the block's threads of one tensor and chunk in a fixed order, then (next kernel) the blocks: no atomics
    float* part = reinterpret_cast<float*>(angles);  // [thread][16], padded
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[threadIdx.x * 17 + (INTER ? 2 * i : i)] = da[i];
      part[threadIdx.x * 17 + (INTER ? 2 * i + 1 : 8 + i)] = db[i];
    }
    __syncthreads();
    const int col0 = blockIdx.y * g.cols;
    for (int e = threadIdx.x; e < 2 * g.head_dim; e += blockDim.x) {
      const int w = e >= g.head_dim, d = e - w * g.head_dim;
      const int pair = INTER ? d / 2 : d % half, slot = INTER ? d % 16 : (d / half) * 8 + pair % 8;
      float sum = 0.f;
      for (int h = w ? g.t[0].heads : 0; h < g.t[0].heads + (w ? g.t[1].heads : 0); ++h) {
        const int c = h * lanes + pair / 8 - col0;
        if (c < 0 || c >= g.cols) continue;
        for (int k = 0; k < g.step; ++k) sum += part[(k * g.cols + c) * 17 + slot];
      }
      g.partial[((int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 + w) * g.head_dim + d] = sum;
    }
  }
}

// Block (w, c): 32 elements of the gain of queries (w = 0) or keys (1), summed over the rows of [blocks][2][head_dim].
__global__ void __launch_bounds__(1024) k_qk_gain_sum(const float* __restrict__ partial, int blocks, int head_dim, float* dq_gain, float* dk_gain) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, r = threadIdx.x >> 5, d = blockIdx.y * 32 + lane;
  float s = 0.f;
  if (d < head_dim) {
#pragma unroll 4
    for (int b = r; b < blocks; b += 32) s += partial[((int64_t)b * 2 + blockIdx.x) * head_dim + d];
  }
  part[lane][r] = s;
  __syncthreads();
  s = part[r][lane];  // warp r: element r, its 32 partial sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0 && blockIdx.y * 32 + r < head_dim) (blockIdx.x ? dk_gain : dq_gain)[blockIdx.y * 32 + r] = s;
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
  if (a->position_bits != 0 && !a->positions && a->batch > 0 && a->tokens > 0) return MGBS_ERR_ARG;  // no token: null is an empty tensor's address
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

// How a block's threads lie over columns and tokens; returns the grid's second dimension.
int qk_layout(QkArgs& g, int in_flight) {
  const int row = (g.t[0].heads + g.t[1].heads) * g.lanes;
  const int parts = (row + QK_THREADS - 1) / QK_THREADS;
  g.cols = parts == 1 ? row : QK_THREADS;
  g.step = QK_THREADS / g.cols;
  g.step_b = g.step / g.tokens;
  g.step_t = g.step % g.tokens;
  // few tokens: one per thread, over more blocks
  g.span = (int64_t)g.batch * g.tokens * parts > (int64_t)g.step * device_sms() * 2 ? g.step * in_flight : g.step;
  while (g.span > g.step && 2 * g.span * (g.head_dim / 2) * (int64_t)sizeof(float2) > 32768) g.span -= g.step;  // two buffers of angles
  return parts;
}

constexpr int QK_BWD_BLOCKS = 592;  // at most, also the number of partial sums of the gains' gradients

// Blocks per SM of one kernel (a template argument, because all of them have one type), asked once per number of warps and
// 8 KB of shared memory at the most of both: the grid, and with it the order of the gains' partial sums, depends on
// nothing that was called before.
template <void (*KERNEL)(QkArgs)> int qk_resident(int threads, size_t smem) {
  static std::atomic<int> known[9][9];
  const size_t step = (smem + 8191) / 8192;  // of at most 49152 bytes without a raised limit
  std::atomic<int>& n = known[threads / 32][step > 8 ? 8 : step];
  int v = n.load(std::memory_order_relaxed);
  if (!v) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v, KERNEL, threads, step * 8192) != cudaSuccess || v < 1) v = 1;
    n.store(v, std::memory_order_relaxed);
  }
  return v;
}

template <typename T, bool INTER, bool VEC, int U, bool BWD, bool SHARED> int qk_start(QkArgs& g, int parts, int* blocks, cudaStream_t st) {
  constexpr auto kernel = k_qk_norm_rope<T, INTER, VEC, U, BWD, SHARED>;
  const int threads = (g.cols * g.step + 31) / 32 * 32;
  size_t smem = (size_t)(SHARED ? g.tokens : 2 * g.span) * (g.head_dim / 2) * sizeof(float2);
  if (BWD && smem < QK_THREADS * 17 * sizeof(float)) smem = QK_THREADS * 17 * sizeof(float);
  const int64_t turns = ((int64_t)g.batch * g.tokens + g.span - 1) / g.span;
  int64_t most = (int64_t)device_sms() * qk_resident<k_qk_norm_rope<T, INTER, VEC, U, BWD, SHARED>>(threads, smem);  // one wave: every block has the same work
  if (BWD && most > QK_BWD_BLOCKS) most = QK_BWD_BLOCKS;
  most = most < parts ? 1 : most / parts;
  if (BWD && parts > QK_BWD_BLOCKS) return MGBS_ERR_TOO_LARGE;
  if (turns < most) most = turns;
  kernel<<<dim3((unsigned)most, parts), threads, smem, st>>>(g);
  *blocks = (int)most * parts;
  return (int)cudaGetLastError();
}
template <typename T, bool INTER, bool VEC, bool BWD> int qk_launch(QkArgs& g, int* blocks, cudaStream_t st) {
  constexpr int U = sizeof(T) == 4 ? (BWD ? 1 : 2) : (BWD ? 2 : 3);
  const int parts = qk_layout(g, U);
  if (VEC && g.pos_sb == 0 && g.batch > 1 && (int64_t)g.tokens * (g.head_dim / 2) * (int64_t)sizeof(float2) <= 16384)
    return qk_start<T, INTER, VEC, U, BWD, VEC>(g, parts, blocks, st);
  return qk_start<T, INTER, VEC, U, BWD, false>(g, parts, blocks, st);
}
template <typename T, bool BWD> int qk_pick(QkArgs& g, bool inter, bool vec, int* blocks, cudaStream_t st) {
  if (inter) return vec ? qk_launch<T, true, true, BWD>(g, blocks, st) : qk_launch<T, true, false, BWD>(g, blocks, st);
  return vec ? qk_launch<T, false, true, BWD>(g, blocks, st) : qk_launch<T, false, false, BWD>(g, blocks, st);
}
template <bool BWD> int qk_dispatch(int dtype, QkArgs& g, bool inter, bool vec, int* blocks, cudaStream_t st) {
  if (dtype == MGBS_DT_BF16) return qk_pick<__nv_bfloat16, BWD>(g, inter, vec, blocks, st);
  if (dtype == MGBS_DT_F16) return qk_pick<__half, BWD>(g, inter, vec, blocks, st);
  return qk_pick<float, BWD>(g, inter, vec, blocks, st);
}

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
  int blocks;
  return qk_dispatch<false>(a->dtype, g, a->interleaved != 0, vec, &blocks, (cudaStream_t)stream);
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
    const int e = qk_dispatch<true>(a->dtype, g, a->interleaved != 0, vec, &blocks, st);
    if (e) return e;
  }
  k_qk_gain_sum<<<dim3(2, (a->head_dim + 31) / 32), 1024, 0, st>>>(a->workspace, blocks, a->head_dim, a->dq_gain, a->dk_gain);
  return (int)cudaGetLastError();
}

}  // extern "C"
