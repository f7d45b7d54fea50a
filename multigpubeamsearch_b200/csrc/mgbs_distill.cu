// Distillation from a teacher's top entries.  For a row of student logits z, K entries (index i_k, teacher logit t_k)
// and a temperature T:
//   p = softmax(t / T) over the held entries (0 <= i_k < V),  q = softmax(z / T),
//   loss = sum_k p_k (log p_k - log q[i_k]),   dloss/dz_j = (q_j - sum_{k: i_k = j} p_k) / T.
// A row without entries has loss 0 and gradient 0; an index given twice counts with both probabilities.
//
// What bounds it: bytes, one read of z and (with the gradient) one write.  Two forms, by the width of a row:
// up to 1024 entries a group of 4 to 32 lanes holds the row in registers; wider rows are split over a block, or over a
// cluster of up to eight, each thread holding up to eight 16-byte pieces in registers between the pass that takes
// maximum and sum and the pass that writes the gradient, so that z is read once.  Rows that not even a cluster holds
// (over 512 KB) are read twice.  Sums are in float32 and in a fixed order; no atomics.

#include <cooperative_groups.h>
#include <math.h>

#include "mgbs_operators.cuh"

namespace mgbs {

namespace cg = cooperative_groups;

struct DistillArgs {
  const void* logits;
  void* grad;           // null: loss only
  const float* teacher;
  const void* index;
  const float* weight;  // null: 1
  float* loss;
  int64_t rows, row_stride, grad_stride, teacher_stride, index_stride;
  int32_t width, entries, index64;
  float c, inv_t;  // log2(e) / T, 1 / T
};

__device__ __forceinline__ int distill_index(const DistillArgs& g, int64_t row, int k) {
  const int64_t at = row * g.index_stride + k;
  const int64_t i = g.index64 ? static_cast<const int64_t*>(g.index)[at] : (int64_t) static_cast<const int32_t*>(g.index)[at];
  return i >= 0 && i < g.width ? (int)i : -1;
}

constexpr int DISTILL_THREADS = 256;

template <typename T, int NPL, bool GRAD>
__global__ void __launch_bounds__(DISTILL_THREADS) k_distill_rows(const __grid_constant__ DistillArgs g, int lanes) {
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t row_any = ((int64_t)blockIdx.x * DISTILL_THREADS + threadIdx.x) / lanes;
  const bool live = row_any < g.rows;
  const int64_t row = live ? row_any : g.rows - 1;  // idle groups repeat the last row and write nothing
  const T* z = static_cast<const T*>(g.logits) + row * g.row_stride;
  float v[NPL], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int e = lane + i * lanes;
    v[i] = e < g.width ? Elem<T>::up(z[e]) : -INFINITY;
    m = fmaxf(m, v[i]);
  }
  float tm = -INFINITY;
  int any = 0;
  for (int k = lane; k < g.entries; k += lanes) {
    const float t = g.teacher[row * g.teacher_stride + k];
    if (distill_index(g, row, k) >= 0 && t != -INFINITY) { any = 1; tm = fmaxf(tm, t); }
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
    any |= __shfl_xor_sync(0xffffffffu, any, o);
  }
  // differences first: entries at the type's lowest value stay finite, and equal ones stay equal
  float s = 0.f, ts = 0.f;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    v[i] = lane + i * lanes < g.width ? fast_exp2((v[i] - m) * g.c) : 0.f;
    s += v[i];
  }
  for (int k = lane; k < g.entries; k += lanes)
    if (distill_index(g, row, k) >= 0) ts += fast_exp2((g.teacher[row * g.teacher_stride + k] - tm) * g.c);
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    ts += __shfl_xor_sync(0xffffffffu, ts, o);
  }
  const float log_ratio = log2f(s) - log2f(ts), inv_ts = 1.f / ts;
  float loss = 0.f;
  if (any)
    for (int k = lane; k < g.entries; k += lanes) {
      const int i = distill_index(g, row, k);
      if (i < 0) continue;
      const float t = (g.teacher[row * g.teacher_stride + k] - tm) * g.c;
      const float p = fast_exp2(t) * inv_ts;
      if (p != 0.f) loss += p * (t - (Elem<T>::up(z[i]) - m) * g.c + log_ratio);
    }
  for (int o = lanes >> 1; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
  if (live && lane == 0) g.loss[row] = loss * kLn2;
  if (GRAD) {
    T* out = static_cast<T*>(g.grad) + row * g.grad_stride;
    const float w = (g.weight ? g.weight[row] : 1.f) * g.inv_t;
    const float scale = any ? w / s : 0.f;
    if (live) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const int e = lane + i * lanes;
        if (e < g.width) out[e] = Elem<T>::down(any ? v[i] * scale : 0.f);
      }
    }
    __syncwarp();
    // the entries' columns once more, from float32: the first of equal indices writes, for all of them
    if (live && any)
      for (int k = lane; k < g.entries; k += lanes) {
        const int i = distill_index(g, row, k);
        if (i < 0) continue;
        float p = 0.f;
        bool first = true;
        for (int n = 0; n < g.entries; ++n)
          if (distill_index(g, row, n) == i) {
            first = first && n >= k;
            p += fast_exp2((g.teacher[row * g.teacher_stride + n] - tm) * g.c);
          }
        if (first) out[i] = Elem<T>::down(fast_exp2((Elem<T>::up(z[i]) - m) * g.c) * scale - p * inv_ts * w);
      }
  }
}

// ---------------------------------------------------------------------------------------------------------------

constexpr int DISTILL_WIDE = 512;  // threads of a block

struct MaxSum { float m, s; };  // maximum and sum of 2^((x - m) c)

__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float base = m == -INFINITY ? 0.f : m;  // nothing yet on either side: both sums are 0
  return {m, a.s * fast_exp2((a.m - base) * c) + b.s * fast_exp2((b.m - base) * c)};
}

// One row per cluster of gridDim-given size; piece p of the row holds 16 bytes.  A row that does not start on a
// 16-byte boundary is read from the boundary before it, its first and last piece element by element.
template <typename T, int NV, bool GRAD>
__global__ void __launch_bounds__(DISTILL_WIDE) k_distill_wide(const __grid_constant__ DistillArgs g, int pieces_per_block) {
  constexpr int E = Vec16<T>::N;
  __shared__ MaxSum warp_part[DISTILL_WIDE / 32];
  __shared__ MaxSum block_part;
  __shared__ float s_t[MGBS_DISTILL_MAX_ENTRIES];
  __shared__ int s_i[MGBS_DISTILL_MAX_ENTRIES];
  __shared__ float s_tm, s_ts;
  __shared__ int s_any;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / ranks;
  const int tid = threadIdx.x;
  const T* z = static_cast<const T*>(g.logits) + row * g.row_stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  for (int k = tid; k < g.entries; k += DISTILL_WIDE) {
    s_i[k] = distill_index(g, row, k);
    s_t[k] = g.teacher[row * g.teacher_stride + k];
  }
  const int pieces = (g.width + skew + E - 1) / E;
  const int p0 = rank * pieces_per_block, p1 = min(pieces, p0 + pieces_per_block);
  uint4 raw[NV];
  auto fetch = [&](int base) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = base + i * DISTILL_WIDE + tid;
      const int e = p * E - skew;
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (p < p1) {
        if (e >= 0 && e + E <= g.width) raw[i] = __ldg(reinterpret_cast<const uint4*>(z + e));
        else {
          T* part = reinterpret_cast<T*>(&raw[i]);
#pragma unroll
          for (int j = 0; j < E; ++j) part[j] = e + j >= 0 && e + j < g.width ? z[e + j] : Elem<T>::down(-INFINITY);
        }
      }
    }
  };
  MaxSum mine{-INFINITY, 0.f};
  for (int base = p0; base < p1; base += NV * DISTILL_WIDE) {
    fetch(base);
    float top = mine.m;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (base + i * DISTILL_WIDE + tid < p1) {
        float v[E];
        Vec16<T>::up(raw[i], v);
#pragma unroll
        for (int j = 0; j < E; ++j) top = fmaxf(top, v[j]);
      }
    const float seen = top == -INFINITY ? 0.f : top;
    mine.s *= fast_exp2((mine.m - seen) * g.c);
    mine.m = top;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (base + i * DISTILL_WIDE + tid < p1) {
        float v[E];
        Vec16<T>::up(raw[i], v);
#pragma unroll
        for (int j = 0; j < E; ++j) mine.s += fast_exp2((v[j] - seen) * g.c);
      }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const MaxSum other{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o)};
    mine = merge(mine, other, g.c);
  }
  const int warp = tid >> 5, lane = tid & 31;
  if (lane == 0) warp_part[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    mine = lane < DISTILL_WIDE / 32 ? warp_part[lane] : MaxSum{-INFINITY, 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const MaxSum other{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o)};
      mine = merge(mine, other, g.c);
    }
    if (lane == 0) block_part = mine;
  } else if (warp == 1) {  // the teacher's softmax
    float tm = -INFINITY, ts = 0.f;
    int any = 0;
    for (int k = lane; k < g.entries; k += 32)
      if (s_i[k] >= 0 && s_t[k] != -INFINITY) { any = 1; tm = fmaxf(tm, s_t[k]); }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
      any |= __shfl_xor_sync(0xffffffffu, any, o);
    }
    for (int k = lane; k < g.entries; k += 32)
      if (s_i[k] >= 0) ts += fast_exp2((s_t[k] - tm) * g.c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ts += __shfl_xor_sync(0xffffffffu, ts, o);
    if (lane == 0) { s_tm = tm; s_ts = ts; s_any = any; }
  }
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  MaxSum all = block_part;
  if (ranks > 1) {
    all = *cluster.map_shared_rank(&block_part, 0);
    for (int r = 1; r < ranks; ++r) all = merge(all, *cluster.map_shared_rank(&block_part, r), g.c);
  }
  const float m = all.m, tm = s_tm, inv_ts = 1.f / s_ts;
  const bool any = s_any != 0;
  if (rank == 0 && warp == 0) {
    const float log_ratio = log2f(all.s) - log2f(s_ts);
    float loss = 0.f;
    if (any)
      for (int k = lane; k < g.entries; k += 32) {
        if (s_i[k] < 0) continue;
        const float t = (s_t[k] - tm) * g.c, p = fast_exp2(t) * inv_ts;
        if (p != 0.f) loss += p * (t - (Elem<T>::up(z[s_i[k]]) - m) * g.c + log_ratio);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
    if (lane == 0) g.loss[row] = loss * kLn2;
  }
  if (GRAD) {
    T* out = static_cast<T*>(g.grad) + row * g.grad_stride;
    const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(z)) & 15) == 0;
    const float w = (g.weight ? g.weight[row] : 1.f) * g.inv_t;
    const float scale = any ? w / all.s : 0.f;
    for (int base = p0; base < p1; base += NV * DISTILL_WIDE) {
      if (p1 - p0 > NV * DISTILL_WIDE) fetch(base);  // the row does not stay in registers
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int p = base + i * DISTILL_WIDE + tid;
        if (p >= p1) continue;
        const int e = p * E - skew;
        float v[E];
        Vec16<T>::up(raw[i], v);
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = any ? fast_exp2((v[j] - m) * g.c) * scale : 0.f;
        if (same && e >= 0 && e + E <= g.width) *reinterpret_cast<uint4*>(out + e) = Vec16<T>::down(v);
        else {
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (e + j >= 0 && e + j < g.width) out[e + j] = Elem<T>::down(v[j]);
        }
      }
    }
    __syncthreads();
    if (any)
      for (int k = tid; k < g.entries; k += DISTILL_WIDE) {
        const int i = s_i[k];
        if (i < 0) continue;
        const int piece = (i + skew) / E;
        if (piece < p0 || piece >= p1) continue;  // another block's column
        float p = 0.f;
        bool first = true;
        for (int n = 0; n < g.entries; ++n)
          if (s_i[n] == i) {
            first = first && n >= k;
            p += fast_exp2((s_t[n] - tm) * g.c);
          }
        if (first) out[i] = Elem<T>::down(fast_exp2((Elem<T>::up(z[i]) - m) * g.c) * scale - p * inv_ts * w);
      }
  }
  if (ranks > 1) cluster.sync();  // a block's sums stay until all have read them
}

namespace {

template <typename T, bool GRAD> int distill_rows(const DistillArgs& g, cudaStream_t st) {
  int lanes = 4;
  while (lanes < 32 && lanes * 4 < g.width) lanes *= 2;
  const int64_t blocks = (g.rows * lanes + DISTILL_THREADS - 1) / DISTILL_THREADS;
  if (blocks > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  if (g.width <= 4 * lanes) k_distill_rows<T, 4, GRAD><<<(unsigned)blocks, DISTILL_THREADS, 0, st>>>(g, lanes);
  else if (g.width <= 8 * lanes) k_distill_rows<T, 8, GRAD><<<(unsigned)blocks, DISTILL_THREADS, 0, st>>>(g, lanes);
  else k_distill_rows<T, 32, GRAD><<<(unsigned)blocks, DISTILL_THREADS, 0, st>>>(g, lanes);
  return (int)cudaGetLastError();
}

template <typename T, int NV, bool GRAD> int distill_wide_as(const DistillArgs& g, int ranks, int per_block, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.rows * ranks));
  cfg.blockDim = dim3(DISTILL_WIDE);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, k_distill_wide<T, NV, GRAD>, g, per_block);
}

template <typename T, bool GRAD> int distill_wide(const DistillArgs& g, int sms, cudaStream_t st) {
  const int64_t pieces = ((int64_t)g.width + 2 * Vec16<T>::N - 2) / Vec16<T>::N;  // whatever the row's first byte
  // the fewest blocks that hold the row in eight pieces per thread; more of them while that leaves SMs without work
  int ranks = 1;
  while (ranks < 8 && pieces > (int64_t)ranks * 8 * DISTILL_WIDE) ranks *= 2;
  while (ranks < 8 && g.rows * ranks < sms && pieces > (int64_t)ranks * DISTILL_WIDE) ranks *= 2;
  if (g.rows * ranks > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  const int per_block = (int)((pieces + ranks - 1) / ranks);
  if (per_block <= DISTILL_WIDE) return distill_wide_as<T, 1, GRAD>(g, ranks, per_block, st);
  if (per_block <= 2 * DISTILL_WIDE) return distill_wide_as<T, 2, GRAD>(g, ranks, per_block, st);
  if (per_block <= 4 * DISTILL_WIDE) return distill_wide_as<T, 4, GRAD>(g, ranks, per_block, st);
  return distill_wide_as<T, 8, GRAD>(g, ranks, per_block, st);
}

template <typename T> int distill_typed(const DistillArgs& g, cudaStream_t st) {
  if (g.width <= 1024) return g.grad ? distill_rows<T, true>(g, st) : distill_rows<T, false>(g, st);
  const int sms = device_sms();
  return g.grad ? distill_wide<T, true>(g, sms, st) : distill_wide<T, false>(g, sms, st);
}

}  // namespace
}  // namespace mgbs

extern "C" int mgbs_distill_top_logits(const MgbsDistillArgs* a, void* stream) {
  using namespace mgbs;
  if (!a) return MGBS_ERR_ARG;
  if (a->dtype < MGBS_DT_BF16 || a->dtype > MGBS_DT_F32) return MGBS_ERR_UNSUPPORTED;
  if (a->rows < 0 || a->width < 1 || a->entries < 1) return MGBS_ERR_ARG;
  if (a->entries > MGBS_DISTILL_MAX_ENTRIES || a->width > (1 << 30)) return MGBS_ERR_TOO_LARGE;
  if (a->index_bits != 32 && a->index_bits != 64) return MGBS_ERR_ARG;
  if (!(a->temperature > 0.f) || isinf(a->temperature)) return MGBS_ERR_ARG;
  if (a->rows == 0) return 0;
  if (!a->logits || !a->teacher || !a->index || !a->loss) return MGBS_ERR_ARG;
  if (a->grad && a->grad == a->logits) return MGBS_ERR_ARG;  // the entries' columns are read after the row is written
  const uintptr_t elem = a->dtype == MGBS_DT_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->grad)) % elem) return MGBS_ERR_ARG;
  DistillArgs g;
  g.logits = a->logits; g.grad = a->grad; g.teacher = a->teacher; g.index = a->index; g.weight = a->row_weight; g.loss = a->loss;
  g.rows = a->rows; g.row_stride = a->row_stride; g.grad_stride = a->grad_stride;
  g.teacher_stride = a->teacher_stride; g.index_stride = a->index_stride;
  g.width = a->width; g.entries = a->entries; g.index64 = a->index_bits == 64;
  g.c = kLog2e / a->temperature;
  g.inv_t = 1.f / a->temperature;
  if (isinf(g.c) || isinf(g.inv_t)) return MGBS_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == MGBS_DT_BF16) return distill_typed<__nv_bfloat16>(g, st);
  if (a->dtype == MGBS_DT_F16) return distill_typed<__half>(g, st);
  return distill_typed<float>(g, st);
}
extern "C" int mgbs_sizeof_distill_args(void) { return (int)sizeof(MgbsDistillArgs); }
