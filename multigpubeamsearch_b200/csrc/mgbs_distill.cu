// Distillation from a teacher's top entries.  For a row of student logits z, K entries (index i_k, teacher logit t_k)
// and a temperature T:
//   p = softmax(t / T) over the held entries (0 <= i_k < V),  q = softmax(z / T),
//   loss = sum_k p_k (log p_k - log q[i_k]),   dloss/dz_j = (q_j - sum_{k: i_k = j} p_k) / T.
// A row without entries has loss 0 and gradient 0; an index given twice counts with both probabilities.
//
// What bounds it: bytes, one read of z and (with the gradient) one write.  Two forms, by the width of a row:
// up to 1024 entries a group of 4 to 32 lanes holds the row in registers; a wider row is held in the shared memory of a
// block, or of a cluster of up to eight, between the pass that takes maximum and sum and the pass that writes the
// gradient, so that z is read once.  Rows that not even a cluster holds (over 864 KB) are read twice.  Sums are in float32 and in a fixed order; no atomics.

#include <math.h>

#include "mgbs_operators.cuh"

namespace mgbs {

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

// 2^(x c) relative to the row's maximum m.  Where |m c| is out of all proportion (rows at the type's lowest value, where
// x c would overflow) differences come first, so that equal logits still get equal weights.
struct Scale {
  float c, m, k;
  bool huge;
  __device__ __forceinline__ Scale(float m_, float c_) : c(c_), m(m_) {
    k = rintf(m_ * c_);
    huge = !(fabsf(k) <= 0x1p20f);
  }
  __device__ __forceinline__ float arg(float x) const { return huge ? (x - m) * c : fmaf(x, c, -k); }
  // what a sum taken relative to maximum `other` is multiplied with
  __device__ __forceinline__ float from(float other) const {
    const Scale o(other, c);
    return fast_exp2(huge || o.huge ? (other - m) * c : o.k - k);
  }
};

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
  const Scale sc(m, g.c);
  float s = 0.f, ts = 0.f;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    v[i] = lane + i * lanes < g.width ? fast_exp2(sc.arg(v[i])) : 0.f;
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
      if (p != 0.f) loss += p * (t - sc.arg(Elem<T>::up(z[i])) + log_ratio);
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
        if (first) out[i] = Elem<T>::down(fast_exp2(sc.arg(Elem<T>::up(z[i]))) * scale - p * inv_ts * w);
      }
  }
}

// ---------------------------------------------------------------------------------------------------------------

constexpr int DISTILL_WIDE = 512;  // threads of a block at most

// Maximum m of some logits and the sum of 2^(x c - k), k = m c rounded to a whole number: sums of different m differ by
// exact powers of two, and a term costs one fused step without an error of its own in k.
struct MaxSum { float m, s; };

__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  const Scale to(m == -INFINITY ? 0.f : m, c);  // nothing yet on either side: both sums are 0
  return {m, a.s * to.from(a.m) + b.s * to.from(b.m)};
}

// n of them in shared memory, in order.
__device__ __forceinline__ MaxSum gather(const MaxSum* v, int n, float c) {
  float m = v[0].m;
  for (int i = 1; i < n; ++i) m = fmaxf(m, v[i].m);
  const float k = rintf(m * c);
  if (fabsf(k) <= 0x1p20f) {
    float s = 0.f;
    for (int i = 0; i < n; ++i) s += v[i].m == -INFINITY ? 0.f : v[i].s * fast_exp2(fmaxf(rintf(v[i].m * c), -0x1p30f) - k);
    return {m, s};
  }
  MaxSum all = v[0];
  for (int i = 1; i < n; ++i) all = merge(all, v[i], c);
  return all;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void put_remote(MaxSum* local, int rank, MaxSum v) {  // the same address in block `rank`
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(local)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(v.m), "f"(v.s) : "memory");
}

// One row per cluster of `ranks` blocks, in pieces of 16 bytes on 16-byte boundaries; the elements before the first and
// after the last boundary belong to single threads of the first and the last block.  Shared memory stands in for
// registers: a thread copies its own pieces there asynchronously, in four groups, and reads only those, first for maximum
// and sum as the groups arrive, then for the gradient.  Two blocks of an SM cover one another's waits.  Blocks of a
// cluster send one another their maximum and sum and meet once; everything about the teacher's entries is fetched while
// the row is on its way.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(DISTILL_WIDE, 2) k_distill_wide(const __grid_constant__ DistillArgs g, int ranks, int pieces_per_block, int capacity) {
  constexpr int E = Vec16<T>::N;
  extern __shared__ __align__(16) uint8_t held[];  // [capacity] pieces, then the entries
  __shared__ MaxSum warp_part[DISTILL_WIDE / 32];
  __shared__ MaxSum parts[8];                       // maximum and sum of every block of the cluster
  __shared__ float s_tm, s_ts;
  __shared__ int s_any;
  const int entries4 = (g.entries + 3) / 4;
  int* s_i = reinterpret_cast<int*>(held + (size_t)capacity * 16);
  float* s_t = reinterpret_cast<float*>(s_i + 4 * entries4);  // teacher logits
  float* s_z = s_t + 4 * entries4;                            // the student's at the same columns
  const int rank = ranks > 1 ? (int)(blockIdx.x % ranks) : 0;
  const int64_t row = blockIdx.x / ranks;
  const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31;
  if (ranks > 1) cluster_arrive_relaxed();  // "this block runs": waited for before anything is sent to it
  const T* z = static_cast<const T*>(g.logits) + row * g.row_stride;
  const int head = (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T));  // elements before the first boundary
  const int pieces = (g.width - head) / E, tail = g.width - head - pieces * E;
  const uint4* body = reinterpret_cast<const uint4*>(z + head);
  const int p0 = min(pieces, rank * pieces_per_block), p1 = min(pieces, p0 + pieces_per_block);
  const bool last = rank == ranks - 1;
  const int edge = rank == 0 && tid < head ? tid : last && tid >= 32 && tid < 32 + tail ? g.width - tail + tid - 32 : -1;
  const float edge_z = edge >= 0 ? Elem<T>::up(z[edge]) : -INFINITY;
  const uint4* mine16 = reinterpret_cast<const uint4*>(held) + tid;
  const uint32_t mine_at = smem_addr(mine16);
  const int turns = (min(capacity, p1 - p0) + threads - 1) / threads, group = (turns + 3) / 4;  // pieces per thread, and of them per group
  auto fetch = [&](int base) {
    const int end = min(p1, base + capacity);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll 2
      for (int i = q * group; i < (q + 1) * group; ++i) {
        const int p = base + i * threads + tid;
        if (p < end) copy16(mine_at + i * threads * 16, body + p, 16);
      }
      copy_commit();
    }
  };
  fetch(p0);
  for (int k = tid; k < 4 * entries4; k += threads) {
    const int i = k < g.entries ? distill_index(g, row, k) : -1;
    s_i[k] = i;
    s_t[k] = k < g.entries ? g.teacher[row * g.teacher_stride + k] : -INFINITY;
    s_z[k] = i >= 0 ? Elem<T>::up(z[i]) : 0.f;
  }
  const float w = GRAD ? (g.weight ? g.weight[row] : 1.f) * g.inv_t : 0.f;
  MaxSum mine{-INFINITY, 0.f};
  auto take = [&](int base, int q, float extra) {  // group q of the pieces held from `base` on
    const int end = min(p1, base + capacity);
    float top = fmaxf(mine.m, extra);
#pragma unroll 2
    for (int i = q * group; i < (q + 1) * group; ++i)
      if (base + i * threads + tid < end) top = fmaxf(top, Vec16<T>::top(mine16[i * threads]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const Scale sc(top == -INFINITY ? 0.f : top, g.c);  // one for the warp
    mine.s = mine.s * sc.from(mine.m) + fast_exp2(sc.arg(extra));
    mine.m = top;
    if (!sc.huge) {
      const Pair c2 = pair(g.c, g.c), k2 = pair(-sc.k, -sc.k);
      Pair part[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll 2
      for (int i = q * group; i < (q + 1) * group; ++i)
        if (base + i * threads + tid < end) {
          float v[E];
          Vec16<T>::up(mine16[i * threads], v);
#pragma unroll
          for (int j = 0; j < E; j += 2) part[j / 2 & 1] = add2(part[j / 2 & 1], exp2_2(fma2(pair(v[j], v[j + 1]), c2, k2)));
        }
      const float2 sum = both(add2(part[0], part[1]));
      mine.s += sum.x + sum.y;
    } else {
#pragma unroll 1
      for (int i = q * group; i < (q + 1) * group; ++i)
        if (base + i * threads + tid < end) {
          float v[E];
          Vec16<T>::up(mine16[i * threads], v);
#pragma unroll
          for (int j = 0; j < E; ++j) mine.s += fast_exp2(sc.arg(v[j]));
        }
    }
  };
  for (int base = p0; base == p0 || base < p1; base += capacity) {
    if (base != p0) fetch(base);
    copy_wait<3>();
    take(base, 0, base == p0 ? edge_z : -INFINITY);
    copy_wait<2>();
    take(base, 1, -INFINITY);
    copy_wait<1>();
    take(base, 2, -INFINITY);
    copy_wait<0>();
    take(base, 3, -INFINITY);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine.s += __shfl_xor_sync(0xffffffffu, mine.s, o);
  if (lane == 0) warp_part[warp] = mine;
  __syncthreads();
  if (ranks > 1) cluster_wait();
  if (warp == 0) {
    const MaxSum whole = gather(warp_part, threads / 32, g.c);
    if (ranks == 1) { if (lane == 0) parts[0] = whole; }
    else if (lane < ranks) put_remote(&parts[rank], lane, whole);
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
  if (ranks > 1) { cluster_arrive(); cluster_wait(); }
  else __syncthreads();
  const MaxSum all = gather(parts, ranks, g.c);
  const Scale sc(all.m, g.c);
  const float tm = s_tm, inv_ts = 1.f / s_ts;
  const bool any = s_any != 0;
  if (rank == 0 && warp == 0) {
    const float log_ratio = log2f(all.s) - log2f(s_ts);
    float loss = 0.f;
    if (any)
      for (int k = lane; k < g.entries; k += 32) {
        if (s_i[k] < 0) continue;
        const float t = (s_t[k] - tm) * g.c, p = fast_exp2(t) * inv_ts;
        if (p != 0.f) loss += p * (t - sc.arg(s_z[k]) + log_ratio);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
    if (lane == 0) g.loss[row] = loss * kLn2;
  }
  if (GRAD) {
    T* out = static_cast<T*>(g.grad) + row * g.grad_stride;
    const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(z)) & 15) == 0;
    const float scale = any ? w / all.s : 0.f;
    if (edge >= 0) out[edge] = Elem<T>::down(any ? fast_exp2(sc.arg(edge_z)) * scale : 0.f);
    T* out_body = out + head;
    const Pair c2 = pair(g.c, g.c), k2 = pair(-sc.k, -sc.k), w2 = pair(scale, scale);
    for (int base = p0; base < p1; base += capacity) {
      const int end = min(p1, base + capacity);
      if (p1 - p0 > capacity) {  // the row is not all held
        fetch(base);
        copy_wait<0>();
      }
      if (same && any && !sc.huge) {
#pragma unroll 2
        for (int p = base + tid, i = 0; p < end; p += threads, i += threads) {
          float v[E];
          Vec16<T>::up(mine16[i], v);
#pragma unroll
          for (int j = 0; j < E; j += 2) {
            const float2 q = both(mul2(exp2_2(fma2(pair(v[j], v[j + 1]), c2, k2)), w2));
            v[j] = q.x; v[j + 1] = q.y;
          }
          reinterpret_cast<uint4*>(out_body)[p] = Vec16<T>::down(v);
        }
      } else {
#pragma unroll 1
        for (int p = base + tid, i = 0; p < end; p += threads, i += threads) {
          float v[E];
          Vec16<T>::up(mine16[i], v);
#pragma unroll
          for (int j = 0; j < E; ++j) out_body[p * E + j] = Elem<T>::down(any ? fast_exp2(sc.arg(v[j])) * scale : 0.f);
        }
      }
    }
    __syncthreads();
    // the entries' columns once more, from float32: the first of equal indices writes, for all of them
    if (any)
      for (int k = tid; k < g.entries; k += threads) {
        const int i = s_i[k];
        if (i < 0) continue;
        const int piece = i < head ? -1 : (i - head) / E;  // -1 and `pieces`: the edges
        if (piece < 0 ? rank != 0 : piece >= pieces ? !last : piece < p0 || piece >= p1) continue;  // another block's column
        float p = 0.f;
        bool first = true;
        for (int n = 0; n < entries4; ++n) {
          const int4 four = reinterpret_cast<const int4*>(s_i)[n];
          if (four.x != i && four.y != i && four.z != i && four.w != i) continue;
          const int f[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (f[j] == i) {
              first = first && 4 * n + j >= k;
              p += fast_exp2((s_t[4 * n + j] - tm) * g.c);
            }
        }
        if (first) out[i] = Elem<T>::down(fast_exp2(sc.arg(s_z[k])) * scale - p * inv_ts * w);
      }
  }
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

constexpr int DISTILL_HELD = 108 * 1024;  // bytes of a row per block: two blocks and their entries fit an SM
template <typename T, bool GRAD> int distill_wide(const DistillArgs& g, int sms, cudaStream_t st) {
  static std::atomic<uint64_t> raised{0};
  const int rc = raise_smem(k_distill_wide<T, GRAD>, DISTILL_HELD + 12 * MGBS_DISTILL_MAX_ENTRIES, raised);
  if (rc) return rc;
  const int64_t pieces = g.width / Vec16<T>::N;  // at most, whatever the row's first byte
  // the fewest blocks that hold the row; more of them while that leaves SMs without work
  int64_t ranks = (pieces * 16 + DISTILL_HELD - 1) / DISTILL_HELD;
  if (ranks > 8) ranks = 8;
  while (ranks < 8 && g.rows * ranks < sms && pieces > ranks * 1024) ++ranks;
  if (g.rows * ranks > 0x7fffffffll) return MGBS_ERR_TOO_LARGE;
  const int per_block = (int)((pieces + ranks - 1) / ranks);
  const int capacity = per_block * 16 <= DISTILL_HELD ? per_block : DISTILL_HELD / 16;
  int threads = 128;  // some four pieces per thread and more
  while (threads < DISTILL_WIDE && threads * 8 <= per_block) threads *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.rows * ranks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)capacity * 16 + (size_t)(g.entries + 3) / 4 * 4 * 12;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, k_distill_wide<T, GRAD>, g, (int)ranks, per_block, capacity);
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
