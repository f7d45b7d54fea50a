// Distillation from a teacher's top entries.  For a row of student logits z, K entries (index i_k, teacher logit t_k)
// and a temperature T:
//   p = softmax(t / T) over the held entries (0 <= i_k < V),  q = softmax(z / T),
//   loss = sum_k p_k (log p_k - log q[i_k]),   dloss/dz_j = (q_j - sum_{k: i_k = j} p_k) / T.
// A row without entries has loss 0 and gradient 0; an index given twice counts with both probabilities.
//
// What bounds it: bytes, one read of z and (with the gradient) one write.  Two forms, by the width of a row:
// up to 1024 entries a group of 4 to 32 lanes holds the row in registers; a wider row is held in the shared memory of a
// block, or of a cluster of up to eight, between the pass that takes maximum and sum and the pass that writes the
// gradient, so that z is read once.  Rows that not even a cluster holds (over 832 KB) are read twice.  Sums are in float32 and in a fixed order; no atomics.

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
};

constexpr int DISTILL_THREADS = 256;

// A group of `lanes` lanes has a row.  Each lane keeps its first entry in registers from the start, so that a row with no
// more entries than lanes waits for memory once.
template <typename T, int NPL, bool GRAD>
__global__ void __launch_bounds__(DISTILL_THREADS) k_distill_rows(const __grid_constant__ DistillArgs g, int lanes) {
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t row_any = ((int64_t)blockIdx.x * DISTILL_THREADS + threadIdx.x) / lanes;
  const bool live = row_any < g.rows;
  const int64_t row = live ? row_any : g.rows - 1;  // idle groups repeat the last row and write nothing
  const T* z = static_cast<const T*>(g.logits) + row * g.row_stride;
  const float* teacher = g.teacher + row * g.teacher_stride;
  const int i0 = lane < g.entries ? distill_index(g, row, lane) : -1;
  const float t0 = i0 >= 0 ? teacher[lane] : -INFINITY;
  const float w = GRAD ? (g.weight ? g.weight[row] : 1.f) * g.inv_t : 0.f;
  float v[NPL], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int e = lane + i * lanes;
    v[i] = e < g.width ? Elem<T>::up(z[e]) : -INFINITY;
    m = fmaxf(m, v[i]);
  }
  const float z0 = i0 >= 0 ? Elem<T>::up(z[i0]) : 0.f;
  auto index = [&](int k) { return k == lane ? i0 : distill_index(g, row, k); };
  auto logit = [&](int k) { return k == lane ? t0 : teacher[k]; };
  float tm = t0;
  int any = t0 != -INFINITY;
  for (int k = lane + lanes; k < g.entries; k += lanes) {
    const float t = teacher[k];
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
    if (index(k) >= 0) ts += fast_exp2((logit(k) - tm) * g.c);
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    ts += __shfl_xor_sync(0xffffffffu, ts, o);
  }
  const float log_ratio = log2f(s) - log2f(ts), inv_ts = 1.f / ts;
  float loss = 0.f;
  if (any)
    for (int k = lane; k < g.entries; k += lanes) {
      const int i = index(k);
      if (i < 0) continue;
      const float t = (logit(k) - tm) * g.c;
      const float p = fast_exp2(t) * inv_ts;
      if (p != 0.f) loss += p * (t - sc.arg(k == lane ? z0 : Elem<T>::up(z[i])) + log_ratio);
    }
  for (int o = lanes >> 1; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
  if (live && lane == 0) g.loss[row] = loss * kLn2;
  if (GRAD) {
    T* out = static_cast<T*>(g.grad) + row * g.grad_stride;
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
    const int group = threadIdx.x & 31 & ~(lanes - 1);
    for (int k = lane; k - lane < g.entries; k += lanes) {  // whole groups, for the exchange
      const int i = k < g.entries ? index(k) : -1;
      float p = 0.f;
      bool first = true;
      for (int n = 0; n < g.entries; ++n) {
        const int other = n < lanes ? __shfl_sync(0xffffffffu, i0, group + n) : distill_index(g, row, n);
        const float t = n < lanes ? __shfl_sync(0xffffffffu, t0, group + n) : 0.f;
        if (other == i) {
          first = first && n >= k;
          p += fast_exp2(((n < lanes ? t : teacher[n]) - tm) * g.c);
        }
      }
      if (live && any && i >= 0 && first) out[i] = Elem<T>::down(fast_exp2(sc.arg(k == lane ? z0 : Elem<T>::up(z[i]))) * scale - p * inv_ts * w);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------

constexpr int DISTILL_WIDE = 512;  // threads of a block at most

// Sum of 2^(x c - k) over some logits, k whole: sums of different k differ by exact powers of two, and a term costs one
// fused step without an error of its own in k.
struct __align__(8) Sum { int k; float s; };  // one 8-byte store to another block
constexpr int DISTILL_FAR = 1 << 24;  // |k| of logits out of all proportion: the row takes the slow way

// n <= 32 of them in shared memory, in a fixed order; the whole warp calls.
__device__ __forceinline__ Sum gather(const Sum* v, int n) {
  const int lane = threadIdx.x & 31;
  const Sum own = lane < n ? v[lane] : Sum{-2 * DISTILL_FAR, 0.f};
  const int k = __reduce_max_sync(0xffffffffu, own.k);
  float s = own.s * fast_exp2((float)(own.k - k));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return {k, s};
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void put_remote(Sum* local, int rank, Sum v) {  // the same address in block `rank`
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(local)), "r"(rank));
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(v.k), "r"(__float_as_int(v.s)) : "memory");
}

// One row per cluster of `ranks` blocks, in pieces of 16 bytes on 16-byte boundaries; the elements before the first and
// after the last boundary belong to single threads of the first and the last block.  Shared memory stands in for
// registers: a thread copies its own pieces there asynchronously and reads only those, first for the sum as they arrive,
// then for the gradient.  Two blocks of an SM cover one another's waits.  The sum's scale is a warp's maximum over its
// first pieces alone: float32 has room for 2^100 above it, so no further maximum is taken; a warp whose sum leaves that
// room (logits far above its first ones, or nothing but masks among those) makes it anew with its true maximum.  Blocks
// of a cluster send one another their sums and meet once; the last warp sees to the teacher's entries while the row is on
// its way.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(DISTILL_WIDE, 2) k_distill_wide(const __grid_constant__ DistillArgs g, int ranks, int pieces_per_block, int capacity) {
  constexpr int E = Vec16<T>::N;
  extern __shared__ __align__(16) uint8_t held[];  // [capacity] pieces, then the entries
  __shared__ Sum warp_part[DISTILL_WIDE / 32];
  __shared__ Sum parts[8];  // of every block of the cluster
  __shared__ __align__(16) uint32_t s_seen[1024];  // one bit per column modulo 2^15: whether an index may be there twice; cleared 16 bytes at a time
  __shared__ float s_ts;
  __shared__ int s_any, s_twice;
  const int entries4 = (g.entries + 3) / 4;
  int* s_i = reinterpret_cast<int*>(held + (size_t)capacity * 16);
  float* s_p = reinterpret_cast<float*>(s_i + 4 * entries4);  // the entry's probability times s_ts
  float* s_z = s_p + 4 * entries4;                            // the student's logit there
  const int rank = ranks > 1 ? (int)(blockIdx.x % ranks) : 0;
  const int64_t row = blockIdx.x / ranks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int threads = (int)blockDim.x - 32, warps = threads / 32;  // that work on the row; the last warp has the teacher
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
  constexpr int TURN = 4;  // pieces per thread and turn: one group of copies
  // Turns in which every thread has all its pieces need no test; the rest, at most TURN pieces per thread, is the last group.
  auto fetch = [&](int base) {
    const int count = min(capacity, p1 - base), full = count / (TURN * threads);
    const uint4* from = body + base + tid;
    uint32_t to = mine_at;
    for (int t = 0; t < full; ++t, from += TURN * threads, to += TURN * threads * 16) {
#pragma unroll
      for (int i = 0; i < TURN; ++i) copy16(to + i * threads * 16, from + i * threads, 16);
      copy_commit();
    }
#pragma unroll 1
    for (int at = full * TURN * threads + tid; at < count; at += threads, from += threads, to += threads * 16) copy16(to, from, 16);
    copy_commit();
  };
  if (warp < warps) fetch(p0);
  const float w = GRAD ? (g.weight ? g.weight[row] : 1.f) * g.inv_t : 0.f;
  float entropy = 0.f;  // the last warp: sum p log2 p
  if (warp == warps) {
    float tm = -INFINITY, ts = 0.f;
    int any = 0;
    bool twice = false;
    for (int k = lane; k < 256; k += 32) reinterpret_cast<uint4*>(s_seen)[k] = make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
    for (int k = lane; k < 4 * entries4; k += 32) {
      const int i = k < g.entries ? distill_index(g, row, k) : -1;
      const float t = i >= 0 ? g.teacher[row * g.teacher_stride + k] : -INFINITY;
      s_i[k] = i;
      s_p[k] = t;
      if (i >= 0) twice |= (atomicOr(&s_seen[(i & 32767) >> 5], 1u << (i & 31)) >> (i & 31)) & 1u;
      s_z[k] = i >= 0 ? Elem<T>::up(z[i]) : 0.f;
      any |= t != -INFINITY;
      tm = fmaxf(tm, t);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
    any = __any_sync(0xffffffffu, any);
    twice = __any_sync(0xffffffffu, twice);
    for (int k = lane; k < 4 * entries4; k += 32) {
      const float t = any ? (s_p[k] - tm) * g.c : -INFINITY, p = fast_exp2(t);
      ts += p;
      if (p != 0.f) entropy += p * t;
      s_p[k] = p;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ts += __shfl_xor_sync(0xffffffffu, ts, o);
      entropy += __shfl_xor_sync(0xffffffffu, entropy, o);
    }
    if (lane == 0) { s_ts = ts; s_any = any; s_twice = twice; }
    __syncwarp();
  }
  Sum mine{0, 0.f};
  if (warp < warps) {
    const Pair c2 = pair(g.c, g.c);
    Pair k2 = pair(0.f, 0.f), part[2] = {k2, k2};
    auto add16 = [&](const uint4& raw) {
      float v[E];
      Vec16<T>::up(raw, v);
#pragma unroll
      for (int j = 0; j < E; j += 2) part[j / 2 & 1] = add2(part[j / 2 & 1], exp2_2(fma2(pair(v[j], v[j + 1]), c2, k2)));
    };
    auto scale_from = [&](float top) {  // the first pieces' maximum over the warp
      top = fmaxf(top, edge_z);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float k = rintf(top * g.c);
      mine.k = fabsf(k) <= 0x1p20f ? (int)k : 0;
      k2 = pair(-(float)mine.k, -(float)mine.k);
      part[0] = pair(fast_exp2(fmaf(edge_z, g.c, -(float)mine.k)), 0.f);
    };
    for (int base = p0; base == p0 || base < p1; base += capacity) {
      if (base != p0) fetch(base);
      const int count = min(capacity, p1 - base), full = count / (TURN * threads);
      const uint4* from = mine16;
      for (int t = 0; t < full; ++t, from += TURN * threads) {
        const int left = full - t;  // groups still on their way after this one
        if (left >= 3) copy_wait<3>();
        else if (left == 2) copy_wait<2>();
        else copy_wait<1>();
        uint4 raw[TURN];
#pragma unroll
        for (int i = 0; i < TURN; ++i) raw[i] = from[i * threads];
        if (t == 0 && base == p0) {
          float top = Vec16<T>::top(raw[0]);
#pragma unroll
          for (int i = 1; i < TURN; ++i) top = fmaxf(top, Vec16<T>::top(raw[i]));
          scale_from(top);
        }
#pragma unroll
        for (int i = 0; i < TURN; ++i) add16(raw[i]);
      }
      copy_wait<0>();
      const int rest = full * TURN * threads;
      if (full == 0 && base == p0) {
        float top = -INFINITY;
#pragma unroll 1
        for (int at = rest; at + tid < count; at += threads) top = fmaxf(top, Vec16<T>::top(mine16[at]));
        scale_from(top);
      }
#pragma unroll 1
      for (int at = rest; at + tid < count; at += threads) add16(mine16[at]);
    }
    const float2 sum = both(add2(part[0], part[1]));
    mine.s = sum.x + sum.y;
  }
  // The slow way, from global memory: this thread's maximum, and its sum relative to a given one.
  auto maximum = [&]() {
    float top = edge_z;
#pragma unroll 1
    for (int p = p0 + tid; p < p1; p += threads) top = fmaxf(top, Vec16<T>::top(__ldg(body + p)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    return top;
  };
  auto sum_to = [&](const Scale& sc) {
    float sum = edge >= 0 ? fast_exp2(sc.arg(edge_z)) : 0.f;
#pragma unroll 1
    for (int p = p0 + tid; p < p1; p += threads) {
      float v[E];
      Vec16<T>::up(__ldg(body + p), v);
#pragma unroll
      for (int j = 0; j < E; ++j) sum += fast_exp2(sc.arg(v[j]));
    }
    return sum;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine.s += __shfl_xor_sync(0xffffffffu, mine.s, o);
  // The whole warp; a NaN stays, as every sum and the row's results are NaN with it, while a maximum would pass over it.
  if (warp < warps && (mine.s < 0x1p-40f || mine.s > 0x1p100f)) {
    const Scale sc(maximum(), g.c);
    mine.k = sc.huge ? (sc.m > 0.f ? DISTILL_FAR : -DISTILL_FAR) : (int)sc.k;
    mine.s = sc.huge ? 0.f : sum_to(sc);
    if (!sc.huge) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mine.s += __shfl_xor_sync(0xffffffffu, mine.s, o);
    }
  }
  // sums of the block, and of the cluster: every warp ends with the same
  bool first = true;
  auto collect = [&](Sum v) {
    __syncthreads();
    if (lane == 0) warp_part[warp] = v;
    __syncthreads();
    if (ranks == 1) return gather(warp_part, warps);
    if (first) cluster_wait();  // all blocks run
    first = false;
    if (warp == 0) {
      const Sum whole = gather(warp_part, warps);
      if (lane < ranks) put_remote(&parts[rank], lane, whole);
    }
    cluster_arrive();
    cluster_wait();
    const Sum all = gather(parts, ranks);
    return all;
  };
  Sum all = collect(mine);
  Scale sc(0.f, g.c);
  sc.k = (float)all.k;
  if (abs(all.k) >= DISTILL_FAR) {  // the whole cluster: once more, relative to the row's maximum
    const float top = warp < warps ? maximum() : -INFINITY;
    __syncthreads();
    if (lane == 0) warp_part[warp] = Sum{0, top};
    __syncthreads();
    float m = warp_part[0].s;
    for (int i = 1; i < warps; ++i) m = fmaxf(m, warp_part[i].s);
    if (ranks > 1) {
      cluster_arrive();  // all have read the parts before
      cluster_wait();
      if (tid < ranks) put_remote(&parts[rank], tid, Sum{0, m});
      cluster_arrive();
      cluster_wait();
      for (int i = 0; i < ranks; ++i) m = fmaxf(m, parts[i].s);
      cluster_arrive();
      cluster_wait();
    }
    sc = Scale(m, g.c);
    sc.huge = true;
    float sum = warp < warps ? sum_to(sc) : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    all = collect(Sum{0, sum});
  }
  const bool any = s_any != 0;
  const float inv_ts = 1.f / s_ts;
  if (rank == 0 && warp == warps) {
    // sum p (log p - log q) = (sum e t - sum e arg) / ts - log ts + log s, e = 2^t unnormalised
    float cross = 0.f;
    for (int k = lane; k < g.entries; k += 32)
      if (s_p[k] != 0.f) cross += s_p[k] * sc.arg(s_z[k]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cross += __shfl_xor_sync(0xffffffffu, cross, o);
    if (lane == 0) g.loss[row] = any ? ((entropy - cross) * inv_ts + (log2f(all.s) - log2f(s_ts))) * kLn2 : 0.f;
  }
  if (GRAD) {
    T* out = static_cast<T*>(g.grad) + row * g.grad_stride;
    const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(z)) & 15) == 0;
    const float scale = any ? w / all.s : 0.f;
    if (edge >= 0) out[edge] = Elem<T>::down(any ? fast_exp2(sc.arg(edge_z)) * scale : 0.f);
    T* out_body = out + head;
    const Pair c2 = pair(g.c, g.c), k2 = pair(-sc.k, -sc.k), w2 = pair(scale, scale);
    for (int base = warp < warps ? p0 : p1; base < p1; base += capacity) {
      const int end = min(p1, base + capacity);
      if (p1 - p0 > capacity) {  // the row is not all held
        fetch(base);
        copy_wait<0>();
      }
      if (same && any && !sc.huge) {
#pragma unroll 4
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
      for (int k = tid; k < g.entries; k += blockDim.x) {
        const int i = s_i[k];
        if (i < 0) continue;
        const int piece = i < head ? -1 : (i - head) / E;  // -1 and `pieces`: the edges
        if (piece < 0 ? rank != 0 : piece >= pieces ? !last : piece < p0 || piece >= p1) continue;  // another block's column
        float p = s_twice ? 0.f : s_p[k];
        bool is_first = true;
        for (int n = 0; s_twice && n < entries4; ++n) {
          const int4 four = reinterpret_cast<const int4*>(s_i)[n];
          if (four.x != i && four.y != i && four.z != i && four.w != i) continue;
          const int f[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (f[j] == i) {
              is_first = is_first && 4 * n + j >= k;
              p += s_p[4 * n + j];
            }
        }
        if (is_first) out[i] = Elem<T>::down(fast_exp2(sc.arg(s_z[k])) * scale - p * inv_ts * w);
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

constexpr int DISTILL_HELD = 104 * 1024;  // bytes of a row per block: two blocks and 256 entries fit an SM
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
  int threads = 128;  // some four pieces per thread and more
  while (threads < DISTILL_WIDE && threads * 8 <= per_block) threads *= 2;
  // of a row that is not all held, whole turns of the threads: the slow way deals the pieces out without these limits, and
  // a thread must come to the same pieces on both
  const int turn = threads - 32, capacity = per_block * 16 <= DISTILL_HELD ? per_block : DISTILL_HELD / 16 / turn * turn;
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
