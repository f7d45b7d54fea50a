// What the forms of the attention with a relative bias share: the kernels' argument block, lengths, buckets, biases.
#pragma once
#include "mgbs_operators.cuh"

namespace mgbs {

struct RelArgs {
  const void* q; const void* k; const void* v; const void* table; const void* dout;
  const int32_t* map; const int32_t* order; const int32_t* start; const int32_t* lengths;
  void* out; void* dq; void* dk; void* dv;
  float2* stats; float* delta; float* partial;
  int64_t qs[3], ks[3], vs[3], ds[3];
  const uint32_t* count_dev; int64_t count_offset;
  int* error;  // or null: first code of a bounded wait that gave up
  int32_t batch, tokens, heads, heads_kv, buckets, reach, causal;  // reach: max_distance
  float scale, sl2;  // sl2: scale * log2(e)
};

constexpr float REL_BIG = 3.0e38f;
__device__ __forceinline__ int rel_batch(const RelArgs& g) {
  if (!g.count_dev) return g.batch;
  const int64_t left = (int64_t)*g.count_dev - g.count_offset;
  return (int)(left < 0 ? 0 : (left < g.batch ? left : g.batch));
}
__device__ __forceinline__ int rel_length(const RelArgs& g, int b) {
  return g.lengths ? min(max(__ldg(g.lengths + b), 0), g.tokens) : g.tokens;
}
__device__ __forceinline__ int rel_bucket(const RelArgs& g, int off) {
  const int at = min(max(off, -g.reach), g.reach) + g.reach;
  return min(max(__ldg(g.map + at), 0), g.buckets - 1);
}
template <typename T> __device__ __forceinline__ float rel_bias(const RelArgs& g, int off, int h) {
  return Elem<T>::up(static_cast<const T*>(g.table)[(int64_t)rel_bucket(g, off) * g.heads + h]);
}
// x * f where finite values stay finite (the type's lowest value is a usual mask and must not become -inf)
__device__ __forceinline__ float scaled_bias(float x, float f, float most) {
  return isinf(x) ? x : fminf(fmaxf(x * f, -most), most);
}

// bias * log2(e) by offset: bt[off + side] for offsets of at most `side`, by `threads` threads.  A tile of n x n that is not
// beyond the reach has offsets below reach + 2 n.
template <typename T> __device__ __forceinline__ void fill_bias(const RelArgs& g, int h, float* bt, int side, int thread, int threads) {
#pragma unroll 4
  for (int i = thread; i < 2 * side + 1; i += threads) bt[i] = scaled_bias(rel_bias<T>(g, i - side, h), kLog2e, REL_BIG);
}

// Block n's tile of one (sequence, head).  Tiles are dealt out to groups of 64 heads, the heads fastest: under a causal
// mask the longest tiles of a whole group start first (dq 143 us against 111 us head by head, the forward 42 us against
// 34 us, at 6 x 1501 tokens x 8 heads).  The group bounds what the L2 cache has to hold of k and v.
constexpr int REL_DEAL = 64;
struct Where { int tile, head, b; };
__device__ __forceinline__ Where rel_where(int64_t n, int tiles, int heads, int batch) {
  const int64_t first = n / ((int64_t)tiles * REL_DEAL) * REL_DEAL, left = (int64_t)heads * batch - first;
  const int in = (int)(n - first * tiles), members = left < REL_DEAL ? (int)left : REL_DEAL;
  const int64_t unit = first + in % members;
  return {in / members, (int)(unit % heads), (int)(unit / heads)};
}

__device__ __forceinline__ void rel_cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 get_remote(const float* local, int rank) {  // the same address in block `rank` of the cluster
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(local)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
inline int rel_ranks(const RelArgs& g) {  // the most blocks of a cluster that the heads of one key head can be dealt to
  int ranks = 1;
  for (int r = 2; r <= 8; ++r)
    if (g.heads / g.heads_kv % r == 0) ranks = r;
  return ranks;
}

constexpr int REL_TC_ROWS = 128;  // rows of a tile of the tcgen05 forms

// The forward on the fifth-generation tensor cores, and whether TMA can describe the strides (it knows no stride of 0).
bool rel_attention_tc_fits(const RelArgs& g);
int rel_attention_tc(const RelArgs& g, int dtype, int head_dim, cudaStream_t st);
// Its backward: dq, dk, dv, delta and the table's partial sums; the same for dout's strides.
bool rel_attention_tc_backward_fits(const RelArgs& g);
int rel_attention_tc_backward(const RelArgs& g, int dtype, int head_dim, cudaStream_t st);

}  // namespace mgbs
