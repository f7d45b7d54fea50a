// What the tcgen05 forms of the attention with a relative bias share: tiles, matrix descriptors, tensor memory, bounded
// waits, TMA maps.
#pragma once
#include "mgbs_rel_attention.cuh"
#include "mgbs_tc.cuh"

namespace mgbs {

constexpr int TC_Q = REL_TC_ROWS, TC_K = 64;        // rows of a block, rows of a tile of the other side
constexpr int TC_THREADS = 192;
constexpr int TC_RIM = 256;                         // a tile that is not beyond the reach has offsets below reach + 2 * TC_Q
constexpr int ERR_TC_LOAD = 21, ERR_TC_FREE = 22, ERR_TC_S = 23, ERR_TC_P = 24, ERR_TC_O = 25;

// Matrix descriptor of rows of D 16-bit elements, swizzled in their own width: groups of 8 rows D * 16 bytes apart.  The
// same for K-major (rows are M or N) and MN-major operands (rows are K): the leading offset is unused in both, as a row is
// one swizzle atom wide.  Version 1; layout 128-byte swizzle = 2, 64-byte swizzle = 4.
template <int D> __device__ __forceinline__ uint64_t tc_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | (1ull << 16) | ((uint64_t)(D * 16 >> 4) << 32) | (1ull << 46) | ((D == 64 ? 2ull : 4ull) << 61);
}
template <typename T> struct TcType { static constexpr uint32_t FORMAT = 1; };
template <> struct TcType<__half> { static constexpr uint32_t FORMAT = 0; };
// kind::f16 instruction descriptor: float32 accumulators; operand types; B MN-major or not; N; M = 128
template <typename T> __device__ __forceinline__ constexpr uint32_t tc_idesc(int n, bool b_mn) {
  return (1u << 4) | (TcType<T>::FORMAT << 7) | (TcType<T>::FORMAT << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(TC_Q >> 4) << 24);
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int row, int head, int batch, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(head), "r"(batch), "r"(bar)
      : "memory");
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
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
      ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
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
  for (int i = 0; i < 256; ++i)  // the clock is slow to read: not in an ordinary wait
    if (mbar_try_wait(bar, parity)) return true;
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

// Where a block has given up: its own copies and products on their way still come to an end.
static __device__ __noinline__ void tc_settle(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < 4096; ++i)
    if (mbar_try_wait(bar, parity)) return;
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}

// Rows of one head of a [batch, tokens, heads, D] tensor as TMA boxes of `rows` tokens.
inline int tc_map(CUtensorMap* map, const void* base, const int64_t (&stride)[3], const RelArgs& g, int heads, int d, int rows, bool bf16) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return MGBS_ERR_STATE;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)g.tokens, (cuuint64_t)heads, (cuuint64_t)g.batch};
  const int64_t by[3] = {stride[1], stride[2], stride[0]};  // token, head, batch
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] > 1 ? (cuuint64_t)by[i] * 2 : (cuuint64_t)d * 2;
  const cuuint32_t box[4] = {(cuuint32_t)d, (cuuint32_t)rows, 1, 1}, each[4] = {1, 1, 1, 1};
  auto encode = [&]() {
    return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, each,
               CU_TENSOR_MAP_INTERLEAVE_NONE, d == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  int device;
  // a thread that has made no runtime call yet (autograd's, on its first backward pass) has no context for the driver
  if (r != CUDA_SUCCESS && cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) r = encode();
  return r == CUDA_SUCCESS ? 0 : MGBS_ERR_STATE;
}

inline bool tc_stride_fits(const int64_t (&s)[3], const RelArgs& g, int heads) {
  const int64_t n[3] = {g.batch, g.tokens, heads};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] >= (1ll << 38))) return false;
  return true;
}

}  // namespace mgbs
