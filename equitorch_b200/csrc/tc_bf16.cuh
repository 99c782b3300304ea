// bfloat16 tiles for tcgen05: descriptors, MMAs and maps of operands that lie along k or along the rows.
#pragma once

#include "tc_common.cuh"

namespace eqt {
namespace tc {

// kind::f16 of bfloat16 operands, float32 sums, m x n; `a_rows`, `b_rows`: the operand lies along M or N (MN-major)
__host__ __device__ inline uint32_t idesc_bf16(int m, int n, bool a_rows = false, bool b_rows = false) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_rows << 15) | ((uint32_t)b_rows << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Along the rows, 128-byte swizzle: 64 values of M or N a line, eight k a group of 1024 bytes, the next 64 values `group_bytes` on.  The low
// word of the descriptor; the high word is that of tiles along k, UMMA_DESC_HI.  16 of k are 2048 bytes.
__device__ __forceinline__ uint32_t umma_lo_rows(uint32_t at, uint32_t group_bytes) { return ((at & 0x3FFFF) >> 4) | ((group_bytes >> 4) << 16); }
constexpr uint32_t K_STEP = 2, ROWS_STEP = 128;          // 16 of k in units of 16 bytes, along k and along the rows

// One thread issues all MMAs, and what it does between two of them counts: low words stepped by immediates, as for TF32.
template <bool ACCUMULATE> __device__ __forceinline__ void umma_bf16(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(UMMA_DESC_HI), "n"(ACCUMULATE ? 1 : 0) : "memory");
}
// A in tensor memory: a lane is a row, two values of k a column
template <bool ACCUMULATE> __device__ __forceinline__ void umma_bf16_ta(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "r"(b_lo), "r"(idesc), "n"(UMMA_DESC_HI), "n"(ACCUMULATE ? 1 : 0) : "memory");
}

// Loads of 32 columns, and the wait that the values of the loads before it pass through.
__device__ __forceinline__ void tmem_issue32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_arrived32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :: "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {    // results below 2^-126 are zero, which saves their scaling
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// `parts` matrices (rows, cols) of bfloat16, columns next to each other, rows `pitch` values apart and parts rows * pitch, in boxes of 64
// columns by `lines` rows, 128-byte swizzle; what is outside reads as zero.
inline int map_bf16(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int64_t part_stride, int parts, int lines) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(EQT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaSetDevice(dev);          // the encoder needs a current context (see make_map)
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)parts}, strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)part_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)lines, 1}, ones[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? EQT_OK : fail(EQT_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}

}  // namespace tc
}  // namespace eqt
