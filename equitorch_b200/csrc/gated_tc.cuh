// Gated linear layer on the 5th-generation tensor cores: one kernel of warp roles for its four products.
//
//   FORWARD      [a | u] = x [W0 | W1]           epilogue h = act(a) u
//   PARTIALS     the same product                epilogue da, du from g
//   INPUT_GRAD   dx = [da | du] [W0 | W1]^T      one sum over both halves
//   WEIGHT_GRAD  dWj = x^T dj                    over parts of the rows, float32 partial results
//
// A CTA per SM strides through tiles of 128 rows; a k-block of 128 bytes a row (64 bfloat16, 32 float32) is a stage of the ring.
// Warp 0 copies tiles (TMA), warp 1 issues the MMAs, the last warps (sixteen, eight for float32) empty the accumulators while the next
// tile is multiplied; the dual products have both halves of the columns in one MMA, so the activation and the product never leave the SM.
//
// bfloat16: the MMA reads tiles as they lie in memory, along k or along the rows (both majors, 128-byte swizzle): 128 x 256 results
// a tile, four stages of 48 KB.  What bounds that is L2: a k-block of 48 KB per 512 cycles of MMA and SM is 12 to 14 TB/s over all
// SMs, and no more arrived.  So where there is work for all of them, two CTAs of a cluster share a tile of 256 x 256: each copies its
// 128 rows of A and half of B, 32 KB a k-block, the first one's MMAs read both SMs' shared memory, and each SM has the results of its
// rows (100k x 256 -> 1024: gradient of x 101 -> 93 us, of the weights 90 -> 83; 8192 x 1024 -> 4096: 115 -> 103).
// float32: operands are split into TF32 pairs, three MMAs each, as everywhere in this library.  Eight warps split a stage between the
// copy and the MMA, big parts in place; a tile that lies along the rows is turned on the way, 32 x 32 values a warp at a time, so the
// MMA always finds k along the row.  128 x 128 results a tile, three stages of 64 KB.  The adder of the tensor cores truncates, so the
// products with small parts have a sum of their own, which leaves one truncation for eight terms in place of three, and a sum is taken
// in pieces of 128 terms that the epilogue adds with ordinary rounding (128 terms: 4.5e-6 of the norm with one sum, 7e-7 so).
//
// Every wait is bounded, as in the other tensor-core kernels; on expiry the status flag is raised and the kernel ends.
#pragma once

#include <algorithm>

#include "gated.cuh"

namespace eqt {
namespace gated {
namespace {
using namespace tc;

enum Mode { FORWARD, PARTIALS, INPUT_GRAD, WEIGHT_GRAD };

// k-blocks of a piece: float32 sums are always taken in pieces; bfloat16 ones (SHAPE LONG) where more than LONGEST terms would be one sum,
// which loses up to 1.8e-7 of itself every 16 terms: 3.6e-4 for 32768, a tenth of its rounding, 1.2e-2 for the 2^20 channels allowed.
// The pieces cost the registers of a tile and pairs of CTAs: 2048 x 32776 -> 2048 forward 571 us, 32768 channels in pairs 407; gradient of x at
// 8192 x 1024, hidden 16392 657 us, 16384 in pairs 437.
constexpr int PIECE = 4, LONG_PIECE = 128;
constexpr int64_t LONGEST = 32768;

// HELD: the k-blocks of B stay in shared memory for all tiles of a column, only A comes by (100k x 256 -> 1024 forward: 123 -> 106 us).
enum Shape { ALONE, PAIR, HELD, LONG };
template <typename T> struct Form;
template <> struct Form<__nv_bfloat16> {
  static constexpr int BK = 64, COLS = 256, FIRST = 2, SPLITTERS = 0, EPI = 16, A_BYTES = 16384, HELD_BLOCKS = 4;
  static constexpr int A_STAGE = A_BYTES, B_STAGE = 32768;
};
template <> struct Form<float> {                         // big and small parts
  static constexpr int BK = 32, COLS = 128, FIRST = 4, SPLITTERS = 8, EPI = 8, A_BYTES = 16384, HELD_BLOCKS = 2;
  static constexpr int A_STAGE = 2 * A_BYTES, B_STAGE = 32768;
};
template <typename T> constexpr int threads() { return 32 * (Form<T>::FIRST + Form<T>::SPLITTERS + Form<T>::EPI); }
// Results leave by 32 columns: a warp's patch is 32 rows of them; PARTIALS has two, so that the next tile's g is on its way.  What is
// left of the shared memory are stages: of both operands, of half of B (PAIR), of A alone (HELD).
template <typename T, int MODE> constexpr int patch_bytes() { return (MODE == PARTIALS ? 2 : 1) * Form<T>::EPI * 1024 * (int)sizeof(T); }
template <typename T, int SHAPE> constexpr int held_bytes() { return SHAPE == HELD ? Form<T>::HELD_BLOCKS * Form<T>::B_STAGE : 0; }
template <typename T, int SHAPE> constexpr int stage_bytes() {
  return Form<T>::A_STAGE + (SHAPE == HELD ? 0 : SHAPE == PAIR ? Form<T>::B_STAGE / 2 : Form<T>::B_STAGE);
}
template <typename T, int MODE, int SHAPE> constexpr int stages() {
  return (231424 - 1024 - patch_bytes<T, MODE>() - held_bytes<T, SHAPE>()) / stage_bytes<T, SHAPE>();
}
template <typename T, int MODE, int SHAPE> constexpr size_t shared_bytes() {
  return 1024 + patch_bytes<T, MODE>() + held_bytes<T, SHAPE>() + (size_t)stages<T, MODE, SHAPE>() * stage_bytes<T, SHAPE>();
}

struct alignas(64) Launch {
  CUtensorMap a[2], b[2];                                // WEIGHT_GRAD: a[0] x, b da and du; INPUT_GRAD: a da and du, b W0 and W1
  void *out, *out2;
  const void* g;
  int64_t rows, out_pitch, g_pitch;                      // rows of the results, values between two of theirs and of g's
  unsigned items;
  int64_t part;                                          // WEIGHT_GRAD: results between two partial ones
  int cols, width;                                       // width: columns a tile (of each half, where there are two)
  int row_tiles, col_tiles, kblocks;                     // kblocks: of one half for INPUT_GRAD, of all rows for WEIGHT_GRAD
  int split_blocks;                                      // WEIGHT_GRAD: k-blocks a part
  int whole;                                             // rows of the results and of g start on 16-byte boundaries
  int* status;
};

// What tile a work item is.
struct Item {
  int64_t row;
  int col, half, part, kb0, kb1;
};
template <int MODE, int SHAPE> __device__ __forceinline__ Item item_of(const Launch& p, unsigned i) {
  constexpr int CTAS = SHAPE == PAIR ? 2 : 1;
  Item t{};
  t.col = (int)(i % (unsigned)p.col_tiles) * p.width;
  i /= (unsigned)p.col_tiles;
  t.row = (int64_t)(MODE == WEIGHT_GRAD ? i % (unsigned)p.row_tiles : i) * (CTAS * TILE_M);
  t.kb1 = MODE == INPUT_GRAD ? 2 * p.kblocks : p.kblocks;
  if (MODE == WEIGHT_GRAD) {
    i /= (unsigned)p.row_tiles;
    t.half = (int)(i & 1);
    t.part = (int)(i >> 1);
    t.kb0 = t.part * p.split_blocks;
    t.kb1 = min(p.kblocks, t.kb0 + p.split_blocks);
  }
  return t;
}

__device__ __forceinline__ uint32_t idesc_bf16(int m, int n, bool a_rows, bool b_rows) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_rows << 15) | ((uint32_t)b_rows << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
// Along the rows (MN-major), 128-byte swizzle: 64 values of M or N a line, eight k a group of 1024 bytes, the next 64 values `BK` lines
// on.  The low word of the descriptor; the high word is that of tiles along k, UMMA_DESC_HI.
__device__ __forceinline__ uint32_t lo_rows(uint32_t at) { return ((at & 0x3FFFF) >> 4) | (uint32_t)((Form<__nv_bfloat16>::BK * 128) >> 4) << 16; }
// One thread issues all MMAs, and what it does between two of them counts: low words stepped by immediates, as for TF32.
template <bool TWO, bool ACCUMULATE> __device__ __forceinline__ void mma_bf16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  if constexpr (TWO)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "n"(UMMA_DESC_HI), "n"(ACCUMULATE ? 1 : 0) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "n"(UMMA_DESC_HI), "n"(ACCUMULATE ? 1 : 0) : "memory");
}

// A block of 32 lines of 128 bytes, one warp: float32 to TF32 pairs, the big ones in place, the small ones `small` bytes on.
__device__ __forceinline__ void split_block(unsigned char* block, int small, bool turn, int lane) {
  if (!turn) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float4* at = reinterpret_cast<float4*>(block) + i * 32 + lane;
      float4 hi, lo;
      split_tf32(*at, hi, lo);
      *at = hi;
      *reinterpret_cast<float4*>(reinterpret_cast<unsigned char*>(at) + small) = lo;
    }
    return;
  }
  // lines are k, values along them rows: lane r collects row r and lays it down in the swizzled order of a row
  float v[32];
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = reinterpret_cast<const float*>(block + k * 128)[lane];
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    float4 hi, lo;
    split_tf32(make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]), hi, lo);
    unsigned char* at = block + lane * 128 + ((c ^ (lane & 7)) << 4);
    *reinterpret_cast<float4*>(at) = hi;
    *reinterpret_cast<float4*>(at + small) = lo;
  }
}

// 32 lines of 32 values (or, as float32 from a bfloat16 kernel, of 16) between global memory and a warp's patch, line r at row r of
// `base`, pieces of 16 bytes; in the patch the pieces of a line are permuted so that eight lanes' lines, and the lines that eight lanes
// copy, fall on all banks.
template <typename T> __device__ __forceinline__ uint4* patch_at(unsigned char* patch, int line, int piece) {
  if constexpr (sizeof(T) == 4) return reinterpret_cast<uint4*>(patch + line * 128 + ((piece ^ (line & 7)) << 4));
  return reinterpret_cast<uint4*>(patch + line * 64 + ((piece ^ ((line >> 1) & 3)) << 4));
}
template <typename T> __device__ __forceinline__ void patch_out(unsigned char* patch, unsigned char* base, int64_t pitch, int lines, int pieces, int lane) {
  constexpr int PER = 2 * (int)sizeof(T), STEP = 32 / PER;       // pieces of a line, lines at a time
  __syncwarp();
  const int piece = lane % PER;
#pragma unroll
  for (int i = 0; i < 32 / STEP; ++i) {
    const int line = i * STEP + lane / PER;
    if (line < lines && piece < pieces) *reinterpret_cast<uint4*>(base + line * pitch + piece * 16) = *patch_at<T>(patch, line, piece);
  }
  __syncwarp();
}
// The same for rows that start anywhere: a lane is a column.
template <typename T> __device__ __forceinline__ T* patch_value(unsigned char* patch, int line, int column) {
  constexpr int GROUP = 16 / (int)sizeof(T);
  return reinterpret_cast<T*>(patch_at<T>(patch, line, column / GROUP)) + column % GROUP;
}
template <typename T> __device__ __forceinline__ void patch_out_any(unsigned char* patch, T* base, int64_t pitch, int lines, int columns, int lane) {
  __syncwarp();
#pragma unroll 4
  for (int line = 0; line < lines; ++line)
    if (lane < columns) base[line * pitch + lane] = *patch_value<T>(patch, line, lane);
  __syncwarp();
}
template <typename T> __device__ __forceinline__ void patch_in_any(unsigned char* patch, const T* base, int64_t pitch, int lines, int columns, int lane) {
#pragma unroll 8
  for (int line = 0; line < 32; ++line)
    *patch_value<T>(patch, line, lane) = line < lines && lane < columns ? base[line * pitch + lane] : static_cast<T>(0.f);
}
template <typename T>
__device__ __forceinline__ void patch_in(unsigned char* patch, const unsigned char* base, int64_t pitch, int lines, int pieces, int lane) {
  constexpr int PER = 2 * (int)sizeof(T), STEP = 32 / PER;
  const int piece = lane % PER;
#pragma unroll
  for (int i = 0; i < 32 / STEP; ++i) {
    const int line = i * STEP + lane / PER;
    const bool there = line < lines && piece < pieces;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 ::"r"(s32(patch_at<T>(patch, line, piece))), "l"(there ? base + line * pitch + piece * 16 : base), "r"(there ? 16 : 0) : "memory");
  }
}
// Loads of 16 columns of two accumulators, and the wait that the values of the loads before it pass through.
__device__ __forceinline__ void tmem_issue16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[16], uint32_t (&q)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(q[0]), "+r"(q[1]), "+r"(q[2]), "+r"(q[3]),
                 "+r"(q[4]), "+r"(q[5]), "+r"(q[6]), "+r"(q[7]), "+r"(q[8]), "+r"(q[9]), "+r"(q[10]), "+r"(q[11]), "+r"(q[12]), "+r"(q[13]),
                 "+r"(q[14]), "+r"(q[15])
               :: "memory");
}

// 16 bytes of values
template <typename T> __device__ __forceinline__ uint4 to16(const float (&v)[16 / sizeof(T)]) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      r[i] = __float_as_uint(v[i]);
    } else {
      const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      r[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
template <typename T> __device__ __forceinline__ void from16(const uint4& u, float (&v)[16 / sizeof(T)]) {
  const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(r[i]);
    } else {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
}
// A lane's 32 values to its line of the patch.
template <typename T> __device__ __forceinline__ void line_put(unsigned char* patch, int lane, const float (&v)[32]) {
  constexpr int GROUP = 16 / (int)sizeof(T);
#pragma unroll
  for (int q = 0; q < 32 / GROUP; ++q) {
    float x[GROUP];
#pragma unroll
    for (int i = 0; i < GROUP; ++i) x[i] = v[q * GROUP + i];
    *patch_at<T>(patch, lane, q) = to16<T>(x);
  }
}

// ---- pairs of CTAs ------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival at the barrier of the same place in the first CTA of the pair.
__device__ __forceinline__ void bar_arrive_first(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 at;\n\tmapa.shared::cluster.u32 at, %0, 0;\n\tmbarrier.arrive.release.cluster.shared::cluster.b64 _, [at];\n\t}"
      ::"r"(s32(bar)) : "memory");
}
__device__ __forceinline__ bool bar_try_cluster(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(s32(b)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool bar_wait_cluster(uint64_t* b, uint32_t parity, volatile int* abort_flag) {
  for (int i = 0; i < TC_WAIT_SPINS; ++i) {
    if (bar_try_cluster(b, parity)) return true;
    if ((i & 63) == 63) {
      if (*abort_flag) return false;
      __nanosleep(128);
    }
  }
  *abort_flag = 1;
  return false;
}
// A copy to this CTA's shared memory whose bytes count at the first CTA's barrier: bit 24 of a shared address is the place in the pair.
template <bool TWO> __device__ __forceinline__ void copy_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  if constexpr (!TWO) {
    tma_load_2d(dst, map, c0, c1, bar);
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(s32(dst)), "l"(map), "r"(s32(bar) & 0xFEFFFFFFu), "r"(c0), "r"(c1) : "memory");
  }
}
template <bool TWO> __device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (!TWO) {
    umma_commit(bar);
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(s32(bar)), "h"((uint16_t)3) : "memory");
  }
}

template <typename T, int MODE, int ACT, int SHAPE>
__global__ void __launch_bounds__(threads<T>(), 1) gated_tc_kernel(const __grid_constant__ Launch p) {
  using S = Form<T>;
  constexpr bool F32 = sizeof(T) == 4, TWO = SHAPE == PAIR, PIECES = F32 || SHAPE == LONG, DUAL = MODE == FORWARD || MODE == PARTIALS;
  constexpr bool A_TURNED = MODE == WEIGHT_GRAD, B_TURNED = MODE != INPUT_GRAD;      // the operand lies along the rows
  constexpr int LINE = 128 / (int)sizeof(T);                                          // values of a line
  constexpr int STAGES = stages<T, MODE, SHAPE>(), STAGE = stage_bytes<T, SHAPE>();
  static_assert(STAGES >= 2 && (SHAPE != HELD || DUAL), "two stages at least; B stays for the dual products");
  static_assert(SHAPE != LONG || (!F32 && MODE != WEIGHT_GRAD), "rows are summed in parts, float32 in pieces anyway");
  constexpr int ACC_COLS = F32 ? 2 * S::COLS : S::COLS;                               // of tensor memory: float32 has two sums
  constexpr int CTAS = TWO ? 2 : 1, BLOCKS = F32 ? PIECE : LONG_PIECE;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[STAGES], ready[STAGES], empty[STAGES], acc_full[2], acc_empty[2], held_full, held_ready;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = TWO ? (int)cluster_rank() : 0;
  const unsigned first_item = blockIdx.x / CTAS, item_step = gridDim.x / CTAS;        // HELD: a multiple of the columns, so a CTA has one
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *held = base, *ring = base + held_bytes<T, SHAPE>();
  const int n_mma = DUAL ? 2 * p.width : p.width;                                     // columns of an MMA
  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      bar_init(&full[s], 1);
      bar_init(&ready[s], F32 ? S::SPLITTERS : 1);
      bar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      bar_init(&acc_full[a], 1);
      bar_init(&acc_empty[a], CTAS * S::EPI);
    }
    bar_init(&held_full, 1);
    bar_init(&held_ready, F32 ? S::SPLITTERS : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (TWO) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&tmem_slot)), "r"(2 * ACC_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&tmem_slot)), "r"(2 * ACC_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (TWO) cluster_sync();                              // barriers and tensor memory of both are there
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* ab = &abort_flag;

  // float32: 640 threads of 96 registers, of which those that copy and issue and those that split leave some to the epilogue (all three
  // shares are of whole groups of four warps: 40 + 2 * 64 + 2 * 152 = 472 <= 5 * 96).
  if (warp < S::FIRST) {
    if constexpr (F32) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      // ---------------- copies ----------------
      if (lane == 0) {
        int s = 0;
        uint32_t ph = 1;
        bool ok = true;
        const uint32_t bytes = CTAS * S::A_BYTES + (SHAPE == HELD ? 0 : (uint32_t)n_mma * 128);
        if (SHAPE == HELD && first_item < p.items) {
          const int col = item_of<MODE, SHAPE>(p, first_item).col;
          bar_expect_tx(&held_full, (uint32_t)(p.kblocks * n_mma) * 128);
          for (int kb = 0; kb < p.kblocks; ++kb)
            for (int q = 0; q < 2; ++q)
              for (int c = 0; c < p.width / LINE; ++c)
                tma_load_2d(held + kb * S::B_STAGE + (q * (p.width / LINE) + c) * S::BK * 128, &p.b[q], col + c * LINE, kb * S::BK, &held_full);
        }
        for (unsigned i = first_item; i < p.items && ok && !*ab; i += item_step) {
          const Item t = item_of<MODE, SHAPE>(p, i);
          const int row = (int)t.row + rank * TILE_M;
          // Columns of B that this CTA copies: all, or its half; of the dual products' pair, one weight's.
          const int b_cols = TWO && !DUAL ? p.width / 2 : p.width, col = t.col + (TWO && !DUAL ? rank * b_cols : 0);
          for (int kb = t.kb0; kb < t.kb1; ++kb) {
            if (!bar_wait(&empty[s], ph, ab)) { ok = false; break; }
            unsigned char* st = ring + (size_t)s * STAGE;
            uint64_t* bar = &full[s];
            if (rank == 0) bar_expect_tx(bar, bytes);
            const int h = MODE == INPUT_GRAD ? kb >= p.kblocks : t.half, k = (MODE == INPUT_GRAD && h ? kb - p.kblocks : kb) * S::BK;
            if (A_TURNED) {
#pragma unroll
              for (int c = 0; c < TILE_M / LINE; ++c) copy_2d<TWO>(st + c * S::BK * 128, &p.a[0], row + c * LINE, k, bar);
            } else {
              copy_2d<TWO>(st, &p.a[MODE == INPUT_GRAD ? h : 0], k, row, bar);
            }
            unsigned char* sb = st + S::A_STAGE;
            if (SHAPE == HELD) {
            } else if (MODE == INPUT_GRAD) {
              copy_2d<TWO>(sb, &p.b[h], k, col, bar);
            } else {
              const int q0 = DUAL ? rank : t.half, q1 = DUAL && !TWO ? 2 : q0 + 1;
              for (int q = q0; q < q1; ++q)
                for (int c = 0; c < b_cols / LINE; ++c, sb += S::BK * 128) copy_2d<TWO>(sb, &p.b[q], col + c * LINE, k, bar);
            }
            if (++s == STAGES) s = 0, ph ^= 1;
          }
        }
      }
    } else if (warp == 1) {
      // ---------------- MMAs ----------------
      if (lane == 0 && rank == 0) {
        int s = 0;
        uint32_t ph = 0;
        int piece = 0;
        bool ok = true;
        const uint32_t idesc = F32 ? umma_idesc_tf32(n_mma) : idesc_bf16(CTAS * TILE_M, n_mma, A_TURNED, B_TURNED);
        if (SHAPE == HELD) {
          ok = bar_wait(F32 ? &held_ready : &held_full, 0, ab);
          tc_fence_after();
        }
        for (unsigned i = first_item; i < p.items && ok && !*ab; i += item_step) {
          const Item t = item_of<MODE, SHAPE>(p, i);
          for (int k0 = t.kb0; k0 < t.kb1 && ok; ++piece) {
            const int k1 = PIECES ? min(k0 + BLOCKS, t.kb1) : t.kb1, a = piece & 1;
            const uint32_t parity = (uint32_t)(((piece >> 1) & 1) ^ 1);
            if (!(TWO ? bar_wait_cluster(&acc_empty[a], parity, ab) : bar_wait(&acc_empty[a], parity, ab))) { ok = false; break; }
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(a * ACC_COLS);
            for (int kb = k0; kb < k1; ++kb) {
              if (!(TWO ? bar_wait_cluster(&full[s], ph, ab) : bar_wait(F32 ? &ready[s] : &full[s], ph, ab))) { ok = false; break; }
              tc_fence_after();
              const uint32_t at = s32(ring + (size_t)s * STAGE), bt = SHAPE == HELD ? s32(held + kb * S::B_STAGE) : at + S::A_STAGE;
              if constexpr (F32) {
                const uint32_t ah = umma_lo(at), al = ah + S::A_BYTES / 16, bh = umma_lo(bt), bl = bh + S::COLS * 8;
                if (kb == k0) {
                  umma_tf32_lo<false>(d, ah, bh, idesc);
                  umma_tf32_lo<false>(d + S::COLS, al, bh, idesc);
                } else {
                  umma_tf32_lo<true>(d, ah, bh, idesc);
                  umma_tf32_lo<true>(d + S::COLS, al, bh, idesc);
                }
                umma_tf32_lo<true>(d + S::COLS, ah, bl, idesc);
#pragma unroll
                for (int q = 1; q < 4; ++q) {
                  umma_tf32_lo<true>(d, ah + q * 2, bh + q * 2, idesc);
                  umma_tf32_lo<true>(d + S::COLS, al + q * 2, bh + q * 2, idesc);
                  umma_tf32_lo<true>(d + S::COLS, ah + q * 2, bl + q * 2, idesc);
                }
              } else {
                constexpr int A_STEP = A_TURNED ? 128 : 2, B_STEP = B_TURNED ? 128 : 2;                // 16 of k, in 16 bytes
                const uint32_t a_lo = A_TURNED ? lo_rows(at) : umma_lo(at), b_lo = B_TURNED ? lo_rows(bt) : umma_lo(bt);
                if (kb == k0) mma_bf16<TWO, false>(d, a_lo, b_lo, idesc);
                else mma_bf16<TWO, true>(d, a_lo, b_lo, idesc);
#pragma unroll
                for (int q = 1; q < 4; ++q) mma_bf16<TWO, true>(d, a_lo + q * A_STEP, b_lo + q * B_STEP, idesc);
              }
              commit<TWO>(&empty[s]);
              if (++s == STAGES) s = 0, ph ^= 1;
            }
            if (ok) commit<TWO>(&acc_full[a]);
            k0 = k1;
          }
        }
      }
    }
  } else if (warp < S::FIRST + S::SPLITTERS) {
    if constexpr (F32) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ---------------- float32 to TF32 pairs ----------------
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    const int w = warp - S::FIRST;
    if (SHAPE == HELD && first_item < p.items) {
      ok = bar_wait(&held_full, 0, ab);
      for (int b = w; b < p.kblocks * (n_mma / 32) && ok; b += S::SPLITTERS)
        split_block(held + b / (n_mma / 32) * S::B_STAGE + b % (n_mma / 32) * 4096, S::COLS * 128, B_TURNED, lane);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(&held_ready);
    }
    for (unsigned i = first_item; i < p.items && ok && !*ab; i += item_step) {
      const Item t = item_of<MODE, SHAPE>(p, i);
      for (int kb = t.kb0; kb < t.kb1; ++kb) {
        if (!bar_wait(&full[s], ph, ab)) { ok = false; break; }
        unsigned char* st = ring + (size_t)s * STAGE;
        // four blocks of A, up to four of B: one a warp
        if (w < 4) split_block(st + w * 4096, S::A_BYTES, A_TURNED, lane);
        else if (SHAPE != HELD && w - 4 < n_mma / 32) split_block(st + S::A_STAGE + (w - 4) * 4096, S::COLS * 128, B_TURNED, lane);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(&ready[s]);
        if (++s == STAGES) s = 0, ph ^= 1;
      }
    }
  } else {
    // ---------------- epilogue ----------------
    if constexpr (F32) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
    // Warps of the same quarter of the lanes share a tile's columns, 32 at a time in turn; of the dual products, 32 of each half.
    constexpr int SHARES = S::EPI / 4, GROUP = 16 / (int)sizeof(T), TURNS = S::COLS / (DUAL ? 64 : 32) / SHARES;
    const int e = warp - S::FIRST - S::SPLITTERS, quarter = warp & 3, share = e >> 2;
    unsigned char* patch = ring + (size_t)STAGES * STAGE + (size_t)e * 1024 * sizeof(T);
    unsigned char* other = patch + S::EPI * 1024 * sizeof(T);                         // PARTIALS
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const int64_t pitch = p.out_pitch * (int)sizeof(T);
    int piece = 0;
    bool ok = true;
    // PARTIALS: g of a turn, asked for a turn before it is used
    auto fetch = [&](unsigned item, int turn, unsigned char* where) {
      if (item < p.items) {
        const Item x = item_of<MODE, SHAPE>(p, item);
        const int64_t r = x.row + rank * TILE_M + quarter * 32;
        const int c0 = (share + turn * SHARES) * 32, c = x.col + c0, here = (int)max((int64_t)0, min((int64_t)32, p.rows - r));
        const int valid = c0 < p.width ? max(0, min(32, p.cols - c)) : 0;
        const T* from = static_cast<const T*>(p.g) + (here > 0 && valid > 0 ? r * p.g_pitch + c : 0);
        if (p.whole) patch_in<T>(where, reinterpret_cast<const unsigned char*>(from), p.g_pitch * (int)sizeof(T), here, valid / GROUP, lane);
        else patch_in_any<T>(where, from, p.g_pitch, here, valid, lane);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (MODE == PARTIALS) fetch(first_item, 0, patch);
    for (unsigned i = first_item; i < p.items && ok && !*ab; i += item_step) {
      const Item t = item_of<MODE, SHAPE>(p, i);
      const int64_t row = t.row + rank * TILE_M + quarter * 32;
      const int lines = (int)max((int64_t)0, min((int64_t)32, p.rows - row));
      // sums that come in pieces gather in registers: the share's two turns, or its turn of each half
      float sum[PIECES ? 2 : 1][32];
      uint32_t d = 0;
      const int pieces = PIECES ? (t.kb1 - t.kb0 + BLOCKS - 1) / BLOCKS : 1;
      for (int q = 0; q < pieces; ++q, ++piece) {
        const int a = piece & 1;
        if (!bar_wait(&acc_full[a], (uint32_t)((piece >> 1) & 1), ab)) { ok = false; break; }
        tc_fence_after();
        d = lanes + (uint32_t)(a * ACC_COLS);
        if constexpr (PIECES) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int at = DUAL ? b * p.width + share * 32 : (share + b * SHARES) * 32;
            if (at >= n_mma) continue;                                                // a narrow tile: the share has no such columns
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              float v[16];
              tmem_ld16(d + (F32 ? S::COLS : 0) + at + h, v);
#pragma unroll
              for (int c = 0; c < 16; ++c) sum[b][h + c] = q ? sum[b][h + c] + v[c] : v[c];
              if constexpr (F32) {
                tmem_ld16(d + at + h, v);
#pragma unroll
                for (int c = 0; c < 16; ++c) sum[b][h + c] += v[c];
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(&acc_empty[a]);
        }
      }
      if (!ok) break;
#pragma unroll
      for (int turn = 0; turn < TURNS; ++turn) {
        const int c0 = (share + turn * SHARES) * 32;
        if (c0 >= p.width) break;
        if (MODE == PARTIALS) {
          if (turn + 1 < TURNS && c0 + SHARES * 32 < p.width) fetch(i, turn + 1, other);
          else fetch(i + item_step, 0, other);
        }
        const int col = t.col + c0, valid = max(0, min(32, p.cols - col));            // columns of this turn in the results
        const int64_t at = row * p.out_pitch + col;
        if (!DUAL) {
          float v[32];
          if constexpr (PIECES) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = sum[turn][c];
          } else {
            tmem_ld32(d + c0, v);
          }
          if (MODE == INPUT_GRAD || F32) {
            line_put<T>(patch, lane, v);
            T* out = static_cast<T*>(p.out) + at + (MODE == WEIGHT_GRAD ? (t.part * 2 + t.half) * p.part : 0);
            if (MODE == WEIGHT_GRAD || p.whole) patch_out<T>(patch, reinterpret_cast<unsigned char*>(out), pitch, lines, (valid + GROUP - 1) / GROUP, lane);
            else patch_out_any<T>(patch, out, p.out_pitch, lines, valid, lane);
          } else {                                                                    // partial results are float32: 16 columns at a time
            float* out = static_cast<float*>(p.out) + at + (t.part * 2 + t.half) * p.part;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float x[4] = {v[h * 16 + 4 * c], v[h * 16 + 4 * c + 1], v[h * 16 + 4 * c + 2], v[h * 16 + 4 * c + 3]};
                *patch_at<T>(patch, lane, c) = to16<float>(x);
              }
              patch_out<T>(patch, reinterpret_cast<unsigned char*>(out + h * 16), p.out_pitch * 4, lines, (min(16, max(0, valid - h * 16)) + 3) / 4, lane);
            }
          }
          continue;
        }
        // du waits in registers while da leaves through the patch, in which it takes the place of g
        uint4 second[F32 ? 1 : 4];
        if (MODE == PARTIALS) {
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t a[16], u[16];
          if constexpr (!PIECES) {
            tmem_issue16(d + c0 + b * 16, a);
            tmem_issue16(d + p.width + c0 + b * 16, u);
            tmem_arrived(a, u);
          }
#pragma unroll
          for (int q = 0; q < 16 / GROUP; ++q) {
            uint4* at16 = patch_at<T>(patch, lane, b * (16 / GROUP) + q);
            float x[GROUP], y[GROUP], g[GROUP];
            if (MODE == PARTIALS) from16<T>(*at16, g);
#pragma unroll
            for (int c = 0; c < GROUP; c += 2) {
              const int j = q * GROUP + c;
              float ai[2], ui[2];
              Value<float> v[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if constexpr (PIECES) {
                  ai[h] = sum[0][b * 16 + j + h];
                  ui[h] = sum[1][b * 16 + j + h];
                } else {
                  ai[h] = __uint_as_float(a[j + h]);
                  ui[h] = __uint_as_float(u[j + h]);
                }
              }
              v[0] = activate(ai[0], ACT);
              v[1] = activate(ai[1], ACT);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (MODE == FORWARD) {
                  x[c + h] = v[h].y * ui[h];
                } else {
                  x[c + h] = g[c + h] * ui[h] * v[h].dy;
                  y[c + h] = g[c + h] * v[h].y;
                  if (F32) sum[F32 ? 1 : 0][b * 16 + j + h] = y[c + h];
                }
              }
            }
            *at16 = to16<T>(x);
            if (MODE == PARTIALS && !F32) second[F32 ? 0 : b * (16 / GROUP) + q] = to16<T>(y);
          }
        }
        // da and du have rows of their own, wide enough for the last piece; h lies as it has to
        if (MODE == PARTIALS || p.whole) patch_out<T>(patch, reinterpret_cast<unsigned char*>(static_cast<T*>(p.out) + at), pitch, lines, (valid + GROUP - 1) / GROUP, lane);
        else patch_out_any<T>(patch, static_cast<T*>(p.out) + at, p.out_pitch, lines, valid, lane);
        if (MODE == PARTIALS) {
          if constexpr (F32) {
            line_put<T>(patch, lane, sum[1]);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) *patch_at<T>(patch, lane, c) = second[c];
          }
          patch_out<T>(patch, reinterpret_cast<unsigned char*>(static_cast<T*>(p.out2) + at), pitch, lines, (valid + GROUP - 1) / GROUP, lane);
          unsigned char* t0 = patch;
          patch = other;
          other = t0;
        }
      }
      if (!PIECES) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (TWO && rank) bar_arrive_first(&acc_empty[(piece - 1) & 1]);
          else bar_arrive(&acc_empty[(piece - 1) & 1]);
        }
      }
    }
    if (MODE == PARTIALS) asm volatile("cp.async.wait_all;" ::: "memory");
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && abort_flag) {
    atomicExch(p.status, 2);
    let_copies_land(full, STAGES);
    if (SHAPE == HELD) let_copies_land(&held_full, 1);
  }
  __syncthreads();
  if (TWO) cluster_sync();                              // nothing of the other CTA reaches this one's memory any more
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (TWO)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * ACC_COLS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * ACC_COLS) : "memory");
  }
}

// ---- host side ----------------------------------------------------------------------------------
// A (rows, columns) matrix, columns next to each other, rows `pitch` values apart, in boxes of `line` columns by `lines` rows.
template <typename T>
int map_of(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int line, int lines, bool swizzle) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(EQT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch * sizeof(T)};
  const cuuint32_t box[2] = {(cuuint32_t)line, (cuuint32_t)lines}, ones[2] = {1, 1};
  const CUresult r = enc(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                         strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? EQT_OK : fail(EQT_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}

// Columns a tile: as few tiles as `most` allows, of one width, a multiple of the columns of a line.  Narrower ones where that leaves
// SMs idle: a small call is bound by how long one tile takes.
int width_of(int cols, int most, int line, bool narrow, int64_t others) {
  int width;
  for (;; most /= 2) {
    const int tiles = (int)ceil_div(cols, most);
    width = (int)ceil_div(ceil_div(cols, tiles), line) * line;
    if (!narrow || others * ceil_div(cols, width) * 2 > tc::sm_count() || most / 2 < line) return width;
  }
}

template <typename T, int MODE, int SHAPE, int ACT> int launch_form(const GatedArgs& a, cudaStream_t s) {
  using S = Form<T>;
  constexpr bool TWO = SHAPE == PAIR;
  constexpr int ROWS = TWO ? 2 * TILE_M : TILE_M;       // of a tile
  constexpr int LINE = 128 / (int)sizeof(T);
  constexpr bool DUAL = MODE == FORWARD || MODE == PARTIALS, F32 = sizeof(T) == 4;
  const size_t size = sizeof(T);
  const char *w = static_cast<const char*>(a.w), *d = static_cast<const char*>(a.d);
  const char* w1 = w + (size_t)a.c * a.w_pitch * size;
  const char* d1 = d ? d + (size_t)a.n * a.d_pitch * size : nullptr;
  Launch p{};
  int rc = EQT_OK, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaSetDevice(dev);          // the encoder of the maps needs a current context (see make_map)
  // Operands that lie along the rows come in boxes of one line of values by a k-block; for float32 they are turned on the way and
  // need no swizzle.
  if (DUAL) {
    p.cols = a.f, p.rows = a.n, p.kblocks = (int)ceil_div(a.c, S::BK);
    p.width = width_of(a.f, S::COLS / 2, LINE, !TWO, ceil_div(a.n, ROWS));
    rc = map_of<T>(&p.a[0], a.x, a.n, a.c, a.x_pitch, LINE, TILE_M, true);
    if (!rc) rc = map_of<T>(&p.b[0], w, a.c, a.f, a.w_pitch, LINE, S::BK, !F32);
    if (!rc) rc = map_of<T>(&p.b[1], w1, a.c, a.f, a.w_pitch, LINE, S::BK, !F32);
    p.out = MODE == FORWARD ? a.h : a.d;
    p.out2 = const_cast<char*>(d1);
    p.g = a.g;
  } else if (MODE == INPUT_GRAD) {
    p.cols = a.c, p.rows = a.n, p.kblocks = (int)ceil_div(a.f, S::BK);
    p.width = width_of(a.c, S::COLS, LINE, !TWO, ceil_div(a.n, ROWS));
    rc = map_of<T>(&p.a[0], d, a.n, a.f, a.d_pitch, LINE, TILE_M, true);
    if (!rc) rc = map_of<T>(&p.a[1], d1, a.n, a.f, a.d_pitch, LINE, TILE_M, true);
    if (!rc) rc = map_of<T>(&p.b[0], w, a.c, a.f, a.w_pitch, LINE, TWO ? p.width / 2 : p.width, true);
    if (!rc) rc = map_of<T>(&p.b[1], w1, a.c, a.f, a.w_pitch, LINE, TWO ? p.width / 2 : p.width, true);
    p.out = a.dx;
  } else {
    p.cols = a.f, p.rows = a.c, p.kblocks = (int)ceil_div(a.n, S::BK);
    p.width = width_of(a.f, S::COLS, TWO ? 2 * LINE : LINE, !TWO, 2 * a.splits * ceil_div(a.c, ROWS));    // a pair halves it
    p.split_blocks = (int)(a.split_rows / S::BK);
    p.part = (int64_t)a.c * a.d_pitch;
    rc = map_of<T>(&p.a[0], a.x, a.n, a.c, a.x_pitch, LINE, S::BK, !F32);
    if (!rc) rc = map_of<T>(&p.b[0], d, a.n, a.f, a.d_pitch, LINE, S::BK, !F32);
    if (!rc) rc = map_of<T>(&p.b[1], d1, a.n, a.f, a.d_pitch, LINE, S::BK, !F32);
    p.out = a.parts;
  }
  if (rc) return rc;
  p.out_pitch = MODE == PARTIALS || MODE == WEIGHT_GRAD ? a.d_pitch : p.cols;
  p.g_pitch = a.f;
  p.whole = p.cols * sizeof(T) % 16 == 0;
  p.row_tiles = (int)ceil_div(p.rows, ROWS);
  p.col_tiles = (int)ceil_div(p.cols, p.width);
  const int64_t items = (int64_t)p.row_tiles * p.col_tiles * (MODE == WEIGHT_GRAD ? 2 * a.splits : 1);
  if (items > INT32_MAX / 2) return fail(EQT_ERR_UNSUPPORTED, "gated: %lld tiles are more than one launch takes", (long long)items);
  p.items = (unsigned)items;
  p.status = a.status;
  const size_t shared = shared_bytes<T, MODE, SHAPE>();
  auto kernel = gated_tc_kernel<T, MODE, ACT, SHAPE>;
  static std::atomic<uint64_t> allowed{0};               // this kernel's
  if (int r = allow_shared_once(kernel, shared, allowed)) return r;
  constexpr int CTAS = TWO ? 2 : 1;
  cudaLaunchConfig_t config{};
  int64_t at_once = std::min<int64_t>(items, tc::sm_count() / CTAS);
  if (SHAPE == HELD) at_once = std::min<int64_t>(items, tc::sm_count() / p.col_tiles * p.col_tiles);
  config.gridDim = dim3((unsigned)(at_once * CTAS));
  config.blockDim = dim3(threads<T>());
  config.dynamicSmemBytes = shared;
  config.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = CTAS;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = TWO ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, p);
  if (e != cudaSuccess) return fail(EQT_ERR_CUDA, "gated_tc: %s", cudaGetErrorString(e));
  return check_launch("gated_tc");
}

// HELD for the forward pass where B's k-blocks fit and the columns' tiles divide the SMs with little left over (123 -> 106 us at 100k x
// 256 -> 1024; the partial results 149 -> 167 us, since their patches leave A two stages).  Pairs of CTAs from the size on that gives most
// SMs a tile of 256 rows, below it tiles of 128 rows fill more of them; not for the dual products of short sums, whose tiles change hands
// too often (the same call in pairs: forward 132, partial results 171 us).  Both sides at the borders, tiles of 128 rows | pairs | held, us:
//   forward, 100k rows x 384 -> 1024 161 | 147, x 448 -> 2048 367 | 319; 50k x 512 -> 1024 116 | 104; 2048 x 512 -> 1024 10.2 | 11.2
//   forward, 20k x 256 -> 512 18.9 | 21.8 | 17.7, 5000 x 256 -> 512 10.4 | 11.8 | 10.5; float32 50k x 64 -> 200 37.6 | - | 35.6, 20k x 64 -> 64 11.4 | - | 11.3
//   partial results, 100k x 384 -> 1024 194 | 203, x 448 -> 2048 435 | 424; 50k x 512 -> 1024 131 | 132, 640 -> 2048 289 | 249
//   gradient of x, 100k x 256 -> 1024 106 | 96; 8192 x 512 -> 1024 20.9 | 20.9; 4096 x 512 -> 1024 17.5 | 19.3; 20k x 256 -> 512 18.5 | 19.4
//   of the weights, 100k x 256 -> 1024 100 | 84, x 384 -> 1024 144 | 177 (a quarter of the pairs' rows are empty), 50k x 512 -> 2048 191 | 166; 5000
//   x 256 -> 512 10.2 | 11.4
// So the rule is off by up to a fifth where channels are no multiple of 256 (weights), and forward sums of 257 to 511 channels would gain a tenth.
template <typename T, int MODE> Shape shape_of(const GatedArgs& a) {
  constexpr bool DUAL = MODE == FORWARD || MODE == PARTIALS;
  const int64_t sms = tc::sm_count();
  if (MODE == FORWARD) {
    const int64_t columns = ceil_div(a.f, Form<T>::COLS / 2);
    if (a.c <= Form<T>::BK * Form<T>::HELD_BLOCKS && sms / columns * columns * 10 >= sms * 9 && ceil_div(a.n, TILE_M) * columns >= 2 * sms) return HELD;
  }
  if (sizeof(T) == 4) return ALONE;
  if (MODE != WEIGHT_GRAD && (DUAL ? (int64_t)a.c : 2 * (int64_t)a.f) > LONGEST) return LONG;
  const int64_t rows = MODE == WEIGHT_GRAD ? a.c : a.n, cols = MODE == INPUT_GRAD ? a.c : a.f;
  const int64_t tiles = ceil_div(rows, 256) * ceil_div(cols, DUAL ? 128 : 256) * (MODE == WEIGHT_GRAD ? 2 * a.splits : 1);
  return rows > TILE_M && tiles * 5 >= sms * 2 && (!DUAL || a.c >= 512) ? PAIR : ALONE;
}
template <typename T> Shape shape_of(const GatedArgs& a, int product) {
  return product == FORWARD ? shape_of<T, FORWARD>(a) : product == PARTIALS ? shape_of<T, PARTIALS>(a)
         : product == INPUT_GRAD ? shape_of<T, INPUT_GRAD>(a) : shape_of<T, WEIGHT_GRAD>(a);
}

template <typename T, int MODE, int ACT = EQT_ACT_SILU> int launch(const GatedArgs& a, cudaStream_t s) {
  const Shape shape = shape_of<T, MODE>(a);
  if constexpr (MODE == FORWARD) {
    if (shape == HELD) return launch_form<T, MODE, HELD, ACT>(a, s);
  }
  if constexpr (sizeof(T) == 2) {
    if (shape == PAIR) return launch_form<T, MODE, PAIR, ACT>(a, s);
    if constexpr (MODE != WEIGHT_GRAD) {
      if (shape == LONG) return launch_form<T, MODE, LONG, ACT>(a, s);
    }
  }
  return launch_form<T, MODE, ALONE, ACT>(a, s);
}

template <typename T, int MODE> int launch_dual(const GatedArgs& a, cudaStream_t s) {
  switch (a.act) {
    case EQT_ACT_SILU: return launch<T, MODE, EQT_ACT_SILU>(a, s);
    case EQT_ACT_GELU: return launch<T, MODE, EQT_ACT_GELU>(a, s);
    case EQT_ACT_RELU: return launch<T, MODE, EQT_ACT_RELU>(a, s);
    default: return launch<T, MODE, EQT_ACT_SIGMOID>(a, s);
  }
}

template <typename T> int backward(const GatedArgs& a, cudaStream_t s) {
  if (int rc = launch_dual<T, PARTIALS>(a, s)) return rc;
  if (a.dx)
    if (int rc = launch<T, INPUT_GRAD>(a, s)) return rc;
  return a.dw ? launch<T, WEIGHT_GRAD>(a, s) : EQT_OK;
}

}  // namespace
}  // namespace gated
}  // namespace eqt
