// Cross entropy over the types of a table, without keeping the logits.
//
//     z = x w^T  (n, t)      lse_i = log sum_t exp z_it      loss_i = lse_i - z_i,target
//     backward, with r_i the row's share of the result (zero where the target is negative):
//         G_it = r_i (exp(z_it - lse_i) - [t = target_i])        dx = G w        dw = G^T x
//
// A share that all rows have (a sum's, a mean's) is left out of G and multiplied to the sums: early in training G is -r_i at the target and little elsewhere, and
// the rounding of one r would be every row's (1000 rows, 2-norm of dx's error 3.3e-3 | 2.3e-3, of a result's rounding 1.7e-3).
//
// One kernel of warp roles on the 5th-generation tensor cores makes all four products:
//
//   LOGITS   z, tile by tile; a thread of the epilogue has a row's 64 logits of a tile in registers and carries their maximum, in units of log2, and sum of
//            exponentials over a run of tiles, which is all that leaves the SM (8 bytes for 64 to 2048 logits)
//   SCORES   z again for a piece of the types, and from it G, rounded to bfloat16 (of few types to two, float32 to three parts of it), to scratch
//   INPUT    dx += G w of the piece         WEIGHT   dw = G^T x of the piece
//
// G of a piece is at most PIECE_BYTES (or, of over a million rows, of 128 types), and pieces add to one float32 dx, which the last one rounds, so scratch does not grow with the
// table; a piece that has a wave of WEIGHT's tiles has whole ones.  Sums that would leave SMs idle are cut into parts, float32 partial results that one kernel adds
// in their order.  Floor: 8 n t c flops for both passes.
// At most MOST_TERMS channels.  Bound by the tensor cores: 16,384 rows, 32,768 types, 512 bfloat16 channels 573 us of LOGITS (0.96 PFLOP/s, the exponentials
// at the same time), four pieces of 124, 130 and 120 (1.06 to 1.15 PFLOP/s); pairs of CTAs for a tile of 256 x 256 took 532, 151, 114 and 122 (2100 | 2130 us in
// all).  float32 5003 x 14,161 x 128: LOGITS 102, then 81, 74 and 57 twice, bound by the shared memory that six products of split operands read.
//
// A CTA per SM; warp 0 copies tiles (TMA), warp 1 issues the MMAs, the other eight (float32: sixteen) are the epilogue.  A k-block is 64
// values of k; operands lie along k or along the rows, as they are in memory.  bfloat16: tiles of 128 x 256, four stages of 48 KB, two sums of 256 columns in tensor memory.
// float32: operands are split once into three bfloat16 parts (24 bits), six products of which leave 2^-26 of a term; a stage has all parts of
// both operands, 96 KB for 128 x 128 results, and products with small parts have a sum of their own, so that the truncation of the tensor cores' adder counts once every
// 16 terms.  A float32 sum is taken out of the tensor cores every `fold` k-blocks (512 terms lose at most 4e-6); bfloat16 sums are of at most MOST_TERMS, which
// lose 2e-4, a tenth of the rounding of a result: longer ones are cut into parts.
//
// Rows whose target is negative may hold anything: their G is set, not multiplied, to zero, and the backward pass reads x from a copy in which they are zero.
#include <algorithm>
#include <type_traits>

#include "tc_bf16.cuh"

namespace eqt {
namespace type_loss {
namespace {
using namespace tc;

enum Mode { LOGITS, SCORES, INPUT, WEIGHT };
constexpr int BK = 64;                                   // k of a block
constexpr float LOG2E = 1.4426950408889634f;
constexpr int64_t PIECE_BYTES = int64_t(256) << 20, MOST_TERMS = 16384;

template <int PARTS> constexpr int cols() { return PARTS == 1 ? 256 : 128; }             // of a tile
template <int PARTS> constexpr int epilogue_warps() { return PARTS == 1 ? 8 : 16; }
template <int PARTS> constexpr int share() { return 4 * cols<PARTS>() / epilogue_warps<PARTS>(); }     // of a tile's columns, that a thread of the epilogue has
template <int PARTS> constexpr int threads() { return 32 * (2 + epilogue_warps<PARTS>()); }
template <int PARTS> constexpr int a_bytes() { return PARTS * TILE_M * BK * 2; }
template <int PARTS> constexpr int stage_bytes() { return a_bytes<PARTS>() + PARTS * cols<PARTS>() * BK * 2; }
constexpr int PATCH = 2048;                              // a warp's: 32 rows of 64 bytes
template <int PARTS> constexpr int stages() { return (232448 - 1024 - epilogue_warps<PARTS>() * PATCH - 1024) / stage_bytes<PARTS>(); }
template <int PARTS> constexpr size_t shared_bytes() { return 1024 + (size_t)stages<PARTS>() * stage_bytes<PARTS>() + epilogue_warps<PARTS>() * PATCH; }

struct alignas(64) Launch {
  CUtensorMap a, b;
  int64_t rows;                                          // of the results
  int columns, width;                                    // of the results, of a tile
  int planes, plane_blocks;                              // of G, bfloat16: what rounding its first leaves is in the second; k-blocks of each
  int row_tiles, col_tiles, run, kblocks, part_blocks, fold;       // run: LOGITS, column tiles of an item
  unsigned items;
  int a_first, b_first;                                  // SCORES: the piece's first type; INPUT: of w's rows
  // LOGITS: states [run and share][row]; SCORES: g (parts, rows, pitch); INPUT, WEIGHT: results, or partial ones [slot][row][pitch]
  void* out;
  int64_t out_pitch, out_part;
  int whole, typed;                                      // typed: results of the tensors' type, else float32 partial ones
  const float* before;                                   // INPUT: the sums of the pieces before this one, NULL for the first
  int64_t before_pitch, before_part;
  const int64_t* target;
  int64_t types;
  float* target_logit;
  const float *lse, *grad, *count;
  int reduction;
  int* status;
};

__host__ __device__ inline int shares_of(int width, int share) { return (width + share - 1) / share; }

struct Item {
  int64_t row;
  int tile0, tile1, part, kb0, kb1;                      // column tiles
};
template <int MODE> __device__ __forceinline__ Item item_of(const Launch& p, unsigned i) {
  Item t{};
  t.kb1 = p.kblocks;
  if (MODE == LOGITS || MODE == SCORES) {                // rows first: SMs share the tiles of w
    t.row = (int64_t)(i % (unsigned)p.row_tiles) * TILE_M;
    t.tile0 = (int)(i / (unsigned)p.row_tiles) * p.run;
    t.tile1 = min(p.col_tiles, t.tile0 + p.run);
    return t;
  }
  t.tile0 = (int)(i % (unsigned)p.col_tiles);            // columns first: SMs share the tiles of G
  t.tile1 = t.tile0 + 1;
  i /= (unsigned)p.col_tiles;
  t.row = (int64_t)(i % (unsigned)p.row_tiles) * TILE_M;
  t.part = (int)(i / (unsigned)p.row_tiles);
  t.kb0 = t.part * p.part_blocks;
  t.kb1 = min(p.kblocks, t.kb0 + p.part_blocks);
  return t;
}

// x as bfloat16 parts: what the first leaves is in the second, what these leave in the third
__device__ __forceinline__ void split3(float x, float& a, float& b, float& c) {
  a = __bfloat162float(__float2bfloat16_rn(x));
  b = __bfloat162float(__float2bfloat16_rn(x - a));
  c = (x - a) - b;
}

// 32 rows of a warp, 64 bytes of each: 16 bytes a piece, permuted so that eight lanes' rows, and the rows that eight lanes copy, fall on all banks.
__device__ __forceinline__ uint4* patch_at(unsigned char* patch, int row, int piece) {
  return reinterpret_cast<uint4*>(patch + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}
// A warp's 32 rows by 64 / sizeof(T) columns, a lane a row, to `out` (row 0, first column); `valid` columns and `lines` rows exist.
template <typename T> __device__ __forceinline__ void store_block(unsigned char* patch, const float* v, T* out, int64_t pitch, int lines, int valid, bool whole, int lane) {
  constexpr int N = 64 / (int)sizeof(T), V = 16 / (int)sizeof(T);
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 u;
    if constexpr (sizeof(T) == 4) u = make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
    else u = make_uint4(two_bf16(v[8 * q], v[8 * q + 1]), two_bf16(v[8 * q + 2], v[8 * q + 3]), two_bf16(v[8 * q + 4], v[8 * q + 5]), two_bf16(v[8 * q + 6], v[8 * q + 7]));
    *patch_at(patch, lane, q) = u;
  }
  __syncwarp();
  if (whole) {
    const int piece = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 8 + (lane >> 2);
      if (row < lines && piece * V < valid) *reinterpret_cast<uint4*>(out + row * pitch + piece * V) = *patch_at(patch, row, piece);
    }
  } else {
    const int column = lane % N, step = 32 / N;
#pragma unroll 4
    for (int row = lane / N; row < lines; row += step)
      if (column < valid) out[row * pitch + column] = reinterpret_cast<const T*>(patch_at(patch, row, column / V))[column % V];
  }
}

// PLANES: parts of G that SCORES makes of bfloat16
template <int PARTS, int MODE, int PLANES> __global__ void __launch_bounds__(threads<PARTS>(), 1) loss_kernel(const __grid_constant__ Launch p) {
  constexpr bool F32 = PARTS == 3, A_TURNED = MODE == WEIGHT, B_TURNED = MODE == INPUT || MODE == WEIGHT;
  constexpr int STAGES = stages<PARTS>(), STAGE = stage_bytes<PARTS>(), COLS = cols<PARTS>();
  static_assert(STAGES >= 2, "two stages at least");
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      bar_init(&full[s], 1);
      bar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      bar_init(&acc_full[a], 1);
      bar_init(&acc_empty[a], epilogue_warps<PARTS>());
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* ab = &abort_flag;

  if (warp == 0) {
    // ---------------- copies ----------------
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 1;
      bool ok = true;
      const uint32_t bytes = (uint32_t)(a_bytes<PARTS>() + PARTS * p.width * BK * 2);
      for (unsigned i = blockIdx.x; i < p.items && ok && !*ab; i += gridDim.x) {
        const Item t = item_of<MODE>(p, i);
        for (int tile = t.tile0; tile < t.tile1 && ok; ++tile) {
          const int col = tile * p.width;
          for (int kb = t.kb0; kb < t.kb1; ++kb) {
            if (!bar_wait(&empty[s], ph, ab)) { ok = false; break; }
            const int plane = (MODE == INPUT || MODE == WEIGHT) && kb >= p.plane_blocks, k = (kb - plane * p.plane_blocks) * BK;
            unsigned char* at = ring + (size_t)s * STAGE;
            bar_expect_tx(&full[s], bytes);
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
              unsigned char *sa = at + q * TILE_M * BK * 2, *sb = at + a_bytes<PARTS>() + q * COLS * BK * 2;
              if (A_TURNED) {
                tma_load_3d(sa, &p.a, (int)t.row, k, q + plane, &full[s]);
                tma_load_3d(sa + 8192, &p.a, (int)t.row + 64, k, q + plane, &full[s]);
              } else {
                tma_load_3d(sa, &p.a, k, (int)t.row, q + plane, &full[s]);
              }
              if (B_TURNED) {
                for (int c = 0; c < p.width / 64; ++c) tma_load_3d(sb + c * 8192, &p.b, col + c * 64, p.b_first + k, q, &full[s]);
              } else {
                tma_load_3d(sb, &p.b, k, p.b_first + col, q, &full[s]);
              }
            }
            if (++s == STAGES) s = 0, ph ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMAs ----------------
    if (lane == 0) {
      int s = 0, piece = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t idesc = idesc_bf16(TILE_M, p.width, A_TURNED, B_TURNED);
      constexpr uint32_t A_STEP = A_TURNED ? ROWS_STEP : K_STEP, B_STEP = B_TURNED ? ROWS_STEP : K_STEP;
      for (unsigned i = blockIdx.x; i < p.items && ok && !*ab; i += gridDim.x) {
        const Item t = item_of<MODE>(p, i);
        for (int tile = t.tile0; tile < t.tile1 && ok; ++tile) {
          for (int k0 = t.kb0; k0 < t.kb1 && ok; k0 += p.fold, ++piece) {
            const int k1 = min(k0 + p.fold, t.kb1), a = piece & 1;
            if (!bar_wait(&acc_empty[a], (uint32_t)(((piece >> 1) & 1) ^ 1), ab)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(a * 256);
            for (int kb = k0; kb < k1; ++kb) {
              if (!bar_wait(&full[s], ph, ab)) { ok = false; break; }
              tc_fence_after();
              const uint32_t at = s32(ring + (size_t)s * STAGE), bt = at + a_bytes<PARTS>();
              const uint32_t a_lo = A_TURNED ? umma_lo_rows(at, 8192) : umma_lo(at), b_lo = B_TURNED ? umma_lo_rows(bt, 8192) : umma_lo(bt);
              constexpr uint32_t A_PART = TILE_M * BK * 2 / 16, B_PART = COLS * BK * 2 / 16;
              auto parts_of = [&](int q, auto first) {
                constexpr bool MORE = !decltype(first)::value;
                const uint32_t an = a_lo + q * A_STEP, bn = b_lo + q * B_STEP;
                umma_bf16<MORE>(d, an, bn, idesc);
                if constexpr (F32) {
                  umma_bf16<MORE>(d + COLS, an, bn + 2 * B_PART, idesc);
                  umma_bf16<true>(d + COLS, an + 2 * A_PART, bn, idesc);
                  umma_bf16<true>(d + COLS, an + A_PART, bn + B_PART, idesc);
                  umma_bf16<true>(d + COLS, an, bn + B_PART, idesc);
                  umma_bf16<true>(d + COLS, an + A_PART, bn, idesc);
                }
              };
              if (kb == k0) parts_of(0, std::true_type());
              else parts_of(0, std::false_type());
#pragma unroll
              for (int q = 1; q < 4; ++q) parts_of(q, std::false_type());
              umma_commit(&empty[s]);
              if (++s == STAGES) s = 0, ph ^= 1;
            }
            if (ok) umma_commit(&acc_full[a]);
          }
        }
      }
    }
  } else {
    // ---------------- epilogue ----------------
    // Warps of the same quarter of the lanes have a share of a tile's columns each, 32 at a time.
    constexpr int SHARE = share<PARTS>();
    const int e = warp - 2, quarter = warp & 3, part_of = e >> 2;
    unsigned char* patch = ring + (size_t)STAGES * STAGE + (size_t)e * PATCH;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(part_of * SHARE);
    const int mine = max(0, min(SHARE, p.width - part_of * SHARE));                         // columns of a narrow tile may be none
    int piece = 0;
    bool ok = true;
    for (unsigned i = blockIdx.x; i < p.items && ok && !*ab; i += gridDim.x) {
      const Item t = item_of<MODE>(p, i);
      const int64_t row0 = t.row + quarter * 32, row = row0 + lane;
      const int lines = (int)max((int64_t)0, min((int64_t)32, p.rows - row0));
      const bool there = row < p.rows;
      int64_t target = -1;
      float top = -INFINITY, sum = 0.f, lse = 0.f, part = 0.f;
      if (MODE != WEIGHT && there) target = p.target[row];
      if (MODE == SCORES && target >= 0) {
        lse = p.lse[row];
        part = p.reduction == 0 ? p.grad[row] : 1.f;
        if (target >= p.types) part = NAN;
      }
      float factor = 1.f;
      if (MODE == INPUT || MODE == WEIGHT) factor = p.reduction == 0 ? 1.f : p.reduction == 1 ? p.grad[0] : p.count[0] > 0.f ? p.grad[0] / p.count[0] : 0.f;
      // 32 columns from `col` on, of which `valid` exist
      auto block = [&](float* v, int col, int valid) {
        if constexpr (MODE == LOGITS) {
          if (valid < 32) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = c < valid ? v[c] : -INFINITY;
          }
          const int64_t at = target - col;
          if (at >= 0 && at < min(valid, 32)) {
            float z = 0.f;
#pragma unroll
            for (int c = 0; c < 32; ++c) z = c == (int)at ? v[c] : z;
            p.target_logit[row] = z;
          }
          float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 32; ++c) most[c & 3] = fmaxf(most[c & 3], v[c]);
          // The unit of the sum is the rounded product, so a sum whose unit stays is multiplied by one: with the greatest logit as the unit it was by what the
          // product's rounding left, every 32 columns in the same direction (greatest logit 100 of 32,768: the loss 2.7e-4 off).
          const float now = fmaxf(top, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * LOG2E), base = now == -INFINITY ? 0.f : now;
#pragma unroll
          for (int c = 0; c < 32; ++c) add[c & 3] += exp2_fast(fmaf(v[c], LOG2E, -base));
          sum = sum * exp2_fast(top - base) + ((add[0] + add[1]) + (add[2] + add[3]));
          top = now;
        } else if constexpr (MODE == SCORES) {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = part * exp2_fast(fmaf(v[c], LOG2E, -lse));
          if (__any_sync(0xffffffffu, target < 0)) {     // set, whatever the product
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = target < 0 ? 0.f : v[c];
          }
          const int64_t at = target - p.a_first - col;
          if (at >= 0 && at < min(valid, 32)) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = c == (int)at ? v[c] - part : v[c];
          }
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + row0 * p.out_pitch + col;
#pragma unroll
          for (int q = 0; q < PARTS * PLANES; ++q) {
            store_block<__nv_bfloat16>(patch, v, out + q * p.out_part, p.out_pitch, lines, valid, true, lane);
            if constexpr (PARTS * PLANES > 1) {
#pragma unroll
              for (int c = 0; c < 32; ++c) v[c] -= __bfloat162float(__float2bfloat16_rn(v[c]));
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] *= factor;
          if (MODE == INPUT && p.before && there) {      // the place may be the one that is written: store_block has a warp's barrier before it
            const float* from = p.before + t.part * p.before_part + row * p.before_pitch + col;
#pragma unroll
            for (int c = 0; c < 32; c += 4)
              if (col + c < p.before_pitch) {
                const float4 a = *reinterpret_cast<const float4*>(from + c);
                v[c] += a.x, v[c + 1] += a.y, v[c + 2] += a.z, v[c + 3] += a.w;
              }
          }
          if (MODE == INPUT && p.typed && target < 0) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = 0.f;
          }
          if (F32 || !p.typed) {
            float* out = static_cast<float*>(p.out) + (p.typed ? 0 : t.part * p.out_part) + row0 * p.out_pitch + col;
            store_block<float>(patch, v, out, p.out_pitch, lines, valid, p.whole, lane);
            store_block<float>(patch, v + 16, out + 16, p.out_pitch, lines, valid - 16, p.whole, lane);
          } else {
            store_block<__nv_bfloat16>(patch, v, static_cast<__nv_bfloat16*>(p.out) + row0 * p.out_pitch + col, p.out_pitch, lines, valid, p.whole, lane);
          }
        }
      };
      for (int tile = t.tile0; tile < t.tile1 && ok; ++tile) {
        const int col = tile * p.width + part_of * SHARE, valid = min(p.columns, (tile + 1) * p.width) - col;
        auto release = [&](int a) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(&acc_empty[a]);
        };
        if constexpr (F32) {                             // pieces of the sum, of two sums each, gather in registers
          float v[SHARE];
          for (int k0 = t.kb0; k0 < t.kb1; k0 += p.fold, ++piece) {
            const int a = piece & 1;
            if (!bar_wait(&acc_full[a], (uint32_t)((piece >> 1) & 1), ab)) { ok = false; break; }
            tc_fence_after();
            if (mine) {
#pragma unroll
              for (int h = 0; h < SHARE; h += 32) {
                uint32_t r[32];
                tmem_issue32(lanes + (uint32_t)(a * 256 + h), r);
                tmem_arrived32(r);
#pragma unroll
                for (int c = 0; c < 32; ++c) v[h + c] = k0 > t.kb0 ? v[h + c] + __uint_as_float(r[c]) : __uint_as_float(r[c]);
                tmem_issue32(lanes + (uint32_t)(a * 256 + COLS + h), r);
                tmem_arrived32(r);
#pragma unroll
                for (int c = 0; c < 32; ++c) v[h + c] += __uint_as_float(r[c]);
              }
            }
            release(a);
          }
          if (!ok) break;
          if (mine) {
#pragma unroll
            for (int h = 0; h < SHARE; h += 32) block(v + h, col + h, valid - h);
          }
        } else {                                         // one sum; the next columns are on their way while these are worked on
          const int a = piece & 1;
          if (!bar_wait(&acc_full[a], (uint32_t)((piece >> 1) & 1), ab)) { ok = false; break; }
          ++piece;
          tc_fence_after();
          uint32_t r[2][32];
          if (mine) {
            tmem_issue32(lanes + (uint32_t)(a * 256), r[0]);
#pragma unroll
            for (int h = 0; h < SHARE; h += 32) {
              if (h >= mine) break;
              uint32_t(&now)[32] = r[(h / 32) & 1];
              tmem_arrived32(now);
              if (h + 32 < mine) tmem_issue32(lanes + (uint32_t)(a * 256 + h + 32), r[(h / 32 + 1) & 1]);
              else release(a);
              float v[32];
#pragma unroll
              for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(now[c]);
              block(v, col + h, valid - h);
            }
          } else {
            release(a);
          }
        }
      }
      if (MODE == LOGITS && ok && there && mine)
        static_cast<float2*>(p.out)[(int64_t)(t.tile0 / p.run * shares_of(p.width, SHARE) + part_of) * p.rows + row] = make_float2(top, sum);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && abort_flag) {
    atomicExch(p.status, 2);
    let_copies_land(full, STAGES);
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---- before and after ---------------------------------------------------------------------------
// Matrices (rows, cols) to rows of `pitch` bfloat16 values, in three parts of float32 ones; rows whose target is negative as zeros.  Two at once.
struct Prepare {
  const void* from;
  __nv_bfloat16* to;
  int64_t rows;
  const int64_t* target;
};
template <typename T> __global__ void __launch_bounds__(256) prepare_kernel(const Prepare first, const Prepare second, int cols, int pitch) {
  const Prepare& p = blockIdx.y ? second : first;
  const int64_t part = p.rows * pitch;
  const unsigned pieces = pitch / 8;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < p.rows * pieces; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i <= UINT32_MAX ? (unsigned)i / pieces : i / pieces;
    const int col = (int)(i - row * pieces) * 8;
    const bool none = p.target && p.target[row] < 0;
    const T* from = static_cast<const T*>(p.from) + row * cols + col;
    float v[8], w[8], u[8];
    if (cols % 8 == 0) {
      if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        const uint4 a = *reinterpret_cast<const uint4*>(from);
        const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(r[j] << 16), v[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = col + j < cols ? ld(from + j) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (none) v[j] = 0.f;
      if constexpr (sizeof(T) == 4) split3(v[j], v[j], w[j], u[j]);
    }
    auto put = [&](const float (&x)[8], int q) {
      *reinterpret_cast<uint4*>(p.to + q * part + row * pitch + col) = make_uint4(two_bf16(x[0], x[1]), two_bf16(x[2], x[3]), two_bf16(x[4], x[5]), two_bf16(x[6], x[7]));
    };
    put(v, 0);
    if constexpr (sizeof(T) == 4) {
      put(w, 1);
      put(u, 2);
    }
  }
}

// The rows' log sums, in units of log2, and losses from the states of their runs: eight threads a row.  The logits of all of them were multiplied by the float32
// LOG2E, so the target's is as well, and the difference is formed where it is exact.
__global__ void __launch_bounds__(256) rows_kernel(const float2* __restrict__ states, int count, const float* __restrict__ target_logit,
                                                   const int64_t* __restrict__ target, int64_t n, int64_t types, float* __restrict__ lse, float* __restrict__ losses) {
  __shared__ float2 shared[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x * (int64_t)32 + lane;
  float top = -INFINITY, sum = 0.f;
  auto join = [&](float2 s) {
    const float now = fmaxf(top, s.x), base = now == -INFINITY ? 0.f : now;
    sum = sum * exp2_fast(top - base) + s.y * exp2_fast(s.x - base);
    top = now;
  };
  if (row < n)
    for (int i = warp; i < count; i += 8) join(states[i * n + row]);
  shared[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp || row >= n) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) join(shared[w][lane]);
  const double more = log2((double)sum);
  lse[row] = (float)((double)top + more);
  const int64_t t = target[row];
  losses[row] = t < 0 ? 0.f : t >= types ? NAN : (float)((((double)top - (double)target_logit[row] * (double)LOG2E) + more) * 0.693147180559945309);
}
__global__ void __launch_bounds__(1024) reduce_kernel(const float* __restrict__ losses, const int64_t* __restrict__ target, int64_t n, int mean, float* result,
                                                      float* count) {
  __shared__ double sums[32];
  __shared__ int64_t counts[32];
  double sum = 0.0;
  int64_t c = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    sum += losses[i];
    c += target[i] >= 0;
  }
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum, counts[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 32; ++w) sum += sums[w], c += counts[w];
  count[0] = (float)c;
  if (result) result[0] = (float)(mean ? sum / (double)(c ? c : 1) : sum);
}

// Partial results [slots][rows][pitch] added in their order, eight columns a thread; rows of a negative target are zeros.
template <typename T> __global__ void __launch_bounds__(256) sum_kernel(const float* __restrict__ parts, T* __restrict__ out, int64_t rows, int cols, int pitch, int slots,
                                                                        const int64_t* __restrict__ target) {
  const int64_t part = rows * pitch;
  const unsigned pieces = pitch / 8;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < rows * pieces; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i <= UINT32_MAX ? (unsigned)i / pieces : i / pieces;
    const int col = (int)(i - row * pieces) * 8;
    const float4* from = reinterpret_cast<const float4*>(parts + row * pitch + col);
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < slots; ++s) {
      const float4 a = from[s * (part / 4)], b = from[s * (part / 4) + 1];
      sum[0] += a.x, sum[1] += a.y, sum[2] += a.z, sum[3] += a.w, sum[4] += b.x, sum[5] += b.y, sum[6] += b.z, sum[7] += b.w;
    }
    if (target && target[row] < 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] = 0.f;
    }
    T* to = out + row * cols + col;
    if (cols % 8 == 0) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(to)[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
        reinterpret_cast<float4*>(to)[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
      } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(two_bf16(sum[0], sum[1]), two_bf16(sum[2], sum[3]), two_bf16(sum[4], sum[5]), two_bf16(sum[6], sum[7]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < cols) st(to + j, sum[j]);
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------
int size_of(int dtype) { return dtype == EQT_F32 ? 4 : 2; }
size_t up(size_t b) { return (b + 1023) / 1024 * 1024; }
int64_t up_to(int64_t v, int64_t m) { return ceil_div(v, m) * m; }

struct Plan {
  int parts, pitch, cols;                                // of the operands: bfloat16 parts, values a row; columns a tile
  int64_t piece, pieces, g_pitch;
  int width_t, width_c, run, runs;
  int planes, input_parts, input_blocks, weight_parts, weight_blocks;
  size_t x, w, states, logit, g, dx, dw, bytes;          // places in the scratch
};
int width_of(int64_t columns, int most) {
  const int64_t tiles = ceil_div(columns, most);
  return (int)up_to(ceil_div(columns, tiles), 64);
}
// Parts of a sum of `blocks` k-blocks for `tiles` results: as many as fill the SMs, of at least eight blocks, and at most MOST_TERMS.
void cut(int64_t blocks, int64_t tiles, int& parts, int& part_blocks) {
  const int64_t wanted = std::max<int64_t>(1, sm_count() / std::max<int64_t>(1, tiles));
  part_blocks = (int)std::min<int64_t>(MOST_TERMS / BK, std::max<int64_t>(std::min<int64_t>(blocks, 8), ceil_div(blocks, wanted)));
  parts = (int)ceil_div(blocks, part_blocks);
}
// bfloat16 G of few types goes into its products in two parts: a row's few numbers are often of one size, whose rounding does not average out (1000 rows, 2 to
// 10 types: 2-norm of dx's error 2.15e-3 in one part, 1.65e-3 in two, that of a result's rounding); up to 64 types are one k-block a part, so it costs a few microseconds.
int planes_of(const eqt_type_loss_args& a) { return a.dtype == EQT_BF16 && a.t <= BK ? 2 : 1; }
Plan plan_of(const eqt_type_loss_args& a, bool backward) {
  Plan p{};
  const int64_t sms = sm_count(), row_tiles = ceil_div(a.n, TILE_M);
  const bool f32 = a.dtype == EQT_F32;
  p.parts = f32 ? 3 : 1;
  p.cols = f32 ? cols<3>() : cols<1>();
  p.pitch = (int)up_to(a.c, 8);
  p.width_t = width_of(a.t, p.cols);
  p.width_c = width_of(a.c, p.cols);
  const bool copy_x = f32 || backward || p.pitch != a.c, copy_w = f32 || p.pitch != a.c;
  p.w = copy_x ? up((size_t)a.n * p.pitch * 2 * p.parts) : 0;
  size_t at = p.w + (copy_w ? up((size_t)a.t * p.pitch * 2 * p.parts) : 0);
  if (!backward) {
    const int64_t col_tiles = ceil_div(a.t, p.width_t);
    p.run = (int)std::min<int64_t>(32, std::max<int64_t>(1, row_tiles * col_tiles / (sms * 8)));
    p.runs = (int)ceil_div(col_tiles, p.run);
    p.states = at;
    p.logit = p.states + up((size_t)p.runs * shares_of(p.width_t, p.parts == 1 ? share<1>() : share<3>()) * a.n * sizeof(float2));
    p.bytes = p.logit + up((size_t)a.n * 4);
    return p;
  }
  // a piece: whole waves of WEIGHT's tiles, as many as the scratch for G takes
  const int64_t col_tiles = ceil_div(a.c, p.width_c), wave = std::max<int64_t>(1, sms / col_tiles) * TILE_M;
  p.planes = planes_of(a);
  const int64_t most = std::max<int64_t>(TILE_M, PIECE_BYTES / (2 * p.parts) / up_to(a.n, TILE_M) / TILE_M * TILE_M);
  p.piece = std::min<int64_t>(up_to(a.t, TILE_M), most >= wave ? most / wave * wave : most);
  p.pieces = ceil_div(a.t, p.piece);
  p.g_pitch = p.piece;
  cut(p.planes * ceil_div(std::min<int64_t>(p.piece, a.t), BK), row_tiles * col_tiles, p.input_parts, p.input_blocks);
  cut(p.planes * ceil_div(a.n, BK), ceil_div(p.piece, TILE_M) * col_tiles, p.weight_parts, p.weight_blocks);
  p.g = at;
  p.dx = p.g + up((size_t)a.n * p.g_pitch * 2 * p.parts * p.planes);
  p.dw = p.dx + (a.dx && (p.input_parts > 1 || p.pieces > 1) ? up((size_t)p.input_parts * a.n * p.pitch * 4) : 0);
  p.bytes = p.dw + (a.dw && p.weight_parts > 1 ? up((size_t)p.weight_parts * p.piece * p.pitch * 4) : 0);
  return p;
}

int check(const eqt_type_loss_args* a) {
  if (!a) return fail(EQT_ERR_BAD_ARGUMENT, "type_loss: NULL pointer");
  if (a->dtype != EQT_F32 && a->dtype != EQT_BF16) return fail(EQT_ERR_BAD_ARGUMENT, "type_loss: unknown dtype %d", a->dtype);
  if (a->reduction < 0 || a->reduction > 2) return fail(EQT_ERR_BAD_ARGUMENT, "type_loss: unknown reduction %d", a->reduction);
  if (a->n < 0 || a->c < 1 || a->t < 1) return fail(EQT_ERR_BAD_ARGUMENT, "type_loss: sizes");
  if (a->n > INT32_MAX - 256 || a->t > INT32_MAX - 256 || a->c > MOST_TERMS) return fail(EQT_ERR_UNSUPPORTED, "type_loss: at most 2^31 rows and types and 16384 channels");
  if (ceil_div(a->n, TILE_M) * ceil_div(a->t, 64) > INT32_MAX / 2) return fail(EQT_ERR_UNSUPPORTED, "type_loss: rows times types are more than one launch takes");
  return EQT_OK;
}

template <int PARTS, int MODE, int PLANES = 1> int launch(const Launch& p, cudaStream_t s) {
  auto kernel = loss_kernel<PARTS, MODE, PLANES>;
  static std::atomic<uint64_t> allowed{0};
  if (int rc = allow_shared_once(kernel, shared_bytes<PARTS>(), allowed)) return rc;
  kernel<<<std::min<unsigned>(p.items, (unsigned)sm_count()), threads<PARTS>(), shared_bytes<PARTS>(), s>>>(p);
  return check_launch("type_loss");
}
template <int MODE> int launch(int parts, const Launch& p, cudaStream_t s) {
  if constexpr (MODE == SCORES)
    if (parts == 1 && p.planes == 2) return launch<1, MODE, 2>(p, s);
  return parts == 1 ? launch<1, MODE>(p, s) : launch<3, MODE>(p, s);
}

int sum_parts(int dtype, const float* parts, void* out, int64_t rows, int cols, int pitch, int slots, const int64_t* target, cudaStream_t s) {
  const unsigned grid = flat_grid(rows * (pitch / 8), 256);
  if (dtype == EQT_F32) sum_kernel<<<grid, 256, 0, s>>>(parts, static_cast<float*>(out), rows, cols, pitch, slots, target);
  else sum_kernel<<<grid, 256, 0, s>>>(parts, static_cast<__nv_bfloat16*>(out), rows, cols, pitch, slots, target);
  return check_launch("type_loss_sum");
}

// Operands ready for the copies of tiles: as they are, or from the scratch.
int operands(const eqt_type_loss_args& a, const Plan& p, bool backward, const void*& x, const void*& w, cudaStream_t s) {
  unsigned char* base = static_cast<unsigned char*>(a.scratch);
  x = a.x, w = a.w;
  Prepare jobs[2];
  int count = 0;
  if (p.w) {
    jobs[count++] = {a.x, reinterpret_cast<__nv_bfloat16*>(base + p.x), a.n, backward ? a.target : nullptr};
    x = base + p.x;
  }
  if (p.parts > 1 || p.pitch != a.c) {
    jobs[count++] = {a.w, reinterpret_cast<__nv_bfloat16*>(base + p.w), a.t, nullptr};
    w = base + p.w;
  }
  if (!count) return EQT_OK;
  const dim3 grid(flat_grid(std::max(jobs[0].rows, jobs[count - 1].rows) * (p.pitch / 8), 256), (unsigned)count);
  if (a.dtype == EQT_F32) prepare_kernel<float><<<grid, 256, 0, s>>>(jobs[0], jobs[count - 1], (int)a.c, p.pitch);
  else prepare_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(jobs[0], jobs[count - 1], (int)a.c, p.pitch);
  return check_launch("type_loss_prepare");
}

int check_pointers(const eqt_type_loss_args& a, size_t need) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.scratch) | reinterpret_cast<uintptr_t>(a.dx) |
                   reinterpret_cast<uintptr_t>(a.dw);
  if (bits % 16) return fail(EQT_ERR_BAD_ARGUMENT, "type_loss: operands must start on 16-byte boundaries");
  if (a.scratch_bytes < (int64_t)need || !a.scratch)
    return fail(EQT_ERR_BAD_ARGUMENT, "type_loss: %lld bytes of scratch given, %lld needed", (long long)a.scratch_bytes, (long long)need);
  return EQT_OK;
}

constexpr int fold_of(int parts) { return parts == 3 ? 8 : (int)(MOST_TERMS / BK); }

}  // namespace
}  // namespace type_loss
}  // namespace eqt

using namespace eqt;
using namespace eqt::type_loss;

extern "C" int64_t eqt_type_loss_scratch(const eqt_type_loss_args* a, int32_t backward) {
  if (check(a) || a->n == 0) return 0;
  return (int64_t)plan_of(*a, backward != 0).bytes;
}

extern "C" int eqt_type_loss_forward(const eqt_type_loss_args* args, void* stream) {
  if (int rc = check(args)) return rc;
  const eqt_type_loss_args& a = *args;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!a.count || (a.reduction && !a.result)) return fail(EQT_ERR_BAD_ARGUMENT, "type_loss: NULL pointer");
  if (a.n) {
    if (!a.x || !a.w || !a.target || !a.losses || !a.lse || !a.status) return fail(EQT_ERR_BAD_ARGUMENT, "type_loss: NULL pointer");
    const Plan p = plan_of(a, false);
    if (int rc = check_pointers(a, p.bytes)) return rc;
    const void *x, *w;
    if (int rc = operands(a, p, false, x, w, s)) return rc;
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    Launch l{};
    if (int rc = tc::map_bf16(&l.a, x, a.n, p.pitch, p.pitch, a.n * p.pitch, p.parts, tc::TILE_M)) return rc;
    if (int rc = tc::map_bf16(&l.b, w, a.t, p.pitch, p.pitch, a.t * p.pitch, p.parts, p.width_t)) return rc;
    l.rows = a.n, l.columns = (int)a.t, l.width = p.width_t, l.row_tiles = (int)ceil_div(a.n, tc::TILE_M), l.col_tiles = (int)ceil_div(a.t, p.width_t);
    l.run = p.run, l.kblocks = (int)ceil_div(a.c, BK), l.fold = fold_of(p.parts), l.items = (unsigned)(l.row_tiles * p.runs);
    l.out = base + p.states, l.target = a.target, l.types = a.t, l.target_logit = reinterpret_cast<float*>(base + p.logit), l.status = a.status;
    if (int rc = launch<LOGITS>(p.parts, l, s)) return rc;
    rows_kernel<<<(unsigned)ceil_div(a.n, 32), 256, 0, s>>>(reinterpret_cast<const float2*>(base + p.states), p.runs * shares_of(p.width_t, p.parts == 1 ? share<1>() : share<3>()), l.target_logit, a.target, a.n,
                                                            a.t, a.lse, a.losses);
    if (int rc = check_launch("type_loss_rows")) return rc;
  }
  reduce_kernel<<<1, 1024, 0, s>>>(a.losses, a.target, a.n, a.reduction == 2, a.reduction ? a.result : nullptr, a.count);
  return check_launch("type_loss_reduce");
}

extern "C" int eqt_type_loss_backward(const eqt_type_loss_args* args, void* stream) {
  if (int rc = check(args)) return rc;
  const eqt_type_loss_args& a = *args;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.n == 0) {
    if (a.dw && cudaMemsetAsync(a.dw, 0, (size_t)a.t * a.c * size_of(a.dtype), s) != cudaSuccess) return fail(EQT_ERR_CUDA, "cudaMemsetAsync failed");
    return EQT_OK;
  }
  if (!a.x || !a.w || !a.target || !a.lse || !a.grad || !a.status || (a.reduction == 2 && !a.count)) return fail(EQT_ERR_BAD_ARGUMENT, "type_loss backward: NULL pointer");
  if (!a.dx && !a.dw) return EQT_OK;
  const Plan p = plan_of(a, true);
  if (int rc = check_pointers(a, p.bytes)) return rc;
  const void *x, *w;
  if (int rc = operands(a, p, true, x, w, s)) return rc;
  unsigned char* base = static_cast<unsigned char*>(a.scratch);
  float *dx_parts = reinterpret_cast<float*>(base + p.dx), *dw_parts = reinterpret_cast<float*>(base + p.dw);
  const int size = size_of(a.dtype);
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t t0 = i * p.piece, here = std::min<int64_t>(p.piece, a.t - t0);
    Launch l{};
    if (int rc = tc::map_bf16(&l.a, x, a.n, p.pitch, p.pitch, a.n * p.pitch, p.parts, tc::TILE_M)) return rc;
    if (int rc = tc::map_bf16(&l.b, w, a.t, p.pitch, p.pitch, a.t * p.pitch, p.parts, p.width_t)) return rc;
    l.rows = a.n, l.columns = (int)here, l.width = p.width_t, l.row_tiles = (int)ceil_div(a.n, tc::TILE_M), l.col_tiles = (int)ceil_div(here, p.width_t);
    l.run = 1, l.kblocks = (int)ceil_div(a.c, BK), l.fold = fold_of(p.parts), l.items = (unsigned)(l.row_tiles * l.col_tiles);
    l.planes = p.planes, l.a_first = l.b_first = (int)t0, l.out = base + p.g, l.out_pitch = p.g_pitch, l.out_part = a.n * p.g_pitch;
    l.target = a.target, l.types = a.t, l.lse = a.lse, l.grad = a.grad, l.count = a.count, l.reduction = a.reduction, l.status = a.status;
    if (int rc = launch<SCORES>(p.parts, l, s)) return rc;
    if (a.dx) {
      Launch d{};
      if (int rc = tc::map_bf16(&d.a, base + p.g, a.n, here, p.g_pitch, a.n * p.g_pitch, p.parts * p.planes, tc::TILE_M)) return rc;
      if (int rc = tc::map_bf16(&d.b, w, a.t, p.pitch, p.pitch, a.t * p.pitch, p.parts, BK)) return rc;
      d.rows = a.n, d.columns = (int)a.c, d.width = p.width_c, d.row_tiles = l.row_tiles, d.col_tiles = (int)ceil_div(a.c, p.width_c);
      d.plane_blocks = (int)ceil_div(here, BK), d.kblocks = p.planes * d.plane_blocks, d.part_blocks = p.input_blocks, d.fold = l.fold;
      d.items = (unsigned)(d.row_tiles * d.col_tiles * ceil_div(d.kblocks, d.part_blocks));                 // a short last piece adds to the first parts only
      d.b_first = (int)t0, d.typed = p.input_parts == 1 && i == p.pieces - 1, d.target = a.target, d.types = a.t, d.status = a.status;
      d.grad = a.grad, d.count = a.count, d.reduction = a.reduction;
      d.out = d.typed ? a.dx : dx_parts, d.out_pitch = d.typed ? a.c : p.pitch, d.out_part = a.n * p.pitch;
      d.before = i ? dx_parts : nullptr, d.before_pitch = p.pitch, d.before_part = a.n * p.pitch;
      d.whole = !d.typed || a.c * size % 16 == 0;
      if (int rc = launch<INPUT>(p.parts, d, s)) return rc;
    }
    if (a.dw) {
      Launch d{};
      if (int rc = tc::map_bf16(&d.a, base + p.g, a.n, here, p.g_pitch, a.n * p.g_pitch, p.parts * p.planes, BK)) return rc;
      if (int rc = tc::map_bf16(&d.b, x, a.n, p.pitch, p.pitch, a.n * p.pitch, p.parts, BK)) return rc;
      d.rows = here, d.columns = (int)a.c, d.width = p.width_c, d.row_tiles = (int)ceil_div(here, tc::TILE_M), d.col_tiles = (int)ceil_div(a.c, p.width_c);
      d.plane_blocks = (int)ceil_div(a.n, BK), d.kblocks = p.planes * d.plane_blocks, d.part_blocks = p.weight_blocks, d.fold = l.fold, d.items = (unsigned)(d.row_tiles * d.col_tiles * p.weight_parts);
      d.typed = p.weight_parts == 1, d.status = a.status;
      d.grad = a.grad, d.count = a.count, d.reduction = a.reduction;
      void* to = static_cast<unsigned char*>(a.dw) + (size_t)t0 * a.c * size;
      d.out = d.typed ? to : dw_parts, d.out_pitch = d.typed ? a.c : p.pitch, d.out_part = here * p.pitch;
      d.whole = !d.typed || a.c * size % 16 == 0;
      if (int rc = launch<WEIGHT>(p.parts, d, s)) return rc;
      if (!d.typed)
        if (int rc = sum_parts(a.dtype, dw_parts, to, here, (int)a.c, p.pitch, p.weight_parts, nullptr, s)) return rc;
    }
  }
  if (a.dx && p.input_parts > 1) return sum_parts(a.dtype, dx_parts, a.dx, a.n, (int)a.c, p.pitch, p.input_parts, a.target, s);
  return EQT_OK;
}
