// Gated linear layer on the 5th-generation tensor cores: one kernel of warp roles for its four products.
//
//   FORWARD      [a | u] = x [W0 | W1]           epilogue h = act(a) u
//   PARTIALS     the same product                epilogue da, du from g
//   INPUT_GRAD   dx = [da | du] [W0 | W1]^T      one sum over both halves
//   WEIGHT_GRAD  dWj = x^T dj                    over parts of the rows, float32 partial results
//
// A CTA per SM strides through tiles of 128 rows; a k-block of 128 bytes a row (64 bfloat16, 32 float32) is a stage of the ring.
// Warp 0 copies tiles (TMA), warp 1 issues the MMAs, the last eight warps empty the accumulators while the next tile is multiplied;
// the dual products have both halves of the columns in one MMA, so the activation and the product never leave the SM.
//
// bfloat16: the MMA reads tiles as they lie in memory, along k or along the rows (both majors, 128-byte swizzle): 128 x 256 results
// a tile, four stages of 48 KB.
// float32: operands are split into TF32 pairs, three MMAs each, as everywhere in this library.  Four warps split a stage between the
// copy and the MMA, big parts in place; a tile that lies along the rows is turned on the way, 32 x 32 values a warp at a time, so the
// MMA always finds k along the row.  128 x 128 results a tile, three stages of 64 KB.  The adder of the tensor cores truncates, so a
// sum longer than 512 terms is taken in pieces that the epilogue adds with ordinary rounding.
//
// Every wait is bounded, as in the other tensor-core kernels; on expiry the status flag is raised and the kernel ends.
#include <algorithm>

#include "gated.cuh"

namespace eqt {
namespace gated {
namespace {
using namespace tc;

enum Mode { FORWARD, PARTIALS, INPUT_GRAD, WEIGHT_GRAD };

constexpr int EPI_WARPS = 8, PATCH = 32 * 128;           // bytes of a warp's patch: 32 rows of 128
constexpr int PIECE = 16;                                // k-blocks of a float32 piece

template <typename T> struct Form;
template <> struct Form<__nv_bfloat16> {
  static constexpr int BK = 64, STAGES = 4, COLS = 256, SPLITTERS = 0, A_BYTES = 16384, B_AT = 16384, STAGE = 49152;
};
template <> struct Form<float> {                         // A big, A small, B big, B small
  static constexpr int BK = 32, STAGES = 3, COLS = 128, SPLITTERS = 4, A_BYTES = 16384, B_AT = 32768, STAGE = 65536;
};
template <typename T> constexpr int threads() { return 32 * (2 + Form<T>::SPLITTERS + EPI_WARPS); }
template <typename T> constexpr size_t shared_bytes() { return 1024 + (size_t)Form<T>::STAGES * Form<T>::STAGE + EPI_WARPS * PATCH; }

struct alignas(64) Launch {
  CUtensorMap a[2], b[2];                                // WEIGHT_GRAD: a[0] x, b da and du; INPUT_GRAD: a da and du, b W0 and W1
  void *out, *out2;
  const void* g;
  int64_t rows, items, out_pitch;                        // rows and columns of the results
  int64_t part;                                          // WEIGHT_GRAD: results between two partial ones
  int cols, width;                                       // width: columns a tile (of each half, where there are two)
  int row_tiles, col_tiles, kblocks;                     // kblocks: of one half for INPUT_GRAD, of all rows for WEIGHT_GRAD
  int split_blocks;                                      // WEIGHT_GRAD: k-blocks a part
  int act;
  int* status;
};

// What tile a work item is.
struct Item {
  int64_t row;
  int col, half, part, kb0, kb1;
};
template <int MODE> __device__ __forceinline__ Item item_of(const Launch& p, int64_t i) {
  Item t{};
  t.col = (int)(i % p.col_tiles) * p.width;
  i /= p.col_tiles;
  t.row = (i % p.row_tiles) * TILE_M;
  t.kb1 = MODE == INPUT_GRAD ? 2 * p.kblocks : p.kblocks;
  if (MODE == WEIGHT_GRAD) {
    i /= p.row_tiles;
    t.half = (int)(i & 1);
    t.part = (int)(i >> 1);
    t.kb0 = t.part * p.split_blocks;
    t.kb1 = min(p.kblocks, t.kb0 + p.split_blocks);
  }
  return t;
}

__device__ __forceinline__ uint32_t idesc_bf16(int n, bool a_rows, bool b_rows) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_rows << 15) | ((uint32_t)b_rows << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(TILE_M >> 4) << 24);
}
// Along the rows (MN-major), 128-byte swizzle: 64 values of M or N a line, eight k a group of 1024 bytes, the next 64 values `BK` lines on.
__device__ __forceinline__ uint64_t desc_rows(uint32_t at) {
  return (uint64_t)((at & 0x3FFFF) >> 4) | ((uint64_t)((Form<__nv_bfloat16>::BK * 128) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
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

// 32 lines of up to 128 bytes between global memory and a warp's patch, line r at row r of `base`, pieces of 16 bytes; in the patch
// the pieces of a line are permuted so that a lane's line and four lines' pieces fall on all banks.
__device__ __forceinline__ uint4* patch_at(unsigned char* patch, int line, int piece) {
  return reinterpret_cast<uint4*>(patch + line * 128 + ((piece ^ (line & 7)) << 4));
}
__device__ __forceinline__ void patch_out(unsigned char* patch, unsigned char* base, int64_t pitch, int lines, int pieces, int lane) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int line = i * 4 + (lane >> 3), piece = lane & 7;
    if (line < lines && piece < pieces) *reinterpret_cast<uint4*>(base + line * pitch + piece * 16) = *patch_at(patch, line, piece);
  }
  __syncwarp();
}
__device__ __forceinline__ void patch_in(unsigned char* patch, const unsigned char* base, int64_t pitch, int lines, int pieces, int lane) {
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int line = i * 4 + (lane >> 3), piece = lane & 7;
    v[i] = line < lines && piece < pieces ? __ldg(reinterpret_cast<const uint4*>(base + line * pitch + piece * 16)) : make_uint4(0, 0, 0, 0);
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) *patch_at(patch, i * 4 + (lane >> 3), lane & 7) = v[i];
  __syncwarp();
}
// A lane's line: 32 values to or from the patch, for bfloat16 the first or second half of the line.
template <typename T> __device__ __forceinline__ void line_put(unsigned char* patch, int lane, int half, const float (&v)[32]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *patch_at(patch, lane, c) = make_uint4(__float_as_uint(v[4 * c]), __float_as_uint(v[4 * c + 1]), __float_as_uint(v[4 * c + 2]), __float_as_uint(v[4 * c + 3]));
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(v[8 * c + 2 * i], v[8 * c + 2 * i + 1]);
        r[i] = *reinterpret_cast<const uint32_t*>(&two);
      }
      *patch_at(patch, lane, half * 4 + c) = make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
}
template <typename T> __device__ __forceinline__ void line_get(unsigned char* patch, int lane, int half, float (&v)[32]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint4 u = *patch_at(patch, lane, c);
      v[4 * c] = __uint_as_float(u.x), v[4 * c + 1] = __uint_as_float(u.y), v[4 * c + 2] = __uint_as_float(u.z), v[4 * c + 3] = __uint_as_float(u.w);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 u = *patch_at(patch, lane, half * 4 + c);
      const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[8 * c + 2 * i] = __uint_as_float(r[i] << 16);
        v[8 * c + 2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
      }
    }
  }
}

template <typename T, int MODE>
__global__ void __launch_bounds__(threads<T>(), 1) gated_tc_kernel(const __grid_constant__ Launch p) {
  using S = Form<T>;
  constexpr bool F32 = sizeof(T) == 4, DUAL = MODE == FORWARD || MODE == PARTIALS;
  constexpr bool A_TURNED = MODE == WEIGHT_GRAD, B_TURNED = MODE != INPUT_GRAD;      // the operand lies along the rows
  constexpr int LINE = 128 / (int)sizeof(T);                                          // values of a line
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[S::STAGES], ready[S::STAGES], empty[S::STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int n_mma = DUAL ? 2 * p.width : p.width;                                     // columns of an MMA
  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < S::STAGES; ++s) {
      bar_init(&full[s], 1);
      bar_init(&ready[s], F32 ? S::SPLITTERS : 1);
      bar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      bar_init(&acc_full[a], 1);
      bar_init(&acc_empty[a], EPI_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&tmem_slot)), "r"(2 * S::COLS) : "memory");
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
      const uint32_t bytes = S::A_BYTES + (uint32_t)n_mma * 128;
      for (int64_t i = blockIdx.x; i < p.items && ok && !*ab; i += gridDim.x) {
        const Item t = item_of<MODE>(p, i);
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!bar_wait(&empty[s], ph, ab)) { ok = false; break; }
          unsigned char* st = base + (size_t)s * S::STAGE;
          uint64_t* bar = &full[s];
          bar_expect_tx(bar, bytes);
          const int h = MODE == INPUT_GRAD ? kb >= p.kblocks : t.half, k = (MODE == INPUT_GRAD && h ? kb - p.kblocks : kb) * S::BK;
          if (A_TURNED) {
#pragma unroll
            for (int c = 0; c < TILE_M / LINE; ++c) tma_load_2d(st + c * S::BK * 128, &p.a[0], (int)t.row + c * LINE, k, bar);
          } else {
            tma_load_2d(st, &p.a[MODE == INPUT_GRAD ? h : 0], k, (int)t.row, bar);
          }
          unsigned char* sb = st + S::B_AT;
          if (MODE == INPUT_GRAD) {
            tma_load_2d(sb, &p.b[h], k, t.col, bar);
          } else {
            for (int q = 0; q < (DUAL ? 2 : 1); ++q)
              for (int c = 0; c < p.width / LINE; ++c, sb += S::BK * 128) tma_load_2d(sb, &p.b[DUAL ? q : t.half], t.col + c * LINE, k, bar);
          }
          if (++s == S::STAGES) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMAs ----------------
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      int64_t piece = 0;
      bool ok = true;
      const uint32_t idesc = F32 ? umma_idesc_tf32(n_mma) : idesc_bf16(n_mma, A_TURNED, B_TURNED);
      for (int64_t i = blockIdx.x; i < p.items && ok && !*ab; i += gridDim.x) {
        const Item t = item_of<MODE>(p, i);
        for (int k0 = t.kb0; k0 < t.kb1 && ok; ++piece) {
          const int k1 = F32 ? min(k0 + PIECE, t.kb1) : t.kb1, a = (int)(piece & 1);
          if (!bar_wait(&acc_empty[a], (uint32_t)(((piece >> 1) & 1) ^ 1), ab)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(a * S::COLS);
          for (int kb = k0; kb < k1; ++kb) {
            if (!bar_wait(F32 ? &ready[s] : &full[s], ph, ab)) { ok = false; break; }
            tc_fence_after();
            const uint32_t at = s32(base + (size_t)s * S::STAGE), bt = at + S::B_AT;
            if (F32) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint64_t ah = umma_desc(at + q * 32), al = umma_desc(at + S::A_BYTES + q * 32);
                const uint64_t bh = umma_desc(bt + q * 32), bl = umma_desc(bt + S::COLS * 128 + q * 32);
                umma_tf32(d, al, bh, idesc, kb != k0 || q);
                umma_tf32(d, ah, bl, idesc, 1);
                umma_tf32(d, ah, bh, idesc, 1);
              }
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                mma_bf16(d, A_TURNED ? desc_rows(at + q * 2048) : umma_desc(at + q * 32), B_TURNED ? desc_rows(bt + q * 2048) : umma_desc(bt + q * 32),
                         idesc, kb != k0 || q);
            }
            umma_commit(&empty[s]);
            if (++s == S::STAGES) s = 0, ph ^= 1;
          }
          if (ok) umma_commit(&acc_full[a]);
          k0 = k1;
        }
      }
    }
  } else if (warp < 2 + S::SPLITTERS) {
    // ---------------- float32 to TF32 pairs ----------------
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    const int w = warp - 2;
    for (int64_t i = blockIdx.x; i < p.items && ok && !*ab; i += gridDim.x) {
      const Item t = item_of<MODE>(p, i);
      for (int kb = t.kb0; kb < t.kb1; ++kb) {
        if (!bar_wait(&full[s], ph, ab)) { ok = false; break; }
        unsigned char* st = base + (size_t)s * S::STAGE;
        split_block(st + w * 4096, S::A_BYTES, A_TURNED, lane);
        for (int b = w; b < n_mma / 32; b += S::SPLITTERS) split_block(st + S::B_AT + b * 4096, S::COLS * 128, B_TURNED, lane);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(&ready[s]);
        if (++s == S::STAGES) s = 0, ph ^= 1;
      }
    }
  } else {
    // ---------------- epilogue ----------------
    // Warps of the same quarter of the lanes share a tile's columns: 32 at a time of each half (two halves side by side: DUAL).
    const int e = warp - 2 - S::SPLITTERS, quarter = warp & 3, share = e >> 2;
    unsigned char* patch = base + (size_t)S::STAGES * S::STAGE + (size_t)e * PATCH;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    int64_t piece = 0;
    bool ok = true;
    for (int64_t i = blockIdx.x; i < p.items && ok && !*ab; i += gridDim.x) {
      const Item t = item_of<MODE>(p, i);
      const int64_t row = t.row + quarter * 32;
      const int lines = (int)max((int64_t)0, min((int64_t)32, p.rows - row));
      // 32 columns of the sum, read from tensor memory or, where it came in pieces, from registers
      float sum[F32 ? 2 : 1][32];
      uint32_t d = 0;
      int pieces = F32 ? (t.kb1 - t.kb0 + PIECE - 1) / PIECE : 1;
      for (int q = 0; q < pieces; ++q, ++piece) {
        const int a = (int)(piece & 1);
        if (!bar_wait(&acc_full[a], (uint32_t)((piece >> 1) & 1), ab)) { ok = false; break; }
        tc_fence_after();
        d = lanes + (uint32_t)(a * S::COLS);
        if (F32) {
          // float32 tiles have at most 128 columns: a share is 64, or 32 of each half
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int at = DUAL ? b * p.width + share * 32 : share * 64 + b * 32;
            if (at >= n_mma) continue;                                               // a narrow tile: the share has no such columns
            float v[32];
            tmem_ld32(d + at, v);
#pragma unroll
            for (int c = 0; c < 32; ++c) sum[F32 ? b : 0][c] = q ? sum[F32 ? b : 0][c] + v[c] : v[c];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(&acc_empty[a]);
        }
      }
      if (!ok) break;
      const int mine = F32 ? (DUAL ? 32 : 64) : p.width > 64 ? (p.width / 2 + LINE - 1) / LINE * LINE : LINE;    // columns of a share
      const int from = share * mine, to = min(p.width, from + mine);
      for (int c0 = from; c0 < to; c0 += LINE) {
        const int col = t.col + c0, valid = min(LINE, p.cols - col);                  // columns of this line in the results
        const int64_t at = row * p.out_pitch + col;
        if (MODE == WEIGHT_GRAD) {
          // partial results are float32, so a bfloat16 tile's line of 64 leaves as two
#pragma unroll
          for (int b = 0; b < LINE / 32; ++b) {
            float v[32];
            if (F32) {
#pragma unroll
              for (int c = 0; c < 32; ++c) v[c] = c0 == from ? sum[0][c] : sum[F32 ? 1 : 0][c];
            } else {
              tmem_ld32(d + c0 + b * 32, v);
            }
            line_put<float>(patch, lane, 0, v);
            const int here = valid - b * 32;
            float* out = static_cast<float*>(p.out) + (t.part * 2 + t.half) * p.part + at + b * 32;
            patch_out(patch, reinterpret_cast<unsigned char*>(out), p.out_pitch * 4, lines, here > 0 ? min(32, here) / 4 : 0, lane);
          }
          continue;
        }
        const int bytes16 = max(0, valid) * (int)sizeof(T) / 16;
        const int64_t pitch = p.out_pitch * (int)sizeof(T);
        T* out = static_cast<T*>(p.out) + at;
        if (MODE == INPUT_GRAD) {
#pragma unroll
          for (int b = 0; b < LINE / 32; ++b) {
            float v[32];
            if (F32) {
#pragma unroll
              for (int c = 0; c < 32; ++c) v[c] = c0 == from ? sum[0][c] : sum[F32 ? 1 : 0][c];
            } else {
              tmem_ld32(d + c0 + b * 32, v);
            }
            line_put<T>(patch, lane, b, v);
          }
          patch_out(patch, reinterpret_cast<unsigned char*>(out), pitch, lines, bytes16, lane);
          continue;
        }
        if (MODE == PARTIALS) patch_in(patch, reinterpret_cast<const unsigned char*>(static_cast<const T*>(p.g) + at), pitch, lines, bytes16, lane);
        uint32_t second[F32 ? 1 : LINE / 2];                                          // du of the line, while da leaves through the patch
        float keep[32];
#pragma unroll
        for (int b = 0; b < LINE / 32; ++b) {
          float a[32], u[32];
          if (F32) {
#pragma unroll
            for (int c = 0; c < 32; ++c) a[c] = sum[0][c], u[c] = sum[F32 ? 1 : 0][c];
          } else {
            tmem_ld32(d + c0 + b * 32, a);
            tmem_ld32(d + p.width + c0 + b * 32, u);
          }
          if (MODE == FORWARD) {
#pragma unroll
            for (int c = 0; c < 32; ++c) a[c] = activate(a[c], p.act).y * u[c];
          } else {
            float g[32];
            line_get<T>(patch, lane, b, g);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const Value<float> v = activate(a[c], p.act);
              a[c] = g[c] * u[c] * v.dy;
              u[c] = g[c] * v.y;
            }
            if constexpr (F32) {
#pragma unroll
              for (int c = 0; c < 32; ++c) keep[c] = u[c];
            } else {
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(u[2 * c], u[2 * c + 1]);
                second[b * 16 + c] = *reinterpret_cast<const uint32_t*>(&two);
              }
            }
          }
          line_put<T>(patch, lane, b, a);
        }
        patch_out(patch, reinterpret_cast<unsigned char*>(out), pitch, lines, bytes16, lane);
        if (MODE == PARTIALS) {
          if constexpr (F32) {
            line_put<T>(patch, lane, 0, keep);
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) *patch_at(patch, lane, c) = make_uint4(second[4 * c], second[4 * c + 1], second[4 * c + 2], second[4 * c + 3]);
          }
          patch_out(patch, reinterpret_cast<unsigned char*>(static_cast<T*>(p.out2) + at), pitch, lines, bytes16, lane);
        }
      }
      if (!F32) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&acc_empty[(int)(piece - 1) & 1]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * S::COLS) : "memory");
  }
  if (tid == 0 && abort_flag) {
    atomicExch(p.status, 2);
    let_copies_land(full, S::STAGES);
  }
}

// ---- host side ----------------------------------------------------------------------------------
// A (rows, columns) matrix, columns next to each other, in boxes of `line` columns by `lines` rows.
template <typename T>
int map_of(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int line, int lines, bool swizzle) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(EQT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  int dev = 0;                                           // the encoder needs a current context (see make_map)
  if (cudaGetDevice(&dev) == cudaSuccess) cudaSetDevice(dev);
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols * sizeof(T)};
  const cuuint32_t box[2] = {(cuuint32_t)line, (cuuint32_t)lines}, ones[2] = {1, 1};
  const CUresult r = enc(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                         strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? EQT_OK : fail(EQT_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}

// Columns a tile: as few tiles as `most` allows, of one width, a multiple of the columns of a line.
int width_of(int cols, int most, int line) {
  const int tiles = (int)ceil_div(cols, most);
  return (int)ceil_div(ceil_div(cols, tiles), line) * line;
}

template <typename T, int MODE> int launch(const GatedArgs& a, cudaStream_t s) {
  using S = Form<T>;
  constexpr int LINE = 128 / (int)sizeof(T);
  constexpr bool DUAL = MODE == FORWARD || MODE == PARTIALS, F32 = sizeof(T) == 4;
  const size_t size = sizeof(T);
  const char *w = static_cast<const char*>(a.w), *d = static_cast<const char*>(a.d);
  const char* w1 = w + (size_t)a.c * a.f * size;
  const char* d1 = d ? d + (size_t)a.n * a.f * size : nullptr;
  Launch p{};
  int rc = EQT_OK;
  // Operands that lie along the rows come in boxes of one line of values by a k-block; for float32 they are turned on the way and
  // need no swizzle.
  if (DUAL) {
    p.cols = a.f, p.rows = a.n, p.kblocks = (int)ceil_div(a.c, S::BK);
    p.width = width_of(a.f, S::COLS / 2, F32 ? 32 : LINE);
    rc = map_of<T>(&p.a[0], a.x, a.n, a.c, LINE, TILE_M, true);
    if (!rc) rc = map_of<T>(&p.b[0], w, a.c, a.f, LINE, S::BK, !F32);
    if (!rc) rc = map_of<T>(&p.b[1], w1, a.c, a.f, LINE, S::BK, !F32);
    p.out = MODE == FORWARD ? a.h : a.d;
    p.out2 = const_cast<char*>(d1);
    p.g = a.g;
  } else if (MODE == INPUT_GRAD) {
    p.cols = a.c, p.rows = a.n, p.kblocks = (int)ceil_div(a.f, S::BK);
    p.width = width_of(a.c, S::COLS, LINE);
    rc = map_of<T>(&p.a[0], d, a.n, a.f, LINE, TILE_M, true);
    if (!rc) rc = map_of<T>(&p.a[1], d1, a.n, a.f, LINE, TILE_M, true);
    if (!rc) rc = map_of<T>(&p.b[0], w, a.c, a.f, LINE, p.width, true);
    if (!rc) rc = map_of<T>(&p.b[1], w1, a.c, a.f, LINE, p.width, true);
    p.out = a.dx;
  } else {
    p.cols = a.f, p.rows = a.c, p.kblocks = (int)ceil_div(a.n, S::BK);
    p.width = width_of(a.f, S::COLS, LINE);
    p.split_blocks = (int)(a.split_rows / S::BK);
    p.part = (int64_t)a.c * a.f;
    rc = map_of<T>(&p.a[0], a.x, a.n, a.c, LINE, S::BK, !F32);
    if (!rc) rc = map_of<T>(&p.b[0], d, a.n, a.f, LINE, S::BK, !F32);
    if (!rc) rc = map_of<T>(&p.b[1], d1, a.n, a.f, LINE, S::BK, !F32);
    p.out = a.parts;
  }
  if (rc) return rc;
  p.out_pitch = p.cols;
  p.row_tiles = (int)ceil_div(p.rows, TILE_M);
  p.col_tiles = (int)ceil_div(p.cols, p.width);
  p.items = (int64_t)p.row_tiles * p.col_tiles * (MODE == WEIGHT_GRAD ? 2 * a.splits : 1);
  p.act = a.act;
  p.status = a.status;
  if (int r = allow_shared(gated_tc_kernel<T, MODE>, shared_bytes<T>())) return r;
  const unsigned grid = (unsigned)std::min<int64_t>(p.items, tc::sm_count());
  gated_tc_kernel<T, MODE><<<grid, threads<T>(), shared_bytes<T>(), s>>>(p);
  return check_launch("gated_tc");
}

template <typename T> int backward(const GatedArgs& a, cudaStream_t s) {
  if (int rc = launch<T, PARTIALS>(a, s)) return rc;
  if (a.dx)
    if (int rc = launch<T, INPUT_GRAD>(a, s)) return rc;
  return a.dw ? launch<T, WEIGHT_GRAD>(a, s) : EQT_OK;
}

}  // namespace

int tensor_forward(int dtype, const GatedArgs& p, cudaStream_t s) {
  return dtype == EQT_F32 ? launch<float, FORWARD>(p, s) : launch<__nv_bfloat16, FORWARD>(p, s);
}
int tensor_backward(int dtype, const GatedArgs& p, cudaStream_t s) {
  return dtype == EQT_F32 ? backward<float>(p, s) : backward<__nv_bfloat16>(p, s);
}

}  // namespace gated
}  // namespace eqt
