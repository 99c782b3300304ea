// Attention within the graphs of a packed batch, forward and backward.
//
// Features are (nodes, d, C); the channels are split over the heads, and a head's vectors are its D = d C / H values of a node.  Node i
// attends to the nodes j of its own graph:
//
//     z_ij = scale <q_i, k_j>        t_ij = tanh(z_ij / cap)         s_ij = (cap t_ij  or  z_ij) - slope_h |p_i - p_j|
//     P_ij = exp(s_ij) / sum_j exp(s_ij)                             out_i = sum_j P_ij v_j
//
//     dP_ij = <g_i, v_j>             delta_i = <g_i, out_i>          dS_ij = P_ij (dP_ij - delta_i)
//     dz_ij = scale dS_ij (1 - t_ij^2)      dv_j = sum_i P_ij g_i    dq_i = sum_j dz_ij k_j    dk_j = sum_i dz_ij q_i
//     dslope_h = - sum_ij dS_ij r_ij        dp_n = sum_h -slope_h (sum_j dS_nj u_nj - sum_i dS_in u_in),  u_ij = (p_i - p_j) / r_ij
//
// One pass over the keys with the running maximum and sum of the softmax; scores stay in registers.  A CTA of four warps has a tile of
// rows of ONE graph (16 a warp), so nothing that another graph holds, not even a NaN, enters a product.  The backward pass computes the
// scores again, twice: once by rows (dq, delta, the rows' geometry) and once by columns (dk, dv, the columns' geometry), so every
// result is written by one CTA and sums have one order; no atomics.
//
// Matrix instructions are the warp-wide mma.sync.  Measured on this GPU they run at 552 TFLOP/s in bf16 and the special function unit
// at 4.6e12 results/s.  A score costs one root (distance), two results for the cap and one exponential, so a head of 64 values takes
// 256 flops of the tensor cores for up to four results: 0.46 ps against 0.87 ps.  What bounds the calls is the special functions and
// the arithmetic around them, and tiles of 16 rows fit graphs of tens of nodes, where tiles of 128 rows would be three quarters empty.
// float32 operands are split into TF32 pairs, three products each.
#pragma once

#include "tc_common.cuh"

namespace eqt {
namespace attention {

constexpr int THREADS = 128, WARPS = 4;
constexpr float LOG2E = 1.4426950408889634f;

struct Operand {
  const void* p;
  int64_t node, comp;        // strides in elements
};

struct AttentionParams {
  Operand q, k, v, out, g;
  void *out_w, *dq, *dk, *dv;
  float *lse, *delta;        // [head][node]; lse in units of log2
  float4 *geo_row, *geo_col; // [head][node]: (sum dS r, sum dS u) by rows; (0, sum dS u) by columns
  const int4* tiles;         // first row, first and one past the last node of its graph
  const float *pos, *slope;
  int64_t n;
  int heads, comps, size;    // size: channels a head
  float scale, cap;          // cap 0: none
  int vec;                   // 16-byte pieces of every operand lie on 16-byte boundaries
};

// ---- matrix fragments ---------------------------------------------------------------------------
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const float (&a)[4], float b0, float b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(tc::s32(p)) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(tc::s32(p)) : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Rows of a tile in shared memory are DP values and 16 bytes apart from a multiple of 32 banks, so that the eight rows of a matrix
// load, and the four by eight places of a TF32 fragment (and of one transposed), fall on different banks.
template <typename T, int DP> struct Row { static constexpr int LD = DP + 16 / (int)sizeof(T); };

// acc[16 rows][8 NT] = A[16][DP] B[8 NT][DP]^T
template <int DP, int NT>
__device__ __forceinline__ void score_mma(float (&acc)[NT][4], const __nv_bfloat16* a, const __nv_bfloat16* b, int lane) {
  constexpr int LD = Row<__nv_bfloat16, DP>::LD;
  const __nv_bfloat16* ap = a + (lane & 15) * LD + (lane >> 4) * 8;
  const __nv_bfloat16* bp = b + ((lane & 7) + ((lane >> 4) << 3)) * LD + ((lane >> 3) & 1) * 8;
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    uint32_t ra[4];
    ldmatrix4(ra, ap + ks * 16);
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t rb[4];
      ldmatrix4(rb, bp + n * 8 * LD + ks * 16);
      mma_bf16(acc[n], ra, rb[0], rb[1]);
      mma_bf16(acc[n + 1], ra, rb[2], rb[3]);
    }
  }
}
template <int DP, int NT>
__device__ __forceinline__ void score_mma(float (&acc)[NT][4], const float* a, const float* b, int lane) {
  constexpr int LD = Row<float, DP>::LD;
  const int g = lane >> 2, t = lane & 3;
  const float *ap = a + g * LD + t, *bp = b + g * LD + t;
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll 4
  for (int ks = 0; ks < DP / 8; ++ks) {
    float hi[4], lo[4];
    tc::split_tf32(ap[ks * 8], hi[0], lo[0]);
    tc::split_tf32(ap[ks * 8 + 8 * LD], hi[1], lo[1]);
    tc::split_tf32(ap[ks * 8 + 4], hi[2], lo[2]);
    tc::split_tf32(ap[ks * 8 + 8 * LD + 4], hi[3], lo[3]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float h0, l0, h1, l1;
      tc::split_tf32(bp[n * 8 * LD + ks * 8], h0, l0);
      tc::split_tf32(bp[n * 8 * LD + ks * 8 + 4], h1, l1);
      mma_tf32(acc[n], lo, h0, h1);
      mma_tf32(acc[n], hi, l0, l1);
      mma_tf32(acc[n], hi, h0, h1);
    }
  }
}

// o[16 rows][DP] += p[16][8 NT] X[8 NT][DP], p in the layout that score_mma leaves
template <int DP, int NT>
__device__ __forceinline__ void out_mma(float (&o)[DP / 8][4], const float (&p)[NT][4], const __nv_bfloat16* x, int lane) {
  constexpr int LD = Row<__nv_bfloat16, DP>::LD;
  const __nv_bfloat16* xp = x + (lane & 15) * LD + (lane >> 4) * 8;
#pragma unroll
  for (int j = 0; j < NT / 2; ++j) {
    // weights and score gradients are rounded to bfloat16 here, as the operands are; their sums stay in float32
    const uint32_t a[4] = {pack_bf16(p[2 * j][0], p[2 * j][1]), pack_bf16(p[2 * j][2], p[2 * j][3]),
                           pack_bf16(p[2 * j + 1][0], p[2 * j + 1][1]), pack_bf16(p[2 * j + 1][2], p[2 * j + 1][3])};
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      uint32_t rb[4];
      ldmatrix4_trans(rb, xp + j * 16 * LD + d * 16);
      mma_bf16(o[2 * d], a, rb[0], rb[1]);
      mma_bf16(o[2 * d + 1], a, rb[2], rb[3]);
    }
  }
}
// The k-th place of a TF32 fragment may be any row of X as long as both operands agree: place t is row 2 t and place t + 4 row 2 t + 1,
// which is where score_mma left the weights.  The tensor cores' adder truncates, so a tile's sum starts at zero and joins the running
// one with ordinary rounding.
template <int DP, int NT>
__device__ __forceinline__ void out_mma(float (&o)[DP / 8][4], const float (&p)[NT][4], const float* x, int lane) {
  constexpr int LD = Row<float, DP>::LD;
  const float* xp = x + (lane & 3) * 2 * LD + (lane >> 2);
  float hi[NT][4], lo[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    tc::split_tf32(p[j][0], hi[j][0], lo[j][0]);
    tc::split_tf32(p[j][2], hi[j][1], lo[j][1]);
    tc::split_tf32(p[j][1], hi[j][2], lo[j][2]);
    tc::split_tf32(p[j][3], hi[j][3], lo[j][3]);
  }
#pragma unroll
  for (int d = 0; d < DP / 8; d += 4) {
    float s[4][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e][0] = s[e][1] = s[e][2] = s[e][3] = 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float h0, l0, h1, l1;
        tc::split_tf32(xp[j * 8 * LD + (d + e) * 8], h0, l0);
        tc::split_tf32(xp[j * 8 * LD + LD + (d + e) * 8], h1, l1);
        mma_tf32(s[e], lo[j], h0, h1);
        mma_tf32(s[e], hi[j], l0, l1);
        mma_tf32(s[e], hi[j], h0, h1);
      }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d + e][i] += s[e][i];
  }
}

// ---- special functions --------------------------------------------------------------------------
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rsqrt_fast(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh to some 1e-7 absolute, which is what a score needs: (e - 1) / (e + 1), e = exp(2 x), kept finite.
// float32 scores take the function of the library, which keeps small values to the last bit.
template <typename T> __device__ __forceinline__ float tanh_of(float x) {
  const float e = exp2_fast(fminf(x * (2.f * LOG2E), 64.f));
  return __fdividef(e - 1.f, e + 1.f);
}
template <> __device__ __forceinline__ float tanh_of<float>(float x) { return tanhf(x); }

// ---- tiles in shared memory ---------------------------------------------------------------------
__device__ __forceinline__ void copy16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::s32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(void* dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(tc::s32(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Which 16 bytes of a head's row a thread of a head's warps copies: always the same ones.
template <typename T, int DP, int TH> struct Piece {
  static constexpr int V = 16 / (int)sizeof(T);
  static constexpr int PER_ROW = DP / V, ROWS = TH / PER_ROW;        // rows that the head's threads copy at a time
  int row, at, comp, channel;
  bool there;
  __device__ __forceinline__ Piece(int tid, int comps, int size) {
    row = tid / PER_ROW;
    at = (tid % PER_ROW) * V;
    comp = at / size;
    channel = at - comp * size;
    there = row < ROWS && at < comps * size;
  }
};

// Rows [first, first + ROWS_TILE) of one head to shared memory, zeros from `end` on.
template <typename T, int DP, int TH, int ROWS_TILE>
__device__ __forceinline__ void load_rows(T* dst, const Operand& x, const Piece<T, DP, TH>& piece, int first, int end, int head,
                                          const AttentionParams& p, int tid) {
  constexpr int LD = Row<T, DP>::LD;
  if (p.vec) {
    if (!piece.there) return;
    const T* src = static_cast<const T*>(x.p) + piece.comp * x.comp + (int64_t)head * p.size + piece.channel;
#pragma unroll
    for (int r = piece.row; r < ROWS_TILE; r += Piece<T, DP, TH>::ROWS) {
      const bool there = first + r < end;
      copy16(dst + r * LD + piece.at, src + (int64_t)(there ? first + r : 0) * x.node, there);
    }
    return;
  }
  const int d = p.comps * p.size;
  for (int i = tid; i < ROWS_TILE * d; i += TH) {
    const int r = i / d, j = i - r * d, m = j / p.size, c = j - m * p.size;
    dst[r * LD + j] = first + r < end ? static_cast<const T*>(x.p)[(int64_t)(first + r) * x.node + m * x.comp + (int64_t)head * p.size + c]
                                      : static_cast<T>(0.f);
  }
}

// The 16 rows of a warp from the accumulators to shared memory and from there to (n, d, C), contiguous.
template <typename T, int DP>
__device__ __forceinline__ void store_rows(T* buf, void* out, const float (&o)[DP / 8][4], float f0, float f1, int first, int end, int head,
                                           const AttentionParams& p, int lane) {
  constexpr int LD = Row<T, DP>::LD, V = 16 / (int)sizeof(T);
  const int g = lane >> 2, t = lane & 3;
  __syncwarp();
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    T* b = buf + g * LD + n * 8 + 2 * t;
    b[0] = static_cast<T>(o[n][0] * f0);
    b[1] = static_cast<T>(o[n][1] * f0);
    b[8 * LD] = static_cast<T>(o[n][2] * f1);
    b[8 * LD + 1] = static_cast<T>(o[n][3] * f1);
  }
  __syncwarp();
  const int d = p.comps * p.size, channels = p.heads * p.size;
  T* to = static_cast<T*>(out) + (int64_t)head * p.size;
  if (p.vec) {
    const int pieces = d / V;
    for (int i = lane; i < 16 * pieces; i += 32) {
      const int r = i / pieces, j = (i - r * pieces) * V, m = j / p.size, c = j - m * p.size;
      if (first + r < end)
        *reinterpret_cast<uint4*>(to + ((int64_t)(first + r) * p.comps + m) * channels + c) = *reinterpret_cast<const uint4*>(buf + r * LD + j);
    }
    return;
  }
  for (int i = lane; i < 16 * d; i += 32) {
    const int r = i / d, j = i - r * d, m = j / p.size, c = j - m * p.size;
    if (first + r < end) to[((int64_t)(first + r) * p.comps + m) * channels + c] = buf[r * LD + j];
  }
}

// Positions of the rows [first, first + ROWS_TILE), by all threads of the CTA.
template <int ROWS_TILE>
__device__ __forceinline__ void load_positions(float4* dst, const float* pos, int first, int end) {
  for (int i = threadIdx.x; i < ROWS_TILE * 3; i += THREADS) {
    const int r = i / 3, x = i - r * 3;
    const bool there = first + r < end;
    copy4(reinterpret_cast<float*>(dst + r) + x, pos + (int64_t)(there ? first + r : 0) * 3 + x, there);
  }
}

__device__ __forceinline__ float3 position(const float* pos, int row, int end) {
  return row < end ? make_float3(pos[(int64_t)row * 3], pos[(int64_t)row * 3 + 1], pos[(int64_t)row * 3 + 2]) : make_float3(0.f, 0.f, 0.f);
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// WR warps have the rows of one head (a tile of 16 WR rows), so a CTA has 4 / WR heads; KT rows of the other side at a time, two
// tiles of them in shared memory.
template <typename T, int DP, int WR, int KT> struct Shape {
  static constexpr int HEADS = WARPS / WR, TH = WR * 32, TILE = 16 * WR, LD = Row<T, DP>::LD;
  static constexpr size_t STAGE = (size_t)2 * KT * LD;                                       // elements: two matrices
  static constexpr size_t head_elements(int residents) { return (size_t)residents * TILE * LD + 2 * STAGE; }
  static constexpr size_t bytes(int residents, int extra) { return HEADS * head_elements(residents) * sizeof(T) + (size_t)extra; }
};

template <typename T, int DP, int WR, int KT>
__global__ void __launch_bounds__(THREADS) attention_forward_kernel(const __grid_constant__ AttentionParams p) {
  using S = Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int slot = warp / WR, ht = tid - slot * S::TH;                   // the head's place in the CTA, the thread's place in the head
  const int head = blockIdx.y * S::HEADS + slot;
  const int4 tile = p.tiles[blockIdx.x];
  const int first = tile.x, lo = tile.y, hi = tile.z;
  T* base = reinterpret_cast<T*>(smem) + slot * S::head_elements(1);
  T *rows = base, *stage = base + S::TILE * LD;
  float4* spos = reinterpret_cast<float4*>(smem + S::bytes(1, 0));       // two tiles of positions
  const bool here = head < p.heads;
  const int end = here ? hi : 0;                                         // a place without a head copies nothing
  if (p.comps * p.size < DP) {                                           // the columns behind the head's values stay zero
    for (size_t i = tid; i < S::bytes(1, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  const Piece<T, DP, S::TH> piece(ht, p.comps, p.size);
  auto fetch = [&](int key, int s) {
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE, p.k, piece, key, end, head, p, ht);
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, p.v, piece, key, end, head, p, ht);
    if (p.pos) load_positions<KT>(spos + s * KT, p.pos, key, hi);
    copies_commit();
  };
  load_rows<T, DP, S::TH, S::TILE>(rows, p.q, piece, first, end, head, p, ht);
  fetch(lo, 0);

  const int row = first + (warp % WR) * 16;                              // of the warp
  const bool work = here && row < hi;
  const T* mine = rows + (warp % WR) * 16 * LD;
  float o[DP / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  const float scale2 = p.scale * LOG2E, cap2 = p.cap * LOG2E, to_cap = p.cap > 0.f ? p.scale / p.cap : 0.f;
  float slope2 = 0.f;
  float3 p0, p1;
  if (p.pos) {
    slope2 = here ? p.slope[head] * LOG2E : 0.f;
    p0 = position(p.pos, row + g, hi);
    p1 = position(p.pos, row + g + 8, hi);
  }
  int s = 0;
  for (int key = lo; key < hi; key += KT, s ^= 1) {
    if (key + KT < hi) {
      fetch(key + KT, s ^ 1);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncthreads();
    if (work) {
      const T *ks = stage + s * S::STAGE, *vs = ks + KT * LD;
      float z[NT][4];
      score_mma<DP, NT>(z, mine, ks, lane);
      if (p.cap > 0.f) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) z[n][i] = cap2 * tanh_of<T>(z[n][i] * to_cap);
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) z[n][i] *= scale2;
      }
      if (p.pos) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 pk = spos[s * KT + n * 8 + 2 * t + i];
            const float x0 = p0.x - pk.x, y0 = p0.y - pk.y, z0 = p0.z - pk.z, x1 = p1.x - pk.x, y1 = p1.y - pk.y, z1 = p1.z - pk.z;
            const float d0 = x0 * x0 + y0 * y0 + z0 * z0, d1 = x1 * x1 + y1 * y1 + z1 * z1;
            z[n][i] -= slope2 * (d0 > 0.f ? d0 * rsqrt_fast(d0) : 0.f);
            z[n][2 + i] -= slope2 * (d1 > 0.f ? d1 * rsqrt_fast(d1) : 0.f);
          }
      }
      if (key + KT > hi) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (key + n * 8 + 2 * t + i >= hi) z[n][i] = z[n][2 + i] = -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float m = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n) m = fmaxf(m, fmaxf(z[n][2 * r], z[n][2 * r + 1]));
        m = fmaxf(quad_max(m), top[r]);
        const float from = m == -INFINITY ? 0.f : m, keep = exp2_fast(top[r] - from);
        top[r] = m;
        float add = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          z[n][2 * r] = exp2_fast(z[n][2 * r] - from);
          z[n][2 * r + 1] = exp2_fast(z[n][2 * r + 1] - from);
          add += z[n][2 * r] + z[n][2 * r + 1];
        }
        sum[r] = sum[r] * keep + add;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          o[n][2 * r] *= keep;
          o[n][2 * r + 1] *= keep;
        }
      }
      out_mma<DP, NT>(o, z, vs, lane);
    }
    __syncthreads();
  }
  if (!work) return;
  sum[0] = quad_sum(sum[0]);
  sum[1] = quad_sum(sum[1]);
  if (p.lse && t == 0) {
    float* to = p.lse + (int64_t)head * p.n + row + g;
    if (row + g < hi) to[0] = top[0] + log2f(sum[0]);
    if (row + g + 8 < hi) to[8] = top[1] + log2f(sum[1]);
  }
  store_rows<T, DP>(const_cast<T*>(mine), p.out_w, o, 1.f / sum[0], 1.f / sum[1], row, hi, head, p, lane);
}

// Backward by rows: dq, delta, and with positions the rows' sums of dS r and dS u.
// These sums are float32 results also where the features are bfloat16, so they do not go by the delta of the rounded output: with
// w = r or u, sum_j dS w = sum_j P dP w - (sum_j P dP) (sum_j P w), and the columns' pass is given sum_j P dP.
template <typename T, int DP, int WR, int KT, bool GEO>
__global__ void __launch_bounds__(THREADS) attention_rows_kernel(const __grid_constant__ AttentionParams p) {
  using S = Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  static_assert(2 * KT >= S::TILE, "the output's rows fit a stage");
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int slot = warp / WR, ht = tid - slot * S::TH;
  const int head = blockIdx.y * S::HEADS + slot;
  const int4 tile = p.tiles[blockIdx.x];
  const int first = tile.x, lo = tile.y, hi = tile.z;
  T* base = reinterpret_cast<T*>(smem) + slot * S::head_elements(2);
  T *rows = base, *grads = base + S::TILE * LD, *stage = base + 2 * S::TILE * LD;
  float4* spos = reinterpret_cast<float4*>(smem + S::bytes(2, 0));
  const bool here = head < p.heads;
  const int end = here ? hi : 0;
  if (p.comps * p.size < DP) {
    for (size_t i = tid; i < S::bytes(2, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  const Piece<T, DP, S::TH> piece(ht, p.comps, p.size);
  auto fetch = [&](int key, int s) {
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE, p.k, piece, key, end, head, p, ht);
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, p.v, piece, key, end, head, p, ht);
    if (p.pos) load_positions<KT>(spos + s * KT, p.pos, key, hi);
    copies_commit();
  };
  load_rows<T, DP, S::TH, S::TILE>(rows, p.q, piece, first, end, head, p, ht);
  load_rows<T, DP, S::TH, S::TILE>(grads, p.g, piece, first, end, head, p, ht);
  load_rows<T, DP, S::TH, S::TILE>(stage + S::STAGE, p.out, piece, first, end, head, p, ht);   // the output, where the second tile will be
  fetch(lo, 0);
  copies_wait<0>();
  __syncthreads();

  const int row = first + (warp % WR) * 16;
  const bool work = here && row < hi;
  const T *mq = rows + (warp % WR) * 16 * LD, *mg = grads + (warp % WR) * 16 * LD;
  float delta[2] = {0.f, 0.f}, lse[2] = {INFINITY, INFINITY};
  {
    const T *a = mg + g * LD, *b = stage + S::STAGE + ((warp % WR) * 16 + g) * LD;
    for (int c = t; c < DP; c += 4) {
      delta[0] += static_cast<float>(a[c]) * static_cast<float>(b[c]);
      delta[1] += static_cast<float>(a[8 * LD + c]) * static_cast<float>(b[8 * LD + c]);
    }
    delta[0] = quad_sum(delta[0]);
    delta[1] = quad_sum(delta[1]);
  }
  __syncthreads();                                                       // the output has been read
  const bool is[2] = {work && row + g < hi, work && row + g + 8 < hi};
  const int64_t at = (int64_t)head * p.n + row + g;
  if (is[0]) lse[0] = p.lse[at];
  if (is[1]) lse[1] = p.lse[at + 8];
  float dq[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) dq[n][0] = dq[n][1] = dq[n][2] = dq[n][3] = 0.f;
  float all[2] = {0.f, 0.f}, pw[2][4], pdw[2][4];                          // sum P dP, sum P w, sum P dP w; w = (r, u)
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) pw[r][i] = pdw[r][i] = 0.f;
  const float scale2 = p.scale * LOG2E, cap2 = p.cap * LOG2E, to_cap = p.cap > 0.f ? p.scale / p.cap : 0.f;
  float slope2 = 0.f;
  float3 pr[2];
  if (p.pos) {
    slope2 = here ? p.slope[head] * LOG2E : 0.f;
    pr[0] = position(p.pos, row + g, hi);
    pr[1] = position(p.pos, row + g + 8, hi);
  }
  int s = 0;
  for (int key = lo; key < hi; key += KT, s ^= 1) {
    if (key + KT < hi) {
      fetch(key + KT, s ^ 1);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncthreads();
    if (work) {
      const T *ks = stage + s * S::STAGE, *vs = ks + KT * LD;
      float z[NT][4], dp[NT][4];
      score_mma<DP, NT>(z, mq, ks, lane);
      score_mma<DP, NT>(dp, mg, vs, lane);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 pk = p.pos ? spos[s * KT + n * 8 + 2 * t + i] : make_float4(0.f, 0.f, 0.f, 0.f);
          const bool there = key + n * 8 + 2 * t + i < hi;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float& zz = z[n][2 * r + i];
            float slant = p.scale, score;
            if (p.cap > 0.f) {
              const float th = tanh_of<T>(zz * to_cap);
              score = cap2 * th;
              slant = p.scale * (1.f - th * th);
            } else {
              score = zz * scale2;
            }
            float dx, dy, dz, inv = 0.f, dist = 0.f;
            if (p.pos) {
              dx = pr[r].x - pk.x, dy = pr[r].y - pk.y, dz = pr[r].z - pk.z;
              const float d2 = dx * dx + dy * dy + dz * dz;
              inv = d2 > 0.f ? rsqrt_fast(d2) : 0.f;
              dist = d2 * inv;
              score -= slope2 * dist;
            }
            const float w = there ? exp2_fast(score - lse[r]) : 0.f, d = dp[n][2 * r + i];
            if (GEO) {
              const float wd = w * d, wi = w * inv, wdi = wd * inv;
              all[r] += wd;
              pw[r][0] += w * dist;
              pw[r][1] += wi * dx;
              pw[r][2] += wi * dy;
              pw[r][3] += wi * dz;
              pdw[r][0] += wd * dist;
              pdw[r][1] += wdi * dx;
              pdw[r][2] += wdi * dy;
              pdw[r][3] += wdi * dz;
            }
            zz = w * (d - delta[r]) * slant;
          }
        }
      out_mma<DP, NT>(dq, z, ks, lane);
    }
    __syncthreads();
  }
  if (!work) return;
  if (GEO) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      delta[r] = quad_sum(all[r]);
#pragma unroll
      for (int i = 0; i < 4; ++i) pdw[r][i] = quad_sum(pdw[r][i]) - delta[r] * quad_sum(pw[r][i]);
      if (is[r] && t == 0) p.geo_row[at + 8 * r] = make_float4(pdw[r][0], pdw[r][1], pdw[r][2], pdw[r][3]);
    }
  }
  if (t == 0) {
    if (is[0]) p.delta[at] = delta[0];
    if (is[1]) p.delta[at + 8] = delta[1];
  }
  store_rows<T, DP>(const_cast<T*>(mq), p.dq, dq, 1.f, 1.f, row, hi, head, p, lane);
}

// Backward by columns: dk, dv, and with positions the columns' sums of dS u.  The CTA's rows are keys; queries and the output's
// gradients come by in tiles, and the products are the transposed ones.
template <typename T, int DP, int WR, int KT, bool GEO>
__global__ void __launch_bounds__(THREADS) attention_columns_kernel(const __grid_constant__ AttentionParams p) {
  using S = Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int slot = warp / WR, ht = tid - slot * S::TH;
  const int head = blockIdx.y * S::HEADS + slot;
  const int4 tile = p.tiles[blockIdx.x];
  const int first = tile.x, lo = tile.y, hi = tile.z;
  T* base = reinterpret_cast<T*>(smem) + slot * S::head_elements(2);
  T *keys = base, *values = base + S::TILE * LD, *stage = base + 2 * S::TILE * LD;
  float4* spos = reinterpret_cast<float4*>(smem + S::bytes(2, 0));
  float* stats = reinterpret_cast<float*>(spos + 2 * KT) + slot * 4 * KT;           // [tile][lse, delta][KT]
  const bool here = head < p.heads;
  const int end = here ? hi : 0;
  if (p.comps * p.size < DP) {
    for (size_t i = tid; i < S::bytes(2, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  const Piece<T, DP, S::TH> piece(ht, p.comps, p.size);
  auto fetch = [&](int query, int s) {
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE, p.q, piece, query, end, head, p, ht);
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, p.g, piece, query, end, head, p, ht);
    for (int i = ht; i < KT; i += S::TH) {
      const bool there = query + i < end;
      const int64_t at = there ? (int64_t)head * p.n + query + i : 0;
      copy4(stats + (2 * s) * KT + i, p.lse + at, there);
      copy4(stats + (2 * s + 1) * KT + i, p.delta + at, there);
    }
    if (p.pos) load_positions<KT>(spos + s * KT, p.pos, query, hi);
    copies_commit();
  };
  load_rows<T, DP, S::TH, S::TILE>(keys, p.k, piece, first, end, head, p, ht);
  load_rows<T, DP, S::TH, S::TILE>(values, p.v, piece, first, end, head, p, ht);
  fetch(lo, 0);

  const int row = first + (warp % WR) * 16;
  const bool work = here && row < hi;
  const T *mk = keys + (warp % WR) * 16 * LD, *mv = values + (warp % WR) * 16 * LD;
  float dk[DP / 8][4], dv[DP / 8][4], geo[2][3] = {{0.f, 0.f, 0.f}, {0.f, 0.f, 0.f}};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    dk[n][0] = dk[n][1] = dk[n][2] = dk[n][3] = 0.f;
    dv[n][0] = dv[n][1] = dv[n][2] = dv[n][3] = 0.f;
  }
  const float scale2 = p.scale * LOG2E, cap2 = p.cap * LOG2E, to_cap = p.cap > 0.f ? p.scale / p.cap : 0.f;
  float slope2 = 0.f;
  float3 pr[2];
  if (p.pos) {
    slope2 = here ? p.slope[head] * LOG2E : 0.f;
    pr[0] = position(p.pos, row + g, hi);
    pr[1] = position(p.pos, row + g + 8, hi);
  }
  int s = 0;
  for (int query = lo; query < hi; query += KT, s ^= 1) {
    if (query + KT < hi) {
      fetch(query + KT, s ^ 1);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncthreads();
    if (work) {
      const T *qs = stage + s * S::STAGE, *gs = qs + KT * LD;
      const float *ls = stats + 2 * s * KT, *ds = ls + KT;
      float z[NT][4], dp[NT][4];
      score_mma<DP, NT>(z, mk, qs, lane);
      score_mma<DP, NT>(dp, mv, gs, lane);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = n * 8 + 2 * t + i;
          const float4 pk = p.pos ? spos[s * KT + c] : make_float4(0.f, 0.f, 0.f, 0.f);
          const bool there = query + c < hi;
          const float lse = ls[c], delta = ds[c];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float &zz = z[n][2 * r + i], &dd = dp[n][2 * r + i];
            float slant = p.scale, score;
            if (p.cap > 0.f) {
              const float th = tanh_of<T>(zz * to_cap);
              score = cap2 * th;
              slant = p.scale * (1.f - th * th);
            } else {
              score = zz * scale2;
            }
            float dx, dy, dz, inv = 0.f;
            if (p.pos) {                                                 // from the key to the query
              dx = pk.x - pr[r].x, dy = pk.y - pr[r].y, dz = pk.z - pr[r].z;
              const float d2 = dx * dx + dy * dy + dz * dz;
              inv = d2 > 0.f ? rsqrt_fast(d2) : 0.f;
              score -= slope2 * (d2 * inv);
            }
            const float w = there ? exp2_fast(score - lse) : 0.f, e = w * (dd - delta);
            if (GEO) {
              const float ei = e * inv;
              geo[r][0] += ei * dx;
              geo[r][1] += ei * dy;
              geo[r][2] += ei * dz;
            }
            zz = w;
            dd = e * slant;
          }
        }
      out_mma<DP, NT>(dv, z, gs, lane);
      out_mma<DP, NT>(dk, dp, qs, lane);
    }
    __syncthreads();
  }
  if (!work) return;
  if (GEO) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float4 v = make_float4(0.f, quad_sum(geo[r][0]), quad_sum(geo[r][1]), quad_sum(geo[r][2]));
      if (t == 0 && row + g + 8 * r < hi) p.geo_col[(int64_t)head * p.n + row + g + 8 * r] = v;
    }
  }
  store_rows<T, DP>(const_cast<T*>(mk), p.dk, dk, 1.f, 1.f, row, hi, head, p, lane);
  store_rows<T, DP>(const_cast<T*>(mv), p.dv, dv, 1.f, 1.f, row, hi, head, p, lane);
}

// ---- host side ----------------------------------------------------------------------------------
enum Pass { FORWARD, ROWS, COLUMNS };

template <typename T, int DP, int WR, int KT>
int launch(Pass pass, const AttentionParams& p, int64_t tiles, bool geo, cudaStream_t s) {
  using S = Shape<T, DP, WR, KT>;
  const dim3 grid((unsigned)tiles, (unsigned)ceil_div(p.heads, S::HEADS));
  auto run = [&](auto kernel, size_t bytes, const char* what) {
    if (int rc = allow_shared(kernel, bytes)) return rc;
    kernel<<<grid, THREADS, bytes, s>>>(p);
    return check_launch(what);
  };
  constexpr int POS = 2 * KT * 16, STATS = S::HEADS * 4 * KT * 4;
  if (pass == FORWARD) return run(attention_forward_kernel<T, DP, WR, KT>, S::bytes(1, POS), "attention_forward");
  if (pass == ROWS)
    return geo ? run(attention_rows_kernel<T, DP, WR, KT, true>, S::bytes(2, POS), "attention_rows")
               : run(attention_rows_kernel<T, DP, WR, KT, false>, S::bytes(2, POS), "attention_rows");
  return geo ? run(attention_columns_kernel<T, DP, WR, KT, true>, S::bytes(2, POS + STATS), "attention_columns")
             : run(attention_columns_kernel<T, DP, WR, KT, false>, S::bytes(2, POS + STATS), "attention_columns");
}

template <typename T, int DP>
int launch_rows(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s) {
  constexpr int KT = sizeof(T) == 2 && DP <= 64 ? 64 : 32;       // wide heads need the registers; float32 needs twice the registers and shared memory a value
  if (tile_rows == 64) return launch<T, DP, 4, KT>(pass, p, tiles, geo, s);
  if (tile_rows == 32) return launch<T, DP, 2, 32>(pass, p, tiles, geo, s);
  return launch<T, DP, 1, 16>(pass, p, tiles, geo, s);
}

template <typename T>
int launch_width(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s) {
  const int d = p.comps * p.size;
  if (d <= 32) return launch_rows<T, 32>(pass, p, tiles, tile_rows, geo, s);
  if (d <= 64) return launch_rows<T, 64>(pass, p, tiles, tile_rows, geo, s);
  if (d <= 96) return launch_rows<T, 96>(pass, p, tiles, tile_rows, geo, s);
  return launch_rows<T, 128>(pass, p, tiles, tile_rows, geo, s);
}

// Defined in graph_attention_f32.cu and graph_attention_bf16.cu, which compile side by side.
int launch_f32(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s);
int launch_bf16(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s);

}  // namespace attention
}  // namespace eqt
