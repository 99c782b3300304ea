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
// at 4.6e12 results/s.  A score costs one root (distance) and one exponential, the cap two results more unless its polynomial does, so
// a head of 64 values takes 256 flops of the tensor cores, 0.46 ps, for two to four results, 0.43 to 0.87 ps, and some twenty
// instructions of arithmetic.  Tiles of 16 rows fit graphs of tens of nodes, where tiles of 128 rows would be three quarters empty.  float32
// operands are split into TF32 pairs, three products each.
//
// One graph of 5001 nodes, 8 heads of 64 bfloat16 values, distance and cap: forward 355 us (144 TFLOP/s), by rows 667, by columns 652;
// 16 graphs of up to 2000 nodes, 8 heads of 32, forward with distance: 173 us, the special functions half busy.  No pipe is full: what
// bounds them is the latency of dependent instructions at the two to seven warps a scheduler that the registers leave.  For graphs of some hundred
// nodes and more, tcgen05 with accumulators in tensor memory would take them out of the registers; that has not been built or measured.
//
// Operands whose 16-byte pieces do not lie on 16-byte boundaries (12 bfloat16 channels a head, say) are read value by value, without
// asynchronous copies: 2000 molecules, 8 heads of 12 channels 1268 us a forward and backward pass, of 16 channels 387.
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
  Operand q, k, v, g;
  void *out, *dq, *dk, *dv;
  float *top, *inverse;      // [head][node]: the row's greatest score in units of log2, one over its sum of weights from there
  float* delta;              // [head][node]
  float4 *geo_row, *geo_col; // [head][node]: (sum dS r, sum dS u) by rows; (0, sum dS u) by columns
  const int4* tiles;         // first row, first and one past the last node of its graph
  const float *pos, *slope;
  int64_t n;
  int heads, comps, size;    // size: channels a head
  float scale, cap;          // cap 0: none
  int folds;                 // bfloat16: a graph of more than FOLD nodes
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

// acc[16 rows][8 NT] = A[16][DP] B[8 NT][DP]^T.  The pass by columns has the operands the other way round (TURNED) and takes the products in
// the same order: a score has the same bits in all passes, so its weight belongs to the saved statistics however large it is.
template <int DP, int NT, bool TURNED = false>
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
// The tensor cores' adder truncates, so the products with small parts have a sum of their own: one truncation for eight terms.
template <int DP, int NT, bool TURNED = false>
__device__ __forceinline__ void score_mma(float (&acc)[NT][4], const float* a, const float* b, int lane) {
  constexpr int LD = Row<float, DP>::LD;
  const int g = lane >> 2, t = lane & 3;
  const float *ap = a + g * LD + t, *bp = b + g * LD + t;
  float fine[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    fine[n][0] = fine[n][1] = fine[n][2] = fine[n][3] = 0.f;
  }
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
      mma_tf32(acc[n], hi, h0, h1);
      if (TURNED) mma_tf32(fine[n], hi, l0, l1);
      mma_tf32(fine[n], lo, h0, h1);
      if (!TURNED) mma_tf32(fine[n], hi, l0, l1);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] += fine[n][i];
}

// o[16 rows][DP] += p[16][8 NT] X[8 NT][DP], p in the layout that score_mma leaves.  Weights and score gradients are rounded to bfloat16
// here, as the operands are; their sums stay in float32.  FINE: what the rounding left goes in too.
template <int DP, int NT, bool FINE = false>
__device__ __forceinline__ void out_mma(float (&o)[DP / 8][4], const float (&p)[NT][4], const __nv_bfloat16* x, int lane) {
  constexpr int LD = Row<__nv_bfloat16, DP>::LD;
  const __nv_bfloat16* xp = x + (lane & 15) * LD + (lane >> 4) * 8;
#pragma unroll
  for (int j = 0; j < NT / 2; ++j) {
    const uint32_t a[4] = {pack_bf16(p[2 * j][0], p[2 * j][1]), pack_bf16(p[2 * j][2], p[2 * j][3]),
                           pack_bf16(p[2 * j + 1][0], p[2 * j + 1][1]), pack_bf16(p[2 * j + 1][2], p[2 * j + 1][3])};
    uint32_t rest[4];
    if (FINE) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        rest[i] = pack_bf16(p[2 * j + (i >> 1)][2 * (i & 1)] - __uint_as_float(a[i] << 16),
                            p[2 * j + (i >> 1)][2 * (i & 1) + 1] - __uint_as_float(a[i] & 0xffff0000u));
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      uint32_t rb[4];
      ldmatrix4_trans(rb, xp + j * 16 * LD + d * 16);
      mma_bf16(o[2 * d], a, rb[0], rb[1]);
      mma_bf16(o[2 * d + 1], a, rb[2], rb[3]);
      if (FINE) {
        mma_bf16(o[2 * d], rest, rb[0], rb[1]);
        mma_bf16(o[2 * d + 1], rest, rb[2], rb[3]);
      }
    }
  }
}
// The k-th place of a TF32 fragment may be any row of X as long as both operands agree: place t is row 2 t and place t + 4 row 2 t + 1,
// which is where score_mma left the weights.  The tensor cores' adder truncates, so a tile's sum starts at zero and joins the running
// one with ordinary rounding.
template <int DP, int NT, bool FINE = false>
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
  for (int d = 0; d < DP / 8; d += 2) {
    float s[2][4], h[2][NT][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) s[e][0] = s[e][1] = s[e][2] = s[e][3] = 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l0, l1;
        tc::split_tf32(xp[j * 8 * LD + (d + e) * 8], h[e][j][0], l0);
        tc::split_tf32(xp[j * 8 * LD + LD + (d + e) * 8], h[e][j][1], l1);
        mma_tf32(s[e], lo[j], h[e][j][0], h[e][j][1]);
        mma_tf32(s[e], hi[j], l0, l1);
      }
#pragma unroll
    for (int j = 0; j < NT; ++j)                         // large products last: truncations before them are of small sums
#pragma unroll
      for (int e = 0; e < 2; ++e) mma_tf32(s[e], hi[j], h[e][j][0], h[e][j][1]);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d + e][i] += s[e][i];
  }
}

// The bfloat16 products add up in the matrix instructions, whose adder truncates: a sum of one sign loses 1.2e-7 of itself at every step of
// 16 terms (outputs of 400,000 nodes: 3e-3, as much as their rounding).  So every FOLD terms a sum joins, with ordinary rounding, another
// one that waits in local memory; 8192 terms lose 6e-5.  Only the kernels for graphs that are longer do so (FOLDS), which take tiles of 64 rows:
// the code costs the others 3 % in registers.  float32 sums join after every tile anyway.
constexpr int FOLD = 8192;
template <int DP, int MORE = 0> struct Far {             // a thread's sums, and MORE numbers beside them
  float values[DP / 2 + MORE];
  __device__ __forceinline__ float* at() {
    float* p = values;
    asm volatile("" : "+l"(p));                          // values stay in memory: their address is known to no one
    return p;
  }
};
template <int DP> __device__ __forceinline__ void fold(float* far, float (&o)[DP / 8][4], bool first, float keep0 = 1.f, float keep1 = 1.f) {
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      far[4 * n + i] = first ? o[n][i] : fmaf(far[4 * n + i], i < 2 ? keep0 : keep1, o[n][i]);
      o[n][i] = 0.f;
    }
}
template <int DP> __device__ __forceinline__ void unfold(const float* far, float (&o)[DP / 8][4], float keep0 = 1.f, float keep1 = 1.f) {
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = fmaf(far[4 * n + i], i < 2 ? keep0 : keep1, o[n][i]);
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
// Two float32 values an instruction: what the warps issue is the bound beside the special functions, and packed arithmetic is half of it.
using pair = unsigned long long;
__device__ __forceinline__ pair both(float x, float y) {
  pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void parts(pair v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ pair add2(pair a, pair b) {
  pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair mul2(pair a, pair b) {
  pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair fma2(pair a, pair b, pair c) {
  pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// From products to scores without the distance, in units of log2: unit z, or unit tanh(x) with x = z to_cap.  tanh is up to a half an odd
// polynomial (fitted for the least relative error, 7.4e-8 in float32 arithmetic), above it 1 - 2 / (e^2x + 1).  Scores mostly stay below
// half the cap, and a warp whose tile does so needs no special function for them.  The polynomial's argument is x itself: to_cap may be
// anything from 0 to 1e24, and powers of it, as factors of the coefficients, leave the range of float32.  Both branches take the same steps
// for an x below a half, so that a score has the same bits whatever tile it is in, in the forward and in both backward passes.
constexpr float TANH3 = -0.333331435918808f, TANH5 = 0.13325878977775574f, TANH7 = -0.05304549261927605f, TANH9 = 0.01724148727953434f;
__device__ __forceinline__ float capped(float x, float unit) {
  const float y = fabsf(x), w = x * x, large = copysignf(1.f - __fdividef(2.f, exp2_fast(fminf(y * (2.f * LOG2E), 64.f)) + 1.f), x);
  const float z = x * unit, more = w * fmaf(w, fmaf(w, fmaf(w, TANH9, TANH7), TANH5), TANH3);
  return y <= 0.5f ? fmaf(z, more, z) : x == x ? unit * large : x;
}
template <int NT> __device__ __forceinline__ void cap_tile(float (&z)[NT][4], float unit, float to_cap, bool has_cap) {
  // The assembler joins a packed product with a packed addition that is its only use, rounding modifiers or not (measured).  These products have
  // another use in every pass (the row's maximum, the distance), so scores are rounded before the greatest is taken off, all alike.
  if (!has_cap) {
    const pair u = both(unit, unit);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) parts(mul2(both(z[n][2 * r], z[n][2 * r + 1]), u), z[n][2 * r], z[n][2 * r + 1]);
    return;
  }
  const pair to = both(to_cap, to_cap);
  float most = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int r = 0; r < 2; ++r) parts(mul2(both(z[n][2 * r], z[n][2 * r + 1]), to), z[n][2 * r], z[n][2 * r + 1]);
    most = fmaxf(fmaxf(most, fmaxf(fabsf(z[n][0]), fabsf(z[n][1]))), fmaxf(fabsf(z[n][2]), fabsf(z[n][3])));
  }
  if (__all_sync(0xffffffffu, most <= 0.5f)) {           // the maximum drops NaNs; they stay NaN either way
    const pair k0 = both(TANH3, TANH3), k1 = both(TANH5, TANH5), k2 = both(TANH7, TANH7), k3 = both(TANH9, TANH9), u = both(unit, unit);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const pair x = both(z[n][2 * r], z[n][2 * r + 1]), w = mul2(x, x), y = mul2(x, u);
        parts(fma2(y, mul2(w, fma2(w, fma2(w, fma2(w, k3, k2), k1), k0)), y), z[n][2 * r], z[n][2 * r + 1]);
      }
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) z[n][i] = capped(z[n][i], unit);
  }
}

// The way from a row to two columns, one over the distances and the distances.  One over is finite where two nodes coincide, so that
// the distance comes out as zero, and the way over it too.
struct Way { pair x, y, z, inverse, length; };
struct Place { pair x, y, z; };                          // of two columns, or twice that of a row
__device__ __forceinline__ Place columns_at(const float* columns, int stride) {
  return {*reinterpret_cast<const pair*>(columns), *reinterpret_cast<const pair*>(columns + stride), *reinterpret_cast<const pair*>(columns + 2 * stride)};
}
__device__ __forceinline__ Way way_to(const Place& columns, const Place& minus_row) {
  Way w;
  w.x = add2(columns.x, minus_row.x);
  w.y = add2(columns.y, minus_row.y);
  w.z = add2(columns.z, minus_row.z);
  const pair square = fma2(w.z, w.z, fma2(w.y, w.y, mul2(w.x, w.x)));
  float a, b;
  parts(square, a, b);
  w.inverse = both(rsqrt_fast(fmaxf(a, 1e-30f)), rsqrt_fast(fmaxf(b, 1e-30f)));
  w.length = mul2(square, w.inverse);
  return w;
}

__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

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

// Where a thread's pieces of an operand's rows begin, moved on from tile to tile by additions.
template <typename T, int DP, int TH> struct Source {
  const T* at;
  int64_t step;              // between the rows that the thread copies
  __device__ __forceinline__ Source(const Operand& x, const Piece<T, DP, TH>& piece, int first, int head, const AttentionParams& p)
      : at(static_cast<const T*>(x.p) + (int64_t)(first + piece.row) * x.node + piece.comp * x.comp + (int64_t)head * p.size + piece.channel),
        step(x.node * Piece<T, DP, TH>::ROWS) {}
};

// The next ROWS_TILE rows of one head to shared memory, zeros from the `left`-th on; `first` is the row of the first.
template <typename T, int DP, int TH, int ROWS_TILE>
__device__ __forceinline__ void load_rows(T* dst, Source<T, DP, TH>& source, const Operand& x, const Piece<T, DP, TH>& piece, int first, int left, int head,
                                          const AttentionParams& p, int tid) {
  constexpr int LD = Row<T, DP>::LD, ROWS = Piece<T, DP, TH>::ROWS;
  if (p.vec) {
    if (piece.there) {
      T* to = dst + piece.row * LD + piece.at;
      const T* from = source.at;
#pragma unroll
      for (int r = 0; r < ROWS_TILE; r += ROWS, from += source.step) {
        if (ROWS_TILE % ROWS && r + piece.row >= ROWS_TILE) break;
        const bool there = r + piece.row < left;
        copy16(to + r * LD, there ? from : static_cast<const T*>(x.p), there);
      }
    }
    source.at += x.node * ROWS_TILE;
    return;
  }
  const int d = p.comps * p.size;
  for (int i = tid; i < ROWS_TILE * d; i += TH) {
    const int r = i / d, j = i - r * d, m = j / p.size, c = j - m * p.size;
    dst[r * LD + j] = r < left ? static_cast<const T*>(x.p)[(int64_t)(first + r) * x.node + m * x.comp + (int64_t)head * p.size + c]
                               : static_cast<T>(0.f);
  }
}

// The 16 rows of a warp from the accumulators to shared memory and from there to (n, d, C), contiguous.
template <typename T, int DP>
__device__ __forceinline__ void store_rows(T* buf, void* out, const float (&o)[DP / 8][4], float f0, float f1, int first, int end, int head,
                                           const AttentionParams& p, int lane) {
  constexpr int LD = Row<T, DP>::LD;
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
    const Piece<T, DP, 32> piece(lane, p.comps, p.size);
    if (!piece.there) return;
    to += (int64_t)piece.comp * channels + piece.channel;
    for (int r = piece.row; r < 16 && first + r < end; r += Piece<T, DP, 32>::ROWS)
      *reinterpret_cast<uint4*>(to + (int64_t)(first + r) * p.comps * channels) = *reinterpret_cast<const uint4*>(buf + r * LD + piece.at);
    return;
  }
  for (int i = lane; i < 16 * d; i += 32) {
    const int r = i / d, j = i - r * d, m = j / p.size, c = j - m * p.size;
    if (first + r < end) to[((int64_t)(first + r) * p.comps + m) * channels + c] = buf[r * LD + j];
  }
}

// Sum over a head's values of g and the result, for rows g and g + 8 of a warp: four lanes a row.
template <typename T, int DP>
__device__ __forceinline__ void row_delta(const T* grads, int first, int end, int head, const AttentionParams& p, int lane, float (&delta)[2]) {
  constexpr int LD = Row<T, DP>::LD;
  const int g = lane >> 2, t = lane & 3, d = p.comps * p.size, channels = p.heads * p.size;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float sum = 0.f;
    if (first + g + 8 * r < end) {
      const T* o = static_cast<const T*>(p.out) + (int64_t)(first + g + 8 * r) * p.comps * channels + (int64_t)head * p.size;
      const T* a = grads + (g + 8 * r) * LD;
      constexpr int V = 16 / (int)sizeof(T);
      for (int j0 = t * V; j0 < d; j0 += 4 * V) {        // the same order of sums with any alignment
        if (p.vec) {
          const int m = j0 / p.size;
          const uint4 raw = *reinterpret_cast<const uint4*>(o + (int64_t)m * channels + j0 - m * p.size);
          const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
          for (int i = 0; i < V; ++i) sum += static_cast<float>(a[j0 + i]) * static_cast<float>(v[i]);
        } else {
          for (int j = j0; j < min(d, j0 + V); ++j) {
            const int m = j / p.size;
            sum += static_cast<float>(a[j]) * static_cast<float>(o[(int64_t)m * channels + j - m * p.size]);
          }
        }
      }
    }
    delta[r] = quad_sum(sum);
  }
}

// Positions of the rows [first, first + ROWS_TILE), all x, all y, all z, by all threads of the CTA.
template <int ROWS_TILE>
__device__ __forceinline__ void load_positions(float* dst, const float* pos, int first, int end) {
  for (int i = threadIdx.x; i < ROWS_TILE * 3; i += THREADS) {
    const int x = i / ROWS_TILE, r = i % ROWS_TILE;
    const bool there = first + r < end;
    copy4(dst + i, pos + (int64_t)(there ? first + r : 0) * 3 + x, there);
  }
}

// Minus the position of a row, each coordinate twice.
__device__ __forceinline__ Place minus_position(const float* pos, int row, int end) {
  float x = 0.f, y = 0.f, z = 0.f;
  if (row < end) x = -pos[(int64_t)row * 3], y = -pos[(int64_t)row * 3 + 1], z = -pos[(int64_t)row * 3 + 2];
  return {both(x, x), both(y, y), both(z, z)};
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

// CTAs an SM, here and below: as measured, against one more or fewer (forward, heads of 32: ragged graphs 167 us with 5, 175 with 6, 190 with
// 7, molecules 81, 76 and 74; backward, molecules: by rows 141 with 4, 158 with 3, 164 with 5).
template <typename T, int DP, int WR, int KT, bool FOLDS>
__global__ void __launch_bounds__(THREADS, DP <= 32 ? (WR == 4 ? 5 : sizeof(T) == 2 ? 7 : 6) : DP <= 64 ? 4 : 3) attention_forward_kernel(const __grid_constant__ AttentionParams p) {
  using S = Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int slot = warp / WR, ht = tid - slot * S::TH;                   // the head's place in the CTA, the thread's place in the head
  const unsigned groups = (p.heads + S::HEADS - 1) / S::HEADS;           // all heads of a tile first: the largest graphs' tiles come first
  const int head = (int)(blockIdx.x % groups) * S::HEADS + slot;
  const int4 tile = p.tiles[blockIdx.x / groups];
  const int first = tile.x, lo = tile.y, hi = tile.z;
  T* base = reinterpret_cast<T*>(smem) + slot * S::head_elements(1);
  T *rows = base, *stage = base + S::TILE * LD;
  float* spos = reinterpret_cast<float*>(smem + S::bytes(1, 0));         // two tiles of positions
  const bool here = head < p.heads;
  const int end = here ? hi : 0;                                         // a place without a head copies nothing
  if (p.comps * p.size < DP) {                                           // the columns behind the head's values stay zero
    for (size_t i = tid; i < S::bytes(1, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  const Piece<T, DP, S::TH> piece(ht, p.comps, p.size);
  Source<T, DP, S::TH> from_k(p.k, piece, lo, head, p), from_v(p.v, piece, lo, head, p);
  auto fetch = [&](int key, int s) {
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE, from_k, p.k, piece, key, end - key, head, p, ht);
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, from_v, p.v, piece, key, end - key, head, p, ht);
    if (p.pos) load_positions<KT>(spos + s * 3 * KT, p.pos, key, hi);
    copies_commit();
  };
  auto load_tile = [&](T* dst, const Operand& x) {       // the CTA's own rows
    Source<T, DP, S::TH> from(x, piece, first, head, p);
    load_rows<T, DP, S::TH, S::TILE>(dst, from, x, piece, first, end - first, head, p, ht);
  };
  load_tile(rows, p.q);
  fetch(lo, 0);

  const int row = first + (warp % WR) * 16;                              // of the warp
  const bool work = here && row < hi;
  const T* mine = rows + (warp % WR) * 16 * LD;
  float o[DP / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  const float to_cap = p.cap > 0.f ? p.scale / p.cap : 0.f, unit = (p.cap > 0.f ? p.cap : p.scale) * LOG2E;   // of a score: the tanh, or the product
  pair slope2 = 0;                                                       // minus the slope, twice, in units of log2
  Place at[2];
  if (p.pos) {
    const float f = here ? -p.slope[head] * LOG2E : 0.f;
    slope2 = both(f, f);
    at[0] = minus_position(p.pos, row + g, hi);
    at[1] = minus_position(p.pos, row + g + 8, hi);
  }
  Far<DP, 2> waiting;                                                    // and the greatest scores that it goes by
  auto keep_far = [&](const float* far, int r) { return exp2_fast(far[DP / 2 + r] - (top[r] == -INFINITY ? 0.f : top[r])); };
  int s = 0, key = lo;
  do {
    const int stop = FOLDS && hi - key > FOLD ? key + FOLD : hi;
    for (; key < stop; key += KT, s ^= 1) {
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
        cap_tile<NT>(z, unit, to_cap, p.cap > 0.f);
        if (p.pos) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const Place columns = columns_at(spos + s * 3 * KT + n * 8 + 2 * t, KT);
#pragma unroll
            for (int r = 0; r < 2; ++r)
              parts(fma2(way_to(columns, at[r]).length, slope2, both(z[n][2 * r], z[n][2 * r + 1])), z[n][2 * r], z[n][2 * r + 1]);
          }
        }
        if (key + KT > hi) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (key + n * 8 + 2 * t + i >= hi) z[n][i] = z[n][2 + i] = -INFINITY;
        }
        float most[2], keep[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float m = top[r];
#pragma unroll
          for (int n = 0; n < NT; ++n) m = fmaxf(m, fmaxf(z[n][2 * r], z[n][2 * r + 1]));
          most[r] = quad_max(m);
        }
        if (__any_sync(0xffffffffu, most[0] > top[0] || most[1] > top[1])) {             // the running sums have a new unit
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            keep[r] = exp2_fast(top[r] - (most[r] == -INFINITY ? 0.f : most[r]));
            sum[r] *= keep[r];
            top[r] = most[r];
          }
#pragma unroll
          for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= keep[i >> 1];
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float from = top[r] == -INFINITY ? 0.f : -top[r];
          const pair shift = both(from, from);
          pair add = 0;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float x, y;
            parts(add2(both(z[n][2 * r], z[n][2 * r + 1]), shift), x, y);
            z[n][2 * r] = exp2_fast(x);
            z[n][2 * r + 1] = exp2_fast(y);
            add = add2(add, both(z[n][2 * r], z[n][2 * r + 1]));
          }
          float x, y;
          parts(add, x, y);
          sum[r] += x + y;
        }
        out_mma<DP, NT>(o, z, vs, lane);
      }
      __syncthreads();
    }
    if (FOLDS && key < hi && work) {
      float* far = waiting.at();
      const bool first_time = key - lo == FOLD;
      fold<DP>(far, o, first_time, first_time ? 1.f : keep_far(far, 0), first_time ? 1.f : keep_far(far, 1));
      far[DP / 2] = top[0], far[DP / 2 + 1] = top[1];
    }
  } while (FOLDS && key < hi);
  if (!work) return;
  if (FOLDS && hi - lo > FOLD) {
    const float* far = waiting.at();
    unfold<DP>(far, o, keep_far(far, 0), keep_far(far, 1));
  }
  sum[0] = quad_sum(sum[0]);
  sum[1] = quad_sum(sum[1]);
  const float f0 = 1.f / sum[0], f1 = 1.f / sum[1];
  if (p.top && t == 0) {                                                 // apart: their sum would lose the logarithm beside a large score
    const int64_t to = (int64_t)head * p.n + row + g;
    if (row + g < hi) p.top[to] = top[0], p.inverse[to] = f0;
    if (row + g + 8 < hi) p.top[to + 8] = top[1], p.inverse[to + 8] = f1;
  }
  store_rows<T, DP>(const_cast<T*>(mine), p.out, o, f0, f1, row, hi, head, p, lane);
}

// Backward by rows: dq, delta, and with positions the rows' sums of dS r and dS u.  Weights are taken from the row's greatest score, and
// one over their sum follows at the end.
// bfloat16: dq goes by the delta of rounded weights and outputs, which are at hand; the columns' pass is given sum_j P dP, which is known at the
// end, and so do the sums for slopes and positions, float32 results, go: with w = r or u, sum_j dS w = sum_j P dP w - (sum_j P dP) (sum_j P w).
// As dq has that error already, its score gradients go into the product in two parts (one graph of 5001 nodes, 2-norm of the error: 2.75e-3
// with one part, 2.08e-3 with two, which cost 610 -> 666 us; a rounding of the result alone is 1.7e-3).
template <typename T, int DP, int WR, int KT, bool FOLDS, bool GEO, bool CAP>
__global__ void __launch_bounds__(THREADS, DP <= 32 ? 4 : DP <= 96 ? 3 : 2) attention_rows_kernel(const __grid_constant__ AttentionParams p) {
  using S = Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int slot = warp / WR, ht = tid - slot * S::TH;
  const unsigned groups = (p.heads + S::HEADS - 1) / S::HEADS;           // all heads of a tile first: the largest graphs' tiles come first
  const int head = (int)(blockIdx.x % groups) * S::HEADS + slot;
  const int4 tile = p.tiles[blockIdx.x / groups];
  const int first = tile.x, lo = tile.y, hi = tile.z;
  T* base = reinterpret_cast<T*>(smem) + slot * S::head_elements(2);
  T *rows = base, *grads = base + S::TILE * LD, *stage = base + 2 * S::TILE * LD;
  float* spos = reinterpret_cast<float*>(smem + S::bytes(2, 0));
  const bool here = head < p.heads;
  const int end = here ? hi : 0;
  if (p.comps * p.size < DP) {
    for (size_t i = tid; i < S::bytes(2, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  const Piece<T, DP, S::TH> piece(ht, p.comps, p.size);
  Source<T, DP, S::TH> from_k(p.k, piece, lo, head, p), from_v(p.v, piece, lo, head, p);
  auto fetch = [&](int key, int s) {
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE, from_k, p.k, piece, key, end - key, head, p, ht);
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, from_v, p.v, piece, key, end - key, head, p, ht);
    if (p.pos) load_positions<KT>(spos + s * 3 * KT, p.pos, key, hi);
    copies_commit();
  };
  auto load_tile = [&](T* dst, const Operand& x) {       // the CTA's own rows
    Source<T, DP, S::TH> from(x, piece, first, head, p);
    load_rows<T, DP, S::TH, S::TILE>(dst, from, x, piece, first, end - first, head, p, ht);
  };
  load_tile(rows, p.q);
  load_tile(grads, p.g);
  copies_commit();
  fetch(lo, 0);
  copies_wait<1>();
  __syncthreads();

  const int row = first + (warp % WR) * 16;
  const bool work = here && row < hi;
  const T *mq = rows + (warp % WR) * 16 * LD, *mg = grads + (warp % WR) * 16 * LD;
  float delta[2] = {0.f, 0.f}, top[2] = {INFINITY, INFINITY}, inverse[2] = {0.f, 0.f};
  if (work) row_delta<T, DP>(mg, row, hi, head, p, lane, delta);
  const bool is[2] = {work && row + g < hi, work && row + g + 8 < hi};
  const int64_t at = (int64_t)head * p.n + row + g;
  if (is[0]) top[0] = p.top[at], inverse[0] = p.inverse[at];
  if (is[1]) top[1] = p.top[at + 8], inverse[1] = p.inverse[at + 8];
  float dq[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) dq[n][0] = dq[n][1] = dq[n][2] = dq[n][3] = 0.f;
  pair geo[2][4], flat[2][4], all[2] = {0, 0};                             // sum dS w, or of P dP w; sum P w; sum P dP; two columns' each
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) geo[r][i] = flat[r][i] = 0;
  constexpr bool APART = sizeof(T) == 2;
  const float to_cap = CAP ? p.scale / p.cap : 0.f, unit = (CAP ? p.cap : p.scale) * LOG2E;   // of a score: the tanh, or the product
  const float bend = -1.f / (unit * unit);                                 // 1 - tanh^2, from unit tanh; the scale follows at the end
  const pair one2 = both(1.f, 1.f), bend2 = both(bend, bend);
  pair slope2 = 0;
  Place place[2];
  if (p.pos) {
    const float f = here ? -p.slope[head] * LOG2E : 0.f;
    slope2 = both(f, f);
    place[0] = minus_position(p.pos, row + g, hi);
    place[1] = minus_position(p.pos, row + g + 8, hi);
  }
  Far<DP> waiting;
  int s = 0, key = lo;
  do {
    const int stop = FOLDS && hi - key > FOLD ? key + FOLD : hi;
    for (; key < stop; key += KT, s ^= 1) {
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
        cap_tile<NT>(z, unit, to_cap, CAP);
        const bool last = key + KT > hi;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          Place columns;
          if (p.pos) columns = columns_at(spos + s * 3 * KT + n * 8 + 2 * t, KT);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const pair score0 = both(z[n][2 * r], z[n][2 * r + 1]), d = both(dp[n][2 * r], dp[n][2 * r + 1]);
            pair score = score0;
            Way v;
            if (p.pos) {
              v = way_to(columns, place[r]);
              score = fma2(v.length, slope2, score);
            }
            float x, y;
            parts(add2(score, both(-top[r], -top[r])), x, y);
            if (last) {
              if (key + n * 8 + 2 * t >= hi) x = -INFINITY;
              if (key + n * 8 + 2 * t + 1 >= hi) y = -INFINITY;
            }
            const pair w = both(exp2_fast(x), exp2_fast(y)), e = mul2(w, add2(d, both(-delta[r], -delta[r])));
            if (APART) all[r] = fma2(w, d, all[r]);
            if (GEO) {
              const pair f = APART ? mul2(w, d) : e, fi = mul2(f, v.inverse), wi = mul2(w, v.inverse);
              if (APART) {
                flat[r][0] = fma2(w, v.length, flat[r][0]);
                flat[r][1] = fma2(wi, v.x, flat[r][1]);
                flat[r][2] = fma2(wi, v.y, flat[r][2]);
                flat[r][3] = fma2(wi, v.z, flat[r][3]);
              }
              geo[r][0] = fma2(f, v.length, geo[r][0]);
              geo[r][1] = fma2(fi, v.x, geo[r][1]);
              geo[r][2] = fma2(fi, v.y, geo[r][2]);
              geo[r][3] = fma2(fi, v.z, geo[r][3]);
            }
            pair dz = e;                                                   // without a cap a score may be minus infinity, its weight zero
            if (CAP) dz = mul2(e, fma2(mul2(score0, bend2), score0, one2));
            parts(dz, z[n][2 * r], z[n][2 * r + 1]);
          }
        }
        out_mma<DP, NT, true>(dq, z, ks, lane);
      }
      __syncthreads();
    }
    if (FOLDS && key < hi && work) fold<DP>(waiting.at(), dq, key - lo == FOLD);
  } while (FOLDS && key < hi);
  if (!work) return;
  if (FOLDS && hi - lo > FOLD) unfold<DP>(waiting.at(), dq);
  if (APART) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float x, y;
      parts(all[r], x, y);
      delta[r] = quad_sum(x + y) * inverse[r];
    }
  }
  if (GEO) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float x, y, sums[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        parts(geo[r][i], x, y);
        sums[i] = quad_sum(x + y);
        if (APART) {
          parts(flat[r][i], x, y);
          sums[i] -= delta[r] * quad_sum(x + y);
        }
        sums[i] *= inverse[r];
      }
      const float4 v = make_float4(sums[0], -sums[1], -sums[2], -sums[3]);   // u points from the column to the row
      if (is[r] && t == 0) p.geo_row[at + 8 * r] = v;
    }
  }
  if (t == 0) {
    if (is[0]) p.delta[at] = delta[0];
    if (is[1]) p.delta[at + 8] = delta[1];
  }
  store_rows<T, DP>(const_cast<T*>(mq), p.dq, dq, p.scale * inverse[0], p.scale * inverse[1], row, hi, head, p, lane);
}

// Backward by columns: dk, dv, and with positions the columns' sums of dS u.  The CTA's rows are keys; queries and the output's
// gradients come by in tiles, and the products are the transposed ones.
template <typename T, int DP, int WR, int KT, bool FOLDS, bool GEO, bool CAP>
__global__ void __launch_bounds__(THREADS, DP <= 32 ? 4 : DP <= 64 ? 3 : 2) attention_columns_kernel(const __grid_constant__ AttentionParams p) {
  using S = Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int slot = warp / WR, ht = tid - slot * S::TH;
  const unsigned groups = (p.heads + S::HEADS - 1) / S::HEADS;           // all heads of a tile first: the largest graphs' tiles come first
  const int head = (int)(blockIdx.x % groups) * S::HEADS + slot;
  const int4 tile = p.tiles[blockIdx.x / groups];
  const int first = tile.x, lo = tile.y, hi = tile.z;
  T* base = reinterpret_cast<T*>(smem) + slot * S::head_elements(2);
  T *keys = base, *values = base + S::TILE * LD, *stage = base + 2 * S::TILE * LD;
  float* spos = reinterpret_cast<float*>(smem + S::bytes(2, 0));
  float* stats = spos + 6 * KT + slot * 6 * KT;           // [tile][top, inverse, delta][KT]
  const bool here = head < p.heads;
  const int end = here ? hi : 0;
  if (p.comps * p.size < DP) {
    for (size_t i = tid; i < S::bytes(2, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  const Piece<T, DP, S::TH> piece(ht, p.comps, p.size);
  Source<T, DP, S::TH> from_q(p.q, piece, lo, head, p), from_g(p.g, piece, lo, head, p);
  auto fetch = [&](int query, int s) {
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE, from_q, p.q, piece, query, end - query, head, p, ht);
    load_rows<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, from_g, p.g, piece, query, end - query, head, p, ht);
    for (int i = ht; i < KT; i += S::TH) {
      const bool there = query + i < end;
      const int64_t at = there ? (int64_t)head * p.n + query + i : 0;
      copy4(stats + (3 * s) * KT + i, p.top + at, there);
      copy4(stats + (3 * s + 1) * KT + i, p.inverse + at, there);
      copy4(stats + (3 * s + 2) * KT + i, p.delta + at, there);
    }
    if (p.pos) load_positions<KT>(spos + s * 3 * KT, p.pos, query, hi);
    copies_commit();
  };
  auto load_tile = [&](T* dst, const Operand& x) {       // the CTA's own rows
    Source<T, DP, S::TH> from(x, piece, first, head, p);
    load_rows<T, DP, S::TH, S::TILE>(dst, from, x, piece, first, end - first, head, p, ht);
  };
  load_tile(keys, p.k);
  load_tile(values, p.v);
  fetch(lo, 0);

  const int row = first + (warp % WR) * 16;
  const bool work = here && row < hi;
  const T *mk = keys + (warp % WR) * 16 * LD, *mv = values + (warp % WR) * 16 * LD;
  float dk[DP / 8][4], dv[DP / 8][4];
  pair geo[2][3] = {{0, 0, 0}, {0, 0, 0}};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    dk[n][0] = dk[n][1] = dk[n][2] = dk[n][3] = 0.f;
    dv[n][0] = dv[n][1] = dv[n][2] = dv[n][3] = 0.f;
  }
  const float to_cap = CAP ? p.scale / p.cap : 0.f, unit = (CAP ? p.cap : p.scale) * LOG2E;
  const float bend = -1.f / (unit * unit);
  const pair one2 = both(1.f, 1.f), bend2 = both(bend, bend), minus = both(-1.f, -1.f);
  pair slope2 = 0;
  Place place[2];
  if (p.pos) {
    const float f = here ? -p.slope[head] * LOG2E : 0.f;
    slope2 = both(f, f);
    place[0] = minus_position(p.pos, row + g, hi);
    place[1] = minus_position(p.pos, row + g + 8, hi);
  }
  Far<DP> waiting_k, waiting_v;
  int s = 0, query = lo;
  do {
    const int stop = FOLDS && hi - query > FOLD ? query + FOLD : hi;
    for (; query < stop; query += KT, s ^= 1) {
      if (query + KT < hi) {
        fetch(query + KT, s ^ 1);
        copies_wait<1>();
      } else {
        copies_wait<0>();
      }
      __syncthreads();
      if (work) {
        const T *qs = stage + s * S::STAGE, *gs = qs + KT * LD;
        const float* st = stats + 3 * s * KT;
        float z[NT][4], dp[NT][4];
        score_mma<DP, NT, true>(z, mk, qs, lane);
        score_mma<DP, NT, true>(dp, mv, gs, lane);
        cap_tile<NT>(z, unit, to_cap, CAP);
        const bool last = query + KT > hi;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int c = n * 8 + 2 * t;
          const pair top = *reinterpret_cast<const pair*>(st + c), inverse = *reinterpret_cast<const pair*>(st + KT + c),
                     delta = *reinterpret_cast<const pair*>(st + 2 * KT + c);
          Place columns;
          if (p.pos) columns = columns_at(spos + s * 3 * KT + c, KT);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const pair score0 = both(z[n][2 * r], z[n][2 * r + 1]), d = both(dp[n][2 * r], dp[n][2 * r + 1]);
            pair score = score0;
            Way v;
            if (p.pos) {                                                   // from the key to the query
              v = way_to(columns, place[r]);
              score = fma2(v.length, slope2, score);
            }
            float x, y;
            parts(fma2(top, minus, score), x, y);
            if (last) {
              if (query + c >= hi) x = -INFINITY;
              if (query + c + 1 >= hi) y = -INFINITY;
            }
            const pair w = mul2(both(exp2_fast(x), exp2_fast(y)), inverse), e = mul2(w, fma2(delta, minus, d));
            if (GEO) {
              const pair ei = mul2(e, v.inverse);
              geo[r][0] = fma2(ei, v.x, geo[r][0]);
              geo[r][1] = fma2(ei, v.y, geo[r][1]);
              geo[r][2] = fma2(ei, v.z, geo[r][2]);
            }
            parts(w, z[n][2 * r], z[n][2 * r + 1]);
            pair dz = e;
            if (CAP) dz = mul2(e, fma2(mul2(score0, bend2), score0, one2));
            parts(dz, dp[n][2 * r], dp[n][2 * r + 1]);
          }
        }
        out_mma<DP, NT>(dv, z, gs, lane);
        out_mma<DP, NT>(dk, dp, qs, lane);
      }
      __syncthreads();
    }
    if (FOLDS && query < hi && work) {
      fold<DP>(waiting_k.at(), dk, query - lo == FOLD);
      fold<DP>(waiting_v.at(), dv, query - lo == FOLD);
    }
  } while (FOLDS && query < hi);
  if (!work) return;
  if (FOLDS && hi - lo > FOLD) {
    unfold<DP>(waiting_k.at(), dk);
    unfold<DP>(waiting_v.at(), dv);
  }
  if (GEO) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float x, y, sums[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        parts(geo[r][i], x, y);
        sums[i] = quad_sum(x + y);
      }
      const float4 v = make_float4(0.f, sums[0], sums[1], sums[2]);
      if (t == 0 && row + g + 8 * r < hi) p.geo_col[(int64_t)head * p.n + row + g + 8 * r] = v;
    }
  }
  store_rows<T, DP>(const_cast<T*>(mk), p.dk, dk, p.scale, p.scale, row, hi, head, p, lane);
  store_rows<T, DP>(const_cast<T*>(mv), p.dv, dv, 1.f, 1.f, row, hi, head, p, lane);
}

// ---- host side ----------------------------------------------------------------------------------
enum Pass { FORWARD, ROWS, COLUMNS };

// KF and KB: keys, or queries, of a tile in the forward and in the backward pass
template <typename T, int DP, int WR, int KF, int KB, bool FOLDS = false>
int launch(Pass pass, const AttentionParams& p, int64_t tiles, bool geo, cudaStream_t s) {
  using F = Shape<T, DP, WR, KF>;
  using B = Shape<T, DP, WR, KB>;
  const int64_t ctas = tiles * ceil_div(p.heads, F::HEADS);
  if (ctas > INT32_MAX) return fail(EQT_ERR_UNSUPPORTED, "attention: %lld tiles and heads are more than one launch takes", (long long)ctas);
  const unsigned grid = (unsigned)ctas;
  static std::atomic<uint64_t> allowed[9];                               // of the kernels below
  auto run = [&](auto kernel, size_t bytes, const char* what, int which) {
    if (int rc = allow_shared_once(kernel, bytes, allowed[which])) return rc;
    kernel<<<grid, THREADS, bytes, s>>>(p);
    return check_launch(what);
  };
  constexpr int POSITIONS = 2 * 12 * KB, STATS = B::HEADS * 24 * KB;     // two tiles each
  if (pass == FORWARD) return run(attention_forward_kernel<T, DP, WR, KF, FOLDS>, F::bytes(1, 2 * 12 * KF), "attention_forward", 0);
  const bool cap = p.cap > 0.f;
  const int which = 2 * geo + cap;
  if (pass == ROWS) {
    constexpr size_t bytes = B::bytes(2, POSITIONS);
    if (geo) return cap ? run(attention_rows_kernel<T, DP, WR, KB, FOLDS, true, true>, bytes, "attention_rows", 1 + which)
                        : run(attention_rows_kernel<T, DP, WR, KB, FOLDS, true, false>, bytes, "attention_rows", 1 + which);
    return cap ? run(attention_rows_kernel<T, DP, WR, KB, FOLDS, false, true>, bytes, "attention_rows", 1 + which)
               : run(attention_rows_kernel<T, DP, WR, KB, FOLDS, false, false>, bytes, "attention_rows", 1 + which);
  }
  constexpr size_t bytes = B::bytes(2, POSITIONS + STATS);
  if (geo) return cap ? run(attention_columns_kernel<T, DP, WR, KB, FOLDS, true, true>, bytes, "attention_columns", 5 + which)
                      : run(attention_columns_kernel<T, DP, WR, KB, FOLDS, true, false>, bytes, "attention_columns", 5 + which);
  return cap ? run(attention_columns_kernel<T, DP, WR, KB, FOLDS, false, true>, bytes, "attention_columns", 5 + which)
             : run(attention_columns_kernel<T, DP, WR, KB, FOLDS, false, false>, bytes, "attention_columns", 5 + which);
}

template <typename T, int DP>
int launch_rows(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s) {
  // Wide heads, float32 and the backward pass need the registers; float32's backward pass also the shared memory (48 graphs of 40 to
  // 250 nodes, heads of 72 values: by rows 184 us with 32, 170 with 16, by columns the same).
  constexpr int KF = sizeof(T) == 2 && DP <= 64 ? 64 : 32, KB = sizeof(T) == 2 ? 32 : 16;
  if constexpr (sizeof(T) == 2) {
    if (p.folds) return launch<T, DP, 4, KF, KB, true>(pass, p, tiles, geo, s);
  }
  if (tile_rows == 64) return launch<T, DP, 4, KF, KB>(pass, p, tiles, geo, s);
  if (tile_rows == 32) return launch<T, DP, 2, 32, 32>(pass, p, tiles, geo, s);
  return launch<T, DP, 1, 16, 16>(pass, p, tiles, geo, s);
}

template <typename T>
int launch_width(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s) {
  const int d = p.comps * p.size;
  if (d <= 32) return launch_rows<T, 32>(pass, p, tiles, tile_rows, geo, s);
  if (d <= 64) return launch_rows<T, 64>(pass, p, tiles, tile_rows, geo, s);
  if (d <= 80) return launch_rows<T, 80>(pass, p, tiles, tile_rows, geo, s);       // nine components of eight channels
  if (d <= 96) return launch_rows<T, 96>(pass, p, tiles, tile_rows, geo, s);
  return launch_rows<T, 128>(pass, p, tiles, tile_rows, geo, s);
}

// Defined in graph_attention_f32.cu and graph_attention_bf16.cu, which compile side by side.
int launch_f32(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s);
int launch_bf16(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s);

}  // namespace attention
}  // namespace eqt
