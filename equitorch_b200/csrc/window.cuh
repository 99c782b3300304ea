// Attention within windows of packed chains: what its kernels share.
//
// Node i of a chain [lo, hi) sees the nodes j of it with  j <= i + after  and  (j >= i - before  or  j < lo + sinks):
//
//     s_ij = scale <q_i, k_j>      P_ij = exp(s_ij) / sum_j exp(s_ij)      out_i = sum_j P_ij v_j
//     dP_ij = <g_i, v_j>           delta_i = sum_j P_ij dP_ij              dS_ij = P_ij (dP_ij - delta_i)
//     dv_j = sum_i P_ij g_i        dq_i = scale sum_j dS_ij k_j            dk_j = scale sum_i dS_ij q_i
//
// over the heads that share k and v, for dk and dv.
//
// Where a weight is almost one, dP - delta is what two such numbers leave, and delta has to be that of the very weights: sum_j P_ij dP_ij.  bfloat16 weights are
// rounded for their product with v, so the forward pass divides by the sum of the rounded ones and keeps what the rounding of its result left; the rows' pass takes
// the same rounded weights, whose delta is <g, out + rest>.  The forward pass rounds a weight in the unit that its row has at that moment,
// so a row's units differ by whole powers of two.  On its way it sums P, and P dP, of the weights before rounding, by which the columns go.
//
// A tile's products run over nodes that some of its rows do not see, with weights of zero, and zero times infinity or a NaN is a NaN.  So a row whose
// result is not finite is done again, one visible node at a time (`again_*`): a NaN that is not seen does not reach it, and one that is seen does.
#pragma once

#include "graph_attention.cuh"

namespace eqt {
namespace window {
using attention::AttentionParams;
using attention::Operand;
using attention::exp2_fast;
using attention::LOG2E;

struct WindowParams {
  AttentionParams q, kv;     // of the heads of queries; of the heads of keys (dk and dv)
  int before, after, sinks, group;
  // Gradients of the first nodes of long chains from queries behind their windows, made apart (SPLIT) because a chain may have any number of those: sums of dS q and of P g
  // by blocks of FAR_BLOCK nodes of the batch, [pair of a block and a chain][head of keys][16 first nodes][dk, dv][node][value], then joined in the chain's first place.
  void* rest;                // what the rounding of the results left (bfloat16, for the backward pass)
  float* inverse;            // [head][node]: one over the sum of weights as the columns have them, not rounded
  const int64_t* ptr;
  int64_t chains;
  float* far;
  int split, apart;          // apart: nodes of a chain from which it is such a long one, none where not SPLIT
  int folds_rows, folds_columns;   // bfloat16: sums of results and dq, and of dk and dv, of more than FOLD terms
};
constexpr int FAR_BLOCK = 512, FAR_ROWS = 16, MOST_SPLIT_SINKS = 64;
__host__ __device__ inline int far_groups(const WindowParams& p) { return (p.sinks + FAR_ROWS - 1) / FAR_ROWS; }
// Chains of at least that many nodes start so far from one another that no two have the same slot, start / far_length, so places go by the nodes and not by the chains, of which
// a batch may have any number; a block b and a chain of slot g that has nodes in it are pair b + g, which no other two are: going on, the block or the slot moves on.
__host__ __device__ inline int far_length(const WindowParams& p) { return p.before + 1 + FAR_BLOCK; }
__host__ __device__ inline int64_t far_slots(const WindowParams& p) { return p.q.n / far_length(p) + 1; }
__host__ __device__ inline int64_t far_pairs(const WindowParams& p) { return (p.q.n + FAR_BLOCK - 1) / FAR_BLOCK + far_slots(p); }
__device__ __forceinline__ bool apart(const WindowParams& p, int lo, int hi) { return hi - lo >= p.apart; }
__device__ __forceinline__ int64_t far_place(const WindowParams& p, int64_t pair, int kv, int group) {
  return ((pair * p.kv.heads + kv) * far_groups(p) + group) * (2 * FAR_ROWS * (int64_t)(p.q.comps * p.q.size));
}
// The last chain g with `of(g)` at most `x`, `of` ascending; -1 if there is none.
template <typename F> __device__ __forceinline__ int64_t last_chain(int64_t chains, int64_t x, F of) {
  int64_t lo = -1, hi = chains - 1;
  while (lo < hi) {
    const int64_t mid = lo + (hi - lo + 1) / 2;
    if (of(mid) <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// What queries behind its window give a first node j of the chain [lo, hi): dk, with dv FAR_ROWS rows on; none: NULL.
__device__ __forceinline__ const float* far_of(const WindowParams& p, int j, int kv, int lo, int hi) {
  if (!apart(p, lo, hi) || j >= lo + p.sinks || j + p.before + 1 >= hi) return nullptr;
  const int group = (j - lo) / FAR_ROWS, first = lo + group * FAR_ROWS;
  return p.far + far_place(p, (first + p.before + 1) / FAR_BLOCK + lo / far_length(p), kv, group) + (int64_t)(j - first) * (p.q.comps * p.q.size);
}

__device__ __forceinline__ bool sees(const WindowParams& p, int i, int j, int lo) { return j <= i + p.after && (j >= i - p.before || j < lo + p.sinks); }

// A lane's values (every 32nd) of a head's row; and of an operand with contiguous rows of `heads` heads.
template <typename T> __device__ __forceinline__ void lane_row(float (&v)[4], const Operand& x, int node, int head, const AttentionParams& p, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int e = lane + 32 * c, comp = e / p.size;
    v[c] = comp < p.comps ? static_cast<float>(static_cast<const T*>(x.p)[node * x.node + comp * x.comp + (int64_t)head * p.size + e - comp * p.size]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void lane_put(void* out, const float (&v)[4], float f, int node, int head, const AttentionParams& p, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int e = lane + 32 * c, comp = e / p.size;
    if (comp < p.comps) st(static_cast<T*>(out) + (((int64_t)node * p.comps + comp) * p.heads + head) * p.size + e - comp * p.size, v[c] * f);
  }
}
__device__ __forceinline__ float lanes_dot(const float (&a)[4], const float (&b)[4]) {
  float s = a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// One row, by a warp.
template <typename T> __device__ __noinline__ void again_forward(const WindowParams& p, int i, int head, int lo, int hi, int lane) {
  const int kv = head / p.group;
  float q[4], k[4], v[4], o[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, sum = 0.f;
  lane_row<T>(q, p.q.q, i, head, p.q, lane);
  const int end = (int)min((int64_t)hi, (int64_t)i + p.after + 1);
  for (int j = lo; j < end; ++j) {
    if (j >= lo + p.sinks && j < i - p.before) j = i - p.before;
    lane_row<T>(k, p.q.k, j, kv, p.q, lane);
    lane_row<T>(v, p.q.v, j, kv, p.q, lane);
    const float s = lanes_dot(q, k) * (p.q.scale * LOG2E), now = fmaxf(top, s), base = now == -INFINITY ? 0.f : now;
    const float keep = exp2_fast(top - base), w = exp2_fast(s - base);
    sum = sum * keep + w;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = w == 0.f ? o[c] * keep : fmaf(w, v[c], o[c] * keep);      // a score of minus infinity is no part of the sum
    top = now;
  }
  lane_put<T>(p.q.out, o, 1.f / sum, i, head, p.q, lane);
  if (!p.rest) return;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float x = o[c] / sum;
    o[c] = x - static_cast<float>(static_cast<T>(x));
  }
  lane_put<T>(p.rest, o, 1.f, i, head, p.q, lane);
}
template <typename T> __device__ __noinline__ void again_rows(const WindowParams& p, int i, int head, int lo, int hi, int lane) {
  const int kv = head / p.group;
  const int64_t at = (int64_t)head * p.q.n + i;
  const float top = p.q.top[at], inverse = p.inverse[at], delta = p.q.delta[at];
  float q[4], k[4], v[4], g[4], dq[4] = {0.f, 0.f, 0.f, 0.f};
  lane_row<T>(q, p.q.q, i, head, p.q, lane);
  lane_row<T>(g, p.q.g, i, head, p.q, lane);
  const int end = (int)min((int64_t)hi, (int64_t)i + p.after + 1);
  for (int j = lo; j < end; ++j) {
    if (j >= lo + p.sinks && j < i - p.before) j = i - p.before;
    lane_row<T>(k, p.q.k, j, kv, p.q, lane);
    lane_row<T>(v, p.q.v, j, kv, p.q, lane);
    const float w = exp2_fast(lanes_dot(q, k) * (p.q.scale * LOG2E) - top) * inverse, ds = w * (lanes_dot(g, v) - delta);
#pragma unroll
    for (int c = 0; c < 4; ++c) dq[c] = fmaf(ds, k[c], dq[c]);
  }
  lane_put<T>(p.q.dq, dq, p.q.scale, i, head, p.q, lane);
}
template <typename T> __device__ __noinline__ void again_columns(const WindowParams& p, int j, int kv, int lo, int hi, int lane, bool put_dv = true, bool put_dk = true) {
  float q[4], k[4], v[4], g[4], dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
  lane_row<T>(k, p.q.k, j, kv, p.q, lane);
  lane_row<T>(v, p.q.v, j, kv, p.q, lane);
  const int start = (int)max((int64_t)lo, (int64_t)j - p.after), end = j < lo + p.sinks ? hi : (int)min((int64_t)hi, (int64_t)j + p.before + 1);
  for (int head = kv * p.group; head < (kv + 1) * p.group; ++head)
    for (int i = start; i < end; ++i) {
      const int64_t at = (int64_t)head * p.q.n + i;
      lane_row<T>(q, p.q.q, i, head, p.q, lane);
      lane_row<T>(g, p.q.g, i, head, p.q, lane);
      const float w = exp2_fast(lanes_dot(q, k) * (p.q.scale * LOG2E) - p.q.top[at]) * p.inverse[at], ds = w * (lanes_dot(g, v) - p.q.delta[at]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        dv[c] = fmaf(w, g[c], dv[c]);
        dk[c] = fmaf(ds, q[c], dk[c]);
      }
    }
  if (put_dk) lane_put<T>(p.kv.dk, dk, p.q.scale, j, kv, p.kv, lane);
  if (put_dv) lane_put<T>(p.kv.dv, dv, 1.f, j, kv, p.kv, lane);
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }

int far_bf16(const WindowParams& p, cudaStream_t s);                                                             // window_f32.cu and window_bf16.cu
int tiles_forward_f32(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s);
int tiles_forward_bf16(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s);
int tiles_backward_f32(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s);
int tiles_backward_bf16(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s);

}  // namespace window
}  // namespace eqt
