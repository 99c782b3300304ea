// Attention within windows by tiles of one chain (16 to 64 nodes, as for attention within whole graphs), on the warp-wide matrix instructions: any
// type, alignment and length of chains.  One pass over the visible keys forward; the backward pass once by rows (dq, delta) and once by
// columns (dk, dv, over the heads that share them); every result is written by one warp and sums have one order.
//
// A tile walks two stretches of keys, the chain's first ones and those of its rows' windows, so its work goes by the window, not by the chain.  What a
// tile of 64 rows sees of 64 + before + after keys it uses in full but for the two triangles at its ends.  32 chains of 30 float32 nodes: 48 us for three kernels and
// the call bound by the host; bfloat16 that the 5th-generation tensor cores take (window_tc.cu) come here only unaligned, or with a scale that is not positive.
#pragma once

#include <algorithm>

#include "window.cuh"

namespace eqt {
namespace window {
namespace {
using namespace attention;

// The other side's rows that a tile meets, as steps of KT: [from0, to0), then [from1, to1).
struct Walk {
  int from0, to0, from1, to1, steps0, steps;
  template <int KT> __device__ __forceinline__ void set() {
    steps0 = max(0, (to0 - from0 + KT - 1) / KT);
    steps = steps0 + max(0, (to1 - from1 + KT - 1) / KT);
  }
  template <int KT> __device__ __forceinline__ int at(int step, int& end) const {
    const bool second = step >= steps0;
    end = second ? to1 : to0;
    return second ? from1 + (step - steps0) * KT : from0 + step * KT;
  }
};
__device__ __forceinline__ Walk keys_of(const WindowParams& p, int first, int last, int lo, int hi) {        // rows [first, last)
  Walk w;
  w.from1 = max(lo, first - p.before);
  w.to1 = min(hi, last + p.after);
  w.from0 = lo;
  w.to0 = min(w.from1, lo + p.sinks);
  return w;
}
__device__ __forceinline__ Walk queries_of(const WindowParams& p, int first, int last, int lo, int hi) {     // keys [first, last)
  Walk w;
  w.from0 = w.to0 = lo;
  w.from1 = max(lo, first - p.after);
  w.to1 = first < lo + p.sinks && !apart(p, lo, hi) ? hi : min(hi, last + p.before);
  return w;
}

template <typename T, int DP, int TH, int ROWS> __device__ __forceinline__ void load_tile(T* dst, const Operand& x, int first, int left, int head, const AttentionParams& p, int ht) {
  const Piece<T, DP, TH> piece(ht, p.comps, p.size);
  Source<T, DP, TH> from(x, piece, first, head, p);
  load_rows<T, DP, TH, ROWS>(dst, from, x, piece, first, left, head, p, ht);
}

// Rows of a warp whose results are not finite: bits of row g in `bad[0]`, of row g + 8 in `bad[1]`, four lanes a row.
template <int N> __device__ __forceinline__ bool finite_rows(const float (&o)[N][4], int r) {
  bool ok = true;
#pragma unroll
  for (int n = 0; n < N; ++n) ok = ok && is_finite(o[n][2 * r]) && is_finite(o[n][2 * r + 1]);
  return ok;
}
template <typename F> __device__ __forceinline__ void each_bad_row(bool bad0, bool bad1, int row, int end, F again) {
  const unsigned b0 = __ballot_sync(0xffffffffu, bad0), b1 = __ballot_sync(0xffffffffu, bad1);
  if (!(b0 | b1)) return;
  __syncwarp();
  for (int r = 0; r < 16; ++r)
    if ((((r < 8 ? b0 : b1) >> (4 * (r & 7))) & 15) && row + r < end) again(row + r);
}

// Whether the sums of bfloat16 products are taken out of the matrix instructions before a step, so that they are of at most FOLD terms.
template <int KT> __device__ __forceinline__ bool fold_now(int step) { return step > 0 && step % (FOLD / KT) == 0; }

template <typename T> __device__ __forceinline__ float rounded(float x) { return sizeof(T) == 4 ? x : __bfloat162float(__float2bfloat16_rn(x)); }

template <typename T, int DP, int WR, int KT, bool FOLDS>
__global__ void __launch_bounds__(THREADS, DP <= 64 ? 4 : 3) window_forward_kernel(const __grid_constant__ WindowParams p) {
  using S = attention::Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, slot = warp / WR, ht = tid - slot * S::TH;
  const unsigned groups = (p.q.heads + S::HEADS - 1) / S::HEADS;
  const int head = (int)(blockIdx.x % groups) * S::HEADS + slot;
  const int4 tile = p.q.tiles[blockIdx.x / groups];
  const int first = tile.x, lo = tile.y, hi = tile.z, last = min(hi, first + S::TILE);
  T *rows = reinterpret_cast<T*>(smem) + slot * S::head_elements(1), *stage = rows + S::TILE * LD;
  const bool here = head < p.q.heads;
  const int kv = here ? head / p.group : 0;
  if (p.q.comps * p.q.size < DP) {                       // the columns behind the head's values stay zero
    for (size_t i = tid; i < S::bytes(1, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  Walk walk = keys_of(p, first, last, lo, hi);
  walk.set<KT>();
  auto fetch = [&](int step, int s) {
    int end;
    const int key = walk.at<KT>(step, end);
    load_tile<T, DP, S::TH, KT>(stage + s * S::STAGE, p.q.k, key, here ? end - key : 0, kv, p.q, ht);
    load_tile<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, p.q.v, key, here ? end - key : 0, kv, p.q, ht);
    copies_commit();
  };
  load_tile<T, DP, S::TH, S::TILE>(rows, p.q.q, first, here ? hi - first : 0, here ? head : 0, p.q, ht);
  fetch(0, 0);
  const int row = first + (warp % WR) * 16;
  const bool work = here && row < hi;
  const T* mine = rows + (warp % WR) * 16 * LD;
  const float unit = p.q.scale * LOG2E;
  float o[DP / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, kept[2] = {1.f, 1.f};
  Far<FOLDS ? DP : 2> waiting;                           // FOLDS: the sums of the steps before, in a unit that was `kept` times as great
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  for (int step = 0, s = 0; step < walk.steps; ++step, s ^= 1) {
    if constexpr (FOLDS) {
      if (fold_now<KT>(step) && work) {
        fold<DP>(waiting.at(), o, step == FOLD / KT, kept[0], kept[1]);
        kept[0] = kept[1] = 1.f;
      }
    }
    if (step + 1 < walk.steps) {
      fetch(step + 1, s ^ 1);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncthreads();
    int end;
    const int key = walk.at<KT>(step, end);
    // a warp whose rows see none of the keys has nothing to do
    if (work && key <= row + 15 + p.after && (key + KT > row - p.before || key < lo + p.sinks)) {
      const T *ks = stage + s * S::STAGE, *vs = ks + KT * LD;
      float z[NT][4];
      score_mma<DP, NT>(z, mine, ks, lane);
      const bool all = key + KT <= end && key + KT - 1 <= row + p.after && key >= row + 15 - p.before;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = key + n * 8 + 2 * t + (i & 1);
          z[n][i] = all || (j < end && sees(p, row + g + 8 * (i >> 1), j, lo)) ? z[n][i] * unit : -INFINITY;
        }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float most = top[r];
#pragma unroll
        for (int n = 0; n < NT; ++n) most = fmaxf(most, fmaxf(z[n][2 * r], z[n][2 * r + 1]));
        most = quad_max(most);
        if constexpr (sizeof(T) == 2) {                  // by whole steps, if float32 has the step: a weight's rounding is the same in any unit
          const float rise = most - top[r];
          if (rise > 0.f && rise < INFINITY) most = top[r] + ceilf(rise);
        }
        const float base = most == -INFINITY ? 0.f : most, keep = exp2_fast(top[r] - base);
        float add = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            z[n][2 * r + i] = rounded<T>(exp2_fast(z[n][2 * r + i] - base));
            add += z[n][2 * r + i];
          }
        sum[r] = sum[r] * keep + add;
        if (FOLDS) kept[r] *= keep;
        top[r] = most;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) o[n][2 * r] *= keep, o[n][2 * r + 1] *= keep;
      }
      out_mma<DP, NT>(o, z, vs, lane);
    }
    __syncthreads();
  }
  if (!work) return;
  if constexpr (FOLDS)
    if (walk.steps > FOLD / KT) unfold<DP>(waiting.at(), o, kept[0], kept[1]);
  float f[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) f[r] = 1.f / quad_sum(sum[r]);
  if (p.q.top && t == 0) {
    const int64_t at = (int64_t)head * p.q.n + row + g;
    if (row + g < hi) p.q.top[at] = top[0], p.q.inverse[at] = f[0];
    if (row + g + 8 < hi) p.q.top[at + 8] = top[1], p.q.inverse[at + 8] = f[1];
  }
  const bool ok0 = finite_rows(o, 0), ok1 = finite_rows(o, 1);
  store_rows<T, DP>(const_cast<T*>(mine), p.q.out, o, f[0], f[1], row, hi, head, p.q, lane);
  if (p.rest) {
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = o[n][i] * f[i >> 1];
        o[n][i] = x - rounded<T>(x);
      }
    store_rows<T, DP>(const_cast<T*>(mine), p.rest, o, 1.f, 1.f, row, hi, head, p.q, lane);
  }
  each_bad_row(!ok0, !ok1, row, hi, [&](int i) { again_forward<T>(p, i, head, lo, hi, lane); });
}

template <typename T, int DP, int WR, int KT, bool FOLDS>
__global__ void __launch_bounds__(THREADS, DP <= 32 ? 4 : DP <= 96 ? 3 : 2) window_rows_kernel(const __grid_constant__ WindowParams p) {
  using S = attention::Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, slot = warp / WR, ht = tid - slot * S::TH;
  const unsigned groups = (p.q.heads + S::HEADS - 1) / S::HEADS;
  const int head = (int)(blockIdx.x % groups) * S::HEADS + slot;
  const int4 tile = p.q.tiles[blockIdx.x / groups];
  const int first = tile.x, lo = tile.y, hi = tile.z, last = min(hi, first + S::TILE);
  T *rows = reinterpret_cast<T*>(smem) + slot * S::head_elements(2), *grads = rows + S::TILE * LD, *stage = grads + S::TILE * LD;
  const bool here = head < p.q.heads;
  const int kv = here ? head / p.group : 0;
  if (p.q.comps * p.q.size < DP) {
    for (size_t i = tid; i < S::bytes(2, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  Walk walk = keys_of(p, first, last, lo, hi);
  walk.set<KT>();
  auto fetch = [&](int step, int s) {
    int end;
    const int key = walk.at<KT>(step, end);
    load_tile<T, DP, S::TH, KT>(stage + s * S::STAGE, p.q.k, key, here ? end - key : 0, kv, p.q, ht);
    load_tile<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, p.q.v, key, here ? end - key : 0, kv, p.q, ht);
    copies_commit();
  };
  load_tile<T, DP, S::TH, S::TILE>(rows, p.q.q, first, here ? hi - first : 0, here ? head : 0, p.q, ht);
  load_tile<T, DP, S::TH, S::TILE>(grads, p.q.g, first, here ? hi - first : 0, here ? head : 0, p.q, ht);
  copies_commit();
  fetch(0, 0);
  copies_wait<1>();
  __syncthreads();
  const int row = first + (warp % WR) * 16;
  const bool work = here && row < hi;
  const T *mq = rows + (warp % WR) * 16 * LD, *mg = grads + (warp % WR) * 16 * LD;
  const float unit = p.q.scale * LOG2E;
  float delta[2] = {0.f, 0.f}, top[2] = {INFINITY, INFINITY}, inverse[2] = {0.f, 0.f};
  if (work) {
    row_delta<T, DP>(mg, row, hi, head, p.q, lane, delta);
    if (p.rest) {
      AttentionParams rest = p.q;
      rest.out = p.rest;
      float more[2];
      row_delta<T, DP>(mg, row, hi, head, rest, lane, more);
      delta[0] += more[0], delta[1] += more[1];
    }
  }
  const int64_t at = (int64_t)head * p.q.n + row + g;
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (work && row + g + 8 * r < hi) {
      top[r] = p.q.top[at + 8 * r];
      inverse[r] = p.q.inverse[at + 8 * r];
    }
  float sums[2] = {0.f, 0.f}, exact[2] = {0.f, 0.f};     // of weights before rounding, and of these times dP: for the columns
  float dq[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) dq[n][0] = dq[n][1] = dq[n][2] = dq[n][3] = 0.f;
  Far<FOLDS ? DP : 2> waiting;
  for (int step = 0, s = 0; step < walk.steps; ++step, s ^= 1) {
    if constexpr (FOLDS)
      if (fold_now<KT>(step) && work) fold<DP>(waiting.at(), dq, step == FOLD / KT);
    if (step + 1 < walk.steps) {
      fetch(step + 1, s ^ 1);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncthreads();
    int end;
    const int key = walk.at<KT>(step, end);
    if (work && key <= row + 15 + p.after && (key + KT > row - p.before || key < lo + p.sinks)) {
      const T *ks = stage + s * S::STAGE, *vs = ks + KT * LD;
      float z[NT][4], dp[NT][4];
      score_mma<DP, NT>(z, mq, ks, lane);
      score_mma<DP, NT>(dp, mg, vs, lane);
      const bool all = key + KT <= end && key + KT - 1 <= row + p.after && key >= row + 15 - p.before;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i >> 1, j = key + n * 8 + 2 * t + (i & 1);
          const bool on = all || (j < end && sees(p, row + g + 8 * r, j, lo));
          const float weight = exp2_fast(z[n][i] * unit - top[r]);
          z[n][i] = on ? rounded<T>(weight) * inverse[r] * (dp[n][i] - delta[r]) : 0.f;
          sums[r] += on ? weight : 0.f;
          exact[r] += on ? weight * dp[n][i] : 0.f;
        }
      out_mma<DP, NT, true>(dq, z, ks, lane);
    }
    __syncthreads();
  }
  if (!work) return;
  if constexpr (FOLDS)
    if (walk.steps > FOLD / KT) unfold<DP>(waiting.at(), dq);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float all = quad_sum(exact[r]), sum = 1.f / quad_sum(sums[r]);
    if (t == 0 && row + g + 8 * r < hi) p.q.delta[at + 8 * r] = all * sum, p.inverse[at + 8 * r] = sum;
  }
  const bool ok0 = finite_rows(dq, 0), ok1 = finite_rows(dq, 1);
  store_rows<T, DP>(const_cast<T*>(mq), p.q.dq, dq, p.q.scale, p.q.scale, row, hi, head, p.q, lane);
  each_bad_row(!ok0, !ok1, row, hi, [&](int i) { again_rows<T>(p, i, head, lo, hi, lane); });
}

template <typename T, int DP, int WR, int KT, bool FOLDS>
__global__ void __launch_bounds__(THREADS, DP <= 64 ? 3 : 2) window_columns_kernel(const __grid_constant__ WindowParams p) {
  using S = attention::Shape<T, DP, WR, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, slot = warp / WR, ht = tid - slot * S::TH;
  const unsigned groups = (p.kv.heads + S::HEADS - 1) / S::HEADS;
  const int kv = (int)(blockIdx.x % groups) * S::HEADS + slot;
  const int4 tile = p.q.tiles[blockIdx.x / groups];
  const int first = tile.x, lo = tile.y, hi = tile.z, last = min(hi, first + S::TILE);
  T *keys = reinterpret_cast<T*>(smem) + slot * S::head_elements(2), *values = keys + S::TILE * LD, *stage = values + S::TILE * LD;
  float* numbers = reinterpret_cast<float*>(smem + S::bytes(2, 0)) + slot * 6 * KT;      // of the queries: two tiles of greatest score, inverse sum, delta
  const bool here = kv < p.kv.heads;
  if (p.q.comps * p.q.size < DP) {
    for (size_t i = tid; i < S::bytes(2, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  Walk walk = queries_of(p, first, last, lo, hi);
  walk.set<KT>();
  const int steps = walk.steps * p.group;                // the heads one after the other
  const bool far_apart = apart(p, lo, hi);
  const int first_end = far_apart ? lo : lo + p.sinks;   // nodes before it are seen from behind their windows here
  auto fetch = [&](int step, int s) {
    int end;
    const int i = walk.at<KT>(step % walk.steps, end), head = here ? kv * p.group + step / walk.steps : 0;
    load_tile<T, DP, S::TH, KT>(stage + s * S::STAGE, p.q.q, i, here ? end - i : 0, head, p.q, ht);
    load_tile<T, DP, S::TH, KT>(stage + s * S::STAGE + KT * LD, p.q.g, i, here ? end - i : 0, head, p.q, ht);
    for (int c = ht; c < 3 * KT; c += S::TH) {
      const int r = c % KT;
      const float* from = c < KT ? p.q.top : c < 2 * KT ? p.inverse : p.q.delta;
      const bool there = here && i + r < end;
      copy4(numbers + s * 3 * KT + c, from + (there ? (int64_t)head * p.q.n + i + r : 0), there);
    }
    copies_commit();
  };
  load_tile<T, DP, S::TH, S::TILE>(keys, p.q.k, first, here ? hi - first : 0, here ? kv : 0, p.q, ht);
  load_tile<T, DP, S::TH, S::TILE>(values, p.q.v, first, here ? hi - first : 0, here ? kv : 0, p.q, ht);
  fetch(0, 0);
  const int row = first + (warp % WR) * 16;
  const bool work = here && row < hi;
  const T *mk = keys + (warp % WR) * 16 * LD, *mv = values + (warp % WR) * 16 * LD;
  const float unit = p.q.scale * LOG2E;
  float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) dk[n][i] = dv[n][i] = 0.f;
  Far<FOLDS ? DP : 2> waiting_k, waiting_v;
  for (int step = 0, s = 0; step < steps; ++step, s ^= 1) {
    if constexpr (FOLDS)
      if (fold_now<KT>(step) && work) {
        fold<DP>(waiting_k.at(), dk, step == FOLD / KT);
        fold<DP>(waiting_v.at(), dv, step == FOLD / KT);
      }
    if (step + 1 < steps) {
      fetch(step + 1, s ^ 1);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncthreads();
    int end;
    const int query = walk.at<KT>(step % walk.steps, end);
    if (work && row <= query + KT - 1 + p.after && (row + 15 >= query - p.before || row < first_end)) {
      const T *qs = stage + s * S::STAGE, *gs = qs + KT * LD;
      const float* num = numbers + s * 3 * KT;
      float z[NT][4], dp[NT][4];
      score_mma<DP, NT, true>(z, mk, qs, lane);
      score_mma<DP, NT, true>(dp, mv, gs, lane);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = n * 8 + 2 * t + (i & 1), q = query + c;
          const int j = row + g + 8 * (i >> 1);
          const bool on = q < end && j <= q + p.after && (j >= q - p.before || j < first_end);
          z[n][i] = on ? exp2_fast(z[n][i] * unit - num[c]) * num[KT + c] : 0.f;
          dp[n][i] = on ? z[n][i] * (dp[n][i] - num[2 * KT + c]) : 0.f;
        }
      out_mma<DP, NT>(dv, z, gs, lane);
      out_mma<DP, NT>(dk, dp, qs, lane);
    }
    __syncthreads();
  }
  if (!work) return;
  if constexpr (FOLDS)
    if (steps > FOLD / KT) {
      unfold<DP>(waiting_k.at(), dk);
      unfold<DP>(waiting_v.at(), dv);
    }
  if (far_apart && row < lo + p.sinks) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int j = row + g + 8 * r, values = p.q.comps * p.q.size;
      const float* far = j < hi ? far_of(p, j, kv, lo, hi) : nullptr;
      if (!far) continue;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = n * 8 + 2 * t + i;
          if (c >= values) continue;
          dk[n][2 * r + i] += far[c];
          dv[n][2 * r + i] += far[FAR_ROWS * values + c];
        }
    }
  }
  const bool ok0 = finite_rows(dk, 0) && finite_rows(dv, 0), ok1 = finite_rows(dk, 1) && finite_rows(dv, 1);
  store_rows<T, DP>(const_cast<T*>(mk), p.kv.dk, dk, p.q.scale, p.q.scale, row, hi, kv, p.kv, lane);
  store_rows<T, DP>(const_cast<T*>(mv), p.kv.dv, dv, 1.f, 1.f, row, hi, kv, p.kv, lane);
  each_bad_row(!ok0, !ok1, row, hi, [&](int j) { again_columns<T>(p, j, kv, lo, hi, lane); });
}

// 16 first nodes of a chain and the queries behind their windows in one block of the batch: a CTA, whose warps take the steps of all heads in turn and
// add their sums up in order.
template <typename T, int DP, int KT, bool FOLDS> __global__ void __launch_bounds__(THREADS) window_far_kernel(const __grid_constant__ WindowParams p) {
  using S = attention::Shape<T, DP, 1, KT>;
  constexpr int LD = S::LD, NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int64_t chain;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, kv = blockIdx.y, values = p.q.comps * p.q.size;
  // The only chain that may be that pair's: what comes behind a long chain has a greater number than its last pair.
  if (tid == 0) chain = last_chain(p.chains, blockIdx.x, [&](int64_t c) { return p.ptr[c] / FAR_BLOCK + p.ptr[c] / far_length(p); });
  if (values < DP)
    for (size_t i = tid; i < S::bytes(2, 0) / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (chain < 0) return;
  const int lo = (int)p.ptr[chain], hi = (int)p.ptr[chain + 1];
  const int64_t block = blockIdx.x - lo / far_length(p);
  const int first = lo + (int)blockIdx.z * FAR_ROWS, last = min(min(lo + p.sinks, hi), first + FAR_ROWS);
  if (!apart(p, lo, hi) || block > (hi - 1) / FAR_BLOCK || first >= last) return;
  const int from = max((int)(block * FAR_BLOCK), first + p.before + 1), to = (int)min((block + 1) * FAR_BLOCK, (int64_t)hi);
  if (from >= to) return;
  T *keys = reinterpret_cast<T*>(smem) + warp * S::head_elements(2), *vals = keys + 16 * LD, *stage = vals + 16 * LD;
  float* numbers = reinterpret_cast<float*>(smem + S::bytes(2, 0)) + warp * 6 * KT;
  const int blocks = (to - from + KT - 1) / KT, steps = blocks * p.group;
  auto fetch = [&](int step, int s) {
    const int head = kv * p.group + step / blocks, i = from + step % blocks * KT;
    load_tile<T, DP, 32, KT>(stage + s * S::STAGE, p.q.q, i, to - i, head, p.q, lane);
    load_tile<T, DP, 32, KT>(stage + s * S::STAGE + KT * LD, p.q.g, i, to - i, head, p.q, lane);
    for (int c = lane; c < 3 * KT; c += 32) {
      const int r = c % KT;
      const float* x = c < KT ? p.q.top : c < 2 * KT ? p.inverse : p.q.delta;
      const bool there = i + r < to;
      copy4(numbers + s * 3 * KT + c, x + (there ? (int64_t)head * p.q.n + i + r : 0), there);
    }
    copies_commit();
  };
  load_tile<T, DP, 32, 16>(keys, p.q.k, first, last - first, kv, p.q, lane);
  load_tile<T, DP, 32, 16>(vals, p.q.v, first, last - first, kv, p.q, lane);
  if (warp < steps) fetch(warp, 0);
  const float unit = p.q.scale * LOG2E;
  float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) dk[n][i] = dv[n][i] = 0.f;
  Far<FOLDS ? DP : 2> waiting_k, waiting_v;
  for (int step = warp, s = 0; step < steps; step += WARPS, s ^= 1) {
    if constexpr (FOLDS)
      if (fold_now<KT>(step / WARPS)) {
        fold<DP>(waiting_k.at(), dk, step / WARPS == FOLD / KT);
        fold<DP>(waiting_v.at(), dv, step / WARPS == FOLD / KT);
      }
    if (step + WARPS < steps) {
      fetch(step + WARPS, s ^ 1);
      copies_wait<1>();
    } else {
      copies_wait<0>();
    }
    __syncwarp();
    const int query = from + step % blocks * KT;
    const T *qs = stage + s * S::STAGE, *gs = qs + KT * LD;
    const float* num = numbers + s * 3 * KT;
    float z[NT][4], dp[NT][4];
    score_mma<DP, NT, true>(z, keys, qs, lane);
    score_mma<DP, NT, true>(dp, vals, gs, lane);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = n * 8 + 2 * t + (i & 1), j = first + g + 8 * (i >> 1);
        const bool on = query + c < to && j < last && query + c > j + p.before;
        z[n][i] = on ? exp2_fast(z[n][i] * unit - num[c]) * num[KT + c] : 0.f;
        dp[n][i] = on ? z[n][i] * (dp[n][i] - num[2 * KT + c]) : 0.f;
      }
    out_mma<DP, NT>(dv, z, gs, lane);
    out_mma<DP, NT>(dk, dp, qs, lane);
    __syncwarp();
  }
  copies_wait<0>();
  if constexpr (FOLDS)
    if ((steps - warp + WARPS - 1) / WARPS > FOLD / KT) {
      unfold<DP>(waiting_k.at(), dk);
      unfold<DP>(waiting_v.at(), dv);
    }
  float* sums = reinterpret_cast<float*>(smem);          // [dk, dv][node][value], where the tiles were
  for (int w = 0; w < WARPS; ++w) {
    __syncthreads();
    if (warp != w) continue;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (g + 8 * (i >> 1)) * DP + n * 8 + 2 * t + (i & 1);
        sums[at] = w ? sums[at] + dk[n][i] : dk[n][i];
        sums[FAR_ROWS * DP + at] = w ? sums[FAR_ROWS * DP + at] + dv[n][i] : dv[n][i];
      }
  }
  __syncthreads();
  float* out = p.far + far_place(p, blockIdx.x, kv, blockIdx.z);
  for (int i = tid; i < 2 * FAR_ROWS * values; i += THREADS) out[i] = sums[i / values * DP + i % values];
}
// The blocks of a slot's chain, in their order, into its first one: a thread has one number.
__global__ void __launch_bounds__(256) window_far_join_kernel(const __grid_constant__ WindowParams p, int groups) {
  __shared__ int64_t found;
  if (threadIdx.x == 0) found = last_chain(p.chains, blockIdx.x, [&](int64_t c) { return p.ptr[c] / far_length(p); });
  __syncthreads();
  const int64_t chain = found;
  if (chain < 0) return;
  const int group = blockIdx.z % groups, at = blockIdx.z / groups * 256 + threadIdx.x;
  const int lo = (int)p.ptr[chain], hi = (int)p.ptr[chain + 1], first = lo + group * FAR_ROWS;
  if (!apart(p, lo, hi) || lo / far_length(p) != blockIdx.x || first >= lo + p.sinks || first + p.before + 1 >= hi || at >= 2 * FAR_ROWS * p.q.comps * p.q.size) return;
  const int64_t begin = (first + p.before + 1) / FAR_BLOCK, end = (hi - 1) / FAR_BLOCK;
  const int64_t step = far_place(p, 1, 0, 0);
  float* to = p.far + far_place(p, begin + blockIdx.x, blockIdx.y, group) + at;
  float sum = 0.f;
#pragma unroll 16
  for (int64_t b = 0; b <= end - begin; ++b) sum += to[b * step];
  *to = sum;
}

// ---- host side ----------------------------------------------------------------------------------
template <typename T, int DP> int launch_far(const WindowParams& p, cudaStream_t s) {
  constexpr int KT = DP > 32 ? 16 : 32;
  using S = attention::Shape<T, DP, 1, KT>;
  const int64_t pairs = far_pairs(p);                    // fewer than 2^22
  const size_t shared = S::bytes(2, WARPS * 6 * KT * 4);
  auto kernel = window_far_kernel<T, DP, KT, false>;
  bool folds = false;                                    // a warp has a quarter of a block's queries of all heads
  if constexpr (sizeof(T) == 2) {
    folds = p.group > FOLD / (FAR_BLOCK / WARPS);
    if (folds) kernel = window_far_kernel<T, DP, KT, true>;
  }
  static std::atomic<uint64_t> allowed[2]{};
  if (int rc = allow_shared_once(kernel, shared, allowed[folds])) return rc;
  kernel<<<dim3((unsigned)pairs, (unsigned)p.kv.heads, (unsigned)far_groups(p)), THREADS, shared, s>>>(p);
  if (int rc = check_launch("window_far")) return rc;
  const int groups = far_groups(p), chunks = (int)ceil_div(2 * FAR_ROWS * p.q.comps * p.q.size, 256);
  window_far_join_kernel<<<dim3((unsigned)far_slots(p), (unsigned)p.kv.heads, (unsigned)(groups * chunks)), 256, 0, s>>>(p, groups);
  return check_launch("window_far_join");
}
template <typename T> int far(const WindowParams& p, cudaStream_t s) {
  const int values = p.q.comps * p.q.size;
  return values <= 16 ? launch_far<T, 16>(p, s) : values <= 32 ? launch_far<T, 32>(p, s) : values <= 64 ? launch_far<T, 64>(p, s) : launch_far<T, 128>(p, s);
}

enum Pass { FORWARD, ROWS, COLUMNS };
template <typename T, int DP, int WR, int KT, int PASS, bool FOLDS = false> int launch(const WindowParams& p, int64_t num_tiles, cudaStream_t s) {
  using S = attention::Shape<T, DP, WR, KT>;
  const int heads = PASS == COLUMNS ? p.kv.heads : p.q.heads;
  const int64_t grid = num_tiles * ceil_div(heads, S::HEADS);
  if (grid > INT32_MAX) return fail(EQT_ERR_UNSUPPORTED, "window_attention: %lld tiles are more than one launch takes", (long long)grid);
  const size_t shared = S::bytes(PASS == FORWARD ? 1 : 2, PASS == COLUMNS ? S::HEADS * 6 * KT * 4 : 0);
  auto kernel = PASS == FORWARD ? window_forward_kernel<T, DP, WR, KT, FOLDS> : PASS == ROWS ? window_rows_kernel<T, DP, WR, KT, FOLDS> : window_columns_kernel<T, DP, WR, KT, FOLDS>;
  static std::atomic<uint64_t> allowed{0};
  if (int rc = allow_shared_once(kernel, shared, allowed)) return rc;
  kernel<<<(unsigned)grid, THREADS, shared, s>>>(p);
  return check_launch("window_attention");
}
// Keys a step: 32, of wide float32 rows 16, whose two stages would not fit three CTAs an SM.
template <typename T, int DP, int PASS> int by_rows(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s) {
  constexpr int KT = sizeof(T) == 4 && DP > 64 ? 16 : 32;
  // Long sums, in kernels of their own, whose registers the others need not pay for: by columns of chains of any length, since heads add up; of rows where chains are so long
  // that tiles have 64 rows.
  if constexpr (sizeof(T) == 2) {
    if constexpr (PASS == COLUMNS)
      if (p.folds_columns)
        return tile_rows == 16 ? launch<T, DP, 1, KT, COLUMNS, true>(p, num_tiles, s) : tile_rows == 32 ? launch<T, DP, 2, KT, COLUMNS, true>(p, num_tiles, s)
                                                                                                         : launch<T, DP, 4, KT, COLUMNS, true>(p, num_tiles, s);
    if constexpr (PASS != COLUMNS)
      if (p.folds_rows) return launch<T, DP, 4, KT, PASS, true>(p, num_tiles, s);
  }
  switch (tile_rows) {
    case 16: return launch<T, DP, 1, KT, PASS>(p, num_tiles, s);
    case 32: return launch<T, DP, 2, KT, PASS>(p, num_tiles, s);
    default: return launch<T, DP, 4, KT, PASS>(p, num_tiles, s);
  }
}
template <typename T, int PASS> int by_values(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s) {
  const int values = p.q.comps * p.q.size;
  if (values <= 16) return by_rows<T, 16, PASS>(p, tile_rows, num_tiles, s);
  if (values <= 32) return by_rows<T, 32, PASS>(p, tile_rows, num_tiles, s);
  if (values <= 64) return by_rows<T, 64, PASS>(p, tile_rows, num_tiles, s);
  return by_rows<T, 128, PASS>(p, tile_rows, num_tiles, s);
}

template <typename T> int tiles_backward(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s) {
  if (int rc = by_values<T, ROWS>(p, tile_rows, num_tiles, s)) return rc;
  if (p.split)
    if (int rc = far<T>(p, s)) return rc;
  return by_values<T, COLUMNS>(p, tile_rows, num_tiles, s);
}

}  // namespace
}  // namespace window
}  // namespace eqt
