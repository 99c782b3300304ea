// Attention of one new node of every chain over a cache: the last `before` nodes and the new one, and the chain's first `sinks`.
//
//     s_j = scale <q, k_j>,   out = sum_j softmax(s)_j v_j,      j in [len - 1 - before, len) or j < sinks,  j < len
//
// Bound by HBM: every visible key and value is read once, for all the heads that share it.  The visible keys of a chain are two stretches (first nodes,
// window) of steps of 32 keys, cut into parts so that the chains' parts fill the SMs; a CTA takes a part and up to 16 heads of a head of keys, whose queries
// are the rows of the warp-wide matrix instructions.  Each of its four warps takes every fourth step, with copies of its own three ahead, and has the
// maxima, sums and weighted values of its keys; warps, and then parts, are joined by their maxima, in one order.
// 64 chains of up to 8192 nodes, window 4096, 16 heads on 4 of 64 bfloat16 values: 56 us (3.7 TB/s) and 6 for the join; with products by the threads 87.
#include <algorithm>

#include "graph_attention.cuh"

namespace eqt {
namespace window_step {
namespace {

using namespace attention;
constexpr int MOST_VALUES = 128, STAGES = 3, ROWS = 16;

struct StepArgs {
  Operand q, k, v;                                       // of one chain
  int64_t q_chain, k_chain, v_chain;                     // strides between chains, in values
  void* out;
  float* parts;                                          // [chain][head][part]: maximum, sum, sums of the values
  const int64_t* lengths;
  int64_t capacity, before, sinks, part_steps;
  int group, num_parts;                                  // group: heads of a head of keys
  AttentionParams a;                                     // heads, components, channels a head, alignment
};

// Keys a step, such that three stages of four warps leave two CTAs an SM.
template <typename T, int DP> constexpr int step_keys() { return sizeof(T) * DP > 256 ? 8 : sizeof(T) * DP > 128 ? 16 : 32; }
template <typename T, int DP> constexpr size_t stage_values() { return (size_t)2 * step_keys<T, DP>() * Row<T, DP>::LD; }
template <typename T, int DP> constexpr size_t shared_bytes() {
  const size_t tiles = (ROWS * Row<T, DP>::LD + WARPS * STAGES * stage_values<T, DP>()) * sizeof(T), sums = (size_t)WARPS * ROWS * (DP + 2) * 4;
  return tiles > sums ? tiles : sums;
}

template <typename T, int DP, int ROWS_TILE> __device__ __forceinline__ void load_some(T* dst, const Operand& x, int first, int left, int head, const AttentionParams& p, int lane) {
  const Piece<T, DP, 32> piece(lane, p.comps, p.size);
  Source<T, DP, 32> from(x, piece, first, head, p);
  load_rows<T, DP, 32, ROWS_TILE>(dst, from, x, piece, first, left, head, p, lane);
}

template <typename T, int DP> __global__ void __launch_bounds__(THREADS) step_kernel(const __grid_constant__ StepArgs p) {
  constexpr int LD = Row<T, DP>::LD, KT = step_keys<T, DP>(), NT = KT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, values = p.a.comps * p.a.size;
  const int part = blockIdx.x, blocks = (p.group + ROWS - 1) / ROWS, kv = blockIdx.y / blocks, head0 = kv * p.group + blockIdx.y % blocks * ROWS;
  const int here = min(ROWS, (kv + 1) * p.group - head0);
  const int64_t chain = blockIdx.z;
  const int length = (int)max((int64_t)0, min(p.lengths[chain], p.capacity)), low = (int)max((int64_t)0, length - 1 - p.before), sinks = (int)min((int64_t)low, p.sinks);
  const int steps0 = (sinks + KT - 1) / KT, steps = steps0 + (length - low + KT - 1) / KT;
  const int first = (int)min((int64_t)steps, part * p.part_steps), end = (int)min((int64_t)steps, first + p.part_steps);
  T *rows = reinterpret_cast<T*>(smem), *stage = rows + ROWS * LD + warp * STAGES * stage_values<T, DP>();
  if (values < DP) {                                     // the columns behind a head's values stay zero
    for (size_t i = tid; i < shared_bytes<T, DP>() / 16; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  auto of = [&](const Operand& x, int64_t stride) { return Operand{static_cast<const T*>(x.p) + chain * stride, x.node, x.comp}; };
  const Operand q = of(p.q, p.q_chain), k = of(p.k, p.k_chain), v = of(p.v, p.v_chain);
  for (int i = tid; i < ROWS * values; i += THREADS) {
    const int h = i / values, e = i - h * values, comp = e / p.a.size;
    rows[h * LD + e] = h < here ? static_cast<const T*>(q.p)[comp * q.comp + (int64_t)(head0 + h) * p.a.size + e - comp * p.a.size] : static_cast<T>(0.f);
  }
  auto key_of = [&](int step, int& stop) {
    stop = step < steps0 ? sinks : length;
    return step < steps0 ? step * KT : low + (step - steps0) * KT;
  };
  auto ask = [&](int step, int place) {
    if (step < end) {
      int stop;
      const int key = key_of(step, stop);
      T* to = stage + place * stage_values<T, DP>();
      load_some<T, DP, KT>(to, k, key, stop - key, kv, p.a, lane);
      load_some<T, DP, KT>(to + KT * LD, v, key, stop - key, kv, p.a, lane);
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) ask(first + warp + i * WARPS, i);
  __syncthreads();
  const float unit = p.a.scale * LOG2E;
  float o[DP / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  int place = 0;
  for (int step = first + warp; step < end; step += WARPS) {
    ask(step + (STAGES - 1) * WARPS, place == 0 ? STAGES - 1 : place - 1);
    copies_wait<STAGES - 1>();
    __syncwarp();
    const T *ks = stage + place * stage_values<T, DP>(), *vs = ks + KT * LD;
    int stop;
    const int key = key_of(step, stop);
    float z[NT][4];
    score_mma<DP, NT>(z, rows, ks, lane);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) z[n][i] = key + n * 8 + 2 * t + (i & 1) < stop ? z[n][i] * unit : -INFINITY;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float most = top[r];
#pragma unroll
      for (int n = 0; n < NT; ++n) most = fmaxf(most, fmaxf(z[n][2 * r], z[n][2 * r + 1]));
      most = quad_max(most);
      const float base = most == -INFINITY ? 0.f : most, keep = exp2_fast(top[r] - base);
      float add = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float &x = z[n][2 * r], &y = z[n][2 * r + 1];
        x = exp2_fast(x - base), y = exp2_fast(y - base);
        add += x + y;
      }
      sum[r] = sum[r] * keep + add;
      top[r] = most;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) o[n][2 * r] *= keep, o[n][2 * r + 1] *= keep;
    }
    out_mma<DP, NT, true>(o, z, vs, lane);              // in two parts: a result has no rounding but its own (2-norm of its error 1.85e-3 | 1.64e-3; 53.2 | 55.9 us)
    __syncwarp();
    if (++place == STAGES) place = 0;
  }
  copies_wait<0>();
  __syncthreads();                                       // the tiles' place is the sums' now: [warp][head] maximum, sum, values
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float* to = sums + (warp * ROWS + g + 8 * r) * (DP + 2);
    const float all = quad_sum(sum[r]);
    if (t == 0) to[0] = top[r], to[1] = all;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) to[2 + n * 8 + 2 * t] = o[n][2 * r], to[2 + n * 8 + 2 * t + 1] = o[n][2 * r + 1];
  }
  __syncthreads();
  for (int i = tid; i < here * values; i += THREADS) {
    const int h = i / values, e = i - h * values;
    float most = -INFINITY, total = 0.f, value = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) most = fmaxf(most, sums[(w * ROWS + h) * (DP + 2)]);
    const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* from = sums + (w * ROWS + h) * (DP + 2);
      const float f = exp2_fast(from[0] - base);
      total += f * from[1];
      value += f * from[2 + e];
    }
    const int head = head0 + h, comp = e / p.a.size;
    if (p.num_parts > 1) {
      float* to = p.parts + ((chain * p.a.heads + head) * p.num_parts + part) * (2 + values);
      if (e == 0) to[0] = most, to[1] = total;
      to[2 + e] = value;
    } else {
      st(static_cast<T*>(p.out) + ((chain * p.a.comps + comp) * p.a.heads + head) * p.a.size + e - comp * p.a.size, length > 0 ? value / total : 0.f);
    }
  }
}

// The parts of a chain and head, one warp: the maxima and sums by the lanes, then a lane has every 32nd value.
template <typename T> __global__ void __launch_bounds__(THREADS) step_join_kernel(const __grid_constant__ StepArgs p, int64_t rows) {
  const int64_t row = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, head = (int)(row % p.a.heads), values = p.a.comps * p.a.size;
  const int64_t chain = row / p.a.heads;
  const float* parts = p.parts + row * p.num_parts * (2 + values);
  float most = -INFINITY, total = 0.f;
  for (int i = lane; i < p.num_parts; i += 32) most = fmaxf(most, parts[i * (2 + values)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  const float base = most == -INFINITY ? 0.f : most;
  for (int i = lane; i < p.num_parts; i += 32) total += exp2_fast(parts[i * (2 + values)] - base) * parts[i * (2 + values) + 1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  float value[MOST_VALUES / 32];
#pragma unroll
  for (int c = 0; c < MOST_VALUES / 32; ++c) value[c] = 0.f;
#pragma unroll 4
  for (int i = 0; i < p.num_parts; ++i) {
    const float* from = parts + i * (2 + values);
    const float f = exp2_fast(from[0] - base);
#pragma unroll
    for (int c = 0; c < MOST_VALUES / 32; ++c) value[c] += f * (lane + 32 * c < values ? from[2 + lane + 32 * c] : 0.f);
  }
  const bool any = p.lengths[chain] > 0 && p.capacity > 0;
#pragma unroll
  for (int c = 0; c < MOST_VALUES / 32; ++c) {
    const int at = lane + 32 * c, comp = at / p.a.size, channel = at - comp * p.a.size;
    if (at < values) st(static_cast<T*>(p.out) + ((chain * p.a.comps + comp) * p.a.heads + head) * p.a.size + channel, any ? value[c] / total : 0.f);
  }
}

// ---- host side ----------------------------------------------------------------------------------
int width_of(int values) { return values <= 16 ? 16 : values <= 32 ? 32 : values <= 64 ? 64 : 128; }
int keys_of(int dtype, int width) { return (dtype == EQT_F32 ? 4 : 2) * width > 256 ? 8 : (dtype == EQT_F32 ? 4 : 2) * width > 128 ? 16 : 32; }

// Parts of the visible keys: so many that SMs with shorter chains take more of them, a step for each warp, and of a warp no more than what bfloat16 products may add up in
// the matrix instructions, whose adder truncates (1,048,576 keys in one part: 1e-3 of a sum of one sign).
void cut(StepArgs& p, int dtype, int64_t chains, int kv_heads) {
  const int kt = keys_of(dtype, width_of(p.a.comps * p.a.size));
  const int64_t window = std::min<int64_t>(p.capacity, p.before + 1), first = std::min<int64_t>(p.capacity, p.sinks);
  const int64_t steps = std::max<int64_t>(1, ceil_div(window, kt) + ceil_div(first, kt));
  const int64_t others = std::max<int64_t>(1, chains * kv_heads), wanted = ceil_div((int64_t)sm_count() * 8, others);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(wanted, ceil_div(steps, WARPS)), 1024));
  p.part_steps = std::min<int64_t>(ceil_div(ceil_div(steps, parts), WARPS), FOLD / kt) * WARPS;
  p.num_parts = (int)ceil_div(steps, p.part_steps);
}

template <typename T, int DP> int launch(const StepArgs& p, int64_t chains, int kv_heads, cudaStream_t s) {
  auto kernel = step_kernel<T, DP>;
  static std::atomic<uint64_t> allowed{0};
  if (int rc = allow_shared_once(kernel, shared_bytes<T, DP>(), allowed)) return rc;
  const dim3 grid((unsigned)p.num_parts, (unsigned)(kv_heads * ceil_div(p.group, ROWS)), (unsigned)chains);
  kernel<<<grid, THREADS, shared_bytes<T, DP>(), s>>>(p);
  if (int rc = check_launch("window_step")) return rc;
  if (p.num_parts == 1) return EQT_OK;
  const int64_t rows = chains * p.a.heads;
  step_join_kernel<T><<<(unsigned)ceil_div(rows, WARPS), THREADS, 0, s>>>(p, rows);
  return check_launch("window_step_join");
}
template <typename T> int run(const StepArgs& p, int64_t chains, int kv_heads, cudaStream_t s) {
  switch (width_of(p.a.comps * p.a.size)) {
    case 16: return launch<T, 16>(p, chains, kv_heads, s);
    case 32: return launch<T, 32>(p, chains, kv_heads, s);
    case 64: return launch<T, 64>(p, chains, kv_heads, s);
    default: return launch<T, 128>(p, chains, kv_heads, s);
  }
}

int fill(StepArgs& p, const eqt_window_step_args* a) {
  if (!a) return fail(EQT_ERR_BAD_ARGUMENT, "window_step: NULL pointer");
  if (a->dtype != EQT_F32 && a->dtype != EQT_BF16) return fail(EQT_ERR_BAD_ARGUMENT, "window_step: unknown dtype %d", a->dtype);
  if (a->chains < 0 || a->capacity < 0 || a->before < 0 || a->sinks < 0 || a->heads < 1 || a->kv_heads < 1 || a->comps < 1 || a->head_channels < 1 ||
      a->heads % a->kv_heads)
    return fail(EQT_ERR_BAD_ARGUMENT, "window_step: sizes");
  if ((int64_t)a->comps * a->head_channels > MOST_VALUES || a->chains > 65535 || a->heads > 65535 || a->capacity > INT32_MAX - 64 || a->before > INT32_MAX ||
      a->sinks > INT32_MAX)
    return fail(EQT_ERR_UNSUPPORTED, "window_step: at most %d values a head, 65535 chains and heads, 2^31 nodes a chain", MOST_VALUES);
  const int v = a->dtype == EQT_F32 ? 4 : 8;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v);
  const int64_t strides = a->k_chain | a->k_node | a->k_comp | a->v_chain | a->v_node | a->v_comp;
  p.q = {a->q, 0, a->q_comp}, p.k = {a->k, a->k_node, a->k_comp}, p.v = {a->v, a->v_node, a->v_comp};
  p.q_chain = a->q_chain, p.k_chain = a->k_chain, p.v_chain = a->v_chain;
  p.out = a->out, p.parts = a->scratch, p.lengths = a->lengths, p.capacity = a->capacity, p.before = a->before, p.sinks = a->sinks;
  p.group = a->heads / a->kv_heads;
  p.a.heads = a->heads, p.a.comps = a->comps, p.a.size = a->head_channels, p.a.scale = a->scale;
  p.a.vec = bits % 16 == 0 && strides % v == 0 && a->head_channels % v == 0;
  cut(p, a->dtype, a->chains, a->kv_heads);
  return EQT_OK;
}

}  // namespace
}  // namespace window_step
}  // namespace eqt

using namespace eqt;
using namespace eqt::window_step;

extern "C" int64_t eqt_window_step_scratch(const eqt_window_step_args* a) {
  StepArgs p{};
  if (fill(p, a) || p.num_parts == 1) return 0;
  return a->chains * p.a.heads * p.num_parts * (2 + p.a.comps * p.a.size);
}

extern "C" int eqt_window_step(const eqt_window_step_args* a, void* stream) {
  StepArgs p{};
  if (int rc = fill(p, a)) return rc;
  if (a->chains == 0) return EQT_OK;
  if (!a->q || !a->out || !a->lengths || (a->capacity && (!a->k || !a->v))) return fail(EQT_ERR_BAD_ARGUMENT, "window_step: NULL pointer");
  const int64_t need = p.num_parts == 1 ? 0 : a->chains * p.a.heads * p.num_parts * (2 + p.a.comps * p.a.size);
  if (need && (!a->scratch || a->scratch_floats < need))
    return fail(EQT_ERR_BAD_ARGUMENT, "window_step: %lld values of scratch given, %lld needed", (long long)a->scratch_floats, (long long)need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == EQT_F32 ? run<float>(p, a->chains, a->kv_heads, s) : run<__nv_bfloat16>(p, a->chains, a->kv_heads, s);
}
