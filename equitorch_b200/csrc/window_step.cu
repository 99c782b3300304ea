// Attention of one new node of every chain over a cache: the last `before` nodes and the new one, and the chain's first `sinks`.
//
//     s_j = scale <q, k_j>,   out = sum_j softmax(s)_j v_j,      j in [len - 1 - before, len) or j < sinks,  j < len
//
// Bound by HBM: every visible key and value is read once, for all the heads that share it; 2 D values a key against 4 D flops a head.  The
// visible keys of a chain are one list (sinks, then the window), cut into parts so that the chains' parts fill the SMs; a CTA takes a part of
// a chain and the heads of one head of keys, up to MOST at a time.  The threads that a key's row takes by pieces of 16 bytes form a team; a team
// takes key after key with the softmax's maximum and sum, and its sums of the values, in its own registers, so that nothing but the product
// itself crosses threads on the way.  Teams, and then parts, are joined by their maxima at the end, in one order.
#include <algorithm>

#include "graph_attention.cuh"

namespace eqt {
namespace window_step {
namespace {

constexpr int THREADS = 128, MOST_VALUES = 128, AHEAD = 6;
using attention::LOG2E;

struct StepArgs {
  const void *q, *k, *v;
  void* out;
  float* parts;                                          // [chain][head][part]: maximum, sum, sums of the values
  const int64_t* lengths;
  int64_t q_chain, q_comp, k_chain, k_node, k_comp, v_chain, v_node, v_comp, capacity, before, sinks;
  int64_t part_keys;
  int heads, group, comps, size, values, num_parts;      // group: heads of a head of keys; values: of a head
  float scale;                                           // times log2 e
};

using attention::add2;
using attention::both;
using attention::exp2_fast;
using attention::fma2;
using attention::mul2;
using attention::pair;
using attention::parts;

// V values from memory: 16 bytes, or one
template <int V> __device__ __forceinline__ void unpack(const uint4& u, float (&v)[V]) {
  if constexpr (V > 1) {
    const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 4) v[i] = __uint_as_float(r[i]);
      else v[2 * i] = __uint_as_float(r[i] << 16), v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
}
template <typename T, int V> __device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  if constexpr (V == 1) v[0] = static_cast<float>(*p);
  else unpack<V>(__ldg(reinterpret_cast<const uint4*>(p)), v);
}

// What a softmax over some keys leaves.  Without a key the maximum is minus infinity and the sums are zero.
template <int N> struct State {
  float top, sum, o[N];
};
template <int N> __device__ __forceinline__ void join(State<N>& a, float top, float sum, const float* o) {
  const float t = top > a.top || top != top ? top : a.top, keep = a.top == -INFINITY ? 0.f : exp2_fast(a.top - t), take = top == -INFINITY ? 0.f : exp2_fast(top - t);
  a.sum = a.sum * keep + sum * take;
#pragma unroll
  for (int i = 0; i < N; ++i) a.o[i] = a.o[i] * keep + o[i] * take;
  a.top = t;
}

// TEAM threads a key, PIECES pieces of V values each; H heads at a time
template <typename T, int V, int TEAM, int PIECES, int H> __global__ void __launch_bounds__(THREADS) step_kernel(const StepArgs p) {
  constexpr int N = V * PIECES, TEAMS = THREADS / TEAM;
  __shared__ float tops[THREADS / 32][H], sums[THREADS / 32][H], values[THREADS / 32][H][TEAM * N];
  __shared__ uint4 ring[V > 1 ? AHEAD : 1][2][V > 1 ? THREADS : 1];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM, warp = threadIdx.x >> 5;
  const int part = blockIdx.x, blocks = (p.group + H - 1) / H, kv = blockIdx.y / blocks, head0 = kv * p.group + blockIdx.y % blocks * H;
  const int here = min(H, (kv + 1) * p.group - head0);
  const int64_t chain = blockIdx.z, length = max((int64_t)0, min(p.lengths[chain], p.capacity));
  const int64_t low = max((int64_t)0, length - 1 - p.before), sinks = min(low, p.sinks), visible = sinks + length - low;
  const int64_t first = part * p.part_keys, end = min(visible, first + p.part_keys);
  // this thread's places in a head's row
  int64_t k_at[PIECES], v_at[PIECES];
  bool on[PIECES];
  float q[H][N];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int at = (lane + i * TEAM) * V;
    on[i] = at < p.values;
    const int comp = on[i] ? at / p.size : 0, channel = on[i] ? at - comp * p.size : 0;
    k_at[i] = chain * p.k_chain + comp * p.k_comp + (int64_t)kv * p.size + channel;
    v_at[i] = chain * p.v_chain + comp * p.v_comp + (int64_t)kv * p.size + channel;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float t[V];
#pragma unroll
      for (int j = 0; j < V; ++j) t[j] = 0.f;
      if (on[i] && h < here) load<T, V>(static_cast<const T*>(p.q) + chain * p.q_chain + comp * p.q_comp + (int64_t)(head0 + h) * p.size + channel, t);
#pragma unroll
      for (int j = 0; j < V; ++j) q[h][i * V + j] = t[j] * p.scale;
    }
  }
  pair q2[H][N / 2], o2[H][N / 2];
  float tops_[H], sums_[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    tops_[h] = -INFINITY;
    sums_[h] = 0.f;
#pragma unroll
    for (int c = 0; c < N / 2; ++c) {
      q2[h][c] = both(q[h][2 * c], q[h][2 * c + 1]);
      o2[h][c] = 0;
    }
  }
  auto key_of = [&](int64_t i) { return i < sinks ? i : low + i - sinks; };
  // Pieces of 16 bytes are on their way AHEAD rounds before they are used, each thread's to a place of its own, so that no thread waits for another.
  auto ask = [&](int64_t round, int place) {
    if constexpr (V > 1) {
      if (round + team < end && on[0]) {
        const int64_t j = key_of(round + team);
        attention::copy16(&ring[place][0][threadIdx.x], static_cast<const T*>(p.k) + k_at[0] + j * p.k_node, true);
        attention::copy16(&ring[place][1][threadIdx.x], static_cast<const T*>(p.v) + v_at[0] + j * p.v_node, true);
      }
      attention::copies_commit();
    }
  };
  if constexpr (V > 1) {
    if (!on[0])
      for (int i = 0; i < AHEAD; ++i) ring[i][0][threadIdx.x] = ring[i][1][threadIdx.x] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < AHEAD - 1; ++i) ask(first + i * TEAMS, i);
  }
  // all threads of a warp take as many rounds, so that the shuffles find them; teams without a key add nothing
  int place = 0;
  for (int64_t round = first; round < end; round += TEAMS) {
    const int64_t i = round + team;
    const bool there = i < end;
    float k[N], v[N];
    if constexpr (V > 1) {
      ask(round + (AHEAD - 1) * TEAMS, place == 0 ? AHEAD - 1 : place - 1);
      attention::copies_wait<AHEAD - 1>();
      unpack<V>(ring[place][0][threadIdx.x], k);
      unpack<V>(ring[place][1][threadIdx.x], v);
      if (++place == AHEAD) place = 0;
    } else {
      const int64_t j = there ? key_of(i) : 0;
#pragma unroll
      for (int m = 0; m < PIECES; ++m) {
        k[m] = there && on[m] ? static_cast<float>(static_cast<const T*>(p.k)[k_at[m] + j * p.k_node]) : 0.f;
        v[m] = there && on[m] ? static_cast<float>(static_cast<const T*>(p.v)[v_at[m] + j * p.v_node]) : 0.f;
      }
    }
    float score[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      pair sum = mul2(q2[h][0], both(k[0], k[1]));
#pragma unroll
      for (int c = 1; c < N / 2; ++c) sum = fma2(q2[h][c], both(k[2 * c], k[2 * c + 1]), sum);
      float x, y;
      parts(sum, x, y);
      score[h] = x + y;
    }
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1)
#pragma unroll
      for (int h = 0; h < H; ++h) score[h] += __shfl_xor_sync(0xffffffffu, score[h], o);
    if (there) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        if (score[h] > tops_[h] || score[h] != score[h]) {                // a new maximum (or not a number, which stays)
          const float keep = exp2_fast(tops_[h] - score[h]);
          sums_[h] *= keep;
          const pair keeps = both(keep, keep);
#pragma unroll
          for (int c = 0; c < N / 2; ++c) o2[h][c] = mul2(o2[h][c], keeps);
          tops_[h] = score[h];
        }
        const float w = score[h] == -INFINITY ? 0.f : exp2_fast(score[h] - tops_[h]);
        const pair weights = both(w, w);
        sums_[h] += w;
        if (w != 0.f) {                                  // of a weight of zero, nothing, whatever the value
#pragma unroll
          for (int c = 0; c < N / 2; ++c) o2[h][c] = fma2(weights, both(v[2 * c], v[2 * c + 1]), o2[h][c]);
        }
      }
    }
  }
  if constexpr (V > 1) attention::copies_wait<0>();
  State<N> state[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    state[h].top = tops_[h];
    state[h].sum = sums_[h];
#pragma unroll
    for (int c = 0; c < N / 2; ++c) parts(o2[h][c], state[h].o[2 * c], state[h].o[2 * c + 1]);
  }
  // teams of a warp by shuffles, then warps through shared memory
#pragma unroll
  for (int o = TEAM; o < 32; o <<= 1)
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float other[N];
      const float top = __shfl_xor_sync(0xffffffffu, state[h].top, o), sum = __shfl_xor_sync(0xffffffffu, state[h].sum, o);
#pragma unroll
      for (int c = 0; c < N; ++c) other[c] = __shfl_xor_sync(0xffffffffu, state[h].o[c], o);
      join<N>(state[h], top, sum, other);
    }
  if ((threadIdx.x & 31) < TEAM) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (lane == 0) tops[warp][h] = state[h].top, sums[warp][h] = state[h].sum;
#pragma unroll
      for (int c = 0; c < N; ++c) values[warp][h][lane * N + c] = state[h].o[c];
    }
  }
  __syncthreads();
  for (int h = warp; h < here; h += THREADS / 32) {
    if ((threadIdx.x & 31) >= TEAM) continue;
    State<N> s;
    s.top = tops[0][h];
    s.sum = sums[0][h];
#pragma unroll
    for (int c = 0; c < N; ++c) s.o[c] = values[0][h][lane * N + c];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) join<N>(s, tops[w][h], sums[w][h], &values[w][h][lane * N]);
    const int head = head0 + h;
    if (p.num_parts > 1) {
      float* to = p.parts + ((chain * p.heads + head) * p.num_parts + part) * (2 + p.values);
      if (lane == 0) to[0] = s.top, to[1] = s.sum;
#pragma unroll
      for (int m = 0; m < PIECES; ++m)
#pragma unroll
        for (int c = 0; c < V; ++c)
          if (on[m]) to[2 + (lane + m * TEAM) * V + c] = s.o[m * V + c];
    } else {
      const float inverse = visible > 0 ? 1.f / s.sum : 0.f;
#pragma unroll
      for (int m = 0; m < PIECES; ++m) {
        const int at = (lane + m * TEAM) * V, comp = at / p.size, channel = at - comp * p.size;
#pragma unroll
        for (int c = 0; c < V; ++c)
          if (on[m]) st(static_cast<T*>(p.out) + ((chain * p.comps + comp) * p.heads + head) * p.size + channel + c, s.o[m * V + c] * inverse);
      }
    }
  }
}

// The parts of a chain and head, one warp: a lane has every 32nd value.
template <typename T> __global__ void __launch_bounds__(THREADS) step_join_kernel(const StepArgs p, int64_t rows) {
  const int64_t row = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, head = (int)(row % p.heads);
  const int64_t chain = row / p.heads;
  const float* parts = p.parts + row * p.num_parts * (2 + p.values);
  State<MOST_VALUES / 32> s;
  s.top = -INFINITY;
  s.sum = 0.f;
#pragma unroll
  for (int c = 0; c < MOST_VALUES / 32; ++c) s.o[c] = 0.f;
#pragma unroll 2
  for (int i = 0; i < p.num_parts; ++i, parts += 2 + p.values) {
    float o[MOST_VALUES / 32];
#pragma unroll
    for (int c = 0; c < MOST_VALUES / 32; ++c) o[c] = lane + 32 * c < p.values ? parts[2 + lane + 32 * c] : 0.f;
    join<MOST_VALUES / 32>(s, parts[0], parts[1], o);
  }
  const float inverse = p.lengths[chain] > 0 && p.capacity > 0 ? 1.f / s.sum : 0.f;
#pragma unroll
  for (int c = 0; c < MOST_VALUES / 32; ++c) {
    const int at = lane + 32 * c, comp = at / p.size, channel = at - comp * p.size;
    if (at < p.values) st(static_cast<T*>(p.out) + ((chain * p.comps + comp) * p.heads + head) * p.size + channel, s.o[c] * inverse);
  }
}

constexpr int64_t LEAST_KEYS = 64;                       // of a part: joining costs as much as some keys
// Parts of the visible keys: so many that SMs with shorter chains take more of them.
void cut(StepArgs& p, int64_t chains, int kv_heads) {
  const int64_t visible = std::max<int64_t>(1, std::min<int64_t>(p.capacity, p.before + 1 + p.sinks));
  const int64_t others = std::max<int64_t>(1, chains * kv_heads), wanted = ceil_div((int64_t)sm_count() * 16, others);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(wanted, ceil_div(visible, LEAST_KEYS)), 1024));
  p.part_keys = ceil_div(ceil_div(visible, parts), 16) * 16;
  p.num_parts = (int)ceil_div(visible, p.part_keys);
}

template <typename T, int V, int TEAM, int PIECES, int H> int launch(const StepArgs& p, int64_t chains, int kv_heads, cudaStream_t s) {
  const dim3 grid((unsigned)p.num_parts, (unsigned)(kv_heads * ceil_div(p.group, H)), (unsigned)chains);
  step_kernel<T, V, TEAM, PIECES, H><<<grid, THREADS, 0, s>>>(p);
  if (int rc = check_launch("window_step")) return rc;
  if (p.num_parts == 1) return EQT_OK;
  const int64_t rows = chains * p.heads;
  step_join_kernel<T><<<(unsigned)ceil_div(rows, THREADS / 32), THREADS, 0, s>>>(p, rows);
  return check_launch("window_step_join");
}
template <typename T, int V, int TEAM, int PIECES> int by_group(const StepArgs& p, int64_t chains, int kv_heads, cudaStream_t s) {
  if (p.group == 1) return launch<T, V, TEAM, PIECES, 1>(p, chains, kv_heads, s);
  if (p.group == 2) return launch<T, V, TEAM, PIECES, 2>(p, chains, kv_heads, s);
  return launch<T, V, TEAM, PIECES, 4>(p, chains, kv_heads, s);
}
template <typename T> int run(const StepArgs& p, int64_t chains, int kv_heads, bool whole, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (!whole) return by_group<T, 1, 32, 4>(p, chains, kv_heads, s);
  const int pieces = (int)ceil_div(p.values, V);
  if (pieces <= 4) return by_group<T, V, 4, 1>(p, chains, kv_heads, s);
  if (pieces <= 8) return by_group<T, V, 8, 1>(p, chains, kv_heads, s);
  if (pieces <= 16) return by_group<T, V, 16, 1>(p, chains, kv_heads, s);
  return by_group<T, V, 32, 1>(p, chains, kv_heads, s);
}

int fill(StepArgs& p, const eqt_window_step_args* a) {
  if (!a) return fail(EQT_ERR_BAD_ARGUMENT, "window_step: NULL pointer");
  if (a->dtype != EQT_F32 && a->dtype != EQT_BF16) return fail(EQT_ERR_BAD_ARGUMENT, "window_step: unknown dtype %d", a->dtype);
  if (a->chains < 0 || a->capacity < 0 || a->before < 0 || a->sinks < 0 || a->heads < 1 || a->kv_heads < 1 || a->comps < 1 || a->head_channels < 1 ||
      a->heads % a->kv_heads)
    return fail(EQT_ERR_BAD_ARGUMENT, "window_step: sizes");
  if ((int64_t)a->comps * a->head_channels > MOST_VALUES || a->chains > 65535 || a->heads > 65535 || a->capacity > INT32_MAX || a->before > INT32_MAX ||
      a->sinks > INT32_MAX)
    return fail(EQT_ERR_UNSUPPORTED, "window_step: at most %d values a head, 65535 chains and heads, 2^31 nodes a chain", MOST_VALUES);
  p.q = a->q, p.k = a->k, p.v = a->v, p.out = a->out, p.parts = a->scratch, p.lengths = a->lengths;
  p.q_chain = a->q_chain, p.q_comp = a->q_comp, p.k_chain = a->k_chain, p.k_node = a->k_node, p.k_comp = a->k_comp;
  p.v_chain = a->v_chain, p.v_node = a->v_node, p.v_comp = a->v_comp;
  p.capacity = a->capacity, p.before = a->before, p.sinks = a->sinks, p.heads = a->heads, p.group = a->heads / a->kv_heads;
  p.comps = a->comps, p.size = a->head_channels, p.values = a->comps * a->head_channels, p.scale = a->scale * LOG2E;
  cut(p, a->chains, a->kv_heads);
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
  return a->chains * p.heads * p.num_parts * (2 + p.values);
}

extern "C" int eqt_window_step(const eqt_window_step_args* a, void* stream) {
  StepArgs p{};
  if (int rc = fill(p, a)) return rc;
  if (a->chains == 0) return EQT_OK;
  if (!a->q || !a->out || !a->lengths || (a->capacity && (!a->k || !a->v))) return fail(EQT_ERR_BAD_ARGUMENT, "window_step: NULL pointer");
  const int64_t need = p.num_parts == 1 ? 0 : a->chains * p.heads * p.num_parts * (2 + p.values);
  if (need && (!a->scratch || a->scratch_floats < need))
    return fail(EQT_ERR_BAD_ARGUMENT, "window_step: %lld values of scratch given, %lld needed", (long long)a->scratch_floats, (long long)need);
  const int v = a->dtype == EQT_F32 ? 4 : 8;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v);
  const int64_t strides = a->q_chain | a->q_comp | a->k_chain | a->k_node | a->k_comp | a->v_chain | a->v_node | a->v_comp;
  const bool whole = bits % 16 == 0 && strides % v == 0 && a->head_channels % v == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == EQT_F32 ? run<float>(p, a->chains, a->kv_heads, whole, s) : run<__nv_bfloat16>(p, a->chains, a->kv_heads, whole, s);
}
