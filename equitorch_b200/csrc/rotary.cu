// Rotary positions: channel pairs of every head turned by an angle that goes with the node's position along its chain.
//
//     (a, b) -> m (a cos t - b sin t,  a sin t + b cos t),     t = position * frequency[pair]
//
// of the first 2 `half` channels of a head, pairs (j, j + half) or (2 j, 2 j + 1); the other channels are passed on.  All components of a
// node's features turn alike, so that rotations of space and these commute.  The gradient is the same with -t.
//
// Bound by HBM: every value is read and written once.  A CTA's angles go to shared memory as (cos, sin), each computed once for all heads and
// components of q and k, in pairs of float64 up to what is left of whole turns, for any position (the product of a position of a million and a frequency has no
// place in float32: half an ulp of it is 0.03 of a radian; one of 2^40 loses 2e-4 in float64).  A thread has the same piece of a head of four nodes in registers, on their way while the angles
// are made: two times 16 bytes of both halves, or 16 bytes of neighbouring pairs; single values where these do not lie on 16-byte boundaries.
// 65,536 nodes, 8 and 2 heads of 64 bfloat16 values: 34 us (4.9 TB/s) each way, 33.5 with angles in single float64 numbers.
#include <algorithm>

#include "common.cuh"

namespace eqt {
namespace rotary {
namespace {

constexpr int THREADS = 128, AT_ONCE = 4;                // AT_ONCE: nodes whose pieces a thread has in registers

struct Rows {                                            // q or k
  const void* in;
  void* out;
  int64_t node, comp, out_node, out_comp;                // strides in values
  int heads;
};
struct RotaryArgs {
  Rows side[2];
  const int64_t* positions;
  const double* frequencies;
  int64_t n;
  int comps, size, half, sides, units;                   // units: pieces of a head
  float magnitude;
  float sign;                                            // negative for the gradient
};

// What a position's angle is of a turn, within half of one.  Position, their product and one over a whole turn are sums of two float64 numbers each, and what the
// first parts' product is of whole turns goes before anything is added to it.
__device__ __forceinline__ float part_of_turn(int64_t position, double frequency) {
  constexpr double TURN = 0.15915494309189533577, TURN_REST = -9.839338337591243e-18;          // 1 / 2 pi
  const double at = (double)position;
  const uint64_t whole = at == 9223372036854775808.0 ? uint64_t(1) << 63 : (uint64_t)(int64_t)at;
  const double rest = (double)(int64_t)((uint64_t)position - whole);
  const double angle = at * frequency, angle_rest = fma(at, frequency, -angle) + rest * frequency;
  const double turns = angle * TURN, turns_rest = fma(angle, TURN, -turns) + (angle * TURN_REST + angle_rest * TURN);
  const double left = turns - rint(turns) + turns_rest;
  return (float)(left - rint(left));
}

// A piece as it lies in memory: 16 bytes, or one value, of each of the two places that turn together (interleaved: of the one place).
template <typename T, int V> struct Raw { using type = uint4; };
template <typename T> struct Raw<T, 1> { using type = T; };
template <typename T, int V> __device__ __forceinline__ void open(const typename Raw<T, V>::type& raw, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = static_cast<float>(raw);
  } else {
    const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 4) v[i] = __uint_as_float(r[i]);
      else v[2 * i] = __uint_as_float(r[i] << 16), v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
}
template <typename T, int V> __device__ __forceinline__ void put(T* to, const float (&v)[V]) {
  if constexpr (V == 1) {
    st(to, v[0]);
  } else {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 4) r[i] = __float_as_uint(v[i]);
      else {
        const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        r[i] = *reinterpret_cast<const uint32_t*>(&two);
      }
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

// The same roundings wherever it is called, so that results do not go by alignment.
__device__ __forceinline__ void turn(float a, float b, float2 t, float& x, float& y) {
  x = fmaf(a, t.x, -__fmul_rn(b, t.y));
  y = fmaf(a, t.y, __fmul_rn(b, t.x));
}

// Where a thread's piece of a head is.
template <typename T, int V, bool INTERLEAVED> struct Place {
  const T* from;
  T* to;
  int64_t in_step, out_step;                             // between nodes
  int first, second, pair;                               // channels of the two places (of the one: `second` < 0), their first pair; none turns: `pair` < 0
  __device__ __forceinline__ Place(const RotaryArgs& p, int piece, int a_side, int64_t node) {
    const bool other = piece >= a_side;
    const Rows& rows = p.side[other];
    if (other) piece -= a_side;
    const int unit = piece % p.units, head = piece / p.units % rows.heads, comp = piece / p.units / rows.heads;
    in_step = rows.node;
    out_step = rows.out_node;
    from = static_cast<const T*>(rows.in) + node * in_step + comp * rows.comp + (int64_t)head * p.size;
    to = static_cast<T*>(rows.out) + node * out_step + comp * rows.out_comp + (int64_t)head * p.size;
    if constexpr (V == 1) {                              // a pair, or one channel behind the pairs
      const bool turns = unit < p.half;
      pair = turns ? unit : -1;
      first = !turns ? p.half + unit : INTERLEAVED ? 2 * unit : unit;
      second = !turns ? -1 : INTERLEAVED ? 2 * unit + 1 : unit + p.half;
    } else if constexpr (INTERLEAVED) {
      first = unit * V;
      second = -1;
      pair = first < 2 * p.half ? first / 2 : -1;
    } else {
      const bool turns = unit * V < p.half;
      pair = turns ? unit * V : -1;
      first = turns ? unit * V : unit * V + p.half;
      second = turns ? unit * V + p.half : -1;
    }
  }
};

template <typename T, int V, bool INTERLEAVED> __global__ void __launch_bounds__(THREADS) rotary_kernel(const RotaryArgs p, int together) {
  using R = typename Raw<T, V>::type;
  using Q = Place<T, V, INTERLEAVED>;
  extern __shared__ float2 angles[];                     // [node][pair]
  const int a_side = p.comps * p.side[0].heads * p.units, per_node = a_side + (p.sides > 1 ? p.comps * p.side[1].heads * p.units : 0);
  const int nodes = together * AT_ONCE, pieces = together * per_node;
  for (int64_t first = (int64_t)blockIdx.x * nodes; first < p.n; first += (int64_t)gridDim.x * nodes) {
    const int here = (int)min((int64_t)nodes, p.n - first);
    bool ready = false;                                  // the angles
    // all threads take as many rounds: the first one's pieces are on their way while the angles are made
    for (int at0 = 0; at0 < pieces; at0 += THREADS) {
      const int at = at0 + threadIdx.x, sub = at / per_node;
      const bool mine = at < pieces;
      const Q place(p, mine ? at - sub * per_node : 0, a_side, first + (mine ? sub : 0));
      R a[AT_ONCE], b[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        if (mine && sub + i * together < here) {
          const T* from = place.from + (int64_t)i * together * place.in_step;
          a[i] = *reinterpret_cast<const R*>(from + place.first);
          if (place.second >= 0) b[i] = *reinterpret_cast<const R*>(from + place.second);
        }
      if (!ready) {
        __syncthreads();
        for (int i = threadIdx.x; i < here * p.half; i += THREADS) {
          const int node = i / p.half, pair = i - node * p.half;
          float s, c;
          sincospif(2.f * p.sign * part_of_turn(p.positions[first + node], p.frequencies[pair]), &s, &c);
          angles[i] = make_float2(c * p.magnitude, s * p.magnitude);
        }
        __syncthreads();
        ready = true;
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        if (mine && sub + i * together < here) {
          T* to = place.to + (int64_t)i * together * place.out_step;
          if (place.pair < 0) {
            *reinterpret_cast<R*>(to + place.first) = a[i];
            continue;
          }
          const float2* t = angles + (sub + i * together) * p.half + place.pair;
          float x[V], y[V];
          open<T, V>(a[i], x);
          if constexpr (INTERLEAVED && V > 1) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
              const float u = x[j], v = x[j + 1];
              turn(u, v, t[j / 2], x[j], x[j + 1]);
            }
          } else {
            open<T, V>(b[i], y);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float u = x[j], v = y[j];
              turn(u, v, t[j], x[j], y[j]);
            }
            put<T, V>(to + place.second, y);
          }
          put<T, V>(to + place.first, x);
        }
    }
  }
}

template <typename T, int V> int launch(const RotaryArgs& p, bool interleaved, cudaStream_t s) {
  int64_t heads = p.side[0].heads + (p.sides > 1 ? p.side[1].heads : 0);
  const int together = (int)std::max<int64_t>(1, std::min<int64_t>(THREADS / (p.comps * heads * p.units), 8192 / (std::max(1, p.half) * AT_ONCE * sizeof(float2))));
  const size_t shared = (size_t)together * AT_ONCE * p.half * sizeof(float2);
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(p.n, together * AT_ONCE), (int64_t)sm_count() * 64);
  if (interleaved) rotary_kernel<T, V, true><<<grid, THREADS, shared, s>>>(p, together);
  else rotary_kernel<T, V, false><<<grid, THREADS, shared, s>>>(p, together);
  return check_launch("rotary");
}
template <typename T> int run(RotaryArgs& p, bool interleaved, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  bool whole = p.size % V == 0 && (interleaved ? 2 * p.half : p.half) % V == 0;
  for (int i = 0; i < p.sides; ++i) {
    const Rows& r = p.side[i];
    whole = whole && (reinterpret_cast<uintptr_t>(r.in) | reinterpret_cast<uintptr_t>(r.out)) % 16 == 0 && (r.node | r.comp | r.out_node | r.out_comp) % V == 0;
  }
  if (whole) {
    p.units = interleaved ? p.size / V : p.half / V + (p.size - 2 * p.half) / V;
    return launch<T, V>(p, interleaved, s);
  }
  p.units = p.size - p.half;                             // pairs and single channels
  return launch<T, 1>(p, interleaved, s);
}

}  // namespace
}  // namespace rotary
}  // namespace eqt

using namespace eqt;
using namespace eqt::rotary;

extern "C" int eqt_rotary(const eqt_rotary_args* a, void* stream) {
  if (!a) return fail(EQT_ERR_BAD_ARGUMENT, "rotary: NULL pointer");
  if (a->dtype != EQT_F32 && a->dtype != EQT_BF16) return fail(EQT_ERR_BAD_ARGUMENT, "rotary: unknown dtype %d", a->dtype);
  if (a->n < 0 || a->comps < 0 || a->heads < 0 || a->kv_heads < 0 || a->size < 1 || a->half < 0 || 2 * (int64_t)a->half > a->size)
    return fail(EQT_ERR_BAD_ARGUMENT, "rotary: sizes");
  const bool pair = a->k != nullptr;
  if ((int64_t)a->comps * ((int64_t)a->heads + a->kv_heads) * a->size > 1 << 24 || a->half > 512 || a->n > INT32_MAX)
    return fail(EQT_ERR_UNSUPPORTED, "rotary: at most 2^31 nodes of 2^24 values and 512 pairs a head");
  if (a->n == 0 || a->comps == 0 || (int64_t)a->heads + (pair ? a->kv_heads : 0) == 0) return EQT_OK;
  if (!a->q || !a->q_out || (pair && !a->k_out) || !a->positions || (a->half && !a->frequencies)) return fail(EQT_ERR_BAD_ARGUMENT, "rotary: NULL pointer");
  RotaryArgs p{};
  const int64_t width = (int64_t)a->heads * a->size, kv_width = (int64_t)a->kv_heads * a->size;
  p.side[0] = {a->q, a->q_out, a->q_node, a->q_comp, a->comps * width, width, a->heads};
  p.side[1] = {a->k, a->k_out, a->k_node, a->k_comp, a->comps * kv_width, kv_width, a->kv_heads};
  p.sides = pair ? 2 : 1;
  p.positions = a->positions, p.frequencies = a->frequencies, p.n = a->n, p.comps = a->comps, p.size = a->size, p.half = a->half;
  p.magnitude = a->magnitude;
  p.sign = a->backward ? -1.f : 1.f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == EQT_F32 ? run<float>(p, a->interleaved != 0, s) : run<__nv_bfloat16>(p, a->interleaved != 0, s);
}
