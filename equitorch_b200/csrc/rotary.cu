// Rotary positions: channel pairs of every head turned by an angle that goes with the node's position along its chain.
//
//     (a, b) -> m (a cos t - b sin t,  a sin t + b cos t),     t = position * frequency[pair]
//
// of the first 2 `half` channels of a head, pairs (j, j + half) or (2 j, 2 j + 1); the other channels are passed on.  All components of a
// node's features turn alike, so that rotations of space and these commute.  The gradient is the same with -t.
//
// Bound by HBM: every value is read and written once.  A CTA takes 32 nodes at a time: their angles go to shared memory as (cos, sin), each
// computed once for all heads and components of q and k, in float64 up to what is left of whole turns (the product of a position of a
// million and a frequency has no place in float32: half an ulp of it is 0.03 of a radian).  Then a thread takes the same piece of a head for
// node after node: two times 16 bytes of both halves, or 16 bytes of neighbouring pairs; single values where these do not lie on 16-byte boundaries.
#include <algorithm>

#include "common.cuh"

namespace eqt {
namespace rotary {
namespace {

constexpr int NODES = 32, THREADS = 256;

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
  double turns;                                          // one over a whole turn, negative for the gradient
};

template <typename T> __device__ __forceinline__ float get(const T* p) { return static_cast<float>(*p); }

// V values of a head at `from`: pairs of places (first, second) and the angles' places
template <typename T, int V, bool INTERLEAVED>
__device__ __forceinline__ void turn_piece(const T* from, T* to, const float2* angles, int unit, int half, float magnitude) {
  if constexpr (V == 1) {
    const int pairs = half;
    if (unit < pairs) {
      const int i = INTERLEAVED ? 2 * unit : unit, j = INTERLEAVED ? 2 * unit + 1 : unit + half;
      const float a = get(from + i) * magnitude, b = get(from + j) * magnitude;
      const float2 t = angles[unit];
      st(to + i, a * t.x - b * t.y);
      st(to + j, a * t.y + b * t.x);
    } else {
      to[half + unit] = from[half + unit];
    }
  } else {
    constexpr int W = 4;                                 // words of 16 bytes
    auto words = [](const T* p, float (&v)[V]) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t r[W] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (V == 4) v[i] = __uint_as_float(r[i]);
        else v[2 * i] = __uint_as_float(r[i] << 16), v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
      }
    };
    auto put = [](T* p, const float (&v)[V]) {
      uint32_t r[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (V == 4) r[i] = __float_as_uint(v[i]);
        else {
          const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          r[i] = *reinterpret_cast<const uint32_t*>(&two);
        }
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    };
    const int turned = INTERLEAVED ? 2 * half / V : half / V;
    if (unit >= turned) {
      const int at = (INTERLEAVED ? unit : unit + turned) * V;
      *reinterpret_cast<uint4*>(to + at) = __ldg(reinterpret_cast<const uint4*>(from + at));
      return;
    }
    float a[V];
    words(from + unit * V, a);
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float2 t = angles[(unit * V + i) / 2];
        const float x = a[i] * magnitude, y = a[i + 1] * magnitude;
        a[i] = x * t.x - y * t.y;
        a[i + 1] = x * t.y + y * t.x;
      }
    } else {
      float b[V];
      words(from + half + unit * V, b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 t = angles[unit * V + i];
        const float x = a[i] * magnitude, y = b[i] * magnitude;
        a[i] = x * t.x - y * t.y;
        b[i] = x * t.y + y * t.x;
      }
      put(to + half + unit * V, b);
    }
    put(to + unit * V, a);
  }
}

template <typename T, int V, bool INTERLEAVED> __global__ void __launch_bounds__(THREADS) rotary_kernel(const RotaryArgs p) {
  extern __shared__ float2 angles[];                     // [node][pair]
  const int a_side = p.comps * p.side[0].heads * p.units, per_node = a_side + (p.sides > 1 ? p.comps * p.side[1].heads * p.units : 0);
  const int together = max(1, THREADS / per_node);       // nodes that the CTA's threads take at a time
  for (int64_t first = (int64_t)blockIdx.x * NODES; first < p.n; first += (int64_t)gridDim.x * NODES) {
    const int here = (int)min((int64_t)NODES, p.n - first);
    __syncthreads();
    for (int i = threadIdx.x; i < here * p.half; i += THREADS) {
      const int node = i / p.half, pair = i - node * p.half;
      double t = (double)p.positions[first + node] * (p.frequencies[pair] * p.turns);
      t -= rint(t);
      float s, c;
      sincospif(2.f * (float)t, &s, &c);
      angles[i] = make_float2(c, s);
    }
    __syncthreads();
    for (int at = threadIdx.x; at < together * per_node; at += THREADS) {
      const int sub = at / per_node;
      int piece = at - sub * per_node;
      const bool second = piece >= a_side;
      const Rows& rows = p.side[second];
      if (second) piece -= a_side;
      const int unit = piece % p.units, head = piece / p.units % rows.heads, comp = piece / p.units / rows.heads;
      const T* from = static_cast<const T*>(rows.in) + (first + sub) * rows.node + comp * rows.comp + (int64_t)head * p.size;
      T* to = static_cast<T*>(rows.out) + (first + sub) * rows.out_node + comp * rows.out_comp + (int64_t)head * p.size;
#pragma unroll 4
      for (int node = sub; node < here; node += together, from += together * rows.node, to += together * rows.out_node)
        turn_piece<T, V, INTERLEAVED>(from, to, angles + node * p.half, unit, p.half, p.magnitude);
    }
  }
}

template <typename T, int V> int launch(const RotaryArgs& p, bool interleaved, cudaStream_t s) {
  const size_t shared = (size_t)NODES * p.half * sizeof(float2);
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(p.n, NODES), (int64_t)sm_count() * 16);
  if (interleaved) rotary_kernel<T, V, true><<<grid, THREADS, shared, s>>>(p);
  else rotary_kernel<T, V, false><<<grid, THREADS, shared, s>>>(p);
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
  p.turns = (a->backward ? -1.0 : 1.0) * 0.15915494309189533577;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == EQT_F32 ? run<float>(p, a->interleaved != 0, s) : run<__nv_bfloat16>(p, a->interleaved != 0, s);
}
