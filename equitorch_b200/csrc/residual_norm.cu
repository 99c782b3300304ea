// Root-mean-square norm of a node's values with the residual's addition before it, forward, backward, and with the result in 8 bits.
//
// A row is a node's D = d C values (components times channels), so that the norm of equivariant features is invariant:
//
//     h = x + res      r = (mean h^2 + eps)^-1/2      y = h r w[channel]
//     backward, from g = dL/dy and gh = dL/dh (the stream goes on):  gw = g w,  u = h r
//         dx = dres = gh + r (gw - u mean(gw u))        dw[channel] = sum over nodes and components of g u
//     8 bits: of every group of values, t = h w, m = max |t|:   value = e4m3(448 t / m), scale = m r / 448
//
// All of it is bound by HBM: 18 bytes a bfloat16 value forward and backward (x, res, out, h; g, gh, x, res, dx).  Of bfloat16 the backward pass reads x and the
// residual and not the sum as it was returned, whose rounding would go into dw beside dw's own (2-norm of the error 2.5e-3 | 1.7e-3; backward pass
// 137 | 158 us).  A row stays in the registers of 32, 128 or 512 threads, one, two or four pieces of 16 bytes each: one reads x and the residual,
// adds, reduces by shuffles and writes.  A CTA strides over the rows, so the weight is read once and the backward pass has the weight's gradient in
// registers, summed over the CTA's rows; the CTAs' sums are added in their order by a second kernel (no atomics).  Rows that are no whole pieces of 16
// bytes, or longer than 2048 pieces, are read twice by loops.
// 100,003 nodes of 4 x 256 bfloat16 values: forward 130 us (6.3 TB/s), backward 158 (6.5 TB/s), the weight's sums 15.  8 bits, 32,768 x 2048 in groups of 128:
// 123 us (3.9 TB/s), where the exact quotients' instructions count.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace eqt {
namespace residual_norm {
namespace {

constexpr float E4M3_MAX = 448.f;

struct NormArgs {
  const void *x, *res, *w, *g, *gh;
  void *y, *total, *dx, *dw;
  uint8_t* values;
  float *scales, *rstd, *parts;
  int64_t n;
  int length, channels, group;                           // values of a row; of a group of 8-bit values
  float eps;
};

template <typename T> constexpr int VALUES = 16 / (int)sizeof(T);

template <typename T> __device__ __forceinline__ void unpack(const uint4& u, float (&v)[VALUES<T>]) {
  const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(r[i]);
    } else {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
}
template <typename T> __device__ __forceinline__ void add_to(const uint4& u, float (&v)[VALUES<T>]) {
  float a[VALUES<T>];
  unpack<T>(u, a);
#pragma unroll
  for (int j = 0; j < VALUES<T>; ++j) v[j] += a[j];
}
template <typename T> __device__ __forceinline__ uint4 pack(const float (&v)[VALUES<T>]) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      r[i] = __float_as_uint(v[i]);
    } else {
      const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      r[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

struct Sum {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Max {                                             // drops NaNs
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
};
// Over `lanes` neighbouring threads of a warp, a power of two.
template <typename V, typename F> __device__ __forceinline__ V across_lanes(V v, int lanes, F f) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Over the THREADS of a row, all of which call it; `buffer` holds a value a warp and is not the one of the call before.
template <int THREADS, typename V, typename F> __device__ __forceinline__ V across_row(V v, V* buffer, F f) {
  v = across_lanes(v, 32, f);
  if constexpr (THREADS > 32) {
    if ((threadIdx.x & 31) == 0) buffer[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buffer[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) v = f(v, buffer[i]);
  }
  return v;
}

// One over the root, as rounded once.
__device__ __forceinline__ float inverse_root(float sum, int length, float eps) { return __frsqrt_rn(sum / (float)length + eps); }

// ---- 8 bits -------------------------------------------------------------------------------------
// The result is the nearest of 8 bits to 448 t / m, ties to even, as if computed without rounding before.  In float32, with at most six
// roundings, the quotient is within 2^-21 of itself; where that leaves two answers (two or three values in 100,000, more where t and m have
// few bits and ties are real) it is formed in float64 and brought to float32 rounding to odd, which keeps on which side of a border it is.
__device__ __forceinline__ uint8_t to_e4m3(float v) { return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint16_t to_e4m3(float v, float w) { return (uint16_t)__nv_cvt_float2_to_fp8x2(make_float2(v, w), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint8_t to_e4m3_exact(double t, double m) {
  const double q = t * (double)E4M3_MAX / m;
  float f = __double2float_rz(q);
  if ((double)f != q) f = __uint_as_float(__float_as_uint(f) | 1u);
  return to_e4m3(f);
}
constexpr float NEAR = 4.76837158203125e-7f;             // 2^-21
constexpr float TINY = 1e-30f;                           // below it 448 / m may be infinite
// m r / 448, whose last steps must not round to a number below the normal ones before the others have brought it up.
__device__ __forceinline__ float scale_of(float most, float inverse) { return (float)((double)most * (double)inverse * (1.0 / (double)E4M3_MAX)); }
__device__ __forceinline__ double exact_value(float x, float res, float w) { return ((double)x + (double)res) * (double)w; }

// ---- rows in registers --------------------------------------------------------------------------
// The 8-bit values of a piece, the long way, from memory (`x` NULL: no piece).  The group's greatest |t| comes from the threads whose values are within an error of `m`,
// the greatest in float32, in float64; the group is `lanes` threads, or (0) known: `known`.  A call and not in line: in line it takes the kernel from 68 to 168
// registers a thread, and all rows pay for it (32,768 x 2048: 85 | 138 us).
template <typename T> __device__ __forceinline__ double exact_most(const uint4& x, const uint4& res, const uint4& w, float m) {
  constexpr int V = VALUES<T>;
  float a[V], b[V], c[V];
  unpack<T>(x, a);
  unpack<T>(res, b);
  unpack<T>(w, c);
  double most = 0.0;
#pragma unroll 1
  for (int j = 0; j < V; ++j) {
    float ta = a[0], tb = b[0], tc = c[0];
#pragma unroll
    for (int i = 1; i < V; ++i)
      if (i == j) ta = a[i], tb = b[i], tc = c[i];
    if (fabsf((ta + tb) * tc) >= m * (1.f - NEAR)) most = fmax(most, fabs(exact_value(ta, tb, tc)));
  }
  return most;
}
template <typename T> __device__ __forceinline__ void load_piece(const uint4* x, const uint4* res, const uint4* w, uint4& a, uint4& b, uint4& c) {
  a = b = c = make_uint4(0, 0, 0, 0);
  if (!x) return;
  a = __ldg(x);
  if (res) b = __ldg(res);
  if (w) c = __ldg(w);
  else if constexpr (sizeof(T) == 4) c = make_uint4(0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u);
  else c = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
}
template <typename T> __device__ __noinline__ double exact_greatest(const uint4* x, const uint4* res, const uint4* w, float m) {
  uint4 a, b, c;
  load_piece<T>(x, res, w, a, b, c);
  return exact_most<T>(a, b, c, m);
}
template <typename T> __device__ __noinline__ uint2 exact_piece(const uint4* x, const uint4* res, const uint4* w, float m, int lanes, double known) {
  constexpr int V = VALUES<T>;
  uint4 x4, r4, w4;
  load_piece<T>(x, res, w, x4, r4, w4);
  const double most = lanes ? across_lanes(exact_most<T>(x4, r4, w4, m), lanes, Max()) : known;
  float a[V], b[V], c[V];
  unpack<T>(x4, a);
  unpack<T>(r4, b);
  unpack<T>(w4, c);
  const float to = m > 0.f ? __fdiv_rn(E4M3_MAX, m) : 0.f;
  uint32_t words[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float t = (a[j] + b[j]) * c[j];
    uint32_t held = to_e4m3(t * (to * (1.f - NEAR)));
    if (held != to_e4m3(t * (to * (1.f + NEAR))) || (m < TINY && m > 0.f)) held = to_e4m3_exact(exact_value(a[j], b[j], c[j]), most);
    words[j / 4] |= held << (8 * (j & 3));
  }
  return make_uint2(words[0], words[1]);
}

// OUT: 0 values of the type, 1 8 bits with a scale a row, 2 with a scale every p.group values (whole pieces, a power of two of at most 32)
template <typename T, int ROW_THREADS, int PIECES, int OUT, bool RES>
__global__ void __launch_bounds__(ROW_THREADS < 128 ? 128 : ROW_THREADS, OUT != 0 && PIECES <= 2 && ROW_THREADS < 512 ? 6 : 1) forward_kernel(const NormArgs p) {
  constexpr int V = VALUES<T>, ROWS = ROW_THREADS < 128 ? 128 / ROW_THREADS : 1;
  __shared__ float buffer[2][ROW_THREADS / 32], most_of[2][ROW_THREADS / 32];
  __shared__ double exact_of[2][ROW_THREADS / 32];
  const int at = threadIdx.x % ROW_THREADS, pieces = p.length / V;
  float c[PIECES][V];                                    // weights
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int k = at + i * ROW_THREADS;
#pragma unroll
    for (int j = 0; j < V; ++j) c[i][j] = 1.f;
    if (p.w && k < pieces) unpack<T>(reinterpret_cast<const uint4*>(p.w)[k % (p.channels / V)], c[i]);
  }
  bool bad_weight = false;                               // one that is not finite: no scale is a number then
  if constexpr (OUT != 0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) bad_weight = bad_weight || !(fabsf(c[i][j]) < INFINITY);
    bad_weight = __syncthreads_or(bad_weight);
  }
  int turn = 0;
  constexpr bool AHEAD = PIECES <= 2;                    // the next row is on its way while this one is worked on
  uint4 x[PIECES], r[PIECES], next_x[PIECES], next_r[PIECES];
  auto ask = [&](int64_t row, uint4 (&a)[PIECES], uint4 (&b)[PIECES]) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int k = at + i * ROW_THREADS;
      const bool on = row < p.n && k < pieces;
      a[i] = on ? __ldg(reinterpret_cast<const uint4*>(p.x) + row * pieces + k) : make_uint4(0, 0, 0, 0);
      if (RES) b[i] = on ? __ldg(reinterpret_cast<const uint4*>(p.res) + row * pieces + k) : make_uint4(0, 0, 0, 0);
    }
  };
  const int64_t step = (int64_t)gridDim.x * ROWS;
  if (AHEAD) ask((int64_t)blockIdx.x * ROWS + threadIdx.x / ROW_THREADS, next_x, next_r);
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < p.n; row0 += step, turn ^= 1) {
    const int64_t row = row0 + threadIdx.x / ROW_THREADS;
    const bool there = row < p.n;
    const int64_t first = row * pieces;
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        x[i] = next_x[i];
        if (RES) r[i] = next_r[i];
      }
      ask(row + step, next_x, next_r);
    } else {
      ask(row, x, r);
    }
    float h[PIECES][V], sum = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      unpack<T>(x[i], h[i]);
      if (RES) {
        float b[V];
        unpack<T>(r[i], b);
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] += b[j];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum = fmaf(h[i][j], h[i][j], sum);
    }
    sum = across_row<ROW_THREADS>(sum, buffer[turn], Sum());
    const float inverse = inverse_root(sum, p.length, p.eps);
    if (p.rstd && at == 0 && there) p.rstd[row] = inverse;
    if (RES && p.total) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int k = at + i * ROW_THREADS;
        if (there && k < pieces) reinterpret_cast<uint4*>(p.total)[first + k] = pack<T>(h[i]);
      }
    }
    if constexpr (OUT == 0) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int k = at + i * ROW_THREADS;
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = h[i][j] * inverse * c[i][j];
        if (there && k < pieces) reinterpret_cast<uint4*>(p.y)[first + k] = pack<T>(y);
      }
    } else {
      const int lanes = OUT == 2 ? p.group / V : 32;
      float most[PIECES], all = 0.f;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        most[i] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          h[i][j] *= c[i][j];
          most[i] = Max()(most[i], fabsf(h[i][j]));
        }
        if (OUT == 2) most[i] = across_lanes(most[i], lanes, Max());
        else all = Max()(all, most[i]);
      }
      if (OUT == 1) all = across_row<ROW_THREADS>(all, most_of[turn], Max());
      // both ends of what the quotient may be: one answer, or the long way round
      uint16_t held[PIECES][V / 2];
      unsigned unsure = 0;                               // no branches: any difference leaves a bit
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        if (OUT == 1) most[i] = all;
        const float to = most[i] > 0.f ? __fdiv_rn(E4M3_MAX, most[i]) : 0.f, less = to * (1.f - NEAR), more = to * (1.f + NEAR);
        unsure |= (unsigned)(most[i] < TINY) & (unsigned)(most[i] > 0.f);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          held[i][j / 2] = to_e4m3(h[i][j] * less, h[i][j + 1] * less);
          unsure |= held[i][j / 2] ^ to_e4m3(h[i][j] * more, h[i][j + 1] * more);
        }
      }
      const bool again = OUT == 1 ? __syncthreads_or(unsure != 0) : __any_sync(0xffffffffu, unsure != 0);
      if (again) {
        auto of = [&](const void* base, int64_t from, bool on) { return base && on ? reinterpret_cast<const uint4*>(base) + from : nullptr; };
        double known = 0.0;
        for (int step = OUT == 1 ? 0 : 1; step < 2; ++step) {             // a row's greatest first
#pragma unroll 1
          for (int i = 0; i < PIECES; ++i) {
            const int k = at + i * ROW_THREADS;
            const bool on = there && k < pieces;
            const uint4 *px = of(p.x, first + k, on), *pr = of(p.res, first + k, on), *pw = of(p.w, k % (p.channels / V), on);
            float m = most[0];
#pragma unroll
            for (int q = 1; q < PIECES; ++q) m = q == i ? most[q] : m;
            if (step == 0) {
              known = fmax(known, exact_greatest<T>(px, pr, pw, m));
              continue;
            }
            const uint2 words = exact_piece<T>(px, pr, pw, m, OUT == 2 ? lanes : 0, known);
            if (!on) continue;
            if constexpr (V == 8) reinterpret_cast<uint2*>(p.values)[first + k] = words;
            else reinterpret_cast<uint32_t*>(p.values)[first + k] = words.x;
          }
          if (OUT == 1 && step == 0) known = across_row<ROW_THREADS>(known, exact_of[turn], Max());
        }
      }
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int k = at + i * ROW_THREADS;
        if (!there || k >= pieces) continue;
        uint8_t* to_values = p.values + (first + k) * V;
        if (again) {
        } else if constexpr (V == 8) *reinterpret_cast<uint2*>(to_values) = make_uint2(held[i][0] | (uint32_t)held[i][1] << 16, held[i][2] | (uint32_t)held[i][3] << 16);
        else
          *reinterpret_cast<uint32_t*>(to_values) = held[i][0] | (uint32_t)held[i][1] << 16;
        const float scale = bad_weight || !(sum < INFINITY) ? NAN : scale_of(most[i], inverse);
        if (OUT == 2 && k % lanes == 0) p.scales[(first + k) / lanes] = scale;
        if (OUT == 1 && k == 0) p.scales[row] = scale;
      }
    }
  }
}

// parts [CTA][values of a row]: the CTA's sums of g u
template <typename T, int ROW_THREADS, int PIECES, bool RES>
__global__ void __launch_bounds__(ROW_THREADS < 128 ? 128 : ROW_THREADS) backward_kernel(const NormArgs p) {
  constexpr int V = VALUES<T>, ROWS = ROW_THREADS < 128 ? 128 / ROW_THREADS : 1;
  __shared__ float buffer[2][ROW_THREADS / 32];
  __shared__ float sums[ROWS > 1 ? PIECES * 32 * V : 1];
  const int at = threadIdx.x % ROW_THREADS, pieces = p.length / V;
  uint4 w[PIECES];
  float dw[PIECES][V];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int k = at + i * ROW_THREADS;
    w[i] = make_uint4(0, 0, 0, 0);
    if (p.w && k < pieces) w[i] = reinterpret_cast<const uint4*>(p.w)[k % (p.channels / V)];
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = 0.f;
  }
  int turn = 0;
  constexpr bool AHEAD = PIECES <= 2;
  uint4 g[PIECES], t[PIECES], e[PIECES], s[PIECES], next_g[PIECES], next_t[PIECES], next_e[PIECES], next_s[PIECES];
  float inverse, next_inverse = 0.f;
  auto ask = [&](int64_t row, uint4 (&a)[PIECES], uint4 (&b)[PIECES], uint4 (&d)[PIECES], uint4 (&c)[PIECES], float& root) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int k = at + i * ROW_THREADS;
      const bool on = row < p.n && k < pieces;
      a[i] = on ? __ldg(reinterpret_cast<const uint4*>(p.g) + row * pieces + k) : make_uint4(0, 0, 0, 0);
      b[i] = on ? __ldg(reinterpret_cast<const uint4*>(p.total) + row * pieces + k) : make_uint4(0, 0, 0, 0);
      if (RES) d[i] = on ? __ldg(reinterpret_cast<const uint4*>(p.res) + row * pieces + k) : make_uint4(0, 0, 0, 0);
      c[i] = p.gh && on ? __ldg(reinterpret_cast<const uint4*>(p.gh) + row * pieces + k) : make_uint4(0, 0, 0, 0);
    }
    root = row < p.n ? __ldg(p.rstd + row) : 0.f;
  };
  const int64_t step = (int64_t)gridDim.x * ROWS;
  if (AHEAD) ask((int64_t)blockIdx.x * ROWS + threadIdx.x / ROW_THREADS, next_g, next_t, next_e, next_s, next_inverse);
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < p.n; row0 += step, turn ^= 1) {
    const int64_t row = row0 + threadIdx.x / ROW_THREADS;
    const bool there = row < p.n;
    const int64_t first = row * pieces;
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        g[i] = next_g[i], t[i] = next_t[i], s[i] = next_s[i];
        if (RES) e[i] = next_e[i];
      }
      inverse = next_inverse;
      ask(row + step, next_g, next_t, next_e, next_s, next_inverse);
    } else {
      ask(row, g, t, e, s, inverse);
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      float a[V], c[V], h[V];
      unpack<T>(g[i], a);
      unpack<T>(w[i], c);
      unpack<T>(t[i], h);
      if (RES) add_to<T>(e[i], h);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float u = h[j] * inverse;
        dw[i][j] = fmaf(a[j], u, dw[i][j]);
        sum = fmaf(p.w ? a[j] * c[j] : a[j], u, sum);
      }
    }
    const float mean = across_row<ROW_THREADS>(sum, buffer[turn], Sum()) / (float)p.length;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int k = at + i * ROW_THREADS;
      float a[V], c[V], h[V], more[V], out[V];
      unpack<T>(g[i], a);
      unpack<T>(w[i], c);
      unpack<T>(t[i], h);
      if (RES) add_to<T>(e[i], h);
      unpack<T>(s[i], more);
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = fmaf(inverse, fmaf(-(h[j] * inverse), mean, p.w ? a[j] * c[j] : a[j]), more[j]);
      if (there && k < pieces) reinterpret_cast<uint4*>(p.dx)[first + k] = pack<T>(out);
    }
  }
  if (!p.parts) return;
  float* part = p.parts + (int64_t)blockIdx.x * p.length;
  if constexpr (ROWS > 1) {                              // the CTA's rows in their order
    for (int q = 0; q < ROWS; ++q) {
      if ((int)threadIdx.x / ROW_THREADS == q) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float& sum = sums[(i * 32 + at) * V + j];
            sum = q ? sum + dw[i][j] : dw[i][j];
          }
      }
      __syncthreads();
    }
    for (int k = threadIdx.x; k < p.length; k += blockDim.x) part[k] = sums[k];
  } else {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int k = at + i * ROW_THREADS;
      if (k >= pieces) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) part[k * V + j] = dw[i][j];
    }
  }
}

// ---- rows of any length and alignment -----------------------------------------------------------
constexpr int LONG_THREADS = 256;
template <typename T, bool EIGHT> __global__ void __launch_bounds__(LONG_THREADS) forward_long_kernel(const NormArgs p) {
  __shared__ float buffer[2][LONG_THREADS / 32], most_of[2][LONG_THREADS / 32];
  __shared__ double exact_of[2][LONG_THREADS / 32];
  const T *x = static_cast<const T*>(p.x), *res = static_cast<const T*>(p.res), *w = static_cast<const T*>(p.w);
  bool bad_weight = false;
  if constexpr (EIGHT) {
    if (w)
      for (int k = threadIdx.x; k < p.channels; k += LONG_THREADS) bad_weight = bad_weight || !(fabsf(ld(w + k)) < INFINITY);
    bad_weight = __syncthreads_or(bad_weight);
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x, turn ^= 1) {
    const int64_t first = row * p.length;
    auto value = [&](int k) { return ld(x + first + k) + (res ? ld(res + first + k) : 0.f); };
    auto weight = [&](int k) { return w ? ld(w + k % p.channels) : 1.f; };
    auto exact_at = [&](int k) { return fabs(exact_value(ld(x + first + k), res ? ld(res + first + k) : 0.f, weight(k))); };
    float sum = 0.f;
    for (int k = threadIdx.x; k < p.length; k += LONG_THREADS) {
      const float h = value(k);
      sum = fmaf(h, h, sum);
    }
    sum = across_row<LONG_THREADS>(sum, buffer[turn], Sum());
    const float inverse = inverse_root(sum, p.length, p.eps);
    if (p.rstd && threadIdx.x == 0) p.rstd[row] = inverse;
    if constexpr (!EIGHT) {
      for (int k = threadIdx.x; k < p.length; k += LONG_THREADS) {
        const float h = value(k);
        st(static_cast<T*>(p.y) + first + k, w ? h * inverse * weight(k) : h * inverse);
        if (res && p.total) st(static_cast<T*>(p.total) + first + k, h);
      }
    } else {
      const bool whole = p.group == p.length;
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
      float most = 0.f;
      double exact = 0.0;
      if (whole) {                                       // one group: by all threads
        for (int k = threadIdx.x; k < p.length; k += LONG_THREADS) most = Max()(most, fabsf(value(k) * weight(k)));
        most = across_row<LONG_THREADS>(most, most_of[turn], Max());
        for (int k = threadIdx.x; k < p.length; k += LONG_THREADS)
          if (fabsf(value(k) * weight(k)) >= most * (1.f - NEAR)) exact = Max()(exact, exact_at(k));
        exact = across_row<LONG_THREADS>(exact, exact_of[turn], Max());
      }
      for (int start = whole ? 0 : warp * p.group; start < p.length; start += whole ? p.length : LONG_THREADS / 32 * p.group) {
        const int from = whole ? (int)threadIdx.x : start + lane, step = whole ? LONG_THREADS : 32, end = start + p.group;
        if (!whole) {
          most = 0.f;
          exact = 0.0;
          for (int k = from; k < end; k += step) most = Max()(most, fabsf(value(k) * weight(k)));
          most = across_lanes(most, 32, Max());
          for (int k = from; k < end; k += step)
            if (fabsf(value(k) * weight(k)) >= most * (1.f - NEAR)) exact = Max()(exact, exact_at(k));
          exact = across_lanes(exact, 32, Max());
        }
        const float to = most > 0.f ? __fdiv_rn(E4M3_MAX, most) : 0.f;
        for (int k = from; k < end; k += step) {
          const float h = value(k), q = h * weight(k) * to;
          uint8_t held = to_e4m3(q * (1.f - NEAR));
          if (held != to_e4m3(q * (1.f + NEAR)) || (most < TINY && most > 0.f))
            held = to_e4m3_exact(exact_value(ld(x + first + k), res ? ld(res + first + k) : 0.f, weight(k)), exact);
          p.values[first + k] = held;
          if (res && p.total) st(static_cast<T*>(p.total) + first + k, h);
        }
        if (whole ? threadIdx.x == 0 : lane == 0) p.scales[row * (p.length / p.group) + start / p.group] = bad_weight || !(sum < INFINITY) ? NAN : scale_of(most, inverse);
      }
    }
  }
}

template <typename T> __global__ void __launch_bounds__(LONG_THREADS) backward_long_kernel(const NormArgs p) {
  __shared__ float buffer[2][LONG_THREADS / 32];
  const T *g = static_cast<const T*>(p.g), *gh = static_cast<const T*>(p.gh), *total = static_cast<const T*>(p.total), *res = static_cast<const T*>(p.res), *w = static_cast<const T*>(p.w);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x, turn ^= 1) {
    const int64_t first = row * p.length;
    const float inverse = p.rstd[row];
    auto weighted = [&](int k) { return w ? ld(g + first + k) * ld(w + k % p.channels) : ld(g + first + k); };
    auto unit = [&](int k) { return (ld(total + first + k) + (res ? ld(res + first + k) : 0.f)) * inverse; };
    float sum = 0.f;
    for (int k = threadIdx.x; k < p.length; k += LONG_THREADS) sum = fmaf(weighted(k), unit(k), sum);
    const float mean = across_row<LONG_THREADS>(sum, buffer[turn], Sum()) / (float)p.length;
    for (int k = threadIdx.x; k < p.length; k += LONG_THREADS)
      st(static_cast<T*>(p.dx) + first + k, fmaf(inverse, fmaf(-unit(k), mean, weighted(k)), gh ? ld(gh + first + k) : 0.f));
  }
}
// The weight's gradient of such rows: a thread has a place of the row, a CTA a part of the rows.
template <typename T> __global__ void __launch_bounds__(LONG_THREADS) weight_long_kernel(const NormArgs p, int64_t part_rows) {
  const T *g = static_cast<const T*>(p.g), *total = static_cast<const T*>(p.total), *res = static_cast<const T*>(p.res);
  const int k = blockIdx.x * LONG_THREADS + threadIdx.x;          // a row may have more pieces than a grid's y
  if (k >= p.length) return;
  const int64_t end = min(p.n, (int64_t)(blockIdx.y + 1) * part_rows);
  float sum = 0.f;
#pragma unroll 4
  for (int64_t row = blockIdx.y * part_rows; row < end; ++row) {
    const int64_t at = row * p.length + k;
    sum = fmaf(ld(g + at), (ld(total + at) + (res ? ld(res + at) : 0.f)) * __ldg(p.rstd + row), sum);
  }
  p.parts[(int64_t)blockIdx.y * p.length + k] = sum;
}

// dw[c] = the parts' sums over the components: a CTA has eight channels, 64 slices of the parts each
constexpr int SLICES = 64;
template <typename T> __global__ void __launch_bounds__(8 * SLICES) weight_sum_kernel(const NormArgs p, int parts) {
  __shared__ float sums[SLICES / 4][8];
  const int c = blockIdx.x * 8 + (threadIdx.x & 7), comps = p.length / p.channels;
  float sum = 0.f;
  if (c < p.channels)
    for (int m = 0; m < comps; ++m) {
      const float* from = p.parts + m * p.channels + c;
#pragma unroll 8
      for (int q = threadIdx.x >> 3; q < parts; q += SLICES) sum += from[(int64_t)q * p.length];
    }
  sum += __shfl_xor_sync(0xffffffffu, sum, 8);
  sum += __shfl_xor_sync(0xffffffffu, sum, 16);
  if ((threadIdx.x & 31) < 8) sums[threadIdx.x >> 5][threadIdx.x & 7] = sum;
  __syncthreads();
  if (threadIdx.x >= 8 || c >= p.channels) return;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < SLICES / 4; ++i) sum += sums[i][threadIdx.x];
  st(static_cast<T*>(p.dw) + c, sum);
}

// ---- host side ----------------------------------------------------------------------------------
int size_of(int dtype) { return dtype == EQT_F32 ? 4 : 2; }

// Threads of a row held in registers, and pieces of 16 bytes a thread; 0 threads where it is read by loops.
struct Rows { int threads, pieces; };
Rows rows_of(int dtype, int64_t length, int64_t channels, uintptr_t bits) {
  const int v = 16 / size_of(dtype);
  if (bits % 16 || length % v || channels % v) return {0, 0};
  const int64_t pieces = length / v;
  if (pieces <= 64) return {32, pieces <= 32 ? 1 : 2};
  if (pieces <= 512) return {128, pieces <= 128 ? 1 : pieces <= 256 ? 2 : 4};
  return pieces <= 2048 ? Rows{512, pieces <= 1024 ? 2 : 4} : Rows{0, 0};
}
// A call of `f` with the threads and pieces as constants.
template <int N> using Constant = std::integral_constant<int, N>;
template <typename F> void with_rows(Rows r, F f) {
  if (r.threads == 32 && r.pieces == 1) f(Constant<32>(), Constant<1>());
  else if (r.threads == 32) f(Constant<32>(), Constant<2>());
  else if (r.threads == 128 && r.pieces == 1) f(Constant<128>(), Constant<1>());
  else if (r.threads == 128 && r.pieces == 2) f(Constant<128>(), Constant<2>());
  else if (r.threads == 128) f(Constant<128>(), Constant<4>());
  else if (r.pieces == 2) f(Constant<512>(), Constant<2>());
  else f(Constant<512>(), Constant<4>());
}
// CTAs of the backward pass, whose sums of the weight's gradient are added afterwards: two waves of what fits an SM.
unsigned part_ctas(int threads, int64_t n) {
  const int64_t rows = threads == 32 ? 4 : 1;
  return (unsigned)std::min<int64_t>(ceil_div(n, rows), (int64_t)sm_count() * (threads == 512 ? 2 : 6));
}
// Parts of the rows where they are read by loops.
int64_t long_parts(int64_t n) { return std::min<int64_t>(ceil_div(n, 16), 128); }

int check_eps(double eps) {
  return (float)eps > 0.f && (float)eps < INFINITY ? EQT_OK : fail(EQT_ERR_BAD_ARGUMENT, "add_rms_norm: eps of %g is no positive float32", eps);
}
int check(int dtype, int64_t n, int64_t comps, int64_t channels) {
  if (dtype != EQT_F32 && dtype != EQT_BF16) return fail(EQT_ERR_BAD_ARGUMENT, "add_rms_norm: unknown dtype %d", dtype);
  if (n < 0 || comps < 0 || channels < 0) return fail(EQT_ERR_BAD_ARGUMENT, "add_rms_norm: negative size");
  if (n > INT32_MAX || comps > 1 << 24 || channels > 1 << 24 || comps * channels > 1 << 24)
    return fail(EQT_ERR_UNSUPPORTED, "add_rms_norm: at most 2^31 nodes of 2^24 values");
  return EQT_OK;
}

template <typename T, int OUT> int launch_forward(const NormArgs& p, Rows r, cudaStream_t s) {
  if (r.threads) {
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(p.n, r.threads == 32 ? 4 : 1), (int64_t)sm_count() * (r.threads == 512 ? 4 : 16));
    with_rows(r, [&](auto threads, auto pieces) {
      constexpr int N = decltype(threads)::value, K = decltype(pieces)::value;
      if (p.res) forward_kernel<T, N, K, OUT, true><<<grid, N < 128 ? 128 : N, 0, s>>>(p);
      else forward_kernel<T, N, K, OUT, false><<<grid, N < 128 ? 128 : N, 0, s>>>(p);
    });
  } else {
    forward_long_kernel<T, OUT != 0><<<(unsigned)std::min<int64_t>(p.n, (int64_t)sm_count() * 8), LONG_THREADS, 0, s>>>(p);
  }
  return check_launch("add_rms_norm");
}
template <typename T> int launch_backward(const NormArgs& p, Rows r, cudaStream_t s) {
  int parts;
  if (r.threads) {
    parts = (int)part_ctas(r.threads, p.n);
    with_rows(r, [&](auto threads, auto pieces) {
      constexpr int N = decltype(threads)::value, K = decltype(pieces)::value;
      if (p.res) backward_kernel<T, N, K, true><<<parts, N < 128 ? 128 : N, 0, s>>>(p);
      else backward_kernel<T, N, K, false><<<parts, N < 128 ? 128 : N, 0, s>>>(p);
    });
    if (int rc = check_launch("add_rms_norm_backward")) return rc;
  } else {
    backward_long_kernel<T><<<(unsigned)std::min<int64_t>(p.n, (int64_t)sm_count() * 8), LONG_THREADS, 0, s>>>(p);
    if (int rc = check_launch("add_rms_norm_backward")) return rc;
    if (!p.parts) return EQT_OK;
    parts = (int)long_parts(p.n);
    weight_long_kernel<T><<<dim3((unsigned)ceil_div(p.length, LONG_THREADS), (unsigned)parts), LONG_THREADS, 0, s>>>(p, ceil_div(p.n, parts));
    if (int rc = check_launch("add_rms_norm_weight")) return rc;
  }
  if (!p.parts) return EQT_OK;
  weight_sum_kernel<T><<<(unsigned)ceil_div(p.channels, 8), 8 * SLICES, 0, s>>>(p, parts);
  return check_launch("add_rms_norm_weight_sum");
}

uintptr_t bits_of(std::initializer_list<const void*> pointers) {
  uintptr_t bits = 0;
  for (const void* p : pointers) bits |= reinterpret_cast<uintptr_t>(p);
  return bits;
}

}  // namespace
}  // namespace residual_norm
}  // namespace eqt

using namespace eqt;
using namespace eqt::residual_norm;

extern "C" int eqt_add_rms_norm_forward(int32_t dtype, const void* x, const void* residual, const void* weight, void* out, void* total, float* rstd,
                                        int64_t n, int64_t comps, int64_t channels, double eps, void* stream) {
  if (int rc = check(dtype, n, comps, channels)) return rc;
  if (int rc = check_eps(eps)) return rc;
  if (n == 0 || comps * channels == 0) return EQT_OK;
  if (!x || !out) return fail(EQT_ERR_BAD_ARGUMENT, "add_rms_norm: NULL pointer");
  NormArgs p{};
  p.x = x, p.res = residual, p.w = weight, p.y = out, p.total = total, p.rstd = rstd, p.n = n, p.eps = (float)eps;
  p.length = (int)(comps * channels), p.channels = (int)channels;
  const Rows rows = rows_of(dtype, p.length, channels, bits_of({x, residual, weight, out, total}));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == EQT_F32 ? launch_forward<float, 0>(p, rows, s) : launch_forward<__nv_bfloat16, 0>(p, rows, s);
}

extern "C" int eqt_add_rms_norm_e4m3(int32_t dtype, const void* x, const void* residual, const void* weight, void* values, float* scales, void* total,
                                     int64_t n, int64_t comps, int64_t channels, int64_t group, double eps, void* stream) {
  if (int rc = check(dtype, n, comps, channels)) return rc;
  if (int rc = check_eps(eps)) return rc;
  if (n == 0 || comps * channels == 0) return EQT_OK;
  if (!x || !values || !scales) return fail(EQT_ERR_BAD_ARGUMENT, "add_rms_norm: NULL pointer");
  if (group < 1 || (comps * channels) % group) return fail(EQT_ERR_BAD_ARGUMENT, "add_rms_norm: rows of %lld values are no groups of %lld", (long long)(comps * channels), (long long)group);
  NormArgs p{};
  p.x = x, p.res = residual, p.w = weight, p.values = static_cast<uint8_t*>(values), p.scales = scales, p.total = total, p.n = n, p.eps = (float)eps;
  p.length = (int)(comps * channels), p.channels = (int)channels, p.group = (int)group;
  Rows rows = rows_of(dtype, p.length, channels, bits_of({x, residual, weight, values, total}));
  const int64_t lanes = group * size_of(dtype) / 16;
  const bool whole = group == p.length, pieces = group * size_of(dtype) % 16 == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0;
  if (!whole && !pieces) rows = {0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == EQT_F32) return whole ? launch_forward<float, 1>(p, rows, s) : launch_forward<float, 2>(p, rows, s);
  return whole ? launch_forward<__nv_bfloat16, 1>(p, rows, s) : launch_forward<__nv_bfloat16, 2>(p, rows, s);
}

extern "C" int64_t eqt_add_rms_norm_scratch(int32_t dtype, int64_t n, int64_t comps, int64_t channels) {
  if (check(dtype, n, comps, channels)) return 0;
  const Rows rows = rows_of(dtype, comps * channels, channels, 0);
  return std::max<int64_t>(rows.threads ? part_ctas(rows.threads, n) : 0, long_parts(n)) * comps * channels;
}

extern "C" int eqt_add_rms_norm_backward(int32_t dtype, const void* grad, const void* grad_total, const void* total, const void* residual, const void* weight,
                                         const float* rstd, void* dx, void* dweight, float* scratch, int64_t scratch_floats, int64_t n, int64_t comps, int64_t channels,
                                         void* stream) {
  if (int rc = check(dtype, n, comps, channels)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0 || comps * channels == 0) {
    if (dweight && channels && cudaMemsetAsync(dweight, 0, (size_t)channels * size_of(dtype), s) != cudaSuccess) return fail(EQT_ERR_CUDA, "cudaMemsetAsync failed");
    return EQT_OK;
  }
  if (!grad || !total || !rstd || !dx || (dweight && !scratch)) return fail(EQT_ERR_BAD_ARGUMENT, "add_rms_norm backward: NULL pointer");
  if (dweight && scratch_floats < eqt_add_rms_norm_scratch(dtype, n, comps, channels))
    return fail(EQT_ERR_BAD_ARGUMENT, "add_rms_norm backward: %lld values of scratch given, %lld needed", (long long)scratch_floats,
                (long long)eqt_add_rms_norm_scratch(dtype, n, comps, channels));
  NormArgs p{};
  p.g = grad, p.gh = grad_total, p.total = const_cast<void*>(total), p.res = residual, p.w = weight, p.rstd = const_cast<float*>(rstd), p.dx = dx, p.dw = dweight;
  p.parts = dweight ? scratch : nullptr, p.n = n, p.length = (int)(comps * channels), p.channels = (int)channels;
  const Rows rows = rows_of(dtype, p.length, channels, bits_of({grad, grad_total, total, residual, weight, dx}));
  return dtype == EQT_F32 ? launch_backward<float>(p, rows, s) : launch_backward<__nv_bfloat16>(p, rows, s);
}
