// Gated linear layer: the C entry points, and the kernels for float64, which have no tensor cores.
//
// The tensor memory accelerator copies tiles of operands whose rows start on 16-byte boundaries, so x and W of other widths are first
// copied to scratch with wider rows; da, du and the partial results have such rows anyway, and results are stored as they are to lie.
//
// The float64 kernel is a tiled product of strided operands, 64 x 64 results a CTA of 256 threads, 4 x 4 a thread, 16 terms at a time;
// it is bound by the multiply-adds.
#include <algorithm>

#include "gated.cuh"

namespace eqt {
namespace gated {
namespace {

enum Mode { FORWARD, PARTIALS, INPUT_GRAD, WEIGHT_GRAD };

constexpr int TILE = 64, TERMS = 16;

// Results [m][n] = sum_k A[m][k] B[k][n]; two products side by side (FORWARD, PARTIALS) or one.
template <int MODE>
__global__ void __launch_bounds__(256) double_kernel(const GatedArgs p, int64_t row_tiles) {
  using T = double;
  using A = double;
  constexpr bool DUAL = MODE == FORWARD || MODE == PARTIALS;
  __shared__ A sa[TERMS][TILE + 1], sb[DUAL ? 2 : 1][TERMS][TILE + 1];
  const int tid = threadIdx.x, tm = tid / 16, tn = tid % 16;
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *d = static_cast<const T*>(p.d);
  const int64_t nf = p.n * p.f, cf = (int64_t)p.c * p.f;
  int64_t m0, rows = MODE == WEIGHT_GRAD ? p.c : p.n, k0 = 0, k1;
  const int n0 = blockIdx.y * TILE, cols = MODE == INPUT_GRAD ? p.c : p.f;
  int j = 0, split = 0;
  if (MODE == WEIGHT_GRAD) {
    j = blockIdx.z & 1;
    split = blockIdx.z >> 1;
    m0 = (int64_t)blockIdx.x * TILE;
    k0 = split * p.split_rows;
    k1 = min(p.n, k0 + p.split_rows);
  } else {
    k1 = MODE == INPUT_GRAD ? 2 * (int64_t)p.f : p.c;
  }
  for (int64_t tile = MODE == WEIGHT_GRAD ? 0 : blockIdx.x; tile < row_tiles; tile += MODE == WEIGHT_GRAD ? row_tiles : gridDim.x) {
    if (MODE != WEIGHT_GRAD) m0 = tile * TILE;
    A acc[DUAL ? 2 : 1][4][4];
#pragma unroll
    for (int q = 0; q < (DUAL ? 2 : 1); ++q)
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[q][a][b] = A(0);
    for (int64_t kb = k0; kb < k1; kb += TERMS) {
      for (int i = tid; i < TILE * TERMS; i += 256) {
        // neighbouring threads read neighbouring values of each operand
        const int mk = MODE == WEIGHT_GRAD ? i / TILE : i % TERMS, mm = MODE == WEIGHT_GRAD ? i % TILE : i / TERMS;
        const int64_t k = kb + mk, m = m0 + mm;
        A v = A(0);
        if (k < k1 && m < rows) {
          if (DUAL) v = static_cast<A>(x[m * p.c + k]);
          if (MODE == INPUT_GRAD) v = static_cast<A>(k < p.f ? d[m * p.f + k] : d[nf + m * p.f + k - p.f]);
          if (MODE == WEIGHT_GRAD) v = static_cast<A>(x[k * p.c + m]);
        }
        sa[mk][mm] = v;
        const int nk = MODE == INPUT_GRAD ? i % TERMS : i / TILE, nn = MODE == INPUT_GRAD ? i / TERMS : i % TILE;
        const int64_t kn = kb + nk, n = n0 + nn;
        A b0 = A(0), b1 = A(0);
        if (kn < k1 && n < cols) {
          if (DUAL) {
            b0 = static_cast<A>(w[kn * p.f + n]);
            b1 = static_cast<A>(w[cf + kn * p.f + n]);
          }
          if (MODE == INPUT_GRAD) b0 = static_cast<A>(kn < p.f ? w[n * p.f + kn] : w[cf + n * p.f + kn - p.f]);
          if (MODE == WEIGHT_GRAD) b0 = static_cast<A>(d[j * nf + kn * p.f + n]);
        }
        sb[0][nk][nn] = b0;
        if (DUAL) sb[DUAL ? 1 : 0][nk][nn] = b1;
      }
      __syncthreads();
#pragma unroll 4
      for (int k = 0; k < TERMS; ++k) {
        A a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = sa[k][tm * 4 + i];
#pragma unroll
        for (int q = 0; q < (DUAL ? 2 : 1); ++q)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const A v = sb[q][k][tn + 16 * b];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[q][i][b] += a[i] * v;
          }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int64_t m = m0 + tm * 4 + i, n = n0 + tn + 16 * b;
        if (m >= rows || n >= cols) continue;
        if (MODE == FORWARD) {
          static_cast<T*>(p.h)[m * p.f + n] = static_cast<T>(activate(acc[0][i][b], p.act).y * acc[DUAL ? 1 : 0][i][b]);
        } else if (MODE == PARTIALS) {
          const Value<A> v = activate(acc[0][i][b], p.act);
          const A g = static_cast<A>(static_cast<const T*>(p.g)[m * p.f + n]);
          static_cast<T*>(p.d)[m * p.f + n] = static_cast<T>(g * acc[DUAL ? 1 : 0][i][b] * v.dy);
          static_cast<T*>(p.d)[nf + m * p.f + n] = static_cast<T>(g * v.y);
        } else if (MODE == INPUT_GRAD) {
          static_cast<T*>(p.dx)[m * p.c + n] = static_cast<T>(acc[0][i][b]);
        } else {
          static_cast<A*>(p.parts)[(split * 2 + j) * cf + m * p.f + n] = acc[0][i][b];
        }
      }
  }
}

// dW = the sum over the parts of the rows, in their order
template <typename T>
__global__ void __launch_bounds__(256) sum_parts_kernel(const typename Acc<T>::type* __restrict__ parts, T* __restrict__ dw, int rows, int f, int pitch,
                                                        int splits) {
  using A = typename Acc<T>::type;
  const int64_t size = (int64_t)rows * f, part = (int64_t)rows * pitch;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < size; i += (int64_t)gridDim.x * blockDim.x) {
    int64_t at = i;
    if (pitch != f) {
      const int64_t row = size <= UINT32_MAX ? (unsigned)i / (unsigned)f : i / f;
      at = row * pitch + (i - row * f);
    }
    const A* from = parts + at;
    A sum = A(0);
#pragma unroll 8
    for (int s = 0; s < splits; ++s) sum += from[s * part];
    dw[i] = static_cast<T>(sum);
  }
}
template <typename T> int sum_parts(const GatedArgs& p, cudaStream_t s) {
  sum_parts_kernel<T><<<flat_grid(2 * (int64_t)p.c * p.f, 256, 8), 256, 0, s>>>(static_cast<const typename Acc<T>::type*>(p.parts), static_cast<T*>(p.dw),
                                                                                 2 * p.c, p.f, p.d_pitch, p.splits);
  return check_launch("gated_sum_parts");
}

// rows of `cols` values to rows of `pitch`; what lies between is not read
template <typename T>
__global__ void __launch_bounds__(256) widen_kernel(const T* __restrict__ from, T* __restrict__ to, int64_t rows, int cols, int pitch) {
  const int64_t size = rows * cols;
#pragma unroll 4
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < size; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = size <= UINT32_MAX ? (unsigned)i / (unsigned)cols : i / cols;
    to[row * pitch + (i - row * cols)] = from[i];
  }
}
int widen(int dtype, const void* from, void* to, int64_t rows, int cols, int pitch, cudaStream_t s) {
  const unsigned grid = flat_grid(ceil_div(rows * cols, 4), 256);
  if (dtype == EQT_F32) widen_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(from), static_cast<float*>(to), rows, cols, pitch);
  else widen_kernel<<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(from), static_cast<uint16_t*>(to), rows, cols, pitch);
  return check_launch("gated_widen");
}

template <int MODE> int run_double(const GatedArgs& p, cudaStream_t s) {
  const int64_t tiles = ceil_div(p.n, TILE);
  dim3 grid((unsigned)std::min<int64_t>(tiles, 1 << 20), (unsigned)ceil_div(MODE == INPUT_GRAD ? p.c : p.f, TILE));
  if (MODE == WEIGHT_GRAD) grid = dim3((unsigned)ceil_div(p.c, TILE), grid.y, (unsigned)(2 * p.splits));
  double_kernel<MODE><<<grid, 256, 0, s>>>(p, MODE == WEIGHT_GRAD ? 1 : tiles);
  return check_launch("gated_double");
}
int backward_double(const GatedArgs& p, cudaStream_t s) {
  if (int rc = run_double<PARTIALS>(p, s)) return rc;
  if (p.dx)
    if (int rc = run_double<INPUT_GRAD>(p, s)) return rc;
  return p.dw ? run_double<WEIGHT_GRAD>(p, s) : EQT_OK;
}

int size_of(int dtype) { return dtype == EQT_F64 ? 8 : dtype == EQT_F32 ? 4 : 2; }

int check_sizes(int dtype, int64_t n, int64_t c, int64_t f, int act) {
  if (dtype != EQT_F32 && dtype != EQT_F64 && dtype != EQT_BF16) return fail(EQT_ERR_BAD_ARGUMENT, "gated: unknown dtype %d", dtype);
  if (act < EQT_ACT_SILU || act > EQT_ACT_SIGMOID) return fail(EQT_ERR_BAD_ARGUMENT, "gated: unknown activation %d", act);
  if (n < 0 || c < 0 || f < 0) return fail(EQT_ERR_BAD_ARGUMENT, "gated: negative size");
  if (n > INT32_MAX - 128 || c > 1 << 20 || f > 1 << 20) return fail(EQT_ERR_UNSUPPORTED, "gated: at most 2^31 rows and 2^20 channels");
  return EQT_OK;
}

// Rows are summed in parts so that the tiles of the weights' gradient fill the SMs evenly: as many parts as make the longest SM's work
// shortest, where an item costs its rows and about 256 rows' time for its start, its end and its partial results.  A part of bfloat16 is one
// sum of the tensor cores, whose adder truncates: up to 1.8e-7 of the sum are lost every 16 rows where the terms have one sign (100,000 rows:
// 1.1e-3 of the gradient, a third of its rounding).  16384 rows, which lose 1.8e-4, are the most; the parts are added with ordinary rounding.
constexpr int64_t MOST_ROWS = 16384;
void split_rows(GatedArgs& p, int dtype, int64_t n, int64_t c, int64_t f) {
  const int64_t tiles = 2 * ceil_div(c, 128) * ceil_div(f, dtype == EQT_BF16 ? 256 : 128), sms = sm_count();
  const int64_t least = dtype == EQT_BF16 ? ceil_div(n, MOST_ROWS) : 1;
  int64_t best = INT64_MAX;
  for (int64_t s = least; s <= std::max(least, std::min<int64_t>(sms, ceil_div(n, 128))); ++s) {
    const int64_t rows = ceil_div(ceil_div(n, s), 64) * 64, cost = ceil_div(tiles * s, sms) * (rows + 256);
    if (cost < best) best = cost, p.split_rows = rows;
  }
  p.splits = (int)ceil_div(n, p.split_rows);
}

size_t up(size_t b) { return (b + 1023) / 1024 * 1024; }

// Scratch: x and W with wider rows where theirs do not start on 16-byte boundaries, and for the backward pass da, du and the parts.
struct Scratch { size_t x, w, d, parts, bytes; };
Scratch lay_out(GatedArgs& p, int dtype, int64_t n, int64_t c, int64_t f, bool backward) {
  const size_t size = size_of(dtype);
  const int group = dtype == EQT_F64 ? 1 : (int)(16 / size);
  auto wide = [&](int64_t v) { return (int)(ceil_div(v, group) * group); };
  p.x_pitch = wide(c);
  p.w_pitch = p.d_pitch = wide(f);
  Scratch s{};
  s.w = p.x_pitch == c ? 0 : up((size_t)n * p.x_pitch * size);
  s.d = s.w + (p.w_pitch == f ? 0 : up((size_t)2 * c * p.w_pitch * size));
  s.parts = s.bytes = s.d;
  if (backward) {
    split_rows(p, dtype, n, c, f);
    s.parts = s.d + up((size_t)2 * n * p.d_pitch * size);
    s.bytes = s.parts + (size_t)p.splits * 2 * c * p.d_pitch * (dtype == EQT_F64 ? 8 : 4);
  }
  return s;
}

// Puts x and W of the right pitch into p.
int widen_operands(GatedArgs& p, int dtype, const Scratch& at, void* scratch, cudaStream_t s) {
  unsigned char* base = static_cast<unsigned char*>(scratch);
  if (p.x_pitch != p.c) {
    if (int rc = widen(dtype, p.x, base + at.x, p.n, p.c, p.x_pitch, s)) return rc;
    p.x = base + at.x;
  }
  if (p.w_pitch != p.f) {
    if (int rc = widen(dtype, p.w, base + at.w, 2 * (int64_t)p.c, p.f, p.w_pitch, s)) return rc;
    p.w = base + at.w;
  }
  return EQT_OK;
}

int check_pointers(int dtype, std::initializer_list<const void*> pointers) {
  uintptr_t bits = 0;
  for (const void* p : pointers) bits |= reinterpret_cast<uintptr_t>(p);
  return dtype == EQT_F64 || bits % 16 == 0 ? EQT_OK : fail(EQT_ERR_BAD_ARGUMENT, "gated: operands must start on 16-byte boundaries");
}

}  // namespace
}  // namespace gated
}  // namespace eqt

using namespace eqt;
using namespace eqt::gated;

extern "C" int64_t eqt_gated_scratch(int32_t dtype, int64_t n, int64_t c, int64_t f, int32_t backward) {
  if (check_sizes(dtype, n, c, f, 0) || n == 0 || f == 0 || c == 0) return 0;
  GatedArgs p{};
  return (int64_t)lay_out(p, dtype, n, c, f, backward != 0).bytes;
}

extern "C" int32_t eqt_gated_form(int32_t dtype, int64_t n, int64_t c, int64_t f, int32_t product) {
  if (check_sizes(dtype, n, c, f, 0) || dtype == EQT_F64 || n == 0 || f == 0 || c == 0 || product < FORWARD || product > WEIGHT_GRAD) return -1;
  GatedArgs p{};
  lay_out(p, dtype, n, c, f, true);
  p.n = n, p.c = (int)c, p.f = (int)f;
  return dtype == EQT_F32 ? tensor_form_f32(p, product) : tensor_form_bf16(p, product);
}

extern "C" int eqt_gated_forward(int32_t dtype, const void* x, const void* w, void* h, void* scratch, int64_t scratch_bytes, int64_t n, int64_t c,
                                 int64_t f, int32_t act, int32_t* status, void* stream) {
  if (int rc = check_sizes(dtype, n, c, f, act)) return rc;
  if (n == 0 || f == 0) return EQT_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!h) return fail(EQT_ERR_BAD_ARGUMENT, "gated: NULL pointer");
  if (c == 0) return cudaMemsetAsync(h, 0, (size_t)n * f * size_of(dtype), s) == cudaSuccess ? EQT_OK : fail(EQT_ERR_CUDA, "cudaMemsetAsync failed");
  GatedArgs p{};
  const Scratch at = lay_out(p, dtype, n, c, f, false);
  if (!x || !w || !status || (at.bytes && !scratch)) return fail(EQT_ERR_BAD_ARGUMENT, "gated: NULL pointer");
  if (scratch_bytes < (int64_t)at.bytes)
    return fail(EQT_ERR_BAD_ARGUMENT, "gated: %lld bytes of scratch given, %lld needed", (long long)scratch_bytes, (long long)at.bytes);
  if (int rc = check_pointers(dtype, {x, w, h, scratch})) return rc;
  p.x = x, p.w = w, p.h = h, p.n = n, p.c = (int)c, p.f = (int)f, p.act = act, p.status = status;
  if (dtype == EQT_F64) return run_double<FORWARD>(p, s);
  if (int rc = widen_operands(p, dtype, at, scratch, s)) return rc;
  return dtype == EQT_F32 ? tensor_forward_f32(p, s) : tensor_forward_bf16(p, s);
}

extern "C" int eqt_gated_backward(int32_t dtype, const void* x, const void* w, const void* g, void* dx, void* dw, void* scratch,
                                  int64_t scratch_bytes, int64_t n, int64_t c, int64_t f, int32_t act, int32_t* status, void* stream) {
  if (int rc = check_sizes(dtype, n, c, f, act)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0 || f == 0 || c == 0) {
    if (dx && n && c && cudaMemsetAsync(dx, 0, (size_t)n * c * size_of(dtype), s) != cudaSuccess) return fail(EQT_ERR_CUDA, "cudaMemsetAsync failed");
    if (dw && f && c && cudaMemsetAsync(dw, 0, (size_t)2 * c * f * size_of(dtype), s) != cudaSuccess) return fail(EQT_ERR_CUDA, "cudaMemsetAsync failed");
    return EQT_OK;
  }
  if (!x || !w || !g || !scratch || !status) return fail(EQT_ERR_BAD_ARGUMENT, "gated backward: NULL pointer");
  GatedArgs p{};
  const Scratch at = lay_out(p, dtype, n, c, f, true);
  if (scratch_bytes < (int64_t)at.bytes)
    return fail(EQT_ERR_BAD_ARGUMENT, "gated backward: %lld bytes of scratch given, %lld needed", (long long)scratch_bytes, (long long)at.bytes);
  if (int rc = check_pointers(dtype, {x, w, g, dx, dw, scratch})) return rc;
  p.x = x, p.w = w, p.g = g, p.dx = dx, p.dw = dw, p.n = n, p.c = (int)c, p.f = (int)f, p.act = act, p.status = status;
  p.d = static_cast<unsigned char*>(scratch) + at.d;
  p.parts = static_cast<unsigned char*>(scratch) + at.parts;
  if (dtype == EQT_F64) {
    if (int rc = backward_double(p, s)) return rc;
    return dw ? sum_parts<double>(p, s) : EQT_OK;
  }
  if (int rc = widen_operands(p, dtype, at, scratch, s)) return rc;
  if (int rc = dtype == EQT_F32 ? tensor_backward_f32(p, s) : tensor_backward_bf16(p, s)) return rc;
  if (!dw) return EQT_OK;
  return dtype == EQT_F32 ? sum_parts<float>(p, s) : sum_parts<__nv_bfloat16>(p, s);
}
