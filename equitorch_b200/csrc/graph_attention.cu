// Attention within packed graphs: checks of the arguments, order of the launches, sums over the heads.
#include "graph_attention.cuh"

namespace eqt {
namespace {
using namespace attention;

// Geometry over the heads: the first `heads` CTAs sum a head's slope gradient in a fixed order, the others the positions' gradients.
constexpr int GEO_THREADS = 1024;
__global__ void __launch_bounds__(GEO_THREADS) attention_geometry_kernel(const float4* __restrict__ row, const float4* __restrict__ col,
                                                                         const float* __restrict__ slope, float* __restrict__ dslope,
                                                                         float* __restrict__ dpos, int64_t n, int heads) {
  if (blockIdx.x < heads) {
    __shared__ double part[GEO_THREADS / 32];
    double sum = 0.0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < n; i += GEO_THREADS) sum += row[(int64_t)blockIdx.x * n + i].x;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < GEO_THREADS / 32; ++w) sum += part[w];
      dslope[blockIdx.x] = (float)-sum;
    }
    return;
  }
  const int64_t i = (int64_t)(blockIdx.x - heads) * GEO_THREADS + threadIdx.x;
  if (i >= n) return;
  float x = 0.f, y = 0.f, z = 0.f;
#pragma unroll 4
  for (int h = 0; h < heads; ++h) {
    const float4 a = row[(int64_t)h * n + i], b = col[(int64_t)h * n + i];
    const float f = -slope[h];
    x += f * (a.y - b.y);
    y += f * (a.z - b.z);
    z += f * (a.w - b.w);
  }
  dpos[3 * i] = x;
  dpos[3 * i + 1] = y;
  dpos[3 * i + 2] = z;
}

// ---- tiles of a packed batch --------------------------------------------------------------------
constexpr int PACK_THREADS = 1024, CLASSES = 64;
// Graphs of about one size: two classes an octave, the largest first.
__device__ __forceinline__ int size_class(int64_t size) {
  const int octave = 63 - __clzll(size);
  return CLASSES - 1 - min(CLASSES - 1, 2 * octave + (octave ? (int)(size >> (octave - 1)) & 1 : 0));
}

// stats: first boundary, last boundary, least and greatest size, and how many tiles of 16, 32 and 64 rows there are.
__global__ void __launch_bounds__(PACK_THREADS) pack_stats_kernel(const int64_t* __restrict__ ptr, int64_t graphs, int64_t* __restrict__ stats) {
  __shared__ long long least, greatest, tiles[3];
  if (threadIdx.x == 0) least = INT64_MAX, greatest = 0, tiles[0] = tiles[1] = tiles[2] = 0;
  __syncthreads();
  long long low = INT64_MAX, high = 0, sum[3] = {0, 0, 0};
  for (int64_t g = threadIdx.x; g < graphs; g += PACK_THREADS) {
    const int64_t size = ptr[g + 1] - ptr[g];
    low = min(low, (long long)size);
    high = max(high, (long long)size);
    for (int i = 0; i < 3; ++i) sum[i] += size > 0 ? (size + (16 << i) - 1) >> (4 + i) : 0;
  }
  atomicMin(&least, low);
  atomicMax(&greatest, high);
  for (int i = 0; i < 3; ++i) atomicAdd(reinterpret_cast<unsigned long long*>(&tiles[i]), (unsigned long long)sum[i]);
  __syncthreads();
  if (threadIdx.x == 0) {
    stats[0] = ptr[0];
    stats[1] = ptr[graphs];
    stats[2] = graphs ? least : 0;
    stats[3] = greatest;
    for (int i = 0; i < 3; ++i) stats[4 + i] = tiles[i];
  }
}

// The tiles, those of the larger classes first; within a class a graph's place is any, which changes no result.
__global__ void __launch_bounds__(PACK_THREADS) pack_tiles_kernel(const int64_t* __restrict__ ptr, int64_t graphs, int4* __restrict__ tiles,
                                                                  int64_t num_tiles, int rows) {
  __shared__ unsigned long long place[CLASSES];
  const int lane = threadIdx.x & 31;
  auto tiles_of = [&](int64_t size) { return size > 0 ? (size + rows - 1) / rows : 0; };
  if (threadIdx.x < CLASSES) place[threadIdx.x] = 0;
  __syncthreads();
  for (int64_t g = threadIdx.x; g < graphs; g += PACK_THREADS) {
    const int64_t size = ptr[g + 1] - ptr[g];
    if (size > 0) atomicAdd(&place[size_class(size)], (unsigned long long)tiles_of(size));
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned long long run = 0;
    for (int c = 0; c < CLASSES; ++c) {
      const unsigned long long here = place[c];
      place[c] = run;
      run += here;
    }
  }
  __syncthreads();
  for (int64_t g0 = threadIdx.x - lane; g0 < graphs; g0 += PACK_THREADS) {
    const int64_t g = g0 + lane;
    const int64_t lo = g < graphs ? ptr[g] : 0, hi = g < graphs ? ptr[g + 1] : 0, count = tiles_of(hi - lo);
    const int64_t at = count ? (int64_t)atomicAdd(&place[size_class(hi - lo)], (unsigned long long)count) : 0;
    constexpr int ALONE = 4;                             // tiles that a lane writes by itself; the warp writes those of larger graphs
    for (int64_t t = 0; t < count && count <= ALONE; ++t)
      if (at + t < num_tiles) tiles[at + t] = make_int4((int)(lo + t * rows), (int)lo, (int)hi, 0);
    unsigned many = __ballot_sync(0xffffffffu, count > ALONE);
    while (many) {
      const int who = __ffs(many) - 1;
      many &= many - 1;
      const int64_t l = __shfl_sync(0xffffffffu, lo, who), h = __shfl_sync(0xffffffffu, hi, who), a = __shfl_sync(0xffffffffu, at, who);
      for (int64_t t = lane; l + t * rows < h; t += 32)
        if (a + t < num_tiles) tiles[a + t] = make_int4((int)(l + t * rows), (int)l, (int)h, 0);
    }
  }
}

int launch_all(Pass pass, const eqt_attention_args* a, const AttentionParams& p, bool geo, cudaStream_t s) {
  return a->dtype == EQT_F32 ? launch_f32(pass, p, a->num_tiles, a->tile_rows, geo, s)
                             : launch_bf16(pass, p, a->num_tiles, a->tile_rows, geo, s);
}

int fill(const eqt_attention_args* a, AttentionParams& p, bool backward) {
  if (!a) return fail(EQT_ERR_BAD_ARGUMENT, "attention: NULL arguments");
  if (a->dtype != EQT_F32 && a->dtype != EQT_BF16) return fail(EQT_ERR_UNSUPPORTED, "attention: float32 or bfloat16 features expected");
  if (a->n < 0 || a->longest < 0 || a->num_tiles < 0 || a->heads < 1 || a->comps < 1 || a->head_channels < 1)
    return fail(EQT_ERR_BAD_ARGUMENT, "attention: sizes must be positive");
  if (a->tile_rows != 16 && a->tile_rows != 32 && a->tile_rows != 64) return fail(EQT_ERR_BAD_ARGUMENT, "attention: tiles have 16, 32 or 64 rows");
  if (a->n > INT32_MAX - 64 || a->num_tiles > INT32_MAX || a->heads > 65535)
    return fail(EQT_ERR_UNSUPPORTED, "attention: nodes and tiles are numbered in 32 bits, heads in 16");
  if ((int64_t)a->comps * a->head_channels > 128)
    return fail(EQT_ERR_UNSUPPORTED, "attention: a head has at most 128 values a node, got %lld", (long long)a->comps * a->head_channels);
  if (a->cap != 0.f && !(a->cap >= 1e-12f && a->cap <= 1e12f)) return fail(EQT_ERR_BAD_ARGUMENT, "attention: the cap must be 0 or from 1e-12 to 1e12");
  if (!(fabsf(a->scale) <= 1e12f)) return fail(EQT_ERR_BAD_ARGUMENT, "attention: the scale must be at most 1e12");
  if (a->n && (a->pos != nullptr) != (a->slope != nullptr)) return fail(EQT_ERR_BAD_ARGUMENT, "attention: positions and slopes come together");
  if (a->num_tiles && (!a->q || !a->k || !a->v || !a->out || !a->tiles || (backward && (!a->grad_out || !a->stats || !a->dq || !a->dk || !a->dv || !a->delta))))
    return fail(EQT_ERR_BAD_ARGUMENT, "attention: NULL pointer");
  const bool geo = a->dpos || a->dslope;
  if (backward && geo && a->n && (!a->pos || !a->dpos || !a->dslope || !a->geo))
    return fail(EQT_ERR_BAD_ARGUMENT, "attention: the gradients of positions and slopes come together, with positions and scratch");
  const int64_t channels = (int64_t)a->heads * a->head_channels;
  const int size = a->dtype == EQT_F32 ? 4 : 2;
  p = AttentionParams{};
  p.q = {a->q, a->q_node, a->q_comp};
  p.k = {a->k, a->k_node, a->k_comp};
  p.v = {a->v, a->v_node, a->v_comp};
  p.g = {a->grad_out, a->comps * channels, channels};
  p.out = a->out;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  p.top = a->stats;
  p.inverse = a->stats ? a->stats + a->heads * a->n : nullptr;
  p.delta = a->delta;
  p.geo_row = static_cast<float4*>(a->geo);
  p.geo_col = p.geo_row ? p.geo_row + a->heads * a->n : nullptr;
  p.tiles = static_cast<const int4*>(static_cast<const void*>(a->tiles));
  p.pos = a->pos;
  p.slope = a->slope;
  p.n = a->n;
  p.heads = a->heads;
  p.comps = a->comps;
  p.size = a->head_channels;
  const int64_t longest = a->longest ? a->longest : a->n;
  p.folds = a->dtype == EQT_BF16 && longest > FOLD;
  if (p.folds && a->num_tiles && a->tile_rows != 64)
    return fail(EQT_ERR_UNSUPPORTED, "attention: bfloat16 with graphs of more than %d nodes needs tiles of 64 rows, got %d", FOLD, a->tile_rows);
  p.scale = a->scale;
  p.cap = a->cap;
  uintptr_t bits = (uintptr_t)a->head_channels * size;
  for (const void* q : {a->q, a->k, a->v, (const void*)a->out, a->grad_out, (const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
    bits |= reinterpret_cast<uintptr_t>(q);
  for (int64_t st : {a->q_node, a->q_comp, a->k_node, a->k_comp, a->v_node, a->v_comp}) bits |= (uintptr_t)st * size;
  p.vec = bits % 16 == 0;
  return EQT_OK;
}

}  // namespace
}  // namespace eqt

using namespace eqt;

extern "C" int eqt_attention_forward(const eqt_attention_args* a, void* stream) {
  AttentionParams p;
  if (int rc = fill(a, p, false)) return rc;
  if (a->num_tiles == 0) return EQT_OK;
  return launch_all(FORWARD, a, p, false, static_cast<cudaStream_t>(stream));
}

extern "C" int eqt_attention_backward(const eqt_attention_args* a, void* stream) {
  AttentionParams p;
  if (int rc = fill(a, p, true)) return rc;
  const bool geo = a->dslope != nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->num_tiles) {
    if (int rc = launch_all(ROWS, a, p, geo, s)) return rc;
    if (int rc = launch_all(COLUMNS, a, p, geo, s)) return rc;
  }
  if (!geo) return EQT_OK;
  attention_geometry_kernel<<<(unsigned)(a->heads + ceil_div(a->n, GEO_THREADS)), GEO_THREADS, 0, s>>>(
      p.geo_row, p.geo_col, a->slope, a->dslope, a->dpos, a->n, a->heads);
  return check_launch("attention_geometry");
}

extern "C" int eqt_pack_graphs_stats(const int64_t* ptr, int64_t graphs, int64_t* stats, void* stream) {
  if (!ptr || !stats || graphs < 0) return fail(EQT_ERR_BAD_ARGUMENT, "pack_graphs: NULL pointer or negative size");
  pack_stats_kernel<<<1, PACK_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(ptr, graphs, stats);
  return check_launch("pack_stats");
}

extern "C" int eqt_pack_graphs_tiles(const int64_t* ptr, int64_t graphs, int32_t* tiles, int64_t num_tiles, int32_t rows, void* stream) {
  if (num_tiles == 0 || graphs == 0) return EQT_OK;
  if (!ptr || !tiles || graphs < 0 || num_tiles < 0) return fail(EQT_ERR_BAD_ARGUMENT, "pack_graphs: NULL pointer or negative size");
  if (rows != 16 && rows != 32 && rows != 64) return fail(EQT_ERR_BAD_ARGUMENT, "pack_graphs: tiles have 16, 32 or 64 rows");
  pack_tiles_kernel<<<1, PACK_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(ptr, graphs, reinterpret_cast<int4*>(tiles), num_tiles, rows);
  return check_launch("pack_tiles");
}
