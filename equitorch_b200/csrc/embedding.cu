// Rows of a table by type, scaled, and the gradient of the table.
//
//   forward:   out[n, :] = scale * weight[index[n], :]              (a row of zeros where index[n] is no type)
//   gradient:  gw[t, :]  = scale * sum over n with index[n] = t of g[n, :]
//
// Both are bound by memory: one read of g (or one write of out) and of the indices.  The gradient uses no atomics on values, so two
// calls give the same bits.  Rows of whole 16 bytes on 16-byte boundaries go by pieces of 16 bytes, others by single values (2.0M bfloat16 rows,
// 14161 types, both directions: 32 values 240 us, 31 values 386, 33 values 507).  Few rows: a CTA per type looks through all indices.  Otherwise the rows are sorted by type (a counting
// sort of one digit of up to eight bits a pass, least digit first, in the order of the rows within a type), teams of lanes add up
// equal pieces of the sorted rows whatever types they hold, and sums that cross the border of a piece are joined afterwards in the
// order of the pieces.
#include <algorithm>

#include "common.cuh"

namespace eqt {
namespace {

constexpr int SORT_THREADS = 256, SORT_WARPS = SORT_THREADS / 32;
constexpr int MAX_BINS = 256;
constexpr int TEAM_THREADS = 128;
constexpr int UNROLL = 8;
constexpr unsigned FULL = 0xffffffffu;

template <typename T, int V> struct Pack { T v[V]; };
template <typename T, int V> struct alignas(sizeof(T) * V) Packed : Pack<T, V> {};

// ---- forward ------------------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(256) embedding_kernel(const T* __restrict__ weight, const int64_t* __restrict__ index,
                                                        T* __restrict__ out, int64_t n, int64_t types, int64_t pitch, unsigned cols,
                                                        typename Acc<T>::type scale) {
  using A = typename Acc<T>::type;
  // neighbouring threads hold neighbouring pieces of a row; four pieces a thread are on their way at a time
  const int64_t total = n * cols, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t at = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; at < total; at += 4 * step) {
    int64_t row[4], type[4];
    unsigned col[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = at + u * step;
      row[u] = total <= UINT32_MAX ? (unsigned)i / cols : i / cols;
      col[u] = (unsigned)(i - row[u] * cols);
      type[u] = i < total ? __ldg(index + row[u]) : -1;
    }
    Packed<T, V> v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if ((uint64_t)type[u] < (uint64_t)types) {
        v[u] = *reinterpret_cast<const Packed<T, V>*>(weight + type[u] * pitch + (int64_t)col[u] * V);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[u].v[i] = static_cast<T>(A(0));
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (at + u * step >= total) break;
#pragma unroll
      for (int i = 0; i < V; ++i) v[u].v[i] = static_cast<T>(static_cast<A>(v[u].v[i]) * scale);
      *reinterpret_cast<Packed<T, V>*>(out + row[u] * pitch + (int64_t)col[u] * V) = v[u];
    }
  }
}

// ---- sort by type -------------------------------------------------------------------------------
// A row that names no type gets the key `types`, which sorts behind all others.
// Key and row travel as one value of eight bytes: places are scattered, so a store costs a sector whatever its size.
__device__ __forceinline__ int2 entry_of(const int64_t* index, const int2* sorted, int64_t i, int64_t types) {
  if (sorted) return __ldg(sorted + i);
  const int64_t t = __ldg(index + i);
  return make_int2((int)((uint64_t)t < (uint64_t)types ? t : types), (int)i);
}

// Each warp owns `rows` rows in a row; within[warp][bin] is how many rows of the digit the warps of its CTA before it own,
// counts[CTA][bin] how many the CTA does.
__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const int64_t* __restrict__ index, const int2* __restrict__ sorted,
                                                                  int* __restrict__ within, int* __restrict__ counts, int64_t n,
                                                                  int64_t types, int64_t rows, int shift, int bins) {
  extern __shared__ int tally[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* mine = tally + warp * bins;
  for (int b = lane; b < bins; b += 32) mine[b] = 0;
  __syncwarp();
  const int64_t w = (int64_t)blockIdx.x * SORT_WARPS + warp, lo = w * rows, hi = min(n, lo + rows);
#pragma unroll 4
  for (int64_t i = lo + lane; i < hi; i += 32) atomicAdd(&mine[(entry_of(index, sorted, i, types).x >> shift) & (bins - 1)], 1);   // counts: order is free
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += SORT_THREADS) {
    int run = 0;
#pragma unroll
    for (int v = 0; v < SORT_WARPS; ++v) {
      within[((int64_t)blockIdx.x * SORT_WARPS + v) * bins + b] = run;
      run += tally[v * bins + b];
    }
    counts[(int64_t)blockIdx.x * bins + b] = run;
  }
}

// before[CTA][bin] is the number of rows of the digit that the CTAs before own, totals[bin] their number over all CTAs.
// A lane is a digit, the 32 warps of the CTA share the rows of `counts`.
__global__ void __launch_bounds__(1024) sort_scan_kernel(const int* __restrict__ counts, int* __restrict__ before, int* __restrict__ totals, int ctas,
                                                         int bins) {
  __shared__ int part[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bin = blockIdx.x * 32 + lane;
  const int each = (ctas + 31) / 32, lo = min(ctas, warp * each), hi = min(ctas, lo + each);
  const bool there = bin < bins;
  int sum = 0;
#pragma unroll 8
  for (int w = lo; w < hi; ++w) sum += there ? __ldg(counts + (int64_t)w * bins + bin) : 0;
  part[warp][lane] = sum;
  __syncthreads();
  int run = 0, all = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) run += part[w][lane];
    all += part[w][lane];
  }
  if (warp == 0 && there) totals[bin] = all;
#pragma unroll 8
  for (int w = lo; w < hi; ++w) {
    const int v = there ? __ldg(counts + (int64_t)w * bins + bin) : 0;
    if (there) before[(int64_t)w * bins + bin] = run;
    run += v;
  }
}

// Rows to their places, in their order within a digit: a warp takes 32 rows at a time, lanes of the same digit rank by lane.
__global__ void __launch_bounds__(SORT_THREADS) sort_place_kernel(const int64_t* __restrict__ index, const int2* __restrict__ sorted,
                                                                  const int* __restrict__ within, const int* __restrict__ before,
                                                                  const int* __restrict__ totals, int2* __restrict__ out, int64_t n,
                                                                  int64_t types, int64_t rows, int shift, int bins) {
  extern __shared__ int place[];                // [warp][bin]
  __shared__ int first[MAX_BINS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {                              // exclusive sums of the digits' totals
    int run = 0;
    for (int b0 = 0; b0 < bins; b0 += 32) {
      const int v = b0 + lane < bins ? totals[b0 + lane] : 0;
      int s = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(FULL, s, o);
        if (lane >= o) s += t;
      }
      if (b0 + lane < bins) first[b0 + lane] = run + s - v;
      run += __shfl_sync(FULL, s, 31);
    }
  }
  __syncthreads();
  int* mine = place + warp * bins;
  const int64_t w = (int64_t)blockIdx.x * SORT_WARPS + warp, lo = w * rows, hi = min(n, lo + rows);
  for (int b = lane; b < bins; b += 32) mine[b] = first[b] + before[(int64_t)blockIdx.x * bins + b] + within[w * bins + b];
  __syncwarp();
  for (int64_t i0 = lo; i0 < hi; i0 += 128) {
    int2 entry[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {               // the loads of four steps together
      const int64_t i = i0 + u * 32 + lane;
      entry[u] = i < hi ? entry_of(index, sorted, i, types) : make_int2(0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool there = i0 + u * 32 + lane < hi;
      const int digit = there ? (entry[u].x >> shift) & (bins - 1) : bins;     // lanes past the end are a digit of their own
      const unsigned same = __match_any_sync(FULL, digit);
      const int rank = __popc(same & ((1u << lane) - 1));
      const int to = there ? mine[digit] + rank : 0;
      __syncwarp();
      if (there && rank == 0) mine[digit] += __popc(same);
      __syncwarp();
      if (there) out[to] = entry[u];
    }
  }
}

// ---- sums over the sorted rows ------------------------------------------------------------------
template <typename T, int V>
__device__ __forceinline__ void put(T* p, const typename Acc<T>::type (&sum)[V], typename Acc<T>::type scale) {
  Packed<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.v[i] = static_cast<T>(sum[i] * scale);
  *reinterpret_cast<Packed<T, V>*>(p) = v;
}
template <typename A, int V>
__device__ __forceinline__ void put_part(A* p, const A (&sum)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] = sum[i];
}

// A team of `team` lanes (a power of two) adds up the sorted rows [c * piece, (c + 1) * piece), V columns a lane.  A type whose rows
// all lie in the piece is written at once; what began in a piece before goes to head[c], what goes on in the next to tail[c].
template <typename T, int V>
__global__ void __launch_bounds__(TEAM_THREADS) piece_sum_kernel(const T* __restrict__ g, const int2* __restrict__ sorted, T* __restrict__ gw,
                                                                 typename Acc<T>::type* __restrict__ head,
                                                                 typename Acc<T>::type* __restrict__ tail, int64_t n, int types,
                                                                 int64_t pitch, int cols, int team, int piece, int64_t pieces,
                                                                 typename Acc<T>::type scale) {
  using A = typename Acc<T>::type;
  const int64_t c = ((int64_t)blockIdx.x * TEAM_THREADS + threadIdx.x) / team;
  const int col = (blockIdx.y * team + threadIdx.x % team);
  if (c >= pieces || col >= cols) return;
  const int64_t lo = c * piece, hi = min(n, lo + piece);
  const T* gc = g + (int64_t)col * V;
  A sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = A(0);
  int now = sorted[lo].x;
  bool open = lo > 0 && sorted[lo - 1].x == now;                                   // the run began in a piece before
  auto close = [&](int key, bool goes_on) {
    if (key < types) {
      if (open) put_part(head + c * pitch + (int64_t)col * V, sum);
      else if (goes_on) put_part(tail + c * pitch + (int64_t)col * V, sum);
      else put(gw + key * pitch + (int64_t)col * V, sum, scale);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = A(0);
    open = false;
  };
  for (int64_t i = lo; i < hi; i += UNROLL) {
    int2 entry[UNROLL];
    Packed<T, V> row[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) entry[u] = i + u < hi ? __ldg(sorted + i + u) : make_int2(types, 0);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (entry[u].x < types) row[u] = *reinterpret_cast<const Packed<T, V>*>(gc + (int64_t)entry[u].y * pitch);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (i + u >= hi) break;
      if (entry[u].x != now) {
        close(now, false);
        now = entry[u].x;
      }
      if (now < types) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += static_cast<A>(row[u].v[j]);
      }
    }
  }
  close(now, hi < n && sorted[hi].x == now);
}

// Adds up parts tail[c], head[c + 1 .. last] of a run, V columns a lane: team `mine` of `teams` takes every teams-th part in order.
template <typename A, int V>
__device__ __forceinline__ void add_parts(const A* __restrict__ head, const A* __restrict__ tail, int64_t c, int64_t last, int64_t pitch,
                                          int64_t at, int mine, int teams, A (&sum)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = mine == 0 ? tail[c * pitch + at + i] : A(0);
#pragma unroll 8
  for (int64_t p = c + 1 + mine; p <= last; p += teams) {
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] += head[p * pitch + at + i];
  }
}

// A warp looks at a piece: where a run begins in it that goes on behind it, the warp adds up the run's parts, or the whole CTA does
// where they are many.  Teams of lanes take the parts in turn and are added up in a fixed order.
constexpr int JOIN_WARPS = 8, JOIN_ALONE = 64;
template <typename T, int V>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const int2* __restrict__ sorted, T* __restrict__ gw,
                                                               const typename Acc<T>::type* __restrict__ head,
                                                               const typename Acc<T>::type* __restrict__ tail, int64_t n, int types,
                                                               int64_t pitch, int cols, int team, int piece, int64_t pieces,
                                                               typename Acc<T>::type scale) {
  using A = typename Acc<T>::type;
  __shared__ A part[JOIN_WARPS][32 * V];
  __shared__ int64_t long_last[JOIN_WARPS];     // of the runs left to the whole CTA, else -1
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int teams = 32 / team, mine = lane / team, tl = lane % team;
  const int64_t c = (int64_t)blockIdx.x * JOIN_WARPS + warp, lo = c * piece, hi = min(n, lo + piece);
  auto fold = [&](A(&sum)[V]) {                 // sums of the teams of a warp to team 0
    for (int o = 16; o >= team; o >>= 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += __shfl_down_sync(FULL, sum[i], o);
    }
  };
  int64_t last = -1;
  int key = types;
  if (c < pieces) {
    key = sorted[hi - 1].x;
    if (key < types && hi < n && sorted[hi].x == key && !(lo > 0 && sorted[lo - 1].x == key)) {
      // The run reaches into the pieces whose first row has its type: 32 of them are looked at a step, first the next ones, then by
      // 32nds of what is left.
      last = c + 1;                             // reaches in
      int64_t past = pieces;                    // does not
      for (int64_t step = 1; past - last > 1; step = (past - last + 31) / 32) {
        const int64_t at = last + (lane + 1) * step;
        const unsigned in = __ballot_sync(FULL, at < past && __ldg(&sorted[at * piece].x) == key);     // a run of ones from lane 0 on
        const int reach = __popc(in);
        if (reach < 32) past = min(past, last + (reach + 1) * step);
        last += reach * step;
      }
    }
  }
  const bool all = last - c >= JOIN_ALONE;
  if (lane == 0) long_last[warp] = all ? last : -1;
  if (last >= 0 && !all) {
    for (int col0 = 0; col0 < cols; col0 += team) {
      const int col = col0 + tl;
      A sum[V];
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = A(0);
      if (col < cols) add_parts(head, tail, c, last, pitch, (int64_t)col * V, mine, teams, sum);
      fold(sum);
      if (mine == 0 && col < cols) put(gw + key * pitch + (int64_t)col * V, sum, scale);
    }
  }
  __syncthreads();
  for (int w = 0; w < JOIN_WARPS; ++w) {
    const int64_t end = long_last[w];
    if (end < 0) continue;
    const int64_t first = (int64_t)blockIdx.x * JOIN_WARPS + w;
    const int64_t type = sorted[min(n, (first + 1) * piece) - 1].x;
    for (int col0 = 0; col0 < cols; col0 += team) {
      const int col = col0 + tl;
      A sum[V];
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = A(0);
      if (col < cols) add_parts(head, tail, first, end, pitch, (int64_t)col * V, warp * teams + mine, JOIN_WARPS * teams, sum);
      fold(sum);
      __syncthreads();
      if (mine == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) part[warp][tl * V + i] = sum[i];
      }
      __syncthreads();
      if (warp == 0 && mine == 0 && col < cols) {
        for (int v = 1; v < JOIN_WARPS; ++v) {
#pragma unroll
          for (int i = 0; i < V; ++i) sum[i] += part[v][tl * V + i];
        }
        put(gw + type * pitch + (int64_t)col * V, sum, scale);
      }
    }
  }
}

// ---- few rows: a CTA per type and slab of columns looks through all indices ----------------------
template <typename T, int V>
__global__ void __launch_bounds__(256) type_sum_kernel(const T* __restrict__ g, const int64_t* __restrict__ index, T* __restrict__ gw,
                                                       int n, int64_t pitch, int cols, typename Acc<T>::type scale) {
  using A = typename Acc<T>::type;
  __shared__ A part[8][32 * V];
  const int64_t type = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y * 32 + lane;
  const int each = ((n + 7) / 8 + 31) & ~31, lo = warp * each, hi = min(n, lo + each);
  A sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = A(0);
  for (int i0 = lo; i0 < hi; i0 += 32) {
    unsigned hits = __ballot_sync(FULL, i0 + lane < hi && __ldg(index + i0 + lane) == type);
    while (hits) {                                                             // rows in order, up to four on their way
      Packed<T, V> row[4];
      int m = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (!hits) break;
        const int at = i0 + __ffs(hits) - 1;
        hits &= hits - 1;
        if (col < cols) row[u] = *reinterpret_cast<const Packed<T, V>*>(g + at * pitch + (int64_t)col * V);
        m = u + 1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (u >= m || col >= cols) break;
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += static_cast<A>(row[u].v[j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) part[warp][lane * V + i] = sum[i];
  __syncthreads();
  if (warp == 0 && col < cols) {
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = A(0);
    for (int w = 0; w < 8; ++w) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += part[w][lane * V + i];
    }
    put(gw + type * pitch + (int64_t)col * V, sum, scale);
  }
}

// ---- host side ----------------------------------------------------------------------------------
struct GradPlan {
  bool small;               // one launch of type_sum_kernel
  int passes, digit_bits;
  int64_t warps, rows;      // of the sort
  int piece;
  int64_t pieces;
  size_t sorted, within, counts, before, totals, parts, bytes;       // scratch: two buffers of sorted rows
};

int size_of(int dtype) { return dtype == EQT_F64 ? 8 : dtype == EQT_F32 ? 4 : 2; }

GradPlan grad_plan(int dtype, int64_t n, int64_t types, int64_t width) {
  GradPlan p{};
  // Every type's CTA reads all n indices: few rows, and a bounded number of reads altogether.
  p.small = n <= 4096 && types <= 65535 && n * types <= (int64_t)1 << 22;
  if (p.small) return p;
  int bits = 1;
  while (((int64_t)1 << bits) <= types) ++bits;           // keys 0 .. types
  p.passes = (bits + 7) / 8;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  const int64_t most = (int64_t)sm_count() * 16;
  p.rows = std::max<int64_t>(128, ceil_div(ceil_div(n, most), 32) * 32);
  p.warps = ceil_div(ceil_div(n, p.rows), SORT_WARPS) * SORT_WARPS;
  int team = 1;                                           // lanes that have a row: one 16 bytes, at most 32
  while (team < 32 && team * 16 < width * size_of(dtype)) team *= 2;
  // Pieces so short that 256 threads an SM have one, but not so short that their borders cost more than their rows (2.0M rows of 64
  // bytes, 14161 types, sums and joins: 100 us with 256 threads, 107 with 512, 104 with 1024, 121 with 2048).
  p.piece = (int)std::max<int64_t>(32, ceil_div(ceil_div(n, (int64_t)sm_count() * 256 / team), UNROLL) * UNROLL);
  p.pieces = ceil_div(n, p.piece);
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  p.sorted = 0;
  p.within = up((size_t)n * 8) * 2;
  const size_t bins = (size_t)4 << p.digit_bits, ctas = (size_t)p.warps / SORT_WARPS;
  p.counts = p.within + up(p.warps * bins);
  p.before = p.counts + up(ctas * bins);
  p.totals = p.before + up(ctas * bins);
  p.parts = p.totals + up((size_t)MAX_BINS * 4);
  p.bytes = p.parts + 2 * up((size_t)p.pieces * width * (dtype == EQT_F64 ? 8 : 4));
  return p;
}

template <typename T, int V>
int run_forward(const void* weight, const int64_t* index, void* out, int64_t n, int64_t types, int64_t width, double scale, cudaStream_t s) {
  const int64_t cols = width / V;
  embedding_kernel<T, V><<<flat_grid(ceil_div(n * cols, 4), 256), 256, 0, s>>>(
      static_cast<const T*>(weight), index, static_cast<T*>(out), n, types, width, (unsigned)cols, static_cast<typename Acc<T>::type>(scale));
  return check_launch("embedding");
}

template <typename T, int V>
int run_grad(int dtype, const void* g, const int64_t* index, void* gw, int64_t n, int64_t types, int64_t width, double scale_,
             unsigned char* scratch, cudaStream_t s) {
  using A = typename Acc<T>::type;
  const A scale = static_cast<A>(scale_);
  const int cols = (int)(width / V);
  const GradPlan p = grad_plan(dtype, n, types, width);
  if (p.small) {
    type_sum_kernel<T, V><<<dim3((unsigned)types, (unsigned)ceil_div(cols, 32)), 256, 0, s>>>(
        static_cast<const T*>(g), index, static_cast<T*>(gw), (int)n, width, cols, scale);
    return check_launch("type_sum");
  }
  if (cudaMemsetAsync(gw, 0, (size_t)types * width * sizeof(T), s) != cudaSuccess) return fail(EQT_ERR_CUDA, "cudaMemsetAsync failed");
  int2* sorted[2] = {reinterpret_cast<int2*>(scratch + p.sorted), reinterpret_cast<int2*>(scratch + p.sorted + ((size_t)n * 8 + 255) / 256 * 256)};
  int* within = reinterpret_cast<int*>(scratch + p.within);
  int* counts = reinterpret_cast<int*>(scratch + p.counts);
  int* before = reinterpret_cast<int*>(scratch + p.before);
  int* totals = reinterpret_cast<int*>(scratch + p.totals);
  const int bins = 1 << p.digit_bits;
  const unsigned grid = (unsigned)(p.warps / SORT_WARPS);
  const size_t shared = (size_t)SORT_WARPS * bins * 4;     // at most 8 KB
  int at = 0;
  for (int pass = 0; pass < p.passes; ++pass, at ^= 1) {
    const int2* from = pass ? sorted[at ^ 1] : nullptr;
    const int shift = pass * p.digit_bits;
    sort_count_kernel<<<grid, SORT_THREADS, shared, s>>>(index, from, within, counts, n, types, p.rows, shift, bins);
    if (int rc = check_launch("sort_count")) return rc;
    sort_scan_kernel<<<(unsigned)ceil_div(bins, 32), 1024, 0, s>>>(counts, before, totals, (int)grid, bins);
    if (int rc = check_launch("sort_scan")) return rc;
    sort_place_kernel<<<grid, SORT_THREADS, shared, s>>>(index, from, within, before, totals, sorted[at], n, types, p.rows, shift, bins);
    if (int rc = check_launch("sort_place")) return rc;
  }
  at ^= 1;
  int team = 1;
  while (team < cols && team < 32) team *= 2;
  A* head = reinterpret_cast<A*>(scratch + p.parts);
  A* tail = reinterpret_cast<A*>(scratch + p.parts + ((size_t)p.pieces * width * sizeof(A) + 255) / 256 * 256);
  const dim3 sums((unsigned)ceil_div(p.pieces * team, TEAM_THREADS), (unsigned)ceil_div(cols, team));
  piece_sum_kernel<T, V><<<sums, TEAM_THREADS, 0, s>>>(static_cast<const T*>(g), sorted[at], static_cast<T*>(gw), head, tail, n,
                                                        (int)types, width, cols, team, p.piece, p.pieces, scale);
  if (int rc = check_launch("piece_sum")) return rc;
  join_kernel<T, V><<<(unsigned)ceil_div(p.pieces, JOIN_WARPS), JOIN_WARPS * 32, 0, s>>>(
      sorted[at], static_cast<T*>(gw), head, tail, n, (int)types, width, cols, team, p.piece, p.pieces, scale);
  return check_launch("join");
}

int check_sizes(int dtype, int64_t n, int64_t types, int64_t width) {
  if (dtype != EQT_F32 && dtype != EQT_F64 && dtype != EQT_BF16) return fail(EQT_ERR_BAD_ARGUMENT, "embedding: unknown dtype %d", dtype);
  if (n < 0 || types < 0 || width < 0) return fail(EQT_ERR_BAD_ARGUMENT, "embedding: negative size");
  if (n > INT32_MAX - 1 || types > INT32_MAX - 1 || width > 1 << 20)
    return fail(EQT_ERR_UNSUPPORTED, "embedding: rows and types are numbered in 32 bits, a row has at most 2^20 values");
  return EQT_OK;
}

bool wide(const void* a, const void* b, int64_t width, int dtype) {
  return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % 16 == 0 && width * size_of(dtype) % 16 == 0;
}

}  // namespace
}  // namespace eqt

using namespace eqt;

extern "C" int eqt_embedding_forward(int32_t dtype, const void* weight, const int64_t* index, void* out, int64_t n, int64_t types,
                                     int64_t width, double scale, void* stream) {
  if (int rc = check_sizes(dtype, n, types, width)) return rc;
  if (n == 0 || width == 0) return EQT_OK;
  if (!index || !out || (!weight && types)) return fail(EQT_ERR_BAD_ARGUMENT, "embedding: NULL pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool w = wide(weight, out, width, dtype);
  if (dtype == EQT_F64)
    return w ? run_forward<double, 2>(weight, index, out, n, types, width, scale, s) : run_forward<double, 1>(weight, index, out, n, types, width, scale, s);
  if (dtype == EQT_F32)
    return w ? run_forward<float, 4>(weight, index, out, n, types, width, scale, s) : run_forward<float, 1>(weight, index, out, n, types, width, scale, s);
  return w ? run_forward<__nv_bfloat16, 8>(weight, index, out, n, types, width, scale, s)
           : run_forward<__nv_bfloat16, 1>(weight, index, out, n, types, width, scale, s);
}

extern "C" int64_t eqt_embedding_grad_scratch(int32_t dtype, int64_t n, int64_t types, int64_t width) {
  if (check_sizes(dtype, n, types, width) || n == 0 || types == 0 || width == 0) return 0;
  return (int64_t)grad_plan(dtype, n, types, width).bytes;
}

extern "C" int eqt_embedding_grad(int32_t dtype, const void* g, const int64_t* index, void* gw, int64_t n, int64_t types, int64_t width,
                                  double scale, void* scratch, int64_t scratch_bytes, void* stream) {
  if (int rc = check_sizes(dtype, n, types, width)) return rc;
  if (types == 0 || width == 0) return EQT_OK;
  if (!gw || ((!g || !index) && n)) return fail(EQT_ERR_BAD_ARGUMENT, "embedding gradient: NULL pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0)
    return cudaMemsetAsync(gw, 0, (size_t)types * width * size_of(dtype), s) == cudaSuccess ? EQT_OK : fail(EQT_ERR_CUDA, "cudaMemsetAsync failed");
  const int64_t need = (int64_t)grad_plan(dtype, n, types, width).bytes;
  if (need && (!scratch || scratch_bytes < need))
    return fail(EQT_ERR_BAD_ARGUMENT, "embedding gradient: %lld bytes of scratch given, %lld needed", (long long)scratch_bytes, (long long)need);
  unsigned char* sc = static_cast<unsigned char*>(scratch);
  const bool w = wide(g, gw, width, dtype);
  if (dtype == EQT_F64)
    return w ? run_grad<double, 2>(dtype, g, index, gw, n, types, width, scale, sc, s) : run_grad<double, 1>(dtype, g, index, gw, n, types, width, scale, sc, s);
  if (dtype == EQT_F32)
    return w ? run_grad<float, 4>(dtype, g, index, gw, n, types, width, scale, sc, s) : run_grad<float, 1>(dtype, g, index, gw, n, types, width, scale, sc, s);
  return w ? run_grad<__nv_bfloat16, 8>(dtype, g, index, gw, n, types, width, scale, sc, s)
           : run_grad<__nv_bfloat16, 1>(dtype, g, index, gw, n, types, width, scale, sc, s);
}
