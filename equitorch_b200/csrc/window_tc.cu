// Attention within windows of packed chains on the 5th-generation tensor cores, bfloat16: tiles of 128 nodes of the packed batch, whatever chains they
// belong to, against 64 of the other side at a time.
//
//   FORWARD   S = q k^T          P = exp(S - base)             out += P v
//   ROWS      S, dP = g v^T      dS = P (dP - delta)           dq += dS k
//   COLUMNS   S^T = k q^T, dP^T = v g^T       P^T, dS^T        dv += P^T g,  dk += dS^T q      over the heads that share k and v
//
// A thread of the softmax has one row of the tile (a lane of tensor memory), so maxima, sums and masks cross no threads; what it sees of 64 others
// is one word of 64 bits, made of the row's one or two intervals, and only words that are not full cost selects.  P and dS go back to tensor memory, over
// the scores, as the first operand of the second product.  Windows of neighbouring nodes overlap, so the tile's walk over the others is one stretch, and
// forward and by rows the first nodes of the chain that the tile begins in, before it.  Tiles do not stop at the chains' ends: many short chains fill them.
//
// The forward pass keeps its unit of the exponentials until a row's greatest score is over 2^8 of it, and only then rescales the sums in tensor memory;
// the sum and the result have the same unit, so that loses nothing.  The scores of the next 64 keys are made while the softmax works on these.
// dS goes into dq's product in two parts, as within whole graphs: dq has the error of rounded weights already.  2-norm of the errors 2.3e-3 to 2.4e-3, a rounding of the result
// alone 1.7e-3 (dk and dv have that where there are few tiles, see `launch`); with a delta of rounded results and weights not rounded, dq's was 3.4e-3 where windows are of few nodes, and dk's 2.7e-3.
//
// Two CTAs an SM hide each other's chain of copy, product, softmax and product.  By columns two or three groups of softmax warps take turns in one CTA, which
// has all the tensor memory (64 values a head: 247 -> 217 us for 240 chains of 50 to 500 nodes against two CTAs of one group; by rows, where one thread has
// half the products to issue, that lost: 189 -> 325).  By rows, with one buffer of scores, two warps share a row's 64 others (64 values 196 -> 172 us, 128 values
// 430 -> 406); forward and by columns that lost (128 values 240 -> 266 us, 408 -> 441), for want of registers and of room for the instructions.
// The first 4 (8, 12) warps: softmax; then two that issue MMAs and two that copy.
//
// Two bounds: the special functions (a score is one exponential, 0.22 ps of the GPU; of 4 x 64 flops, 0.16 ps of the tensor cores), and the tensor cores, whose MMA
// of 128 x 64 takes as long as one of 128 x 128: S and dP run at half the rate.  128 keys at a time have the full rate, and lost forward (240 -> 267 us), where tensor
// memory then has one buffer of scores.  One chain of 32,781 nodes, 8 heads of 128, window of 1024 and 4 first nodes: forward 240 us, by rows 395, by columns
// 393, tensor pipe 33 to 37 % busy; a step of 64 takes a CTA 2200 cycles, 1400 of them softmax, the rest the way to the MMAs and back.
// The tensor cores' adder truncates, 1.2e-7 of a sum of one sign at every 16 terms, so sums that may be of more than 8192 terms are taken out every 126 steps, in kernels of
// their own (one chain of 32,781 nodes, window of 16,384, 8 heads of 128: 9.0 -> 9.8 ms; of 64, two heads of keys: 7.5 -> 7.8).
// Every wait is bounded; on expiry the status flag is raised and the kernel ends.
#include <algorithm>

#include "tc_bf16.cuh"
#include "window_tc.cuh"

namespace eqt {
namespace window {
namespace {
using namespace tc;
using attention::copy4;
using T = __nv_bfloat16;

enum Mode { FORWARD, ROWS, COLUMNS };
constexpr int KEYS = 64, LOADERS = 64;                   // of the other side at a time; threads that copy
constexpr int MOST_TILES = 16;                           // of a CTA
constexpr float FAR = 8.f;                               // of log2, that a score may be above the unit

// What a tile walks over: `ns` first nodes of the chain that its first row is in, from `from0` on, to `wide` places (whole eights, what the 128-byte swizzle repeats
// by), then [from1, to1), as one sequence.
struct Stretch {
  int from0, ns, wide, from1, to1, total, steps;
};
constexpr int STRETCHES = 8;

template <int DP, int MODE> struct Form {
  static constexpr int GROUPS = MODE == COLUMNS ? (DP == 128 ? 2 : 3) : 1;             // of softmax warps, each with a buffer of scores
  static constexpr int BUFFERS = MODE == FORWARD ? 2 : GROUPS;
  static constexpr int HALVES = MODE == ROWS ? 2 : 1;                               // warps that share a row's others
  static constexpr int SOFT = 4 * HALVES * GROUPS, THREADS = 32 * (SOFT + 2) + LOADERS, CTAS = GROUPS > 1 ? 1 : 2;
  static constexpr int OWN = MODE == FORWARD ? 1 : 2;                                // operands of the tile's rows
  static constexpr int OWN_BYTES = TILE_M * DP * 2, SLOT_BYTES = KEYS * DP * 2;
  static constexpr int SLOTS = MODE == FORWARD && DP == 128 ? 4 : MODE == ROWS && DP == 128 ? 3 : 8;
  static constexpr int NUMBERS = MODE == COLUMNS ? SLOTS / 2 * 3 * KEYS * 4 : 0;     // bytes: a query's greatest score, inverse sum, delta
  static constexpr int BUFFER = MODE == FORWARD ? KEYS : 2 * KEYS;                   // columns of tensor memory: S, or S and dP
  static constexpr int SUM_AT = BUFFERS * BUFFER, COLS = CTAS == 1 ? 512 : 256;
  static constexpr int BARRIERS = 384;                                               // bytes, with the tensor memory's address and the abort flag
  static constexpr size_t bytes() {
    return (size_t)OWN * OWN_BYTES + (size_t)SLOTS * SLOT_BYTES + NUMBERS + BARRIERS + STRETCHES * sizeof(Stretch) + 4 * GROUPS * MOST_TILES * 4;
  }
  static_assert((2 * SLOTS + 3 * BUFFERS + 4 + STRETCHES) * 8 + 8 <= BARRIERS, "barriers");
  static_assert(SUM_AT + (MODE == COLUMNS ? 2 : 1) * DP <= COLS, "tensor memory");
};

// What a thread copies of an operand's rows: in each group of 64 values the same 16 bytes of every fourth or eighth row (32 or 64 threads), so that where they come
// from moves on by additions; and goes to, but for the 128-byte swizzle (a line of 128 bytes a row).  Zeros behind the head's values, up to whole
// sixteens.  Loops are short on purpose: with all copies laid out one after the other the kernel's code is more than the SM's instruction cache
// holds, and every warp of it waits (by columns, 128 values: 473 -> 604 us).
template <int DP> struct Copier {
  static constexpr int GROUPS = DP / 64;
  const T* from[GROUPS];
  int64_t node;
  int row, col, every, size;
  bool on[GROUPS], there[GROUPS];                        // has values; has a place
  __device__ __forceinline__ Copier(const Operand& x, const AttentionParams& p, int thread, int threads)
      : node(x.node), row(thread >> 3), col(thread & 7), every(threads >> 3), size(p.size) {
    const int values = p.comps * p.size;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int at = (col + 8 * g) * 8;
      on[g] = at < values;
      there[g] = at < (values + 15) / 16 * 16;
      const int comp = on[g] ? at / p.size : 0;
      from[g] = static_cast<const T*>(x.p) + comp * x.comp + (on[g] ? at - comp * p.size : 0);
    }
  }
  __device__ __forceinline__ uint32_t place(int r) const { return (uint32_t)(r * 128 + ((col ^ (r & 7)) << 4)); }
  __device__ __forceinline__ void copy(uint32_t d, const T* f, int g, bool in) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(in ? f : from[g]), "r"(in ? 16 : 0) : "memory");
  }
  // KEYS rows of a head from `first` on, zeros from the `left`-th on
  __device__ __forceinline__ void next(unsigned char* dst, int first, int left, int head) const {
    const int64_t move = (int64_t)(first + row) * node + (int64_t)head * size, step = every * node;
    const uint32_t d = s32(dst);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (!there[g]) continue;
      const T* f = from[g] + move;
#pragma unroll 2
      for (int r = row; r < KEYS; r += every, f += step) copy(d + g * (KEYS * 128) + place(r), f, g, on[g] && r < left);
    }
  }
  // the same of a stretch from its `at`-th row on
  __device__ __forceinline__ void mixed(unsigned char* dst, int at, const Stretch& s, int left, int head) const {
    const uint32_t d = s32(dst);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (!there[g]) continue;
#pragma unroll 2
      for (int r = row; r < KEYS; r += every) {
        const int v = at + r;
        copy(d + g * (KEYS * 128) + place(r), from[g] + (int64_t)(v < s.ns ? s.from0 + v : s.from1 + v - s.wide) * node + (int64_t)head * size, g, on[g] && r < left && (v < s.ns || v >= s.wide));
      }
    }
  }
  // the tile's own: `high` rows of one head after the other
  __device__ __forceinline__ void own(unsigned char* dst, int first, int left, int head, int high) const {
    const uint32_t d = s32(dst);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (!there[g]) continue;
#pragma unroll 2
      for (int r = row; r < TILE_M; r += every) {
        const int h = r / high, q = r - h * high;
        copy(d + g * (TILE_M * 128) + place(r), from[g] + (int64_t)(first + q) * node + (int64_t)(head + h) * size, g, on[g] && q < left);
      }
    }
  }
};

// The barrier has an arrival of this thread when its copies so far have landed.
__device__ __forceinline__ void land_at(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(s32(bar)) : "memory");
}

// The bits of [lo, hi) within 32
__device__ __forceinline__ uint32_t bits_of(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi > lo ? (~0u >> (32 - (hi - lo))) << lo : 0;
}

template <int MODE> __device__ __forceinline__ Stretch stretch_of(const WindowParams& w, int first, int last, int2 a, int2 b) {       // rows first to last, their chains
  Stretch s;
  s.from0 = s.from1 = first;
  s.ns = 0;
  s.to1 = last + 1;
  if (MODE == COLUMNS) {
    if (a.y > a.x) s.from1 = max(a.x, first - w.after);
    if (b.y > b.x) s.to1 = !apart(w, b.x, b.y) && max(b.x, first) < b.x + w.sinks ? b.y : min(b.y, last + w.before + 1);
  } else {
    if (a.y > a.x) {
      s.from1 = max(a.x, first - w.before);
      s.from0 = a.x;
      s.ns = min(s.from1, a.x + w.sinks) - a.x;
    }
    if (b.y > b.x) s.to1 = min(b.y, last + w.after + 1);
  }
  s.wide = (s.ns + 7) & ~7;
  s.total = s.wide + s.to1 - s.from1;
  s.steps = (s.total + KEYS - 1) / KEYS;
  return s;
}

// 32 columns of a lane from and to tensor memory
__device__ __forceinline__ void tmem_put16(uint32_t at, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two float32 values in a pair of registers: packed instructions take half the issue slots, which bound the softmax beside the exponentials.
struct Two {
  uint64_t v;
  __device__ __forceinline__ Two() = default;
  __device__ __forceinline__ Two(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ void apart(float& x, float& y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
};
__device__ __forceinline__ Two two_of(const uint32_t* r) { return Two(__uint_as_float(r[0]), __uint_as_float(r[1])); }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Two bf16_values(uint32_t u) { return Two(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }

// Rows of 64 bytes, a lane each, to lines that four lanes write: piece lane & 3 of the rows of lanes lane, lane ^ 1, lane ^ 2 and lane ^ 3.
__device__ __forceinline__ void across_lanes(uint32_t (&u)[16], int lane) {
  const bool b0 = lane & 1, b1 = lane & 2;
#pragma unroll
  for (int k = 0; k < 8; ++k) {                          // halves of the rows
    const uint32_t keep = b1 ? u[8 + k] : u[k], send = b1 ? u[k] : u[8 + k];
    u[k] = keep;
    u[8 + k] = __shfl_xor_sync(0xffffffffu, send, 2);
  }
#pragma unroll
  for (int h = 0; h < 16; h += 8)                        // and of the halves
#pragma unroll
    for (int k = h; k < h + 4; ++k) {
      const uint32_t keep = b0 ? u[4 + k] : u[k], send = b0 ? u[k] : u[4 + k];
      u[k] = keep;
      u[4 + k] = __shfl_xor_sync(0xffffffffu, send, 1);
    }
}

// FOLDS: a lane's WIDE sums out of tensor memory, onto those that wait in local memory (in a unit that was `kept` times as great), so that the tensor cores' adder, which
// truncates, adds up at most 128 steps (8192 terms).  Before a tile's step of the group's first turn and FOLD_STEPS, and every FOLD_STEPS from there.
constexpr int FOLD_STEPS = 126;                          // a multiple of the groups, which are one, two or three
template <int WIDE> __device__ __noinline__ void take_out(float* beside, uint32_t sum, int wide, bool first, float kept) {
#pragma unroll 1
  for (int h = 0; h < WIDE; h += 32) {
    if (h >= wide) break;
    uint32_t r[32];
    tmem_issue32(sum + h, r);
    tmem_arrived32(r);
    float4* to = reinterpret_cast<float4*>(beside + h);
    float4 v[8];                                         // all of them on their way at once: memory is far
    if (!first) {
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = to[c];
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int c = 0; c < 8; ++c)
      to[c] = make_float4(fmaf(v[c].x, kept, __uint_as_float(r[4 * c])), fmaf(v[c].y, kept, __uint_as_float(r[4 * c + 1])), fmaf(v[c].z, kept, __uint_as_float(r[4 * c + 2])),
                          fmaf(v[c].w, kept, __uint_as_float(r[4 * c + 3])));
  }
}
// Of the lanes' rows of results the WIDE values from the `first` on, with `more` and those `beside` where given, `f` times, to (n, components, heads, channels), and what the rounding
// left to `rest`; whether they were finite.  Loops are not unrolled: code that runs once a tile comes from beyond the instruction cache.
template <int WIDE> __device__ __forceinline__ bool put_row(uint32_t sum, int first, float f, bool on, void* out, int row, int head, const AttentionParams& p, int lane,
                                                            const float* more = nullptr, void* rest = nullptr, const float* beside = nullptr, float kept = 1.f) {
  const int values = p.comps * p.size;
  const int64_t place = on ? ((int64_t)row * p.comps * p.heads + head) * p.size : -1;
  int64_t to[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) to[e] = __shfl_xor_sync(0xffffffffu, place, e);
  const Two times(f, f), zero(0.f, 0.f), less(-1.f, -1.f);
  Two nought = zero;                                     // or NaN, once a sum is not finite
#pragma unroll 1
  for (int h = first; h < min(first + WIDE, values); h += 32) {
    uint32_t r[32];
    tmem_issue32(sum + h, r);
    tmem_arrived32(r);
#pragma unroll
    for (int c = 0; c < 32; c += 8) {
      if (h + c >= values) break;
      if (beside) {
#pragma unroll
        for (int j = c; j < c + 8; ++j) r[j] = __float_as_uint(fmaf(beside[h - first + j], kept, __uint_as_float(r[j])));
      }
      if (more) {
#pragma unroll
        for (int j = c; j < c + 8; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + more[h + j]);
      }
#pragma unroll
      for (int j = c; j < c + 8; j += 2) nought = fma2(two_of(&r[j]), zero, nought);
    }
    const int at = h + 8 * (lane & 3), comp = at / p.size;
    const int64_t offset = (int64_t)comp * (p.heads - 1) * p.size + at;
    void* base = out;
#pragma unroll 1
    for (int t = 0; t < 2 && base; ++t, base = rest) {
      uint32_t u[16];
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const Two v = mul2(two_of(&r[c]), times);
        float x, y;
        v.apart(x, y);
        u[c / 2] = two_bf16(x, y);
        if (t) {
          fma2(bf16_values(u[c / 2]), less, v).apart(x, y);
          u[c / 2] = two_bf16(x, y);
        }
      }
      across_lanes(u, lane);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (to[e] >= 0 && at < values) *reinterpret_cast<uint4*>(static_cast<T*>(base) + to[e] + offset) = make_uint4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]);
    }
  }
  float x, y;
  nought.apart(x, y);
  return x + y == 0.f;
}

// FINE, by columns: weights and score gradients go into their products in two parts.  FOLDS: sums may be of more than 8192 terms.
template <int DP, int MODE, bool FINE, bool FOLDS> __global__ void __launch_bounds__(Form<DP, MODE>::THREADS, Form<DP, MODE>::CTAS) window_tc_kernel(const __grid_constant__ TcParams p) {
  using F = Form<DP, MODE>;
  constexpr int SLOTS = F::SLOTS, GROUPS = F::GROUPS, BUFFERS = F::BUFFERS;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *own = smem, *ring = own + F::OWN * F::OWN_BYTES;
  float* numbers = reinterpret_cast<float*>(ring + SLOTS * F::SLOT_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + SLOTS * F::SLOT_BYTES + F::NUMBERS);
  uint64_t *full = bars, *empty = full + SLOTS, *scores = empty + SLOTS, *weights = scores + BUFFERS, *freed = weights + BUFFERS, *own_full = freed + BUFFERS,
           *own_empty = own_full + 1, *done = own_empty + 1, *sums_free = done + 1, *known = sums_free + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(known + STRETCHES);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  Stretch* stretches = reinterpret_cast<Stretch*>(reinterpret_cast<unsigned char*>(bars) + F::BARRIERS);
  unsigned* bad_rows = reinterpret_cast<unsigned*>(stretches + STRETCHES);                                       // [group's quarter][tile of the CTA]

  const WindowParams& w = p.w;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // A tile is `pack` heads that share their keys by `high` nodes: with fewer nodes, the walk over what any of them sees is shorter.
  const int pack = MODE == COLUMNS ? 1 : p.pack, high = TILE_M / pack, heads = (MODE == COLUMNS ? w.kv.heads : w.q.heads) / pack;
  const int values = w.q.comps * w.q.size, wide = (values + 15) / 16 * 16;
  // A CTA takes every gridDim-th tile.  All roles go through the same tiles and steps and count them, and their barriers' phases, on.  The warps that copy find
  // a tile's stretch, a tile ahead, and leave it for the others; these are fewer tiles behind than there are places, since scores have at most three buffers (and a barrier
  // each: a wait by parity must not be two phases behind, as the softmax may be behind the tile's own rows).
  struct Tile {
    int head, kv, first, last;
  };
  auto tile_of = [&](unsigned i) {
    Tile t;
    t.head = (int)(i % (unsigned)heads) * pack;
    t.kv = MODE == COLUMNS ? t.head : t.head / w.group;
    t.first = (int)(i / (unsigned)heads) * high;
    t.last = min((int)w.q.n, t.first + high) - 1;
    return t;
  };

  if (tid == 0) {
    *abort_flag = (s32(smem) & 1023) != 0;                // the swizzle goes by addresses
    for (int s = 0; s < SLOTS; ++s) {
      bar_init(&full[s], !p.tma ? LOADERS : MODE == COLUMNS && !(s & 1) ? 33 : 1);
      bar_init(&empty[s], 1);
    }
    bar_init(own_full, p.tma ? 1 : LOADERS);
    for (int b = 0; b < BUFFERS; ++b) {
      bar_init(&scores[b], 1);
      bar_init(&weights[b], 4 * F::HALVES);
      bar_init(&freed[b], 1);
    }
    for (int k = 0; k < STRETCHES; ++k) bar_init(&known[k], 1);
    bar_init(own_empty, 1);                              // a tile's scores have been made
    bar_init(done, 1);                                   // and its sums
    bar_init(sums_free, (GROUPS > 1 ? 8 : 4) * F::HALVES);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int b = tid; b < 4 * GROUPS * MOST_TILES; b += F::THREADS) bad_rows[b] = 0;
  if (warp == F::SOFT) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(tmem_slot)), "r"(F::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  volatile int* ab = abort_flag;

  if (warp >= F::SOFT + 2) {
    // ---------------- copies ----------------
    // Items in the order of their use: FORWARD k, v; ROWS v, k; COLUMNS q with its numbers, g.  Heads of 64 or 128 values in one component are
    // copied by TMA, eight rows a lane where a stretch's first nodes are among them; other heads by the threads: their copies arrive at the item's barrier when they have landed, and
    // the thread that issues the MMAs, which sees them all there, puts the fence between them and the tensor cores.  Copying by hand takes the warps
    // issue slots that the softmax wants (one chain of 32,781 nodes, 8 heads of 128 values, by hand and by TMA: 1270 | 1197 us of kernels).
    const int thread = tid - 32 * (F::SOFT + 2), threads = p.tma ? 32 : LOADERS;
    const Copier<DP> even(MODE == FORWARD ? w.q.k : MODE == ROWS ? w.q.v : w.q.q, w.q, thread, threads);
    const Copier<DP> odd(MODE == FORWARD ? w.q.v : MODE == ROWS ? w.q.k : w.q.g, w.q, thread, threads);
    unsigned item = 0, i = blockIdx.x;
    Tile next = tile_of(i);
    int2 a = p.spans[next.first], b = p.spans[next.last];
    auto copy_tile = [&](const Tile& t, const Stretch& walk, int steps, int number) {
      // All threads wait for every place, also where one copies: who skips waits gets phases ahead, and a wait by parity cannot tell a phase from the one but next.
      if (!__all_sync(0xffffffffu, number == 0 || bar_wait(own_empty, (uint32_t)((number - 1) & 1), ab))) return false;
      if (thread == 0) {
        stretches[number % STRETCHES] = walk;
        bar_arrive(&known[number % STRETCHES]);
      }
      if (!p.tma) {
        const int left = t.last + 1 - t.first;
        Copier<DP>(MODE == COLUMNS ? w.q.k : w.q.q, w.q, thread, threads).own(own, t.first, left, t.head, high);
        if (MODE != FORWARD) Copier<DP>(MODE == COLUMNS ? w.q.v : w.q.g, w.q, thread, threads).own(own + F::OWN_BYTES, t.first, left, t.head, high);
        land_at(own_full);
      } else if (thread == 0) {
        bar_expect_tx(own_full, F::OWN * F::OWN_BYTES);
        for (int x = 0; x < F::OWN; ++x)
          for (int h = 0; h < pack; ++h)
            for (int g = 0; g < DP / 64; ++g)
              tma_load_3d(own + x * F::OWN_BYTES + g * (TILE_M * 128) + h * high * 128, &p.own[x], (t.head + h) * DP + g * 64, t.first, 0, own_full);
      }
      int at = 0, h = MODE == COLUMNS ? t.kv * w.group : t.kv;
      for (int k = 0; k < 2 * steps; ++k, ++item) {
        const unsigned slot = item % SLOTS;
        const bool mixed = MODE != COLUMNS && at < walk.wide, numbered = MODE == COLUMNS && !(k & 1);
        if (!__all_sync(0xffffffffu, item < SLOTS || bar_wait(&empty[slot], (uint32_t)((item / SLOTS - 1) & 1), ab))) return false;
        unsigned char* to = ring + slot * F::SLOT_BYTES;
        const Copier<DP>& x = k & 1 ? odd : even;
        if (mixed && p.tma) {                            // eight rows a copy, each lane its own: all of them by hand took longer than a step
          if (thread == 0) bar_expect_tx(&full[slot], F::SLOT_BYTES);
          __syncwarp();
          const int v = at + 8 * thread;
          if (8 * thread < KEYS)
            for (int g = 0; g < DP / 64; ++g)
              tma_load_3d(to + g * (KEYS * 128) + thread * 1024, &p.eight[k & 1], h * DP + g * 64, v < walk.wide ? walk.from0 + v : walk.from1 + v - walk.wide, 0, &full[slot]);
        } else if (mixed) {
          x.mixed(to, at, walk, walk.total - at, h);
        } else if (!p.tma) {
          x.next(to, walk.from1 + at - walk.wide, walk.total - at, h);
        } else if (thread == 0) {
          bar_expect_tx(&full[slot], F::SLOT_BYTES);
          for (int g = 0; g < DP / 64; ++g) tma_load_3d(to + g * (KEYS * 128), &p.ring[k & 1], h * DP + g * 64, walk.from1 + at - walk.wide, 0, &full[slot]);
        }
        if (numbered) {
          for (int c = thread; c < KEYS; c += threads) {
            const int query = walk.from1 + at + c;
            const bool there = query < walk.to1;
            const int64_t from = there ? (int64_t)h * w.q.n + query : 0;
            float* num = numbers + slot / 2 * 3 * KEYS + c;
            copy4(num, w.q.top + from, there);
            copy4(num + KEYS, w.inverse + from, there);
            copy4(num + 2 * KEYS, w.q.delta + from, there);
          }
        }
        if (!p.tma || numbered) land_at(&full[slot]);
        if ((k & 1) && (at += KEYS) >= walk.total) at = 0, ++h;          // COLUMNS: the next head
      }
      return true;
    };
    for (int number = 0; thread < threads; ++number) {
      const Tile t = next;
      const Stretch walk = stretch_of<MODE>(w, t.first, t.last, a, b);
      const bool more = p.tiles - i > gridDim.x;
      if (more) {
        next = tile_of(i += gridDim.x);
        a = p.spans[next.first], b = p.spans[next.last];
      }
      if (!copy_tile(t, walk, walk.steps * (MODE == COLUMNS ? w.group : 1), number) || !more) break;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= F::SOFT) {
    // ---------------- MMAs ----------------
    // One thread makes S and dP, another adds weighted rows up: each MMA costs its thread some ninety cycles whatever its size, and a step has up to 24.
    if (lane == 0) {
      const uint32_t to_scores = idesc_bf16(TILE_M, KEYS), to_sums = idesc_bf16(TILE_M, wide, false, true);
      const uint32_t own_at = s32(own), ring_at = s32(ring), sum = tmem + F::SUM_AT;
      const int ksteps = wide / 16;
      // of steps counted over all tiles
      auto slot_at = [&](unsigned item) { return ring_at + item % SLOTS * F::SLOT_BYTES; };
      auto arrived = [&](unsigned item) { return bar_wait(&full[item % SLOTS], (item / SLOTS) & 1, ab); };
      auto fence = [] { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); };
      // scores of a step are free when the products that read them BUFFERS steps before are done
      auto free_again = [&](unsigned j) { return j < BUFFERS || bar_wait(&freed[j % BUFFERS], (j / BUFFERS - 1) & 1, ab); };
      auto weighted = [&](unsigned j) { return bar_wait(&weights[j % BUFFERS], (j / BUFFERS) & 1, ab); };
      // d (128 rows x 64) = rows of the tile times rows of the slot
      auto score = [&](uint32_t d, uint32_t a, uint32_t b) {
        const uint32_t a_lo = umma_lo(a), b_lo = umma_lo(b);
        umma_bf16<false>(d, a_lo, b_lo, to_scores);
#pragma unroll
        for (int k = 1; k < DP / 16; ++k)
          if (k < ksteps) umma_bf16<true>(d, a_lo + (k >> 2) * (TILE_M * 128 / 16) + (k & 3) * K_STEP, b_lo + (k >> 2) * (KEYS * 128 / 16) + (k & 3) * K_STEP, to_scores);
      };
      // d (128 rows x values) += weights in tensor memory, 32 at the front of every 32 columns, times the slot
      auto add = [&](uint32_t d, uint32_t a, uint32_t b, bool more) {
        const uint32_t b_lo = umma_lo_rows(b, KEYS * 128);
        if (more) umma_bf16_ta<true>(d, a, b_lo, to_sums);
        else umma_bf16_ta<false>(d, a, b_lo, to_sums);
#pragma unroll
        for (int k = 1; k < KEYS / 16; ++k) umma_bf16_ta<true>(d, a + (k >> 1) * 32 + (k & 1) * 8, b_lo + k * ROWS_STEP, to_sums);
      };
      bool ok = true;
      constexpr int S_ITEM = MODE == ROWS ? 1 : 0;
      auto make_s = [&](unsigned j) {
        ok = ok && arrived(2 * j + S_ITEM) && free_again(j);
        if (!ok) return;
        fence();
        tc_fence_after();
        score(tmem + (j % BUFFERS) * F::BUFFER, own_at, slot_at(2 * j + S_ITEM));
        if (MODE == FORWARD) umma_commit(&empty[2 * j % SLOTS]);
      };
      // By rows, the place of dP is free when the softmax has read it.
      auto make_dp = [&](unsigned j) {
        ok = ok && arrived(2 * j + 1 - S_ITEM) && (MODE == COLUMNS || j < BUFFERS || weighted(j - BUFFERS));
        if (!ok) return;
        fence();
        tc_fence_after();
        score(tmem + (j % BUFFERS) * F::BUFFER + KEYS, own_at + F::OWN_BYTES, slot_at(2 * j + 1 - S_ITEM));
        if (MODE == ROWS) umma_commit(&empty[2 * j % SLOTS]);
      };
      unsigned j = 0;
      int number = 0;
      for (unsigned i = blockIdx.x; i < p.tiles && ok; i += gridDim.x, ++number) {
        ok = bar_wait(&known[number % STRETCHES], (uint32_t)(number / STRETCHES & 1), ab) && (warp != F::SOFT || bar_wait(own_full, (uint32_t)(number & 1), ab));
        if (!ok) break;
        const unsigned end = j + stretches[number % STRETCHES].steps * (MODE == COLUMNS ? w.group : 1);
        if (warp == F::SOFT) {
          for (; j < end && ok; ++j) {
            if (MODE == ROWS) make_dp(j);
            make_s(j);
            if (MODE == COLUMNS) make_dp(j);
            if (ok) umma_commit(&scores[j % BUFFERS]);
          }
          if (ok) umma_commit(own_empty);
          continue;
        }
        ok = number == 0 || bar_wait(sums_free, (uint32_t)((number - 1) & 1), ab);
        const unsigned start = j;
        // a sum starts anew where a group takes out what there is: that of dk the last group, others the first
        unsigned anew = start + (GROUPS - start % GROUPS) % GROUPS + FOLD_STEPS, anew_k = start + (GROUPS - 1 + GROUPS - start % GROUPS) % GROUPS + FOLD_STEPS;
        auto goes_on = [&](unsigned& next) {
          if (!FOLDS || j != next) return j != start;
          next += FOLD_STEPS;
          return false;
        };
        for (; j < end && ok; ++j) {
          const uint32_t d = tmem + (j % BUFFERS) * F::BUFFER;
          ok = arrived(2 * j + 1) && (MODE != COLUMNS || arrived(2 * j));
          if (!ok) break;
          fence();
          ok = weighted(j);
          if (!ok) break;
          tc_fence_after();
          add(sum, d, slot_at(2 * j + 1), goes_on(anew));
          if (MODE == ROWS || FINE) add(sum, d + 16, slot_at(2 * j + 1), true);
          if (MODE == COLUMNS) {
            add(sum + DP, d + KEYS, slot_at(2 * j), goes_on(anew_k));
            if (FINE) add(sum + DP, d + KEYS + 16, slot_at(2 * j), true);
            umma_commit(&empty[2 * j % SLOTS]);
          }
          umma_commit(&empty[(2 * j + 1) % SLOTS]);
          umma_commit(&freed[j % BUFFERS]);
        }
        if (ok) umma_commit(done);
      }
    }
  } else {
    // ---------------- softmax ----------------
    constexpr int HALVES = F::HALVES, WIDE = DP / HALVES, CHUNKS = KEYS / HALVES / 32;         // a thread's part of the results and of 64 others
    const int quarter = warp & 3, half = (warp >> 2) % HALVES, group = warp / (4 * HALVES), place = quarter * 32 + lane, first_value = half * WIDE;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), sum_at = lanes + F::SUM_AT;
    // whether all threads of a row's two warps have it so; they meet here
    auto both = [&](bool x) {
      if (HALVES == 1) return __all_sync(0xffffffffu, x) != 0;
      int r;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, 64, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
                   : "=r"(r) : "r"((int)x), "r"(1 + group * 4 + quarter) : "memory");
      return r != 0;
    };
    const float unit = w.q.scale * LOG2E;
    bool ok = true;
    unsigned j0 = 0;                                     // steps of the tiles before
    int tiles_done = 0;
    // the lane's node, and a tile ahead its chain
    const int in_tile = place % high, in_pack = place / high;
    auto span_of = [&](unsigned i) {
      const int row = (int)(i / (unsigned)heads) * high + in_tile;
      return i < p.tiles && row < w.q.n ? p.spans[row] : make_int2(0, 0);
    };
    int2 next_span = span_of(blockIdx.x);
    int number = 0;
    alignas(16) attention::Far<FOLDS ? 2 * WIDE : 2> waiting;
    float* const beside = FOLDS ? waiting.at() : nullptr;
    for (unsigned i = blockIdx.x; i < p.tiles; i += gridDim.x, ++number) {
    const Tile tile = tile_of(i);
    bool taken = false;                                  // some of the tile's sums are beside
    int take_next = FOLD_STEPS;
    // before the tile's k-th step, once all products of those before it are there
    auto take_out_sums = [&](unsigned j, uint32_t sum, float kept) {
      take_next += FOLD_STEPS;
      ok = __all_sync(0xffffffffu, bar_wait(&freed[(j - 1) % BUFFERS], ((j - 1) / BUFFERS) & 1, ab));
      if (!ok) return false;
      tc_fence_after();
      take_out<WIDE>(beside, sum, values - first_value, !taken, kept);
      taken = true;
      return true;
    };
    const int row = tile.first + in_tile, mine = tile.head + in_pack;
    const int2 span = next_span;
    next_span = span_of(i + gridDim.x);
    const bool on = span.y > span.x;
    ok = both(bar_wait(&known[number % STRETCHES], (uint32_t)(number / STRETCHES & 1), ab));       // both warps go on or neither
    if (!ok) break;
    const Stretch walk = stretches[number % STRETCHES];
    const int steps = walk.steps * (MODE == COLUMNS ? w.group : 1);
    // what the row sees: [lo, hi), and the first nodes [span.x, far)
    const int lo = !on ? 0 : max(span.x, row - (MODE == COLUMNS ? w.after : w.before));
    const int hi = !on ? 0 : MODE == COLUMNS ? (!apart(w, span.x, span.y) && row < span.x + w.sinks ? span.y : min(span.y, row + w.before + 1)) : min(span.y, row + w.after + 1);
    const int far = on && MODE != COLUMNS ? min(lo, span.x + w.sinks) : 0;
    // as bits of the 32 from the stretch's `at`-th on; first nodes are before `from1`, or in the stretch behind it, or both
    auto seen = [&](int at) {
      const int shift = walk.from1 - walk.wide + at;
      uint32_t bits = bits_of(lo - shift, hi - shift);
      if (MODE != COLUMNS) {
        bits |= bits_of(max(span.x, walk.from1) - shift, far - shift);
        if (at < walk.ns && span.x < walk.from1) bits |= bits_of(span.x - walk.from0 - at, min(far - walk.from0, walk.ns) - at);
      }
      return bits;
    };
    // all sums of the tile are there; after reading them they may be written again
    auto sums_there = [&] {
      ok = both(ok);
      if (ok) ok = both(bar_wait(done, (uint32_t)(number & 1), ab));
      tc_fence_after();
      return ok;
    };
    auto sums_read = [&](bool bad) {
      tc_fence_before();
      const unsigned rows = __ballot_sync(0xffffffffu, bad);
      if (lane == 0) {
        bar_arrive(sums_free);
        if (rows) atomicOr(&bad_rows[(group * 4 + quarter) * MOST_TILES + number], rows);
      }
      tiles_done = number + 1;
    };
    if (MODE == FORWARD) {
      float base = -INFINITY, total = 0.f, kept = 1.f;
      for (int k = 0; k < steps; ++k) {
        const unsigned j = j0 + k, b = j % BUFFERS;
        ok = __all_sync(0xffffffffu, bar_wait(&scores[b], (j / BUFFERS) & 1, ab));
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_at = lanes + b * F::BUFFER;
        uint32_t raw[CHUNKS][32];
#pragma unroll
        for (int h = 0; h < CHUNKS; ++h) tmem_issue32(s_at + 32 * h, raw[h]);
        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < CHUNKS; ++h) {
          tmem_arrived32(raw[h]);
          const uint32_t bits = seen(k * KEYS + 32 * h);
          if (!__all_sync(0xffffffffu, bits == ~0u)) {
#pragma unroll
            for (int c = 0; c < 32; ++c) raw[h][c] = (bits >> c) & 1 ? raw[h][c] : 0xff800000u;
          }
#pragma unroll
          for (int c = 0; c < 32; ++c) most[c & 3] = fmaxf(most[c & 3], __uint_as_float(raw[h][c]));
        }
        if (FOLDS && k == take_next) {
          if (!take_out_sums(j, sum_at, kept)) break;
          kept = 1.f;
        }
        const float now = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * unit;
        const bool higher = now > base + FAR || (base == -INFINITY && now > base);
        if (__any_sync(0xffffffffu, higher)) {           // another unit: what there is so far goes by it
          // by whole steps, if float32 has the step: the rounding of a weight is the same in any unit of a row
          const float rise = now - base, unit_now = rise < INFINITY ? base + ceilf(rise) : now;
          const float keep = !higher ? 1.f : base == -INFINITY ? 0.f : exp2_fast(base - unit_now);
          total *= keep;
          if (FOLDS) kept *= keep;
          if (higher) base = unit_now;
          if (k > 0) {
            ok = __all_sync(0xffffffffu, bar_wait(&freed[(j - 1) % BUFFERS], ((j - 1) / BUFFERS) & 1, ab));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < DP; h += 32) {
              if (h >= wide) break;
              float v[32];
              tmem_ld32(sum_at + h, v);
#pragma unroll
              for (int c = 0; c < 32; ++c) v[c] *= keep;
              tmem_st32(sum_at + h, v);
            }
          }
        }
        const float minus = base == -INFINITY ? 0.f : -base;
        const Two units(unit, unit), minuses(minus, minus);
        Two add[2] = {Two(0.f, 0.f), Two(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < CHUNKS; ++h) {
          uint32_t out[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float x, y;
            fma2(two_of(&raw[h][c]), units, minuses).apart(x, y);
            out[c >> 1] = two_bf16(exp2_fast(x), exp2_fast(y));
            add[(c >> 1) & 1] = add2(add[(c >> 1) & 1], bf16_values(out[c >> 1]));     // the sum is that of the rounded weights
          }
          tmem_put16(s_at + 32 * h, out);
        }
        float even, odd;
        add2(add[0], add[1]).apart(even, odd);
        total += even + odd;
        tmem_stored();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&weights[b]);
      }
      if (sums_there()) {
        const float inverse = 1.f / total;
        const bool finite = put_row<WIDE>(sum_at, first_value, inverse, on, w.q.out, row, mine, w.q, lane, nullptr, w.rest, taken ? beside : nullptr, kept);
        sums_read(on && !finite);
        if (on && w.q.top) w.q.top[(int64_t)mine * w.q.n + row] = base, w.q.inverse[(int64_t)mine * w.q.n + row] = inverse;
      }
    } else if (MODE == ROWS) {
      const int64_t at_row = (int64_t)mine * w.q.n + row;
      float top = INFINITY, inverse = 0.f, delta = 0.f;
      if (on) top = w.q.top[at_row], inverse = w.q.inverse[at_row], delta = w.q.delta[at_row];
      Two sums(0.f, 0.f), exact(0.f, 0.f);               // of weights before rounding, and of these times dP: for the columns
      const Two units(unit, unit), minuses(-top, -top), inverses(inverse, inverse), deltas(-delta * inverse, -delta * inverse), less(-1.f, -1.f);
      static_assert(MODE != ROWS || GROUPS == 1, "one group by rows");
      for (int k = 0; k < steps; ++k) {
        const unsigned j = j0 + k, b = j % BUFFERS;
        ok = bar_wait(&scores[b], (j / BUFFERS) & 1, ab);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        if (FOLDS && k == take_next && !take_out_sums(j, sum_at + first_value, 1.f)) break;
        const uint32_t word = seen(k * KEYS + 32 * half);
        const bool all = __all_sync(0xffffffffu, word == ~0u);
        uint32_t s[32], d[32], large[16], small[16];
        const uint32_t s_at = lanes + b * F::BUFFER + 32 * half;
        tmem_issue32(s_at, s);
        tmem_issue32(s_at + KEYS, d);
        tmem_arrived32(s);
        tmem_arrived32(d);
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          float e[2], x[2];
          fma2(two_of(&s[c]), units, minuses).apart(e[0], e[1]);
          Two dp = two_of(&d[c]);
          e[0] = exp2_fast(e[0]), e[1] = exp2_fast(e[1]);
          if (!all) {                                  // zero times zero for what is not seen
            const bool see[2] = {(bool)((word >> c) & 1), (bool)((word >> (c + 1)) & 1)};
            e[0] = see[0] ? e[0] : 0.f, e[1] = see[1] ? e[1] : 0.f;
            dp = Two(see[0] ? __uint_as_float(d[c]) : 0.f, see[1] ? __uint_as_float(d[c + 1]) : 0.f);
          }
          const Two before(e[0], e[1]);
          sums = add2(sums, before);
          exact = fma2(before, dp, exact);
          const Two ds = mul2(bf16_values(two_bf16(e[0], e[1])), fma2(dp, inverses, deltas));
          ds.apart(x[0], x[1]);
          large[c / 2] = two_bf16(x[0], x[1]);
          fma2(bf16_values(large[c / 2]), less, ds).apart(x[0], x[1]);
          small[c / 2] = two_bf16(x[0], x[1]);
        }
        tmem_put16(s_at, large);
        tmem_put16(s_at + 16, small);
        tmem_stored();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&weights[b]);
      }
      if (sums_there()) {
        const bool finite = put_row<WIDE>(sum_at, first_value, w.q.scale, on, w.q.dq, row, mine, w.q, lane, nullptr, nullptr, taken ? beside : nullptr);
        sums_read(on && !finite);
        // One half leaves its sums where the other's go, whose threads have had delta and wait for it (there is no more shared memory at 128 values).
        float s[2], x[2];
        sums.apart(s[0], s[1]), exact.apart(x[0], x[1]);
        float weight = s[0] + s[1], weighted = x[0] + x[1];
        if (half && on) w.inverse[at_row] = weight, w.q.delta[at_row] = weighted;
        both(true);
        if (!half && on) {
          weight = 1.f / (weight + w.inverse[at_row]);
          w.q.delta[at_row] = (weighted + w.q.delta[at_row]) * weight;
          w.inverse[at_row] = weight;
        }
      }
    } else {
      const int skip = (int)((group + GROUPS - j0 % GROUPS) % GROUPS);      // the groups take turns over all tiles' steps
      int at = skip % walk.steps * KEYS;
      take_next += skip;
      const Two minus_units(-unit, -unit), less(-1.f, -1.f);
      for (int k = skip; k < steps; k += GROUPS) {
        const unsigned j = j0 + k, b = j % BUFFERS, slot = 2 * j % SLOTS;
        ok = bar_wait(&full[slot], (2 * j / SLOTS) & 1, ab) && bar_wait(&scores[b], (j / BUFFERS) & 1, ab);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        if (FOLDS && (group == 0 || group == GROUPS - 1) && k == take_next && !take_out_sums(j, group == 0 ? sum_at : sum_at + DP, 1.f)) break;
        const int from = at;
        for (at += GROUPS * KEYS; at >= walk.steps * KEYS;) at -= walk.steps * KEYS;
        const float* num = numbers + slot / 2 * 3 * KEYS;
        const uint32_t s_at = lanes + b * F::BUFFER;
#pragma unroll 1
        for (int h = half * CHUNKS; h < (half + 1) * CHUNKS; ++h) {
          const uint32_t word = seen(from + 32 * h);
          const bool all = __all_sync(0xffffffffu, word == ~0u);
          uint32_t s[32], d[32], pt[2][16], dst[2][16];  // large and small parts
          tmem_issue32(s_at + 32 * h, s);
          tmem_issue32(s_at + KEYS + 32 * h, d);
          tmem_arrived32(s);
          tmem_arrived32(d);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 top = *reinterpret_cast<const float4*>(num + 32 * h + c), inverse = *reinterpret_cast<const float4*>(num + KEYS + 32 * h + c),
                         delta = *reinterpret_cast<const float4*>(num + 2 * KEYS + 32 * h + c);
            const Two tops[2] = {Two(top.x, top.y), Two(top.z, top.w)}, inverses[2] = {Two(inverse.x, inverse.y), Two(inverse.z, inverse.w)},
                      deltas[2] = {Two(delta.x, delta.y), Two(delta.z, delta.w)};
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              fma2(two_of(&s[c + i]), minus_units, tops[i / 2]).apart(x[i], x[i + 1]);
              const Two weight = mul2(Two(exp2_fast(-x[i]), exp2_fast(-x[i + 1])), inverses[i / 2]);
              weight.apart(x[i], x[i + 1]);
              mul2(weight, fma2(deltas[i / 2], less, two_of(&d[c + i]))).apart(y[i], y[i + 1]);
            }
            if (!all) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool see = (word >> (c + i)) & 1;
                x[i] = see ? x[i] : 0.f;
                y[i] = see ? y[i] : 0.f;
              }
            }
            auto parts = [&](uint32_t(&to)[2][16], int at, float a, float b) {
              to[0][at] = two_bf16(a, b);
              if (FINE) {
                float a1, b1;
                fma2(bf16_values(to[0][at]), less, Two(a, b)).apart(a1, b1);
                to[1][at] = two_bf16(a1, b1);
              }
            };
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              parts(pt, (c + i) / 2, x[i], x[i + 1]);
              parts(dst, (c + i) / 2, y[i], y[i + 1]);
            }
          }
#pragma unroll
          for (int part = 0; part < (FINE ? 2 : 1); ++part) {
            tmem_put16(s_at + 32 * h + 16 * part, pt[part]);
            tmem_put16(s_at + KEYS + 32 * h + 16 * part, dst[part]);
          }
        }
        tmem_stored();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&weights[b]);
      }
      // one group stores each sum, the others go on
      ok = both(ok);
      if ((group == 0 || group == GROUPS - 1) && sums_there()) {
        bool finite = true;
        const float* more = on ? far_of(w, row, tile.kv, span.x, span.y) : nullptr;
        if (group == 0) finite = put_row<WIDE>(sum_at, first_value, 1.f, on, w.kv.dv, row, tile.kv, w.kv, lane, more ? more + FAR_ROWS * values : nullptr, nullptr, taken ? beside : nullptr);
        if (group == GROUPS - 1) finite = put_row<WIDE>(sum_at + DP, first_value, w.q.scale, on, w.kv.dk, row, tile.kv, w.kv, lane, more, nullptr, taken ? beside : nullptr) && finite;
        sums_read(on && !finite);
      }
    }
    j0 += steps;
    if (!__all_sync(0xffffffffu, ok)) break;
    }
    // Rows that are not finite, when no role waits for this one any more and both halves have theirs: a row takes long.
    asm volatile("barrier.cta.sync 15, %0;" ::"n"(32 * F::SOFT) : "memory");
    for (int number = half; number < tiles_done; number += HALVES) {
      const Tile tile = tile_of(blockIdx.x + number * gridDim.x);
      for (unsigned bad = bad_rows[(group * 4 + quarter) * MOST_TILES + number]; bad; bad &= bad - 1) {
        const int at = quarter * 32 + __ffs(bad) - 1, row = tile.first + at % high, mine = tile.head + at / high;
        const int2 span = p.spans[row];
        if (MODE == FORWARD) again_forward<T>(w, row, mine, span.x, span.y, lane);
        if (MODE == ROWS) again_rows<T>(w, row, mine, span.x, span.y, lane);
        if (MODE == COLUMNS) again_columns<T>(w, row, tile.kv, span.x, span.y, lane, group == 0, group == GROUPS - 1);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) {
    atomicExch(p.status, 2);
    let_copies_land(full, SLOTS);
    let_copies_land(own_full, 1);
  }
  __syncthreads();
  if (warp == F::SOFT) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::COLS) : "memory");
  }
}

// delta = <g, out + rest> of every node and head: `lanes` threads a head (a power of two), 16 bytes each, neighbouring heads side by side.  Apart from the rows' pass, whose
// threads have a row each and would read both with a line for every 16 bytes.
__global__ void __launch_bounds__(256) delta_kernel(const __grid_constant__ WindowParams p, int lanes) {
  const int values = p.q.comps * p.q.size, lane = threadIdx.x & (lanes - 1);
  const int64_t count = p.q.n * p.q.heads, step = (int64_t)gridDim.x * 256 / lanes, rounds = ceil_div(count, step);
  int64_t at = (blockIdx.x * (int64_t)256 + threadIdx.x) / lanes;
  for (int64_t k = 0; k < rounds; ++k, at += step) {     // as many for all: the shuffles want whole warps
    const int64_t node = count <= UINT32_MAX ? (unsigned)at / (unsigned)p.q.heads : at / p.q.heads;
    const int head = (int)(at - node * p.q.heads), e = lane * 8, comp = e / p.q.size;
    float sum = 0.f;
    if (at < count && e < values) {
      const int64_t place = ((node * p.q.comps + comp) * p.q.heads + head) * p.q.size + e - comp * p.q.size;
      auto words = [&](const void* base) { return __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(base) + place)); };
      const uint4 a = words(p.q.out), b = words(p.q.g.p), c = words(p.rest);
      const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w}, z[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum = fmaf(__uint_as_float(x[i] << 16) + __uint_as_float(z[i] << 16), __uint_as_float(y[i] << 16), sum);
        sum = fmaf(__uint_as_float(x[i] & 0xffff0000u) + __uint_as_float(z[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), sum);
      }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (at < count && lane == 0) p.q.delta[(int64_t)head * p.q.n + node] = sum;
  }
}

// The chain of every node, [0, 0) of none.
__global__ void __launch_bounds__(256) spans_kernel(const int64_t* __restrict__ ptr, int64_t chains, int2* __restrict__ spans, int64_t n) {
  const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (i >= n) return;
  int64_t lo = 0, hi = chains;                           // the last boundary at or before the node
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) / 2;
    if (ptr[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  const bool in = lo < chains && ptr[lo] <= i;
  spans[i] = in ? make_int2((int)ptr[lo], (int)ptr[lo + 1]) : make_int2(0, 0);
}

template <int DP, int MODE> int launch(const TcParams& p, cudaStream_t s) {
  using F = Form<DP, MODE>;
  const int64_t tiles = MODE == COLUMNS ? ceil_div(p.w.q.n, TILE_M) * p.w.kv.heads : ceil_div(p.w.q.n, TILE_M / p.pack) * (p.w.q.heads / p.pack);
  if (tiles > INT32_MAX) return fail(EQT_ERR_UNSUPPORTED, "window_attention: %lld tiles are more than one launch takes", (long long)tiles);
  // Tiles of a CTA are settled beforehand, which is for even ones: by columns, those with first nodes walk further (217 us with a CTA each, 234 so; of even ones 470
  // and 416; one chain of 32,781 and 400 of 300: 447 and 561), unless chains are on average so short that it is not far (100,000 chains of 20: 7970 and 5620 us) or so long
  // that they are taken apart.
  const bool even = MODE != COLUMNS || p.w.sinks == 0 || p.w.q.n / TILE_M <= p.w.chains || (p.w.split && p.w.q.n / p.w.apart >= p.w.chains);
  const int64_t grid = even ? std::min<int64_t>(tiles, std::max<int64_t>((int64_t)sm_count() * F::CTAS, ceil_div(tiles, MOST_TILES))) : tiles;
  TcParams t = p;
  t.tiles = (unsigned)tiles;
  const int64_t width = (int64_t)p.w.q.heads * DP, kv_width = (int64_t)p.w.kv.heads * DP;
  t.tma = p.w.q.comps == 1 && p.w.q.size == DP && p.w.q.q.node >= width && p.w.q.k.node >= kv_width && p.w.q.v.node >= kv_width;
  if (t.tma) {
    const AttentionParams& q = p.w.q;
    auto map = [&](CUtensorMap* m, const Operand& x, int heads, int lines) { return map_bf16(m, x.p, q.n, (int64_t)heads * DP, x.node, x.node, 1, lines); };
    const int kv_heads = p.w.kv.heads, high = TILE_M / p.pack;
    int rc;
    if (MODE == COLUMNS) {
      (void)((rc = map(&t.own[0], q.k, kv_heads, TILE_M)) || (rc = map(&t.own[1], q.v, kv_heads, TILE_M)) || (rc = map(&t.ring[0], q.q, q.heads, KEYS)) ||
             (rc = map(&t.ring[1], q.g, q.heads, KEYS)));
    } else {
      (void)((rc = map(&t.own[0], q.q, q.heads, high)) || (MODE == ROWS && (rc = map(&t.own[1], q.g, q.heads, high))) ||
             (rc = map(&t.ring[MODE == ROWS], q.k, kv_heads, KEYS)) || (rc = map(&t.ring[MODE == FORWARD], q.v, kv_heads, KEYS)) ||
             (rc = map(&t.eight[MODE == ROWS], q.k, kv_heads, 8)) || (rc = map(&t.eight[MODE == FORWARD], q.v, kv_heads, 8)));
    }
    if (rc) return rc;
  }
  // In two parts, dk and dv have no rounding but their own, and a step by columns a fifth more to do.  Where there are no more tiles than SMs, what a call takes is
  // latency, and where few nodes share a chain their roundings do not average out (2-norm of the errors up to 2.6e-3 | 1.7e-3; one chain of 2000 nodes, 8
  // heads of 64: 84 | 89 us of kernels; one chain of 32,781, 128 values, dS alone in two: 1131 | 1180).
  const bool fine = MODE == COLUMNS && tiles <= sm_count(), folds = MODE == COLUMNS ? p.w.folds_columns : p.w.folds_rows;
  auto kernel = folds ? window_tc_kernel<DP, MODE, false, true> : window_tc_kernel<DP, MODE, false, false>;
  if constexpr (MODE == COLUMNS)
    if (fine) kernel = folds ? window_tc_kernel<DP, MODE, true, true> : window_tc_kernel<DP, MODE, true, false>;
  static std::atomic<uint64_t> allowed[4]{};
  if (int rc = allow_shared_once(kernel, F::bytes(), allowed[2 * folds + fine])) return rc;
  kernel<<<(unsigned)grid, F::THREADS, F::bytes(), s>>>(t);
  return check_launch("window_tc");
}

}  // namespace
}  // namespace window
}  // namespace eqt

int eqt::window::spans(const int64_t* ptr, int64_t chains, int2* out, int64_t n, cudaStream_t s) {
  spans_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(ptr, chains, out, n);
  return check_launch("window_spans");
}
int eqt::window::tc_forward(const TcParams& p, cudaStream_t s) {
  return p.w.q.comps * p.w.q.size <= 64 ? launch<64, FORWARD>(p, s) : launch<128, FORWARD>(p, s);
}
int eqt::window::tc_backward(const TcParams& p, cudaStream_t s) {
  const bool narrow = p.w.q.comps * p.w.q.size <= 64;
  int lanes = 1;
  while (lanes * 8 < p.w.q.comps * p.w.q.size) lanes *= 2;
  delta_kernel<<<flat_grid(ceil_div(p.w.q.n * p.w.q.heads * lanes, 2), 256), 256, 0, s>>>(p.w, lanes);
  if (int rc = check_launch("window_delta")) return rc;
  if (int rc = narrow ? launch<64, ROWS>(p, s) : launch<128, ROWS>(p, s)) return rc;
  if (p.w.split)
    if (int rc = far_bf16(p.w, s)) return rc;
  return narrow ? launch<64, COLUMNS>(p, s) : launch<128, COLUMNS>(p, s);
}
