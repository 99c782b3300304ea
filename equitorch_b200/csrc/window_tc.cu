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
// dS goes into dq's product in two parts, as within whole graphs: dq has the error of delta, which goes by the rounded result, already.
//
// Two CTAs an SM hide each other's chain of copy, product, softmax and product.  By columns two or three groups of softmax warps take turns in one CTA, which
// has all the tensor memory (64 values a head: 247 -> 217 us for 240 chains of 50 to 500 nodes against two CTAs of one group; by rows, where one thread has
// half the products to issue, that lost: 189 -> 325).  Warps 0 to 3 (7, 11): softmax; then two that issue MMAs and two that copy.
//
// Bound by the special functions at 64 values a head (a score is 4 x 64 flops, 0.16 ps of the tensor cores, and one exponential, 0.22 ps) and by the
// tensor cores at 128.  Every wait is bounded; on expiry the status flag is raised and the kernel ends.
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
constexpr float FAR = 8.f;                               // of log2, that a score may be above the unit

template <int DP, int MODE> struct Form {
  static constexpr int GROUPS = MODE == COLUMNS ? (DP == 128 ? 2 : 3) : 1;             // of softmax warps, each with a buffer of scores
  static constexpr int BUFFERS = MODE == FORWARD ? 2 : GROUPS;
  static constexpr int SOFT = 4 * GROUPS, THREADS = 32 * (SOFT + 2) + LOADERS, CTAS = GROUPS > 1 ? 1 : 2;
  static constexpr int OWN = MODE == FORWARD ? 1 : 2;                                // operands of the tile's rows
  static constexpr int OWN_BYTES = TILE_M * DP * 2, SLOT_BYTES = KEYS * DP * 2;
  static constexpr int SLOTS = MODE == FORWARD && DP == 128 ? 4 : MODE == ROWS && DP == 128 ? 3 : 8;
  static constexpr int NUMBERS = MODE == COLUMNS ? SLOTS / 2 * 3 * KEYS * 4 : 0;     // bytes: a query's greatest score, inverse sum, delta
  static constexpr int BUFFER = MODE == FORWARD ? KEYS : 2 * KEYS;                   // columns of tensor memory: S, or S and dP
  static constexpr int SUM_AT = BUFFERS * BUFFER, COLS = CTAS == 1 ? 512 : 256;
  static constexpr size_t bytes() { return (size_t)OWN * OWN_BYTES + (size_t)SLOTS * SLOT_BYTES + NUMBERS + 512; }
  static_assert(LOADERS == KEYS, "a number of a query each");
  static_assert(SUM_AT + (MODE == COLUMNS ? 2 : 1) * DP <= COLS, "tensor memory");
};

// What a thread copies of an operand's rows: in each group of 64 values the same 16 bytes of every eighth row, so that where they come from and go
// (128-byte swizzle, a line of 128 bytes a row) moves on by additions.  Zeros behind the head's values, up to whole sixteens.
template <int DP> struct Copier {
  static constexpr int GROUPS = DP / 64;
  const T* from[GROUPS];
  int64_t node;
  int row, size;
  uint32_t to;
  bool on[GROUPS], there[GROUPS];                        // has values; has a place
  __device__ __forceinline__ Copier(const Operand& x, const AttentionParams& p, int thread) : node(x.node), row(thread >> 3), size(p.size) {
    const int col = thread & 7, values = p.comps * p.size;
    to = (uint32_t)(row * 128 + ((col ^ row) << 4));
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int at = (col + 8 * g) * 8;
      on[g] = at < values;
      there[g] = at < (values + 15) / 16 * 16;
      const int comp = on[g] ? at / p.size : 0;
      from[g] = static_cast<const T*>(x.p) + comp * x.comp + (on[g] ? at - comp * p.size : 0) + row * node;
    }
  }
  // KEYS rows of a head from `first` on, zeros from the `left`-th on
  __device__ __forceinline__ void next(unsigned char* dst, int first, int left, int head) const {
    const int64_t move = first * node + (int64_t)head * size, step = 8 * node;
    const T* f[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) f[g] = from[g] + move;
    uint32_t d = s32(dst) + to;
#pragma unroll 2
    for (int r = row; r < KEYS; r += 8, d += 1024) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g, f[g - 1] += step)
        if (there[g]) copy(d + g * (KEYS * 128), f[g], g, on[g] && r < left);
    }
  }
  // the same of a stretch that begins with `ns` rows from `from0` on and goes on at `from1`, from its `at`-th row on
  __device__ __forceinline__ void mixed(unsigned char* dst, int at, int ns, int from0, int from1, int left, int head) const {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (!there[g]) continue;
      const uint32_t d = s32(dst) + to + g * (KEYS * 128);
#pragma unroll 1
      for (int r = 0; r < KEYS; r += 8) {
        const int v = at + r + row, first = (v < ns ? from0 + v : from1 + v - ns) - row;
        copy(d + r * 128, from[g] + first * node + (int64_t)head * size, g, on[g] && r + row < left);
      }
    }
  }
  // the tile's own: `high` rows of one head after the other
  __device__ __forceinline__ void own(unsigned char* dst, int first, int left, int head, int high) const {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (!there[g]) continue;
      const uint32_t d = s32(dst) + to + g * (TILE_M * 128);
      const T* f = from[g] + first * node + (int64_t)head * size;
      int q = 0;
#pragma unroll 2
      for (int r = 0; r < TILE_M; r += 8) {
        copy(d + r * 128, f + q * node, g, on[g] && q + row < left);
        if ((q += 8) == high) q = 0, f += size;
      }
    }
  }
  __device__ __forceinline__ void copy(uint32_t d, const T* f, int g, bool in) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(in ? f : from[g]), "r"(in ? 16 : 0) : "memory");
  }
};

// The barrier has an arrival of this thread when its copies so far have landed.
__device__ __forceinline__ void land_at(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(s32(bar)) : "memory");
}

// The bits of [lo, hi) within 64
__device__ __forceinline__ uint64_t bits_of(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 64);
  return hi > lo ? (~uint64_t(0) >> (64 - (hi - lo))) << lo : 0;
}

// What a tile walks over: `ns` first nodes of the chain that its first row is in, from `from0` on, then [from1, to1), as one sequence.
struct Stretch {
  int from0, ns, from1, to1, total, steps;
};
template <int MODE> __device__ __forceinline__ Stretch stretch_of(const TcParams& p, int first, int last) {       // rows first to last
  const WindowParams& w = p.w;
  const int2 a = p.spans[first], b = p.spans[last];
  Stretch s;
  s.from0 = s.from1 = first;
  s.ns = 0;
  s.to1 = last + 1;
  if (MODE == COLUMNS) {
    if (a.y > a.x) s.from1 = max(a.x, first - w.after);
    if (b.y > b.x) s.to1 = !w.split && max(b.x, first) < b.x + w.sinks ? b.y : min(b.y, last + w.before + 1);
  } else {
    if (a.y > a.x) {
      s.from1 = max(a.x, first - w.before);
      s.from0 = a.x;
      s.ns = min(s.from1, a.x + w.sinks) - a.x;
    }
    if (b.y > b.x) s.to1 = min(b.y, last + w.after + 1);
  }
  s.total = s.ns + s.to1 - s.from1;
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

// A lane's row of results, with `more` where given, `f` times, to (n, components, heads, channels); whether all of it was finite.
template <int DP> __device__ __forceinline__ bool put_row(uint32_t sum, float f, bool on, void* out, int row, int head, const AttentionParams& p, const float* more = nullptr) {
  bool finite = true;
  const int values = p.comps * p.size;
  T* to = static_cast<T*>(out) + ((int64_t)row * p.comps * p.heads + head) * p.size;
#pragma unroll
  for (int h = 0; h < DP; h += 32) {
    if (h >= values) break;
    uint32_t r[32];
    tmem_issue32(sum + h, r);
    tmem_arrived32(r);
#pragma unroll
    for (int c = 0; c < 32; c += 8) {
      const int at = h + c;
      if (at >= values) break;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = __uint_as_float(r[c + j]) + (more ? more[at + j] : 0.f);
        finite = finite && is_finite(v[j]);
        v[j] *= f;
      }
      const int comp = at / p.size;
      if (on)
        *reinterpret_cast<uint4*>(to + (int64_t)comp * p.heads * p.size + at - comp * p.size) =
            make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7]));
    }
  }
  return finite;
}

template <int DP, int MODE> __global__ void __launch_bounds__(Form<DP, MODE>::THREADS, Form<DP, MODE>::CTAS) window_tc_kernel(const __grid_constant__ TcParams p) {
  using F = Form<DP, MODE>;
  constexpr int SLOTS = F::SLOTS, GROUPS = F::GROUPS, BUFFERS = F::BUFFERS;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *own = smem, *ring = own + F::OWN * F::OWN_BYTES;
  float* numbers = reinterpret_cast<float*>(ring + SLOTS * F::SLOT_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + SLOTS * F::SLOT_BYTES + F::NUMBERS);
  uint64_t *full = bars, *empty = full + SLOTS, *own_full = empty + SLOTS, *scores = own_full + 1, *weights = scores + BUFFERS, *freed = weights + BUFFERS, *done = freed + BUFFERS, *gathered = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gathered + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  static_assert((2 * SLOTS + 3 + 3 * BUFFERS) * 8 + 8 <= 512, "barriers");

  const WindowParams& w = p.w;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // A tile is `pack` heads that share their keys by `high` nodes: with fewer nodes, the walk over what any of them sees is shorter.
  const int pack = MODE == COLUMNS ? 1 : p.pack, high = TILE_M / pack, heads = (MODE == COLUMNS ? w.kv.heads : w.q.heads) / pack;
  const int head = (int)(blockIdx.x % (unsigned)heads) * pack, kv = MODE == COLUMNS ? head : head / w.group;
  const int first = (int)(blockIdx.x / (unsigned)heads) * high, last = min((int)w.q.n, first + high) - 1;
  const Stretch walk = stretch_of<MODE>(p, first, last);
  const int steps = walk.steps * (MODE == COLUMNS ? w.group : 1);
  const int values = w.q.comps * w.q.size, wide = (values + 15) / 16 * 16;

  if (tid == 0) {
    *abort_flag = (s32(smem) & 1023) != 0;                // the swizzle goes by addresses
    for (int s = 0; s < SLOTS; ++s) {
      bar_init(&full[s], !p.tma ? LOADERS : MODE == COLUMNS && !(s & 1) ? LOADERS + 1 : 1);
      bar_init(&empty[s], 1);
    }
    bar_init(own_full, p.tma ? 1 : LOADERS);
    for (int b = 0; b < BUFFERS; ++b) {
      bar_init(&scores[b], 1);
      bar_init(&weights[b], 4);
      bar_init(&freed[b], 1);
    }
    bar_init(done, 1);                                   // all products
    bar_init(gathered, LOADERS);                         // a mixed item where others are copied by TMA
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
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
    // copied by one thread (TMA); a stretch's first nodes, and all of other heads, by the threads: their copies arrive at the item's barrier when they have landed, and
    // the thread that issues the MMAs, which sees them all there, puts the fence between them and the tensor cores.  Copying by hand takes the warps
    // issue slots that the softmax wants (one chain of 32,781 nodes, 8 heads of 128 values, by hand and by TMA: HAND | TMA us).
    const int thread = tid - 32 * (F::SOFT + 2);
    const int left = last + 1 - first;
    const Copier<DP> even(MODE == FORWARD ? w.q.k : MODE == ROWS ? w.q.v : w.q.q, w.q, thread);
    const Copier<DP> odd(MODE == FORWARD ? w.q.v : MODE == ROWS ? w.q.k : w.q.g, w.q, thread);
    if (!p.tma) {
      Copier<DP>(MODE == COLUMNS ? w.q.k : w.q.q, w.q, thread).own(own, first, left, head, high);
      if (MODE != FORWARD) Copier<DP>(MODE == COLUMNS ? w.q.v : w.q.g, w.q, thread).own(own + F::OWN_BYTES, first, left, head, high);
      land_at(own_full);
    } else if (thread == 0) {
      bar_expect_tx(own_full, F::OWN * F::OWN_BYTES);
      for (int x = 0; x < F::OWN; ++x)
        for (int h = 0; h < pack; ++h)
          for (int g = 0; g < DP / 64; ++g)
            tma_load_3d(own + x * F::OWN_BYTES + g * (TILE_M * 128) + h * high * 128, &p.own[x], (head + h) * DP + g * 64, first, 0, own_full);
    }
    int at = 0, h = MODE == COLUMNS ? kv * w.group : kv;
    for (int item = 0; item < 2 * steps; ++item) {
      const int slot = item % SLOTS;
      const bool mixed = MODE != COLUMNS && at < walk.ns, numbered = MODE == COLUMNS && !(item & 1);
      if (!p.tma || mixed || numbered || thread == 0) {  // the others have nothing to do with tiles that are copied whole
        if (item >= SLOTS && !bar_wait(&empty[slot], (uint32_t)((item / SLOTS - 1) & 1), ab)) break;
        unsigned char* to = ring + slot * F::SLOT_BYTES;
        const Copier<DP>& x = item & 1 ? odd : even;
        if (mixed) {
          x.mixed(to, at, walk.ns, walk.from0, walk.from1, walk.total - at, h);
          if (p.tma) {                                   // one arrival for all, none of whom is an item ahead
            land_at(gathered);
            if (!bar_wait(gathered, (uint32_t)(item & 1), ab)) break;
            if (thread == 0) bar_arrive(&full[slot]);
          }
        } else if (!p.tma) {
          x.next(to, walk.from1 + at - walk.ns, walk.total - at, h);
        } else if (thread == 0) {
          bar_expect_tx(&full[slot], F::SLOT_BYTES);
          for (int g = 0; g < DP / 64; ++g) tma_load_3d(to + g * (KEYS * 128), &p.ring[item & 1], h * DP + g * 64, walk.from1 + at - walk.ns, 0, &full[slot]);
        }
        if (numbered) {
          const int i = walk.from1 + at + thread;
          const bool there = i < walk.to1;
          const int64_t from = there ? (int64_t)h * w.q.n + i : 0;
          float* num = numbers + slot / 2 * 3 * KEYS + thread;
          copy4(num, w.q.top + from, there);
          copy4(num + KEYS, w.q.inverse + from, there);
          copy4(num + 2 * KEYS, w.q.delta + from, there);
        }
        if (!p.tma || numbered) land_at(&full[slot]);
      }
      if ((item & 1) && (at += KEYS) >= walk.total) at = 0, ++h;         // COLUMNS: the next head
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= F::SOFT) {
    // ---------------- MMAs ----------------
    // One thread makes S and dP, another adds weighted rows up: each MMA costs its thread some ninety cycles whatever its size, and a step has up to 24.
    if (lane == 0) {
      const uint32_t to_scores = idesc_bf16(TILE_M, KEYS), to_sums = idesc_bf16(TILE_M, wide, false, true);
      const uint32_t own_at = s32(own), ring_at = s32(ring), sum = tmem + F::SUM_AT;
      const int ksteps = wide / 16;
      auto slot_at = [&](int item) { return ring_at + (uint32_t)(item % SLOTS) * F::SLOT_BYTES; };
      auto arrived = [&](int item) { return bar_wait(&full[item % SLOTS], (uint32_t)((item / SLOTS) & 1), ab); };
      auto fence = [] { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); };
      // scores of a step are free when the products that read them BUFFERS steps before are done
      auto free_again = [&](int j) { return j < BUFFERS || bar_wait(&freed[j % BUFFERS], (uint32_t)((j / BUFFERS - 1) & 1), ab); };
      auto weighted = [&](int j) { return bar_wait(&weights[j % BUFFERS], (uint32_t)((j / BUFFERS) & 1), ab); };
      // d (128 rows x 64) = rows of the tile times rows of the slot
      auto score = [&](uint32_t d, uint32_t a, uint32_t b) {
        const uint32_t a_lo = umma_lo(a), b_lo = umma_lo(b);
        umma_bf16<false>(d, a_lo, b_lo, to_scores);
#pragma unroll
        for (int k = 1; k < DP / 16; ++k)
          if (k < ksteps) umma_bf16<true>(d, a_lo + (k >> 2) * (TILE_M * 128 / 16) + (k & 3) * K_STEP, b_lo + (k >> 2) * (KEYS * 128 / 16) + (k & 3) * K_STEP, to_scores);
      };
      // d (128 rows x values) += weights in tensor memory times the slot
      auto add = [&](uint32_t d, uint32_t a, uint32_t b, bool more) {
        const uint32_t b_lo = umma_lo_rows(b, KEYS * 128);
        if (more) umma_bf16_ta<true>(d, a, b_lo, to_sums);
        else umma_bf16_ta<false>(d, a, b_lo, to_sums);
#pragma unroll
        for (int k = 1; k < KEYS / 16; ++k) umma_bf16_ta<true>(d, a + k * 8, b_lo + k * ROWS_STEP, to_sums);
      };
      bool ok = true;
      constexpr int S_ITEM = MODE == ROWS ? 1 : 0;
      auto make_s = [&](int j) {
        ok = ok && arrived(2 * j + S_ITEM) && free_again(j);
        if (!ok) return;
        fence();
        tc_fence_after();
        score(tmem + (j % BUFFERS) * F::BUFFER, own_at, slot_at(2 * j + S_ITEM));
        if (MODE == FORWARD) umma_commit(&empty[2 * j % SLOTS]);
      };
      // By rows, the place of dP is free when the softmax has read it.
      auto make_dp = [&](int j) {
        ok = ok && arrived(2 * j + 1 - S_ITEM) && (MODE == COLUMNS || j < BUFFERS || weighted(j - BUFFERS));
        if (!ok) return;
        fence();
        tc_fence_after();
        score(tmem + (j % BUFFERS) * F::BUFFER + KEYS, own_at + F::OWN_BYTES, slot_at(2 * j + 1 - S_ITEM));
        if (MODE == ROWS) umma_commit(&empty[2 * j % SLOTS]);
      };
      if (warp == F::SOFT) {
        ok = bar_wait(own_full, 0, ab);
        for (int j = 0; j < steps && ok; ++j) {
          if (MODE == ROWS) make_dp(j);
          make_s(j);
          if (MODE == COLUMNS) make_dp(j);
          if (ok) umma_commit(&scores[j % BUFFERS]);
        }
      } else {
        for (int j = 0; j < steps && ok; ++j) {
          const uint32_t d = tmem + (j % BUFFERS) * F::BUFFER;
          ok = arrived(2 * j + 1) && (MODE != COLUMNS || arrived(2 * j));
          if (!ok) break;
          fence();
          ok = weighted(j);
          if (!ok) break;
          tc_fence_after();
          add(sum, d, slot_at(2 * j + 1), j > 0);
          if (MODE == ROWS) add(sum, d + 32, slot_at(2 * j + 1), true);
          if (MODE == COLUMNS) {
            add(sum + DP, d + KEYS, slot_at(2 * j), j > 0);
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
    const int quarter = warp & 3, group = warp >> 2, place = quarter * 32 + lane, row = first + place % high, mine = head + place / high;       // its head
    const bool there = row <= last;
    const int2 span = there ? p.spans[row] : make_int2(0, 0);
    const bool on = span.y > span.x;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), sum_at = lanes + F::SUM_AT;
    const float unit = w.q.scale * LOG2E;
    // what the row sees: [lo, hi), and the first nodes [span.x, far)
    const int lo = !on ? 0 : max(span.x, row - (MODE == COLUMNS ? w.after : w.before));
    const int hi = !on ? 0 : MODE == COLUMNS ? (!w.split && row < span.x + w.sinks ? span.y : min(span.y, row + w.before + 1)) : min(span.y, row + w.after + 1);
    const int far = on && MODE != COLUMNS ? min(lo, span.x + w.sinks) : 0;
    bool ok = true;
    // as bits of the 64 from the stretch's `at`-th on; first nodes are before `from1`, or in the stretch behind it, or both
    auto seen = [&](int at) {
      const int shift = walk.from1 - walk.ns + at;
      uint64_t bits = bits_of(lo - shift, hi - shift);
      if (MODE != COLUMNS) {
        bits |= bits_of(max(span.x, walk.from1) - shift, far - shift);
        if (at < walk.ns && span.x < walk.from1) bits |= bits_of(span.x - walk.from0 - at, min(far - walk.from0, walk.ns) - at);
      }
      return bits;
    };
    if (MODE == FORWARD) {
      float base = -INFINITY, total = 0.f;
      for (int j = 0; j < steps; ++j) {
        const int b = j & 1;
        ok = bar_wait(&scores[b], (uint32_t)((j >> 1) & 1), ab);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint32_t s_at = lanes + b * F::BUFFER;
        uint32_t raw[2][32];
        tmem_issue32(s_at, raw[0]);
        tmem_issue32(s_at + 32, raw[1]);
        const uint64_t bits = seen(j * KEYS);
        tmem_arrived32(raw[0]);
        tmem_arrived32(raw[1]);
        if (!__all_sync(0xffffffffu, bits == ~uint64_t(0))) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t word = (uint32_t)(bits >> (32 * h));
#pragma unroll
            for (int c = 0; c < 32; ++c) raw[h][c] = (word >> c) & 1 ? raw[h][c] : 0xff800000u;
          }
        }
        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; ++c) most[c & 3] = fmaxf(most[c & 3], __uint_as_float(raw[c >> 5][c & 31]));
        const float now = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * unit;
        const bool higher = now > base + FAR || (base == -INFINITY && now > base);
        if (__any_sync(0xffffffffu, higher)) {           // another unit: what there is so far goes by it
          const float keep = !higher ? 1.f : base == -INFINITY ? 0.f : exp2_fast(base - now);
          total *= keep;
          if (higher) base = now;
          if (j > 0) {
            ok = bar_wait(&freed[(j - 1) & 1], (uint32_t)(((j - 1) >> 1) & 1), ab);
            if (!__all_sync(0xffffffffu, ok)) break;
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
        float add[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t out[32];
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float x = exp2_fast(fmaf(__uint_as_float(raw[c >> 5][c & 31]), unit, minus)), y = exp2_fast(fmaf(__uint_as_float(raw[c >> 5][(c & 31) + 1]), unit, minus));
          add[(c >> 1) & 3] += x + y;
          out[c >> 1] = two_bf16(x, y);
        }
        total += (add[0] + add[1]) + (add[2] + add[3]);
        tmem_put16(s_at, out);
        tmem_put16(s_at + 16, out + 16);
        tmem_stored();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&weights[b]);
      }
      ok = __all_sync(0xffffffffu, ok);
      if (ok && steps) ok = __all_sync(0xffffffffu, bar_wait(done, 0, ab));
      if (ok && steps) {
        tc_fence_after();
        const float inverse = 1.f / total;
        const bool finite = put_row<DP>(sum_at, inverse, on, w.q.out, row, mine, w.q);
        if (on && w.q.top) w.q.top[(int64_t)mine * w.q.n + row] = base, w.q.inverse[(int64_t)mine * w.q.n + row] = inverse;
        __syncwarp();
        for (unsigned bad = __ballot_sync(0xffffffffu, on && !finite); bad; bad &= bad - 1) {
          const int r = __ffs(bad) - 1;
          again_forward<T>(w, __shfl_sync(0xffffffffu, row, r), __shfl_sync(0xffffffffu, mine, r), __shfl_sync(0xffffffffu, span.x, r), __shfl_sync(0xffffffffu, span.y, r), lane);
        }
      }
    } else if (MODE == ROWS) {
      const int64_t number = (int64_t)mine * w.q.n + row;
      float top = INFINITY, inverse = 0.f, delta = 0.f;
      if (on) {
        top = w.q.top[number];
        inverse = w.q.inverse[number];
        const int64_t at = ((int64_t)row * w.q.comps * w.q.heads + mine) * w.q.size;
        for (int e = 0; e < values; e += 8) {
          const int comp = e / w.q.size;
          const int64_t place = at + (int64_t)comp * w.q.heads * w.q.size + e - comp * w.q.size;
          const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const T*>(w.q.out) + place), b = *reinterpret_cast<const uint4*>(static_cast<const T*>(w.q.g.p) + place);
          const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            delta = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), delta);
            delta = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), delta);
          }
        }
        if (group == 0) w.q.delta[number] = delta;
      }
      for (int j = group; j < steps; j += GROUPS) {
        const int b = j % BUFFERS;
        ok = bar_wait(&scores[b], (uint32_t)((j / BUFFERS) & 1), ab);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint64_t bits = seen(j * KEYS);
        const bool all = __all_sync(0xffffffffu, bits == ~uint64_t(0));
        uint32_t s[2][32], d[32], large[16], small[16];
        const uint32_t s_at = lanes + b * F::BUFFER;
        tmem_issue32(s_at, s[0]);
        tmem_issue32(s_at + 32, s[1]);
        tmem_arrived32(s[0]);
        tmem_arrived32(s[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tmem_issue32(s_at + KEYS + 32 * h, d);
          tmem_arrived32(d);
          const uint32_t word = (uint32_t)(bits >> (32 * h));
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              x[i] = exp2_fast(fmaf(__uint_as_float(s[h][c + i]), unit, -top)) * inverse * (__uint_as_float(d[c + i]) - delta);
              if (!all) x[i] = (word >> (c + i)) & 1 ? x[i] : 0.f;
            }
            const uint32_t two = two_bf16(x[0], x[1]);
            large[c / 2] = two;
            small[c / 2] = two_bf16(x[0] - __uint_as_float(two << 16), x[1] - __uint_as_float(two & 0xffff0000u));
          }
          tmem_put16(s_at + 16 * h, large);
          tmem_put16(s_at + 32 + 16 * h, small);
        }
        tmem_stored();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&weights[b]);
      }
      ok = __all_sync(0xffffffffu, ok);
      if (ok && steps) ok = __all_sync(0xffffffffu, bar_wait(done, 0, ab));
      if (ok && steps && group == 0) {
        tc_fence_after();
        const bool finite = put_row<DP>(sum_at, w.q.scale, on, w.q.dq, row, mine, w.q);

        __syncwarp();
        for (unsigned bad = __ballot_sync(0xffffffffu, on && !finite); bad; bad &= bad - 1) {
          const int r = __ffs(bad) - 1;
          again_rows<T>(w, __shfl_sync(0xffffffffu, row, r), __shfl_sync(0xffffffffu, mine, r), __shfl_sync(0xffffffffu, span.x, r), __shfl_sync(0xffffffffu, span.y, r), lane);
        }
      }
    } else {
      int at = group % walk.steps * KEYS;
      for (int j = group; j < steps; j += GROUPS) {
        const int b = j % BUFFERS, slot = 2 * j % SLOTS;
        ok = bar_wait(&full[slot], (uint32_t)((2 * j / SLOTS) & 1), ab) && bar_wait(&scores[b], (uint32_t)((j / BUFFERS) & 1), ab);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint64_t bits = seen(at);
        for (at += GROUPS * KEYS; at >= walk.steps * KEYS;) at -= walk.steps * KEYS;
        const bool all = __all_sync(0xffffffffu, bits == ~uint64_t(0));
        const float* num = numbers + slot / 2 * 3 * KEYS;
        const uint32_t s_at = lanes + b * F::BUFFER;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t s[32], d[32], pt[16], dst[16];
          tmem_issue32(s_at + 32 * h, s);
          tmem_issue32(s_at + KEYS + 32 * h, d);
          tmem_arrived32(s);
          tmem_arrived32(d);
          const uint32_t word = (uint32_t)(bits >> (32 * h));
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 top = *reinterpret_cast<const float4*>(num + 32 * h + c), inverse = *reinterpret_cast<const float4*>(num + KEYS + 32 * h + c),
                         delta = *reinterpret_cast<const float4*>(num + 2 * KEYS + 32 * h + c);
            const float tops[4] = {top.x, top.y, top.z, top.w}, inverses[4] = {inverse.x, inverse.y, inverse.z, inverse.w}, deltas[4] = {delta.x, delta.y, delta.z, delta.w};
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x[i] = exp2_fast(fmaf(__uint_as_float(s[c + i]), unit, -tops[i])) * inverses[i];
              y[i] = x[i] * (__uint_as_float(d[c + i]) - deltas[i]);
              if (!all) {
                const bool see = (word >> (c + i)) & 1;
                x[i] = see ? x[i] : 0.f;
                y[i] = see ? y[i] : 0.f;
              }
            }
            pt[c / 2] = two_bf16(x[0], x[1]);
            pt[c / 2 + 1] = two_bf16(x[2], x[3]);
            dst[c / 2] = two_bf16(y[0], y[1]);
            dst[c / 2 + 1] = two_bf16(y[2], y[3]);
          }
          tmem_put16(s_at + 16 * h, pt);
          tmem_put16(s_at + KEYS + 16 * h, dst);
        }
        tmem_stored();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&weights[b]);
      }
      ok = __all_sync(0xffffffffu, ok);
      if (ok && steps) ok = __all_sync(0xffffffffu, bar_wait(done, 0, ab));
      if (ok && steps) {                                  // of two groups, one stores each sum
        tc_fence_after();
        bool finite = true;
        const float* more = on ? far_of(w, row, kv, span.x, span.y) : nullptr;
        if (group == 0) finite = put_row<DP>(sum_at, 1.f, on, w.kv.dv, row, kv, w.kv, more ? more + FAR_ROWS * values : nullptr);
        if (group == GROUPS - 1) finite = put_row<DP>(sum_at + DP, w.q.scale, on, w.kv.dk, row, kv, w.kv, more) && finite;
        __syncwarp();
        for (unsigned bad = __ballot_sync(0xffffffffu, on && !finite); bad; bad &= bad - 1) {
          const int r = __ffs(bad) - 1;
          again_columns<T>(w, row - lane + r, kv, __shfl_sync(0xffffffffu, span.x, r), __shfl_sync(0xffffffffu, span.y, r), lane, group == 0, group == GROUPS - 1);
        }
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
  const int64_t grid = MODE == COLUMNS ? ceil_div(p.w.q.n, TILE_M) * p.w.kv.heads : ceil_div(p.w.q.n, TILE_M / p.pack) * (p.w.q.heads / p.pack);
  if (grid > INT32_MAX) return fail(EQT_ERR_UNSUPPORTED, "window_attention: %lld tiles are more than one launch takes", (long long)grid);
  TcParams t = p;
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
             (rc = map(&t.ring[MODE == ROWS], q.k, kv_heads, KEYS)) || (rc = map(&t.ring[MODE == FORWARD], q.v, kv_heads, KEYS)));
    }
    if (rc) return rc;
  }
  auto kernel = window_tc_kernel<DP, MODE>;
  static std::atomic<uint64_t> allowed{0};
  if (int rc = allow_shared_once(kernel, F::bytes(), allowed)) return rc;
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
  if (int rc = narrow ? launch<64, ROWS>(p, s) : launch<128, ROWS>(p, s)) return rc;
  if (p.w.split)
    if (int rc = far_bf16(p.w, s)) return rc;
  return narrow ? launch<64, COLUMNS>(p, s) : launch<128, COLUMNS>(p, s);
}
