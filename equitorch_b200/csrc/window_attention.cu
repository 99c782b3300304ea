// Attention within windows of packed chains: the C entry points.
#include <algorithm>

#include "window_tc.cuh"

namespace eqt {
namespace window {
namespace {

size_t up(size_t b) { return (b + 1023) / 1024 * 1024; }

int check(const eqt_window_attention_args* a) {
  if (!a) return fail(EQT_ERR_BAD_ARGUMENT, "window_attention: NULL pointer");
  if (a->dtype != EQT_F32 && a->dtype != EQT_BF16) return fail(EQT_ERR_BAD_ARGUMENT, "window_attention: unknown dtype %d", a->dtype);
  if (a->n < 0 || a->num_graphs < 0 || a->num_tiles < 0 || a->before < 0 || a->after < 0 || a->sinks < 0 || a->heads < 1 || a->kv_heads < 1 || a->comps < 1 ||
      a->head_channels < 1 || a->heads % a->kv_heads || (a->tile_rows != 16 && a->tile_rows != 32 && a->tile_rows != 64))
    return fail(EQT_ERR_BAD_ARGUMENT, "window_attention: sizes");
  if (a->n >= 1 << 30 || (int64_t)a->comps * a->head_channels > 128 || a->heads > 65535)
    return fail(EQT_ERR_UNSUPPORTED, "window_attention: fewer than 2^30 nodes, 128 values a head and 65535 heads");
  return EQT_OK;
}

// What all kernels take.  Windows reach no further than the longest chain, so a place and a reach, both below 2^30, add up in 32 bits.
WindowParams params(const eqt_window_attention_args& a) {
  WindowParams p{};
  const int64_t reach = std::min<int64_t>(std::max<int64_t>(a.longest, 1), a.n);
  p.before = (int)std::min(a.before, reach), p.after = (int)std::min(a.after, reach), p.sinks = (int)std::min(a.sinks, reach);
  p.group = a.heads / a.kv_heads;
  AttentionParams& q = p.q;
  const int64_t width = (int64_t)a.heads * a.head_channels;
  q.q = {a.q, a.q_node, a.q_comp}, q.k = {a.k, a.k_node, a.k_comp}, q.v = {a.v, a.v_node, a.v_comp}, q.g = {a.grad, a.comps * width, width};
  q.out = a.out, q.dq = a.dq, q.dk = a.dk, q.dv = a.dv, q.top = a.stats, q.inverse = a.stats ? a.stats + a.heads * a.n : nullptr, q.delta = nullptr;
  q.tiles = reinterpret_cast<const int4*>(a.tiles), q.n = a.n, q.heads = a.heads, q.comps = a.comps, q.size = a.head_channels, q.scale = a.scale;
  const int v = a.dtype == EQT_F32 ? 4 : 8;
  const int64_t strides = a.q_node | a.q_comp | a.k_node | a.k_comp | a.v_node | a.v_comp;
  uintptr_t bits = 0;
  for (const void* x : {a.q, a.k, a.v, a.grad, (const void*)a.out, (const void*)a.rest, (const void*)a.dq, (const void*)a.dk, (const void*)a.dv}) bits |= reinterpret_cast<uintptr_t>(x);
  q.vec = bits % 16 == 0 && strides % v == 0 && a.head_channels % v == 0;
  p.kv = q;
  p.kv.heads = a.kv_heads;
  // A tile of keys that holds a chain's first nodes would walk to the chain's end, alone, while the others are done (one chain of 32,781 nodes, 8 heads of 128
  // values, window of 1024: by columns 876 us; with these queries apart 473 and 62 for them).  Two launches more, so not for batches whose chains are all walked in a few steps (240
  // chains of 50 to 500 nodes, window of 64 on both sides: 217 us walked, 164 and 61 apart), nor for such chains beside a longer one (`apart`), which would take scratch each;
  // and not for so many first nodes that tiles are full of them.
  p.ptr = a.ptr, p.chains = a.num_graphs, p.rest = a.dtype == EQT_BF16 ? a.rest : nullptr;
  p.split = p.sinks > 0 && p.sinks <= MOST_SPLIT_SINKS && a.longest - p.before > 2 * FAR_BLOCK;
  p.apart = p.split ? far_length(p) : INT32_MAX;
  if (a.dtype == EQT_BF16) {
    const int64_t window = std::min<int64_t>((int64_t)p.before + p.after + 1, reach);
    p.folds_rows = std::min<int64_t>(window + p.sinks, reach) > attention::FOLD;
    // a first node is seen to its chain's end, or apart to the length from which chains are
    const int64_t far = !p.sinks ? 0 : p.split ? std::min<int64_t>(p.apart, reach) : reach;
    p.folds_columns = p.group * std::max(window, far) > attention::FOLD;
  }
  return p;
}

// Tiles of 128 nodes on the tensor cores: bfloat16 whose pieces lie on 16-byte boundaries, and a positive scale, by which the greatest product is the greatest
// score.
bool on_tensor_cores(const eqt_window_attention_args& a) {
  if (a.dtype != EQT_BF16 || !(a.scale > 0.f)) return false;
  const int64_t strides = a.q_node | a.q_comp | a.k_node | a.k_comp | a.v_node | a.v_comp;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.rest) |
                         reinterpret_cast<uintptr_t>(a.grad) | reinterpret_cast<uintptr_t>(a.dq) | reinterpret_cast<uintptr_t>(a.dk) | reinterpret_cast<uintptr_t>(a.dv);
  return bits % 16 == 0 && strides % 8 == 0 && a.head_channels % 8 == 0;
}

// Scratch: the nodes' chains, and for the backward pass the deltas, the inverse sums and what far queries give first nodes.
int64_t spans_bytes(const eqt_window_attention_args& a) { return a.dtype == EQT_BF16 ? (int64_t)up((size_t)a.n * sizeof(int2)) : 0; }
int64_t delta_bytes(const eqt_window_attention_args& a) { return (int64_t)up((size_t)a.heads * a.n * 4); }
int64_t scratch_bytes(const eqt_window_attention_args& a, bool backward) {
  if (!backward) return spans_bytes(a);
  const WindowParams p = params(a);
  return spans_bytes(a) + 2 * delta_bytes(a) + (p.split ? far_pairs(p) * a.kv_heads * far_groups(p) * 2 * FAR_ROWS * a.comps * a.head_channels * 4 : 0);
}
int check_scratch(const eqt_window_attention_args& a, bool backward) {
  const int64_t need = scratch_bytes(a, backward);
  if (need && (!a.scratch || a.scratch_bytes < need))
    return fail(EQT_ERR_BAD_ARGUMENT, "window_attention: %lld bytes of scratch given, %lld needed", (long long)a.scratch_bytes, (long long)need);
  return reinterpret_cast<uintptr_t>(a.scratch) % 16 ? fail(EQT_ERR_BAD_ARGUMENT, "window_attention: scratch must start on a 16-byte boundary") : EQT_OK;
}
int check_tiles(const eqt_window_attention_args& a, const WindowParams& p) {
  if (p.folds_rows && a.tile_rows != 64)
    return fail(EQT_ERR_UNSUPPORTED, "window_attention: bfloat16 windows of more than %d nodes need tiles of 64 rows, got %d", attention::FOLD, a.tile_rows);
  return EQT_OK;
}
int tensor_params(TcParams& t, const eqt_window_attention_args& a, const WindowParams& p, cudaStream_t s) {
  if (!a.ptr || !a.status) return fail(EQT_ERR_BAD_ARGUMENT, "window_attention: NULL pointer");
  t.w = p;
  t.spans = static_cast<const int2*>(a.scratch);
  t.status = a.status;
  t.pack = p.group % 8 == 0 ? 8 : p.group % 4 == 0 ? 4 : p.group % 2 == 0 ? 2 : 1;
  return spans(a.ptr, a.num_graphs, static_cast<int2*>(a.scratch), a.n, s);
}

}  // namespace
}  // namespace window
}  // namespace eqt

using namespace eqt;
using namespace eqt::window;

extern "C" int64_t eqt_window_attention_scratch(const eqt_window_attention_args* a, int32_t backward) {
  if (check(a)) return 0;
  return scratch_bytes(*a, backward != 0);
}

extern "C" int32_t eqt_window_attention_form(const eqt_window_attention_args* a) {
  if (check(a)) return -1;
  return on_tensor_cores(*a);
}

extern "C" int eqt_window_attention_forward(const eqt_window_attention_args* args, void* stream) {
  if (int rc = check(args)) return rc;
  const eqt_window_attention_args& a = *args;
  if (a.n == 0 || a.num_tiles == 0) return EQT_OK;
  if (!a.q || !a.k || !a.v || !a.out || !a.tiles || (a.dtype == EQT_BF16 && a.stats && !a.rest)) return fail(EQT_ERR_BAD_ARGUMENT, "window_attention: NULL pointer");
  if (int rc = check_scratch(a, false)) return rc;
  const WindowParams p = params(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (on_tensor_cores(a)) {
    TcParams t;
    if (int rc = tensor_params(t, a, p, s)) return rc;
    return tc_forward(t, s);
  }
  if (int rc = check_tiles(a, p)) return rc;
  return a.dtype == EQT_F32 ? tiles_forward_f32(p, a.tile_rows, a.num_tiles, s) : tiles_forward_bf16(p, a.tile_rows, a.num_tiles, s);
}

extern "C" int eqt_window_attention_backward(const eqt_window_attention_args* args, void* stream) {
  if (int rc = check(args)) return rc;
  const eqt_window_attention_args& a = *args;
  if (a.n == 0 || a.num_tiles == 0) return EQT_OK;
  if (!a.q || !a.k || !a.v || !a.grad || !a.out || (a.dtype == EQT_BF16 && !a.rest) || !a.stats || !a.dq || !a.dk || !a.dv || !a.tiles) return fail(EQT_ERR_BAD_ARGUMENT, "window_attention backward: NULL pointer");
  if (int rc = check_scratch(a, true)) return rc;
  WindowParams p = params(a);
  if (p.split && !a.ptr) return fail(EQT_ERR_BAD_ARGUMENT, "window_attention backward: NULL pointer");
  unsigned char* base = static_cast<unsigned char*>(a.scratch) + spans_bytes(a);
  p.q.delta = p.kv.delta = reinterpret_cast<float*>(base);
  p.inverse = reinterpret_cast<float*>(base + delta_bytes(a));
  p.far = reinterpret_cast<float*>(base + 2 * delta_bytes(a));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (on_tensor_cores(a)) {
    TcParams t;
    if (int rc = tensor_params(t, a, p, s)) return rc;
    return tc_backward(t, s);
  }
  if (int rc = check_tiles(a, p)) return rc;
  return a.dtype == EQT_F32 ? tiles_backward_f32(p, a.tile_rows, a.num_tiles, s) : tiles_backward_bf16(p, a.tile_rows, a.num_tiles, s);
}
