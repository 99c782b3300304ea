// Attention within windows by tiles of one chain, bfloat16.
#include "window_tiles.cuh"

int eqt::window::tiles_forward_bf16(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s) {
  return by_values<__nv_bfloat16, FORWARD>(p, tile_rows, num_tiles, s);
}
int eqt::window::tiles_backward_bf16(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s) {
  return tiles_backward<__nv_bfloat16>(p, tile_rows, num_tiles, s);
}
int eqt::window::far_bf16(const WindowParams& p, cudaStream_t s) { return far<__nv_bfloat16>(p, s); }
