// Attention within windows by tiles of one chain, float32.
#include "window_tiles.cuh"

int eqt::window::tiles_forward_f32(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s) {
  return by_values<float, FORWARD>(p, tile_rows, num_tiles, s);
}
int eqt::window::tiles_backward_f32(const WindowParams& p, int tile_rows, int64_t num_tiles, cudaStream_t s) {
  return tiles_backward<float>(p, tile_rows, num_tiles, s);
}
