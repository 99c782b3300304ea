// Attention within packed graphs: the float32 kernels.
#include "graph_attention.cuh"

int eqt::attention::launch_f32(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s) {
  return launch_width<float>(pass, p, tiles, tile_rows, geo, s);
}
