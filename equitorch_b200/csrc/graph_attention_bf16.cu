// Attention within packed graphs: the bfloat16 kernels.
#include "graph_attention.cuh"

int eqt::attention::launch_bf16(Pass pass, const AttentionParams& p, int64_t tiles, int tile_rows, bool geo, cudaStream_t s) {
  return launch_width<__nv_bfloat16>(pass, p, tiles, tile_rows, geo, s);
}
