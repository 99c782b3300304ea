// The tiles of 128 nodes on the 5th-generation tensor cores (window_tc.cu).
#pragma once

#include "tc_bf16.cuh"
#include "window.cuh"

namespace eqt {
namespace window {

struct alignas(64) TcParams {
  CUtensorMap own[2], ring[2], eight[2];   // where `tma`: of the tile's operands, of the others in the order of their use, and of eight rows of these
  WindowParams w;
  const int2* spans;         // [node]: its chain
  unsigned tiles;
  int* status;
  int pack;                  // heads of a tile, by rows: a power of two of at most eight that divides the heads that share keys
  int tma;                   // a head's rows are one or two whole lines of 64 values: tiles are copied by the tensor memory accelerator
};
int spans(const int64_t* ptr, int64_t chains, int2* out, int64_t n, cudaStream_t s);
int tc_forward(const TcParams& p, cudaStream_t s);
int tc_backward(const TcParams& p, cudaStream_t s);

}  // namespace window
}  // namespace eqt
