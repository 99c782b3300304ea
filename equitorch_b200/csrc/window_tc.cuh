// The tiles of 128 nodes on the 5th-generation tensor cores (window_tc.cu).
#pragma once

#include "window.cuh"

namespace eqt {
namespace window {

struct TcParams {
  WindowParams w;
  const int2* spans;         // [node]: its chain
  int* status;
};
int spans(const int64_t* ptr, int64_t chains, int2* out, int64_t n, cudaStream_t s);
int tc_forward(const TcParams& p, cudaStream_t s);
int tc_backward(const TcParams& p, cudaStream_t s);

}  // namespace window
}  // namespace eqt
