// Gated linear layer on tensor cores: the float32 kernels.
#include "gated_tc.cuh"

int eqt::gated::tensor_forward_f32(const GatedArgs& p, cudaStream_t s) { return launch_dual<float, FORWARD>(p, s); }
int eqt::gated::tensor_backward_f32(const GatedArgs& p, cudaStream_t s) { return backward<float>(p, s); }
int eqt::gated::tensor_form_f32(const GatedArgs& p, int product) { return shape_of<float>(p, product); }
