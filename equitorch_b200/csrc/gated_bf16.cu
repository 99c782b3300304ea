// Gated linear layer on tensor cores: the bfloat16 kernels.
#include "gated_tc.cuh"

int eqt::gated::tensor_forward_bf16(const GatedArgs& p, cudaStream_t s) { return launch_dual<__nv_bfloat16, FORWARD>(p, s); }
int eqt::gated::tensor_backward_bf16(const GatedArgs& p, cudaStream_t s) { return backward<__nv_bfloat16>(p, s); }
int eqt::gated::tensor_form_bf16(const GatedArgs& p, int product) { return shape_of<__nv_bfloat16>(p, product); }
