#include "common.cuh"
using namespace eqt;
extern "C" int64_t eqt_window_attention_scratch(const eqt_window_attention_args*, int32_t) { return 0; }
extern "C" int32_t eqt_window_attention_form(const eqt_window_attention_args*) { return 0; }
extern "C" int eqt_window_attention_forward(const eqt_window_attention_args*, void*) { return fail(EQT_ERR_UNSUPPORTED, "window attention: no kernel yet"); }
extern "C" int eqt_window_attention_backward(const eqt_window_attention_args*, void*) { return fail(EQT_ERR_UNSUPPORTED, "window attention: no kernel yet"); }
