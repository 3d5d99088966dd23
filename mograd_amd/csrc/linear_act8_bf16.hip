// Gradients of bf16 Linear layers from an input in 8 bits.
#include "linear_act8_dw.h"
namespace mg {
template int launch_linear_act8<bf16_t>(const Act8Dw<bf16_t>&, const Gemm16Problem<bf16_t>*, int, int64_t, int64_t, hipStream_t);
}  // namespace mg
