// Gradients of f32 Linear layers from an input in 8 bits.
#include "linear_act8_dw.h"
namespace mg {
template int launch_linear_act8<float>(const Act8Dw<float>&, const Gemm16Problem<float>*, int, int64_t, int64_t, hipStream_t);
}  // namespace mg
