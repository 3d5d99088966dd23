#include "residual_norm_impl.h"

MG_DEFINE_RESIDUAL_NORM(f16_t)
