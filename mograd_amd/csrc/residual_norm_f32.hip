#include "residual_norm_impl.h"

MG_DEFINE_RESIDUAL_NORM(float)
