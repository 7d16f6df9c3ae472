// Norms over rows of fp16 (norm_rows.h).
#include "norm_rows.h"

namespace tvae {
int norm_launch_f16(const NormCall& c, int r_dtype, bool bwd, hipStream_t s) {
    return r_dtype == TVAE_F32 ? norm_launch<f16, float>(c, bwd, s) : norm_launch<f16, f16>(c, bwd, s);
}
}  // namespace tvae
