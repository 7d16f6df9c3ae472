// Norms over rows of fp32 (norm_rows.h).
#include "norm_rows.h"

namespace tvae {
int norm_launch_f32(const NormCall& c, bool bwd, hipStream_t s) { return norm_launch<float, float>(c, bwd, s); }
}  // namespace tvae
