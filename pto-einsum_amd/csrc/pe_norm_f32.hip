// Norms and rows in 8 bits of float32 values.
#include "pe_norm.h"

namespace pe {
namespace rows {

int norm_launch_f32(Op op, bool q8, bool, const NormArgs& a, hipStream_t stream) {
    return launch_type<F32>(op, q8, false, a, stream);
}

}  // namespace rows
}  // namespace pe
