// Norms and rows in 8 bits of bfloat16 values.
#include "pe_norm.h"

namespace pe {
namespace rows {

int norm_launch_bf16(Op op, bool q8, bool wide, const NormArgs& a, hipStream_t stream) {
    return launch_type<BF16>(op, q8, wide, a, stream);
}

}  // namespace rows
}  // namespace pe
