// Chunked selective scan of bfloat16 operands (pe_scan_chunk.h).
#include "pe_scan_chunk.h"

namespace pe {
namespace ssm {

int chunks_bf16(const ChunkArgs* g, int nt, int waves, bool main, hipStream_t stream) {
    return chunks<BF16>(g, nt, waves, main, stream);
}

}  // namespace ssm
}  // namespace pe
