// Chunked selective scan of float16 operands (pe_scan_chunk.h).
#include "pe_scan_chunk.h"

namespace pe {
namespace ssm {

int chunks_f16(const ChunkArgs* g, int nt, int waves, bool main, hipStream_t stream) {
    return chunks<F16>(g, nt, waves, main, stream);
}

}  // namespace ssm
}  // namespace pe
