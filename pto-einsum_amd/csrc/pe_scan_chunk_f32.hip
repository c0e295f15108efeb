// Chunked selective scan of float32 operands (pe_scan_chunk.h).
#include "pe_scan_chunk.h"

namespace pe {
namespace ssm {

int chunks_f32(const ChunkArgs* g, int nt, int waves, bool main, hipStream_t stream) {
    return chunks<F32>(g, nt, waves, main, stream);
}

}  // namespace ssm
}  // namespace pe
