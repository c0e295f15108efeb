// Chunked selective scan of float32 operands (pe_scan_chunk.h).
#include "pe_scan_chunk.h"

namespace pe {
namespace ssm {

void launch_chunks_f32(const ChunkArgs& g, int nt, int waves, bool main, hipStream_t stream) {
    switch (nt) {
        case 32: return launch_chunks<F32, 32, 32>(g, waves, main, stream);
        case 64: return launch_chunks<F32, 64, 32>(g, waves, main, stream);
        case 128: return launch_chunks<F32, 128, 32>(g, waves, main, stream);
        default: return launch_chunks<F32, 256, 32>(g, waves, main, stream);
    }
}

}  // namespace ssm
}  // namespace pe
