// Chunked selective scan of float16 operands (pe_scan_chunk.h).
#include "pe_scan_chunk.h"

namespace pe {
namespace ssm {

void launch_chunks_f16(const ChunkArgs& g, int nt, int waves, bool main, hipStream_t stream) {
    switch (nt) {
        case 32: return launch_chunks<F16, 32, 64>(g, waves, main, stream);
        case 64: return launch_chunks<F16, 64, 64>(g, waves, main, stream);
        case 128: return launch_chunks<F16, 128, 64>(g, waves, main, stream);
        default: return launch_chunks<F16, 256, 32>(g, waves, main, stream);
    }
}

}  // namespace ssm
}  // namespace pe
