// Chunked selective scan of bfloat16 operands (pe_scan_chunk.h).
#include "pe_scan_chunk.h"

namespace pe {
namespace ssm {

void launch_chunks_bf16(const ChunkArgs& g, int nt, int waves, bool main, hipStream_t stream) {
    switch (nt) {
        case 32: return launch_chunks<BF16, 32, 64>(g, waves, main, stream);
        case 64: return launch_chunks<BF16, 64, 64>(g, waves, main, stream);
        case 128: return launch_chunks<BF16, 128, 64>(g, waves, main, stream);
        default: return launch_chunks<BF16, 256, 32>(g, waves, main, stream);
    }
}

}  // namespace ssm
}  // namespace pe
