// The paged chunk kernel over pages of 8 bits.
#include "paged_chunk.hpp"

namespace cea {

int launch_paged_chunk8(const ChunkParams& c, hipStream_t st) { return launch_pages<true>(c, st); }

}  // namespace cea
