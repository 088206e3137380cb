#include "decay.cuh"
namespace tbl { namespace stack {
bool decay_chunk_supported(const tbl_decay_mixer&) { return false; }
size_t decay_chunk_workspace(const tbl_decay_mixer&, int, int) { return 0; }
int launch_decay_chunks(const tbl_decay_mixer&, const DecayParams&, void*, cudaStream_t) { return TBL_ERR_UNSUPPORTED; }
} }
