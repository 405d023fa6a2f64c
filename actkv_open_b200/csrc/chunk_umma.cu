// Chunk attention on the sm_100a tensor cores: not there yet, every call takes chunk_simt.cu.
#include "kernels.cuh"

namespace actkv {

size_t chunk_workspace_bytes(int) { return 256; }

bool chunk_umma_supported(const ChunkArgs&, int, const char** why) {
  *why = "not built";
  return false;
}

cudaError_t launch_chunk_umma(const ChunkArgs&, int, cudaStream_t, const char**) { return cudaErrorNotSupported; }

}  // namespace actkv
