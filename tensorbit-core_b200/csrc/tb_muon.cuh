// Orthogonalised updates (tb_muon.cu).
#pragma once

#include <cuda_runtime.h>

namespace tb {
namespace muon {

// Error code recorded by these kernels on this device since the previous call
// (0 none, 1 a bounded wait expired, -1 it could not be read); resets it.
int take_error(cudaStream_t st);

}  // namespace muon
}  // namespace tb
