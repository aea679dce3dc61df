// One-token attention for 16-bit queries: kernels for e4m3 pages.
#include "ma_decode_mma.cuh"

namespace ma {

cudaError_t run_decode_e4m3(const DecodeArgs& a, cudaStream_t st) {
  return launch_pages<Elem::e4m3>(a, st);
}

}  // namespace ma
