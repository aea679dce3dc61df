// One-token attention for 16-bit queries: kernels for int8 pages.
#include "ma_decode_mma.cuh"

namespace ma {

cudaError_t run_decode_i8(const DecodeArgs& a, cudaStream_t st) {
  return launch_pages<Elem::i8>(a, st);
}

}  // namespace ma
