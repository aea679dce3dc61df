// One-token attention for 16-bit queries: kernels for bf16 pages.
#include "ma_decode_mma.cuh"

namespace ma {

cudaError_t run_decode_bf16(const DecodeArgs& a, cudaStream_t st) {
  return launch_pages<Elem::bf16>(a, st);
}

}  // namespace ma
