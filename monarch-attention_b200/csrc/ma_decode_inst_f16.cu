// One-token attention for 16-bit queries: kernels for fp16 pages.
#include "ma_decode_mma.cuh"

namespace ma {

cudaError_t run_decode_f16(const DecodeArgs& a, cudaStream_t st) {
  return launch_pages<Elem::f16>(a, st);
}

}  // namespace ma
