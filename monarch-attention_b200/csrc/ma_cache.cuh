// Paged key-value cache shared by the store / read-back kernels (ma_cache.cu)
// and the one-token attention (ma_decode.cu): the kernels' view of it, page
// look-up with bounds checks, and element conversion.
#pragma once

#include <string>

#include "ma_common.cuh"

namespace ma {

// How an element of the pages is held.
enum class Elem { f32, f16, bf16, e4m3, i8 };

template <Elem K> struct ElemT;
template <> struct ElemT<Elem::f32> { using type = float; };
template <> struct ElemT<Elem::f16> { using type = __half; };
template <> struct ElemT<Elem::bf16> { using type = __nv_bfloat16; };
template <> struct ElemT<Elem::e4m3> { using type = __nv_fp8_e4m3; };
template <> struct ElemT<Elem::i8> { using type = int8_t; };

template <Elem K> constexpr bool is_coded = K == Elem::e4m3 || K == Elem::i8;

template <> __device__ __forceinline__ float to_f<int8_t>(int8_t x) { return static_cast<float>(x); }

constexpr int kMaxCacheDim = 256;

// What the kernels need of an ma_kv_cache.  Offsets are element counts and
// always computed in 64 bits: a cache may hold more than 2^31 elements.
struct CacheView {
  char* pages[2];      // k, v
  float* scale[2];
  int64_t stride[2][3];   // page, head, token
  int64_t sstride[2][3];
  const int32_t* table;
  int64_t tstride[2];
  int E, Hk, D, num_pages, page_size, max_pages;
  int capacity;  // max_pages * page_size
  uint32_t page_mul, page_shift;  // position / page_size without a division
  uint32_t* status;
  uint32_t* status_host;
};

__device__ __forceinline__ void cache_fail(const CacheView& c, uint32_t bit) {
  atomicOr(c.status, bit);
  if (c.status_host) *reinterpret_cast<volatile uint32_t*>(c.status_host) = bit;
}

// The page of a sequence that position pos (0 <= pos < 2^31) lies in.  With s =
// ceil(log2 page_size) and m = ceil(2^(31 + s) / page_size), floor(pos m /
// 2^(31 + s)) is exact: m exceeds the quotient by less than 2^s / page_size
// in units of 2^(31 + s), which times pos stays below 1 / page_size.
__device__ __forceinline__ int page_index(const CacheView& c, int pos) {
  return c.page_size == 1 ? pos : (int)(__umulhi((uint32_t)pos, c.page_mul) >> c.page_shift);
}
inline void page_divisor(CacheView& c) {
  int s = 0;
  while ((int64_t{1} << s) < c.page_size) ++s;
  c.page_mul = s == 0 ? 0 : (uint32_t)(((uint64_t{1} << (31 + s)) + c.page_size - 1) / c.page_size);
  c.page_shift = s == 0 ? 0 : s - 1;
}

// Tokens of sequence e that its pages can hold, at most `len`.
__device__ __forceinline__ int cache_length(const CacheView& c, int len) {
  if (len < 0 || len > c.capacity) {
    cache_fail(c, MA_STATUS_BAD_LENGTH);
    return len < 0 ? 0 : c.capacity;
  }
  return len;
}

// The page that holds position pos (0 <= pos < capacity) of sequence e, or -1
// where the table names none, and the position's slot in it.
__device__ __forceinline__ int cache_page(const CacheView& c, int e, int pos, int& slot) {
  const int i = page_index(c, pos);
  slot = pos - i * c.page_size;
  const int page = __ldg(c.table + (int64_t)e * c.tstride[0] + (int64_t)i * c.tstride[1]);
  if (page < 0 || page >= c.num_pages) {
    cache_fail(c, MA_STATUS_BAD_PAGE);
    return -1;
  }
  return page;
}

// Kernels that follow each other on a stream: one started with launch_early() gets
// its place on the SMs while the one before still runs (every kernel here lets
// it at its own start), and waits in wait_for_earlier() until all its results are
// there; nothing may be read or written before.
__device__ __forceinline__ void wait_for_earlier() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                         const A&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Host side (ma_cache.cu): checks an ma_kv_cache and fills the view; MA_OK or
// an error code with its detail.
int cache_view(const ma_kv_cache& c, CacheView* v, std::string* detail);
Elem cache_elem(int dtype);
// Whether the rows of pages t (0 k, 1 v) start on `bytes`-byte boundaries.
bool cache_rows_aligned(const ma_kv_cache& c, int t, int bytes);
int cache_elem_bytes(int dtype);

}  // namespace ma
