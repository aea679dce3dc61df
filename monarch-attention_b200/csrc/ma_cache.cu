// Paged key-value cache: new tokens stored (quantised as they are written)
// and sequences read back as dense tensors.  C entries ma_cache_write and
// ma_cache_read (include/ma_api.h); the reference's decoder keeps dense
// tensors instead (bart/model.py:67-152).
//
// Store:  scale = max(max_d |x_d|, 1e-12) * (1 / top),  code_d = rn(x_d / scale)
// Read:   x_d = code_d * scale, zero at and behind a sequence's length
//
// Both kernels touch every byte once and compute a few operations a value, so
// HBM bounds them.  A row of D values (one token, head, and k or v) is taken
// by 4 to 32 neighbouring lanes with 8 values each: 16 bytes of a 16-bit row,
// 8 of an 8-bit one; the row's maximum is a shuffle over these lanes.
#include <math.h>

#include "ma_cache.cuh"

namespace ma {

void set_error_detail(const std::string& detail);  // ma_api.cu
void set_launch_count(int n);
int host_word_check(const void* ptr);

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;  // values a lane
constexpr float kAmaxMin = 1e-12f;

// Lanes that share a row of D values: a power of two so that the row's
// maximum is a shuffle reduction.
int row_lanes(int D) {
  int n = 1;
  while (n * kPer < D) n *= 2;
  return n;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* dst, bool vec, int valid, const float (&x)[kPer]) {
  if (vec && valid >= kPer) {
    union {
      uint4 v[sizeof(T) * kPer / 16];
      T t[kPer];
    } u;
#pragma unroll
    for (int i = 0; i < kPer; ++i) u.t[i] = from_f<T>(x[i]);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * kPer / 16); ++i) reinterpret_cast<uint4*>(dst)[i] = u.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < valid) dst[i] = from_f<T>(x[i]);
  }
}

struct WriteArgs {
  CacheView c;
  const char* x[2];
  int64_t xs[2][4];
  const int32_t* start;
  const int32_t* count;
  int T, lanes, rows;  // rows = 2 * T * Hk of one sequence
  bool xvec[2], pvec[2];
};

template <typename X, Elem K>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const WriteArgs a) {
  const CacheView& c = a.c;
  const int sub = threadIdx.x % a.lanes;
  const int row = blockIdx.x * (kThreads / a.lanes) + threadIdx.x / a.lanes;
  for (int e = blockIdx.y; e < c.E; e += gridDim.y) {
    // row -> (token, head, k or v), heads fastest: the projections' order
    const int which = row & 1;
    const int t = (row >> 1) / c.Hk, h = (row >> 1) % c.Hk;
    const int n = a.count ? min(max(__ldg(a.count + e), 0), a.T) : a.T;
    const bool mine = row < a.rows && t < n;
    const int64_t pos = (int64_t)__ldg(a.start + e) + t;
    const int d0 = sub * kPer, valid = c.D - d0;
    float x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = 0.0f;
    int page = -1, slot = 0;
    if (mine) {
      if (pos < 0 || pos >= c.capacity)
        cache_fail(c, MA_STATUS_BAD_LENGTH);
      else
        page = cache_page(c, e, (int)pos, slot);
      const X* src = reinterpret_cast<const X*>(a.x[which]) + e * a.xs[which][0] +
                     h * a.xs[which][1] + t * a.xs[which][2] + d0 * a.xs[which][3];
      if (a.xs[which][3] == 1) {
        load_vec<X, kPer>(src, a.xvec[which], valid, x);
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (i < valid) x[i] = to_f<X>(src[i * a.xs[which][3]]);
      }
    }
    const int64_t at = page * c.stride[which][0] + h * c.stride[which][1] + slot * c.stride[which][2];
    if constexpr (is_coded<K>) {
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        // NaN stays: a row with one gets a NaN scale, as its maximum in torch
        amax = (fabsf(x[i]) > amax || isnan(x[i])) ? fabsf(x[i]) : amax;
      for (int o = a.lanes / 2; o > 0; o /= 2) {
        const float other = __shfl_xor_sync(0xffffffffu, amax, o);
        amax = (other > amax || isnan(other)) ? other : amax;
      }
      const float scale =
          (isnan(amax) ? amax : fmaxf(amax, kAmaxMin)) * (K == Elem::i8 ? 1.0f / 127.0f : 1.0f / 448.0f);
      if (page >= 0 && valid > 0) {
        union {
          uint2 v;
          uint8_t b[kPer];
        } u;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const float y = __fdiv_rn(x[i], scale);
          if (K == Elem::i8)
            u.b[i] = (uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(y, -127.0f), 127.0f));
          else
            u.b[i] = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
        }
        uint8_t* dst = reinterpret_cast<uint8_t*>(c.pages[which]) + at + d0;
        if (a.pvec[which] && valid >= kPer) {
          *reinterpret_cast<uint2*>(dst) = u.v;
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (i < valid) dst[i] = u.b[i];
        }
        if (sub == 0)
          c.scale[which][page * c.sstride[which][0] + h * c.sstride[which][1] +
                         slot * c.sstride[which][2]] = scale;
      }
    } else {
      using P = typename ElemT<K>::type;
      if (page >= 0 && valid > 0)
        store_vec<P>(reinterpret_cast<P*>(c.pages[which]) + at + d0, a.pvec[which], valid, x);
    }
  }
}

struct ReadArgs {
  CacheView c;
  char* x[2];
  int64_t xs[2][4];
  const int32_t* lengths;
  uint8_t* mask;
  int N, lanes;
  int64_t rows;  // 2 * N * Hk of one sequence
  bool xvec[2], pvec[2];
};

template <typename X, Elem K>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const ReadArgs a) {
  using P = typename ElemT<K>::type;
  const CacheView& c = a.c;
  const int sub = threadIdx.x % a.lanes;
  const int row = blockIdx.x * (kThreads / a.lanes) + threadIdx.x / a.lanes;
  if (row >= a.rows) return;
  // row -> (k or v, head, token), tokens fastest: the order of pages and output
  const int t = row % a.N, h = (row / a.N) % c.Hk, which = row / a.N / c.Hk;
  for (int e = blockIdx.y; e < c.E; e += gridDim.y) {
    const int len = cache_length(c, __ldg(a.lengths + e));
    const int d0 = sub * kPer, valid = c.D - d0;
    float x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = 0.0f;
    if (t < len && valid > 0) {
      int slot;
      const int page = cache_page(c, e, t, slot);
      if (page >= 0) {
        load_vec<P, kPer>(reinterpret_cast<const P*>(c.pages[which]) + page * c.stride[which][0] +
                              h * c.stride[which][1] + slot * c.stride[which][2] + d0,
                          a.pvec[which], valid, x);
        if constexpr (is_coded<K>) {
          const float s = c.scale[which][page * c.sstride[which][0] + h * c.sstride[which][1] +
                                         slot * c.sstride[which][2]];
#pragma unroll
          for (int i = 0; i < kPer; ++i) x[i] *= s;
        }
      }
    }
    if (valid > 0) {
      X* dst = reinterpret_cast<X*>(a.x[which]) + e * a.xs[which][0] + h * a.xs[which][1] +
               t * a.xs[which][2] + d0 * a.xs[which][3];
      if (a.xs[which][3] == 1) {
        store_vec<X>(dst, a.xvec[which], valid, x);
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (i < valid) dst[i * a.xs[which][3]] = from_f<X>(x[i]);
      }
    }
    if (a.mask && which == 0 && h == 0 && sub == 0) a.mask[(int64_t)e * a.N + t] = t < len;
  }
}

int refuse(int code, const std::string& detail) {
  set_error_detail(detail);
  return code;
}

int dense_bytes(int dtype) {
  return dtype == MA_DTYPE_F32 ? 4 : dtype == MA_DTYPE_F16 || dtype == MA_DTYPE_BF16 ? 2 : 0;
}

// Whether rows of an (E, Hk, T, D) tensor start on `bytes`-byte boundaries.
bool dense_aligned(const void* p, const int64_t* st, int eb, int bytes) {
  return st[3] == 1 && (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && st[0] * eb % bytes == 0 &&
         st[1] * eb % bytes == 0 && st[2] * eb % bytes == 0;
}

template <typename F> int launch(F&& f) {
  f();
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess)
    return refuse(MA_ERR_CUDA, std::string("CUDA error: ") + cudaGetErrorName(err) + ": " +
                                   cudaGetErrorString(err));
  set_launch_count(1);
  return MA_OK;
}

template <typename X>
int launch_write(const WriteArgs& a, int dtype, dim3 grid, cudaStream_t st) {
  return launch([&] {
    switch (cache_elem(dtype)) {
      case Elem::f32: cache_write_kernel<X, Elem::f32><<<grid, kThreads, 0, st>>>(a); break;
      case Elem::f16: cache_write_kernel<X, Elem::f16><<<grid, kThreads, 0, st>>>(a); break;
      case Elem::bf16: cache_write_kernel<X, Elem::bf16><<<grid, kThreads, 0, st>>>(a); break;
      case Elem::e4m3: cache_write_kernel<X, Elem::e4m3><<<grid, kThreads, 0, st>>>(a); break;
      case Elem::i8: cache_write_kernel<X, Elem::i8><<<grid, kThreads, 0, st>>>(a); break;
    }
  });
}

template <typename X>
int launch_read(const ReadArgs& a, int dtype, dim3 grid, cudaStream_t st) {
  return launch([&] {
    switch (cache_elem(dtype)) {
      case Elem::f32: cache_read_kernel<X, Elem::f32><<<grid, kThreads, 0, st>>>(a); break;
      case Elem::f16: cache_read_kernel<X, Elem::f16><<<grid, kThreads, 0, st>>>(a); break;
      case Elem::bf16: cache_read_kernel<X, Elem::bf16><<<grid, kThreads, 0, st>>>(a); break;
      case Elem::e4m3: cache_read_kernel<X, Elem::e4m3><<<grid, kThreads, 0, st>>>(a); break;
      case Elem::i8: cache_read_kernel<X, Elem::i8><<<grid, kThreads, 0, st>>>(a); break;
    }
  });
}

int check_dense(const char* what, const void* k, const void* v, const int64_t* ks, const int64_t* vs) {
  if (!k || !v) return refuse(MA_ERR_NULL_POINTER, std::string(what) + " is NULL");
  for (int i = 0; i < 4; ++i)
    if (ks[i] < 0 || vs[i] < 0) return refuse(MA_ERR_BAD_STRIDE, "negative stride");
  return MA_OK;
}

}  // namespace

Elem cache_elem(int dtype) {
  switch (dtype) {
    case MA_DTYPE_F16: return Elem::f16;
    case MA_DTYPE_BF16: return Elem::bf16;
    case MA_DTYPE_E4M3: return Elem::e4m3;
    case MA_DTYPE_I8: return Elem::i8;
    default: return Elem::f32;
  }
}

int cache_elem_bytes(int dtype) {
  switch (dtype) {
    case MA_DTYPE_F32: return 4;
    case MA_DTYPE_F16:
    case MA_DTYPE_BF16: return 2;
    case MA_DTYPE_E4M3:
    case MA_DTYPE_I8: return 1;
    default: return 0;
  }
}

bool cache_rows_aligned(const ma_kv_cache& c, int t, int bytes) {
  const int eb = cache_elem_bytes(c.dtype);
  const int64_t* st = t ? c.v_stride : c.k_stride;
  return reinterpret_cast<uintptr_t>(t ? c.v_pages : c.k_pages) % bytes == 0 &&
         st[0] * eb % bytes == 0 && st[1] * eb % bytes == 0 && st[2] * eb % bytes == 0;
}

int cache_view(const ma_kv_cache& c, CacheView* v, std::string* detail) {
  const auto no = [&](int code, const char* why) {
    *detail = why;
    return code;
  };
  if (c.struct_size != sizeof(ma_kv_cache))
    return no(MA_ERR_BAD_PARAMS, "struct_size of the cache is not sizeof(ma_kv_cache)");
  if (cache_elem_bytes(c.dtype) == 0) return no(MA_ERR_BAD_DTYPE, "unknown dtype of the pages");
  if (c.E < 1 || c.Hk < 1 || c.num_pages < 1 || c.page_size < 1 || c.max_pages < 1)
    return no(MA_ERR_BAD_SHAPE, "E, Hk, num_pages, page_size and max_pages must all be >= 1");
  if (c.D < 1 || c.D > kMaxCacheDim)
    return no(MA_ERR_BAD_SHAPE, "head dim of the pages must be in [1, 256]");
  if ((int64_t)c.max_pages * c.page_size > INT32_MAX - 64)
    return no(MA_ERR_BAD_SHAPE, "max_pages * page_size exceeds 2^31 - 65");
  if (!c.k_pages || !c.v_pages || !c.page_table)
    return no(MA_ERR_NULL_POINTER, "pages or page table is NULL");
  if (!c.status) return no(MA_ERR_NULL_POINTER, "status word is NULL");
  const bool coded = c.dtype == MA_DTYPE_E4M3 || c.dtype == MA_DTYPE_I8;
  if (coded && (!c.k_scale || !c.v_scale))
    return no(MA_ERR_NULL_POINTER, "e4m3 / int8 pages need k and v scales");
  for (int i = 0; i < 3; ++i)
    if (c.k_stride[i] < 0 || c.v_stride[i] < 0 || (coded && (c.ks_stride[i] < 0 || c.vs_stride[i] < 0)))
      return no(MA_ERR_BAD_STRIDE, "negative stride of the pages or scales");
  if (c.page_table_stride[0] < 0 || c.page_table_stride[1] < 0)
    return no(MA_ERR_BAD_STRIDE, "negative stride of the page table");
  if (c.status_host && !host_word_check(c.status_host))
    return no(MA_ERR_BAD_PARAMS,
              "status_host is not page-locked host memory the device can write at the same address");
  v->pages[0] = static_cast<char*>(c.k_pages);
  v->pages[1] = static_cast<char*>(c.v_pages);
  v->scale[0] = c.k_scale;
  v->scale[1] = c.v_scale;
  for (int i = 0; i < 3; ++i) {
    v->stride[0][i] = c.k_stride[i];
    v->stride[1][i] = c.v_stride[i];
    v->sstride[0][i] = c.ks_stride[i];
    v->sstride[1][i] = c.vs_stride[i];
  }
  v->table = c.page_table;
  v->tstride[0] = c.page_table_stride[0];
  v->tstride[1] = c.page_table_stride[1];
  v->E = c.E; v->Hk = c.Hk; v->D = c.D;
  v->num_pages = c.num_pages; v->page_size = c.page_size; v->max_pages = c.max_pages;
  v->capacity = c.max_pages * c.page_size;
  page_divisor(*v);
  v->status = c.status;
  v->status_host = c.status_host;
  return MA_OK;
}

}  // namespace ma

using namespace ma;

extern "C" {

int ma_cache_write(const ma_cache_write_params* p, void* stream) try {
  set_error_detail("");
  if (!p) return refuse(MA_ERR_NULL_POINTER, "params is NULL");
  if (p->struct_size != sizeof(*p))
    return refuse(MA_ERR_BAD_PARAMS, "struct_size is not sizeof(ma_cache_write_params)");
  WriteArgs a{};
  std::string why;
  int rc = cache_view(p->cache, &a.c, &why);
  if (rc != MA_OK) return refuse(rc, why);
  const int xb = dense_bytes(p->dtype), pb = cache_elem_bytes(p->cache.dtype);
  if (!xb) return refuse(MA_ERR_BAD_DTYPE, "new keys and values are f32, f16 or bf16");
  if (p->T < 1) return refuse(MA_ERR_BAD_SHAPE, "T must be >= 1");
  rc = check_dense("k or v", p->k, p->v, p->k_stride, p->v_stride);
  if (rc != MA_OK) return rc;
  if (!p->start) return refuse(MA_ERR_NULL_POINTER, "start is NULL");
  const int64_t rows = 2 * (int64_t)p->T * a.c.Hk;
  if (rows > INT32_MAX - kThreads) return refuse(MA_ERR_BAD_SHAPE, "2 * T * Hk exceeds 2^31");
  for (int t = 0; t < 2; ++t) {
    const int64_t* st = t ? p->v_stride : p->k_stride;
    a.x[t] = static_cast<const char*>(t ? p->v : p->k);
    for (int i = 0; i < 4; ++i) a.xs[t][i] = st[i];
    a.xvec[t] = dense_aligned(a.x[t], st, xb, 16);
    a.pvec[t] = cache_rows_aligned(p->cache, t, pb == 1 ? 8 : 16);
  }
  a.start = p->start;
  a.count = p->count;
  a.T = p->T;
  a.lanes = row_lanes(a.c.D);
  a.rows = (int)rows;
  const int per = kThreads / a.lanes;
  const dim3 grid((unsigned)((rows + per - 1) / per), a.c.E < 65535 ? a.c.E : 65535);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return p->dtype == MA_DTYPE_F32    ? launch_write<float>(a, p->cache.dtype, grid, st)
         : p->dtype == MA_DTYPE_F16 ? launch_write<__half>(a, p->cache.dtype, grid, st)
                                    : launch_write<__nv_bfloat16>(a, p->cache.dtype, grid, st);
} catch (...) {
  return MA_ERR_BAD_PARAMS;
}

int ma_cache_read(const ma_cache_read_params* p, void* stream) try {
  set_error_detail("");
  if (!p) return refuse(MA_ERR_NULL_POINTER, "params is NULL");
  if (p->struct_size != sizeof(*p))
    return refuse(MA_ERR_BAD_PARAMS, "struct_size is not sizeof(ma_cache_read_params)");
  ReadArgs a{};
  std::string why;
  int rc = cache_view(p->cache, &a.c, &why);
  if (rc != MA_OK) return refuse(rc, why);
  const int xb = dense_bytes(p->dtype), pb = cache_elem_bytes(p->cache.dtype);
  if (!xb) return refuse(MA_ERR_BAD_DTYPE, "sequences are read back as f32, f16 or bf16");
  if (p->N < 1) return refuse(MA_ERR_BAD_SHAPE, "N must be >= 1");
  rc = check_dense("k or v", p->k, p->v, p->k_stride, p->v_stride);
  if (rc != MA_OK) return rc;
  if (!p->lengths) return refuse(MA_ERR_NULL_POINTER, "lengths is NULL");
  a.rows = 2 * (int64_t)p->N * a.c.Hk;
  if (a.rows > INT32_MAX - kThreads) return refuse(MA_ERR_BAD_SHAPE, "2 * N * Hk exceeds 2^31");
  for (int t = 0; t < 2; ++t) {
    const int64_t* st = t ? p->v_stride : p->k_stride;
    a.x[t] = static_cast<char*>(t ? p->v : p->k);
    for (int i = 0; i < 4; ++i) a.xs[t][i] = st[i];
    a.xvec[t] = dense_aligned(a.x[t], st, xb, 16);
    a.pvec[t] = cache_rows_aligned(p->cache, t, pb == 1 ? 8 : 16);
  }
  a.lengths = p->lengths;
  a.mask = p->mask;
  a.N = p->N;
  a.lanes = row_lanes(a.c.D);
  const int per = kThreads / a.lanes;
  const dim3 grid((unsigned)((a.rows + per - 1) / per), a.c.E < 65535 ? a.c.E : 65535);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return p->dtype == MA_DTYPE_F32    ? launch_read<float>(a, p->cache.dtype, grid, st)
         : p->dtype == MA_DTYPE_F16 ? launch_read<__half>(a, p->cache.dtype, grid, st)
                                    : launch_read<__nv_bfloat16>(a, p->cache.dtype, grid, st);
} catch (...) {
  return MA_ERR_BAD_PARAMS;
}

}  // extern "C"
