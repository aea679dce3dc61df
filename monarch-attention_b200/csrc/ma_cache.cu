// Paged key-value cache: new tokens stored (quantised as they are written)
// and sequences read back as dense tensors.  C entries ma_cache_write and
// ma_cache_read (include/ma_api.h); the reference's decoder keeps dense
// tensors instead (bart/model.py:67-152).
//
// Store:  scale = max(max_d |x_d|, 1e-12) * (1 / top),  code_d = rn(x_d / scale)
// Read:   x_d = code_d * scale, zero at and behind a sequence's length
//
// Both kernels touch every byte once and compute a few operations a value, so
// HBM bounds them, and what counts is bytes in flight and few instructions
// beside the loads and stores.  A row of D values (one token, head, and k or v)
// is taken by 1 to 32 neighbouring lanes with 8 values each (16 of 8-bit
// pages); the row's maximum is a shuffle over these lanes.  The lanes go
// through some heads of their token, up to eight rows in flight at a time as
// they lie in memory: page and slot are looked up once (a chain of three loads,
// longer than the copy of a row), and a row's place is the last one's plus a stride.
// Measured (B200, 4 x 16384 tokens, 16 heads of 128, bf16 in and out): stored as
// e4m3 in 172 us (4.7 TB/s; issue bounds it: 267 instructions for four rows of a
// warp, 40 % of them the exact quotients), read back in 136 us (6.0 TB/s); bf16 pages
// 166 and 200 us (6.5 and 5.4 TB/s).
#include <math.h>

#include <type_traits>

#include "ma_cache.cuh"

namespace ma {

void set_error_detail(const std::string& detail);  // ma_api.cu
void set_launch_count(int n);
int host_word_check(const void* ptr);

namespace {

constexpr int kThreads = 256;
constexpr float kAmaxMin = 1e-12f;
constexpr int64_t kDeviceThreads = 148 * 2048;  // that a B200 holds at a time

// What both kernels need of the dense side, and the split of their work: an
// item is (token, k or v, some heads); items of one sequence lie in blockIdx.x.
struct DenseArgs {
  CacheView c;
  char* x[2];
  int64_t xs[2][4];
  int T;              // tokens a sequence: new ones, or those to read back
  int per;            // values of a lane
  int lanes, lshift;  // of a row: a power of two
  int heads, chunks;  // heads of an item, items of a token
  int items;          // T * 2 * chunks
  bool xvec[2], pvec[2];
};

struct Item {
  int t, which, h0, h1, sub;
  bool valid;
};

// Neighbouring items are neighbouring in the projections' output when tokens are
// stored (heads, k or v first), in the dense result when they are read back
// (tokens first).
__device__ __forceinline__ Item find_item(const DenseArgs& a, bool tokens_first) {
  Item it;
  const int i = blockIdx.x * (kThreads >> a.lshift) + (threadIdx.x >> a.lshift);
  it.sub = threadIdx.x & (a.lanes - 1);
  it.valid = i < a.items;
  const int per = 2 * a.chunks, rest = tokens_first ? i / a.T : i % per;
  it.t = tokens_first ? i % a.T : i / per;
  it.which = rest / a.chunks;
  it.h0 = rest % a.chunks * a.heads;
  it.h1 = min(it.h0 + a.heads, a.c.Hk);
  return it;
}

// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// N values of a lane as they lie in memory.
template <typename X, int N>
struct Raw {
  static constexpr int kWords = sizeof(X) * N / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // All of them, on a 16-byte boundary (8 codes: 8), one behind the other.  No branch around
  // it: loads with one wait for each other.
  __device__ __forceinline__ void load_all(const X* src) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      if constexpr (kWords >= 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + i / 4);
        w[i] = v.x;
        w[i + 1] = v.y;
        w[i + 2] = v.z;
        w[i + 3] = v.w;
      } else {  // 8 codes
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
        w[0] = v.x;
        w[1] = v.y;
      }
    }
  }
  // `valid` of them lie in the row, `step` apart; vec: on a 16-byte boundary,
  // one behind the other
  __device__ __forceinline__ void load(const X* src, int64_t step, bool vec, int valid) {
    if (vec && valid >= N) {
      load_all(src);
    } else if (vec && valid == N / 2 && kWords % 2 == 0) {
      zero();
#pragma unroll
      for (int i = 0; i < kWords / 2; i += 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(src) + i / 2);
        w[i] = v.x;
        w[i + 1] = v.y;
      }
    } else {
      zero();
      constexpr int kIn = 4 / sizeof(X);  // in a word
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < valid) {
          union {
            X x;
            uint8_t b[sizeof(X)];
          } u;
          u.x = src[i * step];
          uint32_t bits = 0;
#pragma unroll
          for (int j = 0; j < (int)sizeof(X); ++j) bits |= (uint32_t)u.b[j] << (8 * j);
          w[i / kIn] |= bits << (8 * (int)sizeof(X) * (i % kIn));
        }
    }
  }
  __device__ __forceinline__ void values(float (&x)[N]) const {
    union {
      uint32_t w[kWords];
      X t[N];
    } u;
#pragma unroll
    for (int i = 0; i < kWords; ++i) u.w[i] = w[i];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f<X>(u.t[i]);
  }
};

// Rows in flight: 32 registers of them.
template <typename X, int N> constexpr int kFlight = 32 / Raw<X, N>::kWords;

template <typename X, int N>
__device__ __forceinline__ void store_values(X* dst, int64_t step, bool vec, int valid,
                                             const float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 8) {
    if (step == 1 && vec && valid - i >= 8) {
      union {
        uint4 v[sizeof(X) / 2];
        X t[8];
      } u;
#pragma unroll
      for (int j = 0; j < 8; ++j) u.t[j] = from_f<X>(x[i + j]);
#pragma unroll
      for (int j = 0; j < (int)sizeof(X) / 2; ++j) reinterpret_cast<uint4*>(dst + i)[j] = u.v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < valid) dst[(i + j) * step] = from_f<X>(x[i + j]);
    }
  }
}

// The values x of a lane, read as `raw`, to an aligned row: as they are where the
// types are the same.
template <typename X, int N, typename R>
__device__ __forceinline__ void store_all(X* dst, const R& raw, const float (&x)[N]) {
  union {
    uint4 v[sizeof(X) * N / 16];
    uint32_t w[sizeof(X) * N / 4];
    X t[N];
  } u;
  if constexpr (std::is_same<R, Raw<X, N>>::value) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(X) * N / 4; ++i) u.w[i] = raw.w[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) u.t[i] = from_f<X>(x[i]);
  }
#pragma unroll
  for (int i = 0; i < (int)sizeof(X) * N / 16; ++i) reinterpret_cast<uint4*>(dst)[i] = u.v[i];
}

// x / scale, correctly rounded, given inv = 1 / scale, correctly rounded: two
// steps of q += inv (x - q scale) with exact remainders (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor",
// 1990: the second one starts from a quotient that is off by less than a unit).
// A remainder that underflows belongs to a quotient far below the smallest code.
__device__ __forceinline__ float quotient(float x, float scale, float inv) {
  float q = x * inv;
  q = fmaf(fmaf(-q, scale, x), inv, q);
  return fmaf(fmaf(-q, scale, x), inv, q);
}

template <Elem K>
__device__ __forceinline__ uint32_t code4(const float* y) {
  if constexpr (K == Elem::e4m3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  } else {
    // |y| <= 127 (1 + 2^-23): 1.5 * 2^23 more rounds it to an integer, ties to
    // even, in the last bits
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(y[i] + 12582912.0f);
    return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
  }
}

struct WriteArgs : DenseArgs {
  const int32_t* start;
  const int32_t* count;
};

// N: values a lane.  EVEN: rows of a multiple of N values on boundaries for their
// loads and stores on both sides.
template <typename X, Elem K, int N, bool EVEN>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const WriteArgs a) {
  const CacheView& c = a.c;
  constexpr int F = kFlight<X, N>;
  const Item it = find_item(a, false);
  wait_for_earlier();
  const int w = it.which, d0 = it.sub * N, valid = c.D - d0;
  const int64_t step = a.xs[w][3];
  for (int e = blockIdx.y; e < c.E; e += gridDim.y) {
    const int n = a.count ? min(max(__ldg(a.count + e), 0), a.T) : a.T;
    const int64_t pos = (int64_t)__ldg(a.start + e) + it.t;
    const bool here = it.valid && it.t < n;
    const X* src = reinterpret_cast<const X*>(a.x[w]) + e * a.xs[w][0];
    if (!EVEN || (here && valid > 0))  // else: any row
      src += it.h0 * a.xs[w][1] + it.t * a.xs[w][2] + d0 * step;
    const int last = EVEN && !(here && valid > 0) ? 0 : it.h1 - it.h0 - 1;
    int64_t at = 0, sat = 0;
    int page = -2;  // not looked up yet: the first rows are asked for before it
    // (every lane takes part in the shuffles: the trip count is the grid's)
#pragma unroll 1
    for (int i0 = 0; i0 < a.heads; i0 += F) {
      Raw<X, N> raw[F];
#pragma unroll
      for (int i = 0; i < F; ++i) {
        if constexpr (EVEN)
          raw[i].load_all(src + min(i0 + i, last) * a.xs[w][1]);
        else if (here && valid > 0 && i0 + i <= last)
          raw[i].load(src + (i0 + i) * a.xs[w][1], step, a.xvec[w], valid);
        else
          raw[i].zero();
      }
      if (page == -2) {
        int slot = 0;
        page = -1;
        if (here) {
          if (pos < 0 || pos >= c.capacity) cache_fail(c, MA_STATUS_BAD_LENGTH);
          else page = cache_page(c, e, (int)pos, slot);
        }
        if (page >= 0) {
          at = page * c.stride[w][0] + it.h0 * c.stride[w][1] + slot * c.stride[w][2] + d0;
          if constexpr (is_coded<K>)
            sat = page * c.sstride[w][0] + it.h0 * c.sstride[w][1] + slot * c.sstride[w][2];
        }
      }
#pragma unroll
      for (int i = 0; i < F; ++i) {
        if (i0 + i >= a.heads) break;
        const bool in = page >= 0 && valid > 0 && i0 + i <= last;
        float x[N];
        raw[i].values(x);
        if (EVEN && is_coded<K> && valid <= 0) {  // a lane behind the row's end
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] = 0.0f;
        }
        if constexpr (is_coded<K>) {
          float amax = 0.0f;
#pragma unroll
          for (int j = 0; j < N; ++j) amax = max_nan(amax, fabsf(x[j]));
          for (int o = a.lanes / 2; o > 0; o /= 2)
            amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const float scale = max_nan(amax, kAmaxMin) * (K == Elem::i8 ? 1.0f / 127.0f : 1.0f / 448.0f);
          if (scale <= 3.4e38f) {
            const float inv = __frcp_rn(scale);
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = quotient(x[j], scale, inv);
          } else {  // infinity or NaN among the values: x / scale is 0 or NaN
            const float f = isnan(scale) ? scale : 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] *= f;
          }
          if (in) {
            uint8_t* dst = reinterpret_cast<uint8_t*>(c.pages[w]) + at + (i0 + i) * c.stride[w][1];
            union {
              uint4 v;
              uint2 h[2];
              uint32_t w4[4];
              uint8_t b[16];
            } u;
#pragma unroll
            for (int j = 0; j < N; j += 4) u.w4[j / 4] = code4<K>(&x[j]);
            if (N == 16 && (EVEN || (a.pvec[w] && valid >= N))) {
              *reinterpret_cast<uint4*>(dst) = u.v;
            } else if (EVEN || (a.pvec[w] && valid == 8)) {
              *reinterpret_cast<uint2*>(dst) = u.h[0];
            } else {
#pragma unroll
              for (int j = 0; j < N; ++j)
                if (j < valid) dst[j] = u.b[j];
            }
            if (it.sub == 0) c.scale[w][sat + (i0 + i) * c.sstride[w][1]] = scale;
          }
        } else if (in) {
          using P = typename ElemT<K>::type;
          P* dst = reinterpret_cast<P*>(c.pages[w]) + at + (i0 + i) * c.stride[w][1];
          if constexpr (EVEN) store_all<P, N>(dst, raw[i], x);
          else store_values<P, N>(dst, 1, a.pvec[w], valid, x);
        }
      }
    }
  }
}

struct ReadArgs : DenseArgs {
  const int32_t* lengths;
  uint8_t* mask;
};

template <typename X, Elem K, int N, bool EVEN>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const ReadArgs a) {
  using P = typename ElemT<K>::type;
  const CacheView& c = a.c;
  constexpr int F = kFlight<P, N> > 8 ? 8 : kFlight<P, N>;
  const Item it = find_item(a, true);
  wait_for_earlier();
  if (!it.valid) return;
  const int w = it.which, d0 = it.sub * N, valid = c.D - d0;
  const int64_t step = a.xs[w][3];
  for (int e = blockIdx.y; e < c.E; e += gridDim.y) {
    const int len = cache_length(c, __ldg(a.lengths + e));
    if (valid <= 0) continue;
    int page = -1, slot = 0;
    if (it.t < len) page = cache_page(c, e, it.t, slot);
    // (not valid where the page is missing, which is reported too)
    if (a.mask && w == 0 && it.h0 == 0 && it.sub == 0) a.mask[(int64_t)e * a.T + it.t] = page >= 0;
    const P* src = reinterpret_cast<const P*>(c.pages[w]) + d0;  // any row
    const float* ssrc = c.scale[w];
    if (page >= 0) {
      src += page * c.stride[w][0] + it.h0 * c.stride[w][1] + slot * c.stride[w][2];
      if constexpr (is_coded<K>)
        ssrc += page * c.sstride[w][0] + it.h0 * c.sstride[w][1] + slot * c.sstride[w][2];
    }
    X* dst = reinterpret_cast<X*>(a.x[w]) + e * a.xs[w][0] + it.h0 * a.xs[w][1] + it.t * a.xs[w][2] +
             d0 * step;
    const int heads = it.h1 - it.h0, last = page >= 0 ? heads - 1 : 0;
#pragma unroll 1
    for (int i0 = 0; i0 < heads; i0 += F) {
      Raw<P, N> raw[F];
      float s[F];
#pragma unroll
      for (int i = 0; i < F; ++i) {
        s[i] = 0.0f;
        if constexpr (EVEN) {
          if constexpr (is_coded<K>) s[i] = __ldg(ssrc + min(i0 + i, last) * c.sstride[w][1]);
          raw[i].load_all(src + min(i0 + i, last) * c.stride[w][1]);
        } else if (page >= 0 && i0 + i < heads) {
          if constexpr (is_coded<K>) s[i] = __ldg(ssrc + (i0 + i) * c.sstride[w][1]);
          raw[i].load(src + (i0 + i) * c.stride[w][1], 1, a.pvec[w], valid);
        } else {
          raw[i].zero();
        }
      }
#pragma unroll
      for (int i = 0; i < F; ++i) {
        if (i0 + i >= heads) break;
        float x[N];
        raw[i].values(x);
        if constexpr (is_coded<K>) {
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] *= s[i];
        }
        X* to = dst + (i0 + i) * a.xs[w][1];
        if constexpr (EVEN) {
          if (page < 0) {
            raw[i].zero();
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = 0.0f;
          }
          store_all<X, N>(to, raw[i], x);
        } else {
          store_values<X, N>(to, step, a.xvec[w], valid, x);
        }
      }
    }
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

int launched(cudaError_t err) {
  if (err != cudaSuccess)
    return refuse(MA_ERR_CUDA, std::string("CUDA error: ") + cudaGetErrorName(err) + ": " +
                                   cudaGetErrorString(err));
  set_launch_count(1);
  return MA_OK;
}

// Splits the work: more heads an item cost its look-up less often, fewer give
// more threads.  Measured best (B200, heads 1 to 16 tried, D 64 and 128, e4m3,
// int8 and bf16): 16 where a row a group fills the SMs' threads over 16 times
// (write and read 16384 e4m3 tokens of 16 heads: 171 and 136 us; with 4 heads 191 and
// 159), 8 from 4 times, 4 from once (512 tokens: 10 and 8.4 us; with one head 14
// and 14), 2 from a third, else 1.  Fills grid; false where the items pass 2^31.
bool split(DenseArgs& a, int T, int per, dim3* grid) {
  a.T = T;
  a.per = per;
  a.lshift = 0;
  while ((per << a.lshift) < a.c.D) ++a.lshift;
  a.lanes = 1 << a.lshift;
  const int64_t all = (int64_t)a.c.E * T * 2 * a.c.Hk * a.lanes, full = kDeviceThreads;
  int64_t heads = all > 16 * full ? 16 : all > 4 * full ? 8 : all > full ? 4 : 3 * all > full ? 2 : 1;
  if (heads > a.c.Hk) heads = a.c.Hk;
  a.chunks = (int)((a.c.Hk + heads - 1) / heads);
  a.heads = (a.c.Hk + a.chunks - 1) / a.chunks;
  const int64_t items = (int64_t)T * 2 * a.chunks;
  if (items > INT32_MAX - kThreads) return false;
  a.items = (int)items;
  const int64_t group = kThreads >> a.lshift;
  *grid = dim3((unsigned)((items + group - 1) / group), a.c.E < 65535 ? a.c.E : 65535);
  return true;
}

// 16 codes a lane, or 8 where rows are whole numbers of 8 but not of 16.
int values_per_lane(const ma_kv_cache& c) {
  return cache_elem_bytes(c.dtype) == 1 && (c.D % 16 == 0 || c.D % 8 != 0) ? 16 : 8;
}

// Whether the kernels' EVEN form fits N values a lane.
bool even(const DenseArgs& a, int n) {
  return a.c.D % n == 0 && a.xvec[0] && a.xvec[1] && a.pvec[0] && a.pvec[1];
}

template <typename X, Elem K, int N>
int launch_write(const WriteArgs& a, dim3 grid, cudaStream_t st) {
  return launched(launch_early(even(a, N) ? cache_write_kernel<X, K, N, true>
                                          : cache_write_kernel<X, K, N, false>,
                               grid, kThreads, 0, st, a));
}
template <typename X, Elem K>
int launch_write(const WriteArgs& a, dim3 grid, cudaStream_t st) {
  if constexpr (is_coded<K>)
    if (a.per == 16) return launch_write<X, K, 16>(a, grid, st);
  return launch_write<X, K, 8>(a, grid, st);
}

template <typename X, Elem K, int N>
int launch_read(const ReadArgs& a, dim3 grid, cudaStream_t st) {
  return launched(launch_early(even(a, N) ? cache_read_kernel<X, K, N, true>
                                          : cache_read_kernel<X, K, N, false>,
                               grid, kThreads, 0, st, a));
}
template <typename X, Elem K>
int launch_read(const ReadArgs& a, dim3 grid, cudaStream_t st) {
  if constexpr (is_coded<K>)
    if (a.per == 16) return launch_read<X, K, 16>(a, grid, st);
  return launch_read<X, K, 8>(a, grid, st);
}

template <typename X>
int launch_write(const WriteArgs& a, int dtype, dim3 grid, cudaStream_t st) {
  switch (cache_elem(dtype)) {
    case Elem::f16: return launch_write<X, Elem::f16>(a, grid, st);
    case Elem::bf16: return launch_write<X, Elem::bf16>(a, grid, st);
    case Elem::e4m3: return launch_write<X, Elem::e4m3>(a, grid, st);
    case Elem::i8: return launch_write<X, Elem::i8>(a, grid, st);
    default: return launch_write<X, Elem::f32>(a, grid, st);
  }
}

template <typename X>
int launch_read(const ReadArgs& a, int dtype, dim3 grid, cudaStream_t st) {
  switch (cache_elem(dtype)) {
    case Elem::f16: return launch_read<X, Elem::f16>(a, grid, st);
    case Elem::bf16: return launch_read<X, Elem::bf16>(a, grid, st);
    case Elem::e4m3: return launch_read<X, Elem::e4m3>(a, grid, st);
    case Elem::i8: return launch_read<X, Elem::i8>(a, grid, st);
    default: return launch_read<X, Elem::f32>(a, grid, st);
  }
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
  for (int t = 0; t < 2; ++t) {
    const int64_t* st = t ? p->v_stride : p->k_stride;
    a.x[t] = static_cast<char*>(const_cast<void*>(t ? p->v : p->k));
    for (int i = 0; i < 4; ++i) a.xs[t][i] = st[i];
    a.xvec[t] = dense_aligned(a.x[t], st, xb, 16);
    a.pvec[t] = cache_rows_aligned(p->cache, t, pb == 1 ? values_per_lane(p->cache) : 16);
  }
  a.start = p->start;
  a.count = p->count;
  dim3 grid;
  if (!split(a, p->T, values_per_lane(p->cache), &grid))
    return refuse(MA_ERR_BAD_SHAPE, "2 * T * Hk exceeds 2^31");
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
  for (int t = 0; t < 2; ++t) {
    const int64_t* st = t ? p->v_stride : p->k_stride;
    a.x[t] = static_cast<char*>(t ? p->v : p->k);
    for (int i = 0; i < 4; ++i) a.xs[t][i] = st[i];
    a.xvec[t] = dense_aligned(a.x[t], st, xb, 16);
    a.pvec[t] = cache_rows_aligned(p->cache, t, pb == 1 ? values_per_lane(p->cache) : 16);
  }
  a.lengths = p->lengths;
  a.mask = p->mask;
  dim3 grid;
  if (!split(a, p->N, values_per_lane(p->cache), &grid))
    return refuse(MA_ERR_BAD_SHAPE, "2 * N * Hk exceeds 2^31");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return p->dtype == MA_DTYPE_F32    ? launch_read<float>(a, p->cache.dtype, grid, st)
         : p->dtype == MA_DTYPE_F16 ? launch_read<__half>(a, p->cache.dtype, grid, st)
                                    : launch_read<__nv_bfloat16>(a, p->cache.dtype, grid, st);
} catch (...) {
  return MA_ERR_BAD_PARAMS;
}

}  // extern "C"
