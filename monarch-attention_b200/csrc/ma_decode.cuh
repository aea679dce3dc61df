// One-token attention over a paged cache: what its two kernels (ma_decode.cu,
// ma_decode_mma.cuh) share -- the work split, page look-up and joins.
//
//   s_j = sm_scale <q, k_j>,  o = sum_j softmax(s)_j v_j,  lse = log sum_j e^{s_j}
//
// Every cached value is used 2 G times (G = H / Hk query heads share it), a
// few operations a byte, so HBM bounds it and the work is to keep every SM
// loading from start to end whatever the lengths are.
//
// Work split.  A row is (sequence, kv head, group of query heads); it has
// ceil(length / 32) tiles of 32 tokens.  All rows' tiles form one line, cut
// into as many equal pieces as there are CTAs (each CTA sums the lengths
// itself: they are device data).  A CTA goes through its piece row by row, its
// warps taking the tiles in turn with one pass over the data (running maximum
// m, sum l and weighted values o); the warps' (m, l, o) meet in shared memory
// at a row's end.  A row that lies in one CTA is finished there.  Otherwise
// each CTA leaves its part in the workspace and the last one to arrive joins
// them in the order of the tiles, so the result does not depend on timing:
// up to kJoinOne parts at once, more by groups of kJoinGroup and then the groups.
// No CTA ever waits for another one.
#pragma once

#include <math.h>

#include <atomic>

#include "ma_cache.cuh"

namespace ma {
namespace decode {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;      // tokens a warp takes at a time
constexpr int kMaxCtas = 592;  // bound of the workspace's parts
constexpr int kPartFloats = 4 * 16 + 2048;  // (m, l) twice for up to 16 heads, o: 16 x 128 or 8 x 256
constexpr int kJoinOne = 24;
constexpr int kJoinGroup = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DecodeArgs {
  CacheView c;
  const void* q;
  void* out;
  float* lse;
  int64_t qs[3], os[3];
  const int32_t* lengths;
  const void* mask;
  int64_t ms[2];
  int mask_dtype, mask_len, dtype;
  int H, G, groups, rows;  // rows: kv heads x groups of one sequence
  float scale2;            // sm_scale * log2(e): exponents are powers of two
  bool kvec, vvec, qvec;  // rows of keys, values on 16-byte, of q on 8-byte boundaries
  uint32_t* count;  // [2][2 * kMaxCtas] arrivals, zero between calls
  float* parts;     // [2 * kMaxCtas][kPartFloats]
};

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^(m - to), 0 where m is -inf (no token): the weight of a part with maximum m.
__device__ __forceinline__ float weight(float m, float to) {
  return m == -INFINITY ? 0.0f : ex2f(m - to);
}

__device__ __forceinline__ float load_dense(const void* p, int dtype, int64_t at) {
  return dtype == MA_DTYPE_F32   ? static_cast<const float*>(p)[at]
         : dtype == MA_DTYPE_F16 ? to_f(static_cast<const __half*>(p)[at])
                                 : to_f(static_cast<const __nv_bfloat16*>(p)[at]);
}

__device__ __forceinline__ void store_dense(void* p, int dtype, int64_t at, float x) {
  if (dtype == MA_DTYPE_F32)
    static_cast<float*>(p)[at] = x;
  else if (dtype == MA_DTYPE_F16)
    static_cast<__half*>(p)[at] = from_f<__half>(x);
  else
    static_cast<__nv_bfloat16*>(p)[at] = from_f<__nv_bfloat16>(x);
}

// Tiles of a row of len tokens: an empty row still has to be written.
__device__ __forceinline__ int row_tiles(int len) {
  return len > 0 ? (len + kTile - 1) / kTile : 1;
}

// Lengths of kHeld sequences from `first` on in shared memory, so that going
// from row to row does not wait for global memory.  (So few: two CTAs of the
// largest rings that fit an SM twice leave 256 bytes.)
constexpr int kHeld = 48;
struct Lengths {
  int first;
  const int* held;
  __device__ __forceinline__ int of(const DecodeArgs& a, int e) const {
    return e - first < kHeld ? held[e - first] : cache_length(a.c, __ldg(a.lengths + e));
  }
};

// The piece of the line of tiles that is this CTA's.
struct Piece {
  int64_t total, t0, t1;  // all tiles, this CTA's
  int n;                  // CTAs that have one
  int e, r, tile;         // where t0 lies: sequence, its row, the row's tile
};

__device__ __forceinline__ int64_t piece_start(int64_t total, int n, int c) { return total * c / n; }
__device__ __forceinline__ int piece_of(int64_t total, int n, int64_t t) {
  return (int)(((t + 1) * n - 1) / total);
}

__device__ __forceinline__ bool find_piece(const DecodeArgs& a, Piece* out, Lengths* lens) {
  __shared__ int64_t wsum[kWarps];
  __shared__ int at[3], held[kHeld];
  const int E = a.c.E, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (E + kThreads - 1) / kThreads;
  const int e0 = min((int)threadIdx.x * per, E), e1 = min(e0 + per, E);
  int64_t mine = 0;
  for (int e = e0; e < e1; ++e) {
    const int len = cache_length(a.c, __ldg(a.lengths + e));
    if (E <= kHeld) held[e] = len;
    mine += row_tiles(len);
  }
  mine *= a.rows;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += wsum[w];
    total += wsum[w];
  }
  before += incl - mine;
  Piece p;
  p.total = total;
  // no more CTAs than rows, or than give each warp a tile
  const int64_t rows = (int64_t)E * a.rows, quads = (total + kWarps - 1) / kWarps;
  const int64_t most = rows > quads ? rows : quads;
  p.n = (int)(most < gridDim.x ? most : gridDim.x);
  if ((int)blockIdx.x >= p.n) return false;
  p.t0 = piece_start(total, p.n, blockIdx.x);
  p.t1 = piece_start(total, p.n, blockIdx.x + 1);
  if (p.t0 >= before && p.t0 < before + mine) {
    int64_t rem = p.t0 - before;
    int e = e0, tiles = row_tiles(cache_length(a.c, __ldg(a.lengths + e)));
    while (rem >= (int64_t)tiles * a.rows) {
      rem -= (int64_t)tiles * a.rows;
      ++e;
      tiles = row_tiles(cache_length(a.c, __ldg(a.lengths + e)));
    }
    at[0] = e;
    at[1] = (int)(rem / tiles);
    at[2] = (int)(rem % tiles);
  }
  __syncthreads();
  p.e = at[0];
  p.r = at[1];
  p.tile = at[2];
  *out = p;
  lens->first = E <= kHeld ? 0 : p.e;
  lens->held = held;
  if (E > kHeld) {
    const int e = p.e + threadIdx.x;
    if (threadIdx.x < kHeld && e < E) held[threadIdx.x] = cache_length(a.c, __ldg(a.lengths + e));
    __syncthreads();
  }
  return true;
}

// One token (lane) of a warp's tile: where its keys and values lie.
struct Token {
  int64_t k, v;  // element offsets of the rows
  float ks, vs;  // their scales
  bool valid;
};

template <Elem K>
__device__ __forceinline__ Token find_token(const DecodeArgs& a, int e, int h, int pos, int len) {
  const CacheView& c = a.c;
  Token t;
  t.k = t.v = 0;
  t.ks = t.vs = 1.0f;
  t.valid = pos < len;
  if (t.valid && a.mask)
    t.valid = pos < a.mask_len && mask_value(a.mask, a.mask_dtype, e * a.ms[0] + pos * a.ms[1]);
  if (t.valid) {
    int slot;
    const int page = cache_page(c, e, pos, slot);
    t.valid = page >= 0;
    if (t.valid) {
      t.k = page * c.stride[0][0] + h * c.stride[0][1] + slot * c.stride[0][2];
      t.v = page * c.stride[1][0] + h * c.stride[1][1] + slot * c.stride[1][2];
      if constexpr (is_coded<K>) {
        t.ks = c.scale[0][page * c.sstride[0][0] + h * c.sstride[0][1] + slot * c.sstride[0][2]];
        t.vs = c.scale[1][page * c.sstride[1][0] + h * c.sstride[1][1] + slot * c.sstride[1][2]];
      }
    }
  }
  return t;
}

// Row parts of a CTA's warps, or of several CTAs, are joined as
//   m = max m_i,  l = sum l_i 2^(m_i - m),  o = sum o_i 2^(m_i - m)
// and a finished row is o / l and (m + log2 l) ln 2.  A part is NC heads' m,
// NC l, room for the m and l of parts joined into it, and o (NC, DP).
template <int NC, int DP>
__device__ __forceinline__ void finish(const DecodeArgs& a, int e, int r, int col, int d, float m,
                                       float l, float4 o) {
  const int hk = r / a.groups, first = (r % a.groups) * NC + col;
  if (first >= a.G) return;
  const int h = hk * a.G + first;
  const float inv = __fdiv_rn(1.0f, l);
  const int64_t at = e * a.os[0] + h * a.os[1];
  const float x[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (d + i < a.c.D)
      store_dense(a.out, a.dtype, at + (d + i) * a.os[2], l == 0.0f ? 0.0f : x[i] * inv);
  if (a.lse && d == 0)
    a.lse[(int64_t)e * a.H + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

__device__ __forceinline__ void add_part(float w, float li, float4 x, float& l, float4& o) {
  l += w * li;
  o.x += w * x.x;
  o.y += w * x.y;
  o.z += w * x.z;
  o.w += w * x.w;
}

// Joins n parts of a row and finishes it (last), or leaves the joined part in
// the first one's slot.  Part i lies in slot0 (i = 0) or in the first half of
// the slots of the CTA i * step behind slot0's.  joined: the parts' (m, l) are
// those of an earlier join.
template <int NC, int DP>
__device__ __forceinline__ void join(const DecodeArgs& a, int e, int r, int slot0, int n, int step, bool joined,
                     bool last) {
  const auto part = [&](int i) {
    return a.parts + (int64_t)(i == 0 ? slot0 : 2 * ((slot0 >> 1) + i * step)) * kPartFloats;
  };
  const int ml = joined ? 2 * NC : 0;
#pragma unroll 1
  for (int it = threadIdx.x; it < NC * DP / 4; it += kThreads) {
    const int col = it / (DP / 4), d = it % (DP / 4) * 4;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = 0; i < n; ++i) m = fmaxf(m, __ldcg(part(i) + ml + col));
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float* p = part(i);
      add_part(weight(__ldcg(p + ml + col), m), __ldcg(p + ml + NC + col),
               __ldcg(reinterpret_cast<const float4*>(p + 4 * NC + col * DP + d)), l, o);
    }
    if (last) {
      finish<NC, DP>(a, e, r, col, d, m, l, o);
    } else {
      // o replaces what only this thread reads; (m, l) go beside the ones
      // that other threads may still read
      float* p = part(0);
      *reinterpret_cast<float4*>(p + 4 * NC + col * DP + d) = o;
      if (d == 0) {
        p[2 * NC + col] = m;
        p[3 * NC + col] = l;
      }
    }
  }
}

// Whether this CTA is the last of n to arrive at a counter, which is zero
// again after it.  What the others wrote before they arrived can then be read.
__device__ __forceinline__ bool arrive(uint32_t* count, int n) {
  __shared__ bool last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicInc(count, n - 1) == (uint32_t)(n - 1);
    __threadfence();
  }
  __syncthreads();
  return last;
}

// The end of a CTA's part of a row, tiles [tile, tile + n) of its `tiles`,
// which begin at pos on the line of tiles: the warps' parts (m, l in sm (warp,
// 2, NC), o in so (warp, NC, OS)) are joined and the row finished, or left in
// the workspace and joined with those of other CTAs by the last one.  A warp
// without a token has m = -inf, and its o is not read.
template <int NC, int DP, int OS>
__device__ __forceinline__ void end_row(const DecodeArgs& a, const Piece& p, int e, int r, int tile,
                                        int tiles, int n, int64_t pos, const float* sm,
                                        const float* so) {
  const int64_t row0 = pos - tile;  // the row's first tile
  const int slot = 2 * blockIdx.x + (pos > p.t0 ? 1 : 0);
  float* part = a.parts + (int64_t)slot * kPartFloats;
#pragma unroll 1
  for (int it = threadIdx.x; it < NC * DP / 4; it += kThreads) {
    const int col = it / (DP / 4), d = it % (DP / 4) * 4;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm[w * 2 * NC + col]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = sm[w * 2 * NC + col];
      if (mw != -INFINITY)
        add_part(ex2f(mw - m), sm[w * 2 * NC + NC + col],
                 *reinterpret_cast<const float4*>(so + (w * NC + col) * OS + d), l, o);
    }
    if (n == tiles) {
      finish<NC, DP>(a, e, r, col, d, m, l, o);
    } else {
      *reinterpret_cast<float4*>(part + 4 * NC + col * DP + d) = o;
      if (d == 0) {
        part[col] = m;
        part[NC + col] = l;
      }
    }
  }
  if (n < tiles) {
    // a row's parts: slot 1 of the first CTA where the row starts inside its
    // piece, slot 0 of all others
    const int first = piece_of(p.total, p.n, row0);
    const int cnt = piece_of(p.total, p.n, row0 + tiles - 1) - first + 1;
    const int i = blockIdx.x - first;
    const int slot0 = 2 * first + (row0 > piece_start(p.total, p.n, first) ? 1 : 0);
    const int group = cnt <= kJoinOne ? cnt : kJoinGroup;
    const int lead = i / group * group;
    const int lslot = lead == 0 ? slot0 : 2 * (first + lead);
    const int members = min(group, cnt - lead);
    if (arrive(a.count + lslot, members)) {
      const bool one = group == cnt;
      join<NC, DP>(a, e, r, lslot, members, 1, false, one);
      if (!one) {
        const int groups = (cnt + group - 1) / group;
        if (arrive(a.count + 2 * kMaxCtas + slot0, groups))
          join<NC, DP>(a, e, r, slot0, groups, group, true, true);
      }
    }
  }
}

// ---- host side: launch shape ---------------------------------------------------------------

// CTAs of a kernel to launch: every SM full, but no more than the longest
// lengths that fit the page table could use; 0 where the device refuses.  known:
// per device, what fits an SM (0: not asked yet).
constexpr int kMaxDevices = 64;
struct Resident {
  std::atomic<int> per_sm[kMaxDevices], sms[kMaxDevices];
};

template <typename F>
int grid_size(const DecodeArgs& a, F* kernel, int smem, Resident& known) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) return 0;
  int per = known.per_sm[dev], sms = known.sms[dev];
  if (per == 0) {
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 smem) != cudaSuccess)
      return 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kThreads, smem) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return 0;
    known.sms[dev] = sms;
    known.per_sm[dev] = per;
  }
  int64_t grid = (int64_t)sms * per;
  const int64_t tiles = ((int64_t)a.c.capacity + kTile - 1) / kTile;
  const int64_t most = (int64_t)a.c.E * a.rows * ((tiles + kWarps - 1) / kWarps);
  if (grid > most) grid = most;
  return (int)(grid < kMaxCtas ? grid : kMaxCtas);
}

}  // namespace decode

// ma_decode_inst_*.cu: 16-bit queries on the tensor cores; the rows of the
// pages must start on 16-byte boundaries.
cudaError_t run_decode_f16(const decode::DecodeArgs& a, cudaStream_t st);
cudaError_t run_decode_bf16(const decode::DecodeArgs& a, cudaStream_t st);
cudaError_t run_decode_e4m3(const decode::DecodeArgs& a, cudaStream_t st);
cudaError_t run_decode_i8(const decode::DecodeArgs& a, cudaStream_t st);

}  // namespace ma
