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
// up to kJoinOne parts at once, more by groups and then the groups.
// No CTA ever waits for another one.
//
// Few short rows (at most one for every place of a CTA, at most 64 tiles and 1 MB if
// they were as long as the page table allows) need no line: a CTA with more warps
// takes one row and finishes it, without the way through the workspace and a join,
// 4 to 5 us of the 10 that such a call takes on pieces.
#pragma once

#include <math.h>

#include <atomic>

#include "ma_cache.cuh"

namespace ma {
namespace decode {

constexpr int kWarps = 4;      // of a CTA that takes a piece
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;      // tokens a warp takes at a time
constexpr int kMaxCtas = 592;  // bound of the workspace's parts
constexpr int kPartFloats = 4 * 16 + 2048;  // (m, l) twice for up to 16 heads, o: 16 x 128 or 8 x 256
// A running maximum m moves, and o with it, when a score exceeds it by this much: weights
// 2^(s - m) reach 2^kSlack.
constexpr float kSlack = 6.0f;
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
  bool few;  // the longest lengths give less than 2^28 tiles
  bool kvec, vvec, qvec, ovec;  // rows of keys, values, q, out start on 16-byte boundaries
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

// The maximum that stands with a part's l.  Maxima leave NaN out, so a part whose scores are
// all NaN has m = -inf as one without a token has; its l is NaN, and with a finite m it counts.
__device__ __forceinline__ float part_max(float m, float l) { return isnan(l) ? 0.0f : m; }

__device__ __forceinline__ float load_dense(const void* p, int dtype, int64_t at) {
  return dtype == MA_DTYPE_F32   ? static_cast<const float*>(p)[at]
         : dtype == MA_DTYPE_F16 ? to_f(static_cast<const __half*>(p)[at])
                                 : to_f(static_cast<const __nv_bfloat16*>(p)[at]);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 x = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
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

// Lengths of kHeld sequences from `first` on in shared memory, so that going from row
// to row does not wait for global memory.
constexpr int kSeqs = 2;  // of a lane in find_piece
constexpr int kHeld = 32 * kSeqs;
struct Lengths {
  int first;
  const int* held;
  __device__ __forceinline__ int of(const DecodeArgs& a, int e) const {
    return e - first < kHeld ? held[e - first] : cache_length(a.c, __ldg(a.lengths + e));
  }
};

// The length of the only row of a CTA.
struct RowLength {
  int len;
  __device__ __forceinline__ int of(const DecodeArgs&, int) const { return len; }
};

// x / y rounded down; 64-bit divisions take several times as long.
__device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}

// The pieces of the line of tiles, one a CTA, are of one size.  Where there are
// more rows than CTAs a row counts as kRowCost tiles more than it has, in front
// of its first tile: the end of one row and the start of the next cost a CTA
// about as much (1.4 to 2 us, a CTA's tile 0.45 us), and a piece of many short rows
// would take several times as long as the others (80 sequences of 10 to 900 fp16
// tokens, 12 heads of 64: 54 us without, 32 with 3, 30 with 6).
constexpr int kRowCost = 6;
struct Piece {
  int64_t size;
  int cost;        // of a row
  int64_t start;   // where the row starts that the piece starts in, from there; <= 0
  int end;         // the piece's end, from its start
  int e, r, tile;  // that row, and the first tile of it in the piece
};

// The tiles of a row (of `tiles`, which starts at `start` from the piece's start)
// that lie before the piece's end.
__device__ __forceinline__ int tiles_before_end(const Piece& p, int64_t start, int tiles) {
  const int64_t n = p.end - start - p.cost;
  return n < tiles ? (int)n : tiles;
}

__device__ __forceinline__ int64_t piece_size(const DecodeArgs& a, int64_t total) {
  int64_t size = divide(total + gridDim.x - 1, gridDim.x);
  // Few tiles: as many a warp in fewer CTAs, whose ends then often are rows' ends
  // too, but a CTA for every row where they last.
  if (size <= 4 * kWarps && total > (int64_t)a.c.E * a.rows)
    size = (size + kWarps - 1) / kWarps * kWarps;
  return size;
}

__device__ __forceinline__ bool find_piece(const DecodeArgs& a, Piece* out, Lengths* lens) {
  const int E = a.c.E, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ int held[kHeld];
  Piece p;
  p.cost = (int64_t)E * a.rows > gridDim.x ? kRowCost : 0;
  if (E <= 32 * kSeqs && a.few) {
    // every warp finds it by itself: kSeqs sequences a lane, in 32 bits
    int len[kSeqs], sum = 0;
#pragma unroll
    for (int i = 0; i < kSeqs; ++i) {
      const int e = lane * kSeqs + i;
      len[i] = e < E ? __ldg(a.lengths + e) : 0;
    }
#pragma unroll
    for (int i = 0; i < kSeqs; ++i)
      if (lane * kSeqs + i < E) {
        len[i] = cache_length(a.c, len[i]);
        sum += row_tiles(len[i]) + p.cost;
      }
    sum *= a.rows;
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    p.size = piece_size(a, total);
    const int64_t t0 = p.size * blockIdx.x;
    if (t0 >= total) return false;
    p.end = (int)(t0 + p.size < total ? p.size : total - t0);
    const int owner = __ffs(__ballot_sync(0xffffffffu, incl > (int)t0)) - 1;
    int rem = (int)t0 - __shfl_sync(0xffffffffu, incl - sum, owner), te = 0;
    p.e = owner * kSeqs;
#pragma unroll
    for (int i = 0; i < kSeqs; ++i) {
      const int x = row_tiles(__shfl_sync(0xffffffffu, len[i], owner)) + p.cost;
      if (i == 0 || rem >= te * a.rows) {
        if (i > 0) {
          rem -= te * a.rows;
          ++p.e;
        }
        te = x;
      } else {
        break;
      }
    }
    p.r = rem / te;
    p.start = p.r * te - rem;
    if (warp == 0) {
#pragma unroll
      for (int i = 0; i < kSeqs; ++i) held[lane * kSeqs + i] = len[i];
    }
    __syncthreads();
    lens->first = 0;
    lens->held = held;
  } else {
    __shared__ int64_t wsum[kWarps], start;
    __shared__ int at[2];
    const int per = (E + kThreads - 1) / kThreads;
    const int e0 = min((int)threadIdx.x * per, E), e1 = min(e0 + per, E);
    const auto tiles_of = [&](int e) {
      return row_tiles(cache_length(a.c, __ldg(a.lengths + e))) + p.cost;
    };
    int64_t mine = 0;
    for (int e = e0; e < e1; ++e) mine += tiles_of(e);
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
    p.size = piece_size(a, total);
    const int64_t t0 = p.size * blockIdx.x;
    if (t0 >= total) return false;
    p.end = (int)(t0 + p.size < total ? p.size : total - t0);
    if (t0 >= before && t0 < before + mine) {
      int64_t rem = t0 - before;
      int e = e0, tiles = tiles_of(e);
      while (rem >= (int64_t)tiles * a.rows) {
        rem -= (int64_t)tiles * a.rows;
        tiles = tiles_of(++e);
      }
      at[0] = e;
      at[1] = (int)divide(rem, tiles);
      start = (int64_t)at[1] * tiles - rem;
    }
    __syncthreads();
    p.e = at[0];
    p.r = at[1];
    p.start = start;
    lens->first = p.e;
    lens->held = held;
    const int e = p.e + threadIdx.x;
    if (threadIdx.x < kHeld && e < E) held[threadIdx.x] = cache_length(a.c, __ldg(a.lengths + e));
    __syncthreads();
  }
  const int64_t in = -p.start - p.cost;
  p.tile = in > 0 ? (int)in : 0;
  *out = p;
  return true;
}

// A CTA's row where it takes just one.
__device__ __forceinline__ bool find_piece(const DecodeArgs& a, Piece* out, RowLength* row) {
  Piece p;
  p.e = blockIdx.x / a.rows;
  p.r = blockIdx.x - p.e * a.rows;
  row->len = cache_length(a.c, __ldg(a.lengths + p.e));
  p.size = p.end = row_tiles(row->len);
  p.cost = p.tile = 0;
  p.start = 0;
  *out = p;
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
// and a finished row is o / l and (m + log2 l) ln 2.  A part without a token has m = -inf
// and is left out; one with a NaN among its scores has a finite m (part_max) and NaN for
// l and o, and so has the row.  A part is NC heads' m, NC l, room for the m and l of parts
// joined into it, and o (NC, DP).
template <int NC, int DP>
__device__ __forceinline__ void finish(const DecodeArgs& a, int e, int r, int col, int d, float m,
                                       float l, float4 o) {
  const int hk = r / a.groups, first = (r % a.groups) * NC + col;
  if (first >= a.G) return;
  const int h = hk * a.G + first;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t at = e * a.os[0] + h * a.os[1] + d * a.os[2];
  o = l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                : make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  if (a.ovec && d + 4 <= a.c.D) {  // rows of out on 16-byte boundaries
    if (a.dtype == MA_DTYPE_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = o;
    } else {
      const bool bf = a.dtype == MA_DTYPE_BF16;
      const uint2 u = make_uint2(bf ? pack_bf16(o.x, o.y) : pack_f16(o.x, o.y),
                                 bf ? pack_bf16(o.z, o.w) : pack_f16(o.z, o.w));
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = u;
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 4 && d + i < a.c.D; ++i)
      store_dense(a.out, a.dtype, at + i * a.os[2], i == 0 ? o.x : i == 1 ? o.y : i == 2 ? o.z : o.w);
  }
  if (a.lse && d == 0)
    a.lse[(int64_t)e * a.H + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

__device__ __forceinline__ void add_part(float w, float4 x, float4& o) {
  o.x += w * x.x;
  o.y += w * x.y;
  o.z += w * x.z;
  o.w += w * x.w;
}

// Joins n parts of a row and finishes it (last), or leaves the joined part in the
// first one's slot.  Part i lies in slot0 (i = 0) or in the first half of the
// slots of the CTA i * step behind slot0's.  joined: the parts' (m, l) are those
// of an earlier join.  One CTA reads all the parts, so the loads' latency is most
// of it: a thread has those of kBatch parts in flight.
template <int NC, int DP>
__device__ __forceinline__ void join(const DecodeArgs& a, int e, int r, int slot0, int n, int step,
                                     bool joined, bool last) {
  constexpr int kCol = kThreads / NC;                  // threads of a column
  constexpr int kItems = (DP / 4 + kCol - 1) / kCol;   // 4 values each
  constexpr int kBatch = kItems == 2 ? 6 : 8;
  const int col = threadIdx.x / kCol, c0 = threadIdx.x % kCol;
  if (c0 < DP / 4) {
    const float* base = a.parts + (joined ? 2 * NC : 0) + col;
    const auto part = [&](int i) {
      return (int64_t)(i == 0 ? slot0 : 2 * ((slot0 >> 1) + i * step)) * kPartFloats;
    };
    float m = -INFINITY, l = 0.0f;
    float4 o[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += kBatch) {
      float mi[kBatch], li[kBatch];
      float4 x[kBatch][kItems];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {  // (no branch around a load: the last part again)
        const int64_t at = part(min(i0 + i, n - 1));
        mi[i] = __ldcg(base + at);
        li[i] = __ldcg(base + at + NC);
#pragma unroll
        for (int k = 0; k < kItems; ++k)
          x[i][k] = __ldcg(reinterpret_cast<const float4*>(a.parts + at + 4 * NC + col * DP) + c0 +
                           k * kCol);
      }
      float to = m;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (i0 + i >= n) mi[i] = -INFINITY;
        to = fmaxf(to, mi[i]);
      }
      const float w = weight(m, to);
      m = to;
      l *= w;
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        o[k].x *= w;
        o[k].y *= w;
        o[k].z *= w;
        o[k].w *= w;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (mi[i] != -INFINITY) {
          const float f = ex2f(mi[i] - m);
          l += f * li[i];
#pragma unroll
          for (int k = 0; k < kItems; ++k) add_part(f, x[i][k], o[k]);
        }
    }
    float* p = a.parts + part(0);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int d = (c0 + k * kCol) * 4;
      if (last) finish<NC, DP>(a, e, r, col, d, m, l, o[k]);
      else *reinterpret_cast<float4*>(p + 4 * NC + col * DP + d) = o[k];
    }
    if (!last && c0 == 0) {  // beside the (m, l) that others may still read
      p[2 * NC + col] = m;
      p[3 * NC + col] = l;
    }
  }
}

// The rows of which a CTA has only a part: at most its first and its last one.
struct LeftRow {
  int e, r, tiles;
  int64_t start;  // on the line of tiles
};
struct Left {
  int n = 0;
  LeftRow first, second;
};

// The end of a CTA's part of a row, n of its `tiles`, which starts at `start` from
// the CTA's piece: the warps' parts (m, l in sm (warp, 2, NC), o in so (warp, NC,
// OS)) are joined and the row finished, or its part left in the workspace.  A warp
// without a token has m = -inf, and its o is not read.  A row that is only in part
// here is noted in `left` and joined when all of the CTA's tiles are done.
template <int NC, int DP, int OS, int W>
__device__ __forceinline__ void end_row(const DecodeArgs& a, const Piece& p, int e, int r, int tiles,
                                        int n, int64_t start, bool first, const float* sm,
                                        const float* so, Left& left) {
  const int slot = 2 * blockIdx.x + (first ? 0 : 1);
  float* part = a.parts + (int64_t)slot * kPartFloats;
#pragma unroll 1
  for (int it = threadIdx.x; it < NC * DP / 4; it += W * 32) {
    const int col = it / (DP / 4), d = it % (DP / 4) * 4;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, sm[w * 2 * NC + col]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = sm[w * 2 * NC + col];
      if (mw != -INFINITY) {
        const float f = ex2f(mw - m);
        l += f * sm[w * 2 * NC + NC + col];
        add_part(f, *reinterpret_cast<const float4*>(so + (w * NC + col) * OS + d), o);
      }
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
    const LeftRow row = {e, r, tiles, p.size * blockIdx.x + start};
    if (left.n++ == 0) left.first = row;
    else left.second = row;
  }
}

// Parts that one CTA joins at once: as many as four batches of loads bring.
template <int NC, int DP>
constexpr int kJoinOne = NC * DP <= 512 ? 32 : NC * DP <= 1024 ? 24 : 16;

// A left row's parts: in slot 1 of the first CTA where the row starts inside its
// piece, in slot 0 of all others.  Up to kJoinOne are joined at once, more by
// groups.  A group's counter and joined part are its first CTA's.
struct Group {
  int first, parts;    // the row's first CTA, its parts
  int slot0;           // the first part's slot
  int size;            // parts a group
  int slot, members;   // this CTA's group
};

template <int NC, int DP>
__device__ __forceinline__ Group group_of(const Piece& p, const LeftRow& row) {
  Group g;
  const int64_t tile0 = row.start + p.cost;
  g.first = (int)divide(tile0, p.size);
  g.parts = (int)divide(tile0 + row.tiles - 1, p.size) - g.first + 1;
  g.slot0 = 2 * g.first + (row.start > p.size * g.first ? 1 : 0);
  g.size = g.parts <= kJoinOne<NC, DP> ? g.parts : g.parts <= 64 ? 8 : 16;
  const int lead = (blockIdx.x - g.first) / g.size * g.size;
  g.slot = lead == 0 ? g.slot0 : 2 * (g.first + lead);
  g.members = min(g.size, g.parts - lead);
  return g;
}

// Arrival at the rows that were left, and their joins where this CTA is the last
// to arrive: it finds the count of the others, and makes it zero again.  What
// they wrote before can then be read: the barrier orders a CTA's writes before
// the fence and the arrival.
template <int NC, int DP>
__device__ __forceinline__ void join_left(const DecodeArgs& a, const Piece& p, const Left& left) {
  __shared__ bool last[2], last_group;
  if (left.n == 0) return;
  __syncthreads();
  if (threadIdx.x < left.n) {
    const Group g = group_of<NC, DP>(p, threadIdx.x == 0 ? left.first : left.second);
    __threadfence();
    last[threadIdx.x] = atomicInc(a.count + g.slot, g.members - 1) == (uint32_t)(g.members - 1);
    __threadfence();
  }
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < left.n; ++k) {
    if (!last[k]) continue;
    const LeftRow row = k == 0 ? left.first : left.second;
    const Group g = group_of<NC, DP>(p, row);
    const bool one = g.size == g.parts;
    join<NC, DP>(a, row.e, row.r, g.slot, g.members, 1, false, one);
    if (one) continue;
    const int groups = (g.parts + g.size - 1) / g.size;
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      last_group = atomicInc(a.count + 2 * kMaxCtas + g.slot0, groups - 1) == (uint32_t)(groups - 1);
      __threadfence();
    }
    __syncthreads();
    if (last_group) join<NC, DP>(a, row.e, row.r, g.slot0, groups, g.size, true, true);
  }
}

// ---- host side: launch shape ---------------------------------------------------------------

// What fits an SM of a kernel, asked for once a device (0: not yet).
constexpr int kMaxDevices = 64;
struct Resident {
  std::atomic<int> per_sm[kMaxDevices], sms[kMaxDevices];
};

// CTAs of a kernel that the device holds at a time; 0 where it refuses.
template <typename F>
int64_t places(F* kernel, int threads, int smem, Resident& known) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) return 0;
  int per = known.per_sm[dev], sms = known.sms[dev];
  if (per == 0) {
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 smem) != cudaSuccess)
      return 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return 0;
    known.sms[dev] = sms;
    known.per_sm[dev] = per;
  }
  return (int64_t)sms * per;
}

// Tiles of the longest sequence that the page table allows.
inline int64_t longest(const DecodeArgs& a) { return ((int64_t)a.c.capacity + kTile - 1) / kTile; }

// Whether rows go to one CTA each, where all find a place: rows of up to 64 tiles
// and 1 MB at the longest.  (fp32, 63 tiles: D 64, 1 MB, 12.4 us where pieces
// took 14.8; D 96, 1.5 MB, 22 us where pieces take 19; D 128, 2 MB, 24 where pieces take
// 25; 16-bit rows of 256, 2 MB, the same.)
inline bool short_rows(const DecodeArgs& a, int bytes) {
  return longest(a) <= 64 && longest(a) * (kTile * 2 * bytes) * a.c.D <= 1 << 20;
}

// CTAs on pieces: every place, but no more than the longest lengths could use.
// Fills a.few.
inline int piece_ctas(DecodeArgs& a, int64_t places) {
  const int64_t tiles = longest(a);
  a.few = (double)a.c.E * a.rows * tiles < (1 << 28);
  const int64_t most = (int64_t)a.c.E * a.rows * ((tiles + kWarps - 1) / kWarps);
  const int64_t grid = places < most ? places : most;
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
