// Attention of one new token a sequence over a paged key-value cache
// (ma_decode, include/ma_api.h).
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
#include <math.h>

#include "ma_cache.cuh"

namespace ma {

void set_error_detail(const std::string& detail);  // ma_api.cu
void set_launch_count(int n);

namespace {

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
  bool kvec, vvec;
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

__device__ __forceinline__ int seq_tiles(const DecodeArgs& a, int e) {
  const int len = cache_length(a.c, __ldg(a.lengths + e));
  return len > 0 ? (len + kTile - 1) / kTile : 1;  // an empty row still has to be written
}

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

__device__ bool find_piece(const DecodeArgs& a, Piece* out) {
  __shared__ int64_t wsum[kWarps];
  __shared__ int at[3];
  const int E = a.c.E, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (E + kThreads - 1) / kThreads;
  const int e0 = min((int)threadIdx.x * per, E), e1 = min(e0 + per, E);
  int64_t mine = 0;
  for (int e = e0; e < e1; ++e) mine += seq_tiles(a, e);
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
    int e = e0, tiles = seq_tiles(a, e);
    while (rem >= (int64_t)tiles * a.rows) {
      rem -= (int64_t)tiles * a.rows;
      tiles = seq_tiles(a, ++e);
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
    const int page = cache_page(c, e, pos), slot = pos % c.page_size;
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
__device__ void join(const DecodeArgs& a, int e, int r, int slot0, int n, int step, bool joined,
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

// ---------------------------------------------------------------------------
// Any type, size and alignment, in 32-bit arithmetic: 8 lanes share a token
// (4 tokens a warp at a time), each with DP / 8 of its values, so that q, o
// and the running sums stay in registers and a token's score is a shuffle over
// 8 lanes.  The four groups of lanes keep their own (m, l, o) and meet at the
// row's end.
// ---------------------------------------------------------------------------
template <Elem K_, int NC_, int DP_>
struct ScalarCore {
  static constexpr Elem K = K_;
  static constexpr int NC = NC_, DP = DP_;
  static constexpr int kPer = DP / 8;  // values of a row in a lane
  using P = typename ElemT<K>::type;
  // values loaded at once: 16 bytes, or the lane's whole share
  static constexpr int kVec = 16 / (int)sizeof(P) < kPer ? 16 / (int)sizeof(P) : kPer;

  // value i of lane l8 is element (i / kVec) * 8 * kVec + l8 * kVec + i % kVec
  static __device__ __forceinline__ int dim(int l8, int i) {
    return i / kVec * 8 * kVec + l8 * kVec + i % kVec;
  }
  static __device__ __forceinline__ void load(const DecodeArgs& a, const P* row, bool vec, int l8,
                                              float (&x)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; i += kVec) {
      float y[kVec];
      load_vec<P, kVec>(row + dim(l8, i), vec, a.c.D - dim(l8, i), y);
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[i + j] = y[j];
    }
  }

  // Tiles [tile + warp, tile + n) of row (e, r), every kWarps-th: the warp's
  // part goes to m, l (NC) and o (NC, DP) in shared memory.
  static __device__ __forceinline__ void run(const DecodeArgs& a, int e, int r, int tile, int n,
                                             float* sm, float* so) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l8 = lane & 7, sub = lane >> 3;
    const int hk = r / a.groups, h0 = hk * a.G + (r % a.groups) * NC;
    const int heads = min(NC, a.G - (r % a.groups) * NC);
    const int len = cache_length(a.c, __ldg(a.lengths + e));
    float q[NC][kPer], o[NC][kPer], m[NC], l[NC];
#pragma unroll
    for (int g = 0; g < NC; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int d = dim(l8, i);
        q[g][i] = g < heads && d < a.c.D
                      ? load_dense(a.q, a.dtype, e * a.qs[0] + (h0 + g) * a.qs[1] + d * a.qs[2])
                      : 0.0f;
        o[g][i] = 0.0f;
      }
    }
    for (int t = tile + warp; t < tile + n; t += kWarps) {
      const Token tok = find_token<K>(a, e, hk, t * kTile + lane, len);
#pragma unroll 1
      for (int j = 0; j < kTile / 4; ++j) {
        const int src = j * 4 + sub;
        const int64_t ko = __shfl_sync(0xffffffffu, tok.k, src);
        const int64_t vo = __shfl_sync(0xffffffffu, tok.v, src);
        const float ks = __shfl_sync(0xffffffffu, tok.ks, src);
        const float vs = __shfl_sync(0xffffffffu, tok.vs, src);
        const bool valid = __shfl_sync(0xffffffffu, (int)tok.valid, src);
        float k[kPer], v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) k[i] = v[i] = 0.0f;
        if (valid) {
          load(a, reinterpret_cast<const P*>(a.c.pages[0]) + ko, a.kvec, l8, k);
          load(a, reinterpret_cast<const P*>(a.c.pages[1]) + vo, a.vvec, l8, v);
        }
#pragma unroll
        for (int g = 0; g < NC; ++g) {
          float s = 0.0f;
#pragma unroll
          for (int i = 0; i < kPer; ++i) s = fmaf(q[g][i], k[i], s);
#pragma unroll
          for (int x = 1; x < 8; x *= 2) s += __shfl_xor_sync(0xffffffffu, s, x);
          if (valid) {
            s *= ks * a.scale2;
            const float to = fmaxf(m[g], s);
            const float c = weight(m[g], to), p = s == -INFINITY ? 0.0f : ex2f(s - to);
            const float pv = p * vs;
            m[g] = to;
            l[g] = l[g] * c + p;
#pragma unroll
            for (int i = 0; i < kPer; ++i) o[g][i] = o[g][i] * c + pv * v[i];
          }
        }
      }
    }
#pragma unroll
    for (int g = 0; g < NC; ++g) {
      float to = m[g];
      to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 8));
      to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 16));
      const float w = weight(m[g], to);
      float lw = l[g] * w;
      lw += __shfl_xor_sync(0xffffffffu, lw, 8);
      lw += __shfl_xor_sync(0xffffffffu, lw, 16);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float x = o[g][i] * w;
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (sub == 0) so[(warp * NC + g) * DP + dim(l8, i)] = x;
      }
      if (lane == 0) {
        sm[warp * 2 * NC + g] = to;
        sm[warp * 2 * NC + NC + g] = lw;
      }
    }
  }
};

template <class Core>
__global__ void __launch_bounds__(kThreads) decode_kernel(const DecodeArgs a) {
  constexpr int NC = Core::NC, DP = Core::DP;
  __shared__ float sm[kWarps * 2 * NC];
  __shared__ __align__(16) float so[kWarps * NC * DP];
  Piece p;
  if (!find_piece(a, &p)) return;
  int e = p.e, r = p.r, tile = p.tile;
  int64_t pos = p.t0;
  while (pos < p.t1) {
    const int tiles = seq_tiles(a, e);
    const int n = (int)(tiles - tile < p.t1 - pos ? tiles - tile : p.t1 - pos);
    Core::run(a, e, r, tile, n, sm, so);
    __syncthreads();
    const int64_t row0 = pos - tile;  // the row's first tile
    const int first = piece_of(p.total, p.n, row0);
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
      for (int w = 0; w < kWarps; ++w)
        add_part(weight(sm[w * 2 * NC + col], m), sm[w * 2 * NC + NC + col],
                 *reinterpret_cast<const float4*>(so + (w * NC + col) * DP + d), l, o);
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
    __syncthreads();
    pos += n;
    tile = 0;
    if (++r == a.rows) {
      r = 0;
      ++e;
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int refuse(int code, const std::string& detail) {
  set_error_detail(detail);
  return code;
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return n;
}

template <class Core>
cudaError_t launch(DecodeArgs a, cudaStream_t st) {
  a.groups = (a.G + Core::NC - 1) / Core::NC;
  a.rows = a.c.Hk * a.groups;
  int per = 0;
  cudaError_t err =
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, decode_kernel<Core>, kThreads, 0);
  if (err != cudaSuccess) return err;
  int64_t grid = (int64_t)sm_count() * per;
  // the most that the lengths can ask for
  const int64_t tiles = ((int64_t)a.c.capacity + kTile - 1) / kTile;
  const int64_t rows = (int64_t)a.c.E * a.rows;
  const int64_t most = tiles > kWarps ? rows * ((tiles + kWarps - 1) / kWarps) : rows;
  if (grid > most) grid = most;
  if (grid > kMaxCtas) grid = kMaxCtas;
  if (grid < 1) return cudaErrorInvalidDevice;
  decode_kernel<Core><<<(unsigned)grid, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

template <Elem K>
cudaError_t launch_scalar(const DecodeArgs& a, cudaStream_t st) {
  // four query heads share a pass over the keys and values where there are
  // that many and their rows of q and o fit the registers
  if (a.c.D <= 64)
    return a.G > 1 ? launch<ScalarCore<K, 4, 64>>(a, st) : launch<ScalarCore<K, 1, 64>>(a, st);
  if (a.c.D <= 128)
    return a.G > 1 ? launch<ScalarCore<K, 4, 128>>(a, st) : launch<ScalarCore<K, 1, 128>>(a, st);
  return launch<ScalarCore<K, 1, 256>>(a, st);
}

constexpr size_t kCountBytes = sizeof(uint32_t) * 4 * kMaxCtas;

}  // namespace
}  // namespace ma

using namespace ma;

extern "C" {

size_t ma_decode_workspace_bytes(void) {
  return align_up(kCountBytes, 256) + sizeof(float) * (size_t)kPartFloats * 2 * kMaxCtas;
}

int ma_decode(const ma_decode_params* p, void* stream) try {
  set_error_detail("");
  if (!p) return refuse(MA_ERR_NULL_POINTER, "params is NULL");
  if (p->struct_size != sizeof(*p))
    return refuse(MA_ERR_BAD_PARAMS, "struct_size is not sizeof(ma_decode_params)");
  DecodeArgs a{};
  std::string why;
  const int rc = cache_view(p->cache, &a.c, &why);
  if (rc != MA_OK) return refuse(rc, why);
  const ma_kv_cache& c = p->cache;
  if (p->dtype != MA_DTYPE_F32 && p->dtype != MA_DTYPE_F16 && p->dtype != MA_DTYPE_BF16)
    return refuse(MA_ERR_BAD_DTYPE, "q and out are f32, f16 or bf16");
  const bool coded = c.dtype == MA_DTYPE_E4M3 || c.dtype == MA_DTYPE_I8;
  if (!coded && c.dtype != p->dtype)
    return refuse(MA_ERR_BAD_DTYPE, "f32, f16 and bf16 pages need q and out of their type");
  if (p->H < 1 || p->H % c.Hk != 0)
    return refuse(MA_ERR_BAD_SHAPE, "H must be a positive multiple of Hk");
  if ((int64_t)c.E * p->H > INT32_MAX) return refuse(MA_ERR_BAD_SHAPE, "E * H exceeds 2^31 - 1");
  if (!p->q || !p->out || !p->lengths) return refuse(MA_ERR_NULL_POINTER, "q, out or lengths is NULL");
  for (int i = 0; i < 3; ++i)
    if (p->q_stride[i] < 0 || p->o_stride[i] < 0) return refuse(MA_ERR_BAD_STRIDE, "negative stride");
  if (p->mask) {
    if (p->mask_dtype <= MA_MASK_NONE || p->mask_dtype > MA_MASK_BF16)
      return refuse(MA_ERR_BAD_MASK, "unknown mask dtype");
    if (p->mask_len < 0) return refuse(MA_ERR_BAD_MASK, "mask_len is negative");
    if (p->mask_stride[0] < 0 || p->mask_stride[1] < 0)
      return refuse(MA_ERR_BAD_STRIDE, "negative mask stride");
  } else if (p->mask_dtype != MA_MASK_NONE) {
    return refuse(MA_ERR_BAD_MASK, "mask_dtype set but mask is NULL");
  }
  if (!(p->sm_scale > 0.0f) || isinf(p->sm_scale))
    return refuse(MA_ERR_BAD_PARAMS, "sm_scale must be positive and finite");
  if (!p->workspace || p->workspace_bytes < ma_decode_workspace_bytes() ||
      reinterpret_cast<uintptr_t>(p->workspace) % 256 != 0)
    return refuse(MA_ERR_WORKSPACE, "workspace needs " + std::to_string(ma_decode_workspace_bytes()) +
                                        " bytes on a 256-byte boundary, got " +
                                        std::to_string(p->workspace_bytes));
  a.q = p->q;
  a.out = p->out;
  a.lse = p->lse;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = p->q_stride[i];
    a.os[i] = p->o_stride[i];
  }
  a.lengths = p->lengths;
  a.mask = p->mask;
  a.ms[0] = p->mask_stride[0];
  a.ms[1] = p->mask_stride[1];
  a.mask_dtype = p->mask_dtype;
  a.mask_len = p->mask_len;
  a.dtype = p->dtype;
  a.H = p->H;
  a.G = p->H / c.Hk;
  a.scale2 = p->sm_scale * kLog2e;
  a.kvec = cache_rows_aligned(c, 0, 16);
  a.vvec = cache_rows_aligned(c, 1, 16);
  a.count = static_cast<uint32_t*>(p->workspace);
  a.parts = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + align_up(kCountBytes, 256));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t err = cudaSuccess;
  switch (cache_elem(c.dtype)) {
    case Elem::f32: err = launch_scalar<Elem::f32>(a, st); break;
    case Elem::f16: err = launch_scalar<Elem::f16>(a, st); break;
    case Elem::bf16: err = launch_scalar<Elem::bf16>(a, st); break;
    case Elem::e4m3: err = launch_scalar<Elem::e4m3>(a, st); break;
    case Elem::i8: err = launch_scalar<Elem::i8>(a, st); break;
  }
  if (err != cudaSuccess)
    return refuse(MA_ERR_CUDA, std::string("CUDA error: ") + cudaGetErrorName(err) + ": " +
                                   cudaGetErrorString(err));
  set_launch_count(1);
  return MA_OK;
} catch (...) {
  return MA_ERR_BAD_PARAMS;
}

}  // extern "C"
