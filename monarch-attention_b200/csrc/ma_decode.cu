// Attention of one new token a sequence over a paged key-value cache: the C
// entry (ma_decode, include/ma_api.h) and the kernel for 32-bit queries and
// for rows that no 16-byte load fits.  The mathematics, the work split and the
// joins stand in ma_decode.cuh, 16-bit queries in ma_decode_mma.cuh.
#include <type_traits>

#include "ma_decode.cuh"

namespace ma {

void set_error_detail(const std::string& detail);  // ma_api.cu
void set_launch_count(int n);

using namespace decode;

namespace {

// ---------------------------------------------------------------------------
// Any type, size and alignment, in 32-bit arithmetic: 8 lanes share a token
// (4 tokens a warp at a time), each with DP / 8 of its values.  The sums o stay in
// registers; q of four heads lies in shared memory, where the 8 lanes' addresses
// are all that is read.  A score is a sum over 8 lanes: of four heads each lane ends
// with one (4 shuffles instead of 12), so that a weight is computed once instead of 8
// times, and gets the others' weights by a shuffle each.  m moves when a score
// exceeds it by kSlack: one vote for all in flight, and a value costs one operation
// for each of q k and p v.  The four groups of lanes keep their own (m, l, o) and meet
// at the row's end.  VEC: rows of whole vectors on 16-byte boundaries; kFlight * 4
// tokens' keys and values are then in flight at a time (no branch around a load: loads
// with one wait for each other).  Every lane takes part in every shuffle and vote,
// whether its token is valid or not.
// Measured (B200, fp32, 8 sequences of 100 to 2000 tokens, 12 kv heads): one query
// head each of 64, 12 us, of 128, 25, of 256, 49; four of 64, 21 us (with a maximum a
// token and every lane its own weights, 34), of 128, 40 (49), of 256, 87 (a pass a head:
// 153).  16000 tokens each, one head of 64: 124 us (6.4 TB/s, HBM).  Passes of 8 heads
// were slower (of 64, 8 heads: 61 us where two passes of four took 43).
// ---------------------------------------------------------------------------
template <Elem K_, int NC_, int DP_, bool VEC_, bool ROW_>
struct ScalarCore {
  static constexpr Elem K = K_;
  static constexpr int NC = NC_, DP = DP_;
  static constexpr bool VEC = VEC_, ROW = ROW_;
  static constexpr int W = !ROW ? kWarps : NC > 1 || DP > 128 ? 8 : DP == 128 ? 12 : 16;  // warps
  static constexpr int kPer = DP / 8;  // values of a row in a lane
  using P = typename ElemT<K>::type;
  // values loaded at once: 16 bytes, or the lane's whole share
  static constexpr int kVec = 16 / (int)sizeof(P) < kPer ? 16 / (int)sizeof(P) : kPer;
  // as many as 64 registers hold, or 32 beside 128 of o
  static constexpr int kFit = (NC * kPer >= 128 ? 32 : 64) / (2 * kPer * (int)sizeof(P) / 4);
  // CTAs an SM
  static constexpr int kMin = ROW ? 1 : DP == 64 ? (NC == 1 ? 4 : 3) : NC == 1 && DP == 128 ? 3 : 2;
  static constexpr int kFlight = !VEC || kFit < 1 ? 1 : kFit > 4 ? 4 : kFit;

  // value i of lane l8 is element (i / kVec) * 8 * kVec + l8 * kVec + i % kVec
  static __device__ __forceinline__ int dim(int l8, int i) {
    return i / kVec * 8 * kVec + l8 * kVec + i % kVec;
  }
  struct Row {
    union {
      uint32_t w[kPer * sizeof(P) / 4];
      P t[kPer];
    };
  };
  // Vectors behind the row's end come from its start: q is 0 there, and o is not used.
  static __device__ __forceinline__ void load(const DecodeArgs& a, const P* row, int l8, Row& x) {
    constexpr int B = kVec * (int)sizeof(P);
#pragma unroll
    for (int i = 0; i < kPer; i += kVec) {
      const P* at = row + (DP == a.c.D || dim(l8, i) < a.c.D ? dim(l8, i) : 0);
      uint32_t* w = x.w + i * (int)sizeof(P) / 4;
      if constexpr (B == 16) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(at));
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
        w[0] = v.x;
        w[1] = v.y;
      }
    }
  }
  static __device__ __forceinline__ void load_singly(const DecodeArgs& a, const P* row, int l8,
                                                     bool valid, Row& x) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      x.t[i] = P();
      if (valid && dim(l8, i) < a.c.D) x.t[i] = row[dim(l8, i)];
    }
  }

  // The sum of head l8 % NC's z over the 8 lanes of a token: with 4 heads each lane
  // gives up two, then one of them, so that 4 shuffles serve all 4.
  static __device__ __forceinline__ float sum_own(const float(&z)[NC], int l8) {
    constexpr uint32_t kAll = 0xffffffffu;
    float s;
    if constexpr (NC == 4) {
      const bool odd = l8 & 1, high = l8 & 2;
      const float a = (odd ? z[1] : z[0]) + __shfl_xor_sync(kAll, odd ? z[0] : z[1], 1);
      const float b = (odd ? z[3] : z[2]) + __shfl_xor_sync(kAll, odd ? z[2] : z[3], 1);
      s = (high ? b : a) + __shfl_xor_sync(kAll, high ? a : b, 2);
    } else {
      static_assert(NC == 1);
      s = z[0] + __shfl_xor_sync(kAll, z[0], 1);
      s += __shfl_xor_sync(kAll, s, 2);
    }
    return s + __shfl_xor_sync(kAll, s, 4);
  }
  // head g's x, which lanes g and g + NC, ... of a token's 8 hold
  static __device__ __forceinline__ float of_head(float x, int g) {
    return NC == 1 ? x : __shfl_sync(0xffffffffu, x, g, 8);
  }

  // Tiles [tile + warp, tile + n) of row (e, r), every W-th: the warp's
  // part goes to m, l (NC) and o (NC, DP) in shared memory.  sq: shared memory for q
  // (NC, DP).
  static __device__ __forceinline__ void run(const DecodeArgs& a, int e, int r, int len, int tile,
                                             int n, float* sm, float* so, float* sq) {
    constexpr uint32_t kAll = 0xffffffffu;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l8 = lane & 7, sub = lane >> 3;
    const int hk = r / a.groups, h0 = hk * a.G + (r % a.groups) * NC;
    const int heads = min(NC, a.G - (r % a.groups) * NC);
    for (int i = threadIdx.x; i < NC * DP; i += W * 32) {
      const int g = i / DP, d = i % DP;
      sq[i] = g < heads && d < a.c.D
                  ? load_dense(a.q, a.dtype, e * a.qs[0] + (h0 + g) * a.qs[1] + d * a.qs[2])
                  : 0.0f;
    }
    __syncthreads();
    const auto load_q = [&](int g, float(&x)[kPer]) {
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(sq + g * DP + dim(l8, i));
        x[i] = v.x;
        x[i + 1] = v.y;
        x[i + 2] = v.z;
        x[i + 3] = v.w;
      }
    };
    float q1[kPer], o[NC][kPer], m = -INFINITY, l = 0.0f;  // m, l: of head l8 % NC
    if constexpr (NC == 1) load_q(0, q1);  // more heads' q stay in shared memory
#pragma unroll
    for (int g = 0; g < NC; ++g)
#pragma unroll
      for (int i = 0; i < kPer; ++i) o[g][i] = 0.0f;
    for (int t = tile + warp; t < tile + n; t += W) {
      const Token tok = find_token<K>(a, e, hk, t * kTile + lane, len);
      const uint32_t in = __ballot_sync(kAll, tok.valid);
      if (in == 0) continue;
#pragma unroll 1
      for (int j0 = 0; j0 < kTile / 4; j0 += kFlight) {
        if ((in >> (4 * j0) & ((1u << (4 * kFlight)) - 1u)) == 0) continue;
        Row k[kFlight], v[kFlight];
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
          const int src = (j0 + j) * 4 + sub;
          const P* kr = reinterpret_cast<const P*>(a.c.pages[0]) + __shfl_sync(kAll, tok.k, src);
          const P* vr = reinterpret_cast<const P*>(a.c.pages[1]) + __shfl_sync(kAll, tok.v, src);
          if constexpr (VEC) {  // an invalid token's row is any row
            load(a, kr, l8, k[j]);
            load(a, vr, l8, v[j]);
          } else {
            load_singly(a, kr, l8, in >> src & 1, k[j]);
            load_singly(a, vr, l8, in >> src & 1, v[j]);
          }
        }
        float s[kFlight], vs[kFlight], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
          const int src = (j0 + j) * 4 + sub;
          float ks = a.scale2;
          vs[j] = 1.0f;
          if constexpr (is_coded<K>) {
            ks *= __shfl_sync(kAll, tok.ks, src);
            vs[j] = __shfl_sync(kAll, tok.vs, src);
          }
          float x[kPer], z[NC];
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            x[i] = DP == a.c.D || dim(l8, i) < a.c.D ? to_f<P>(k[j].t[i]) : 0.0f;
#pragma unroll
          for (int g = 0; g < NC; ++g) {
            float qg[kPer];
            if constexpr (NC > 1) load_q(g, qg);
            z[g] = 0.0f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) z[g] = fmaf(NC > 1 ? qg[i] : q1[i], x[i], z[g]);
          }
          const float sum = sum_own(z, l8) * ks;  // shuffles: by every lane
          s[j] = in >> src & 1 ? sum : -INFINITY;
          top = fmaxf(top, s[j]);
        }
        if (__any_sync(kAll, top - m > kSlack)) {
          const float to = fmaxf(m, top), c = weight(m, to);
          m = to;
          l *= c;
#pragma unroll
          for (int g = 0; g < NC; ++g) {
            const float cg = of_head(c, g);
#pragma unroll
            for (int i = 0; i < kPer; ++i) o[g][i] *= cg;
          }
        }
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
          const bool valid = in >> ((j0 + j) * 4 + sub) & 1;
          const float p = s[j] == -INFINITY ? 0.0f : ex2f(s[j] - m);
          l += p;
#pragma unroll
          for (int g = 0; g < NC; ++g) {
            const float pg = of_head(p * vs[j], g);  // by every lane
            if (valid)
#pragma unroll
              for (int i = 0; i < kPer; ++i) o[g][i] = fmaf(pg, to_f<P>(v[j].t[i]), o[g][i]);
          }
        }
      }
    }
    float to = m;
    to = fmaxf(to, __shfl_xor_sync(kAll, to, 8));
    to = fmaxf(to, __shfl_xor_sync(kAll, to, 16));
    const float w = weight(m, to);
    float lw = l * w;
    lw += __shfl_xor_sync(kAll, lw, 8);
    lw += __shfl_xor_sync(kAll, lw, 16);
    if (lane < NC) {
      sm[warp * 2 * NC + lane] = part_max(to, lw);
      sm[warp * 2 * NC + NC + lane] = lw;
    }
#pragma unroll
    for (int g = 0; g < NC; ++g) {
      const float wg = of_head(w, g);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float x = o[g][i] * wg;
        x += __shfl_xor_sync(kAll, x, 8);
        x += __shfl_xor_sync(kAll, x, 16);
        if (sub == 0) so[(warp * NC + g) * DP + dim(l8, i)] = x;
      }
    }
  }
};

template <class Core>
__global__ void __launch_bounds__(Core::W * 32, Core::kMin) decode_kernel(const DecodeArgs a) {
  constexpr int NC = Core::NC, DP = Core::DP, W = Core::W;
  wait_for_earlier();
  __shared__ float sm[W * 2 * NC];
  __shared__ __align__(16) float so[W * NC * DP], sq[NC * DP];
  Piece p;
  typename std::conditional<Core::ROW, RowLength, Lengths>::type lens;
  if (!find_piece(a, &p, &lens)) return;
  int e = p.e, r = p.r, tile = p.tile;
  int64_t start = p.start;
  Left left;
  for (;;) {
    const int len = lens.of(a, e), tiles = row_tiles(len);
    const int n = tiles_before_end(p, start, tiles) - tile;
    if (n <= 0) break;
    Core::run(a, e, r, len, tile, n, sm, so, sq);
    __syncthreads();
    end_row<NC, DP, DP, W>(a, p, e, r, tiles, n, start, start <= 0, sm, so, left);
    __syncthreads();
    start += tiles + p.cost;
    if (start >= p.end) break;
    tile = 0;
    if (++r == a.rows) {
      r = 0;
      ++e;
    }
  }
  if constexpr (!Core::ROW) join_left<NC, DP>(a, p, left);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int refuse(int code, const std::string& detail) {
  set_error_detail(detail);
  return code;
}

template <class Core>
cudaError_t launch(const DecodeArgs& a, int grid, cudaStream_t st) {
  if (grid < 1) return cudaErrorInvalidDevice;
  return launch_early(decode_kernel<Core>, grid, Core::W * 32, 0, st, a);
}

template <Elem K, int NC, int DP, bool VEC>
cudaError_t launch(DecodeArgs a, cudaStream_t st) {
  using Row = ScalarCore<K, NC, DP, VEC, true>;
  using Cut = ScalarCore<K, NC, DP, VEC, false>;
  static Resident known[2];
  a.groups = (a.G + NC - 1) / NC;
  a.rows = a.c.Hk * a.groups;
  const int64_t rows = (int64_t)a.c.E * a.rows;
  if (short_rows(a, (int)sizeof(typename Row::P)) && rows <= places(decode_kernel<Row>, Row::W * 32, 0, known[0]))
    return launch<Row>(a, (int)rows, st);
  return launch<Cut>(a, piece_ctas(a, places(decode_kernel<Cut>, Cut::W * 32, 0, known[1])), st);
}

template <Elem K, bool VEC>
cudaError_t launch_scalar(const DecodeArgs& a, cudaStream_t st) {
  // four query heads share a pass over the keys and values where there are that many
  if (a.c.D <= 64) return a.G > 1 ? launch<K, 4, 64, VEC>(a, st) : launch<K, 1, 64, VEC>(a, st);
  if (a.c.D <= 128) return a.G > 1 ? launch<K, 4, 128, VEC>(a, st) : launch<K, 1, 128, VEC>(a, st);
  // (codes, widened to 32 bits, leave no registers for four o of 256)
  if constexpr (!is_coded<K>)
    if (a.G > 1) return launch<K, 4, 256, VEC>(a, st);
  return launch<K, 1, 256, VEC>(a, st);
}

// 32-bit queries, and 16-bit ones on rows that start on other boundaries.
template <Elem K>
cudaError_t launch_scalar(const DecodeArgs& a, cudaStream_t st) {
  // 16-bit pages come here for their alignment alone
  if constexpr (K == Elem::f16 || K == Elem::bf16) {
    return launch_scalar<K, false>(a, st);
  } else {
    const int bytes = (int)sizeof(typename ElemT<K>::type);
    const bool vec = a.kvec && a.vvec && a.c.D * bytes % 16 == 0;
    return vec ? launch_scalar<K, true>(a, st) : launch_scalar<K, false>(a, st);
  }
}

static_assert(sizeof(uint32_t) * 4 * kMaxCtas <= MA_DECODE_ZERO_BYTES, "the counters are what is zero");

}  // namespace
}  // namespace ma

using namespace ma;

extern "C" {

size_t ma_decode_workspace_bytes(void) {
  return MA_DECODE_ZERO_BYTES + sizeof(float) * (size_t)kPartFloats * 2 * kMaxCtas;
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
  if ((double)c.E * p->H * a.c.capacity >= 8796093022208.0)  // a CTA's tiles are counted in 32 bits
    return refuse(MA_ERR_BAD_SHAPE, "E * H * max_pages * page_size exceeds 2^43");
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
  const int qb = p->dtype == MA_DTYPE_F32 ? 4 : 2;
  const auto aligned = [&](const void* at, const int64_t* st) {
    return st[2] == 1 && reinterpret_cast<uintptr_t>(at) % 16 == 0 && st[0] * qb % 16 == 0 &&
           st[1] * qb % 16 == 0;
  };
  a.qvec = aligned(p->q, p->q_stride);
  a.ovec = aligned(p->out, p->o_stride);
  a.count = static_cast<uint32_t*>(p->workspace);
  a.parts = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + MA_DECODE_ZERO_BYTES);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t err = cudaSuccess;
  // 16-bit results may come from 16-bit products of the tensor cores
  const bool mma = p->dtype != MA_DTYPE_F32 && a.kvec && a.vvec;
  switch (cache_elem(c.dtype)) {
    case Elem::f32: err = launch_scalar<Elem::f32>(a, st); break;
    case Elem::f16: err = mma ? run_decode_f16(a, st) : launch_scalar<Elem::f16>(a, st); break;
    case Elem::bf16: err = mma ? run_decode_bf16(a, st) : launch_scalar<Elem::bf16>(a, st); break;
    case Elem::e4m3: err = mma ? run_decode_e4m3(a, st) : launch_scalar<Elem::e4m3>(a, st); break;
    case Elem::i8: err = mma ? run_decode_i8(a, st) : launch_scalar<Elem::i8>(a, st); break;
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
