// One-token attention for 16-bit queries (ma_decode, include/ma_api.h), on
// the tensor cores.  Mathematics, work split and joins: ma_decode.cuh.
//
// HBM bounds it; the products are there to keep the arithmetic out of the
// way.  With 8 query heads on a kv head, fp32 FMAs would need 16 a cached
// value where an SM has time for about 10 (16-bit pages; 5 for 8-bit ones); m16n8k16
// products with the tokens (scores) or the values' dimensions (output) as the
// 16 rows and the query heads as the 8 columns need 1/128th of the instructions.
//
// A warp works alone on tiles of 32 tokens.  Each lane copies with cp.async
// exactly the 16-byte pieces that it will feed to the products itself, so
// fragments come out of shared memory without a transposition or a bank
// conflict, and no barrier stands between load and use:
//   keys     lane (g, t) holds rows g, g + 8, ... at bytes 16 t of each 64: the sum
//            over dimensions may run in any order, so they need not be the k
//            index that the product names, only q's fragments the same
//   values   lane (g, t) holds rows 2t, 2t+1, 2t+8, 2t+9 (the product's k index)
//            at bytes 16 g of each 128; byte permutes pair two tokens' values
// Three pieces of a ring (keys, values, next keys) keep two of them in flight.
//
// Weights p = 2^(s - m) are fed in two 16-bit halves (rounded, and what the
// rounding left): with one, its rounding would be as large as the result's own.
// e4m3 and int8 codes become fp16 exactly; a key's scale multiplies its score.
// A value's scale v_s joins its weight as 2^(s + log2 v_s - M) with a running
// maximum M of its own, so the fp16 weights stay in range whatever the scales.
// q becomes fp16 relative to the power of two of its largest value.
#include "ma_decode.cuh"
#include "ma_mma_sync.cuh"

namespace ma {

using namespace decode;

namespace {

template <Elem K> struct Wide { using type = __half; };  // what the products take
template <> struct Wide<Elem::bf16> { using type = __nv_bfloat16; };

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
  return __byte_perm(a, b, s);
}

// The 8x8 matrix of 16-bit elements whose rows' pairs the lanes hold, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Two 8-bit codes (low 16 bits, then high 16 bits of x) as fp16 pairs.
template <Elem K>
__device__ __forceinline__ void widen(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if constexpr (K == Elem::e4m3) {
    asm("{.reg .b16 a, b;\n"
        "mov.b32 {a, b}, %2;\n"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n"
        "cvt.rn.f16x2.e4m3x2 %1, b;}"
        : "=r"(lo), "=r"(hi)
        : "r"(x));
  } else {
    // 1024 + (x + 128) has x + 128 in its last bits
    const uint32_t u = x ^ 0x80808080u;
    const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
    lo = prmt(u, 0x64646464u, 0x4140u);
    hi = prmt(u, 0x64646464u, 0x4342u);
    __half2 a = __hsub2(*reinterpret_cast<__half2*>(&lo), off);
    __half2 b = __hsub2(*reinterpret_cast<__half2*>(&hi), off);
    lo = *reinterpret_cast<uint32_t*>(&a);
    hi = *reinterpret_cast<uint32_t*>(&b);
  }
}

template <int B>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int bytes) {
  if constexpr (B == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(bytes),
                 "n"(B)
                 : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_but() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int B>
__device__ __forceinline__ void load_shared(uint32_t at, uint32_t (&x)[B / 4]) {
  if constexpr (B == 16)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                 : "r"(at)
                 : "memory");
  else
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(at) : "memory");
}
__device__ __forceinline__ float load_shared_f(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}

// A load that is issued where it stands.
template <typename T> __device__ __forceinline__ T load_now(const T* at) {
  static_assert(sizeof(T) == 4, "");
  uint32_t x;
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(x) : "l"(at));
  return static_cast<T>(x);
}

// A mask element as it lies in memory, and later its truth value (mask_value
// in two steps, so that nothing waits for the load).
__device__ __forceinline__ uint64_t load_mask(const void* mask, int dtype, int64_t at) {
  uint64_t x;
  if (dtype == MA_MASK_BOOL)
    asm volatile("ld.global.nc.u8 %0, [%1];" : "=l"(x) : "l"(static_cast<const uint8_t*>(mask) + at));
  else if (dtype == MA_MASK_I64)
    asm volatile("ld.global.nc.u64 %0, [%1];" : "=l"(x) : "l"(static_cast<const int64_t*>(mask) + at));
  else if (dtype == MA_MASK_I32 || dtype == MA_MASK_F32)
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=l"(x) : "l"(static_cast<const int32_t*>(mask) + at));
  else
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=l"(x) : "l"(static_cast<const uint16_t*>(mask) + at));
  return x;
}
__device__ __forceinline__ bool mask_bits(uint64_t x, int dtype) {
  // +0 and -0 are false, everything else (NaN included) is true
  if (dtype == MA_MASK_F32) x &= 0x7fffffffu;
  if (dtype == MA_MASK_F16 || dtype == MA_MASK_BF16) x &= 0x7fffu;
  return x != 0;
}

// NT * 8 query heads a pass, rows of at most DP values.
template <Elem K_, int NT_, int DP_>
struct Mma {
  static constexpr Elem K = K_;
  static constexpr int NT = NT_, DP = DP_, NC = NT * 8;
  static constexpr int kBytes = is_coded<K> ? 1 : 2;
  static constexpr bool kBf16 = K == Elem::bf16;
  static constexpr int kPiece = kTile * DP * kBytes;  // a tile's keys or values
  static constexpr int kScales = is_coded<K> ? 4 * kTile * 4 : 0;  // (keys, values) x 2 tiles
  static constexpr int kWarpBytes = 3 * kPiece + kScales;
  static constexpr int kKeyParts = DP * kBytes / 64;               // 16 bytes a lane each
  static constexpr int kValBytes = DP * kBytes >= 128 ? 16 : 8;    // a lane's part of a row
  static constexpr int kValParts = DP * kBytes / (8 * kValBytes);
  static constexpr int kSteps = DP / 16;
  static constexpr int OS = DP + 4;  // row of o in shared memory
  static constexpr int kOut = kWarps * kWarpBytes;
  static constexpr int kSmem = kOut + kWarps * NC * OS * 4 + kWarps * 2 * NC * 4;
  // as many CTAs as the rings leave room for, at most four
  static constexpr int kFit = 228 * 1024 / (kSmem + 1024 + 256);
  static constexpr int kMin = kFit < 1 ? 1 : kFit > 4 ? 4 : kFit;
};

// A warp's way along the tiles of its CTA's piece.
struct Walk {
  int e, r, tile, tiles, len;
  int64_t pos;
};

__device__ __forceinline__ void enter_row(const DecodeArgs& a, const Lengths& lens, Walk& w) {
  w.len = lens.of(a, w.e);
  w.tiles = row_tiles(w.len);
}

__device__ __forceinline__ void step(const DecodeArgs& a, const Lengths& lens, Walk& w, int n,
                                     int64_t end) {
  w.pos += n;
  if (w.pos >= end) return;
  w.tile += n;
  while (w.tile >= w.tiles) {
    w.tile -= w.tiles;
    if (++w.r == a.rows) {
      w.r = 0;
      ++w.e;
      enter_row(a, lens, w);
    }
  }
}

template <class M>
__global__ void __launch_bounds__(kThreads, M::kMin) decode_mma_kernel(const DecodeArgs a) {
  constexpr Elem K = M::K;
  constexpr int NT = M::NT, DP = M::DP, NC = M::NC;
  constexpr bool BF = M::kBf16;
  extern __shared__ __align__(16) char smem[];
  float* so = reinterpret_cast<float*>(smem + M::kOut);
  float* sm = so + kWarps * NC * M::OS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t ring = mmas::smem_u32(smem) + warp * M::kWarpBytes;
  const uint32_t scales = ring + 3 * M::kPiece;
  Piece p;
  Lengths lens;
  if (!find_piece(a, &p, &lens)) return;

  Walk w;  // the tile whose keys are loaded next
  w.e = p.e;
  w.r = p.r;
  w.tile = p.tile;
  w.pos = p.t0;
  enter_row(a, lens, w);
  step(a, lens, w, warp, p.t1);

  const int row_bytes = a.c.D * M::kBytes;
  int issue = 0, use = 0;      // pieces of the ring
  int parity_k = 0;            // tiles' halves of the scales
  uint32_t valid_next = 0, valid_now = 0;
  // this lane's token of the tile whose keys come next: its page's number and
  // its mask element as they lie in memory, asked for a tile ahead
  int page = -1;
  uint64_t mask = 0;
  int64_t value_at = 0;  // of the tile whose keys were loaded last

  const auto look_ahead = [&] {
    if (w.pos >= p.t1) return;
    const int pos = w.tile * kTile + lane;
    page = -1;
    if (pos < w.len) {
      page = load_now<int>(a.c.table + (int64_t)w.e * a.c.tstride[0] +
                           (int64_t)(pos / a.c.page_size) * a.c.tstride[1]);
      if (a.mask)
        mask = pos < a.mask_len ? load_mask(a.mask, a.mask_dtype, w.e * a.ms[0] + pos * a.ms[1]) : 0;
    }
  };
  const auto load_keys = [&] {
    valid_next = 0;
    if (w.pos < p.t1) {
      const CacheView& c = a.c;
      const int hk = w.r / a.groups, pos = w.tile * kTile + lane, slot = pos % c.page_size;
      bool in = pos < w.len;
      if (in && (unsigned)page >= (unsigned)c.num_pages) {
        cache_fail(c, MA_STATUS_BAD_PAGE);
        in = false;
      }
      if (a.mask) in = in && mask_bits(mask, a.mask_dtype);
      valid_next = __ballot_sync(0xffffffffu, in);
      const int64_t at_page = in ? page : 0;
      const int64_t key_at =
          (at_page * c.stride[0][0] + hk * c.stride[0][1] + slot * c.stride[0][2]) * M::kBytes;
      value_at = (at_page * c.stride[1][0] + hk * c.stride[1][1] + slot * c.stride[1][2]) * M::kBytes;
      const uint32_t at = ring + issue * M::kPiece + lane * 16;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const char* row = c.pages[0] + __shfl_sync(0xffffffffu, key_at, g + 8 * r);
        const bool ok = valid_next >> (g + 8 * r) & 1;
#pragma unroll
        for (int i = 0; i < M::kKeyParts; ++i) {
          const int off = i * 64 + t * 16;
          const int n = ok ? min(max(row_bytes - off, 0), 16) : 0;
          copy_async<16>(at + (r * M::kKeyParts + i) * 512, n ? row + off : c.pages[0], n);
        }
      }
      if constexpr (is_coded<K>) {
        const float* ks = c.scale[0] + at_page * c.sstride[0][0] + hk * c.sstride[0][1] +
                          slot * c.sstride[0][2];
        const float* vs = c.scale[1] + at_page * c.sstride[1][0] + hk * c.sstride[1][1] +
                          slot * c.sstride[1][2];
        copy_async<4>(scales + (parity_k * kTile + lane) * 4, in ? ks : c.scale[0], in ? 4 : 0);
        copy_async<4>(scales + ((2 + parity_k) * kTile + lane) * 4, in ? vs : c.scale[1], in ? 4 : 0);
      }
      parity_k ^= 1;
      step(a, lens, w, kWarps, p.t1);
      look_ahead();
    }
    issue = issue == 2 ? 0 : issue + 1;
    commit();
  };
  const auto load_values = [&] {
    if (valid_next) {
      const uint32_t at = ring + issue * M::kPiece + lane * M::kValBytes;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int key = 16 * (r >> 2) + 8 * ((r >> 1) & 1) + 2 * t + (r & 1);
        const char* row = a.c.pages[1] + __shfl_sync(0xffffffffu, value_at, key);
        const bool in = valid_next >> key & 1;
#pragma unroll
        for (int c = 0; c < M::kValParts; ++c) {
          const int off = (c * 8 + g) * M::kValBytes;
          const int n = in ? min(max(row_bytes - off, 0), M::kValBytes) : 0;
          copy_async<M::kValBytes>(at + (r * M::kValParts + c) * 32 * M::kValBytes,
                                   n ? row + off : a.c.pages[1], n);
        }
      }
    }
    issue = issue == 2 ? 0 : issue + 1;
    commit();
  };

  look_ahead();
  load_keys();
  load_values();
  valid_now = valid_next;
  load_keys();

  int64_t pos = p.t0, mine = p.t0 + warp;  // the row's first tile here, and the warp's next
  int e = p.e, r = p.r, tile = p.tile, parity = 0;
  while (pos < p.t1) {
    const int tiles = row_tiles(lens.of(a, e));
    const int n = (int)(tiles - tile < p.t1 - pos ? tiles - tile : p.t1 - pos);
    float m[NT][2], l[NT][2], mv[NT][2], o[DP / 16][NT][4];
    uint32_t q[M::kSteps][NT][2];
    float qscale[NT][2];
    const bool any = mine < pos + n;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[i][j] = mv[i][j] = -INFINITY;
        l[i][j] = 0.0f;
        qscale[i][j] = a.scale2;
      }
    if (any) {
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[i][j][x] = 0.0f;
      // q: column g of each 8 heads, in the order in which keys are held
      const int hk = r / a.groups, first = (r % a.groups) * NC;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int head = first + 8 * j + g;
        const bool in = head < a.G;
        const int64_t base = e * a.qs[0] + (int64_t)(hk * a.G + (in ? head : 0)) * a.qs[1];
        float x[M::kSteps][4], amax = 0.0f;
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = is_coded<K> ? s / 4 * 64 + t * 16 + s % 4 * 4 + i
                                      : s / 2 * 32 + t * 8 + s % 2 * 4 + i;
            x[s][i] = in && d < a.c.D ? load_dense(a.q, a.dtype, base + d * a.qs[2]) : 0.0f;
            amax = fmaxf(amax, fabsf(x[s][i]));
          }
        if constexpr (is_coded<K>) {
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          const uint32_t ex = min(max(__float_as_uint(amax) >> 23, 1u), 253u);
          const float down = __uint_as_float((254u - ex) << 23), up = __uint_as_float(ex << 23);
#pragma unroll
          for (int s = 0; s < M::kSteps; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[s][i] *= down;
          qscale[j][0] *= __shfl_sync(0xffffffffu, up, 8 * t);
          qscale[j][1] *= __shfl_sync(0xffffffffu, up, 8 * t + 4);
        }
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s) {
          q[s][j][0] = mmas::pack2<BF>(x[s][0], x[s][1]);
          q[s][j][1] = mmas::pack2<BF>(x[s][2], x[s][3]);
        }
      }
    }
    while (mine < pos + n) {
      // ---- scores: tokens g, g + 8 (+ 16 i) x heads 2t, 2t + 1 (+ 8 j)
      float s[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[i][j][x] = 0.0f;
      wait_but<2>();
      __syncwarp();
      {
        const uint32_t at = ring + use * M::kPiece + lane * 16;
#pragma unroll
        for (int c = 0; c < M::kKeyParts; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t x[4], y[4];
            load_shared<16>(at + ((2 * i) * M::kKeyParts + c) * 512, x);
            load_shared<16>(at + ((2 * i + 1) * M::kKeyParts + c) * 512, y);
            if constexpr (is_coded<K>) {
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                uint32_t x0, x1, y0, y1;
                widen<K>(x[h], x0, x1);
                widen<K>(y[h], y0, y1);
#pragma unroll
                for (int j = 0; j < NT; ++j)
                  mmas::mma16816<BF>(s[i][j], x0, y0, x1, y1, q[4 * c + h][j][0], q[4 * c + h][j][1]);
              }
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                  mmas::mma16816<BF>(s[i][j], x[2 * h], y[2 * h], x[2 * h + 1], y[2 * h + 1],
                                     q[2 * c + h][j][0], q[2 * c + h][j][1]);
            }
          }
      }
      use = use == 2 ? 0 : use + 1;
      const uint32_t valid = valid_now;
      load_values();  // of the next tile, where these keys were
      valid_now = valid_next;

      // ---- running maximum, weights and their sum
      float vs[4], top[NT][2], topv[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) top[j][0] = top[j][1] = topv[j][0] = topv[j][1] = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // token g + 8 k
        float ks = 1.0f;
        if constexpr (is_coded<K>) {
          ks = load_shared_f(scales + (parity * kTile + g + 8 * k) * 4);
          vs[k] = log2f(load_shared_f(scales + ((2 + parity) * kTile + g + 8 * k) * 4));
        }
        const bool in = valid >> (g + 8 * k) & 1;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float& z = s[k >> 1][j][2 * (k & 1) + x];
            z = in ? z * (qscale[j][x] * ks) : -INFINITY;
            top[j][x] = fmaxf(top[j][x], z);
            if constexpr (is_coded<K>) topv[j][x] = fmaxf(topv[j][x], in ? z + vs[k] : -INFINITY);
          }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float mm = top[j][x];
          mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 4));
          mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 8));
          mm = fmaxf(fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 16)), m[j][x]);
          const float c = weight(m[j][x], mm);
          m[j][x] = mm;
          l[j][x] *= c;
          float cv = c;
          if constexpr (is_coded<K>) {
            float mt = topv[j][x];
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
            mt = fmaxf(fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16)), mv[j][x]);
            cv = weight(mv[j][x], mt);
            mv[j][x] = mt;
          }
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) {
            o[i][j][x] *= cv;
            o[i][j][2 + x] *= cv;
          }
        }
      uint32_t ph[2][NT][2], pl[2][NT][2];  // the weights' halves, heads x tokens
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float pv[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float z = s[k >> 1][j][2 * (k & 1) + x];
            const float pr = z == -INFINITY ? 0.0f : ex2f(z - m[j][x]);
            l[j][x] += pr;
            pv[x] = pr;
            if constexpr (is_coded<K>) {
              const float zv = z + vs[k];
              pv[x] = z == -INFINITY || zv == -INFINITY ? 0.0f : ex2f(zv - mv[j][x]);
            }
          }
          const uint32_t hi = mmas::pack2<BF>(pv[0], pv[1]);
          float h0, h1;
          if constexpr (BF) {
            h0 = __uint_as_float(hi << 16);
            h1 = __uint_as_float(hi & 0xffff0000u);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            h0 = f.x;
            h1 = f.y;
          }
          ph[k >> 1][j][k & 1] = transpose8(hi);
          pl[k >> 1][j][k & 1] = transpose8(mmas::pack2<BF>(pv[0] - h0, pv[1] - h1));
        }

      // ---- output: dimensions x heads
      wait_but<2>();
      __syncwarp();
      if (valid) {
        const uint32_t at = ring + use * M::kPiece + lane * M::kValBytes;
        constexpr int R = M::kValBytes / 4;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < M::kValParts; ++c) {
            uint32_t v[4][R];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int x = 0; x < 4; ++x)
              load_shared<M::kValBytes>(
                  at + ((4 * i + x) * M::kValParts + c) * 32 * M::kValBytes, v[x]);
#pragma unroll
            for (int h = 0; h < R; ++h) {
              if constexpr (is_coded<K>) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  uint32_t a0, a1, a2, a3;
                  widen<K>(prmt(v[0][h], v[1][h], y ? 0x7362u : 0x5140u), a0, a1);
                  widen<K>(prmt(v[2][h], v[3][h], y ? 0x7362u : 0x5140u), a2, a3);
#pragma unroll
                  for (int j = 0; j < NT; ++j) {
                    float(&d)[4] = o[(c * R + h) * 2 + y][j];
                    mmas::mma16816<BF>(d, a0, a1, a2, a3, ph[i][j][0], ph[i][j][1]);
                    mmas::mma16816<BF>(d, a0, a1, a2, a3, pl[i][j][0], pl[i][j][1]);
                  }
                }
              } else {
                const uint32_t a0 = prmt(v[0][h], v[1][h], 0x5410u), a1 = prmt(v[0][h], v[1][h], 0x7632u);
                const uint32_t a2 = prmt(v[2][h], v[3][h], 0x5410u), a3 = prmt(v[2][h], v[3][h], 0x7632u);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                  float(&d)[4] = o[c * R + h][j];
                  mmas::mma16816<BF>(d, a0, a1, a2, a3, ph[i][j][0], ph[i][j][1]);
                  mmas::mma16816<BF>(d, a0, a1, a2, a3, pl[i][j][0], pl[i][j][1]);
                }
              }
            }
          }
      }
      use = use == 2 ? 0 : use + 1;
      parity ^= 1;
      mine += kWarps;
      load_keys();  // of the tile after the next, where these values were
    }

    // ---- the row's end: (m, l, o) to shared memory
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float ls = l[j][x];
        ls += __shfl_xor_sync(0xffffffffu, ls, 4);
        ls += __shfl_xor_sync(0xffffffffu, ls, 8);
        ls += __shfl_xor_sync(0xffffffffu, ls, 16);
        const int col = 8 * j + 2 * t + x;
        if (g == 0) {
          sm[warp * 2 * NC + col] = m[j][x];
          sm[warp * 2 * NC + NC + col] = ls;
        }
        if (any) {
          // o is relative to M where values have scales
          const float f = is_coded<K> ? weight(mv[j][x], m[j][x]) : 1.0f;
          float* dst = so + (warp * NC + col) * M::OS;
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) {
            // the values' order: see the loads above
            constexpr int per = M::kValBytes / M::kBytes / 2;  // products a lane's part feeds
            const int d = (i / per * 8 + g) * (2 * per) + i % per * 2;
            *reinterpret_cast<float2*>(dst + d) = make_float2(o[i][j][x] * f, o[i][j][2 + x] * f);
          }
        }
      }
    __syncthreads();
    end_row<NC, DP, M::OS>(a, p, e, r, tile, tiles, n, pos, sm, so);
    __syncthreads();
    pos += n;
    tile = 0;
    if (++r == a.rows) {
      r = 0;
      ++e;
    }
  }
}

template <class M>
cudaError_t launch(DecodeArgs a, cudaStream_t st) {
  a.groups = (a.G + M::NC - 1) / M::NC;
  a.rows = a.c.Hk * a.groups;
  static Resident known;
  const int grid = grid_size(a, decode_mma_kernel<M>, M::kSmem, known);
  if (grid < 1) return cudaErrorInvalidDevice;
  decode_mma_kernel<M><<<grid, kThreads, M::kSmem, st>>>(a);
  return cudaGetLastError();
}

template <Elem K>
cudaError_t launch_dim(const DecodeArgs& a, cudaStream_t st) {
  // 16 heads a pass where more than 8 share a kv head and o fits the registers
  if (a.c.D <= 64) return a.G > 8 ? launch<Mma<K, 2, 64>>(a, st) : launch<Mma<K, 1, 64>>(a, st);
  if (a.c.D <= 128) return a.G > 8 ? launch<Mma<K, 2, 128>>(a, st) : launch<Mma<K, 1, 128>>(a, st);
  return launch<Mma<K, 1, 256>>(a, st);
}

}  // namespace

cudaError_t run_decode_mma(const DecodeArgs& a, Elem pages, cudaStream_t st) {
  switch (pages) {
    case Elem::f16: return launch_dim<Elem::f16>(a, st);
    case Elem::bf16: return launch_dim<Elem::bf16>(a, st);
    case Elem::e4m3: return launch_dim<Elem::e4m3>(a, st);
    case Elem::i8: return launch_dim<Elem::i8>(a, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace ma
