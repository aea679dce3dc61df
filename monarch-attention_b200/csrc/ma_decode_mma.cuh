// One-token attention for 16-bit queries (ma_decode, include/ma_api.h), on
// the tensor cores; compiled for one type of pages each (ma_decode_inst_*.cu).
// Mathematics, work split and joins: ma_decode.cuh.
//
// HBM bounds it; the products are there to keep the arithmetic out of the
// way.  With 8 query heads on a kv head, fp32 FMAs would need 16 a cached
// value where an SM has time for about 10 (16-bit pages; 5 for 8-bit ones); m16n8k16
// products with the tokens (scores) or the values' dimensions (output) as the
// 16 rows and the query heads as the 8 columns need 1/128th of the instructions.
//
// A warp works alone on tiles of 32 tokens, and no barrier stands between load and use
// (cp.async, then a warp's own fence).
//   16-bit rows  row by row, their 16-byte chunks swizzled, and read as 8x8 matrices:
//            keys as they lie, values transposed, without a bank conflict
//   codes    each lane copies exactly the bytes that it will feed to the products itself:
//     keys     lane (g, t) holds rows g, g + 8, ... at bytes 16 t of each 64: the sum
//              over dimensions may run in any order, so they need not be the k
//              index that the product names, only q's fragments the same
//     values   lane (g, t) holds rows 2t, 2t+1, 2t+8, 2t+9 (the product's k index)
//              at bytes 16 g of each 128 (8 g of each 64 in rows of 64); byte permutes
//              pair two tokens' values
// Three pieces of a ring (keys, values, next keys) keep two of them in flight.
//
// Weights p = 2^(s - m) are fed in two 16-bit halves (rounded, and what the
// rounding left): with one, its rounding would be as large as the result's own.
// fp16 halves end at 2^-24, where a row of many small weights beside one large one would lose
// them: there m lies kLift below the maximum, so that they reach to the top of fp16's range.
// fp16 pages' second halves go in kUp times as large, with sums of their own, so that a weight
// is right to 2^-44 of the largest: the token that has it may hold values near zero.  (Codes
// need no such sums: their weights are relative to the largest product with a scale, below.
// The sums cost 4 FMAs a product of 5 to 16 heads, 0 to 3 % of a call's time: 64 sequences of 256 to
// 4096 fp16 tokens, 128 heads on 8 of 128, 133 us without, 136 with; 4 heads have their
// second halves in columns of their own.)
// e4m3 and int8 codes become fp16 exactly; a key's scale multiplies its score.
// A value's scale v_s joins its weight as 2^(s + log2 v_s - M) with a running maximum M of its
// own (the largest product of weight and scale), so the fp16 weights stay in range whatever the
// scales, and are right to 2^-33 of the largest product.
// q becomes fp16 with its largest value at the top of fp16's range.
//
// Measured (B200): 4 x 65536 bf16 tokens, 16 heads of 128, 323 us (6.6 TB/s); 64
// sequences of 256 to 4096 e4m3 tokens, 32 heads on 8 of 128, 77 us (4.1 TB/s of
// what they hold; while tiles run, a tile an SM and 197 ns, 6.3); 4 sequences of
// 4096 to 8192 fp16 tokens, 12 heads of 64, 23 us (3.3 TB/s); a single tile a
// row 5 us.  The forms for codes are held to kMin CTAs an SM and spill up to 92 bytes
// a thread there (40 with 4 heads of 128 in blocks).
#pragma once

#include <type_traits>

#include "ma_decode.cuh"
#include "ma_mma_sync.cuh"

namespace ma {

using namespace decode;

namespace {

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
  return __byte_perm(a, b, s);
}

// The 8x8 matrix of 16-bit elements whose rows' pairs the lanes hold, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The m16n8k16 product, for the compiler to place (mmas::mma16816 keeps its order).
template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// A 16-bit element of q (of either type: the products take fp16 for codes).
__device__ __forceinline__ float widen_q(uint32_t bits, bool bf16) {
  return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
}

// NH query heads a pass (4, 8 or 16), rows of at most DP values.  WHOLE: every
// row has DP values, a page's rows of a head follow each other without a gap and
// no tile crosses a page's end, so a tile is one block of memory.  ROW: a CTA with
// twice the warps (four times where 128 registers do) takes one row.
template <Elem K_, int NH_, int DP_, bool WHOLE_, bool ROW_>
struct Mma {
  static constexpr Elem K = K_;
  static constexpr int DP = DP_, NC = NH_;
  static constexpr bool WHOLE = WHOLE_, ROW = ROW_;
  static constexpr int W = !ROW ? kWarps : DP == 64 && NH_ < 16 ? 4 * kWarps : 2 * kWarps;
  // Columns of the products.  4 heads have their weights' second halves in the
  // other 4 columns; more take a second product for them.
  static constexpr int NT = NC > 8 ? 2 : 1;
  static constexpr bool kTwins = NC == 4;
  static constexpr int kBytes = is_coded<K> ? 1 : 2;
  static constexpr bool kBf16 = K == Elem::bf16;
  // fp16 weights are relative to what lies kLift below a maximum, and that moves when a score
  // exceeds it by kOver: they reach 2^15.  bf16 ones have fp32's range.
  static constexpr float kLift = kBf16 ? 0.0f : 9.0f, kOver = kSlack + kLift;
  // Second halves of fp16 pages' weights go in kUp (an fp16's bits) times as large: at most as
  // large as the first ones.
  static constexpr bool kApart = K == Elem::f16;
  static constexpr float kUp = kApart ? 2048.0f : 1.0f, kDown = kApart ? 1.0f / 2048.0f : 1.0f;
  static constexpr int kRow = DP * kBytes;
  static constexpr int kPiece = kTile * kRow;  // a tile's keys or values
  static constexpr int kScales = is_coded<K> ? 4 * kTile * 4 : 0;  // (keys, values) x 2 tiles
  static constexpr int kWarpBytes = 3 * kPiece + kScales;
  static constexpr int kSteps = DP / 16;
  // 16-bit rows: lanes that copy one, rows a copy instruction takes
  static constexpr int kRowLanes = kRow / 16 < 32 ? kRow / 16 : 32;
  static constexpr int kRowsAtOnce = 32 / kRowLanes;
  // codes: 16 bytes a lane and part of a row for keys, kValBytes for values
  static constexpr int kKeyParts = kRow / 64;
  static constexpr int kValBytes = kRow >= 128 ? 16 : 8;
  static constexpr int kValParts = kRow / (8 * kValBytes);
  // Row of o in shared memory, with a shift in the banks where that does not cost
  // a CTA its place on the SM.
  static constexpr int OS = DP == 128 && NC == 8 && !is_coded<K> ? DP : DP + 4;
  static constexpr int kOut = W * kWarpBytes;
  static constexpr int kSmem = kOut + W * NC * OS * 4 + W * 2 * NC * 4;
  static constexpr bool kFits = kSmem + 512 <= 227 * 1024;
  // as many CTAs as the rings leave room for, at most four (three where 128
  // registers would not do)
  static constexpr int kFit = 228 * 1024 / (kSmem + 1024 + 512);
  static constexpr int kMost = is_coded<K> && NC == 16 ? 3 : 4;
  static constexpr int kMin = ROW || kFit < 1 ? 1 : kFit > kMost ? kMost : kFit;

  // kLift below a maximum, or the maximum itself where that would be rounded.
  static __device__ __forceinline__ float below(float top) {
    if (kLift == 0.0f) return top;
    const float b = top - kLift;
    return top - b == kLift ? b : top;
  }
};

// A lane's pairs of q, element by element: any stride and alignment.
template <class M>
__device__ __forceinline__ void load_q_singly(const DecodeArgs& a, const uint16_t* qp, int t,
                                           uint32_t (&u)[M::kSteps][2]) {
#pragma unroll
  for (int s = 0; s < M::kSteps; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = is_coded<M::K> ? s / 4 * 64 + t * 16 + s % 4 * 4 + i
                                   : s * 16 + t * 2 + (i & 1) + (i >> 1) * 8;
      if (d < a.c.D) u[s][i >> 1] |= (uint32_t)qp[d * a.qs[2]] << (16 * (i & 1));
    }
}

// A warp's way along the tiles of its CTA's piece.
struct Walk {
  int e, r, tile, tiles, len;
  int64_t start;  // of the row, from the piece's start
  bool done;
};

template <class L>
__device__ __forceinline__ void enter_row(const DecodeArgs& a, const L& lens, Walk& w) {
  w.len = lens.of(a, w.e);
  w.tiles = row_tiles(w.len);
}

template <class L>
__device__ __forceinline__ void step(const DecodeArgs& a, const L& lens, const Piece& p, Walk& w,
                                     int n) {
  w.tile += n;
  while (w.tile >= w.tiles) {
    w.tile -= w.tiles;
    w.start += w.tiles + p.cost;
    if (w.start >= p.end) {
      w.done = true;
      return;
    }
    if (++w.r == a.rows) {
      w.r = 0;
      ++w.e;
      enter_row(a, lens, w);
    }
  }
  w.done = w.tile >= tiles_before_end(p, w.start, w.tiles);
}

template <class M>
__global__ void __launch_bounds__(M::W * 32, M::kMin) decode_mma_kernel(const DecodeArgs a) {
  constexpr Elem K = M::K;
  constexpr int NT = M::NT, DP = M::DP, NC = M::NC, W = M::W;
  constexpr bool BF = M::kBf16, CODED = is_coded<K>;
  constexpr uint32_t kAll = 0xffffffffu;
  extern __shared__ __align__(128) char smem[];
  float* so = reinterpret_cast<float*>(smem + M::kOut);
  float* sm = so + W * NC * M::OS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t ring = mmas::smem_u32(smem) + warp * M::kWarpBytes;
  const uint32_t scales = ring + 3 * M::kPiece;
  const CacheView& c = a.c;
  wait_for_earlier();
  Piece p;
  typename std::conditional<M::ROW, RowLength, Lengths>::type lens;
  if (!find_piece(a, &p, &lens)) return;

  Walk w;  // the tile whose keys are loaded next
  w.e = p.e;
  w.r = p.r;
  w.tile = p.tile;
  w.start = p.start;
  enter_row(a, lens, w);
  step(a, lens, p, w, warp);

  const int row_bytes = M::WHOLE ? M::kRow : c.D * M::kBytes;

  // ---- loads: the three pieces of the ring are filled in turn
  int issue = 0, use = 1;
  int half = 0;  // of the scales, for the next tile to load
  uint32_t valid_next = 0, valid_now = 0;
  // this lane's token of the tile whose keys come next: its page's number and
  // its mask element as they lie in memory, asked for a tile ahead
  int page = -1;
  uint64_t mask = 0;
  // where the values of the tile lie whose keys were loaded last: this lane's
  // token (WHOLE: the first token)
  int64_t value_at = 0;

  const auto look_ahead = [&] {
    if (w.done) return;
    const int pos = w.tile * kTile + lane;
    page = -1;
    if (pos < w.len) {
      page = load_now<int>(c.table + (int64_t)w.e * c.tstride[0] +
                           (int64_t)page_index(c, pos) * c.tstride[1]);
      if (a.mask)
        mask = pos < a.mask_len ? load_mask(a.mask, a.mask_dtype, w.e * a.ms[0] + pos * a.ms[1]) : 0;
    }
  };
  // Row i of a tile whose rows (WHOLE: first row) lie at `at` bytes.
  const auto row_of = [&](int which, int64_t at, int i) {
    return c.pages[which] + (M::WHOLE ? at + i * M::kRow : __shfl_sync(kAll, at, i));
  };
  // 16-bit rows, row by row, the 16-byte chunks of row i at chunk ^ (i % 8):
  // eight rows' equal chunks, which a matrix load takes at once, lie in
  // different banks
  const auto copy_rows = [&](int which, int64_t at) {
    const int sub = lane / M::kRowLanes, chunk = lane % M::kRowLanes;
    const uint32_t dst = ring + issue * M::kPiece + sub * M::kRow;
    const auto to = [&](int i) {
      return dst + i * M::kRowsAtOnce * M::kRow + ((chunk ^ ((i * M::kRowsAtOnce + sub) & 7)) * 16);
    };
    if (M::WHOLE && valid_next == kAll) {
      const char* src = c.pages[which] + at + lane * 16;
#pragma unroll
      for (int i = 0; i < kTile / M::kRowsAtOnce; ++i)
        copy_async<16>(to(i), src + i * M::kRowsAtOnce * M::kRow, 16);
    } else {
      const int most = M::WHOLE ? 16 : min(max(row_bytes - chunk * 16, 0), 16);
      const int64_t off = most > 0 ? chunk * 16 : 0;
#pragma unroll
      for (int i = 0; i < kTile / M::kRowsAtOnce; ++i) {
        const int row = i * M::kRowsAtOnce + sub;
        copy_async<16>(to(i), row_of(which, at, row) + off, valid_next >> row & 1 ? most : 0);
      }
    }
  };
  // Codes, each lane the bytes that it feeds to the products: B of each 4 B (keys)
  // or 8 B (values) of a row.
  const auto copy_part = [&](auto bytes, uint32_t dst, const char* row, int off, int part_end, bool in) {
    constexpr int B = decltype(bytes)::value;
    if (M::WHOLE || part_end <= row_bytes) {
      copy_async<B>(dst, row + off, in ? B : 0);
    } else {  // zero behind the row's end
      const int n = in ? min(max(row_bytes - off, 0), B) : 0;
      copy_async<B>(dst, n ? row + off : row, n);
    }
  };
  const auto copy_key_codes = [&](int64_t at) {
    const uint32_t dst = ring + issue * M::kPiece + lane * 16;
    if (M::WHOLE && valid_next == kAll) {
      const char* src = c.pages[0] + at + g * M::kRow + t * 16;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int x = 0; x < M::kKeyParts; ++x)
          copy_async<16>(dst + (r * M::kKeyParts + x) * 512, src + r * 8 * M::kRow + x * 64, 16);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = g + 8 * r;
        const char* row = row_of(0, at, i);
#pragma unroll
        for (int x = 0; x < M::kKeyParts; ++x)
          copy_part(std::integral_constant<int, 16>{}, dst + (r * M::kKeyParts + x) * 512, row,
                    x * 64 + t * 16, x * 64 + 64, valid_next >> i & 1);
      }
    }
  };
  const auto copy_value_codes = [&](int64_t at) {
    constexpr int B = M::kValBytes;
    const uint32_t dst = ring + issue * M::kPiece + lane * B;
    if (M::WHOLE && valid_next == kAll) {
      const char* src = c.pages[1] + at + 2 * t * M::kRow + g * B;
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int x = 0; x < M::kValParts; ++x)
          copy_async<B>(dst + (r * M::kValParts + x) * 32 * B,
                        src + (16 * (r >> 2) + 8 * ((r >> 1) & 1) + (r & 1)) * M::kRow + x * 8 * B, B);
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int i = 16 * (r >> 2) + 8 * ((r >> 1) & 1) + 2 * t + (r & 1);
        const char* row = row_of(1, at, i);
#pragma unroll
        for (int x = 0; x < M::kValParts; ++x)
          copy_part(std::integral_constant<int, B>{}, dst + (r * M::kValParts + x) * 32 * B, row,
                    (x * 8 + g) * B, (x * 8 + 8) * B, valid_next >> i & 1);
      }
    }
  };
  const auto load_keys = [&] {
    valid_next = 0;
    if (!w.done) {
      const int hk = a.groups == 1 ? w.r : w.r / a.groups, pos = w.tile * kTile + lane;
      const int slot = pos - page_index(c, pos) * c.page_size;
      bool in = pos < w.len;
      if (a.mask) in = in && mask_bits(mask, a.mask_dtype);  // first: a masked token's page may be gone
      if (in && (unsigned)page >= (unsigned)c.num_pages) {
        cache_fail(c, MA_STATUS_BAD_PAGE);
        in = false;
      }
      valid_next = __ballot_sync(kAll, in);
      if (valid_next) {
        int64_t at_page = in ? page : 0;
        int at_slot = slot;
        if constexpr (CODED) {
          const float* ks = c.scale[0] + at_page * c.sstride[0][0] + hk * c.sstride[0][1] +
                            slot * c.sstride[0][2];
          const float* vs = c.scale[1] + at_page * c.sstride[1][0] + hk * c.sstride[1][1] +
                            slot * c.sstride[1][2];
          copy_async<4>(scales + (half * kTile + lane) * 4, in ? ks : c.scale[0], in ? 4 : 0);
          copy_async<4>(scales + ((2 + half) * kTile + lane) * 4, in ? vs : c.scale[1], in ? 4 : 0);
        }
        if constexpr (M::WHOLE) {  // one page, named by any valid token
          at_page = __shfl_sync(kAll, page, __ffs(valid_next) - 1);
          at_slot = slot - lane;
        }
        const int64_t key_at =
            (at_page * c.stride[0][0] + hk * c.stride[0][1] + at_slot * c.stride[0][2]) * M::kBytes;
        value_at =
            (at_page * c.stride[1][0] + hk * c.stride[1][1] + at_slot * c.stride[1][2]) * M::kBytes;
        if constexpr (CODED) copy_key_codes(key_at);
        else copy_rows(0, key_at);
      }
      half ^= 1;
      step(a, lens, p, w, W);
      look_ahead();
    }
    issue = issue == 2 ? 0 : issue + 1;
    commit();
  };
  const auto load_values = [&] {
    if (valid_next) {
      if constexpr (CODED) copy_value_codes(value_at);
      else copy_rows(1, value_at);
    }
    issue = issue == 2 ? 0 : issue + 1;
    commit();
  };

  look_ahead();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {  // nothing and keys 0, values 0 and keys 1
    load_values();
    valid_now = valid_next;
    load_keys();
  }
  int e = p.e, r = p.r, tile = p.tile, use_half = 0;
  int skip = warp;  // tiles of the row here before the warp's next one
  int64_t start = p.start;
  Left left;
  // the row's q as it lies in memory, the next row's asked for at this one's end:
  // pairs of column g of each 8, in the order in which keys are fed
  uint32_t raw[NT][M::kSteps][2];
  const auto load_q = [&](int e, int r) {
    const int hk = r / a.groups, first = (r % a.groups) * NC;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int head = first + 8 * j + (M::kTwins ? g & 3 : g);
      const bool in = head < a.G;
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + e * a.qs[0] +
                           (int64_t)(hk * a.G + (in ? head : 0)) * a.qs[1];
#pragma unroll
      for (int s = 0; s < M::kSteps; ++s) raw[j][s][0] = raw[j][s][1] = 0;
      if (!a.qvec || (!M::WHOLE && (c.D & 15))) {
        if (in) load_q_singly<M>(a, qp, t, raw[j]);
      } else if (!in) {
        // zero
      } else if constexpr (CODED) {
#pragma unroll
        for (int s = 0; s < M::kSteps; s += 4) {
          const int d = s * 16 + t * 16;
          if (M::WHOLE || d < c.D) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(qp + d));
            const uint4 w4 = __ldg(reinterpret_cast<const uint4*>(qp + d + 8));
            raw[j][s][0] = v.x;
            raw[j][s][1] = v.y;
            raw[j][s + 1][0] = v.z;
            raw[j][s + 1][1] = v.w;
            raw[j][s + 2][0] = w4.x;
            raw[j][s + 2][1] = w4.y;
            raw[j][s + 3][0] = w4.z;
            raw[j][s + 3][1] = w4.w;
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s)
          if (M::WHOLE || s * 16 < c.D) {
            raw[j][s][0] = __ldg(reinterpret_cast<const uint32_t*>(qp + s * 16 + t * 2));
            raw[j][s][1] = __ldg(reinterpret_cast<const uint32_t*>(qp + s * 16 + t * 2 + 8));
          }
      }
    }
  };
  load_q(e, r);
  for (;;) {
    const int tiles = row_tiles(lens.of(a, e));
    const int n = tiles_before_end(p, start, tiles) - tile;
    if (n <= 0) break;
    float m[NT][2], l[NT][2], mv[NT][2], o[DP / 16][NT][4];
    uint32_t q[M::kSteps][NT][2];
    float qscale[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[i][j] = mv[i][j] = -INFINITY;
        l[i][j] = 0.0f;
      }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][j][x] = 0.0f;
    // q as the products take it
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if constexpr (CODED) {
        const bool bf = a.dtype == MA_DTYPE_BF16;
        float amax = 0.0f;
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            amax = fmaxf(amax, fmaxf(fabsf(widen_q(raw[j][s][i] & 0xffffu, bf)),
                                     fabsf(widen_q(raw[j][s][i] >> 16, bf))));
        amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, 2));
        // largest value in [2^15, 2^16): fp16 queries never lose a bit, and bf16 ones only below
        // 2^-32 of it (2^-40 become 0)
        const uint32_t ex = min(max(__float_as_uint(amax) >> 23, 16u), 254u);
        const float to = __uint_as_float((269u - ex) << 23), back = __uint_as_float((ex - 15u) << 23);
        qscale[j][0] = a.scale2 * __shfl_sync(kAll, back, 8 * t);
        qscale[j][1] = a.scale2 * __shfl_sync(kAll, back, 8 * t + 4);
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            q[s][j][i] = mmas::pack2<false>(widen_q(raw[j][s][i] & 0xffffu, bf) * to,
                                            widen_q(raw[j][s][i] >> 16, bf) * to);
      } else {
#pragma unroll
        for (int s = 0; s < M::kSteps; ++s) {
          q[s][j][0] = raw[j][s][0];
          q[s][j][1] = raw[j][s][1];
        }
      }
    }
    for (; skip < n; skip += W) {
      float s[2][NT][4];
      {
        // ---- scores: tokens g, g + 8 (+ 16 i) x heads 2t, 2t + 1 (+ 8 j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[i][j][x] = 0.0f;
        wait_but<2>();
        __syncwarp();
        if constexpr (CODED) {
          const uint32_t at = ring + use * M::kPiece + lane * 16;
#pragma unroll
          for (int x0 = 0; x0 < M::kKeyParts; x0 += 2) {
            constexpr int X = M::kKeyParts < 2 ? 1 : 2;  // parts at hand at a time
            uint32_t u[X][2][4], v[X][2][4];
#pragma unroll
            for (int x = 0; x < X; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                load_shared<16>(at + ((2 * i) * M::kKeyParts + x0 + x) * 512, u[x][i]);
                load_shared<16>(at + ((2 * i + 1) * M::kKeyParts + x0 + x) * 512, v[x][i]);
              }
#pragma unroll
            for (int x = 0; x < X; ++x)
#pragma unroll
              for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  uint32_t u0, u1, v0, v1;
                  widen<K>(u[x][i][h], u0, u1);
                  widen<K>(v[x][i][h], v0, v1);
#pragma unroll
                  for (int j = 0; j < NT; ++j)
                    mma<BF>(s[i][j], u0, v0, u1, v1, q[4 * (x0 + x) + h][j][0], q[4 * (x0 + x) + h][j][1]);
                }
          }
        } else {
          // matrices: (tokens 0-7, 8-15) x (dimensions 0-7, 8-15)
          const uint32_t at = ring + use * M::kPiece + (lane & 15) * M::kRow;
          const uint32_t x0 = (lane >> 4) ^ (lane & 7);
#pragma unroll
          for (int h = 0; h < M::kSteps; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t u[4];
              mmas::ldsm_x4(at + i * 16 * M::kRow + ((x0 ^ (2 * h)) * 16), u[0], u[1], u[2], u[3]);
#pragma unroll
              for (int j = 0; j < NT; ++j)
                mma<BF>(s[i][j], u[0], u[1], u[2], u[3], q[h][j][0], q[h][j][1]);
            }
        }
        use = use == 2 ? 0 : use + 1;
        __syncwarp();  // every lane has read these keys
      }
      const uint32_t valid = valid_now;
      load_values();  // of the next tile, where these keys were
      valid_now = valid_next;

      {
        // ---- running maximum, weights and their sum
        float ls[4], top[NT][2], topv[NT][2];  // ls: log2 of the values' scales
        if constexpr (CODED) {
          const float ks = load_shared_f(scales + (use_half * kTile + lane) * 4);
          const float lv = log2f(load_shared_f(scales + ((2 + use_half) * kTile + lane) * 4));
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // token g + 8 k
            const float f = __shfl_sync(kAll, ks, g + 8 * k);
            ls[k] = __shfl_sync(kAll, lv, g + 8 * k);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int x = 0; x < 2; ++x) s[k >> 1][j][2 * (k & 1) + x] *= qscale[j][x] * f;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) s[i][j][x] *= a.scale2;
        }
        if (valid != kAll) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (!(valid >> (g + 8 * k) & 1)) {
#pragma unroll
              for (int j = 0; j < NT; ++j)
                s[k >> 1][j][2 * (k & 1)] = s[k >> 1][j][2 * (k & 1) + 1] = -INFINITY;
            }
        }
        // m (and M) need only be near the maximum, or where fp16 weights' range wants them:
        // they move, and o with them, when a score exceeds them by kOver
        float over = -INFINITY;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float z = -INFINITY, zv = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              z = fmaxf(z, s[k >> 1][j][2 * (k & 1) + x]);
              if constexpr (CODED) zv = fmaxf(zv, s[k >> 1][j][2 * (k & 1) + x] + ls[k]);
            }
            top[j][x] = z;
            topv[j][x] = zv;
            over = fmaxf(over, z - m[j][x]);
            if constexpr (CODED) over = fmaxf(over, zv - mv[j][x]);
          }
        if (__any_sync(kAll, over > M::kOver)) {
#pragma unroll
          for (int d = 4; d < 32; d *= 2)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                top[j][x] = fmaxf(top[j][x], __shfl_xor_sync(kAll, top[j][x], d));
                if constexpr (CODED) topv[j][x] = fmaxf(topv[j][x], __shfl_xor_sync(kAll, topv[j][x], d));
              }
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float z = fmaxf(CODED ? top[j][x] : M::below(top[j][x]), m[j][x]);
              float f = weight(m[j][x], z);
              l[j][x] *= f;
              m[j][x] = z;
              if constexpr (CODED) {
                const float zv = fmaxf(M::below(topv[j][x]), mv[j][x]);
                f = weight(mv[j][x], zv);
                mv[j][x] = zv;
              }
#pragma unroll
              for (int i = 0; i < DP / 16; ++i) {
                o[i][j][x] *= f;
                o[i][j][2 + x] *= f;
              }
            }
        }
        float from[NT][2], fromv[NT][2];  // no valid token yet: any finite one
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            from[j][x] = m[j][x] == -INFINITY ? 0.0f : m[j][x];
            fromv[j][x] = mv[j][x] == -INFINITY ? 0.0f : mv[j][x];
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
              pv[x] = ex2f(z - from[j][x]);
              l[j][x] += pv[x];
              if constexpr (CODED) pv[x] = ex2f(z + ls[k] - fromv[j][x]);
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
            const uint32_t lo = mmas::pack2<BF>((pv[0] - h0) * M::kUp, (pv[1] - h1) * M::kUp);
            if constexpr (M::kTwins) {
              ph[k >> 1][j][k & 1] = transpose8(t < 2 ? hi : lo);
            } else {
              ph[k >> 1][j][k & 1] = transpose8(hi);
              pl[k >> 1][j][k & 1] = transpose8(lo);
            }
          }

        // ---- output: dimensions x heads
        wait_but<2>();
        __syncwarp();
        const auto product = [&](float(&d)[4], const uint32_t(&u)[4], int i, int j) {
          if constexpr (!M::kTwins && M::kApart) {
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma<BF>(x, u[0], u[1], u[2], u[3], pl[i][j][0], pl[i][j][1]);
#pragma unroll
            for (int y = 0; y < 4; ++y) d[y] = fmaf(x[y], M::kDown, d[y]);
          }
          mma<BF>(d, u[0], u[1], u[2], u[3], ph[i][j][0], ph[i][j][1]);
          if constexpr (!M::kTwins && !M::kApart)
            mma<BF>(d, u[0], u[1], u[2], u[3], pl[i][j][0], pl[i][j][1]);
        };
        if (!valid) {
          // nothing was loaded
        } else if constexpr (CODED) {
          const uint32_t at = ring + use * M::kPiece + lane * M::kValBytes;
          constexpr int R = M::kValBytes / 4;
#pragma unroll
          for (int x = 0; x < M::kValParts; ++x) {
            uint32_t v[2][4][R];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9 (+ 16 i)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                load_shared<M::kValBytes>(
                    at + ((4 * i + y) * M::kValParts + x) * 32 * M::kValBytes, v[i][y]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int h = 0; h < R; ++h)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  uint32_t u[4];
                  widen<K>(prmt(v[i][0][h], v[i][1][h], y ? 0x7362u : 0x5140u), u[0], u[1]);
                  widen<K>(prmt(v[i][2][h], v[i][3][h], y ? 0x7362u : 0x5140u), u[2], u[3]);
#pragma unroll
                  for (int j = 0; j < NT; ++j) product(o[(x * R + h) * 2 + y][j], u, i, j);
                }
          }
        } else {
          // matrices, transposed: (dimensions 0-7, 8-15) x (tokens 0-7, 8-15)
          const uint32_t at =
              ring + use * M::kPiece + ((lane & 7) + (lane >> 4) * 8) * M::kRow;
          const uint32_t x0 = ((lane >> 3) & 1) ^ (lane & 7);
#pragma unroll
          for (int h = 0; h < M::kSteps; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t u[4];
              mmas::ldsm_x4_t(at + i * 16 * M::kRow + ((x0 ^ (2 * h)) * 16), u[0], u[1], u[2], u[3]);
#pragma unroll
              for (int j = 0; j < NT; ++j) product(o[h][j], u, i, j);
            }
        }
        use = use == 2 ? 0 : use + 1;
        use_half ^= 1;
        __syncwarp();  // every lane has read these values
      }
      load_keys();  // of the tile after the next, where these values were
    }

    // ---- the row's end: (m, l, o) to shared memory
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float ls = l[j][x];
        ls += __shfl_xor_sync(kAll, ls, 4);
        ls += __shfl_xor_sync(kAll, ls, 8);
        ls += __shfl_xor_sync(kAll, ls, 16);
        const int col = 8 * j + 2 * t + x;
        if (g == 0 && col < NC) {
          sm[warp * 2 * NC + col] = part_max(m[j][x], ls);
          sm[warp * 2 * NC + NC + col] = ls;
        }
      }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = 8 * j + 2 * t + x;
        // o is relative to M where values have scales
        const float f = CODED ? weight(mv[j][x], m[j][x]) : 1.0f;
        float* dst = so + (warp * NC + (col < NC ? col : 0)) * M::OS;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          float u = o[i][j][x], v = o[i][j][2 + x];
          if constexpr (M::kTwins) {  // the halves' columns are 4 apart: two lanes
            u = fmaf(__shfl_xor_sync(kAll, u, 2), M::kDown, u);
            v = fmaf(__shfl_xor_sync(kAll, v, 2), M::kDown, v);
          }
          if (col < NC) {
            if constexpr (CODED) {
              constexpr int per = M::kValBytes / 2;  // products a lane's part feeds
              const int d = (i / per * 8 + g) * (2 * per) + i % per * 2;
              *reinterpret_cast<float2*>(dst + d) = make_float2(u * f, v * f);
            } else {
              dst[16 * i + g] = u;
              dst[16 * i + 8 + g] = v;
            }
          }
        }
      }
    const int row_e = e, row_r = r;
    const int64_t row_start = start;
    start += tiles + p.cost;
    if (++r == a.rows) {
      r = 0;
      ++e;
    }
    const bool more = start < p.end;
    if (more) load_q(e, r);
    __syncthreads();
    end_row<NC, DP, M::OS, W>(a, p, row_e, row_r, tiles, n, row_start, row_start <= 0, sm, so, left);
    __syncthreads();
    if (!more) break;
    skip -= n;
    tile = 0;
  }
  if constexpr (!M::ROW) join_left<NC, DP>(a, p, left);
}

template <class M>
cudaError_t launch(const DecodeArgs& a, int grid, cudaStream_t st) {
  if (grid < 1) return cudaErrorInvalidDevice;
  return launch_early(decode_mma_kernel<M>, grid, M::W * 32, M::kSmem, st, a);
}

template <Elem K, int NH, int DP, bool WHOLE>
cudaError_t launch(DecodeArgs a, cudaStream_t st) {
  using Row = Mma<K, NH, DP, WHOLE, true>;
  using Cut = Mma<K, NH, DP, WHOLE, false>;
  static Resident known[2];
  a.groups = (a.G + NH - 1) / NH;
  a.rows = a.c.Hk * a.groups;
  const int64_t rows = (int64_t)a.c.E * a.rows;
  if constexpr (Row::kFits)
    if (short_rows(a, Row::kBytes) &&
        rows <= places(decode_mma_kernel<Row>, Row::W * 32, Row::kSmem, known[0]))
      return launch<Row>(a, (int)rows, st);
  return launch<Cut>(
      a, piece_ctas(a, places(decode_mma_kernel<Cut>, Cut::W * 32, Cut::kSmem, known[1])), st);
}

template <Elem K, int DP, bool WHOLE>
cudaError_t launch_heads(const DecodeArgs& a, cudaStream_t st) {
  // as few passes over the keys and values as o's registers allow
  if (a.G <= 4) return launch<K, 4, DP, WHOLE>(a, st);
  if constexpr (DP <= 128)
    if (a.G > 8) return launch<K, 16, DP, WHOLE>(a, st);
  return launch<K, 8, DP, WHOLE>(a, st);
}

template <Elem K, int DP>
cudaError_t launch_dim(const DecodeArgs& a, cudaStream_t st) {
  const bool whole = a.c.D == DP && a.c.page_size % kTile == 0 && a.c.stride[0][2] == DP &&
                     a.c.stride[1][2] == DP;
  return whole ? launch_heads<K, DP, true>(a, st) : launch_heads<K, DP, false>(a, st);
}

template <Elem K>
cudaError_t launch_pages(const DecodeArgs& a, cudaStream_t st) {
  return a.c.D <= 64 ? launch_dim<K, 64>(a, st)
         : a.c.D <= 128 ? launch_dim<K, 128>(a, st)
                        : launch_dim<K, 256>(a, st);
}

}  // namespace

}  // namespace ma
