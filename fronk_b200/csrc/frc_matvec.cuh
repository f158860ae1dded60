// frc_matvec.cuh - products of one dense 4-bit matrix with 1-16 token vectors.
//
// y[t][r] = sum_j W[r][j] x[t][j], W in the row formats of the expert slices:
// Q4_K (w = d sc_g q - dmin mi_g, a 6-bit scale and minimum per 32 weights
// under fp16 super scales per 256) or MXFP4 (w = 2^(e-127) E2M1 per 32).
//
// The weights' bytes bound it, so the work per weight has to stay under the
// ~1.5 integer and ~3 other lane operations that one weight may cost at the
// HBM rate (43 weights a clock and SM).  A warp multiplies 16 rows x 256
// columns ("a span of a tile") on the tensor cores by mma.sync, with the
// vectors as the eight columns.  x is scaled by a power of two per span.
//   Q4_K, up to four tokens: in integers.  The nibbles are the bytes of a u8
//     operand after one mask each; x is held as four signed base-256 digits,
//     a column each: rounded to 2^-30 of the span's largest value, so that the
//     parts of a span's sum that come from digits stay whole numbers (a value
//     2^-7 of the largest loses its last bits, 2^-30 of the sum's size at
//     most, where fp32 sums round 2^-24 at every step); the 6-bit scales
//     multiply the int32 sums of each 32, so a span is exact.
//   Q4_K, more tokens: in fp16, which holds q sc exactly (10 bits): masked
//     nibbles are made 1024 + q and one half2 operation takes the 1024 off
//     (and multiplies by sc where that saves work on the results).
//   MXFP4: in fp16, by the hardware's E2M1 conversion, and per 32 weights one
//     fma with the block's scale.
//   In fp16 a bf16 x fits one value (P = 1); an fp32 x is the sum of two, hi
//     and lo, a column each (P = 2): 22 of its 24 bits, or 2^-34 of the span's
//     largest value where that is more.  A third part would cost half as many
//     products again for 2^-23 of each x, which the sums' rounding hides.
//   The minima of Q4_K are one more fp16 product, of mi with the sums of x
//     over each 32 (hi and lo parts along K, 22 bits like x itself).
// (fp16 subnormals as operands would save the half2 operations, but mma.sync
// aligns its sums by the operands' exponents: measured, q 2^-24 costs 20 times
// the rounding error.)
//
// Measured on one B200, graph replays: 131072 x 2048, one token: Q4_K 27.8 us
// (5.4 TB/s, 84 % of the copy rate), MXFP4 26.7 us; 65536 x 2048, Q4_K, 4, 8
// and 16 fp32 tokens 20.6, 28.2 and 39.2 us (with more columns the products
// and their operands' reads bound it, not the weights); 50021 x 2560, MXFP4,
// 16 tokens: bf16 25.1 us, fp32 39.1 us (its 32 columns spill registers).
#pragma once
#include <atomic>
#include <cuda_bf16.h>

#include "../../include/fronk_b200.h"
#include "frc_device.cuh"

namespace frc {

constexpr unsigned kMvSpan = 256;          // weights of a row in one step
constexpr unsigned kMvTile = 16;           // rows of one step

// Device layout: tile after tile (16 rows, the last one filled up with zero
// rows), in it span after span of [scales][pieces], a piece being 64 weights
// of the 16 rows: lane (g = lane / 4, q = lane % 4) owns 16 bytes {row g
// group 0, row g + 8 group 0, row g group 1, row g + 8 group 1}, a word of
// eight weights 32 group + 8 q + 0..7 each, so that a load is the fragment
// (Q4_K: 0..3 in the low nibbles of its bytes, 4..7 in the high ones).
// The last span stops at the last piece that holds weights.
//   Q4_K scales: the 16 header bytes of each row (d, dmin, packed 6 bits).
//   MXFP4 scales: 8 bytes a row, e + 1 - shift for a block of exponent e, so
//   that each is the exponent field of an fp32 number (twice the scale; the
//   spans' powers of two are halved), and 0 for a block whose weights are all
//   zero.  The shift is 0 but in rows with scales over 2^102: it keeps the
//   byte at or under kMvField, where a span's sum (at most 256 x 6 x 2^14
//   times the scale) stays under 2^128.  127 + shift of the rows are 16 bytes
//   a tile at `shift`.
struct MvLayout {
  unsigned tiles, spans, pieces_last, span_bytes, scale_bytes;
  size_t tile_bytes, shift_at, total;
};
constexpr unsigned kMvField = 230;  // largest scale byte of MXFP4
enum : unsigned { kMvNotFinite = 1, kMvTooFarApart = 2 };  // what matrix_layout_kernel finds
inline MvLayout mv_layout(unsigned type, unsigned rows, unsigned n) {
  MvLayout l;
  l.tiles = (rows + kMvTile - 1) / kMvTile;
  l.spans = (n + kMvSpan - 1) / kMvSpan;
  l.pieces_last = (n - (l.spans - 1) * kMvSpan + 63) / 64;
  l.scale_bytes = type == FRC_Q4_K ? 256 : 128;
  l.span_bytes = l.scale_bytes + 2048;
  l.tile_bytes = static_cast<size_t>(l.spans - 1) * l.span_bytes + l.scale_bytes + 512 * l.pieces_last;
  l.shift_at = l.tile_bytes * l.tiles;
  l.total = l.shift_at + static_cast<size_t>(l.tiles) * kMvTile;
  return l;
}

// Whether an MXFP4 block has a weight other than zero.
__device__ __forceinline__ bool mv_block_counts(const uint8_t* b) {
  unsigned any = 0;
#pragma unroll
  for (unsigned j = 1; j < 17; ++j) any |= b[j];
  return any & 0x77u;
}

// Reference rows -> the layout above, one CTA a tile.  Flags scales that are
// not finite (Q4_K super scales, MXFP4 exponent 255) and MXFP4 rows whose
// smallest scale would not fit the byte.
template <unsigned TYPE>
__global__ void __launch_bounds__(256) matrix_layout_kernel(const uint8_t* __restrict__ src, uint8_t* dst, MvLayout l,
                                                            unsigned rows, unsigned n, unsigned row_bytes,
                                                            unsigned* flag) {
  __shared__ unsigned s_high[kMvTile];  // a row's largest exponent, then its shift
  const unsigned tile = blockIdx.x, tid = threadIdx.x;
  const uint8_t* in = src + static_cast<size_t>(tile) * kMvTile * row_bytes;
  uint8_t* out = dst + tile * l.tile_bytes;
  const unsigned left = rows - tile * kMvTile < kMvTile ? rows - tile * kMvTile : kMvTile;
  bool bad = false, apart = false;
  if (TYPE == kMXFP4) {
    if (tid < kMvTile) s_high[tid] = 0;
    __syncthreads();
    for (unsigned i = tid; i < left * (n / 32); i += 256) {
      const unsigned r = i / (n / 32), b = i % (n / 32);
      const uint8_t* block = in + static_cast<size_t>(r) * row_bytes + 17 * b;
      bad |= block[0] == 255;
      if (mv_block_counts(block)) atomicMax(&s_high[r], static_cast<unsigned>(block[0]));
    }
    __syncthreads();
    if (tid < kMvTile) {
      const unsigned shift = s_high[tid] < kMvField ? 0 : s_high[tid] + 1 - kMvField;
      s_high[tid] = shift;
      dst[l.shift_at + static_cast<size_t>(tile) * kMvTile + tid] = static_cast<uint8_t>(127 + shift);
    }
    __syncthreads();
  }
  for (unsigned s = 0; s < l.spans; ++s) {
    uint8_t* o = out + static_cast<size_t>(s) * l.span_bytes;
    if (TYPE == kQ4K) {
      if (tid < 64) {  // a 4-byte word of a row's header
        const unsigned r = tid / 4, w = tid % 4;
        const uint8_t* b = in + static_cast<size_t>(r) * row_bytes + 144 * s + 4 * w;
        const unsigned v = r < left ? b[0] | b[1] << 8 | b[2] << 16 | static_cast<unsigned>(b[3]) << 24 : 0u;
        if (w == 0) bad |= (v & 0x7c00u) == 0x7c00u || (v & 0x7c000000u) == 0x7c000000u;
        reinterpret_cast<unsigned*>(o)[tid] = v;
      }
    } else if (tid < 128) {
      const unsigned r = tid / 8, b = 8 * s + tid % 8;
      unsigned e = 0;
      if (r < left && b < n / 32) {
        const uint8_t* block = in + static_cast<size_t>(r) * row_bytes + 17 * b;
        if (mv_block_counts(block)) {
          apart |= block[0] < s_high[r];
          e = block[0] + 1 - s_high[r];
        }
      }
      o[tid] = static_cast<uint8_t>(e);
    }
    const unsigned pieces = s + 1 < l.spans ? 4 : l.pieces_last;
    for (unsigned i = tid; i < pieces * 128; i += 256) {
      const unsigned piece = i / 128, lane = i / 4 % 32, part = i % 4;
      const unsigned r = lane / 4 + 8 * (part & 1), grp = 2 * piece + part / 2, k0 = 8 * (lane % 4);
      unsigned v = 0;
      if (r < left && kMvSpan * s + 32 * grp < n) {
        const uint8_t* b = in + static_cast<size_t>(r) * row_bytes;
        if (TYPE == kQ4K) {
          const uint8_t* q = b + 144 * s + 16 + 32 * (grp / 2) + k0;
#pragma unroll
          for (unsigned j = 0; j < 8; ++j) v |= (q[j] >> (4 * (grp & 1)) & 15u) << (8 * (j % 4) + 4 * (j / 4));
        } else {
          const uint8_t* q = b + 17 * (8 * s + grp) + 1 + (k0 & 8);
#pragma unroll
          for (unsigned j = 0; j < 8; ++j) v |= (q[j] >> (k0 < 16 ? 0 : 4) & 15u) << (4 * j);
        }
      }
      reinterpret_cast<unsigned*>(o + l.scale_bytes)[i] = v;
    }
  }
  if (bad) atomicOr(flag, kMvNotFinite);
  if (apart) atomicOr(flag, kMvTooFarApart);
}

struct MatvecParams {
  const uint8_t* w;
  const void* x;
  void* y;
  size_t x_stride, y_stride;  // elements between tokens
  size_t tile_bytes, shift_at;
  unsigned rows, n, tokens, tiles, spans, pieces_last;
  unsigned slice;             // spans of K a CTA works on (all, or a share where a cluster splits K)
  unsigned chunk;             // spans of x in shared memory at a time, at most the slice
  unsigned cluster;           // CTAs that share K
  unsigned x_vec, x_bf16, y_bf16;  // x rows are 16-byte aligned; x, y are bf16
  unsigned* status;
};

// m16n8k16, fp16 inputs, fp32 accumulators: c += a b, or c = a b.
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// m16n8k32, unsigned by signed bytes, int32: c = a b.
__device__ __forceinline__ void mma_u8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Eight E2M1 values -> fp16 pairs.
__device__ __forceinline__ void e2m1_f16(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

// A lane's share of one span of a tile, and the slots of shared memory that a
// warp has its next spans copied to (a lane copies the words it will read;
// the scales are read by other lanes too).
template <unsigned TYPE>
struct MvFrag {
  static constexpr unsigned kScale = TYPE == kQ4K ? 256 : 128, kBytes = kScale + 2048;
  uint4 w[4];
  uint4 s[TYPE == kQ4K ? 2 : 1];  // Q4_K: headers of rows g and g + 8; MXFP4: their exponents, 8 bytes each

  static __device__ __forceinline__ void copy(uint32_t slot, const uint8_t* p, unsigned pieces, unsigned lane) {  // p: the span
    const uint8_t* q = p + 16 * lane + kScale;
    const uint32_t d = slot + 16 * lane + kScale;
#pragma unroll
    for (unsigned j = 0; j < 4; ++j)
      if (TYPE == kQ4K || j < pieces)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + 512 * j), "l"(q + 512 * j) : "memory");
    if (lane < kScale / 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d - kScale), "l"(q - kScale) : "memory");
  }
  __device__ __forceinline__ void read(uint32_t slot, unsigned pieces, unsigned lane) {
    const uint32_t d = slot + 16 * lane + kScale, e = slot + (kScale / 16) * (lane / 4);
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) w[j] = lds128(d + 512 * j);
    if (TYPE == kQ4K) {
      s[0] = lds128(e);
      s[TYPE == kQ4K ? 1 : 0] = lds128(e + 128);
    } else {
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(s[0].x), "=r"(s[0].y) : "r"(e));
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(s[0].z), "=r"(s[0].w) : "r"(e + 64));
      if (pieces < 4) {
#pragma unroll
        for (unsigned j = 1; j < 4; ++j)
          if (j >= pieces) w[j] = make_uint4(0, 0, 0, 0);
      }
    }
  }
};

// The vectors of one K chunk in shared memory, as the products' B fragments:
// per span and group of 32 a block of 8 NT columns of 64 bytes (32 for the
// digits of P = 4).
//
// With few columns (COLS = 1, 2, 4: tokens x parts, rounded up) the eight of
// a product are shared by 8 / COLS groups: the block of group i holds its
// values in columns (i mod (8 / COLS)) COLS + c and zeros elsewhere, so that
// one accumulator keeps the groups' sums apart, each lane has the sums of its
// own group, and a lane applies one scale where it would apply 8 / COLS.  The
// zeros have to be written first: it pays from six spans a warp on (MXFP4,
// bf16 x, one token: 131072 x 2048 26.7 against 27.4 us; 513 x 2048, one span
// a warp, 4.1 against 4.0).
struct MvShared {
  uint8_t* col;     // [chunk][8 groups][NT][8 columns][64 or 32]
  uint8_t* sums;    // Q4_K: [chunk][NT][8 columns][32]: sums over each 32 (x 2^-5, so they fit fp16), eight hi, eight
                    // lo parts, in a token's (first) column of the first group; columns of other groups are zero
  float* scale;     // [tokens][chunk]: the power of two of each span
  float* part;      // [warps][values][32]: sums of tiles that a warp did not begin; in a cluster
                    // [tiles][values][32] behind them: the CTA's share of its tiles
  uint8_t* ring;    // [warps][DEPTH][span]
};

// Spans first .. first + count of every token into shared memory, a warp a
// (token, span) at a time with the values of U of them on their way.
template <unsigned TYPE, unsigned P, unsigned NT, unsigned COLS>
__device__ __forceinline__ void mv_prepare(const MatvecParams& a, const MvShared& sh, unsigned first, unsigned count) {
  constexpr unsigned U = P == 1 ? 8 : 4, R = P == 1 ? 4 : 8;
  const bool bf16 = P == 1 || (P == 4 && a.x_bf16);
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = blockDim.x / 32, units = a.tokens * count;
  for (unsigned u0 = warp; u0 < units; u0 += U * warps) {
    uint32_t raw[U][R];
#pragma unroll
    for (unsigned i = 0; i < U; ++i) {
      const unsigned u = u0 + i * warps, t = u / count, s = u - t * count, k = (first + s) * kMvSpan + 8 * lane;
#pragma unroll
      for (unsigned j = 0; j < R; ++j) raw[i][j] = 0;
      if (u >= units || k >= a.n) continue;
      if (!bf16) {
        const float* x = static_cast<const float*>(a.x) + t * a.x_stride + k;
        if (a.x_vec) {
          const uint4 p = reinterpret_cast<const uint4*>(x)[0], q = reinterpret_cast<const uint4*>(x)[1];
          raw[i][0] = p.x; raw[i][1] = p.y; raw[i][2] = p.z; raw[i][3] = p.w;
          raw[i][R - 4] = q.x; raw[i][R - 3] = q.y; raw[i][R - 2] = q.z; raw[i][R - 1] = q.w;
        } else {
#pragma unroll
          for (unsigned j = 0; j < R; ++j) raw[i][j] = __float_as_uint(x[j]);
        }
      } else {
        const uint16_t* x = static_cast<const uint16_t*>(a.x) + t * a.x_stride + k;
        if (a.x_vec) {
          const uint4 p = *reinterpret_cast<const uint4*>(x);
          raw[i][0] = p.x; raw[i][1] = p.y; raw[i][2] = p.z; raw[i][3] = p.w;
        } else {
#pragma unroll
          for (unsigned j = 0; j < 4; ++j) raw[i][j] = x[2 * j] | static_cast<uint32_t>(x[2 * j + 1]) << 16;
        }
      }
    }
#pragma unroll
    for (unsigned i = 0; i < U; ++i) {
      const unsigned u = u0 + i * warps, t = u / count, s = u - t * count;
      if (u >= units) break;
      float v[8];
#pragma unroll
      for (unsigned j = 0; j < 8; ++j)
        v[j] = __uint_as_float(!bf16 ? raw[i][j % R] : j & 1 ? raw[i][j / 2] & 0xffff0000u : raw[i][j / 2] << 16);
      unsigned top = 0;
#pragma unroll
      for (unsigned j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
      top = __reduce_max_sync(0xffffffffu, top);
      // x = v 2^ex, the largest |v| in [2^13, 2^14), or [2^29, 2^30) as digits; a span that is not finite has the
      // scale NaN and so its results.  The scales of MXFP4's blocks are doubled, so the span's is halved.
      constexpr int TOP = P == 4 ? 29 : 13, HALVED = TYPE == kMXFP4 ? 1 : 0;
      int ex = static_cast<int>(top >> 23) - 127 - TOP;
      // Near the smallest numbers, where 2^-ex is too large for fp32, v is made in two steps and the span's scale is
      // subnormal (131072 x 2048, one token: the same time with and without; 50021 x 2560, 16 tokens 25.1 and 24.8 us).  At 2^-149, the last bit of any x, v is a whole number.
      constexpr int LOW = HALVED - 126;
      const int less = min(max(LOW - ex, 0), 23);
      ex = max(ex, LOW);
      if (less) {
        const float more = __uint_as_float(static_cast<uint32_t>(127 + less) << 23);
#pragma unroll
        for (unsigned j = 0; j < 8; ++j) v[j] *= more;
      }
      const bool finite = top < 0x7f800000u;
      const float inv = finite ? __uint_as_float(static_cast<uint32_t>(127 - ex) << 23) : 0.0f;
#pragma unroll
      for (unsigned j = 0; j < 8; ++j) v[j] = finite ? v[j] * inv : 0.0f;
      const float sum8 = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      const unsigned grp = lane / 4, c0 = COLS < 8 ? (grp % (8 / COLS)) * COLS + t * P : t * P;
      if (P == 4) {
        // signed digits: with 128 added to the three low bytes they are the bytes less 128
        uint32_t w[8];
#pragma unroll
        for (unsigned j = 0; j < 8; ++j) w[j] = (static_cast<uint32_t>(__float2int_rn(v[j])) + 0x00808080u) ^ 0x00808080u;
        uint8_t* c = sh.col + ((s * 8 + grp) * NT + c0 / 8) * 256 + c0 % 8 * 32 + 8 * (lane % 4);
#pragma unroll
        for (unsigned d = 0; d < 4; ++d) {
          const uint32_t sel = d | (4 + d) << 4;
          const uint32_t lo = prmt(prmt(w[0], w[1], sel), prmt(w[2], w[3], sel), 0x5410);
          const uint32_t hi = prmt(prmt(w[4], w[5], sel), prmt(w[6], w[7], sel), 0x5410);
          *reinterpret_cast<uint2*>(c + 32 * d) = make_uint2(lo, hi);
        }
      } else {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) {
          // a Q4_K word gives the pairs 0 2, 4 6, 1 3, 5 7, of them 4..7 as 16 q
          const float f = TYPE == kQ4K && (j & 1) ? 0.0625f : 1.0f;
          const unsigned e0 = TYPE == kQ4K ? 4 * (j & 1) + j / 2 : 2 * j, e1 = TYPE == kQ4K ? e0 + 2 : e0 + 1;
          const float p = v[e0] * f, q = v[e1] * f;
          const __half2 h = __floats2half2_rn(p, q);
          hi[j] = *reinterpret_cast<const uint32_t*>(&h);
          const float2 b = __half22float2(h);
          const __half2 l = __floats2half2_rn(p - b.x, q - b.y);
          lo[j] = *reinterpret_cast<const uint32_t*>(&l);
        }
        uint8_t* c = sh.col + ((s * 8 + grp) * NT + c0 / 8) * 512 + c0 % 8 * 64 + 16 * (lane % 4);
        *reinterpret_cast<uint4*>(c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (P == 2) *reinterpret_cast<uint4*>(c + 64) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      if (lane == 0)
        sh.scale[t * a.chunk + s] = finite ? __uint_as_float(less ? 1u << (23 - less) : static_cast<uint32_t>(127 - HALVED + ex) << 23) : NAN;
      if (TYPE == kQ4K) {
        float sum = sum8;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= P == 4 ? 0x1p-21f : 0x1p-5f;  // fits fp16
        if (lane % 4 == 0) {
          const __half h = __float2half_rn(sum), l = __float2half_rn(sum - __half2float(h));
          __half* o = reinterpret_cast<__half*>(sh.sums + (s * NT * 8 + t * P) * 32) + grp;
          o[0] = h;
          o[8] = l;
        }
      }
    }
  }
}

// A lane's part in the products: its fragment of a block, its tokens' scales
// and, where groups share columns, which group's results it holds.
template <unsigned P, unsigned NT, unsigned COLS>
struct MvLane {
  static constexpr unsigned kTok = P >= 2 || COLS == 1 ? 1 : 2;  // tokens of a lane's results in eight columns
  uint32_t col, sums, scale[NT][kTok];
  unsigned sel;      // bytes 2 q and 2 q + 1
  unsigned mine[2];  // byte of the scale of the lane's first and second column, for a group set that starts at byte 0
  __device__ __forceinline__ unsigned token(unsigned t, unsigned k, unsigned q) const {
    if (COLS == 8) return P == 4 ? 2 * t + q / 2 : P == 2 ? 4 * t + q : 8 * t + 2 * q + k;
    return ((2 * q + k) % COLS) / P;
  }
  // Whether the lane has its column's results when the lanes have been joined.
  __device__ __forceinline__ bool holds(unsigned k, unsigned q) const {
    return (COLS == 8 || (2 * q + k) / COLS == 0) && (P != 4 || q % 2 == 0);
  }
  __device__ __forceinline__ MvLane(const MatvecParams& a, const MvShared& sh, unsigned lane) {
    const unsigned g = lane / 4, q = lane % 4;
    sel = 2 * q | (2 * q + 1) << 4;
    mine[0] = 2 * q / COLS;
    mine[1] = (2 * q + 1) / COLS;
    col = smem_u32(sh.col) + (P == 4 ? 32 * g + 8 * q : 64 * g + 16 * q);
    sums = smem_u32(sh.sums) + 32 * g + 4 * q;
#pragma unroll
    for (unsigned t = 0; t < NT; ++t)
#pragma unroll
      for (unsigned k = 0; k < kTok; ++k) {
        const unsigned tok = token(t, k, q);
        scale[t][k] = smem_u32(sh.scale) + 4 * ((tok < a.tokens ? tok : 0) * a.chunk);
      }
  }
};

// The fp16 operands of 32 columns of a tile from a lane's word of one row: for
// Q4_K 1024 + q (pairs 0, 2) and 1024 + 16 q (pairs 1, 3).
template <unsigned TYPE>
__device__ __forceinline__ void mv_weights(uint32_t w, uint32_t (&av)[4]) {
  if (TYPE == kQ4K) {
    const uint32_t u = w >> 8;
    av[0] = (w & 0x000f000fu) | 0x64006400u;
    av[1] = (w & 0x00f000f0u) | 0x64006400u;
    av[2] = (u & 0x000f000fu) | 0x64006400u;
    av[3] = (u & 0x00f000f0u) | 0x64006400u;
  } else {
    e2m1_f16(w, av);
  }
}
// Byte `at` of the eight in {lo, hi} as a float: a 6-bit scale, or the number
// of that exponent field (0 for 0).
template <unsigned TYPE>
__device__ __forceinline__ float mv_scale(uint32_t lo, uint32_t hi, unsigned at) {
  const uint32_t v = prmt(lo, hi, at);
  if (TYPE == kQ4K) return __uint_as_float(prmt(v, 0x4B000000u, 0x7440u)) - 8388608.0f;
  return __uint_as_float(v << 23 & 0x7f800000u);
}
template <unsigned TYPE>
__device__ __forceinline__ float mv_scale_at(const uint32_t (&b)[2], unsigned at) {  // at known when compiled
  const uint32_t v = b[at / 4];
  if (TYPE == kQ4K) return __uint_as_float(prmt(v, 0x4B000000u, 0x7440u | at % 4)) - 8388608.0f;
  return __uint_as_float((at % 4 == 3 ? v >> 1 : v << (23 - 8 * (at % 4))) & 0x7f800000u);
}

// The header of a Q4_K row's super-block: d, -dmin, the eight 6-bit scales and
// minima as bytes.
__device__ __forceinline__ void mv_header(uint4 b, float& d, float& dm, uint32_t (&sc)[2], uint32_t (&mi)[2]) {
  d = h2f(b.x & 0xffffu);
  dm = -h2f(b.x >> 16);
  sc[0] = b.y & 0x3f3f3f3fu;
  mi[0] = b.z & 0x3f3f3f3fu;
  sc[1] = (b.w & 0x0f0f0f0fu) | (b.y >> 2 & 0x30303030u);
  mi[1] = (b.w >> 4 & 0x0f0f0f0fu) | (b.z >> 2 & 0x30303030u);
}
// Minima of groups 2 q and 2 q + 1 of a row as fp16 (sel: their bytes).
__device__ __forceinline__ uint32_t mv_minima(const uint32_t (&mi)[2], unsigned sel) {
  return hsub2(prmt(prmt(mi[0], mi[1], sel), 0x64646464u, 0x4140u), 0x64006400u);
}

// One span (s of the chunk) of a tile times the columns; acc: [row g | row
// g + 8] of the lane's columns' tokens in each eight columns (the sum of both
// columns for P = 2).  The 6-bit scales of Q4_K go onto the results of each
// 32, or for several groups of columns (where that is more work) into the
// weights.
template <unsigned TYPE, unsigned P, unsigned NT, unsigned COLS>
__device__ __forceinline__ void mv_span(const MvLane<P, NT, COLS>& ln, const MvFrag<TYPE>& f, unsigned s,
                                        float (&acc)[NT * (P >= 2 ? 2 : 4)]) {
  constexpr bool FOLD = TYPE == kQ4K && NT > 1;
  constexpr unsigned SHARE = 8 / COLS;  // groups in one accumulator
  uint32_t sc[2][2];  // eight scale bytes of rows g and g + 8
  float d[2], dm[2], m[NT][4];
  if constexpr (TYPE == kQ4K) {
    uint32_t mi[2][2];
    mv_header(f.s[0], d[0], dm[0], sc[0], mi[0]);
    mv_header(f.s[TYPE == kQ4K ? 1 : 0], d[1], dm[1], sc[1], mi[1]);
    const uint32_t m0 = mv_minima(mi[0], ln.sel), m1 = mv_minima(mi[1], ln.sel);
#pragma unroll
    for (unsigned t = 0; t < NT; ++t) {
      const uint32_t at = ln.sums + 256 * (NT * s + t);
      mma_f16_first(m[t], m0, m1, m0, m1, lds32(at), lds32(at + 16));
    }
    // the sums were scaled down
    dm[0] *= P == 4 ? 0x1p21f : 0x1p5f;
    dm[1] *= P == 4 ? 0x1p21f : 0x1p5f;
  } else {
    sc[0][0] = f.s[0].x; sc[0][1] = f.s[0].y; sc[1][0] = f.s[0].z; sc[1][1] = f.s[0].w;
  }
  if constexpr (P == 4) {
    const uint32_t xc = ln.col + 2048 * NT * s;
    int sum[NT][4];
#pragma unroll
    for (unsigned t = 0; t < NT; ++t) sum[t][0] = sum[t][1] = sum[t][2] = sum[t][3] = 0;
#pragma unroll
    for (unsigned grp = 0; grp < 8; ++grp) {
      const uint4 wv = f.w[grp / 2];
      const uint32_t w0 = grp & 1 ? wv.z : wv.x, w1 = grp & 1 ? wv.w : wv.y;
      const uint32_t a0 = w0 & 0x0f0f0f0fu, a1 = w1 & 0x0f0f0f0fu, a2 = w0 >> 4 & 0x0f0f0f0fu, a3 = w1 >> 4 & 0x0f0f0f0fu;
      const int k0 = static_cast<int>(prmt(sc[0][grp / 4], 0, 0x4440u | grp % 4)), k1 = static_cast<int>(prmt(sc[1][grp / 4], 0, 0x4440u | grp % 4));
#pragma unroll
      for (unsigned t = 0; t < NT; ++t) {
        uint32_t b0, b1;
        int c[4];
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(xc + 256 * (NT * grp + t)));
        mma_u8(c, a0, a1, a2, a3, b0, b1);
        // |c| <= 32 x 15 x 128, times 63, eight times: below 2^25
        sum[t][0] += c[0] * k0;
        sum[t][1] += c[1] * k0;
        sum[t][2] += c[2] * k1;
        sum[t][3] += c[3] * k1;
      }
    }
    const bool upper = threadIdx.x & 1;  // two digits of the four: the upper two are 2^16 up
#pragma unroll
    for (unsigned t = 0; t < NT; ++t) {
      const float x = __uint_as_float(lds32(ln.scale[t][0] + 4 * s)), xd = upper ? x * 65536.0f : x;
#pragma unroll
      for (unsigned h = 0; h < 2; ++h) {
        const float v = fmaf(static_cast<float>(sum[t][2 * h + 1]), 256.0f, static_cast<float>(sum[t][2 * h]));
        // the sums of x are in the first digit's column
        acc[2 * t + h] += fmaf(v * d[h], xd, (upper ? 0.0f : m[t][2 * h] * dm[h]) * x);
      }
    }
    return;
  }
  const uint32_t xc = ln.col + 4096 * NT * s;
  constexpr unsigned SV = P == 2 ? 2 : 4;
  float sum[NT][SV], c[NT][4];
#pragma unroll
  for (unsigned t = 0; t < NT; ++t)
#pragma unroll
    for (unsigned i = 0; i < SV; ++i) sum[t][i] = 0.0f;
#pragma unroll
  for (unsigned grp = 0; grp < 8; ++grp) {
    const uint4 wv = f.w[grp / 2];
    uint32_t a0[4], a1[4];
    mv_weights<TYPE>(grp & 1 ? wv.z : wv.x, a0);
    mv_weights<TYPE>(grp & 1 ? wv.w : wv.y, a1);
    if (FOLD) {
      // sc as 1024 + sc less 1024, and -1024 sc
      const uint32_t sel = 0x4040u | (grp % 4) * 0x0101u;
      const uint32_t k0 = hsub2(prmt(sc[0][grp / 4], 0x64646464u, sel), 0x64006400u), k1 = hsub2(prmt(sc[1][grp / 4], 0x64646464u, sel), 0x64006400u);
      const uint32_t n0 = hmul2(k0, 0xe400e400u), n1 = hmul2(k1, 0xe400e400u);
#pragma unroll
      for (unsigned i = 0; i < 4; ++i) {
        a0[i] = hfma2(a0[i], k0, n0);
        a1[i] = hfma2(a1[i], k1, n1);
      }
    } else if (TYPE == kQ4K) {
#pragma unroll
      for (unsigned i = 0; i < 4; ++i) {
        a0[i] = hsub2(a0[i], 0x64006400u);
        a1[i] = hsub2(a1[i], 0x64006400u);
      }
    }
#pragma unroll
    for (unsigned t = 0; t < NT; ++t) {
      const uint4 b = lds128(xc + 512 * (NT * grp + t));
      if (FOLD ? grp % 4 == 0 : grp % SHARE == 0) mma_f16_first(c[t], a0[0], a1[0], a0[1], a1[1], b.x, b.y);
      else mma_f16(c[t], a0[0], a1[0], a0[1], a1[1], b.x, b.y);
      mma_f16(c[t], a0[2], a1[2], a0[3], a1[3], b.z, b.w);
    }
    if (FOLD && grp % 4 == 3) {  // mma.sync truncates at each step: halves of a span are added in fp32
#pragma unroll
      for (unsigned t = 0; t < NT; ++t) {
        if (P == 2) {
          sum[t][0] += c[t][0] + c[t][1];
          sum[t][1] += c[t][2] + c[t][3];
        } else {
#pragma unroll
          for (unsigned i = 0; i < 4; ++i) sum[t][i % SV] += c[t][i];
        }
      }
    }
    if (!FOLD && grp % SHARE == SHARE - 1) {  // the set's sums, each lane the group of its columns
      constexpr unsigned K = COLS == 1 ? 2 : 1;
      float k[2][K];
#pragma unroll
      for (unsigned h = 0; h < 2; ++h)
#pragma unroll
        for (unsigned i = 0; i < K; ++i) k[h][i] = SHARE > 1 ? mv_scale<TYPE>(sc[h][0], sc[h][1], grp + 1 - SHARE + ln.mine[i]) : mv_scale_at<TYPE>(sc[h], grp);
#pragma unroll
      for (unsigned t = 0; t < NT; ++t)
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
          if (P == 2) {
            sum[t][h] = fmaf(c[t][2 * h] + c[t][2 * h + 1], k[h][0], sum[t][h]);
          } else {
            sum[t][(2 * h) % SV] = fmaf(c[t][2 * h], k[h][0], sum[t][(2 * h) % SV]);
            sum[t][(2 * h + 1) % SV] = fmaf(c[t][2 * h + 1], k[h][K - 1], sum[t][(2 * h + 1) % SV]);
          }
        }
    }
  }
#pragma unroll
  for (unsigned t = 0; t < NT; ++t) {
    constexpr unsigned A = P == 2 ? 1 : 2;  // results of a row a lane keeps
#pragma unroll
    for (unsigned k = 0; k < A; ++k) {
      const float x = __uint_as_float(lds32(ln.scale[t][MvLane<P, NT, COLS>::kTok == 1 ? 0 : k] + 4 * s));
#pragma unroll
      for (unsigned h = 0; h < 2; ++h) {
        float v = P == 2 ? sum[t][h % SV] : sum[t][(2 * h + k) % SV];
        if (TYPE == kQ4K) v = fmaf(v, d[h], (P == 2 ? m[t][2 * h] : m[t][2 * h + k]) * dm[h]);
        acc[(2 * t + h) * A + k] = fmaf(v, x, acc[(2 * t + h) * A + k]);
      }
    }
  }
}

__device__ __forceinline__ void mv_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Stores the results of a tile (acc as mv_span leaves it).
template <unsigned TYPE, unsigned P, unsigned NT, unsigned COLS>
__device__ __forceinline__ bool mv_store(const MatvecParams& a, const MvLane<P, NT, COLS>& ln, unsigned tile, unsigned lane,
                                         const float (&acc)[NT * (P >= 2 ? 2 : 4)]) {
  constexpr unsigned V = NT * (P >= 2 ? 2 : 4), A = P >= 2 ? 1 : 2;
  const unsigned g = lane / 4, q = lane % 4;
  bool bad = false;
#pragma unroll
  for (unsigned h = 0; h < 2; ++h) {
    const unsigned row = tile * kMvTile + g + 8 * h;
    if (row >= a.rows) continue;
    const float f = TYPE == kMXFP4 ? __uint_as_float(static_cast<unsigned>(a.w[a.shift_at + row]) << 23) : 1.0f;
#pragma unroll
    for (unsigned i = 0; i < V / 2; ++i) {
      const unsigned t = i / A, k = i % A, tok = ln.token(t, k, q);
      if (tok >= a.tokens || !ln.holds(k, q)) continue;
      float v = acc[(2 * t + h) * A + k];
      if (TYPE == kMXFP4) v *= f;
      if (a.y_bf16) {
        const __nv_bfloat16 o = __float2bfloat16_rn(v);
        v = __bfloat162float(o);
        static_cast<__nv_bfloat16*>(a.y)[tok * a.y_stride + row] = o;
      } else {
        static_cast<float*>(a.y)[tok * a.y_stride + row] = v;
      }
      bad |= !isfinite(v);
    }
  }
  return bad;
}

// The lanes that hold groups of the same columns together.
template <unsigned P, unsigned NT, unsigned COLS>
__device__ __forceinline__ void mv_join(float (&acc)[NT * (P >= 2 ? 2 : 4)]) {
  constexpr unsigned V = NT * (P >= 2 ? 2 : 4);
  if (COLS == 8 && P != 4) return;
  if (COLS == 1) {
    acc[0] += acc[1];
    acc[2 % V] += acc[3 % V];
  }
#pragma unroll
  for (unsigned i = 0; i < V; ++i) {
    if (COLS == 1 && (i & 1)) continue;
    if (COLS <= 2 || P == 4) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 1);
    if (COLS < 8) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 2);
  }
}

// A CTA (of each cluster: the CTAs of a cluster share K) takes a run of
// tiles, and its W warps equal shares of the run's spans, wherever they fall:
// a tile's sum is finished by the warp that began it, which adds the parts of
// the warps behind it in order.  x is prepared once, while each warp has the
// weights of its first DEPTH spans on their way.  Where the slice of x does
// not fit shared memory (chunk < slice), a warp takes one tile at a time and
// x is prepared anew for every W tiles, chunk by chunk.
template <unsigned TYPE, unsigned P, unsigned NT, unsigned COLS, unsigned W, unsigned DEPTH>
__global__ void __launch_bounds__(32 * W, W == 8 ? 2 : 1) matvec_kernel(const MatvecParams a) {
  constexpr unsigned V = NT * (P >= 2 ? 2 : 4), kBytes = MvFrag<TYPE>::kBytes;
  extern __shared__ __align__(128) uint8_t smem[];
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  MvShared sh;
  sh.ring = smem;
  sh.col = smem + W * DEPTH * kBytes;
  sh.sums = sh.col + (P == 4 ? 2048 : 4096) * NT * a.chunk;
  sh.scale = reinterpret_cast<float*>(sh.sums + (TYPE == kQ4K ? 256 * NT * a.chunk : 0));
  sh.part = sh.scale + a.tokens * a.chunk;
  const MvLane<P, NT, COLS> ln(a, sh, lane);
  const unsigned rank = a.cluster > 1 ? blockIdx.x % a.cluster : 0, cta = blockIdx.x / a.cluster, ctas = gridDim.x / a.cluster;
  const unsigned k_first = rank * a.slice, k_end = min(a.spans, k_first + a.slice);
  const unsigned count = k_first < k_end ? k_end - k_first : 0;
  // 32 bits hold these: tiles up to 2^20, a run of up to tiles / CTAs, 256 spans
  const unsigned t0 = a.tiles * cta / ctas, t1 = a.tiles * (cta + 1) / ctas;
  const uint32_t ring = smem_u32(sh.ring) + warp * DEPTH * kBytes;
  unsigned in = 0, out = 0;
  bool bad = false;
  float acc[V];
#pragma unroll
  for (unsigned i = 0; i < V; ++i) acc[i] = 0.0f;
  const auto fill = [&]() {  // what no value goes to: columns of other groups
    uint4* z = reinterpret_cast<uint4*>(sh.col);
    const unsigned n16 = static_cast<unsigned>(reinterpret_cast<uint8_t*>(sh.scale) - sh.col) / 16;
    for (unsigned i = threadIdx.x; i < n16; i += 32 * W) z[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  };
  const auto place = [&](unsigned tile, unsigned span) {
    return a.w + static_cast<size_t>(tile) * a.tile_bytes + static_cast<size_t>(span) * kBytes;
  };
  if (a.chunk < a.slice) {
    if (COLS < 8) fill();
    for (unsigned base = t0; base < t1; base += W) {
      const unsigned tile = base + warp;
      for (unsigned first = k_first; first < k_end; first += a.chunk) {
        const unsigned part = min(a.chunk, k_end - first);
        __syncthreads();  // every warp has left the chunk before
        mv_prepare<TYPE, P, NT, COLS>(a, sh, first, part);
        __syncthreads();
        if (tile >= t1) continue;
        for (unsigned s = 0; s < part; ++s) {
          const unsigned pieces = first + s + 1 == a.spans ? a.pieces_last : 4;
          MvFrag<TYPE>::copy(ring, place(tile, first + s), pieces, lane);
          asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
          __syncwarp();
          MvFrag<TYPE> f;
          f.read(ring, pieces, lane);
          __syncwarp();
          mv_span<TYPE, P, NT, COLS>(ln, f, s, acc);
        }
      }
      if (tile < t1) {
        mv_join<P, NT, COLS>(acc);
        bad |= mv_store<TYPE, P, NT, COLS>(a, ln, tile, lane, acc);
      }
#pragma unroll
      for (unsigned i = 0; i < V; ++i) acc[i] = 0.0f;
    }
  } else {
    const unsigned work = (t1 - t0) * count;
    const auto share = [&](unsigned w) { return work * w / W; };
    const unsigned l0 = share(warp), l1 = share(warp + 1);
    unsigned tile = count ? t0 + l0 / count : t0, s = count ? l0 % count : 0;
    // the copies run DEPTH spans ahead
    unsigned at_tile = tile, at_s = s, at_left = l1 - l0;
    const uint8_t* at = place(tile, k_first + s);
    const auto copy = [&]() {
      if (at_left) {
        --at_left;
        MvFrag<TYPE>::copy(ring + in, at, k_first + at_s + 1 == a.spans ? a.pieces_last : 4, lane);
        at += kBytes;
        if (++at_s == count) {
          at_s = 0;
          at = place(++at_tile, k_first);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");  // empty groups keep the count
      in = in + kBytes == DEPTH * kBytes ? 0 : in + kBytes;
    };
#pragma unroll
    for (unsigned i = 0; i < DEPTH; ++i) copy();
    if (COLS < 8) fill();
    mv_prepare<TYPE, P, NT, COLS>(a, sh, k_first, count);
    __syncthreads();
    float* mine = sh.part + warp * V * 32 + lane;
    float* tiles = sh.part + W * V * 32 + lane;  // of a cluster's CTA
    const auto finish = [&](unsigned t) {
      if (a.cluster == 1) {
        bad |= mv_store<TYPE, P, NT, COLS>(a, ln, t, lane, acc);
      } else {
#pragma unroll
        for (unsigned i = 0; i < V; ++i) tiles[(t - t0) * V * 32 + 32 * i] = acc[i];
      }
    };
    bool began = s == 0;
    for (unsigned l = l0; l < l1; ++l) {
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
      __syncwarp();
      MvFrag<TYPE> f;
      f.read(ring + out, k_first + s + 1 == a.spans ? a.pieces_last : 4, lane);
      __syncwarp();  // the slot has been read
      out = out + kBytes == DEPTH * kBytes ? 0 : out + kBytes;
      copy();
      mv_span<TYPE, P, NT, COLS>(ln, f, s, acc);
      if (++s == count) {
        mv_join<P, NT, COLS>(acc);
        if (began) {
          finish(tile);
        } else {
#pragma unroll
          for (unsigned i = 0; i < V; ++i) mine[32 * i] = acc[i];
        }
        began = true;
        s = 0;
        ++tile;
#pragma unroll
        for (unsigned i = 0; i < V; ++i) acc[i] = 0.0f;
      }
    }
    if (s && l0 < l1) {
      mv_join<P, NT, COLS>(acc);
      if (!began) {
#pragma unroll
        for (unsigned i = 0; i < V; ++i) mine[32 * i] = acc[i];
      }
    }
    __syncthreads();
    if (s && l0 < l1 && began) {
      const unsigned end = (tile - t0 + 1) * count;
      for (unsigned w = warp + 1; w < W && share(w) < end; ++w) {
        const float* p = sh.part + w * V * 32 + lane;
        if (share(w) < share(w + 1))
#pragma unroll
          for (unsigned i = 0; i < V; ++i) acc[i] += p[32 * i];
      }
      finish(tile);
    }
    if (a.cluster > 1) {
      if (!count) {  // a CTA past the end of K
        for (unsigned i = threadIdx.x; i < (t1 - t0) * V * 32; i += 32 * W) sh.part[W * V * 32 + i] = 0.0f;
      }
      mv_cluster_sync();
      for (unsigned t = t0 + rank + a.cluster * warp; t < t1; t += a.cluster * W) {  // the CTAs share the tiles
#pragma unroll
        for (unsigned i = 0; i < V; ++i) acc[i] = 0.0f;
        for (unsigned r = 0; r < a.cluster; ++r) {
          uint32_t from;
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(smem_u32(tiles + (t - t0) * V * 32)), "r"(r));
#pragma unroll
          for (unsigned i = 0; i < V; ++i) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(from + 128 * i) : "memory");
            acc[i] += v;
          }
        }
        bad |= mv_store<TYPE, P, NT, COLS>(a, ln, t, lane, acc);
      }
      mv_cluster_sync();  // no CTA leaves while another reads its shared memory
    }
  }
  if (bad) atomicOr(a.status, kStNumeric);
}

// ------------------------------------------------------------ host side

struct MvPlan {
  unsigned warps, slice, chunk, cluster, grid, smem, share;
};

// Spans a warp has on their way (131072 x 2048, one token: four are no faster, 28.0 against 27.8 us).
constexpr unsigned kMvDepth = 2;
constexpr unsigned kMvSmemSm = 228 * 1024, kMvSmemCta = 227 * 1024;

// Shared memory of a CTA with `tiles` results kept (in a cluster).
inline size_t mv_smem(unsigned type, unsigned P, unsigned nt, unsigned tokens, unsigned values, unsigned warps,
                      unsigned chunk, unsigned tiles) {
  const unsigned scale = type == FRC_Q4_K ? 256 : 128;
  return static_cast<size_t>(warps) * kMvDepth * (2048 + scale) +
         static_cast<size_t>(chunk) * ((P == 4 ? 2048 : 4096) * nt + (type == FRC_Q4_K ? 256 * nt : 0) + 4 * tokens) +
         (static_cast<size_t>(warps) + tiles) * values * 128;
}
inline unsigned mv_ceil(unsigned a, unsigned b) { return (a + b - 1) / b; }

// Chooses the warps a CTA and the CTAs that share K by an estimate of the
// time in us, fitted to sweeps over both: a span takes a warp 0.06 us (times
// `heavy`, for the columns) for each warp of its SM, at least 0.4; preparing
// x 0.35 a span and warp, a cluster's exchange 0.1 a CTA and 0.02 a tile.
// Measured both ways: 5120 x 2560 and 8 tokens 9.8 us with clusters of 4, 10.4
// without; 513 x 2048 and one token 3.9 and 3.5; 50021 x 2560 and 16 tokens
// 25.8 with clusters of 2, 25.1 without; 4096 x 8192 and one token 8.9 either
// way.
inline MvPlan mv_plan(unsigned type, unsigned P, unsigned nt, unsigned tokens, const MvLayout& l, unsigned sms) {
  const unsigned values = nt * (P >= 2 ? 2 : 4);
  const double heavy = nt == 1 ? 1.0 : nt == 2 ? 1.5 : 2.3;
  MvPlan best{};
  double least = 1e30;
  for (unsigned warps = 8; warps <= 16; warps *= 2) {
    const size_t limit = warps == 8 ? (kMvSmemSm - 2048) / 2 : kMvSmemCta;
    for (unsigned cluster = 1; cluster <= 8 && cluster <= l.spans; cluster *= 2) {
      // clusters of more than two do not tile the SMs of every GPC
      const unsigned resident = sms * (warps == 8 ? 2 : 1) / cluster * (cluster > 2 ? 7 : 8) / 8;
      if (!resident) continue;
      MvPlan p{};
      p.warps = warps;
      p.cluster = cluster;
      p.slice = p.chunk = mv_ceil(l.spans, cluster);
      const unsigned groups = l.tiles < resident ? l.tiles : resident, tiles = mv_ceil(l.tiles, groups);
      const unsigned kept = cluster > 1 ? tiles : 0;
      if (mv_smem(type, P, nt, tokens, values, warps, p.chunk, kept) > limit) {
        if (cluster > 1 || warps == 8) continue;
        while (mv_smem(type, P, nt, tokens, values, warps, p.chunk, kept) > limit) p.chunk = mv_ceil(p.chunk, 2);
      }
      p.grid = groups * cluster;
      p.smem = static_cast<unsigned>(mv_smem(type, P, nt, tokens, values, warps, p.chunk, kept));
      const unsigned steps = mv_ceil(tiles * p.slice, warps), busy = warps * mv_ceil(p.grid, sms);
      const double step = 0.06 * busy * heavy > 0.4 ? 0.06 * busy * heavy : 0.4;
      const double prep = 0.4 + 0.35 * mv_ceil(tokens * p.chunk, warps);
      double t = step * steps + prep + (cluster > 1 ? 0.3 + 0.1 * cluster + 0.02 * tiles : 0.0) + (warps == 16 ? 0.3 : 0.0);
      if (p.chunk < p.slice) t += (step + prep) * mv_ceil(tiles, warps) * mv_ceil(p.slice, p.chunk);
      p.share = steps >= 6;
      if (t < least * 0.98) {
        least = t;
        best = p;
      }
    }
  }
  return best;
}

template <unsigned TYPE, unsigned P, unsigned NT, unsigned COLS, unsigned W>
inline cudaError_t mv_launch(const MatvecParams& a, const MvPlan& p, int device, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed{0};  // devices on which the kernel may use kMvSmemCta bytes
  const unsigned long long bit = 1ull << (device & 63);
  if (p.smem > 48 * 1024 && (device > 63 || !(allowed.load(std::memory_order_relaxed) & bit))) {
    const cudaError_t e = cudaFuncSetAttribute(matvec_kernel<TYPE, P, NT, COLS, W, kMvDepth>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kMvSmemCta);
    if (e != cudaSuccess) return e;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = p.cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.grid);
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, matvec_kernel<TYPE, P, NT, COLS, W, kMvDepth>, a);
}
template <unsigned TYPE, unsigned P, unsigned NT, unsigned COLS>
inline cudaError_t mv_launch_w(const MatvecParams& a, const MvPlan& p, int device, cudaStream_t s) {
  return p.warps == 8 ? mv_launch<TYPE, P, NT, COLS, 8>(a, p, device, s) : mv_launch<TYPE, P, NT, COLS, 16>(a, p, device, s);
}

// Parts of x and groups of eight columns of a call.  The digits' four columns
// a token pay up to four tokens (65536 x 2048, Q4_K: 4 tokens 20.6 us against
// 23.1 in fp16, 8 tokens 28.8 against 28.2).
inline unsigned mv_parts(unsigned type, unsigned tokens, unsigned x_type) {
  return type == FRC_Q4_K && tokens <= 4 ? 4 : x_type == FRC_F32 ? 2 : 1;
}
inline unsigned mv_groups(unsigned cols) { return cols <= 8 ? 1 : cols <= 16 ? 2 : 4; }
inline MvPlan mv_plan(unsigned type, unsigned tokens, unsigned x_type, const MvLayout& l, unsigned sms) {
  const unsigned P = mv_parts(type, tokens, x_type);
  return mv_plan(type, P, mv_groups(tokens * P), tokens, l, sms);
}

template <unsigned TYPE>
inline cudaError_t launch_matvec(MatvecParams& a, const MvLayout& l, const MvPlan& p, unsigned x_type, int device,
                                 cudaStream_t s) {
  const unsigned P = mv_parts(TYPE, a.tokens, x_type), cols = a.tokens * P, nt = mv_groups(cols);
  a.tile_bytes = l.tile_bytes; a.shift_at = l.shift_at; a.tiles = l.tiles; a.spans = l.spans; a.pieces_last = l.pieces_last;
  a.slice = p.slice; a.chunk = p.chunk; a.cluster = p.cluster;
  if constexpr (TYPE == kQ4K) {
    if (P == 4) return nt == 1 ? mv_launch_w<TYPE, 4, 1, 8>(a, p, device, s) : mv_launch_w<TYPE, 4, 2, 8>(a, p, device, s);
  } else {
    if (P == 2 && cols <= 2 && p.share) return mv_launch_w<TYPE, 2, 1, 2>(a, p, device, s);
    if (P == 2 && cols <= 4 && p.share) return mv_launch_w<TYPE, 2, 1, 4>(a, p, device, s);
    if (P == 1 && cols <= 1 && p.share) return mv_launch_w<TYPE, 1, 1, 1>(a, p, device, s);
    if (P == 1 && cols <= 2 && p.share) return mv_launch_w<TYPE, 1, 1, 2>(a, p, device, s);
    if (P == 1 && cols <= 4 && p.share) return mv_launch_w<TYPE, 1, 1, 4>(a, p, device, s);
  }
  if (P == 2) {
    if (nt == 1) return mv_launch_w<TYPE, 2, 1, 8>(a, p, device, s);
    if (nt == 2) return mv_launch_w<TYPE, 2, 2, 8>(a, p, device, s);
    return mv_launch_w<TYPE, 2, 4, 8>(a, p, device, s);
  }
  if (nt == 1) return mv_launch_w<TYPE, 1, 1, 8>(a, p, device, s);
  return mv_launch_w<TYPE, 1, 2, 8>(a, p, device, s);
}

}  // namespace frc
