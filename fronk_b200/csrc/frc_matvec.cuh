// frc_matvec.cuh - products of one dense 4-bit matrix with 1-16 token vectors.
//
// y[t][r] = sum_j W[r][j] x[t][j], W in the row formats of the expert slices:
// Q4_K (w = d sc_g q - dmin mi_g, a 6-bit scale and minimum per 32 weights
// under fp16 super scales per 256) or MXFP4 (w = 2^(e-127) E2M1 per 32).
//
// The weights' bytes bound it, so the work per weight has to stay under the
// ~1.5 integer and ~3 other lane operations that one weight may cost at the
// HBM rate (43 weights a clock and SM).  Both formats are exact in fp16, so a
// warp multiplies 16 rows x 256 columns ("a span of a tile") on the tensor
// cores (m16n8k16, fp32 accumulators) with the vectors as the eight columns:
//   Q4_K: nibble pairs masked out of a word are fp16 subnormals q 2^-24; one
//     half2 product by sc makes q sc 2^-24 (10 bits, exact), so a whole span
//     accumulates without touching the scales, and the minima are one more
//     product, of mi with the sums of x over each 32.
//   MXFP4: the hardware's E2M1 -> fp16 conversion, and per 32 weights one fma
//     with 2^(e - base), base the row's largest exponent.
// x is scaled by a power of two per span (largest value in [2^13, 2^14)) and
// held in fp16: a bf16 value fits (P = 1), an fp32 value is the sum of two
// (P = 2; 22 of its 24 bits, or 2^-34 of the span's largest value where that
// is more: half a step of an fp16 hi, then of an fp16 lo part).  The two parts
// are columns of their own.
#pragma once
#include <cuda_bf16.h>

#include "../../include/fronk_b200.h"
#include "frc_device.cuh"

namespace frc {

constexpr unsigned kMvSpan = 256;          // weights of a row in one step
constexpr unsigned kMvTile = 16;           // rows of one step
constexpr unsigned kMvColPad = 64;         // bytes: columns start in alternate halves of the banks

// Device layout: tile after tile (16 rows, the last one filled up with zero
// rows), in it span after span of [scales][pieces], a piece being 64 weights
// of the 16 rows: lane (g = lane / 4, q = lane % 4) owns 16 bytes {row g
// group 0, row g + 8 group 0, row g group 1, row g + 8 group 1}, a word of
// eight weights 32 group + 8 q + 0..7 each, so that a load is the fragment.
// The last span stops at the last piece that holds weights.
//   Q4_K scales: the 16 header bytes of each row (d, dmin, packed 6 bits).
//   MXFP4 scales: 8 exponents a row, relative to the row's largest (127 is
//   that one, 0 stands for nothing); the largest are 16 bytes a tile at `base`.
struct MvLayout {
  unsigned tiles, spans, pieces_last, span_bytes, scale_bytes;
  size_t tile_bytes, base_at, total;
};
inline MvLayout mv_layout(unsigned type, unsigned rows, unsigned n) {
  MvLayout l;
  l.tiles = (rows + kMvTile - 1) / kMvTile;
  l.spans = (n + kMvSpan - 1) / kMvSpan;
  l.pieces_last = (n - (l.spans - 1) * kMvSpan + 63) / 64;
  l.scale_bytes = type == FRC_Q4_K ? 256 : 128;
  l.span_bytes = l.scale_bytes + 2048;
  l.tile_bytes = static_cast<size_t>(l.spans - 1) * l.span_bytes + l.scale_bytes + 512 * l.pieces_last;
  l.base_at = l.tile_bytes * l.tiles;
  l.total = l.base_at + static_cast<size_t>(l.tiles) * kMvTile;
  return l;
}

// Reference rows -> the layout above, one CTA a tile; scales that are not
// finite (Q4_K super scales, MXFP4 exponent 255) raise the numeric bit.
template <unsigned TYPE>
__global__ void __launch_bounds__(256) matrix_layout_kernel(const uint8_t* __restrict__ src, uint8_t* dst, MvLayout l,
                                                            unsigned rows, unsigned n, unsigned row_bytes,
                                                            unsigned* flag) {
  __shared__ unsigned s_base[kMvTile];
  const unsigned tile = blockIdx.x, tid = threadIdx.x;
  const uint8_t* in = src + static_cast<size_t>(tile) * kMvTile * row_bytes;
  uint8_t* out = dst + tile * l.tile_bytes;
  const unsigned left = rows - tile * kMvTile < kMvTile ? rows - tile * kMvTile : kMvTile;
  bool bad = false;
  if (TYPE == kMXFP4) {
    if (tid < kMvTile) s_base[tid] = 0;
    __syncthreads();
    for (unsigned i = tid; i < left * (n / 32); i += 256) {
      const unsigned r = i / (n / 32), b = i % (n / 32), e = in[static_cast<size_t>(r) * row_bytes + 17 * b];
      bad |= e == 255;
      atomicMax(&s_base[r], e);
    }
    __syncthreads();
    if (tid < kMvTile) dst[l.base_at + static_cast<size_t>(tile) * kMvTile + tid] = static_cast<uint8_t>(s_base[tid]);
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
        const unsigned v = in[static_cast<size_t>(r) * row_bytes + 17 * b], base = s_base[r];
        e = base - v < 127u ? v + 127u - base : 0u;
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
          for (unsigned j = 0; j < 8; ++j)  // pair j / 2: its two weights in the word's halves
            v |= (q[j] >> (4 * (grp & 1)) & 15u) << (4 * (j / 2) + 16 * (j & 1));
        } else {
          const uint8_t* q = b + 17 * (8 * s + grp) + 1 + (k0 & 8);
#pragma unroll
          for (unsigned j = 0; j < 8; ++j) v |= (q[j] >> (k0 < 16 ? 0 : 4) & 15u) << (4 * j);
        }
      }
      reinterpret_cast<unsigned*>(o + l.scale_bytes)[i] = v;
    }
  }
  if (bad) atomicOr(flag, kStNumeric);
}

struct MatvecParams {
  const uint8_t* w;
  const void* x;
  void* y;
  size_t x_stride, y_stride;  // elements between tokens
  size_t tile_bytes, base_at;
  unsigned rows, n, tokens, tiles, spans, pieces_last;
  unsigned slice;             // spans of K a CTA works on (all, or a share where a cluster splits K)
  unsigned chunk;             // spans of x in shared memory at a time, at most the slice
  unsigned split;             // warps that share a tile's spans
  unsigned cluster;           // CTAs that share K
  unsigned x_vec, y_bf16;     // x rows are 16-byte aligned; y is bf16
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
__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
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

// A lane's share of one span of a tile.
template <unsigned TYPE>
struct MvFrag {
  static constexpr unsigned kScale = TYPE == kQ4K ? 256 : 128, kBytes = kScale + 2048;
  uint4 w[4];
  uint4 s[TYPE == kQ4K ? 2 : 1];  // Q4_K: headers of rows g and g + 8; MXFP4: their exponents, 8 bytes each

  __device__ __forceinline__ void load(const uint8_t* p, unsigned pieces, unsigned lane) {  // p: the span
    const uint8_t* q = p + 16 * lane + kScale;
    if (TYPE == kQ4K || pieces == 4) {
#pragma unroll
      for (unsigned j = 0; j < 4; ++j) w[j] = ldg_stream(q + 512 * j);
    } else {
#pragma unroll
      for (unsigned j = 0; j < 4; ++j) w[j] = j < pieces ? ldg_stream(q + 512 * j) : make_uint4(0, 0, 0, 0);
    }
    if (TYPE == kQ4K) {
      s[0] = ldg_stream(p + 16 * (lane / 4));
      s[TYPE == kQ4K ? 1 : 0] = ldg_stream(p + 128 + 16 * (lane / 4));
    } else {
      const uint2 e0 = __ldg(reinterpret_cast<const uint2*>(p) + lane / 4);
      const uint2 e1 = __ldg(reinterpret_cast<const uint2*>(p) + 8 + lane / 4);
      s[0] = make_uint4(e0.x, e0.y, e1.x, e1.y);
    }
  }
};

// The vectors of one K chunk in shared memory: columns of fp16 parts, per
// token and span the power of two, and for Q4_K the sums over each 32 as
// eight hi and eight lo parts (x 2^-5: they fit fp16).
struct MvShared {
  uint8_t* col;     // [tokens * P][chunk * 512 + pad]
  float* scale;     // [tokens][chunk]
  uint8_t* sums;    // [tokens][chunk][32]
  float* part;      // [warps][values][32], when warps or CTAs share a tile
};
inline __host__ __device__ unsigned mv_col_bytes(unsigned chunk) { return chunk * 512 + kMvColPad; }

// Spans first .. first + count of every token into shared memory, a warp a
// (token, span) at a time with the values of U of them on their way.
template <unsigned TYPE, unsigned P>
__device__ __forceinline__ void mv_prepare(const MatvecParams& a, const MvShared& sh, unsigned first, unsigned count) {
  constexpr unsigned U = P == 2 ? 4 : 8, R = P == 2 ? 8 : 4;
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = blockDim.x / 32, units = a.tokens * count;
  for (unsigned u0 = warp; u0 < units; u0 += U * warps) {
    uint32_t raw[U][R];
#pragma unroll
    for (unsigned i = 0; i < U; ++i) {
      const unsigned u = u0 + i * warps, t = u / count, s = u - t * count, k = (first + s) * kMvSpan + 8 * lane;
#pragma unroll
      for (unsigned j = 0; j < R; ++j) raw[i][j] = 0;
      if (u >= units || k >= a.n) continue;
      if (P == 2) {
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
        v[j] = __uint_as_float(P == 2 ? raw[i][j % R] : j & 1 ? raw[i][j / 2] & 0xffff0000u : raw[i][j / 2] << 16);
      unsigned top = 0;
#pragma unroll
      for (unsigned j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
      top = __reduce_max_sync(0xffffffffu, top);
      // x = v 2^ex; a span that is not finite has the scale NaN and so its results
      int ex = static_cast<int>(top >> 23) - 127 - 13;
      if (ex < -126) ex = -126;
      const bool finite = top < 0x7f800000u;
      const float inv = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
      float sum = 0.0f;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (unsigned j = 0; j < 4; ++j) {
        // odd pairs of a Q4_K word carry 16 q
        const float f = TYPE == kQ4K && (j & 1) ? 0.0625f : 1.0f;
        float p = finite ? v[2 * j] * inv : 0.0f, q = finite ? v[2 * j + 1] * inv : 0.0f;
        sum += p + q;
        p *= f;
        q *= f;
        const __half2 h = __floats2half2_rn(p, q);
        hi[j] = *reinterpret_cast<const uint32_t*>(&h);
        const float2 b = __half22float2(h);
        const __half2 l = __floats2half2_rn(p - b.x, q - b.y);
        lo[j] = *reinterpret_cast<const uint32_t*>(&l);
      }
      uint8_t* c = sh.col + (t * P) * mv_col_bytes(a.chunk) + 512 * s + 16 * lane;
      *reinterpret_cast<uint4*>(c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if (P == 2) *reinterpret_cast<uint4*>(c + mv_col_bytes(a.chunk)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      if (lane == 0) sh.scale[t * a.chunk + s] = finite ? __uint_as_float(static_cast<uint32_t>(127 + ex) << 23) : NAN;
      if (TYPE == kQ4K) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= 0.03125f;
        if (lane % 4 == 0) {
          const __half h = __float2half_rn(sum), l = __float2half_rn(sum - __half2float(h));
          __half* o = reinterpret_cast<__half*>(sh.sums + (t * a.chunk + s) * 32) + lane / 4;
          o[0] = h;
          o[8] = l;
        }
      }
    }
  }
}

// A lane's shared-memory addresses: its columns, their sums, its tokens' scales.
template <unsigned P, unsigned NT>
struct MvLane {
  static constexpr unsigned kTok = P == 2 ? 1 : 2;  // tokens of a lane's results in a group of eight columns
  uint32_t col[NT], sums[NT], scale[NT][kTok];
  unsigned sel;  // bytes 2 q and 2 q + 1
  __device__ __forceinline__ MvLane(const MatvecParams& a, const MvShared& sh, unsigned lane) {
    const unsigned g = lane / 4, q = lane % 4, cols = a.tokens * P;
    sel = 2 * q | (2 * q + 1) << 4;
#pragma unroll
    for (unsigned t = 0; t < NT; ++t) {
      const unsigned c = 8 * t + g < cols ? 8 * t + g : 0;  // columns past the tokens are not looked at
      col[t] = smem_u32(sh.col) + c * mv_col_bytes(a.chunk) + 16 * q;
      sums[t] = smem_u32(sh.sums) + (c / P) * a.chunk * 32 + 4 * q;
#pragma unroll
      for (unsigned k = 0; k < kTok; ++k) {
        const unsigned tok = P == 2 ? 4 * t + q : 8 * t + 2 * q + k;
        scale[t][k] = smem_u32(sh.scale) + 4 * ((tok < a.tokens ? tok : 0) * a.chunk);
      }
    }
  }
};

// One span (s of the chunk) of a tile times the columns; acc: [row g | row
// g + 8] of the lane's token(s) in each group of eight columns.  FOLD: the
// 6-bit scales of Q4_K go into the weights (eight half2 products per 32
// columns of a tile), else onto the results (four fma per eight columns).
template <unsigned TYPE, unsigned P, unsigned NT>
__device__ __forceinline__ void mv_span(const MvLane<P, NT>& ln, const MvFrag<TYPE>& f, unsigned s, unsigned lane,
                                        float (&acc)[NT * (P == 2 ? 2 : 4)]) {
  constexpr bool FOLD = TYPE == kQ4K && NT > 2;
  float sum[NT][4];
#pragma unroll
  for (unsigned t = 0; t < NT; ++t) sum[t][0] = sum[t][1] = sum[t][2] = sum[t][3] = 0.0f;
  uint32_t xc[NT];
#pragma unroll
  for (unsigned t = 0; t < NT; ++t) xc[t] = ln.col[t] + 512 * s;
  if constexpr (TYPE == kQ4K) {
    uint32_t sc[2][2], mi[2][2];
    float d[2], dm[2], m[NT][4];
#pragma unroll
    for (unsigned h = 0; h < 2; ++h) {
      const uint4 b = f.s[h];
      d[h] = h2f(b.x & 0xffffu) * 16777216.0f;   // against q sc 2^-24
      dm[h] = h2f(b.x >> 16) * 536870912.0f;     // against mi 2^-24 and sums 2^-5
      sc[h][0] = b.y & 0x3f3f3f3fu;
      mi[h][0] = b.z & 0x3f3f3f3fu;
      sc[h][1] = (b.w & 0x0f0f0f0fu) | (b.y >> 2 & 0x30303030u);
      mi[h][1] = (b.w >> 4 & 0x0f0f0f0fu) | (b.z >> 2 & 0x30303030u);
    }
    // minima of groups 2 q and 2 q + 1 as fp16 subnormals mi 2^-24, against the sums' hi and lo parts; the column
    // of an fp32 token's lo part takes them too and is left out below
    const uint32_t m0 = prmt(prmt(mi[0][0], mi[0][1], ln.sel), 0, 0x4140), m1 = prmt(prmt(mi[1][0], mi[1][1], ln.sel), 0, 0x4140);
#pragma unroll
    for (unsigned t = 0; t < NT; ++t) mma_f16_first(m[t], m0, m1, m0, m1, lds32(ln.sums[t] + 32 * s), lds32(ln.sums[t] + 32 * s + 16));
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const uint32_t w[4] = {f.w[j].x, f.w[j].y, f.w[j].z, f.w[j].w};
#pragma unroll
      for (unsigned e = 0; e < 2; ++e) {
        const unsigned grp = 2 * j + e;
        uint32_t av[2][4];
        float k[2];
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
          const uint32_t v = w[2 * e + h], u = v >> 8;
          av[h][0] = v & 0x000f000fu;
          av[h][1] = v & 0x00f000f0u;
          av[h][2] = u & 0x000f000fu;
          av[h][3] = u & 0x00f000f0u;
          if (FOLD) {
            // 1024 + sc in both halves, less 1024
            const uint32_t c = hsub2(prmt(sc[h][grp / 4], 0x64646464u, 0x4040u | (grp % 4) * 0x0101u), 0x64006400u);
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) av[h][i] = hmul2(av[h][i], c);
          } else {
            k[h] = static_cast<float>(sc[h][grp / 4] >> (8 * (grp % 4)) & 255u);
          }
        }
#pragma unroll
        for (unsigned t = 0; t < NT; ++t) {
          const uint4 b = lds128(xc[t] + 64 * grp);
          if (FOLD) {
            mma_f16(sum[t], av[0][0], av[1][0], av[0][1], av[1][1], b.x, b.y);
            mma_f16(sum[t], av[0][2], av[1][2], av[0][3], av[1][3], b.z, b.w);
          } else {
            float c[4];
            mma_f16_first(c, av[0][0], av[1][0], av[0][1], av[1][1], b.x, b.y);
            mma_f16(c, av[0][2], av[1][2], av[0][3], av[1][3], b.z, b.w);
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) sum[t][i] = fmaf(c[i], k[i / 2], sum[t][i]);
          }
        }
      }
    }
#pragma unroll
    for (unsigned t = 0; t < NT; ++t) {
#pragma unroll
      for (unsigned h = 0; h < 2; ++h) {
        if (P == 2) {
          const float v = d[h] * (sum[t][2 * h] + sum[t][2 * h + 1]) - dm[h] * m[t][2 * h];
          acc[2 * t + h] = fmaf(v, __uint_as_float(lds32(ln.scale[t][0] + 4 * s)), acc[2 * t + h]);
        } else {
#pragma unroll
          for (unsigned c = 0; c < 2; ++c) {
            const float v = d[h] * sum[t][2 * h + c] - dm[h] * m[t][2 * h + c];
            acc[4 * t + 2 * h + c] = fmaf(v, __uint_as_float(lds32(ln.scale[t][P == 2 ? 0 : c] + 4 * s)), acc[4 * t + 2 * h + c]);
          }
        }
      }
    }
  } else {
    const uint32_t ex[2][2] = {{f.s[0].x, f.s[0].y}, {f.s[0].z, f.s[0].w}};
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const uint32_t w[4] = {f.w[j].x, f.w[j].y, f.w[j].z, f.w[j].w};
#pragma unroll
      for (unsigned e = 0; e < 2; ++e) {
        const unsigned grp = 2 * j + e;
        uint32_t av[2][4];
        float k[2];
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
          e2m1_f16(w[2 * e + h], av[h]);
          k[h] = __uint_as_float((ex[h][grp / 4] >> (8 * (grp % 4)) & 255u) << 23);
        }
#pragma unroll
        for (unsigned t = 0; t < NT; ++t) {
          const uint4 b = lds128(xc[t] + 64 * grp);
          float c[4];
          mma_f16_first(c, av[0][0], av[1][0], av[0][1], av[1][1], b.x, b.y);
          mma_f16(c, av[0][2], av[1][2], av[0][3], av[1][3], b.z, b.w);
#pragma unroll
          for (unsigned i = 0; i < 4; ++i) sum[t][i] = fmaf(c[i], k[i / 2], sum[t][i]);
        }
      }
    }
#pragma unroll
    for (unsigned t = 0; t < NT; ++t) {
#pragma unroll
      for (unsigned h = 0; h < 2; ++h) {
        if (P == 2) {
          acc[2 * t + h] = fmaf(sum[t][2 * h] + sum[t][2 * h + 1], __uint_as_float(lds32(ln.scale[t][0] + 4 * s)), acc[2 * t + h]);
        } else {
#pragma unroll
          for (unsigned c = 0; c < 2; ++c)
            acc[4 * t + 2 * h + c] = fmaf(sum[t][2 * h + c], __uint_as_float(lds32(ln.scale[t][P == 2 ? 0 : c] + 4 * s)), acc[4 * t + 2 * h + c]);
        }
      }
    }
  }
}

__device__ __forceinline__ void mv_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CTAs of W warps; `split` of them share the spans of a tile, and the CTAs of
// a cluster share K.  Tiles are dealt round robin; x is prepared once a CTA,
// or once a tile and chunk where it does not fit shared memory as a whole.
// The next span's weights are on their way while one is worked on.
template <unsigned TYPE, unsigned P, unsigned NT, unsigned W>
__global__ void __launch_bounds__(32 * W, W == 8 ? 2 : 1) matvec_kernel(const MatvecParams a) {
  constexpr unsigned V = NT * (P == 2 ? 2 : 4), kBytes = MvFrag<TYPE>::kBytes;
  extern __shared__ __align__(128) uint8_t smem[];
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, q = lane % 4;
  MvShared sh;
  sh.col = smem;
  sh.sums = smem + a.tokens * P * mv_col_bytes(a.chunk);
  sh.scale = reinterpret_cast<float*>(sh.sums + (TYPE == kQ4K ? a.tokens * a.chunk * 32 : 0));
  sh.part = sh.scale + a.tokens * a.chunk;
  const MvLane<P, NT> ln(a, sh, lane);
  const unsigned split = a.split, per_cta = W / split, sub = warp / split, ks = warp % split;
  const unsigned rank = a.cluster > 1 ? blockIdx.x % a.cluster : 0, cta = blockIdx.x / a.cluster, ctas = gridDim.x / a.cluster;
  const unsigned k_first = rank * a.slice, k_end = min(a.spans, k_first + a.slice);
  bool prepared = false, bad = false;
  for (unsigned base = cta * per_cta; base < a.tiles; base += ctas * per_cta) {
    const unsigned tile = base + sub;
    float acc[V];
#pragma unroll
    for (unsigned i = 0; i < V; ++i) acc[i] = 0.0f;
    for (unsigned first = k_first; first < k_end; first += a.chunk) {
      const unsigned count = min(a.chunk, k_end - first);
      const bool any = tile < a.tiles && ks < count;
      MvFrag<TYPE> f0, f1;
      const uint8_t* p = a.w + tile * a.tile_bytes + static_cast<size_t>(first + ks) * kBytes;
      const unsigned last = a.spans - 1 - first;  // the span that may be short
      unsigned s = ks;
      const auto fetch = [&](MvFrag<TYPE>& f, unsigned at) { f.load(p, at == last ? a.pieces_last : 4, lane); };
      if (any) fetch(f0, s);
      if (!prepared || a.chunk < a.slice) {
        __syncthreads();  // every warp has left the chunk before
        mv_prepare<TYPE, P>(a, sh, first, count);
        __syncthreads();
        prepared = true;
      }
      if (any) {
        const size_t step = static_cast<size_t>(split) * kBytes;
        while (true) {
          p += step;
          if (s + split < count) fetch(f1, s + split);
          mv_span<TYPE, P, NT>(ln, f0, s, lane, acc);
          s += split;
          if (s >= count) break;
          p += step;
          if (s + split < count) fetch(f0, s + split);
          mv_span<TYPE, P, NT>(ln, f1, s, lane, acc);
          s += split;
          if (s >= count) break;
        }
      }
    }
    if (split > 1 || a.cluster > 1) {
      float* p = sh.part + (warp * V) * 32 + lane;
#pragma unroll
      for (unsigned i = 0; i < V; ++i) p[32 * i] = acc[i];
      __syncthreads();
      if (ks == 0 && split > 1) {
        for (unsigned w = 1; w < split; ++w)
#pragma unroll
          for (unsigned i = 0; i < V; ++i) acc[i] += p[32 * (w * V + i)];
        if (a.cluster > 1) {
#pragma unroll
          for (unsigned i = 0; i < V; ++i) p[32 * i] = acc[i];
        }
      }
      if (a.cluster > 1) {
        mv_cluster_sync();
        if (rank == 0 && ks == 0) {
          for (unsigned r = 1; r < a.cluster; ++r) {
            uint32_t at;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(r));
#pragma unroll
            for (unsigned i = 0; i < V; ++i) {
              float v;
              asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at + 128 * i) : "memory");
              acc[i] += v;
            }
          }
        }
        mv_cluster_sync();
      } else {
        __syncthreads();
      }
    }
    if (ks == 0 && rank == 0 && tile < a.tiles) {
#pragma unroll
      for (unsigned h = 0; h < 2; ++h) {
        const unsigned row = tile * kMvTile + g + 8 * h;
        if (row >= a.rows) continue;
        float f = 1.0f;
        if (TYPE == kMXFP4) {
          const unsigned e = a.w[a.base_at + row];
          f = __uint_as_float(e ? e << 23 : 0x00400000u);
        }
#pragma unroll
        for (unsigned i = 0; i < V / 2; ++i) {
          const unsigned tok = P == 2 ? 4 * i + q : 8 * (i / 2) + 2 * q + i % 2;
          if (tok >= a.tokens) continue;
          float v = acc[P == 2 ? 2 * i + h : 4 * (i / 2) + 2 * h + i % 2];
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
    }
  }
  if (bad) atomicOr(a.status, kStNumeric);
}

// ------------------------------------------------------------ host side

struct MvPlan {
  unsigned warps, slice, chunk, split, cluster, grid, smem;
};

constexpr unsigned kMvSmemSm = 228 * 1024, kMvSmemCta = 227 * 1024;

// Shared memory of a CTA; the parts only where warps or CTAs share tiles.
inline size_t mv_smem(unsigned type, unsigned P, unsigned tokens, unsigned values, unsigned warps, unsigned chunk, bool part) {
  return static_cast<size_t>(tokens) * P * mv_col_bytes(chunk) +
         static_cast<size_t>(tokens) * chunk * ((type == FRC_Q4_K ? 32 : 0) + 4) + (part ? static_cast<size_t>(warps) * values * 128 : 0);
}

// Chooses the warps a CTA, the CTAs that share K and the warps that share a
// tile by an estimate of the time in steps of one span a warp (about 0.3 us):
// the preparation of x (a batch of spans a warp, three steps), the rounds of
// tiles, and four steps for a cluster's exchange.
inline MvPlan mv_plan(unsigned type, unsigned P, unsigned nt, unsigned tokens, const MvLayout& l, unsigned sms) {
  const unsigned values = nt * (P == 2 ? 2 : 4), batch = P == 2 ? 4 : 8;
  MvPlan best{};
  double least = 1e30;
  for (unsigned warps = 8; warps <= 16; warps *= 2) {
    for (unsigned cluster = 1; cluster <= 8 && cluster <= l.spans; cluster *= 2) {
      MvPlan p{};
      p.warps = warps;
      p.cluster = cluster;
      p.slice = p.chunk = (l.spans + cluster - 1) / cluster;
      const size_t limit = warps == 8 ? (kMvSmemSm - 2048) / 2 : kMvSmemCta;
      if (warps == 8 && mv_smem(type, P, tokens, values, warps, p.chunk, true) > limit) continue;
      while (mv_smem(type, P, tokens, values, warps, p.chunk, true) > limit) p.chunk = (p.chunk + 1) / 2;
      // clusters do not tile the SMs of every GPC
      const unsigned resident = sms * (warps == 8 ? 2 : 1) / cluster * (cluster > 1 ? 7 : 8) / 8;
      if (!resident) continue;
      for (unsigned split = 1; split <= warps && (split == 1 || split / 2 < p.chunk); split *= 2) {
        const unsigned per = warps / split, groups = (l.tiles + per - 1) / per, rounds = (groups + resident - 1) / resident;
        const unsigned steps = (p.chunk + split - 1) / split * ((p.slice + p.chunk - 1) / p.chunk);
        const double prep = 3.0 * ((tokens * p.chunk + warps * batch - 1) / (warps * batch)) * (p.chunk < p.slice ? rounds * ((p.slice + p.chunk - 1) / p.chunk) : 1);
        const double t = prep + static_cast<double>(rounds) * (steps + (split > 1 ? 0.5 : 0.1) + (cluster > 1 ? 4 : 0));
        if (t < least * 0.98) {
          least = t;
          best = p;
          best.split = split;
          best.grid = (groups < resident ? groups : resident) * cluster;
        }
      }
    }
  }
  best.smem = static_cast<unsigned>(mv_smem(type, P, tokens, values, best.warps, best.chunk, best.split > 1 || best.cluster > 1));
  return best;
}

template <unsigned TYPE, unsigned P, unsigned NT, unsigned W>
inline cudaError_t mv_launch(const MatvecParams& a, const MvPlan& p, cudaStream_t s) {
  if (p.smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(matvec_kernel<TYPE, P, NT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(p.smem));
    if (e != cudaSuccess) return e;
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
  return cudaLaunchKernelEx(&cfg, matvec_kernel<TYPE, P, NT, W>, a);
}
template <unsigned TYPE, unsigned P, unsigned NT>
inline cudaError_t mv_launch_w(const MatvecParams& a, const MvPlan& p, cudaStream_t s) {
  return p.warps == 8 ? mv_launch<TYPE, P, NT, 8>(a, p, s) : mv_launch<TYPE, P, NT, 16>(a, p, s);
}

template <unsigned TYPE>
inline cudaError_t launch_matvec(MatvecParams& a, const MvLayout& l, unsigned x_type, unsigned sms, cudaStream_t s) {
  const unsigned P = x_type == FRC_F32 ? 2 : 1, cols = a.tokens * P, nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  MvPlan p = mv_plan(TYPE, P, nt, a.tokens, l, sms);
#ifdef MV_ENV
  if (const char* e = getenv("MV_PLAN")) {  // warps,cluster,split,grid groups per resident
    unsigned w, c, sp;
    if (sscanf(e, "%u,%u,%u", &w, &c, &sp) == 3) {
      const unsigned values = nt * (P == 2 ? 2 : 4);
      p.warps = w; p.cluster = c; p.split = sp; p.slice = p.chunk = (l.spans + c - 1) / c;
      while (mv_smem(TYPE, P, a.tokens, values, w, p.chunk, true) > (w == 8 ? (kMvSmemSm - 2048) / 2 : kMvSmemCta)) p.chunk = (p.chunk + 1) / 2;
      const unsigned per = w / sp, groups = (l.tiles + per - 1) / per, resident = sms * (w == 8 ? 2 : 1) / c * (c > 1 ? 7 : 8) / 8;
      p.grid = (groups < resident ? groups : resident) * c;
      p.smem = mv_smem(TYPE, P, a.tokens, values, w, p.chunk, sp > 1 || c > 1);
    }
    fprintf(stderr, "plan warps %u cluster %u split %u slice %u chunk %u grid %u smem %u\n", p.warps, p.cluster, p.split, p.slice, p.chunk, p.grid, p.smem);
  }
#endif
  a.tile_bytes = l.tile_bytes; a.base_at = l.base_at; a.tiles = l.tiles; a.spans = l.spans; a.pieces_last = l.pieces_last;
  a.slice = p.slice; a.chunk = p.chunk; a.split = p.split; a.cluster = p.cluster;
  if (P == 2) {
    if (nt == 1) return mv_launch_w<TYPE, 2, 1>(a, p, s);
    if (nt == 2) return mv_launch_w<TYPE, 2, 2>(a, p, s);
    return mv_launch_w<TYPE, 2, 4>(a, p, s);
  }
  if (nt == 1) return mv_launch_w<TYPE, 1, 1>(a, p, s);
  return mv_launch_w<TYPE, 1, 2>(a, p, s);
}

}  // namespace frc
