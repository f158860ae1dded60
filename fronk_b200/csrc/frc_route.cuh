// frc_route.cuh - routing of a MoE layer: the ten experts of each token and
// their gates from the expert logits, the per-expert counts and the balance
// loss, and the gradient of both with respect to the logits.
//
// Per token (row) of E logits l (10 <= E <= 512, -inf: masked out):
//   chosen: the ten largest, descending, ties by the lower index;
//   gate_i = exp(l_i - max) / sum over the chosen; 0 where l_i = -inf;
//   p = softmax(l) over all E.
// Over the N valid tokens: count_e = tokens that chose e (never a masked
// expert), prob_e = mean p_e, loss = E sum_e count_e / (10 N) prob_e.
//
// A warp takes a row, 16 logits a lane; the logits' bytes bound it.  Measured
// on one B200, graph replays, 512 experts fp32: statistics of 65,536 rows 27.0
// us (5.0 TB/s), selection and statistics of 16,384 rows 17.2 us and of 65,536
// rows 43.5 (430 instructions a row bound it), both gradients of 16,384 rows
// 14.9 us, one row's selection 2.4 us.  Rows that a shared column puts 513
// elements apart are not 16-byte aligned: selection and statistics of 16,384
// rows 20.8 us, both gradients 16.9.
#pragma once
#include <cuda_bf16.h>

#include "../../include/fronk_b200.h"
#include "frc_device.cuh"

namespace frc {

constexpr unsigned kTopK = 10, kGates = 11, kMaxExperts = 512;
constexpr unsigned kRouteSlots = kMaxExperts / 32;  // logits a lane holds
constexpr unsigned kRouteWarps = 24;                // warps a CTA whose rows pass through registers alone, at most
constexpr unsigned kRouteSums = 16;                 // arrays of sums a CTA folds its warps into; warps of a cluster's CTA
constexpr unsigned kRouteRows = 8;                  // rows a CTA that makes statistics, at least, while SMs are free
constexpr unsigned kRouteCtas = 160;                // CTAs that make statistics (one an SM), at most
constexpr unsigned kRouteCluster = 8;               // CTAs that finish them

struct RouteParams {
  const void* logits;
  size_t stride;         // elements between rows
  const uint8_t* valid;  // null: every row
  const uint16_t* expert_in;
  uint16_t* expert;
  float* gate;
  unsigned tokens, experts, shared;
  // statistics: [CTA][E] {sum of p, count}, [CTA] valid rows
  float2* part;
  unsigned* pvalid;
  unsigned* status;
};

struct RouteFinish {
  const float2* part;
  const unsigned* pvalid;
  unsigned parts, experts;
  float* loss;
  unsigned* count;
  float* prob;
};

struct RouteBackwardParams {
  const void* logits;
  size_t stride, d_stride;
  const uint8_t* valid;
  const uint16_t* expert;
  const float* d_gate;    // null: no gate gradient
  const unsigned* count;  // [E + 1], the last entry N; null: no balance gradient
  const float* d_loss;
  void* d_logits;
  unsigned tokens, experts, shared;
  unsigned* status;
};

template <typename L>
__device__ __forceinline__ float logit(const L* p);
template <>
__device__ __forceinline__ float logit<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float logit<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Unsigned keys in the order of floats (no NaN); 0 lies below every float.
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned b = __float_as_uint(v);
  return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (unsigned o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Over lanes 0-15, for each of them.
__device__ __forceinline__ float chosen_sum(float v) {
#pragma unroll
  for (unsigned o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Maxima that are NaN when a value is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float warp_max_nan(float v) {
  float d;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float warp_max(float v) {
  float d;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float warp_min(float v) {
  float d;
  asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float rcp(float v) {  // within one step; v is a sum of exponentials, at least 1
  float d;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }
// exp(v - m) with v <= m, m finite; v may be -inf.
__device__ __forceinline__ float exp_below(float v, float m) {
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"((v - m) * 1.4426950408889634f));
  return d;
}

// The largest of a lane's slots (NaN when one is), as a tree.
__device__ __forceinline__ float row_max(const float (&v)[kRouteSlots]) {
  static_assert(kRouteSlots == 16, "5 threes and one, then 2 threes");
  float m[5];
#pragma unroll
  for (unsigned i = 0; i < 5; ++i) m[i] = max_nan(v[3 * i], v[3 * i + 1], v[3 * i + 2]);
  return max_nan(max_nan(m[0], m[1], m[2]), max_nan(m[3], m[4], v[15]));
}

// Two fp32 operations an instruction: a row's arithmetic is 16 values a lane.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d.v) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpack2(F2 d, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d.v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}

// A row's E logits over a warp, kRouteSlots a lane: V neighbours a load (V = 1
// where rows are not 16-byte aligned), slot i of a lane being column
// col<V>(i, lane); columns past E are -inf.
template <unsigned V>
__device__ __forceinline__ unsigned col(unsigned i, unsigned lane) {
  return i / V * (32 * V) + V * lane + i % V;
}
// FULL: E is kMaxExperts (the framework's expert count), no slot is past it.
template <typename L, unsigned V, bool FULL>
struct RowLoad {
  static constexpr unsigned kWords = V == 1 ? kRouteSlots : kRouteSlots * sizeof(L) / 4;
  uint32_t w[kWords];  // fp32 bits, or pairs of bf16, or (V = 1) a value's bits each

  static __device__ __forceinline__ uint32_t raw(const float* p) { return *reinterpret_cast<const uint32_t*>(p); }
  static __device__ __forceinline__ uint32_t raw(const __nv_bfloat16* p) { return *reinterpret_cast<const uint16_t*>(p); }
  __device__ __forceinline__ void load(const L* row, unsigned E, unsigned lane) {
    if constexpr (V == 1) {
#pragma unroll
      for (unsigned i = 0; i < kRouteSlots; ++i) {  // as it lies: nothing waits for a value here
        const unsigned c = lane + 32 * i;
        w[i] = FULL || c < E ? raw(row + c) : (sizeof(L) == 4 ? 0xff800000u : 0xff80u);
      }
    } else {
#pragma unroll
      for (unsigned j = 0; j < kRouteSlots / V; ++j) {
        const unsigned c = col<V>(j * V, lane);
        uint4 v;
        if (FULL || c + V <= E) {
          v = *reinterpret_cast<const uint4*>(row + c);
        } else if constexpr (sizeof(L) == 4) {
          uint32_t e[4];
#pragma unroll
          for (unsigned k = 0; k < 4; ++k) e[k] = __float_as_uint(c + k < E ? logit(row + c + k) : -INFINITY);
          v = make_uint4(e[0], e[1], e[2], e[3]);
        } else {
          uint32_t e[4];
#pragma unroll
          for (unsigned k = 0; k < 4; ++k) {
            const float x = c + 2 * k < E ? logit(row + c + 2 * k) : -INFINITY, y = c + 2 * k + 1 < E ? logit(row + c + 2 * k + 1) : -INFINITY;
            e[k] = __float_as_uint(x) >> 16 | (__float_as_uint(y) & 0xffff0000u);
          }
          v = make_uint4(e[0], e[1], e[2], e[3]);
        }
        w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ float value(unsigned i) const {
    if constexpr (sizeof(L) == 4) return __uint_as_float(w[i]);
    else if constexpr (V == 1) return __uint_as_float(w[i] << 16);
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};

// A row on its way through shared memory: a lane fetches the columns that it
// holds into the warp's buffer, columns past E are -inf.
template <typename L, unsigned V, bool FULL>
__device__ __forceinline__ void stage_row(L* buf, const L* row, unsigned E, unsigned lane) {
  static_assert(V * sizeof(L) == 16, "16 bytes a copy");
#pragma unroll
  for (unsigned j = 0; j < kRouteSlots / V; ++j) {
    const unsigned c = col<V>(j * V, lane);
    if (FULL || c + V <= E) {
      cp_async16(buf + c, row + c);
    } else {
#pragma unroll
      for (unsigned k = 0; k < V; ++k) buf[c + k] = c + k < E ? row[c + k] : static_cast<L>(-INFINITY);
    }
  }
}

// e = exp(v - m) of a lane's slots, in pairs; returns their sum.
__device__ __forceinline__ float exp_row(const float (&v)[kRouteSlots], float m, F2 (&e)[kRouteSlots / 2]) {
  const F2 shift = pack2(-m, -m), log2e = pack2(1.4426950408889634f, 1.4426950408889634f);
  F2 z = pack2(0.0f, 0.0f), z1 = z;
#pragma unroll
  for (unsigned i = 0; i < kRouteSlots / 2; ++i) {
    float x, y;
    unpack2(mul2(add2(pack2(v[2 * i], v[2 * i + 1]), shift), log2e), x, y);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y));
    e[i] = pack2(x, y);
    if (i & 1) z1 = add2(z1, e[i]);
    else z = add2(z, e[i]);
  }
  float x, y;
  unpack2(add2(z, z1), x, y);
  return x + y;
}

// A warp's room for its candidates: their columns, then their keys.
constexpr unsigned kLaneCand = 4;
union RouteCand {
  __nv_bfloat16 top[32];
  uint16_t column[32];
  uint64_t key[32];
};
// Slot of a lane's column set whose number is not known when compiled.
template <unsigned V>
__device__ __forceinline__ unsigned col_at(unsigned i, unsigned lane) {
  return V == 1 ? lane + 32 * i : (i / V) * (32 * V) + V * lane + (i & (V - 1));
}

// The ten largest of a row in order, ties by the lower column: lane r < 10
// gets the r-th one's column and value.
//
// The tenth largest of the lanes' maxima bounds the tenth largest logit from
// below (a lane's rank is counted among all lanes' distances from the largest
// rounded to bf16: any rounding leaves ten maxima at or above the bound), so only the logits at or above it (a dozen as a rule) are collected
// and ranked against one another by {order of the value, lower column first}
// as one integer.  Where a lane has more than four of them or the warp more
// than 32 (ties), or the bound is -inf (few logits left), ten searches over
// the whole row choose one by one.
template <typename L, unsigned V>
__device__ __forceinline__ void choose(const float (&v)[kRouteSlots], const L* row, unsigned E, unsigned lane, float top,
                                       float m, RouteCand* cand, unsigned* id, float* val) {
  const __nv_bfloat16 rough = __float2bfloat16_rn(top - m);
  cand->top[lane] = rough;
  __syncwarp();
  const __nv_bfloat162 own = __bfloat162bfloat162(rough);
  __nv_bfloat162 above[4];
#pragma unroll
  for (unsigned k = 0; k < 4; ++k) {
    const uint4 w = reinterpret_cast<const uint4*>(cand->top)[k];
    const uint32_t o[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const __nv_bfloat162 gt = __hgt2(*reinterpret_cast<const __nv_bfloat162*>(&o[j]), own);
      above[j] = k ? __hadd2(above[j], gt) : gt;
    }
  }
  const __nv_bfloat162 sum = __hadd2(__hadd2(above[0], above[1]), __hadd2(above[2], above[3]));
  const float bound = warp_min(__low2float(sum) + __high2float(sum) < kTopK ? top : INFINITY);
  __syncwarp();
  bool done = false;
  if (bound > -INFINITY) {
    unsigned mine = 0, total = 0;  // the lane's slots at or above the bound
    // the signs of v - bound; 0 - bound is +0 for either zero, so that a zero less a zero is +0
    const float less = 0.0f - bound;
    const F2 below = pack2(less, less);
#pragma unroll
    for (unsigned i = kRouteSlots / 2; i-- > 0;) {
      float x, y;
      unpack2(add2(pack2(v[2 * i], v[2 * i + 1]), below), x, y);
      mine = __funnelshift_l(__float_as_uint(y), mine, 1);
      mine = __funnelshift_l(__float_as_uint(x), mine, 1);
    }
    mine ^= (1u << kRouteSlots) - 1u;
    done = !__any_sync(0xffffffffu, __popc(mine) > kLaneCand);
    if (done) {
      const unsigned before = (1u << lane) - 1u;
#pragma unroll
      for (unsigned k = 0; k < kLaneCand; ++k) {
        const unsigned with = __ballot_sync(0xffffffffu, mine);
        if (!with) break;
        const unsigned place = total + __popc(with & before);
        if (mine && place < 32) cand->column[place] = static_cast<uint16_t>(col_at<V>(__ffs(mine) - 1, lane));
        mine &= mine - 1;
        total += __popc(with);
      }
      done = total <= 32;
    }
    if (done) {
      __syncwarp();
      uint64_t key = 0;
      if (lane < total) {
        const unsigned c = cand->column[lane];
        key = static_cast<uint64_t>(order_key(logit(row + c) + 0.0f)) << 32 | ~c;  // -0 becomes +0: equal logits are ties
      }
      __syncwarp();
      cand->key[lane] = key;
      __syncwarp();
      unsigned rank = 0;
      for (unsigned k = 0; k < total; k += 4) {
        const ulonglong2 a = reinterpret_cast<const ulonglong2*>(cand->key)[k / 2], b = reinterpret_cast<const ulonglong2*>(cand->key)[k / 2 + 1];
        rank += a.x > key ? 1u : 0u;
        rank += a.y > key ? 1u : 0u;
        rank += b.x > key ? 1u : 0u;
        rank += b.y > key ? 1u : 0u;
      }
      __syncwarp();
      if (lane < total) cand->key[rank] = key;  // ranks are distinct
      __syncwarp();
      const uint64_t r = cand->key[lane < total ? lane : 0];
      *id = ~static_cast<unsigned>(r);
      *val = key_value(static_cast<unsigned>(r >> 32));
    }
  }
  if (!done) {
    unsigned left = 0;
#pragma unroll
    for (unsigned i = 0; i < kRouteSlots; ++i) left |= (col<V>(i, lane) < E ? 1u : 0u) << i;
    for (unsigned r = 0; r < kTopK; ++r) {
      unsigned best = 0, at = 0;
#pragma unroll
      for (unsigned i = 0; i < kRouteSlots; ++i) {
        const unsigned k = left >> i & 1u ? order_key(v[i] + 0.0f) : 0u;
        if (k > best) { best = k; at = i; }
      }
      const unsigned high = __reduce_max_sync(0xffffffffu, best);
      const unsigned win = __reduce_min_sync(0xffffffffu, best == high ? col<V>(at, lane) : 0xffffffffu);
      if (best == high && col<V>(at, lane) == win) left &= ~(1u << at);
      if (lane == r) { *id = win; *val = key_value(high); }
    }
  }
  __syncwarp();
}

// The cluster that makes prob, count and the loss deals the experts over its CTAs.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of the same shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_map(const void* p, uint32_t rank) {
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(p)), "r"(rank));
  return d;
}
__device__ __forceinline__ unsigned ld_cluster(uint32_t a) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Writes prob and count of one expert and returns its term of the loss.
__device__ __forceinline__ double finish_expert(const RouteFinish& f, unsigned e, double p, unsigned c, unsigned n) {
  p /= n ? n : 1u;
  f.prob[e] = static_cast<float>(p);
  f.count[e] = c;
  return p * c;
}
// The loss from the terms of the first `own` threads (a CTA's experts) of
// each CTA: a warp's sum goes straight to the first CTA of the cluster, which
// adds them in order.  The barrier is the last access to another CTA's memory.
constexpr unsigned kOwnWarps = kMaxExperts / kRouteCluster / 32;
__device__ __forceinline__ void finish_loss(const RouteFinish& f, double term, unsigned n, double (&s_term)[kRouteCluster * kOwnWarps]) {
  const unsigned warp = threadIdx.x / 32;
  if (warp < kOwnWarps) {
#pragma unroll
    for (unsigned o = 16; o; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
    if ((threadIdx.x & 31) == 0)
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(cluster_map(&s_term[cluster_rank() * kOwnWarps + warp], 0)), "d"(term) : "memory");
  }
  cluster_sync();
  if (cluster_rank() == 0 && threadIdx.x == 0) {
    double l = 0.0;
#pragma unroll
    for (unsigned r = 0; r < kRouteCluster * kOwnWarps; ++r) l += s_term[r];
    const double m = n ? n : 1u;
    *f.loss = static_cast<float>(l * f.experts / (kTopK * m));
    f.count[f.experts] = n;
  }
}

// Statistics: none, as parts for route_finish_kernel, or finished by the one
// cluster that runs (few rows).
enum : int { kStatsNone = 0, kStatsParts = 1, kStatsCluster = 2 };
// Warps of a CTA, and whether its rows come through shared memory: many
// aligned rows, two buffers a warp.  Without the next row in registers there is
// room for 32 warps, or 28 where experts are chosen and sums kept (65,536 rows
// of 512, all of it, when this was chosen: 44.7 us; with 24 warps 46.5, with
// 32, which spill, 45.7).
template <unsigned V, bool SELECT, int STATS, bool MANY>
struct RouteShape {
  static constexpr bool kStaged = MANY && V > 1;
  static constexpr unsigned kWarps = !kStaged ? kRouteWarps : SELECT && STATS ? 28 : 32;
};

// One warp a row; SELECT: choose experts and gates; STATS: sums of p and
// counts of the chosen (or given) experts over the CTA's rows.  The next
// row's logits are on their way while one is worked on.  Neighbouring rows go
// to different CTAs: runs of padding rows leave none idle (a ragged batch of
// 16,384 rows 17.1 us, with neighbours in one CTA 18.1).
template <typename L, unsigned V, bool FULL, bool SELECT, int STATS, bool MANY>
__global__ void __launch_bounds__(32 * RouteShape<V, SELECT, STATS, MANY>::kWarps, 1) route_kernel(const RouteParams a, const RouteFinish f) {
  using Shape = RouteShape<V, SELECT, STATS, MANY>;
  extern __shared__ __align__(16) uint8_t s_rows[];  // [warps][2][kMaxExperts] of L where rows are staged
  constexpr unsigned kSums = Shape::kStaged ? Shape::kWarps : kRouteSums;
  constexpr bool kOwnSums = STATS && !Shape::kStaged;  // else they lie where the rows passed through
  __shared__ __align__(16) float s_sums[kOwnSums ? kSums : 1][kOwnSums ? kMaxExperts : 1];
  float(*const s_psum)[kMaxExperts] = reinterpret_cast<float(*)[kMaxExperts]>(Shape::kStaged ? reinterpret_cast<float*>(s_rows) : &s_sums[0][0]);
  __shared__ unsigned s_count[STATS ? kMaxExperts : 1], s_valid;
  __shared__ __align__(16) RouteCand s_cand[SELECT ? Shape::kWarps : 1];
  __shared__ double s_term[kRouteCluster * kOwnWarps];
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = blockDim.x / 32, E = a.experts;
  const L* logits = static_cast<const L*>(a.logits);
  F2 psum[STATS ? kRouteSlots / 2 : 1];
  unsigned nvalid = 0;
  if (STATS) {
#pragma unroll
    for (unsigned i = 0; i < kRouteSlots / 2; ++i) psum[i] = pack2(0.0f, 0.0f);
    for (unsigned e = threadIdx.x; e < E; e += blockDim.x) s_count[e] = 0;
    if (threadIdx.x == 0) s_valid = 0;
    __syncthreads();
  }
  const unsigned step = gridDim.x * warps;
  unsigned t = warp * gridDim.x + blockIdx.x;
  RowLoad<L, V, FULL> next;
  bool next_valid = false;
  unsigned next_id = 0;
  L* stage = reinterpret_cast<L*>(s_rows) + 2 * kMaxExperts * warp;
  unsigned side = 0;  // the buffer that takes the next row
  const auto fetch = [&](unsigned r) {
    next_valid = !a.valid || a.valid[r];
    if (STATS && !SELECT && lane < kTopK) next_id = a.expert_in[r * kTopK + lane];
    if constexpr (Shape::kStaged) {
      stage_row<L, V, FULL>(stage + side, logits + r * a.stride, E, lane);
      side ^= kMaxExperts;
    } else {
      next.load(logits + r * a.stride, E, lane);
    }
  };
  if (t < a.tokens) fetch(t);
  for (; t < a.tokens; t += step) {
    const L* row = logits + t * a.stride;  // where single logits are read again
    const bool valid = next_valid;
    float v[kRouteSlots];
    if constexpr (Shape::kStaged) {
      row = stage + (side ^ kMaxExperts);
      cp_async_wait_all();
      __syncwarp();
      next.load(row, kMaxExperts, lane);
    }
#pragma unroll
    for (unsigned i = 0; i < kRouteSlots; ++i) v[i] = next.value(i);
    unsigned id = lane;
    float val = -INFINITY;
    if (STATS && !SELECT && lane < kTopK) {
      id = next_id;
      if (id < E && valid) val = logit(row + id);
    }
    if (t + step < a.tokens) fetch(t + step);
    const float top = row_max(v), m = warp_max_nan(top);
    const bool bad = valid && !(m < INFINITY);
    if (bad && lane == 0) atomicOr(a.status, kStNumeric);
    const bool use = valid && !bad;
    if (SELECT) {
      float g = 0.0f;
      if (use) {
        choose<L, V>(v, row, E, lane, top, m, &s_cand[warp], &id, &val);
        const float e = lane < kTopK && m > -INFINITY ? expf(val - m) : 0.0f;
        const float sum = chosen_sum(e);
        g = sum > 0.0f ? e * rcp(sum) : 0.0f;
        if (lane == kTopK && a.shared) {
          const float s = logit(logits + t * a.stride + E);
          g = sigmoid(s);
          if (s != s) {
            g = 0.0f;
            atomicOr(a.status, kStNumeric);
          }
        }
      }
      // 32 bits hold the places of 2^24 rows
      if (lane < kTopK) a.expert[t * kTopK + lane] = static_cast<uint16_t>(id);
      if (lane < kGates) a.gate[t * kGates + lane] = g;
    }
    if (STATS && use) {
      if (lane < kTopK) {
        if (!SELECT && id >= E) atomicOr(a.status, kStInvalid);
        if (val > -INFINITY) atomicAdd(&s_count[id], 1u);
      }
      ++nvalid;
      if (m > -INFINITY) {
        F2 e[kRouteSlots / 2];
        const float zi = rcp(warp_sum(exp_row(v, m, e)));
        const F2 z2 = pack2(zi, zi);
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots / 2; ++i) psum[i] = fma2(e[i], z2, psum[i]);
      }
    }
  }
  if (STATS) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (lane == 0) atomicAdd(&s_valid, nvalid);
    if (Shape::kStaged) __syncthreads();
    for (unsigned w = 0; w < warps; w += kSums) {  // in a fixed order
      if (warp >= w && warp < w + kSums)
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots / 2; i += 2) {
          float x[4];
          unpack2(psum[i], x[0], x[1]);
          unpack2(psum[i + 1], x[2], x[3]);
          float* p = &s_psum[warp - w][col<V>(2 * i, lane)];
          if constexpr (V > 1) {
            float4 q = w ? *reinterpret_cast<const float4*>(p) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            q.x += x[0]; q.y += x[1]; q.z += x[2]; q.w += x[3];
            *reinterpret_cast<float4*>(p) = q;
          } else {
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) p[32 * k] = (w ? p[32 * k] : 0.0f) + x[k];
          }
        }
      __syncthreads();
    }
    const unsigned sums = warps < kSums ? warps : kSums;
    if (STATS == kStatsParts) {
      for (unsigned e = threadIdx.x; e < E; e += blockDim.x) {
        float s = 0.0f;
#pragma unroll 8
        for (unsigned w = 0; w < sums; ++w) s += s_psum[w][e];
        a.part[static_cast<size_t>(blockIdx.x) * E + e] = make_float2(s, __uint_as_float(s_count[e]));
      }
      if (threadIdx.x == 0) a.pvalid[blockIdx.x] = s_valid;
    } else {
      for (unsigned e = threadIdx.x; e < E; e += blockDim.x) {
        float s = 0.0f;
        for (unsigned w = 0; w < sums; ++w) s += s_psum[w][e];
        s_psum[0][e] = s;
      }
      cluster_sync();
      const unsigned own = (E + kRouteCluster - 1) / kRouteCluster, e = cluster_rank() * own + threadIdx.x;
      double term = 0.0;
      unsigned n = 0;
      if (threadIdx.x < 32 * kOwnWarps) {
        unsigned v[kRouteCluster], c[kRouteCluster], p[kRouteCluster];
        const bool mine = threadIdx.x < own && e < E;
#pragma unroll
        for (unsigned r = 0; r < kRouteCluster; ++r) {
          v[r] = ld_cluster(cluster_map(&s_valid, r));
          p[r] = mine ? ld_cluster(cluster_map(&s_psum[0][e], r)) : 0u;
          c[r] = mine ? ld_cluster(cluster_map(&s_count[e], r)) : 0u;
        }
        double sum = 0.0;
        unsigned count = 0;
#pragma unroll
        for (unsigned r = 0; r < kRouteCluster; ++r) {
          n += v[r];
          count += c[r];
          sum += __uint_as_float(p[r]);
        }
        if (mine) term = finish_expert(f, e, sum, count, n);
      }
      finish_loss(f, term, n, s_term);
    }
  }
}

// Sums the CTAs' parts in order, in double, and forms the loss: one cluster,
// 16 threads an expert that take every 16th part, all of them in flight.
static_assert(kRouteCtas % 32 == 0, "whole warps of parts");
constexpr unsigned kFinishSplit = 16, kFinishThreads = kMaxExperts / kRouteCluster * kFinishSplit;
__global__ void __cluster_dims__(kRouteCluster, 1, 1) __launch_bounds__(kFinishThreads)
    route_finish_kernel(const RouteFinish f) {
  __shared__ double s_p[kFinishSplit][kMaxExperts / kRouteCluster], s_term[kRouteCluster * kOwnWarps];
  __shared__ unsigned s_c[kFinishSplit][kMaxExperts / kRouteCluster];
  const unsigned own = kMaxExperts / kRouteCluster, i = threadIdx.x % own, k0 = threadIdx.x / own;
  const unsigned e = cluster_rank() * own + i;
  // the first CTA gets the terms of the others in its shared memory: it must have started by then
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double p = 0.0;
  unsigned c = 0, valid[kRouteCtas / 32], n = 0;
#pragma unroll
  for (unsigned j = 0; j < kRouteCtas / 32; ++j) {
    const unsigned k = 32 * j + (threadIdx.x & 31);
    valid[j] = k < f.parts ? f.pvalid[k] : 0u;
  }
  if (e < f.experts) {
    float2 v[kRouteCtas / kFinishSplit];
#pragma unroll
    for (unsigned j = 0; j < kRouteCtas / kFinishSplit; ++j) {
      const unsigned k = k0 + kFinishSplit * j;
      v[j] = k < f.parts ? f.part[static_cast<size_t>(k) * f.experts + e] : make_float2(0.0f, 0.0f);
    }
#pragma unroll
    for (unsigned j = 0; j < kRouteCtas / kFinishSplit; ++j) {
      p += v[j].x;
      c += __float_as_uint(v[j].y);
    }
  }
#pragma unroll
  for (unsigned j = 0; j < kRouteCtas / 32; ++j) n += valid[j];
  n = __reduce_add_sync(0xffffffffu, n);
  s_p[k0][i] = p;
  s_c[k0][i] = c;
  __syncthreads();
  double term = 0.0;
  if (k0 == 0 && e < f.experts) {
    for (unsigned k = 1; k < kFinishSplit; ++k) {
      p += s_p[k][i];
      c += s_c[k][i];
    }
    term = finish_expert(f, e, p, c, n);
  }
  __syncwarp();  // the barriers are a whole warp's
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  finish_loss(f, term, n, s_term);
}

__device__ __forceinline__ void store_grad(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_grad(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
template <typename L, unsigned V, bool FULL>
__device__ __forceinline__ void store_row(L* row, unsigned E, unsigned lane, const float (&d)[kRouteSlots]) {
  if constexpr (V == 1) {
#pragma unroll
    for (unsigned i = 0; i < kRouteSlots; ++i)
      if (FULL || 32 * i + 32 <= E || lane + 32 * i < E) store_grad(row + lane + 32 * i, d[i]);
  } else {
#pragma unroll
    for (unsigned j = 0; j < kRouteSlots / V; ++j) {
      const unsigned c = col<V>(j * V, lane);
      if (FULL || c + V <= E) {
        if constexpr (sizeof(L) == 4) {
          *reinterpret_cast<float4*>(row + c) = make_float4(d[4 * j], d[4 * j + 1], d[4 * j + 2], d[4 * j + 3]);
        } else {
          uint32_t w[4];
#pragma unroll
          for (unsigned k = 0; k < 4; ++k) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(d[8 * j + 2 * k], d[8 * j + 2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t*>(&h);
          }
          *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
#pragma unroll
        for (unsigned k = 0; k < V; ++k)
          if (c + k < E) store_grad(row + c + k, d[j * V + k]);
      }
    }
  }
}

// One warp a row: the balance term of every logit is stored first, then lanes
// 0-9 store the chosen ones' sum with the routing term.  BALANCE off: only
// the chosen logits are read.  Ids are fetched two rows ahead and the chosen
// logits one, like the row itself.
template <typename L, unsigned V, bool FULL, bool BALANCE>
__global__ void __launch_bounds__(256, BALANCE ? 3 : 6) route_backward_kernel(const RouteBackwardParams a) {
  // k = scale count (the balance term is p_e (k_e - sum p k)): by column, and as the lanes' slots
  __shared__ float s_k[BALANCE ? kMaxExperts : 1];
  __shared__ __align__(16) float s_slots[BALANCE ? kRouteSlots / 4 : 1][32][4];
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = blockDim.x / 32, E = a.experts;
  const L* logits = static_cast<const L*>(a.logits);
  const unsigned step = gridDim.x * warps;
  unsigned t = blockIdx.x * warps + warp;
  RowLoad<L, V, FULL> next;
  unsigned id = E + 1, id1 = E + 1;
  float dg = 0.0f, dg1 = 0.0f, val1 = -INFINITY;
  bool valid1 = false, valid2 = false;
  // the chosen experts in lanes 0-9, the shared logit in lane 10
  const auto ids = [&](unsigned r) {
    valid2 = !a.valid || a.valid[r];
    if (a.d_gate) {
      if (lane < kTopK) id1 = a.expert[r * kTopK + lane];
      if (lane < kGates) dg1 = a.d_gate[r * kGates + lane];
    }
  };
  const auto chosen_logit = [&](unsigned r, unsigned e) {
    const L* row = logits + r * a.stride;
    if (a.d_gate && lane < kTopK && e < E) return logit(row + e);
    if (a.d_gate && lane == kTopK && a.shared) return logit(row + E);
    return -INFINITY;
  };
  if (t < a.tokens) {
    ids(t);
    if (BALANCE) next.load(logits + t * a.stride, E, lane);
  }
  if (BALANCE) {
    unsigned count[4];  // all of a thread's loads at once
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const unsigned e = threadIdx.x + j * blockDim.x;
      count[j] = e < E ? a.count[e] : 0u;
    }
    const float n = static_cast<float>(a.count[E]), d_loss = *a.d_loss;
    const float scale = n > 0.0f ? d_loss * static_cast<float>(E) / (static_cast<float>(kTopK) * n * n) : 0.0f;
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const unsigned e = threadIdx.x + j * blockDim.x;
      if (e < kMaxExperts) {
        const unsigned i = e / (32 * V) * V + e % V;  // the column's slot
        s_k[e] = s_slots[i / 4][e / V % 32][i % 4] = scale * static_cast<float>(count[j]);
      }
    }
    __syncthreads();
  }
  if (t < a.tokens) {
    id = id1;
    dg = dg1;
    valid1 = valid2;
    val1 = chosen_logit(t, id);
    if (t + step < a.tokens) ids(t + step);
  }
  for (; t < a.tokens; t += step) {
    L* out = static_cast<L*>(a.d_logits) + t * a.d_stride;
    const bool valid = valid1;
    const float val = val1, cdg = dg;
    const unsigned cid = id;
    float d[kRouteSlots];
#pragma unroll
    for (unsigned i = 0; i < kRouteSlots; ++i) d[i] = BALANCE ? next.value(i) : 0.0f;
    if (t + step < a.tokens) {
      id = id1;
      dg = dg1;
      valid1 = valid2;
      val1 = chosen_logit(t + step, id);
      if (step < a.tokens - t - step) ids(t + 2 * step);
      if (BALANCE) next.load(logits + (t + step) * a.stride, E, lane);
    }
    float m = -INFINITY, zi = 0.0f, dot = 0.0f;
    if (BALANCE) {
      m = warp_max_nan(row_max(d));
      if (valid && !(m < INFINITY) && lane == 0) atomicOr(a.status, kStNumeric);
      if (valid && m > -INFINITY) {
        F2 e[kRouteSlots / 2], s2 = pack2(0.0f, 0.0f);
        const float z = exp_row(d, m, e);
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots / 4; ++i) {
          const float4 k = *reinterpret_cast<const float4*>(s_slots[i][lane]);
          s2 = fma2(e[2 * i], pack2(k.x, k.y), s2);
          s2 = fma2(e[2 * i + 1], pack2(k.z, k.w), s2);
        }
        unpack2(s2, dot, zi);
        dot += zi;
        zi = rcp(warp_sum(z));
        dot = warp_sum(dot) * zi;
        // (e / z) (k - dot) = e (k / z - dot / z)
        const F2 z2 = pack2(zi, zi), c2 = pack2(-dot * zi, -dot * zi);
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots / 4; ++i) {
          const float4 k = *reinterpret_cast<const float4*>(s_slots[i][lane]);
          unpack2(mul2(e[2 * i], fma2(pack2(k.x, k.y), z2, c2)), d[4 * i], d[4 * i + 1]);
          unpack2(mul2(e[2 * i + 1], fma2(pack2(k.z, k.w), z2, c2)), d[4 * i + 2], d[4 * i + 3]);
        }
      } else {
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots; ++i) d[i] = 0.0f;
      }
    }
    __syncwarp();  // d_logits may be logits: every lane has read the row
    store_row<L, V, FULL>(out, E, lane, d);
    if (a.d_gate) {
      if (lane < kTopK && valid) {
        if (cid >= E) atomicOr(a.status, kStInvalid);
        if (!(val < INFINITY)) atomicOr(a.status, kStNumeric);
      }
      const float chosen = lane < kTopK && valid ? val : -INFINITY, mk = warp_max(chosen);
      float g = mk > -INFINITY ? exp2f((chosen - mk) * 1.4426950408889634f) : 0.0f;  // subnormal gates count
      // gates that are 0 by a mask (or an id that is none) are constants: their gradient, which may be anything,
      // does not count.  In lane 10 it is the shared gate's.
      // Taken as sixteenths: the ten products with gates that are not divided by their sum yet stay in range.
      const float d16 = chosen > -INFINITY ? cdg * 0.0625f : 0.0f;
      const float s = warp_sum(g), gd16 = warp_sum(g * d16), si = s > 0.0f ? rcp(s) : 0.0f;
      const float own = g * si * (d16 - gd16 * si) * 16.0f;
      float term = own;
      const unsigned same = __match_any_sync(0xffffffffu, cid) & 0x3ffu;
      const bool twice = lane < kTopK && same != 1u << lane;
      if (__any_sync(0xffffffffu, twice)) {  // the same index twice adds twice
        if (twice) term = 0.0f;
        for (unsigned r = 0; r < kTopK; ++r) {
          const float o = __shfl_sync(0xffffffffu, own, r);
          if (twice && (same >> r & 1u)) term += o;
        }
      }
      if (BALANCE && lane < kTopK && zi > 0.0f && cid < E) term += exp_below(val, m) * fmaf(s_k[cid], zi, -dot * zi);
      __syncwarp();  // behind the row's stores
      if (valid && lane < kTopK && cid < E) store_grad(out + cid, term);
    }
    if (a.shared && lane == kTopK) {
      // an infinite logit's gate is constant, and a NaN one's, which is reported; padding may hold any d_gate
      const bool moves = a.d_gate && valid && fabsf(val) < INFINITY;
      if (a.d_gate && valid && val != val) atomicOr(a.status, kStNumeric);
      // s (1 - s) as e / (1 + e)^2 with e = exp(-|val|): 1 - s would lose what s has rounded away, all of it from 17 on
      const float e = expf(-fabsf(val)), r = 1.0f / (1.0f + e);
      store_grad(out + E, moves ? e * r * r * cdg : 0.0f);
    }
  }
}

// ------------------------------------------------------------ host side

// Whether one cluster makes the statistics in one launch.  Measured at 512
// experts fp32, one cluster against CTAs of eight rows and the launch that
// joins them: statistics of 250 rows 5.0 and 5.1 us, of 512 rows 6.3 and 5.3,
// of 700 rows 7.7 and 5.8; with the selection 100 rows 5.8 and 5.9, 160 rows
// 7.3 and 6.1, 250 rows 7.9 and 6.2.  The second launch costs the host 1.2 us,
// which is what a call that is not replayed from a graph waits for: the rule
// takes the cluster until the device time outweighs that.
inline bool route_one_cluster(unsigned tokens, bool select) { return tokens <= (select ? 160 : 512); }

// CTAs that make statistics of `tokens` rows: one part of the sums each.
inline unsigned route_parts(unsigned tokens, unsigned sms) {
  const unsigned n = (tokens + kRouteRows - 1) / kRouteRows;
  return n < sms ? n : sms;
}
inline bool rows_aligned(const void* p, size_t stride, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}

// route_finish_kernel may start while route_kernel ends (it waits for it).
inline cudaError_t launch_finish(const RouteFinish& f, cudaStream_t s) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kRouteCluster);
  cfg.blockDim = dim3(kFinishThreads);
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, route_finish_kernel, f);
}

// route_kernel for many rows.
template <typename L, unsigned V, bool FULL, bool SELECT, int STATS>
inline cudaError_t launch_many(const RouteParams& a, const RouteFinish& f, unsigned ctas, int device, cudaStream_t s) {
  using Shape = RouteShape<V, SELECT, STATS, true>;
  constexpr unsigned smem = Shape::kStaged ? Shape::kWarps * 2 * kMaxExperts * sizeof(L) : 0;
  static_assert(!smem || Shape::kWarps * kMaxExperts * sizeof(float) <= smem, "the warps' sums");
  const unsigned rows = (a.tokens + ctas - 1) / ctas, warps = rows < Shape::kWarps ? rows : Shape::kWarps;
  static std::atomic<unsigned long long> allowed{0};  // devices on which the kernel may take its shared memory
  const unsigned long long bit = 1ull << (device & 63);
  if (smem && (device > 63 || !(allowed.load(std::memory_order_relaxed) & bit))) {
    const cudaError_t e = cudaFuncSetAttribute(route_kernel<L, V, FULL, SELECT, STATS, true>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  route_kernel<L, V, FULL, SELECT, STATS, true><<<ctas, 32 * warps, smem / Shape::kWarps * warps, s>>>(a, f);
  return cudaGetLastError();
}

template <typename L, unsigned V, bool FULL, bool SELECT>
inline cudaError_t launch_stats(const RouteParams& a, const RouteFinish& f, int device, cudaStream_t s) {
  if (route_one_cluster(a.tokens, SELECT)) {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = kRouteCluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kRouteCluster);
    cfg.blockDim = dim3(32 * kRouteSums);
    cfg.stream = s;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, route_kernel<L, V, FULL, SELECT, kStatsCluster, false>, a, f);
  }
  const cudaError_t e = launch_many<L, V, FULL, SELECT, kStatsParts>(a, f, f.parts, device, s);
  return e == cudaSuccess ? launch_finish(f, s) : e;
}

template <typename L, unsigned V, bool FULL>
inline cudaError_t launch_route(const RouteParams& a, const RouteFinish& f, bool select, bool stats, unsigned sms,
                                int device, cudaStream_t s) {
  if (stats) return select ? launch_stats<L, V, FULL, true>(a, f, device, s) : launch_stats<L, V, FULL, false>(a, f, device, s);
  // few rows: four warps a CTA spread them over the SMs
  if (a.tokens <= 8 * sms) {
    route_kernel<L, V, FULL, true, kStatsNone, false><<<(a.tokens + 3) / 4, 128, 0, s>>>(a, f);
    return cudaGetLastError();
  }
  return launch_many<L, V, FULL, true, kStatsNone>(a, f, sms, device, s);
}
inline cudaError_t launch_route(const RouteParams& a, const RouteFinish& f, unsigned type, bool select, bool stats,
                                unsigned sms, int device, cudaStream_t s) {
  const size_t size = type == FRC_BF16 ? 2 : 4;
  // neighbours a lane only where they leave no lane without logits: the
  // bound on the tenth largest needs the lanes' maxima
  const bool vec = rows_aligned(a.logits, a.stride, size) && a.experts * size >= 512;
  const bool full = a.experts == kMaxExperts;
  if (type == FRC_BF16) {
    if (vec) return full ? launch_route<__nv_bfloat16, 8, true>(a, f, select, stats, sms, device, s) : launch_route<__nv_bfloat16, 8, false>(a, f, select, stats, sms, device, s);
    return full ? launch_route<__nv_bfloat16, 1, true>(a, f, select, stats, sms, device, s) : launch_route<__nv_bfloat16, 1, false>(a, f, select, stats, sms, device, s);
  }
  if (vec) return full ? launch_route<float, 4, true>(a, f, select, stats, sms, device, s) : launch_route<float, 4, false>(a, f, select, stats, sms, device, s);
  return full ? launch_route<float, 1, true>(a, f, select, stats, sms, device, s) : launch_route<float, 1, false>(a, f, select, stats, sms, device, s);
}

template <typename L, unsigned V, bool FULL>
inline cudaError_t launch_backward(const RouteBackwardParams& a, unsigned sms, cudaStream_t s) {
  const unsigned warps = a.tokens <= 8 * sms ? 4 : 8, ctas = (a.tokens + warps - 1) / warps, limit = (a.count ? 3 : 6) * sms, grid = ctas < limit ? ctas : limit;
  if (a.count) route_backward_kernel<L, V, FULL, true><<<grid, 32 * warps, 0, s>>>(a);
  else route_backward_kernel<L, V, FULL, false><<<grid, 32 * warps, 0, s>>>(a);
  return cudaGetLastError();
}
inline cudaError_t launch_backward(const RouteBackwardParams& a, unsigned type, unsigned sms, cudaStream_t s) {
  const size_t size = type == FRC_BF16 ? 2 : 4;
  const bool vec = rows_aligned(a.logits, a.stride, size) && rows_aligned(a.d_logits, a.d_stride, size);
  const bool full = a.experts == kMaxExperts;
  if (type == FRC_BF16) {
    if (vec) return full ? launch_backward<__nv_bfloat16, 8, true>(a, sms, s) : launch_backward<__nv_bfloat16, 8, false>(a, sms, s);
    return full ? launch_backward<__nv_bfloat16, 1, true>(a, sms, s) : launch_backward<__nv_bfloat16, 1, false>(a, sms, s);
  }
  if (vec) return full ? launch_backward<float, 4, true>(a, sms, s) : launch_backward<float, 4, false>(a, sms, s);
  return full ? launch_backward<float, 1, true>(a, sms, s) : launch_backward<float, 1, false>(a, sms, s);
}

}  // namespace frc
