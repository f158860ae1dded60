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
#pragma once
#include <cuda_bf16.h>

#include "frc_device.cuh"

namespace frc {

constexpr unsigned kTopK = 10, kGates = 11, kMaxExperts = 512;
constexpr unsigned kRouteSlots = kMaxExperts / 32;  // logits a lane holds
constexpr unsigned kRouteWarps = 4;                 // warps a CTA
constexpr unsigned kRouteCtas = 296;                // CTAs that make statistics, at most

struct RouteParams {
  const void* logits;
  size_t stride;         // elements between rows
  const uint8_t* valid;  // null: every row
  const uint16_t* expert_in;
  uint16_t* expert;
  float* gate;
  unsigned tokens, experts, shared;
  // statistics: [CTA][E] sums of p, [CTA][E] counts, [CTA] valid rows
  float* psum;
  unsigned* pcount;
  unsigned* pvalid;
  unsigned* status;
};

struct RouteFinish {
  const float* psum;
  const unsigned* pcount;
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
__device__ __forceinline__ void store_grad(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_grad(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

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
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (unsigned o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }
// exp(v - m) with v <= m, both finite or v = -inf.
__device__ __forceinline__ float exp_below(float v, float m) { return exp2f((v - m) * 1.4426950408889634f); }

// One warp a row; SELECT: choose experts and gates, STATS: sum p and counts
// of the chosen (or given) experts over the CTA's rows.
template <typename L, bool SELECT, bool STATS>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const RouteParams a) {
  __shared__ float s_psum[STATS ? kRouteWarps : 1][STATS ? kMaxExperts : 1];
  __shared__ unsigned s_count[STATS ? kMaxExperts : 1], s_valid;
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x & 31, E = a.experts;
  float psum[STATS ? kRouteSlots : 1] = {};
  unsigned nvalid = 0;
  if (STATS) {
    for (unsigned e = threadIdx.x; e < E; e += blockDim.x) s_count[e] = 0;
    if (threadIdx.x == 0) s_valid = 0;
    __syncthreads();
  }
  for (unsigned t = blockIdx.x * kRouteWarps + warp; t < a.tokens; t += gridDim.x * kRouteWarps) {
    const L* row = static_cast<const L*>(a.logits) + t * a.stride;
    const bool valid = !a.valid || a.valid[t];
    float v[kRouteSlots];
    bool bad = false;
#pragma unroll
    for (unsigned i = 0; i < kRouteSlots; ++i) {
      const unsigned e = lane + 32 * i;
      v[i] = e < E && valid ? logit(row + e) + 0.0f : -INFINITY;  // -0 becomes +0: equal logits are ties
      bad |= !(v[i] < INFINITY);
    }
    bad = __any_sync(0xffffffffu, bad);
    if (bad && lane == 0) atomicOr(a.status, kStNumeric);
    const bool use = valid && !bad;
    unsigned id = lane;
    float val = -INFINITY;
    if (SELECT) {
      if (use) {
        unsigned left = 0;
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots; ++i) left |= (lane + 32 * i < E ? 1u : 0u) << i;
        for (unsigned r = 0; r < kTopK; ++r) {
          unsigned best = 0, slot = 0;
#pragma unroll
          for (unsigned i = 0; i < kRouteSlots; ++i) {
            const unsigned k = left >> i & 1u ? order_key(v[i]) : 0u;
            if (k > best) { best = k; slot = i; }
          }
          const unsigned top = __reduce_max_sync(0xffffffffu, best);
          const unsigned win = __reduce_min_sync(0xffffffffu, best == top ? lane + 32 * slot : 0xffffffffu);
          if ((win & 31) == lane) left &= ~(1u << (win >> 5));
          if (lane == r) { id = win; val = key_value(top); }
        }
      }
      const float m = __shfl_sync(0xffffffffu, val, 0);
      const float e = lane < kTopK && m > -INFINITY ? expf(val - m) : 0.0f;
      const float sum = warp_sum(e);
      float g = sum > 0.0f ? e / sum : 0.0f;
      if (lane == kTopK && a.shared && use) {
        const float s = logit(row + E);
        g = sigmoid(s);
        if (s != s) {
          g = 0.0f;
          atomicOr(a.status, kStNumeric);
        }
      }
      if (lane < kTopK) a.expert[static_cast<size_t>(t) * kTopK + lane] = static_cast<uint16_t>(id);
      if (lane < kGates) a.gate[static_cast<size_t>(t) * kGates + lane] = g;
    }
    if (STATS && use) {
      if (lane < kTopK) {
        if (!SELECT) {
          id = a.expert_in[static_cast<size_t>(t) * kTopK + lane];
          if (id < E) val = logit(row + id);
          else atomicOr(a.status, kStInvalid);
        }
        if (val > -INFINITY) atomicAdd(&s_count[id], 1u);
      }
      float m = -INFINITY;
#pragma unroll
      for (unsigned i = 0; i < kRouteSlots; ++i) m = fmaxf(m, v[i]);
      m = warp_max(m);
      ++nvalid;
      if (m > -INFINITY) {
        float z = 0.0f;
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots; ++i) {
          v[i] = exp_below(v[i], m);
          z += v[i];
        }
        z = 1.0f / warp_sum(z);
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots; ++i) psum[i] = fmaf(v[i], z, psum[i]);
      }
    }
  }
  if (STATS) {
#pragma unroll
    for (unsigned i = 0; i < kRouteSlots; ++i) s_psum[warp][lane + 32 * i] = psum[i];
    if (lane == 0) atomicAdd(&s_valid, nvalid);
    __syncthreads();
    for (unsigned e = threadIdx.x; e < E; e += blockDim.x) {
      float s = 0.0f;
#pragma unroll
      for (unsigned w = 0; w < kRouteWarps; ++w) s += s_psum[w][e];
      a.psum[static_cast<size_t>(blockIdx.x) * E + e] = s;
      a.pcount[static_cast<size_t>(blockIdx.x) * E + e] = s_count[e];
    }
    if (threadIdx.x == 0) a.pvalid[blockIdx.x] = s_valid;
  }
}

// Sums the CTAs' parts in order (one thread an expert, in double) and forms
// the loss.
__global__ void __launch_bounds__(kMaxExperts) route_finish_kernel(const RouteFinish a) {
  __shared__ double s_part[kMaxExperts / 32];
  __shared__ unsigned s_n;
  const unsigned e = threadIdx.x, lane = e & 31;
  if (e < 32) {
    unsigned n = 0;
    for (unsigned k = lane; k < a.parts; k += 32) n += a.pvalid[k];
    n = __reduce_add_sync(0xffffffffu, n);
    if (e == 0) s_n = n;
  }
  double p = 0.0;
  unsigned c = 0;
  if (e < a.experts)
    for (unsigned k = 0; k < a.parts; ++k) {
      p += a.psum[static_cast<size_t>(k) * a.experts + e];
      c += a.pcount[static_cast<size_t>(k) * a.experts + e];
    }
  __syncthreads();
  const double n = s_n ? s_n : 1u;
  p /= n;
  if (e < a.experts) {
    a.prob[e] = static_cast<float>(p);
    a.count[e] = c;
  }
  if (e == 0) a.count[a.experts] = s_n;
  double l = p * c;
#pragma unroll
  for (unsigned o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (lane == 0) s_part[e / 32] = l;
  __syncthreads();
  if (e == 0) {
    l = 0.0;
    for (unsigned w = 0; w < kMaxExperts / 32; ++w) l += s_part[w];
    *a.loss = static_cast<float>(l * a.experts / (kTopK * n));
  }
}

// One warp a row: d_logits = routing term + balance term.
template <typename L>
__global__ void __launch_bounds__(32 * kRouteWarps) route_backward_kernel(const RouteBackwardParams a) {
  const unsigned warp = threadIdx.x / 32, lane = threadIdx.x & 31, E = a.experts;
  const float n = a.count ? static_cast<float>(a.count[E]) : 0.0f;
  const float scale = n > 0.0f ? *a.d_loss * static_cast<float>(E) / (static_cast<float>(kTopK) * n * n) : 0.0f;
  for (unsigned t = blockIdx.x * kRouteWarps + warp; t < a.tokens; t += gridDim.x * kRouteWarps) {
    const L* row = static_cast<const L*>(a.logits) + t * a.stride;
    L* out = static_cast<L*>(a.d_logits) + t * a.d_stride;
    const bool valid = !a.valid || a.valid[t];
    float d[kRouteSlots] = {};
    float m = -INFINITY, zi = 0.0f, dot = 0.0f;
    if (valid && a.count) {
      bool bad = false;
#pragma unroll
      for (unsigned i = 0; i < kRouteSlots; ++i) {
        const unsigned e = lane + 32 * i;
        d[i] = e < E ? logit(row + e) : -INFINITY;
        bad |= !(d[i] < INFINITY);
        m = fmaxf(m, d[i]);
      }
      if (bad) atomicOr(a.status, kStNumeric);
      m = warp_max(m);
      float z = 0.0f;
#pragma unroll
      for (unsigned i = 0; i < kRouteSlots; ++i) {
        const unsigned e = lane + 32 * i;
        d[i] = m > -INFINITY ? exp_below(d[i], m) : 0.0f;
        z += d[i];
        if (e < E) dot = fmaf(d[i], static_cast<float>(a.count[e]), dot);
      }
      z = warp_sum(z);
      zi = z > 0.0f ? 1.0f / z : 0.0f;
      dot = warp_sum(dot) * zi;
#pragma unroll
      for (unsigned i = 0; i < kRouteSlots; ++i) {
        const unsigned e = lane + 32 * i;
        if (e < E) d[i] = scale * (d[i] * zi) * (static_cast<float>(a.count[e]) - dot);
      }
    }
    float d_shared = 0.0f;
    if (valid && a.d_gate) {
      unsigned id = 0;
      float val = -INFINITY, dg = 0.0f;
      if (lane < kTopK) {
        id = a.expert[static_cast<size_t>(t) * kTopK + lane];
        dg = a.d_gate[static_cast<size_t>(t) * kGates + lane];
        if (id < E) val = logit(row + id);
        else atomicOr(a.status, kStInvalid);
        if (!(val < INFINITY)) atomicOr(a.status, kStNumeric);
      }
      const float mk = warp_max(val);
      float g = lane < kTopK && mk > -INFINITY ? expf(val - mk) : 0.0f;
      const float s = warp_sum(g);
      g = s > 0.0f ? g / s : 0.0f;
      const float gd = warp_sum(g * dg);
      const float term = g * (dg - gd);
      for (unsigned r = 0; r < kTopK; ++r) {  // the same index twice adds twice
        const unsigned er = __shfl_sync(0xffffffffu, id, r);
        const float tr = __shfl_sync(0xffffffffu, term, r);
#pragma unroll
        for (unsigned i = 0; i < kRouteSlots; ++i) d[i] += lane + 32 * i == er && er < E ? tr : 0.0f;
      }
      if (a.shared) {
        const float sg = sigmoid(logit(row + E));
        d_shared = sg * (1.0f - sg) * a.d_gate[static_cast<size_t>(t) * kGates + kTopK];
      }
    }
    __syncwarp();  // d_logits may be logits: every lane has read the row
#pragma unroll
    for (unsigned i = 0; i < kRouteSlots; ++i) {
      const unsigned e = lane + 32 * i;
      if (e < E) store_grad(out + e, d[i]);
    }
    if (a.shared && lane == 0) store_grad(out + E, d_shared);
  }
}

// CTAs that make statistics of `tokens` rows: one part of the sums each.
inline unsigned route_parts(unsigned tokens) {
  const unsigned n = (tokens + kRouteWarps - 1) / kRouteWarps;
  return n < kRouteCtas ? n : kRouteCtas;
}

template <typename L>
inline void launch_route(const RouteParams& a, bool select, bool stats, cudaStream_t s) {
  const unsigned full = (a.tokens + kRouteWarps - 1) / kRouteWarps, threads = 32 * kRouteWarps;
  if (!stats) route_kernel<L, true, false><<<full, threads, 0, s>>>(a);
  else if (select) route_kernel<L, true, true><<<route_parts(a.tokens), threads, 0, s>>>(a);
  else route_kernel<L, false, true><<<route_parts(a.tokens), threads, 0, s>>>(a);
}

}  // namespace frc
