// Routing of tokens to experts and what surrounds the experts' products: the
// choice (route) and its gradient, the order of rows by expert (plan), the
// weighted sum of a token's rows (combine) and its gradient, and the gradient
// of an activation.  None of them multiplies matrices: they are bound by
// memory, or by launch latency for the few tokens of a decoding step.
//
// All kernels wait for the previous grid before they touch memory and let the
// next one start early (programmatic dependent launch).
#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/opengemm_b200.h"
#include "activation.cuh"
#include "dependent_launch.h"
#include "device_scope.h"
#include "ptx.cuh"

namespace og {
namespace {

constexpr unsigned ALL = 0xFFFFFFFFu;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Two 16-bit values of a 32-bit word, and back.
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return make_float2(half_bits_to_float(w), half_bits_to_float(w >> 16));
}
template <typename T> __device__ __forceinline__ uint32_t pack2_of(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2_of<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack2_of<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }

template <typename T>
__device__ __forceinline__ void load8(const T* at, float* v) {
  const uint4 q = *reinterpret_cast<const uint4*>(at);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* at, float* v) {
  const float4 a = reinterpret_cast<const float4*>(at)[0], b = reinterpret_cast<const float4*>(at)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* at, const float* v) {
  *reinterpret_cast<uint4*>(at) =
      make_uint4(pack2_of<T>(v[0], v[1]), pack2_of<T>(v[2], v[3]), pack2_of<T>(v[4], v[5]), pack2_of<T>(v[6], v[7]));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d /= 2) v += __shfl_xor_sync(ALL, v, d);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d; d /= 2) v = fmaxf(v, __shfl_xor_sync(ALL, v, d));
  return v;
}

// ------------------------------------------------------------------- route

// Order of scores as unsigned integers: 0 for what may not be chosen (a score
// of -infinity included), NaN above everything, -0 equal to 0.
__device__ __forceinline__ uint32_t score_key(float c, bool open) {
  if (!open || c == -INFINITY) return 0u;
  if (c != c) return 0xFFFFFFFFu;
  const uint32_t bits = __float_as_uint(c + 0.0f);
  return (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float key_score(uint32_t key) {
  if (key == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}

struct RouteParams {
  const void* logits;
  const float* bias;
  float* weights;
  int* indices;
  const float* grad_weights;
  void* grad_logits;
  long long tokens;
  int experts, top_k, sigmoid, groups, each, top_groups, group_top, renormalise;
  float scale;
};

// A row's scores: exp(l - top) / sum, or the logistic function.  `top` and
// `inverse` come from row_scale; a row without any finite logit scores 0.
struct RowScale {
  float top, inverse;
};
template <int VALUES>
__device__ __forceinline__ RowScale row_scale(const float (&l)[VALUES], bool sigmoid) {
  RowScale r{0.0f, 1.0f};
  if (sigmoid) return r;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < VALUES; ++j) top = fmaxf(top, l[j]);
  r.top = warp_max(top);
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < VALUES; ++j) sum += l[j] == -INFINITY ? 0.0f : expf(l[j] - r.top);
  sum = warp_sum(sum);
  r.inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
  return r;
}
__device__ __forceinline__ float score_of(float l, const RowScale& r, bool sigmoid) {
  if (l == -INFINITY) return 0.0f;
  return sigmoid ? 1.0f / (1.0f + expf(-l)) : expf(l - r.top) * r.inverse;
}

// s (1 - s) of the logistic function s = 1 / (1 + e): with e = exp(-|l|) it is e / (1 + e)^2, on either side.
__device__ __forceinline__ float logistic_slope(float l) {
  const float e = expf(-fabsf(l)), t = 1.0f + e;
  return e / (t * t);
}

constexpr int ROUTE_WARPS = 4;

// The VALUES consecutive logits of a lane, -infinity past the last expert; one
// vector load (or a few) where rows divide into such pieces.
template <int VALUES, typename T>
__device__ __forceinline__ void load_logits(const T* row, int lane, int experts, float (&l)[VALUES]) {
  constexpr int BYTES = VALUES * int(sizeof(T)), WIDE = BYTES < 16 ? BYTES : 16;
  if (experts % VALUES == 0 && reinterpret_cast<uintptr_t>(row) % WIDE == 0) {
    alignas(16) T v[VALUES];
    if (lane * VALUES < experts) {
      if constexpr (WIDE == 16) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(row + lane * VALUES)[i];
      } else if constexpr (WIDE == 8) {
        *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(row + lane * VALUES);
      } else if constexpr (WIDE == 4) {
        *reinterpret_cast<uint32_t*>(v) = *reinterpret_cast<const uint32_t*>(row + lane * VALUES);
      } else {
        v[0] = row[lane];
      }
#pragma unroll
      for (int j = 0; j < VALUES; ++j) l[j] = to_float(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < VALUES; ++j) l[j] = -INFINITY;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < VALUES; ++j) l[j] = lane * VALUES + j < experts ? to_float(row[lane * VALUES + j]) : -INFINITY;
}

// One step of a sorting network, larger key first.
__device__ __forceinline__ void order_keys(uint32_t& a, uint32_t& b) {
  const uint32_t hi = max(a, b);
  b = min(a, b);
  a = hi;
}

// One warp per token; lane `lane` holds VALUES consecutive experts, so that the
// first lane that reaches a maximum also holds the lowest such index, and a
// choice is one warp-wide maximum, a ballot and a shuffle; only the winning
// lane looks for its next best.
//
// SIMPLE: neither bias nor groups.  The order of the scores is then that of the
// logits, which no rounding blurs, so those are compared, and renormalised
// softmax weights need neither the row's sum nor the other experts' exponentials.
// The key of a 16-bit logit leaves its low bits free: with the (inverted) index
// in there a choice is the maximum alone, and each lane keeps its few keys
// sorted so that the next best moves up.
//
// Bound by instruction issue (16384 tokens of 128 experts, top 8, are 4 MB):
// 690 instructions a warp and 13.2 us before the two shortcuts.
template <int VALUES, typename T, bool SIMPLE>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) route_kernel(const RouteParams p) {
  constexpr bool PACKED = SIMPLE && sizeof(T) == 2;
  constexpr bool SORTED = PACKED && VALUES <= 8;
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long token = (long long)blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + token * p.experts;
  const int id0 = lane * VALUES;
  float l[VALUES];
  load_logits(row, lane, p.experts, l);
  const bool sigmoid = p.sigmoid != 0;
  RowScale r{0.0f, 1.0f};
  const bool by_chosen = SIMPLE && p.renormalise;  // scores relative to the largest chosen one
  if (!by_chosen) r = row_scale(l, sigmoid);
  uint32_t key[VALUES];
#pragma unroll
  for (int j = 0; j < VALUES; ++j) {
    float c = l[j];
    if (!SIMPLE && c != -INFINITY) c = score_of(l[j], r, sigmoid) + (p.bias && id0 + j < p.experts ? p.bias[id0 + j] : 0.0f);
    key[j] = score_key(c, l[j] != -INFINITY);
  }
  if (!SIMPLE && p.groups > 1) {
    uint32_t group_key = 0;  // of group `lane`
    const int span = p.each / VALUES;  // lanes of a group, where groups begin at lanes
    if (p.each % VALUES == 0 && (span & (span - 1)) == 0) {
      // All groups at once: each lane's best two, merged over the lanes of its group
      // (one after another 1 x 256 in 8 groups takes 6.6 us).
      uint32_t best = 0, second = 0;
#pragma unroll
      for (int j = 0; j < VALUES; ++j) {
        second = max(second, min(best, key[j]));
        best = max(best, key[j]);
      }
      for (int d = 1; d < span; d *= 2) {
        const uint32_t best2 = __shfl_xor_sync(ALL, best, d), second2 = __shfl_xor_sync(ALL, second, d);
        second = max(max(second, second2), min(best, best2));
        best = max(best, best2);
      }
      const float score = key_score(best) + (p.group_top == 2 && second ? key_score(second) : 0.0f);
      const uint32_t mine_key = best ? score_key(score, true) : 0u;
      const uint32_t of_lane = __shfl_sync(ALL, mine_key, (lane * span) & 31);
      group_key = lane < p.groups ? of_lane : 0u;
    } else for (int g = 0; g < p.groups; ++g) {
      const int first = g * p.each - id0, last = first + p.each;  // in this lane's values
      uint32_t best = 0, second = 0;
      if (first < VALUES && last > 0) {
#pragma unroll
        for (int j = 0; j < VALUES; ++j) {
          const uint32_t k = j >= first && j < last ? key[j] : 0u;
          second = max(second, min(best, k));
          best = max(best, k);
        }
      }
      const uint32_t one = __reduce_max_sync(ALL, best);
      float score = key_score(one);
      if (p.group_top == 2 && one) {
        const int holder = __ffs(__ballot_sync(ALL, best == one)) - 1;
        const uint32_t two = __reduce_max_sync(ALL, lane == holder ? second : best);
        if (two) score += key_score(two);
      }
      if (lane == g) group_key = one ? score_key(score, true) : 0u;
    }
    uint32_t open = 0;
    for (int i = 0; i < p.top_groups; ++i) {
      const uint32_t best = __reduce_max_sync(ALL, group_key);
      if (!best) break;
      const int winner = __ffs(__ballot_sync(ALL, group_key == best)) - 1;
      open |= 1u << winner;
      if (lane == winner) group_key = 0;
    }
    int g = id0 / p.each, left = p.each - (id0 - g * p.each);
#pragma unroll
    for (int j = 0; j < VALUES; ++j) {
      if (left == 0) ++g, left = p.each;
      --left;
      if (g >= p.groups || !(open >> g & 1)) key[j] = 0;
      if (!p.bias && key[j]) key[j] = score_key(l[j], true);  // inside the open groups the logits decide
    }
  }
  int mine = -1;  // choice number `lane`
  if constexpr (PACKED) {
    constexpr uint32_t LOW = 0x3FFu;  // a 16-bit float's key has at least 13 zeros (or, negative, ones) below
#pragma unroll
    for (int j = 0; j < VALUES; ++j) key[j] = key[j] ? (key[j] & ~LOW) | (LOW - uint32_t(id0 + j)) : 0u;
    if constexpr (SORTED) {
#pragma unroll
      for (int step = 0; step < VALUES; ++step)  // odd-even transposition: neighbours only
#pragma unroll
        for (int j = step & 1; j + 1 < VALUES; j += 2) order_keys(key[j], key[j + 1]);
    }
    uint32_t best = key[0];
    if constexpr (!SORTED) {
#pragma unroll
      for (int j = 1; j < VALUES; ++j) best = max(best, key[j]);
    }
    for (int i = 0; i < p.top_k; ++i) {
      const uint32_t top = __reduce_max_sync(ALL, best);
      if (!top) break;
      if (lane == i) mine = int(LOW - (top & LOW));
      if (best == top) {
        if constexpr (SORTED) {
#pragma unroll
          for (int j = 0; j + 1 < VALUES; ++j) key[j] = key[j + 1];
          key[VALUES - 1] = 0;
          best = key[0];
        } else {
          best = 0;
#pragma unroll
          for (int j = 0; j < VALUES; ++j) {
            key[j] = key[j] == top ? 0u : key[j];
            best = max(best, key[j]);
          }
        }
      }
    }
  } else {
    uint32_t best = 0;
    int at = 0;
    auto rescan = [&] {
      best = key[0], at = id0;
#pragma unroll
      for (int j = 1; j < VALUES; ++j)
        if (key[j] > best) best = key[j], at = id0 + j;
    };
    rescan();
    for (int i = 0; i < p.top_k; ++i) {
      const uint32_t top = __reduce_max_sync(ALL, best);
      if (!top) break;
      const int holder = __ffs(__ballot_sync(ALL, best == top)) - 1;
      const int winner = __shfl_sync(ALL, at, holder);
      if (lane == i) mine = winner;
      if (lane == holder) {
#pragma unroll
        for (int j = 0; j < VALUES; ++j) key[j] = id0 + j == at ? 0u : key[j];
        rescan();
      }
    }
  }
  const float chosen = mine >= 0 ? to_float(row[mine]) : -INFINITY;
  if (by_chosen) r.top = __shfl_sync(ALL, chosen, 0);
  float w = score_of(chosen, r, sigmoid);
  if (p.renormalise) {
    const float total = warp_sum(w);
    w = total == 0.0f ? 0.0f : w / total;
  }
  if (lane < p.top_k) {
    p.weights[token * p.top_k + lane] = w * p.scale;
    p.indices[token * p.top_k + lane] = mine;
  }
}

// d weights -> d logits.  q: the chosen scores, S their sum, g' the incoming
// gradient times the factor:  dq = (g' - sum(g' q) / S) / S when renormalised,
// else g'.  Softmax: dl = s (ds - sum(ds s)), where the sum vanishes after a
// renormalisation; logistic: dl = ds s (1 - s), the slope from the exponential
// itself, as 1 - s has lost its digits where s is next to 1.  Both differences
// are the same with any number taken from all g' (or ds); where one expert has
// more than half of the weight it is that expert's own, so that the gradient of
// the largest score, a sum over the others' small ones, is not what is left of
// two nearly equal numbers.  The few ds are scattered through shared memory (an
// index may be there twice).
template <int VALUES, typename T>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) route_gradient_kernel(const RouteParams p) {
  __shared__ float scattered[ROUTE_WARPS][32 * VALUES];
  float* const ds = scattered[threadIdx.x >> 5];
  const int lane = threadIdx.x & 31, id0 = lane * VALUES;
#pragma unroll
  for (int j = 0; j < VALUES; ++j) ds[j * 32 + lane] = 0.0f;
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const long long token = (long long)blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + token * p.experts;
  int mine = lane < p.top_k ? p.indices[token * p.top_k + lane] : -1;
  if (mine >= p.experts) mine = -1;
  float g = mine >= 0 ? p.grad_weights[token * p.top_k + lane] * p.scale : 0.0f;
  const float chosen = mine >= 0 ? to_float(row[mine]) : -INFINITY;
  float l[VALUES];
  load_logits(row, lane, p.experts, l);
  const bool sigmoid = p.sigmoid != 0;
  const RowScale r = row_scale(l, sigmoid);
  const float q = score_of(chosen, r, sigmoid);
  if (p.renormalise) {
    const float total = warp_sum(q);
    const unsigned lead = __ballot_sync(ALL, q > 0.5f * total);
    if (lead) {
      const float own = __shfl_sync(ALL, g, __ffs(lead) - 1);
      g = mine >= 0 ? g - own : 0.0f;
    }
    const float dot = warp_sum(g * q);
    g = mine >= 0 && total != 0.0f ? (g - dot / total) / total : 0.0f;
  }
  __syncwarp();
  // One after another where an index is repeated, in the order of the choices.
  unsigned todo = __ballot_sync(ALL, mine >= 0);
  const unsigned same = __match_any_sync(ALL, mine);
  while (todo) {
    const bool turn = (todo >> lane & 1) && !(same & todo & ((1u << lane) - 1));
    if (turn) ds[mine] += g;
    todo &= ~__ballot_sync(ALL, turn);
    __syncwarp();
  }
  T* out = static_cast<T*>(p.grad_logits) + token * p.experts;
  alignas(16) T v[VALUES];
  if (sigmoid || p.renormalise) {
#pragma unroll
    for (int j = 0; j < VALUES; ++j) v[j] = from_float<T>(ds[id0 + j] * (sigmoid ? logistic_slope(l[j]) : score_of(l[j], r, false)));
  } else {
    float own = 0.0f, through = 0.0f;  // the leader's ds, in its lane
    bool leads = false;
#pragma unroll
    for (int j = 0; j < VALUES; ++j) {
      l[j] = score_of(l[j], r, false);
      if (l[j] > 0.5f) leads = true, own = ds[id0 + j];
    }
    const unsigned lead = __ballot_sync(ALL, leads);
    if (lead) own = __shfl_sync(ALL, own, __ffs(lead) - 1);
#pragma unroll
    for (int j = 0; j < VALUES; ++j) through = fmaf(l[j], ds[id0 + j] - own, through);
    through = warp_sum(through);
#pragma unroll
    for (int j = 0; j < VALUES; ++j) v[j] = from_float<T>(l[j] * (ds[id0 + j] - own - through));
  }
  constexpr int BYTES = VALUES * int(sizeof(T)), WIDE = BYTES < 16 ? BYTES : 16;
  if (p.experts % VALUES == 0 && reinterpret_cast<uintptr_t>(out) % WIDE == 0) {
    if (id0 < p.experts) {
      if constexpr (WIDE == 16) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(out + id0)[i] = reinterpret_cast<const uint4*>(v)[i];
      } else if constexpr (WIDE == 8) {
        *reinterpret_cast<uint2*>(out + id0) = *reinterpret_cast<const uint2*>(v);
      } else if constexpr (WIDE == 4) {
        *reinterpret_cast<uint32_t*>(out + id0) = *reinterpret_cast<const uint32_t*>(v);
      } else {
        out[id0] = v[0];
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < VALUES; ++j)
    if (id0 + j < p.experts) out[id0 + j] = v[j];
}

// -------------------------------------------------------------------- plan

// Rows in order of their expert, in the order of the pairs inside one: a
// stable counting sort.  A block takes a chunk of pairs and each of its warps a
// contiguous part, so ranks follow from counts in order: before the chunk
// (histograms of a first kernel), before the warp's part (counts in shared
// memory), inside it (lanes with the same expert).  Atomics only count, they
// decide no order, so the plan is the same every time.
// A lane reads its PLAN_EACH pairs at once and keeps them: with a load per step
// the chain of trips to L2 was most of the time (4096 pairs: 6.9 us).
constexpr int PLAN_WARPS = 32;
constexpr int PLAN_CHUNK = 8192;  // pairs per block; up to this many need no histogram
constexpr int PLAN_EACH = PLAN_CHUNK / (PLAN_WARPS * 32);
// Above this many chunks their counts are added up once, by a kernel between the
// two; up to it each block adds up all of them itself, which saves that launch but
// grows with the square of the pairs (256 experts: 16 chunks 11.7 us, 13.2 with the
// kernel between; 64 chunks 13.8 and 13.9; 256 chunks 39 and 24; 1024 chunks 302 and 80).
constexpr int PLAN_SCAN = 64;

struct PlanParams {
  const int* indices;
  int* offsets;    // [experts + 1]
  int* tokens;     // [pairs] the token of each sorted row
  int* positions;  // [pairs] the sorted row of each pair, -1 for one that goes nowhere
  int* histogram;  // [chunks, experts] counts; above PLAN_SCAN chunks then the counts up to and with each chunk
  int pairs, top_k, experts, chunks;
};

__global__ void __launch_bounds__(PLAN_WARPS * 32) plan_histogram_kernel(const PlanParams p) {
  extern __shared__ int counts[];
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) counts[e] = 0;
  __syncthreads();
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int first = blockIdx.x * PLAN_CHUNK, last = min(first + PLAN_CHUNK, p.pairs);
  for (int i = first + threadIdx.x; i < last; i += blockDim.x) {
    const int e = p.indices[i];
    if (e >= 0 && e < p.experts) atomicAdd(&counts[e], 1);  // a count, whatever the order
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) p.histogram[blockIdx.x * p.experts + e] = counts[e];
}

// Counts of each chunk -> counts up to and with it, in place.  A block has 32
// experts, one a lane; its warps each take a run of chunks, add it up, learn from
// one another what comes before it, and go over it again.
__global__ void __launch_bounds__(PLAN_WARPS * 32) plan_scan_kernel(const PlanParams p) {
  __shared__ int sums[PLAN_WARPS][32];
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = blockIdx.x * 32 + lane;
  const int each = (p.chunks + PLAN_WARPS - 1) / PLAN_WARPS, first = min(warp * each, p.chunks), last = min(first + each, p.chunks);
  int* const column = p.histogram + e;
  int sum = 0;
  if (e < p.experts) {
#pragma unroll 8
    for (int c = first; c < last; ++c) sum += column[(long long)c * p.experts];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (e >= p.experts) return;
  int run = 0;
  for (int w = 0; w < warp; ++w) run += sums[w][lane];
  for (int c0 = first; c0 < last; c0 += 8) {  // eight loads in flight
    int n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = c0 + i < last ? column[(long long)(c0 + i) * p.experts] : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      run += n[i];
      if (c0 + i < last) column[(long long)(c0 + i) * p.experts] = run;
    }
  }
}

__global__ void __launch_bounds__(PLAN_WARPS * 32) plan_kernel(const PlanParams p) {
  extern __shared__ int shared[];
  int* const counts = shared;                            // [warps][experts], then the warp's next row
  int* const base = shared + PLAN_WARPS * p.experts;     // [experts] rows of all chunks, then the chunk's first row
  int* const ahead = base + p.experts;                   // [experts] rows of earlier chunks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < PLAN_WARPS * p.experts; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int first = blockIdx.x * PLAN_CHUNK, size = min(PLAN_CHUNK, p.pairs - first);
  const int part = (size + PLAN_WARPS * 32 - 1) / (PLAN_WARPS * 32) * 32;  // at most PLAN_EACH * 32
  const int begin = first + min(warp * part, size), end = first + min((warp + 1) * part, size);
  int* const own = counts + warp * p.experts;
  int expert[PLAN_EACH];
#pragma unroll
  for (int s = 0; s < PLAN_EACH; ++s) {
    const int i = begin + s * 32 + lane;
    expert[s] = i < end ? p.indices[i] : -1;
    if (expert[s] >= p.experts || expert[s] < 0) expert[s] = -1;
  }
#pragma unroll
  for (int s = 0; s < PLAN_EACH; ++s)
    if (expert[s] >= 0) atomicAdd(&own[expert[s]], 1);  // a count, whatever the order
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
    int run = 0;
#pragma unroll 1
    for (int w0 = 0; w0 < PLAN_WARPS; w0 += 16) {  // sixteen loads in flight, not one
      int part_of[16];
#pragma unroll
      for (int w = 0; w < 16; ++w) part_of[w] = counts[(w0 + w) * p.experts + e];
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        counts[(w0 + w) * p.experts + e] = run;
        run += part_of[w];
      }
    }
    int before = 0, total = run;
    if (p.chunks > PLAN_SCAN) {
      if (blockIdx.x) before = p.histogram[(blockIdx.x - 1) * p.experts + e];
      total = p.histogram[(p.chunks - 1) * p.experts + e];
    } else if (p.chunks > 1) {
      total = 0;
#pragma unroll 8
      for (int c = 0; c < p.chunks; ++c) {
        const int n = p.histogram[c * p.experts + e];
        if (c < int(blockIdx.x)) before += n;
        total += n;
      }
    }
    base[e] = total;
    ahead[e] = before;
  }
  __syncthreads();
  if (warp == 0) {  // exclusive sums over the experts
    const int per = (p.experts + 31) / 32, e0 = min(lane * per, p.experts), e1 = min(e0 + per, p.experts);
    int sum = 0;
    for (int e = e0; e < e1; ++e) sum += base[e];
    int run = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(ALL, run, d);
      if (lane >= d) run += other;
    }
    run -= sum;
    for (int e = e0; e < e1; ++e) {
      const int n = base[e];
      if (blockIdx.x == 0) p.offsets[e] = run;
      base[e] = run + ahead[e];
      run += n;
    }
    if (blockIdx.x == 0 && lane == 31) p.offsets[p.experts] = run;
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < PLAN_EACH; ++s) {
    const int i = begin + s * 32 + lane;
    if (i - lane >= end) break;
    const int e = expert[s];
    unsigned same = __ballot_sync(ALL, e >= 0);  // lanes with the same expert: one ballot per bit of its number
    for (int bit = 1; bit < p.experts; bit *= 2) {
      const unsigned set = __ballot_sync(ALL, (e & bit) != 0);
      same &= (e & bit) ? set : ~set;
    }
    const int row = e >= 0 ? base[e] + own[e] + __popc(same & ((1u << lane) - 1)) : -1;
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) own[e] += __popc(same);
    __syncwarp();
    if (i < end) {
      p.positions[i] = row;
      if (e >= 0) p.tokens[row] = i / p.top_k;
    }
  }
}

// ------------------------------------------------------------------ gather

// out[r] = x[tokens[r]] for the plan's rows, 16 bytes a lane, a warp per row: two
// passes over the rows (67 MB each for 8192 rows of 4096 bf16 values) against
// fetching them row by row inside the product, where the copy engine takes some
// 50 cycles for four rows of 128 bytes and a tile of 128 rows then waits for it
// (8 experts, 4096 x 4096, 7675 rows: 660 us gathered there, 199 us on sorted rows).
__global__ void __launch_bounds__(256) gather_kernel(const uint4* x, const int* tokens, const int* limit, uint4* out, int vectors, int rows) {
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= min(rows, *limit)) return;
  const uint4* src = x + (long long)tokens[row] * vectors;
  uint4* dst = out + (long long)row * vectors;
  int i = lane;
  for (; i + 96 < vectors; i += 128) {
    const uint4 a = src[i], b = src[i + 32], c = src[i + 64], d = src[i + 96];
    dst[i] = a, dst[i + 32] = b, dst[i + 64] = c, dst[i + 96] = d;
  }
  for (; i < vectors; i += 32) dst[i] = src[i];
}

// ----------------------------------------------------------------- combine

struct CombineParams {
  const void* y;          // [rows, n]
  const float* weights;   // [tokens, top_k], or null for ones
  const int* positions;   // [tokens, top_k]
  const void* residual;   // [tokens, n], or null
  void* out;              // [tokens, n]; gradient: grad_y [rows, n]
  const void* grad;       // gradient: of out
  float* grad_weights;    // gradient: [tokens, top_k]
  long long tokens;
  int n, top_k;
};

constexpr int COMBINE_THREADS = 128;

// out[t] = residual[t] + sum over j of weights[t, j] * y[positions[t, j]], added
// in the order of j in float32.  A thread takes eight columns (one when rows
// are not multiples of 16 bytes); its top_k loads do not depend on one another.
// Y: type of the rows (float32 where a gradient's parts must not be rounded
// before they are added).
template <typename T, typename Y, bool VECTOR>
__global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(const CombineParams p) {
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  constexpr int WIDE = VECTOR ? 8 : 1;
  const long long token = blockIdx.x;
  const int col = (blockIdx.y * COMBINE_THREADS + threadIdx.x) * WIDE;
  if (col >= p.n) return;
  const Y* y = static_cast<const Y*>(p.y);
  const T* residual = static_cast<const T*>(p.residual);
  float sum[WIDE];
#pragma unroll
  for (int i = 0; i < WIDE; ++i) sum[i] = 0.0f;
#pragma unroll 4
  for (int j = 0; j < p.top_k; ++j) {
    const int row = p.positions[token * p.top_k + j];
    if (row < 0) continue;
    const float w = p.weights ? p.weights[token * p.top_k + j] : 1.0f;
    float v[WIDE];
    if constexpr (VECTOR) load8(y + (long long)row * p.n + col, v);
    else v[0] = to_float(y[(long long)row * p.n + col]);
#pragma unroll
    for (int i = 0; i < WIDE; ++i) sum[i] = fmaf(w, v[i], sum[i]);
  }
  if (residual) {
    float v[WIDE];
    if constexpr (VECTOR) load8(residual + token * p.n + col, v);
    else v[0] = to_float(residual[token * p.n + col]);
#pragma unroll
    for (int i = 0; i < WIDE; ++i) sum[i] += v[i];
  }
  T* out = static_cast<T*>(p.out) + token * p.n + col;
  if constexpr (VECTOR) store8(out, sum);
  else *out = from_float<T>(sum[0]);
}

// grad_y[positions[t, j]] = weights[t, j] * grad[t] and grad_weights[t, j] =
// <grad[t], y[positions[t, j]]>: one block per pair, its threads' parts of the
// product added in a fixed order.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(COMBINE_THREADS) combine_gradient_kernel(const CombineParams p) {
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  constexpr int WIDE = VECTOR ? 8 : 1;
  const long long pair = blockIdx.x;
  const int row = p.positions[pair];
  if (row < 0) {
    if (threadIdx.x == 0) p.grad_weights[pair] = 0.0f;
    return;
  }
  const T* grad = static_cast<const T*>(p.grad) + pair / p.top_k * p.n;
  const T* y = static_cast<const T*>(p.y) + (long long)row * p.n;
  T* out = static_cast<T*>(p.out) + (long long)row * p.n;
  const float w = p.weights[pair];
  float dot = 0.0f;
  for (int col = threadIdx.x * WIDE; col < p.n; col += COMBINE_THREADS * WIDE) {
    float g[WIDE], v[WIDE];
    if constexpr (VECTOR) load8(grad + col, g), load8(y + col, v);
    else g[0] = to_float(grad[col]), v[0] = to_float(y[col]);
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      dot = fmaf(g[i], v[i], dot);
      g[i] *= w;
    }
    if constexpr (VECTOR) store8(out + col, g);
    else out[col] = from_float<T>(g[0]);
  }
  __shared__ float parts[COMBINE_THREADS / 32];
  dot = warp_sum(dot);
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < COMBINE_THREADS / 32; ++i) total += parts[i];
    p.grad_weights[pair] = total;
  }
}

// ---------------------------------------------------- gradient of activation

struct ActGradientParams {
  const void* grad;   // [rows, width]
  const void* z;      // [rows, n], or null without an activation
  void* dz;           // [rows, n], or null when it is grad itself
  float* partial;     // [row blocks, n] column sums, or null
  float* column_sums; // [n] the sums themselves, where one cluster of blocks has all rows
  int block_rows;     // rows a block works on, a multiple of 8
  const int* limit;   // rows to work on (device), or null for all
  long long rows;
  int n, width, shape, glu;
  float a, b;
};

// Rows to work on: all, or those before a limit that an earlier kernel left on the device.
__device__ __forceinline__ long long live_rows(const int* limit, long long rows) { return limit ? min((long long)*limit, rows) : rows; }

constexpr int GRADIENT_CLUSTER = 8;  // up to this many blocks add up their column sums among themselves

// dz = grad * act'(z), eight columns a thread; a gated pair writes both halves,
// gate: grad * up * act'(gate), up: grad * act(gate).  Column sums (of the
// unrounded values) are added per thread down its rows, across the block's row
// lanes in a fixed order, and across blocks by column_sum_kernel; where eight
// blocks have all rows they are one cluster, whose first adds the others' sums
// from their shared memory, which saves that launch.
template <typename T>
__global__ void __launch_bounds__(256) act_gradient_kernel(const ActGradientParams p) {
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const long long rows = live_rows(p.limit, p.rows);
  const long long first = (long long)blockIdx.x * p.block_rows;
  if (first >= rows) return;  // (never with column_sums: its grid is the blocks that have rows)
  const int lane = threadIdx.x & 31, row_lane = threadIdx.x >> 5;
  const int col = (blockIdx.y * 32 + lane) * 8;
  const bool live = col < p.width;
  const T* grad = static_cast<const T*>(p.grad);
  const T* z = static_cast<const T*>(p.z);
  T* dz = static_cast<T*>(p.dz);
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto slopes_as = [&](auto shape, const float* x, float* value, float* slope) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float2 v, d;
      act_both2<decltype(shape)::value>(make_float2(x[i], x[i + 1]), p.a, p.b, &v, &d);
      value[i] = v.x, value[i + 1] = v.y, slope[i] = d.x, slope[i + 1] = d.y;
    }
  };
  auto slopes = [&](const float* x, float* value, float* slope) {
    if (p.shape == SHAPE_SIGMOID) slopes_as(std::integral_constant<int, SHAPE_SIGMOID>{}, x, value, slope);
    else if (p.shape == SHAPE_PHI) slopes_as(std::integral_constant<int, SHAPE_PHI>{}, x, value, slope);
    else slopes_as(std::integral_constant<int, SHAPE_RELU>{}, x, value, slope);
  };
#pragma unroll 2
  for (int r = row_lane; r < p.block_rows; r += 8) {
    const long long row = first + r;
    if (!live || row >= rows) break;
    float g[8], x[8], value[8], slope[8];
    load8(grad + row * p.width + col, g);
    if (p.glu) {
      float up[8];
      load8(z + row * p.n + col, x);
      load8(z + row * p.n + p.width + col, up);
      slopes(x, value, slope);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        slope[i] *= g[i] * up[i];
        value[i] *= g[i];
      }
      store8(dz + row * p.n + col, slope);
      store8(dz + row * p.n + p.width + col, value);
      continue;
    }
    if (z) {
      load8(z + row * p.n + col, x);
      slopes(x, value, slope);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] *= slope[i];
      store8(dz + row * p.n + col, g);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += g[i];
  }
  if (!p.partial && !p.column_sums) return;
  __shared__ float parts[8][256];
#pragma unroll
  for (int i = 0; i < 8; ++i) parts[row_lane][i * 32 + lane] = sum[i];
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) total += parts[i][threadIdx.x];
  const int at = blockIdx.y * 256 + (threadIdx.x & 31) * 8 + (threadIdx.x >> 5);
  if (!p.column_sums) {
    if (at < p.n) p.partial[(long long)blockIdx.x * p.n + at] = total;
    return;
  }
  __syncthreads();  // everyone has read its column of `parts`
  parts[0][threadIdx.x] = total;
  cluster_sync_all();
  if (blockIdx.x == 0 && at < p.n) {
    for (unsigned b = 1; b < gridDim.x; ++b) total += ld_cluster_f32(map_to_cta(smem_u32(&parts[0][threadIdx.x]), b));
    p.column_sums[at] = total;
  }
  cluster_sync_all();  // the others' shared memory stays until it has been read
}

// Sums over the row blocks that have rows (the others wrote no sums): eight
// lanes take every eighth block, added in order.
__global__ void __launch_bounds__(256) column_sum_kernel(const float* partial, float* out, const int* limit, long long rows, int block_rows, int n) {
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const int blocks = int((live_rows(limit, rows) + block_rows - 1) / block_rows);
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (col < n) {
#pragma unroll 8
    for (int b = part; b < blocks; b += 8) sum += partial[(long long)b * n + col];
  }
  __shared__ float parts[8][32];
  parts[part][lane] = sum;
  __syncthreads();
  if (part || col >= n) return;
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) total += parts[i][lane];
  out[col] = total;
}

// -------------------------------------------------------------------- host

thread_local char routing_error[256];

int routing_fail(const char* format, ...) {
  va_list args;
  va_start(args, format);
  vsnprintf(routing_error, sizeof routing_error, format, args);
  va_end(args);
  return OG_ERR_LAUNCH;
}

int check_device(const DeviceScope& on, int device) {
  return on.status() == cudaSuccess ? int(OG_OK) : routing_fail("cudaSetDevice(%d): %s", device, cudaGetErrorString(on.status()));
}

template <typename... Args>
int clustered_launch(void (*kernel)(Args...), dim3 grid, int cluster, int threads, size_t smem, void* stream, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads, 1, 1);
  config.dynamicSmemBytes = smem;
  config.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = dependent_launches();
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t launched = cudaLaunchKernelEx(&config, kernel, args...);
  if (launched != cudaSuccess) return routing_fail("kernel launch failed: %s", cudaGetErrorString(launched));
  return OG_OK;
}

template <typename... Args>
int dependent_launch(void (*kernel)(Args...), dim3 grid, int threads, size_t smem, void* stream, Args... args) {
  return clustered_launch(kernel, grid, 1, threads, smem, stream, args...);
}

enum ElementType : int { TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2 };

template <template <int, typename> class Picker, typename T>
auto pick_values(int experts) {
  const int values = (experts + 31) / 32;
  return values <= 1 ? Picker<1, T>::kernel : values <= 2 ? Picker<2, T>::kernel : values <= 4 ? Picker<4, T>::kernel
         : values <= 8 ? Picker<8, T>::kernel : values <= 16 ? Picker<16, T>::kernel : Picker<32, T>::kernel;
}
template <int VALUES, typename T> struct RouteSimple { static constexpr void (*kernel)(RouteParams) = route_kernel<VALUES, T, true>; };
template <int VALUES, typename T> struct RouteForward { static constexpr void (*kernel)(RouteParams) = route_kernel<VALUES, T, false>; };
template <int VALUES, typename T> struct RouteGradient { static constexpr void (*kernel)(RouteParams) = route_gradient_kernel<VALUES, T>; };

int check_route(const OgRoute& r) {
  if (r.dtype < TYPE_F32 || r.dtype > TYPE_F16) return routing_fail("dtype %d is none of 0 (float32), 1 (bfloat16), 2 (float16)", r.dtype);
  if (r.experts < 1 || r.experts > 1024) return routing_fail("%d experts: 1 to 1024 are served", r.experts);
  if (r.top_k < 1 || r.top_k > 32 || r.top_k > r.experts) return routing_fail("top_k = %d: 1 to 32 of the %d experts", r.top_k, r.experts);
  if (r.tokens < 0 || r.tokens > 0x7FFFFFFFll * ROUTE_WARPS) return routing_fail("tokens = %lld", (long long)r.tokens);
  return OG_OK;
}

}  // namespace
}  // namespace og

using namespace og;

extern "C" {

OG_API const char* og_b200_routing_error(void) { return routing_error; }

OG_API int32_t og_b200_route(const OgRoute* route, const void* logits, const float* bias, float* weights, int32_t* indices,
                             int32_t device, void* stream) {
  if (!route) return routing_fail("null OgRoute");
  const OgRoute& r = *route;
  if (const int bad = check_route(r)) return bad;
  if (r.groups < 1 || r.groups > 32 || r.experts % r.groups) return routing_fail("%d groups: 1 to 32 that divide the %d experts", r.groups, r.experts);
  if (r.top_groups < 1 || r.top_groups > r.groups) return routing_fail("top_groups = %d of %d groups", r.top_groups, r.groups);
  if (r.group_top != 1 && r.group_top != 2) return routing_fail("group_top = %d: 1 or 2", r.group_top);
  if (r.top_k > r.top_groups * (r.experts / r.groups)) return routing_fail("top_k = %d is more than the %d experts of the open groups", r.top_k, r.top_groups * (r.experts / r.groups));
  if (!r.tokens) return OG_OK;
  if (!logits || !weights || !indices) return routing_fail("logits, weights and indices must be device pointers, got null");
  const DeviceScope on(device);
  if (const int bad = check_device(on, device)) return bad;
  RouteParams p{};
  p.logits = logits, p.bias = bias, p.weights = weights, p.indices = indices, p.tokens = r.tokens, p.experts = r.experts;
  p.top_k = r.top_k, p.sigmoid = r.sigmoid, p.groups = r.groups, p.each = r.experts / r.groups, p.top_groups = r.top_groups;
  p.group_top = r.group_top, p.renormalise = r.renormalise, p.scale = r.scale;
  const bool simple = !bias && r.groups == 1;
#define OG_ROUTE(T) (simple ? pick_values<RouteSimple, T>(r.experts) : pick_values<RouteForward, T>(r.experts))
  const auto kernel = r.dtype == TYPE_F32 ? OG_ROUTE(float) : r.dtype == TYPE_BF16 ? OG_ROUTE(__nv_bfloat16) : OG_ROUTE(__half);
#undef OG_ROUTE
  return dependent_launch(kernel, dim3(unsigned((r.tokens + ROUTE_WARPS - 1) / ROUTE_WARPS)), ROUTE_WARPS * 32, 0, stream, p);
}

OG_API int32_t og_b200_route_gradient(const OgRoute* route, const float* grad_weights, const void* logits, const int32_t* indices,
                                      void* grad_logits, int32_t device, void* stream) {
  if (!route) return routing_fail("null OgRoute");
  const OgRoute& r = *route;
  if (const int bad = check_route(r)) return bad;
  if (!r.tokens) return OG_OK;
  if (!grad_weights || !logits || !indices || !grad_logits) return routing_fail("gradients, logits and indices must be device pointers, got null");
  const DeviceScope on(device);
  if (const int bad = check_device(on, device)) return bad;
  RouteParams p{};
  p.logits = logits, p.grad_weights = grad_weights, p.indices = const_cast<int32_t*>(indices), p.grad_logits = grad_logits;
  p.tokens = r.tokens, p.experts = r.experts, p.top_k = r.top_k, p.sigmoid = r.sigmoid, p.renormalise = r.renormalise, p.scale = r.scale;
  const auto kernel = r.dtype == TYPE_F32    ? pick_values<RouteGradient, float>(r.experts)
                      : r.dtype == TYPE_BF16 ? pick_values<RouteGradient, __nv_bfloat16>(r.experts)
                                             : pick_values<RouteGradient, __half>(r.experts);
  return dependent_launch(kernel, dim3(unsigned((r.tokens + ROUTE_WARPS - 1) / ROUTE_WARPS)), ROUTE_WARPS * 32, 0, stream, p);
}

OG_API int32_t og_b200_expert_plan(const int32_t* indices, int64_t tokens, int32_t top_k, int32_t experts, int32_t* offsets,
                                   int32_t* token_of_row, int32_t* positions, int32_t* workspace, int32_t device, void* stream) {
  if (experts < 1 || experts > 1024) return routing_fail("%d experts: 1 to 1024 are served", experts);
  if (top_k < 1 || tokens < 0 || tokens > 0x40000000ll || tokens * top_k > 0x40000000ll) return routing_fail("%lld tokens with %d experts each are too many", (long long)tokens, top_k);
  if (!offsets || (tokens && (!indices || !token_of_row || !positions))) return routing_fail("indices and the plan's arrays must be device pointers, got null");
  if (tokens * top_k > PLAN_CHUNK && !workspace)
    return routing_fail("%lld pairs take a workspace of %lld integers", (long long)(tokens * top_k), (long long)((tokens * top_k + PLAN_CHUNK - 1) / PLAN_CHUNK * experts));
  const DeviceScope on(device);
  if (const int bad = check_device(on, device)) return bad;
  PlanParams p{};
  p.indices = indices, p.offsets = offsets, p.tokens = token_of_row, p.positions = positions, p.histogram = workspace;
  p.pairs = int(tokens * top_k), p.top_k = top_k, p.experts = experts;
  p.chunks = std::max(1, (p.pairs + PLAN_CHUNK - 1) / PLAN_CHUNK);
  if (p.chunks > 1) {
    if (const int bad = dependent_launch(plan_histogram_kernel, dim3(p.chunks), PLAN_WARPS * 32, experts * sizeof(int), stream, p)) return bad;
  }
  if (p.chunks > PLAN_SCAN) {
    if (const int bad = dependent_launch(plan_scan_kernel, dim3((experts + 31) / 32), PLAN_WARPS * 32, 0, stream, p)) return bad;
  }
  const size_t smem = size_t(PLAN_WARPS + 2) * experts * sizeof(int);
  if (smem > 48 * 1024) {  // up to 136 KiB for 1024 experts
    const cudaError_t status = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (PLAN_WARPS + 2) * 1024 * int(sizeof(int)));
    if (status != cudaSuccess) return routing_fail("cudaFuncSetAttribute: %s", cudaGetErrorString(status));
  }
  return dependent_launch(plan_kernel, dim3(p.chunks), PLAN_WARPS * 32, smem, stream, p);
}

static bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }

OG_API int32_t og_b200_expert_gather(const void* x, const int32_t* token_of_row, const int32_t* row_limit, void* out, int64_t row_bytes,
                                     int32_t rows, int32_t device, void* stream) {
  if (rows < 0 || row_bytes < 16 || row_bytes % 16 || row_bytes / 16 > 0x7FFFFFFF) return routing_fail("rows of %lld bytes: a multiple of 16", (long long)row_bytes);
  if (!rows) return OG_OK;
  if (!x || !token_of_row || !row_limit || !out) return routing_fail("x, the plan and out must be device pointers, got null");
  if (!aligned16(x) || !aligned16(out)) return routing_fail("rows must start on 16-byte boundaries");
  const DeviceScope on(device);
  if (const int bad = check_device(on, device)) return bad;
  return dependent_launch(gather_kernel, dim3(unsigned((rows + 7) / 8)), 256, 0, stream, static_cast<const uint4*>(x), token_of_row, row_limit,
                          static_cast<uint4*>(out), int(row_bytes / 16), int(rows));
}

OG_API int32_t og_b200_expert_combine(int32_t dtype, int32_t y_is_f32, const void* y, const float* weights, const int32_t* positions, const void* residual,
                                      void* out, int64_t tokens, int32_t top_k, int32_t n, int32_t device, void* stream) {
  if (dtype != TYPE_BF16 && dtype != TYPE_F16) return routing_fail("dtype %d is none of 1 (bfloat16), 2 (float16)", dtype);
  if (tokens < 0 || tokens > 0x7FFFFFFFll || top_k < 1 || n < 1) return routing_fail("tokens = %lld, top_k = %d, n = %d", (long long)tokens, top_k, n);
  if (!tokens) return OG_OK;
  if (!y || !positions || !out) return routing_fail("y, positions and out must be device pointers, got null");
  const DeviceScope on(device);
  if (const int bad = check_device(on, device)) return bad;
  CombineParams p{};
  p.y = y, p.weights = weights, p.positions = positions, p.residual = residual, p.out = out, p.tokens = tokens, p.n = n, p.top_k = top_k;
  const bool wide = n % 8 == 0 && aligned16(y) && aligned16(residual) && aligned16(out);
  const int columns = COMBINE_THREADS * (wide ? 8 : 1);
  if ((n + columns - 1) / columns > 65535) return routing_fail("n = %d is too wide", n);
  const dim3 grid(unsigned(tokens), unsigned((n + columns - 1) / columns));
#define OG_COMBINE(T) (y_is_f32 ? (wide ? combine_kernel<T, float, true> : combine_kernel<T, float, false>) \
                                : (wide ? combine_kernel<T, T, true> : combine_kernel<T, T, false>))
  const auto kernel = dtype == TYPE_BF16 ? OG_COMBINE(__nv_bfloat16) : OG_COMBINE(__half);
#undef OG_COMBINE
  return dependent_launch(kernel, grid, COMBINE_THREADS, 0, stream, p);
}

OG_API int32_t og_b200_expert_combine_gradient(int32_t dtype, const void* grad, const void* y, const float* weights, const int32_t* positions,
                                               void* grad_y, float* grad_weights, int64_t tokens, int32_t top_k, int32_t n, int32_t device,
                                               void* stream) {
  if (dtype != TYPE_BF16 && dtype != TYPE_F16) return routing_fail("dtype %d is none of 1 (bfloat16), 2 (float16)", dtype);
  if (tokens < 0 || top_k < 1 || n < 1 || tokens * top_k > 0x7FFFFFFFll) return routing_fail("tokens = %lld, top_k = %d, n = %d", (long long)tokens, top_k, n);
  if (!tokens) return OG_OK;
  if (!grad || !y || !weights || !positions || !grad_y || !grad_weights) return routing_fail("the gradient's tensors must be device pointers, got null");
  const DeviceScope on(device);
  if (const int bad = check_device(on, device)) return bad;
  CombineParams p{};
  p.y = y, p.weights = weights, p.positions = positions, p.grad = grad, p.out = grad_y, p.grad_weights = grad_weights;
  p.tokens = tokens, p.n = n, p.top_k = top_k;
  const bool wide = n % 8 == 0 && aligned16(y) && aligned16(grad) && aligned16(grad_y);
  const auto kernel = dtype == TYPE_BF16 ? (wide ? combine_gradient_kernel<__nv_bfloat16, true> : combine_gradient_kernel<__nv_bfloat16, false>)
                                         : (wide ? combine_gradient_kernel<__half, true> : combine_gradient_kernel<__half, false>);
  return dependent_launch(kernel, dim3(unsigned(tokens * top_k)), COMBINE_THREADS, 0, stream, p);
}

OG_API int32_t og_b200_activation_gradient(int32_t dtype, int32_t activation, const void* grad, const void* z, void* dz, float* bias_gradient,
                                           float* workspace, const int32_t* row_limit, int64_t rows, int32_t n, int32_t device, void* stream) {
  if (dtype != TYPE_BF16 && dtype != TYPE_F16) return routing_fail("dtype %d is none of 1 (bfloat16), 2 (float16)", dtype);
  if (activation < ACT_NONE || activation > ACT_GEGLU) return routing_fail("activation %d is none of 0..%d", activation, int(ACT_GEGLU));
  const bool glu = activation == ACT_SWIGLU || activation == ACT_GEGLU;
  if (rows < 0 || n < 1 || n % (glu ? 16 : 8)) return routing_fail("rows = %lld, n = %d: columns come in eights", (long long)rows, n);
  if (glu && bias_gradient) return routing_fail("a gated activation has no bias gradient here");
  if (rows > 0x7FFFFFFFll) return routing_fail("rows = %lld are too many", (long long)rows);
  const DeviceScope on(device);
  if (const int bad = check_device(on, device)) return bad;
  const int block_rows = gradient_block_rows(rows, glu ? n / 2 : n);
  const int blocks = int((rows + block_rows - 1) / block_rows);
  const bool one_cluster = bias_gradient && !row_limit && rows && blocks <= GRADIENT_CLUSTER;
  if (rows) {
    if (!grad || (activation && (!z || !dz)) || (bias_gradient && !workspace)) return routing_fail("the gradient's tensors must be device pointers, got null");
    if (!aligned16(grad) || !aligned16(z) || !aligned16(dz)) return routing_fail("gradients and pre-activations must start on 16-byte boundaries");
    ActGradientParams p{};
    p.grad = grad, p.z = activation ? z : nullptr, p.dz = dz, p.limit = row_limit, p.block_rows = block_rows;
    if (one_cluster) p.column_sums = bias_gradient;
    else if (bias_gradient) p.partial = workspace;
    p.rows = rows, p.n = n, p.width = glu ? n / 2 : n, p.glu = glu;
    act_constants(activation, &p.shape, &p.a, &p.b);
    if (!activation && !bias_gradient) return OG_OK;
    const dim3 grid(unsigned(blocks), unsigned((p.width + 255) / 256));
    if (grid.y > 65535) return routing_fail("n = %d is too wide", n);
    const auto kernel = dtype == TYPE_BF16 ? act_gradient_kernel<__nv_bfloat16> : act_gradient_kernel<__half>;
    if (const int bad = clustered_launch(kernel, grid, one_cluster ? blocks : 1, 256, 0, stream, p)) return bad;
  }
  if (!bias_gradient || one_cluster) return OG_OK;
  return dependent_launch(column_sum_kernel, dim3(unsigned((n + 31) / 32)), 256, 0, stream, (const float*)workspace, bias_gradient, row_limit, (long long)rows, block_rows, int(n));
}

}  // extern "C"
