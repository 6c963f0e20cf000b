// The fused product for up to four rows of A (decoding steps) and 16-bit
// operands: C = act(alpha A.B^T + bias) + residual with plain arithmetic.
//
// Such a product reads B once and computes next to nothing: 134 MB against 67
// million multiply-adds a row at N = K = 8192.  The tiled kernel gives B's rows
// to its MMA in pieces of 128, which leaves 64 tiles for 148 SMs at N = 8192 and
// a whole accumulator to drain at the end.  Here every SM has one block and an
// equal run of B's rows; the block's eight warps cut K between them, take the
// rows in fours and keep the next four rows' 16-byte loads in flight while they
// work on the current ones.  A stays in L1.  Their partial sums meet in shared
// memory, where one thread finishes each value of C.
//
// From five rows of A on the multiply-adds, not the bytes, would set the time.
#include <algorithm>
#include <cstdint>

#include <cuda_runtime.h>

#include "activation.cuh"
#include "launch_common.h"
#include "skinny.h"

namespace og {
namespace {

constexpr int SKINNY_WARPS = 8;
constexpr int SKINNY_ROWS = 4;    // of B at a time
constexpr int SKINNY_DEEP = 4;    // 16-byte vectors of each, per lane
constexpr int SKINNY_ROUND = 128; // rows of B between two reductions

struct SkinnyParams {
  const void* a;
  const void* b;
  const float* bias;
  const void* residual;
  void* preact;
  void* c;
  int n, k, out;  // out: OutType
  float alpha;
  int act_shape;
  float act_a, act_b;
  int pdl;
};

// Two 16-bit floats of a word.
template <bool BF16>
__device__ __forceinline__ void widen2(uint32_t w, float& lo, float& hi) {
  if constexpr (BF16) {
    lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    lo = half_bits_to_float(w), hi = half_bits_to_float(w >> 16);
  }
}

// Read once: no place in L1, which A keeps.  Not a read-only (.nc) load: the
// block may have started while an earlier kernel was still writing B, and such a
// load asks for memory that nobody writes as long as this kernel runs.
__device__ __forceinline__ uint4 load_streamed(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ float load_value(const void* base, size_t at, int out) {
  if (out == OUT_F32) return static_cast<const float*>(base)[at];
  const uint32_t bits = static_cast<const uint16_t*>(base)[at];
  return out == OUT_F16 ? half_bits_to_float(bits) : __uint_as_float(bits << 16);
}
__device__ __forceinline__ void store_value(void* base, size_t at, int out, float v) {
  if (out == OUT_F32) static_cast<float*>(base)[at] = v;
  else static_cast<uint16_t*>(base)[at] = uint16_t((out == OUT_F16 ? pack_f16x2(v, 0.0f) : pack_bf16x2(v, 0.0f)) & 0xFFFFu);
}

template <bool BF16, int M>
__global__ void __launch_bounds__(SKINNY_WARPS * 32) skinny_kernel(const SkinnyParams p) {
  constexpr int ROWS = SKINNY_ROWS, DEEP = SKINNY_DEEP;
  __shared__ float partial[SKINNY_ROUND * M][SKINNY_WARPS + 1];
  if (p.pdl) {
    pdl_launch_dependents();
    pdl_wait_prior_grids();
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_begin = int((long long)p.n * blockIdx.x / gridDim.x), row_end = int((long long)p.n * (blockIdx.x + 1) / gridDim.x);
  const int vectors = p.k / 8;
  const int v_begin = int((long long)vectors * warp / SKINNY_WARPS) + lane, v_end = int((long long)vectors * (warp + 1) / SKINNY_WARPS);
  const uint4* const a = static_cast<const uint4*>(p.a);
  const uint4* const b = static_cast<const uint4*>(p.b);
  const int chunks = max(1, (v_end - (v_begin - lane) + 32 * DEEP - 1) / (32 * DEEP));
  float sum[ROWS][M];
  // One piece of work: ROWS rows from `row` on, 32 * DEEP vectors from chunk `c` on.
  auto load = [&](int row, int c, uint4 (&q)[DEEP][ROWS]) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int v = v_begin + (c * DEEP + d) * 32;
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        q[d][r] = v < v_end ? load_streamed(b + size_t(min(row + r, row_end - 1)) * vectors + v) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  auto add = [&](int c, const uint4 (&q)[DEEP][ROWS]) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int v = v_begin + (c * DEEP + d) * 32;
      if (v >= v_end) break;
      float x[M][8];
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const uint4 w = a[size_t(m) * vectors + v];
        widen2<BF16>(w.x, x[m][0], x[m][1]), widen2<BF16>(w.y, x[m][2], x[m][3]);
        widen2<BF16>(w.z, x[m][4], x[m][5]), widen2<BF16>(w.w, x[m][6], x[m][7]);
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        float y[8];
        widen2<BF16>(q[d][r].x, y[0], y[1]), widen2<BF16>(q[d][r].y, y[2], y[3]);
        widen2<BF16>(q[d][r].z, y[4], y[5]), widen2<BF16>(q[d][r].w, y[6], y[7]);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[r][m] = fmaf(x[m][j], y[j], sum[r][m]);
      }
    }
  };
  auto clear = [&] {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int m = 0; m < M; ++m) sum[r][m] = 0.0f;
  };
  // After the last chunk of four rows: their sums over the warp to shared memory.
  auto publish = [&](int local) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float v = sum[r][m];
#pragma unroll
        for (int d = 16; d; d /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
        if (lane == 0) partial[(local + r) * M + m][warp] = v;
      }
  };
  for (int round = row_begin; round < row_end; round += SKINNY_ROUND) {
    const int round_end = min(round + SKINNY_ROUND, row_end);
    uint4 now[DEEP][ROWS], soon[DEEP][ROWS];
    int row = round, c = 0;
    load(row, c, now);
    clear();
    while (true) {
      int next_row = row, next_c = c + 1;
      if (next_c == chunks) next_row += ROWS, next_c = 0;
      const bool more = next_row < round_end;
      if (more) load(next_row, next_c, soon);
      add(c, now);
      if (next_c == 0) {
        publish(row - round);
        clear();
      }
      if (!more) break;
#pragma unroll
      for (int d = 0; d < DEEP; ++d)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) now[d][r] = soon[d][r];
      row = next_row, c = next_c;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (round_end - round) * M; i += SKINNY_WARPS * 32) {
      // value i: row m = i % M of A, row col of B
      const int m = i % M, col = round + i / M;
      float z = 0.0f;
#pragma unroll
      for (int w = 0; w < SKINNY_WARPS; ++w) z += partial[i][w];
      const size_t at = size_t(m) * p.n + col;
      z *= p.alpha;
      if (p.bias) z += p.bias[col];
      if (p.preact) store_value(p.preact, at, p.out, z);
      if (p.act_shape == SHAPE_SIGMOID) z = act_value<SHAPE_SIGMOID>(z, p.act_a, p.act_b);
      else if (p.act_shape == SHAPE_PHI) z = act_value<SHAPE_PHI>(z, 0.f, 0.f);
      else if (p.act_shape == SHAPE_RELU) z = act_value<SHAPE_RELU>(z, 0.f, 0.f);
      if (p.residual) z += load_value(p.residual, at, p.out);
      store_value(p.c, at, p.out, z);
    }
    __syncthreads();
  }
}

template <bool BF16>
auto pick_kernel(int m) {
  return m == 1 ? skinny_kernel<BF16, 1> : m == 2 ? skinny_kernel<BF16, 2> : m == 3 ? skinny_kernel<BF16, 3> : skinny_kernel<BF16, 4>;
}

}  // namespace

bool skinny_serves(const OgGemm& g, const Format& f, const LaunchPointers& io) {
  return g.m <= SKINNY_MAX_M && f.kind == KIND_F16 && !io.out_quant && ((reinterpret_cast<uintptr_t>(io.a) | reinterpret_cast<uintptr_t>(io.b)) & 15) == 0;
}

cudaError_t launch_skinny(const OgGemm& g, const Format& f, const LaunchPointers& io, const float* alpha, bool pdl, int sm_count, cudaStream_t stream) {
  SkinnyParams p{};
  p.a = io.a, p.b = io.b, p.bias = static_cast<const float*>(io.bias), p.residual = io.residual, p.preact = io.preact, p.c = io.c;
  p.n = g.n, p.k = g.k, p.out = f.out, p.alpha = alpha ? *alpha : 1.0f, p.pdl = pdl;
  act_constants(io.activation, &p.act_shape, &p.act_a, &p.act_b);
  const bool bf16 = element(f.a)->format == 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(std::min(sm_count, ceil_div(g.n, SKINNY_ROWS))), 1, 1);
  config.blockDim = dim3(SKINNY_WARPS * 32, 1, 1);
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = pdl ? 1 : 0;
  const auto kernel = bf16 ? pick_kernel<true>(g.m) : pick_kernel<false>(g.m);
  return cudaLaunchKernelEx(&config, kernel, p);
}

}  // namespace og
