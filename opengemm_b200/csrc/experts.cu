// Host side of the experts' products and of the gradients of products: tile
// choice, tensor maps and the launch (experts.cuh has the kernel).
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <type_traits>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/opengemm_b200.h"
#include "dependent_launch.h"
#include "device_scope.h"
#include "experts_launch.h"
#include "launch_common.h"

namespace og {

extern const ExpertKernel EXPERT_FORWARD16[];
extern const int EXPERT_FORWARD16_COUNT;
extern const ExpertKernel EXPERT_FORWARD8[];
extern const int EXPERT_FORWARD8_COUNT;
extern const ExpertKernel EXPERT_GRADIENT[];
extern const int EXPERT_GRADIENT_COUNT;

namespace {

thread_local char experts_error[320];

int experts_fail(int code, const char* format, ...) {
  va_list args;
  va_start(args, format);
  vsnprintf(experts_error, sizeof experts_error, format, args);
  va_end(args);
  return code;
}

constexpr int XP_DEVICES = 64;
constexpr int XP_STATIC_SMEM = 9 * 1024;  // barriers and the group tables

// What a launch runs with, and its estimated cycles.
struct ExpertPlan {
  int cta_group, tile_n;
  double cost = 0;
};

constexpr ExpertPlan TILES[] = {{2, 256}, {1, 256}, {1, 128}, {1, 64}};

// The tile of a launch: the cheapest of a short menu by an estimate.
//
// With several groups only their number and the number of all rows are known
// here (the table of offsets is on the device): they are taken as equal, a
// group's last tile as half full, and the last wave of tiles as half idle.
// A tile costs its K blocks and some 2000 cycles (its first loads, its last store),
// but no less than storing it takes (16 experts with some 20 rows each, weights'
// gradient of 2608 x 2992: 64 us in tiles of 256, as long as clearing that memory
// takes, 86 us in pairs, 89 and 141 us in narrower ones).  A K block costs what
// fits 63 measured launches of 8 to 32 unevenly filled experts, 20 to 1500 rows
// each, best: pairs of CTAs share the N-side operand, which lets wide tiles run
// nearest the tensor pipe's rate (bf16 4096 x 8192 x 4096, rows' gradient: 190 us
// in pairs, 217 / 237 / 364 us in single CTAs 256 / 128 / 64 wide).  Where a
// group's rows fit one tile its weights are read from memory once and nothing else
// is: the block then costs the SM's share of the memory bandwidth, best used by
// tiles of 128 in the forward product (16 tokens x 8 of 64 experts, 2048 x 2048
// weights: 59 us; 65 us in pairs, 63 us 256 wide, 66 us 64 wide), of 256 in the
// rows' gradient (64 experts, three rows each: 84 us for 89).  Narrow tiles give
// every SM work when there are few.
//
// Measured with every tile (OgExpertProduct.tile) over 27 launches, 8 to 64 experts
// of 2 to 1670 rows: the choice is within 8 % of the best of the four in 19 of them.
// The others are experts of some 100 to 700 rows, where the last, half-filled tile
// counts most: the forward product and the rows' gradient take pairs where one CTA
// of 256 would do (4 x 300 and 4 x 700 rows, 2048 x 2048: rows' gradient 49 us for 36,
// forward 40 for 36; 16 x 100, 1536 x 3000: forward 58 for 45, rows' gradient 40 for
// 34), and the weights' gradient one CTA where a pair would (8 x 512, 2048 x 2048: 36
// us for 31.5): a single cost a block prices a pair's second CTA and its longer
// store alike.
// Gathered rows go to single CTAs: with the few rows an expert for which gathering
// pays, a pair's second CTA has none.
// With `parts` > 1 a single group's work is cut along its reduction into that
// many launches' worth of tiles.
ExpertPlan choose_plan(int mode, bool gather, bool glu, int groups, int rows, int m_out, int cols, int blocks_fixed, int sm_count, int parts = 1) {
  const int busy = std::max(1, std::min(groups, rows));
  const double rows_each = double(std::max(rows, 1)) / busy;
  static const int multiply_cycles[3][4] = {{740, 950, 560, 390}, {750, 1025, 615, 535}, {685, 725, 460, 290}};  // by mode
  static const int stream_cycles[2][4] = {{780, 1430, 680, 525}, {780, 1090, 680, 525}};
  static const int least_cycles[] = {9200, 4900, 2950, 2450};
  const int first = gather ? 1 : 0;
  ExpertPlan best = TILES[first];
  double best_cost = 0;
  for (int i = first; i < 4; ++i) {
    const ExpertPlan& c = TILES[i];
    const int out_n = glu ? c.tile_n / 2 : c.tile_n, tile_m = 128 * c.cta_group;
    const double m_tiles = mode == MODE_DW   ? ceil_div(m_out, tile_m)
                           : groups == 1     ? ceil_div(std::max(rows, 1), tile_m)
                                             : std::max(1.0, rows_each / tile_m + 0.5);
    const double tiles = double(parts) * (mode == MODE_DW ? groups : busy) * m_tiles * ceil_div(cols, out_n);
    const double blocks = (mode == MODE_DW ? std::max(1.0, rows_each / 64) : blocks_fixed) / parts;
    double block = mode != MODE_DW && rows_each <= tile_m ? stream_cycles[mode][i] : multiply_cycles[mode][i];
    if (mode != MODE_DW && c.cta_group == 2 && rows_each <= 128) block *= 1.22;  // the second CTA has no rows
    const double waves = tiles / (sm_count / c.cta_group);
    const double cost = (groups == 1 ? std::ceil(waves) : std::max(1.0, waves + 0.5)) * std::max(blocks * block + 2000, double(least_cycles[i]));
    if (i == first || cost < best_cost) best = c, best_cost = cost;
  }
  best.cost = best_cost;
  return best;
}

int experts_sm_count(int device) {
  static std::atomic<int> known[XP_DEVICES];
  int count = known[device].load(std::memory_order_relaxed);
  if (!count) {
    if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || count <= 0) count = 148;
    known[device].store(count, std::memory_order_relaxed);
  }
  return count;
}

const ExpertKernel* kernel_at(int index) {
  if (index < EXPERT_FORWARD16_COUNT) return &EXPERT_FORWARD16[index];
  index -= EXPERT_FORWARD16_COUNT;
  if (index < EXPERT_FORWARD8_COUNT) return &EXPERT_FORWARD8[index];
  index -= EXPERT_FORWARD8_COUNT;
  return index < EXPERT_GRADIENT_COUNT ? &EXPERT_GRADIENT[index] : nullptr;
}

const ExpertKernel* find_kernel(int kind, int cta_group, int mode, bool gather, bool glu, int out_bytes, int* index) {
  for (int i = 0; const ExpertKernel* k = kernel_at(i); ++i)
    if (k->kind == kind && k->cta_group == cta_group && k->mode == mode && k->gather == int(gather) && k->glu == int(glu) && k->out_bytes == out_bytes) {
      *index = i;
      return k;
    }
  return nullptr;
}

std::atomic<uint64_t> configured[XP_DEVICES];  // bit per kernel

int ensure_expert_kernel(const ExpertKernel& kernel, int index, int device) {
  if (configured[device].load(std::memory_order_acquire) >> index & 1) return OG_OK;
  const cudaError_t status = kernel.configure(SMEM_LIMIT - XP_STATIC_SMEM);
  if (status != cudaSuccess) return experts_fail(OG_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(status));
  configured[device].fetch_or(1ull << index, std::memory_order_release);
  return OG_OK;
}

// Parts that a plain product's gradient is cut into along its reduction: few
// tiles with many K blocks each leave most SMs idle, and a part more costs the
// float32 sums it writes and one short kernel that adds them (some 6000 cycles
// and the sums' bytes, twice, at 3400 a cycle).
int choose_parts(int mode, int m, int n, int k, int sm_count) {
  const int m_out = mode == MODE_DW ? n : m, blocks = ceil_div(mode == MODE_DW ? m : n, 64);
  int best = 1;
  double best_cost = 0;
  for (int parts = 1; parts <= 16 && parts * 4 <= std::max(4, blocks); parts *= 2) {
    const double sums = parts > 1 ? 6000 + double(parts) * m_out * k * 8 / 3400 : 0;
    const double cost = choose_plan(mode, false, false, 1, m, n, k, blocks, sm_count, parts).cost + sums;
    if (parts == 1 || cost < 0.9 * best_cost) best = parts, best_cost = cost;
  }
  return best;
}

// out = sum over `parts` of partial[part], rounded once; in the order of the parts.
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const float4* partial, T* out, long long vectors, int parts) {
  pdl_wait_prior_grids();
  pdl_launch_dependents();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= vectors) return;
  float4 sum = partial[i];
  for (int s = 1; s < parts; ++s) {
    const float4 v = partial[s * vectors + i];
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(out)[i] = sum;
  } else if constexpr (std::is_same<T, __half>::value) {
    reinterpret_cast<uint2*>(out)[i] = make_uint2(pack_f16x2(sum.x, sum.y), pack_f16x2(sum.z, sum.w));
  } else {
    reinterpret_cast<uint2*>(out)[i] = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
  }
}

template <typename T>
cudaError_t add_parts(const void* partial, void* out, long long values, int parts, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned((values / 4 + 255) / 256), 1, 1);
  config.blockDim = dim3(256, 1, 1);
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = dependent_launches();
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, add_parts_kernel<T>, static_cast<const float4*>(partial), static_cast<T*>(out), values / 4, parts);
}

// `parts` > 1 (MODE_DX and MODE_DW of one group): out is the float32 partial sums, one after another.
int launch_product(const OgExpertProduct& g, int device, void* stream, int parts = 1) {
  char why[256];
  const int mode = g.mode;
  if (mode < MODE_FORWARD || mode > MODE_DW) return experts_fail(OG_ERR_LAUNCH, "mode %d is none of 0..2", mode);
  const bool bf16 = !std::strncmp(g.dtype, "bf16", 16), f16 = !std::strncmp(g.dtype, "f16", 16), e4m3 = !std::strncmp(g.dtype, "e4m3", 16);
  if (!bf16 && !f16 && !(e4m3 && mode == MODE_FORWARD))
    return experts_fail(OG_ERR_LAUNCH, "dtype %.16s is not served: bf16, f16, and e4m3 for the forward product", g.dtype);
  if (g.groups < 1 || g.groups > XP_MAX_GROUPS) return experts_fail(OG_ERR_LAUNCH, "%d experts: 1 to %d are served", g.groups, XP_MAX_GROUPS);
  if (!g.offsets && g.groups != 1) return experts_fail(OG_ERR_LAUNCH, "%d experts without a table of their rows", g.groups);
  if (g.rows < 0 || g.n <= 0 || g.k <= 0) return experts_fail(OG_ERR_LAUNCH, "rows = %d, n = %d, k = %d", g.rows, g.n, g.k);
  const int elem = e4m3 ? 1 : 2, multiple = 16 / elem;
  if (g.k % multiple || (mode != MODE_FORWARD && g.n % multiple))
    return experts_fail(OG_ERR_LAUNCH, "n = %d, k = %d: rows must be multiples of 16 bytes", g.n, g.k);
  const bool glu = g.activation == ACT_SWIGLU || g.activation == ACT_GEGLU;
  if (g.activation < ACT_NONE || g.activation > ACT_GEGLU || (g.activation && mode != MODE_FORWARD))
    return experts_fail(OG_ERR_LAUNCH, "activation %d is not one of the forward product's", g.activation);
  if (glu && g.n % 16) return experts_fail(OG_ERR_LAUNCH, "a gated activation takes a multiple of 16 weight rows, got %d", g.n);
  if (g.out_f32 && mode == MODE_FORWARD) return experts_fail(OG_ERR_LAUNCH, "the forward product writes 16-bit values");
  const bool gather = g.tokens != nullptr;
  if (gather && mode != MODE_FORWARD) return experts_fail(OG_ERR_LAUNCH, "only the forward product gathers its rows");
  if (g.tile < 0 || g.tile > 4 || (gather && g.tile == 1)) return experts_fail(OG_ERR_LAUNCH, "tile %d is none of 0..4, or a pair for gathered rows", g.tile);
  if (device < 0 || device >= XP_DEVICES) return experts_fail(OG_ERR_LAUNCH, "device %d is out of range: this library serves devices 0..%d", device, XP_DEVICES - 1);
  const DeviceScope on(device);
  if (on.status() != cudaSuccess) return experts_fail(OG_ERR_LAUNCH, "cudaSetDevice(%d): %s", device, cudaGetErrorString(on.status()));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int out_bytes = g.out_f32 ? 4 : 2;
  if (g.rows == 0 || (gather && g.x_rows == 0)) {  // nothing to multiply: sums over no rows are zero
    if (mode == MODE_DW && cudaMemsetAsync(g.out, 0, size_t(g.groups) * g.n * g.k * out_bytes, s) != cudaSuccess)
      return experts_fail(OG_ERR_LAUNCH, "cudaMemsetAsync failed");
    return OG_OK;
  }
  if (!g.x || !g.w || !g.out) return experts_fail(OG_ERR_LAUNCH, "x, w and out must be device pointers, got null");
  if ((reinterpret_cast<uintptr_t>(g.x) | reinterpret_cast<uintptr_t>(g.w)) & 15)
    return experts_fail(OG_ERR_LAUNCH, "operands must start on 16-byte boundaries");

  ExpertParams p;
  std::memset(&p, 0, sizeof p);
  const int sm_count = experts_sm_count(device);
  p.groups = g.groups;
  p.rows = g.rows;
  p.glu_offset = glu ? g.n / 2 : 0;
  p.cols = mode == MODE_FORWARD ? (glu ? g.n / 2 : g.n) : g.k;
  p.m_out = g.n;
  p.k = mode == MODE_FORWARD ? g.k : g.n;
  p.block_k = 128 / elem;
  p.k_blocks = ceil_div(p.k, p.block_k);
  const ExpertPlan plan = g.tile ? TILES[g.tile - 1] : choose_plan(mode, gather, glu, g.groups, g.rows, p.m_out, p.cols, p.k_blocks, sm_count, parts);
  p.rows_per_group = g.rows;
  if (parts > 1) {
    if (mode == MODE_DW) {
      p.rows_per_group = ceil_div(ceil_div(g.rows, 64), parts) * 64;
      p.groups = ceil_div(g.rows, p.rows_per_group);
    } else {
      p.split_blocks = ceil_div(p.k_blocks, parts);
      p.groups = ceil_div(p.k_blocks, p.split_blocks);
    }
  }
  p.tile_n = plan.tile_n;
  p.out_tile_n = glu ? plan.tile_n / 2 : plan.tile_n;
  p.tiles_n = ceil_div(p.cols, p.out_tile_n);
  p.tiles_m_fixed = ceil_div(p.m_out, 128 * plan.cta_group);
  p.band = 8;
  const int y_rows = plan.tile_n / plan.cta_group;  // of the N side, per CTA: a multiple of 64
  p.y_bytes = y_rows * 128;
  p.stage_bytes = 16384 + p.y_bytes;
  p.stages = std::min(XP_MAX_STAGES, (SMEM_LIMIT - XP_STATIC_SMEM - 1024 - xp_staging_bytes(out_bytes)) / p.stage_bytes);
  p.tmem_cols = pow2_at_least(2 * plan.tile_n);
  const uint32_t x_columns = mode == MODE_DW, y_columns = mode != MODE_FORWARD;
  const uint32_t fmt = bf16 ? 1u : 0u;  // e4m3 is code 0 of its kind, f16 of its own
  p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (x_columns << 15) | (y_columns << 16) | (uint32_t(plan.tile_n >> 3) << 17) |
            (uint32_t(128 * plan.cta_group >> 4) << 24);
  p.offsets = g.offsets;
  p.tokens = g.tokens;
  p.alpha = g.alpha;
  p.factor = g.factor;
  p.beside = g.beside_previous != 0;
  p.d = g.out;
  p.preact = g.preactivation;
  p.wait_limit_ns = current_wait_limit_ns();
  p.ldd = p.cols;
  p.ldz = g.n;
  p.out_f16 = f16 && !g.out_f32;
  p.vec_ok = ((reinterpret_cast<uintptr_t>(g.out) | reinterpret_cast<uintptr_t>(g.preactivation)) & 15) == 0 && (int64_t(p.cols) * out_bytes) % 16 == 0;
  act_constants(g.activation, &p.act_shape, &p.act_a, &p.act_b);

  const int type = e4m3 ? int(CU_TENSOR_MAP_DATA_TYPE_UINT8) : bf16 ? int(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16) : int(CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
  const CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B;
  const uint32_t box = uint32_t(p.block_k);
  const uint64_t k = uint64_t(g.k), n = uint64_t(g.n), x_rows = uint64_t(gather ? g.x_rows : g.rows);
  int rc = OG_OK;
  auto map = [&](CUtensorMap* out, const void* base, uint64_t inner, uint64_t rows, uint32_t box1, const char* which, uint64_t matrices = 0) {
    if (rc == OG_OK) rc = encode_2d(out, base, type, inner, rows, inner * elem, box, box1, swizzle, 2, which, why, sizeof why, matrices);
  };
  if (mode == MODE_DW) {  // dz [rows, n] against x [rows, k], both along their rows
    map(&p.map_x, g.x, n, uint64_t(g.rows), 64, "the output's gradient");
    map(&p.map_y, g.w, k, x_rows, 64, "the rows");
  } else {
    const uint64_t inner = mode == MODE_FORWARD ? k : n;
    map(&p.map_x, g.x, inner, x_rows, 128, "the rows");
    map(&p.map_x32, g.x, inner, x_rows, gather ? 1 : 32, "the rows");
    const uint32_t box_rows = mode == MODE_DX ? 64 : uint32_t(glu ? plan.tile_n / 2 : y_rows);
    map(&p.map_y, g.w, k, n, box_rows, "the weights", uint64_t(g.groups));
  }
  const int64_t out_rows = mode == MODE_DW ? int64_t(p.groups) * g.n : p.split_blocks ? int64_t(p.groups) * g.rows : int64_t(g.rows);
  p.direct = p.vec_ok && out_rows <= 0x7FFFFFFF;
  if (p.direct && rc == OG_OK) {  // swizzled as the epilogue's staging buffers are
    const int out_type = g.out_f32 ? int(CU_TENSOR_MAP_DATA_TYPE_FLOAT32) : f16 ? int(CU_TENSOR_MAP_DATA_TYPE_FLOAT16) : int(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
    rc = encode_2d(&p.map_d, g.out, out_type, uint64_t(p.cols), uint64_t(out_rows), uint64_t(p.cols) * out_bytes, XP_CHUNK, 32,
                   g.out_f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, 0, "the output", why, sizeof why);
  }
  if (rc != OG_OK) return experts_fail(rc, "%s", why);

  int index = 0;
  const ExpertKernel* kernel = find_kernel(e4m3 ? KIND_F8F6F4 : KIND_F16, plan.cta_group, mode, gather, glu, out_bytes, &index);
  if (!kernel) return experts_fail(OG_ERR_NO_KERNEL, "no kernel for this product");
  if (const int bad = ensure_expert_kernel(*kernel, index, device)) return bad;
  // At most this many tiles: every group may end in a partial one.
  const int64_t m_tiles = mode == MODE_DW ? int64_t(p.groups) * p.tiles_m_fixed
                                          : (int64_t(g.rows) / (128 * plan.cta_group) + std::min(g.groups, g.rows)) * parts;
  const int clusters = int(std::min<int64_t>(sm_count / plan.cta_group, m_tiles * p.tiles_n));
  const int smem = p.stages * p.stage_bytes + xp_staging_bytes(out_bytes) + 1024;
  const cudaError_t launched = kernel->launch(p, std::max(1, clusters) * plan.cta_group, smem, s);
  if (launched != cudaSuccess) return experts_fail(OG_ERR_LAUNCH, "kernel launch failed: %s", cudaGetErrorString(launched));
  return OG_OK;
}

}  // namespace

// For og_b200_prepare_device, with the device current.
const char* prepare_experts(int device) {
  for (int i = 0; const ExpertKernel* k = kernel_at(i); ++i)
    if (ensure_expert_kernel(*k, i, device) != OG_OK) return experts_error;
  return nullptr;
}

}  // namespace og

using namespace og;

extern "C" {

OG_API const char* og_b200_experts_error(void) { return experts_error; }

// A workspace's parts: dz, the bias's partial sums, the products' partial sums
// (one product after another uses them).  Each starts on a 16-byte boundary.
struct GradientSpace {
  int64_t dz, bias, sums;  // bytes
  int parts_a, parts_b;
};

static GradientSpace gradient_space(const OgGemmGradients& g, int device) {
  GradientSpace s{};
  auto up = [](int64_t bytes) { return (bytes + 15) / 16 * 16; };
  const int sm_count = device >= 0 && device < XP_DEVICES ? experts_sm_count(device) : 148;
  s.parts_a = g.grad_a && g.m ? choose_parts(MODE_DX, g.m, g.n, g.k, sm_count) : 1;
  s.parts_b = g.grad_b && g.m ? choose_parts(MODE_DW, g.m, g.n, g.k, sm_count) : 1;
  if (g.activation) s.dz = up(int64_t(g.m) * g.n * 2);
  if (g.grad_bias) s.bias = up(int64_t(ceil_div(g.m, gradient_block_rows(g.m, g.n))) * g.n * 4);
  if (s.parts_a > 1) s.sums = up(int64_t(s.parts_a) * g.m * g.k * 4);
  if (s.parts_b > 1) s.sums = std::max(s.sums, up(int64_t(s.parts_b) * g.n * g.k * 4));
  return s;
}

static int check_gradients(const OgGemmGradients& g) {
  if (std::strncmp(g.dtype, "bf16", 16) && std::strncmp(g.dtype, "f16", 16)) return experts_fail(OG_ERR_LAUNCH, "dtype %.16s is not served: bf16 and f16", g.dtype);
  if (g.activation < ACT_NONE || g.activation > ACT_SILU) return experts_fail(OG_ERR_LAUNCH, "activation %d is none of 0..%d", g.activation, int(ACT_SILU));
  if (g.m < 0 || g.n <= 0 || g.k <= 0 || g.n % 8 || g.k % 8) return experts_fail(OG_ERR_LAUNCH, "m = %d, n = %d, k = %d: n and k come in eights", g.m, g.n, g.k);
  return OG_OK;
}

OG_API int64_t og_b200_gemm_gradients_workspace(const OgGemmGradients* g, int32_t device) {
  if (!g) return experts_fail(OG_ERR_LAUNCH, "null OgGemmGradients");
  if (const int rc = check_gradients(*g)) return rc;
  const GradientSpace s = gradient_space(*g, device);
  return s.dz + s.bias + s.sums;
}

OG_API int32_t og_b200_gemm_gradients(const OgGemmGradients* g, int32_t device, void* stream) {
  if (!g) return experts_fail(OG_ERR_LAUNCH, "null OgGemmGradients");
  if (const int rc = check_gradients(*g)) return rc;
  const bool bf16 = !std::strncmp(g->dtype, "bf16", 16);
  if ((reinterpret_cast<uintptr_t>(g->grad_a) | reinterpret_cast<uintptr_t>(g->grad_b)) & 15)
    return experts_fail(OG_ERR_LAUNCH, "gradients must start on 16-byte boundaries");
  const GradientSpace s = gradient_space(*g, device);
  if (s.dz + s.bias + s.sums > 0 && (!g->workspace || (reinterpret_cast<uintptr_t>(g->workspace) & 15) || g->workspace_bytes < s.dz + s.bias + s.sums))
    return experts_fail(OG_ERR_LAUNCH, "these gradients take a 16-byte aligned workspace of %lld bytes, got %lld", (long long)(s.dz + s.bias + s.sums), (long long)g->workspace_bytes);
  const DeviceScope on(device);
  if (on.status() != cudaSuccess) return experts_fail(OG_ERR_LAUNCH, "cudaSetDevice(%d): %s", device, cudaGetErrorString(on.status()));
  uint8_t* const dz = static_cast<uint8_t*>(g->workspace);
  float* const bias_sums = reinterpret_cast<float*>(dz + s.dz);
  uint8_t* const sums = dz + s.dz + s.bias;
  if (g->activation || g->grad_bias) {
    const int rc = og_b200_activation_gradient(bf16 ? 1 : 2, g->activation, g->grad, g->z, dz, g->grad_bias, bias_sums, nullptr, g->m, g->n, device, stream);
    if (rc != OG_OK) return experts_fail(rc, "%s", og_b200_routing_error());
  }
  OgExpertProduct product;
  std::memset(&product, 0, sizeof product);
  product.x = g->activation ? dz : g->grad;
  product.groups = 1, product.rows = g->m, product.n = g->n, product.k = g->k, product.factor = g->factor;
  std::memcpy(product.dtype, g->dtype, sizeof product.dtype);
  for (int mode = MODE_DX; mode <= MODE_DW; ++mode) {
    void* const out = mode == MODE_DX ? g->grad_a : g->grad_b;
    if (!out) continue;
    const int parts = mode == MODE_DX ? s.parts_a : s.parts_b;
    product.mode = mode, product.w = mode == MODE_DX ? g->b : g->a;
    product.out = parts > 1 ? sums : out, product.out_f32 = parts > 1 ? 1 : g->out_f32;
    // The second product reads nothing of the first's, unless they share the partial sums' space.
    product.beside_previous = mode == MODE_DW && g->grad_a && s.parts_a == 1;
    int rc = launch_product(product, device, stream, parts);
    if (rc != OG_OK) return rc;
    if (parts == 1) continue;
    // as many parts as have K blocks
    const int blocks = ceil_div(mode == MODE_DX ? g->n : g->m, 64), live = ceil_div(blocks, ceil_div(blocks, parts));
    const long long values = (long long)(mode == MODE_DX ? g->m : g->n) * g->k;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t launched = g->out_f32 ? add_parts<float>(sums, out, values, live, st)
                                 : bf16     ? add_parts<__nv_bfloat16>(sums, out, values, live, st)
                                            : add_parts<__half>(sums, out, values, live, st);
    if (launched != cudaSuccess) return experts_fail(OG_ERR_LAUNCH, "kernel launch failed: %s", cudaGetErrorString(launched));
  }
  return OG_OK;
}

OG_API int32_t og_b200_expert_product(const OgExpertProduct* product, int32_t device, void* stream) {
  if (!product) return experts_fail(OG_ERR_LAUNCH, "null OgExpertProduct");
  return launch_product(*product, device, stream);
}

}  // extern "C"
