// One persistent, warp-specialised tcgen05 kernel for products whose rows fall
// into groups, each group with its own matrix (experts), and for the gradients
// of such a product.  A single group without an offset table is the plain
// matrix product, which makes it the kernel of gemm's gradients too.
//
//   MODE_FORWARD  out[r, :]    = act(alpha_e * x[r, :] . w_e^T)      r in expert e's rows
//   MODE_DX       out[r, :]    = dz[r, :] . w_e
//   MODE_DW       out[e, :, :] = sum over e's rows r of dz[r, :]^T x[r, :]
//
// The MMA reduces along the innermost (contiguous) extent of both operands in
// the forward product; the gradients reduce along a row extent instead.  The
// 16-bit MMA reads such an operand as it lies: a stage then holds boxes of 64
// reduction rows x 64 columns (128 bytes, swizzled), and the matrix
// descriptor says that the columns, not the reduction, are contiguous.  So no
// operand is transposed through memory.
//
// Rows of a group may start anywhere (offsets come from a table on the device;
// the host never sees them): tiles start at the group's first row, rows past
// its end are computed from whatever lies there and not stored.  Only the
// weight gradient, which sums over rows, has to cut its last block of 64 rows
// short: a warp of its own waits for that stage's data and clears the rows past
// the end in shared memory before the MMA reads it.
//
// Roles as in kernel.cuh: warp 0 loads (one thread; all lanes when rows are
// gathered, four rows a lane and instruction), warp 1 issues the MMAs, warps
// 2-9 store, warp 10 is the weight gradient's.  Every wait is bounded.
//
// What bounds it: with many rows the tensor pipe, under the power limit (bf16, 8
// experts of 960 rows, 4096 x 4096: 200 us, 88-93 % active).  With a few hundred
// rows an expert the ring of stages: a K block moves 32 KB a CTA in pairs, 48 KB
// in a CTA of 128 x 256, against 512 cycles of MMAs, and memory or L2 is over a
// microsecond away (8 experts of 512 rows, weights' gradient 2048 x 2048: 31 us in
// pairs with six stages, 36 us with four of the larger ones, which the estimate of
// experts.cu takes there).  Every stage counts:
// staging two chunks of output a warp, for whole 128-byte lines, takes one and was
// slower (36 -> 39 us), and asking for the weights a few blocks ahead in L2 costs
// the copy engine as much as loading them (35 -> 38 us in the rows' product, 34 ->
// 45 us with eight rows an expert).  Whole slabs of 32 output rows leave by that
// engine too, straight from the staging buffer, which is swizzled as its map says:
// 37 -> 36 us there, and 53 -> 45 us where a tile is one load and one store (16
// experts, 256 rows each); rows by threads where a group ends.
#pragma once

#include "activation.cuh"
#include "ptx.cuh"

namespace og {

enum ExpertMode : int { MODE_FORWARD = 0, MODE_DX = 1, MODE_DW = 2 };

constexpr int XP_MAX_STAGES = 12;
constexpr int XP_MAX_GROUPS = 1024;
constexpr int XP_CHUNK = 32;  // columns an epilogue warp works on at a time

// Two epilogue warps per quarter of the accumulator's rows, taking turns at its
// columns: a weight gradient over few rows is all stores.
constexpr int XP_EPILOGUE_WARPS = 8;
constexpr int xp_staging_bytes(int out_bytes) { return XP_EPILOGUE_WARPS * 32 * XP_CHUNK * out_bytes; }  // each warp's 32 rows of a chunk
__host__ __device__ constexpr int xp_threads(int mode) { return 64 + 32 * XP_EPILOGUE_WARPS + (mode == MODE_DW ? 32 : 0); }

struct alignas(64) ExpertParams {
  CUtensorMap map_x;    // MMA-M side, boxes of 128 rows (64 x 64 in MODE_DW)
  CUtensorMap map_x32;  // the same in boxes of 32 rows, for a group's last, short tile; gathered: of one row
  CUtensorMap map_y;    // MMA-N side
  CUtensorMap map_d;    // output, boxes of 32 rows x XP_CHUNK columns (`direct` only)
  const int* offsets;   // [groups + 1] first row of each group; null: one group of all rows
  const int* tokens;    // gathered operand: its row for each sorted row
  const float* alpha;   // [groups], or null
  float factor;         // on every sum, beside alpha
  void* d;
  void* preact;
  unsigned long long wait_limit_ns;
  int groups, rows;
  int rows_per_group;   // without offsets: rows of each group but the last (MODE_DW cut along its rows)
  int split_blocks;     // MODE_DX of one group cut along its reduction: K blocks of each part, which is then
                        // a "group" with all rows; 0 otherwise
  int cols;             // output columns
  int m_out;            // MODE_DW: output rows of each group
  int k;                // reduction extent (MODE_DW: the group's rows)
  int k_blocks, block_k;
  int tile_n, out_tile_n, tiles_n, tiles_m_fixed;  // tiles_m_fixed: MODE_DW
  int glu_offset;       // first row of the up half of the weights; 0 without a gate
  int stages, stage_bytes, y_bytes;
  unsigned idesc;
  int band;             // M tiles per band of the tile order
  int ldd, ldz;         // elements per row of `d` and `preact`
  int vec_ok;           // rows of d and preact take 16-byte stores
  int direct;           // whole slabs of 32 output rows leave by TMA
  int act_shape;
  float act_a, act_b;
  int out_f16;
  int tmem_cols;
  int beside;           // runs beside the stream's previous launch (see below)
};

// One tile of work: group, its rows, and the tile's place.
struct ExpertTile {
  int group, first_row, rows;  // rows of the group
  int mi, ni;
  int k0;  // first K block
};

// Gathered rows: four rows of `tmap` (one-row boxes) into 512 consecutive bytes.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const void* tmap, int x, int r0, int r1, int r2, int r3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(tmap), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
      : "memory");
}

template <int CTA_GROUP>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, int x, int y, int z, uint32_t bar) {
  if constexpr (CTA_GROUP == 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// Operand whose columns (the M or N extent) are contiguous: 128-byte swizzled
// boxes of 64 columns x 64 reduction rows, 8 KiB each.  Leading offset: from
// one box of 64 columns to the next; stride offset: eight reduction rows on.
__device__ __forceinline__ uint64_t column_operand_desc(uint32_t smem_addr) {
  return uint64_t((smem_addr & 0x3FFFFu) >> 4) | (uint64_t(8192 >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// GATHER and GLU: MODE_FORWARD only; GATHER: single CTAs only.
template <int KIND, int CTA_GROUP, int MODE, bool GATHER, bool GLU, int OUT_BYTES>
__global__ void __launch_bounds__(xp_threads(MODE), 1) expert_kernel(const __grid_constant__ ExpertParams p) {
  static_assert(!GATHER || (MODE == MODE_FORWARD && CTA_GROUP == 1));
  constexpr int TILE_M = 128 * CTA_GROUP;
  constexpr bool X_COLUMNS = MODE == MODE_DW, Y_COLUMNS = MODE != MODE_FORWARD;
  constexpr int CHUNK = XP_CHUNK, ROW_BYTES = CHUNK * OUT_BYTES, UNITS = ROW_BYTES / 16, UNIT = 16 / OUT_BYTES;
  constexpr int ROWS_AT_ONCE = 32 / UNITS, STEPS = 32 / ROWS_AT_ONCE;

  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t bars[4 * XP_MAX_STAGES + 5];
  __shared__ int group_row[XP_MAX_GROUPS + 1];   // first row of each group
  __shared__ int group_tile[XP_MAX_GROUPS + 1];  // first tile of each group
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CTA_GROUP == 2 ? cluster_cta_rank() : 0u;
  const int cluster_id = blockIdx.x / CTA_GROUP, num_clusters = gridDim.x / CTA_GROUP;
  const uint32_t ring = (smem_u32(dyn_smem) + 1023u) & ~1023u;
  const uint32_t staging = ring + p.stages * p.stage_bytes;
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * XP_MAX_STAGES;
  const uint32_t bar_ready = bar_empty + 8 * XP_MAX_STAGES;  // MODE_DW: a short block's rows past the end are cleared
  const uint32_t bar_go = bar_ready + 8 * XP_MAX_STAGES;     // MODE_DW, a short block: asked for (leader), landed (pair's second CTA)
  const uint32_t bar_acc_full = bar_go + 8 * XP_MAX_STAGES, bar_acc_empty = bar_acc_full + 16;
  const uint32_t bar_tmem = bar_acc_empty + 16;
  const WaitCtx ctx{&abort_flag, nullptr, p.wait_limit_ns};

  if (threadIdx.x == 0) {
    prefetch_tmap(&p.map_x);
    prefetch_tmap(&p.map_y);
    if (MODE == MODE_FORWARD) prefetch_tmap(&p.map_x32);
    if (p.direct) prefetch_tmap(&p.map_d);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
      mbar_init(bar_ready + 8 * s, CTA_GROUP);
      mbar_init(bar_go + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_acc_full + 8 * s, 1);
      mbar_init(bar_acc_empty + 8 * s, XP_EPILOGUE_WARPS * CTA_GROUP);
    }
    mbar_init(bar_tmem, CTA_GROUP);
    abort_flag = 0;
    mbar_init_fence();
  }
  __syncthreads();
  if (CTA_GROUP == 2) cluster_sync_all();
  if (warp == 1) {
    tmem_alloc<CTA_GROUP>(smem_u32(&tmem_slot), p.tmem_cols);
    tmem_relinquish<CTA_GROUP>();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(bar_tmem);
      if constexpr (CTA_GROUP == 2) mbar_arrive_cluster(map_to_cta(bar_tmem, rank ^ 1u));
    }
  }
  // The offsets are an earlier kernel's output, like everything else read here.
  //
  // `beside`: the stream's previous launch is such a kernel too, and writes
  // nothing that this one touches.  Its blocks let this grid start only after
  // their own wait has returned, so whatever came before it is complete: this
  // grid need not wait, and fills the SMs that the other's last wave leaves
  // idle.  It waits before it ends, so that completion stays transitive.
  if (!p.beside) pdl_wait_prior_grids();
  if (threadIdx.x == 0) pdl_launch_dependents();

  // Group table: rows and tiles before each group.  Warp 2 sums; a lane takes a
  // contiguous run of groups.
  const int groups = p.groups;
  for (int i = threadIdx.x; i <= groups; i += xp_threads(MODE)) group_row[i] = p.offsets ? p.offsets[i] : min(i * p.rows_per_group, p.rows);
  __syncthreads();
  if (warp == 2) {
    auto tiles_of = [&](int e) {
      const int rows = MODE == MODE_DX && p.split_blocks ? p.rows : group_row[e + 1] - group_row[e];
      const int m_tiles = MODE == MODE_DW ? p.tiles_m_fixed : (rows + TILE_M - 1) / TILE_M;
      return m_tiles * p.tiles_n;
    };
    const int per = (groups + 31) / 32, first = min(lane * per, groups), last = min(first + per, groups);
    int sum = 0;
    for (int e = first; e < last; ++e) sum += tiles_of(e);
    int before = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(0xFFFFFFFFu, before, d);
      if (lane >= d) before += other;
    }
    before -= sum;
    for (int e = first; e < last; ++e) {
      group_tile[e] = before;
      before += tiles_of(e);
    }
    if (lane == 31) group_tile[groups] = before;
  }
  __syncthreads();
  const int num_tiles = group_tile[groups];

  // Tile t: the last group that starts at or before it (empty groups share
  // their successor's start), then bands of `band` M tiles, M fastest inside a
  // band, so that tiles running together share weights and rows in L2.
  auto find_tile = [&](int t, ExpertTile& w) {
    int lo = 0, hi = groups;  // group_tile[lo] <= t < group_tile[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (group_tile[mid] <= t) lo = mid; else hi = mid;
    }
    w.group = lo;
    w.first_row = group_row[lo];
    w.rows = group_row[lo + 1] - w.first_row;
    w.k0 = 0;
    if (MODE == MODE_DX && p.split_blocks) w.first_row = 0, w.rows = p.rows, w.k0 = lo * p.split_blocks;
    const int m_tiles = MODE == MODE_DW ? p.tiles_m_fixed : (w.rows + TILE_M - 1) / TILE_M;
    const int local = t - group_tile[lo];
    const int band = local / (p.band * p.tiles_n);
    const int height = min(p.band, m_tiles - band * p.band);
    const int rest = local - band * p.band * p.tiles_n;
    w.ni = rest / height;
    w.mi = band * p.band + rest - w.ni * height;
  };
  auto k_blocks_of = [&](const ExpertTile& w) {
    if (MODE == MODE_DW) return (w.rows + 63) / 64;
    return MODE == MODE_DX && p.split_blocks ? min(p.split_blocks, p.k_blocks - w.k0) : p.k_blocks;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (GATHER || elect_one()) {
      const int stages = p.stages, block_k = p.block_k, tile_n = p.tile_n;
      const uint32_t stage_bytes = p.stage_bytes, y_bytes = p.y_bytes;
      const int y_rows = tile_n / CTA_GROUP;       // MMA-N rows this CTA loads
      const int y_boxes = y_rows / 64;             // column boxes of a Y_COLUMNS operand
      const bool leads = !GATHER || lane == 0;     // the one thread that credits bytes and loads whole boxes
      int stage = 0;
      uint32_t phase = 0, issued = 0;
      bool ok = true;
      for (int t = cluster_id; ok && t < num_tiles; t += num_clusters) {
        ExpertTile w;
        find_tile(t, w);
        const int blocks = k_blocks_of(w);
        const int left = w.rows - w.mi * TILE_M;   // rows of the group from this tile on
        const int x_row = w.first_row + w.mi * TILE_M + int(rank) * 128;
        // Rows of the M side that each CTA of the pair loads, in pieces of 32 (gathered: 4).
        int mine = 128, whole = 128 * CTA_GROUP;
        if constexpr (MODE != MODE_DW) {
          constexpr int PIECE = GATHER ? 4 : 32;
          const int l0 = min(max(left, 0), 128), l1 = CTA_GROUP == 2 ? min(max(left - 128, 0), 128) : 0;
          const int p0 = (l0 + PIECE - 1) / PIECE * PIECE, p1 = (l1 + PIECE - 1) / PIECE * PIECE;
          mine = rank == 0 ? p0 : p1;
          whole = p0 + p1;
        }
        const uint32_t tx = uint32_t(whole) * 128 + CTA_GROUP * y_bytes;
        int token[4];
        if constexpr (GATHER) {
#pragma unroll
          for (int i = 0; i < 4; ++i)  // rows past the group's end repeat its last row
            token[i] = 4 * lane < mine ? p.tokens[min(x_row + 4 * lane + i, w.first_row + w.rows - 1)] : 0;
        }
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1, ctx, SITE_PRODUCER_EMPTY)) {
            ok = false;
            break;
          }
          const uint32_t full_local = bar_full + 8 * stage;
          const uint32_t full = CTA_GROUP == 2 ? map_to_cta(full_local, 0) : full_local;
          const uint32_t sx = ring + stage * stage_bytes, sy = sx + 16384;
          if (leads) {
            if (rank == 0) mbar_expect_tx(full_local, tx);
            if constexpr (MODE == MODE_FORWARD) {
              const int n0 = w.ni * p.out_tile_n;
              if constexpr (GLU) {  // gate rows first, up rows behind them: one half per CTA of a pair
                if constexpr (CTA_GROUP == 2) {
                  tma_load_3d<2>(sy, &p.map_y, kb * block_k, n0 + (rank ? p.glu_offset : 0), w.group, full);
                } else {
                  tma_load_3d<1>(sy, &p.map_y, kb * block_k, n0, w.group, full);
                  tma_load_3d<1>(sy + y_bytes / 2, &p.map_y, kb * block_k, n0 + p.glu_offset, w.group, full);
                }
              } else {
                tma_load_3d<CTA_GROUP>(sy, &p.map_y, kb * block_k, n0 + int(rank) * y_rows, w.group, full);
              }
            } else if constexpr (MODE == MODE_DX) {
              const int c0 = w.ni * tile_n + int(rank) * y_rows;
              for (int b = 0; b < y_boxes; ++b) tma_load_3d<CTA_GROUP>(sy + b * 8192, &p.map_y, c0 + 64 * b, (w.k0 + kb) * 64, p.split_blocks ? 0 : w.group, full);
            } else {
              const int r = w.first_row + kb * 64, m0 = w.mi * TILE_M + int(rank) * 128;
              tma_load_2d<CTA_GROUP>(sx, &p.map_x, m0, r, full);
              tma_load_2d<CTA_GROUP>(sx + 8192, &p.map_x, m0 + 64, r, full);
              const int c0 = w.ni * tile_n + int(rank) * y_rows;
              for (int b = 0; b < y_boxes; ++b) tma_load_2d<CTA_GROUP>(sy + b * 8192, &p.map_y, c0 + 64 * b, r, full);
            }
            if constexpr (MODE != MODE_DW && !GATHER) {
              const int kx = (w.k0 + kb) * block_k;
              if (mine == 128) tma_load_2d<CTA_GROUP>(sx, &p.map_x, kx, x_row, full);
              else
                for (int r = 0; r < mine; r += 32) tma_load_2d<CTA_GROUP>(sx + r * 128, &p.map_x32, kx, x_row + r, full);
            }
          }
          if constexpr (GATHER) {
            if (4 * lane < mine)
              tma_gather4(sx + lane * 512, &p.map_x32, kb * block_k, token[0], token[1], token[2], token[3], full);
          }
          if constexpr (MODE == MODE_DW) {  // a short block is on its way: the clearing warp may look for it
            if (leads && rank == 0 && kb == blocks - 1 && (w.rows & 63)) mbar_arrive(bar_go + 8 * stage);
          }
          ++issued;
          if (++stage == stages) stage = 0, phase ^= 1;
        }
      }
      if (!ok && rank == 0 && leads) {
        // Loads in flight still land: give each armed barrier a bounded chance before teardown.
        int s = stage;
        uint32_t ph = phase;
        const uint32_t pending = issued < uint32_t(p.stages) ? issued : uint32_t(p.stages);
        for (uint32_t back = 0; back < pending; ++back) {
          if (--s < 0) s = p.stages - 1, ph ^= 1;
          const uint64_t start = global_timer_ns();
          while (!mbar_try_wait(bar_full + 8 * s, ph) && global_timer_ns() - start < 1000000ull) {
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (rank == 0 && elect_one()) {
      const uint64_t desc_stage = uint64_t(p.stage_bytes >> 4);
      const uint64_t dx0 = X_COLUMNS ? column_operand_desc(ring) : operand_desc(ring);
      const uint64_t dy0 = Y_COLUMNS ? column_operand_desc(ring + 16384) : operand_desc(ring + 16384);
      // Operand start from one MMA to the next: 32 bytes of K, or 16 rows of a column box.
      constexpr uint64_t X_STEP = X_COLUMNS ? 128 : 2, Y_STEP = Y_COLUMNS ? 128 : 2;
      const int stages = p.stages, block_k = p.block_k, mma_k = block_k / 4;
      const uint32_t idesc = p.idesc;
      int stage = 0, tile_idx = 0;
      uint32_t phase = 0, cleared = 0;  // bit s: parity of stage s's next short block
      uint64_t stage_off = 0;
      bool ok = mbar_wait(bar_tmem, 0, ctx, SITE_TMEM_READY);
      tc_fence_after_sync();
      const uint32_t tmem_base = tmem_slot;
      for (int t = cluster_id; ok && t < num_tiles; t += num_clusters, ++tile_idx) {
        ExpertTile w;
        find_tile(t, w);
        const int blocks = k_blocks_of(w);
        const int slot = tile_idx & 1;
        if (!mbar_wait(bar_acc_empty + 8 * slot, ((tile_idx >> 1) & 1) ^ 1, ctx, SITE_MMA_ACC_EMPTY)) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + slot * p.tile_n;
        uint32_t accumulate = 0;
        int k_left = MODE == MODE_DW ? w.rows : p.k - w.k0 * block_k;
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(bar_full + 8 * stage, phase, ctx, SITE_MMA_FULL)) {
            ok = false;
            break;
          }
          if constexpr (MODE == MODE_DW) {
            if (k_left < 64) {
              if (!mbar_wait(bar_ready + 8 * stage, (cleared >> stage) & 1, ctx, SITE_MMA_FULL)) {
                ok = false;
                break;
              }
              cleared ^= 1u << stage;
            }
          }
#pragma unroll
          for (int ki = 0; ki < 4; ++ki) {
            if (ki == 0 || ki * mma_k < k_left) {  // an MMA that would read zeros only is skipped
              mma_dense<KIND, CTA_GROUP>(d_tmem, dx0 + stage_off + ki * X_STEP, dy0 + stage_off + ki * Y_STEP, idesc, accumulate);
              accumulate = 1;
            }
          }
          mma_commit<CTA_GROUP>(bar_empty + 8 * stage);
          k_left -= block_k;
          stage_off += desc_stage;
          if (++stage == stages) stage = 0, phase ^= 1, stage_off = 0;
        }
        if (ok) mma_commit<CTA_GROUP>(bar_acc_full + 8 * slot);
      }
    }
  } else if (MODE == MODE_DW && warp == 2 + XP_EPILOGUE_WARPS) {
    // ------------------------------------------------------- short blocks
    // Counts the stages as the producer does.  Once the producer has asked for
    // a short block, the leader waits for its data (its barrier counts both
    // CTAs' bytes), tells the pair's other CTA, and each clears its own rows past
    // the group's end.  The full barrier is looked at only after the producer's
    // word: until the MMA has used the block, its phase then cannot pass by.
    int stage = 0;
    uint32_t phase = 0, told = 0;
    bool ok = true;
    const int boxes = 2 + p.tile_n / CTA_GROUP / 64;
    for (int t = cluster_id; ok && t < num_tiles; t += num_clusters) {
      ExpertTile w;
      find_tile(t, w);
      const int blocks = k_blocks_of(w), tail = w.rows & 63;
      if (blocks == 0) continue;
      for (int kb = 0; kb < blocks; ++kb) {
        if (kb == blocks - 1 && tail) {
          ok = mbar_wait(bar_go + 8 * stage, (told >> stage) & 1, ctx, SITE_MMA_FULL);
          if (ok && rank == 0) ok = mbar_wait(bar_full + 8 * stage, phase, ctx, SITE_MMA_FULL);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          told ^= 1u << stage;
          if (CTA_GROUP == 2 && rank == 0 && lane == 0) mbar_arrive_cluster(map_to_cta(bar_go + 8 * stage, 1));
          // Rows tail .. 63 of every 64 x 128-byte box: whole lines, so the swizzle does not matter.
          const uint32_t base = ring + stage * p.stage_bytes;
          for (int b = 0; b < boxes; ++b)
            for (int i = tail * 8 + lane; i < 512; i += 32) st_shared_v4(base + b * 8192 + i * 16, 0u, 0u, 0u, 0u);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CTA_GROUP == 2) mbar_arrive_cluster(map_to_cta(bar_ready + 8 * stage, 0));
            else mbar_arrive(bar_ready + 8 * stage);
          }
        }
        if (++stage == p.stages) stage = 0, phase ^= 1;
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;
    const uint32_t lane_base = uint32_t(quarter * 32) << 16;
    const uint32_t acc_empty_leader = CTA_GROUP == 2 ? map_to_cta(bar_acc_empty, 0) : bar_acc_empty;
    const uint32_t my_buf = staging + (warp - 2) * 32 * ROW_BYTES;
    const int sub_row = lane / UNITS, unit = lane % UNITS;
    // 16-byte unit u of staging row r, swizzled so that eight lanes on eight rows,
    // or on the units of one row, touch all banks.
    auto at_unit = [&](int r, int u) { return my_buf + r * ROW_BYTES + ((u ^ (UNITS == 8 ? r & 7 : (r >> 1) & 3)) << 4); };
    const int out_tile_n = p.out_tile_n, cols = p.cols;
    const bool out_f16 = p.out_f16 != 0, vec_ok = p.vec_ok != 0;
    auto pack2 = [&](float lo, float hi) { return out_f16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi); };
    const bool allocated = mbar_wait(bar_tmem, 0, ctx, SITE_TMEM_READY);
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    int tile_idx = 0;
    for (int t = cluster_id; __all_sync(0xFFFFFFFFu, allocated) && t < num_tiles; t += num_clusters, ++tile_idx) {
      ExpertTile w;
      find_tile(t, w);
      const int slot = tile_idx & 1;
      const bool ready = mbar_wait(bar_acc_full + 8 * slot, (tile_idx >> 1) & 1, ctx, SITE_EPI_ACC_FULL);
      if (!__all_sync(0xFFFFFFFFu, ready)) break;
      tc_fence_after_sync();
      const int local_row = w.mi * TILE_M + int(rank) * 128 + quarter * 32;  // this warp's first row of the group's output
      const int group_rows = MODE == MODE_DW ? p.m_out : w.rows;
      const int valid = min(max(group_rows - local_row, 0), 32);             // rows this warp stores
      const bool by_part = MODE == MODE_DX && p.split_blocks;                // each part has an output of its own
      const size_t row0 = (MODE == MODE_DW ? size_t(w.group) * p.m_out : by_part ? size_t(w.group) * p.rows : size_t(w.first_row)) + local_row;
      const int col0 = w.ni * out_tile_n;
      const uint32_t acc = tmem_base + lane_base + slot * p.tile_n;
      const bool nothing = MODE == MODE_DW && w.rows == 0;                   // no rows: the sum is zero
      const float alpha = MODE == MODE_FORWARD && p.alpha ? p.alpha[w.group] * p.factor : p.factor;

      // CHUNK columns of this lane's row, through the warp's swizzled buffer, as
      // whole row segments; unaligned rows element by element, side by side.
      auto store = [&](const float* v, uint8_t* base, int ld, int col, int limit, bool direct) {
        if (lane == 0) tma_store_wait_read<0>();  // the buffer's last chunk has left
        __syncwarp();
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          uint32_t q[4];
#pragma unroll
          for (int h = 0; h < 4; ++h)
            q[h] = OUT_BYTES == 4 ? __float_as_uint(v[(4 * u + h) % CHUNK]) : pack2(v[(8 * u + 2 * h) % CHUNK], v[(8 * u + 2 * h + 1) % CHUNK]);
          st_shared_v4(at_unit(lane, u), q[0], q[1], q[2], q[3]);
        }
        if (direct && valid == 32) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.map_d, my_buf, col, int(row0));
            tma_store_commit();
          }
          return;
        }
        __syncwarp();
        if (vec_ok) {
          const int gcol = col + unit * UNIT;
          if (gcol < limit) {
            uint8_t* dst = base + ((row0 + sub_row) * ld + gcol) * OUT_BYTES;
            const size_t step = size_t(ROWS_AT_ONCE) * ld * OUT_BYTES;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
              const int r = i * ROWS_AT_ONCE + sub_row;
              if (r < valid) *reinterpret_cast<uint4*>(dst + i * step) = ld_shared_v4(at_unit(r, unit));
            }
          }
        } else if (col + lane < limit) {
          uint8_t* dst = base + (row0 * ld + col + lane) * OUT_BYTES;
#pragma unroll 8
          for (int r = 0; r < valid; ++r, dst += size_t(ld) * OUT_BYTES) {
            const uint32_t from = at_unit(r, lane / UNIT) + (lane % UNIT) * OUT_BYTES;
            if constexpr (OUT_BYTES == 4) *reinterpret_cast<uint32_t*>(dst) = ld_shared_u32(from);
            else *reinterpret_cast<uint16_t*>(dst) = ld_shared_u16(from);
          }
        }
        __syncwarp();
      };
      auto load = [&](int c, float* v) { tmem_ld_32(acc + c, reinterpret_cast<uint32_t*>(v)); };
      auto settle = [&](float* v) { tmem_ld_settle_32(reinterpret_cast<uint32_t*>(v)); };
      auto activate = [&](float* v) {
        if (p.act_shape == SHAPE_SIGMOID) activate_all<SHAPE_SIGMOID, CHUNK>(v, p.act_a, p.act_b);
        else if (p.act_shape == SHAPE_PHI) activate_all<SHAPE_PHI, CHUNK>(v, 0.f, 0.f);
        else if (p.act_shape == SHAPE_RELU) activate_all<SHAPE_RELU, CHUNK>(v, 0.f, 0.f);
      };

      auto hand_back = [&] {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          // Relaxed: what is handed back is tensor memory, whose loads have completed;
          // a release would wait for this warp's stores as well.
          if constexpr (CTA_GROUP == 2) mbar_arrive_cluster_relaxed(acc_empty_leader + 8 * slot);
          else mbar_arrive(bar_acc_empty + 8 * slot);
        }
      };
      // The next chunk's accumulators are on their way while a chunk is stored
      // (not those of a gated pair, which would be 64 more registers), and the
      // slot goes back once its last columns have arrived.
      constexpr int STRIDE = XP_EPILOGUE_WARPS / 4 * CHUNK;
      const int chunk0 = (warp - 2) / 4 * CHUNK;
      auto live = [&](int c) { return valid > 0 && c < out_tile_n && col0 + c < cols; };
      float coming[CHUNK];
      if (live(chunk0)) load(chunk0, coming);
      else hand_back();
      for (int c = chunk0; live(c); c += STRIDE) {
        const bool last = !live(c + STRIDE);
        float v[CHUNK], up[GLU ? CHUNK : 1];
        if constexpr (GLU) load(out_tile_n + c, up);
        tmem_ld_wait();
        settle(coming);
        if constexpr (GLU) settle(up);
#pragma unroll
        for (int j = 0; j < CHUNK; ++j) v[j] = nothing ? 0.0f : coming[j];
        if (last) hand_back();
        else if (!GLU) load(c + STRIDE, coming);
        if (alpha != 1.0f) {
#pragma unroll
          for (int j = 0; j < CHUNK; ++j) {
            v[j] *= alpha;
            if constexpr (GLU) up[j] *= alpha;
          }
        }
        if constexpr (MODE == MODE_FORWARD) {
          if (p.preact) {
            store(v, static_cast<uint8_t*>(p.preact), p.ldz, col0 + c, cols, false);
            if constexpr (GLU) store(up, static_cast<uint8_t*>(p.preact), p.ldz, p.glu_offset + col0 + c, p.glu_offset + cols, false);
          }
          activate(v);
          if constexpr (GLU) {
#pragma unroll
            for (int j = 0; j < CHUNK; ++j) v[j] *= up[j];
          }
        }
        store(v, static_cast<uint8_t*>(p.d), p.ldd, col0 + c, cols, p.direct != 0);
        if (GLU && !last) load(c + STRIDE, coming);
      }
    }
    if (lane == 0) tma_store_wait<0>();
  }

  if (p.beside) pdl_wait_prior_grids();
  tc_fence_before_sync();
  __syncthreads();
  if (CTA_GROUP == 2) cluster_sync_all();
  tc_fence_after_sync();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc<CTA_GROUP>(tmem_slot, p.tmem_cols);
  }
}

}  // namespace og
