// Products of rows grouped by expert for sm_100a, ragged sizes:
//
//   forward   C[i, n] = sum_k A[i, k] W[g, n, k]        offsets[g] <= i < offsets[g+1]
//   gradient  dW[g, n, k] = sum_i dC[i, n] A[i, k]      over the rows i of group g
//
// (the gradient with respect to A is the forward product with the transposed view of W).  All sums are tcgen05.mma
// chains in fp32 tensor-memory accumulators, K in steps of 16 from the first to the last, rounded once.  With leaves
// every leaf is a chain of its own and the leaves' sums are joined by fp32 adds in the tree of the dense kernel (level 0
// F leaves left to right, binary above), the stack in spare tensor-memory columns.  Neither depends on the group's size,
// the tile or the grid, so a row's bits are those of the dense kernel on the group's rows alone.
//
// What is ragged is only which tiles exist: every CTA builds the table of the groups' tiles in shared memory when it
// starts (offsets are read on the device), then the persistent loop of each role finds its tile's group by binary search.
// A tile's rows end with the group: rows beyond it are multiplied (they are the next group's) and not stored.
//
// Forward tiles put the WEIGHT's rows on the instruction's 128 (256) lanes and the tokens on its columns: the token count
// of an instruction is a run-time field in steps of 16 (32), so a ragged group costs what it holds, and a decode step's
// tiles of a few tokens read W and little else.  A group's tokens are dealt evenly to as few tiles as fit.
//
//   warp 0      TMA producer   128-byte swizzled boxes of 64 reduction steps; of the tokens 16, 32, 64 or 128 rows
//   warp 1      UMMA issuer    two accumulators: tile (or leaf) i+1 runs while i drains
//   warp 2      tensor memory
//   warps 4-11  epilogue       tcgen05.ld, tree, rounding, store
//
// The operands' contiguous index is the reduction index (K-major) or the other one (MN-major); the instruction takes
// either, so the transposed weight and both operands of the weight gradient are read as they lie.  The weight gradient
// reduces over a group's rows: its last step of 16 ends inside the group's last box, and the rows of the next group that the
// box brought along must become zero before the multiply, in both operands (a NaN there must not meet a zero).  That step
// has boxes of its own, loaded when the tile begins and cleared by warp 3, so that nobody waits for it when its turn comes
// (16384 rows of 32 groups, K = N = 2048: cleared in the stage itself by the issuing warps 147 us, so 129 us; groups of whole
// steps 126 us).
//
// PAIR: a cluster of two CTAs per tile (cta_group::2), each with its own 128 rows and half of the columns' operand.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "ptx_sm100a.cuh"
#include "tbik_internal.h"

namespace tbik {
namespace {

constexpr int BM = 128;  // rows of a tile per CTA
constexpr int BK = 64;   // reduction steps per stage
constexpr int UMMA_K = 16;
constexpr int NUM_THREADS = 384;
constexpr int EPI_WARP0 = 4;
constexpr int NUM_EPI_WARPS = 8;
constexpr uint32_t TMEM_COLS = 512;
constexpr int CHUNK = 32;  // accumulator columns per tcgen05.ld
constexpr uint64_t WAIT_LIMIT_NS = 2000000000ull;
constexpr uint32_t STAGING_BYTES_PER_WARP = 4096;  // weight gradient: 32 rows of 128 bytes
constexpr int DEALT = 256;  // tiles of a CTA (pair) that are worked out ahead
constexpr int GROUP_M = 8;  // row tiles that share a sweep over the columns

__device__ uint32_t g_grouped_status[4];  // [0] a bounded wait ran out, [1] block, [2] role

struct Maps {
  CUtensorMap a[4];  // forward: A with boxes of 16, 32, 64, 128 rows; weight gradient: dC, dW, dC and A with boxes of 16 rows
  CUtensorMap b;     // W; weight gradient: A
};

// What every role has to know of the groups, in shared memory: rows first[g] .. last[g] - 1, tiles of `per[g]` rows
// (forward), before[g] tiles in the groups before g (G + 1 entries; forward).
struct Table {
  int *first, *last, *before, *per;
  int* warps;  // 3 x 16 words of scratch
  static constexpr uint32_t bytes(int groups, bool tiles) { return 4u * ((tiles ? 4 * groups + 1 : 2 * groups) + 48); }
  TBIK_DEVICE Table(uint8_t* at, int groups, bool tiles) {
    first = reinterpret_cast<int*>(at);
    last = first + groups;
    per = tiles ? last + groups : nullptr;
    before = tiles ? per + groups : nullptr;
    warps = tiles ? before + groups + 1 : last + groups;
  }
};

TBIK_DEVICE int scan_max(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v = max(v, u);
  }
  return v;
}
TBIK_DEVICE int scan_sum(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Fills the table; all threads of the block, a thread per group.  tiles_of(rows, per) gives a group's tiles and writes the
// rows of one.  Whatever `offsets` holds, the running maximum keeps the groups' rows inside [0, M) and disjoint.  One more
// barrier has to follow before the table is read.
template <typename TilesOf>
TBIK_DEVICE void build_table(const int32_t* offsets, int groups, int M, const Table& t, TilesOf tiles_of) {
  constexpr int WARPS = NUM_THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int end = min(max(offsets[0], 0), M), run = 0;  // rows and tiles of the passes before
  for (int g0 = 0; g0 < groups; g0 += NUM_THREADS) {
    const int g = g0 + static_cast<int>(threadIdx.x);
    int hi = scan_max(g < groups ? min(max(offsets[g + 1], 0), M) : 0, lane);
    if (lane == 31) t.warps[warp] = hi;
    __syncthreads();
    int before_warp = end;
    for (int w = 0; w < warp; ++w) before_warp = max(before_warp, t.warps[w]);
    hi = max(hi, before_warp);
    int lo = __shfl_up_sync(0xFFFFFFFFu, hi, 1);
    if (lane == 0) lo = before_warp;
    int per = 1;
    const int tiles = g < groups ? tiles_of(hi - lo, per) : 0;
    const int sum = scan_sum(tiles, lane);
    if (lane == 31) {
      t.warps[16 + warp] = sum;
      t.warps[32 + warp] = hi;
    }
    __syncthreads();
    int at = run;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) at += t.warps[16 + w];
      run += t.warps[16 + w];
      end = max(end, t.warps[32 + w]);
    }
    if (g < groups) {
      t.first[g] = lo;
      t.last[g] = hi;
      if (t.before == nullptr) continue;
      t.per[g] = per;
      t.before[g] = at + sum - tiles;
      if (g == groups - 1) t.before[groups] = at + sum;
    }
  }
}

// a / b for a >= 0, b > 0, small numbers without the long integer division: (a + 0.5) / b is at least 0.5 / b away from a
// whole number, 2^-21 of itself for a < 2^20, and __fdividef is off by 2 units, 2^-22, at most.
TBIK_DEVICE int quotient(int a, int b) {
  return a < (1 << 20) ? static_cast<int>(__fdividef(static_cast<float>(a) + 0.5f, static_cast<float>(b))) : a / b;
}

// Keeps the compiler from working out all of an unrolled loop's addresses ahead, in registers that are not there.
template <typename V>
TBIK_DEVICE void one_by_one(V*& p) { asm volatile("" : "+l"(p)); }

// The group that a tile belongs to: before[g] <= tile < before[g + 1].
TBIK_DEVICE int group_of(const int* before, int groups, int tile) {
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= tile) lo = mid; else hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------- forward
struct ForwardParams {
  void* C;
  const int32_t* offsets;
  int64_t ldc;
  int M, N, groups;
  int blocks_per_leaf, T, F, L;  // 64-step blocks per leaf; the tree
  int tiles_w;                   // tiles over the weight's rows
  int half;                      // 16-bit type of the operands: 1 bf16, 0 fp16 (the UMMA format code)
  int out32;                     // C is fp32
  int zero_outside;              // rows of no group are set to zero
};

// W_ROWS weight rows per CTA against up to TN tokens.  SUB 64-step blocks share a stage: a barrier round trip of the
// single-thread roles costs about 300 cycles however little a block holds.
template <int W_ROWS, int TN_, int SUB_, int STAGES_, bool PAIR, bool W_MN>
struct ForwardCfg {
  static constexpr int TN = TN_, SUB = SUB_, STAGES = STAGES_;
  static constexpr int W_TILE = PAIR ? 2 * W_ROWS : W_ROWS;
  static constexpr int STEP = PAIR ? 32 : 16;                 // granularity of an instruction's token count
  static constexpr int T_ROWS = PAIR ? TN / 2 : TN;           // token rows this CTA stages
  static constexpr uint32_t W_BYTES = (W_MN && W_ROWS < 64 ? 64 : W_ROWS) * BK * 2;  // one block of W
  static constexpr uint32_t T_BYTES = T_ROWS * BK * 2;        // room for one block of tokens
  static constexpr uint32_t STAGE_BYTES = SUB * (W_BYTES + T_BYTES);
  // The instruction reads 128 rows of W whatever the box brought; with narrow tiles the surplus is whatever follows in
  // the stage, and its results are never read.
  static_assert(W_ROWS == 128 || (SUB - 1) * W_BYTES + 128 * BK * 2 <= STAGE_BYTES, "the surplus rows stay inside the stage");
  static constexpr int EPI_HALVES = TN >= 64 ? 2 : 1;
  static constexpr int CHUNKS = TN / CHUNK / EPI_HALVES;      // token chunks per epilogue warp
  static constexpr uint32_t OFF_FULL = STAGES * STAGE_BYTES;
  static constexpr uint32_t OFF_EMPTY = OFF_FULL + 8 * STAGES;
  static constexpr uint32_t OFF_TFULL = OFF_EMPTY + 8 * STAGES;
  static constexpr uint32_t OFF_TEMPTY = OFF_TFULL + 16;
  static constexpr uint32_t OFF_TMEM_PTR = OFF_TEMPTY + 16;
  static constexpr uint32_t OFF_ABORT = OFF_TMEM_PTR + 4;
  static constexpr uint32_t OFF_DEALT = (OFF_ABORT + 4 + 15) / 16 * 16;
  static constexpr uint32_t OFF_TABLE = OFF_DEALT + DEALT * 16;
  static constexpr uint32_t smem_bytes(int groups) { return OFF_TABLE + Table::bytes(groups, true) + 1024; }
  static_assert(smem_bytes(TBIK_MAX_GROUPS) <= 232448, "shared memory budget");
  // tokens per tile of a group of m rows: as few tiles as TN allows, evenly filled (m may be close to 2^31: m plus the number
  // of tiles would not fit)
  static TBIK_DEVICE int tokens(int m) {
    const int tiles = (m + TN - 1) / TN;
    return tiles == 0 ? STEP : (quotient(m - 1, tiles) + STEP) / STEP * STEP;
  }
};

template <int W_ROWS, int TN, int SUB, int STAGES, bool PAIR, bool W_MN, bool TREE>
__global__ void __launch_bounds__(NUM_THREADS, 1) forward_kernel(const __grid_constant__ Maps maps, const ForwardParams p) {
  using C_ = ForwardCfg<W_ROWS, TN, SUB, STAGES, PAIR, W_MN>;
  constexpr uint32_t STAGE_BYTES = C_::STAGE_BYTES, T_OFF = SUB * C_::W_BYTES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int cta_rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int num_units = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  const bool leader = cta_rank == 0;

  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem_gen + C_::OFF_ABORT);
  volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(smem_gen + C_::OFF_TMEM_PTR);
  auto full_bar = [&](int s) { return smem_base + C_::OFF_FULL + 8u * s; };
  auto empty_bar = [&](int s) { return smem_base + C_::OFF_EMPTY + 8u * s; };
  auto tfull_bar = [&](int a) { return smem_base + C_::OFF_TFULL + 8u * a; };
  auto tempty_bar = [&](int a) { return smem_base + C_::OFF_TEMPTY + 8u * a; };
  const Table table(smem_gen + C_::OFF_TABLE, p.groups, true);

  if constexpr (PAIR) cluster_sync_all();
  if (threadIdx.x == 0) {
    *abort_flag = 0u;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), (PAIR && leader) ? 2 : 1);  // pair, leader: its own producer and the partner's relay
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), PAIR ? 2 * NUM_EPI_WARPS : NUM_EPI_WARPS);
    }
    fence_mbar_init();
  }
  if (warp == 2) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_base + C_::OFF_TMEM_PTR, TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_base + C_::OFF_TMEM_PTR, TMEM_COLS);
      tmem_relinquish();
    }
  }
  build_table(p.offsets, p.groups, p.M, table, [&](int m, int& per) {
    per = C_::tokens(m);
    return quotient(m + per - 1, per) * p.tiles_w;
  });
  __syncthreads();
  const int num_tiles = table.before[p.groups];
  const int my_tiles = num_tiles > unit ? quotient(num_tiles - unit - 1, num_units) + 1 : 0;

  struct alignas(16) Tile {
    int g, t0, tokens, w0;  // group; first token row and number of rows; first weight row
  };
  // The i-th tile of this unit.  Every role walks the same list, and to work a tile out takes 950 cycles, a tenth of a tile's
  // time with leaves: the first ones are worked out at once, by as many threads.
  Tile* dealt = reinterpret_cast<Tile*>(smem_gen + C_::OFF_DEALT);
  auto work_out = [&](int i) {
    const int tile = unit + i * num_units;
    const int g = group_of(table.before, p.groups, tile);
    const int n = table.per[g], lo = table.first[g], hi = table.last[g];
    int in = tile - table.before[g], first_tt = 0, height = quotient(hi - lo + n - 1, n);
    if (height > GROUP_M) {  // GROUP_M token tiles share a sweep over the weight's rows
      first_tt = quotient(in, GROUP_M * p.tiles_w) * GROUP_M;
      in -= first_tt * p.tiles_w;
      height = min(height - first_tt, GROUP_M);
    }
    const int tw = quotient(in, height);
    Tile t;
    t.g = g;
    t.t0 = lo + (first_tt + in - tw * height) * n;
    t.tokens = min(n, hi - t.t0);
    t.w0 = tw * C_::W_TILE;
    return t;
  };
  for (int i = threadIdx.x; i < min(my_tiles, DEALT); i += NUM_THREADS) dealt[i] = work_out(i);
  auto tile_at = [&](int i) { return i < DEALT ? dealt[i] : work_out(i); };
  tc_fence_before_sync();
  if constexpr (PAIR) cluster_sync_all(); else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_ptr_smem;

  // token count of the instructions: whole steps
  auto issue_tokens = [&](const Tile& t) { return (t.tokens + C_::STEP - 1) / C_::STEP * C_::STEP; };

  int role_failed = 0;

  // The tree's epilogue holds a node and a whole leaf in registers: with 128 tokens per tile it takes registers from the
  // warps that issue.
  constexpr bool SPLIT = TREE && C_::CHUNKS > 1;
  if (warp < EPI_WARP0) {
  if constexpr (SPLIT) setmaxnreg_dec<56>();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t policy = l2_policy(0);
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile t = tile_at(i);
        const int rows = PAIR ? issue_tokens(t) / 2 : issue_tokens(t);  // token rows of this CTA
        const int box = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
        const int box_rows = 16 << box;
        const CUtensorMap* map_t = &maps.a[box];
        const int t0 = t.t0 + cta_rank * rows, w0 = t.w0 + cta_rank * W_ROWS;
        const uint32_t block_bytes = C_::W_BYTES + static_cast<uint32_t>(box_rows) * BK * 2;
        // one stage: up to SUB blocks
        auto load = [&](int x, int blocks) -> bool {
          if (!mbar_wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, WAIT_LIMIT_NS)) {
            ok = false;
            role_failed = 1;
            return false;
          }
          const uint32_t sw = smem_base + stage * STAGE_BYTES, st = sw + T_OFF, bar = full_bar(stage);
          mbar_arrive_expect_tx(bar, static_cast<uint32_t>(blocks) * block_bytes);
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
            if (SUB == 1 || u < blocks) {
              const int k = x + u * BK;
              if constexpr (W_MN) {
#pragma unroll
                for (int v = 0; v < (W_ROWS + 63) / 64; ++v)
                  tma_load_3d_hint(sw + u * C_::W_BYTES + v * 8192, &maps.b, w0 + v * 64, k, t.g, bar, policy);
              } else {
                tma_load_3d_hint(sw + u * C_::W_BYTES, &maps.b, k, w0, t.g, bar, policy);
              }
              tma_load_2d_hint(st + u * C_::T_BYTES, map_t, k, t0, bar, policy);
            }
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
          return true;
        };
        if constexpr (SUB == 1) {
          // straight-line code for four blocks: a taken branch per block costs more than issuing its loads.  Leaves follow
          // each other in K, so they do not matter here.
          const int blocks = p.T * p.blocks_per_leaf;
          int b = 0;
          for (; ok && b + 4 <= blocks; b += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (!load((b + u) * BK, 1)) break;
          }
          for (; ok && b < blocks; ++b)
            if (!load(b * BK, 1)) break;
        } else {
          for (int l = 0; ok && l < p.T; ++l) {
            for (int b = 0; b < p.blocks_per_leaf; b += SUB)
              if (!load((l * p.blocks_per_leaf + b) * BK, min(SUB, p.blocks_per_leaf - b))) break;
          }
        }
      }
      if (!ok) {  // copies that are still in flight get time to land before the CTA retires
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (PAIR && !leader) {
      // ------------------------------------------------------------ partner: relay "stage landed" to the leader
      if (elect_one()) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        const int stages_per_tile = p.T * ((p.blocks_per_leaf + SUB - 1) / SUB);
        for (int i = 0; ok && i < my_tiles; ++i) {
          for (int s = 0; s < stages_per_tile; ++s) {
            if (!mbar_wait_bounded(full_bar(stage), phase, abort_flag, WAIT_LIMIT_NS)) {
              ok = false;
              role_failed = 5;
              break;
            }
            mbar_arrive_cluster(map_to_cta(full_bar(stage), 0));
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
    } else if (elect_one()) {
      // ------------------------------------------------------------ UMMA issuer
      const uint64_t desc_w0 = W_MN ? umma_desc_sw128_mnmajor(smem_base, 8192u) : umma_desc_sw128_kmajor(smem_base);
      const uint64_t desc_t0 = umma_desc_sw128_kmajor(smem_base + T_OFF);
      constexpr uint64_t W_STEP = W_MN ? 2048 >> 4 : (UMMA_K * 2) >> 4, T_STEP = (UMMA_K * 2) >> 4;
      int stage = 0;
      uint32_t phase = 0, chain = 0;
      bool ok = true;
      auto commit = [&](uint32_t bar) {
        if constexpr (PAIR) {
          umma_commit_pair(bar);
          umma_commit_pair(map_to_cta(bar, 1));
        } else {
          umma_commit(bar);
        }
      };
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile t = tile_at(i);
        const uint32_t idesc = umma_idesc_f16(static_cast<uint32_t>(p.half), PAIR ? 256 : 128, static_cast<uint32_t>(issue_tokens(t))) |
                               (W_MN ? kUmmaTransposeA : 0u);
        for (int l = 0; ok && l < p.T; ++l, ++chain) {
          const uint32_t a = chain & 1u;
          if (!mbar_wait_bounded(tempty_bar(a), ((chain >> 1) & 1u) ^ 1u, abort_flag, WAIT_LIMIT_NS)) {
            ok = false;
            role_failed = 2;
            break;
          }
          tc_fence_after_sync();
          const uint32_t tmem_d = tmem_base + a * TN;
          auto stage_of = [&](int b, int blocks) -> bool {
            if (!mbar_wait_bounded(full_bar(stage), phase, abort_flag, WAIT_LIMIT_NS)) {
              ok = false;
              role_failed = 3;
              return false;
            }
            tc_fence_after_sync();
            const uint64_t sd = static_cast<uint64_t>(stage) * (STAGE_BYTES >> 4);
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              if (SUB == 1 || u < blocks) {
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k) {
                  const uint64_t dw = desc_w0 + sd + u * (C_::W_BYTES >> 4) + k * W_STEP;
                  const uint64_t dt = desc_t0 + sd + u * (C_::T_BYTES >> 4) + k * T_STEP;
                  const uint32_t acc = (b | u | k) != 0 ? 1u : 0u;
                  if constexpr (PAIR) umma_f16_ss_pair(tmem_d, dw, dt, idesc, acc);
                  else umma_f16_ss(tmem_d, dw, dt, idesc, acc);
                }
              }
            }
            commit(empty_bar(stage));
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
            return true;
          };
          if constexpr (SUB == 1) {
            int b = 0;
            for (; ok && b + 4 <= p.blocks_per_leaf; b += 4) {
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (!stage_of(b + u, 1)) break;
            }
#pragma unroll
            for (int u = 0; u < 3; ++u)
              if (ok && b + u < p.blocks_per_leaf) stage_of(b + u, 1);
          } else {
            for (int b = 0; b < p.blocks_per_leaf; b += SUB)
              if (!stage_of(b, min(SUB, p.blocks_per_leaf - b))) break;
          }
          if (ok) commit(tfull_bar(a));
        }
      }
    }
  }
  } else {
    // ------------------------------------------------------------ epilogue: lanes are weight rows, columns are tokens
    if constexpr (SPLIT) setmaxnreg_inc<224>();
    const int q = warp & 3;                 // tensor-memory lane quadrant of this warp
    const int h = (warp - EPI_WARP0) >> 2;  // it drains every second chunk of tokens
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tempty0 = PAIR ? map_to_cta(tempty_bar(0), 0) : tempty_bar(0);
    const int es = p.out32 ? 4 : 2;
    const bool pairs_ok = !p.out32 && p.ldc % 2 == 0 && (reinterpret_cast<uintptr_t>(p.C) & 3u) == 0;
    bool ok = true;

    if (p.zero_outside) {
      // rows of no group, before the first and behind the last: one warp per row
      const bool vec = (p.ldc * es) % 16 == 0 && (static_cast<int64_t>(p.N) * es) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.C) & 15u) == 0;
      const int lo = table.first[0], hi = table.last[p.groups - 1];
      for (int64_t i = static_cast<int64_t>(blockIdx.x) * NUM_EPI_WARPS + warp - EPI_WARP0; i < static_cast<int64_t>(lo) + (p.M - hi);
           i += static_cast<int64_t>(gridDim.x) * NUM_EPI_WARPS) {
        const int64_t row = i < lo ? i : hi + (i - lo);
        uint8_t* dst = static_cast<uint8_t*>(p.C) + row * p.ldc * es;
        if (vec) {
          for (int64_t c = lane; c < static_cast<int64_t>(p.N) * es / 16; c += 32) reinterpret_cast<uint4*>(dst)[c] = make_uint4(0u, 0u, 0u, 0u);
        } else {
          for (int64_t c = lane; c < static_cast<int64_t>(p.N) * es / 2; c += 32) reinterpret_cast<uint16_t*>(dst)[c] = 0;
        }
      }
    }

    uint32_t chain = 0;
    for (int i = 0; ok && i < my_tiles; ++i) {
      const Tile t = tile_at(i);
      const int n0 = t.w0 + cta_rank * W_ROWS + q * 32;  // this warp's 32 columns of C
      const bool busy = h < C_::EPI_HALVES && q * 32 < W_ROWS && n0 < p.N;
      const bool whole = pairs_ok && n0 + 32 <= p.N;
      // v[j]: column n0 + lane of token row tok + j.  A lane holds one column of 32 rows: lanes 2i and 2i + 1 swap halves
      // of two rows, so that a store instruction writes 64 whole bytes of each of two rows.
      auto store_chunk = [&](const float (&v)[CHUNK], int tok) {
        const int left = t.tokens - tok;
        if (p.out32) {
          float* dst = static_cast<float*>(p.C) + static_cast<int64_t>(t.t0 + tok) * p.ldc + n0 + lane;
          const bool in = n0 + lane < p.N;
#pragma unroll
          for (int j = 0; j < CHUNK; ++j, dst += p.ldc)
          {
            if (j < left && in) *dst = v[j];
            one_by_one(dst);
          }
          return;
        }
        if (whole) {
          // every column exists and pairs of columns are aligned: straight-line code, a store is predicated on its row alone
          const bool odd = (lane & 1) != 0;
          uint16_t* dst = static_cast<uint16_t*>(p.C) + static_cast<int64_t>(t.t0 + tok + (lane & 1)) * p.ldc + n0 + (lane & ~1);
#pragma unroll
          for (int j = 0; j < CHUNK; j += 2, dst += 2 * p.ldc) {
            const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[j] : v[j + 1], 1);
            const float lo = odd ? other : v[j], hi = odd ? v[j + 1] : other;
            const uint32_t w = p.half ? Pack16<__nv_bfloat16>::from_f32(lo, hi) : Pack16<__half>::from_f32(lo, hi);
            if (j + (lane & 1) < left) *reinterpret_cast<uint32_t*>(dst) = w;
            one_by_one(dst);
          }
          return;
        }
        uint16_t* dst = static_cast<uint16_t*>(p.C) + static_cast<int64_t>(t.t0 + tok) * p.ldc + n0 + lane;
        const bool in = n0 + lane < p.N;
#pragma unroll
        for (int j = 0; j < CHUNK; ++j, dst += p.ldc) {
          const uint32_t w = p.half ? Pack16<__nv_bfloat16>::from_f32(v[j], 0.0f) : Pack16<__half>::from_f32(v[j], 0.0f);
          if (j < left && in) *dst = static_cast<uint16_t>(w & 0xFFFFu);
          one_by_one(dst);
        }
      };
      // the open level-0 group, then the node that climbs the tree: fp32 in the registers that tcgen05.ld fills
      [[maybe_unused]] uint32_t node[TREE ? C_::CHUNKS : 1][CHUNK];
      int in_group = 0;
      uint32_t closed = 0;
      for (int l = 0; ok && l < p.T; ++l, ++chain) {
        const uint32_t a = chain & 1u;
        if (!mbar_wait_bounded(tfull_bar(a), (chain >> 1) & 1u, abort_flag, WAIT_LIMIT_NS)) {
          ok = false;
          role_failed = 4;
          break;
        }
        tc_fence_after_sync();
        const uint32_t tacc = tmem_base + lane_off + a * TN + h * CHUNK;
        auto release = [&]() {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * a);
        };
        // chunks of this warp that hold tokens: h, h + 2, ...
        const int have = busy ? ((t.tokens + CHUNK - 1) / CHUNK - h + C_::EPI_HALVES - 1) / C_::EPI_HALVES : 0;
        if (have <= 0) {
          release();
          continue;
        }
        if constexpr (!TREE) {
          // A loop, not unrolled code: with few tiles per SM this runs once or twice, and fetching four copies of the body
          // took longer than draining (one 256-token tile per SM, N = 1000: 13000 cycles).
#pragma unroll 1
          for (int c = 0; c < have; ++c) {
            uint32_t raw[CHUNK];
            tmem_ld32(tacc + c * C_::EPI_HALVES * CHUNK, raw);
            tmem_wait_ld();
            if (c + 1 == have) release();
            float v[CHUNK];
#pragma unroll
            for (int j = 0; j < CHUNK; ++j) v[j] = __uint_as_float(raw[j]);
            store_chunk(v, (c * C_::EPI_HALVES + h) * CHUNK);
          }
        } else {
          tmem_wait_st();  // stack stores of earlier leaves have landed
          // one fp32 add per node (commutative: which side is the earlier one does not matter)
          auto add = [&](uint32_t (&x)[CHUNK], const uint32_t (&y)[CHUNK]) {
#pragma unroll
            for (int j = 0; j < CHUNK; ++j) x[j] = __float_as_uint(__fadd_rn(__uint_as_float(x[j]), __uint_as_float(y[j])));
          };
          // 32 columns per chunk from tensor memory, all chunks requested before the first is waited for
          auto fetch = [&](uint32_t (&v)[C_::CHUNKS][CHUNK], uint32_t col) {
#pragma unroll
            for (int c = 0; c < C_::CHUNKS; ++c)
              if (c < have) tmem_ld32(col + c * C_::EPI_HALVES * CHUNK, v[c]);
            tmem_wait_ld();
          };
          if (in_group == 0) {
            fetch(node, tacc);
            release();
          } else {
            uint32_t raw[C_::CHUNKS][CHUNK];
            fetch(raw, tacc);
            release();
#pragma unroll
            for (int c = 0; c < C_::CHUNKS; ++c)
              if (c < have) add(node[c], raw[c]);  // level 0: F leaves left to right
          }
          if (++in_group < p.F) continue;
          in_group = 0;
          uint32_t gb = closed++;
          int lvl = 1;
          auto stack_col = [&](int level) -> uint32_t { return tmem_base + lane_off + (1 + level) * TN + h * CHUNK; };
          while (lvl < p.L && (gb & 1u)) {
            uint32_t raw[C_::CHUNKS][CHUNK];
            fetch(raw, stack_col(lvl));
#pragma unroll
            for (int c = 0; c < C_::CHUNKS; ++c)
              if (c < have) add(node[c], raw[c]);
            gb >>= 1;
            ++lvl;
          }
#pragma unroll
          for (int c = 0; c < C_::CHUNKS; ++c) {
            if (c < have) {
              if (lvl < p.L) {
                tmem_st32(stack_col(lvl) + c * C_::EPI_HALVES * CHUNK, node[c]);
              } else {
                float v[CHUNK];
#pragma unroll
                for (int j = 0; j < CHUNK; ++j) v[j] = __uint_as_float(node[c][j]);
                store_chunk(v, (c * C_::EPI_HALVES + h) * CHUNK);
              }
            }
          }
        }
      }
    }
  }

  // ---------------------------------------------------------------- tear-down
  tc_fence_before_sync();
  __syncwarp();
  if constexpr (PAIR) cluster_sync_all(); else __syncthreads();
  if (role_failed != 0 && atomicCAS(&g_grouped_status[0], 0u, 1u) == 0u) {
    g_grouped_status[1] = blockIdx.x;
    g_grouped_status[2] = static_cast<uint32_t>(role_failed);
  }
  if (warp == 2) {
    tc_fence_after_sync();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS); else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------- weight gradient
struct WgradParams {
  void* C;
  const int32_t* offsets;
  int M, groups;
  int rows, cols;        // N, K: dW[g] is [N, K]
  int tiles_r, tiles_c;
  int half, out32;
  int tma_store;         // dW leaves through tensor map a[1]
};

template <int BN, int STAGES_, bool PAIR>
struct WgradCfg {
  static constexpr int STAGES = STAGES_;
  static constexpr int TILE_M = PAIR ? 2 * BM : BM;
  static constexpr int B_COLS = PAIR ? BN / 2 : BN;  // columns of A that this CTA stages
  static constexpr uint32_t A_BYTES = BM * BK * 2;
  static constexpr uint32_t STAGE_BYTES = A_BYTES + B_COLS * BK * 2;
  static constexpr int CW = BN / 2;  // columns per epilogue warp
  static constexpr int NCH = CW / CHUNK;
  static constexpr uint32_t TAIL_BYTES = STAGE_BYTES / BK * UMMA_K;  // a group's last step, of two tiles
  static constexpr uint32_t OFF_TAIL = STAGES * STAGE_BYTES;
  static constexpr uint32_t OFF_STAGING = OFF_TAIL + 2 * TAIL_BYTES;
  static constexpr uint32_t OFF_FULL = OFF_STAGING + NUM_EPI_WARPS * STAGING_BYTES_PER_WARP;
  static constexpr uint32_t OFF_EMPTY = OFF_FULL + 8 * STAGES;
  static constexpr uint32_t OFF_TFULL = OFF_EMPTY + 8 * STAGES;
  static constexpr uint32_t OFF_TEMPTY = OFF_TFULL + 16;
  static constexpr uint32_t OFF_TAIL_BARS = OFF_TEMPTY + 16;  // landed, free, cleared: two each
  static constexpr uint32_t OFF_TMEM_PTR = OFF_TAIL_BARS + 48;
  static constexpr uint32_t OFF_ABORT = OFF_TMEM_PTR + 4;
  static constexpr uint32_t OFF_DEALT = (OFF_ABORT + 4 + 15) / 16 * 16;
  static constexpr uint32_t OFF_TABLE = OFF_DEALT + DEALT * 32;
  static constexpr uint32_t smem_bytes(int groups) { return OFF_TABLE + Table::bytes(groups, false) + 1024; }
  static_assert(smem_bytes(TBIK_MAX_GROUPS) <= 232448, "shared memory budget");
};

template <int BN, int STAGES, bool PAIR>
__global__ void __launch_bounds__(NUM_THREADS, 1) wgrad_kernel(const __grid_constant__ Maps maps, const WgradParams p) {
  using C_ = WgradCfg<BN, STAGES, PAIR>;
  constexpr uint32_t STAGE_BYTES = C_::STAGE_BYTES;
  constexpr int TILE_M = C_::TILE_M;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int cta_rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int num_units = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  const bool leader = cta_rank == 0;

  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem_gen + C_::OFF_ABORT);
  volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(smem_gen + C_::OFF_TMEM_PTR);
  auto full_bar = [&](int s) { return smem_base + C_::OFF_FULL + 8u * s; };
  auto empty_bar = [&](int s) { return smem_base + C_::OFF_EMPTY + 8u * s; };
  auto tfull_bar = [&](int a) { return smem_base + C_::OFF_TFULL + 8u * a; };
  auto tempty_bar = [&](int a) { return smem_base + C_::OFF_TEMPTY + 8u * a; };
  auto tail_landed_bar = [&](int b) { return smem_base + C_::OFF_TAIL_BARS + 8u * b; };
  auto tail_free_bar = [&](int b) { return smem_base + C_::OFF_TAIL_BARS + 16 + 8u * b; };
  auto tail_cleared_bar = [&](int b) { return smem_base + C_::OFF_TAIL_BARS + 32 + 8u * b; };
  const Table table(smem_gen + C_::OFF_TABLE, p.groups, false);

  if constexpr (PAIR) cluster_sync_all();
  if (threadIdx.x == 0) {
    *abort_flag = 0u;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), (PAIR && leader) ? 2 : 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), PAIR ? 2 * NUM_EPI_WARPS : NUM_EPI_WARPS);
      mbar_init(tail_landed_bar(a), 1);
      mbar_init(tail_free_bar(a), 1);
      mbar_init(tail_cleared_bar(a), PAIR ? 2 : 1);  // pair: each CTA's warp 3, the leader's barrier alone
    }
    fence_mbar_init();
  }
  if (warp == 2) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_base + C_::OFF_TMEM_PTR, TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_base + C_::OFF_TMEM_PTR, TMEM_COLS);
      tmem_relinquish();
    }
  }
  build_table(p.offsets, p.groups, p.M, table, [&](int, int&) { return 0; });
  __syncthreads();
  const int num_tiles = p.groups * p.tiles_r * p.tiles_c;
  const int my_tiles = num_tiles > unit ? quotient(num_tiles - unit - 1, num_units) + 1 : 0;

  struct alignas(16) Tile {
    int g, r0, count, row, col;  // group, its first row and their number; first row and column of dW[g]
  };
  Tile* dealt = reinterpret_cast<Tile*>(smem_gen + C_::OFF_DEALT);
  auto work_out = [&](int i) {  // the i-th tile of this unit, as in the forward kernel
    const int tile = unit + i * num_units;
    const int per = p.tiles_r * p.tiles_c;
    const int g = quotient(tile, per);
    int in = tile - g * per, first_row = 0, height = p.tiles_r;
    if (height > GROUP_M) {
      first_row = quotient(in, GROUP_M * p.tiles_c) * GROUP_M;
      in -= first_row * p.tiles_c;
      height = min(height - first_row, GROUP_M);
    }
    const int col = quotient(in, height);
    return Tile{g, table.first[g], table.last[g] - table.first[g], (first_row + in - col * height) * TILE_M, col * BN};
  };
  for (int i = threadIdx.x; i < min(my_tiles, DEALT); i += NUM_THREADS) dealt[i] = work_out(i);
  auto tile_at = [&](int i) { return i < DEALT ? dealt[i] : work_out(i); };
  tc_fence_before_sync();
  if constexpr (PAIR) cluster_sync_all(); else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_ptr_smem;

  int role_failed = 0;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0, tails = 0;
      bool ok = true;
      const uint64_t policy = l2_policy(0);
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile t = tile_at(i);
        const int whole = t.count / UMMA_K * UMMA_K;  // rows in whole steps
        const int row = t.row + cta_rank * BM, col = t.col + cta_rank * C_::B_COLS;
        if (whole < t.count) {
          const uint32_t buf = tails & 1u, bar = tail_landed_bar(buf);
          if (!mbar_wait_bounded(tail_free_bar(buf), ((tails >> 1) & 1u) ^ 1u, abort_flag, WAIT_LIMIT_NS)) {
            ok = false;
            role_failed = 6;
            break;
          }
          ++tails;
          const uint32_t sa = smem_base + C_::OFF_TAIL + buf * C_::TAIL_BYTES, sb = sa + C_::A_BYTES / BK * UMMA_K;
          mbar_arrive_expect_tx(bar, C_::TAIL_BYTES);
#pragma unroll
          for (int u = 0; u < BM / 64; ++u) tma_load_2d_hint(sa + u * 2048, &maps.a[2], row + u * 64, t.r0 + whole, bar, policy);
#pragma unroll
          for (int u = 0; u < C_::B_COLS / 64; ++u) tma_load_2d_hint(sb + u * 2048, &maps.a[3], col + u * 64, t.r0 + whole, bar, policy);
        }
        for (int b = 0; b < whole; b += BK) {
          if (!mbar_wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, WAIT_LIMIT_NS)) {
            ok = false;
            role_failed = 1;
            break;
          }
          const uint32_t sa = smem_base + stage * STAGE_BYTES, sb = sa + C_::A_BYTES, bar = full_bar(stage);
          mbar_arrive_expect_tx(bar, STAGE_BYTES);
#pragma unroll
          for (int u = 0; u < BM / 64; ++u)
            tma_load_2d_hint(sa + u * 8192, &maps.a[0], row + u * 64, t.r0 + b, bar, policy);
#pragma unroll
          for (int u = 0; u < C_::B_COLS / 64; ++u)
            tma_load_2d_hint(sb + u * 8192, &maps.b, col + u * 64, t.r0 + b, bar, policy);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (PAIR && !leader) {
      // ------------------------------------------------------------ partner: relay "stage landed" to the leader
      if (elect_one()) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = 0; ok && i < my_tiles; ++i) {
          const int whole = tile_at(i).count / UMMA_K * UMMA_K;
          for (int b = 0; b < whole; b += BK) {
            if (!mbar_wait_bounded(full_bar(stage), phase, abort_flag, WAIT_LIMIT_NS)) {
              ok = false;
              role_failed = 5;
              break;
            }
            mbar_arrive_cluster(map_to_cta(full_bar(stage), 0));
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
    } else if (elect_one()) {
      // ------------------------------------------------------------ UMMA issuer
      const uint32_t idesc = umma_idesc_f16(static_cast<uint32_t>(p.half), TILE_M, BN) | kUmmaTransposeA | kUmmaTransposeB;
      const uint64_t desc_a0 = umma_desc_sw128_mnmajor(smem_base, 8192u);
      const uint64_t desc_b0 = umma_desc_sw128_mnmajor(smem_base + C_::A_BYTES, 8192u);
      const uint64_t tail_a0 = umma_desc_sw128_mnmajor(smem_base + C_::OFF_TAIL, 2048u);
      const uint64_t tail_b0 = umma_desc_sw128_mnmajor(smem_base + C_::OFF_TAIL + C_::A_BYTES / BK * UMMA_K, 2048u);
      constexpr uint64_t STEP = 2048 >> 4;
      int stage = 0;
      uint32_t phase = 0, chain = 0, tails = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity, int role) {
        ok = mbar_wait_bounded(bar, parity, abort_flag, WAIT_LIMIT_NS);
        if (!ok) role_failed = role;
        return ok;
      };
      auto commit = [&](uint32_t bar) {
        if constexpr (PAIR) {
          umma_commit_pair(bar);
          umma_commit_pair(map_to_cta(bar, 1));
        } else {
          umma_commit(bar);
        }
      };
      auto multiply = [&](uint32_t d, uint64_t a, uint64_t b, bool first) {
        if constexpr (PAIR) umma_f16_ss_pair(d, a, b, idesc, first ? 0u : 1u); else umma_f16_ss(d, a, b, idesc, first ? 0u : 1u);
      };
      for (int i = 0; ok && i < my_tiles; ++i) {
        const int count = tile_at(i).count, whole = count / UMMA_K * UMMA_K;
        if (count == 0) continue;  // an empty group: the epilogue writes zeros
        const uint32_t a = chain & 1u;
        if (!wait(tempty_bar(a), ((chain >> 1) & 1u) ^ 1u, 2)) break;
        ++chain;
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + a * BN;
        for (int b = 0; b < whole; b += BK) {
          if (!wait(full_bar(stage), phase, 3)) break;
          tc_fence_after_sync();
          const uint64_t sd = static_cast<uint64_t>(stage) * (STAGE_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            if (b + k * UMMA_K < whole) multiply(tmem_d, desc_a0 + sd + k * STEP, desc_b0 + sd + k * STEP, (b | k) == 0);
          commit(empty_bar(stage));
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok && whole < count) {
          const uint32_t buf = tails & 1u;
          const uint32_t parity = (tails >> 1) & 1u;
          if (!wait(tail_cleared_bar(buf), parity, 7)) break;
          if (PAIR && !mbar_acquire_cluster(tail_cleared_bar(buf), parity)) {  // the partner's zeros
            ok = false;
            role_failed = 7;
            break;
          }
          ++tails;
          tc_fence_after_sync();
          const uint64_t sd = static_cast<uint64_t>(buf) * (C_::TAIL_BYTES >> 4);
          multiply(tmem_d, tail_a0 + sd, tail_b0 + sd, whole == 0);
          commit(tail_free_bar(buf));
        }
        if (ok) commit(tfull_bar(a));
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------ clears what follows the group in its last step
    constexpr int BOXES = static_cast<int>(C_::TAIL_BYTES / 2048);
    uint32_t tails = 0;
    for (int i = 0; i < my_tiles; ++i) {
      const int left = tile_at(i).count % UMMA_K;
      if (left == 0) continue;
      const uint32_t buf = tails & 1u;
      // the lanes have to agree on the outcome
      if (!__all_sync(0xFFFFFFFFu, mbar_wait_bounded(tail_landed_bar(buf), (tails >> 1) & 1u, abort_flag, WAIT_LIMIT_NS))) {
        role_failed = 8;
        break;
      }
      ++tails;
      uint8_t* at = smem_gen + C_::OFF_TAIL + buf * C_::TAIL_BYTES;
      for (int j = lane; j < (UMMA_K - left) * 8 * BOXES; j += 32) {
        const int piece = j & 7, box = (j >> 3) % BOXES, row = left + (j >> 3) / BOXES;
        *reinterpret_cast<uint4*>(at + box * 2048 + row * 128 + piece * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_cluster_release(map_to_cta(tail_cleared_bar(buf), 0)); else mbar_arrive(tail_cleared_bar(buf));
      }
    }
  } else if (warp >= EPI_WARP0) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;
    const int h = (warp - EPI_WARP0) >> 2;
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tempty0 = PAIR ? map_to_cta(tempty_bar(0), 0) : tempty_bar(0);
    uint8_t* staging = smem_gen + C_::OFF_STAGING + (warp - EPI_WARP0) * STAGING_BYTES_PER_WARP;
    const int es = p.out32 ? 4 : 2;
    const bool vec_ok = (static_cast<int64_t>(p.cols) * es) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.C) & 15u) == 0;
    bool ok = true;

    // 32 columns of this warp's 32 rows from registers to C.  64 bytes of each row at a time meet in shared memory (their
    // 16-byte pieces permuted against bank conflicts) and leave as whole pieces of 8 rows per instruction.
    auto store_chunk = [&](const float (&v)[CHUNK], uint8_t* c_row0, int rows_left, int col0) {
      // c_row0: element (first row of this warp, column 0); rows_left, p.cols: what exists
      const int passes = p.out32 ? 2 : 1;
      for (int ps = 0; ps < passes; ++ps) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 w;
          if (p.out32) {
            w = ps == 0 ? make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]))
                        : make_uint4(__float_as_uint(v[16 + 4 * j]), __float_as_uint(v[17 + 4 * j]), __float_as_uint(v[18 + 4 * j]), __float_as_uint(v[19 + 4 * j]));
          } else if (p.half) {
            w = make_uint4(Pack16<__nv_bfloat16>::from_f32(v[8 * j], v[8 * j + 1]), Pack16<__nv_bfloat16>::from_f32(v[8 * j + 2], v[8 * j + 3]),
                           Pack16<__nv_bfloat16>::from_f32(v[8 * j + 4], v[8 * j + 5]), Pack16<__nv_bfloat16>::from_f32(v[8 * j + 6], v[8 * j + 7]));
          } else {
            w = make_uint4(Pack16<__half>::from_f32(v[8 * j], v[8 * j + 1]), Pack16<__half>::from_f32(v[8 * j + 2], v[8 * j + 3]),
                           Pack16<__half>::from_f32(v[8 * j + 4], v[8 * j + 5]), Pack16<__half>::from_f32(v[8 * j + 6], v[8 * j + 7]));
          }
          *reinterpret_cast<uint4*>(staging + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = w;
        }
        __syncwarp();
        const int c0 = col0 + ps * 16;                      // first column of the 64 bytes
        const int per = 16 / es;                            // columns of one piece
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int r = it * 8 + (lane >> 2), piece = lane & 3;
          const uint4 w = *reinterpret_cast<const uint4*>(staging + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
          const int c = c0 + piece * per;
          if (r < rows_left && c < p.cols) {
            uint8_t* dst = c_row0 + (static_cast<int64_t>(r) * p.cols + c) * es;
            if (vec_ok && c + per <= p.cols) {
              *reinterpret_cast<uint4*>(dst) = w;
            } else {
              const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if (i < per && c + i < p.cols) {
                  if (p.out32) reinterpret_cast<uint32_t*>(dst)[i] = u[i & 3];
                  else reinterpret_cast<uint16_t*>(dst)[i] = static_cast<uint16_t>(i & 1 ? u[i >> 1] >> 16 : u[i >> 1] & 0xFFFFu);
                }
              }
            }
          }
        }
        __syncwarp();
      }
    };

    // 128 bytes of each of this warp's 32 rows (64 columns, or 32 of fp32) to shared memory in the tensor map's swizzle, and
    // from there as one tiled store, which stops at the edges of the group's matrix.  (Pieces of 64 bytes stored by the
    // threads themselves wrote an all-zero gradient of 268 MB in 64 us.)
    const uint32_t stage_addr = smem_u32(staging);
    auto staging_free = [&]() {  // the store before has read the staging buffer
      if (lane == 0) bulk_wait_read_all();
      __syncwarp();
    };
    auto put = [&](int j, const uint4& w) {  // piece j of this lane's row
      *reinterpret_cast<uint4*>(staging + lane * 128 + ((j ^ (lane & 7)) << 4)) = w;
    };
    auto send = [&](const Tile& t, int row0, int col) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(&maps.a[1], stage_addr, col, row0, t.g);
        bulk_commit_group();
      }
    };

    uint32_t chain = 0;
    for (int i = 0; ok && i < my_tiles; ++i) {
      const Tile t = tile_at(i);
      const int row0 = t.row + cta_rank * BM + q * 32;  // first row of this warp
      const int rows_left = p.rows - row0;
      uint8_t* c_row0 = static_cast<uint8_t*>(p.C) + (static_cast<int64_t>(t.g) * p.rows + row0) * p.cols * es;
      const int col0 = t.col + h * C_::CW;
      const bool here = rows_left > 0 && col0 < p.cols;  // this warp has something to write
      if (t.count == 0 && p.tma_store) {
        if (here) {
          staging_free();
#pragma unroll
          for (int j = 0; j < 8; ++j) put(j, make_uint4(0u, 0u, 0u, 0u));
          const int step = p.out32 ? 32 : 64;
          fence_proxy_async_smem();
          __syncwarp();
          for (int c = col0; c < min(col0 + C_::CW, p.cols); c += step) send(t, row0, c);
        }
        continue;
      }
      if (t.count == 0) {
        float zero[CHUNK];
#pragma unroll
        for (int j = 0; j < CHUNK; ++j) zero[j] = 0.0f;
        for (int c = 0; c < C_::NCH; ++c) store_chunk(zero, c_row0, rows_left, col0 + c * CHUNK);
        continue;
      }
      const uint32_t a = chain & 1u;
      if (!mbar_wait_bounded(tfull_bar(a), (chain >> 1) & 1u, abort_flag, WAIT_LIMIT_NS)) {
        ok = false;
        role_failed = 4;
        break;
      }
      ++chain;
      tc_fence_after_sync();
      const uint32_t tacc = tmem_base + lane_off + a * BN + h * C_::CW;
      auto release = [&]() {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * a);
      };
      if (!here) {
        release();
        continue;
      }
      if (p.tma_store) {
#pragma unroll
        for (int c = 0; c < C_::NCH; c += 2) {  // 64 columns at a time
          uint32_t raw[2][CHUNK];
          tmem_ld32(tacc + c * CHUNK, raw[0]);
          tmem_ld32(tacc + (c + 1) * CHUNK, raw[1]);
          tmem_wait_ld();
          if (c + 2 >= C_::NCH) release();
          const int col = col0 + c * CHUNK;
          if (p.out32) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              staging_free();
#pragma unroll
              for (int j = 0; j < 8; ++j) put(j, make_uint4(raw[u][4 * j], raw[u][4 * j + 1], raw[u][4 * j + 2], raw[u][4 * j + 3]));
              if (col + u * CHUNK < p.cols) send(t, row0, col + u * CHUNK);
            }
          } else {
            uint32_t w[CHUNK];
#pragma unroll
            for (int j = 0; j < CHUNK; ++j) {
              const float lo = __uint_as_float(raw[j / 16][2 * (j % 16)]), hi = __uint_as_float(raw[j / 16][2 * (j % 16) + 1]);
              w[j] = p.half ? Pack16<__nv_bfloat16>::from_f32(lo, hi) : Pack16<__half>::from_f32(lo, hi);
            }
            staging_free();
#pragma unroll
            for (int j = 0; j < 8; ++j) put(j, make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]));
            if (col < p.cols) send(t, row0, col);
          }
        }
        continue;
      }
      uint32_t raw[2][CHUNK];
      tmem_ld32(tacc, raw[0]);
#pragma unroll
      for (int c = 0; c < C_::NCH; ++c) {
        tmem_wait_ld();
        if (c + 1 < C_::NCH) tmem_ld32(tacc + (c + 1) * CHUNK, raw[(c + 1) & 1]); else release();
        float v[CHUNK];
#pragma unroll
        for (int j = 0; j < CHUNK; ++j) v[j] = __uint_as_float(raw[c & 1][j]);
        store_chunk(v, c_row0, rows_left, col0 + c * CHUNK);
      }
    }
  }

  // ---------------------------------------------------------------- tear-down
  if (warp >= EPI_WARP0 && lane == 0) bulk_wait_read_all();  // staged stores have left shared memory
  tc_fence_before_sync();
  __syncwarp();
  if constexpr (PAIR) cluster_sync_all(); else __syncthreads();
  if (role_failed != 0 && atomicCAS(&g_grouped_status[0], 0u, 1u) == 0u) {
    g_grouped_status[1] = blockIdx.x;
    g_grouped_status[2] = static_cast<uint32_t>(role_failed);
  }
  if (warp == 2) {
    tc_fence_after_sync();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS); else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}


// ==================================================================== host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(ptr);
    return static_cast<EncodeTiledFn>(nullptr);
  }();
  return fn;
}

// `rank` 2 or 3 dimensions of a tensor, innermost first, strides in elements; box 128 bytes wide, `box_rows` high.
int make_map(CUtensorMap* tm, int dtype, const void* base, int rank, const int64_t* dims, const int64_t* strides, int box_rows) {
  const bool f32 = dtype == TBIK_DTYPE_FP32;  // (results only) 32 wide: 128 bytes either way
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(TBIK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t d[3], s[2];
  cuuint32_t box[3] = {f32 ? 32u : 64u, static_cast<cuuint32_t>(box_rows), 1}, one[3] = {1, 1, 1};
  for (int i = 0; i < rank; ++i) d[i] = static_cast<cuuint64_t>(dims[i]);
  for (int i = 0; i + 1 < rank; ++i) s[i] = static_cast<cuuint64_t>(strides[i]) * (f32 ? 4 : 2);
  auto encode = [&]() {
    return fn(tm, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == TBIK_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
              static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, s, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
    // The first CUDA call of a host thread (a backward pass runs in one of its own): the runtime binds the device's
    // context when it is told the device, the driver call above does not.
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
  }
  if (r != CUDA_SUCCESS) {
    char msg[160];
    snprintf(msg, sizeof(msg), "cuTensorMapEncodeTiled failed with CUresult %d (%lld x %lld, stride %lld)", static_cast<int>(r),
             static_cast<long long>(dims[1]), static_cast<long long>(dims[0]), static_cast<long long>(strides[0]));
    return set_error(TBIK_ERR_CUDA, msg);
  }
  return TBIK_OK;
}

constexpr int kMaxDevices = 64;

// `most`: more tiles than that cannot exist
template <typename Kernel, typename P>
int launch(Kernel kernel, std::atomic<bool>* configured, size_t smem_max, size_t smem, bool pair, const Maps& maps, const P& p,
           int64_t most, int max_ctas, cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices || !configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_max));
    if (e != cudaSuccess) return set_cuda_error(e, "cudaFuncSetAttribute(grouped product)");
    if (dev >= 0 && dev < kMaxDevices) configured[dev].store(true, std::memory_order_release);
  }
  int ctas = sm_count();
  if (max_ctas > 0 && max_ctas < ctas) ctas = max_ctas;
  int64_t units = pair ? (ctas / 2 > 0 ? ctas / 2 : 1) : ctas;
  if (units > most) units = most > 0 ? most : 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(pair ? 2 * units : units));
  cfg.blockDim = dim3(NUM_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pair ? 2 : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pair ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps, p);
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, "grouped product launch");
}

template <int W_ROWS, int TN, int SUB, int STAGES, bool PAIR, bool W_MN, bool TREE>
int launch_forward(const Maps& maps, const ForwardParams& p, int64_t most, int max_ctas, cudaStream_t stream) {
  using C_ = ForwardCfg<W_ROWS, TN, SUB, STAGES, PAIR, W_MN>;
  static std::atomic<bool> configured[kMaxDevices];
  return launch(forward_kernel<W_ROWS, TN, SUB, STAGES, PAIR, W_MN, TREE>, configured, C_::smem_bytes(TBIK_MAX_GROUPS),
                C_::smem_bytes(p.groups), PAIR, maps, p, most, max_ctas, stream);
}

template <int BN, int STAGES, bool PAIR>
int launch_wgrad(const Maps& maps, const WgradParams& p, int64_t most, int max_ctas, cudaStream_t stream) {
  using C_ = WgradCfg<BN, STAGES, PAIR>;
  static std::atomic<bool> configured[kMaxDevices];
  return launch(wgrad_kernel<BN, STAGES, PAIR>, configured, C_::smem_bytes(TBIK_MAX_GROUPS), C_::smem_bytes(p.groups), PAIR,
                maps, p, most, max_ctas, stream);
}

bool bad_align(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check_common(const char* what, int64_t M, int N, int K, int groups, int dtype, int out_dtype) {
  char msg[160];
  if (dtype != TBIK_DTYPE_BF16 && dtype != TBIK_DTYPE_FP16) {
    snprintf(msg, sizeof(msg), "%s supports bf16 and fp16 operands", what);
    return set_error(TBIK_ERR_DTYPE, msg);
  }
  if (out_dtype != dtype && out_dtype != TBIK_DTYPE_FP32) {
    snprintf(msg, sizeof(msg), "%s: the result has the operand type or fp32", what);
    return set_error(TBIK_ERR_DTYPE, msg);
  }
  if (M < 0 || M >= (int64_t(1) << 31) - 256 || N < 0 || N >= (1 << 30) || K <= 0 || K >= (1 << 30)) {
    snprintf(msg, sizeof(msg), "%s: M below 2^31 - 256, N below 2^30, K in 1 .. 2^30 - 1", what);
    return set_error(TBIK_ERR_SHAPE, msg);
  }
  if (groups < 1 || groups > TBIK_MAX_GROUPS) {
    snprintf(msg, sizeof(msg), "%s: 1 .. %d groups", what, TBIK_MAX_GROUPS);
    return set_error(TBIK_ERR_SHAPE, msg);
  }
  return TBIK_OK;
}

// Tile shape of a forward product, from the sizes alone (the groups' sizes are on the device).
struct Shape {
  int w_rows, tokens;
  bool pair;
};
constexpr Shape kPair{128, 256, true}, kPairTree{128, 128, true}, kWide{128, 64, false}, kNarrow{32, 32, false};

Shape choose(int64_t M, int N, int groups, int T, int L) {
  // Tree levels above level 0 that the tensor-memory columns beside the accumulators hold: none, 2, 6 and 14.
  if (L - 1 > 6) return kNarrow;
  const int64_t rows = M / groups;  // per group, were they even
  if (rows >= 48 && L - 1 <= 2) return T == 1 ? kPair : kPairTree;
  // Few rows: W streams from HBM.  An instruction takes about 70 cycles however few rows and tokens it covers, so the full
  // 128 rows pay even where that leaves SMs without a tile.
  return kWide;
}

template <bool W_MN>
int forward(const Shape& c, const Maps& maps, const ForwardParams& p, int64_t most, int max_ctas, cudaStream_t stream) {
  if (c.pair && c.tokens == 256) return launch_forward<128, 256, 1, 6, true, W_MN, false>(maps, p, most, max_ctas, stream);
  if (c.pair) return launch_forward<128, 128, 1, 8, true, W_MN, true>(maps, p, most, max_ctas, stream);
  if (c.w_rows == 128) return launch_forward<128, 64, 2, 4, false, W_MN, true>(maps, p, most, max_ctas, stream);
  return launch_forward<32, 32, W_MN ? 2 : 4, W_MN ? 7 : 6, false, W_MN, true>(maps, p, most, max_ctas, stream);
}

}  // namespace

int sm_count() {
  static std::atomic<int> cached[kMaxDevices];
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) dev = 0;
  n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = 148;
    }
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int grouped_gemm(const void* A, const void* W, void* C, const int32_t* offsets, int64_t M, int N, int K, int groups,
                 int64_t lda, int64_t ldw, int64_t stride_w, int64_t ldc, int w_layout, int dtype, int out_dtype, int leaf,
                 int outside, int max_ctas, cudaStream_t stream) {
  int rc = check_common("tbik_grouped_gemm", M, N, K, groups, dtype, out_dtype);
  if (rc != TBIK_OK) return rc;
  if (w_layout != TBIK_W_K_CONTIGUOUS && w_layout != TBIK_W_N_CONTIGUOUS)
    return set_error(TBIK_ERR_ARG, "tbik_grouped_gemm: unknown layout of W");
  if (leaf < 0 || leaf % BK != 0 || (leaf > 0 && K % leaf != 0))
    return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm: leaf must be 0 or a multiple of 64 that divides K");
  int T = 1, F = 1, L = 1;
  if (leaf > 0) (void)tree_shape(K, leaf, &T, &F, &L);
  if (L > 15) return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm: at most 15 tree levels: use a wider leaf");
  if (M == 0 || N == 0) return TBIK_OK;
  if (!A || !W || !C || !offsets) return set_error(TBIK_ERR_ARG, "tbik_grouped_gemm: null pointer");
  const bool kc = w_layout == TBIK_W_K_CONTIGUOUS;
  const int64_t w_row = kc ? K : N, w_rows = kc ? N : K;
  // one group behind the other, or their rows in turn ([N, G, K] seen as [G, N, K]): a tensor map steps over either
  const bool behind = stride_w >= (w_rows - 1) * ldw + w_row, in_turn = stride_w >= w_row && ldw >= (groups - 1) * stride_w + w_row;
  if (lda < K || ldw < w_row || ldc < N || (groups > 1 && !behind && !in_turn))
    return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm: stride smaller than what it steps over");
  if (bad_align(A) || bad_align(W) || lda % 8 || ldw % 8 || stride_w % 8)
    return set_error(TBIK_ERR_ALIGN, "tbik_grouped_gemm: A and W must be 16-byte aligned with strides that are multiples of 8 elements");
  if (reinterpret_cast<uintptr_t>(C) % (out_dtype == TBIK_DTYPE_FP32 ? 4 : 2))
    return set_error(TBIK_ERR_ALIGN, "tbik_grouped_gemm: C must be aligned to its element size");

  const Shape c = choose(M, N, groups, T, L);
  Maps maps;
  const int64_t da[2] = {K, M}, sa[1] = {lda};
  for (int i = 0; i < 4; ++i) {
    rc = make_map(&maps.a[i], dtype, A, 2, da, sa, 16 << i);
    if (rc != TBIK_OK) return rc;
  }
  const int64_t dw[3] = {w_row, w_rows, groups}, sw[2] = {ldw, groups > 1 ? stride_w : w_rows * ldw};
  rc = make_map(&maps.b, dtype, W, 3, dw, sw, kc ? c.w_rows : BK);
  if (rc != TBIK_OK) return rc;

  ForwardParams p{};
  p.C = C;
  p.offsets = offsets;
  p.ldc = ldc;
  p.M = static_cast<int>(M);
  p.N = N;
  p.groups = groups;
  p.blocks_per_leaf = leaf > 0 ? leaf / BK : (K + BK - 1) / BK;
  p.T = T;
  p.F = F;
  p.L = L;
  const int w_tile = c.pair ? 2 * c.w_rows : c.w_rows;
  p.tiles_w = (N + w_tile - 1) / w_tile;
  p.half = dtype == TBIK_DTYPE_BF16 ? 1 : 0;
  p.out32 = out_dtype == TBIK_DTYPE_FP32 ? 1 : 0;
  p.zero_outside = outside;
  // token tiles: at most one ragged one per group that has rows
  const int64_t most = (M / c.tokens + (M < groups ? M : groups)) * p.tiles_w;
  if (most >= (int64_t(1) << 31)) return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm: too many tiles");
  return kc ? forward<false>(c, maps, p, most, max_ctas, stream) : forward<true>(c, maps, p, most, max_ctas, stream);
}

int grouped_gemm_wgrad(const void* dC, const void* A, void* dW, const int32_t* offsets, int64_t M, int N, int K, int groups,
                       int64_t lddc, int64_t lda, int dtype, int out_dtype, int max_ctas, cudaStream_t stream) {
  int rc = check_common("tbik_grouped_gemm_wgrad", M, N, K, groups, dtype, out_dtype);
  if (rc != TBIK_OK || N == 0) return rc;
  if (M == 0) return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm_wgrad: no rows: the gradient is zero");
  if (!dC || !A || !dW || !offsets) return set_error(TBIK_ERR_ARG, "tbik_grouped_gemm_wgrad: null pointer");
  if (lddc < N || lda < K) return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm_wgrad: leading dimension smaller than the row");
  if (bad_align(A) || bad_align(dC) || lda % 8 || lddc % 8)
    return set_error(TBIK_ERR_ALIGN, "tbik_grouped_gemm_wgrad: operands must be 16-byte aligned with row strides that are multiples of 8 elements");
  if (reinterpret_cast<uintptr_t>(dW) % (out_dtype == TBIK_DTYPE_FP32 ? 4 : 2))
    return set_error(TBIK_ERR_ALIGN, "tbik_grouped_gemm_wgrad: dW must be aligned to its element size");
  Maps maps;
  const int64_t dd[2] = {N, M}, sd[1] = {lddc}, da[2] = {K, M}, sa[1] = {lda};
  rc = make_map(&maps.a[0], dtype, dC, 2, dd, sd, BK);
  if (rc != TBIK_OK) return rc;
  maps.a[1] = maps.a[0];
  rc = make_map(&maps.a[2], dtype, dC, 2, dd, sd, UMMA_K);
  if (rc != TBIK_OK) return rc;
  rc = make_map(&maps.a[3], dtype, A, 2, da, sa, UMMA_K);
  if (rc != TBIK_OK) return rc;
  const int es = out_dtype == TBIK_DTYPE_FP32 ? 4 : 2;
  const bool tma_store = !bad_align(dW) && static_cast<int64_t>(K) * es % 16 == 0;
  if (tma_store) {
    const int64_t dw[3] = {K, N, groups}, sw[2] = {K, static_cast<int64_t>(N) * K};
    rc = make_map(&maps.a[1], out_dtype, dW, 3, dw, sw, 32);
    if (rc != TBIK_OK) return rc;
  }
  rc = make_map(&maps.b, dtype, A, 2, da, sa, BK);
  if (rc != TBIK_OK) return rc;
  const bool pair = N > BM && K > BM;
  const int bn = pair ? 256 : 128, tile_m = pair ? 2 * BM : BM;
  WgradParams p{};
  p.C = dW;
  p.offsets = offsets;
  p.M = static_cast<int>(M);
  p.groups = groups;
  p.rows = N;
  p.cols = K;
  p.tiles_r = (N + tile_m - 1) / tile_m;
  p.tiles_c = (K + bn - 1) / bn;
  p.half = dtype == TBIK_DTYPE_BF16 ? 1 : 0;
  p.out32 = out_dtype == TBIK_DTYPE_FP32 ? 1 : 0;
  p.tma_store = tma_store ? 1 : 0;
  const int64_t most = static_cast<int64_t>(groups) * p.tiles_r * p.tiles_c;
  if (most >= (int64_t(1) << 31)) return set_error(TBIK_ERR_SHAPE, "tbik_grouped_gemm_wgrad: too many tiles");
  return pair ? launch_wgrad<256, 5, true>(maps, p, most, max_ctas, stream) : launch_wgrad<128, 5, false>(maps, p, most, max_ctas, stream);
}

int grouped_status(uint32_t out[4]) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_grouped_status, sizeof(uint32_t) * 4);
  if (e != cudaSuccess) return set_cuda_error(e, "cudaMemcpyFromSymbol(g_grouped_status)");
  if (out[0] != 0) {
    const uint32_t zero[4] = {0, 0, 0, 0};
    cudaMemcpyToSymbol(g_grouped_status, zero, sizeof(zero));
  }
  return TBIK_OK;
}

}  // namespace tbik
