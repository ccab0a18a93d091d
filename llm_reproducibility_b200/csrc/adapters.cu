// Low-rank adapters of many requests beside a shared projection:
//
//   h[t]   = A_a x[t]                       fp32, K cut into at most 8 leaves, ((0+1)+(2+3))+((4+5)+(6+7))
//   out[t] = round(y[t] + s_a B_a h[t])     fp32, a = adapter of row t
//
// Both products are skinny (R = 8 .. 128), so what has to move is x, y, out and the adapters in use, and mma.sync m16n8k16 takes its
// operands straight from global memory -- no tensor-memory round trip for 16 columns (8192 rows, rank 32, K = N = 4096: 52 us, HBM
// 41 % busy, tensor pipe 37 %, issue slots 34 %: the loads that 14 warps per SM have in flight are the limit; rank 128: 180 us, tensor
// pipe 41 %).  The k index of an instruction may be permuted as long as both operands agree: a lane takes 8 neighbouring elements
// of its row as its share of two instructions, which makes every operand load 16 bytes wide; in the second product the columns are
// permuted the same way, so that a lane ends up with 8 neighbouring results.
//
// One cluster of 1 .. 8 CTAs per (adapter, tile of rows), both products in one launch.  The CTAs split K by leaves, add
// the leaves through distributed shared memory, and split N for the second product.  Few rows: 16-row tiles and
// asynchronous copies of a leaf into shared memory, so that a decode step pays one memory latency; many rows: 32-row tiles,
// whose warps take a leaf or a part of its columns of h each, operands straight into registers.  Either way a leaf is one
// chain of instructions over its columns, so a row's bits depend on the row and its adapter alone.
//
// h is held in fp32 and multiplied whole: the second product reads it as the sum of three values of the operand type, each the
// rounding of what the ones before leave (three times 8 bits for bf16, 11 for fp16, whose rows are scaled by a power of two
// into its range first), the smallest first.  Two values, 16 bits for bf16, lost the result's last bits where the adapter's
// terms or y nearly cancel; the third costs what its instructions cost (8192 rows, K = N = 4096: rank 32 51.7 -> 52.8 us, rank 64
// 80 -> 87, rank 128 137 -> 182).
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "ptx_sm100a.cuh"
#include "tbik_internal.h"

namespace tbik {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kLeaves = 8;
constexpr int kParts = 3;  // values of the operand type that make up one of h
// One of the two buffers of a staged leaf.  Three CTAs per SM for the usual ranks, whose leaf then comes in one piece (96 rows of 48
// adapters, rank 16, K = 12288: 24 KiB 18.5 us, 30 KiB 17.4 us, 36 KiB and two CTAs 22.6 us); more columns at a time for the large
// ones, of which two CTAs (rank 64) or one (rank 128) are resident.
__host__ __device__ constexpr uint32_t stage_bytes(int R) { return R <= 32 ? 30720 : 49152; }

struct Params {
  const void *x, *y, *A, *B;
  void* out;
  const float* scales;
  float* h;
  const int32_t *order, *offsets;
  int64_t T, ldx, ldy, ldo;
  int N, K, R, adapters, leaf;
  int cluster;     // CTAs per item
  int rest;        // rows of no adapter have work to do too (copy y, or zero h)
};

constexpr float kInf = __builtin_huge_valf();

template <bool B> struct Bool { static constexpr bool value = B; };
template <typename V> struct Four { V v[4]; };

template <typename T> struct Half;
template <> struct Half<__nv_bfloat16> {
  static constexpr float kLargest = 0x1.FEp127f;
  TBIK_DEVICE static float f32(uint32_t w, int hi) { return __uint_as_float(hi ? (w & 0xFFFF0000u) : (w << 16)); }
  TBIK_DEVICE static uint32_t pack(float lo, float hi) { return Pack16<__nv_bfloat16>::from_f32(lo, hi); }
  TBIK_DEVICE static float round(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
  TBIK_DEVICE static bool any_nan(const uint32_t (&w)[4]) {
    const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(w);
    const __nv_bfloat162 top = __hmax2_nan(__hmax2_nan(v[0], v[1]), __hmax2_nan(v[2], v[3]));
    return !__hbeq2(top, top);
  }
  TBIK_DEVICE static void mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  }
};
template <> struct Half<__half> {
  static constexpr float kLargest = 65504.0f;
  TBIK_DEVICE static float f32(uint32_t w, int hi) {
    const __half2 v = *reinterpret_cast<const __half2*>(&w);
    return hi ? __high2float(v) : __low2float(v);
  }
  TBIK_DEVICE static uint32_t pack(float lo, float hi) { return Pack16<__half>::from_f32(lo, hi); }
  TBIK_DEVICE static float round(float v) { return __half2float(__float2half_rn(v)); }
  TBIK_DEVICE static bool any_nan(const uint32_t (&w)[4]) {
    const __half2* v = reinterpret_cast<const __half2*>(w);
    const __half2 top = __hmax2_nan(__hmax2_nan(v[0], v[1]), __hmax2_nan(v[2], v[3]));
    return !__hbeq2(top, top);
  }
  TBIK_DEVICE static void mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  }
};

TBIK_DEVICE void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)) : "memory");
}
TBIK_DEVICE void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> TBIK_DEVICE void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// A row is read 64 bytes at a time by lanes of eight rows: L2 is asked for the 256 bytes around at once.
TBIK_DEVICE uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
TBIK_DEVICE void prefetch_l2(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(reinterpret_cast<uint64_t>(src)), "r"(bytes) : "memory");
}

TBIK_DEVICE float4 add(const float4& a, const float4& b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
TBIK_DEVICE int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Shared memory: [rows TM][item 4], at 512 [row factors TM] | leaf sums [8 / cluster][TM][R] | h [TM][R] |
// h as operand [TM / 16][ceil(R / 16)][32 lanes] x 48 bytes | two staging buffers
struct Layout {
  uint32_t sums, h, frags, stage, total;
};
template <int MT, bool STAGED>
__host__ __device__ inline Layout layout(int R, int cluster) {
  constexpr int TM = MT * 16;
  Layout l;
  l.sums = 1024;
  l.h = l.sums + (kLeaves / cluster) * TM * R * 4;
  l.frags = l.h + TM * R * 4;
  l.stage = (l.frags + MT * ((R + 15) / 16) * kParts * 512 + 127) / 128 * 128;
  l.total = l.stage + (STAGED ? 2 * stage_bytes(R) : 0);
  return l;
}

// Staged: three CTAs per SM are what shared memory leaves room for, and 80 registers (the case above 16.5 us; 64 registers, which would
// let a fourth in, 17.5 us: more spills).
template <typename T, int MT, bool STAGED>
__global__ void __launch_bounds__(kThreads, STAGED ? 3 : 2) adapters_kernel(const Params p) {
  constexpr int TM = MT * 16;  // rows of the tile
  extern __shared__ __align__(128) uint8_t smem[];
  const Layout lay = layout<MT, STAGED>(p.R, p.cluster);
  int* rows = reinterpret_cast<int*>(smem);                 // row index or -1
  int* item = rows + TM;                                    // adapter, first place, rows
  float* factor = reinterpret_cast<float*>(smem + 512);     // what a row of h was multiplied by (fp16)
  float* sums = reinterpret_cast<float*>(smem + lay.sums);
  float* hs = reinterpret_cast<float*>(smem + lay.h);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = p.cluster, rank = static_cast<int>(blockIdx.x) % C, want = static_cast<int>(blockIdx.x) / C;
  const int R = p.R, K = p.K;

  if (tid == 0) item[0] = -2;  // no item
  // ---- which adapter and rows: tiles of the groups in order, then tiles of the rows of no adapter
  {
    int* warp_sum = reinterpret_cast<int*>(smem + lay.sums);  // free until the leaves' sums
    const int all = static_cast<int>(p.T);
    const int per = ceil_div(p.adapters, kThreads);
    int first[4], count[4], mine = 0;                         // adapters <= 1024 = 4 x 256
    int carry = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int g = tid * per + u;
      first[u] = count[u] = 0;
      if (u < per && g < p.adapters) {
        const int lo = min(max(p.offsets[g], 0), all), hi = min(max(p.offsets[g + 1], lo), all);
        first[u] = lo;
        count[u] = hi - lo;
        mine += ceil_div(hi - lo, TM);
      }
    }
    int run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, run, o);
      if (lane >= o) run += v;
    }
    if (lane == 31) warp_sum[warp] = run;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) carry += warp_sum[w];
      total += warp_sum[w];
    }
    int at = carry + run - mine;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int tiles = ceil_div(count[u], TM);
      if (want >= at && want < at + tiles) {
        item[1] = first[u] + (want - at) * TM;
        item[2] = min(TM, first[u] + count[u] - item[1]);
        item[0] = tid * per + u;
      }
      at += tiles;
    }
    if (p.rest && tid == 0 && want >= total) {
      const int lo = min(max(p.offsets[0], 0), all), hi = min(max(p.offsets[p.adapters], lo), all);
      const int i = (want - total) * TM;  // i-th row of no adapter
      if (i < lo + all - hi) {
        item[0] = -1;
        item[1] = i;
        item[2] = min(TM, lo + all - hi - i);
        item[3] = lo;
      }
    }
    __syncthreads();
  }
  const int adapter = item[0], place = item[1], count = item[2];
  if (adapter < -1) return;  // the whole cluster has no item
  if (tid < TM) {
    int t = -1;
    if (tid < count) {
      int at = place + tid;
      if (adapter < 0 && at >= item[3]) at += min(max(p.offsets[p.adapters], item[3]), static_cast<int>(p.T)) - item[3];
      t = p.order[at];
      if (t < 0 || t >= p.T) t = -1;
    }
    rows[tid] = t;
  }
  __syncthreads();
  const bool shrink = p.x != nullptr, expand = p.y != nullptr;

  if (adapter < 0) {
    // rows of no adapter: out = y, or h = 0
    for (int i = warp * C + rank; i < count; i += kWarps * C) {
      const int t = rows[i];
      if (t < 0) continue;
      if (expand) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.y) + static_cast<int64_t>(t) * p.ldy);
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + static_cast<int64_t>(t) * p.ldo);
        for (int c0 = lane; c0 < p.N / 8; c0 += 32 * 8) {  // eight pieces in flight
          uint4 v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (c0 + u * 32 < p.N / 8) v[u] = src[c0 + u * 32];
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (c0 + u * 32 < p.N / 8) dst[c0 + u * 32] = v[u];
        }
      } else {
        for (int r = lane; r < R; r += 32) p.h[static_cast<int64_t>(t) * R + r] = 0.0f;
      }
    }
    return;
  }

  const int g = lane >> 2, c = lane & 3;  // the lane's row (and row + 8) and its place in a row
  const int nblocks = ceil_div(p.N, 32);
  const T* B = static_cast<const T*>(p.B) + static_cast<int64_t>(adapter) * p.N * R;

  // ---- first product
  if (shrink) {
    const T* A = static_cast<const T*>(p.A) + static_cast<int64_t>(adapter) * R * K;
    const T* x = static_cast<const T*>(p.x);
    const int own = kLeaves / C;  // leaves of this CTA
    const int ntiles = R / 8;
    if (STAGED && expand && warp == 1) {
      // this CTA's share of B and of the rows of y is wanted right after: on its way to L2 meanwhile
      const int per = ceil_div(nblocks, C) * 32, n0 = min(rank * per, p.N), n1 = min(n0 + per, p.N);
      if (lane == 0 && n1 > n0) prefetch_l2(B + static_cast<int64_t>(n0) * R, static_cast<uint32_t>(n1 - n0) * R * 2);
      if (lane < TM && n1 > n0 && rows[lane] >= 0)
        prefetch_l2(static_cast<const T*>(p.y) + static_cast<int64_t>(rows[lane]) * p.ldy + n0, static_cast<uint32_t>(n1 - n0) * 2);
    }
    if constexpr (STAGED) {
      // A buffer holds `cols` columns of the adapter's R rows and of the tile's `count` rows: the whole leaf where it fits in
      // both buffers together, else alternating halves.  A row's pitch is 64 bytes off a multiple of 128, so that the
      // 16-byte pieces that 8 lanes read together lie in different banks.
      const uint32_t stage = stage_bytes(R), lines = static_cast<uint32_t>(R + count);
      const int whole = (p.leaf + 63) / 64 * 64;
      const bool once = whole <= static_cast<int>((2 * stage / lines - 64) / 2);
      const int cols = once ? whole : static_cast<int>((stage / lines - 64) / 128 * 64);
      const uint32_t pitch = static_cast<uint32_t>(cols) * 2 + 64, second = once ? 0u : stage;
      const int per_leaf = ceil_div(p.leaf, cols), steps = own * per_leaf, ahead = once ? 1 : 2;
      auto range = [&](int s, int& k0, int& k1) {
        const int l = rank * own + s / per_leaf;
        const int64_t b = static_cast<int64_t>(l) * p.leaf, e = min(b + p.leaf, static_cast<int64_t>(K));
        const int64_t f = min(b + static_cast<int64_t>(s % per_leaf) * cols, e);
        k0 = static_cast<int>(f);
        k1 = max(static_cast<int>(min(f + cols, e)), k0);
      };
      // A warp per row, 16 bytes per lane; one group of asynchronous copies per step, empty or not.
      auto load = [&](int s) {
        int k0, k1;
        range(s, k0, k1);
        const uint32_t buf = smem_u32(smem + lay.stage) + (s & 1) * second;
        for (int i = warp; i < R + count; i += kWarps) {
          const int t = i < R ? 0 : rows[i - R];
          if (t < 0) continue;
          const T* src = (i < R ? A + static_cast<int64_t>(i) * K : x + static_cast<int64_t>(t) * p.ldx) + k0;
          for (int k = lane * 8; k < k1 - k0; k += 256) copy16(buf + i * pitch + k * 2, src + k);
        }
        copy_commit();
      };
      load(0);
      if (ahead == 2 && steps > 1) load(1);
      // Rows of the instruction beyond the tile repeat its last one: a row's results depend on no other row, and theirs are
      // not read.  Columns between the end of K and the next multiple of 32 are cleared below.
      const int row0 = R + min(g, count - 1), row1 = R + min(g + 8, count - 1);
      float acc[2][4];  // this warp's column tiles: warp, warp + 8
      auto chain = [&](const uint8_t* buf, int n, auto two) {
        const uint8_t *x0 = buf + row0 * pitch + c * 16, *x1 = buf + row1 * pitch + c * 16, *b0 = buf + (warp * 8 + g) * pitch + c * 16;
#pragma unroll 4
        for (int k = 0; k < n; k += 32) {
          const uint4 a0 = *reinterpret_cast<const uint4*>(x0 + k * 2), a1 = *reinterpret_cast<const uint4*>(x1 + k * 2);
          const uint4 b = *reinterpret_cast<const uint4*>(b0 + k * 2);
          Half<T>::mma(acc[0], make_uint4(a0.x, a1.x, a0.y, a1.y), b.x, b.y);
          Half<T>::mma(acc[0], make_uint4(a0.z, a1.z, a0.w, a1.w), b.z, b.w);
          if constexpr (decltype(two)::value) {
            const uint4 d = *reinterpret_cast<const uint4*>(b0 + 64 * pitch + k * 2);
            Half<T>::mma(acc[1], make_uint4(a0.x, a1.x, a0.y, a1.y), d.x, d.y);
            Half<T>::mma(acc[1], make_uint4(a0.z, a1.z, a0.w, a1.w), d.z, d.w);
          }
        }
      };
      for (int s = 0; s < steps; ++s) {
        int k0, k1;
        range(s, k0, k1);
        if (s % per_leaf == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
        }
        if (ahead == 2 && s + 1 < steps) copy_wait<1>(); else copy_wait<0>();
        uint8_t* buf = smem + lay.stage + (s & 1) * second;
        const int n = k1 - k0, pad = (32 - n % 32) % 32 / 8;  // 16-byte pieces to clear per row
        if (pad > 0)
          for (int i = tid; i < (R + count) * pad; i += kThreads)
            *reinterpret_cast<uint4*>(buf + i / pad * pitch + n * 2 + i % pad * 16) = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        if (warp + 8 < ntiles) chain(buf, n, Bool<true>{});
        else if (warp < ntiles) chain(buf, n, Bool<false>{});
        if ((s + 1) % per_leaf == 0) {
          float* out = sums + (s / per_leaf) * TM * R;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n8 = (warp + 8 * i) * 8 + c * 2;
            if (warp + 8 * i < ntiles) {
              *reinterpret_cast<float2*>(out + g * R + n8) = make_float2(acc[i][0], acc[i][1]);
              *reinterpret_cast<float2*>(out + (g + 8) * R + n8) = make_float2(acc[i][2], acc[i][3]);
            }
          }
        }
        if (s + ahead < steps) {
          __syncthreads();  // everyone is done with the buffer
          load(s + ahead);
        }
      }
    } else {
      // Eight leaves and eight warps: a warp takes one, or with C CTAs every C-th column tile of one.
      static_assert(kWarps == kLeaves, "a warp per leaf");
      const int slot = warp / C, parts = C, part = warp % C;
      const int leaf = rank * own + slot;
      const int64_t kb = min(static_cast<int64_t>(leaf) * p.leaf, static_cast<int64_t>(K));
      const int k0 = static_cast<int>(kb), k1 = static_cast<int>(min(kb + p.leaf, static_cast<int64_t>(K)));
      // rows and column tiles beyond what there is repeat the last one; their results are not read
      const T* xr[2 * MT];
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) xr[i] = x + static_cast<int64_t>(max(rows[min(i * 8 + g, count - 1)], 0)) * p.ldx + c * 8;
      float* out = sums + slot * TM * R;
      for (int n0 = part; n0 < ntiles; n0 += 4 * parts) {
        float acc[MT][4][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[m][i][j] = 0.0f;
        const T* ar[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ar[i] = A + static_cast<int64_t>(min(n0 + i * parts, ntiles - 1) * 8 + g) * K + c * 8;
        // `in`: the lane's piece of the run of 32 columns exists
        auto load = [&](int k, bool in, uint4 (&a)[2 * MT], uint4 (&b)[4]) {
#pragma unroll
          for (int i = 0; i < 2 * MT; ++i) a[i] = in ? load_stream(xr[i] + k) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int i = 0; i < 4; ++i) b[i] = in ? __ldg(reinterpret_cast<const uint4*>(ar[i] + k)) : make_uint4(0u, 0u, 0u, 0u);
        };
        auto multiply = [&](const uint4 (&a)[2 * MT], const uint4 (&b)[4]) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) Half<T>::mma(acc[m][i], make_uint4(a[2 * m].x, a[2 * m + 1].x, a[2 * m].y, a[2 * m + 1].y), b[i].x, b[i].y);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) Half<T>::mma(acc[m][i], make_uint4(a[2 * m].z, a[2 * m + 1].z, a[2 * m].w, a[2 * m + 1].w), b[i].z, b[i].w);
        };
        // The next run is on its way while one is multiplied; whole runs go without a thought for the end of the leaf (1500 rows,
        // rank 32, K = 12288: 41 us, without this loop 45; 8192 rows, K = 4096: 53 and 52).
        uint4 a[2][2 * MT], b[2][4];
        load(k0, k0 + c * 8 < k1, a[0], b[0]);
        int k = k0;
#pragma unroll 1
        for (; k + 96 <= k1; k += 64) {
          load(k + 32, true, a[1], b[1]);
          multiply(a[0], b[0]);
          load(k + 64, true, a[0], b[0]);
          multiply(a[1], b[1]);
        }
#pragma unroll 1
        for (; k < k1; k += 64) {
          if (k + 32 < k1) load(k + 32, k + 32 + c * 8 < k1, a[1], b[1]);
          multiply(a[0], b[0]);
          if (k + 32 < k1) {
            if (k + 64 < k1) load(k + 64, k + 64 + c * 8 < k1, a[0], b[0]);
            multiply(a[1], b[1]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (n0 + i * parts < ntiles) {
            const int n = (n0 + i * parts) * 8 + c * 2;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              *reinterpret_cast<float2*>(out + (m * 16 + g) * R + n) = make_float2(acc[m][i][0], acc[m][i][1]);
              *reinterpret_cast<float2*>(out + (m * 16 + g + 8) * R + n) = make_float2(acc[m][i][2], acc[m][i][3]);
            }
          }
        }
      }
    }
    // ---- the leaves' sums: this CTA's own first, a subtree of theirs, then one node from each CTA of the cluster
    cg::cluster_group cluster = cg::this_cluster();
    if (own > 1) {
      __syncthreads();
      for (int i = tid; i < TM * R / 4; i += kThreads) {
        float4 s[kLeaves];
#pragma unroll
        for (int l = 0; l < kLeaves; ++l)
          if (l < own) s[l] = reinterpret_cast<const float4*>(sums + l * TM * R)[i];
#pragma unroll
        for (int d = 1; d < kLeaves; d *= 2)
#pragma unroll
          for (int l = 0; l < kLeaves; l += 2 * d)
            if (l + d < own) s[l] = add(s[l], s[l + d]);
        reinterpret_cast<float4*>(C > 1 ? sums : hs)[i] = s[0];
      }
    }
    if (C > 1) {
      cluster.sync();
      for (int i = tid; i < TM * R / 4; i += kThreads) {
        float4 s[kLeaves];
#pragma unroll
        for (int c = 0; c < kLeaves; ++c)
          if (c < C) s[c] = reinterpret_cast<const float4*>(cluster.map_shared_rank(sums, c))[i];
#pragma unroll
        for (int d = 1; d < kLeaves; d *= 2)
#pragma unroll
          for (int c = 0; c < kLeaves; c += 2 * d)
            if (c + d < C) s[c] = add(s[c], s[c + d]);
        reinterpret_cast<float4*>(hs)[i] = s[0];
      }
    }
    if (C > 1) cluster.sync(); else __syncthreads();  // nobody leaves while its sums may still be read
    if (!expand) {
      for (int i = tid; i < TM * R / 4; i += kThreads) {
        const int t = rows[i / (R / 4)];
        if (t >= 0 && i / (R / 4) % C == rank)
          reinterpret_cast<float4*>(p.h + static_cast<int64_t>(t) * R)[i % (R / 4)] = reinterpret_cast<const float4*>(hs)[i];
      }
      return;
    }
  } else {
    for (int i = tid; i < TM * R / 4; i += kThreads) {
      const int t = rows[i / (R / 4)];
      reinterpret_cast<float4*>(hs)[i] = t >= 0 ? reinterpret_cast<const float4*>(p.h + static_cast<int64_t>(t) * R)[i % (R / 4)]
                                               : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    __syncthreads();
  }

  // ---- h as an operand: its parts, arranged per lane
  constexpr bool kScaled = sizeof(T) == 2 && Pack16<T>::kUmmaFmt == 0;  // fp16
  if constexpr (kScaled) {
    for (int i = warp; i < TM; i += kWarps) {
      float top = 0.0f;
      for (int r = lane; r < R; r += 32) top = fmaxf(top, fabsf(hs[i * R + r]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      // the largest of the row to about 2^14; 0 and infinity as they are
      int e = 0;
      if (top > 0.0f && top < kInf) e = min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 100);
      if (lane == 0) factor[i] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    }
    __syncthreads();
  }
  // Instruction s of a run of 16 columns of h: lane c's four columns.  Where R is a multiple of 32 the lane's columns of two
  // instructions are 8 neighbours, so that its piece of a row of B is 16 bytes; else it is 8.
  const bool wide = R % 32 == 0;
  auto column = [&](int s, int at) { return wide ? 32 * (s >> 1) + 8 * at + 4 * (s & 1) : 16 * s + 4 * at; };
  uint4* frags = reinterpret_cast<uint4*>(smem + lay.frags);
  const int ksteps = (R + 15) / 16;
  for (int i = tid; i < MT * ksteps * 32; i += kThreads) {
    const int ln = i & 31, s = (i >> 5) % ksteps, m = (i >> 5) / ksteps;
    const int r = column(s, ln & 3);
    uint32_t part[kParts][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // rows ln / 4 and + 8
      const int row = m * 16 + (ln >> 2) + 8 * u;
      const float4 v = r < R ? *reinterpret_cast<const float4*>(hs + row * R + r) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float left[4] = {v.x, v.y, v.z, v.w};
      if constexpr (kScaled) {
        const float f = factor[row];
#pragma unroll
        for (int j = 0; j < 4; ++j) left[j] *= f;
      }
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          t[j] = Half<T>::round(left[j]);
          // a number beyond the type's largest starts with that one; infinity and NaN have no further parts
          if (fabsf(t[j]) == kInf && fabsf(left[j]) < kInf) t[j] = copysignf(Half<T>::kLargest, left[j]);
          left[j] = fabsf(t[j]) < kInf ? left[j] - t[j] : 0.0f;
        }
        part[k][u] = Half<T>::pack(t[0], t[1]);
        part[k][u + 2] = Half<T>::pack(t[2], t[3]);
      }
    }
#pragma unroll
    for (int k = 0; k < kParts; ++k) frags[kParts * i + k] = make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
  }
  __syncthreads();

  // ---- second product, 32 columns per warp and trip
  const float scale = p.scales[adapter];
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out);
  const int per = ceil_div(nblocks, C), b1 = min((rank + 1) * per, nblocks);
  int row[2 * MT];
  [[maybe_unused]] float s_row[kScaled ? 2 * MT : 1];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    row[i] = i * 8 + g < count ? rows[i * 8 + g] : -1;
    if constexpr (kScaled) s_row[i] = scale / factor[i * 8 + g];  // a power of two: exact
  }
  auto load_y = [&](int blk, uint4 (&v)[2 * MT]) {
    const int col = blk * 32 + c * 8;  // the lane's 8 columns
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i)
      if (col < p.N && row[i] >= 0) v[i] = *reinterpret_cast<const uint4*>(y + row[i] * p.ldy + col);
  };
  // row of B, i.e. column of the result, that this lane brings for instruction j: 8 (g / 2) + 2 j + g % 2 (N is a multiple of 8:
  // all four are in or out, and where they are out their results are not stored)
  auto row_of_b = [&](int blk) {
    const int n0 = blk * 32 + 8 * (g >> 1) + (g & 1);
    return B + static_cast<int64_t>(n0 < p.N ? n0 : 0) * R;
  };
  auto load_wide = [&](int blk, int s2, uint4 (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __ldg(reinterpret_cast<const uint4*>(row_of_b(blk) + 2 * j * R + 32 * s2 + 8 * c));
  };
  auto load_narrow = [&](int blk, int s, uint2 (&v)[4]) {
    const bool ok = 16 * s + 4 * c < R;  // R may end inside the run
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = ok ? __ldg(reinterpret_cast<const uint2*>(row_of_b(blk) + 2 * j * R + 16 * s + 4 * c)) : make_uint2(0u, 0u);
  };
  // acc += rows 16 m .. of h, run s, times the four instructions' operands
  auto multiply = [&](int m, int s, const uint2 (&v)[4], float (&acc)[4][4]) {
#pragma unroll
    for (int k = kParts - 1; k >= 0; --k) {
      const uint4 part = frags[kParts * ((m * ksteps + s) * 32 + lane) + k];
#pragma unroll
      for (int j = 0; j < 4; ++j) Half<T>::mma(acc[j], part, v[j].x, v[j].y);
    }
  };
  auto multiply_wide = [&](int m, int s2, const uint4 (&v)[4], float (&acc)[4][4]) {
    const uint2 lo8[4] = {{v[0].x, v[0].y}, {v[1].x, v[1].y}, {v[2].x, v[2].y}, {v[3].x, v[3].y}};
    const uint2 hi8[4] = {{v[0].z, v[0].w}, {v[1].z, v[1].w}, {v[2].z, v[2].w}, {v[3].z, v[3].w}};
    multiply(m, 2 * s2, lo8, acc);
    multiply(m, 2 * s2 + 1, hi8, acc);
  };
  auto finish = [&](int blk, int m, const uint4 (&yv)[2 * MT], const float (&acc)[4][4]) {
    const int col = blk * 32 + c * 8;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = 2 * m + u;
      if (col >= p.N || row[i] < 0) continue;
      const float s = kScaled ? s_row[kScaled ? i : 0] : scale;
      const uint32_t yw[4] = {yv[i].x, yv[i].y, yv[i].z, yv[i].w};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = Half<T>::pack(fmaf(s, acc[j][2 * u], Half<T>::f32(yw[j], 0)), fmaf(s, acc[j][2 * u + 1], Half<T>::f32(yw[j], 1)));
      T* dst = out + row[i] * p.ldo + col;
      if (!Half<T>::any_nan(o)) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
        continue;
      }
      // An infinite entry of B against a part of h that is zero, or against parts of either sign, is NaN where their sum
      // times it is not: such elements are taken again from h itself.  (In place, y is read just before it is written.)
      const T* yp = y + row[i] * p.ldy + col;
#pragma unroll 1
      for (int q = 0; q < 8; ++q) {
        const uint32_t w = q < 4 ? (q < 2 ? o[0] : o[1]) : (q < 6 ? o[2] : o[3]);
        float v = Half<T>::f32(w, q & 1);
        if (v != v) {
          const float* hr = hs + (i * 8 + g) * R;
          const T* br = B + static_cast<int64_t>(col + q) * R;
          float sum = 0.0f;
#pragma unroll 1
          for (int r = 0; r < R; ++r) sum = fmaf(hr[r], static_cast<float>(br[r]), sum);
          v = fmaf(scale, sum, static_cast<float>(yp[q]));
        }
        dst[q] = static_cast<T>(v);
      }
    }
    __syncwarp();  // (the instructions of the next trip are the warp's)
  };
  auto clear = [](float (&acc)[4][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  };
  const int b0 = rank * per + warp;
  bool done = false;
  if constexpr (!STAGED) {
    if (R <= 16 || R == 32) {
      // h in one load of B per trip: the next trip's y and B are on their way while one is multiplied
      auto run = [&](auto load_b, auto times, auto sample) {
        uint4 yv[2][2 * MT];
        decltype(sample) bv[2];
        auto trip = [&](int blk, int at) {
          if (blk + kWarps < b1) {
            load_y(blk + kWarps, yv[1 - at]);
            load_b(blk + kWarps, bv[1 - at].v);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            float acc[4][4];
            clear(acc);
            times(m, bv[at].v, acc);
            finish(blk, m, yv[at], acc);
          }
        };
        if (b0 < b1) {
          load_y(b0, yv[0]);
          load_b(b0, bv[0].v);
        }
#pragma unroll 1
        for (int blk = b0; blk < b1; blk += 2 * kWarps) {
          trip(blk, 0);
          if (blk + kWarps < b1) trip(blk + kWarps, 1);
        }
      };
      if (R == 32) run([&](int blk, uint4 (&v)[4]) { load_wide(blk, 0, v); }, [&](int m, const uint4 (&v)[4], float (&acc)[4][4]) { multiply_wide(m, 0, v, acc); }, Four<uint4>{});
      else run([&](int blk, uint2 (&v)[4]) { load_narrow(blk, 0, v); }, [&](int m, const uint2 (&v)[4], float (&acc)[4][4]) { multiply(m, 0, v, acc); }, Four<uint2>{});
      done = true;
    }
  } else if (R <= 16) {  // a trip or two: nothing to run ahead of
#pragma unroll 1
    for (int blk = b0; blk < b1; blk += kWarps) {
      uint4 yv[2 * MT];
      uint2 v[4];
      load_y(blk, yv);
      load_narrow(blk, 0, v);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float acc[4][4];
        clear(acc);
        multiply(m, 0, v, acc);
        finish(blk, m, yv, acc);
      }
    }
    done = true;
  }
  if (!done) {
#pragma unroll 1
    for (int blk = b0; blk < b1; blk += kWarps) {
      uint4 yv[2 * MT];
      load_y(blk, yv);
      float acc[MT][4][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) clear(acc[m]);
      if (wide) {
#pragma unroll 2
        for (int s2 = 0; s2 < ksteps / 2; ++s2) {
          uint4 v[4];
          load_wide(blk, s2, v);
#pragma unroll
          for (int m = 0; m < MT; ++m) multiply_wide(m, s2, v, acc[m]);
        }
      } else {
#pragma unroll 2
        for (int s = 0; s < ksteps; ++s) {
          uint2 v[4];
          load_narrow(blk, s, v);
#pragma unroll
          for (int m = 0; m < MT; ++m) multiply(m, s, v, acc[m]);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) finish(blk, m, yv, acc[m]);
    }
  }
}

// ---------------------------------------------------------------- host side
constexpr int kMaxDevices = 64;

// A launch of `items` clusters; the kernel may use as much shared memory as there is.
template <typename T, int MT, bool STAGED>
int configure(int R, int cluster, int64_t items, cudaStream_t stream, cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr) {
  static std::atomic<bool> configured[kMaxDevices];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices || !configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(adapters_kernel<T, MT, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return set_cuda_error(e, "cudaFuncSetAttribute(adapters_kernel)");
    if (dev >= 0 && dev < kMaxDevices) configured[dev].store(true, std::memory_order_release);
  }
  *cfg = cudaLaunchConfig_t{};
  cfg->gridDim = dim3(static_cast<unsigned>(items * cluster));
  cfg->blockDim = dim3(kThreads);
  cfg->dynamicSmemBytes = layout<MT, STAGED>(R, cluster).total;
  cfg->stream = stream;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = static_cast<unsigned>(cluster);
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg->attrs = attr;
  cfg->numAttrs = 1;
  return TBIK_OK;
}

template <typename T, int MT, bool STAGED>
int launch(const Params& p, int64_t items, cudaStream_t stream) {
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  const int rc = configure<T, MT, STAGED>(p.R, p.cluster, items, stream, &cfg, &attr);
  if (rc != TBIK_OK) return rc;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, adapters_kernel<T, MT, STAGED>, p);
  return e == cudaSuccess ? TBIK_OK : set_cuda_error(e, "adapters_kernel launch");
}

// Clusters of staged CTAs that the device holds at once, asked once per device, rank and cluster (0: it could not be asked).
template <typename T>
int resident(int R, int cluster) {
  static std::atomic<int> known[kMaxDevices][TBIK_MAX_RANK / 8][2];
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  const bool keep = dev >= 0 && dev < kMaxDevices;
  if (keep) n = known[dev][R / 8 - 1][cluster == 8].load(std::memory_order_relaxed);
  if (n > 0) return n - 1;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  if (configure<T, 1, true>(R, cluster, 1, nullptr, &cfg, &attr) != TBIK_OK) return 0;
  if (cudaOccupancyMaxActiveClusters(&n, adapters_kernel<T, 1, true>, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  if (keep) known[dev][R / 8 - 1][cluster == 8].store(n + 1, std::memory_order_relaxed);
  return n;
}

template <typename T>
int choose_and_launch(Params p, cudaStream_t stream) {
  const bool shrink = p.x != nullptr, expand = p.y != nullptr;
  const int R = p.R, N = p.N, K = p.K;
  const int64_t rows = p.T, groups = rows < p.adapters ? rows : p.adapters;
  // Tiles of 16 rows from shared memory, for few rows that are done in one wave: its chain of latencies once, eight CTAs per tile, or
  // four up to rank 32.  What rows can be expected to make, drawn from `adapters`: one tile per adapter in use, or every adapter's
  // last one half full (the grid has room for the most that there can be).  K = N = 4096, staged and straight: 96 rows of 48
  // adapters, rank 32 18 and 23 us, rank 64 (not one wave) 36 and 31, rank 128 87 and 43; 300 rows of 48, rank 32 19 and 23; 64 rows
  // of 32 adapters, rank 64 21 and 30; 300 rows of 1000, rank 16 42 and 32.  What few rows are: 8 adapters, rank 16, 1000 rows 17
  // and 23, 1500 rows 20 and 23 (K = 512: 18 and 14); rank 32, 500 rows 17 and 25.
  if (rows <= (R <= 16 ? 1024 : 512)) {
    const double used = p.adapters * -std::expm1(-static_cast<double>(rows) / p.adapters);
    const int tiles = static_cast<int>(std::max(used, rows / 16.0 + used / 2) + 0.5);
    for (p.cluster = kLeaves; p.cluster >= (R <= 32 ? 4 : kLeaves); p.cluster /= 2)
      if (tiles <= resident<T>(R, p.cluster)) return launch<T, 1, true>(p, rows / 16 + groups + p.rest, stream);
  }
  // Tiles of 32 rows, straight.  No more CTAs than one wave of two per SM, and few per tile, because the eight warps of a CTA that has
  // fewer leaves share a leaf by columns of h and each reads all of x: two (1500 rows, rank 32, K = 12288, N = 4096: 39 us, with four
  // 43), one where K is long (3000 rows, K = 6 N: 46 us, with two 59), eight for a wide result (1100 rows, N = 8 K: 23 us, with two 28);
  // with large ranks a warp has that many passes over x to share.  The first product alone is the case of a long K (600 rows, rank
  // 32, K = 4096: one, two and four CTAs 11.9, 12.4 and 12.1 us; 4000 rows 13.3, 16.7 and 31.7), the second alone that of a wide
  // result (N = 4096, two, four and eight: 600 rows 13.5, 8.8 and 7.7 us; 2000 rows, where eight are more than a wave, 14.8, 12.8 and
  // 16.7).  The leaves' sums have to leave room for the second CTA.
  const int64_t items = rows / 32 + groups + p.rest, most = 2 * sm_count();
  const int cap = !shrink || (expand && N >= 4 * K) ? kLeaves : std::max(!expand || K >= 4 * N ? 1 : 2, R / 32);
  p.cluster = 1;
  while (p.cluster < kLeaves && ((p.cluster < cap && items * p.cluster * 2 <= most) || kLeaves / p.cluster * R > 512)) p.cluster *= 2;
  return launch<T, 2, false>(p, items, stream);
}

bool bad_align(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace

int adapters(const void* x, int64_t ldx, const void* y, int64_t ldy, void* out, int64_t ldo, const void* A, const void* B,
             const float* scales, float* h, const int32_t* order, const int32_t* offsets, int64_t T, int N, int K, int R,
             int adapters, int dtype, int leaf, cudaStream_t stream) {
  if (dtype != TBIK_DTYPE_BF16 && dtype != TBIK_DTYPE_FP16) return set_error(TBIK_ERR_DTYPE, "tbik_adapters supports bf16 and fp16");
  if (T < 0 || T >= (int64_t(1) << 25) || N < 8 || N % 8 || N >= (1 << 24) || K < 8 || K % 8 || K >= (1 << 24))
    return set_error(TBIK_ERR_SHAPE, "tbik_adapters: T in 0 .. 2^25 - 1, N and K positive multiples of 8 below 2^24");
  if (R < 8 || R % 8 || R > TBIK_MAX_RANK) return set_error(TBIK_ERR_SHAPE, "tbik_adapters: R must be a multiple of 8 up to 128");
  if (adapters < 1 || adapters > TBIK_MAX_GROUPS) return set_error(TBIK_ERR_SHAPE, "tbik_adapters: 1 .. 1024 adapters");
  if (leaf == 0) leaf = (K + 255) / 256 * 32;
  if (leaf < 0 || leaf % 32 || (static_cast<int64_t>(K) + leaf - 1) / leaf > kLeaves)
    return set_error(TBIK_ERR_SHAPE, "tbik_adapters: leaf must be a multiple of 32 with at most 8 leaves covering K");
  leaf = std::min(leaf, (K + 31) / 32 * 32);  // one leaf of all K, however wide it was said to be
  if (T == 0) return TBIK_OK;
  const bool shrink = x != nullptr, expand = y != nullptr;
  if (!order || !offsets || (!shrink && !expand) || (shrink && !A) || (expand && (!out || !B || !scales)) || (shrink != expand && !h))
    return set_error(TBIK_ERR_ARG, "tbik_adapters: null pointer");
  if ((shrink && ldx < K) || (expand && (ldy < N || ldo < N)))
    return set_error(TBIK_ERR_SHAPE, "tbik_adapters: row stride smaller than the row");
  if (bad_align(x) || bad_align(y) || bad_align(out) || bad_align(A) || bad_align(B) || bad_align(h) || ldx % 8 || ldy % 8 || ldo % 8)
    return set_error(TBIK_ERR_ALIGN, "tbik_adapters: pointers must be 16-byte aligned, row strides multiples of 8 elements");
  Params p{x, y, A, B, out, scales, h, order, offsets, T, ldx, ldy, ldo, N, K, R, adapters, leaf, 1, 0};
  p.rest = (expand ? out != y : 1) ? 1 : 0;
  return dtype == TBIK_DTYPE_BF16 ? choose_and_launch<__nv_bfloat16>(p, stream) : choose_and_launch<__half>(p, stream);
}

}  // namespace tbik
