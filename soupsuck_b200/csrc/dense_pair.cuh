// Two-SM (cta_group::2) dense GEMM for the distillation loss: fp16 or bf16 operands,
// fp32 sums, 256 x 256 tiles of a CTA pair.
//
// As in the NF4 pair kernel, each CTA of a pair holds 128 rows of A and 128 of the
// tile's 256 B columns; the rank-0 CTA issues 256 x 256 x 16 UMMAs that read both
// CTAs' halves and leave 128 accumulator rows in each CTA's TMEM.  Operands arrive by
// TMA (no multicast) in a ring of six 32 KB stages.
//
// Sums.  The tensor core adds in fp32 but cuts each addition off (towards zero): over
// the 96 steps of K = 1536 a sum of equal signs loses 8.5e-6 of itself, over K = 8192
// 5.3e-5 (fp16 operands, against 64 bits).  A logit that far off would dominate the
// error of a divergence, so a TMEM accumulation covers `seg` 64-wide k-blocks only: the
// two TMEM buffers take turns, and eight epilogue warps add each finished one into
// registers (128 fp32 per thread, rounded to nearest) while the next accumulates.
// Registers for that come from the four other warps (setmaxnreg).
//
// Warps: 0 TMA, 1 UMMA issue (rank 0), 2-3 idle, 4-11 epilogue: warp w holds TMEM lanes
// 32 (w % 4) .. +31, columns 128 ((w - 4) / 4) .. +127 of its CTA's 128 x 256 tile.
// Barriers:
//   full[s]      rank 0: its producer's arrival, bytes of both CTAs
//   empty[s]     both: rank 0's commit
//   acc_full[b]  both: rank 0's commit
//   acc_empty[b] rank 0: one arrival per epilogue warp of both CTAs (16)
// Waits are bounded, and the exits drain, as in the NF4 pair kernel.
//
// Measured (one launch, H = 1536, V = 151936): logits of 3300 rows 1.02 ms, 1.51 PFLOP/s
// with the tensor pipe 91 % active; of 48 rows 95 us, 5.0 TB/s of the head; the product
// for 1221 rows 417 us.  Long runs of either settle at the board's power limit (8192 x
// 3584: 1.44 and 1.41 PFLOP/s).  What an epilogue warp does for a logits tile of 12,288
// cycles of matrix work: four runs drained 2250 cycles, listed columns 1030, maximum 320,
// exponentials and sums 1950, hidden behind the next tile's first two runs.
#pragma once

#include <cuda_bf16.h>

#include <mutex>

#include "gemm_pair.cuh"

namespace sb {
namespace dense {

using gemm::kBK;
using gemm::kTileRows;

constexpr int kTile = 256;
constexpr int kHalf = 128;
constexpr int kStages = 6;
constexpr int kThreads = 384;
constexpr int kOperandBytes = kTileRows * kBK * 2;    // 16 KB, A or B of one stage
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kBoxBytes = 32 * 128;                   // one staging box per epilogue warp
constexpr int kSmemBytes = kStages * kStageBytes + 8 * kBoxBytes + 1024 + 1024;
static_assert(kSmemBytes <= 232448, "shared memory");

// Registers: 384 threads are launched with 168 each; the epilogue's two warpgroups
// take 224, the first keeps 56 (128 * 56 + 256 * 224 = 64,512 = 384 * 168).
constexpr int kRegsFew = 56, kRegsMany = 224;
static_assert(128 * kRegsFew + 256 * kRegsMany <= kThreads * 168, "register split");

struct Params {
  const int* count;      // rows of all blocks, known on the device
  int row_base;          // first of them in this block
  int rows_cap;          // rows this block's buffers hold
  int cols;              // N
  int n_tiles;
  int k_blocks;
  int seg;               // k-blocks of one TMEM accumulation
  int64_t room;          // product: elements of the output buffer
  // logits
  float scale;           // log2(e) / temperature
  int list;              // list length K
  const int* columns;    // [rows of the call, K] listed columns, rising
  const float* reference;  // [compact rows] exponent that the rows' exponentials share
  const uint32_t* lookup;  // [compact rows, 2 n_tiles] which columns of each 128 are listed (listed_word)
  float* listed;         // [compact rows, K] logits of the listed columns
  float2* stats;         // [2 n_tiles, rows_cap] exponent M and sum of 2^(y - M + 14)
  int store;             // write the exponentials too
};

// Splits of the product's K: as few as keep the last wave of units full, counting a
// unit's k-blocks, its start and end (8 k-blocks) and the traffic of its partial tile.
// A pair's k-block takes about 0.28 us.  `room`: what the buffer holds, at least one split.
// Called by whole warps: the lanes try different counts.
__device__ inline int product_splits(int rows, int cols, int k_blocks, int pairs, int64_t room) {
  const int tiles = ((rows + kTile - 1) / kTile) * ((cols + kTile - 1) / kTile);
  const int64_t elements = static_cast<int64_t>((rows + kTile - 1) / kTile * kTile) * cols;
  const int64_t fit = room / elements;
  const int most = fit < pairs ? static_cast<int>(fit) : pairs;
  int best = 1;
  float best_cost = 3.0e38f;
  for (int s = 1 + (threadIdx.x & 31); s <= most && (s == 1 || k_blocks / s >= 32); s += 32) {
    const int waves = (tiles * s + pairs - 1) / pairs;
    const float cost = waves * (static_cast<float>(k_blocks) / s + 8.0f) + s * static_cast<float>(elements) * 4.4e-6f;
    if (cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  for (int o = 16; o; o >>= 1) {
    const float cost = __shfl_xor_sync(0xffffffffu, best_cost, o);
    const int s = __shfl_xor_sync(0xffffffffu, best, o);
    if (cost < best_cost || (cost == best_cost && s < best)) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

struct Unit {
  int m0, nt, k0, k1, split;
};

// Logits: whole-K tiles, rows fastest (the pairs of a wave share columns of W).
// Product: (split, tile) with columns fastest, so the pairs of a wave walk the same
// k-blocks together and share their operands in L2.  Split s takes every splits-th block,
// from the last one down: each begins with what the logits launch left in L2.
template <bool PRODUCT>
struct Units {
  int m_tiles, tiles, splits, cursor, end, stride;
  __device__ Units(const Params& p, int rows, int splits_, int id, int count) {
    m_tiles = (rows + kTile - 1) / kTile;
    tiles = m_tiles * p.n_tiles;
    splits = splits_;
    cursor = id;
    end = tiles * splits;
    stride = count;
  }
  __device__ bool next(const Params& p, Unit& u) {
    if (cursor >= end) return false;
    if (PRODUCT) {
      u.split = cursor / tiles;
      const int t = cursor % tiles;
      u.m0 = t / p.n_tiles * kTile;
      u.nt = t % p.n_tiles;
      u.k0 = 0;
      u.k1 = (p.k_blocks - u.split + splits - 1) / splits;
    } else {
      u.split = 0;
      u.m0 = cursor % m_tiles * kTile;
      u.nt = cursor / m_tiles;
      u.k0 = 0;
      u.k1 = p.k_blocks;
    }
    cursor += stride;
    return true;
  }
};

__device__ __forceinline__ int block_rows(const Params& p) {
  const int left = *p.count - p.row_base;
  return left < 0 ? 0 : (left < p.rows_cap ? left : p.rows_cap);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in one 64-bit register pair: one instruction adds or scales both.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 values_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  } else {
    __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  }
}

// Exponentials are 2^(y - M + 14), y = z log2(e) / tau, with a whole exponent M: the row's
// reference, a guess of its log-sum-exp and a little more, where the tile's maximum
// (rounded up) lies from 26 below it to 1 above, else the tile's own maximum.  So fp16
// holds them without overflow (2^15) and, within a tile, down to 2^-12 of the maximum
// with an error below 2^-13 of it.  Rows whose tiles all keep the reference need no
// rescaling afterwards.
constexpr float kLift = 14.0f;
constexpr float kBelow = 26.0f, kAbove = 1.0f;

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// The list entries of one row in one tile of 128 columns: columns of the first three (7
// bits each), the first one's number in the list (8), how many (2, at most 3), whether
// there are more (1).  One load per row and tile; finding them from the list itself was
// three dependent ones, a tenth of the kernel.
__device__ __forceinline__ uint32_t listed_word(int first, int n, int c0, int c1, int c2) {
  uint32_t w = static_cast<uint32_t>(first & 255) << 21 | static_cast<uint32_t>(n < 3 ? n : 3) << 29 | (n > 3 ? 1u << 31 : 0u);
  if (n > 0) w |= static_cast<uint32_t>(c0 & 127);
  if (n > 1) w |= static_cast<uint32_t>(c1 & 127) << 7;
  if (n > 2) w |= static_cast<uint32_t>(c2 & 127) << 14;
  return w;
}

// ---------------------------------------------------------------- logits epilogue
// acc: this thread's row, columns col0 .. col0 + 127.  Listed columns leave their logit
// in p.listed and count as absent; the others give the tile's exponent M and sum of
// 2^(y - M + 14), which are also stored.
template <bool BF16>
__device__ __forceinline__ void logits_epilogue(const Params& p, uint64_t (&acc)[64], int row, int rows, int col0, int jt,
                                                uint32_t listed_here, float reference, uint8_t* box, const CUtensorMap* tm_out,
                                                int row_box, int lane) {
  const int ncol = p.cols - col0;
  if (ncol < 128) {
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      const float2 y = values_of(acc[i]);
      acc[i] = pair_of(2 * i < ncol ? y.x : -INFINITY, 2 * i + 1 < ncol ? y.y : -INFINITY);
    }
  }
  const bool valid = row < rows;
  // Listed columns: every lane its first one, then the lanes that have another, ...  The
  // column's register is found by comparing, in those groups of 32 that any lane needs
  // (with 64 of 151936 listed, one or two of a tile's four), by all lanes together: a
  // branch per column took 2900 of a tile's 16,000 cycles, a jump per entry 1650.
  {
    const int64_t list_at = (static_cast<int64_t>(p.row_base) + row) * p.list;
    int entry = (listed_here >> 21) & 255;
    int left = (listed_here >> 29) & 3;
    uint32_t columns = listed_here;
    int c = left ? static_cast<int>(columns & 127u) : 128;
    while (__any_sync(0xffffffffu, c < 128)) {
      float z = 0.0f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (__any_sync(0xffffffffu, c >> 5 == g)) {
#pragma unroll
          for (int i = 16 * g; i < 16 * g + 16; ++i) {
            const float2 y = values_of(acc[i]);
            const bool is_x = c == 2 * i, is_y = c == 2 * i + 1;
            z = is_x ? y.x : z;
            z = is_y ? y.y : z;
            acc[i] = pair_of(is_x ? -INFINITY : y.x, is_y ? -INFINITY : y.y);
          }
        }
      }
      if (c < 128) {
        p.listed[list_at + entry] = z;
        ++entry;
        columns >>= 7;
        c = 128;
        if (--left > 0) {
          c = columns & 127u;
        } else if (listed_here >> 31 && entry < p.list) {
          c = p.columns[list_at + entry] - col0;  // 128 or more past the tile's last
        }
      }
      __syncwarp();
    }
  }
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const float2 y = values_of(acc[i]);
    top[i & 3] = fmaxf(fmaxf(top[i & 3], y.x), y.y);
  }
  const float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  float m = t == -INFINITY ? 0.0f : ceilf(t * p.scale);
  m = m >= reference - kBelow && m <= reference + kAbove ? reference : m;
  const uint64_t scale = pair_of(p.scale, p.scale), off = pair_of(kLift - m, kLift - m);
  uint64_t s0 = 0, s1 = 0;
  const uint32_t swz = static_cast<uint32_t>(lane & 7);
  // A panel of 64 columns at a time: the first one's store reads the box while the
  // second one's exponentials are formed.
#pragma unroll
  for (int panel = 0; panel < 2; ++panel) {
#pragma unroll
    for (int i = 32 * panel; i < 32 * panel + 32; ++i) {
      const float2 e = values_of(fma_pair(acc[i], scale, off));
      acc[i] = pair_of(exp2_fast(e.x), exp2_fast(e.y));
      if (i & 1) {
        s1 = add_pair(s1, acc[i]);
      } else {
        s0 = add_pair(s0, acc[i]);
      }
    }
    if (p.store) {
      if (lane == 0) gemm::pair::bulk_wait_read0();
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 e = values_of(acc[panel * 32 + c * 4 + j]);
          w[j] = pack2<BF16>(e.x, e.y);
        }
        *reinterpret_cast<uint4*>(box + lane * 128 + ((static_cast<uint32_t>(c) ^ swz) << 4)) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && col0 + panel * 64 < p.cols) {
        gemm::pair::tma_store_2d(tm_out, box, col0 + panel * 64, row_box);
        gemm::pair::bulk_commit();
      }
    }
  }
  const float2 s = values_of(add_pair(s0, s1));
  if (valid) p.stats[static_cast<int64_t>(jt) * p.rows_cap + row] = make_float2(m, s.x + s.y);
}

// ---------------------------------------------------------------- product epilogue
__device__ __forceinline__ void product_epilogue(const Params& p, uint64_t (&acc)[64], int col0, uint8_t* box,
                                                 const CUtensorMap* tm_out, int row_box, int lane) {
  const uint32_t swz = static_cast<uint32_t>(lane & 7);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (lane == 0) gemm::pair::bulk_wait_read0();
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 a = values_of(acc[c * 16 + j * 2]), b = values_of(acc[c * 16 + j * 2 + 1]);
      *reinterpret_cast<float4*>(box + lane * 128 + ((static_cast<uint32_t>(j) ^ swz) << 4)) =
          make_float4(a.x, a.y, b.x, b.y);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && col0 + c * 32 < p.cols) {
      gemm::pair::tma_store_2d(tm_out, box, col0 + c * 32, row_box);
      gemm::pair::bulk_commit();
    }
  }
}

// ---------------------------------------------------------------- the kernel
// PRODUCT false: out = exponentials of A[rows, K] . B[cols, K]^T; true: partial sums of
// A[rows, K] . B[K, cols] (B's panels MN-major).
template <bool PRODUCT, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    dense_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                 const __grid_constant__ CUtensorMap tm_out, const Params p) {
  using namespace gemm::pair;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + kStages * kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + 8 * kBoxBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pair_id = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 16);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_holder, 2 * kTile);
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  // Launched with programmatic stream serialisation (launch_after): the set-up above
  // overlaps the previous kernel; its results are read from here on.
  grid_dependency_wait();
  launch_dependents();
  const int rows = block_rows(p);
  const int splits = PRODUCT && rows > 0 ? product_splits(rows, p.cols, p.k_blocks, pairs, p.room) : 1;
  const uint32_t leader_full = map_to_rank(smem_addr(full), 0);
  const uint32_t leader_acc_empty = map_to_rank(smem_addr(acc_empty), 0);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
    if (warp == 0) {
      // ---------------------------------------------------------- TMA producer (both CTAs)
      if (lane == 0) {
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_b);
        uint32_t it = 0;
        bool ok = true;
        Units<PRODUCT> units(p, rows, splits, pair_id, pairs);
        Unit u;
        while (ok && units.next(p, u)) {
          const int arow = u.m0 + static_cast<int>(rank) * kTileRows;
          const int bcol = u.nt * kTile + static_cast<int>(rank) * kHalf;
          for (int kb = u.k0; kb < u.k1; ++kb, ++it) {
            const int s = it % kStages;
            if (!mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, kErrWaitEmpty, abort_flag)) {
              ok = false;
              break;
            }
            uint8_t* a_s = smem + s * kStageBytes;
            uint8_t* b_s = a_s + kOperandBytes;
            if (leader) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
            const int k = PRODUCT ? ((u.k1 - 1 - kb) * splits + u.split) * kBK : kb * kBK;
            tma_load_2d_pair(a_s, &tm_a, leader_full + 8u * s, k, arow);
            if constexpr (PRODUCT) {
              tma_load_2d_pair(b_s, &tm_b, leader_full + 8u * s, bcol, k);
              tma_load_2d_pair(b_s + kOperandBytes / 2, &tm_b, leader_full + 8u * s, bcol + 64, k);
            } else {
              tma_load_2d_pair(b_s, &tm_b, leader_full + 8u * s, k, bcol);
            }
          }
        }
        // Every stage filled above released by the UMMA (its bytes landed, the peer's
        // commits arrived) before exit; after an abort wait out the loads in flight.
        volatile int drain_abort = 0;
        bool clean = ok && !*abort_flag;
        for (uint32_t j = it; clean && j < it + kStages; ++j) {
          clean = mbar_wait(&empty[j % kStages], ((j / kStages) & 1) ^ 1, kErrWaitDrain, abort_flag);
        }
        if (!clean) {
          const uint32_t first = it > static_cast<uint32_t>(kStages) ? it - kStages : 0;
          for (uint32_t j = first; j < it; ++j) {
            if (leader) mbar_wait(&full[j % kStages], (j / kStages) & 1, kErrWaitDrain, &drain_abort);
          }
        }
      }
    } else if (warp == 1 && leader) {
      // ---------------------------------------------------------- UMMA issuer (rank 0)
      constexpr uint32_t kType = BF16 ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t kIdesc = idesc_f16_f32(kTile, kTile, 0, PRODUCT ? 1 : 0) | kType;
      const uint64_t ad0 = smem_desc(smem_addr(smem), 16, 1024, kSwizzle128B);
      const uint64_t bd0 = PRODUCT ? smem_desc(smem_addr(smem) + kOperandBytes, 64 * 128, 1024, kSwizzle128B)
                                   : smem_desc(smem_addr(smem) + kOperandBytes, 16, 1024, kSwizzle128B);
      const uint32_t a_lo0 = static_cast<uint32_t>(ad0), a_hi = static_cast<uint32_t>(ad0 >> 32);
      const uint32_t b_lo0 = static_cast<uint32_t>(bd0), b_hi = static_cast<uint32_t>(bd0 >> 32);
      const uint32_t empty_addr = smem_addr(empty);
      uint32_t st = 0, ph = 0, acc = 0;
      bool ok = true;
      Units<PRODUCT> units(p, rows, splits, pair_id, pairs);
      Unit u;
      while (ok && units.next(p, u)) {
        for (int kb = u.k0; ok && kb < u.k1; ++acc) {
          const int stop = kb + p.seg < u.k1 ? kb + p.seg : u.k1;
          const uint32_t buf = acc & 1;
          if (!warp_wait(&acc_empty[buf], ((acc >> 1) & 1) ^ 1, kErrWaitAccEmpty, abort_flag, lane)) {
            ok = false;
            break;
          }
          tc_fence_after();
          for (uint32_t first = 0; kb < stop; ++kb, first = 1) {
            if (!warp_wait(full + st, ph, kErrWaitFull, abort_flag, lane)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t off = st * (kStageBytes >> 4);
            umma_kstep_pair_warp(tmem_base + buf * kTile, a_lo0 + off, a_hi, b_lo0 + off, b_hi, 32 >> 4,
                                 PRODUCT ? (16 * 128) >> 4 : 32 >> 4, kIdesc, first, empty_addr + 8u * st);
            if (++st == static_cast<uint32_t>(kStages)) {
              st = 0;
              ph ^= 1u;
            }
          }
          if (ok) umma_commit_both_warp(&acc_full[buf]);
        }
      }
      // Both accumulators released by both epilogues, then every UMMA complete.
      if (ok && !*abort_flag) {
        if (warp_wait(&acc_empty[acc & 1], ((acc >> 1) & 1) ^ 1, kErrWaitDrain, abort_flag, lane)) {
          warp_wait(&acc_empty[(acc + 1) & 1], (((acc + 1) >> 1) & 1) ^ 1, kErrWaitDrain, abort_flag, lane);
        }
      }
      umma_commit_local_warp(drain);
      volatile int no_abort = 0;
      warp_wait(drain, 0, kErrWaitDrain, &no_abort, lane);
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMany));
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint8_t* box = staging + (warp - 4) * kBoxBytes;
    const uint32_t tlane = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + half * kHalf;
    uint32_t accs = 0;
    bool ok = true;
    Units<PRODUCT> units(p, rows, splits, pair_id, pairs);
    Unit u;
    while (ok && units.next(p, u)) {
      const int row_box = u.m0 + static_cast<int>(rank) * kTileRows + q * 32;
      const int row = row_box + lane;
      const int col0 = u.nt * kTile + half * kHalf;
      const int jt = u.nt * 2 + half;
      uint32_t listed_here = 0;
      float reference = 0.0f;
      if constexpr (!PRODUCT) {
        if (row < rows) {
          const int64_t at = static_cast<int64_t>(p.row_base) + row;
          listed_here = p.lookup[at * (2 * p.n_tiles) + jt];
          reference = p.reference[at];
        }
      }
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
#pragma unroll 1
      for (int kb = u.k0; kb < u.k1; kb += p.seg, ++accs) {
        const uint32_t buf = accs & 1;
        if (!warp_wait(&acc_full[buf], (accs >> 1) & 1, kErrWaitAccFull, abort_flag, lane)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t tacc = tlane + buf * kTile;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[32], w[32];
          tmem_ld32(tacc + c * 64, v);
          tmem_ld32(tacc + c * 64 + 32, w);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            acc[32 * c + i] = add_pair(acc[32 * c + i], pair_of(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])));
            acc[32 * c + 16 + i] =
                add_pair(acc[32 * c + 16 + i], pair_of(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(leader_acc_empty + 8u * buf);
      }
      if (!ok) break;
      if constexpr (PRODUCT) {
        product_epilogue(p, acc, col0, box, &tm_out, u.split * units.m_tiles * kTile + row_box, lane);
      } else {
        logits_epilogue<BF16>(p, acc, row, rows, col0, jt, listed_here, reference, box, &tm_out, row_box, lane);
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kTile);
  }
}

// A launch that may begin while the previous kernel of the stream ends; the kernel waits
// for it (grid_dependency_wait) before it touches memory.  Every kernel launched this way
// waits, so a kernel's results are complete for all later ones, not only the next.
template <typename... P, typename... A>
int launch_after(const char* name, void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e != cudaSuccess) return fail(SB_ECUDA, std::string(name) + ": " + cudaGetErrorString(e));
  count_launch();
  return check_launch(name);
}

template <bool PRODUCT, bool BF16>
int launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out, const Params& p, cudaStream_t st,
           const char* name) {
  auto kern = dense_kernel<PRODUCT, BF16>;
  static std::mutex mu;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
      // The register split counts on the launch's total: with fewer it would wait forever.
      cudaFuncAttributes attributes{};
      if (e == cudaSuccess) e = cudaFuncGetAttributes(&attributes, kern);
      if (e != cudaSuccess) return fail(SB_ECUDA, std::string(name) + " attributes: " + cudaGetErrorString(e));
      if (attributes.numRegs * kThreads < 128 * kRegsFew + 256 * kRegsMany) {
        return fail(SB_EUNSUPPORTED, std::string(name) + " was compiled with too few registers for its split");
      }
      if (dev >= 0 && dev < 64) configured[dev] = true;
    }
  }
  return launch_after(name, kern, device_sm_count() / 2 * 2, kThreads, kSmemBytes, st, a, b, out, p);
}

}  // namespace dense
}  // namespace sb
