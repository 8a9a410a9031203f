// Distillation from a teacher's listed logits through a frozen head, with its gradient.
//
// Row n: student logits z_v = h . W_v / tau, q = softmax(z); the teacher lists columns J
// with logits t_j.  With its log-sum-exp L: p_j = exp(t_j / tau - L) and one bucket of all
// other columns, p_rest = max(0, 1 - sum p_j); without: p = softmax over J, p_rest = 0.
//
//   loss = sum_J g(p_j, q_j) + g(p_rest, q_rest),   g(p, q) = p log(p / q) - p + q
//   mass = sum_J q_j
//   d loss / d z_v = q_v - p_v on J,   q_v (1 - p_rest / q_rest) elsewhere
//
// The -p + q terms sum to zero over both distributions; with them every term is at
// least zero and nothing cancels where student and teacher are close.
//
// Forward.  prepare gathers the answered rows (the others are left out of everything
// else), sorts each one's list and computes log p.  One tensor-core launch forms the
// logits tile by tile (dense_pair.cuh): listed ones are written out, the others leave an
// exponent and a sum of exponentials per row and 128 columns, and, where a gradient is
// wanted, the exponentials themselves in 16 bits [rows, V].  merge joins them per row.
// The gradient does not wait for the upstream one, which only scales rows: dz is the
// stored exponentials with the listed columns written in, du = dz . W on the tensor
// cores, and the row's remaining factor is applied to the fp32 sums.  A row whose tiles
// used different exponents, or whose listed columns would overflow beside the others,
// is first multiplied by powers of two (exact), 4 bytes of traffic per logit that most
// rows do without: prepare guesses the row's log-sum-exp (from the student's logit of
// the teacher's best token, as if their probabilities of it were equal) and the tiles
// use that exponent.  Keeping the exponentials instead of forming the logits a second
// time saves a third of the matrix work.
// Backward.  dhidden = upstream * du, rounded once.
//
// Measured (one pass, V = 151936): 1221 answered of 3300 rows, H = 1536: logits 432, product
// 417, all others 62 us; 48 rows 95, 87 and 45; the two products are what bounds it
// (dense_pair.cuh), the small kernels (4 to 20 us each) wait for dependent loads.
#pragma once

#include <type_traits>

#include "dense_pair.cuh"
#include "gemm_host.cuh"

namespace sb {
namespace distill {

constexpr int kMaxList = 256;
constexpr int kNone = 0x7fffffff;             // an unused entry of a sorted list
constexpr int64_t kBlockBytes = int64_t(4) << 30;  // 16-bit exponentials of one row block
constexpr int kMaxRowBlocks = 256;
constexpr int kFixes = 4;
constexpr int kPadAtOnce = 4;  // vectors of a thread in flight
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T> __device__ __forceinline__ float logit_at(const void* p, int64_t i);
template <> __device__ __forceinline__ float logit_at<float>(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
template <> __device__ __forceinline__ float logit_at<__half>(const void* p, int64_t i) {
  return __half2float(static_cast<const __half*>(p)[i]);
}
template <> __device__ __forceinline__ float logit_at<__nv_bfloat16>(const void* p, int64_t i) {
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ float warp_sum(float x) {
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
  for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// out[rows, width] = in[rows, h] (row stride `pitch`, any alignment of 2 bytes) with zero
// columns behind: the layout that the tensor maps need.  A thread writes 16 bytes from
// the two aligned 16-byte words around them; words past the last element are not read.
__global__ void __launch_bounds__(256) pad_kernel(const uint16_t* __restrict__ in, int64_t rows, int64_t h, int64_t pitch,
                                                  int64_t width, uint16_t* __restrict__ out) {
  const uint32_t per_row = static_cast<uint32_t>(width / 8);
  const uint16_t* end = in + (rows - 1) * pitch + h;
  const int64_t vecs = rows * per_row, step = static_cast<int64_t>(gridDim.x) * 256 * kPadAtOnce;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * 256 * kPadAtOnce + threadIdx.x; first < vecs; first += step) {
    const uint16_t* from[kPadAtOnce];
    int have[kPadAtOnce];
    uint4 x[kPadAtOnce], y[kPadAtOnce];
#pragma unroll
    for (int u = 0; u < kPadAtOnce; ++u) {
      const int64_t i = first + u * 256;
      const int64_t row = vecs <= 0xffffffffll ? static_cast<uint32_t>(i) / per_row : i / per_row;
      const int64_t col = (i - row * per_row) * 8;
      from[u] = in + row * pitch + col;
      have[u] = i < vecs ? (h - col < 8 ? static_cast<int>(h - col) : 8) : 0;
      const uint16_t* base = from[u] - static_cast<int>(reinterpret_cast<uintptr_t>(from[u]) & 15) / 2;
      if (have[u] == 8 && base >= in && base + 16 <= end) {
        x[u] = __ldg(reinterpret_cast<const uint4*>(base));
        y[u] = __ldg(reinterpret_cast<const uint4*>(base) + 1);
      } else {
        have[u] |= 16;
      }
    }
#pragma unroll
    for (int u = 0; u < kPadAtOnce; ++u) {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
      if (have[u] < 16) {
        const int off = static_cast<int>(reinterpret_cast<uintptr_t>(from[u]) & 15) / 2;
        // Words off / 2 .. off / 2 + 4 of the eight, shifted by half a word where off is odd.
        uint32_t a[5] = {x[u].x, x[u].y, x[u].z, x[u].w, y[u].x};
        if (off & 2) { a[0] = a[1]; a[1] = a[2]; a[2] = a[3]; a[3] = a[4]; a[4] = y[u].y; }
        if (off & 4) {
          const uint32_t next = off & 2 ? y[u].z : y[u].y, then = off & 2 ? y[u].w : y[u].z;
          a[0] = a[2]; a[1] = a[3]; a[2] = a[4]; a[3] = next; a[4] = then;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = off & 1 ? __funnelshift_r(a[j], a[j + 1], 16) : a[j];
      } else {
        for (int j = 0; j < (have[u] & 15); ++j) w[j / 2] |= static_cast<uint32_t>(from[u][j]) << (16 * (j & 1));
      }
      if (first + u * 256 < vecs) reinterpret_cast<uint4*>(out)[first + u * 256] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// faults[0]: indices that are neither -1 nor a column; faults[1]: repeats within a row.
__global__ void check_kernel(const int64_t* __restrict__ indices, int64_t rows, int k, int64_t v,
                             unsigned long long* __restrict__ faults) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int64_t* list = indices + row * k;
  unsigned long long outside = 0, repeats = 0;
  for (int j = lane; j < k; j += 32) {
    const int64_t c = list[j];
    if (c < -1 || c >= v) ++outside;
    if (c >= 0) {
      for (int i = 0; i < j; ++i) {
        if (list[i] == c) {
          ++repeats;
          break;
        }
      }
    }
  }
  if (outside) atomicAdd(&faults[0], outside);
  if (repeats) atomicAdd(&faults[1], repeats);
}

// Which rows are answered: a listed column, and on the list some teacher probability.
// One warp per row; `blocks` counts the answered rows of each CTA's eight.
constexpr int kRowsPerBlock = 8;
template <typename T>
__global__ void __launch_bounds__(256) answered_kernel(const int64_t* __restrict__ indices, const void* __restrict__ logits,
                                                       const float* __restrict__ lse, int64_t rows, int k, int64_t v,
                                                       int* __restrict__ place, int* __restrict__ blocks) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock + warp;
  bool some = false;
  if (row < rows) {
    for (int j = lane; j < k; j += 32) {
      const int64_t c = indices[row * k + j];
      some |= c >= 0 && c < v && (lse || !(logit_at<T>(logits, row * k + j) == -INFINITY));
    }
    some = __any_sync(0xffffffffu, some) && !(lse && lse[row] == -INFINITY);
    if (lane == 0) place[row] = some ? 1 : -1;
  }
  const int n = __syncthreads_count(some && lane == 0);
  if (threadIdx.x == 0) blocks[blockIdx.x] = n;
}

// What the other kernels need of each answered row, in the rows' order without gaps: its
// hidden state, its list sorted by column, log p of each entry, p_rest, how many entries
// are used, and which entries each 128-column tile has.  Rows that are not answered get zero
// loss and mass here.  One warp per row; an entry's place is the number of entries
// before it (K <= 256).
template <typename T, bool BF16>
__global__ void __launch_bounds__(256) prepare_kernel(const uint16_t* __restrict__ hidden, int64_t h,
                                                      const uint16_t* __restrict__ weight,
                                                      const int64_t* __restrict__ indices, const void* __restrict__ logits,
                                                      const float* __restrict__ lse, int64_t rows, int k, int64_t v,
                                                      float inv_tau, int tiles, const int* __restrict__ blocks,
                                                      int* __restrict__ place, int* __restrict__ source,
                                                      int* __restrict__ count, uint16_t* __restrict__ gathered,
                                                      int* __restrict__ columns, float* __restrict__ logp,
                                                      float* __restrict__ rest, int* __restrict__ used,
                                                      uint32_t* __restrict__ lookup, float* __restrict__ reference,
                                                      int* __restrict__ uneven, int row_blocks, float* __restrict__ loss,
                                                      float* __restrict__ mass) {
  __shared__ int s_col[kRowsPerBlock][kMaxList];
  __shared__ float s_t[kRowsPerBlock][kMaxList];
  __shared__ int s_before[kRowsPerBlock], s_in[kRowsPerBlock];
  grid_dependency_wait();
  launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock + warp;
  int before = 0;
  for (int i = threadIdx.x; i < static_cast<int>(blockIdx.x); i += 256) before += blocks[i];
  for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const bool in = row < rows && place[row] > 0;
  if (lane == 0) {
    s_before[warp] = before;
    s_in[warp] = in ? 1 : 0;
  }
  __syncthreads();
  int at = 0;
  for (int i = 0; i < kRowsPerBlock; ++i) at += s_before[i] + (i < warp ? s_in[i] : 0);
  if (lane == 0 && warp == kRowsPerBlock - 1 && blockIdx.x == gridDim.x - 1) *count = at + s_in[warp];
  if (blockIdx.x == 0 && threadIdx.x < row_blocks) uneven[threadIdx.x] = 0;
  if (row >= rows) return;
  if (lane == 0) {
    place[row] = in ? at : -1;
    if (in) {
      source[at] = static_cast<int>(row);
    } else {
      loss[row] = 0.0f;
      mass[row] = 0.0f;
    }
  }
  if (!in) return;
  int* col = s_col[warp];
  float* tv = s_t[warp];
  int n = 0, best = kNone;  // best: the column of this lane's largest logit
  float top = -INFINITY;
  for (int j = lane; j < k; j += 32) {
    const int64_t c = indices[row * k + j];
    const bool used_here = c >= 0 && c < v;
    const float t = used_here ? logit_at<T>(logits, row * k + j) * inv_tau : -INFINITY;
    col[j] = used_here ? static_cast<int>(c) : kNone;
    tv[j] = t;
    n += used_here ? 1 : 0;
    if (used_here && (best == kNone || t > top)) best = static_cast<int>(c);
    top = t == t ? fmaxf(top, t) : INFINITY;  // a NaN makes the row NaN
  }
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  const float mine = top;
  top = warp_max(top);
  best = __shfl_sync(0xffffffffu, best, __ffs(__ballot_sync(0xffffffffu, best != kNone && mine == top) | 0x80000000u) - 1);
  if (best == kNone) best = 0;  // (a lane's NaN: any column will do)
  // The hidden state, and its logit of that column.
  float dot = 0.0f;
  {
    const uint4* from = reinterpret_cast<const uint4*>(hidden + row * h);
    const uint4* w = reinterpret_cast<const uint4*>(weight + static_cast<int64_t>(best) * h);
    uint4* to = reinterpret_cast<uint4*>(gathered + at * h);
    for (int64_t i = lane; i < h / 8; i += 32) {
      const uint4 a = from[i], b = w[i];
      to[i] = a;
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = dense::unpack2<BF16>(aw[j]), y = dense::unpack2<BF16>(bw[j]);
        dot = fmaf(x.x, y.x, fmaf(x.y, y.y, dot));
      }
    }
    dot = warp_sum(dot);
  }
  __syncwarp();
  // The normaliser: the teacher's, or the list's own.
  float norm;
  if (lse) {
    norm = lse[row];
  } else {
    float s = 0.0f;
    for (int j = lane; j < k; j += 32) s += expf(tv[j] - top);
    norm = top + logf(warp_sum(s));
  }
  int* row_columns = columns + static_cast<int64_t>(at) * k;
  float* row_logp = logp + static_cast<int64_t>(at) * k;
  float sum = 0.0f;
  for (int j = lane; j < k; j += 32) {
    const int c = col[j];
    int where = 0;
    for (int i = 0; i < k; ++i) where += (col[i] < c || (col[i] == c && i < j)) ? 1 : 0;
    const float lp = c == kNone ? -INFINITY : tv[j] - norm;
    row_columns[where] = c;
    row_logp[where] = lp;
    if (c != kNone) sum += expf(lp);
  }
  sum = warp_sum(sum);
  if (lane == 0) {
    const float left = 1.0f - sum;
    rest[at] = !lse || n == v ? 0.0f : (left < 0.0f ? 0.0f : left);
    used[at] = n;
    // log2 of the student's exponential sum if it gave the teacher's best token the
    // teacher's probability, and four more for the listed columns' room in 16 bits.
    reference[at] = ceilf((dot * inv_tau - (top - norm)) * kLog2e) + 4.0f;
  }
  // The tiles' lookups: zeros, then each tile's from its first entry.
  uint32_t* row_lookup = lookup + static_cast<int64_t>(at) * tiles;
  for (int j = lane; j < tiles / 2; j += 32) reinterpret_cast<uint2*>(row_lookup)[j] = make_uint2(0u, 0u);
  __syncwarp();
  for (int j = lane; j < n; j += 32) {
    const int c = row_columns[j], tile = c >> 7;
    if (j > 0 && row_columns[j - 1] >> 7 == tile) continue;
    int next[3], here = 1;
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      next[e] = j + 1 + e < n ? row_columns[j + 1 + e] : kNone;
      here += next[e] >> 7 == tile ? 1 : 0;
    }
    row_lookup[tile] = dense::listed_word(j, here, c, next[0], next[1]);
  }
}

// g(p, q) from logarithms: q (r e^r - e^r + 1) with r = log(p / q), by its series
// r^2/2 + r^3/3 + r^4/8 + ... where the closed form would cancel, and as p r - p + q where
// e^r would be large.
__device__ __forceinline__ float gap(float p, float logp, float q, float logq) {
  if (!(p > 0.0f) && p == p) return q;
  const float r = logp - logq;
  if (fabsf(r) < 0.25f) {
    const float poly =
        r * r * (0.5f + r * (1.0f / 3 + r * (0.125f + r * (1.0f / 30 + r * (1.0f / 144 + r * (1.0f / 840 + r * (1.0f / 5760)))))));
    return q * poly;
  }
  if (r > 1.0f) return fmaf(p, r, q - p);
  return q * (r * expf(r) - expm1f(r));
}

// Four rows per CTA.  Joins a row's tile statistics and listed logits into its loss and
// mass, and for the gradient: `unit`, dz's factor, and the listed columns' dz / unit,
// written in among the exponentials.  The unit is a power of two times the factor all
// unlisted columns share,
//   b = 2^(R - lse2) - p_rest / S     (R the largest M, S the sum of 2^(y - R)),
// so only the listed columns' values are rounded anew, and is such that neither passes
// 2^15 in fp16.  Rows whose exponentials have to change for that, by 2^(M + shift) in a
// tile, go to the list `uneven` (its count first); their listed values are kept over
// their logits for the kernel that does it.
constexpr int kMergeThreads = 512, kMergeRows = 4;
constexpr float kLow = -1e9f;  // below every exponent

// 2^x for a whole x <= 0 (zero below -126; NaN stays).
__device__ __forceinline__ float power(float x) {
  return x > -127.0f ? __int_as_float((static_cast<int>(x) + 127) << 23) : (x == x ? 0.0f : x);
}

template <bool BF16>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(
    const float2* __restrict__ stats, int64_t ld, int tiles, const int* __restrict__ count, int row_base,
    const int* __restrict__ source, const int* __restrict__ used, const float* __restrict__ logp,
    const float* __restrict__ rest, int k, float scale, float* __restrict__ listed, float* __restrict__ loss,
    float* __restrict__ mass, const float* __restrict__ reference, const int* __restrict__ columns,
    uint16_t* __restrict__ dz, int64_t pitch, float* __restrict__ unit, int* __restrict__ shift,
    int2* __restrict__ fixes, int* __restrict__ uneven_count, int* __restrict__ uneven) {
  __shared__ float s_r[kMergeThreads], s_s[kMergeThreads];
  __shared__ int s_mixed[kMergeRows];
  grid_dependency_wait();
  launch_dependents();
  const int n = *count - row_base;
  const int r = threadIdx.x % kMergeRows, g = threadIdx.x / kMergeRows;
  constexpr int kGroups = kMergeThreads / kMergeRows;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kMergeRows + r;
  if (static_cast<int64_t>(blockIdx.x) * kMergeRows >= n) return;
  if (threadIdx.x < kMergeRows) s_mixed[threadIdx.x] = 0;
  __syncthreads();
  float R = kLow, S = 0.0f;
  if (row < n) {
    const float ref = reference[row_base + row];
    bool mixed = false;
    // Loads first, several at a time; every factor is a power of two (exact).
    constexpr int kAtOnce = 10;
    for (int j0 = g; j0 < tiles; j0 += kAtOnce * kGroups) {
      float2 t[kAtOnce];
      float top = R;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int64_t j = j0 + i * kGroups;
        t[i] = j < tiles ? stats[j * ld + row] : make_float2(kLow, 0.0f);
        if (t[i].y != 0.0f) top = fmaxf(top, t[i].x);
        mixed |= t[i].y != 0.0f && t[i].x != ref;
      }
      S *= power(R - top);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (t[i].y != 0.0f) S += t[i].y * power(t[i].x - top);
      }
      R = top;
    }
    if (mixed) s_mixed[r] = 1;
  }
  s_r[threadIdx.x] = R;
  s_s[threadIdx.x] = S;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp >= kMergeRows) return;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kMergeRows + warp;
  if (at >= n) return;
  R = kLow;
  S = 0.0f;
  for (int i = lane; i < kGroups; i += 32) R = fmaxf(R, s_r[i * kMergeRows + warp]);
  R = warp_max(R);
  for (int i = lane; i < kGroups; i += 32) {
    const float s = s_s[i * kMergeRows + warp];
    if (s != 0.0f) S += s * power(s_r[i * kMergeRows + warp] - R);
  }
  S = warp_sum(S) * exp2f(-dense::kLift);
  const int64_t src = source[row_base + at];
  const int m = used[row_base + at];
  float* z = listed + (row_base + at) * k;
  const float* lp = logp + (row_base + at) * k;
  float top = S > 0.0f ? R : -INFINITY;
  for (int j = lane; j < m; j += 32) top = fmaxf(top, z[j] * scale);
  top = warp_max(top);
  float total = 0.0f;
  for (int j = lane; j < m; j += 32) total += exp2f(fmaf(z[j], scale, -top));
  total = warp_sum(total);
  if (S != 0.0f) total += S * exp2f(R - top);
  const float lse2 = top + log2f(total);
  float gaps = 0.0f, covered = 0.0f, largest = 0.0f;
  for (int j = lane; j < m; j += 32) {
    const float y = fmaf(z[j], scale, -lse2);
    const float q = exp2f(y), p = expf(lp[j]);
    gaps += gap(p, lp[j], q, y * kLn2);
    covered += q;
    const float d = q - p;
    largest = fmaxf(largest, fabsf(d));
    z[j] = d;
  }
  gaps = warp_sum(gaps);
  covered = warp_sum(covered);
  largest = warp_max(largest);
  const float p_rest = rest[row_base + at];
  const float head = exp2f(R - lse2);
  if (lane == 0) {
    if (S > 0.0f || !(S == S)) gaps += gap(p_rest, logf(p_rest), S * head, (R - lse2 + log2f(S)) * kLn2);
    loss[src] = gaps;
    mass[src] = covered;
  }
  if (!unit) return;
  const float a = S == 0.0f ? 0.0f : (head - p_rest / S) * exp2f(-dense::kLift);
  float f;
  int e;
  if (a == 0.0f) {
    e = -100000;  // no unlisted share: the stored exponentials become zeros
    f = largest > 0.0f ? exp2f(static_cast<float>(ilogbf(largest)) - dense::kLift) : 1.0f;
  } else {
    int down = largest > 0.0f ? 14 + ilogbf(a) - ilogbf(largest) : 0;
    if (!(a == a) || isinf(a) || !(largest < INFINITY)) down = 0;
    down = down > 0 ? 0 : down;
    e = down - static_cast<int>(R);
    f = ldexpf(a, -down);
  }
  const bool even = S == 0.0f || (s_mixed[warp] == 0 && e == -static_cast<int>(R));
  const int* row_columns = columns + (row_base + at) * k;
  for (int j = lane; j < m; j += 32) {
    const float x = z[j] / f;
    z[j] = x;
    if (even) dz[at * pitch + row_columns[j]] = static_cast<uint16_t>(dense::pack2<BF16>(x, 0.0f) & 0xffffu);
  }
  __syncwarp();
  // What the rounding to 16 bits takes from the listed columns is most of dz's error; the
  // largest four amounts are kept, for the product's sums.
  uint64_t before = ~0ull;
  for (int i = 0; i < kFixes; ++i) {
    uint64_t best = 0;
    for (int j = lane; j < m; j += 32) {
      const float x = z[j];
      const float lost = x - dense::unpack2<BF16>(dense::pack2<BF16>(x, 0.0f)).x;
      const uint64_t key = static_cast<uint64_t>(__float_as_uint(fabsf(lost))) << 32 | static_cast<uint32_t>(j + 1);
      if (key < before && key > best) best = key;
    }
    for (int o = 16; o; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    before = best;
    const int j = static_cast<int>(best & 0xffffffffu) - 1;
    if (lane == 0) {
      int2 fix = make_int2(0, 0);
      if (j >= 0) {
        const float x = z[j];
        const float lost = x - dense::unpack2<BF16>(dense::pack2<BF16>(x, 0.0f)).x;
        fix = make_int2(row_columns[j], __float_as_int(lost * f));
      }
      fixes[(row_base + at) * kFixes + i] = fix;
    }
  }
  if (lane == 0) {
    unit[row_base + at] = f;
    shift[row_base + at] = e;
    if (!even) uneven[atomicAdd(uneven_count, 1)] = static_cast<int>(at);
  }
}

// The uneven rows' dz in place, a segment of a row at a time: each tile's exponentials
// times 2^(M + shift), then the listed columns.
constexpr int kScaleThreads = 256, kScaleVecs = 4;
template <bool BF16>
__global__ void __launch_bounds__(kScaleThreads) scale_kernel(
    uint16_t* __restrict__ dz, int64_t pitch, const float2* __restrict__ stats, int64_t ld,
    const int* __restrict__ uneven_count, const int* __restrict__ uneven, int row_base, const int* __restrict__ used,
    const int* __restrict__ columns, const float* __restrict__ listed, int k, const int* __restrict__ shift) {
  constexpr int kSegment = kScaleThreads * kScaleVecs;  // vectors
  grid_dependency_wait();
  launch_dependents();
  const int segments = static_cast<int>((pitch / 8 + kSegment - 1) / kSegment);
  const int64_t items = static_cast<int64_t>(*uneven_count) * segments;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = uneven[item / segments];
    const int e = shift[row_base + row];
    uint16_t* line = dz + row * pitch;
    const int64_t v0 = item % segments * kSegment;
#pragma unroll
    for (int i = 0; i < kScaleVecs; ++i) {
      const int64_t vec = v0 + i * kScaleThreads + threadIdx.x;
      if (vec * 8 >= pitch) break;
      const float2 t = stats[(vec >> 4) * ld + row];
      const int by = static_cast<int>(t.x) + e;
      if (by == 0 || t.y == 0.0f) continue;
      const float f = exp2f(static_cast<float>(by));
      uint4* at = reinterpret_cast<uint4*>(line) + vec;
      uint4 w = *at;
      uint32_t* x = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 y = dense::unpack2<BF16>(x[j]);
        x[j] = dense::pack2<BF16>(y.x * f, y.y * f);
      }
      *at = w;
    }
    __syncthreads();
    const int64_t c0 = v0 * 8, c1 = c0 + kSegment * 8;
    const int n = used[row_base + row];
    for (int j = threadIdx.x; j < n; j += kScaleThreads) {
      const int c = columns[(row_base + row) * k + j];
      if (c >= c0 && c < c1) {
        line[c] = static_cast<uint16_t>(dense::pack2<BF16>(listed[(row_base + row) * k + j], 0.0f) & 0xffffu);
      }
    }
  }
}

// du[compact row] = (unit * sum of the splits, in their order + the listed columns' lost
// amounts times their rows of W) / tau.
template <bool BF16>
__global__ void __launch_bounds__(256) sum_kernel(const float* __restrict__ parts, int64_t h, int k_blocks, int pairs,
                                                  int64_t room, const int* __restrict__ count, int row_base, int rows_cap,
                                                  const float* __restrict__ unit, const int2* __restrict__ fixes,
                                                  const uint16_t* __restrict__ weight, float inv_tau,
                                                  float* __restrict__ du) {
  grid_dependency_wait();
  launch_dependents();
  const int left = *count - row_base;
  const int rows = left < rows_cap ? left : rows_cap;
  if (rows <= 0) return;
  const int splits = dense::product_splits(rows, static_cast<int>(h), k_blocks, pairs, room);
  const int64_t part = static_cast<int64_t>((rows + dense::kTile - 1) / dense::kTile * dense::kTile) * h;
  const int per_row = static_cast<int>(h / 4);
  const int64_t vecs = static_cast<int64_t>(rows) * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < vecs;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row = static_cast<int>(i / per_row);
    const int col = static_cast<int>(i - static_cast<int64_t>(row) * per_row) * 4;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = 0; s < splits; ++s) {
      const float4 x = reinterpret_cast<const float4*>(parts + s * part)[i];
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    }
    const float f = unit[row_base + row];
    a = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
#pragma unroll
    for (int j = 0; j < kFixes; ++j) {
      const int2 fix = fixes[(static_cast<int64_t>(row_base) + row) * kFixes + j];
      const float x = __int_as_float(fix.y);
      if (x == 0.0f) continue;
      const uint2 w = *reinterpret_cast<const uint2*>(weight + static_cast<int64_t>(fix.x) * h + col);
      const float2 lo = dense::unpack2<BF16>(w.x), hi = dense::unpack2<BF16>(w.y);
      a = make_float4(fmaf(x, lo.x, a.x), fmaf(x, lo.y, a.y), fmaf(x, hi.x, a.z), fmaf(x, hi.y, a.w));
    }
    reinterpret_cast<float4*>(du + static_cast<int64_t>(row_base) * h)[i] =
        make_float4(a.x * inv_tau, a.y * inv_tau, a.z * inv_tau, a.w * inv_tau);
  }
}

// dhidden = grad * du for rows with a list, exact zeros for the others whatever their grad.
template <bool BF16>
__global__ void __launch_bounds__(256) backward_kernel(const float* __restrict__ du, const int* __restrict__ place,
                                                       const float* __restrict__ grad, int64_t rows, int64_t h,
                                                       uint16_t* __restrict__ out) {
  const int64_t vecs = rows * h / 8;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < vecs;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i * 8 / h, col = i * 8 - row * h;
    const int c = place[row];
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (c >= 0) {
      const float g = grad[row];
      const float4* from = reinterpret_cast<const float4*>(du + c * h + col);
      const float4 a = from[0], b = from[1];
      w = make_uint4(dense::pack2<BF16>(a.x * g, a.y * g), dense::pack2<BF16>(a.z * g, a.w * g),
                     dense::pack2<BF16>(b.x * g, b.y * g), dense::pack2<BF16>(b.z * g, b.w * g));
    }
    reinterpret_cast<uint4*>(out)[i] = w;
  }
}

// ----------------------------------------------------------------- workspace
struct Layout {
  int64_t tiles, pitch, cap, room;
  int n_tiles, out_tiles, k_blocks;
  size_t columns, logp, listed, rest, used, source, blocks, count, unit, shift, fixes, reference, uneven, uneven_counts, hidden, lookup, stats, dz, parts, total;
};

inline Layout layout(int64_t t, int64_t h, int64_t v, int k, bool train) {
  Layout L{};
  L.n_tiles = static_cast<int>((v + dense::kTile - 1) / dense::kTile);
  L.tiles = 2 * static_cast<int64_t>(L.n_tiles);
  L.pitch = (v + 63) / 64 * 64;
  L.cap = t;
  if (train) {
    int64_t rows = kBlockBytes / (L.pitch * 2) / dense::kTile * dense::kTile;
    const int64_t least = ((t + kMaxRowBlocks - 1) / kMaxRowBlocks + dense::kTile - 1) / dense::kTile * dense::kTile;
    if (rows < least) rows = least;
    if (rows < t) L.cap = rows;
  }
  L.out_tiles = static_cast<int>((h + dense::kTile - 1) / dense::kTile);
  L.k_blocks = static_cast<int>(L.pitch / 64);
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o = gemm::align256(o + bytes);
    return at;
  };
  L.columns = take(t * k * 4);
  L.logp = take(t * k * 4);
  L.listed = take(t * k * 4);
  L.rest = take(t * 4);
  L.used = take(t * 4);
  L.source = take(t * 4);
  L.blocks = take((t + kRowsPerBlock - 1) / kRowsPerBlock * 4);
  L.count = take(16);
  L.unit = take(t * 4);
  L.shift = take(t * 4);
  L.reference = take(t * 4);
  L.fixes = take(t * kFixes * 8);
  L.uneven = take(L.cap * 4);
  L.uneven_counts = take(kMaxRowBlocks * 4);
  L.hidden = take(t * h * 2);
  L.lookup = take(L.tiles * t * 4);
  L.stats = take(L.tiles * L.cap * 8);
  if (train) {
    L.dz = take(L.cap * L.pitch * 2);
    // Partial sums of the product, whose splits are chosen on the device from the
    // answered rows: 512 MB while that holds four splits of the whole block, and no
    // more than one split per pair of SMs can use.
    const int64_t one = (L.cap + dense::kTile - 1) / dense::kTile * dense::kTile * h;
    int64_t splits = (int64_t(1) << 27) / one;
    splits = splits < 4 ? 4 : splits;
    const int pairs = device_sm_count() / 2;
    L.room = one * (splits < pairs ? splits : pairs);
    L.parts = take(L.room * 4);
  }
  L.total = o;
  return L;
}

template <bool BF16>
int forward(int64_t t, int64_t h, const uint16_t* weight, int64_t v, int k, float temperature, const Layout& L, uint8_t* ws,
            float* loss, float* mass, float* du, cudaStream_t st) {
  using namespace gemm;
  auto ptr = [&](size_t at) { return ws + at; };
  int* columns = reinterpret_cast<int*>(ptr(L.columns));
  float* logp = reinterpret_cast<float*>(ptr(L.logp));
  float* listed = reinterpret_cast<float*>(ptr(L.listed));
  float* rest = reinterpret_cast<float*>(ptr(L.rest));
  int* used = reinterpret_cast<int*>(ptr(L.used));
  int* source = reinterpret_cast<int*>(ptr(L.source));
  int* count = reinterpret_cast<int*>(ptr(L.count));
  float* unit = reinterpret_cast<float*>(ptr(L.unit));
  int* shift = reinterpret_cast<int*>(ptr(L.shift));
  const float* reference = reinterpret_cast<const float*>(ptr(L.reference));
  int* uneven = reinterpret_cast<int*>(ptr(L.uneven));
  int2* fixes = reinterpret_cast<int2*>(ptr(L.fixes));
  uint16_t* hc = reinterpret_cast<uint16_t*>(ptr(L.hidden));
  uint32_t* lookup = reinterpret_cast<uint32_t*>(ptr(L.lookup));
  float2* stats = reinterpret_cast<float2*>(ptr(L.stats));
  const bool train = du != nullptr;
  uint16_t* dz = train ? reinterpret_cast<uint16_t*>(ptr(L.dz)) : nullptr;
  float* parts = train ? reinterpret_cast<float*>(ptr(L.parts)) : nullptr;
  const CUtensorMapDataType dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const float scale = kLog2e / temperature;
  const int pairs = device_sm_count() / 2;

  CUtensorMap m_w;
  int rc = make_map(&m_w, dt, weight, h, v, h * 2, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  for (int64_t r0 = 0; r0 < t; r0 += L.cap) {
    const int64_t rows = t - r0 < L.cap ? t - r0 : L.cap;
    CUtensorMap m_h, m_dz, m_dz_out, m_wn, m_parts;
    rc = make_map(&m_h, dt, hc + r0 * h, h, rows, h * 2, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc && train) rc = make_map(&m_dz_out, dt, dz, L.pitch, rows, L.pitch * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    dense::Params p{};
    p.count = count;
    p.row_base = static_cast<int>(r0);
    p.rows_cap = static_cast<int>(rows);
    p.cols = static_cast<int>(v);
    p.n_tiles = L.n_tiles;
    p.k_blocks = static_cast<int>((h + 63) / 64);
    // Four runs at least, six k-blocks (384 products) each at most.  Of a loss at T = 400,
    // V = 20000, tau = 2 the error is then 0.7 to 1.2 times that of products and sums in
    // fp32 throughout (in one run 2.2 times at H = 128 and 250); shorter runs are more
    // exact and slower (H = 1536: three k-blocks 1.22 against 1.09 ms at T = 3300).
    // Of 1 to 48 rows the error is 0.71 times fp32's on average (40 inputs; single ones 4
    // times over 1.5, 23 times below 1 / 1.5); three k-blocks 0.43, for 3 to 8 % of the time
    // at 48 rows.
    p.seg = (p.k_blocks + 3) / 4;
    if (p.seg > 6) p.seg = 6;
    p.scale = scale;
    p.list = k;
    p.columns = columns;
    p.lookup = lookup;
    p.reference = reference;
    p.listed = listed;
    p.stats = stats;
    p.store = train ? 1 : 0;
    rc = dense::launch<false, BF16>(m_h, m_w, train ? m_dz_out : m_h, p, st, "distill_logits");
    if (rc) return rc;
    int* uneven_count = reinterpret_cast<int*>(ptr(L.uneven_counts)) + r0 / L.cap;
    rc = dense::launch_after("distill_merge", merge_kernel<BF16>, static_cast<unsigned>((rows + kMergeRows - 1) / kMergeRows),
                             kMergeThreads, 0, st, stats, rows, static_cast<int>(L.tiles), count, static_cast<int>(r0), source,
                             used, logp, rest, k, scale, listed, loss, mass, reference, columns, dz, L.pitch,
                             train ? unit : nullptr, shift, fixes, uneven_count, uneven);
    if (rc) return rc;
    if (!train) continue;
    rc = dense::launch_after("distill_scale", scale_kernel<BF16>, static_cast<unsigned>(device_sm_count() * 8), kScaleThreads, 0,
                             st, dz, L.pitch, stats, rows, uneven_count, uneven, static_cast<int>(r0), used, columns, listed, k,
                             shift);
    if (rc) return rc;
    rc = make_map(&m_dz, dt, dz, L.pitch, rows, L.pitch * 2, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) rc = make_map(&m_wn, dt, weight, h, v, h * 2, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) {
      rc = make_map(&m_parts, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, parts, h, L.room / h, h * 4, 32, 32,
                    CU_TENSOR_MAP_SWIZZLE_128B);
    }
    if (rc) return rc;
    dense::Params d{};
    d.count = count;
    d.row_base = static_cast<int>(r0);
    d.rows_cap = static_cast<int>(rows);
    d.cols = static_cast<int>(h);
    d.n_tiles = L.out_tiles;
    d.k_blocks = L.k_blocks;
    d.seg = 16;
    d.room = L.room;
    rc = dense::launch<true, BF16>(m_dz, m_wn, m_parts, d, st, "distill_product");
    if (rc) return rc;
    rc = dense::launch_after("distill_sum", sum_kernel<BF16>, static_cast<unsigned>(device_sm_count() * 8), 256, 0, st, parts, h,
                             L.k_blocks, pairs, L.room, count, static_cast<int>(r0), static_cast<int>(rows), unit, fixes, weight,
                             1.0f / temperature, du);
    if (rc) return rc;
  }
  return SB_OK;
}

}  // namespace distill
}  // namespace sb

extern "C" {

size_t sb_distill_workspace_bytes(int64_t t, int64_t h, int64_t v, int k, int gradient) {
  if (t <= 0 || h <= 0 || v <= 0 || k <= 0) return 0;
  return sb::distill::layout(t, h, v, k, gradient != 0).total;
}

int sb_pad_rows(const uint16_t* in, int64_t rows, int64_t h, int64_t row_stride, int64_t width, uint16_t* out, void* stream) {
  SB_REQUIRE(rows >= 0 && h > 0 && width >= h && width % 8 == 0, "expected rows >= 0, h > 0 and width a multiple of 8, at least h");
  if (rows == 0) return SB_OK;
  SB_REQUIRE(in && out, "NULL pointer argument");
  SB_REQUIRE(row_stride >= 0 && sb::aligned(in, 2) && sb::aligned(out, 16), "bad stride or alignment");
  cudaStream_t st = sb::as_stream(stream);
  const int64_t blocks = (rows * (width / 8) + 256 * sb::distill::kPadAtOnce - 1) / (256 * sb::distill::kPadAtOnce), most = static_cast<int64_t>(sb::device_sm_count()) * 16;
  sb::distill::pad_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, st>>>(in, rows, h, row_stride, width, out);
  sb::count_launch();
  return sb::check_launch("pad_rows");
}

int sb_distill_check(const int64_t* indices, int64_t t, int k, int64_t v, int64_t* faults, void* stream) {
  SB_REQUIRE(faults != nullptr, "NULL faults");
  SB_REQUIRE(t >= 0 && k >= 1 && v > 0, "expected t >= 0, k >= 1, v > 0");
  cudaStream_t st = sb::as_stream(stream);
  cudaError_t e = cudaMemsetAsync(faults, 0, 2 * sizeof(int64_t), st);
  if (e != cudaSuccess) return sb::fail(SB_ECUDA, cudaGetErrorString(e));
  if (t == 0) return SB_OK;
  SB_REQUIRE(indices != nullptr, "NULL indices");
  SB_REQUIRE(t <= 0x7fffffff, "size out of range");
  sb::distill::check_kernel<<<static_cast<unsigned>((t + 7) / 8), 256, 0, st>>>(indices, t, k, v,
                                                                                reinterpret_cast<unsigned long long*>(faults));
  sb::count_launch();
  return sb::check_launch("distill check");
}

int sb_distill_forward(const uint16_t* hidden, int64_t t, int64_t h, const uint16_t* weight, int64_t v, int dtype,
                       const int64_t* indices, const void* logits, int logits_dtype, int k, const float* teacher_lse,
                       float temperature, float* loss, float* mass, float* du, int* place, void* workspace,
                       size_t workspace_bytes, void* stream) {
  using namespace sb::distill;
  SB_REQUIRE(t >= 0 && h > 0 && v > 0, "expected t >= 0, h > 0, v > 0");
  SB_REQUIRE(dtype == SB_F16 || dtype == SB_BF16, "hidden and weight must be fp16 or bf16");
  SB_REQUIRE(logits_dtype == SB_F16 || logits_dtype == SB_BF16 || logits_dtype == SB_F32, "logits must be fp16, bf16 or fp32");
  SB_REQUIRE(k >= 1 && k <= kMaxList, "k must be between 1 and 256");
  SB_REQUIRE(temperature > 0.0f && temperature < INFINITY, "temperature must be positive and finite");
  if (t == 0) return SB_OK;
  SB_REQUIRE(hidden && weight && indices && logits && loss && mass && place, "NULL pointer argument");
  SB_REQUIRE(h % 8 == 0, "hidden size must be a multiple of 8 (pad with zeros)");
  SB_REQUIRE(sb::aligned(hidden, 16) && sb::aligned(weight, 16), "operands must be 16-byte aligned");
  SB_REQUIRE(t <= (int64_t(1) << 30) && v <= (int64_t(1) << 30) && h <= (int64_t(1) << 20), "size out of range");
  const Layout L = layout(t, h, v, k, du != nullptr);
  SB_REQUIRE(!du || L.room / h < 0x7fffffff, "size out of range");
  if (!workspace || workspace_bytes < L.total) return sb::fail(SB_EWORKSPACE, "distillation workspace too small");
  cudaStream_t st = sb::as_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const unsigned blocks = static_cast<unsigned>((t + kRowsPerBlock - 1) / kRowsPerBlock);
  const int row_blocks = static_cast<int>((t + L.cap - 1) / L.cap);
  auto lists = [&](auto type, auto half) {
    using T = decltype(type);
    int* answered = reinterpret_cast<int*>(ws + L.blocks);
    answered_kernel<T><<<blocks, 256, 0, st>>>(indices, logits, teacher_lse, t, k, v, place, answered);
    sb::count_launch();
    if (int rc = sb::check_launch("distill_answered")) return rc;
    return sb::dense::launch_after(
        "distill_prepare", prepare_kernel<T, decltype(half)::value>, blocks, 256, 0, st, hidden, h, weight, indices, logits,
        teacher_lse, t, k, v, 1.0f / temperature, static_cast<int>(L.tiles), answered, place,
        reinterpret_cast<int*>(ws + L.source), reinterpret_cast<int*>(ws + L.count), reinterpret_cast<uint16_t*>(ws + L.hidden),
        reinterpret_cast<int*>(ws + L.columns), reinterpret_cast<float*>(ws + L.logp), reinterpret_cast<float*>(ws + L.rest),
        reinterpret_cast<int*>(ws + L.used), reinterpret_cast<uint32_t*>(ws + L.lookup),
        reinterpret_cast<float*>(ws + L.reference), reinterpret_cast<int*>(ws + L.uneven_counts), row_blocks, loss, mass);
  };
  auto typed = [&](auto half) {
    return logits_dtype == SB_F32 ? lists(float{}, half) : logits_dtype == SB_F16 ? lists(__half{}, half) : lists(__nv_bfloat16{}, half);
  };
  if (int rc = dtype == SB_BF16 ? typed(std::true_type{}) : typed(std::false_type{})) return rc;
  return dtype == SB_BF16
             ? forward<true>(t, h, weight, v, k, temperature, L, ws, loss, mass, du, st)
             : forward<false>(t, h, weight, v, k, temperature, L, ws, loss, mass, du, st);
}

int sb_distill_backward(const float* du, const int* place, const float* grad, int64_t t, int64_t h, void* dhidden, int dtype,
                        void* stream) {
  SB_REQUIRE(t >= 0 && h > 0 && h % 8 == 0, "expected t >= 0 and h a positive multiple of 8");
  SB_REQUIRE(dtype == SB_F16 || dtype == SB_BF16, "dhidden must be fp16 or bf16");
  if (t == 0) return SB_OK;
  SB_REQUIRE(du && place && grad && dhidden, "NULL pointer argument");
  cudaStream_t st = sb::as_stream(stream);
  const int64_t blocks = (t * h / 8 + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < sb::device_sm_count() * 8 ? blocks : sb::device_sm_count() * 8);
  if (dtype == SB_BF16) {
    sb::distill::backward_kernel<true><<<grid, 256, 0, st>>>(du, place, grad, t, h, static_cast<uint16_t*>(dhidden));
  } else {
    sb::distill::backward_kernel<false><<<grid, 256, 0, st>>>(du, place, grad, t, h, static_cast<uint16_t*>(dhidden));
  }
  sb::count_launch();
  return sb::check_launch("distill backward");
}

}  // extern "C"
