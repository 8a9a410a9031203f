// The k largest logits of each row, in falling order, and log sum exp(logits / tau).
//
// Order: by value, equal values by the lower index (+0 and -0 are equal, NaN counts
// above +inf).  Every element has a 64-bit key that carries exactly this order, its
// value's order-preserving bits above the complement of its index, so keys never
// tie and "the k largest" is unique: the result does not depend on the schedule.
//
// One pass over the row.  A CTA streams its row (or its share of one; a cluster of
// CTAs splits a row when there are few) in 16-byte vectors, kVecs per thread and round:
//   * log-sum-exp: each thread keeps a running maximum m and the sums of
//     2^((z - m) log2(e) / tau), rescaled only when a round's maximum passes m;
//   * selection: vectors with an element at or above a threshold go to a list in shared
//     memory, which is sorted out when the row has been read.
// The threshold is a guess.  The 32 streams of a CTA (warp, vector) lie side by side in
// the row, so the first round is an even sample of it; with s of n elements sampled, a
// threshold that k s / n + 2.5 to 5 sqrt(k s / n) + 3 of them pass (taken from the
// threads' maxima) leaves a few times k candidates and seldom fewer than k.  Where it does
// leave fewer, or the list overflows (a row of equal or masked logits; where a cluster shares a row, where
// fewer than k of all parts' candidates lie above each part's threshold), the row is read
// again with the
// threshold that cannot fail: the k-th largest of the threads' maxima over a first chunk
// in index order, raised to the k-th of all so far whenever the candidates have doubled;
// the list then holds a whole chunk and is worked off at its end, so any row is handled.
//
// Measured, k = 64 (copy rate in brackets): 3300 rows of 151936 fp16 203 us (154; the safe
// form alone 259, taking the vectors apart in the loop instead of listing them 703), fp32
// about 330 (307), one row 10.  What bounds it: for 16-bit logits instruction issue and the
// exponentials' unit, each about two thirds busy; for fp32 memory; for one row the chain of
// load, threshold, sort and exchange.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace sb {
namespace top {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kMaxK = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kVecs = 4;                      // 16-byte vectors per thread and chunk
constexpr int kChunk = kThreads * kVecs;      // vectors
constexpr int kBuffer = 2048;
constexpr int kRankable = 512;                // candidates that are sorted without a selection
constexpr int kMaxParts = 8;                  // CTAs of a row (the portable cluster limit)
constexpr int kPerSm = 4;

using u64 = unsigned long long;

// Order-preserving bits: negative values complemented, others with the top bit set.
__device__ __forceinline__ uint32_t rising32(uint32_t b) {
  if ((b << 1) == 0u) return 0x80000000u;                 // +0 and -0
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;  // NaN
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint32_t bits_of_rising32(uint32_t k) {
  return (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k;
}

// A logit type: vectors of kPer elements, keys, and "is any element above t".
// above(v, t) is true for every vector that holds a NaN, and for all when t is NaN.
template <typename T> struct Kind;

template <> struct Kind<float> {
  static constexpr int kPer = 4;
  static constexpr bool kBrain = false;
  static __device__ __forceinline__ uint32_t stored_key(const uint4* v, int i) {
    return rising32(reinterpret_cast<const uint32_t*>(v)[i]);
  }
  static __device__ __forceinline__ uint32_t key_at_most(float f) { return rising32(__float_as_uint(f)); }
  struct Limit { float t; };
  static __device__ __forceinline__ float value(const uint4& v, int i) {
    return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ float2 pair_value(const uint4& v, int i) {
    return make_float2(value(v, 2 * i), value(v, 2 * i + 1));
  }
  static __device__ __forceinline__ uint32_t scalar_key(const float* p) { return rising32(__float_as_uint(*p)); }
  static __device__ __forceinline__ float top(const uint4& v) {
    return fmaxf(fmaxf(value(v, 0), value(v, 1)), fmaxf(value(v, 2), value(v, 3)));
  }
  static __device__ __forceinline__ float top4(const uint4 (&q)[kVecs]) {
    return fmaxf(fmaxf(top(q[0]), top(q[1])), fmaxf(top(q[2]), top(q[3])));
  }
  static __device__ __forceinline__ Limit limit(float t) { return Limit{t}; }
  static __device__ __forceinline__ bool above(const uint4& v, Limit l) {
    return !(value(v, 0) <= l.t && value(v, 1) <= l.t && value(v, 2) <= l.t && value(v, 3) <= l.t);
  }
  static __device__ __forceinline__ void store(void* out, int64_t i, uint32_t key) {
    static_cast<uint32_t*>(out)[i] = bits_of_rising32(key);
  }
};

// The 16-bit types: the key sits in the upper half of the 32-bit one, so that the
// comparisons of the two are alike.
template <typename T, typename T2> struct Kind16 {
  static constexpr int kPer = 8;
  struct Limit { T2 t; };
  static __device__ __forceinline__ uint32_t word(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
  }
  static __device__ __forceinline__ T2 pair(const uint4& v, int i) {
    const uint32_t w = word(v, i);
    return *reinterpret_cast<const T2*>(&w);
  }
  static __device__ __forceinline__ Limit limit_of(T t) { return Limit{T2(t, t)}; }
};

template <> struct Kind<__half> : Kind16<__half, __half2> {
  static constexpr bool kBrain = false;
  static __device__ __forceinline__ uint32_t stored_key(const uint4* v, int i) {
    return rising(reinterpret_cast<const unsigned short*>(v)[i]);
  }
  static __device__ __forceinline__ uint32_t key_at_most(float f) { return rising(__half_as_ushort(__float2half_rd(f))); }
  static __device__ __forceinline__ uint32_t rising(uint32_t b) {
    if ((b & 0x7fffu) == 0u) return 0x80000000u;
    if ((b & 0x7fffu) > 0x7c00u) return 0xffff0000u;
    return ((b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u)) << 16;
  }
  static __device__ __forceinline__ float2 pair_value(const uint4& v, int i) { return __half22float2(pair(v, i)); }
  static __device__ __forceinline__ uint32_t scalar_key(const __half* p) { return rising(__half_as_ushort(*p)); }
  static __device__ __forceinline__ __half2 top2(const uint4& v) {
    return __hmax2_nan(__hmax2_nan(pair(v, 0), pair(v, 1)), __hmax2_nan(pair(v, 2), pair(v, 3)));
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const float2 f = __half22float2(top2(v));
    return fmaxf(f.x, f.y);
  }
  // (Of the numbers: a NaN is left out.)
  static __device__ __forceinline__ float top4(const uint4 (&q)[kVecs]) {
    const float2 f = __half22float2(__hmax2(__hmax2(top2(q[0]), top2(q[1])), __hmax2(top2(q[2]), top2(q[3]))));
    return fmaxf(f.x, f.y);
  }
  // Every threshold is a value of the type (or NaN), so the rounding is exact.
  static __device__ __forceinline__ Limit limit(float t) { return limit_of(__float2half_rn(t)); }
  static __device__ __forceinline__ bool above(const uint4& v, Limit l) { return !__hble2(top2(v), l.t); }
  static __device__ __forceinline__ void store(void* out, int64_t i, uint32_t key) {
    const uint32_t k = key >> 16;
    static_cast<unsigned short*>(out)[i] = static_cast<unsigned short>((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu));
  }
};

template <> struct Kind<__nv_bfloat16> : Kind16<__nv_bfloat16, __nv_bfloat162> {
  static constexpr bool kBrain = true;
  static __device__ __forceinline__ uint32_t stored_key(const uint4* v, int i) {
    return rising(reinterpret_cast<const unsigned short*>(v)[i]);
  }
  static __device__ __forceinline__ uint32_t key_at_most(float f) { return rising(__bfloat16_as_ushort(__float2bfloat16_rd(f))); }
  static __device__ __forceinline__ uint32_t rising(uint32_t b) {
    if ((b & 0x7fffu) == 0u) return 0x80000000u;
    if ((b & 0x7fffu) > 0x7f80u) return 0xffff0000u;
    return ((b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u)) << 16;
  }
  static __device__ __forceinline__ float2 pair_value(const uint4& v, int i) {
    const uint32_t w = word(v, i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t scalar_key(const __nv_bfloat16* p) { return rising(__bfloat16_as_ushort(*p)); }
  static __device__ __forceinline__ __nv_bfloat162 top2(const uint4& v) {
    return __hmax2_nan(__hmax2_nan(pair(v, 0), pair(v, 1)), __hmax2_nan(pair(v, 2), pair(v, 3)));
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const float2 f = __bfloat1622float2(top2(v));
    return fmaxf(f.x, f.y);
  }
  // (Of the numbers: a NaN is left out.)
  static __device__ __forceinline__ float top4(const uint4 (&q)[kVecs]) {
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(top2(q[0]), top2(q[1])), __hmax2(top2(q[2]), top2(q[3]))));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ Limit limit(float t) { return limit_of(__float2bfloat16_rn(t)); }
  static __device__ __forceinline__ bool above(const uint4& v, Limit l) { return !__hble2(top2(v), l.t); }
  static __device__ __forceinline__ void store(void* out, int64_t i, uint32_t key) {
    const uint32_t k = key >> 16;
    static_cast<unsigned short*>(out)[i] = static_cast<unsigned short>((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu));
  }
};

// The value whose key is `key` (as fp32; exact for the 16-bit types), NaN for NaN.
template <typename T> __device__ __forceinline__ float value_of_key(uint32_t key);
template <> __device__ __forceinline__ float value_of_key<float>(uint32_t key) { return __uint_as_float(bits_of_rising32(key)); }
template <> __device__ __forceinline__ float value_of_key<__nv_bfloat16>(uint32_t key) {
  const uint32_t k = key >> 16;
  return __uint_as_float(((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu)) << 16);
}
template <> __device__ __forceinline__ float value_of_key<__half>(uint32_t key) {
  const uint32_t k = key >> 16;
  return __half2float(__ushort_as_half(static_cast<unsigned short>((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu))));
}

__device__ __forceinline__ u64 full_key(uint32_t key, int64_t index) {
  return (static_cast<u64>(key) << 32) | (0xffffffffull - static_cast<u64>(index));
}

struct Scratch {
  uint4 list[kChunk];    // listed vectors of a chunk
  int list_at[kChunk];   // and where they are
  u64 buf[kBuffer];      // candidates
  u64 sel[kMaxK];
  int hist[256];
  int listed[3];         // of chunk c: entry c % 3, cleared while chunk c - 1 lists
  int count, picked, digit, need, bin;
  uint32_t bound;
  u64 limit;             // keys at or below it may be missing among the candidates
  float warp_m[kThreads / 32], warp_s[kThreads / 32];
  float m, s;            // this CTA's log-sum-exp parts
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ u64 pack2(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(u64 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Cut sc.buf[0, n) to its `want` largest keys (all of them when n <= want): they end in
// sc.sel, in no order; returns how many.  Radix selection from the top digit, left as
// soon as a digit's entries are exactly those still wanted; digits in which all keys
// agree (a 16-bit type's lower value bits, an index's leading ones) are left out.
// All threads call it; they have passed a barrier since the last write to the buffer.
template <int VALUE_BITS>
__device__ __forceinline__ int select(int n, int want, int64_t v, Scratch& sc) {
  const int tid = threadIdx.x;
  if (tid == 0) sc.picked = 0;
  u64 prefix = 0, mask = 0;
  if (n > want) {
    int need = want;
    for (int shift = 56; shift >= 0; shift -= 8) {
      if (shift >= 32 ? shift < 64 - VALUE_BITS : (shift > 0 && v <= (int64_t(1) << shift))) continue;
      sc.hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const u64 k = sc.buf[i];
        if ((k & mask) == prefix) atomicAdd(&sc.hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid < 32) {
        // Lane l owns digits 255 - 8 l .. 248 - 8 l: falling order.
        int own[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          own[j] = sc.hist[255 - 8 * tid - j];
          sum += own[j];
        }
        int before = sum;
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, before, o);
          if (tid >= o) before += up;
        }
        before -= sum;
        if (before < need && need <= before + sum) {
          bool open = true;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (open && before + own[j] >= need) {
              sc.digit = 255 - 8 * tid - j;
              sc.need = need - before;
              sc.bin = own[j];
              open = false;
            }
            before += own[j];
          }
        }
      }
      __syncthreads();
      prefix |= static_cast<u64>(sc.digit) << shift;
      mask |= 255ull << shift;
      need = sc.need;
      if (sc.bin == need) break;
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const u64 k = sc.buf[i];
    if ((k & mask) >= prefix) sc.sel[atomicAdd(&sc.picked, 1)] = k;
  }
  __syncthreads();
  return n < want ? n : want;
}

// sc.buf[0, n) as runs of 32, each in falling order (the last filled up with zeros).
// Run i is warp i % 8's.
__device__ __forceinline__ void sort_runs(int n, Scratch& sc) {
  const int lane = threadIdx.x & 31;
  for (int at = (threadIdx.x & ~31); at < n; at += kThreads) {
    u64 key = at + lane < n ? sc.buf[at + lane] : 0;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
      for (int o = size / 2; o; o /= 2) {
        const u64 other = __shfl_xor_sync(0xffffffffu, key, o);
        const bool upper = (lane & o) != 0, falling = (lane & size) == 0;
        key = (upper == falling) == (key > other) ? other : key;
      }
    }
    sc.buf[at + lane] = key;
  }
}

// The r-th largest of the threads' keys: each warp's sorted, then the smallest key that
// fewer than r keys exceed.  Ends with a barrier.
__device__ __forceinline__ uint32_t rth_largest(uint32_t key, int r, Scratch& sc) {
  const int lane = threadIdx.x & 31;
  uint32_t* sorted = reinterpret_cast<uint32_t*>(sc.buf);
  if (threadIdx.x == 0) sc.bound = 0xffffffffu;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
    for (int o = size / 2; o; o /= 2) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, key, o);
      const bool keep_large = ((lane & o) == 0) == ((lane & size) == 0);
      key = keep_large ? max(key, other) : min(key, other);
    }
  }
  sorted[threadIdx.x] = key;
  __syncthreads();
  int above = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t* run = sorted + 32 * w;
    int here = 0;
#pragma unroll
    for (int o = 16; o; o /= 2) here += run[here + o - 1] > key ? o : 0;
    above += here + (run[here] > key ? 1 : 0);
  }
  uint32_t low = above < r ? key : 0xffffffffu;
  low = __reduce_min_sync(0xffffffffu, low);
  if (lane == 0) atomicMin(&sc.bound, low);
  __syncthreads();
  return sc.bound;
}

// emit(key, number of keys above it) for every key of the sorted runs.
template <typename F>
__device__ __forceinline__ void rank_runs(int n, const Scratch& sc, F emit) {
  const int lane = threadIdx.x & 31;
  for (int at = (threadIdx.x & ~31); at < n; at += kThreads) {
    const u64 key = sc.buf[at + lane];
    int rank = lane;
    for (int run = 0; run < n; run += 32) {
      if (run == at) continue;
      int above = 0;
#pragma unroll
      for (int o = 16; o; o /= 2) above += sc.buf[run + above + o - 1] > key ? o : 0;
      rank += above + (sc.buf[run + above] > key ? 1 : 0);
    }
    if (at + lane < n) emit(key, rank);
  }
}

// PARTS: the CTAs of a cluster that share each row (with one per row, the code keeps
// nothing for a second attempt and needs fewer registers).
template <typename T, int PARTS>
__global__ void __launch_bounds__(kThreads, PARTS > 1 ? 3 : kPerSm) top_kernel(const T* __restrict__ logits, int64_t v, int64_t pitch,
                                                          int k, float slack, float scale, float inv_tau, void* __restrict__ values,
                                                          int64_t* __restrict__ indices, float* __restrict__ lse) {
  using K = Kind<T>;
  constexpr int kBits = 8 * sizeof(T);
  __shared__ __align__(16) Scratch sc;
  cg::cluster_group cluster = cg::this_cluster();
  constexpr bool CLUSTER = PARTS > 1;
  constexpr int parts = PARTS;
  const int part = CLUSTER ? static_cast<int>(cluster.block_rank()) : 0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t low16 = sizeof(T) == 4 ? 0xff800000u : (K::kBrain ? 0xff80ff80u : 0xfc00fc00u);
  const uint4 nothing = make_uint4(low16, low16, low16, low16);  // -inf
  uint4 cur[kVecs];

  // [0, head) and [tail, v) are read one element at a time, the vectors between them
  // are shared among the parts in runs of whole vectors.
  const int64_t row = blockIdx.x / parts;
  const T* x = logits + row * pitch;
  int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
  if (head > v) head = static_cast<int>(v);
  const int vecs = static_cast<int>((v - head) / K::kPer);
  const int tail = head + vecs * K::kPer;
  const int w0 = static_cast<int>(static_cast<int64_t>(vecs) * part / parts);
  const int w1 = static_cast<int>(static_cast<int64_t>(vecs) * (part + 1) / parts);
  // Stream j of this warp is vectors [(j kWarps + warp) rounds 32, + 32 rounds) of the part.
  const int rounds = (w1 - w0 + kChunk - 1) / kChunk;
  const uint4* xs = reinterpret_cast<const uint4*>(x + head) + w0 + (warp * rounds) * 32 + lane;
  const int left = w1 - w0 - (warp * rounds) * 32 - lane;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) cur[j] = rounds && j * kWarps * rounds * 32 < left ? __ldcs(xs + j * kWarps * rounds * 32) : nothing;
  if (tid == 0) sc.count = sc.listed[0] = sc.listed[1] = sc.listed[2] = 0;
  // scale = log2(e) / tau.  The reference m2 is the rounded product the exponents
  // use, so that log2(sum) + m2 carries no error from rounding it.
  float m = -1e30f, m2 = fmaxf(-1e30f * scale, -3e38f);
  float s = 0.0f;
  const u64 scale2 = pack2(scale, scale);
  u64 s2 = 0;  // two running sums
  auto raise = [&](float to) {
    const float n2 = to * scale;
    const float f = exp2_fast(m2 - n2);
    const float2 both = unpack2(s2);
    s *= f;
    s2 = pack2(both.x * f, both.y * f);
    m = to;
    m2 = n2;
  };
  u64 limit_key = 0;  // elements whose key is above it are candidates
  typename K::Limit limit = K::limit(__int_as_float(0x7fffffff));
  // Vectors with an element above the value of `key`; NaN (all of them) for none.  A
  // value between -0 and +0 does not exist: the one below stands in.
  auto set_limit = [&](uint32_t key) {
    uint32_t as = key;
    if constexpr (kBits == 16) as = key & 0xffff0000u;
    if (as == 0x7fffffffu || as == 0x7fff0000u) as -= kBits == 16 ? 0x10000u : 1u;
    limit = K::limit(value_of_key<T>(as));
  };
  // Cut the buffer to k and raise the threshold to the k-th.
  auto cut = [&](int n) {
    const int kept = select<kBits>(n, k, v, sc);
    u64 low = ~0ull;
    for (int i = tid; i < kept; i += kThreads) sc.buf[i] = sc.sel[i];
    for (int i = lane; i < kept; i += 32) low = sc.sel[i] < low ? sc.sel[i] : low;
    for (int o = 16; o; o >>= 1) {
      const u64 other = __shfl_xor_sync(0xffffffffu, low, o);
      low = other < low ? other : low;
    }
    if (kept == k) limit_key = low;
    if (tid == 0) sc.count = kept;
    __syncthreads();
    return kept;
  };
  // The first threshold: the r-th largest of the threads' maxima over `cur`.
  auto threshold = [&](bool any, int r) {
    float best = K::top4(cur);
    if (!(best == best)) best = -INFINITY;
    // The maximum of rank r - 1 among all.  A NaN only lowers the maximum seen here,
    // which a bound may be; threads without an element come last.
    const uint32_t t = rth_largest(any ? rising32(__float_as_uint(best)) : 0u, r, sc);
    limit_key = 0;
    limit = K::limit(__int_as_float(0x7fffffff));
    // As a value of the type, rounded down; candidates are at or above it.  (Below the
    // key of -inf there is no value, and no bound.)
    const float f = __uint_as_float(bits_of_rising32(t));
    if (t && f == f) {
      const uint32_t key = K::key_at_most(f);
      limit_key = static_cast<u64>(key) << 32;
      set_limit(key - 1);
    }
  };
  auto one = [&](int i) {  // an element of the row's unaligned ends
    const uint32_t key = K::scalar_key(x + i);
    const float f = value_of_key<T>(key);
    if (f > m) raise(f);
    s += exp2_fast(fmaf(f, scale, -m2));
    if (full_key(key, i) > limit_key) sc.buf[atomicAdd(&sc.count, 1)] = full_key(key, i);
  };
  auto add = [&](const uint4& q, u64 minus) {
#pragma unroll
    for (int i = 0; i < K::kPer; i += 2) {
      const float2 z = K::pair_value(q, i / 2);
      const float2 e = unpack2(fma2(pack2(z.x, z.y), scale2, minus));
      s2 = add2(s2, pack2(exp2_fast(e.x), exp2_fast(e.y)));
    }
  };
  // Listed vectors' elements that pass to the buffer, in batches that it has room for.
  // All threads call it, behind a barrier; ends with one.
  auto work_off = [&](int listed) {
    int done = 0, count = sc.count;
    __syncthreads();
    while (done < listed) {
      const int batch = min(listed - done, kBuffer - count);
      for (int i = done + tid; i < done + batch; i += kThreads) {
        const u64 key = full_key(K::stored_key(&sc.list[i / K::kPer], i % K::kPer), sc.list_at[i / K::kPer] + i % K::kPer);
        if (key > limit_key) sc.buf[atomicAdd(&sc.count, 1)] = key;
      }
      done += batch;
      __syncthreads();
      count = sc.count;
      __syncthreads();
      if (count >= kBuffer / 2) count = cut(count);
    }
    return count;
  };
  const bool ends = part == 0;
  bool safe = true;
  {
    // The guess (its first round is loaded already).
    // `want` elements of the sample above the threshold; as they fall into the threads at
    // random, so many threads' maxima are above it too.  (k maxima would never fail.)
    const float share = static_cast<float>(k) / max(rounds * parts, 1);
    const float want = share + slack * sqrtf(share) + 3.0f;
    const float groups = static_cast<float>(max(min(kThreads, w1 - w0), 1));
    const int r = min(k, static_cast<int>(groups * (1.0f - __expf(-want / groups))) + 1);
    threshold(left > 0, r);
    if (ends && tid < head) one(tid);
    // Every stream of the thread full (all but the part's last ones): no bounds to look at.
    auto stream = [&](auto whole) {
      constexpr bool full = decltype(whole)::value;
      const uint4* at = xs;  // of the round that is loaded next
      const int stride = kWarps * rounds * 32;
      auto load = [&](uint4 (&q)[kVecs], int c) {
        at += 32;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          if (full) {
            if (c < rounds) q[j] = __ldcs(at + j * stride);
          } else {
            q[j] = c < rounds && j * stride + c * 32 < left ? __ldcs(at + j * stride) : nothing;
          }
        }
      };
      auto eat = [&](const uint4 (&q)[kVecs], int c) {
        const float tops = K::top4(q);
        if (tops > m) raise(tops);
        const u64 minus = pack2(-m2, -m2);
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          if (K::above(q[j], limit) && (full || j * stride + c * 32 < left)) {
            const int slot = atomicAdd(&sc.listed[0], 1);
            if (slot < kChunk) {
              sc.list[slot] = q[j];
              sc.list_at[slot] = head + (w0 + warp * rounds * 32 + lane + j * stride + c * 32) * K::kPer;
            }
          }
          add(q[j], minus);
        }
      };
      // Two rounds in registers by turns.  (Past an overflow of the list it is of no use to
      // go on: the other form will do it.)
      uint4 other[kVecs];
      for (int c = 0; c < rounds; c += 2) {
        load(other, c + 1);
        eat(cur, c);
        if (c + 1 >= rounds) break;
        load(cur, c + 2);
        eat(other, c + 1);
        if (*reinterpret_cast<volatile int*>(&sc.listed[0]) > kChunk) break;
      }
    };
    if (__all_sync(0xffffffffu, ((kVecs - 1) * kWarps * rounds + rounds - 1) * 32 < left)) {
      stream(std::true_type{});
    } else {
      stream(std::false_type{});
    }
    __syncthreads();
    const int listed = sc.listed[0];
    if (listed <= kChunk) {
      const int count = work_off(listed * K::kPer);
      // (The tail's elements are still to come, the guess counts without them.  A part
      // among others need not have k: the parts are judged together below.)
      safe = parts == 1 && count < k && limit_key != 0;
    }
  }
  int kept = 0, rank = 0;
  u64 own_key = 0;
  for (bool again = false;; again = true) {
    if (safe || (CLUSTER && again)) {
      const uint4* xv = reinterpret_cast<const uint4*>(x + head) + w0 + tid;
      const int own = w1 - w0 - tid;  // vectors from this thread's first on
      __syncthreads();
      if (tid == 0) sc.count = sc.listed[0] = sc.listed[1] = sc.listed[2] = 0;
      m = -1e30f;
      m2 = fmaxf(-1e30f * scale, -3e38f);
      s = 0.0f;
      s2 = 0;
      auto load = [&](int first) {
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          const int w = first + j * kThreads;
          cur[j] = w < own ? __ldg(xv + w) : nothing;
        }
      };
      load(0);
      threshold(own > 0, k);
      // The head before the vectors and the tail behind them: in index order, as the
      // strict threshold asks.
      if (ends && tid < head) one(tid);
      int turn = 0;
      for (int first = 0; first < w1 - w0; first += kChunk) {
        const int next_turn = turn == 2 ? 0 : turn + 1;
        if (tid == 0) sc.listed[next_turn] = 0;  // read last before the previous barrier
        const float tops = K::top4(cur);
        if (tops > m) raise(tops);
        const u64 minus = pack2(-m2, -m2);
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          if (K::above(cur[j], limit) && first + j * kThreads < own) {
            const int at = atomicAdd(&sc.listed[turn], 1);
            sc.list[at] = cur[j];
            sc.list_at[at] = head + (w0 + tid + first + j * kThreads) * K::kPer;
          }
          add(cur[j], minus);
        }
        load(first + kChunk);
        __syncthreads();
        const int listed = sc.listed[turn] * K::kPer;
        turn = next_turn;
        if (listed) {
          const int count = work_off(listed);
          if (count >= 2 * k) cut(count);
          // Strictly: later vectors have higher indices.
          if (limit_key & 0xffffffffull) set_limit(static_cast<uint32_t>(limit_key >> 32));
        }
      }
    }
    if (ends && tid < v - tail) one(tail + tid);

    // Log-sum-exp of this CTA.
    {
      const float2 both = unpack2(s2);
      s += both.x + both.y;
    }
    for (int o = 16; o; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m2, o), os = __shfl_xor_sync(0xffffffffu, s, o);
      const float big = fmaxf(m2, om);
      s = s * exp2_fast(m2 - big) + os * exp2_fast(om - big);
      m2 = big;
    }
    if (lane == 0) {
      sc.warp_m[warp] = m2;
      sc.warp_s[warp] = s;
    }
    __syncthreads();
    // This CTA's k largest in falling order.
    int n = sc.count;
    __syncthreads();
    if (n > kRankable) n = cut(n);
    sort_runs(n, sc);
    __syncthreads();
    kept = n < k ? n : k;
    rank_runs(n, sc, [&](u64 key, int rank) {
      if (rank < kept) sc.sel[rank] = key;
    });
    for (int i = kept + tid; i < kMaxK; i += kThreads) sc.sel[i] = 0;
    if (tid == 0) {
      float big = sc.warp_m[0];
      for (int w = 1; w < kThreads / 32; ++w) big = fmaxf(big, sc.warp_m[w]);
      float sum = 0.0f;
      for (int w = 0; w < kThreads / 32; ++w) sum += sc.warp_s[w] * exp2_fast(sc.warp_m[w] - big);
      sc.m = big;
      sc.s = sum;
      sc.limit = kept == k || safe || again ? 0 : limit_key;
    }
    if constexpr (CLUSTER) {
      cluster.sync();
    } else {
      __syncthreads();
    }
    // An entry's place in the output: its place here and the entries above it in the
    // other parts' lists, searched side by side (a remote load takes about as long as
    // eight at once).
    static_assert(kMaxK <= kThreads, "an entry per thread");
    rank = tid;
    own_key = tid < kept ? sc.sel[tid] : 0;
    if constexpr (!CLUSTER) {
      break;
    } else {
      const int first_o = 1 << (31 - __clz(k));
      if (tid < kept) {
        int above[parts] = {};
        for (int o = first_o; o; o >>= 1) {
          u64 at[parts];
#pragma unroll
          for (int c = 0; c < parts; ++c) at[c] = above[c] + o <= k ? cluster.map_shared_rank(&sc, c)->sel[above[c] + o - 1] : 0;
#pragma unroll
          for (int c = 0; c < parts; ++c) above[c] += at[c] > own_key ? o : 0;
        }
        rank = 0;
#pragma unroll
        for (int c = 0; c < parts; ++c) rank += above[c];
      }
      // Nothing is missing if k entries lie above every part's limit (lane c counts part c's).
      const Scratch* theirs = cluster.map_shared_rank(&sc, lane & (parts - 1));
      u64 limit_of_all = theirs->limit;
#pragma unroll
      for (int o = parts / 2; o; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, limit_of_all, o);
        limit_of_all = other > limit_of_all ? other : limit_of_all;
      }
      if (limit_of_all == 0) break;
      int above = 0;
      for (int o = first_o; o; o >>= 1) above += above + o <= k && theirs->sel[above + o - 1] > limit_of_all ? o : 0;
#pragma unroll
      for (int o = parts / 2; o; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
      if (above >= k) break;
      cluster.sync();  // all have read the lists that are made anew
    }
  }
  if (tid < kept && rank < k) {
    K::store(values, row * k + rank, static_cast<uint32_t>(own_key >> 32));
    indices[row * k + rank] = static_cast<int64_t>(0xffffffffull - (own_key & 0xffffffffull));
  }
  if (part == 0 && warp == 0) {
    const Scratch* from = CLUSTER && lane < parts ? cluster.map_shared_rank(&sc, lane) : &sc;
    u64 top = from->sel[0];
    float big = from->m, sum = lane < parts ? from->s : 0.0f;
    for (int o = parts / 2; o; o >>= 1) {
      const u64 t = __shfl_xor_sync(0xffffffffu, top, o);
      top = t > top ? t : top;
      const float om = __shfl_xor_sync(0xffffffffu, big, o), os = __shfl_xor_sync(0xffffffffu, sum, o);
      const float to = fmaxf(big, om);
      sum = sum * exp2_fast(big - to) + os * exp2_fast(om - to);
      big = to;
    }
    // The largest logit decides the cases that the sum cannot: NaN and infinities as
    // they are, and logits beyond 1e30 (a row of the type's lowest value), where the
    // logarithm of the count is below the logit's rounding.
    const float topv = value_of_key<T>(static_cast<uint32_t>(top >> 32));
    if (lane == 0) {
      lse[row] = (isnan(topv) || isinf(topv)) ? topv
                 : sum > 0.0f && !isinf(big)     ? (big + log2f(sum)) * 0.6931471805599453f
                                                  : topv * inv_tau;
    }
  }
  if (CLUSTER) cluster.sync();  // the others' lists stay until all have read them
}

template <typename T>
int launch(const void* logits, int64_t rows, int64_t v, int64_t pitch, int k, float temperature, void* values,
           int64_t* indices, float* lse, cudaStream_t st) {
  // Few rows are split over a cluster (at most the portable eight CTAs): to an SM's one
  // CTA in parts of half a chunk, to eight in parts of two (300 rows of 151936 fp16: four
  // parts 40 us, two 51; 600 rows in two 83, in one 68).
  int parts = 1;
  const int64_t sms = device_sm_count(), chunk = kChunk * Kind<T>::kPer;
  while (parts < kMaxParts && rows * parts * 2 <= 8 * sms &&
         v / (parts * 2) >= (rows * parts * 2 <= sms ? chunk / 2 : 2 * chunk)) {
    parts *= 2;
  }
  // How far the guess stays on the safe side, in standard deviations of the sample's count.
  // While every row is resident, one that is read again is the whole call's time: 592 rows
  // of 32001 bf16, k = 200, take 31.1 us at 2.5 and 24.6 at 4 (means of 16 inputs); 37 rows,
  // whose parts are judged together, took 21 us at 2.5 for 6 of 32 inputs and 10.6 at 5 for
  // all.  With more rows the others hide part of it and fewer candidates count for more:
  // fp16, 2.5 against 4, 1000 rows of 151936 73 and 80 us, 2000 rows 129 and 137, 3300 203
  // and 210; but only where the sample holds few of the k, so that the constant 3 is most of
  // the margin (bf16: 16 of them, 2000 rows of 32001, k = 64, 49 and 51; 50 of them, 1000
  // rows of 32001, k = 200, 46 and 40).  (It costs where the guess would have held: 300
  // rows of 151936 34.3 and 35.7.)
  const bool spare = rows > static_cast<int64_t>(kPerSm) * sms && k * chunk <= 32 * v;
  const float slack = spare ? 2.5f : parts > 1 ? 5.0f : 4.0f;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  auto kern = parts == 1 ? top_kernel<T, 1> : parts == 2 ? top_kernel<T, 2> : parts == 4 ? top_kernel<T, 4> : top_kernel<T, 8>;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<const T*>(logits), v, pitch, k, slack,
                                           1.4426950408889634f / temperature, 1.0f / temperature, values, indices, lse);
  if (e != cudaSuccess) return fail(SB_ECUDA, std::string("top_kernel: ") + cudaGetErrorString(e));
  count_launch();
  return check_launch("top_kernel");
}

}  // namespace top
}  // namespace sb

extern "C" {

int sb_top_logits(const void* logits, int dtype, int64_t rows, int64_t v, int64_t row_stride, int k, float temperature,
                  void* values, int64_t* indices, float* lse, void* stream) {
  SB_REQUIRE(dtype == SB_F16 || dtype == SB_F32 || dtype == SB_BF16, "logits must be fp16, bf16 or fp32");
  SB_REQUIRE(rows >= 0 && v > 0 && v <= 0x7fffffff, "expected rows >= 0 and 0 < v < 2^31");
  SB_REQUIRE(k >= 1 && k <= sb::top::kMaxK && k <= v, "k must be between 1 and min(v, 256)");
  SB_REQUIRE(temperature > 0.0f && temperature < INFINITY, "temperature must be positive and finite");
  if (rows == 0) return SB_OK;
  SB_REQUIRE(rows <= (int64_t(1) << 26), "too many rows");
  SB_REQUIRE(logits && values && indices && lse, "NULL pointer argument");
  cudaStream_t st = sb::as_stream(stream);
  if (dtype == SB_F32) return sb::top::launch<float>(logits, rows, v, row_stride, k, temperature, values, indices, lse, st);
  if (dtype == SB_F16) return sb::top::launch<__half>(logits, rows, v, row_stride, k, temperature, values, indices, lse, st);
  return sb::top::launch<__nv_bfloat16>(logits, rows, v, row_stride, k, temperature, values, indices, lse, st);
}

}  // extern "C"
