// The k largest logits of each row, in falling order, and log sum exp(logits / tau).
//
// Order: by value, equal values by the lower index (+0 and -0 are equal, NaN counts
// above +inf).  Every element has a 64-bit key that carries exactly this order, its
// value's order-preserving bits above the complement of its index, so keys never
// tie and "the k largest" is unique: the result does not depend on the schedule.
//
// One pass over the row.  A CTA streams its row (or its share of one; a cluster of
// CTAs splits a row when there are few) in 16-byte vectors:
//   * log-sum-exp: each thread keeps a running maximum m and the sum of
//     2^((z - m) log2(e) / tau), rescaled only when a vector's maximum passes m;
//   * selection: elements above a threshold go to a shared-memory buffer.  The first
//     threshold is the k-th largest of the threads' maxima over their first vectors
//     (k different elements reach it, so nothing that belongs to the k largest is
//     below it); whenever the buffer has passed kKeep entries at a chunk's end it is
//     cut to its k largest and the k-th becomes the threshold, strictly, because
//     later elements of equal value have higher indices.  A chunk adds at most its
//     own size, so the buffer cannot overflow for any input.
// The test costs one packed maximum per two 16-bit elements; the buffer sees a few
// hundred elements of a row of 10^5.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"

namespace sb {
namespace top {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kMaxK = 256;
constexpr int kKeep = 2048;
constexpr int kVecs = 2;  // 16-byte vectors per thread and chunk

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
  struct Limit { float t; };
  static __device__ __forceinline__ float value(const uint4& v, int i) {
    return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ uint32_t key(const uint4& v, int i) {
    return rising32(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ uint32_t scalar_key(const float* p) { return rising32(__float_as_uint(*p)); }
  static __device__ __forceinline__ float top(const uint4& v) {
    return fmaxf(fmaxf(value(v, 0), value(v, 1)), fmaxf(value(v, 2), value(v, 3)));
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
  static __device__ __forceinline__ uint32_t bits(const uint4& v, int i) {
    const uint32_t w = word(v, i >> 1);
    return (i & 1) ? w >> 16 : w & 0xffffu;
  }
  static __device__ __forceinline__ Limit limit_of(T t) { return Limit{T2(t, t)}; }
};

template <> struct Kind<__half> : Kind16<__half, __half2> {
  static __device__ __forceinline__ uint32_t rising(uint32_t b) {
    if ((b & 0x7fffu) == 0u) return 0x80000000u;
    if ((b & 0x7fffu) > 0x7c00u) return 0xffff0000u;
    return ((b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u)) << 16;
  }
  static __device__ __forceinline__ float value(const uint4& v, int i) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits(v, i))));
  }
  static __device__ __forceinline__ uint32_t key(const uint4& v, int i) { return rising(bits(v, i)); }
  static __device__ __forceinline__ uint32_t scalar_key(const __half* p) { return rising(__half_as_ushort(*p)); }
  static __device__ __forceinline__ __half2 top2(const uint4& v) {
    return __hmax2_nan(__hmax2_nan(pair(v, 0), pair(v, 1)), __hmax2_nan(pair(v, 2), pair(v, 3)));
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const float2 f = __half22float2(top2(v));
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
  static __device__ __forceinline__ uint32_t rising(uint32_t b) {
    if ((b & 0x7fffu) == 0u) return 0x80000000u;
    if ((b & 0x7fffu) > 0x7f80u) return 0xffff0000u;
    return ((b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u)) << 16;
  }
  static __device__ __forceinline__ float value(const uint4& v, int i) {
    const uint32_t w = word(v, i >> 1);
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ uint32_t key(const uint4& v, int i) { return rising(bits(v, i)); }
  static __device__ __forceinline__ uint32_t scalar_key(const __nv_bfloat16* p) { return rising(__bfloat16_as_ushort(*p)); }
  static __device__ __forceinline__ __nv_bfloat162 top2(const uint4& v) {
    return __hmax2_nan(__hmax2_nan(pair(v, 0), pair(v, 1)), __hmax2_nan(pair(v, 2), pair(v, 3)));
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const float2 f = __bfloat1622float2(top2(v));
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

template <typename T> constexpr int chunk_elems() { return kThreads * kVecs * Kind<T>::kPer; }
// The buffer: what one chunk (and the row's unaligned ends) can add to kKeep entries.
template <typename T> constexpr int capacity() { return kKeep + chunk_elems<T>() + 32; }

struct Scratch {
  int hist[256];
  int count;    // entries in the buffer
  int picked;   // entries of the selection below
  int digit, need;
  float warp_m[kThreads / 32], warp_s[kThreads / 32];
  float m, s;   // this CTA's log-sum-exp parts
  int out_count;
  u64 sel[kMaxK];
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Cut buf[0, n) to its `want` largest keys (all of them when n <= want): they end in
// sc.sel, in no order; returns how many.  Radix selection from the top digit, left as
// soon as the digit's entries are exactly those still wanted.  All threads call it.
__device__ __forceinline__ int select(const u64* buf, int n, int want, Scratch& sc) {
  const int tid = threadIdx.x;
  if (tid == 0) sc.picked = 0;
  u64 prefix = 0, mask = 0;
  if (n > want) {
    int need = want;
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) sc.hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const u64 k = buf[i];
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
          int j = 0;
          while (before + own[j] < need) before += own[j++];
          sc.digit = 255 - 8 * tid - j;
          sc.need = need - before;
          sc.count = own[j];  // scratch use; the caller sets it again
        }
      }
      __syncthreads();
      prefix |= static_cast<u64>(sc.digit) << shift;
      mask |= 255ull << shift;
      need = sc.need;
      const bool done = sc.count == need;
      __syncthreads();
      if (done) break;
    }
  } else {
    __syncthreads();
  }
  for (int i = tid; i < n; i += kThreads) {
    const u64 k = buf[i];
    if (n <= want || (k & mask) >= prefix) sc.sel[atomicAdd(&sc.picked, 1)] = k;
  }
  __syncthreads();
  return n < want ? n : want;
}

// The smallest key in sc.sel[0, n): what a later element has to pass.
__device__ __forceinline__ u64 lowest(const Scratch& sc, int n) {
  u64 low = ~0ull;
  for (int i = threadIdx.x & 31; i < n; i += 32) low = sc.sel[i] < low ? sc.sel[i] : low;
  for (int o = 16; o; o >>= 1) {
    const u64 other = __shfl_xor_sync(0xffffffffu, low, o);
    low = other < low ? other : low;
  }
  return low;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) top_kernel(const T* __restrict__ logits, int64_t v, int64_t pitch, int k,
                                                       float scale, float inv_tau, void* __restrict__ values,
                                                       int64_t* __restrict__ indices, float* __restrict__ lse) {
  using K = Kind<T>;
  extern __shared__ __align__(16) uint8_t smem[];
  Scratch& sc = *reinterpret_cast<Scratch*>(smem);
  u64* buf = reinterpret_cast<u64*>(smem + ((sizeof(Scratch) + 15) & ~size_t(15)));
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks());
  const int part = static_cast<int>(cluster.block_rank());
  const int64_t row = blockIdx.x / parts;
  const T* x = logits + row * pitch;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // [0, head) and [tail, v) are read one element at a time, the vectors between
  // them are shared among the parts in runs of whole vectors.
  int64_t head = static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T);
  if (head > v) head = v;
  const int64_t vecs = (v - head) / K::kPer;
  const int64_t tail = head + vecs * K::kPer;
  const int64_t w0 = vecs * part / parts, w1 = vecs * (part + 1) / parts;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);

  if (tid == 0) sc.count = 0;
  __syncthreads();
  // scale = log2(e) / tau.  The reference m2 is the rounded product the exponents
  // use, so that log2(sum) + m2 carries no error from rounding it.
  float m = -1e30f, m2 = fmaxf(-1e30f * scale, -3e38f), s = 0.0f;
  auto raise = [&](float to) {
    const float n2 = to * scale;
    s *= exp2_fast(m2 - n2);
    m = to;
    m2 = n2;
  };
  uint32_t limit_key = 0;  // elements with a key above it (strictly) are candidates
  typename K::Limit limit = K::limit(__int_as_float(0x7fffffff));
  auto offer = [&](uint32_t key, int64_t index) {
    if (key > limit_key) {
      const int at = atomicAdd(&sc.count, 1);
      buf[at] = full_key(key, index);
    }
  };
  auto set_limit = [&](uint32_t key) {
    // The value just below `key + 1`; a key between -0 and +0 does not exist.
    limit_key = key;
    uint32_t as = key;
    if constexpr (sizeof(T) == 2) as = key & 0xffff0000u;
    if (as == 0x7fffffffu || as == 0x7fff0000u) as -= sizeof(T) == 2 ? 0x10000u : 1u;
    limit = K::limit(key == 0 ? __int_as_float(0x7fffffff) : value_of_key<T>(as));
  };
  auto add_vec = [&](const uint4& q) {
    const float t = K::top(q);
    if (t > m) raise(t);
#pragma unroll
    for (int i = 0; i < K::kPer; ++i) s += exp2_fast(fmaf(K::value(q, i), scale, -m2));
  };
  auto offer_vec = [&](const uint4& q, int64_t vec) {
    if (K::above(q, limit)) {
      const int64_t base = head + vec * K::kPer;
#pragma unroll
      for (int i = 0; i < K::kPer; ++i) offer(K::key(q, i), base + i);
    }
  };

  // First vectors: the threads' maxima give the first threshold.
  uint4 cur[kVecs], nxt[kVecs];
  auto load = [&](uint4 (&q)[kVecs], int64_t chunk) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int64_t w = w0 + (chunk * kVecs + j) * kThreads + tid;
      if (w < w1) q[j] = __ldg(xv + w);
    }
  };
  const int64_t chunks = (w1 - w0 + kThreads * kVecs - 1) / (kThreads * kVecs);
  load(cur, 0);
  {
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (w0 + j * kThreads + tid < w1) {
#pragma unroll
        for (int i = 0; i < K::kPer; ++i) best = max(best, K::key(cur[j], i));
      }
    }
    // Largest t, in steps of 2^16, that k threads' maxima reach: bit by bit.
    uint32_t t = 0;
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t with = t | (1u << bit);
      if (__syncthreads_count(best >= with) >= k) t = with;
    }
    if (t) set_limit(t - 1);
  }
  // The row's unaligned ends belong to the first part: the head before the vectors
  // and the tail behind them, in index order, as the strict threshold asks.
  auto one = [&](int64_t i) {
    const uint32_t key = K::scalar_key(x + i);
    const float f = value_of_key<T>(key);
    if (f > m) raise(f);
    s += exp2_fast(fmaf(f, scale, -m2));
    offer(key, i);
  };
  if (part == 0 && tid < head) one(tid);
  for (int64_t c = 0; c < chunks; ++c) {
    if (c + 1 < chunks) load(nxt, c + 1);
    bool many = false;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int64_t w = (c * kVecs + j) * kThreads + tid;
      if (w0 + w < w1) {
        add_vec(cur[j]);
        offer_vec(cur[j], w0 + w);
      }
    }
    // A thread that finds the count above kKeep after its own entries: the last to
    // add one does, so the vote is the same as reading the final count.
    many = *reinterpret_cast<volatile int*>(&sc.count) > kKeep;
    if (__syncthreads_or(many)) {
      const int n = sc.count;
      __syncthreads();
      const int kept = select(buf, n, k, sc);
      for (int i = tid; i < kept; i += kThreads) buf[i] = sc.sel[i];
      if (kept == k) {
        const u64 low = lowest(sc, kept);
        set_limit(static_cast<uint32_t>(low >> 32));
      }
      __syncthreads();
      if (tid == 0) sc.count = kept;
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kVecs; ++j) cur[j] = nxt[j];
  }

  if (part == 0 && tid < v - tail) one(tail + tid);

  // Log-sum-exp of this CTA.
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
  const int n = sc.count;
  __syncthreads();
  int kept = select(buf, n, k, sc);
  if (tid == 0) {
    float big = sc.warp_m[0];
    for (int w = 1; w < kThreads / 32; ++w) big = fmaxf(big, sc.warp_m[w]);
    float sum = 0.0f;
    for (int w = 0; w < kThreads / 32; ++w) sum += sc.warp_s[w] * exp2_fast(sc.warp_m[w] - big);
    sc.m = big;
    sc.s = sum;
    sc.out_count = kept;
  }
  if (parts > 1) {
    cluster.sync();
    if (part == 0) {
      // Gather the other parts' selections behind this one's.
      for (int i = tid; i < kept; i += kThreads) buf[i] = sc.sel[i];
      int at = kept;
      for (int c = 1; c < parts; ++c) {
        const Scratch* other = cluster.map_shared_rank(&sc, c);
        const int theirs = other->out_count;
        for (int i = tid; i < theirs; i += kThreads) buf[at + i] = other->sel[i];
        at += theirs;
      }
      if (tid == 0) {
        float big = sc.m;
        for (int c = 1; c < parts; ++c) big = fmaxf(big, cluster.map_shared_rank(&sc, c)->m);
        float sum = 0.0f;
        for (int c = 0; c < parts; ++c) {
          const Scratch* other = cluster.map_shared_rank(&sc, c);
          sum += other->s * exp2_fast(other->m - big);
        }
        sc.m = big;
        sc.s = sum;
      }
      __syncthreads();
      kept = select(buf, at, k, sc);
    }
    cluster.sync();
    if (part != 0) return;
  } else {
    __syncthreads();
  }
  // Rank of each selected key among them: its place in the output.
  for (int i = tid; i < kept; i += kThreads) {
    const u64 key = sc.sel[i];
    int rank = 0;
    for (int j = 0; j < kept; ++j) rank += sc.sel[j] > key ? 1 : 0;
    const uint32_t high = static_cast<uint32_t>(key >> 32);
    K::store(values, row * k + rank, high);
    indices[row * k + rank] = static_cast<int64_t>(0xffffffffull - (key & 0xffffffffull));
    if (rank == 0) {
      // The largest logit decides the cases that the sum cannot: NaN and infinities
      // as they are, and logits beyond 1e30 (a row of the type's lowest value), where
      // the logarithm of the count is below the logit's rounding.
      const float topv = value_of_key<T>(high);
      const float sum = sc.s;
      lse[row] = (isnan(topv) || isinf(topv)) ? topv
                 : sum > 0.0f && !isinf(sc.m)     ? (sc.m + log2f(sum)) * 0.6931471805599453f
                                                   : topv * inv_tau;
    }
  }
}

template <typename T>
int launch(const void* logits, int64_t rows, int64_t v, int64_t pitch, int k, float temperature, void* values,
           int64_t* indices, float* lse, cudaStream_t st) {
  auto kern = top_kernel<T>;
  const int smem = static_cast<int>(((sizeof(Scratch) + 15) & ~size_t(15)) + capacity<T>() * sizeof(u64));
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return fail(SB_ECUDA, std::string("top_kernel attributes: ") + cudaGetErrorString(e));
  // Few rows are split over a cluster while the parts keep a chunk of work each.
  int parts = 1;
  const int sms = device_sm_count();
  while (parts < 8 && rows * parts * 2 <= 2 * sms && v / (parts * 2) >= chunk_elems<T>() / 2) parts *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, static_cast<const T*>(logits), v, pitch, k, 1.4426950408889634f / temperature,
                         1.0f / temperature, values, indices, lse);
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
