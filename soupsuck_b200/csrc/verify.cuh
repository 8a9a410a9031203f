// Verification of drafted tokens against the target model's probabilities.
//
// Per sequence, with target rows p_0..p_S, draft rows q_0..q_{S-1}, drafted tokens
// x_s, uniforms u_s in [0, 1) and exponential noise e_v > 0:
//
//   a      = number of leading s < len with  u_s q_s(x_s) < p_s(x_s)
//   r      = max(p_a - q_a, 0)  if a < len,  p_a otherwise  (p_a too where r is all zero)
//   token  = argmax_v r_v / e_v        (lowest v among equals; -1 where no score is above zero)
//
// which is a draw from r / sum(r) (an exponential race), so the emitted tokens
// follow p whatever q is.  Without a draft distribution q_s is the one-hot of x_s.
// The race needs no sum over the vocabulary: every score is one subtraction and one
// correctly rounded division in fp32, and a maximum does not depend on its order,
// so the result is the same for every split of the row.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"

namespace sb {
namespace verify {

namespace cg = cooperative_groups;

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

struct Args {
  const void* target;
  const void* draft;
  const int64_t* tokens;
  const float* uniforms;
  const float* noise;
  const int64_t* lens;
  int64_t* accepted;
  int64_t* out;
  int64_t v, t_b, t_s, d_b, d_s, n_b;
  int drafts;
};

// Best (score, lowest index) as one ordered key: the bits of a positive float rise
// with its value, and a larger complement means a smaller index.  0: no candidate.
__device__ __forceinline__ unsigned long long pack(float score, int64_t v) {
  return (static_cast<unsigned long long>(__float_as_uint(score)) << 32) |
         (0xffffffffull - static_cast<unsigned long long>(v));
}

// A thread's best so far.  `bar` is a little below it: r / e can only beat the best where
// r > bar e, so the division is left to the few elements that pass (in fp32 rounding;
// bests below 1e-30 keep no bar).
struct Best {
  float score = 0.0f, bar = 0.0f;
  int at = 0;
  __device__ __forceinline__ void race(float p, float q, float e, int v) {
    const float r = __fsub_rn(p, q);
    // (-1e-44: a product among the denormals may be rounded up by a whole one.)
    if (r > fmaf(bar, e, -1e-44f) && r > 0.0f) {
      const float s = __fdiv_rn(r, e);
      if (s > score) {
        score = s;
        bar = s < 1e-30f ? 0.0f : s * 0.999999f;
        at = v;
      }
    }
  }
};

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kPer = 4;
  static __device__ __forceinline__ float get(const uint4& q, int i) {
    return __uint_as_float(i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w);
  }
};
template <typename T> struct Vec16 {
  static constexpr int kPer = 8;
  static __device__ __forceinline__ float get(const uint4& q, int i) {
    const uint32_t w = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    const unsigned short b = static_cast<unsigned short>((i & 1) ? w >> 16 : w & 0xffffu);
    return to_f32<T>(*reinterpret_cast<const T*>(&b));
  }
};
template <> struct Vec<__half> : Vec16<__half> {};
template <> struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16> {};

// One CTA's share [v0, v1) of the row.  16-byte loads where the three rows reach a
// 16-byte boundary at the same element, single elements elsewhere (rows of an odd
// vocabulary differ).  256 sequences x 5 drafts of 151936 fp32, 71 us at the copy rate:
// 72 us in vectors, two in flight per row and thread so that four CTAs fit an SM (four
// in flight, two CTAs: 114); of 151935 in single elements 84; with a division for every
// element 155.  One sequence takes 8 us, most of it the dependent loads of the acceptance
// test and the exchange.
template <typename T, bool DRAFT, int THREADS>
__device__ __forceinline__ void scan(const T* p, const T* q, int hot, const float* e, int v0, int v1, Best& best) {
  using V = Vec<T>;
  constexpr int kPer = V::kPer;
  auto single = [&](int v) { best.race(v == hot ? 0.0f : to_f32<T>(p[v]), DRAFT ? to_f32<T>(q[v]) : 0.0f, e[v], v); };
  auto off = [](const void* x, int size, int mod) { return static_cast<int>(reinterpret_cast<uintptr_t>(x) / size % mod); };
  const int at_p = off(p + v0, sizeof(T), kPer);
  int tid = threadIdx.x;
  if ((!DRAFT || off(q + v0, sizeof(T), kPer) == at_p) && off(e + v0, 4, 4) == at_p % 4) {
    const int head = min((kPer - at_p) % kPer, v1 - v0);
    const int vecs = (v1 - v0 - head) / kPer;
    const int base = v0 + head;
    if (tid < head) single(v0 + tid);
    constexpr int kUnroll = 2;
    constexpr int kE = kPer / 4;
    const uint4* pv = reinterpret_cast<const uint4*>(p + base);
    const uint4* qv = reinterpret_cast<const uint4*>(q + base);
    const uint4* ev = reinterpret_cast<const uint4*>(e + base);
    auto eat = [&](const uint4& a, const uint4& b, const uint4 (&c)[kE], int w) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int v = base + w * kPer + i;
        best.race(!DRAFT && v == hot ? 0.0f : V::get(a, i), DRAFT ? V::get(b, i) : 0.0f, Vec<float>::get(c[i / 4], i % 4), v);
      }
    };
    int w = tid;
    for (; w + (kUnroll - 1) * THREADS < vecs; w += kUnroll * THREADS) {
      uint4 a[kUnroll], b[kUnroll], c[kUnroll][kE];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        a[u] = __ldcs(pv + w + u * THREADS);
        if (DRAFT) b[u] = __ldcs(qv + w + u * THREADS);
#pragma unroll
        for (int i = 0; i < kE; ++i) c[u][i] = __ldcs(ev + (w + u * THREADS) * kE + i);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) eat(a[u], b[u], c[u], w + u * THREADS);
    }
    for (; w < vecs; w += THREADS) {
      uint4 b = make_uint4(0, 0, 0, 0), c[kE];
      const uint4 a = __ldcs(pv + w);
      if (DRAFT) b = __ldcs(qv + w);
#pragma unroll
      for (int i = 0; i < kE; ++i) c[i] = __ldcs(ev + w * kE + i);
      eat(a, b, c, w);
    }
    const int v = base + vecs * kPer + tid;
    if (v < v1) single(v);
    return;
  }
  constexpr int kUnroll = 8;
  int v = v0 + tid;
  for (; v + (kUnroll - 1) * THREADS < v1; v += kUnroll * THREADS) {
    float pv[kUnroll], qv[kUnroll], ev[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int x = v + i * THREADS;
      pv[i] = to_f32<T>(p[x]);
      qv[i] = DRAFT ? to_f32<T>(q[x]) : 0.0f;
      ev[i] = e[x];
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int x = v + i * THREADS;
      best.race(!DRAFT && x == hot ? 0.0f : pv[i], qv[i], ev[i], x);
    }
  }
  for (; v < v1; v += THREADS) single(v);
}

// A cluster of CTAs per sequence: each repeats the short acceptance test, scans its
// share of the vocabulary, and the best keys meet in distributed shared memory.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) verify_kernel(const Args a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks());
  const int part = static_cast<int>(cluster.block_rank());
  const int64_t b = blockIdx.x / parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ int s_accepted, s_len;
  __shared__ unsigned long long s_warp[THREADS / 32];
  __shared__ unsigned long long s_best;
  const T* target = static_cast<const T*>(a.target) + b * a.t_b;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + b * a.d_b : nullptr;
  const int64_t* tokens = a.tokens + b * a.drafts;
  if (warp == 0) {
    int64_t len = a.drafts;
    if (a.lens) {
      len = a.lens[b];
      len = len < 0 ? 0 : (len > a.drafts ? a.drafts : len);
    }
    int accepted = static_cast<int>(len);
    for (int s0 = 0; s0 < len; s0 += 32) {
      const int s = s0 + lane;
      bool ok = true;
      if (s < len) {
        const int64_t x = tokens[s];
        ok = x >= 0 && x < a.v;
        if (ok) {
          const float p = to_f32<T>(target[s * a.t_s + x]);
          const float q = draft ? to_f32<T>(draft[s * a.d_s + x]) : 1.0f;
          ok = __fmul_rn(a.uniforms[b * a.drafts + s], q) < p;
        }
      }
      const unsigned no = __ballot_sync(0xffffffffu, !ok);
      if (no) {
        accepted = s0 + __ffs(no) - 1;
        break;
      }
    }
    if (lane == 0) {
      s_accepted = accepted;
      s_len = static_cast<int>(len);
    }
  }
  __syncthreads();
  const int n = s_accepted;
  const bool rejected = n < s_len;
  const T* p = target + n * a.t_s;
  const T* q = rejected && draft ? draft + n * a.d_s : nullptr;
  int hot = -1;
  if (rejected && !draft && tokens[n] >= 0 && tokens[n] < a.v) hot = static_cast<int>(tokens[n]);
  const float* e = a.noise + b * a.n_b;
  // Shares of whole vectors of every type, in order.
  const int64_t share = ((a.v + parts - 1) / parts + 7) / 8 * 8;
  const int v0 = static_cast<int>(part * share < a.v ? part * share : a.v);
  const int v1 = static_cast<int>(v0 + share < a.v ? v0 + share : a.v);
  unsigned long long key = 0;
  // The second round only where the residual is zero everywhere: p itself then.
  for (int round = 0; round < 2; ++round) {
    Best best;
    if (q) {
      scan<T, true, THREADS>(p, q, -1, e, v0, v1, best);
    } else {
      scan<T, false, THREADS>(p, p, hot, e, v0, v1, best);
    }
    key = best.score > 0.0f ? pack(best.score, best.at) : 0;
    for (int o = 16; o; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      key = other > key ? other : key;
    }
    if (lane == 0) s_warp[warp] = key;
    __syncthreads();
    if (warp == 0) {
      key = lane < THREADS / 32 ? s_warp[lane] : 0;
      for (int o = 16; o; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
        key = other > key ? other : key;
      }
      if (lane == 0) s_best = key;
    }
    cluster.sync();
    // Lane c takes part c's best (remote loads: all at once).
    key = lane < parts ? *cluster.map_shared_rank(&s_best, lane) : 0;
    for (int o = 4; o; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      key = other > key ? other : key;
    }
    key = __shfl_sync(0xffffffffu, key, 0);
    cluster.sync();
    if (key || !rejected) break;
    q = nullptr;
    hot = -1;
  }
  if (part == 0) {
    int64_t* out = a.out + b * (a.drafts + 1);
    for (int s = threadIdx.x; s <= a.drafts; s += THREADS) {
      out[s] = s < n ? tokens[s] : (s == n && key ? static_cast<int64_t>(0xffffffffull - (key & 0xffffffffull)) : -1);
    }
    if (threadIdx.x == 0) a.accepted[b] = n;
  }
}

template <typename T, int THREADS>
int launch(const Args& a, int64_t batch, int parts, cudaStream_t st) {
  auto kern = verify_kernel<T, THREADS>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return fail(SB_ECUDA, std::string("verify_kernel: ") + cudaGetErrorString(e));
  count_launch();
  return check_launch("verify_kernel");
}

}  // namespace verify
}  // namespace sb

extern "C" {

int sb_verify_drafts(const void* target, int64_t target_batch, int64_t target_row, const void* draft,
                     int64_t draft_batch, int64_t draft_row, int dtype, int64_t batch, int64_t drafts, int64_t v,
                     const int64_t* tokens, const float* uniforms, const float* noise, int64_t noise_batch,
                     const int64_t* lens, int64_t* accepted, int64_t* out_tokens, void* stream) {
  SB_REQUIRE(dtype == SB_F16 || dtype == SB_F32 || dtype == SB_BF16, "probabilities must be fp16, bf16 or fp32");
  SB_REQUIRE(batch >= 0 && drafts >= 0 && v > 0, "expected batch >= 0, drafts >= 0, v > 0");
  if (batch == 0) return SB_OK;
  SB_REQUIRE(target && noise && accepted && out_tokens, "NULL pointer argument");
  SB_REQUIRE(drafts == 0 || (tokens && uniforms), "NULL pointer argument");
  SB_REQUIRE(batch <= (int64_t(1) << 27) && drafts <= 0x7ffffffe && v <= 0x7fffffff, "size out of range");
  sb::verify::Args a{};
  a.target = target;
  a.draft = draft;
  a.tokens = tokens;
  a.uniforms = uniforms;
  a.noise = noise;
  a.lens = lens;
  a.accepted = accepted;
  a.out = out_tokens;
  a.v = v;
  a.t_b = target_batch;
  a.t_s = target_row;
  a.d_b = draft_batch;
  a.d_s = draft_row;
  a.n_b = noise_batch;
  a.drafts = static_cast<int>(drafts);
  // Eight CTAs (the portable cluster limit) while that is at most eight per SM (each
  // starts with the dependent loads of the acceptance test: 256 sequences of 151936
  // fp32 take 82 us with eight parts, 73.5 with four) and each keeps some rounds of loads.
  int parts = 8;
  while (parts > 1 && batch * parts > 8 * sb::device_sm_count()) parts /= 2;
  while (parts > 1 && v / parts < 2048) parts /= 2;
  cudaStream_t st = sb::as_stream(stream);
  // Few sequences: a CTA has an SM to itself, and fewer rounds of loads end sooner.
  const bool few = batch * parts <= sb::device_sm_count();
  auto run = [&](auto type) {
    using T = decltype(type);
    return few ? sb::verify::launch<T, 1024>(a, batch, parts, st) : sb::verify::launch<T, 256>(a, batch, parts, st);
  };
  if (dtype == SB_F32) return run(float{});
  if (dtype == SB_F16) return run(__half{});
  return run(__nv_bfloat16{});
}

}  // extern "C"
