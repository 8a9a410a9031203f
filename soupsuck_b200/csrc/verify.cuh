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

constexpr int kThreads = 512;

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

template <typename T>
__device__ __forceinline__ void race(float p, float q, float e, int64_t v, float& best, int64_t& at) {
  const float r = __fsub_rn(p, q);
  if (r > 0.0f) {
    const float s = __fdiv_rn(r, e);
    if (s > best) {
      best = s;
      at = v;
    }
  }
}

// One CTA's share [v0, v1) of the row: elements v0 + tid, v0 + tid + kThreads, ...
template <typename T>
__device__ void scan(const T* p, const T* q, int64_t hot, const float* e, int64_t v0, int64_t v1, float& best,
                     int64_t& at) {
  constexpr int kUnroll = 8;
  int64_t v = v0 + threadIdx.x;
  for (; v + (kUnroll - 1) * kThreads < v1; v += kUnroll * kThreads) {
    float pv[kUnroll], qv[kUnroll], ev[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int64_t x = v + i * kThreads;
      pv[i] = to_f32<T>(p[x]);
      qv[i] = q ? to_f32<T>(q[x]) : 0.0f;
      ev[i] = e[x];
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int64_t x = v + i * kThreads;
      race<T>(x == hot ? 0.0f : pv[i], qv[i], ev[i], x, best, at);
    }
  }
  for (; v < v1; v += kThreads) race<T>(v == hot ? 0.0f : to_f32<T>(p[v]), q ? to_f32<T>(q[v]) : 0.0f, e[v], v, best, at);
}

// A cluster of CTAs per sequence: each repeats the short acceptance test, scans its
// share of the vocabulary, and the best keys meet in distributed shared memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const Args a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks());
  const int part = static_cast<int>(cluster.block_rank());
  const int64_t b = blockIdx.x / parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ int s_accepted, s_len;
  __shared__ unsigned long long s_warp[kThreads / 32];
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
  int64_t hot = rejected && !draft ? tokens[n] : -1;
  const float* e = a.noise + b * a.n_b;
  const int64_t share = (a.v + parts - 1) / parts;
  const int64_t v0 = part * share, v1 = v0 + share < a.v ? v0 + share : a.v;
  unsigned long long key = 0;
  // The second round only where the residual is zero everywhere: p itself then.
  for (int round = 0; round < 2; ++round) {
    float best = 0.0f;
    int64_t at = 0;
    scan<T>(p, q, hot, e, v0, v1, best, at);
    key = best > 0.0f ? pack(best, at) : 0;
    for (int o = 16; o; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      key = other > key ? other : key;
    }
    if (lane == 0) s_warp[warp] = key;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kThreads / 32; ++w) key = s_warp[w] > key ? s_warp[w] : key;
      s_best = key;
    }
    cluster.sync();
    key = 0;
    for (int c = 0; c < parts; ++c) {
      const unsigned long long other = *cluster.map_shared_rank(&s_best, c);
      key = other > key ? other : key;
    }
    cluster.sync();
    if (key || !rejected) break;
    q = nullptr;
    hot = -1;
  }
  if (part == 0) {
    int64_t* out = a.out + b * (a.drafts + 1);
    for (int s = threadIdx.x; s <= a.drafts; s += kThreads) {
      out[s] = s < n ? tokens[s] : (s == n && key ? static_cast<int64_t>(0xffffffffull - (key & 0xffffffffull)) : -1);
    }
    if (threadIdx.x == 0) a.accepted[b] = n;
  }
}

template <typename T>
int launch(const Args& a, int64_t batch, int parts, cudaStream_t st) {
  auto kern = verify_kernel<T>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * parts));
  cfg.blockDim = dim3(kThreads);
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
  // Eight CTAs (the portable cluster limit) while each keeps some rounds of loads.
  int parts = 8;
  while (parts > 1 && v / parts < 2 * sb::verify::kThreads) parts /= 2;
  cudaStream_t st = sb::as_stream(stream);
  if (dtype == SB_F32) return sb::verify::launch<float>(a, batch, parts, st);
  if (dtype == SB_F16) return sb::verify::launch<__half>(a, batch, parts, st);
  return sb::verify::launch<__nv_bfloat16>(a, batch, parts, st);
}

}  // extern "C"
