// wp_logprobs.cu -- log probability, rank and entropy of given tokens and the
// top alternatives of each row of logits, in one launch.
//
//   M = max x, l = sum e^(x - M)
//   log p(token) = (x_token - M) - log l
//   entropy      = log l - sum e^(x - M) (x - M) / l
//   rank         = 1 + #(x > x_token)
//   alternatives: the `top` largest logits, equal ones by ascending index
//
// x - M comes first and is exact for the values that matter, so neither a
// large common offset nor rows of the type's lowest value lose anything. A
// logit of minus infinity has probability 0; a row of nothing else is empty:
// log probabilities -inf, entropy 0. NaN and plus infinity make a row NaN.
//
// What bounds it: T * V logits from HBM once; in 16 bits the instructions per
// logit (7-8 of the 11 that fit in its time at the memory rate) come close
// behind. The row is read a second time, from L2, for the alternatives only:
// every thread's own maximum is known after the first pass, so the top-th
// largest of those is a lower bound that at least `top` logits reach and few
// others do.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stddef.h>
#include <stdint.h>

#include "wp_device.cuh"
#include "wp_internal.h"

namespace wp {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpCands = 1024;  // candidates for the alternatives in one CTA

// 16 bytes of logits as fp32.
template <typename T>
struct Vec {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);  // NaN if either is
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T>::unpack2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float largest(const uint4& v) {
    const float2 f = Elem<T>::unpack2(max2(max2(v.x, v.y), max2(v.z, v.w)));
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(f.x), "f"(f.y));
    return m;
  }
};
template <>
__device__ __forceinline__ uint32_t Vec<__nv_bfloat16>::max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t Vec<__half>::max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float largest(const uint4& v) {
    float a, b;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(__uint_as_float(v.x)), "f"(__uint_as_float(v.y)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(b));
    return a;
  }
};

template <typename T>
__device__ __forceinline__ float load1(const T* p) {
  if constexpr (sizeof(T) == 4)
    return __ldg(reinterpret_cast<const float*>(p));
  else
    return Elem<T>::to_f(*p);
}

// Floats as integers in the same order, NaN above all, both zeros equal.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return k == 0xffffffffu ? NAN : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Larger logits first, of equal ones the lower index: unique, and never 0.
__device__ __forceinline__ unsigned long long key_of(float x, int index) {
  return (static_cast<unsigned long long>(ordered(x)) << 32) | static_cast<uint32_t>(0x7fffffff - index);
}

struct Stat {
  float m;  // maximum (at least -FLT_MAX: a reference that is always finite)
  float l;  // sum e^(x - m)
  float s;  // sum e^(x - m) (x - m)
  int above;  // logits above the given one
  float raw;  // maximum, -inf while there is none
};

__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  r.raw = fmaxf(a.raw, b.raw);
  r.above = a.above + b.above;
  // a side that is far below contributes 0, not 0 * infinity
  const float da = fmaxf(a.m - r.m, -1e4f), db = fmaxf(b.m - r.m, -1e4f);
  const float fa = ex2(da * kLog2e), fb = ex2(db * kLog2e);
  r.l = fa * a.l + fb * b.l;
  r.s = fa * fmaf(a.l, da, a.s) + fb * fmaf(b.l, db, b.s);
  return r;
}

__device__ __forceinline__ Stat shfl_xor(const Stat& a, int o) {
  Stat r;
  r.m = __shfl_xor_sync(~0u, a.m, o);
  r.l = __shfl_xor_sync(~0u, a.l, o);
  r.s = __shfl_xor_sync(~0u, a.s, o);
  r.above = __shfl_xor_sync(~0u, a.above, o);
  r.raw = __shfl_xor_sync(~0u, a.raw, o);
  return r;
}

// What one CTA of a row's cluster hands to the first one.
struct alignas(16) Share {
  Stat stat;
  unsigned long long top[kMaxTop];
};

// Elements of one row that this CTA visits: f(x, index) for the unaligned
// head and tail, g(vector, first index) for the 16-byte vectors between.
template <typename T, typename F, typename G>
__device__ __forceinline__ void for_row(const T* row, int vocab, int rank, int ranks, F&& f, G&& g) {
  constexpr int N = Vec<T>::N;
  const int head = min(static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)), vocab);
  const int nvec = (vocab - head) / N;
  const int tail = head + nvec * N;
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  const int step = ranks * kLpThreads;
  int i = rank * kLpThreads + threadIdx.x;
  // four loads in flight
  for (; i + 3 * step < nvec; i += 4 * step) {
    uint4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __ldg(v + i + j * step);
#pragma unroll
    for (int j = 0; j < 4; ++j) g(x[j], head + (i + j * step) * N);
  }
  for (; i < nvec; i += step) g(__ldg(v + i), head + i * N);
  if (rank == ranks - 1) {
    const int t = threadIdx.x;
    if (t < head) f(load1(row + t), t);
    if (tail + t < vocab) f(load1(row + tail + t), tail + t);
  }
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 2) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int N = Vec<T>::N;
  __shared__ Stat s_stat[kLpWarps];
  __shared__ uint32_t s_max[kLpThreads];  // each thread's maximum
  __shared__ unsigned long long s_cand[kLpCands];
  __shared__ int s_ncand;
  __shared__ uint32_t s_bound;
  __shared__ unsigned long long s_best[kLpWarps];
  __shared__ Share s_share[8];  // on the cluster's first CTA: every CTA's result
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ranks = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  if (ranks > 1) cluster_arrive();  // every CTA runs before the first one's shared memory is written
  const int64_t t = blockIdx.x / ranks;
  const T* row = static_cast<const T*>(a.logits) + t * a.ld;

  const long long token = a.tokens64 ? __ldg(static_cast<const long long*>(a.tokens) + t)
                                     : static_cast<long long>(__ldg(static_cast<const int*>(a.tokens) + t));
  const bool known = token >= 0 && token < a.vocab;
  const float given = known ? load1(row + token) : -INFINITY;

  // ---- pass 1: running maximum, sums, rank
  Stat st{-FLT_MAX, 0.f, 0.f, 0, -INFINITY};
  auto add = [&](float x) {
    // x - m, kept finite where x is far below (minus infinity has e^(x - m)
    // = 0 and adds 0 to both sums); NaN stays NaN
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x - st.m), "f"(-1e38f));
    const float e = ex2(d * kLog2e);
    st.l += e;
    st.s = fmaf(e, d, st.s);
  };
  auto raise = [&](float x) {
    st.raw = fmaxf(st.raw, x);
    const float m = fmaxf(st.m, x), d = fmaxf(st.m - m, -1e4f), f = ex2(d * kLog2e);
    st.s = f * fmaf(st.l, d, st.s);
    st.l *= f;
    st.m = m;
  };
  for_row(
      row, a.vocab, rank, ranks,
      [&](float x, int) {
        if (x > st.raw) raise(x);
        add(x);
        st.above += x > given;
      },
      [&](const uint4& v, int) {
        float x[N];
        Vec<T>::unpack(v, x);
        const float top = Vec<T>::largest(v);
        if (top > st.raw) raise(top);
        if (top > given) {
#pragma unroll
          for (int i = 0; i < N; ++i) st.above += x[i] > given;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) add(x[i]);
      });
  s_max[tid] = st.raw == -INFINITY ? 0u : ordered(st.raw);
#pragma unroll
  for (int o = 16; o; o >>= 1) st = merge(st, shfl_xor(st, o));
  if (lane == 0) s_stat[warp] = st;
  if (tid == 0) s_ncand = 0;
  __syncthreads();
  if (warp == 0) {
    Stat w = lane < kLpWarps ? s_stat[lane] : Stat{-FLT_MAX, 0.f, 0.f, 0, -INFINITY};
#pragma unroll
    for (int o = kLpWarps / 2; o; o >>= 1) w = merge(w, shfl_xor(w, o));
    if (lane == 0) s_stat[0] = w;
  } else if (warp == 1 && a.top > 0) {
    // top-th largest of the threads' maxima (0: fewer than that have one)
    uint32_t k[kLpThreads / 32];
#pragma unroll
    for (int i = 0; i < kLpThreads / 32; ++i) k[i] = s_max[i * 32 + lane];
    uint32_t best = 0;
    for (int n = 0; n < a.top; ++n) {
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < kLpThreads / 32; ++i) mine = max(mine, k[i]);
      best = __reduce_max_sync(~0u, mine);
      const int owner = __ffs(__ballot_sync(~0u, mine == best)) - 1;
      if (lane == owner) {
        bool gone = false;
#pragma unroll
        for (int i = 0; i < kLpThreads / 32; ++i)
          if (!gone && k[i] == best) {
            k[i] = 0;
            gone = true;
          }
      }
    }
    if (lane == 0) s_bound = best;
  }
  __syncthreads();

  // ---- pass 2: the largest `top` of this CTA's part of the row
  unsigned long long mine = 0;  // thread i < top: the i-th largest key
  if (a.top > 0) {
    const float bound = s_bound == 0 ? -INFINITY : unordered(s_bound);
    auto keep = [&](float x, int i) {
      if (!(x < bound)) {
        const int at = atomicAdd(&s_ncand, 1);
        if (at < kLpCands) s_cand[at] = key_of(x, i);
      }
    };
    for_row(row, a.vocab, rank, ranks, keep, [&](const uint4& v, int i0) {
      if (!(Vec<T>::largest(v) < bound)) {
        float x[N];
        Vec<T>::unpack(v, x);
#pragma unroll
        for (int i = 0; i < N; ++i) keep(x[i], i0 + i);
      }
    });
    __syncthreads();
    const int n = s_ncand;
    if (n <= kLpCands) {
      // a candidate's place is the number of larger keys
      __shared__ unsigned long long s_top[kMaxTop];
      if (tid < kMaxTop) s_top[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kLpThreads) {
        const unsigned long long k = s_cand[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += s_cand[j] > k;
        if (place < a.top) s_top[place] = k;
      }
      __syncthreads();
      if (tid < a.top) mine = s_top[tid];
    } else {
      // long runs of equal logits: one pass over the row for each place
      unsigned long long last = ~0ull;
      for (int p = 0; p < a.top; ++p) {
        unsigned long long b = 0;
        auto look = [&](float x, int i) {
          const unsigned long long k = key_of(x, i);
          if (k < last && k > b) b = k;
        };
        for_row(row, a.vocab, rank, ranks, look, [&](const uint4& v, int i0) {
          float x[N];
          Vec<T>::unpack(v, x);
#pragma unroll
          for (int i = 0; i < N; ++i) look(x[i], i0 + i);
        });
#pragma unroll
        for (int o = 16; o; o >>= 1) b = max(b, __shfl_xor_sync(~0u, b, o));
        if (lane == 0) s_best[warp] = b;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kLpWarps; ++i) b = max(b, s_best[i]);
        __syncthreads();
        last = b;
        if (tid == p) mine = b;
      }
    }
  }

  // ---- the cluster's first CTA gathers
  if (ranks > 1) {
    cluster_wait();
    const uint32_t dst = mapa(smem_u32(&s_share[rank]), 0);
    if (tid == 0) {
      const Stat w = s_stat[0];
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(w.m), "f"(w.l), "f"(w.s),
                   "f"(__int_as_float(w.above))
                   : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 16), "f"(w.raw) : "memory");
    }
    if (tid < a.top)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(
                       dst + static_cast<uint32_t>(offsetof(Share, top)) + 8u * tid),
                   "l"(mine)
                   : "memory");
    cluster_sync_hw();
    if (rank != 0) return;
  }
  Stat r = ranks > 1 ? s_share[0].stat : s_stat[0];
  for (int i = 1; i < ranks; ++i) r = merge(r, s_share[i].stat);
  const bool empty = r.raw == -INFINITY && r.l == 0.f;
  const float log_l = logf(r.l);
  auto log_prob = [&](float x) { return x == -INFINITY && r.l == r.l ? -INFINITY : (x - r.m) - log_l; };
  if (tid == 0) {
    a.logprob[t] = log_prob(given);
    if (a.entropy) a.entropy[t] = empty ? 0.f : log_l - r.s / r.l;
    if (a.rank) a.rank[t] = r.above + 1;
  }
  auto put = [&](int place, unsigned long long k) {
    a.top_ids[t * a.top + place] = k == 0 ? -1 : 0x7fffffff - static_cast<int>(k & 0xffffffffu);
    a.top_logprobs[t * a.top + place] = k == 0 ? -INFINITY : log_prob(unordered(static_cast<uint32_t>(k >> 32)));
  };
  if (ranks == 1) {
    if (tid < a.top) put(tid, mine);
  } else {
    for (int i = tid; i < ranks * a.top; i += kLpThreads) {
      const unsigned long long k = s_share[i / a.top].top[i % a.top];
      int place = 0;
      for (int j = 0; j < ranks; ++j)
        for (int p = 0; p < a.top; ++p) {
          const unsigned long long o = s_share[j].top[p];
          place += o > k || (o == k && j * a.top + p < i);  // ties only between places that are empty (0)
        }
      if (place < a.top) put(place, k);
    }
  }
}

template <typename T>
cudaError_t launch(const LogprobArgs& a, int num_sms, cudaStream_t stream) {
  // CTAs per row: enough to fill the GPU with few rows, while a CTA still has
  // a vector for each of its threads
  int ranks = 1;
  while (ranks < 8 && static_cast<int64_t>(a.rows) * ranks < 4 * num_sms &&
         static_cast<int64_t>(a.vocab) >= static_cast<int64_t>(2 * ranks) * kLpThreads * Vec<T>::N)
    ranks *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows * ranks);
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a);
}

}  // namespace

cudaError_t launch_token_logprobs(int dtype, const LogprobArgs& a, int num_sms, cudaStream_t stream) {
  if (dtype == 2) return launch<float>(a, num_sms, stream);
  return dtype == 1 ? launch<__nv_bfloat16>(a, num_sms, stream) : launch<__half>(a, num_sms, stream);
}

}  // namespace wp
