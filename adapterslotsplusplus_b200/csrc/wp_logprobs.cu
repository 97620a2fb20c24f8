// wp_logprobs.cu -- log probability, rank and entropy of given tokens and the
// top alternatives of each row of logits, in one launch.
//
//   M = max x, l = sum e^(x - M)
//   log p(token) = (x_token - M) - log l
//   entropy      = log l - sum e^(x - M) (x - M) / l
//   rank         = 1 + #(x > x_token)
//   alternatives: the `top` largest logits, equal ones by ascending index
//
// A logit of minus infinity has probability 0; a row of nothing else is empty:
// log probabilities -inf, entropy 0. NaN and plus infinity make a row NaN.
//
// What bounds it: T * V logits from HBM once, and close behind it in 16 bits
// the instructions per logit (6.5 of the 11 that fit into its time at the
// memory rate). So the pass works in log2 units, where e^(x - M) is one fused
// multiply-add and one 2^y, with a running reference R = fl(M log2 e): its own
// rounding is the same for every logit of a thread and is taken out of its sums
// again. It is at most 2^-4 because the pass only holds for maxima within
// 2^20 of 0 (a rounding of R beyond 2^31 could exceed the exponents of fp32):
// logits below -2^20, the large negative numbers that stand for masked ones
// among them, count as -2^20, and parts of rows whose maximum is not within
// that range are summed again with x - M exact, M being known then. The row is
// not read a second time for the alternatives: after
// the pass every thread knows its own maximum, the top-th largest of 32 groups'
// maxima is a bound that at least `top` logits reach and few others do, and
// only the threads whose maximum reaches it look at their logits again (a warp
// together for each). 256 x 128000 in bf16 with 20 alternatives: 28 us (floor
// 10), about 8 of them start-up and selection; 2048 x 32003 in fp32 with one:
// 57 us, 72% of the copy rate.

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

constexpr int kLpThreads = 256;
constexpr int kLpPerSm = 4;  // CTAs of one SM (64 registers; 5 and 6 measured the same or slower)
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpAhead = 4;  // vectors that a thread has in flight
constexpr int kLpCands = 1024;  // candidates for the alternatives in one CTA

// 16 bytes of logits as fp32.
template <typename T>
struct Vec {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);  // NaN if either is
  // The lowest logit that the fast pass tells from minus infinity; a part of a
  // row whose maximum is not well above it takes the exact pass.
  static constexpr float kLow = Elem<T>::is_bf16 ? -0x1p20f : -65504.f;
  static constexpr uint32_t kNone = Elem<T>::is_bf16 ? 0xff80ff80u : 0xfc00fc00u;  // minus infinity
  static constexpr uint32_t kLow2 = Elem<T>::is_bf16 ? 0xc980c980u : 0xfbfffbffu;
  // -1 in each half that is above the same half of g
  static __device__ __forceinline__ uint32_t above2(uint32_t v, uint32_t g);
  static __device__ __forceinline__ int above(const uint4& v, uint32_t g2, float) {
    int n = __dp4a(static_cast<int>(above2(v.x, g2)), 0x00010001, 0);
    n = __dp4a(static_cast<int>(above2(v.y, g2)), 0x00010001, n);
    n = __dp4a(static_cast<int>(above2(v.z, g2)), 0x00010001, n);
    return -__dp4a(static_cast<int>(above2(v.w, g2)), 0x00010001, n);
  }
  static __device__ __forceinline__ uint4 raised(const uint4& v) {
    return make_uint4(max2(v.x, kLow2), max2(v.y, kLow2), max2(v.z, kLow2), max2(v.w, kLow2));
  }
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
__device__ __forceinline__ uint32_t Vec<__nv_bfloat16>::above2(uint32_t v, uint32_t g) {
  return __hgt2_mask(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<__nv_bfloat162*>(&g));
}
template <>
__device__ __forceinline__ uint32_t Vec<__half>::above2(uint32_t v, uint32_t g) {
  return __hgt2_mask(*reinterpret_cast<__half2*>(&v), *reinterpret_cast<__half2*>(&g));
}
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr float kLow = -0x1p20f;
  static constexpr uint32_t kNone = 0xff800000u;
  static __device__ __forceinline__ int above(const uint4& v, uint32_t, float g) {
    return (__uint_as_float(v.x) > g) + (__uint_as_float(v.y) > g) + (__uint_as_float(v.z) > g) + (__uint_as_float(v.w) > g);
  }
  static __device__ __forceinline__ float raised1(uint32_t v) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(v)), "f"(kLow));
    return r;
  }
  static __device__ __forceinline__ uint4 raised(const uint4& v) {
    return make_uint4(__float_as_uint(raised1(v.x)), __float_as_uint(raised1(v.y)), __float_as_uint(raised1(v.z)),
                      __float_as_uint(raised1(v.w)));
  }
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

// Maxima up to here take the fast pass (see the top).
constexpr float kHigh = 0x1p20f;

struct Stat {
  float raw;  // maximum, -inf while there is none
  float ref;  // raw, or a finite number above it where raw is too low for the pass
  float l;  // sum 2^y, y = (x - ref) log2 e
  float s;  // sum 2^y y
  int above;  // logits above the given one
};

__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b) {
  Stat r;
  r.raw = fmaxf(a.raw, b.raw);
  r.ref = fmaxf(a.ref, b.ref);
  r.above = a.above + b.above;
  // a side that is far below contributes 0, not 0 * infinity
  const float da = fmaxf((a.ref - r.ref) * kLog2e, -1e4f), db = fmaxf((b.ref - r.ref) * kLog2e, -1e4f);
  const float fa = ex2(da), fb = ex2(db);
  r.l = fa * a.l + fb * b.l;
  r.s = fa * fmaf(a.l, da, a.s) + fb * fmaf(b.l, db, b.s);
  return r;
}

__device__ __forceinline__ Stat shfl_xor(const Stat& a, int o) {
  Stat r;
  r.raw = __shfl_xor_sync(~0u, a.raw, o);
  r.ref = __shfl_xor_sync(~0u, a.ref, o);
  r.l = __shfl_xor_sync(~0u, a.l, o);
  r.s = __shfl_xor_sync(~0u, a.s, o);
  r.above = __shfl_xor_sync(~0u, a.above, o);
  return r;
}

// What one CTA of a row's cluster hands to the first one.
struct alignas(16) Share {
  Stat stat;
  alignas(16) unsigned long long top[kMaxTop];  // descending, 0 past the last
};

// Where the 16-byte vectors of a row start and end.
template <typename T>
struct Row {
  const T* p;
  int vocab, head, nvec, tail;
  __device__ __forceinline__ Row(const T* row, int v) : p(row), vocab(v) {
    head = min(static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)), vocab);
    nvec = (vocab - head) / Vec<T>::N;
    tail = head + nvec * Vec<T>::N;
  }
  __device__ __forceinline__ uint4 vec(int i) const { return __ldg(reinterpret_cast<const uint4*>(p + head) + i); }
};

// Elements of one row that this thread visits: f(x, index) for the unaligned
// head and tail, g(vector, first index) for the 16-byte vectors between.
template <typename T, typename F, typename G>
__device__ __forceinline__ void for_row(const Row<T>& row, int rank, int ranks, F&& f, G&& g) {
  constexpr int N = Vec<T>::N;
  const int step = ranks * kLpThreads;
  // the next kLpAhead vectors load while these are worked on; those past the
  // end count as minus infinity
  uint4 x[kLpAhead];
  auto load = [&](int i) {
#pragma unroll
    for (int j = 0; j < kLpAhead; ++j)
      x[j] = i + j * step < row.nvec ? row.vec(i + j * step) : make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
  };
  int i = rank * kLpThreads + threadIdx.x;
  load(i);
#pragma unroll 1
  for (; i < row.nvec; i += kLpAhead * step) {
    uint4 y[kLpAhead];
#pragma unroll
    for (int j = 0; j < kLpAhead; ++j) y[j] = x[j];
    load(i + kLpAhead * step);
#pragma unroll
    for (int j = 0; j < kLpAhead; ++j) g(y[j], row.head + (i + j * step) * N);
  }
  if (rank == ranks - 1) {
    const int t = threadIdx.x;
    if (t < row.head) f(load1(row.p + t), t);
    if (row.tail + t < row.vocab) f(load1(row.p + row.tail + t), row.tail + t);
  }
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, kLpPerSm) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int N = Vec<T>::N;
  __shared__ Stat s_stat[kLpWarps], s_all;
  __shared__ uint32_t s_max[kLpThreads];  // each thread's maximum
  __shared__ unsigned long long s_cand[kLpCands], s_top[kMaxTop], s_best[kLpWarps];
  __shared__ uint16_t s_hit[kLpThreads];
  __shared__ int s_ncand, s_nhit;
  __shared__ uint32_t s_bound;
  __shared__ Share s_share[8];  // on the cluster's first CTA: every CTA's result
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ranks = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  pdl_wait_prior();
  if (ranks > 1) cluster_arrive();  // every CTA runs before the first one's shared memory is written
  const int64_t t = blockIdx.x / ranks;
  const Row<T> row(static_cast<const T*>(a.logits) + t * a.ld, a.vocab);

  const long long token = a.tokens64 ? __ldg(static_cast<const long long*>(a.tokens) + t)
                                     : static_cast<long long>(__ldg(static_cast<const int*>(a.tokens) + t));
  const bool known = token >= 0 && token < a.vocab;
  const float given = known ? load1(row.p + token) : -INFINITY;

  uint32_t given2 = 0;
  if constexpr (sizeof(T) == 2) given2 = Elem<T>::pack2(given, given);

  // ---- the pass: running maximum, sums, rank
  Stat st{-INFINITY, 0.f, 0.f, 0.f, 0};
  float r2 = Vec<T>::kLow * kLog2e;  // the reference, in log2 units
  uint64_t l2 = 0, s2 = 0, neg2 = pack_f2(-r2, -r2);  // sums of even and odd elements; -r2 twice
  const uint64_t log2e2 = pack_f2(kLog2e, kLog2e);
  auto raise = [&](float x) {
    st.raw = fmaxf(st.raw, x);
    const float old = r2;
    r2 = fmaxf(r2, x * kLog2e);
    const float d = fmaxf(old - r2, -1e30f), f = ex2(d);  // 0 * finite
    const uint64_t f2 = pack_f2(f, f);
    s2 = fma_f2(f2, fma_f2(l2, pack_f2(d, d), s2), 0);
    l2 = fma_f2(f2, l2, 0);
    neg2 = pack_f2(-r2, -r2);
  };
  auto add2 = [&](float x, float y) {
    const uint64_t d = fma_f2(pack_f2(x, y), log2e2, neg2);
    float d0, d1;
    unpack_f2(d, d0, d1);
    const uint64_t e = pack_f2(ex2(d0), ex2(d1));
    l2 = add_f2(l2, e);
    s2 = fma_f2(e, d, s2);
  };
  for_row(
      row, rank, ranks,
      [&](float x, int) {
        if (x > st.raw) raise(x);
        st.above += x > given;
        add2(x == x ? fmaxf(x, Vec<T>::kLow) : x, Vec<T>::kLow);
      },
      [&](const uint4& v, int) {
        float x[N];
        const float top = Vec<T>::largest(v);
        if (top > st.raw) raise(top);
        if (top > given) st.above += Vec<T>::above(v, given2, given);
        Vec<T>::unpack(Vec<T>::raised(v), x);
#pragma unroll
        for (int i = 0; i < N; i += 2) add2(x[i], x[i + 1]);
      });
  {
    float p, q;
    unpack_f2(l2, p, q);
    st.l = p + q;
    unpack_f2(s2, p, q);
    st.s = p + q;
    // from the rounded reference to the maximum itself
    st.ref = fmaxf(st.raw, Vec<T>::kLow);
    const float d = fmaf(st.ref, kLog2e, -r2), f = ex2(-d);
    st.s = f * fmaf(-d, st.l, st.s);
    st.l *= f;
  }
  const bool nan = st.l != st.l;
  s_max[tid] = st.raw == -INFINITY ? 0u : ordered(st.raw);
  const uint32_t my_max = nan ? 0xffffffffu : s_max[tid];
  Stat w = st;
#pragma unroll
  for (int o = 16; o; o >>= 1) w = merge(w, shfl_xor(w, o));
  if (lane == 0) s_stat[warp] = w;
  if (tid == 0) s_ncand = s_nhit = 0;
  if (tid < kMaxTop) s_top[tid] = 0;
  __syncthreads();
  if (a.top > 0 && warp == 0) {
    // 32 groups of threads: the top-th largest of their maxima (0: fewer have one)
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kLpWarps; ++i) mine = max(mine, s_max[i * 32 + lane]);
    int place = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint32_t o = __shfl_sync(~0u, mine, i);
      place += o > mine || (o == mine && i < lane);
    }
    if (place == a.top - 1) s_bound = mine;
  } else if (warp == kLpWarps - 1) {
    w = s_stat[lane % kLpWarps];
#pragma unroll
    for (int o = kLpWarps / 2; o; o >>= 1) w = merge(w, shfl_xor(w, o));
    if (lane == 0) s_all = w;
  }
  __syncthreads();
  w = s_all;
  // Where nothing is well above the lowest logit (masked rows), or the maximum
  // is enormous, the sums again with x - M exact: M is known now. NaN stays.
  if (!(w.raw > Vec<T>::kLow + 200.f && w.raw < kHigh)) {
    float l = 0.f, s = 0.f;
    const float m = fmaxf(w.raw, -FLT_MAX);
    auto exact = [&](float x) {
      float d = (x - m) * kLog2e;
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(-1e30f));
      const float e = ex2(d);
      l += e;
      s = fmaf(e, d, s);
    };
    for_row(
        row, rank, ranks, [&](float x, int) { exact(x); },
        [&](const uint4& v, int) {
          float x[N];
          Vec<T>::unpack(v, x);
#pragma unroll
          for (int i = 0; i < N; ++i) exact(x[i]);
        });
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      l += __shfl_xor_sync(~0u, l, o);
      s += __shfl_xor_sync(~0u, s, o);
    }
    if (lane == 0) s_stat[warp].l = l, s_stat[warp].s = s;
    __syncthreads();
    w.ref = m;
    w.l = w.s = 0.f;
#pragma unroll
    for (int i = 0; i < kLpWarps; ++i) w.l += s_stat[i].l, w.s += s_stat[i].s;
  }

  // ---- the largest `top` of this CTA's part of the row
  unsigned long long mine = 0;  // thread i < top: the i-th largest key
  if (a.top > 0) {
    const uint32_t bound = s_bound;
    const float low = bound == 0 ? -INFINITY : unordered(bound);
    auto keep = [&](float x, int i) {
      if (!(x < low)) {
        const int at = atomicAdd(&s_ncand, 1);
        if (at < kLpCands) s_cand[at] = key_of(x, i);
      }
    };
    // the threads to look at again, each with `per` vectors and perhaps an
    // element of the row's head and tail; all threads share the work
    if (my_max >= bound) s_hit[atomicAdd(&s_nhit, 1)] = static_cast<uint16_t>(tid);
    __syncthreads();
    const int step = ranks * kLpThreads, per = (row.nvec + step - 1) / step, hits = s_nhit;
#pragma unroll 4
    for (int i = tid; i < hits * per; i += kLpThreads) {
      const int at = rank * kLpThreads + s_hit[i % hits] + i / hits * step;
      const uint4 v = at < row.nvec ? row.vec(at) : make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
      if (at < row.nvec && !(Vec<T>::largest(v) < low)) {
        float x[N];
        Vec<T>::unpack(v, x);
#pragma unroll
        for (int j = 0; j < N; ++j) keep(x[j], row.head + at * N + j);
      }
    }
    if (rank == ranks - 1 && my_max >= bound) {
      if (tid < row.head) keep(load1(row.p + tid), tid);
      if (row.tail + tid < row.vocab) keep(load1(row.p + row.tail + tid), row.tail + tid);
    }
    __syncthreads();
    const int n = s_ncand;
    if (n <= kLpCands) {
      // a candidate's place is the number of larger keys
      for (int i = tid; i < n; i += kLpThreads) {
        const unsigned long long k = s_cand[i];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) place += s_cand[j] > k;
        if (place < a.top) s_top[place] = k;
      }
      __syncthreads();
      if (tid < a.top) mine = s_top[tid];
    } else {
      // long runs of equal logits: one pass over the row for each place
      unsigned long long last = ~0ull;
#pragma unroll 1
      for (int p = 0; p < a.top; ++p) {
        unsigned long long b = 0;
        auto look = [&](float x, int i) {
          const unsigned long long k = key_of(x, i);
          if (k < last && k > b) b = k;
        };
        for_row(row, rank, ranks, look, [&](const uint4& v, int i0) {
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
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(w.raw), "f"(w.ref), "f"(w.l), "f"(w.s)
                   : "memory");
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + 16), "r"(w.above) : "memory");
    }
    if (tid < kMaxTop)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(
                       dst + static_cast<uint32_t>(offsetof(Share, top)) + 8u * tid),
                   "l"(mine)
                   : "memory");
    cluster_sync_hw();
    if (rank != 0) return;
    w = s_share[0].stat;
    for (int i = 1; i < ranks; ++i) w = merge(w, s_share[i].stat);
  }
  const bool empty = w.raw == -INFINITY && w.l == w.l;
  const float log_l = logf(w.l);
  auto log_prob = [&](float x) { return empty || (x == -INFINITY && w.l == w.l) ? -INFINITY : (x - w.raw) - log_l; };
  if (tid == 0) {
    a.logprob[t] = log_prob(given);
    if (a.entropy) a.entropy[t] = empty ? 0.f : log_l - kLn2 * (w.s / w.l);
    if (a.rank) a.rank[t] = w.above + 1;
  }
  auto put = [&](int place, unsigned long long k) {
    a.top_ids[t * a.top + place] = k == 0 ? -1 : 0x7fffffff - static_cast<int>(k & 0xffffffffu);
    a.top_logprobs[t * a.top + place] = k == 0 ? -INFINITY : log_prob(unordered(static_cast<uint32_t>(k >> 32)));
  };
  if (ranks == 1) {
    if (tid < a.top) put(tid, mine);
  } else {
    for (int i = tid; i < ranks * kMaxTop; i += kLpThreads) {
      const unsigned long long k = s_share[i / kMaxTop].top[i % kMaxTop];
      if (k == 0) continue;
      int place = 0;
      for (int j = 0; j < ranks; ++j) {
        const ulonglong2* o = reinterpret_cast<const ulonglong2*>(s_share[j].top);
#pragma unroll
        for (int p = 0; p < kMaxTop / 2; ++p) place += (o[p].x > k) + (o[p].y > k);
      }
      if (place < a.top) put(place, k);
    }
  }
}

template <typename T>
cudaError_t launch(const LogprobArgs& a, int num_sms, cudaStream_t stream) {
  // CTAs per row: as many as run at once, while each still has a vector for
  // each of its threads
  int ranks = 1;
  while (ranks < 8 && static_cast<int64_t>(a.rows) * 2 * ranks <= kLpPerSm * num_sms &&
         static_cast<int64_t>(a.vocab) >= static_cast<int64_t>(2 * ranks) * kLpThreads * Vec<T>::N)
    ranks *= 2;
  return launch_after(token_logprobs_kernel<T>, dim3(a.rows * ranks), kLpThreads, 0, stream, a.pdl, ranks, a);
}

}  // namespace

cudaError_t launch_token_logprobs(int dtype, const LogprobArgs& a, int num_sms, cudaStream_t stream) {
  if (dtype == 2) return launch<float>(a, num_sms, stream);
  return dtype == 1 ? launch<__nv_bfloat16>(a, num_sms, stream) : launch<__half>(a, num_sms, stream);
}

}  // namespace wp
