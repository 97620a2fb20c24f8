// wp_attention.cu -- causal attention over packed prompts of different lengths,
// with grouped heads.
//
//   out[i, h] = sum_j p_ij v[j, h / G] / sum_j p_ij,
//   p_ij = 2^((scale q[i, h] . k[j, h / G] - m_i) log2 e),  j <= i + nk - nq
// per sequence of nq query and nk key tokens (bottom-right causal: a chunk of a
// prompt follows its context). Scores, maxima, sums and outputs are fp32; the
// weights p are rounded to the inputs' 16-bit type for the second product (at
// most 1, so the rounding is relative, as the output's own is) while their sum
// is taken before the rounding. A row that sees no key is 0.
//
// Query rows of one kv head are packed: row r of a sequence's (kv head) is
// token r / G, head r % G of the group, so grouped heads share every K and V
// tile and a few tokens of many heads fill a tile's rows.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "wp_device.cuh"
#include "wp_internal.h"

namespace wp {
namespace {

struct PromptSeq {
  int q0, nq, k0, nk;
};

// A sequence's rows, forced into the packed tensors (offsets outside them
// raise the error bit).
__device__ __forceinline__ PromptSeq prompt_seq(const PromptArgs& a, int b) {
  int q0 = __ldg(a.cu_q + b), q1 = __ldg(a.cu_q + b + 1), k0 = __ldg(a.cu_k + b), k1 = __ldg(a.cu_k + b + 1);
  if (q0 < 0 || q1 < q0 || q1 > a.q_tokens || k0 < 0 || k1 < k0 || k1 > a.k_tokens) {
    if (a.err) atomicOr(a.err, kErrBadSegment);
    q0 = min(max(q0, 0), a.q_tokens);
    q1 = min(max(q1, q0), a.q_tokens);
    k0 = min(max(k0, 0), a.k_tokens);
    k1 = min(max(k1, k0), a.k_tokens);
  }
  return PromptSeq{q0, q1 - q0, k0, k1 - k0};
}

// One row by one warp, over its visible keys only, element by element. The
// tiled kernels multiply the weight 0 of a key that a row must not see with
// that key's V, which is NaN where V is not finite; rows whose result is not
// finite come here, so only a row's own keys decide what it is.
template <typename T>
__device__ __noinline__ void prompt_row(const PromptArgs& a, const PromptSeq& s, int token, int head) {
  const int lane = threadIdx.x & 31, d0 = lane * 4, kvh = head / (a.heads / a.kv_heads);
  const bool on = d0 < a.dim;
  auto load = [&](const T* p, float (&x)[4]) {
    const uint2 w = on ? __ldg(reinterpret_cast<const uint2*>(p + d0)) : make_uint2(0, 0);
    const float2 f = Elem<T>::unpack2(w.x), g = Elem<T>::unpack2(w.y);
    x[0] = f.x, x[1] = f.y, x[2] = g.x, x[3] = g.y;
  };
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  load(static_cast<const T*>(a.q) + static_cast<int64_t>(s.q0 + token) * a.q_ts + head * a.q_hs, q);
  const int end = min(token + s.nk - s.nq + 1, s.nk);
  for (int j = 0; j < end; ++j) {
    float k[4], v[4];
    load(static_cast<const T*>(a.k) + static_cast<int64_t>(s.k0 + j) * a.k_ts + kvh * a.k_hs, k);
    load(static_cast<const T*>(a.v) + static_cast<int64_t>(s.k0 + j) * a.v_ts + kvh * a.v_hs, v);
    float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
    for (int off = 16; off; off >>= 1) x += __shfl_xor_sync(~0u, x, off);
    x *= a.scale * kLog2e;
    const float mn = x > m ? x : m, base = mn == -INFINITY ? 0.f : mn;
    const float f = ex2(m - base), p = ex2(x - base);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + p * v[i];
  }
  const int64_t at = static_cast<int64_t>(s.q0 + token) * a.heads + head;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (on)
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.dim + d0) =
        make_uint2(Elem<T>::pack2(o[0] * inv, o[1] * inv), Elem<T>::pack2(o[2] * inv, o[3] * inv));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---- few query rows: warp-level MMA ---------------------------------------------
//
// NW warps share 64-key tiles of K and V (two of each, loaded asynchronously);
// a warp has 16 packed rows. For sequences of a few tokens, where a tcgen05
// tile of 128 rows would be nearly empty and latency is everything.

template <typename T, int D, int NW>
struct SmallCfg {
  static constexpr int BN = 64;
  static constexpr int LD = D * 2 + 16;  // padded row: eight rows of one ldmatrix fall into different banks
  static constexpr int TILE = BN * LD;
  static constexpr int SMEM = 4 * TILE + NW * 16 * LD;
};

template <typename T, int D, int NW>
__global__ void __launch_bounds__(NW * 32) prompt_small_kernel(const __grid_constant__ PromptArgs a) {
  using C = SmallCfg<T, D, NW>;
  using E = Elem<T>;
  constexpr int BN = C::BN, LD = C::LD, KS = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.y, group = a.heads / a.kv_heads;
  const uint32_t ring = smem_u32(smem), qs = ring + 4 * C::TILE + warp * 16 * LD;
  const int chunks = a.dim / 8;  // 16-byte pieces of a row; dimensions past dim are zero

  int b = blockIdx.z, rb = blockIdx.x;
  PromptSeq s = prompt_seq(a, b);
  while (true) {
    const int rows = s.nq * group;
    if (rb * NW * 16 >= rows) {
      if ((b += gridDim.z) >= a.num_seqs) break;
      rb = blockIdx.x;
      s = prompt_seq(a, b);
      continue;
    }
    const int r0 = rb * NW * 16;
    // keys that the block's last row sees
    const int last = (min(r0 + NW * 16, rows) - 1) / group;
    const int end = min(max(last + s.nk - s.nq + 1, 0), s.nk);
    auto load_tile = [&](int j0, int buf) {
      const T* kb = static_cast<const T*>(a.k) + static_cast<int64_t>(s.k0 + j0) * a.k_ts + kvh * a.k_hs;
      const T* vb = static_cast<const T*>(a.v) + static_cast<int64_t>(s.k0 + j0) * a.v_ts + kvh * a.v_hs;
      const int n = (min(end - j0, BN) + 15) & ~15;
      for (int i = tid; i < n * (D / 8); i += NW * 32) {
        const int j = i / (D / 8), d = i % (D / 8);
        const bool on = j0 + j < end && d < chunks;
        const uint32_t off = buf * C::TILE + j * LD + d * 16;
        cp_async16(ring + off, on ? kb + j * a.k_ts + d * 8 : kb, on);
        cp_async16(ring + 2 * C::TILE + off, on ? vb + j * a.v_ts + d * 8 : vb, on);
      }
    };
    for (int i = lane; i < 16 * (D / 8); i += 32) {
      const int j = i / (D / 8), d = i % (D / 8), r = r0 + warp * 16 + j;
      const bool on = r < rows && d < chunks;
      const T* p = static_cast<const T*>(a.q) + (on ? static_cast<int64_t>(s.q0 + r / group) * a.q_ts +
                                                          (kvh * group + r % group) * a.q_hs + d * 8
                                                    : 0);
      cp_async16(qs + j * LD + d * 16, p, on);
    }
    if (end > 0) load_tile(0, 0);
    cp_async_commit();

    // rows g and g + 8 of the warp: the keys they see
    int lim[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) lim[i] = min((r0 + warp * 16 + g + 8 * i) / group + s.nk - s.nq + 1, s.nk);
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    uint32_t qf[KS][4];
    const float sc = a.scale * kLog2e;

    for (int j0 = 0, buf = 0; j0 < end; j0 += BN, buf ^= 1) {
      if (j0 + BN < end) load_tile(j0 + BN, buf ^ 1);
      cp_async_commit();
      cp_async_wait<1>();
      __syncthreads();
      if (j0 == 0) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
          ldsm_x4(qs + (lane & 15) * LD + k * 32 + (lane >> 4) * 16, qf[k][0], qf[k][1], qf[k][2], qf[k][3]);
      }
      const uint32_t ks = ring + buf * C::TILE, vs = ks + 2 * C::TILE;
      const int n16 = (min(end - j0, BN) + 15) / 16;  // groups of 16 keys
      float p[BN / 16][8];
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int t = 0; t < BN / 16; ++t) {
        if (t >= n16) break;
        float x[2][4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t b0, b1, b2, b3;  // keys 0-7: dims 0-7, 8-15; keys 8-15 the same
          ldsm_x4(ks + (t * 16 + (lane & 7) + (lane >> 4) * 8) * LD + k * 32 + ((lane >> 3) & 1) * 16, b0, b1, b2, b3);
          mma_k16<T>(x[0], qf[k], b0, b1);
          mma_k16<T>(x[1], qf[k], b2, b3);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = j0 + t * 16 + h * 8 + 2 * c + (j & 1);
            const float y = key < lim[j >> 1] ? x[h][j] * sc : -INFINITY;
            p[t][h * 4 + j] = y;
            top[j >> 1] = fmaxf(top[j >> 1], y);
          }
      }
      float base[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 2));
        const float mn = fmaxf(m[i], top[i]);
        base[i] = mn == -INFINITY ? 0.f : mn;
        const float f = ex2(m[i] - base[i]);
        m[i] = mn;
        l[i] *= f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][2 * i] *= f;
          o[d][2 * i + 1] *= f;
        }
      }
#pragma unroll
      for (int t = 0; t < BN / 16; ++t) {
        if (t >= n16) break;
        uint32_t pa[4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float e0 = ex2(p[t][h * 4 + 2 * i] - base[i]), e1 = ex2(p[t][h * 4 + 2 * i + 1] - base[i]);
            l[i] += e0 + e1;
            pa[h * 2 + i] = E::pack2(e0, e1);
          }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t b0, b1, b2, b3;  // dims 0-7: keys 0-7, 8-15; dims 8-15 the same
          ldsm_x4_t(vs + (t * 16 + (lane & 15)) * LD + d * 32 + (lane >> 4) * 16, b0, b1, b2, b3);
          mma_k16<T>(o[2 * d], pa, b0, b1);
          mma_k16<T>(o[2 * d + 1], pa, b2, b3);
        }
      }
      __syncthreads();
    }
    cp_async_wait<0>();  // Q of a block that sees no key

    bool bad[2] = {false, false};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(~0u, l[i], 1);
      l[i] += __shfl_xor_sync(~0u, l[i], 2);
      const int r = r0 + warp * 16 + g + 8 * i;
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
      const int64_t at = static_cast<int64_t>(s.q0 + r / group) * a.heads + kvh * group + r % group;
      T* op = static_cast<T*>(a.out) + at * a.dim + 2 * c;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        const float x = o[d][2 * i] * inv, y = o[d][2 * i + 1] * inv;
        bad[i] |= !(fabsf(x) <= 3e38f) || !(fabsf(y) <= 3e38f);
        if (r < rows && d < chunks) *reinterpret_cast<uint32_t*>(op + d * 8) = E::pack2(x, y);
      }
      if (a.lse && c == 0 && r < rows) a.lse[at] = l[i] == 0.f ? -INFINITY : (m[i] + __log2f(l[i])) * kLn2;
      bad[i] &= r < rows;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      for (unsigned todo = __ballot_sync(~0u, bad[i]); todo;) {
        const int lead = __ffs(todo) - 1, r = r0 + warp * 16 + (lead >> 2) + 8 * i;
        todo &= ~(0xfu << (lead & ~3));
        prompt_row<T>(a, s, r / group, kvh * group + r % group);
      }
    __syncthreads();  // the next block's loads overwrite Q and the tiles
    rb += gridDim.x;
  }
}

template <typename T, int D, int NW>
cudaError_t launch_small(const PromptArgs& a, cudaStream_t stream) {
  using C = SmallCfg<T, D, NW>;
  static std::atomic<bool> ready{false};
  if (!ready.load()) {
    cudaError_t e = cudaFuncSetAttribute(prompt_small_kernel<T, D, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    ready.store(true);
  }
  const int group = a.heads / a.kv_heads;
  const int64_t blocks = (static_cast<int64_t>(a.max_q) * group + NW * 16 - 1) / (NW * 16);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(blocks, 1), 4096)), a.kv_heads,
                  std::min(a.num_seqs, 65535));
  prompt_small_kernel<T, D, NW><<<grid, NW * 32, C::SMEM, stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_prompt(const PromptArgs& a, int num_sms, cudaStream_t stream) {
  (void)num_sms;
  const int64_t rows = static_cast<int64_t>(a.max_q) * (a.heads / a.kv_heads);
  if (a.dim <= 64)
    return rows <= 16 ? launch_small<T, 64, 1>(a, stream) : launch_small<T, 64, 4>(a, stream);
  return rows <= 16 ? launch_small<T, 128, 1>(a, stream) : launch_small<T, 128, 4>(a, stream);
}

}  // namespace

cudaError_t launch_prompt_attention(int dtype, const PromptArgs& a, int num_sms, cudaStream_t stream) {
  return dtype == 1 ? launch_prompt<__nv_bfloat16>(a, num_sms, stream) : launch_prompt<__half>(a, num_sms, stream);
}

}  // namespace wp
