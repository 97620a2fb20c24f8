// wp_attention.cu -- causal attention over packed prompts of different lengths,
// with grouped heads.
//
//   out[i, h] = sum_j p_ij v[j, h / G] / sum_j p_ij,
//   p_ij = 2^((scale q[i, h] . k[j, h / G] - m_i) log2 e),  j <= i + nk - nq
// per sequence of nq query and nk key tokens (bottom-right causal: a chunk of a
// prompt follows its context). Scores, maxima, sums and outputs are fp32; the
// weights p are rounded to the inputs' 16-bit type for the second product
// while their sum is taken before the rounding. The rounding is relative, as
// the output's own is: bf16 has fp32's exponents, and in fp16 weights and sum
// have a power of two as a factor (`kWeightUp`) that uses its range up to 2^15:
// weights down to 2^-22 of the row's largest are normal numbers, and those down
// to 2^-33 count. A row that sees no key is 0.
//
// Query rows of one kv head are packed: row r of a sequence's (kv head) is
// token r / G, head r % G of the group, so grouped heads share every K and V
// tile and a few tokens of many heads fill a tile's rows.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "wp_device.cuh"
#include "wp_internal.h"
#include "wp_once.h"

namespace wp {
namespace {

struct PromptSeq {
  int q0, nq, k0, nk;
};

// log2 of what a weight of 2^0 is multiplied by, for weights up to 2^lazy.
template <typename T>
__device__ constexpr float weight_up(float lazy) {
  return Elem<T>::is_bf16 ? 0.f : 15.f - lazy;
}

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

// One row by one warp, over its visible keys only. The tiled kernels multiply
// the weight 0 of a key that a row must not see with that key's V, which is NaN
// where V is not finite; rows whose result is not finite come here, so only a
// row's own keys decide what it is. 32 keys at a time: a lane has the score of
// one of them, then four dimensions of the output. The caller has passed a
// __syncwarp since the row's first stores.
template <typename T>
__device__ __forceinline__ void prompt_row(const PromptArgs& a, const PromptSeq& s, int token, int head) {
  const int lane = threadIdx.x & 31, d0 = lane * 4, kvh = head / (a.heads / a.kv_heads);
  const bool on = d0 < a.dim;
  const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(s.q0 + token) * a.q_ts + head * a.q_hs;
  const T* k = static_cast<const T*>(a.k) + static_cast<int64_t>(s.k0) * a.k_ts + kvh * a.k_hs;
  const T* v = static_cast<const T*>(a.v) + static_cast<int64_t>(s.k0) * a.v_ts + kvh * a.v_hs + (on ? d0 : 0);
  float o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  const int end = min(token + s.nk - s.nq + 1, s.nk);
#pragma unroll 1
  for (int j0 = 0; j0 < end; j0 += 32) {
    float x = -INFINITY;
    if (j0 + lane < end) {
      const T* kr = k + (j0 + lane) * a.k_ts;
      x = 0.f;
#pragma unroll 2
      for (int d = 0; d < a.dim; d += 8) {
        const uint4 kw = __ldg(reinterpret_cast<const uint4*>(kr + d)), qw = __ldg(reinterpret_cast<const uint4*>(q + d));
        const uint32_t ku[4] = {kw.x, kw.y, kw.z, kw.w}, qu[4] = {qw.x, qw.y, qw.z, qw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Elem<T>::unpack2(ku[i]), g = Elem<T>::unpack2(qu[i]);
          x = fmaf(f.x, g.x, x);
          x = fmaf(f.y, g.y, x);
        }
      }
      x *= a.scale * kLog2e;
    }
    float top = x;
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, off));
    top = fmaxf(m, top);
    const float base = top == -INFINITY ? 0.f : top, f = ex2(m - base), p = ex2(x - base);
    m = top;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= f;
    const int n = min(end - j0, 32);
#pragma unroll 4
    for (int t = 0; t < n; ++t) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(v + (j0 + t) * a.v_ts));
      const float2 f0 = Elem<T>::unpack2(w.x), f1 = Elem<T>::unpack2(w.y);
      const float pt = __shfl_sync(~0u, p, t);
      o[0] = fmaf(pt, f0.x, o[0]);
      o[1] = fmaf(pt, f0.y, o[1]);
      o[2] = fmaf(pt, f1.x, o[2]);
      o[3] = fmaf(pt, f1.y, o[3]);
    }
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) l += __shfl_xor_sync(~0u, l, off);
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
// tile of 128 rows would be nearly empty and latency is everything: 5 us for 64
// sequences of 4 tokens, 12 heads of 64 (0.24 us of traffic), of which about 4
// are the launch and three dependent loads (offsets, tiles, result).

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
  constexpr float kWeightUp = weight_up<T>(0.f);
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.y, group = a.heads / a.kv_heads;
  const uint32_t ring = smem_u32(smem), qs = ring + 4 * C::TILE + warp * 16 * LD;
  const int chunks = a.dim / 8;  // 16-byte pieces of a row; dimensions past dim are zero

  pdl_wait_prior();
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
        base[i] -= kWeightUp;
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
      if (a.lse && c == 0 && r < rows) a.lse[at] = l[i] == 0.f ? -INFINITY : (m[i] + (__log2f(l[i]) - kWeightUp)) * kLn2;
      bad[i] &= r < rows && l[i] == l[i];  // a NaN among the row's own scores: all of it is NaN
    }
    __syncwarp();  // a row's first stores come from other lanes
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
  static PerDevice ready;
  if (!ready.get([] {
        return cudaFuncSetAttribute(prompt_small_kernel<T, D, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) ==
               cudaSuccess;
      }))
    return cudaGetLastError();
  const int group = a.heads / a.kv_heads;
  const int64_t blocks = (static_cast<int64_t>(a.max_q) * group + NW * 16 - 1) / (NW * 16);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(blocks, 1), 4096)), a.kv_heads,
                  std::min(a.num_seqs, 65535));
  return launch_after(prompt_small_kernel<T, D, NW>, grid, NW * 32, C::SMEM, stream, a.pdl, 1, a);
}

// ---- many query rows: tcgen05 -----------------------------------------------------
//
// A work item is (sequence, kv head, pair of 128-row tiles of packed query
// rows). Per 128 keys: S_i = Q_i K^T and O_i += P_i V for both tiles i, four
// tcgen05.mma groups of 128 x 128 x D. S and O live in TMEM (2 x 128 + 2 x D
// columns of 512); the weights P go back into S's own columns as 16-bit pairs
// and are the second product's A operand from there, so they never touch
// shared memory.
//
// Warps (384 threads): 0-3 softmax of tile 0, 4-7 of tile 1 (one thread per
// row: no exchange between lanes), 8 TMA producer, 9 and 10 MMA issuers of tile
// 0 and 1, 11 fetches items. The last four give registers to the softmax warps,
// which hold a row's 128 scores (256 x 216 + 128 x 72 = the launch's 384 x 168). While one tile's
// softmax runs, the other's P V and next Q K^T keep the tensor core busy. Each
// tile has its own issuer because the tensor core queues only a few products,
// so one issuer's waits for both tiles would drain it; the issuers take turns
// (`turn`), because two tiles whose products interleave end up with their
// softmaxes at the same time (8192 tokens, when introduced: 608 against 494 us). The
// products of one issuer run in order, so S_i(j + 1) may follow P_i(j) V into
// the same columns, and the arrival of S_i(j) tells that O_i holds all blocks
// before j. P V starts on the first 64 keys' weights.
//
// The running maximum is only raised when a row's grows by more than 8 (in
// log2 units; 7 in fp16): weights then reach 2^8 at most (2^15 with fp16's
// factor), and O is rescaled in a few blocks at the start instead of in most.
//
// The grid has a CTA per item, in the order (sequence, pairs from the last one,
// kv head), so long items come first within a sequence. A resident CTA that
// has issued an item's last load cancels the launch of one of the CTAs that
// still wait for an SM and takes over its item next (warp 11, which also looks
// it up for the others). So an SM is set up once, its next item's loads run
// while the current one ends, and no SM is left with two long items at the end.
// When introduced, against one CTA per SM with a fixed share of the items, which
// every warp looked up for itself (32 query / 8 kv heads of 128, device time): 4
// sequences of 2048 tokens 151 against 204 us, 64 of 100-400 tokens 123 / 136,
// one of 8192 469 / 499, 16 of 1-1500 tokens 42.3 / 50.4; 64 of 256, 12 heads of
// 64: 38 / 44. Taking the next item when the current one begins: 159, 123, 474,
// 50.7 and 38 us; two ahead, 175 us in the first case. Now: 145 us in the first
// case, 437-443 for one of 8192, 38 for 64 of 256.

// Limit of the waits: rows that are computed again (prompt_row) hold the other
// warps of the CTA up for as long as their sequence is long. The 32 rows of a
// warp take 8 us per key with 64 dimensions and 10-12 with 128, when every warp
// of the GPU is at it (50000 and 200000 keys). The limit is 16 polls of 4 us
// per key of the call, and a second for the rest. (A limit that starts anew
// while such rows come further cost every call 1-9%, in the waits' code.)
constexpr int kPollsBase = 1 << 18, kPollsPerKey = 16;
constexpr unsigned long long kPollNs = 4000;

constexpr int kPaWarps = 12;
constexpr int kPaThreads = kPaWarps * 32;
constexpr int kPaProd = 8;
constexpr int kPaMma = 9;
constexpr int kPaRows = 128;  // rows of a tile
constexpr int kPaKeys = 128;  // keys of a block
template <typename T>
constexpr float kPaLazy = Elem<T>::is_bf16 ? 8.f : 7.f;
// Of 8 pairs of weights, those that take the FMA pipe instead of the special-
// function unit. 32 query / 8 kv heads of 128, bf16, for 0, 1, 2 and 3: 4 x 2048
// tokens 150, 156, 145 and 149 us, 64 x 100-400 tokens 129, 134, 131 and 135, 1
// x 1000 25.5, 26.4, 24.8 and 25.6, 1 x 8192 472, 482, 437 and 453 (437: 1.26
// PFLOP/s, 76% of the measured matrix rate). What bounds it is the chain scores
// -> maximum -> weights -> products of a tile, 3300 cycles per 128 keys of two
// tiles against 2100 of the products alone; in long runs also the power cap.
constexpr int kPaFma = 2;

template <int DP>
struct PaCfg {
  static constexpr int SL = DP / 64;  // 64-column slices of a row
  static constexpr int SLICE = 128 * 128;  // bytes of one slice of 128 rows
  static constexpr int TILE = SL * SLICE;
  static constexpr int S = DP == 128 ? 5 : 8;  // ring stages; K and V tiles alternate
  static constexpr int HEAD = 2048;  // barriers, prefix sums
  static constexpr int SMEM = HEAD + 1024 + (2 + S) * TILE;
  static constexpr uint32_t COL_O = 256;
  static_assert(SMEM <= 232448, "shared memory budget");
};

struct PaMaps {
  CUtensorMap q;  // [tokens][heads][dim], box 64 columns x group x tokens of a tile
  CUtensorMap k, v;  // [tokens][kv heads][dim], box 64 columns x 1 x 128
};

struct __align__(16) PaItem {
  PromptSeq s;
  int kvh;
  int t0;  // first token of the pair; -1: no item any more
  int n[2];  // key blocks of each tile (0: no tokens, or none that sees a key)
};

template <typename T, int DP>
__global__ void __launch_bounds__(kPaThreads, 1)
    prompt_tile_kernel(const __grid_constant__ PromptArgs a, const __grid_constant__ PaMaps maps) {
  using C = PaCfg<DP>;
  using E = Elem<T>;
  constexpr int S = C::S;
  constexpr float kWeightUp = weight_up<T>(kPaLazy<T>);
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem);  // [S]
  uint64_t* kv_empty = kv_full + 8;  // [S]
  uint64_t* q_full = kv_full + 16;  // [2]
  uint64_t* q_empty = kv_full + 18;
  uint64_t* s_full = kv_full + 20;
  uint64_t* p_full = kv_full + 22;  // [2 tiles][2 halves of the keys]
  uint64_t* turn = kv_full + 26;  // whose products are next
  uint64_t* o_full = kv_full + 28;
  uint64_t* o_free = kv_full + 30;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(kv_full + 32);
  volatile int* s_bad = reinterpret_cast<volatile int*>(kv_full + 33);
  uint64_t* next_full = kv_full + 40;  // *s_item is the next item
  uint64_t* next_empty = kv_full + 41;
  uint64_t* taken = kv_full + 42;  // a cancellation's answer is there
  uint64_t* drained = kv_full + 50;  // an issuer's products have ended (where a wait ran out)
  uint4* s_answer = reinterpret_cast<uint4*>(kv_full + 44);
  PaItem* s_item = reinterpret_cast<PaItem*>(kv_full + 46);
  int* s_warp = reinterpret_cast<int*>(kv_full + 34);  // [kPaWarps]
  int* s_sum = reinterpret_cast<int*>(smem + 512);  // items before thread i's slice of sequences
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem) + C::HEAD + 1023) & ~uintptr_t(1023));
  uint8_t* ring = tiles + 2 * C::TILE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.heads / a.kv_heads;
  const int tpt = kPaRows / group;  // tokens of a tile

  if (tid == 0) {
#pragma unroll 1
    for (int i = 0; i < S; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 2);  // both issuers
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&turn[i], 1);
      mbar_init(&drained[i], 1);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], 4);
    }
    mbar_init(next_full, 1);
    mbar_init(next_empty, kPaWarps - 1);
    mbar_init(taken, 1);
    *s_bad = 0;
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(s_tmem, 512);
  pdl_wait_prior();

  // ---- items of each thread's slice of sequences, and their prefix sums
  const int slice = (a.num_seqs + kPaThreads - 1) / kPaThreads;
  auto pairs_of = [&](int nq) { return (nq + 2 * tpt - 1) / (2 * tpt); };
  int mine = 0;
#pragma unroll 1
  for (int b = tid * slice; b < min((tid + 1) * slice, a.num_seqs); ++b) mine += pairs_of(prompt_seq(a, b).nq) * a.kv_heads;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_warp[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *s_tmem;
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kPaWarps; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  s_sum[tid] = before + incl - mine;
  __syncthreads();

  // Waits of a warp and of one lane.
  auto wait_warp = [&](uint32_t bar, uint32_t parity) { return mbar_wait_warp(bar, parity, a.err, a.polls); };
  auto wait_lane = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait_bounded(bar, parity, a.err, a.polls * kPollNs);
  };
  // Waits for the CTA's n-th item, a whole warp together; false past the last one.
  auto item = [&](int n, PaItem& it) {
    if (!wait_warp(smem_u32(next_full), n & 1)) {
      *s_bad = 1;
      return false;
    }
    it = *s_item;
    __syncwarp();
    if (lane == 0 && warp != kPaProd) mbar_arrive(next_empty);
    return it.t0 >= 0;
  };

  PaItem it;
  if (warp >= kPaProd) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kPaProd) {
      // ============================ TMA producer ==============================
      if (lane == 0) {
        prefetch_tmap(&maps.q);
        prefetch_tmap(&maps.k);
        prefetch_tmap(&maps.v);
      }
      const uint32_t q_bytes = static_cast<uint32_t>(C::SL * group * tpt * 128);
      int u = 0, qn[2] = {0, 0};
#pragma unroll 1
      for (int n = 0; item(n, it); ++n) {
        const int blocks = max(it.n[0], it.n[1]);
        if (lane == 0 && !*s_bad) {
          for (int i = 0; i < 2; ++i) {
            if (it.n[i] <= 0) continue;
            if (qn[i] > 0 && !wait_lane(&q_empty[i], (qn[i] - 1) & 1)) *s_bad = 1;
            ++qn[i];
            mbar_arrive_expect_tx(&q_full[i], q_bytes);
            for (int sl = 0; sl < C::SL; ++sl)
              tma_load_3d(tiles + i * C::TILE + sl * C::SLICE, &maps.q, sl * 64, it.kvh * group, it.s.q0 + it.t0 + i * tpt,
                          &q_full[i]);
          }
#pragma unroll 1
          for (int j = 0; j < 2 * blocks && !*s_bad; ++j, ++u) {
            const int st = u % S;
            if (u >= S && !wait_lane(&kv_empty[st], ((u / S) - 1) & 1)) {
              *s_bad = 1;
              break;
            }
            mbar_arrive_expect_tx(&kv_full[st], C::TILE);
            for (int sl = 0; sl < C::SL; ++sl)
              tma_load_3d(ring + st * C::TILE + sl * C::SLICE, j & 1 ? &maps.v : &maps.k, sl * 64, it.kvh,
                          it.s.k0 + (j >> 1) * kPaKeys, &kv_full[st]);
          }
        }
        if (lane == 0) mbar_arrive(next_empty);
        __syncwarp();
      }
      if (lane == 0) {  // copies in flight land before the CTA leaves, also where a wait ran out
        for (int i = max(u - S, 0); i < u; ++i) mbar_wait_bounded(&kv_full[i % S], (i / S) & 1, a.err);
        for (int i = 0; i < 2; ++i)
          if (qn[i] > 0) mbar_wait_bounded(&q_full[i], (qn[i] - 1) & 1, a.err);
      }
    } else if (warp < kPaMma + 2) {
      // ==================== MMA issuer of tile i ============================
      // Runs converged and issues from one lane; descriptors are sums of
      // precomputed halves, so little stands between two products (with whole
      // descriptors built for each, one came every 130-170 cycles, not 65).
      constexpr uint32_t kAb = E::is_bf16 ? 1u : 0u;
      constexpr uint32_t id_s = (1u << 4) | (kAb << 7) | (kAb << 10) | ((kPaKeys >> 3) << 17) | ((kPaRows >> 4) << 24);
      constexpr uint32_t id_o = (1u << 4) | (kAb << 7) | (kAb << 10) | ((DP >> 3) << 17) | ((kPaRows >> 4) << 24) | kUmmaBMajorN;
      // descriptor halves (see umma_desc): K-major Q and K tiles; V as it lies,
      // its dimensions contiguous, SLICE bytes between groups of 64 of them
      constexpr uint32_t hi_d = (1024u >> 4) | (1u << 14) | (2u << 29), lo_k = 1u << 16;
      constexpr uint32_t lo_v = static_cast<uint32_t>(C::SLICE >> 4) << 16;
      const uint32_t tm = __shfl_sync(~0u, tbase, 0);
      const uint32_t q_base = __shfl_sync(~0u, smem_u32(tiles) >> 4, 0), kv_base = q_base + 2 * (C::TILE >> 4);
      const uint32_t bars = __shfl_sync(~0u, smem_u32(smem), 0);
      auto bar = [&](const uint64_t* p) { return bars + static_cast<uint32_t>(p - kv_full) * 8; };
      const int i = __shfl_sync(~0u, warp - kPaMma, 0);
      const uint32_t ts = tm + i * kPaKeys, to = tm + C::COL_O + i * DP;
      const uint32_t q_lo = (q_base + i * (C::TILE >> 4)) | lo_k;
      uint32_t st = 0, ph = 0;  // ring position of the next block
      uint32_t q_par = 0, p_par = 0, o_par = 1, t_par = i ? 0 : 1;
      bool ok = true;
      auto wait = [&](uint32_t at, uint32_t parity) { ok = ok && wait_warp(at, parity); };
      auto next = [&] {
        if (++st == S) {
          st = 0;
          ph ^= 1;
        }
      };
#pragma unroll 1
      for (int n = 0; ok && item(n, it); ++n) {
        const int mine = __shfl_sync(~0u, i ? it.n[1] : it.n[0], 0);
        const int blocks = __shfl_sync(~0u, max(it.n[0], it.n[1]), 0);
        // step j: O_i += P_i(j - 1) V(j - 1), then S_i(j) = Q_i K(j)^T
        uint32_t v_st = 0;
#pragma unroll 1
        for (int j = 0; j <= blocks && blocks > 0 && ok; ++j) {
          if (j > 0) {
            v_st = st;
            wait(bar(kv_full) + 8 * st, ph);  // V(j - 1)
            next();
          }
          const uint32_t k_st = st;
          if (j < blocks) {
            wait(bar(kv_full) + 8 * st, ph);  // K(j)
            next();
          }
          const bool pv = j > 0 && j <= mine, qk = j < mine;
          if (j == 0 && qk) {
            wait(bar(q_full) + 8 * i, q_par);
            q_par ^= 1;
          }
          if (pv) {
            if (j == 1) {  // the tile's previous output was read (the first time: nothing to wait for)
              wait(bar(o_free) + 8 * i, o_par);
              o_par ^= 1;
            }
          }
          const uint32_t v_lo = (kv_base + v_st * (C::TILE >> 4)) | lo_v, k_lo = (kv_base + k_st * (C::TILE >> 4)) | lo_k;
          auto weighted = [&](int h) {  // O_i += P_i V for half of the keys
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma_f16_ts_lo(to, ts + h * 32 + ks * 8, v_lo + h * 512 + ks * 128, hi_d, id_o, ks + h > 0 || j > 1 ? 1u : 0u);
          };
          if (pv) {
            wait(bar(p_full) + 16 * i, p_par);
            tc_fence_after();
            if (ok && elect_one()) weighted(0);
            __syncwarp();
          }
          wait(bar(turn) + 8 * i, t_par);
          t_par ^= 1;
          if (pv) {
            wait(bar(p_full) + 16 * i + 8, p_par);
            p_par ^= 1;
          }
          tc_fence_after();
          if (ok && elect_one()) {
            if (pv) {
              weighted(1);
              if (!qk) {
                umma_commit_at(bar(o_full) + 8 * i);
                mbar_arrive(turn + 1 - i);
              }
            }
            if (qk) {
#pragma unroll
              for (int ks = 0; ks < DP / 16; ++ks) {
                const uint32_t at = (ks >> 2) * (C::SLICE >> 4) + 2 * (ks & 3);
                umma_f16_lo(ts, q_lo + at, hi_d, k_lo + at, hi_d, id_s, ks > 0 ? 1u : 0u);
              }
              umma_commit_at(bar(s_full) + 8 * i);
              mbar_arrive(turn + 1 - i);
              if (j + 1 == mine) umma_commit_at(bar(q_empty) + 8 * i);
            }
            if (!pv && !qk) mbar_arrive(turn + 1 - i);
            if (j > 0) umma_commit_at(bar(kv_empty) + 8 * v_st);
            if (j < blocks) umma_commit_at(bar(kv_empty) + 8 * k_st);
          }
          __syncwarp();
        }
      }
      if (!ok || *s_bad) {
        // a wait ran out: stop the others, and let the products in flight end
        // before TMEM is freed
        *s_bad = 1;
        __syncwarp();
        if (elect_one()) umma_commit_at(bar(drained) + 8 * i);
        mbar_wait_bounded(drained + i, 0, a.err, 1000000ull);
      }
    } else {
      // ============================ items ====================================
      // Fetched when every warp has begun the current one and its last load has
      // been issued.
      uint32_t par = 0;
#pragma unroll 1
      for (int n = 0, x = blockIdx.x; x >= 0; ++n) {
        if (lane == 0) {
          bool ok = n == 0 || wait_lane(next_empty, (n - 1) & 1);
          for (bool more = n > 0; ok && (more || x >= total); more = false) {
            mbar_arrive_expect_tx(taken, 16);
            cancel_cta(s_answer, taken);
            ok = mbar_wait_bounded(taken, par, a.err);
            par ^= 1;
            if (ok) x = cancelled_cta(s_answer);
            fence_proxy_async_smem();  // read before the next answer is written
          }
          if (!ok) {
            *s_bad = 1;
            x = -1;
          }
        }
        x = __shfl_sync(~0u, x, 0);
        it.t0 = -1;
        if (x >= 0) {
          int sl = 0;
#pragma unroll 1
          for (int i = lane; i < kPaThreads; i += 32)
            if (s_sum[i] <= x) sl = i;
          sl = __reduce_max_sync(~0u, sl);
          int b = sl * slice, y = x - s_sum[sl], pairs;
          while (true) {
            it.s = prompt_seq(a, b);
            pairs = pairs_of(it.s.nq);
            if (y < pairs * a.kv_heads) break;
            y -= pairs * a.kv_heads;
            ++b;
          }
          it.kvh = y % a.kv_heads;
          it.t0 = (pairs - 1 - y / a.kv_heads) * 2 * tpt;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int first = it.t0 + i * tpt, last = min(first + tpt, it.s.nq) - 1;
            const int end = first < it.s.nq ? min(max(last + it.s.nk - it.s.nq + 1, 0), it.s.nk) : 0;
            it.n[i] = (end + kPaKeys - 1) / kPaKeys;
          }
        }
        if (lane == 0) {
          *s_item = it;
          mbar_arrive(next_full);
        }
        __syncwarp();
      }
    }
  } else {
    // ============================ softmax, one thread per row ================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int i = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t ts = tbase + i * kPaKeys + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t to = tbase + C::COL_O + i * DP + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float sc = a.scale * kLog2e;
    int sn = 0, on = 0;
#pragma unroll 1
    for (int n = 0; item(n, it) && __all_sync(~0u, !*s_bad); ++n) {
      const int first = it.t0 + i * tpt;
      const int blocks = i ? it.n[1] : it.n[0];
      if (first >= it.s.nq) continue;
      const int token = first + row / group, head = it.kvh * group + row % group;
      const bool live = row < tpt * group && token < it.s.nq;
      const int shift = it.s.nk - it.s.nq + 1;
      const int lim = min(token + shift, it.s.nk);  // keys this row sees
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = 0; j < blocks; ++j) {
        if (!wait_warp(smem_u32(&s_full[i]), sn++ & 1)) {
          *s_bad = 1;
          break;
        }
        tc_fence_after();
        uint32_t x[4][32];
        tmem_ld32_nowait(ts, x[0]);
        tmem_ld32_nowait(ts + 32, x[1]);
        tmem_wait_ld32(x[0]);
        tmem_wait_ld32(x[1]);
        tmem_ld32_nowait(ts + 64, x[2]);
        tmem_ld32_nowait(ts + 96, x[3]);
        const int left = lim - j * kPaKeys;
        const bool masked = (j + 1) * kPaKeys > first + shift;  // some row of the tile sees less than the whole block
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto row_max = [&](uint32_t(&y)[32], int at) {
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (at + e >= left) y[e] = 0xff800000u;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            t[e / 2 % 4] = max3(t[e / 2 % 4], __uint_as_float(y[e]), __uint_as_float(y[e + 1]));
        };
        row_max(x[0], 0);
        row_max(x[1], 32);
        tmem_wait_ld32(x[2]);
        tmem_wait_ld32(x[3]);
        row_max(x[2], 64);
        row_max(x[3], 96);
        const float top = max3(max3(t[0], t[1], t[2]), t[3], -INFINITY);
        if (__any_sync(~0u, (top - m) * sc > kPaLazy<T> || (m == -INFINITY && top > m))) {
          const float mn = fmaxf(m, top);
          const float f = m == -INFINITY ? 0.f : ex2((m - mn) * sc);
          m = mn;
          l *= f;
          if (j > 0) {
#pragma unroll 1
            for (int q = 0; q < DP / 32; ++q) {
              uint32_t o[32];
              tmem_ld32_nowait(to + q * 32, o);
              tmem_wait_ld32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32_nowait(to + q * 32, o);
            }
          }
        }
        if (!(top < INFINITY)) l = NAN;  // NaN and infinite scores: the polynomial would lose them
        const float off = m == -INFINITY ? 0.f : fmaf(-m, sc, kWeightUp);
        const uint64_t sc2 = pack_f2(sc, sc), off2 = pack_f2(off, off);
        uint64_t sum[2] = {0, 0};
        // 64 keys at a time, so that the second product starts on the first half
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t p[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const uint32_t* y = &x[2 * h + e / 16][(2 * e) % 32];
            const uint64_t z = fma_f2(pack_f2(__uint_as_float(y[0]), __uint_as_float(y[1])), sc2, off2);
            float p0, p1;
            if (e % 8 < kPaFma) {
              ex2_fma2(z, p0, p1);
            } else {
              unpack_f2(z, p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
            }
            sum[e & 1] = add_f2(sum[e & 1], pack_f2(p0, p1));
            p[e] = E::pack2(p0, p1);
          }
          tmem_st32_nowait(ts + h * 32, p);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * i + h]);
        }
        float l0, l1;
        unpack_f2(add_f2(sum[0], sum[1]), l0, l1);
        l += l0 + l1;
      }
      // ---- the tile's output
      const int64_t at = static_cast<int64_t>(it.s.q0 + token) * a.heads + head;
      T* op = static_cast<T*>(a.out) + at * a.dim;
      bool odd = false;
      if (blocks > 0) {
        if (__any_sync(~0u, *s_bad) || !wait_warp(smem_u32(&o_full[i]), on++ & 1)) {
          *s_bad = 1;
          break;
        }
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int q = 0; q < DP / 32; ++q) {
          uint32_t o[32];
          tmem_ld32_nowait(to + q * 32, o);
          tmem_wait_ld32(o);
          if (q == DP / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[i]);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              y[e] = __uint_as_float(o[8 * w + e]) * inv;
              odd |= !(fabsf(y[e]) <= 3e38f);
            }
            if (live && q * 32 + w * 8 < a.dim)
              *reinterpret_cast<uint4*>(op + q * 32 + w * 8) =
                  make_uint4(E::pack2(y[0], y[1]), E::pack2(y[2], y[3]), E::pack2(y[4], y[5]), E::pack2(y[6], y[7]));
          }
        }
      } else if (live) {  // no row of the tile sees a key
#pragma unroll 1
        for (int d = 0; d < a.dim; d += 8) *reinterpret_cast<uint4*>(op + d) = make_uint4(0, 0, 0, 0);
      }
      if (a.lse && live) a.lse[at] = l == 0.f ? -INFINITY : (m * sc + (__log2f(l) - kWeightUp)) * kLn2;
      // (where l is NaN, one of the row's own scores is, and all of it is NaN)
      __syncwarp();  // a row's first stores come from another lane
      for (unsigned todo = __ballot_sync(~0u, odd && live && l == l); todo; todo &= todo - 1) {
        const int r = (warp & 3) * 32 + __ffs(todo) - 1;
        prompt_row<T>(a, it.s, first + r / group, it.kvh * group + r % group);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// A [tokens][heads][dim] tensor in boxes of 64 columns x box_heads x box_tokens.
bool prompt_map(CUtensorMap* m, int dtype, const void* base, int dim, int heads, int tokens, int64_t ts, int64_t hs,
                int box_heads, int box_tokens) {
  const uint64_t dims[3] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens)};
  const uint64_t strides[2] = {static_cast<uint64_t>(hs) * 2, static_cast<uint64_t>(ts) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(box_heads), static_cast<uint32_t>(box_tokens)};
  return encode_tiled_map(m, dtype, 3, base, dims, strides, box);
}

template <typename T, int DP>
cudaError_t launch_tiles(int dtype, PromptArgs a, cudaStream_t stream) {
  using C = PaCfg<DP>;
  a.polls = static_cast<int>(std::min<int64_t>(kPollsBase + int64_t{kPollsPerKey} * a.k_tokens, 0x7fffffff));
  static PerDevice ready;
  if (!ready.get([] {
        return cudaFuncSetAttribute(prompt_tile_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) ==
               cudaSuccess;
      }))
    return cudaGetLastError();
  const int group = a.heads / a.kv_heads, tpt = kPaRows / group;
  PaMaps maps;
  if (!prompt_map(&maps.q, dtype, a.q, a.dim, a.heads, a.q_tokens, a.q_ts, a.q_hs, group, tpt) ||
      !prompt_map(&maps.k, dtype, a.k, a.dim, a.kv_heads, a.k_tokens, a.k_ts, a.k_hs, 1, kPaKeys) ||
      !prompt_map(&maps.v, dtype, a.v, a.dim, a.kv_heads, a.k_tokens, a.v_ts, a.v_hs, 1, kPaKeys))
    return cudaErrorInvalidValue;
  // The items are not known here: their bound, for offsets that ascend (768 CTAs
  // too many cost nothing that was measured). Of offsets that do not, which
  // raise the error bit, items past the grid are left out.
  const int64_t ctas = (static_cast<int64_t>(a.q_tokens) / (2 * tpt) + a.num_seqs) * a.kv_heads;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  return launch_after(prompt_tile_kernel<T, DP>, dim3(static_cast<unsigned>(ctas)), kPaThreads, C::SMEM, stream, a.pdl, 1, a,
                      maps);
}

// The tiled kernel takes sequences of more than one tile of packed rows, and
// shorter ones over long contexts, whose keys are what counts. Measured, tiled
// against warp-level kernel (bf16, device time), 32 query / 8 kv heads of 128,
// 32 / 64 / 128 / 256 tokens (128 to 1024 rows):
//   16 sequences  9.6 / 12.0 / 18.6 / 34.9 us   6.1 / 13.2 / 29.6 / 77.6
//   64 sequences 22.0 / 30.7 / 53.2 / 109      20.8 / 42.9 / 103 / 285
//   4 sequences   8.7 / 11.1 / 11.4 / 13.7      4.9 /  5.9 / 10.4 / 26.9
//   1 sequence    8.6 / 11.1 / 11.1 / 12.8      4.9 /  5.8 /  8.3 / 13.5
// 12 heads of 64, 128 / 256 / 512 tokens: 64 sequences 24.8 / 37.8 / 86.1
// against 21.5 / 53.3 / 155, one 8.1 / 10.2 / 14.0 against 5.2 / 7.8 / 12.9. 16
// sequences of 4 tokens (16 rows) behind 500 / 2000 keys: 14.1 / 34.1 against
// 30.6 / 111; 64 of 4 tokens, 12 heads of 64, behind 500 / 1000: 46.1 / 77.8
// against 35.8 / 66.9. So the crossover is that of 16 and more sequences. The
// rule is off where the number of CTAs decides: 1 to 4 prompts of 129 to 500
// rows lose 1 to 5 us by it, short contexts of 1000 keys without grouped heads a
// sixth, and a few tokens of grouped heads behind 500 keys take twice as long as
// in the other kernel. The tiled kernel needs strides that a tensor map can
// express, and a positive scale, because its maxima are of unscaled scores.
constexpr int64_t kTileRows = 128, kTileKeys = 1024;

bool use_tiles(const PromptArgs& a) {
  const int group = a.heads / a.kv_heads;
  const int64_t rows = static_cast<int64_t>(a.max_q) * group;
  const int64_t most = int64_t{1} << 38;
  auto ok = [&](int64_t s) { return s > 0 && s < most; };
  return (rows > kTileRows || a.k_tokens >= kTileKeys * a.num_seqs) && group <= kPaRows && a.k_tokens > 0 &&
         a.scale > 0.f && a.scale < 1e30f && ok(a.q_ts) && ok(a.q_hs) && ok(a.k_ts) && ok(a.k_hs) && ok(a.v_ts) && ok(a.v_hs);
}

template <typename T>
cudaError_t launch_prompt(int dtype, const PromptArgs& a, cudaStream_t stream) {
  if (use_tiles(a))
    return a.dim <= 64 ? launch_tiles<T, 64>(dtype, a, stream) : launch_tiles<T, 128>(dtype, a, stream);
  const int64_t rows = static_cast<int64_t>(a.max_q) * (a.heads / a.kv_heads);
  if (a.dim <= 64)
    return rows <= 16 ? launch_small<T, 64, 1>(a, stream) : launch_small<T, 64, 4>(a, stream);
  return rows <= 16 ? launch_small<T, 128, 1>(a, stream) : launch_small<T, 128, 4>(a, stream);
}

}  // namespace

cudaError_t launch_prompt_attention(int dtype, const PromptArgs& a, cudaStream_t stream) {
  return dtype == 1 ? launch_prompt<__nv_bfloat16>(dtype, a, stream)
                    : launch_prompt<__half>(dtype, a, stream);
}

}  // namespace wp
