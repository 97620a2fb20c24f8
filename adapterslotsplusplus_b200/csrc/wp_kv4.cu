// wp_kv4.cu -- a paged key/value cache held in 4 bits: appending tokens,
// reading a range back in 16 bits, and attention over it for one or a few
// query tokens per sequence.
//
// Format. Every token and kv head has one (scale, zero) pair for K and one for
// V: zero = min, scale = round16((max - min) / 15), code = rint((x - zero) /
// scale) in 0..15, and a code stands for zero + scale * code. Scale and zero
// are kept in the cache's own 16-bit type, so a bf16 cache has bf16's range;
// the codes are computed with the rounded scale, so its rounding only moves
// the steps (by 2^-9 of a step in bf16), never the code's nearest value. The
// arithmetic is fp32 in this order everywhere, so codes are reproducible.
//
// Layout (declared with wp_kv4_append in include/wp_api.h). The unit is a tile
// of 16 tokens of one kv head, contiguous in memory: K's codes, V's codes,
// K's and V's (scale, zero) pairs. Both code blocks are laid out as operand
// fragments of mma.sync m16n8k16, so the attention kernel reads them from
// shared memory with 16-byte loads that no two lanes conflict on, and turns 8
// codes into four operand registers with four ANDs and one shift: a nibble in
// bits 0-3 of an fp16 is the subnormal code * 2^-24 and in bits 4-7 code *
// 2^-20, exact operands both, so the codes are never converted.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "wp_device.cuh"
#include "wp_internal.h"
#include "wp_once.h"

namespace wp {
namespace {

// ---- format -----------------------------------------------------------------

// Byte of V's code block that holds dimensions (64 h + 16 m + g, + 8) of token t.
__device__ __forceinline__ int v_byte(int h, int m, int g, int t) {
  return (((h * 8 + g) * 4 + ((t & 7) >> 1)) * 4 + m) * 4 + ((t & 1) << 1) + (t >> 3);
}

template <typename T>
__device__ __forceinline__ float to_float(uint32_t bits16) {
  const unsigned short u = static_cast<unsigned short>(bits16);
  return Elem<T>::to_f(*reinterpret_cast<const T*>(&u));
}

// x / group for the packed rows of a kv head (x * group < 2^32), without a division.
struct GroupDiv {
  uint32_t group, magic;
  __device__ __forceinline__ explicit GroupDiv(int g) : group(g), magic(g == 1 ? 0 : 0xffffffffu / g + 1) {}
  __device__ __forceinline__ int div(int x) const { return group == 1 ? x : static_cast<int>(__umulhi(x, magic)); }
};

struct Seq {
  int first;  // packed row of its first token
  int n;  // tokens of this call
  int len;  // tokens in the cache, those included
};

// A sequence's place, with every value forced into the range of its arrays:
// lengths past the table and rows past the packed tensor raise the error bit
// and are dropped.
__device__ __forceinline__ Seq load_seq(const Kv4Args& a, int b) {
  Seq s;
  int lo = b, hi = b + 1;
  if (a.cu) {
    lo = __ldg(a.cu + b);
    hi = __ldg(a.cu + b + 1);
  }
  s.len = __ldg(a.lens + b);
  const long long cap = static_cast<long long>(a.table_ld) * a.page_tiles * kKv4Tile;
  if (lo < 0 || hi > a.tokens || hi < lo || s.len < 0 || s.len > cap) {
    if (a.err) atomicOr(a.err, kErrBadSegment);
    lo = min(max(lo, 0), a.tokens);
    hi = min(max(hi, lo), a.tokens);
    s.len = static_cast<int>(min(static_cast<long long>(max(s.len, 0)), cap));
  }
  s.first = lo;
  s.n = hi - lo;
  return s;
}

// Address of tile `tile` (16 tokens) of sequence b, head h; null (and the
// error bit) for a page number outside the cache.
__device__ __forceinline__ uint8_t* tile_ptr(const Kv4Args& a, int b, int h, int tile, int tile_bytes) {
  const int slot = tile / a.page_tiles;
  const int page = __ldg(a.table + static_cast<int64_t>(b) * a.table_ld + slot);
  if (page < 0 || page >= a.num_pages) {
    if (a.err) atomicOr(a.err, kErrBadSegment);
    return nullptr;
  }
  return a.pages + ((static_cast<int64_t>(page) * a.kv_heads + h) * a.page_tiles + (tile - slot * a.page_tiles)) * tile_bytes;
}

// ---- append and read ----------------------------------------------------------
//
// One CTA per (sequence, head) and tile of 16 tokens. A lane has 16 dimensions
// of one token of K or V: 32 contiguous bytes in 16 bits, 8 bytes of codes (of
// V, whole bytes: dimensions g and g + 8 share one), and the minimum and
// maximum of a row need log2(D / 16) exchanges. Bound by memory: 4 D bytes of K
// and V in, D + 8 out (append), or the reverse. A tile whose 16 tokens are all
// new leaves shared memory in 16-byte stores; in a tile that is shared with
// older tokens only the new tokens' bytes are written (a token owns whole bytes
// of both blocks). 8 heads of 128, fp16: 512 new tokens of each of 8 sequences
// appended in 13 us, 12000 tokens read back in 18 (59% of the copy rate; the
// latency of one tile after another).

constexpr int kMoveThreads = 128;

// The nearest code to d / step, as rint of the correctly rounded quotient: the
// product with the reciprocal (inv) is within 2^-17 of it and decides unless it
// is about half-way between two codes.
__device__ __forceinline__ uint32_t code_of(float d, float step, float inv) {
  float r = d * inv, k = rintf(r);
  if (!(fabsf(r - k) <= 0.4999f)) k = step > 0.f ? rintf(__fdiv_rn(d, step)) : 0.f;
  return static_cast<uint32_t>(fminf(fmaxf(k, 0.f), 15.f));
}

// NaN if either is: a row with a NaN gets a NaN zero and scale, so that all its
// values are NaN and no step after it looks healthy.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_append_kernel(Kv4Args a, int per_seq) {
  pdl_wait_prior();
  constexpr int TB = kv4_tile_bytes(D);
  constexpr int PER = D / 16;  // lanes per row
  constexpr int RW = 32 / PER;  // rows per warp; even warps take K, odd ones V
  constexpr int N = kKv4Tile / (kMoveThreads / 64 * RW);
  __shared__ __align__(16) uint8_t tile[TB];
  const int b = blockIdx.x / per_seq, h = blockIdx.y;
  const int warp = threadIdx.x >> 5, part = threadIdx.x % PER, is_v = warp & 1;
  const int tok0 = (warp >> 1) * RW + (threadIdx.x & 31) / PER;  // tokens tok0 + kMoveThreads / 64 * RW * n
  const Seq s = load_seq(a, b);
  if (s.n > s.len) {  // more new tokens than the sequence has
    if (threadIdx.x == 0 && a.err) atomicOr(a.err, kErrBadSegment);
    return;
  }
  const int start = s.len - s.n;
  const int t_end = (s.len + kKv4Tile - 1) / kKv4Tile;
  for (int t = start / kKv4Tile + static_cast<int>(blockIdx.x) % per_seq; t < t_end; t += per_seq) {
    const int lo = max(start - t * kKv4Tile, 0), hi = min(s.len - t * kKv4Tile, kKv4Tile);
    uint8_t* dst = tile_ptr(a, b, h, t, TB);
    if (dst == nullptr) continue;  // the same for the whole CTA
    uint4 w[N][2];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int tok = tok0 + kMoveThreads / 64 * RW * n;
      if (tok >= lo && tok < hi) {
        const int64_t row = s.first + (t * kKv4Tile + tok - start);
        const T* src = static_cast<const T*>(is_v ? a.v : a.k) + row * (is_v ? a.v_ts : a.k_ts) +
                       static_cast<int64_t>(h) * (is_v ? a.v_hs : a.k_hs) + part * 16;
        w[n][0] = __ldg(reinterpret_cast<const uint4*>(src));
        w[n][1] = __ldg(reinterpret_cast<const uint4*>(src) + 1);
      } else {
        w[n][0] = w[n][1] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int tok = tok0 + kMoveThreads / 64 * RW * n;
      if (__all_sync(~0u, tok < lo || tok >= hi)) continue;
      float x[16];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t u[4] = {w[n][i].x, w[n][i].y, w[n][i].z, w[n][i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = Elem<T>::unpack2(u[j]);
          x[8 * i + 2 * j] = f.x;
          x[8 * i + 2 * j + 1] = f.y;
        }
      }
      float mn = x[0], mx = x[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mn = min_nan(mn, x[i]), mx = max_nan(mx, x[i]);
#pragma unroll
      for (int o = PER / 2; o; o >>= 1) {
        mn = min_nan(mn, __shfl_xor_sync(~0u, mn, o));
        mx = max_nan(mx, __shfl_xor_sync(~0u, mx, o));
      }
      const uint32_t pair = Elem<T>::pack2(__fmul_rn(__fsub_rn(mx, mn), 1.0f / 15.0f), mn);
      const float step = Elem<T>::unpack2(pair).x, inv = __frcp_rn(step);
      if (tok < lo || tok >= hi) continue;
      if (!is_v) {
        uint32_t c[2] = {0, 0};  // one nibble per dimension
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i >> 3] |= code_of(__fsub_rn(x[i], mn), step, inv) << (4 * (i & 7));
        *reinterpret_cast<uint2*>(tile + tok * (D / 2) + part * 8) = make_uint2(c[0], c[1]);
      } else {
#pragma unroll
        for (int g = 0; g < 8; ++g)
          tile[8 * D + v_byte(part >> 2, part & 3, g, tok)] = static_cast<uint8_t>(
              code_of(__fsub_rn(x[g], mn), step, inv) | (code_of(__fsub_rn(x[g + 8], mn), step, inv) << 4));
      }
      if (part == 0) *reinterpret_cast<uint32_t*>(tile + 16 * D + is_v * 64 + tok * 4) = pair;
    }
    __syncthreads();
    if (lo == 0 && hi == kKv4Tile) {
      for (int i = threadIdx.x; i < TB / 16; i += kMoveThreads)
        reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(tile)[i];
    } else {
      const int nt = hi - lo;
      for (int i = threadIdx.x; i < nt * (D / 8); i += kMoveThreads) {  // K rows, 4 bytes each
        const int o = lo * (D / 2) + i * 4;
        *reinterpret_cast<uint32_t*>(dst + o) = *reinterpret_cast<const uint32_t*>(tile + o);
      }
      for (int i = threadIdx.x; i < nt * 2; i += kMoveThreads) {  // scales
        const int o = 16 * D + (i & 1) * 64 + (lo + (i >> 1)) * 4;
        *reinterpret_cast<uint32_t*>(dst + o) = *reinterpret_cast<const uint32_t*>(tile + o);
      }
      for (int i = threadIdx.x; i < nt * (D / 2); i += kMoveThreads) {  // V: single bytes
        const int r = i % (D / 2), o = 8 * D + v_byte(r >> 5, r & 3, (r >> 2) & 7, lo + i / (D / 2));
        dst[o] = tile[o];
      }
    }
    __syncthreads();
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_read_kernel(Kv4Args a, int per_seq) {
  pdl_wait_prior();
  constexpr int TB = kv4_tile_bytes(D);
  constexpr int PER = D / 16;
  __shared__ __align__(16) uint8_t tile[TB];
  const int b = blockIdx.x / per_seq, h = blockIdx.y;
  const Seq s = load_seq(a, b);
  if (s.n > s.len) {
    if (threadIdx.x == 0 && a.err) atomicOr(a.err, kErrBadSegment);
    return;
  }
  const int start = s.len - s.n;
  const int t_end = (s.len + kKv4Tile - 1) / kKv4Tile;
  for (int t = start / kKv4Tile + static_cast<int>(blockIdx.x) % per_seq; t < t_end; t += per_seq) {
    const int lo = max(start - t * kKv4Tile, 0), hi = min(s.len - t * kKv4Tile, kKv4Tile);
    const uint8_t* src = tile_ptr(a, b, h, t, TB);
    if (src == nullptr) continue;
    for (int i = threadIdx.x; i < TB / 16; i += kMoveThreads)
      reinterpret_cast<uint4*>(tile)[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
    __syncthreads();
    // 16 dimensions of one token of K or V per thread and pass
    for (int i = threadIdx.x; i < 2 * kKv4Tile * PER; i += kMoveThreads) {
      const int part = i % PER, tok = (i / PER) & 15, is_v = i / (PER * kKv4Tile);
      if (tok < lo || tok >= hi) continue;
      const float2 sz = Elem<T>::unpack2(*reinterpret_cast<const uint32_t*>(tile + 16 * D + is_v * 64 + tok * 4));
      auto value = [&](uint32_t c) { return fmaf(sz.x, static_cast<float>(c & 15u), sz.y); };
      uint32_t w[8];  // the 16 values, in pairs
      if (!is_v) {
        const uint2 c = *reinterpret_cast<const uint2*>(tile + tok * (D / 2) + part * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t u = (j < 4 ? c.x : c.y) >> (8 * (j & 3));
          w[j] = Elem<T>::pack2(value(u), value(u >> 4));
        }
      } else {
        const uint8_t* v = tile + 8 * D + v_byte(part >> 2, part & 3, 0, tok);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u0 = v[128 * j], u1 = v[128 * j + 64];  // dimensions 2j, 2j + 1 (and + 8)
          w[j] = Elem<T>::pack2(value(u0), value(u1));
          w[4 + j] = Elem<T>::pack2(value(u0 >> 4), value(u1 >> 4));
        }
      }
      const int64_t row = s.first + (t * kKv4Tile + tok - start);
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(is_v ? a.v : a.k) + (row * a.kv_heads + h) * D + part * 16);
      dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
      dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
    __syncthreads();
  }
}

// ---- attention -----------------------------------------------------------------
//
// For a query row q (one head of one token) over the visible tokens t:
//   s_t = scale * (zeroK_t * sum(q) + scaleK_t * q . codeK_t)
//   out = (sum_t p_t midV_t + sum_t w_t codeV_t - 7.5 sum_t w_t) / sum_t p_t,
//   p_t = 2^(s_t log2 e - m), w_t = p_t scaleV_t, midV_t = zeroV_t + 7.5 scaleV_t
// so both products take the codes as they are; scales and zeros are applied to
// their results in fp32. w_t is rounded to fp16 on its way into the tensor
// core; the sum that is subtracted is that of the rounded weights (one more
// row of ones in the product), so the rounding acts on codes centred around 0,
// as it would on V itself: without it the error is three times as large.
//
// What bounds it: D + 8 bytes per token and kv head from HBM, and, close
// behind, the instructions that feed the tensor cores (0.6 per code). Each
// warp is on its own: it walks a contiguous range of 64-token chunks of
// (sequence, kv head, block of query rows), the same number of chunks for
// every warp of the grid, with a private ring of bulk copies, so no warp waits
// for another. A query row block is the 8 NT rows (head in group, query token)
// that share a kv head. Sequences that span several warps leave partial rows,
// which kv4_combine_kernel adds in order (no atomics: results do not depend on
// timing). 32 contexts of 4096-32768 tokens, 32 query / 8 kv heads of 128: 92
// us (70% of the copy rate), 1090 instructions per chunk, the schedulers
// issuing in 56% of the cycles.
//
// Sums are not divided by the weights' before the end, and a weight reaches 2^8
// (the reference is raised lazily): V beyond 2^119 / tokens, which only bf16
// holds, may overflow them.

// Twelve warps of 168 registers hide the latencies of the short dependent steps
// (softmax, scales) that eight did not (two per scheduler issued in 47% of the
// cycles); 16 query rows need 255 registers and stay at eight.
template <int D, int NT>
struct AttnCfg {
  static constexpr int WARPS = NT == 1 ? 12 : 8;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int TB = kv4_tile_bytes(D);
  static constexpr int TILES = kKv4Chunk / kKv4Tile;  // tiles of one chunk
  static constexpr int STAGE = TILES * TB;
  static constexpr int S = (NT == 1 ? 2 : 3) * (D == 64 ? 2 : 1);  // stages of a warp's ring
  static constexpr int BARS = 1024;  // mbarriers
  static constexpr int HEAD = BARS + THREADS * 4;  // and the block's prefix sums (see the kernel)
  static constexpr int SMEM = HEAD + WARPS * S * STAGE;
  static_assert(SMEM <= 232448 && HEAD % 16 == 0, "shared memory budget");
  static constexpr int ROWS = 8 * NT;
};

// Position in the order (sequence, kv head, row block, chunk).
struct Cursor {
  int b, h, rb, t;
  int chunks;  // of the sequence (at least 1, so that an empty one writes its zeros)
  int blocks;  // row blocks of the sequence (0: no query tokens)
  Seq s;

  __device__ __forceinline__ void load(const Kv4Args& a, int group, int rows) {
    s = load_seq(a, b);
    chunks = max((s.len + kKv4Chunk - 1) / kKv4Chunk, 1);
    blocks = (s.n * group + rows - 1) / rows;
  }
  __device__ __forceinline__ void next(const Kv4Args& a, int group, int rows) {
    if (++t < chunks) return;
    t = 0;
    if (++rb < blocks) return;
    rb = 0;
    if (++h < a.kv_heads) return;
    h = 0;
    do {
      if (++b >= a.num_seqs) return;
      load(a, group, rows);
    } while (blocks == 0);
  }
};

// Range of warp w of n over `total` chunks starts here; n <= total.
__device__ __forceinline__ long long range_start(long long total, int w, int n) { return total * w / n; }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(AttnCfg<D, NT>::THREADS, 1) kv4_attention_kernel(const Kv4Args a) {
  using C = AttnCfg<D, NT>;
  constexpr int kAttnWarps = C::WARPS, kAttnThreads = C::THREADS;
  using E = Elem<T>;
  constexpr int MT = D / 16;  // 16-dimension tiles of the output
  constexpr int KW = D / 32;  // code words (8 dimensions) of a lane's K row; two k16 steps each
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);  // [warps][S]
  int* s_sum = reinterpret_cast<int*>(smem + C::BARS);  // chunks of the sequences of thread i's slice, then their prefix
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int group = a.heads / a.kv_heads;
  const GroupDiv by(group);

  if (lane < C::S) mbar_init(&bars[warp * C::S + lane], 1);
  fence_mbar_init();
  pdl_wait_prior();

  // ---- the call's chunks: each thread counts a contiguous slice of sequences
  const int slice = (a.num_seqs + kAttnThreads - 1) / kAttnThreads;
  auto seq_chunks = [&](int b) {
    Cursor q;
    q.b = b;
    q.load(a, group, C::ROWS);
    return q.chunks * q.blocks * a.kv_heads;
  };
  int mine = 0;
  for (int b = tid * slice; b < min((tid + 1) * slice, a.num_seqs); ++b) mine += seq_chunks(b);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += v;
  }
  __shared__ int s_warp[kAttnWarps];
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  s_sum[tid] = before + incl - mine;
  __syncthreads();
  pdl_launch_dependents();

  const int wg = blockIdx.x * kAttnWarps + warp;
  const int warps = min(static_cast<int>(gridDim.x) * kAttnWarps, total);
  if (lane == 0) a.part_desc[2 * wg] = make_int4(0, 0, 0, 0);
  if (wg >= warps) return;
  const long long w0 = range_start(total, wg, warps), w1 = range_start(total, wg + 1, warps);

  // ---- where the range starts
  int sl = 0;  // last slice that starts at or before w0 and is not empty from there
  for (int i = lane; i < kAttnThreads; i += 32)
    if (s_sum[i] <= w0) sl = i;
  sl = __reduce_max_sync(~0u, sl);
  Cursor con;
  con.b = sl * slice;
  con.h = con.rb = con.t = 0;
  long long at = s_sum[sl];  // chunk index of the start of sequence con.b
  while (true) {
    con.load(a, group, C::ROWS);
    const int n = con.chunks * con.blocks * a.kv_heads;
    if (w0 < at + n) break;
    at += n;
    ++con.b;
  }
  {
    int r = static_cast<int>(w0 - at);
    con.h = r / (con.blocks * con.chunks);
    r -= con.h * con.blocks * con.chunks;
    con.rb = r / con.chunks;
    con.t = r - con.rb * con.chunks;
  }

  // ---- the ring
  uint8_t* ring = smem + C::HEAD + warp * C::S * C::STAGE;
  uint64_t* bar = bars + warp * C::S;
  const int count = static_cast<int>(w1 - w0);
  Cursor pro = con;
  int issued = 0;
  const uint8_t* src = nullptr;  // lane i < TILES: tile i of the next chunk to issue
  int slot = 0, off = 0;  // its page slot and the tile's place in the page
  auto find = [&](bool jump) {
    const int tile = pro.t * C::TILES + lane;
    if (jump) {
      slot = tile / a.page_tiles;
      off = tile - slot * a.page_tiles;
    } else {
      for (off += C::TILES; off >= a.page_tiles; off -= a.page_tiles) ++slot;
    }
    src = nullptr;
    if (lane < C::TILES && tile * kKv4Tile < pro.s.len) {
      const int page = __ldg(a.table + static_cast<int64_t>(pro.b) * a.table_ld + slot);
      src = a.pages;  // a bad page number: any readable tile, and the error bit
      if (page >= 0 && page < a.num_pages)
        src += ((static_cast<int64_t>(page) * a.kv_heads + pro.h) * a.page_tiles + off) * C::TB;
      else if (a.err)
        atomicOr(a.err, kErrBadSegment);
    }
    if (jump && lane < C::ROWS) {  // the segment's query rows will be wanted soon
      const int r = pro.rb * C::ROWS + lane;
      if (r < pro.s.n * group) {
        const T* qp = static_cast<const T*>(a.q) + static_cast<int64_t>(pro.s.first + by.div(r)) * a.q_ts +
                      static_cast<int64_t>(pro.h * group + r - by.div(r) * group) * a.q_hs;
        asm volatile("prefetch.global.L1 [%0];" ::"l"(qp));
        if (D == 128) asm volatile("prefetch.global.L1 [%0];" ::"l"(qp + 64));
      }
    }
  };
  auto issue = [&] {  // src was found one chunk earlier, so its page number has arrived
    const int st = issued % C::S;
    const unsigned have = __ballot_sync(~0u, src != nullptr);
    if (lane == 0) mbar_arrive_expect_tx(&bar[st], __popc(have) * C::TB);
    __syncwarp();
    if (src != nullptr) bulk_g2s(ring + st * C::STAGE + lane * C::TB, src, C::TB, &bar[st]);
    if (++issued < count) {
      pro.next(a, group, C::ROWS);
      find(pro.t == 0);
    }
  };
  find(true);
  for (int i = 0; i < C::S - 1 && issued < count; ++i) issue();

  // ---- the range, segment by segment
  uint32_t qf[NT][KW][4];  // B fragments of the query rows: k16 steps (2i, 2i+1) of code word i
  float qa[NT][2], qb[NT][2];  // rows 2c, 2c+1 of each n-tile: score = zero * qa + scale * acc * qb
  int lim[NT][2];  // tokens that row may see
  float acc[MT][NT][4];  // out^T: dimensions (g, g + 8) x rows (2c, 2c + 1)
  float sumw[NT][4];  // sum of the rounded weights of rows (2c, 2c + 1), times 2^10 of acc's unit ([2], [3] are copies)
  float m[NT][2], l[NT][2], pz[NT][2];
  // p * scaleV enters the tensor core in fp16, rounded once, as p * scaleV /
  // 2^e * 2^14 with 2^(e + 1) above the row's largest such weight: at most
  // 2^15, and a normal number down to 2^-28 of the largest
  float wtop[NT][2];  // a bound of the weights so far, relative to the present m
  uint32_t wexp[NT][2];  // biased exponent of 2^e, in place
  bool ok = true;
  long long seg0 = 0;  // chunk index of the segment's first chunk
  for (int it = 0; it < count; ++it) {
    const bool first = it == 0 || con.t == 0;
    if (first) {
      seg0 = w0 + it - con.t;
      // query rows as fp16 B fragments. A row is scaled by a power of two so
      // that its largest element is in [2^14, 2^15): bf16's 8 bits and fp16's
      // 11 stay exact down to 2^-28 of the row's maximum.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = con.rb * C::ROWS + nt * 8 + g;
        uint4 w[KW];
        float mx = 0.f, sum = 0.f;
        const bool row = r < con.s.n * group;
        const T* qp = static_cast<const T*>(a.q) + static_cast<int64_t>(con.s.first + by.div(r)) * a.q_ts +
                      static_cast<int64_t>(con.h * group + r - by.div(r) * group) * a.q_hs + c * (D / 4);
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          w[i] = row ? __ldg(reinterpret_cast<const uint4*>(qp) + i) : make_uint4(0, 0, 0, 0);
          const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = E::unpack2(u[j]);
            mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
            sum += f.x + f.y;
          }
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
          sum += __shfl_xor_sync(~0u, sum, o);
        }
        const int e = min(max(static_cast<int>(__float_as_uint(mx) >> 23), 40), 240);  // biased exponent of the maximum
        const float down = __uint_as_float(static_cast<uint32_t>(254 + 14 - e) << 23);  // 2^(14 - (e - 127))
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const float2 d01 = E::unpack2(w[i].x), d23 = E::unpack2(w[i].y), d45 = E::unpack2(w[i].z),
                       d67 = E::unpack2(w[i].w);
          const float lo = down, hi = down * 0.0625f;  // the odd dimensions' codes enter times 16
          qf[nt][i][0] = Elem<__half>::pack2(d01.x * lo, d45.x * lo);
          qf[nt][i][1] = Elem<__half>::pack2(d23.x * lo, d67.x * lo);
          qf[nt][i][2] = Elem<__half>::pack2(d01.y * hi, d45.y * hi);
          qf[nt][i][3] = Elem<__half>::pack2(d23.y * hi, d67.y * hi);
        }
        const float sc = a.scale * kLog2e;
        const float up = sc * __uint_as_float(static_cast<uint32_t>(e - 14 + 24) << 23);  // sc * 2^(e - 127 - 14 + 24)
        sum *= sc;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          qa[nt][j] = __shfl_sync(~0u, sum, (2 * c + j) * 4);
          qb[nt][j] = __shfl_sync(~0u, up, (2 * c + j) * 4);
          const int rr = con.rb * C::ROWS + nt * 8 + 2 * c + j;
          lim[nt][j] = min(con.s.len - (con.s.n - 1) + by.div(rr), con.s.len);
          m[nt][j] = -INFINITY;
          l[nt][j] = pz[nt][j] = wtop[nt][j] = 0.f;
          wexp[nt][j] = 40u << 23;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[mt][nt][j] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sumw[nt][j] = 0.f;
      }
    }

    const int st = it % C::S;
    // once a wait has run out (in any lane: the whole warp goes on alike),
    // nothing is loaded any more
    if (ok && issued < count) issue();
    if (ok) ok = __all_sync(~0u, mbar_wait_bounded(&bar[st], (it / C::S) & 1, a.err));
    const uint8_t* sp = ring + st * C::STAGE;
    const int left = con.s.len - con.t * kKv4Chunk;  // tokens from here on
    if (ok && left > 0) {
      const bool masked = con.t * kKv4Chunk + kKv4Chunk > con.s.len - con.s.n + 1;
      // ---- scores^T [16 tokens x 8 rows] of four tiles
      float s[C::TILES][NT][4];
      float top[NT][2];
      float2 vs[C::TILES][2];  // (scale, middle) of V for tokens g, g + 8
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
      for (int ti = 0; ti < C::TILES; ++ti) {
        if (ti * kKv4Tile >= left) {  // no token of the tile is left
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[ti][nt][j] = -INFINITY;
          vs[ti][0] = vs[ti][1] = make_float2(0.f, 0.f);
          continue;
        }
        const uint8_t* tp = sp + ti * C::TB;
        uint32_t k0[KW], k1[KW];
        if constexpr (KW == 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(tp + g * 64 + c * 16);
          const uint4 v = *reinterpret_cast<const uint4*>(tp + 512 + g * 64 + c * 16);
          k0[0] = u.x, k0[1] = u.y, k0[2] = u.z, k0[3] = u.w;
          k1[0] = v.x, k1[1] = v.y, k1[2] = v.z, k1[3] = v.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(tp + g * 32 + c * 8);
          const uint2 v = *reinterpret_cast<const uint2*>(tp + 256 + g * 32 + c * 8);
          k0[0] = u.x, k0[1] = u.y, k1[0] = v.x, k1[1] = v.y;
        }
        float s2[NT][4];  // a second accumulator: half as long a chain of dependent products
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[ti][nt][j] = s2[nt][j] = 0.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint32_t x0 = k0[i] >> 8, x1 = k1[i] >> 8;
          const uint32_t fa[4] = {k0[i] & 0x000f000fu, k1[i] & 0x000f000fu, x0 & 0x000f000fu, x1 & 0x000f000fu};
          const uint32_t fb[4] = {k0[i] & 0x00f000f0u, k1[i] & 0x00f000f0u, x0 & 0x00f000f0u, x1 & 0x00f000f0u};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_k16<__half>(s[ti][nt], fa, qf[nt][i][0], qf[nt][i][1]);
            mma_k16<__half>(s2[nt], fb, qf[nt][i][2], qf[nt][i][3]);
          }
        }
        const float2 kz0 = E::unpack2(*reinterpret_cast<const uint32_t*>(tp + 16 * D + g * 4));
        const float2 kz1 = E::unpack2(*reinterpret_cast<const uint32_t*>(tp + 16 * D + g * 4 + 32));
        vs[ti][0] = E::unpack2(*reinterpret_cast<const uint32_t*>(tp + 16 * D + 64 + g * 4));
        vs[ti][1] = E::unpack2(*reinterpret_cast<const uint32_t*>(tp + 16 * D + 64 + g * 4 + 32));
        vs[ti][0].y = fmaf(vs[ti][0].x, 7.5f, vs[ti][0].y);
        vs[ti][1].y = fmaf(vs[ti][1].x, 7.5f, vs[ti][1].y);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[ti][nt][j] = fmaf((s[ti][nt][j] + s2[nt][j]) * kz0.x, qb[nt][j], kz0.y * qa[nt][j]);
            s[ti][nt][2 + j] = fmaf((s[ti][nt][2 + j] + s2[nt][2 + j]) * kz1.x, qb[nt][j], kz1.y * qa[nt][j]);
          }
        if (masked) {
          // what a row must not see counts as minus infinity whatever the
          // cache holds there; a tile past the end was never loaded
          const int t0 = con.t * kKv4Chunk + ti * kKv4Tile + g;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (t0 >= lim[nt][j]) s[ti][nt][j] = -INFINITY;
              if (t0 + 8 >= lim[nt][j]) s[ti][nt][2 + j] = -INFINITY;
            }
          if (t0 >= con.s.len) vs[ti][0] = make_float2(0.f, 0.f);
          if (t0 + 8 >= con.s.len) vs[ti][1] = make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) top[nt][j] = fmaxf(top[nt][j], fmaxf(s[ti][nt][j], s[ti][nt][2 + j]));
      }
      // ---- the running maximum. It is only a reference, and raised when a
      // row's grows by more than 8 (log2 units): no exchange between lanes, and
      // no rescaling, in nearly all chunks.
      bool grew = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) grew |= top[nt][j] > m[nt][j] + 8.f;
      grew = __any_sync(~0u, grew);
      float f[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) f[nt][0] = f[nt][1] = 1.f;
      if (grew) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) top[nt][j] = fmaxf(top[nt][j], __shfl_xor_sync(~0u, top[nt][j], o));
            const float mn = fmaxf(m[nt][j], top[nt][j]);
            f[nt][j] = m[nt][j] == -INFINITY ? 0.f : ex2(m[nt][j] - mn);
            m[nt][j] = mn;
            l[nt][j] *= f[nt][j];
            pz[nt][j] *= f[nt][j];
          }
      }
      // ---- weights: p = 2^(s - m), s[][][] becomes p * scaleV
      bool move = grew;
      float big[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float base[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          base[j] = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
          big[nt][j] = 0.f;
        }
#pragma unroll
        for (int ti = 0; ti < C::TILES; ++ti) {
          if (ti * kKv4Tile >= left) break;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = ex2(s[ti][nt][j] - base[j & 1]);
            float w = p * vs[ti][j >> 1].x;
            if (masked && s[ti][nt][j] == -INFINITY) {  // 0 * infinity: an unseen token adds nothing
              w = 0.f;
            } else {
              pz[nt][j & 1] = fmaf(p, vs[ti][j >> 1].y, pz[nt][j & 1]);
            }
            l[nt][j & 1] += p;
            s[ti][nt][j] = w;
            big[nt][j & 1] = fmaxf(big[nt][j & 1], w);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) move |= big[nt][j] > 2.f * __uint_as_float(wexp[nt][j]);
      }
      if (__any_sync(~0u, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) big[nt][j] = fmaxf(big[nt][j], __shfl_xor_sync(~0u, big[nt][j], o));
            wtop[nt][j] = fmaxf(wtop[nt][j] * f[nt][j], big[nt][j]);
            const uint32_t e = min(max((__float_as_uint(wtop[nt][j]) & 0x7f800000u) + 0x00800000u, 40u << 23), 254u << 23);
            const int d = static_cast<int>(wexp[nt][j] >> 23) - static_cast<int>(e >> 23);  // 2^(old - new), in two factors
            const float up = __uint_as_float(static_cast<uint32_t>(127 + d / 2) << 23);
            const float r = f[nt][j] * up * __uint_as_float(static_cast<uint32_t>(127 + d - d / 2) << 23);
            wexp[nt][j] = e;
            wtop[nt][j] = __uint_as_float(e - 1);  // just below 2^e: what the weights so far stay under
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              acc[mt][nt][j] *= r;
              acc[mt][nt][2 + j] *= r;
            }
            sumw[nt][j] *= r;
          }
      }
      // ---- out^T += codeV^T . (p scaleV)
      float down[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) down[nt][j] = __uint_as_float(((254u + 14u) << 23) - wexp[nt][j]);  // 2^(14 - e)
#pragma unroll
      for (int ti = 0; ti < C::TILES; ++ti) {
        if (ti * kKv4Tile >= left) break;
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            pb[nt][i] = movmatrix_t(
                Elem<__half>::pack2(s[ti][nt][2 * i] * down[nt][0], s[ti][nt][2 * i + 1] * down[nt][1]));
        // A subnormal operand costs the product its low bits (the tensor core
        // aligns by nominal exponents), which the codes do not need; this sum,
        // which is subtracted, does: 2^-14 is the smallest normal number.
        const uint32_t ones[4] = {0x04000400u, 0x04000400u, 0x04000400u, 0x04000400u};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_k16<__half>(sumw[nt], ones, pb[nt][0], pb[nt][1]);
        const uint8_t* vp = sp + ti * C::TB + 8 * D + lane * 16;
#pragma unroll
        for (int hh = 0; hh < D / 64; ++hh) {
          const uint4 u = *reinterpret_cast<const uint4*>(vp + hh * 512);
          const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = wd[j] >> 8;
            const uint32_t f[4] = {wd[j] & 0x000f000fu, wd[j] & 0x00f000f0u, x & 0x000f000fu, x & 0x00f000f0u};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_k16<__half>(acc[hh * 4 + j][nt], f, pb[nt][0], pb[nt][1]);
          }
        }
      }
    }
    __syncwarp();  // the stage is free for the next issue

    // ---- the segment's end, or the range's
    const bool seg_end = con.t + 1 == con.chunks;
    if (seg_end || it + 1 == count) {
      const bool whole = seg_end && seg0 >= w0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) {
            l[nt][j] += __shfl_xor_sync(~0u, l[nt][j], o);
            pz[nt][j] += __shfl_xor_sync(~0u, pz[nt][j], o);
          }
      // 2^e * 2^24 / 2^14; dimensions g + 8 have their codes times 16
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[mt][nt][j] = fmaf(fmaf(acc[mt][nt][j], j < 2 ? 1024.f : 64.f, -7.5f * sumw[nt][j & 1]),
                                  __uint_as_float(wexp[nt][j & 1]), pz[nt][j & 1]);
      const int rows = con.s.n * group;
      if (whole) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float inv[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) inv[j] = l[nt][j] == 0.f ? 0.f : 1.f / l[nt][j];
          const int r = con.rb * C::ROWS + nt * 8 + g;  // after the transpose this lane has row g, dimensions 2c, 2c + 1
          const int64_t tok = con.s.first + by.div(r);
          T* op = static_cast<T*>(a.out) + (tok * a.heads + con.h * group + r - by.div(r) * group) * D + 2 * c;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t tr =
                  movmatrix_t(E::pack2(acc[mt][nt][2 * half] * inv[0], acc[mt][nt][2 * half + 1] * inv[1]));
              if (r < rows) *reinterpret_cast<uint32_t*>(op + mt * 16 + half * 8) = tr;
            }
          if (a.lse && g < 2) {  // lanes (j, c) write rows 2c + j
            const int rr = con.rb * C::ROWS + nt * 8 + 2 * c + g;
            const float lj = g ? l[nt][1] : l[nt][0], mj = g ? m[nt][1] : m[nt][0];
            if (rr < rows)
              a.lse[(con.s.first + by.div(rr)) * static_cast<int64_t>(a.heads) + con.h * group + rr - by.div(rr) * group] =
                  lj == 0.f ? -INFINITY : (mj + __log2f(lj)) * kLn2;
          }
        }
      } else {
        const int slot = 2 * wg + (seg0 > w0 ? 1 : 0);  // 0: the segment holds this range's first chunk
        float* pp = a.part + static_cast<int64_t>(slot) * C::ROWS * D;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = nt * 8 + 2 * c + j;
            if (con.rb * C::ROWS + r < rows) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                  __stcg(pp + r * D + mt * 16 + half * 8 + g, acc[mt][nt][2 * half + j]);
              if (g == 0) __stcg(a.part_ml + slot * C::ROWS + r, make_float2(m[nt][j], l[nt][j]));
            }
          }
        if (seg0 >= w0 && lane == 0) {
          // the segment starts here and goes on in the warps up to the one with its last chunk
          const long long last = seg0 + con.chunks - 1;
          const int wl = static_cast<int>(((last + 1) * warps - 1) / total);
          a.part_desc[2 * wg] = make_int4(wl - wg + 1, slot - 2 * wg, con.s.first, min(rows - con.rb * C::ROWS, C::ROWS));
          a.part_desc[2 * wg + 1] = make_int4(con.rb * C::ROWS, con.h, 0, 0);
        }
      }
    }
    if (it + 1 < count) con.next(a, group, C::ROWS);
  }
  if (!ok)  // let the copies in flight land before the CTA leaves
    for (int i = max(issued - C::S, 0); i < issued; ++i) mbar_wait_bounded(&bar[i % C::S], (i / C::S) & 1, a.err);
}

// Adds the partial rows of segments that several warps shared, in warp order.
// Most warps' ranges hold no start of such a segment, so descriptors are read
// 32 at a time. A segment of few parts (the usual case with many sequences)
// takes one warp per row, whose loads are all issued together; one of many
// parts (few sequences) takes four, each a quarter of the dimensions.

constexpr int kJoinWarps = 8;
constexpr int kJoinFew = 16;  // parts that one warp joins

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_combine_kernel(const Kv4Args a, int warps) {
  using C = AttnCfg<D, NT>;
  const int lane = threadIdx.x & 31;
  const int group = a.heads / a.kv_heads;
  const int gw = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  const int quarter = gw & 3, row = (gw >> 2) % C::ROWS, grp = gw / (4 * C::ROWS);
  const int ngrp = gridDim.x * kJoinWarps / (4 * C::ROWS);
  pdl_wait_prior();
  for (int base = grp; base < warps; base += ngrp * 32) {
    const int w0 = base + lane * ngrp;
    const int4 none = make_int4(0, 0, 0, 0);
    const int4 m0 = w0 < warps ? __ldcg(a.part_desc + 2 * w0) : none, m1 = w0 < warps ? __ldcg(a.part_desc + 2 * w0 + 1) : none;
    const bool mine = m0.x != 0 && row < m0.w && (m0.x > kJoinFew || (lane & 3) == quarter);
    for (unsigned todo = __ballot_sync(~0u, mine); todo; todo &= todo - 1) {
      const int from = __ffs(todo) - 1, w = base + from * ngrp;
      const int parts = __shfl_sync(~0u, m0.x, from), slot0 = 2 * w + __shfl_sync(~0u, m0.y, from);
      const int first = __shfl_sync(~0u, m0.z, from), r = __shfl_sync(~0u, m1.x, from) + row;
      const int h = __shfl_sync(~0u, m1.y, from);
      auto at = [&](int i) { return static_cast<int64_t>(i == 0 ? slot0 : 2 * (w + i)) * C::ROWS + row; };
      const int64_t to = (static_cast<int64_t>(first) + r / group) * a.heads + h * group + r % group;
      auto put = [&](int d, float4 o, float sum) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + to * D + d) =
            make_uint2(Elem<T>::pack2(o.x * inv, o.y * inv), Elem<T>::pack2(o.z * inv, o.w * inv));
      };
      auto add = [&](float4& o, float f, float4 v) {
        if (f != 0.f) {  // a part that saw nothing adds nothing
          o.x += f * v.x;
          o.y += f * v.y;
          o.z += f * v.z;
          o.w += f * v.w;
        }
      };
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f, top = -INFINITY;
      if (parts <= kJoinFew) {
        const int d = lane * 4;
        const float2 ml = lane < parts ? __ldcg(a.part_ml + at(lane)) : make_float2(-INFINITY, 0.f);
        float4 v[kJoinFew / 2];
        auto load = [&](int i0) {
#pragma unroll
          for (int i = 0; i < kJoinFew / 2; ++i)
            if (i0 + i < parts && d < D) v[i] = __ldcg(reinterpret_cast<const float4*>(a.part + at(i0 + i) * D + d));
        };
        load(0);
        top = ml.x;
#pragma unroll
        for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, s));
        const float f = ex2(ml.x - (top == -INFINITY ? 0.f : top));
        sum = f * ml.y;
#pragma unroll
        for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(~0u, sum, s);
        for (int i0 = 0; i0 < parts; i0 += kJoinFew / 2) {
          if (i0 > 0) load(i0);
#pragma unroll
          for (int i = 0; i < kJoinFew / 2; ++i) {
            const float fi = __shfl_sync(~0u, f, (i0 + i) & 31);
            if (i0 + i < parts) add(o, fi, v[i]);
          }
        }
        if (d < D) put(d, o, sum);
      } else {
        constexpr int LANES = D / 16, PARTS = 32 / LANES;  // a quarter of the dimensions; parts at a time
        const int d = quarter * (D / 4) + lane % LANES * 4;
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, __ldcg(a.part_ml + at(i)).x);
#pragma unroll
        for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, s));
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 8
        for (int i = lane / LANES; i < parts; i += PARTS) {
          const float2 ml = __ldcg(a.part_ml + at(i));
          const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part + at(i) * D + d));
          const float f = ex2(ml.x - ref);
          sum += f * ml.y;
          add(o, f, v);
        }
#pragma unroll
        for (int s = LANES; s < 32; s <<= 1) {
          sum += __shfl_xor_sync(~0u, sum, s);
          o.x += __shfl_xor_sync(~0u, o.x, s);
          o.y += __shfl_xor_sync(~0u, o.y, s);
          o.z += __shfl_xor_sync(~0u, o.z, s);
          o.w += __shfl_xor_sync(~0u, o.w, s);
        }
        if (lane < LANES) put(d, o, sum);
      }
      if (a.lse && (parts <= kJoinFew || quarter == 0) && lane == 0)
        a.lse[to] = sum == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + __log2f(sum)) * kLn2;
    }
  }
}

// Query rows per block: 8, or 16 where a sequence brings more than 8 rows.
int row_tiles(int group, int max_q) { return static_cast<long long>(group) * max_q > 8 ? 2 : 1; }

template <typename T, int D, int NT>
struct Attn {
  // CTAs that one SM holds (0: the kernel cannot run here)
  static int per_sm() {
    static PerDevice known;
    return known.get([] {
      using C = AttnCfg<D, NT>;
      int n = 0;
      if (cudaFuncSetAttribute(kv4_attention_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) !=
              cudaSuccess ||
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv4_attention_kernel<T, D, NT>, C::THREADS, C::SMEM) !=
              cudaSuccess)
        return 0;
      return n;
    });
  }
  static int64_t workspace(int num_sms) {
    using C = AttnCfg<D, NT>;
    const int64_t warps = static_cast<int64_t>(per_sm()) * num_sms * C::WARPS;
    return warps * (2 * C::ROWS * (D * 4 + 8) + 32);
  }
  static cudaError_t launch(Kv4Args a, void* ws, int num_sms, cudaStream_t stream) {
    using C = AttnCfg<D, NT>;
    const int grid = per_sm() * num_sms;
    if (grid == 0) return cudaErrorInvalidConfiguration;
    const int64_t warps = static_cast<int64_t>(grid) * C::WARPS;
    a.part_desc = static_cast<int4*>(ws);
    a.part = reinterpret_cast<float*>(a.part_desc + 2 * warps);
    a.part_ml = reinterpret_cast<float2*>(a.part + 2 * warps * C::ROWS * D);
    cudaError_t e = launch_after(kv4_attention_kernel<T, D, NT>, dim3(grid), C::THREADS, C::SMEM, stream, a.pdl, 1, a);
    if (e != cudaSuccess) return e;
    // 8 CTAs per SM: nearly every shared row finds a warp of its own
    return launch_after(kv4_combine_kernel<T, D, NT>, dim3(num_sms * 8), kJoinWarps * 32, 0, stream, a.pdl, 1, a,
                        static_cast<int>(warps));
  }
};

template <template <typename, int> class F, typename... A>
cudaError_t by_type(int dtype, int head_dim, A... args) {
  if (head_dim == 128)
    return dtype == 1 ? F<__nv_bfloat16, 128>::run(args...) : F<__half, 128>::run(args...);
  return dtype == 1 ? F<__nv_bfloat16, 64>::run(args...) : F<__half, 64>::run(args...);
}

// CTAs per sequence and head: the average number of tiles, so that a batch of
// one-token appends launches no idle CTAs; longer sequences loop.
int move_per_seq(const Kv4Args& a) {
  if (!a.cu) return 1;
  const int64_t avg = (static_cast<int64_t>(a.tokens) + a.num_seqs - 1) / a.num_seqs;
  return static_cast<int>(avg <= 1 ? 1 : (avg + kKv4Tile - 1) / kKv4Tile + 1);
}

template <typename T, int D>
struct Append {
  static cudaError_t run(const Kv4Args& a, cudaStream_t stream) {
    const int per = move_per_seq(a);
    return launch_after(kv4_append_kernel<T, D>, dim3(a.num_seqs * per, a.kv_heads), kMoveThreads, 0, stream, a.pdl, 1, a, per);
  }
};
template <typename T, int D>
struct Read {
  static cudaError_t run(const Kv4Args& a, cudaStream_t stream) {
    const int per = move_per_seq(a);
    return launch_after(kv4_read_kernel<T, D>, dim3(a.num_seqs * per, a.kv_heads), kMoveThreads, 0, stream, a.pdl, 1, a, per);
  }
};
template <typename T, int D>
struct Workspace {
  static cudaError_t run(int rows8, int num_sms, int64_t* bytes) {
    *bytes = rows8 == 2 ? Attn<T, D, 2>::workspace(num_sms) : Attn<T, D, 1>::workspace(num_sms);
    return cudaSuccess;
  }
};
template <typename T, int D>
struct Attend {
  static cudaError_t run(int max_q, const Kv4Args& a, void* ws, int num_sms, cudaStream_t stream) {
    return row_tiles(a.heads / a.kv_heads, max_q) == 2 ? Attn<T, D, 2>::launch(a, ws, num_sms, stream)
                                                       : Attn<T, D, 1>::launch(a, ws, num_sms, stream);
  }
};

}  // namespace

cudaError_t launch_kv4_append(int dtype, int head_dim, const Kv4Args& a, cudaStream_t stream) {
  return by_type<Append>(dtype, head_dim, a, stream);
}

cudaError_t launch_kv4_read(int dtype, int head_dim, const Kv4Args& a, cudaStream_t stream) {
  return by_type<Read>(dtype, head_dim, a, stream);
}

int64_t kv4_attention_workspace(int dtype, int head_dim, int group, int max_q, int num_sms) {
  int64_t bytes = 0;
  by_type<Workspace>(dtype, head_dim, row_tiles(group, max_q), num_sms, &bytes);
  return bytes;
}

cudaError_t launch_kv4_attention(int dtype, int head_dim, int max_q, Kv4Args a, void* workspace, int num_sms,
                                 cudaStream_t stream) {
  return by_type<Attend>(dtype, head_dim, max_q, a, workspace, num_sms, stream);
}

}  // namespace wp
