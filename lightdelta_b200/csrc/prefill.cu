// Gated delta rule attention over whole prompts for sm_100a: the chunked form of the recurrence that
// ld_decode runs token by token, with the same gated RMSNorm on its outputs.
//
// Mathematics.  Per (request, value head), with k and q L2-normalised (q also scaled by 128^-1/2),
// g_t = -exp(a_log) softplus(a_t + dt_bias) and beta_t = sigmoid(b_t), the recurrence is
//   u_t = beta_t (v_t - e^{g_t} S_{t-1} k_t),   S_t = e^{g_t} S_{t-1} + u_t k_t^T,   o_t = S_t q_t.
// For a chunk of C tokens entered with state S, and G_i the sum of g over the chunk's tokens up to i,
//   (I + L) U = R,   R_i = beta_i (v_i - e^{G_i} S k_i),   L_ij = beta_i e^{G_i - G_j} k_i.k_j  (i > j),
//   o_i = e^{G_i} S q_i + sum_{j <= i} P_ij u_j,           P_ij = e^{G_i - G_j} q_i.k_j,
//   S  <- e^{G_C} S + sum_j e^{G_C - G_j} u_j k_j^T,
// so a chunk is a handful of matrix products and one inverse T = (I + L)^{-1} of a unit triangular
// matrix, and only the state passes from chunk to chunk.
//
// Precision.  The state and every sum stay in fp32.  Matrix instructions take fp16 operands with
// fp32 accumulation.  q and k rows are bf16 and become fp16 exactly after scaling by a power of two
// per row (which the fp32 factors fk, fq undo).  Operands on the way to the state (S itself, R, U and
// T, L) go in as two fp16 terms, hi + lo, 22 bits together, after scaling each state row by a power of
// two, so the state follows the fp32 recurrence to under 1e-6.  The two products that only reach the
// bf16 output (S q and P u) take the hi term alone: 11 bits against the output's 8.  G is summed in
// fp64 and kept as two floats, so differences of large sums stay exact to fp32.
//
// Two kernels.  What does not depend on the state is computed first, for all chunks side by side:
// gdn_prefill_pairs_kernel, one CTA per (chunk, key head), scales q and k, forms their products once for
// all value heads of the key head, and leaves q, k, T, P and the rows' factors in a workspace, as the
// images that the second kernel copies to shared memory.  gdn_prefill_chain_kernel, one CTA per
// (request, value head), then carries the state from chunk to chunk: eight chain warps hold the 128 x
// 128 state as accumulator fragments, 16 value rows each.  S k, T R and the update all have the state's
// value rows as M, so every warp carries its rows through all chunks without exchanging anything with
// the others (an accumulator fragment is the next product's A fragment).  Four more warps copy the next
// chunk in and normalise and store the chunk before's outputs.  A first form that prepared each chunk
// inside the chain's CTA took 1,242 us on 24 prompts of 16,000 tokens in all (16 key, 32 value heads):
// its preparation, 33,000 cycles a chunk of short dependent steps, held the chain's 10,500 up.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "internal.h"
#include "launch.cuh"
#include "lightdelta_b200.h"

namespace ldb {
namespace {

constexpr int kDim = LD_HEAD_DIM;
constexpr int kChunk = LD_PREFILL_CHUNK;
constexpr int kPairThreads = 128;
constexpr int kCopyThreads = 128;
constexpr int kChainWarps = 8;
constexpr int kChainThreads = kCopyThreads + 32 * kChainWarps;
constexpr int kORow = kDim + 4;  // floats per row of the output tile: the +4 spreads its rows over the banks
static_assert(kChunk == 64, "fragment loops below are written for chunks of 64 tokens");

__device__ unsigned int g_prefill_faults;

// Workspace images.  Tiles of 128 columns are swizzled (swz), triangular matrices are packed 16 x 16
// blocks (tri), exactly as the chain reads them from shared memory.
struct __align__(128) KeyImage {  // per (chunk, key head)
  __half k[kChunk * kDim];        // k rows x 2^-e
  __half q[kChunk * kDim];        // q rows x 2^-e
};

constexpr int kTriBlocks = 10;  // 16 x 16 blocks on and below the diagonal of a 64 x 64 matrix
struct __align__(128) PairImage {  // per (chunk, value head)
  __half t_hi[kTriBlocks * 256];
  __half t_lo[kTriBlocks * 256];
  __half p[kTriBlocks * 256];
  float beta[kChunk];
  float k_in[kChunk];   // e^{G_i} fk_i: scales S k~
  float q_in[kChunk];   // e^{G_i} fq_i 128^-1/2: scales S q~
  float k_out[kChunk];  // e^{G_C - G_j} fk_j: scales u_j on its way into the state
  float decay;          // e^{G_C}
};
static_assert(sizeof(KeyImage) % 16 == 0 && sizeof(PairImage) % 16 == 0, "images are copied 16 bytes at a time");

struct PrefillArgs {
  const __nv_bfloat16* qkv;
  int64_t qkv_row;
  const __nv_bfloat16* a;
  int64_t a_row;
  const __nv_bfloat16* b;
  int64_t b_row;
  const float* a_log;
  const void* dt_bias;
  const int32_t* table;
  int64_t table_row;
  int64_t table_width;
  const int32_t* context;
  const int32_t* cu;
  void* state;
  int64_t n_slots;
  int64_t slot_stride;
  const __nv_bfloat16* gate;
  int64_t gate_row;
  const void* weight;
  __nv_bfloat16* out;
  int64_t n_tokens;
  int64_t block_size;
  KeyImage* keys;    // [chunk places, num_k_heads]
  PairImage* pairs;  // [chunk places, num_v_heads]
  int n_requests;
  int num_k_heads;
  int num_v_heads;
  int heads_ratio;
  int dt_bias_bf16;
  int weight_bf16;
  float q_scale;
  float eps;
};

// Chunk c of request r is kept at place chunk_base(cu[r], r) + c.  A request of n tokens has at most
// n / 64 + 2 chunks (both ends may be short), so places never overlap, and nobody has to count chunks.
__host__ __device__ __forceinline__ int64_t chunk_base(int64_t first_token, int64_t request) {
  return first_token / kChunk + 2 * request;
}

// A request that runs.
struct Request {
  int64_t first;    // its first token
  int64_t tokens;
  int64_t context;
  int64_t chunks;
  int lead;         // rows of the first chunk in front of the first token
  int32_t source;   // state slot to start from (0: from nothing)
  const int32_t* row;
};

// ------------------------------------------------------------------------------------------
// instructions
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// D[16 x 8] += A[16 x 16] B[16 x 8], fp16 operands, fp32 accumulators.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void bar_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kChainThreads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kChainThreads) : "memory");
}
// Named barriers of the chain kernel, which hand its buffers over (two each of full and empty).
constexpr int kBarFull = 1, kBarEmpty = 3, kBarOReady = 5, kBarOFree = 6;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int bytes = live ? 16 : 0;  // 0: the 16 bytes are filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ------------------------------------------------------------------------------------------
// swizzled tiles: 16-byte pieces of a row are stored at piece ^ (row mod 8), so that the eight rows
// of an 8 x 8 matrix lie in different banks
// ------------------------------------------------------------------------------------------
template <int kCols>
__device__ __forceinline__ int swz(int row, int col) {
  constexpr int kPieces = kCols / 8;
  static_assert(kPieces >= 8, "rows of eight pieces at least");
  return row * kCols + ((((col >> 3) ^ (row & 7)) << 3) | (col & 7));
}

// Address that this lane gives to ldmatrix.x4 for the 16 x 16 block at (0, 0) of a tile: matrices in the
// order (rows 0-7, cols 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15), or with kRowsFirst
// (0-7, 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15).  Row blocks start at multiples of 8, so the swizzle
// depends on the lane alone and the block at (16 rb, 16 cb) is at block<kCols>(address, rb, cb).
template <int kCols, bool kRowsFirst>
__device__ __forceinline__ uint32_t lane_addr(const void* tile, int lane) {
  const int m = lane >> 3;
  const int row = (lane & 7) + 8 * (kRowsFirst ? (m & 1) : (m >> 1));
  const int piece = (kRowsFirst ? (m >> 1) : (m & 1)) ^ (lane & 7);
  return smem_u32(tile) + row * kCols * 2 + (piece << 4);
}

template <int kCols>
__device__ __forceinline__ uint32_t block(uint32_t addr, int rb, int cb) {
  return (addr ^ (cb << 5)) + rb * (16 * kCols * 2);
}

// Packed triangular matrices: block (ib, jb), jb <= ib, of 16 rows of 32 bytes; the two 16-byte pieces of
// rows 4-7 and 12-15 are exchanged, so that eight rows' pieces lie in different banks.
__device__ __forceinline__ int tri(int row, int col) {
  const int ib = row >> 4, jb = col >> 4, r = row & 15, c = col & 15;
  return (ib * (ib + 1) / 2 + jb) * 256 + r * 16 + ((((c >> 3) ^ ((r >> 2) & 1)) << 3) | (c & 7));
}

// This lane's ldmatrix.x4 address in block 0 of a packed matrix, matrices in the order of lane_addr with
// kRowsFirst false; block b is 512 bytes on per block.
__device__ __forceinline__ uint32_t tri_addr(const __half* m, int lane) {
  return smem_u32(m) + 2 * tri((lane & 7) + 8 * (lane >> 4), 8 * ((lane >> 3) & 1));
}
__host__ __device__ constexpr int tri_block(int ib, int jb) { return (ib * (ib + 1) / 2 + jb) * 512; }

__device__ __forceinline__ uint32_t pack_half(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// x, y as two fp16 terms: hi the nearest, lo the nearest to what hi leaves.
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// 2^s with s such that the largest magnitude m lands in [2^13, 2^14), and 2^-s: fp16's two terms then
// resolve 2^-25 of a range of 2^14.  m of 0 (or too small for the exponent) takes the largest scale.
__device__ __forceinline__ void row_scale(float m, float& up, float& down) {
  int e = static_cast<int>((__float_as_uint(m) >> 23) & 0xff);
  e = max(e, 14);
  e = min(e, 253);
  up = __uint_as_float(static_cast<uint32_t>(267 - e) << 23);    // 2^(140 - e) = 2^13 / 2^(e - 127)
  down = __uint_as_float(static_cast<uint32_t>(e - 13) << 23);
}

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

__device__ __forceinline__ float load_param(const void* p, int index, int is_bf16) {
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[index])
                 : static_cast<const float*>(p)[index];
}

__device__ __forceinline__ float softplus(float x) { return x > 20.0f ? x : log1pf(expf(x)); }

// 2^x of non-positive x, within 2 ulp of the fp32 value (0 below 2^-126).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// z sigmoid(z) with the fast exponential and division: a few fp32 ulps, far below bf16's rounding.
__device__ __forceinline__ float silu(float z) { return __fdividef(z, 1.0f + __expf(-z)); }

// ------------------------------------------------------------------------------------------
// pairs: what a chunk's tokens mean to one another
// ------------------------------------------------------------------------------------------
constexpr int kGroup = 4;  // value heads whose gates are computed together, one per warp

struct PairSmem {
  __align__(256) __half k[kChunk * kDim];
  __align__(256) __half q[kChunk * kDim];
  PairImage image;
  __align__(128) __half l_hi[6 * 256];  // L's blocks below the diagonal ones, packed row by row
  __align__(128) __half l_lo[6 * 256];
  __align__(16) float diag[4][16 * 16];  // L's diagonal blocks
  float g_hi[kGroup][kChunk], g_lo[kGroup][kChunk], beta[kGroup][kChunk];
  float fk[kChunk], fq[kChunk];
};

// Element (row, col) of a block strictly below the diagonal of the packed L, and the byte offset of a block.
__host__ __device__ constexpr int low_block(int ib, int jb) { return (ib * (ib - 1) / 2 + jb) * 512; }
__device__ __forceinline__ int low(int row, int col) {
  const int r = row & 15, c = col & 15;
  return low_block(row >> 4, col >> 4) / 2 + r * 16 + ((((c >> 3) ^ ((r >> 2) & 1)) << 3) | (c & 7));
}

template <bool kVec>
__device__ __forceinline__ void load_rows(const __nv_bfloat16* base, int64_t row_stride, int row_lo, int row_hi,
                                          uint16_t* tile, int tid) {
#pragma unroll
  for (int pass = 0; pass < kChunk / 8; ++pass) {
    const int i = pass * 8 + (tid >> 4);
    const int col = (tid & 15) * 8;
    const bool live = i >= row_lo && i < row_hi;
    uint16_t* dst = tile + swz<kDim>(i, col);
    const __nv_bfloat16* src = base + static_cast<int64_t>(live ? i : row_lo) * row_stride + col;
    if constexpr (kVec) {
      cp_async16(smem_u32(dst), src, live);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = live ? __bfloat16_as_ushort(src[e]) : 0;
    }
  }
}

// Scales one row from bf16 to fp16 in place, by one thread: exact, since a power of two brings the row's
// largest magnitude to [1, 2).  Returns that power's inverse.
__device__ __forceinline__ float scale_row(uint16_t* tile, int i) {
  uint16_t* row = tile + i * kDim;
  uint32_t top2 = 0;  // the largest magnitudes so far of even and odd columns; bf16 magnitudes order as integers
#pragma unroll
  for (int piece = 0; piece < kDim / 8; ++piece) {
    const uint4 raw = *reinterpret_cast<const uint4*>(row + ((piece ^ (i & 7)) << 3));
    top2 = __vmaxu2(__vmaxu2(top2, raw.x & 0x7fff7fffu), raw.y & 0x7fff7fffu);
    top2 = __vmaxu2(__vmaxu2(top2, raw.z & 0x7fff7fffu), raw.w & 0x7fff7fffu);
  }
  const int e = min(max(static_cast<int>(max(top2 >> 16, top2 & 0xffffu) >> 7), 1), 253);
  const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);  // 2^(127 - e)
#pragma unroll
  for (int piece = 0; piece < kDim / 8; ++piece) {
    uint4* at = reinterpret_cast<uint4*>(row + ((piece ^ (i & 7)) << 3));
    const uint4 raw = *at;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t y[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      y[n] = pack_half(__uint_as_float(w[n] << 16) * down, __uint_as_float(w[n] & 0xffff0000u) * down);
    }
    *at = make_uint4(y[0], y[1], y[2], y[3]);
  }
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

// g and beta of the chunk's tokens for one value head and G's running sums (in powers of two), by one
// warp (lane: rows lane and lane + 32).
__device__ __forceinline__ void chunk_gates(const PrefillArgs& p, PairSmem& s, int place, int64_t token0, int row_lo,
                                            int row_hi, int head, int lane) {
  const float rate = -expf(p.a_log[head]);
  const float bias = load_param(p.dt_bias, head, p.dt_bias_bf16);
  constexpr double kLog2e = 1.4426950408889634;
  float a[2], b[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = lane + 32 * half;
    a[half] = b[half] = 0.0f;
    if (i >= row_lo && i < row_hi) {
      a[half] = __bfloat162float(p.a[(token0 + i) * p.a_row + head]);
      b[half] = __bfloat162float(p.b[(token0 + i) * p.b_row + head]);
    }
  }
  double sum[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = lane + 32 * half;
    float g = 0.0f, beta = 0.0f;
    if (i >= row_lo && i < row_hi) {
      g = rate * softplus(a[half] + bias);
      // e^-1000 is 0 in fp32: a floor keeps differences of sums finite and changes no value.
      if (g < -1000.0f) g = -1000.0f;
      beta = __fdividef(1.0f, 1.0f + __expf(-b[half]));
    }
    s.beta[place][i] = beta;
    double x = static_cast<double>(g) * kLog2e;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    sum[half] = x;
  }
  sum[1] += __shfl_sync(0xffffffffu, sum[0], 31);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float hi = static_cast<float>(sum[half]);
    s.g_hi[place][lane + 32 * half] = hi;
    s.g_lo[place][lane + 32 * half] = static_cast<float>(sum[half] - static_cast<double>(hi));
  }
}

// Products of this warp's 16 rows of k~ and q~ with the rows of k~ up to its own, and the rows' factors
// (the L2 norm's reciprocal times the power of two that the scaling took) from the diagonals of k~ k~^T
// and q~ q~^T.
__device__ __forceinline__ void row_products(PairSmem& s, int w, int lane, float (&kk)[4][2][4],
                                             float (&qk)[4][2][4]) {
  const uint32_t k_a = lane_addr<kDim, true>(s.k, lane) + w * 16 * kDim * 2;
  const uint32_t q_a = lane_addr<kDim, true>(s.q, lane) + w * 16 * kDim * 2;
  const uint32_t k_b = lane_addr<kDim, false>(s.k, lane);
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int e = 0; e < 4; ++e) kk[nb][m][e] = qk[nb][m][e] = 0.0f;
    }
  }
  float qq[2][4] = {};
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    uint32_t ak[4], aq[4];
    ldsm4(block<kDim>(k_a, 0, ks), ak);
    ldsm4(block<kDim>(q_a, 0, ks), aq);
    // A fragments are (rows 0-7, cols 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15): as B, rows 0-7 are 0, 2.
    mma(qq[0], aq, aq[0], aq[2]);
    mma(qq[1], aq, aq[1], aq[3]);
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      if (nb <= w) {
        uint32_t b[4];
        ldsm4(block<kDim>(k_b, nb, ks), b);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          mma(kk[nb][m], ak, b[2 * m], b[2 * m + 1]);
          mma(qk[nb][m], aq, b[2 * m], b[2 * m + 1]);
        }
      }
    }
  }
  // Element (g, g) of the diagonal block is with t = g / 2 (of 8 columns), and (g + 8, g + 8) likewise.
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float k2 = 0.0f;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      if (nb == w) k2 = (g & 1) ? kk[nb][half][2 * half + 1] : kk[nb][half][2 * half];
    }
    const float q2 = (g & 1) ? qq[half][2 * half + 1] : qq[half][2 * half];
    if (t == g / 2) {
      const int i = 16 * w + g + 8 * half;
      const float up_k = s.fk[i], up_q = s.fq[i];
      s.fk[i] = up_k * rsqrtf(k2 * up_k * up_k + 1e-6f);
      s.fq[i] = up_q * rsqrtf(q2 * up_q * up_q + 1e-6f);
    }
  }
}

// L and P of this warp's rows for one value head.
__device__ __forceinline__ void decayed_pairs(const PrefillArgs& p, PairSmem& s, int place, int w, int lane,
                                              const float (&kk)[4][2][4], const float (&qk)[4][2][4]) {
  const int g = lane >> 2, t = lane & 3;
  float g_hi[2], g_lo[2], row_k[2], row_q[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = 16 * w + g + 8 * half;
    g_hi[half] = s.g_hi[place][i];
    g_lo[half] = s.g_lo[place][i];
    row_k[half] = s.beta[place][i] * s.fk[i];
    row_q[half] = p.q_scale * s.fq[i];
  }
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
    if (nb > w) continue;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int j = 16 * nb + 8 * m + 2 * t;
      const float2 hj = *reinterpret_cast<const float2*>(&s.g_hi[place][j]);
      const float2 lj = *reinterpret_cast<const float2*>(&s.g_lo[place][j]);
      const float2 fj = *reinterpret_cast<const float2*>(&s.fk[j]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = 16 * w + g + 8 * half;
        const float d0 = fj.x * exp2_fast((g_hi[half] - hj.x) + (g_lo[half] - lj.x));
        const float d1 = fj.y * exp2_fast((g_hi[half] - hj.y) + (g_lo[half] - lj.y));
        const float l0 = j < i ? row_k[half] * d0 * kk[nb][m][2 * half] : 0.0f;
        const float l1 = j + 1 < i ? row_k[half] * d1 * kk[nb][m][2 * half + 1] : 0.0f;
        const float p0 = j <= i ? row_q[half] * d0 * qk[nb][m][2 * half] : 0.0f;
        const float p1 = j + 1 <= i ? row_q[half] * d1 * qk[nb][m][2 * half + 1] : 0.0f;
        *reinterpret_cast<uint32_t*>(&s.image.p[tri(i, j)]) = pack_half(p0, p1);
        if (nb == w) {
          *reinterpret_cast<float2*>(&s.diag[w][(g + 8 * half) * 16 + (j & 15)]) = make_float2(l0, l1);
        } else {
          uint32_t hi, lo;
          split(l0, l1, hi, lo);
          *reinterpret_cast<uint32_t*>(&s.l_hi[low(i, j)]) = hi;
          *reinterpret_cast<uint32_t*>(&s.l_lo[low(i, j)]) = lo;
        }
      }
    }
  }
}

// Inverse of this warp's diagonal block of I + L by forward substitution, one column per lane.
__device__ __forceinline__ void invert_diagonal(PairSmem& s, int w, int lane) {
  const int c = lane & 15;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float sum0 = i == c ? 1.0f : 0.0f, sum1 = 0.0f;
#pragma unroll
    for (int j = 0; j < i; ++j) {
      const float l = s.diag[w][i * 16 + j];
      if (j & 1) {
        sum1 = fmaf(-l, x[j], sum1);
      } else {
        sum0 = fmaf(-l, x[j], sum0);
      }
    }
    x[i] = sum0 + sum1;
  }
  if (lane < 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __half hi = __float2half_rn(x[i]);
      s.image.t_hi[tri(16 * w + i, 16 * w + c)] = hi;
      s.image.t_lo[tri(16 * w + i, 16 * w + c)] = __float2half_rn(x[i] - __half2float(hi));
    }
  }
}

// The 16 x 16 blocks of T below diagonal block w, top to bottom:
//   T_iw = -T_ii sum_{k=w}^{i-1} L_ik T_kw,  held transposed so that each result is the next A operand.
__device__ __forceinline__ void invert_column(PairSmem& s, int w, int lane) {
  const uint32_t t_hi = tri_addr(s.image.t_hi, lane), t_lo = tri_addr(s.image.t_lo, lane);
  const uint32_t l_hi = tri_addr(s.l_hi, lane), l_lo = tri_addr(s.l_lo, lane);
  uint32_t x_hi[3][4], x_lo[3][4];  // T_kw^T as A fragments, k = w, w + 1, w + 2
  // ldmatrix.trans of T_ww: matrices (cols 0-7, rows 0-7), (cols 8-15, rows 0-7), (0-7, 8-15), (8-15, 8-15).
  ldsm4_t(t_hi + tri_block(w, w), x_hi[0]);
  ldsm4_t(t_lo + tri_block(w, w), x_lo[0]);
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    const int i = w + d;
    if (i < 4) {
      float m[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < d; ++kk) {
        uint32_t b_hi[4], b_lo[4];
        ldsm4(l_hi + low_block(i, w + kk), b_hi);
        ldsm4(l_lo + low_block(i, w + kk), b_lo);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          mma(m[n], x_hi[kk], b_lo[2 * n], b_lo[2 * n + 1]);
          mma(m[n], x_lo[kk], b_hi[2 * n], b_hi[2 * n + 1]);
          mma(m[n], x_hi[kk], b_hi[2 * n], b_hi[2 * n + 1]);
        }
      }
      uint32_t a_hi[4], a_lo[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        split(m[n][0], m[n][1], a_hi[2 * n], a_lo[2 * n]);
        split(m[n][2], m[n][3], a_hi[2 * n + 1], a_lo[2 * n + 1]);
      }
      float y[2][4] = {};
      uint32_t b_hi[4], b_lo[4];
      ldsm4(t_hi + tri_block(i, i), b_hi);
      ldsm4(t_lo + tri_block(i, i), b_lo);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        mma(y[n], a_hi, b_lo[2 * n], b_lo[2 * n + 1]);
        mma(y[n], a_lo, b_hi[2 * n], b_hi[2 * n + 1]);
        mma(y[n], a_hi, b_hi[2 * n], b_hi[2 * n + 1]);
      }
      // y[n] is -T_iw^T: row m = column of T_iw (g, g + 8), column = row of T_iw (8n + 2t, + 1).
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          split(-y[n][2 * half], -y[n][2 * half + 1], hi[half], lo[half]);
          const int col = 16 * w + g + 8 * half, row = 16 * i + 8 * n + 2 * t;
          const __half2 h = *reinterpret_cast<const __half2*>(&hi[half]);
          const __half2 l = *reinterpret_cast<const __half2*>(&lo[half]);
          s.image.t_hi[tri(row, col)] = __low2half(h);
          s.image.t_hi[tri(row + 1, col)] = __high2half(h);
          s.image.t_lo[tri(row, col)] = __low2half(l);
          s.image.t_lo[tri(row + 1, col)] = __high2half(l);
        }
        if (d < 3) {
          x_hi[d < 3 ? d : 0][2 * n] = hi[0];
          x_hi[d < 3 ? d : 0][2 * n + 1] = hi[1];
          x_lo[d < 3 ? d : 0][2 * n] = lo[0];
          x_lo[d < 3 ? d : 0][2 * n + 1] = lo[1];
        }
      }
    }
  }
}

// Request r, when its tokens, context, blocks and source slot are in order.  Otherwise false, with the
// fault bit to report, and `skip` when its outputs stay as they are (no tokens, or none to write to).
__device__ __forceinline__ bool find_request(const PrefillArgs& p, int64_t r, Request& rq, unsigned int& fault,
                                             bool& skip) {
  const int64_t begin = p.cu[r], end = p.cu[r + 1];
  fault = 0;
  skip = true;
  if (end <= begin) return false;
  if (begin < 0 || end > p.n_tokens) {
    fault = LD_FAULT_DECODE_TOKENS;
    return false;
  }
  skip = false;
  rq.first = begin;
  rq.tokens = end - begin;
  rq.context = p.context[r];
  rq.row = p.table + r * p.table_row;
  rq.source = 0;
  if (rq.context < 0 || (rq.context + rq.tokens - 1) / p.block_size >= p.table_width) {
    fault = LD_FAULT_TABLE_BLOCKS;
    return false;
  }
  if (rq.context > 0) {
    rq.source = rq.row[(rq.context - 1) / p.block_size];
    if (rq.source >= p.n_slots) fault = LD_FAULT_DECODE_SLOT_RANGE;
    if (rq.source <= 0 || rq.source >= p.n_slots) return false;
  }
  rq.lead = static_cast<int>(rq.context % kChunk);
  rq.chunks = (rq.lead + rq.tokens + kChunk - 1) / kChunk;
  return true;
}

template <bool kVec>
__global__ void __launch_bounds__(kPairThreads, 3) gdn_prefill_pairs_kernel(const PrefillArgs p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  PairSmem& s = *reinterpret_cast<PairSmem*>(raw);
  grid_dependency_wait();
  allow_dependent_launch();
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int64_t place = blockIdx.x / p.num_k_heads;
  const int kh = static_cast<int>(blockIdx.x - place * p.num_k_heads);
  // The request of this place: the last r whose places start at or before it, by 32-way bisection.
  int lo = 0, hi = p.n_requests;
  while (hi - lo > 1) {
    const int width = (hi - lo + 31) / 32;
    const int probe = lo + (lane + 1) * width;
    const bool below = probe < hi && chunk_base(p.cu[probe], probe) <= place;
    const int passed = __popc(__ballot_sync(0xffffffffu, below));
    const int next = lo + passed * width;
    hi = min(hi, next + width);
    lo = next;
  }
  Request rq;
  unsigned int fault;
  bool skip;
  if (!find_request(p, lo, rq, fault, skip)) return;
  const int64_t chunk = place - chunk_base(rq.first, lo);
  if (chunk < 0 || chunk >= rq.chunks) return;

  // Row i of the chunk is token token0 + i; rows outside [row_lo, row_hi) belong to no token.
  const int64_t local0 = chunk * kChunk - rq.lead;
  const int64_t token0 = rq.first + local0;
  const int row_lo = chunk == 0 ? rq.lead : 0;
  const int row_hi = static_cast<int>(min(static_cast<int64_t>(kChunk), rq.tokens - local0));
  const __nv_bfloat16* rows = p.qkv + token0 * p.qkv_row;
  load_rows<kVec>(rows + (p.num_k_heads + kh) * kDim, p.qkv_row, row_lo, row_hi, reinterpret_cast<uint16_t*>(s.k), tid);
  load_rows<kVec>(rows + kh * kDim, p.qkv_row, row_lo, row_hi, reinterpret_cast<uint16_t*>(s.q), tid);
  const int head0 = kh * p.heads_ratio;
  if (w < p.heads_ratio) chunk_gates(p, s, w, token0, row_lo, row_hi, head0 + w, lane);
  if constexpr (kVec) cp_async_wait();
  __syncthreads();
  if (tid < kChunk) {
    s.fk[tid] = scale_row(reinterpret_cast<uint16_t*>(s.k), tid);
  } else {
    s.fq[tid - kChunk] = scale_row(reinterpret_cast<uint16_t*>(s.q), tid - kChunk);
  }
  __syncthreads();
  {
    uint4* to = reinterpret_cast<uint4*>(p.keys + place * p.num_k_heads + kh);
    const uint4* k = reinterpret_cast<const uint4*>(s.k);
    const uint4* q = reinterpret_cast<const uint4*>(s.q);
    constexpr int kPieces = kChunk * kDim / 8;
#pragma unroll
    for (int i = 0; i < kPieces / kPairThreads; ++i) {
      to[i * kPairThreads + tid] = k[i * kPairThreads + tid];
      to[kPieces + i * kPairThreads + tid] = q[i * kPairThreads + tid];
    }
  }
  float kk[4][2][4], qk[4][2][4];
  row_products(s, w, lane, kk, qk);
  __syncthreads();
#pragma unroll 1
  for (int n = 0; n < p.heads_ratio; ++n) {
    const int at = n % kGroup;
    if (n > 0) {
      __syncthreads();  // the image and, every fourth head, the gates are taken over
      if (at == 0) {
        if (n + w < p.heads_ratio) chunk_gates(p, s, w, token0, row_lo, row_hi, head0 + n + w, lane);
        __syncthreads();
      }
    }
    if (tid < kChunk) {
      const float in = exp2_fast(s.g_hi[at][tid] + s.g_lo[at][tid]);
      s.image.beta[tid] = s.beta[at][tid];
      s.image.k_in[tid] = in * s.fk[tid];
      s.image.q_in[tid] = in * s.fq[tid] * p.q_scale;
      const float left = (s.g_hi[at][kChunk - 1] - s.g_hi[at][tid]) + (s.g_lo[at][kChunk - 1] - s.g_lo[at][tid]);
      s.image.k_out[tid] = exp2_fast(left) * s.fk[tid];
      if (tid == kChunk - 1) s.image.decay = in;
    }
    decayed_pairs(p, s, at, w, lane, kk, qk);
    __syncwarp();
    invert_diagonal(s, w, lane);
    __syncthreads();
    invert_column(s, w, lane);
    __syncthreads();
    uint4* to = reinterpret_cast<uint4*>(p.pairs + place * p.num_v_heads + head0 + n);
    const uint4* from = reinterpret_cast<const uint4*>(&s.image);
    for (int i = tid; i < static_cast<int>(sizeof(PairImage) / 16); i += kPairThreads) to[i] = from[i];
  }
}

// ------------------------------------------------------------------------------------------
// chain: the state through the chunks, 16 value rows per warp
// ------------------------------------------------------------------------------------------
struct Stage {
  KeyImage key;
  __align__(256) __nv_bfloat16 v[kChunk * kDim];  // swizzled
  PairImage pair;
};

struct ChainSmem {
  __align__(256) Stage stage[2];
  __align__(16) float o[kChunk * kORow];
};

template <typename Image>
__device__ __forceinline__ void copy_image(Image& to, const Image* from, int tid) {
  constexpr int kPieces = sizeof(Image) / 16, kWhole = kPieces / kCopyThreads;
  const uint32_t dst = smem_u32(&to) + 16 * tid;
  const unsigned char* src = reinterpret_cast<const unsigned char*>(from) + 16 * tid;
#pragma unroll
  for (int i = 0; i < kWhole; ++i) cp_async16(dst + 16 * kCopyThreads * i, src + 16 * kCopyThreads * i);
  if (tid < kPieces % kCopyThreads) cp_async16(dst + 16 * kCopyThreads * kWhole, src + 16 * kCopyThreads * kWhole);
}

template <bool kVec>
__device__ __forceinline__ void copy_chunk(const PrefillArgs& p, Stage& st, const Request& rq, int64_t chunk,
                                           int64_t place, int head, int tid) {
  const int kh = head / p.heads_ratio;
  copy_image(st.key, p.keys + place * p.num_k_heads + kh, tid);
  copy_image(st.pair, p.pairs + place * p.num_v_heads + head, tid);
  const int64_t local0 = chunk * kChunk - rq.lead;
  const int row_lo = chunk == 0 ? rq.lead : 0;
  const int row_hi = static_cast<int>(min(static_cast<int64_t>(kChunk), rq.tokens - local0));
  load_rows<kVec>(p.qkv + (rq.first + local0) * p.qkv_row + (2 * p.num_k_heads + head) * kDim, p.qkv_row, row_lo,
                  row_hi, reinterpret_cast<uint16_t*>(st.v), tid);
}

// Gated RMSNorm of the chunk's outputs.  A warp takes two rows at a time, 16 lanes and twice four values
// per lane each; gate rows are loaded first, so that they arrive while the chain finishes the tile (`wait`
// returns then).
template <bool kVec, typename Wait>
__device__ __forceinline__ void store_outputs(const PrefillArgs& p, const ChainSmem& s, const Request& rq,
                                              int64_t chunk, int head, const float (&wt)[8], int tid, Wait wait) {
  const int w = tid >> 5, lane = tid & 31, part = lane & 15;
  const int64_t local0 = chunk * kChunk - rq.lead;
  const int row_lo = chunk == 0 ? rq.lead : 0;
  const int row_hi = static_cast<int>(min(static_cast<int64_t>(kChunk), rq.tokens - local0));
  constexpr int kSteps = kChunk / 8;
  const __nv_bfloat16* gate = p.gate + (rq.first + local0) * p.gate_row + head * kDim + 4 * part;
  uint2 z[kSteps][2];
#pragma unroll
  for (int n = 0; n < kSteps; ++n) {
    const int i = 8 * n + 2 * w + (lane >> 4);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      z[n][half] = make_uint2(0, 0);
      if (i >= row_lo && i < row_hi) {
        const __nv_bfloat16* at = gate + i * p.gate_row + 64 * half;
        if constexpr (kVec) {
          z[n][half] = *reinterpret_cast<const uint2*>(at);
        } else {
          z[n][half].x = __bfloat16_as_ushort(at[0]) | (static_cast<uint32_t>(__bfloat16_as_ushort(at[1])) << 16);
          z[n][half].y = __bfloat16_as_ushort(at[2]) | (static_cast<uint32_t>(__bfloat16_as_ushort(at[3])) << 16);
        }
      }
    }
  }
  wait();
  __nv_bfloat16* out = p.out + ((rq.first + local0) * p.num_v_heads + head) * kDim + 4 * part;
#pragma unroll
  for (int n = 0; n < kSteps; ++n) {
    const int i = 8 * n + 2 * w + (lane >> 4);
    float4 o[2];
    float sq = 0.0f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      o[half] = *reinterpret_cast<const float4*>(&s.o[i * kORow + 64 * half + 4 * part]);
      sq = fmaf(o[half].x, o[half].x, sq);
      sq = fmaf(o[half].y, o[half].y, sq);
      sq = fmaf(o[half].z, o[half].z, sq);
      sq = fmaf(o[half].w, o[half].w, sq);
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    const float rstd = rsqrtf(sq * (1.0f / kDim) + p.eps);
    const bool live = i >= row_lo && i < row_hi;
    __nv_bfloat16* row = out + static_cast<int64_t>(i) * p.num_v_heads * kDim;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint2 zz = z[n][half];
      const float y0 = o[half].x * rstd * wt[4 * half + 0] * silu(__uint_as_float(zz.x << 16));
      const float y1 = o[half].y * rstd * wt[4 * half + 1] * silu(__uint_as_float(zz.x & 0xffff0000u));
      const float y2 = o[half].z * rstd * wt[4 * half + 2] * silu(__uint_as_float(zz.y << 16));
      const float y3 = o[half].w * rstd * wt[4 * half + 3] * silu(__uint_as_float(zz.y & 0xffff0000u));
      __nv_bfloat16* at = row + 64 * half;
      if constexpr (kVec) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(y0, y1), hi = __floats2bfloat162_rn(y2, y3);
        if (live) {
          *reinterpret_cast<uint2*>(at) =
              make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        }
      } else if (live) {
        at[0] = __float2bfloat16_rn(y0);
        at[1] = __float2bfloat16_rn(y1);
        at[2] = __float2bfloat16_rn(y2);
        at[3] = __float2bfloat16_rn(y3);
      }
    }
  }
}

__device__ __forceinline__ void load_pair(const float* at, float& x, float& y) {
  const float2 v = *reinterpret_cast<const float2*>(at);
  x = v.x;
  y = v.y;
}
__device__ __forceinline__ void load_pair(const __nv_bfloat16* at, float& x, float& y) {
  const uint32_t v = *reinterpret_cast<const uint32_t*>(at);
  x = __uint_as_float(v << 16);
  y = __uint_as_float(v & 0xffff0000u);
}
__device__ __forceinline__ void store_pair(float* at, float x, float y) {
  *reinterpret_cast<float2*>(at) = make_float2(x, y);
}
__device__ __forceinline__ void store_pair(__nv_bfloat16* at, float x, float y) {
  *reinterpret_cast<__nv_bfloat162*>(at) = __floats2bfloat162_rn(x, y);
}

// One chunk on this warp's rows of S.  The output tile is free when `wait_o` says so.
template <typename WaitO>
__device__ __forceinline__ void chain_chunk(float (&S)[16][4], const Stage& st, float* o_tile, int v0, int lane,
                                            WaitO wait_o) {
  const int g = lane >> 2, t = lane & 3;
  const uint32_t k_base = lane_addr<kDim, false>(st.key.k, lane), q_base = lane_addr<kDim, false>(st.key.q, lane);
  const uint32_t k_trans = lane_addr<kDim, true>(st.key.k, lane), v_base = lane_addr<kDim, false>(st.v, lane);
  const uint32_t th_base = tri_addr(st.pair.t_hi, lane), tl_base = tri_addr(st.pair.t_lo, lane);
  const uint32_t p_base = tri_addr(st.pair.p, lane);

  // Y = S k~ (two terms) and O = S q~ (hi term), columns = the chunk's rows.
  float top0 = 0.0f, top1 = 0.0f;
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    top0 = fmaxf(top0, fmaxf(fabsf(S[n][0]), fabsf(S[n][1])));
    top1 = fmaxf(top1, fmaxf(fabsf(S[n][2]), fabsf(S[n][3])));
  }
  float up0, down0, up1, down1;
  row_scale(quad_max(top0), up0, down0);
  row_scale(quad_max(top1), up1, down1);
  float Y[8][4], O[8][4];
#pragma unroll
  for (int n = 0; n < 8; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) Y[n][e] = O[n][e] = 0.0f;
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      split(S[2 * ks + m][0] * up0, S[2 * ks + m][1] * up0, hi[2 * m], lo[2 * m]);
      split(S[2 * ks + m][2] * up1, S[2 * ks + m][3] * up1, hi[2 * m + 1], lo[2 * m + 1]);
    }
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      uint32_t b[4];
      ldsm4(block<kDim>(k_base, nb, ks), b);
      mma(Y[2 * nb], lo, b[0], b[1]);
      mma(Y[2 * nb + 1], lo, b[2], b[3]);
      mma(Y[2 * nb], hi, b[0], b[1]);
      mma(Y[2 * nb + 1], hi, b[2], b[3]);
      ldsm4(block<kDim>(q_base, nb, ks), b);
      mma(O[2 * nb], hi, b[0], b[1]);
      mma(O[2 * nb + 1], hi, b[2], b[3]);
    }
  }

  // R = beta (v - k_in Y), in place.
  top0 = top1 = 0.0f;
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
    uint32_t vt[4];  // v transposed: (rows 16nb.., cols v0..), (.., v0 + 8..), (rows 16nb + 8.., ...)
    ldsm4_t(block<kDim>(v_base, nb, v0 / 16), vt);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int n = 2 * nb + m;
      const float2 kin = *reinterpret_cast<const float2*>(&st.pair.k_in[8 * n + 2 * t]);
      const float2 beta = *reinterpret_cast<const float2*>(&st.pair.beta[8 * n + 2 * t]);
      const uint32_t r0 = vt[2 * m], r1 = vt[2 * m + 1];
      Y[n][0] = beta.x * (__uint_as_float(r0 << 16) - kin.x * (Y[n][0] * down0));
      Y[n][1] = beta.y * (__uint_as_float(r0 & 0xffff0000u) - kin.y * (Y[n][1] * down0));
      Y[n][2] = beta.x * (__uint_as_float(r1 << 16) - kin.x * (Y[n][2] * down1));
      Y[n][3] = beta.y * (__uint_as_float(r1 & 0xffff0000u) - kin.y * (Y[n][3] * down1));
      top0 = fmaxf(top0, fmaxf(fabsf(Y[n][0]), fabsf(Y[n][1])));
      top1 = fmaxf(top1, fmaxf(fabsf(Y[n][2]), fabsf(Y[n][3])));
    }
  }
  // O into fp32 units of the first read-out.
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const float2 qin = *reinterpret_cast<const float2*>(&st.pair.q_in[8 * n + 2 * t]);
    O[n][0] *= qin.x * down0;
    O[n][1] *= qin.y * down0;
    O[n][2] *= qin.x * down1;
    O[n][3] *= qin.y * down1;
  }
  row_scale(quad_max(top0), up0, down0);
  row_scale(quad_max(top1), up1, down1);

  // U = T R (both in two terms; the product of the two lo terms is below fp32's last bit).
  float U[8][4];
  {
    uint32_t hi[4][4], lo[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        split(Y[2 * ks + m][0] * up0, Y[2 * ks + m][1] * up0, hi[ks][2 * m], lo[ks][2 * m]);
        split(Y[2 * ks + m][2] * up1, Y[2 * ks + m][3] * up1, hi[ks][2 * m + 1], lo[ks][2 * m + 1]);
      }
    }
#pragma unroll
    for (int ib = 0; ib < 4; ++ib) {
#pragma unroll
      for (int e = 0; e < 4; ++e) U[2 * ib][e] = U[2 * ib + 1][e] = 0.0f;
#pragma unroll
      for (int ks = 0; ks <= ib; ++ks) {
        uint32_t bh[4], bl[4];
        ldsm4(th_base + tri_block(ib, ks), bh);
        ldsm4(tl_base + tri_block(ib, ks), bl);
        mma(U[2 * ib], hi[ks], bl[0], bl[1]);
        mma(U[2 * ib + 1], hi[ks], bl[2], bl[3]);
        mma(U[2 * ib], lo[ks], bh[0], bh[1]);
        mma(U[2 * ib + 1], lo[ks], bh[2], bh[3]);
        mma(U[2 * ib], hi[ks], bh[0], bh[1]);
        mma(U[2 * ib + 1], hi[ks], bh[2], bh[3]);
      }
    }
  }

  // O += P U (hi term), in units of U's own row scale.
  top0 = top1 = 0.0f;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    U[n][0] *= down0;
    U[n][1] *= down0;
    U[n][2] *= down1;
    U[n][3] *= down1;
    top0 = fmaxf(top0, fmaxf(fabsf(U[n][0]), fabsf(U[n][1])));
    top1 = fmaxf(top1, fmaxf(fabsf(U[n][2]), fabsf(U[n][3])));
  }
  row_scale(quad_max(top0), up0, down0);
  row_scale(quad_max(top1), up1, down1);
  {
    uint32_t hi[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        hi[ks][2 * m] = pack_half(U[2 * ks + m][0] * up0, U[2 * ks + m][1] * up0);
        hi[ks][2 * m + 1] = pack_half(U[2 * ks + m][2] * up1, U[2 * ks + m][3] * up1);
      }
    }
#pragma unroll
    for (int ib = 0; ib < 4; ++ib) {
      float acc[2][4] = {};
#pragma unroll
      for (int ks = 0; ks <= ib; ++ks) {
        uint32_t b[4];
        ldsm4(p_base + tri_block(ib, ks), b);
        mma(acc[0], hi[ks], b[0], b[1]);
        mma(acc[1], hi[ks], b[2], b[3]);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        O[2 * ib + m][0] = fmaf(acc[m][0], down0, O[2 * ib + m][0]);
        O[2 * ib + m][1] = fmaf(acc[m][1], down0, O[2 * ib + m][1]);
        O[2 * ib + m][2] = fmaf(acc[m][2], down1, O[2 * ib + m][2]);
        O[2 * ib + m][3] = fmaf(acc[m][3], down1, O[2 * ib + m][3]);
      }
    }
  }
  wait_o();
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    float* at = o_tile + (8 * n + 2 * t) * kORow + v0 + g;
    at[0] = O[n][0];
    at[kORow] = O[n][1];
    at[8] = O[n][2];
    at[kORow + 8] = O[n][3];
  }
  bar_arrive(kBarOReady);

  // S <- decay S + (k_out u) k~^T, u in two terms.  Each column block sums in fresh accumulators and
  // meets the state in one fp32 fused multiply-add.
  top0 = top1 = 0.0f;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const float2 kout = *reinterpret_cast<const float2*>(&st.pair.k_out[8 * n + 2 * t]);
    U[n][0] *= kout.x;
    U[n][1] *= kout.y;
    U[n][2] *= kout.x;
    U[n][3] *= kout.y;
    top0 = fmaxf(top0, fmaxf(fabsf(U[n][0]), fabsf(U[n][1])));
    top1 = fmaxf(top1, fmaxf(fabsf(U[n][2]), fabsf(U[n][3])));
  }
  row_scale(quad_max(top0), up0, down0);
  row_scale(quad_max(top1), up1, down1);
  {
    uint32_t hi[4][4], lo[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        split(U[2 * ks + m][0] * up0, U[2 * ks + m][1] * up0, hi[ks][2 * m], lo[ks][2 * m]);
        split(U[2 * ks + m][2] * up1, U[2 * ks + m][3] * up1, hi[ks][2 * m + 1], lo[ks][2 * m + 1]);
      }
    }
    const float decay = st.pair.decay;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      float acc[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t b[4];  // k~ transposed: (rows 0-7, cols 0-7), (rows 8-15, cols 0-7), (0-7, 8-15), (8-15, 8-15)
        ldsm4_t(block<kDim>(k_trans, ks, nb), b);
        mma(acc[0], lo[ks], b[0], b[1]);
        mma(acc[1], lo[ks], b[2], b[3]);
        mma(acc[0], hi[ks], b[0], b[1]);
        mma(acc[1], hi[ks], b[2], b[3]);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        S[2 * nb + m][0] = fmaf(S[2 * nb + m][0], decay, acc[m][0] * down0);
        S[2 * nb + m][1] = fmaf(S[2 * nb + m][1], decay, acc[m][1] * down0);
        S[2 * nb + m][2] = fmaf(S[2 * nb + m][2], decay, acc[m][2] * down1);
        S[2 * nb + m][3] = fmaf(S[2 * nb + m][3], decay, acc[m][3] * down1);
      }
    }
  }
}

template <typename StateT, bool kVec>
__global__ void __launch_bounds__(kChainThreads, 1) gdn_prefill_chain_kernel(const PrefillArgs p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  ChainSmem& s = *reinterpret_cast<ChainSmem*>(raw);
  grid_dependency_wait();
  allow_dependent_launch();
  const int64_t r = blockIdx.x / p.num_v_heads;
  const int head = static_cast<int>(blockIdx.x - r * p.num_v_heads);
  Request rq;
  unsigned int fault;
  bool skip;
  if (!find_request(p, r, rq, fault, skip)) {
    if (fault != 0 && threadIdx.x == 0 && head == 0) atomicOr(&g_prefill_faults, fault);
    if (skip) return;
    for (int64_t i = threadIdx.x; i < rq.tokens * kDim; i += kChainThreads) {
      p.out[((rq.first + i / kDim) * p.num_v_heads + head) * kDim + i % kDim] = __float2bfloat16_rn(0.0f);
    }
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Launched with 384 x 168 registers; 128 x 88 + 256 x 208 is the same 64,512.
  if (warp < kCopyThreads / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int tid = threadIdx.x;
    const int64_t base = chunk_base(rq.first, r);
    float wt[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) wt[e] = load_param(p.weight, 64 * (e >> 2) + 4 * (lane & 15) + (e & 3), p.weight_bf16);
    // Chunk c is copied in while the chain works on chunk c - 1, then chunk c - 1's outputs are stored.
    for (int64_t c = 0; c <= rq.chunks; ++c) {
      if (c < rq.chunks) {
        const int stage = static_cast<int>(c & 1);
        if (c >= 2) bar_sync(kBarEmpty + stage);
        copy_chunk<kVec>(p, s.stage[stage], rq, c, base + c, head, tid);
        cp_async_wait();
        bar_arrive(kBarFull + stage);
      }
      if (c >= 1) {
        store_outputs<kVec>(p, s, rq, c - 1, head, wt, tid, [] { bar_sync(kBarOReady); });
        if (c < rq.chunks) bar_arrive(kBarOFree);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int g = lane >> 2, t = lane & 3;
    const int v0 = 16 * (warp - kCopyThreads / 32);
    StateT* pool = static_cast<StateT*>(p.state) + static_cast<int64_t>(head) * kDim * kDim + (v0 + g) * kDim + 2 * t;
    float S[16][4];
    if (rq.source > 0) {
      const StateT* at = pool + rq.source * p.slot_stride;
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        load_pair(at + 8 * n, S[n][0], S[n][1]);
        load_pair(at + 8 * kDim + 8 * n, S[n][2], S[n][3]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < 16; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) S[n][e] = 0.0f;
      }
    }
    // Chunks end at absolute positions that are multiples of 64, and so do blocks.
    const int64_t per_block = p.block_size / kChunk;
    const int32_t* slot_at = rq.row + rq.context / p.block_size;
    int64_t left = per_block - (rq.context / kChunk) % per_block;
    for (int64_t c = 0; c < rq.chunks; ++c) {
      const int stage = static_cast<int>(c & 1);
      bar_sync(kBarFull + stage);
      chain_chunk(S, s.stage[stage], s.o, v0, lane, [&] {
        if (c >= 1) bar_sync(kBarOFree);
      });
      if (c + 2 < rq.chunks) bar_arrive(kBarEmpty + stage);
      if (c + 1 == rq.chunks || --left == 0) {  // a block or the request ends here: its slot takes the state
        const int32_t slot = *slot_at++;
        left = per_block;
        if (slot > 0 && slot < p.n_slots) {
          StateT* at = pool + slot * p.slot_stride;
#pragma unroll
          for (int n = 0; n < 16; ++n) {
            store_pair(at + 8 * n, S[n][0], S[n][1]);
            store_pair(at + 8 * kDim + 8 * n, S[n][2], S[n][3]);
          }
        } else if (slot >= p.n_slots && head == 0 && lane == 0) {
          atomicOr(&g_prefill_faults, LD_FAULT_DECODE_SLOT_RANGE);
        }
      }
    }
  }
}

bool aligned(const void* ptr, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }

int64_t chunk_places(int64_t n_tokens, int64_t n_requests) { return chunk_base(n_tokens, n_requests); }

int64_t workspace_bytes(int64_t n_tokens, int64_t n_requests, int64_t num_k_heads, int64_t num_v_heads) {
  const int64_t per_place = num_k_heads * static_cast<int64_t>(sizeof(KeyImage)) +
                            num_v_heads * static_cast<int64_t>(sizeof(PairImage));
  return chunk_places(n_tokens, n_requests) * per_place;
}

template <typename StateT, bool kVec>
cudaError_t launch_prefill(const PrefillArgs& args, cudaStream_t stream) {
  // Set on every call: the attributes belong to the current device, and setting them is a table write.
  auto pairs = gdn_prefill_pairs_kernel<kVec>;
  cudaError_t err = cudaFuncSetAttribute(pairs, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(PairSmem));
  if (err != cudaSuccess) return err;
  auto chain = gdn_prefill_chain_kernel<StateT, kVec>;
  err = cudaFuncSetAttribute(chain, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ChainSmem));
  if (err != cudaSuccess) return err;
  const int64_t places = chunk_places(args.n_tokens, args.n_requests);
  err = launch(pairs, dim3(static_cast<unsigned int>(places * args.num_k_heads)), dim3(kPairThreads), sizeof(PairSmem),
               stream, 1, args);
  if (err != cudaSuccess) return err;
  return launch(chain, dim3(static_cast<unsigned int>(args.n_requests) * args.num_v_heads), dim3(kChainThreads),
                sizeof(ChainSmem), stream, 1, args);
}

}  // namespace

int prefill_faults(uint32_t* flags, int clear) {
  uint32_t value = 0;
  cudaError_t err = cudaMemcpyFromSymbol(&value, g_prefill_faults, sizeof(value));
  if (err == cudaSuccess && clear) {
    const uint32_t zero = 0;
    err = cudaMemcpyToSymbol(g_prefill_faults, &zero, sizeof(zero));
  }
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "ld_fault_flags: %s", cudaGetErrorString(err));
  *flags = value;
  return LD_OK;
}

}  // namespace ldb

extern "C" int64_t ld_prefill_workspace(int64_t n_tokens, int64_t n_requests, int64_t num_k_heads,
                                        int64_t num_v_heads) {
  if (n_tokens < 0 || n_requests < 0 || num_k_heads < 1 || num_v_heads < 1 || n_tokens > INT32_MAX ||
      n_requests > INT32_MAX || num_k_heads > 65536 || num_v_heads > 65536) {
    return -ldb::set_error(LD_ERR_INVALID, "prefill workspace: token, request or head count out of range");
  }
  ldb::ok();
  return ldb::workspace_bytes(n_tokens, n_requests, num_k_heads, num_v_heads);
}

extern "C" int ld_prefill(const void* qkv, int64_t qkv_row_stride, const void* a, int64_t a_row_stride, const void* b,
                          int64_t b_row_stride, const float* a_log, const void* dt_bias, int dt_bias_dtype,
                          const int32_t* table, int64_t table_row_stride, int64_t table_width, int64_t block_size,
                          const int32_t* context, const int32_t* cu, int64_t n_requests, void* state,
                          int state_dtype, int64_t n_slots, int64_t slot_stride, const void* gate,
                          int64_t gate_row_stride, const void* weight, int weight_dtype, void* out, int64_t n_tokens,
                          int64_t num_k_heads, int64_t num_v_heads, float eps, void* workspace,
                          int64_t workspace_size, void* stream) {
  using namespace ldb;
  if (num_k_heads < 1 || num_v_heads < 1 || num_v_heads > 65536 || num_v_heads % num_k_heads != 0) {
    return set_error(LD_ERR_INVALID, "prefill: num_v_heads must be a positive multiple of num_k_heads");
  }
  if (!(eps > 0.0f)) return set_error(LD_ERR_INVALID, "prefill: norm epsilon must be positive");
  if (block_size < 1 || block_size % kChunk != 0) {
    return set_error(LD_ERR_INVALID, "prefill: block_size must be a positive multiple of %d", kChunk);
  }
  if (n_requests < 0 || n_tokens < 0 || n_requests > INT32_MAX / num_v_heads || n_tokens > INT32_MAX ||
      chunk_places(n_tokens, n_requests) > INT32_MAX / num_v_heads) {
    return set_error(LD_ERR_INVALID, "prefill: request or token count out of range");
  }
  for (const int dtype : {dt_bias_dtype, weight_dtype, state_dtype}) {
    if (dtype != LD_DTYPE_F32 && dtype != LD_DTYPE_BF16) {
      return set_error(LD_ERR_INVALID, "prefill: state, dt_bias and weight are fp32 or bf16");
    }
  }
  const bool bf16_pool = state_dtype == LD_DTYPE_BF16;
  const int64_t slot_elems = num_v_heads * kDim * kDim;
  if (n_slots < 1 || slot_stride < slot_elems || slot_stride % (bf16_pool ? 8 : 4) != 0) {
    return set_error(LD_ERR_INVALID,
                     "prefill: the pool needs at least one slot and a slot stride of at least HV*128*128 elements, "
                     "divisible by 4 (fp32) or 8 (bf16)");
  }
  if (table_width < 1 || table_row_stride < table_width) {
    return set_error(LD_ERR_INVALID, "prefill: the table needs at least one block per row and rows that do not overlap");
  }
  if (qkv_row_stride < (2 * num_k_heads + num_v_heads) * kDim || a_row_stride < num_v_heads ||
      b_row_stride < num_v_heads || gate_row_stride < num_v_heads * kDim) {
    return set_error(LD_ERR_INVALID, "prefill: activation row strides are smaller than the rows");
  }
  if (n_requests == 0 || n_tokens == 0) return ok();
  for (const void* ptr : {qkv, a, b, static_cast<const void*>(a_log), dt_bias, static_cast<const void*>(table),
                          static_cast<const void*>(context), static_cast<const void*>(cu),
                          static_cast<const void*>(state), gate, weight, static_cast<const void*>(out)}) {
    if (ptr == nullptr) return set_error(LD_ERR_INVALID, "prefill: a required pointer is NULL");
  }
  const int64_t needed = workspace_bytes(n_tokens, n_requests, num_k_heads, num_v_heads);
  if (workspace == nullptr || !aligned(workspace, 128) || workspace_size < needed) {
    return set_error(LD_ERR_INVALID, "prefill: needs a 128-byte aligned workspace of %lld bytes (got %lld)",
                     static_cast<long long>(needed), static_cast<long long>(workspace == nullptr ? 0 : workspace_size));
  }
  if (!aligned(state, 16) || !aligned(qkv, 2) || !aligned(a, 2) || !aligned(b, 2) || !aligned(gate, 2) ||
      !aligned(out, 2)) {
    return set_error(LD_ERR_INVALID, "prefill: the pool must be 16-byte aligned and bf16 tensors 2-byte aligned");
  }
  PrefillArgs args;
  args.qkv = static_cast<const __nv_bfloat16*>(qkv);
  args.qkv_row = qkv_row_stride;
  args.a = static_cast<const __nv_bfloat16*>(a);
  args.a_row = a_row_stride;
  args.b = static_cast<const __nv_bfloat16*>(b);
  args.b_row = b_row_stride;
  args.a_log = a_log;
  args.dt_bias = dt_bias;
  args.table = table;
  args.table_row = table_row_stride;
  args.table_width = table_width;
  args.context = context;
  args.cu = cu;
  args.state = state;
  args.n_slots = n_slots;
  args.slot_stride = slot_stride;
  args.gate = static_cast<const __nv_bfloat16*>(gate);
  args.gate_row = gate_row_stride;
  args.weight = weight;
  args.out = static_cast<__nv_bfloat16*>(out);
  args.n_tokens = n_tokens;
  args.block_size = block_size;
  args.keys = static_cast<KeyImage*>(workspace);
  args.pairs = reinterpret_cast<PairImage*>(args.keys + chunk_places(n_tokens, n_requests) * num_k_heads);
  args.n_requests = static_cast<int>(n_requests);
  args.num_k_heads = static_cast<int>(num_k_heads);
  args.num_v_heads = static_cast<int>(num_v_heads);
  args.heads_ratio = static_cast<int>(num_v_heads / num_k_heads);
  args.dt_bias_bf16 = dt_bias_dtype == LD_DTYPE_BF16;
  args.weight_bf16 = weight_dtype == LD_DTYPE_BF16;
  args.q_scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(kDim)));
  args.eps = eps;
  // 16-byte copies of the q, k, v rows and 8-byte accesses to gate and out where every row allows them.
  const bool vec = aligned(qkv, 16) && qkv_row_stride % 8 == 0 && aligned(gate, 8) && gate_row_stride % 4 == 0 &&
                   aligned(out, 8);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  if (bf16_pool) {
    err = vec ? launch_prefill<__nv_bfloat16, true>(args, s) : launch_prefill<__nv_bfloat16, false>(args, s);
  } else {
    err = vec ? launch_prefill<float, true>(args, s) : launch_prefill<float, false>(args, s);
  }
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "prefill launch failed: %s", cudaGetErrorString(err));
  return ok();
}
