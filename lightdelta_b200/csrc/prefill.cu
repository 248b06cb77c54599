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
// Layout.  One CTA of 12 warps per (request, value head).  Eight chain warps hold the 128 x 128 state
// as accumulator fragments, 16 value rows each: S k, T R and the update all have the state's value
// rows as M, so every warp carries its rows through all chunks without exchanging anything with the
// others (an accumulator fragment is the next product's A fragment).  Four prep warps work one chunk
// ahead: load and scale q and k, form L, P and T, and normalise and store the chunk before's outputs.
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
constexpr int kPrepThreads = 128;
constexpr int kChainWarps = 8;
constexpr int kThreads = kPrepThreads + 32 * kChainWarps;
constexpr int kORow = kDim + 4;  // floats per row of the output tile: the +4 spreads its rows over the banks
static_assert(kChunk == 64, "fragment loops below are written for chunks of 64 tokens");

__device__ unsigned int g_prefill_faults;

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
  int num_k_heads;
  int num_v_heads;
  int heads_ratio;
  int dt_bias_bf16;
  int weight_bf16;
  float q_scale;
  float eps;
};

// What one chunk's prep leaves for the chain.
struct Stage {
  __align__(128) __half k[kChunk * kDim];          // k rows x 2^-e, swizzled
  __align__(128) __half q[kChunk * kDim];          // q rows x 2^-e, swizzled
  __align__(128) __nv_bfloat16 v[kChunk * kDim];   // swizzled
  __align__(128) __half t_hi[kChunk * kChunk];     // T, lower 16 x 16 blocks, swizzled
  __align__(128) __half t_lo[kChunk * kChunk];
  __align__(128) __half p[kChunk * kChunk];        // P, lower 16 x 16 blocks, swizzled
  float beta[kChunk];
  float k_in[kChunk];   // e^{G_i} fk_i: scales S k~
  float q_in[kChunk];   // e^{G_i} fq_i 128^-1/2: scales S q~
  float k_out[kChunk];  // e^{G_C - G_j} fk_j: scales u_j on its way into the state
  float decay;          // e^{G_C}
};

struct Smem {
  Stage stage[2];
  __align__(128) __half l_hi[kChunk * kChunk];  // L below the diagonal blocks
  __align__(128) __half l_lo[kChunk * kChunk];
  __align__(16) float diag[4][16 * 16];         // L's diagonal blocks
  __align__(16) float o[kChunk * kORow];
  float g_hi[kChunk], g_lo[kChunk];
  float fk[kChunk], fq[kChunk];
};

// The request's place in the launch; `live` is false when it writes nothing further.
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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int kId, int kCount>
__device__ __forceinline__ void bar_sync() {
  asm volatile("bar.sync %0, %1;" ::"n"(kId), "n"(kCount) : "memory");
}
__device__ __forceinline__ void bar_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kThreads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kThreads) : "memory");
}
// Named barriers: 1 joins the prep warps; the others hand buffers between prep and chain.
constexpr int kBarPrep = 1, kBarFull = 2, kBarEmpty = 4, kBarOReady = 6, kBarOFree = 7;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int bytes = live ? 16 : 0;  // 0: the 16 bytes are filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// Address that this lane gives to ldmatrix.x4 for the 16 x 16 block at (row0, col0): matrices in the
// order (rows 0-7, cols 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15), or with kRowsFirst
// (0-7, 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15).
template <int kCols, bool kRowsFirst>
__device__ __forceinline__ uint32_t block_addr(uint32_t base, int row0, int col0, int lane) {
  const int m = lane >> 3;
  const int r = row0 + (lane & 7) + 8 * (kRowsFirst ? (m & 1) : (m >> 1));
  const int c = col0 + 8 * (kRowsFirst ? (m >> 1) : (m & 1));
  return base + 2 * swz<kCols>(r, c);
}

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

// ------------------------------------------------------------------------------------------
// prep: one chunk's operands
// ------------------------------------------------------------------------------------------
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

// Scales this thread's pieces of the tile's rows from bf16 to fp16 in place (rows are exact: a power
// of two per row brings the largest magnitude to [1, 2)) and leaves each row's factor, its L2 norm's
// reciprocal times that power, in `factor`.
__device__ __forceinline__ void scale_rows(uint16_t* tile, float* factor, int tid) {
#pragma unroll
  for (int pass = 0; pass < kChunk / 8; ++pass) {
    const int i = pass * 8 + (tid >> 4);
    uint16_t* piece = tile + swz<kDim>(i, (tid & 15) * 8);
    const uint4 raw = *reinterpret_cast<const uint4*>(piece);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = __uint_as_float(w[e] << 16);
      x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum = fmaf(x[e], x[e], sum);
      top = fmaxf(top, fabsf(x[e]));
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, off);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xff);
    e = min(max(e, 1), 253);
    const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);  // 2^(127 - e)
    const float up = __uint_as_float(static_cast<uint32_t>(e) << 23);
    uint4 y;
    y.x = pack_half(x[0] * down, x[1] * down);
    y.y = pack_half(x[2] * down, x[3] * down);
    y.z = pack_half(x[4] * down, x[5] * down);
    y.w = pack_half(x[6] * down, x[7] * down);
    *reinterpret_cast<uint4*>(piece) = y;
    if ((tid & 15) == 0) factor[i] = up * (1.0f / sqrtf(sum + 1e-6f));
  }
}

// g and beta of the chunk's tokens and G's running sums, by one warp (lane: rows lane and lane + 32).
__device__ __forceinline__ void chunk_gates(const PrefillArgs& p, Smem& s, Stage& st, int64_t token0, int row_lo,
                                            int row_hi, int head, int lane) {
  const float rate = -expf(p.a_log[head]);
  const float bias = load_param(p.dt_bias, head, p.dt_bias_bf16);
  double sum[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = lane + 32 * half;
    float g = 0.0f, beta = 0.0f;
    if (i >= row_lo && i < row_hi) {
      g = rate * softplus(__bfloat162float(p.a[(token0 + i) * p.a_row + head]) + bias);
      // e^-1000 is 0 in fp32: a floor keeps differences of sums finite and changes no value.
      if (g < -1000.0f) g = -1000.0f;
      beta = 1.0f / (1.0f + expf(-__bfloat162float(p.b[(token0 + i) * p.b_row + head])));
    }
    st.beta[i] = beta;
    double x = static_cast<double>(g);
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
    s.g_hi[lane + 32 * half] = hi;
    s.g_lo[lane + 32 * half] = static_cast<float>(sum[half] - static_cast<double>(hi));
  }
}

// L (kKeys) or P of this warp's 16 rows from the products of the scaled rows.
template <bool kKeys>
__device__ __forceinline__ void pair_products(Smem& s, Stage& st, int w, int lane, float q_scale) {
  const uint32_t a_base = smem_u32(kKeys ? st.k : st.q), b_base = smem_u32(st.k);
  float acc[8][4];
#pragma unroll
  for (int n = 0; n < 8; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    uint32_t a[4];
    ldsm4(block_addr<kDim, true>(a_base, 16 * w, 16 * ks, lane), a);
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      if (nb <= w) {
        uint32_t b[4];
        ldsm4(block_addr<kDim, false>(b_base, 16 * nb, 16 * ks, lane), b);
        mma(acc[2 * nb], a, b[0], b[1]);
        mma(acc[2 * nb + 1], a, b[2], b[3]);
      }
    }
  }
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = 16 * w + g + 8 * half;
    const float gi_hi = s.g_hi[i], gi_lo = s.g_lo[i];
    const float row = kKeys ? st.beta[i] * s.fk[i] : q_scale * s.fq[i];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      if (n / 2 > w) continue;
      float x[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = 8 * n + 2 * t + e;
        const bool in = kKeys ? j < i : j <= i;
        const float d = expf((gi_hi - s.g_hi[j]) + (gi_lo - s.g_lo[j]));
        x[e] = in ? row * s.fk[j] * d * acc[n][2 * half + e] : 0.0f;
      }
      const int j = 8 * n + 2 * t;
      if constexpr (kKeys) {
        if (n / 2 == w) {
          *reinterpret_cast<float2*>(&s.diag[w][(g + 8 * half) * 16 + (j & 15)]) = make_float2(x[0], x[1]);
        } else {
          uint32_t hi, lo;
          split(x[0], x[1], hi, lo);
          *reinterpret_cast<uint32_t*>(&s.l_hi[swz<kChunk>(i, j)]) = hi;
          *reinterpret_cast<uint32_t*>(&s.l_lo[swz<kChunk>(i, j)]) = lo;
        }
      } else {
        *reinterpret_cast<uint32_t*>(&st.p[swz<kChunk>(i, j)]) = pack_half(x[0], x[1]);
      }
    }
  }
}

// Inverse of this warp's diagonal block of I + L by forward substitution, one column per lane.
__device__ __forceinline__ void invert_diagonal(Smem& s, Stage& st, int w, int lane) {
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
      st.t_hi[swz<kChunk>(16 * w + i, 16 * w + c)] = hi;
      st.t_lo[swz<kChunk>(16 * w + i, 16 * w + c)] = __float2half_rn(x[i] - __half2float(hi));
    }
  }
}

// The 16 x 16 blocks of T below diagonal block w, top to bottom:
//   T_iw = -T_ii sum_{k=w}^{i-1} L_ik T_kw,  held transposed so that each result is the next A operand.
__device__ __forceinline__ void invert_column(Smem& s, Stage& st, int w, int lane) {
  const uint32_t t_hi = smem_u32(st.t_hi), t_lo = smem_u32(st.t_lo);
  const uint32_t l_hi = smem_u32(s.l_hi), l_lo = smem_u32(s.l_lo);
  uint32_t x_hi[3][4], x_lo[3][4];  // T_kw^T as A fragments, k = w, w + 1, w + 2
  // ldmatrix.trans of T_ww: matrices (cols 0-7, rows 0-7), (cols 8-15, rows 0-7), (0-7, 8-15), (8-15, 8-15).
  ldsm4_t(block_addr<kChunk, false>(t_hi, 16 * w, 16 * w, lane), x_hi[0]);
  ldsm4_t(block_addr<kChunk, false>(t_lo, 16 * w, 16 * w, lane), x_lo[0]);
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    const int i = w + d;
    if (i < 4) {
      float m[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < d; ++kk) {
        uint32_t b_hi[4], b_lo[4];
        ldsm4(block_addr<kChunk, false>(l_hi, 16 * i, 16 * (w + kk), lane), b_hi);
        ldsm4(block_addr<kChunk, false>(l_lo, 16 * i, 16 * (w + kk), lane), b_lo);
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
      ldsm4(block_addr<kChunk, false>(t_hi, 16 * i, 16 * i, lane), b_hi);
      ldsm4(block_addr<kChunk, false>(t_lo, 16 * i, 16 * i, lane), b_lo);
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
          st.t_hi[swz<kChunk>(row, col)] = __low2half(h);
          st.t_hi[swz<kChunk>(row + 1, col)] = __high2half(h);
          st.t_lo[swz<kChunk>(row, col)] = __low2half(l);
          st.t_lo[swz<kChunk>(row + 1, col)] = __high2half(l);
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

template <bool kVec>
__device__ void prepare_chunk(const PrefillArgs& p, Smem& s, Stage& st, const Request& rq, int64_t chunk, int head,
                              int tid) {
  const int w = tid >> 5, lane = tid & 31;
  // Row i of the chunk is token token0 + i; rows outside [row_lo, row_hi) belong to no token.
  const int64_t local0 = chunk * kChunk - rq.lead;
  const int64_t token0 = rq.first + local0;
  const int row_lo = chunk == 0 ? rq.lead : 0;
  const int row_hi = static_cast<int>(min(static_cast<int64_t>(kChunk), rq.tokens - local0));
  const int kh = head / p.heads_ratio;
  const __nv_bfloat16* rows = p.qkv + token0 * p.qkv_row;
  load_rows<kVec>(rows + (p.num_k_heads + kh) * kDim, p.qkv_row, row_lo, row_hi, reinterpret_cast<uint16_t*>(st.k), tid);
  load_rows<kVec>(rows + kh * kDim, p.qkv_row, row_lo, row_hi, reinterpret_cast<uint16_t*>(st.q), tid);
  load_rows<kVec>(rows + (2 * p.num_k_heads + head) * kDim, p.qkv_row, row_lo, row_hi,
                  reinterpret_cast<uint16_t*>(st.v), tid);
  if (w == 0) chunk_gates(p, s, st, token0, row_lo, row_hi, head, lane);
  if constexpr (kVec) cp_async_wait();
  scale_rows(reinterpret_cast<uint16_t*>(st.k), s.fk, tid);  // each thread scales the pieces that it loaded
  scale_rows(reinterpret_cast<uint16_t*>(st.q), s.fq, tid);
  bar_sync<kBarPrep, kPrepThreads>();
  if (tid < kChunk) {
    const float in = expf(s.g_hi[tid] + s.g_lo[tid]);
    st.k_in[tid] = in * s.fk[tid];
    st.q_in[tid] = in * s.fq[tid] * p.q_scale;
    const float left = (s.g_hi[kChunk - 1] - s.g_hi[tid]) + (s.g_lo[kChunk - 1] - s.g_lo[tid]);
    st.k_out[tid] = expf(left) * s.fk[tid];
    if (tid == kChunk - 1) st.decay = in;
  }
  pair_products<true>(s, st, w, lane, p.q_scale);
  pair_products<false>(s, st, w, lane, p.q_scale);
  __syncwarp();
  invert_diagonal(s, st, w, lane);
  bar_sync<kBarPrep, kPrepThreads>();
  invert_column(s, st, w, lane);
}

// Gated RMSNorm of the chunk's outputs: warp w takes rows w, w + 4, ...; four values per lane.
template <bool kVec>
__device__ void store_outputs(const PrefillArgs& p, const Smem& s, const Request& rq, int64_t chunk, int head,
                              const float (&wt)[4], int tid) {
  const int w = tid >> 5, lane = tid & 31;
  const int64_t local0 = chunk * kChunk - rq.lead;
  const int row_lo = chunk == 0 ? rq.lead : 0;
  const int row_hi = static_cast<int>(min(static_cast<int64_t>(kChunk), rq.tokens - local0));
#pragma unroll 4
  for (int i = w; i < kChunk; i += 4) {
    if (i < row_lo || i >= row_hi) continue;
    const int64_t token = rq.first + local0 + i;
    const __nv_bfloat16* zrow = p.gate + token * p.gate_row + head * kDim + 4 * lane;
    float z[4];
    if constexpr (kVec) {
      const uint2 raw = *reinterpret_cast<const uint2*>(zrow);
      z[0] = __uint_as_float(raw.x << 16);
      z[1] = __uint_as_float(raw.x & 0xffff0000u);
      z[2] = __uint_as_float(raw.y << 16);
      z[3] = __uint_as_float(raw.y & 0xffff0000u);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = __bfloat162float(zrow[e]);
    }
    const float4 o = *reinterpret_cast<const float4*>(&s.o[i * kORow + 4 * lane]);
    float sq = o.x * o.x + o.y * o.y + o.z * o.z + o.w * o.w;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    const float rstd = 1.0f / sqrtf(sq / static_cast<float>(kDim) + p.eps);
    const float x[4] = {o.x, o.y, o.z, o.w};
    __align__(8) __nv_bfloat16 y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __float2bfloat16_rn(x[e] * rstd * wt[e] * (z[e] / (1.0f + expf(-z[e]))));
    __nv_bfloat16* at = p.out + (token * p.num_v_heads + head) * kDim + 4 * lane;
    if constexpr (kVec) {
      *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(y);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) at[e] = y[e];
    }
  }
}

// ------------------------------------------------------------------------------------------
// chain: the state through one chunk, 16 value rows per warp
// ------------------------------------------------------------------------------------------
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
  const uint32_t k_base = smem_u32(st.k), q_base = smem_u32(st.q), v_base = smem_u32(st.v);
  const uint32_t th_base = smem_u32(st.t_hi), tl_base = smem_u32(st.t_lo), p_base = smem_u32(st.p);

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
      ldsm4(block_addr<kDim, false>(k_base, 16 * nb, 16 * ks, lane), b);
      mma(Y[2 * nb], lo, b[0], b[1]);
      mma(Y[2 * nb + 1], lo, b[2], b[3]);
      mma(Y[2 * nb], hi, b[0], b[1]);
      mma(Y[2 * nb + 1], hi, b[2], b[3]);
      ldsm4(block_addr<kDim, false>(q_base, 16 * nb, 16 * ks, lane), b);
      mma(O[2 * nb], hi, b[0], b[1]);
      mma(O[2 * nb + 1], hi, b[2], b[3]);
    }
  }

  // R = beta (v - k_in Y), in place.
  top0 = top1 = 0.0f;
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
    uint32_t vt[4];  // v transposed: (rows 16nb.., cols v0..), (.., v0 + 8..), (rows 16nb + 8.., ...)
    ldsm4_t(block_addr<kDim, false>(v_base, 16 * nb, v0, lane), vt);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int n = 2 * nb + m;
      const float2 kin = *reinterpret_cast<const float2*>(&st.k_in[8 * n + 2 * t]);
      const float2 beta = *reinterpret_cast<const float2*>(&st.beta[8 * n + 2 * t]);
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
    const float2 qin = *reinterpret_cast<const float2*>(&st.q_in[8 * n + 2 * t]);
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
        ldsm4(block_addr<kChunk, false>(th_base, 16 * ib, 16 * ks, lane), bh);
        ldsm4(block_addr<kChunk, false>(tl_base, 16 * ib, 16 * ks, lane), bl);
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
        ldsm4(block_addr<kChunk, false>(p_base, 16 * ib, 16 * ks, lane), b);
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
    const float2 kout = *reinterpret_cast<const float2*>(&st.k_out[8 * n + 2 * t]);
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
    const float decay = st.decay;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      float acc[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t b[4];  // k~ transposed: (rows 0-7, cols 0-7), (rows 8-15, cols 0-7), (0-7, 8-15), (8-15, 8-15)
        ldsm4_t(block_addr<kDim, true>(k_base, 16 * ks, 16 * nb, lane), b);
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

// The request of this CTA, or false when there is nothing to compute (after reporting a fault and
// zeroing the outputs of a request that cannot run).
__device__ bool find_request(const PrefillArgs& p, int64_t r, int head, Request& rq) {
  const int64_t begin = p.cu[r], end = p.cu[r + 1];
  if (end <= begin) return false;
  if (begin < 0 || end > p.n_tokens) {
    if (threadIdx.x == 0 && head == 0) atomicOr(&g_prefill_faults, LD_FAULT_DECODE_TOKENS);
    return false;
  }
  rq.first = begin;
  rq.tokens = end - begin;
  rq.context = p.context[r];
  rq.row = p.table + r * p.table_row;
  unsigned int fault = 0;
  bool ok = rq.context >= 0;
  if (!ok || (rq.context + rq.tokens - 1) / p.block_size >= p.table_width) {
    fault = LD_FAULT_TABLE_BLOCKS;
    ok = false;
  }
  rq.source = 0;
  if (ok && rq.context > 0) {
    rq.source = rq.row[(rq.context - 1) / p.block_size];
    if (rq.source >= p.n_slots) fault = LD_FAULT_DECODE_SLOT_RANGE;
    ok = rq.source > 0 && rq.source < p.n_slots;
  }
  if (!ok) {
    if (fault != 0 && threadIdx.x == 0 && head == 0) atomicOr(&g_prefill_faults, fault);
    for (int64_t i = threadIdx.x; i < rq.tokens * kDim; i += kThreads) {
      p.out[((begin + i / kDim) * p.num_v_heads + head) * kDim + i % kDim] = __float2bfloat16_rn(0.0f);
    }
    return false;
  }
  rq.lead = static_cast<int>(rq.context % kChunk);
  rq.chunks = (rq.lead + rq.tokens + kChunk - 1) / kChunk;
  return true;
}

template <typename StateT, bool kVec>
__global__ void __launch_bounds__(kThreads, 1) gdn_prefill_kernel(const PrefillArgs p) {
  extern __shared__ __align__(128) unsigned char raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  grid_dependency_wait();
  allow_dependent_launch();
  const int64_t r = blockIdx.x / p.num_v_heads;
  const int head = static_cast<int>(blockIdx.x - r * p.num_v_heads);
  Request rq;
  if (!find_request(p, r, head, rq)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Launched with 384 x 168 registers; 128 x 88 + 256 x 208 is the same 64,512.
  if (warp < kPrepThreads / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int tid = threadIdx.x;
    float wt[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) wt[e] = load_param(p.weight, 4 * lane + e, p.weight_bf16);
    prepare_chunk<kVec>(p, s, s.stage[0], rq, 0, head, tid);
    bar_arrive(kBarFull);
    for (int64_t c = 0; c < rq.chunks; ++c) {
      if (c + 1 < rq.chunks) {
        const int next = static_cast<int>((c + 1) & 1);
        if (c >= 1) bar_sync(kBarEmpty + next);
        prepare_chunk<kVec>(p, s, s.stage[next], rq, c + 1, head, tid);
        bar_arrive(kBarFull + next);
      }
      bar_sync(kBarOReady);
      store_outputs<kVec>(p, s, rq, c, head, wt, tid);
      if (c + 1 < rq.chunks) bar_arrive(kBarOFree);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int g = lane >> 2, t = lane & 3;
    const int v0 = 16 * (warp - kPrepThreads / 32);
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
    for (int64_t c = 0; c < rq.chunks; ++c) {
      const int stage = static_cast<int>(c & 1);
      bar_sync(kBarFull + stage);
      chain_chunk(S, s.stage[stage], s.o, v0, lane, [&] {
        if (c >= 1) bar_sync(kBarOFree);
      });
      if (c + 2 < rq.chunks) bar_arrive(kBarEmpty + stage);
      // The state after the chunk's last token belongs to a slot when a block or the request ends there.
      const int64_t end = min(rq.context - rq.lead + (c + 1) * kChunk, rq.context + rq.tokens);
      if (c + 1 == rq.chunks || end % p.block_size == 0) {
        const int32_t slot = rq.row[(end - 1) / p.block_size];
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

template <typename StateT, bool kVec>
cudaError_t launch_prefill(const PrefillArgs& args, int64_t n_requests, cudaStream_t stream) {
  auto kernel = gdn_prefill_kernel<StateT, kVec>;
  // Set on every call: the attribute belongs to the current device, and setting it is a table write.
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem));
  if (err != cudaSuccess) return err;
  const dim3 grid(static_cast<unsigned int>(n_requests * args.num_v_heads));
  return launch(kernel, grid, dim3(kThreads), sizeof(Smem), stream, 1, args);
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

extern "C" int ld_prefill(const void* qkv, int64_t qkv_row_stride, const void* a, int64_t a_row_stride, const void* b,
                          int64_t b_row_stride, const float* a_log, const void* dt_bias, int dt_bias_dtype,
                          const int32_t* table, int64_t table_row_stride, int64_t table_width, int64_t block_size,
                          const int32_t* context, const int32_t* cu, int64_t n_requests, void* state,
                          int state_dtype, int64_t n_slots, int64_t slot_stride, const void* gate,
                          int64_t gate_row_stride, const void* weight, int weight_dtype, void* out, int64_t n_tokens,
                          int64_t num_k_heads, int64_t num_v_heads, float eps, void* stream) {
  using namespace ldb;
  if (num_k_heads < 1 || num_v_heads < 1 || num_v_heads % num_k_heads != 0) {
    return set_error(LD_ERR_INVALID, "prefill: num_v_heads must be a positive multiple of num_k_heads");
  }
  if (!(eps > 0.0f)) return set_error(LD_ERR_INVALID, "prefill: norm epsilon must be positive");
  if (block_size < 1 || block_size % kChunk != 0) {
    return set_error(LD_ERR_INVALID, "prefill: block_size must be a positive multiple of %d", kChunk);
  }
  if (n_requests < 0 || n_tokens < 0 || n_requests > INT32_MAX / num_v_heads || n_tokens > INT32_MAX) {
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
    err = vec ? launch_prefill<__nv_bfloat16, true>(args, n_requests, s)
              : launch_prefill<__nv_bfloat16, false>(args, n_requests, s);
  } else {
    err = vec ? launch_prefill<float, true>(args, n_requests, s) : launch_prefill<float, false>(args, n_requests, s);
  }
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "prefill launch failed: %s", cudaGetErrorString(err));
  return ok();
}
