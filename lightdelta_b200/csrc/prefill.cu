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
// fp32 accumulation.  q and k rows are bf16 and become fp16 after scaling by a power of two per row (which
// the fp32 factors fk, fq undo), exactly but for elements below 2^-30 of their row's largest.  All other
// operands (S, R, u, T, L, P) go in as two fp16 terms, hi + lo, 22 bits together (P 19), after scaling each
// state row by a power of two, so the state follows the fp32 recurrence to under 1e-6, and so do the outputs
// until they are rounded to bf16.  (With one term for S q and P u, 11 bits, one output in ten was rounded
// elsewhere, and where a query is nearly orthogonal to what the state holds, or a chunk's keys are all but
// equal, the gated norm made that a few 1e-3 to 1e-2 of the output; that took 377 us for the 24 prompts
// below.)  G is summed in fp64 and kept as two floats, so differences of large sums stay exact to fp32.
//
// Two kernels.  What does not depend on the state is computed first, for all chunks side by side:
// gdn_prefill_pairs_kernel, one CTA per (chunk, key head), scales q and k, forms their products once for
// all value heads of the key head, and leaves q, k, T, P and the rows' factors in a workspace, as the
// images that the second kernel copies to shared memory.  gdn_prefill_chain_kernel then carries the state
// of a (request, value head) from chunk to chunk on the tensor cores' tcgen05 instructions, value rows as
// the M = 128 of every product:
//   Y = S k~, O = S q~   A = S hi, lo in TMEM      B = k~, q~ (K-major)
//   U = T R              A = R hi, lo in TMEM      B = T hi, lo
//   P u                  A = u hi, lo in TMEM      B = P hi, lo
//   dS = u k~            A = k_out u hi, lo        B = the same k~ tile, read MN-major
// It is one persistent CTA per SM that takes (request, value head) items from a queue, longest first.
// Eight warps keep the fp32 state in registers, 16 value rows each, in the layout that 16-lane TMEM
// loads and stores use; between products they scale, split and store the next A operand, and two of them
// issue.  The other eight copy the next chunk in, issue P u, and normalise and store the chunk before's outputs.
//
// What bounds it: 24 prompts of 16,000 tokens in all, 16 key and 32 value heads, take 400-414 us, 124 in
// the pairs kernel (47% of issue slots, 14,600 warp instructions a CTA: latency, at the four CTAs per SM
// that 128 registers allow) and 304 in the chain (7,900 cycles a chunk: the four steps between its products,
// and the moving threads' own loop, which is nearly as long; 46% of issue slots, 24% of the tensor pipe).
// History of the split (and of one prompt of 16,384): one kernel that prepared each chunk inside the
// chain's CTA, 1,242 us (4,878); pairs apart and the chain on mma.sync with the state as its fragments, 555
// (1,646); the chain on tcgen05, 430 (1,181); outputs gathered off the chain's path 418, the queue 412, one
// warp that waits for products 400, issue with constant operands 390 (1,137); the pairs of two heads at a
// time, blocks dealt out evenly, 374 (1,104); long prompts in pieces (742); second terms for the outputs
// 407 (751), of which 30 are what unpacking them takes from the moving threads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "internal.h"
#include "launch.cuh"
#include "lightdelta_b200.h"
#include "math.cuh"

namespace ldb {
namespace {

constexpr int kDim = LD_HEAD_DIM;
constexpr int kChunk = LD_PREFILL_CHUNK;
constexpr int kPairThreads = 128;
constexpr int kMoveThreads = 256;   // chain kernel: warps 0-7 copy chunks in and store outputs,
constexpr int kStateThreads = 256;  // warps 8-15 carry the state
constexpr int kChainThreads = kMoveThreads + kStateThreads;
constexpr int kORow = kDim + 4;  // floats per row of the output tile: the +4 spreads its rows over the banks
static_assert(kChunk == 64, "fragment loops below are written for chunks of 64 tokens");

constexpr int kHalf = kChunk * 64;    // elements of half a 128-column tile
constexpr int kKeyHalf = 2 * kHalf;   // from a half of k (or q) to its other half

__device__ unsigned int g_prefill_faults;

// Workspace images, byte for byte what the chain's products read: tiles of 128 columns are swizzled (swz), triangular
// matrices are packed 16 x 16 blocks (tri_block, core).
struct __align__(128) KeyImage {  // per (chunk, key head)
  __half kq[2 * kChunk * kDim];   // columns 0-63 of k x 2^-e, then of q x 2^-e, then columns 64-127 likewise
};

constexpr int kTriBlocks = 10;  // 16 x 16 blocks on and below the diagonal of a 64 x 64 matrix
constexpr int kLowBlocks = 6;   // of them, below it
// Per (chunk, value head).  The stage that a chunk is worked from has T and P as two fp16 terms each; here the terms share
// what room there is (unpack_chunk takes them apart again):
//   T is a unit triangle, so the lo terms of its diagonal blocks lie transposed above the diagonal of t_hi's;
//   P's lo terms are bytes, in 256ths of the hi term's last bit: 19 bits together.  Of a diagonal block's four core
//   matrices the one above the diagonal is left out, and three numbers lie in bytes of others that are above it, too.
struct PairMain {
  __half t_hi[kTriBlocks * 256];
  __half p_hi[kTriBlocks * 256];
  float beta[kChunk];
  float k_in[kChunk];   // e^{G_i} fk_i: scales S k~
  float q_in[kChunk];   // e^{G_i} fq_i 128^-1/2: scales S q~
  float k_out[kChunk];  // e^{G_C - G_j} fk_j / k_scale: scales u_j on its way into the state
  uint8_t p_lo[kLowBlocks * 256 + 4 * 192];  // blocks below the diagonal, then three core matrices per diagonal block

  // Columns 4-7 of rows 0, 1 and 2 of the first diagonal block.
  __device__ __forceinline__ float* numbers() { return reinterpret_cast<float*>(p_lo + kLowBlocks * 256); }
  __device__ __forceinline__ const float* numbers() const { return reinterpret_cast<const float*>(p_lo + kLowBlocks * 256); }
  __device__ __forceinline__ float& decay() { return numbers()[1]; }    // e^{G_C}
  __device__ __forceinline__ float& k_scale() { return numbers()[3]; }  // the power of two that brings the largest of k_out to [1, 2)
  __device__ __forceinline__ float& p_scale() { return numbers()[5]; }  // the powers of two that P was divided by
  __device__ __forceinline__ float decay() const { return numbers()[1]; }
  __device__ __forceinline__ float k_scale() const { return numbers()[3]; }
  __device__ __forceinline__ float p_scale() const { return numbers()[5]; }
};
struct __align__(128) PairImage {
  PairMain main;
  __half t_lo[kLowBlocks * 256];  // blocks below the diagonal
};
static_assert(sizeof(KeyImage) % 16 == 0 && sizeof(PairMain) % 16 == 0, "images are copied 16 bytes at a time");
static_assert(sizeof(PairImage) == sizeof(PairMain) + sizeof(PairImage::t_lo), "without gaps");

// Splitting a long prompt.  The chain takes a value head's chunks one after the other, so few requests with few heads
// leave most SMs idle.  A chunk's step is linear in the state, S <- S M + B, and so is a run of chunks: M is what it
// makes of the identity with all v taken as zero, B what it makes of zero.  A request in pieces is run in two passes:
// the first runs piece 0 for good and carries M_k and B_k through each middle piece k, all at once; then
// S_1 = the end of piece 0 and S_{k+1} = S_k M_k + B_k are joined, and the second pass runs the pieces from 1 on from
// their states, all at once.  That is three times the work for the middle pieces, in the time of two pieces.
// With room for `slots` CTAs per value head there are (slots - 1) / 2 middle pieces, and one more of half their length,
// whose M and B share a CTA, where a slot is left over: 16,384 tokens of one request with 32 value heads (4 slots,
// 4 pieces, 2 of 3.5 parts of the chain's time) take 751 us, unsplit 1,189; with 4 value heads (16 pieces) 225 instead of
// 1,085, and 1,600 tokens with 8 value heads 81 instead of 121.
struct Pieces {
  int count;       // 1: no request is split
  bool half_last;  // the last middle piece has half the length of the others

  // Piece k begins with chunk chunks * cut(k) / cut(count).
  __host__ __device__ int64_t cut(int k) const { return 2 * k - (half_last && k >= count - 1 ? 1 : 0); }
  // What the first pass runs per request and value head, a matrix each: piece 0, then M_k and B_k, k = 1 .. count - 2.
  __host__ __device__ int first_parts() const { return count > 1 ? 2 * count - 3 : 1; }
};

constexpr int kPieceChunks = 5;   // a whole piece has at least so many: every piece adds 2 us to the joins
constexpr int kSavedChunks = 10;  // chunk times that splitting saves at least: the launches cost about nine
constexpr int kPiecesMost = 16;
constexpr int kPieceSms = 148;

// Splitting pays for a request of so many chunks: 2 whole pieces' time, 4 of cut's units, instead of all.
__host__ __device__ __forceinline__ bool worth_splitting(const Pieces& pieces, int64_t chunks) {
  const int64_t units = pieces.cut(pieces.count);
  return pieces.count > 1 && chunks >= kPieceChunks * pieces.count && chunks * (units - 4) >= kSavedChunks * units;
}

Pieces pieces_of(int64_t n_tokens, int64_t n_requests, int64_t num_v_heads) {
  const int64_t slots = kPieceSms / std::max<int64_t>(n_requests * num_v_heads, 1), chunks = n_tokens / kChunk;
  const int64_t most = std::min<int64_t>(kPiecesMost, chunks / kPieceChunks), whole = 2 + (slots - 1) / 2;
  if (slots < 2 || most < 3) return {1, false};
  const bool half = slots % 2 == 0 && whole < most;
  const Pieces pieces{static_cast<int>(half ? whole + 1 : std::min(whole, most)), half};
  return worth_splitting(pieces, chunks) ? pieces : Pieces{1, false};
}

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
  int32_t* order;    // requests, longest first
  uint32_t* next;    // items that the chain's CTAs have taken, per pass, and whether a wait has run out
  float* states;     // fp32 states between the pieces of split requests, first_parts() per request and value head
  Pieces pieces;     // of long requests
  int pass;          // of the chain kernel: 1 for the pieces that begin with a joined state
  int64_t places;
  int n_requests;
  int num_k_heads;
  int num_v_heads;
  int heads_ratio;
  int dt_bias_bf16;
  int weight_bf16;
  float q_scale;
  float eps;
  uint64_t wait_ns;   // bound of every in-kernel wait (ld_decode_wait_test)
  uint32_t extra_tx;  // test only: bytes that a chunk's copies announce beyond what they copy (normally 0)
};

// Chunk c of request r is kept at place chunk_base(cu[r], r) + c.  A request of n tokens has at most n / 64 + 2 chunks (both
// ends may be short) and at most n, so places never overlap, and nobody has to count chunks.
__host__ __device__ __forceinline__ int64_t chunk_base(int64_t first_token, int64_t request) {
  const int64_t whole = first_token / kChunk + 2 * request;
  return first_token < whole ? first_token : whole;
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

// Named barriers of the chain kernel: the first ones and kBarFull hand over between the threads that move data
// and those that carry the state, kBarState and kBarMove join each.
constexpr int kBarChunkDone = 1, kBarTaken = 2, kBarState = 3, kBarMove = 4, kBarFull = 5;
__device__ __forceinline__ void bar_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kChainThreads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kChainThreads) : "memory");
}
__device__ __forceinline__ void bar_move() {
  asm volatile("bar.sync %0, %1;" ::"n"(kBarMove), "n"(kMoveThreads) : "memory");
}
__device__ __forceinline__ void bar_state() {
  asm volatile("bar.sync %0, %1;" ::"n"(kBarState), "n"(kStateThreads) : "memory");
}

// ---- tcgen05: products with A and D in TMEM and B in shared memory.  One warp calls, with the same values in
// every lane, and its elected lane issues.
// Instruction descriptor of kind::f16: fp16 A and B, fp32 D, M = 128; bit 16 reads B MN-major.
__host__ __device__ constexpr uint32_t mma_shape(int n, bool b_mn_major) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24) | (b_mn_major ? 1u << 16 : 0u);
}

// Shared-memory descriptor of a 128-byte swizzled tile: atoms of 8 rows x 128 bytes, 1024 bytes apart along
// the rows; 64-column halves (MN-major only) kKeyHalf apart.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3fff) | (static_cast<uint64_t>(2 * kKeyHalf >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// The same of a packed triangular matrix's 16-column block, without swizzle: core matrices 128 bytes apart along
// the columns, 256 along the rows.
__device__ __forceinline__ uint64_t tri_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3fff) | (static_cast<uint64_t>(128 >> 4) << 16) |
         (static_cast<uint64_t>(256 >> 4) << 32) | (1ull << 46);
}

__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t elected;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
  return elected;
}

// D[128 x n] (+)= A[128 x 16] B[16 x n].
__device__ __forceinline__ void umma(uint32_t elected, uint32_t d, uint32_t a, uint64_t b, uint32_t shape,
                                     bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(accumulate)), "r"(elected)
      : "memory");
}

// The barrier's phase completes when every product issued so far has.
__device__ __forceinline__ void umma_commit(uint32_t elected, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(elected)
      : "memory");
}

__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 64 fp32 columns of this warp's 16 lanes, as eight accumulator fragments (row g: columns 8n + 2t, + 1 in
// elements 0, 1; row g + 8 in 2, 3).  Loads and their wait are one statement, so nothing reads too early.
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&r)[8][4]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0][0]), "=f"(r[0][1]), "=f"(r[0][2]), "=f"(r[0][3]), "=f"(r[1][0]), "=f"(r[1][1]), "=f"(r[1][2]),
        "=f"(r[1][3]), "=f"(r[2][0]), "=f"(r[2][1]), "=f"(r[2][2]), "=f"(r[2][3]), "=f"(r[3][0]), "=f"(r[3][1]),
        "=f"(r[3][2]), "=f"(r[3][3]), "=f"(r[4][0]), "=f"(r[4][1]), "=f"(r[4][2]), "=f"(r[4][3]), "=f"(r[5][0]),
        "=f"(r[5][1]), "=f"(r[5][2]), "=f"(r[5][3]), "=f"(r[6][0]), "=f"(r[6][1]), "=f"(r[6][2]), "=f"(r[6][3]),
        "=f"(r[7][0]), "=f"(r[7][1]), "=f"(r[7][2]), "=f"(r[7][3])
      : "r"(addr)
      : "memory");
}

// 16 columns from each of two places.
__device__ __forceinline__ void tmem_load(uint32_t x_at, uint32_t y_at, float (&x)[2][4], float (&y)[2][4]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%16];\n\t"
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%17];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=&f"(x[0][0]), "=&f"(x[0][1]), "=&f"(x[0][2]), "=&f"(x[0][3]), "=&f"(x[1][0]), "=&f"(x[1][1]), "=&f"(x[1][2]),
        "=&f"(x[1][3]), "=&f"(y[0][0]), "=&f"(y[0][1]), "=&f"(y[0][2]), "=&f"(y[0][3]), "=&f"(y[1][0]), "=&f"(y[1][1]),
        "=&f"(y[1][2]), "=&f"(y[1][3])
      : "r"(x_at), "r"(y_at)
      : "memory");
}

// Four k-steps of packed A fragments to 32 columns of this warp's 16 lanes.
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&a)[4][4]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(a[0][0]), "r"(a[0][1]), "r"(a[0][2]), "r"(a[0][3]), "r"(a[1][0]), "r"(a[1][1]), "r"(a[1][2]), "r"(a[1][3]),
      "r"(a[2][0]), "r"(a[2][1]), "r"(a[2][2]), "r"(a[2][3]), "r"(a[3][0]), "r"(a[3][1]), "r"(a[3][2]), "r"(a[3][3])
      : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int bytes = live ? 16 : 0;  // 0: the 16 bytes are filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All groups but the last `kLast`.
template <int kLast>
__device__ __forceinline__ void cp_async_wait_groups() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLast) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t arrivals = 1) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// ------------------------------------------------------------------------------------------
// swizzled tiles: 64 rows of 64 16-bit columns, 128 bytes a row, whose 16-byte pieces are stored at
// piece ^ (row mod 8): the 128-byte swizzle of matrix descriptors, free of bank conflicts for ldmatrix too.
// A 128-column tile is two such halves, kStride elements apart (kKeyHalf for k and q, which alternate).
// ------------------------------------------------------------------------------------------
template <int kStride>
__device__ __forceinline__ int swz(int row, int col) {
  return (col >> 6) * kStride + row * 64 + (((((col >> 3) & 7) ^ (row & 7)) << 3) | (col & 7));
}

// Address that this lane gives to ldmatrix.x4 for the 16 x 16 block at (0, 0) of a tile: matrices in the
// order (rows 0-7, cols 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15), or with kRowsFirst
// (0-7, 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15).  Row blocks start at multiples of 8, so the swizzle
// depends on the lane alone and the block at (16 rb, 16 cb) is at block<kStride>(address, rb, cb).
template <bool kRowsFirst>
__device__ __forceinline__ uint32_t lane_addr(const void* tile, int lane) {
  const int m = lane >> 3;
  const int row = (lane & 7) + 8 * (kRowsFirst ? (m & 1) : (m >> 1));
  const int piece = (kRowsFirst ? (m >> 1) : (m & 1)) ^ (lane & 7);
  return smem_u32(tile) + row * 128 + (piece << 4);
}

template <int kStride>
__device__ __forceinline__ uint32_t block(uint32_t addr, int rb, int cb) {
  return (addr ^ ((cb & 3) << 5)) + (cb >> 2) * (2 * kStride) + rb * (16 * 128);
}

// Packed triangular matrices: 16-column blocks one after the other, each from its diagonal block down, in 8 x 8
// core matrices of 128 contiguous bytes, the two of a row group side by side: matrix descriptors without
// swizzle read a column block's rows from any row group on, and ldmatrix reads core matrices without bank
// conflicts.
__host__ __device__ constexpr int tri_block(int ib, int jb) { return 256 * (4 * jb - jb * (jb - 1) / 2 + (ib - jb)); }

// The blocks below the diagonal in the order of their places, and block i's number among all ten.
__host__ __device__ constexpr int below_block(int ib, int jb) { return jb == 0 ? ib - 1 : jb == 1 ? ib + 1 : 5; }
__host__ __device__ constexpr int below_place(int i) { return i + 1 + (i >= 3) + (i >= 5); }
static_assert(256 * below_place(below_block(3, 0)) == tri_block(3, 0) && 256 * below_place(below_block(2, 1)) == tri_block(2, 1) &&
                  256 * below_place(below_block(3, 1)) == tri_block(3, 1) && 256 * below_place(below_block(3, 2)) == tri_block(3, 2),
              "column by column");

__device__ __forceinline__ int core(int row, int col) {  // within a 16 x 16 block
  return (row >> 3) * 128 + (col >> 3) * 64 + (row & 7) * 8 + (col & 7);
}

// This lane's ldmatrix.x4 address in the 16 x 16 block at `m`, matrices in the order of lane_addr with
// kRowsFirst false.
__device__ __forceinline__ uint32_t core_addr(const __half* m, int lane) {
  return smem_u32(m) + 2 * core((lane & 7) + 8 * (lane >> 4), 8 * ((lane >> 3) & 1));
}

__device__ __forceinline__ uint32_t pack_half(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// x.x, x.y as two fp16 terms: hi the nearest, lo the nearest to what hi leaves.
__device__ __forceinline__ void split(float2 x, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  const float2 f = __half22float2(h);
  const float2 r = fma2(f, make_float2(-1.0f, -1.0f), x);  // exact
  const __half2 l = __floats2half2_rn(r.x, r.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// The same with hi cut off instead of rounded, 22 bits together instead of 23, which spares the way back from fp16: the
// chain's splits are on the state's path (one prompt of 16,384 tokens: 777 -> 750 us).
__device__ __forceinline__ void split_masked(float2 x, uint32_t& hi, uint32_t& lo) {
  const float2 f = make_float2(__uint_as_float(__float_as_uint(x.x) & 0xffffe000u),
                               __uint_as_float(__float_as_uint(x.y) & 0xffffe000u));
  hi = pack_half(f.x, f.y);
  const float2 r = fma2(f, make_float2(-1.0f, -1.0f), x);
  lo = pack_half(r.x, r.y);
}

// x as a fp16 term and a byte: what that leaves, in 256ths of its last bit, plus 128.  A last bit is 2^(e - 25), e the
// biased exponent; terms below fp16's normal range keep no byte.
__device__ __forceinline__ void split_byte(float2 x, uint32_t& hi, uint32_t& bytes) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  const float2 f = __half22float2(h);
  const float2 r = fma2(f, make_float2(-1.0f, -1.0f), x);  // exact
  hi = *reinterpret_cast<const uint32_t*>(&h);
  const float s0 = __uint_as_float((160u << 23) - ((hi & 0x7c00u) << 13));  // 2^(33 - e)
  const float s1 = __uint_as_float((160u << 23) - ((hi & 0x7c000000u) >> 3));
  // The sum's last mantissa bits are the rounded byte; half a last bit would be 256.
  constexpr float kShift = 8388608.0f + 128.0f;
  const uint32_t b0 = __float_as_uint(fminf(fmaf(r.x, s0, kShift), kShift + 127.0f));
  const uint32_t b1 = __float_as_uint(fminf(fmaf(r.y, s1, kShift), kShift + 127.0f));
  bytes = __byte_perm(b0, b1, 0x0040) & 0xffffu;
}

// The lo terms of two elements from their hi terms and bytes (the low ones of 16-bit halves).
__device__ __forceinline__ uint32_t lo_terms(uint32_t hi, uint32_t bytes) {
  const uint32_t last = hi & 0x7c007c00u, shifted = bytes | 0x64006400u;  // 2^(e - 15) each; 1024 + byte
  const __half2 bit = __hmul2(*reinterpret_cast<const __half2*>(&last), __float2half2_rn(0x1p-10f));
  const __half2 part = __hfma2(*reinterpret_cast<const __half2*>(&shifted), __float2half2_rn(0x1p-8f), __float2half2_rn(-4.5f));
  const __half2 lo = __hmul2(bit, part);
  return *reinterpret_cast<const uint32_t*>(&lo);
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
// pairs: what a chunk's tokens mean to one another
// ------------------------------------------------------------------------------------------
constexpr int kGroup = 4;  // value heads whose gates are computed together, one per warp

// What a value head's inverse is made in; heads are worked on two at a time.
struct PairHead {
  __align__(16) __half t_hi[kTriBlocks * 256];
  __half t_lo[kTriBlocks * 256];
  __half l_hi[6 * 256];   // L's blocks below the diagonal ones, packed row by row
  __half l_lo[6 * 256];
  float diag[4][16 * 16];  // L's diagonal blocks
  float pad[16];           // the two heads' diagonal blocks, read side by side, lie in different banks
};

struct PairSmem {
  union {
    __align__(128) unsigned char tiles[sizeof(KeyImage)];  // the key image, then, its products in registers,
    unsigned char heads[2 * sizeof(PairHead)];
    uint32_t counts[64];  // of order_requests
  };
  float g_hi[kGroup][kChunk], g_lo[kGroup][kChunk], beta[kGroup][kChunk];
  float fk[kChunk], fq[kChunk];
  float fk_unit[kChunk], fq_unit[kChunk];  // divided by the power of two of the longest normalised row
  float fk_power, fq_power;

  __device__ __forceinline__ __half* kq() { return reinterpret_cast<__half*>(tiles); }
  __device__ __forceinline__ PairHead& head(int i) { return reinterpret_cast<PairHead*>(heads)[i]; }
};
static_assert(sizeof(PairHead) % 128 == 64, "heads differ in banks, and matrices stay 16-byte aligned");

// The 16 x 16 blocks on and below the diagonal that a warp has: the diagonal one of its number and one or two side by
// side below, so that no warp has more than three of the ten.
struct Blocks {
  int w;      // diagonal block
  int row;    // row block of the others
  int col;    // column block of the first
  bool two;   // and of a second, col + 1
  __device__ __forceinline__ explicit Blocks(int warp)
      : w(warp), row(warp == 1 ? 2 : warp == 3 ? 1 : 3), col(warp == 2 ? 2 : 0), two(warp < 2) {}
  __device__ __forceinline__ int ib(int b) const { return b == 0 ? w : row; }
  __device__ __forceinline__ int jb(int b) const { return b == 0 ? w : col + b - 1; }
};

// Rows' products divided by the longest lengths' powers of two are below 4, and with q's 128^-1/2 below 0.36: times this
// they fill fp16's range, and P's terms reach down to 2^-37 of the longest rows' product.
constexpr float kPUp = 16384.0f;

// L's blocks below the diagonal ones, row by row.
__host__ __device__ constexpr int low_block(int ib, int jb) { return 256 * (ib * (ib - 1) / 2 + jb); }

// Rows [row_lo, row_hi) of 128 bf16 to shared memory, the others as zeros, 16 bytes a thread at a time; `at` gives
// the element that (row, column) goes to.
template <bool kVec, int kThreads, typename At>
__device__ __forceinline__ void load_rows(const __nv_bfloat16* base, int64_t row_stride, int row_lo, int row_hi,
                                          uint16_t* tile, int tid, At at) {
#pragma unroll 2
  for (int pass = 0; pass < kChunk / (kThreads / 16); ++pass) {
    const int i = pass * (kThreads / 16) + (tid >> 4);
    const int col = (tid & 15) * 8;
    const bool live = i >= row_lo && i < row_hi;
    uint16_t* dst = tile + at(i, col);
    const __nv_bfloat16* src = base + static_cast<int64_t>(live ? i : row_lo) * row_stride + col;
    if constexpr (kVec) {
      cp_async16(smem_u32(dst), src, live);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = live ? __bfloat16_as_ushort(src[e]) : 0;
    }
  }
}

// Scales one row from bf16 to fp16 in place, by one thread: a power of two brings the row's largest magnitude to
// [2^13, 2^14), so that elements down to 2^-30 of it keep bf16's eight bits above fp16's smallest step, 2^-24, and sums
// of 128 products of two rows stay below 2^35.  Returns that power's inverse.
__device__ __forceinline__ float scale_row(uint16_t* tile, int i) {
  uint16_t* row = tile + i * 64;
  __nv_bfloat162 top = __floats2bfloat162_rn(0.0f, 0.0f);  // the largest magnitudes so far of even and odd columns
#pragma unroll
  for (int piece = 0; piece < kDim / 8; ++piece) {
    const uint4 raw = *reinterpret_cast<const uint4*>(row + (piece >> 3) * kKeyHalf + (((piece & 7) ^ (i & 7)) << 3));
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int n = 0; n < 4; ++n) top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[n])));
  }
  const uint32_t top2 = *reinterpret_cast<const uint32_t*>(&top);  // bf16 magnitudes order as integers
  const int e = min(max(static_cast<int>(max(top2 >> 16, top2 & 0xffffu) >> 7), 14), 253);
  const float down = __uint_as_float(static_cast<uint32_t>(267 - e) << 23);  // 2^(140 - e)
#pragma unroll
  for (int piece = 0; piece < kDim / 8; ++piece) {
    uint4* at = reinterpret_cast<uint4*>(row + (piece >> 3) * kKeyHalf + (((piece & 7) ^ (i & 7)) << 3));
    const uint4 raw = *at;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t y[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float2 x = mul2(make_float2(bf16_low(w[n]), bf16_high(w[n])), make_float2(down, down));
      y[n] = pack_half(x.x, x.y);
    }
    *at = make_uint4(y[0], y[1], y[2], y[3]);
  }
  return __uint_as_float(static_cast<uint32_t>(e - 13) << 23);
}

// The power of two at or below the largest of 64 positive floats, of which each lane of a warp has two.  Operands that
// become fp16 are divided by it, so that keys or queries of any size (the L2 norm's 1e-6 lets short ones stay short)
// have the same bits there.
__device__ __forceinline__ float largest_power(float x, float y) {
  const uint32_t top = __reduce_max_sync(0xffffffffu, max(__float_as_uint(x), __float_as_uint(y)));
  return __uint_as_float(min(max(top >> 23, 1u), 253u) << 23);
}
__device__ __forceinline__ float inverse_power(float power) {
  return __uint_as_float(0x7f000000u - __float_as_uint(power));  // 2^(254 - e - 127)
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

// This warp's blocks of k~ k~^T and q~ k~^T, and its rows' factors (the L2 norm's reciprocal times the power of two that
// the scaling took) from the diagonals of k~ k~^T and q~ q~^T.
__device__ __forceinline__ void row_products(PairSmem& s, const Blocks& mine, int lane, float (&kk)[3][2][4],
                                             float (&qk)[3][2][4]) {
  const uint32_t k_a = lane_addr<true>(s.kq(), lane), q_a = lane_addr<true>(s.kq() + kHalf, lane);
  const uint32_t k_b = lane_addr<false>(s.kq(), lane);
#pragma unroll
  for (int b = 0; b < 3; ++b) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int e = 0; e < 4; ++e) kk[b][m][e] = qk[b][m][e] = 0.0f;
    }
  }
  float qq[2][4] = {};
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    uint32_t ak[4], aq[4], b[4];
    ldsm4(block<kKeyHalf>(k_a, mine.w, ks), ak);
    ldsm4(block<kKeyHalf>(q_a, mine.w, ks), aq);
    // A fragments are (rows 0-7, cols 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15): as B, rows 0-7 are 0, 2.
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      mma(kk[0][m], ak, ak[m], ak[2 + m]);
      mma(qk[0][m], aq, ak[m], ak[2 + m]);
      mma(qq[m], aq, aq[m], aq[2 + m]);
    }
    ldsm4(block<kKeyHalf>(k_a, mine.row, ks), ak);
    ldsm4(block<kKeyHalf>(q_a, mine.row, ks), aq);
#pragma unroll
    for (int n = 1; n < 3; ++n) {
      if (n == 1 || mine.two) {
        ldsm4(block<kKeyHalf>(k_b, mine.jb(n), ks), b);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          mma(kk[n][m], ak, b[2 * m], b[2 * m + 1]);
          mma(qk[n][m], aq, b[2 * m], b[2 * m + 1]);
        }
      }
    }
  }
  // Element (g, g) of the diagonal block is with t = g / 2 (of 8 columns), and (g + 8, g + 8) likewise.
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float k2 = (g & 1) ? kk[0][half][2 * half + 1] : kk[0][half][2 * half];
    const float q2 = (g & 1) ? qq[half][2 * half + 1] : qq[half][2 * half];
    if (t == g / 2) {
      const int i = 16 * mine.w + g + 8 * half;
      const float up_k = s.fk[i], up_q = s.fq[i];
      const float fk = up_k * rsqrtf(k2 * up_k * up_k + 1e-6f), fq = up_q * rsqrtf(q2 * up_q * up_q + 1e-6f);
      s.fk[i] = fk;
      s.fq[i] = fq;
      s.fk_unit[i] = fk * sqrt_fast(k2);  // the normalised row's length, for now
      s.fq_unit[i] = fq * sqrt_fast(q2);
    }
  }
}

// The factors of the chunk's rows for one value head, row i = 0..63 by two warps, straight to its image.
__device__ __forceinline__ void row_factors(const PrefillArgs& p, PairSmem& s, int place, int i, PairMain& image) {
  const float in = exp2_fast(s.g_hi[place][i] + s.g_lo[place][i]);
  image.beta[i] = s.beta[place][i];
  image.k_in[i] = in * s.fk[i];
  image.q_in[i] = in * s.fq[i] * p.q_scale;
  const auto out = [&](int j) {
    const float left = (s.g_hi[place][kChunk - 1] - s.g_hi[place][j]) + (s.g_lo[place][kChunk - 1] - s.g_lo[place][j]);
    return exp2_fast(left) * s.fk[j];
  };
  const float k_out = out(i), power = largest_power(k_out, out(i ^ 32));
  image.k_out[i] = k_out * inverse_power(power);
  if (i == kChunk - 1) {
    image.decay() = in;
    image.k_scale() = power;
    image.p_scale() = s.fk_power * s.fq_power * (1.0f / kPUp);
  }
}

// L and P of this warp's blocks for one value head, two terms each; P goes straight to the image, 128 and 64 bytes a store.
__device__ __forceinline__ void decayed_pairs(const PrefillArgs& p, PairSmem& s, PairHead& head, int place,
                                              const Blocks& mine, int lane, const float (&kk)[3][2][4],
                                              const float (&qk)[3][2][4], PairMain& image) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int b = 0; b < 3; ++b) {
    if (b == 2 && !mine.two) continue;
    const int row0 = 16 * mine.ib(b) + g, col0 = 16 * mine.jb(b) + 2 * t;
    float g_hi[2], g_lo[2], row_k[2], row_q[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = row0 + 8 * half;
      g_hi[half] = s.g_hi[place][i];
      g_lo[half] = s.g_lo[place][i];
      row_k[half] = s.beta[place][i] * s.fk[i] * s.fk_power;
      row_q[half] = kPUp * p.q_scale * s.fq_unit[i];
    }
    const int to_p = tri_block(mine.ib(b), mine.jb(b)) + core(g, 2 * t);
    const int to_byte = (b > 0 ? 256 * below_block(mine.row, mine.jb(b)) : 256 * kLowBlocks + 192 * mine.w) + core(g, 2 * t);
    const int to_l = low_block(mine.row, mine.jb(b)) + core(g, 2 * t);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int j = col0 + 8 * m;
      const float2 hj = *reinterpret_cast<const float2*>(&s.g_hi[place][j]);
      const float2 lj = *reinterpret_cast<const float2*>(&s.g_lo[place][j]);
      const float2 fj = *reinterpret_cast<const float2*>(&s.fk_unit[j]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float d0 = fj.x * exp2_fast((g_hi[half] - hj.x) + (g_lo[half] - lj.x));
        const float d1 = fj.y * exp2_fast((g_hi[half] - hj.y) + (g_lo[half] - lj.y));
        float l0 = row_k[half] * d0 * kk[b][m][2 * half], l1 = row_k[half] * d1 * kk[b][m][2 * half + 1];
        float p0 = row_q[half] * d0 * qk[b][m][2 * half], p1 = row_q[half] * d1 * qk[b][m][2 * half + 1];
        if (b == 0) {
          const int i = row0 + 8 * half;
          l0 = j < i ? l0 : 0.0f;
          l1 = j + 1 < i ? l1 : 0.0f;
          p0 = j <= i ? p0 : 0.0f;
          p1 = j + 1 <= i ? p1 : 0.0f;
          *reinterpret_cast<float2*>(&head.diag[mine.w][(g + 8 * half) * 16 + 8 * m + 2 * t]) = make_float2(l0, l1);
        } else {
          uint32_t hi, lo;
          split(make_float2(l0, l1), hi, lo);
          *reinterpret_cast<uint32_t*>(&head.l_hi[to_l + core(8 * half, 8 * m)]) = hi;
          *reinterpret_cast<uint32_t*>(&head.l_lo[to_l + core(8 * half, 8 * m)]) = lo;
        }
        uint32_t hi, bytes;
        split_byte(make_float2(p0, p1), hi, bytes);
        *reinterpret_cast<uint32_t*>(&image.p_hi[to_p + core(8 * half, 8 * m)]) = hi;
        // Of a diagonal block, pairs with an element on or below the diagonal.
        const bool kept = b > 0 || half > m || (half == m && 2 * t <= g);
        if (kept) *reinterpret_cast<uint16_t*>(&image.p_lo[to_byte + (b > 0 ? core(8 * half, 8 * m) : 64 * (half + m))]) = bytes;
      }
    }
  }
}

// Inverse of a diagonal block of I + L by forward substitution: one column per lane, a head per half warp.
__device__ __forceinline__ void invert_diagonal(PairHead& head, int w, int c) {
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float sum0 = i == c ? 1.0f : 0.0f, sum1 = 0.0f;
#pragma unroll
    for (int j = 0; j < i; j += 4) {
      const float4 l = *reinterpret_cast<const float4*>(&head.diag[w][i * 16 + j]);
      sum0 = fmaf(-l.x, x[j], sum0);
      if (j + 1 < i) sum1 = fmaf(-l.y, x[j + 1], sum1);
      if (j + 2 < i) sum0 = fmaf(-l.z, x[j + 2], sum0);
      if (j + 3 < i) sum1 = fmaf(-l.w, x[j + 3], sum1);
    }
    x[i] = sum0 + sum1;
  }
  __half* to_hi = head.t_hi + tri_block(w, w) + core(0, c);
  __half* to_lo = head.t_lo + tri_block(w, w) + core(0, c);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const __half hi = __float2half_rn(x[i]);
    to_hi[core(i, 0)] = hi;
    to_lo[core(i, 0)] = __float2half_rn(x[i] - __half2float(hi));
  }
}

// The 16 x 16 blocks of T below diagonal block w, top to bottom:
//   T_iw = -T_ii sum_{k=w}^{i-1} L_ik T_kw,  held transposed so that each result is the next A operand.
__device__ __forceinline__ void invert_column(PairHead& head, int w, int lane) {
  const uint32_t t_hi = core_addr(head.t_hi, lane), t_lo = core_addr(head.t_lo, lane);
  const uint32_t l_hi = core_addr(head.l_hi, lane), l_lo = core_addr(head.l_lo, lane);
  uint32_t x_hi[3][4], x_lo[3][4];  // T_kw^T as A fragments, k = w, w + 1, w + 2
  // ldmatrix.trans of T_ww: matrices (cols 0-7, rows 0-7), (cols 8-15, rows 0-7), (0-7, 8-15), (8-15, 8-15).
  ldsm4_t(t_hi + 2 * tri_block(w, w), x_hi[0]);
  ldsm4_t(t_lo + 2 * tri_block(w, w), x_lo[0]);
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    const int i = w + d;
    if (i < 4) {
      float m[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < d; ++kk) {
        uint32_t b_hi[4], b_lo[4];
        ldsm4(l_hi + 2 * low_block(i, w + kk), b_hi);
        ldsm4(l_lo + 2 * low_block(i, w + kk), b_lo);
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
        split(make_float2(m[n][0], m[n][1]), a_hi[2 * n], a_lo[2 * n]);
        split(make_float2(m[n][2], m[n][3]), a_hi[2 * n + 1], a_lo[2 * n + 1]);
      }
      float y[2][4] = {};
      uint32_t b_hi[4], b_lo[4];
      ldsm4(t_hi + 2 * tri_block(i, i), b_hi);
      ldsm4(t_lo + 2 * tri_block(i, i), b_lo);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        mma(y[n], a_hi, b_lo[2 * n], b_lo[2 * n + 1]);
        mma(y[n], a_lo, b_hi[2 * n], b_hi[2 * n + 1]);
        mma(y[n], a_hi, b_hi[2 * n], b_hi[2 * n + 1]);
      }
      // y[n] is -T_iw^T: row m = column of T_iw (g, g + 8), column = row of T_iw (8n + 2t, + 1).
      __half* to_hi = head.t_hi + tri_block(i, w) + core(2 * t, g);
      __half* to_lo = head.t_lo + tri_block(i, w) + core(2 * t, g);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          split(make_float2(-y[n][2 * half], -y[n][2 * half + 1]), hi[half], lo[half]);
          const __half2 h = *reinterpret_cast<const __half2*>(&hi[half]);
          const __half2 l = *reinterpret_cast<const __half2*>(&lo[half]);
          to_hi[core(8 * n, 8 * half)] = __low2half(h);
          to_hi[core(8 * n + 1, 8 * half)] = __high2half(h);
          to_lo[core(8 * n, 8 * half)] = __low2half(l);
          to_lo[core(8 * n + 1, 8 * half)] = __high2half(l);
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

// Requests by their chunk counts, longest first (to half an octave), for the chain to take in this order;
// equal ones in any order.  One CTA.
__device__ __forceinline__ void order_requests(const PrefillArgs& p, uint32_t (&counts)[64], int tid) {
  if (tid < 64) counts[tid] = 0;
  if (tid < 3) p.next[tid] = 0;
  __syncthreads();
  const auto bucket = [&](int r) {
    const int tokens = max(p.cu[r + 1] - p.cu[r], 1);
    const int chunks = tokens / kChunk + 1;  // to one
    const int octave = 31 - __clz(chunks);
    return 63 - (2 * octave + (octave > 0 ? (chunks >> (octave - 1)) & 1 : 0));
  };
  for (int r = tid; r < p.n_requests; r += kPairThreads) atomicAdd(&counts[bucket(r)], 1u);
  __syncthreads();
  if (tid == 0) {
    uint32_t sum = 0;
    for (int b = 0; b < 64; ++b) {
      const uint32_t n = counts[b];
      counts[b] = sum;
      sum += n;
    }
  }
  __syncthreads();
  for (int r = tid; r < p.n_requests; r += kPairThreads) p.order[atomicAdd(&counts[bucket(r)], 1u)] = r;
}

template <bool kVec>
__global__ void __launch_bounds__(kPairThreads, 4) gdn_prefill_pairs_kernel(const __grid_constant__ PrefillArgs p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  PairSmem& s = *reinterpret_cast<PairSmem*>(raw);
  grid_dependency_wait();
  allow_dependent_launch();
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  if (blockIdx.x == 0) {
    order_requests(p, s.counts, tid);
    return;
  }
  const int64_t place = (blockIdx.x - 1) / p.num_k_heads;
  const int kh = static_cast<int>(blockIdx.x - 1 - place * p.num_k_heads);
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
  uint16_t* tiles = reinterpret_cast<uint16_t*>(s.kq());
  const auto at = [](int row, int col) { return swz<kKeyHalf>(row, col); };
  load_rows<kVec, kPairThreads>(rows + (p.num_k_heads + kh) * kDim, p.qkv_row, row_lo, row_hi, tiles, tid, at);
  load_rows<kVec, kPairThreads>(rows + kh * kDim, p.qkv_row, row_lo, row_hi, tiles + kHalf, tid, at);
  const int head0 = kh * p.heads_ratio;
  if (w < p.heads_ratio) chunk_gates(p, s, w, token0, row_lo, row_hi, head0 + w, lane);
  if constexpr (kVec) cp_async_wait();
  __syncthreads();
  if (tid < kChunk) {
    s.fk[tid] = scale_row(tiles, tid);
  } else {
    s.fq[tid - kChunk] = scale_row(tiles + kHalf, tid - kChunk);
  }
  __syncthreads();
  {
    uint4* to = reinterpret_cast<uint4*>(p.keys + place * p.num_k_heads + kh);
    const uint4* from = reinterpret_cast<const uint4*>(s.kq());
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(KeyImage)) / (16 * kPairThreads); ++i) {
      to[i * kPairThreads + tid] = from[i * kPairThreads + tid];
    }
  }
  const Blocks mine(w);
  float kk[3][2][4], qk[3][2][4];
  row_products(s, mine, lane, kk, qk);
  __syncthreads();
  if (w < 2) {
    const float* f = w == 0 ? s.fk : s.fq;
    float* unit = w == 0 ? s.fk_unit : s.fq_unit;
    const float power = largest_power(unit[lane], unit[lane + 32]), down = inverse_power(power);
    unit[lane] = f[lane] * down;
    unit[lane + 32] = f[lane + 32] * down;
    if (lane == 0) (w == 0 ? s.fk_power : s.fq_power) = power;
  }
  __syncthreads();
#pragma unroll 1
  for (int n = 0; n < p.heads_ratio; n += 2) {
    const int at = n % kGroup;
    const int heads = min(p.heads_ratio - n, 2);
    PairImage* images = p.pairs + place * p.num_v_heads + head0 + n;
    if (n > 0) {
      __syncthreads();  // the heads' inverses and, every fourth head, the gates are taken over
      if (at == 0) {
        if (n + w < p.heads_ratio) chunk_gates(p, s, w, token0, row_lo, row_hi, head0 + n + w, lane);
        __syncthreads();
      }
    }
    if ((w >> 1) < heads) row_factors(p, s, at + (w >> 1), tid & (kChunk - 1), images[w >> 1].main);
#pragma unroll 1
    for (int i = 0; i < heads; ++i) decayed_pairs(p, s, s.head(i), at + i, mine, lane, kk, qk, images[i].main);
    __syncwarp();
    if ((lane >> 4) < heads) invert_diagonal(s.head(lane >> 4), w, lane & 15);
    __syncthreads();
    // Columns 0, 1 and 2 have 3, 2 and 1 blocks: a warp takes the first, another the other two.
    if ((w & 1) < heads) {
      for (int col = w >> 1; col <= (w & 2); ++col) invert_column(s.head(w & 1), col, lane);
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < heads; ++i) {
      PairHead& head = s.head(i);
#pragma unroll
      for (int k = 0; k < 2 * kLowBlocks * 32 / kPairThreads; ++k) {  // 16 bytes of the blocks below the diagonal
        const int at = k * kPairThreads + tid, low = at % (kLowBlocks * 32);
        const int from = 256 * below_place(low >> 5) + 8 * (low & 31);
        if (at < kLowBlocks * 32) {
          *reinterpret_cast<uint4*>(&images[i].main.t_hi[from]) = *reinterpret_cast<const uint4*>(&head.t_hi[from]);
        } else {
          *reinterpret_cast<uint4*>(&images[i].t_lo[8 * low]) = *reinterpret_cast<const uint4*>(&head.t_lo[from]);
        }
      }
      // This warp's diagonal block, its lo terms transposed above the diagonal, where hi has zeros and lo has none below.
      uint32_t hi[4], lo[4];
      ldsm4(core_addr(head.t_hi, lane) + 2 * tri_block(w, w), hi);
      ldsm4_t(core_addr(head.t_lo, lane) + 2 * tri_block(w, w), lo);
      uint32_t* to = reinterpret_cast<uint32_t*>(&images[i].main.t_hi[tri_block(w, w) + core(lane >> 2, 2 * (lane & 3))]);
      to[0] = hi[0] | lo[0];
      to[32] = lo[2];  // the upper right core matrix: the lower left one's
      to[64] = hi[2];
      to[96] = hi[3] | lo[3];
    }
  }
}

// ------------------------------------------------------------------------------------------
// chain: the state through the chunks
// ------------------------------------------------------------------------------------------
constexpr int kIssuers = 3;   // warps that issue products
// Moving warps with a task of their own beside the common ones: warp 0 issues P u, these ask for a stage's bulk copies and
// wait for them, and find out the upcoming work.  All by warp 0, the moving threads took longer than the chain.
constexpr int kCopyWarp = 3, kTakeWarp = 5;
constexpr int kVRow = kDim + 8;  // bf16 per row of a stage's v and gate: the 16 bytes spread their rows over the banks

// What a stage holds: one chunk of one item.
struct Work {
  int64_t token0;      // the token of row 0 (rows in front of row_lo have none)
  int64_t place;       // the chunk's place in the workspace; kWorkZero: the item's tokens
  int32_t row_lo, row_hi;
  int32_t head;
  int32_t source;      // the slot that the state starts from (0: from nothing), or one of these:
  int32_t matrix;      // kSourceMatrix: the matrix of `states`
  int32_t save;        // the matrix of `states` that takes the state after the chunk (-1: none)
  int32_t quiet;       // no outputs
  int32_t slot;        // the slot that takes the state after the chunk (0: none)
  int32_t kind;
};
constexpr int kSourceOn = -1, kSourceIdentity = -2, kSourceMatrix = -3;  // the state goes on; identity; a matrix
constexpr int kWorkChunk = 0, kWorkEnd = 1, kWorkZero = 2;  // a chunk; no more items; an item whose outputs are zeros

// Where the item in work is, kept and used by one thread.
struct Cursor {
  const int32_t* slot_at;  // the slot of the block that the next chunk is in
  uint32_t ahead;          // the item after this one, taken with this one's last chunk
  int32_t rest;            // tokens behind the upcoming chunk
  int32_t left;            // chunks to the end of the block, the upcoming one not counted
  int32_t per_block;
  int32_t save;            // the matrix of `states` that takes the item's last state (-1: none)
  bool last;               // the item ends with its request
  bool blind;              // no v: every row counts as one of no token
};

struct __align__(1024) Stage {
  __half kq[2 * kChunk * kDim];
  PairMain pair;  // t_hi without lo terms above the diagonal once it is unpacked
  __align__(16) __half t_lo[kTriBlocks * 256];
  __half p_lo[kTriBlocks * 256];
  __align__(16) __nv_bfloat16 v[kChunk * kVRow];
  __align__(16) __nv_bfloat16 gate[kChunk * kVRow];
  Work work;
};

struct ChainSmem {
  Stage stage[2];
  __align__(16) float o[kChunk * kORow];
  float s_down[kDim], u_down[kDim];  // what S q and P u of the chunk in work are scaled by, per value row
  uint64_t full[2];  // a stage's copies have landed
  uint64_t done[3];  // products finished: [0] what the state waits for, [1] P u, [2] S q
  uint64_t drained;  // after a wait that ran out: every product, a commit of each warp that issues some
  uint32_t tmem;
  Cursor at;
  Work upcoming;      // what the next free stage takes
  volatile int stop;  // a wait ran out: nothing is stored any more
  int keep;           // the issuing warp's answer for the chunk in work: no wait ran out, its state may be stored
};

static_assert(sizeof(ChainSmem) <= 227 * 1024, "shared memory of a CTA");

// TMEM columns (32 bits x 128 lanes, lane = value row); all 512 are allocated, so they start at 0.  dS takes
// the place of Y and T R, which are in registers by then, and P u that of R.
constexpr uint32_t kTmemS = 0, kTmemR = 128, kTmemPu = 128, kTmemU = 192, kTmemW = 224, kTmemY = 288, kTmemTr = 352,
                   kTmemDs = 288, kTmemO = 416, kTmemUlo = 480, kTmemColumns = 512;

// The chunk's images to a stage by bulk copies, its v rows by the moving threads.
template <bool kVec>
__device__ __forceinline__ void copy_chunk(const PrefillArgs& p, Stage& st, const Work& d, uint32_t full, int tid, bool late) {
  // What was read and written in this stage so far comes before the bulk copies, which go through the async
  // proxy (a barrier lies between that and this thread).
  if (tid == 32 * kCopyWarp && !late) {  // after a wait that ran out there are no more of them, and the ones before have landed
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    barrier_expect(full, sizeof(KeyImage) + sizeof(PairImage) + p.extra_tx);
    bulk_copy(smem_u32(st.kq), p.keys + d.place * p.num_k_heads + d.head / p.heads_ratio, sizeof(KeyImage), full);
    const PairImage* pair = p.pairs + d.place * p.num_v_heads + d.head;
    bulk_copy(smem_u32(&st.pair), &pair->main, sizeof(PairMain), full);
#pragma unroll
    for (int col = 0; col < 3; ++col) {  // a column's blocks below its diagonal one
      bulk_copy(smem_u32(&st.t_lo[tri_block(col + 1, col)]), &pair->t_lo[256 * below_block(col + 1, col)], (3 - col) * 512, full);
    }
  }
  // Rows of no token are zeros: their beta is 0, but 0 times what lies there need not be 0.
  load_rows<kVec, kMoveThreads>(p.qkv + d.token0 * p.qkv_row + (2 * p.num_k_heads + d.head) * kDim, p.qkv_row, d.row_lo,
                                d.row_hi, reinterpret_cast<uint16_t*>(st.v), tid,
                                [](int row, int col) { return row * kVRow + col; });
}

// The lo terms of a stage's T and P from what their image has of them, and zeros where T's were, by the moving threads.  The
// upper right core matrices of diagonal blocks of t_lo and p_lo are zeros from the start and stay so.
__device__ __forceinline__ void unpack_chunk(Stage& st, int tid) {
  const int warp = tid >> 5, lane = tid & 31;
  constexpr int kUnits = 8 * (4 * kLowBlocks + 3 * 4);  // rows of 8 elements
#pragma unroll 1
  for (int unit = tid; unit < kUnits; unit += kMoveThreads) {
    int at = 256 * below_place(unit >> 5) + 8 * (unit & 31);
    if (unit >= 32 * kLowBlocks) {
      const int diagonal = unit - 32 * kLowBlocks, block = diagonal / 24, row = diagonal - 24 * block;
      at = tri_block(block, block) + 8 * row + (row >= 8 ? 64 : 0);
    }
    const uint2 b = *reinterpret_cast<const uint2*>(&st.pair.p_lo[8 * unit]);
    const uint4 h = *reinterpret_cast<const uint4*>(&st.pair.p_hi[at]);
    *reinterpret_cast<uint4*>(&st.p_lo[at]) =
        make_uint4(lo_terms(h.x, __byte_perm(b.x, 0, 0x4140)), lo_terms(h.y, __byte_perm(b.x, 0, 0x4342)),
                   lo_terms(h.z, __byte_perm(b.y, 0, 0x4140)), lo_terms(h.w, __byte_perm(b.y, 0, 0x4342)));
  }
  if (warp >= kMoveThreads / 32 - 4) {
    const int w = warp & 3, g = lane >> 2, t = lane & 3;
    const uint32_t from = core_addr(st.pair.t_hi, lane) + 2 * tri_block(w, w);
    uint32_t m[4], turned[4];
    ldsm4(from, m);
    ldsm4_t(from, turned);
    __syncwarp();
    const uint32_t below = 2 * t + 1 < g ? 0xffffffffu : 2 * t < g ? 0xffffu : 0u;
    const uint32_t upto = 2 * t + 1 <= g ? 0xffffffffu : 2 * t <= g ? 0xffffu : 0u;
    const int at = tri_block(w, w) + core(g, 2 * t);
    uint32_t* hi = reinterpret_cast<uint32_t*>(&st.pair.t_hi[at]);
    uint32_t* lo = reinterpret_cast<uint32_t*>(&st.t_lo[at]);
    lo[0] = turned[0] & below;
    lo[64] = turned[1];  // lower left
    lo[96] = turned[3] & below;
    hi[0] = m[0] & upto;
    hi[32] = 0;
    hi[96] = m[3] & upto;
  }
}

// The chunk's gate rows, which only the moving threads read, when the ones before have been used.
template <bool kVec>
__device__ __forceinline__ void copy_gates(const PrefillArgs& p, Stage& st, int tid) {
  const Work& d = st.work;
  if (d.kind == kWorkChunk && !d.quiet) {
    load_rows<kVec, kMoveThreads>(p.gate + d.token0 * p.gate_row + d.head * kDim, p.gate_row, d.row_lo, d.row_hi,
                                  reinterpret_cast<uint16_t*>(st.gate), tid,
                                  [](int row, int col) { return row * kVRow + col; });
  }
}

// The chunk's outputs S q + P u from TMEM to the output tile: this warp's 16 value rows, 16 columns at a time.
__device__ __forceinline__ void gather_outputs(ChainSmem& s, const Stage& st, int v0, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const uint32_t tmem = static_cast<uint32_t>(v0) << 16;
  const float2 s0 = make_float2(s.s_down[v0 + g], s.s_down[v0 + g]);
  const float2 s1 = make_float2(s.s_down[v0 + g + 8], s.s_down[v0 + g + 8]);
  const float2 u0 = make_float2(s.u_down[v0 + g], s.u_down[v0 + g]);
  const float2 u1 = make_float2(s.u_down[v0 + g + 8], s.u_down[v0 + g + 8]);
#pragma unroll 1
  for (int nb = 0; nb < 4; ++nb) {
    float o[2][4], pu[2][4];
    tmem_load(tmem + kTmemO + 16 * nb, tmem + kTmemPu + 16 * nb, o, pu);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int col = 16 * nb + 8 * m + 2 * t;
      const float2 qin = *reinterpret_cast<const float2*>(&st.pair.q_in[col]);
      const float2 x0 = fma2(make_float2(o[m][0], o[m][1]), mul2(qin, s0), mul2(make_float2(pu[m][0], pu[m][1]), u0));
      const float2 x1 = fma2(make_float2(o[m][2], o[m][3]), mul2(qin, s1), mul2(make_float2(pu[m][2], pu[m][3]), u1));
      float* at = s.o + col * kORow + v0 + g;
      at[0] = x0.x;
      at[kORow] = x0.y;
      at[8] = x1.x;
      at[kORow + 8] = x1.y;
    }
  }
}

// Gated RMSNorm of the output tile.  A warp takes two rows at a time, 16 lanes and twice four values per lane each, and
// two such turns are unrolled, no more: the chain's warps run through so much straight code that the instruction cache is
// what they compete for.
template <bool kVec>
__device__ __forceinline__ void store_outputs(const PrefillArgs& p, const ChainSmem& s, const Stage& st, const Work& d,
                                              const float2 (&wt)[4], int tid) {
  const int part = tid & 15;
  const bool stop = s.stop != 0 || d.quiet;
  __nv_bfloat16* out = p.out + (d.token0 * p.num_v_heads + d.head) * kDim + 4 * part;
#pragma unroll 2
  for (int i = tid >> 4; i < kChunk; i += kMoveThreads / 16) {
    float2 o[2][2], sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const float4 x = *reinterpret_cast<const float4*>(&s.o[i * kORow + 64 * half + 4 * part]);
      o[half][0] = make_float2(x.x, x.y);
      o[half][1] = make_float2(x.z, x.w);
      sum = fma2(o[half][0], o[half][0], sum);
      sum = fma2(o[half][1], o[half][1], sum);
    }
    float sq = sum.x + sum.y;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    const float rstd = rsqrtf(sq * (1.0f / kDim) + p.eps);
    const bool live = i >= d.row_lo && i < d.row_hi && !stop;
    __nv_bfloat16* row = out + static_cast<int64_t>(i) * p.num_v_heads * kDim;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint2 z = *reinterpret_cast<const uint2*>(&st.gate[i * kVRow + 64 * half + 4 * part]);
      const float2 r = make_float2(rstd, rstd);
      const float2 y0 = mul2(mul2(o[half][0], r), mul2(wt[2 * half], silu_fast(make_float2(bf16_low(z.x), bf16_high(z.x)))));
      const float2 y1 =
          mul2(mul2(o[half][1], r), mul2(wt[2 * half + 1], silu_fast(make_float2(bf16_low(z.y), bf16_high(z.y)))));
      const uint32_t lo = pack_bf16(y0.x, y0.y), hi = pack_bf16(y1.x, y1.y);
      __nv_bfloat16* at = row + 64 * half;
      if (live) {
        if constexpr (kVec) {
          *reinterpret_cast<uint2*>(at) = make_uint2(lo, hi);
        } else {
          at[0] = __ushort_as_bfloat16(static_cast<unsigned short>(lo));
          at[1] = __ushort_as_bfloat16(static_cast<unsigned short>(lo >> 16));
          at[2] = __ushort_as_bfloat16(static_cast<unsigned short>(hi));
          at[3] = __ushort_as_bfloat16(static_cast<unsigned short>(hi >> 16));
        }
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

// Waits until the barrier's phase has completed, the warp together.  After limit_ns it gives up for good:
// it raises the fault, and from then on this warp stores nothing and waits for no product.
__device__ __forceinline__ void wait_done(uint32_t bar, uint32_t parity, ChainSmem& s, bool& dead, uint64_t limit_ns) {
  if (dead) return;
  uint64_t start = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, ok != 0)) break;
    uint64_t now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now)::"memory");
    if (start == 0) start = now;
    if (__any_sync(0xffffffffu, now - start > limit_ns)) {
      dead = true;
      s.stop = 1;
      atomicOr(&g_prefill_faults, LD_FAULT_WAIT_TIMEOUT);
      break;
    }
  }
  tmem_after();
}

__device__ __forceinline__ float largest(float x, float y, float z) {  // of the magnitudes
  float m;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
  return m;
}

// Largest magnitudes of the two rows of a fragment array, over the row's four lanes, as row scales.
template <int kTiles>
__device__ __forceinline__ void scale_rows(const float (&x)[kTiles][4], float& up0, float& down0, float& up1,
                                           float& down1) {
  float top0[2] = {}, top1[2] = {};  // of even and odd tiles: shorter chains
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    top0[n & 1] = largest(top0[n & 1], x[n][0], x[n][1]);
    top1[n & 1] = largest(top1[n & 1], x[n][2], x[n][3]);
  }
  row_scale(quad_max(fmaxf(top0[0], top0[1])), up0, down0);
  row_scale(quad_max(fmaxf(top1[0], top1[1])), up1, down1);
}

// Four k-steps (64 columns) of a fragment array, scaled, as hi and lo A operands in TMEM.
template <int kTiles>
__device__ __forceinline__ void store_split(const float (&x)[kTiles][4], int first, float up0, float up1,
                                            uint32_t hi_at, uint32_t lo_at) {
  uint32_t hi[4][4], lo[4][4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float(&f)[4] = x[first + 2 * ks + m];
      split_masked(mul2(make_float2(f[0], f[1]), make_float2(up0, up0)), hi[ks][2 * m], lo[ks][2 * m]);
      split_masked(mul2(make_float2(f[2], f[3]), make_float2(up1, up1)), hi[ks][2 * m + 1], lo[ks][2 * m + 1]);
    }
  }
  tmem_store(hi_at, hi);
  tmem_store(lo_at, lo);
}

// f = a f + b x, a pair of columns of two rows at a time.
__device__ __forceinline__ void scale_add(float (&f)[4], float2 a0, float2 a1, const float (&x)[4], float2 b0, float2 b1) {
  const float2 lo = fma2(make_float2(f[0], f[1]), a0, mul2(make_float2(x[0], x[1]), b0));
  const float2 hi = fma2(make_float2(f[2], f[3]), a1, mul2(make_float2(x[2], x[3]), b1));
  f[0] = lo.x;
  f[1] = lo.y;
  f[2] = hi.x;
  f[3] = hi.y;
}

// What the threads that carry the state keep between chunks.
struct StateWarp {
  float S[16][4];  // rows v0 + g, v0 + g + 8; columns 8n + 2t, + 1
  uint32_t phase;
  bool dead;
  bool issuer;  // issues what the state waits for
  bool reader;  // issues S q
};

extern __shared__ __align__(1024) unsigned char chain_raw[];

// The products of one chunk.  Three warps issue them, since a warp issues one every 30 to 45 cycles whatever its size: one
// state warp those that the state waits for, another one S q beside T R, and a moving warp P u when the chunk is done.  All by
// the first, the 28 products that only the outputs need took 750 cycles a chunk.
struct Products {
  const Stage& st;
  uint32_t elected;

  __device__ __forceinline__ explicit Products(const Stage& stage) : st(stage), elected(elect_lane()) { tmem_after(); }
  static __device__ __forceinline__ uint32_t done(int i) { return smem_u32(&reinterpret_cast<ChainSmem*>(chain_raw)->done[i]); }

  // D = S x~, two terms, for k~ or q~.
  __device__ __forceinline__ void of_state(uint32_t d, const __half* tile, uint32_t bar) const {
    const uint64_t b = tile_desc(smem_u32(tile));
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {  // k-steps of lo, then of hi
      const uint32_t ks = i & 7;
      umma(elected, d, kTmemS + 64 - 8 * (i & 8) + 8 * ks, b + ((ks >> 2) * (2 * kKeyHalf >> 4) + (ks & 3) * 2),
           mma_shape(64, false), i > 0);
    }
    umma_commit(elected, bar);
  }

  // D = X M for a triangle M, two terms each (the product of the two lo terms is below fp32's last bit).  M's column block
  // ks starts at row block ks.
  __device__ __forceinline__ void of_triangle(uint32_t d, uint32_t x_hi, uint32_t x_lo, const __half* m_hi, const __half* m_lo,
                                              uint32_t bar) const {
    const uint64_t b_hi = tri_desc(smem_u32(m_hi)), b_lo = tri_desc(smem_u32(m_lo));
#pragma unroll
    for (uint32_t ks = 0; ks < 4; ++ks) {  // small terms first in each column block
      const uint32_t at = 2 * tri_block(ks, ks) >> 4, shape = mma_shape(64 - 16 * ks, false);
      umma(elected, d + 16 * ks, x_hi + 8 * ks, b_lo + at, shape, ks > 0);
      umma(elected, d + 16 * ks, x_lo + 8 * ks, b_hi + at, shape, true);
      umma(elected, d + 16 * ks, x_hi + 8 * ks, b_hi + at, shape, true);
    }
    umma_commit(elected, bar);
  }

  __device__ __forceinline__ void state_keys() const { of_state(kTmemY, st.kq, done(0)); }
  __device__ __forceinline__ void state_queries() const { of_state(kTmemO, st.kq + kHalf, done(2)); }
  __device__ __forceinline__ void corrections() const {
    of_triangle(kTmemTr, kTmemR, kTmemR + 32, st.pair.t_hi, st.t_lo, done(0));
  }
  __device__ __forceinline__ void within() const { of_triangle(kTmemPu, kTmemU, kTmemUlo, st.pair.p_hi, st.p_lo, done(1)); }

  // dS = (k_out u) k~, two terms.
  __device__ __forceinline__ void update() const {
    const uint64_t k = tile_desc(smem_u32(st.kq));
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {  // k-steps of lo, then of hi
      umma(elected, kTmemDs, kTmemW + 32 - 8 * (i & 4) + 8 * (i & 3), k + (i & 3) * (2048 >> 4), mma_shape(128, true), i > 0);
    }
    umma_commit(elected, done(0));
  }
};

// The products that the state waits for are done.  One warp asks the barrier, the others wait for it at a named
// barrier: asking, eight warps took so many issue slots from the one that issues that a product of 32 cycles
// (N = 64) was issued every 48.
//
// With kLast, the chunk's last ones, the issuing warp also says whether the chunk's state may be stored.  `stop` may be set
// at any moment, by the moving threads too: were every warp to read it, a slot could take some warps' rows alone.
//
// S q, which reads S where the next chunk's goes, is over with the chunk, too: its issuer waits for it here.
template <bool kLast = false>
__device__ __forceinline__ void wait_products(StateWarp& x, ChainSmem& s, uint64_t limit_ns) {
  if (x.issuer) {
    wait_done(smem_u32(&s.done[0]), x.phase, s, x.dead, limit_ns);
    x.phase ^= 1;
    if constexpr (kLast) s.keep = s.stop == 0;
  }
  if (kLast && x.reader) {
    wait_done(smem_u32(&s.done[2]), x.phase, s, x.dead, limit_ns);
    x.phase ^= 1;
  }
  bar_state();
  tmem_after();
}

// One chunk.  `tmem` carries this warp's lanes.  `taken` returns when the outputs of the chunk before have left TMEM.
//
// Parity waits are sound because the warp that waits on a barrier has seen a phase before the next one can begin: each
// has one warp that both commits and waits.
template <typename Taken>
__device__ __forceinline__ void chain_chunk(StateWarp& x, ChainSmem& s, int stage, uint32_t tmem, int v0, int lane,
                                            uint64_t limit_ns, Taken taken) {
  const int g = lane >> 2, t = lane & 3;
  const Stage& st = s.stage[stage];

  // Y = S k~ (two terms).
  float up0, down0, up1, down1;
  scale_rows(x.S, up0, down0, up1, down1);
  store_split(x.S, 0, up0, up1, tmem + kTmemS, tmem + kTmemS + 64);
  store_split(x.S, 8, up0, up1, tmem + kTmemS + 32, tmem + kTmemS + 96);
  tmem_stored();
  tmem_before();
  bar_state();
  if (x.issuer && !x.dead) Products(st).state_keys();

  // R = beta (v - k_in Y).
  wait_products(x, s, limit_ns);
  float Y[8][4];
  tmem_load(tmem + kTmemY, Y);
  const uint32_t v_base =
      smem_u32(st.v) + 2 * (((lane & 7) + 8 * (lane >> 4)) * kVRow + v0 + 8 * ((lane >> 3) & 1));
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
    uint32_t vt[4];  // v transposed: (rows 16nb.., cols v0..), (.., v0 + 8..), (rows 16nb + 8.., ...)
    ldsm4_t(v_base + nb * (16 * kVRow * 2), vt);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float(&f)[4] = Y[2 * nb + m];
      const float2 kin = *reinterpret_cast<const float2*>(&st.pair.k_in[16 * nb + 8 * m + 2 * t]);
      const float2 beta = *reinterpret_cast<const float2*>(&st.pair.beta[16 * nb + 8 * m + 2 * t]);
      const uint32_t r0 = vt[2 * m], r1 = vt[2 * m + 1];
      const float2 y0 = fma2(mul2(kin, make_float2(-down0, -down0)), make_float2(f[0], f[1]),
                             make_float2(bf16_low(r0), bf16_high(r0)));
      const float2 y1 = fma2(mul2(kin, make_float2(-down1, -down1)), make_float2(f[2], f[3]),
                             make_float2(bf16_low(r1), bf16_high(r1)));
      const float2 z0 = mul2(beta, y0), z1 = mul2(beta, y1);
      f[0] = z0.x;
      f[1] = z0.y;
      f[2] = z1.x;
      f[3] = z1.y;
    }
  }
  taken();  // R takes the place of the chunk before's P u
  if (t == 0) {
    s.s_down[v0 + g] = down0;
    s.s_down[v0 + g + 8] = down1;
  }
  scale_rows(Y, up0, down0, up1, down1);
  store_split(Y, 0, up0, up1, tmem + kTmemR, tmem + kTmemR + 32);
  tmem_stored();
  tmem_before();
  bar_state();
  // U = T R, and S q beside it.
  if (x.issuer && !x.dead) Products(st).corrections();
  if (x.reader && !x.dead) Products(st).state_queries();

  // k_out u, in two terms.  The largest k_out is in [1, 2), so u's row scale serves both.
  wait_products(x, s, limit_ns);
  tmem_load(tmem + kTmemTr, Y);
  const float r_down0 = down0, r_down1 = down1;
  scale_rows(Y, up0, down0, up1, down1);
  const float w0 = r_down0 * down0, w1 = r_down1 * down1;
  if (t == 0) {
    s.u_down[v0 + g] = w0 * st.pair.p_scale();
    s.u_down[v0 + g + 8] = w1 * st.pair.p_scale();
  }
  {
    uint32_t hi[4][4], lo[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float(&f)[4] = Y[2 * ks + m];
        const float2 u0 = mul2(make_float2(f[0], f[1]), make_float2(up0, up0));
        const float2 u1 = mul2(make_float2(f[2], f[3]), make_float2(up1, up1));
        f[0] = u0.x;
        f[1] = u0.y;
        f[2] = u1.x;
        f[3] = u1.y;
        const float2 kout = *reinterpret_cast<const float2*>(&st.pair.k_out[16 * ks + 8 * m + 2 * t]);
        split_masked(mul2(u0, kout), hi[ks][2 * m], lo[ks][2 * m]);
        split_masked(mul2(u1, kout), hi[ks][2 * m + 1], lo[ks][2 * m + 1]);
      }
    }
    tmem_store(tmem + kTmemW, hi);
    tmem_store(tmem + kTmemW + 32, lo);
  }
  tmem_stored();
  tmem_before();
  bar_state();
  if (x.issuer && !x.dead) Products(st).update();
  // u, in two terms, for P u, while dS is at work.
  store_split(Y, 0, 1.0f, 1.0f, tmem + kTmemU, tmem + kTmemUlo);
  tmem_stored();
  tmem_before();
  // S <- decay S + dS, one fp32 fused multiply-add per element.
  const float2 decay = make_float2(st.pair.decay(), st.pair.decay());
  const float k0 = w0 * st.pair.k_scale(), k1 = w1 * st.pair.k_scale();
  const float2 w02 = make_float2(k0, k0), w12 = make_float2(k1, k1);
  wait_products<true>(x, s, limit_ns);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    tmem_load(tmem + kTmemDs + 64 * half, Y);
#pragma unroll
    for (int n = 0; n < 8; ++n) scale_add(x.S[8 * half + n], decay, decay, Y[n], w02, w12);
  }
}

// Where the state goes after the upcoming chunk: to a slot when a block or the request ends with it, and to a matrix
// when a split request's piece does.
template <bool kSplit>
__device__ __forceinline__ void work_ends(const PrefillArgs& p, Cursor& at, Work& d) {
  d.slot = 0;
  if constexpr (kSplit) {
    d.save = at.rest <= 0 ? at.save : -1;
    if (at.blind) d.row_lo = d.row_hi = 0;
  }
  const bool last = !kSplit || at.last, quiet = kSplit && d.quiet;
  if (!quiet && (at.left == 0 || (at.rest <= 0 && last))) {
    d.slot = *at.slot_at++;
    at.left = at.per_block;
    if (d.slot >= p.n_slots) {
      if (d.head == 0) atomicOr(&g_prefill_faults, LD_FAULT_DECODE_SLOT_RANGE);
      d.slot = 0;
    }
  }
  --at.left;
}

// The first chunk of the next item that has some, the end, or an item whose outputs are zeros.  One thread.
template <bool kSplit>
__device__ __noinline__ void next_item(const PrefillArgs& p, Cursor& at, Work& d) {
  const int64_t per_block = p.block_size / kChunk;
  const uint32_t heads = p.num_v_heads, parts = !kSplit ? 1 : p.pass == 0 ? p.pieces.first_parts() : p.pieces.count - 1;
  while (true) {
    const uint32_t item = at.ahead;
    if (item >= p.n_requests * parts * heads) {
      d.kind = kWorkEnd;
      return;
    }
    const auto take = [&] { at.ahead = atomicAdd(p.next + p.pass, 1u); };
    const int part = static_cast<int>(item / heads % parts);
    const int r = p.order[item / heads / parts];
    const bool first = !kSplit || (p.pass == 0 && part == 0);
    d.head = static_cast<int>(item % heads);
    at.rest = 0;
    Request rq;
    unsigned int fault;
    bool skip;
    if (find_request(p, r, rq, fault, skip)) {
      // Chunks [lo, hi) of the request.
      const bool split = kSplit && worth_splitting(p.pieces, rq.chunks);
      if (!split && !first) {
        take();
        continue;
      }
      const int piece = p.pass == 0 ? (part + 1) / 2 : part + 1;
      const int64_t cuts = p.pieces.cut(p.pieces.count);
      const int64_t lo = split ? rq.chunks * p.pieces.cut(piece) / cuts : 0;
      const int64_t hi = split ? rq.chunks * p.pieces.cut(piece + 1) / cuts : rq.chunks;
      // Chunks end at absolute positions that are multiples of 64, and so do blocks.
      const int64_t position = rq.context / kChunk + lo;
      at.per_block = static_cast<int32_t>(min(per_block, static_cast<int64_t>(INT32_MAX)));
      at.left = static_cast<int32_t>(min(per_block - 1 - position % per_block, static_cast<int64_t>(INT32_MAX)));
      at.slot_at = rq.row + position / per_block;
      at.last = hi == rq.chunks;
      const int64_t before = lo * kChunk - rq.lead;  // tokens in front of row 0
      at.rest = static_cast<int32_t>((at.last ? rq.tokens : hi * kChunk - rq.lead) - before - kChunk);
      const int32_t matrices = static_cast<int32_t>(r * heads + d.head) * p.pieces.first_parts();
      at.save = split && p.pass == 0 ? matrices + part : -1;
      at.blind = p.pass == 0 && (part & 1) != 0;
      d.quiet = p.pass == 0 && part != 0;
      d.token0 = rq.first + before;
      d.place = chunk_base(rq.first, r) + lo;
      d.row_lo = lo == 0 ? rq.lead : 0;
      d.row_hi = kChunk + min(at.rest, 0);
      d.source = first ? rq.source : p.pass != 0 ? kSourceMatrix : at.blind ? kSourceIdentity : 0;
      d.matrix = matrices + 2 * part;  // S_1 is where piece 0 left it, S_{k+1} in the place of B_k
      d.kind = kWorkChunk;
      work_ends<kSplit>(p, at, d);
      if (at.rest <= 0) take();
      return;
    }
    take();
    if (!first) continue;
    if (fault != 0 && d.head == 0) atomicOr(&g_prefill_faults, fault);
    if (!skip) {
      d.token0 = rq.first;
      d.place = rq.tokens;
      d.kind = kWorkZero;
      return;
    }
  }
}

// The upcoming work after the one in `d`.  One thread.
template <bool kSplit>
__device__ __forceinline__ void next_work(const PrefillArgs& p, Cursor& at, Work& d) {
  if (at.rest <= 0) {
    next_item<kSplit>(p, at, d);
    return;
  }
  d.token0 += kChunk;
  d.place += 1;
  d.row_lo = 0;
  d.row_hi = min(at.rest, kChunk);
  d.source = kSourceOn;
  at.rest -= kChunk;
  work_ends<kSplit>(p, at, d);
  if (at.rest <= 0) at.ahead = atomicAdd(p.next + p.pass, 1u);
}

// Writes the zero outputs of upcoming items that cannot run, until a chunk or the end is next.  The moving
// threads together.
__device__ __noinline__ void zero_item(const PrefillArgs& p, const Work& d, int tid) {
  // `place` rows of 256 bytes, one warp a row.
  for (int64_t i = tid >> 5; i < d.place; i += kMoveThreads / 32) {
    __nv_bfloat16* row = p.out + ((d.token0 + i) * p.num_v_heads + d.head) * kDim;
    for (int c = tid & 31; c < kDim; c += 32) row[c] = __float2bfloat16_rn(0.0f);
  }
}

template <bool kSplit>
__device__ __forceinline__ void skip_items(const PrefillArgs& p, ChainSmem& s, int tid) {
  while (s.upcoming.kind == kWorkZero) {
    if (s.stop == 0) zero_item(p, s.upcoming, tid);
    bar_move();
    if (tid == 0) next_item<kSplit>(p, s.at, s.upcoming);
    bar_move();
  }
}

// Gives a free stage the upcoming work and starts its copies.  The moving threads together.
template <typename StateT, bool kVec>
__device__ __forceinline__ void load_stage(const PrefillArgs& p, Stage& st, const Work& d, uint32_t full, int tid, bool late) {
  if (tid == 0) st.work = d;
  if (d.kind == kWorkEnd) return;
  if (d.source > 0 && tid < 32) {  // a new item's state: into L2 by the time that it is read
    const char* state = reinterpret_cast<const char*>(static_cast<const StateT*>(p.state) + d.source * p.slot_stride +
                                                      static_cast<int64_t>(d.head) * kDim * kDim);
    constexpr int kBytes = kDim * kDim * sizeof(StateT) / 32;
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(state + tid * kBytes), "n"(kBytes) : "memory");
  }
  copy_chunk<kVec>(p, st, d, full, tid, late);
}

// A persistent CTA per SM: the moving threads take items (a request's value head each), longest first, and
// feed their chunks through two stages without a gap between items.
template <typename StateT, bool kVec, bool kSplit>
__global__ void __launch_bounds__(kChainThreads, 1) gdn_prefill_chain_kernel(const __grid_constant__ PrefillArgs p) {
  ChainSmem& s = *reinterpret_cast<ChainSmem*>(chain_raw);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kStateWarp = kMoveThreads / 32;

  // Launched with 512 x 128 registers; 256 x 96 + 256 x 160 is the same 65,536.
  if (warp < kStateWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    const int tid = threadIdx.x;
    const auto full = [&](int stage) { return smem_u32(&s.full[stage]); };
    // A stage is handed over when its copies have landed (every thread waits for its own, one warp for the bulk
    // copies) and its second terms are unpacked.
    uint32_t landed = 0;
    bool late = false;
    uint32_t owed = 0, owed_parity = 0;  // the barrier of copies that a wait ran out for
    const auto hand_over = [&](int stage, bool chunk) {
      cp_async_wait_groups<1>();  // but not for the gates, which were asked for last
      if (chunk) {
        if (warp == kCopyWarp) {
          const uint32_t parity = (landed >> stage) & 1;
          const bool before = late;
          wait_done(full(stage), parity, s, late, p.wait_ns);
          if (late && !before) {
            owed = full(stage);
            owed_parity = parity;
          }
          landed ^= 1u << stage;
        }
        bar_move();  // they have landed for everybody
        unpack_chunk(s.stage[stage], tid);
        // Products read what was written here, and later copies write over it, both through the async proxy.
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      bar_arrive(kBarFull + stage);
    };
    {  // the core matrices that unpack_chunk leaves alone: 32 words in each of two stages' eight diagonal blocks
      Stage& st = s.stage[tid >> 7];
      const int block = (tid >> 5) & 3, at = tri_block(block, block) + 64 + 2 * lane;
      *reinterpret_cast<uint32_t*>(&st.t_lo[at]) = 0;
      *reinterpret_cast<uint32_t*>(&st.p_lo[at]) = 0;
    }
    if (tid == 0) {
      for (int i = 0; i < 2; ++i) barrier_init(full(i));
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    grid_dependency_wait();
    allow_dependent_launch();
    if (tid == 0) {
      s.at.ahead = atomicAdd(p.next + p.pass, 1u);
      s.at.rest = 0;
      next_item<kSplit>(p, s.at, s.upcoming);
    }
    __syncthreads();  // the barriers are there
    bool more = true;
#pragma unroll 1
    for (int stage = 0; stage < 2 && more; ++stage) {
      skip_items<kSplit>(p, s, tid);
      load_stage<StateT, kVec>(p, s.stage[stage], s.upcoming, full(stage), tid, late);
      cp_async_commit();
      more = s.upcoming.kind == kWorkChunk;
      bar_move();
      copy_gates<kVec>(p, s.stage[stage], tid);
      cp_async_commit();
      if (stage == 0 && more && tid == 0) next_work<kSplit>(p, s.at, s.upcoming);
      __syncwarp();
      hand_over(stage, more);
      bar_move();
    }
    float2 wt[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = 64 * (e >> 1) + 4 * (lane & 15) + 2 * (e & 1);
      wt[e] = make_float2(load_param(p.weight, at, p.weight_bf16), load_param(p.weight, at + 1, p.weight_bf16));
    }
    const int v0 = 32 * (warp & 3) + 16 * (warp >> 2);  // the TMEM lanes of a warp, as below
    uint32_t phase = 0;
    bool dead = false;
    for (int stage = 0;; stage ^= 1) {
      // Without this the compiler turns the loop around its first test and keeps code twice, and the chain's warps compete
      // for the instruction cache: 884 us instead of 777 (one prompt of 16,384 tokens).
      asm volatile("" ::: "memory");
      Stage& st = s.stage[stage];
      const Work d = st.work;
      if (d.kind == kWorkEnd) break;
      const bool refill = more;
      bar_sync(kBarChunkDone);
      if (refill && tid == 32 * kTakeWarp) next_work<kSplit>(p, s.at, s.upcoming);  // while P u is at work
      __syncwarp();
      if (warp == 0) {  // P u, and with it the outputs are whole
        if (!dead) Products(st).within();
        wait_done(smem_u32(&s.done[1]), phase, s, dead, p.wait_ns);
        phase ^= 1;
      }
      bar_move();
      tmem_after();
      gather_outputs(s, st, v0, lane);
      tmem_before();
      cp_async_wait();  // the gates
      bar_move();  // the tile is whole, the stage read for the last time, the upcoming work known
      if (s.stage[stage ^ 1].work.kind == kWorkChunk) bar_arrive(kBarTaken);
      if (refill) {
        skip_items<kSplit>(p, s, tid);
        load_stage<StateT, kVec>(p, st, s.upcoming, full(stage), tid, late);
        more = s.upcoming.kind == kWorkChunk;
      }
      cp_async_commit();
      store_outputs<kVec>(p, s, st, d, wt, tid);
      bar_move();  // the tile and the stage's gates are free again, and its work written
      if (refill) {
        copy_gates<kVec>(p, st, tid);
        cp_async_commit();
        hand_over(stage, more);
      }
    }
    // Copies that are still under way must not land in shared memory that is another CTA's by then.  There is one set at
    // most: each is waited for before the next is asked for, and after a wait that ran out there is no next.
    if (owed != 0) {
      bool over = false;
      wait_done(owed, owed_parity, s, over, p.wait_ns);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    const int g = lane >> 2, t = lane & 3;
    // A warp reaches the TMEM lanes of its number mod 4; two warps share them, 16 lanes each.
    const int v0 = 32 * (warp & 3) + 16 * ((warp - kStateWarp) >> 2);
    StateWarp x;
    x.phase = 0;
    x.dead = false;
    x.issuer = warp == kStateWarp;
    x.reader = warp == kStateWarp + 1;
    if (x.issuer) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)),
                   "n"(kTmemColumns)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
      if (lane == 0) {
        for (int i = 0; i < 3; ++i) barrier_init(smem_u32(&s.done[i]));
        barrier_init(smem_u32(&s.drained), kIssuers);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      }
      __syncwarp();
      tmem_before();
    }
    grid_dependency_wait();
    if (x.issuer && lane == 0) s.stop = p.pass == 0 ? 0 : static_cast<int>(p.next[2]);  // ran out in the first pass
    __syncthreads();  // the barriers are there
    tmem_after();
    const uint32_t tmem = static_cast<uint32_t>(v0) << 16;
    for (int64_t n = 0;; ++n) {
      const int stage = static_cast<int>(n & 1);
      bar_sync(kBarFull + stage);
      // A copy, for this chunk's store too: from the arrival at kBarChunkDone on, the moving threads may refill the
      // stage and write its next work, so nothing of the stage is read behind that.
      const Work work = s.stage[stage].work;
      if (work.kind == kWorkEnd) break;
      const int32_t source = work.source, slot = work.slot;
      [[maybe_unused]] int32_t save = work.save;
      const int64_t element = (v0 + g) * kDim + 2 * t;
      const auto pool_at = [&](int32_t i) {
        return static_cast<StateT*>(p.state) + i * p.slot_stride + static_cast<int64_t>(work.head) * kDim * kDim + element;
      };
      const auto matrix_at = [&](int32_t i) { return p.states + static_cast<int64_t>(i) * kDim * kDim + element; };
      const auto load = [&](const auto* at) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          load_pair(at + 8 * i, x.S[i][0], x.S[i][1]);
          load_pair(at + 8 * kDim + 8 * i, x.S[i][2], x.S[i][3]);
        }
      };
      const auto store = [&](auto* at) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          store_pair(at + 8 * i, x.S[i][0], x.S[i][1]);
          store_pair(at + 8 * kDim + 8 * i, x.S[i][2], x.S[i][3]);
        }
      };
      // Where the pool has the matrices' type they share its code: instructions are what the chain's warps compete for.
      constexpr bool kShared = kSplit && std::is_same<StateT, float>::value;
      if (source > 0 || (kShared && source == kSourceMatrix)) {
        if constexpr (kShared) {
          load(source > 0 ? pool_at(source) : matrix_at(work.matrix));
        } else {
          load(pool_at(source));
        }
      } else if (kSplit && !kShared && source == kSourceMatrix) {
        load(matrix_at(work.matrix));
      } else if (source != kSourceOn) {  // zeros, or the identity
#pragma unroll
        for (int i = 0; i < 16; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool one = kSplit && source == kSourceIdentity && v0 + g + 8 * (e >> 1) == 8 * i + 2 * t + (e & 1);
            x.S[i][e] = one ? 1.0f : 0.0f;
          }
        }
      }
      chain_chunk(x, s, stage, tmem, v0, lane, p.wait_ns, [&] {
        if (n >= 1) {
          bar_sync(kBarTaken);
          tmem_after();
        }
      });
      bar_arrive(kBarChunkDone);
      const bool to_pool = slot > 0 && s.keep != 0;  // read before the next chunk's answer: bar_state lies between
      if constexpr (kShared) {
        float* at = to_pool ? pool_at(slot) : nullptr;
#pragma unroll 1
        while (at != nullptr || save >= 0) {
          if (at == nullptr) {
            at = matrix_at(save);
            save = -1;
          }
          store(at);
          at = nullptr;
        }
      } else {
        if (to_pool) store(pool_at(slot));
        if (kSplit && save >= 0) store(matrix_at(save));
      }
    }
  }
  // Everybody has taken what it needs from TMEM.
  tmem_before();
  __syncthreads();
  if (threadIdx.x == 0 && s.stop != 0) p.next[2] = 1;
  // Products that nobody waited for may still read the stages and write TMEM.
  const bool drain = s.stop != 0;
  if (drain && (warp == 0 || warp == kStateWarp || warp == kStateWarp + 1)) umma_commit(elect_lane(), smem_u32(&s.drained));
  if (warp == kStateWarp) {
    tmem_after();
    if (drain) {
      bool over = false;
      wait_done(smem_u32(&s.drained), 0, s, over, p.wait_ns);
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem), "n"(kTmemColumns));
  }
}

// S_{k+1} = S_k M_k + B_k for a split request's value head, 8 rows of S per CTA, which takes them through all its pieces.
// A warp multiplies 16 columns of S_k by M_k's rows of their numbers, which it alone reads and which go from global
// memory to registers while the piece before is at work; the warps' partial sums meet in shared memory.
constexpr int kJoinRows = 8, kJoinThreads = 256;

__global__ void __launch_bounds__(kJoinThreads) gdn_prefill_join_kernel(const __grid_constant__ PrefillArgs p) {
  constexpr int kWarps = kJoinThreads / 32, kDepth = kDim / kWarps, kBlocks = kDim / kJoinRows;
  __shared__ __align__(16) float rows[kJoinRows][kDim];
  __shared__ __align__(16) float4 part[kWarps][kJoinRows][32];
  static_assert(kWarps == kJoinRows, "the warps add up a row each");
  grid_dependency_wait();
  allow_dependent_launch();
  const int item = blockIdx.x / kBlocks, row0 = static_cast<int>(blockIdx.x % kBlocks) * kJoinRows;
  Request rq;
  unsigned int fault;
  bool skip;
  if (!find_request(p, item / p.num_v_heads, rq, fault, skip) || !worth_splitting(p.pieces, rq.chunks)) return;
  float* states = p.states + static_cast<int64_t>(item) * p.pieces.first_parts() * kDim * kDim;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const auto matrix = [&](int i, int row) { return reinterpret_cast<float4*>(states + (i * kDim + row) * kDim) + lane; };
  reinterpret_cast<float4*>(rows[w])[lane] = *matrix(0, row0 + w);
  float4 m[kDepth], b = *matrix(2, row0 + w);
#pragma unroll
  for (int i = 0; i < kDepth; ++i) m[i] = *matrix(1, kDepth * w + i);
  __syncthreads();
  for (int k = 1; k < p.pieces.count - 1; ++k) {
    float4 sum[kJoinRows];
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r) {
      sum[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        const float x = rows[r][kDepth * w + i];
        sum[r].x = fmaf(x, m[i].x, sum[r].x);
        sum[r].y = fmaf(x, m[i].y, sum[r].y);
        sum[r].z = fmaf(x, m[i].z, sum[r].z);
        sum[r].w = fmaf(x, m[i].w, sum[r].w);
      }
    }
    float4 total = b;
    if (k + 1 < p.pieces.count - 1) {
      b = *matrix(2 * k + 2, row0 + w);
#pragma unroll
      for (int i = 0; i < kDepth; ++i) m[i] = *matrix(2 * k + 1, kDepth * w + i);
    }
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r) part[w][r][lane] = sum[r];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float4 x = part[i][w][lane];
      total.x += x.x;
      total.y += x.y;
      total.z += x.z;
      total.w += x.w;
    }
    *matrix(2 * k, row0 + w) = total;
    reinterpret_cast<float4*>(rows[w])[lane] = total;
    __syncthreads();
  }
}

bool aligned(const void* ptr, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }

int64_t chunk_places(int64_t n_tokens, int64_t n_requests) { return chunk_base(n_tokens, n_requests); }

// The workspace: key images, pair images, the chain's counters and the requests' order, then split requests' states.
int64_t order_offset(int64_t n_tokens, int64_t n_requests, int64_t num_k_heads, int64_t num_v_heads) {
  return chunk_places(n_tokens, n_requests) * (num_k_heads * static_cast<int64_t>(sizeof(KeyImage)) +
                                               num_v_heads * static_cast<int64_t>(sizeof(PairImage)));
}

constexpr int kCounters = 3;

int64_t states_offset(int64_t n_tokens, int64_t n_requests, int64_t num_k_heads, int64_t num_v_heads) {
  return (order_offset(n_tokens, n_requests, num_k_heads, num_v_heads) + 4 * (n_requests + kCounters) + 127) / 128 * 128;
}

int64_t workspace_bytes(int64_t n_tokens, int64_t n_requests, int64_t num_k_heads, int64_t num_v_heads) {
  const Pieces pieces = pieces_of(n_tokens, n_requests, num_v_heads);
  const int64_t matrices = pieces.count > 1 ? n_requests * num_v_heads * pieces.first_parts() : 0;
  return states_offset(n_tokens, n_requests, num_k_heads, num_v_heads) +
         matrices * kDim * kDim * static_cast<int64_t>(sizeof(float));
}

// Streaming multiprocessors of the current device, asked once per device.
int sm_count(int& sms) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> known[kMaxDevices];
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err == cudaSuccess && device >= 0 && device < kMaxDevices) {
    sms = known[device].load(std::memory_order_relaxed);
    if (sms > 0) return LD_OK;
  }
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "prefill: device query failed: %s", cudaGetErrorString(err));
  if (device >= 0 && device < kMaxDevices) known[device].store(sms, std::memory_order_relaxed);
  return LD_OK;
}

template <typename StateT, bool kVec>
cudaError_t launch_prefill(PrefillArgs& args, int sms, cudaStream_t stream) {
  // Set on every call: the attributes belong to the current device, and setting them is a table write.
  auto pairs = gdn_prefill_pairs_kernel<kVec>;
  cudaError_t err = cudaFuncSetAttribute(pairs, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(PairSmem));
  if (err != cudaSuccess) return err;
  const auto chain = args.pieces.count > 1 ? gdn_prefill_chain_kernel<StateT, kVec, true> : gdn_prefill_chain_kernel<StateT, kVec, false>;
  err = cudaFuncSetAttribute(chain, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ChainSmem));
  if (err != cudaSuccess) return err;
  err = launch(pairs, dim3(static_cast<unsigned int>(1 + args.places * args.num_k_heads)), dim3(kPairThreads),
               sizeof(PairSmem), stream, 1, args);
  if (err != cudaSuccess) return err;
  const int64_t heads = static_cast<int64_t>(args.n_requests) * args.num_v_heads;
  const auto run_chain = [&](int64_t items) {
    return launch(chain, dim3(static_cast<unsigned int>(std::min<int64_t>(items, sms))), dim3(kChainThreads),
                  sizeof(ChainSmem), stream, 1, args);
  };
  err = run_chain(heads * args.pieces.first_parts());
  if (err != cudaSuccess || args.pieces.count == 1) return err;
  err = launch(gdn_prefill_join_kernel, dim3(static_cast<unsigned int>(heads * (kDim / kJoinRows))), dim3(kJoinThreads),
               0, stream, 1, args);
  if (err != cudaSuccess) return err;
  args.pass = 1;
  return run_chain(heads * (args.pieces.count - 1));
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
  // Heads of a token are written while others are still read, so outputs need memory of their own.
  const auto begin_of = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
  const uintptr_t out_end = begin_of(out) + static_cast<uintptr_t>(2 * n_tokens * num_v_heads * kDim);
  const auto overlaps = [&](const void* rows, int64_t stride, int64_t width) {
    return begin_of(rows) < out_end &&
           begin_of(out) < begin_of(rows) + static_cast<uintptr_t>(2 * ((n_tokens - 1) * stride + width));
  };
  if (overlaps(qkv, qkv_row_stride, (2 * num_k_heads + num_v_heads) * kDim) ||
      overlaps(gate, gate_row_stride, num_v_heads * kDim)) {
    return set_error(LD_ERR_INVALID, "prefill: out must not overlap qkv or gate");
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
  unsigned char* order = static_cast<unsigned char*>(workspace) + order_offset(n_tokens, n_requests, num_k_heads, num_v_heads);
  args.next = reinterpret_cast<uint32_t*>(order);
  args.order = reinterpret_cast<int32_t*>(order) + kCounters;
  args.pieces = pieces_of(n_tokens, n_requests, num_v_heads);
  args.pass = 0;
  args.states = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) +
                                         states_offset(n_tokens, n_requests, num_k_heads, num_v_heads));
  args.places = chunk_places(n_tokens, n_requests);
  args.n_requests = static_cast<int>(n_requests);
  args.num_k_heads = static_cast<int>(num_k_heads);
  args.num_v_heads = static_cast<int>(num_v_heads);
  args.heads_ratio = static_cast<int>(num_v_heads / num_k_heads);
  args.dt_bias_bf16 = dt_bias_dtype == LD_DTYPE_BF16;
  args.weight_bf16 = weight_dtype == LD_DTYPE_BF16;
  args.q_scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(kDim)));
  args.eps = eps;
  args.wait_ns = wait_limit_ns();
  args.extra_tx = wait_test_extra_bytes();
  // 16-byte copies of the q, k, v and gate rows and 8-byte stores to out where every row allows them.
  const bool vec = aligned(qkv, 16) && qkv_row_stride % 8 == 0 && aligned(gate, 16) && gate_row_stride % 8 == 0 &&
                   aligned(out, 8);
  int sms = 0;
  const int rc = sm_count(sms);
  if (rc != LD_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  if (bf16_pool) {
    err = vec ? launch_prefill<__nv_bfloat16, true>(args, sms, s) : launch_prefill<__nv_bfloat16, false>(args, sms, s);
  } else {
    err = vec ? launch_prefill<float, true>(args, sms, s) : launch_prefill<float, false>(args, sms, s);
  }
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "prefill launch failed: %s", cudaGetErrorString(err));
  return ok();
}
