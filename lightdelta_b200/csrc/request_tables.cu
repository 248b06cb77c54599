// Block tables, token offsets, positions and slot maps of a batch from its request lengths, in one
// launch and without the host: what the prompt path and a paged cache read before they touch a token.
//
// Per request r with q_r new tokens behind c_r held ones and blocks of `bs` positions:
//   cu = prefix sums of q;  have_r = ceil(c_r / bs), want_r = ceil((c_r + q_r) / bs), need_r = want_r - have_r;
//   table[r, have_r + i] = free[sum_{s<r} need_s + i] for i < need_r;
//   token t of r: position c_r + t - cu_r, slot = table[r, position / bs] * bs + position % bs.
//
// The work is a scan of the requests and about 16 bytes written per token, a few microseconds of
// latency at most sizes, so there is one launch and no scratch: every CTA scans all lengths for itself
// (32 KB from L2 at 4096 requests), keeps one running sum per thread's stretch of requests in shared
// memory, and then takes its share of tokens, new blocks and requests, each found by bisection of the
// stretches and a short walk.  A token's block comes from the free list directly where it is new, so no
// CTA reads what another one writes.
//
// Back to back, 8 one-token requests or 256 prompts of 64,000 tokens take 6.1 us, which is the host's
// launch; 4,096 requests of 400,000 tokens take 11.6 us (0.66 TB/s), the chain of scan, search and
// dependent loads.  One CTA per SM: with twice as many, which do not fit beside one another, 13.1; four
// consecutive tokens a thread with one search for all of them, 12.4.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "internal.h"
#include "launch.cuh"
#include "lightdelta_b200.h"

namespace ldb {
namespace {

constexpr int kThreads = 1024;

__device__ unsigned int g_tables_faults;

struct TablesArgs {
  const int32_t* query;
  const int32_t* context;
  const int32_t* free_blocks;
  int64_t n_free;
  int32_t* table;
  int64_t table_row;
  int64_t table_width;
  int32_t* cu;
  int64_t* positions;
  int64_t* slot_map;
  int64_t n_tokens;
  int32_t* state_slots;
  int32_t* used;
  int n_requests;
  int stretch;  // requests per thread of the scan
  uint32_t block_size;
  int shift;    // log2(block_size) when it is a power of two, else -1
};

// Lengths of one request: new and held tokens (negative ones count as 0), held and wanted blocks.
struct Lengths {
  uint32_t query, context, have, want;
};

// Whole blocks in front of a position (a uniform choice: the division is about twenty instructions).
__device__ __forceinline__ uint32_t block_index(const TablesArgs& p, uint32_t position) {
  return p.shift >= 0 ? position >> p.shift : position / p.block_size;
}

__device__ __forceinline__ uint32_t blocks_of(const TablesArgs& p, uint32_t tokens) {
  const uint32_t whole = block_index(p, tokens);
  return whole + (whole * p.block_size != tokens);
}

__device__ __forceinline__ Lengths lengths_of(const TablesArgs& p, int r) {
  Lengths l;
  l.query = static_cast<uint32_t>(max(p.query[r], 0));
  l.context = static_cast<uint32_t>(max(p.context[r], 0));
  l.have = blocks_of(p, l.context);
  l.want = blocks_of(p, l.context + l.query);  // two int32: no wrap
  return l;
}

// Block `b` of request r, whose new blocks start at free_blocks[first]: the kept entry of its row or the
// free list's, 0 where neither exists.
__device__ __forceinline__ int32_t block_of(const TablesArgs& p, int r, uint32_t b, const Lengths& l, int64_t first) {
  if (b >= p.table_width) return 0;
  if (b < l.have) return p.table[r * p.table_row + b];
  const int64_t at = first + (b - l.have);
  return at < p.n_free ? p.free_blocks[at] : 0;
}

struct Smem {
  int64_t tokens[kThreads + 1];  // tokens in front of each stretch
  int64_t blocks[kThreads + 1];  // new blocks in front of each stretch
  int64_t warp_tokens[kThreads / 32], warp_blocks[kThreads / 32];
};

// The last stretch whose sum is at most x: the one that holds item x.
__device__ __forceinline__ int find_stretch(const int64_t* sums, int64_t x) {
  int lo = 0, hi = kThreads;  // sums[lo] <= x < sums[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) request_tables_kernel(const TablesArgs p) {
  __shared__ Smem s;
  grid_dependency_wait();
  allow_dependent_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = static_cast<int>(min(static_cast<int64_t>(tid) * p.stretch, static_cast<int64_t>(p.n_requests)));
  const int r1 = min(r0 + p.stretch, p.n_requests);

  // This thread's stretch, then the sums in front of it.
  unsigned int fault = 0;
  int64_t tokens = 0, blocks = 0;
#pragma unroll 4
  for (int r = r0; r < r1; ++r) {
    const Lengths l = lengths_of(p, r);
    tokens += l.query;
    blocks += l.want - l.have;
    if (p.query[r] < 0 || p.context[r] < 0) fault |= LD_FAULT_TABLE_LENGTHS;
    if (l.want > p.table_width) fault |= LD_FAULT_TABLE_BLOCKS;
  }
  int64_t tokens_to = tokens, blocks_to = blocks;  // inclusive
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, tokens_to, off), b = __shfl_up_sync(0xffffffffu, blocks_to, off);
    if (lane >= off) {
      tokens_to += a;
      blocks_to += b;
    }
  }
  if (lane == 31) {
    s.warp_tokens[warp] = tokens_to;
    s.warp_blocks[warp] = blocks_to;
  }
  __syncthreads();
  // Every warp adds up the ones in front of it, a warp's sums per lane.
  static_assert(kThreads / 32 == 32, "one warp per lane");
  int64_t tokens_in = lane < warp ? s.warp_tokens[lane] : 0, blocks_in = lane < warp ? s.warp_blocks[lane] : 0;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    tokens_in += __shfl_xor_sync(0xffffffffu, tokens_in, off);
    blocks_in += __shfl_xor_sync(0xffffffffu, blocks_in, off);
  }
  tokens_to += tokens_in;
  blocks_to += blocks_in;
  s.tokens[tid] = tokens_to - tokens;
  s.blocks[tid] = blocks_to - blocks;
  if (tid == kThreads - 1) {
    s.tokens[kThreads] = tokens_to;
    s.blocks[kThreads] = blocks_to;
  }
  __syncthreads();
  const int64_t all_tokens = s.tokens[kThreads], all_blocks = s.blocks[kThreads];

  if (blockIdx.x == 0) {
    if (tid == 0) {
      p.cu[p.n_requests] = static_cast<int32_t>(min(all_tokens, static_cast<int64_t>(INT32_MAX)));
      p.used[0] = static_cast<int32_t>(min(all_blocks, static_cast<int64_t>(INT32_MAX)));
      if (all_tokens > p.n_tokens) fault |= LD_FAULT_TABLE_LENGTHS;
      if (all_blocks > p.n_free) fault |= LD_FAULT_TABLE_BLOCKS;
    }
    if (fault != 0) atomicOr(&g_tables_faults, fault);
  }

  const int64_t start = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = start; i < p.n_requests; i += step) {  // offsets and state slots
    const int r = static_cast<int>(i), f = r / p.stretch;
    int64_t at = s.tokens[f], first = s.blocks[f];
    for (int k = f * p.stretch; k < r; ++k) {
      const Lengths l = lengths_of(p, k);
      at += l.query;
      first += l.want - l.have;
    }
    const Lengths l = lengths_of(p, r);
    p.cu[r] = static_cast<int32_t>(min(at, static_cast<int64_t>(INT32_MAX)));
    p.state_slots[2 * r] = l.query > 0 ? block_of(p, r, l.want - 1, l, first) : 0;
    p.state_slots[2 * r + 1] = l.context > 0 ? block_of(p, r, l.have - 1, l, first) : 0;
  }
  // New blocks past the end of their row are left out.  Lengths that ask for more blocks than the table has entries, up to
  // 2^31 a request, must not keep the GPU busy counting them: there the entries are gone through instead.
  const int64_t width = min(p.table_width, static_cast<int64_t>(1) << 32);  // a request has fewer blocks than 2^32
  const int64_t entries = p.n_requests * width;
  if (all_blocks <= entries) {
    for (int64_t i = start; i < all_blocks; i += step) {
      const int f = find_stretch(s.blocks, i);
      int r = f * p.stretch;
      int64_t first = s.blocks[f];
      Lengths l = lengths_of(p, r);
      while (first + (l.want - l.have) <= i) {
        first += l.want - l.have;
        l = lengths_of(p, ++r);
      }
      const int64_t b = l.have + (i - first);
      if (b < p.table_width) p.table[r * p.table_row + b] = i < p.n_free ? p.free_blocks[i] : 0;
    }
  } else {
    for (int64_t i = start; i < entries; i += step) {
      const int r = static_cast<int>(i / width), f = r / p.stretch;
      const uint32_t b = static_cast<uint32_t>(i - r * width);
      int64_t first = s.blocks[f];
      for (int k = f * p.stretch; k < r; ++k) {
        const Lengths l = lengths_of(p, k);
        first += l.want - l.have;
      }
      const Lengths l = lengths_of(p, r);
      if (b >= l.have && b < l.want) p.table[r * p.table_row + b] = block_of(p, r, b, l, first);
    }
  }
  for (int64_t i = start; i < p.n_tokens; i += step) {
    int64_t position = -1, slot = -1;
    if (i < all_tokens) {
      const int f = find_stretch(s.tokens, i);
      int r = f * p.stretch;
      int64_t at = s.tokens[f], first = s.blocks[f];
      Lengths l = lengths_of(p, r);
      while (at + l.query <= i) {
        at += l.query;
        first += l.want - l.have;
        l = lengths_of(p, ++r);
      }
      const uint32_t pos = l.context + static_cast<uint32_t>(i - at);
      const uint32_t index = block_index(p, pos);
      const int32_t block = block_of(p, r, index, l, first);
      position = pos;
      if (block > 0) slot = static_cast<int64_t>(block) * p.block_size + (pos - index * p.block_size);
    }
    p.positions[i] = position;
    p.slot_map[i] = slot;
  }
}

bool aligned(const void* ptr, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }

}  // namespace

int tables_faults(uint32_t* flags, int clear) {
  uint32_t value = 0;
  cudaError_t err = cudaMemcpyFromSymbol(&value, g_tables_faults, sizeof(value));
  if (err == cudaSuccess && clear) {
    const uint32_t zero = 0;
    err = cudaMemcpyToSymbol(g_tables_faults, &zero, sizeof(zero));
  }
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "ld_fault_flags: %s", cudaGetErrorString(err));
  *flags = value;
  return LD_OK;
}

}  // namespace ldb

extern "C" int ld_request_tables(const int32_t* query_lens, const int32_t* context, int64_t n_requests,
                                 const int32_t* free_blocks, int64_t n_free, int32_t* table, int64_t table_row_stride,
                                 int64_t table_width, int64_t block_size, int32_t* cu, int64_t* positions,
                                 int64_t* slot_map, int64_t n_tokens, int32_t* state_slots, int32_t* used,
                                 void* stream) {
  using namespace ldb;
  if (n_requests < 0 || n_requests > INT32_MAX / 2 || n_tokens < 0 || n_tokens > INT32_MAX || n_free < 0) {
    return set_error(LD_ERR_INVALID, "request_tables: request, token or free block count out of range");
  }
  if (block_size < 1 || block_size > (1 << 30)) {
    return set_error(LD_ERR_INVALID, "request_tables: block_size must be 1 through 2^30");
  }
  if (table_width < 1 || table_row_stride < table_width) {
    return set_error(LD_ERR_INVALID,
                     "request_tables: the table needs at least one block per row and rows that do not overlap");
  }
  if (cu == nullptr || used == nullptr ||
      (n_requests > 0 && (query_lens == nullptr || context == nullptr || table == nullptr || state_slots == nullptr)) ||
      (n_free > 0 && free_blocks == nullptr) || (n_tokens > 0 && (positions == nullptr || slot_map == nullptr))) {
    return set_error(LD_ERR_INVALID, "request_tables: a required pointer is NULL");
  }
  for (const void* ptr : {static_cast<const void*>(query_lens), static_cast<const void*>(context),
                          static_cast<const void*>(free_blocks), static_cast<const void*>(table),
                          static_cast<const void*>(cu), static_cast<const void*>(state_slots),
                          static_cast<const void*>(used)}) {
    if (!aligned(ptr, 4)) return set_error(LD_ERR_INVALID, "request_tables: int32 arrays must be 4-byte aligned");
  }
  if (!aligned(positions, 8) || !aligned(slot_map, 8)) {
    return set_error(LD_ERR_INVALID, "request_tables: int64 arrays must be 8-byte aligned");
  }
  TablesArgs args;
  args.query = query_lens;
  args.context = context;
  args.free_blocks = free_blocks;
  args.n_free = n_free;
  args.table = table;
  args.table_row = table_row_stride;
  args.table_width = table_width;
  args.cu = cu;
  args.positions = positions;
  args.slot_map = slot_map;
  args.n_tokens = n_tokens;
  args.state_slots = state_slots;
  args.used = used;
  args.n_requests = static_cast<int>(n_requests);
  args.stretch = static_cast<int>(std::max<int64_t>((n_requests + kThreads - 1) / kThreads, 1));
  args.block_size = static_cast<uint32_t>(block_size);
  args.shift = -1;
  for (int bit = 0; bit <= 30; ++bit) {
    if (block_size == 1LL << bit) args.shift = bit;
  }
  // One item per thread, at most one CTA per SM.
  const int64_t items = std::max<int64_t>(std::max(n_tokens, n_requests), 1);
  const int64_t ctas = std::min<int64_t>((items + kThreads - 1) / kThreads, 148);
  const cudaError_t err = launch(request_tables_kernel, dim3(static_cast<unsigned int>(ctas)), dim3(kThreads), 0,
                                 static_cast<cudaStream_t>(stream), 1, args);
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "request tables launch failed: %s", cudaGetErrorString(err));
  return ok();
}
