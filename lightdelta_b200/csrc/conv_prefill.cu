// Causal depthwise conv1d and silu over whole prompts: the step between the projection and ld_prefill.
//
//   y_t = silu(bias + sum_{j<w} W[:, j] x_{t-w+1+j}),  x before the request's first token taken from the
//   convolution window in its source slot (zeros without context); wherever a block or the request ends,
//   the last w - 1 inputs become the window in the block's slot, positions 0 .. w - 2, which is where
//   ld_conv_update with accepted = 1 (and the next piece of the prompt) finds them.
//
// Products and sums are fp32, rounded once at the end.  (ld_conv_update rounds each product to bf16, as
// the host engine's kernel that it replaces does.)
//
// One pass bound by HBM: 2 bytes read and 2 written per (token, channel).  A thread owns 4 channels of a
// tile of consecutive tokens, whatever requests they belong to, and slides the window along, so a tile
// reads w - 1 rows beyond its own.  Rows come in batches of 8, a batch's loads while the one before is at
// work, and a whole batch is straight code.  24 prompts of 16,000 tokens in all with 8,192 channels take
// 97.8 us, 5.4 TB/s, at six CTAs on an SM (80 registers a thread); five (96 registers) take 101.4, four
// 103.3, batches of 4 rows at eight CTAs 101.  Without loads ahead six CTAs took 108.5 and five 124; 8
// channels a thread took 222 registers and 299 us.  What is left is instructions, silu's two
// special-function operations per value above all, and the tile's start.
// A request's first w - 1 tokens all go to the thread that has its first one: only that thread reads the
// history, so it can also write the slot when a request goes on inside a block and its source slot is
// its first destination.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "internal.h"
#include "launch.cuh"
#include "lightdelta_b200.h"
#include "math.cuh"

namespace ldb {
namespace {

constexpr int kThreads = 128;
constexpr int kBatch = 8;   // rows loaded together
constexpr int kVector = 4;  // channels per thread where rows allow 8-byte accesses

__device__ unsigned int g_conv_prefill_faults;

struct ConvPrefillArgs {
  const __nv_bfloat16* x;
  int64_t x_row;
  int64_t n_tokens;
  int64_t dim;
  __nv_bfloat16* state;  // element (slot, channel, position) at slot*s_slot + channel*s_dim + position*s_pos
  int64_t n_slots, s_slot, s_dim, s_pos;
  const __nv_bfloat16* weight;
  const __nv_bfloat16* bias;
  const int32_t* table;
  int64_t table_row, table_width;
  uint32_t block_size;  // larger ones as the largest of these: every position is below it
  const int32_t* context;
  const int32_t* cu;
  int n_requests;
  int tile;  // tokens per thread
  __nv_bfloat16* out;
};

// kVec consecutive channels of one token: bf16 pairs in memory order (one channel alone: the low half).
template <int kVec>
struct Row {
  static constexpr int kWords = (kVec + 1) / 2;
  uint32_t w[kWords];
};

template <int kVec>
__device__ __forceinline__ Row<kVec> load_row(const __nv_bfloat16* at) {
  Row<kVec> r;
  if constexpr (kVec == 4) {
    const uint2 raw = *reinterpret_cast<const uint2*>(at);
    r.w[0] = raw.x;
    r.w[1] = raw.y;
  } else {
    r.w[0] = __bfloat16_as_ushort(*at);
  }
  return r;
}

template <int kVec>
__device__ __forceinline__ void store_row(__nv_bfloat16* at, const Row<kVec>& r) {
  if constexpr (kVec == 4) {
    *reinterpret_cast<uint2*>(at) = make_uint2(r.w[0], r.w[1]);
  } else {
    *at = __ushort_as_bfloat16(static_cast<unsigned short>(r.w[0]));
  }
}

template <int kVec>
__device__ __forceinline__ Row<kVec> zero_row() {
  Row<kVec> r;
#pragma unroll
  for (int i = 0; i < Row<kVec>::kWords; ++i) r.w[i] = 0;
  return r;
}

// One position of a slot's window for this thread's channels.
template <int kVec>
__device__ __forceinline__ Row<kVec> load_window(const ConvPrefillArgs& p, int32_t slot, int64_t channel, int position) {
  const __nv_bfloat16* at = p.state + slot * p.s_slot + channel * p.s_dim + position * p.s_pos;
  Row<kVec> r = zero_row<kVec>();
#pragma unroll
  for (int c = 0; c < kVec; ++c) {
    r.w[c / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(at[c * p.s_dim])) << (16 * (c & 1));
  }
  return r;
}

template <int kVec>
__device__ __forceinline__ void store_window(const ConvPrefillArgs& p, int32_t slot, int64_t channel, int position,
                                             const Row<kVec>& r) {
  __nv_bfloat16* at = p.state + slot * p.s_slot + channel * p.s_dim + position * p.s_pos;
#pragma unroll
  for (int c = 0; c < kVec; ++c) {
    at[c * p.s_dim] = __ushort_as_bfloat16(static_cast<unsigned short>(r.w[c / 2] >> (16 * (c & 1))));
  }
}

// The request that a thread is in.
struct Place {
  int64_t begin, end;   // its tokens
  uint32_t context;     // a position, context + token, is below 2^32 - 1
  int64_t next_end;     // the next token after which a block or the request ends
  const int32_t* row;
  int32_t source;       // slot of the history (0: none)
  int32_t kept;         // block that the request's first thread writes because it is also read (-1: none)
  bool ok;              // false: zero outputs, nothing else
};

__device__ __forceinline__ void enter(const ConvPrefillArgs& p, int r, int64_t token, bool report, Place& at) {
  at.begin = p.cu[r];
  at.end = p.cu[r + 1];
  const int32_t context = p.context[r];
  at.context = static_cast<uint32_t>(context);
  at.row = p.table + r * p.table_row;
  at.source = 0;
  at.kept = -1;
  at.next_end = at.end;
  unsigned int fault = 0;
  at.ok = context >= 0 && (at.context + static_cast<uint32_t>(at.end - at.begin) - 1) / p.block_size < p.table_width;
  if (!at.ok) {
    fault = LD_FAULT_TABLE_BLOCKS;
  } else {
    uint32_t block = 0;
    if (context > 0) {
      block = (at.context - 1) / p.block_size;
      at.source = at.row[block];
      if (at.source >= p.n_slots) fault = LD_FAULT_CONV_SLOT_RANGE;
      at.ok = at.source > 0 && at.source < p.n_slots;
      if (at.context - block * p.block_size < p.block_size) at.kept = static_cast<int32_t>(block);
    }
    if (token != at.begin) block = (at.context + static_cast<uint32_t>(token - at.begin)) / p.block_size;
    if (token == at.begin && context > 0 && at.kept < 0) ++block;  // the context fills its block
    at.next_end = min(at.end, at.begin + (static_cast<int64_t>(block) + 1) * p.block_size - at.context);
  }
  if (fault != 0 && report) atomicOr(&g_conv_prefill_faults, fault);
}

// The input `back` >= 1 tokens before token t of the request: an earlier row, or its history.
template <int kVec, int kWidth>
__device__ __forceinline__ Row<kVec> earlier(const ConvPrefillArgs& p, const Place& at, int64_t t, int back,
                                             int64_t channel) {
  const int64_t i = t - back;
  if (i >= at.begin) return load_row<kVec>(p.x + i * p.x_row + channel);
  if (at.source == 0) return zero_row<kVec>();
  return load_window<kVec>(p, at.source, channel, static_cast<int>(kWidth - 1 + (i - at.begin)));
}

// Outputs of one token from it and the inputs before it.
template <int kVec, int kWidth>
__device__ __forceinline__ Row<kVec> convolve(const Row<kVec>* rows, const float2 (&wt)[kWidth][Row<kVec>::kWords],
                                              const float2 (&bias)[Row<kVec>::kWords]) {
  Row<kVec> y;
#pragma unroll
  for (int c = 0; c < Row<kVec>::kWords; ++c) {
    float2 acc = bias[c];
#pragma unroll
    for (int j = 0; j < kWidth; ++j) {
      acc = fma2(make_float2(bf16_low(rows[j].w[c]), bf16_high(rows[j].w[c])), wt[j][c], acc);
    }
    const float2 z = silu_fast(acc);
    y.w[c] = pack_bf16(z.x, z.y);
  }
  return y;
}

// Outputs of `count` tokens and the window behind them.  Whole batches are straight code in which every input is
// unpacked once, and a batch's rows are loaded while the one before is at work.
template <int kVec, int kWidth>
__device__ __forceinline__ void convolve_run(const __nv_bfloat16* x, int64_t x_row, __nv_bfloat16* out, int64_t out_row,
                                             int count, const float2 (&wt)[kWidth][Row<kVec>::kWords],
                                             const float2 (&bias)[Row<kVec>::kWords], Row<kVec> (&window)[kWidth - 1]) {
  Row<kVec> rows[kWidth - 1 + kBatch], next[kBatch];
#pragma unroll
  for (int j = 0; j < kWidth - 1; ++j) rows[j] = window[j];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    if (i < count) next[i] = load_row<kVec>(x + i * x_row);
  }
  x += kBatch * x_row;
#pragma unroll 1
  for (; count >= kBatch; count -= kBatch) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) rows[kWidth - 1 + i] = next[i];
    if (count >= 2 * kBatch) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) next[i] = load_row<kVec>(x + i * x_row);
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (kBatch + i < count) next[i] = load_row<kVec>(x + i * x_row);
      }
    }
    x += kBatch * x_row;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      store_row<kVec>(out, convolve<kVec, kWidth>(rows + i, wt, bias));
      out += out_row;
    }
#pragma unroll
    for (int j = 0; j < kWidth - 1; ++j) rows[j] = rows[kBatch + j];
  }
#pragma unroll
  for (int i = 0; i < kBatch - 1; ++i) {
    if (i < count) {
      rows[kWidth - 1] = next[i];
      store_row<kVec>(out, convolve<kVec, kWidth>(rows, wt, bias));
      out += out_row;
#pragma unroll
      for (int j = 0; j < kWidth - 1; ++j) rows[j] = rows[j + 1];
    }
  }
#pragma unroll
  for (int j = 0; j < kWidth - 1; ++j) window[j] = rows[j];
}

template <int kVec, int kWidth>
__global__ void __launch_bounds__(kThreads, 6) conv_prefill_kernel(const ConvPrefillArgs p) {
  grid_dependency_wait();
  allow_dependent_launch();
  const int64_t channel = (static_cast<int64_t>(blockIdx.y) * kThreads + threadIdx.x) * kVec;
  int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tile;
  const int64_t t1 = min(t0 + p.tile, p.n_tokens);

  // The request of the first token: the last r with cu[r] <= t0, by 32-way bisection (the warp's lanes
  // probe together).  Offsets that are out of order or range are caught by the checks below.
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.n_requests;  // cu[lo] <= t0 (or lo is 0), cu[hi] > t0 (or hi is the end)
  while (hi - lo > 1) {
    const int width = (hi - lo + 31) / 32;
    const int probe = lo + (lane + 1) * width;
    const bool below = probe < hi && p.cu[probe] <= t0;
    const unsigned int votes = __ballot_sync(0xffffffffu, below);
    const int passed = __popc(votes);  // probes are in order, so the votes are a prefix
    const int next = lo + passed * width;
    hi = min(hi, next + width);
    lo = next;
  }
  int r = lo;
  if (channel >= p.dim) return;
  // The tile before takes what is left of a request's first w - 1 tokens (a first token at t0 - 1 or so).
  const int64_t begun = p.cu[r];
  if (begun >= 0 && begun < t0 && t0 < begun + kWidth - 1) {
    t0 = max(t0, min(static_cast<int64_t>(p.cu[r + 1]), begun + kWidth - 1));
  }
  int64_t limit = t1;
  const bool report = channel == 0;

  constexpr int kWords = Row<kVec>::kWords;
  float2 wt[kWidth][kWords], bias[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const int64_t c0 = channel + 2 * i, c1 = kVec > 1 ? c0 + 1 : c0;
#pragma unroll
    for (int j = 0; j < kWidth; ++j) {
      wt[j][i] = make_float2(__bfloat162float(p.weight[c0 * kWidth + j]), __bfloat162float(p.weight[c1 * kWidth + j]));
    }
    bias[i] = p.bias != nullptr ? make_float2(__bfloat162float(p.bias[c0]), __bfloat162float(p.bias[c1]))
                                : make_float2(0.0f, 0.0f);
  }

  Place at;
  at.end = -1;  // no request yet
  Row<kVec> window[kWidth - 1];  // inputs t - w + 1 .. t - 1
#pragma unroll
  for (int j = 0; j < kWidth - 1; ++j) window[j] = zero_row<kVec>();
  for (int64_t t = t0; t < limit;) {
    if (t >= at.end) {  // first token of the tile, or of another request
      while (r < p.n_requests && p.cu[r + 1] <= t) ++r;
      if (r >= p.n_requests) return;  // rows behind the last request stay as they are
      const int64_t begin = p.cu[r], end = p.cu[r + 1];
      if (begin > t || begin < 0 || end > p.n_tokens) {
        if (report && begin <= t) atomicOr(&g_conv_prefill_faults, LD_FAULT_DECODE_TOKENS);
        t = max(t + 1, begin > t ? begin : end);  // rows of no request
        continue;
      }
      enter(p, r, t, report, at);
      if (t == at.begin) limit = max(limit, min(at.end, t + kWidth - 1));
      if (at.ok) {
#pragma unroll
        for (int j = 0; j < kWidth - 1; ++j) window[j] = earlier<kVec, kWidth>(p, at, t, kWidth - 1 - j, channel);
        if (t == at.begin && at.kept >= 0) {
          // This thread has read the source slot, which is the request's first destination too: it
          // writes it now, whichever tile its block's last token lies in.
          const int64_t stop = min(at.end, at.begin + static_cast<int64_t>(at.kept + 1) * p.block_size - at.context);
          Row<kVec> last[kWidth - 1];
#pragma unroll
          for (int j = 0; j < kWidth - 1; ++j) last[j] = earlier<kVec, kWidth>(p, at, stop, kWidth - 1 - j, channel);
#pragma unroll
          for (int j = 0; j < kWidth - 1; ++j) store_window<kVec>(p, at.source, channel, j, last[j]);
        }
      }
    }
    // The tokens to the end of their block, request or tile.
    const int64_t stop = min(limit, at.ok ? at.next_end : at.end);
    const int count = static_cast<int>(stop - t);
    const __nv_bfloat16* x = p.x + t * p.x_row + channel;
    __nv_bfloat16* out = p.out + t * p.dim + channel;
    if (!at.ok) {
      for (int i = 0; i < count; ++i) store_row<kVec>(out + i * p.dim, zero_row<kVec>());
      t += count;
      continue;
    }
    convolve_run<kVec, kWidth>(x, p.x_row, out, p.dim, count, wt, bias, window);
    t += count;
    if (t == at.next_end) {
      const int64_t block = (at.context + static_cast<uint32_t>(t - 1 - at.begin)) / p.block_size;
      if (block != at.kept) {
        const int32_t slot = at.row[block];
        if (slot > 0 && slot < p.n_slots) {
#pragma unroll
          for (int j = 0; j < kWidth - 1; ++j) store_window<kVec>(p, slot, channel, j, window[j]);
        } else if (slot >= p.n_slots && report) {
          atomicOr(&g_conv_prefill_faults, LD_FAULT_CONV_SLOT_RANGE);
        }
      }
      at.next_end = min(at.end, at.next_end + p.block_size);
    }
  }
}

bool aligned(const void* ptr, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }

template <int kWidth>
cudaError_t launch_width(ConvPrefillArgs& args, bool vec, cudaStream_t stream) {
  const int channels = (vec ? kVector : 1) * kThreads;
  const int64_t groups = (args.dim + channels - 1) / channels;
  // A tile's thread reads 3 rows that the tile before reads too, and finds its request and its weights: 24 prompts of
  // 16,000 tokens in all (8,192 channels) take 98.3 us at 64 tokens per thread, 104.0 at 32.  Smaller batches are
  // spread over the SMs (six CTAs each) before their tiles grow.
  const int64_t work = args.n_tokens * groups;
  args.tile = work >= 64 * 6 * 148 ? 64 : work >= 32 * 4 * 148 ? 32 : 8;
  const dim3 grid(static_cast<unsigned int>((args.n_tokens + args.tile - 1) / args.tile),
                  static_cast<unsigned int>(groups));
  if (vec) return launch(conv_prefill_kernel<kVector, kWidth>, grid, dim3(kThreads), 0, stream, 1, args);
  return launch(conv_prefill_kernel<1, kWidth>, grid, dim3(kThreads), 0, stream, 1, args);
}

}  // namespace

int conv_prefill_faults(uint32_t* flags, int clear) {
  uint32_t value = 0;
  cudaError_t err = cudaMemcpyFromSymbol(&value, g_conv_prefill_faults, sizeof(value));
  if (err == cudaSuccess && clear) {
    const uint32_t zero = 0;
    err = cudaMemcpyToSymbol(g_conv_prefill_faults, &zero, sizeof(zero));
  }
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "ld_fault_flags: %s", cudaGetErrorString(err));
  *flags = value;
  return LD_OK;
}

}  // namespace ldb

extern "C" int ld_conv_prefill(const void* x, int64_t x_row_stride, int64_t n_tokens, int64_t dim, void* conv_state,
                               int64_t n_conv_slots, int64_t conv_slot_stride, int64_t conv_dim_stride,
                               int64_t conv_pos_stride, int64_t conv_state_len, const void* conv_weight,
                               const void* conv_bias, int64_t conv_width, const int32_t* table,
                               int64_t table_row_stride, int64_t table_width, int64_t block_size,
                               const int32_t* context, const int32_t* cu, int64_t n_requests, void* out,
                               void* stream) {
  using namespace ldb;
  if (conv_width < 2 || conv_width > 4) {
    return set_error(LD_ERR_INVALID, "conv_prefill: kernel width must be 2 through 4");
  }
  if (conv_state_len < conv_width - 1) {
    return set_error(LD_ERR_INVALID, "conv_prefill: the conv state holds fewer than width - 1 positions");
  }
  if (block_size < 1) return set_error(LD_ERR_INVALID, "conv_prefill: block_size must be positive");
  if (n_requests < 0 || n_requests > INT32_MAX / 2 || n_tokens < 0 || n_tokens > INT32_MAX || dim < 1 ||
      dim > INT32_MAX / 2) {
    return set_error(LD_ERR_INVALID, "conv_prefill: request, token or channel count out of range");
  }
  if (table_width < 1 || table_row_stride < table_width) {
    return set_error(LD_ERR_INVALID,
                     "conv_prefill: the table needs at least one block per row and rows that do not overlap");
  }
  if (x_row_stride < dim || n_conv_slots < 1 || conv_slot_stride < 0 || conv_dim_stride < 1 || conv_pos_stride < 1) {
    return set_error(LD_ERR_INVALID, "conv_prefill: invalid strides or slot count");
  }
  const bool dims_disjoint =
      conv_dim_stride >= conv_state_len * conv_pos_stride || conv_pos_stride >= dim * conv_dim_stride;
  const int64_t slot_extent = (dim - 1) * conv_dim_stride + (conv_state_len - 1) * conv_pos_stride + 1;
  if (!dims_disjoint || (n_conv_slots > 1 && conv_slot_stride < slot_extent)) {
    return set_error(LD_ERR_INVALID, "conv_prefill: the conv state's strides make slots, channels or positions overlap");
  }
  if (n_requests == 0 || n_tokens == 0) return ok();
  if (x == nullptr || conv_state == nullptr || conv_weight == nullptr || table == nullptr || context == nullptr ||
      cu == nullptr || out == nullptr) {
    return set_error(LD_ERR_INVALID, "conv_prefill: a required pointer is NULL");
  }
  if (!aligned(x, 2) || !aligned(conv_state, 2) || !aligned(conv_weight, 2) || !aligned(conv_bias, 2) ||
      !aligned(out, 2)) {
    return set_error(LD_ERR_INVALID, "conv_prefill: bf16 tensors must be 2-byte aligned");
  }
  // Neighbouring tiles read the same inputs, so the outputs cannot take their place.
  const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), o0 = reinterpret_cast<uintptr_t>(out);
  const uintptr_t x1 = x0 + 2 * static_cast<uintptr_t>((n_tokens - 1) * x_row_stride + dim);
  const uintptr_t o1 = o0 + 2 * static_cast<uintptr_t>(n_tokens * dim);
  if (x0 < o1 && o0 < x1) return set_error(LD_ERR_INVALID, "conv_prefill: out must not overlap x");
  ConvPrefillArgs args;
  args.x = static_cast<const __nv_bfloat16*>(x);
  args.x_row = x_row_stride;
  args.n_tokens = n_tokens;
  args.dim = dim;
  args.state = static_cast<__nv_bfloat16*>(conv_state);
  args.n_slots = n_conv_slots;
  args.s_slot = conv_slot_stride;
  args.s_dim = conv_dim_stride;
  args.s_pos = conv_pos_stride;
  args.weight = static_cast<const __nv_bfloat16*>(conv_weight);
  args.bias = static_cast<const __nv_bfloat16*>(conv_bias);
  args.table = table;
  args.table_row = table_row_stride;
  args.table_width = table_width;
  args.block_size = static_cast<uint32_t>(std::min<int64_t>(block_size, UINT32_MAX));
  args.context = context;
  args.cu = cu;
  args.n_requests = static_cast<int>(n_requests);
  args.tile = 0;
  args.out = static_cast<__nv_bfloat16*>(out);
  const bool vec = dim % kVector == 0 && aligned(x, 8) && x_row_stride % kVector == 0 && aligned(out, 8);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  switch (conv_width) {
    case 2: err = launch_width<2>(args, vec, s); break;
    case 3: err = launch_width<3>(args, vec, s); break;
    default: err = launch_width<4>(args, vec, s); break;
  }
  if (err != cudaSuccess) return set_error(LD_ERR_CUDA, "conv prefill launch failed: %s", cudaGetErrorString(err));
  return ok();
}
