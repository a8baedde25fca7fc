// Token embedding with scaling, and its gradient by sorted tokens.
//
//   y[t]  = scale * W[id[t]]                                   (0 in masked rows)
//   dW[v] = scale * sum over valid t with id[t] = v of dy[t]   (the padding row 0)
//
// Forward: a gather, bound by HBM (write of y; a small table is read from the
// caches).  A warp takes a run of tokens, reads their ids at once and keeps
// several rows in flight.
//
// Gradient: tokens are brought into the order of their ids by a stable radix
// sort, so that the tokens of one row are adjacent and in their original order
// (up to 8192 tokens in one block's shared memory; more in per-digit kernels:
// count, scan, scatter, where a scatter also counts the next digit).  A group
// of lanes then sums a fixed chunk of sorted tokens with FP32 accumulators in
// registers and writes each row that lies inside its chunk once; rows that
// cross chunks are joined from per-chunk FP32 partials in chunk order.
// Nothing depends on the order in which blocks run (no floating-point
// atomics): two runs give the same bits.  dy is read once and dW written once,
// apart from the zero fill beside the first sorting kernel.
#include "elements.cuh"
#include "mixer.h"
#include "shell_ops.h"
#include "tc.cuh"

namespace lsso {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSmallTokens = 8192;        // sorted by one block
constexpr int kSmallThreads = 1024;
constexpr int kSmallItems = kSmallTokens / kSmallThreads;
constexpr int kMaxBits = 9;               // digit width limit
constexpr int kMaxBins = 1 << kMaxBits;

// An id outside [0, vocab) gives a zero row; it must not hide a report of
// undefined outputs (any other value of the status word).
__device__ __forceinline__ void report_token_range(int* status) { atomicCAS(status, kStatusOk, kStatusTokenRange); }

__device__ __forceinline__ int64_t read_id(const void* ids, int ids64, int64_t t) {
  return ids64 ? __ldg(static_cast<const long long*>(ids) + t) : static_cast<int64_t>(__ldg(static_cast<const int*>(ids) + t));
}

// Lanes that share a row and the columns each takes: the widest vector that
// leaves the fewest lanes without columns.
struct RowSplit {
  int vec, lanes, slabs;  // lanes: 8, 16 or 32
};
RowSplit split_row(int64_t width, bool aligned, int widest) {
  RowSplit best{1, 32, 1};
  double best_use = -1.0;
  for (int vec : {8, 4, 1}) {
    if (vec > widest || (vec > 1 && (width % vec != 0 || !aligned))) continue;
    const int64_t items = (width + vec - 1) / vec;
    for (int lanes : {32, 16, 8}) {
      const int64_t slabs = (items + lanes - 1) / lanes;
      const double use = static_cast<double>(items) / (slabs * lanes);
      if (use > best_use + 0.01) {
        best_use = use;
        best = {vec, lanes, static_cast<int>(slabs)};
      }
    }
    if (vec > 1 && best_use >= 0.7) break;  // narrower accesses cost more than a quarter of the lanes
  }
  return best;
}

// ---------------------------------------------------------------- forward
// `lanes` lanes per token, 32 / lanes tokens side by side, `per` tokens per warp.
template <typename W, typename O, int V>
__global__ void __launch_bounds__(kThreads, 4) embed_kernel(const EmbeddingCall c, int lanes, int slabs, int per, int wide) {
  pdl_wait();
  const W* __restrict__ weight = static_cast<const W*>(c.weight);
  O* __restrict__ out = static_cast<O*>(c.out);
  const int lane = threadIdx.x & 31;
  const int64_t base = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * per;
  if (base >= c.tokens) return;
  int row_id = -1;  // of token base + lane; -1: zero row
  if (lane < per && base + lane < c.tokens && (c.row_mask == nullptr || c.row_mask[base + lane] != 0)) {
    const int64_t id = read_id(c.ids, c.ids64, base + lane);
    if (id < 0 || id >= c.vocab) {
      report_token_range(c.status);
    } else {
      row_id = static_cast<int>(id);
    }
  }
  const int side = 32 / lanes, mine = lane / lanes;
  const int count = static_cast<int>(min(static_cast<int64_t>(per), c.tokens - base));
  out += base * c.width;
  constexpr int kAhead = 4;
  for (int i0 = 0; i0 < per; i0 += side * kAhead) {
    int row[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) row[k] = __shfl_sync(0xffffffffu, row_id, (i0 + k * side + mine) & 31);
    for (int s = 0; s < slabs; ++s) {
      const int64_t col = static_cast<int64_t>(s * lanes + (lane & (lanes - 1))) * V;
      if (col >= c.width) continue;
      Run<W, V> w[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        w[k] = load_run<W, V>(weight + max(row[k], 0) * c.width + col, wide);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = i0 + k * side + mine;
        if (i >= count) continue;
        float v[V];
        run_to_float(w[k], v);
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = row[k] >= 0 ? v[q] * c.scale : 0.0f;
        store_run<O, V>(out + i * c.width + col, v, wide);
      }
    }
  }
}

template <typename W, typename O>
cudaError_t launch_embed_types(const EmbeddingCall& c, int sm_count, cudaStream_t stream) {
  const uintptr_t both = reinterpret_cast<uintptr_t>(c.weight) | reinterpret_cast<uintptr_t>(c.out);
  const RowSplit r = split_row(c.width, (both & 15u) == 0, 8);
  const int wide = (both & 31u) == 0 ? 1 : 0;
  // tokens per warp: 32 when that still gives every SM sixteen warps
  int per = 32;
  while (per > 32 / r.lanes && (c.tokens + per - 1) / per < 16 * static_cast<int64_t>(sm_count)) per /= 2;
  const int64_t warps = (c.tokens + per - 1) / per;
  const unsigned grid = static_cast<unsigned>((warps + kWarps - 1) / kWarps);
  LaunchScope scope("embedding", stream);
  if (r.vec == 8) {
    launch_pdl(embed_kernel<W, O, 8>, grid, kThreads, 0, stream, c, r.lanes, r.slabs, per, wide);
  } else if (r.vec == 4) {
    launch_pdl(embed_kernel<W, O, 4>, grid, kThreads, 0, stream, c, r.lanes, r.slabs, per, wide);
  } else {
    launch_pdl(embed_kernel<W, O, 1>, grid, kThreads, 0, stream, c, r.lanes, r.slabs, per, wide);
  }
  return cudaGetLastError();
}

// ---------------------------------------------------------------- sort
struct SortArgs {
  const void* ids;          // first pass: the ids (keys_in null)
  int ids64;
  const uint8_t* row_mask;
  int64_t padding;
  int tokens, vocab;
  const uint32_t* keys_in;  // later passes
  const uint32_t* order_in;
  uint32_t* keys_out;
  uint32_t* order_out;
  uint32_t* counts;         // [bins][blocks]
  uint32_t* next_counts;    // of the next pass, cleared before; null in the last
  uint32_t* totals;         // [bins]
  int blocks, block_tokens, bits, shift, passes;
  uint4* zero;              // the gradient (and the later passes' counts), cleared beside the first kernel
  int64_t zero_vectors;
  uint8_t* zero_tail;
  int zero_tail_bytes;
  uint4* zero_counts;
  int64_t zero_count_vectors;
  int* status;
};

// Sorting key of a token: its id, or `vocab` for a token without a gradient.
__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int t) {
  if (a.row_mask != nullptr && a.row_mask[t] == 0) return static_cast<uint32_t>(a.vocab);
  const int64_t id = read_id(a.ids, a.ids64, t);
  if (id < 0 || id >= a.vocab) {
    report_token_range(a.status);
    return static_cast<uint32_t>(a.vocab);
  }
  return id == a.padding ? static_cast<uint32_t>(a.vocab) : static_cast<uint32_t>(id);
}

// Clears what the blocks from `first` on are asked to (rows that no token uses
// stay zero; a row in use is written over by the summation).
__device__ __forceinline__ void clear(const SortArgs& a, int first) {
  const int64_t stride = static_cast<int64_t>(gridDim.x - first) * blockDim.x;
  const int64_t at = static_cast<int64_t>(blockIdx.x - first) * blockDim.x + threadIdx.x;
  for (int64_t i = at; i < a.zero_count_vectors; i += stride) a.zero_counts[i] = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t i = at; i < a.zero_vectors; i += stride) a.zero[i] = make_uint4(0u, 0u, 0u, 0u);
  if (at < a.zero_tail_bytes) a.zero_tail[at] = 0;
}

// Lanes of the warp that hold the same digit, and this lane's place among them.
__device__ __forceinline__ uint32_t peers_of(uint32_t digit, bool in) {
  return __match_any_sync(0xffffffffu, in ? digit : 0xFFFFFFFFu);
}

// Up to kSmallTokens tokens: all passes in one block, keys and order in shared
// memory.  Warps hold consecutive runs of tokens; a token's rank is the count
// of equal digits before it, in earlier warps and rounds (whist) and in lower
// lanes of its round (match).
__global__ void __launch_bounds__(kSmallThreads) sort_small_kernel(const SortArgs a) {
  pdl_wait();
  if (blockIdx.x > 0) {
    clear(a, 1);
    return;
  }
  extern __shared__ uint32_t sm[];
  uint32_t* skey = sm;                      // [kSmallTokens]
  uint32_t* sorder = sm + kSmallTokens;     // [kSmallTokens]
  uint16_t* whist = reinterpret_cast<uint16_t*>(sm + 2 * kSmallTokens);  // [warps][bins]
  __shared__ uint32_t wsum[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t lower = (1u << lane) - 1u;
  const int bins = 1 << a.bits;
  const int per = (a.tokens + kSmallThreads - 1) / kSmallThreads;  // rounds of 32 tokens per warp
  const int mine = warp * per * 32 + lane;
  uint32_t key[kSmallItems], order[kSmallItems], rank[kSmallItems];
#pragma unroll
  for (int i = 0; i < kSmallItems; ++i) {
    const int t = mine + i * 32;
    key[i] = i < per && t < a.tokens ? sort_key(a, t) : 0u;
    order[i] = static_cast<uint32_t>(t);
  }
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.bits;
    for (int i = threadIdx.x; i < 32 * bins / 2; i += kSmallThreads) reinterpret_cast<uint32_t*>(whist)[i] = 0;
    __syncthreads();
    uint16_t* own = whist + warp * bins;
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
      if (i >= per) break;
      const bool in = mine + i * 32 < a.tokens;
      const uint32_t digit = (key[i] >> shift) & (bins - 1);
      const uint32_t peers = peers_of(digit, in);
      const uint32_t first = in ? own[digit] : 0u;
      __syncwarp();
      rank[i] = first + __popc(peers & lower);
      if (in && (peers & lower) == 0) own[digit] = static_cast<uint16_t>(first + __popc(peers));
      __syncwarp();
    }
    __syncthreads();
    // per digit value (one thread each, bins <= 512): its count over the warps, then all exclusive prefixes
    uint32_t sum = 0;
    if (static_cast<int>(threadIdx.x) < bins) {
      for (int w = 0; w < 32; ++w) sum += whist[w * bins + threadIdx.x];
    }
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < bins) {
      uint32_t at = inc - sum;
      for (int w = 0; w < warp; ++w) at += wsum[w];
      for (int w = 0; w < 32; ++w) {
        const uint32_t n = whist[w * bins + threadIdx.x];
        whist[w * bins + threadIdx.x] = static_cast<uint16_t>(at);
        at += n;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
      if (i >= per || mine + i * 32 >= a.tokens) break;
      const uint32_t at = own[(key[i] >> shift) & (bins - 1)] + rank[i];
      skey[at] = key[i];
      sorder[at] = order[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
      if (i >= per || mine + i * 32 >= a.tokens) break;
      key[i] = skey[mine + i * 32];
      order[i] = sorder[mine + i * 32];
    }
  }
#pragma unroll
  for (int i = 0; i < kSmallItems; ++i) {
    if (i >= per || mine + i * 32 >= a.tokens) break;
    a.keys_out[mine + i * 32] = key[i];
    a.order_out[mine + i * 32] = order[i];
  }
}

// First digit's counts of each block's tokens; the blocks past `blocks` clear.
__global__ void __launch_bounds__(kThreads) sort_count_kernel(const SortArgs a) {
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= a.blocks) {
    clear(a, a.blocks);
    return;
  }
  __shared__ uint32_t hist[kMaxBins];
  const int bins = 1 << a.bits;
  for (int b = threadIdx.x; b < bins; b += kThreads) hist[b] = 0;
  __syncthreads();
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.block_tokens;
  const int64_t end = min(static_cast<int64_t>(a.tokens), begin + a.block_tokens);
  for (int64_t t = begin + threadIdx.x; t < end; t += kThreads) {
    atomicAdd(&hist[sort_key(a, static_cast<int>(t)) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kThreads) a.counts[static_cast<size_t>(b) * a.blocks + blockIdx.x] = hist[b];
}

// Per digit value: exclusive prefix of its counts over the blocks, in place,
// and its total.  One warp per digit value.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(uint32_t* counts, uint32_t* totals, int blocks, int bins) {
  pdl_wait();
  const int bin = static_cast<int>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (bin >= bins) return;
  uint32_t* row = counts + static_cast<size_t>(bin) * blocks;
  uint32_t sum = 0;
#pragma unroll 4
  for (int b0 = 0; b0 < blocks; b0 += 32) {
    const uint32_t v = b0 + lane < blocks ? row[b0 + lane] : 0u;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (b0 + lane < blocks) row[b0 + lane] = sum + inc - v;
    sum += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) totals[bin] = sum;
}

// Stable scatter by one digit, kItems tokens per thread at a time: as in the
// small sort, with the counts of earlier blocks (counts) and of this block's
// earlier sub-tiles (base) added.  Each token also counts its next digit for
// the block that will hold it (integer atomics: the same sums in any order).
template <int kItems>
__global__ void __launch_bounds__(kThreads) sort_scatter_kernel(const SortArgs a) {
  pdl_wait();
  __shared__ uint32_t base[kMaxBins];
  __shared__ uint32_t whist[kWarps][kMaxBins];
  __shared__ uint32_t wsum[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bins = 1 << a.bits;
  constexpr int kTile = kItems * kThreads;
  constexpr int kBinsPerThread = kMaxBins / kThreads;
  // exclusive prefix of the digit totals over the digit values
  uint32_t own[kBinsPerThread], sum = 0;
#pragma unroll
  for (int q = 0; q < kBinsPerThread; ++q) {
    const int b = threadIdx.x * kBinsPerThread + q;
    own[q] = b < bins ? a.totals[b] : 0u;
    sum += own[q];
  }
  uint32_t inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  uint32_t before = inc - sum;
  for (int w = 0; w < warp; ++w) before += wsum[w];
#pragma unroll
  for (int q = 0; q < kBinsPerThread; ++q) {
    const int b = threadIdx.x * kBinsPerThread + q;
    if (b < bins) base[b] = before + a.counts[static_cast<size_t>(b) * a.blocks + blockIdx.x];
    before += own[q];
  }
  const uint32_t lower = (1u << lane) - 1u;
  const int64_t block_begin = static_cast<int64_t>(blockIdx.x) * a.block_tokens;
  const int64_t block_end = min(static_cast<int64_t>(a.tokens), block_begin + a.block_tokens);
  for (int64_t tile = block_begin; tile < block_end; tile += kTile) {
    for (int i = threadIdx.x; i < kWarps * kMaxBins; i += kThreads) (&whist[0][0])[i] = 0;
    __syncthreads();
    const int64_t mine = tile + warp * (kTile / kWarps) + lane;
    uint32_t key[kItems], order[kItems], rank[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int64_t t = mine + i * 32;
      const bool in = t < block_end;
      key[i] = !in ? 0u : a.keys_in != nullptr ? a.keys_in[t] : sort_key(a, static_cast<int>(t));
      order[i] = !in ? 0u : a.order_in != nullptr ? a.order_in[t] : static_cast<uint32_t>(t);
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const bool in = mine + i * 32 < block_end;
      const uint32_t digit = (key[i] >> a.shift) & (bins - 1);
      const uint32_t peers = peers_of(digit, in);
      const uint32_t first = in ? whist[warp][digit] : 0u;
      __syncwarp();
      rank[i] = first + __popc(peers & lower);
      if (in && (peers & lower) == 0) whist[warp][digit] = first + __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) {
      uint32_t at = base[b];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t n = whist[w][b];
        whist[w][b] = at;
        at += n;
      }
      base[b] = at;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (mine + i * 32 >= block_end) continue;
      const uint32_t at = whist[warp][(key[i] >> a.shift) & (bins - 1)] + rank[i];
      a.keys_out[at] = key[i];
      a.order_out[at] = order[i];
      if (a.next_counts != nullptr) {
        const uint32_t next = (key[i] >> (a.shift + a.bits)) & (bins - 1);
        atomicAdd(&a.next_counts[static_cast<size_t>(next) * a.blocks + at / a.block_tokens], 1u);
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- summation
struct SumArgs {
  const uint32_t* keys;   // sorted
  const uint32_t* order;  // token of each sorted position
  const void* grad;
  void* out;
  float* head;            // [chunks][width]: a row continued from the chunk before
  float* tail;            // [chunks][width]: a row begun here and continued in the next chunk
  int64_t width;
  int tokens, vocab, chunk, chunks;
  float scale;
};

// One group of `lanes` lanes per (chunk, slab of lanes V columns).  The group
// reads `lanes` sorted positions at a time (one key and one token per lane)
// and keeps kAhead rows in flight.
template <typename O, typename W, int V>
__global__ void __launch_bounds__(kThreads, 4) embed_sum_kernel(const SumArgs a, int lanes, int slabs) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int side = 32 / lanes, sub = lane & (lanes - 1), group0 = lane & ~(lanes - 1);
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * side + lane / lanes;
  const int64_t chunk = unit / slabs;
  const int64_t col = ((unit - chunk * slabs) * lanes + sub) * V;
  const uint32_t none = static_cast<uint32_t>(a.vocab);
  const int64_t begin = chunk * a.chunk;
  const int64_t end = chunk < a.chunks ? min(static_cast<int64_t>(a.tokens), begin + a.chunk) : begin;
  uint32_t key = end > begin ? a.keys[begin] : none;  // `none`: this group has nothing (more) to do
  if (__all_sync(0xffffffffu, key == none)) return;   // tokens without a gradient sort to the end
  bool from_before = key != none && begin > 0 && a.keys[begin - 1] == key;
  const bool inside = col < a.width;
  const O* grad = static_cast<const O*>(a.grad) + (inside ? col : 0);
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;

  auto finish = [&](bool goes_on) {
    if (inside) {
      if (from_before || goes_on) {
        store_run<float, V>((from_before ? a.head : a.tail) + chunk * a.width + col, acc);
      } else {
        float v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = acc[k] * a.scale;
        store_run<W, V>(static_cast<W*>(a.out) + static_cast<int64_t>(key) * a.width + col, v);
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    from_before = false;
  };

  constexpr int kAhead = 8;  // divides every `lanes`
  for (int64_t at = begin; at < begin + a.chunk; at += lanes) {  // the same trip count in every group
    const bool in = at + sub < end;
    const uint32_t my_key = in ? a.keys[at + sub] : none;
    const uint32_t my_token = in ? a.order[at + sub] : 0u;
    for (int j = 0; j < lanes; j += kAhead) {
      // Every load is issued, a skipped position's too (its token exists): a
      // load under a condition would wait for the one before it.
      Run<O, V> rows[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const uint32_t token = __shfl_sync(0xffffffffu, my_token, group0 + j + i);
        rows[i] = load_run<O, V>(grad + static_cast<int64_t>(token) * a.width);
      }
      if (__all_sync(0xffffffffu, __shfl_sync(0xffffffffu, my_key, group0 + j + kAhead - 1) == key)) {
        // sorted keys: the last of the eight continues the row, so all do
        if (key != none) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            float f[V];
            run_to_float(rows[i], f);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += f[k];
          }
        }
        continue;
      }
      // A row ends among the eight: one position at a time, the rows read
      // again (they are in L1), which keeps one copy of finish() here and
      // the registers low enough for four blocks per SM.
#pragma unroll 1
      for (int i = 0; i < kAhead; ++i) {
        const uint32_t next = __shfl_sync(0xffffffffu, my_key, group0 + j + i);
        const uint32_t token = __shfl_sync(0xffffffffu, my_token, group0 + j + i);
        const Run<O, V> again = load_run<O, V>(grad + static_cast<int64_t>(token) * a.width);
        if (next != key && at + j + i < end && key != none) {
          finish(false);
          key = next;
        }
        if (next != none) {
          float f[V];
          run_to_float(again, f);
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] += f[k];
        }
      }
    }
  }
  if (key != none) finish(end < a.tokens && a.keys[end] == key);
}

// Sum of column `col` of the partials of chunks begin, begin + step, ... < end,
// in that order, sixteen loads in flight.
__device__ __forceinline__ float sum_partials(const float* __restrict__ head, int64_t width, int64_t col, int64_t begin,
                                              int64_t end, int step) {
  float sum = 0.0f;
  for (int64_t c = begin; c < end; c += 16 * step) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __ldg(head + min(c + i * step, end - 1) * width + col);
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += c + i * step < end ? v[i] : 0.0f;
  }
  return sum;
}

// Rows that cross chunks: the warp of the chunk in which such a row begins
// adds its partials in chunk order; a row over more than 32 further chunks is
// left to the whole block (each warp takes every eighth partial, then the
// warps' sums are added in warp order).  Blocks: eight chunks by 32 columns
// (by 512 columns the few long rows of a skewed vocabulary took longer: 65536
// tokens, 50021 x 512, 10 -> 14 us).
template <typename W>
__global__ void __launch_bounds__(kThreads) embed_join_kernel(const SumArgs a) {
  pdl_wait();
  __shared__ uint32_t long_key[kWarps];
  __shared__ int long_any;
  __shared__ float part[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t none = static_cast<uint32_t>(a.vocab);
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  const int64_t col0 = static_cast<int64_t>(blockIdx.y) * 32;
  const int columns = static_cast<int>(min(static_cast<int64_t>(32), a.width - col0));
  if (threadIdx.x == 0) long_any = 0;
  __syncthreads();
  uint32_t key = none;
  if (chunk + 1 < a.chunks) {
    const int64_t begin = chunk * a.chunk, end = begin + a.chunk;  // not the last chunk: whole
    key = a.keys[end - 1];
    if (key != none && (a.keys[end] != key || (begin > 0 && a.keys[begin - 1] == key))) key = none;
  }
  if (lane == 0) long_key[warp] = none;
  if (key != none) {
    const int64_t c = chunk + 1 + lane;
    const uint32_t more = __ballot_sync(0xffffffffu, c < a.chunks && a.keys[c * a.chunk] == key);
    if (more == 0xffffffffu) {
      if (lane == 0) {
        long_key[warp] = key;
        long_any = 1;
      }
    } else {
      const int n = __ffs(~more) - 1;  // chunk + 1 .. chunk + n hold a head partial each
      if (lane < columns) {
        const int64_t at = col0 + lane;
        const float sum = a.tail[chunk * a.width + at] + sum_partials(a.head, a.width, at, chunk + 1, chunk + 1 + n, 1);
        static_cast<W*>(a.out)[static_cast<int64_t>(key) * a.width + at] = from_float<W>(sum * a.scale);
      }
    }
  }
  __syncthreads();
  if (!long_any) return;
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t k = long_key[w];
    if (k == none) continue;  // the same for the whole block
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kWarps + w;
    // the first chunk past `first` that does not continue the row, by 256-way search
    int64_t low = first + 1, high = a.chunks;
    while (low < high) {
      const int64_t step = (high - low + kThreads - 1) / kThreads;
      const int64_t at = low + threadIdx.x * step;
      const int n = __syncthreads_count(at < high && a.keys[at * a.chunk] == k);
      if (n == 0) {
        high = low;
      } else {
        high = min(high, low + n * step);
        low = low + (n - 1) * step + 1;
      }
    }
    if (lane < columns) part[warp][lane] = sum_partials(a.head, a.width, col0 + lane, first + 1 + warp, low, kWarps);
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < columns) {
      const int64_t col = col0 + threadIdx.x;
      float sum = a.tail[first * a.width + col];
#pragma unroll
      for (int g = 0; g < kWarps; ++g) sum += part[g][threadIdx.x];
      static_cast<W*>(a.out)[static_cast<int64_t>(k) * a.width + col] = from_float<W>(sum * a.scale);
    }
    __syncthreads();
  }
}

template <typename O, typename W, int V>
cudaError_t launch_sum(const SumArgs& s, const RowSplit& r, cudaStream_t stream) {
  const int64_t groups = static_cast<int64_t>(s.chunks) * r.slabs;
  const int64_t per_block = kThreads / r.lanes;
  LaunchScope scope("embedding_sum", stream);
  launch_pdl(embed_sum_kernel<O, W, V>, static_cast<unsigned>((groups + per_block - 1) / per_block), kThreads, 0, stream,
             s, r.lanes, r.slabs);
  return cudaGetLastError();
}

template <typename O, typename W>
cudaError_t launch_sum_types(const SumArgs& s, const RowSplit& r, cudaStream_t stream) {
  constexpr int kWidest = sizeof(O) == 4 ? 4 : 8;  // 16-byte loads
  const cudaError_t e = r.vec == 8   ? launch_sum<O, W, kWidest>(s, r, stream)
                        : r.vec == 4 ? launch_sum<O, W, 4>(s, r, stream)
                                     : launch_sum<O, W, 1>(s, r, stream);
  if (e != cudaSuccess || s.chunks < 2) return e;
  LaunchScope scope("embedding_join", stream);
  launch_pdl(embed_join_kernel<W>,
             dim3(static_cast<unsigned>((s.chunks - 1 + kWarps - 1) / kWarps), static_cast<unsigned>((s.width + 31) / 32)),
             kThreads, 0, stream, s);
  return cudaGetLastError();
}

template <typename F>
cudaError_t by_type(int type, F&& f) {
  if (type == kBf16) return f(__nv_bfloat16());
  if (type == kFp16) return f(__half());
  return f(float());
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace

cudaError_t launch_embedding_forward(const EmbeddingCall& c, int sm_count, cudaStream_t stream) {
  return by_type(c.weight_type, [&](auto w) {
    return by_type(c.out_type, [&](auto o) { return launch_embed_types<decltype(w), decltype(o)>(c, sm_count, stream); });
  });
}

EmbeddingGradPlan make_embedding_grad_plan(int64_t tokens, int64_t vocab, int64_t width, int sm_count) {
  EmbeddingGradPlan p{};
  int bits = 1;
  while ((int64_t(1) << bits) < vocab + 1) ++bits;  // keys 0 .. vocab
  p.passes = (bits + kMaxBits - 1) / kMaxBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  // tokens per thread of a sorting block: as few as leave two blocks per SM (a
  // block's time is a chain of shared-memory rounds, one per token)
  p.items = 1;
  const int64_t most = 2 * static_cast<int64_t>(sm_count);
  while (p.items < 8 && (tokens + p.items * kThreads - 1) / (p.items * kThreads) > most) p.items *= 2;
  const int64_t tile = p.items * kThreads;
  const int64_t tiles = (tokens + tile - 1) / tile;
  const int64_t rounds = (tiles + most - 1) / most;
  p.block_tokens = static_cast<int>(rounds * tile);
  p.blocks = static_cast<int>((tokens + p.block_tokens - 1) / p.block_tokens);
  // sorted tokens per group of lanes: few enough chunks to keep the partials small, enough to fill the SMs
  const RowSplit r = split_row(width, true, 8);
  p.chunk = 32;
  while (p.chunk < 256 && (tokens / (2 * p.chunk)) * r.slabs * r.lanes / 32 >= 16 * static_cast<int64_t>(sm_count)) p.chunk *= 2;
  p.chunks = static_cast<int>((tokens + p.chunk - 1) / p.chunk);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = align256(off + bytes);
    return at;
  };
  for (int i = 0; i < 2; ++i) {
    p.keys[i] = take(sizeof(uint32_t) * tokens);
    p.order[i] = take(sizeof(uint32_t) * tokens);
  }
  p.count_bytes = align256((sizeof(uint32_t) << p.bits) * p.blocks);
  p.counts = take(p.count_bytes * p.passes);
  p.totals = take(sizeof(uint32_t) << p.bits);
  p.head = take(sizeof(float) * p.chunks * width);
  p.tail = take(sizeof(float) * p.chunks * width);
  p.total = off;
  return p;
}

cudaError_t launch_embedding_backward(const EmbeddingGradPlan& p, const EmbeddingCall& c, uint8_t* workspace,
                                      int sm_count, cudaStream_t stream) {
  SortArgs a{};
  a.ids = c.ids;
  a.ids64 = c.ids64;
  a.row_mask = c.row_mask;
  a.padding = c.padding;
  a.tokens = static_cast<int>(c.tokens);
  a.vocab = static_cast<int>(c.vocab);
  a.totals = reinterpret_cast<uint32_t*>(workspace + p.totals);
  a.blocks = p.blocks;
  a.block_tokens = p.block_tokens;
  a.bits = p.bits;
  a.passes = p.passes;
  a.status = c.status;
  const int bins = 1 << p.bits;
  const int64_t out_bytes = c.vocab * c.width * (c.weight_type == kFp32 ? 4 : 2);
  a.zero = static_cast<uint4*>(c.out);
  a.zero_vectors = out_bytes / 16;
  a.zero_tail = static_cast<uint8_t*>(c.out) + out_bytes / 16 * 16;
  a.zero_tail_bytes = static_cast<int>(out_bytes % 16);
  const bool small = c.tokens <= kSmallTokens;
  if (!small && p.passes > 1) {
    a.zero_counts = reinterpret_cast<uint4*>(workspace + p.counts + p.count_bytes);
    a.zero_count_vectors = static_cast<int64_t>(p.count_bytes * (p.passes - 1) / 16);
  }
  const int64_t need = (a.zero_vectors + a.zero_count_vectors) / 1024 + 1;
  const int clears = static_cast<int>(need < 4 * sm_count ? need : 4 * sm_count);
  const uint32_t *keys = nullptr, *order = nullptr;
  if (small) {
    a.keys_out = reinterpret_cast<uint32_t*>(workspace + p.keys[0]);
    a.order_out = reinterpret_cast<uint32_t*>(workspace + p.order[0]);
    keys = a.keys_out;
    order = a.order_out;
    const size_t smem = sizeof(uint32_t) * 2 * kSmallTokens + sizeof(uint16_t) * 32 * bins;
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(&sort_small_kernel), smem);
    if (e != cudaSuccess) return e;
    LaunchScope scope("embedding_sort_small", stream);
    launch_pdl(sort_small_kernel, static_cast<unsigned>(1 + clears), kSmallThreads, smem, stream, a);
  } else {
    for (int pass = 0; pass < p.passes; ++pass) {
      a.shift = pass * p.bits;
      a.keys_in = keys;
      a.order_in = order;
      a.keys_out = reinterpret_cast<uint32_t*>(workspace + p.keys[pass & 1]);
      a.order_out = reinterpret_cast<uint32_t*>(workspace + p.order[pass & 1]);
      a.counts = reinterpret_cast<uint32_t*>(workspace + p.counts + pass * p.count_bytes);
      a.next_counts =
          pass + 1 < p.passes ? reinterpret_cast<uint32_t*>(workspace + p.counts + (pass + 1) * p.count_bytes) : nullptr;
      if (pass == 0) {
        LaunchScope scope("embedding_sort_count", stream);
        launch_pdl(sort_count_kernel, static_cast<unsigned>(p.blocks + clears), kThreads, 0, stream, a);
      }
      {
        LaunchScope scope("embedding_sort_scan", stream);
        launch_pdl(sort_scan_kernel, static_cast<unsigned>((bins + kWarps - 1) / kWarps), kThreads, 0, stream, a.counts,
                   a.totals, p.blocks, bins);
      }
      auto scatter = p.items == 1   ? &sort_scatter_kernel<1>
                     : p.items == 2 ? &sort_scatter_kernel<2>
                     : p.items == 4 ? &sort_scatter_kernel<4>
                                    : &sort_scatter_kernel<8>;
      {
        LaunchScope scope("embedding_sort_scatter", stream);
        launch_pdl(scatter, static_cast<unsigned>(p.blocks), kThreads, 0, stream, a);
      }
      keys = a.keys_out;
      order = a.order_out;
    }
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  SumArgs s{};
  s.keys = keys;
  s.order = order;
  s.grad = c.grad;
  s.out = c.out;
  s.head = reinterpret_cast<float*>(workspace + p.head);
  s.tail = reinterpret_cast<float*>(workspace + p.tail);
  s.width = c.width;
  s.tokens = static_cast<int>(c.tokens);
  s.vocab = static_cast<int>(c.vocab);
  s.chunk = p.chunk;
  s.chunks = p.chunks;
  s.scale = c.scale;
  const uintptr_t both = reinterpret_cast<uintptr_t>(c.grad) | reinterpret_cast<uintptr_t>(c.out);
  const RowSplit r = split_row(c.width, (both & 15u) == 0, c.out_type == kFp32 ? 4 : 8);
  return by_type(c.out_type, [&](auto o) {
    return by_type(c.weight_type, [&](auto w) { return launch_sum_types<decltype(o), decltype(w)>(s, r, stream); });
  });
}

}  // namespace lsso
