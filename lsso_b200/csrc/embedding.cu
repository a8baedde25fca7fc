// Token embedding with scaling, and its gradient by sorted tokens.
//
//   y[t]  = scale * W[id[t]]                                   (0 in masked rows)
//   dW[v] = scale * sum over valid t with id[t] = v of dy[t]   (the padding row 0)
//
// Forward: a gather, bound by HBM (write of y; a small table is read from L2).
//
// Gradient: tokens are brought into the order of their ids by a stable radix
// sort (per digit: count, scan, scatter), so that the tokens of one row are
// adjacent and in their original order.  One warp then sums a fixed chunk of
// sorted tokens with FP32 accumulators in registers and writes each row that
// lies inside its chunk once; rows that cross chunks are joined from per-chunk
// FP32 partials in chunk order.  Nothing depends on the order in which blocks
// run (no floating-point atomics): two runs give the same bits.  dy is read
// once and dW written once, apart from the zero fill below.
#include "elements.cuh"
#include "mixer.h"
#include "shell_ops.h"
#include "tc.cuh"

namespace lsso {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 2048;               // tokens a sorting block ranks at a time
constexpr int kMaxBits = 9;               // digit width limit
constexpr int kMaxBins = 1 << kMaxBits;
constexpr int kStatusTokenRange = 3;      // an id outside [0, vocab)

__device__ __forceinline__ int64_t read_id(const void* ids, int ids64, int64_t t) {
  return ids64 ? __ldg(static_cast<const long long*>(ids) + t) : static_cast<int64_t>(__ldg(static_cast<const int*>(ids) + t));
}

// ---------------------------------------------------------------- forward
template <typename W, typename O, int V>
__global__ void __launch_bounds__(kThreads) embed_kernel(const EmbeddingCall c, int64_t items, int per_row) {
  pdl_wait();
  const W* weight = static_cast<const W*>(c.weight);
  O* out = static_cast<O*>(c.out);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < items; i += stride) {
    const int64_t t = items <= 0xFFFFFFFFll
                          ? static_cast<int64_t>(static_cast<uint32_t>(i) / static_cast<uint32_t>(per_row))
                          : i / per_row;
    const int col = static_cast<int>(i - t * per_row) * V;
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.0f;
    if (c.row_mask == nullptr || c.row_mask[t] != 0) {
      const int64_t id = read_id(c.ids, c.ids64, t);
      if (id >= 0 && id < c.vocab) {
        const Run<W, V> w = load_run<W, V>(weight + id * c.width + col);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = to_float(w.v[k]) * c.scale;
      } else if (col == 0) {
        atomicExch(c.status, kStatusTokenRange);
      }
    }
    store_run<O, V>(out + t * c.width + col, v);
  }
}

template <typename W, typename O, int V>
cudaError_t launch_embed(const EmbeddingCall& c, int sm_count, cudaStream_t stream) {
  const int64_t items = c.tokens * (c.width / V);
  const int64_t need = (items + kThreads - 1) / kThreads;
  const int64_t most = static_cast<int64_t>(sm_count) * 64;
  LaunchScope scope("embedding", stream);
  launch_pdl(embed_kernel<W, O, V>, static_cast<unsigned>(need < most ? need : most), kThreads, 0, stream, c, items,
             static_cast<int>(c.width / V));
  return cudaGetLastError();
}

template <typename W, typename O>
cudaError_t launch_embed_types(const EmbeddingCall& c, int sm_count, cudaStream_t stream) {
  const uintptr_t both = reinterpret_cast<uintptr_t>(c.weight) | reinterpret_cast<uintptr_t>(c.out);
  if (c.width % 8 == 0 && (both & 15u) == 0) return launch_embed<W, O, 8>(c, sm_count, stream);
  if (c.width % 4 == 0 && (both & 15u) == 0) return launch_embed<W, O, 4>(c, sm_count, stream);
  return launch_embed<W, O, 1>(c, sm_count, stream);
}

// ---------------------------------------------------------------- sort
// Sorting key of a token: its id, or `vocab` for a token without a gradient.
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
  uint32_t* totals;         // [bins]
  int blocks, rounds, shift, bins;
  uint4* zero;              // first pass: the gradient, cleared beside the count
  int64_t zero_vectors;
  void* zero_tail;
  int zero_tail_bytes;
  int* status;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int t) {
  if (a.keys_in != nullptr) return a.keys_in[t];
  if (a.row_mask != nullptr && a.row_mask[t] == 0) return static_cast<uint32_t>(a.vocab);
  const int64_t id = read_id(a.ids, a.ids64, t);
  if (id < 0 || id >= a.vocab) {
    atomicExch(a.status, kStatusTokenRange);
    return static_cast<uint32_t>(a.vocab);
  }
  return id == a.padding ? static_cast<uint32_t>(a.vocab) : static_cast<uint32_t>(id);
}

// Digit counts of each block's tokens.  In the first pass the blocks past
// `blocks` clear the weight gradient meanwhile (rows that no token uses stay
// zero; a row in use is written over by the summation).
__global__ void __launch_bounds__(kThreads) sort_count_kernel(const SortArgs a) {
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= a.blocks) {
    const int64_t stride = static_cast<int64_t>(gridDim.x - a.blocks) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - a.blocks) * kThreads + threadIdx.x; i < a.zero_vectors;
         i += stride) {
      a.zero[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (static_cast<int>(blockIdx.x) == a.blocks && static_cast<int>(threadIdx.x) < a.zero_tail_bytes) {
      static_cast<uint8_t*>(a.zero_tail)[threadIdx.x] = 0;
    }
    return;
  }
  __shared__ uint32_t hist[kMaxBins];
  for (int b = threadIdx.x; b < a.bins; b += kThreads) hist[b] = 0;
  __syncthreads();
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.rounds * kTile;
  const int64_t end = min(static_cast<int64_t>(a.tokens), begin + static_cast<int64_t>(a.rounds) * kTile);
  for (int64_t t = begin + threadIdx.x; t < end; t += kThreads) {
    atomicAdd(&hist[(sort_key(a, static_cast<int>(t)) >> a.shift) & (a.bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < a.bins; b += kThreads) a.counts[static_cast<size_t>(b) * a.blocks + blockIdx.x] = hist[b];
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

// Stable scatter by one digit.  Warps hold consecutive runs of the block's
// tokens; a token's rank is the count of equal digits before it: in earlier
// blocks (counts), in earlier sub-tiles (base), in earlier warps and rounds of
// this sub-tile (whist), and in lower lanes of its round (match).
__global__ void __launch_bounds__(kThreads) sort_scatter_kernel(const SortArgs a) {
  pdl_wait();
  __shared__ uint32_t base[kMaxBins];
  __shared__ uint32_t whist[kWarps][kMaxBins];
  __shared__ uint32_t wsum[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kPerThread = kTile / kThreads;
  constexpr int kBinsPerThread = kMaxBins / kThreads;
  // exclusive prefix of the digit totals over the digit values
  uint32_t own[kBinsPerThread], sum = 0;
#pragma unroll
  for (int q = 0; q < kBinsPerThread; ++q) {
    const int b = threadIdx.x * kBinsPerThread + q;
    own[q] = b < a.bins ? a.totals[b] : 0u;
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
    if (b < a.bins) base[b] = before + a.counts[static_cast<size_t>(b) * a.blocks + blockIdx.x];
    before += own[q];
  }
  const uint32_t lower = (1u << lane) - 1u;
  for (int round = 0; round < a.rounds; ++round) {
    const int64_t tile = (static_cast<int64_t>(blockIdx.x) * a.rounds + round) * kTile;
    if (tile >= a.tokens) break;
    for (int i = threadIdx.x; i < kWarps * kMaxBins; i += kThreads) (&whist[0][0])[i] = 0;
    __syncthreads();
    const int64_t mine = tile + warp * (kTile / kWarps) + lane;
    uint32_t key[kPerThread], order[kPerThread], rank[kPerThread];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int64_t t = mine + i * 32;
      const bool in = t < a.tokens;
      key[i] = in ? sort_key(a, static_cast<int>(t)) : 0u;
      order[i] = !in ? 0u : a.order_in != nullptr ? a.order_in[t] : static_cast<uint32_t>(t);
    }
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const bool in = mine + i * 32 < a.tokens;
      const uint32_t digit = (key[i] >> a.shift) & (a.bins - 1);
      const uint32_t peers = __match_any_sync(0xffffffffu, in ? digit : 0xFFFFFFFFu);
      const uint32_t first = in ? whist[warp][digit] : 0u;
      __syncwarp();
      rank[i] = first + __popc(peers & lower);
      if (in && (peers & lower) == 0) whist[warp][digit] = first + __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    for (int b = threadIdx.x; b < a.bins; b += kThreads) {
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
    for (int i = 0; i < kPerThread; ++i) {
      if (mine + i * 32 >= a.tokens) continue;
      const uint32_t at = whist[warp][(key[i] >> a.shift) & (a.bins - 1)] + rank[i];
      a.keys_out[at] = key[i];
      a.order_out[at] = order[i];
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

// One warp per (chunk, slab of 32 V columns).
template <typename O, typename W, int V>
__global__ void __launch_bounds__(kThreads) embed_sum_kernel(const SumArgs a, int slabs) {
  pdl_wait();
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int chunk = static_cast<int>(unit / slabs);
  const int64_t col = (static_cast<int64_t>(unit - static_cast<int64_t>(chunk) * slabs) * 32 + lane) * V;
  if (chunk >= a.chunks) return;
  const int begin = chunk * a.chunk, end = min(a.tokens, begin + a.chunk);
  const uint32_t none = static_cast<uint32_t>(a.vocab);
  uint32_t key = a.keys[begin];
  if (key == none) return;  // tokens without a gradient sort to the end
  bool from_before = begin > 0 && a.keys[begin - 1] == key;
  const bool inside = col < a.width;
  const O* grad = static_cast<const O*>(a.grad) + col;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;

  auto finish = [&](bool goes_on) {
    if (inside) {
      if (from_before || goes_on) {
        float* part = (from_before ? a.head : a.tail) + static_cast<int64_t>(chunk) * a.width + col;
        store_run<float, V>(part, acc);
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

  constexpr int kAhead = 8;  // rows in flight
  for (int at = begin; at < end; at += kAhead) {
    uint32_t keys[kAhead];
    Run<O, V> rows[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const bool in = at + i < end;
      keys[i] = in ? a.keys[at + i] : none;
      if (keys[i] != none && inside) rows[i] = load_run<O, V>(grad + static_cast<int64_t>(a.order[at + i]) * a.width);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (at + i >= end) break;
      if (keys[i] != key) {
        finish(false);
        key = keys[i];
      }
      if (key == none) return;
      if (inside) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += to_float(rows[i].v[k]);
      }
    }
  }
  finish(end < a.tokens && a.keys[end] == key);
}

// Rows that cross chunks: the block of the chunk in which such a row begins
// adds its partials in chunk order (lane groups take every kGroups-th chunk,
// then their sums are added in group order).
constexpr int kGroups = 8;
template <typename W>
__global__ void __launch_bounds__(kThreads) embed_join_kernel(const SumArgs a) {
  pdl_wait();
  const int chunk = blockIdx.x;
  const int end = min(a.tokens, (chunk + 1) * a.chunk);
  if (end >= a.tokens) return;
  const uint32_t key = a.keys[end - 1];
  if (key == static_cast<uint32_t>(a.vocab) || a.keys[end] != key) return;
  const int begin = chunk * a.chunk;
  if (begin > 0 && a.keys[begin - 1] == key && a.keys[begin] == key) return;  // begun before this chunk
  // first sorted position past the row
  int low = end, high = a.tokens;
  while (low < high) {
    const int mid = low + (high - low) / 2;
    if (a.keys[mid] == key) {
      low = mid + 1;
    } else {
      high = mid;
    }
  }
  const int last = (low - 1) / a.chunk;  // chunk + 1 .. last hold a head partial each
  __shared__ float part[kGroups][32];
  const int group = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t c0 = static_cast<int64_t>(blockIdx.y) * 32; c0 < a.width; c0 += static_cast<int64_t>(gridDim.y) * 32) {
    const int64_t col = c0 + lane;
    float sum = 0.0f;
    if (col < a.width) {
      if (group == 0) sum = a.tail[static_cast<int64_t>(chunk) * a.width + col];
#pragma unroll 4
      for (int c = chunk + 1 + group; c <= last; c += kGroups) sum += a.head[static_cast<int64_t>(c) * a.width + col];
    }
    part[group][lane] = sum;
    __syncthreads();
    if (group == 0 && col < a.width) {
#pragma unroll
      for (int g = 1; g < kGroups; ++g) sum += part[g][lane];
      static_cast<W*>(a.out)[static_cast<int64_t>(key) * a.width + col] = from_float<W>(sum * a.scale);
    }
    __syncthreads();
  }
}

template <typename O, typename W, int V>
cudaError_t launch_sum(const SumArgs& s, cudaStream_t stream) {
  const int slabs = static_cast<int>((s.width + 32 * V - 1) / (32 * V));
  const int64_t units = static_cast<int64_t>(s.chunks) * slabs;
  {
    LaunchScope scope("embedding_sum", stream);
    launch_pdl(embed_sum_kernel<O, W, V>, static_cast<unsigned>((units + kWarps - 1) / kWarps), kThreads, 0, stream, s,
               slabs);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || s.chunks < 2) return e;
  const int64_t columns = (s.width + 31) / 32;
  LaunchScope scope("embedding_join", stream);
  launch_pdl(embed_join_kernel<W>, dim3(static_cast<unsigned>(s.chunks - 1), static_cast<unsigned>(columns < 64 ? columns : 64)),
             kThreads, 0, stream, s);
  return cudaGetLastError();
}

template <typename O, typename W>
cudaError_t launch_sum_types(const SumArgs& s, cudaStream_t stream) {
  const uintptr_t both = reinterpret_cast<uintptr_t>(s.grad) | reinterpret_cast<uintptr_t>(s.out);
  if (s.width % 8 == 0 && (both & 15u) == 0) return launch_sum<O, W, 8>(s, stream);
  if (s.width % 4 == 0 && (both & 15u) == 0) return launch_sum<O, W, 4>(s, stream);
  return launch_sum<O, W, 1>(s, stream);
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
  const int64_t tiles = (tokens + kTile - 1) / kTile;
  const int64_t most = 4 * static_cast<int64_t>(sm_count);
  p.tile_rounds = static_cast<int>((tiles + most - 1) / most);
  p.blocks = static_cast<int>((tiles + p.tile_rounds - 1) / p.tile_rounds);
  p.chunk = 32;
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
  p.counts = take(sizeof(uint32_t) * (size_t(1) << p.bits) * p.blocks);
  p.totals = take(sizeof(uint32_t) * (size_t(1) << p.bits));
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
  a.counts = reinterpret_cast<uint32_t*>(workspace + p.counts);
  a.totals = reinterpret_cast<uint32_t*>(workspace + p.totals);
  a.blocks = p.blocks;
  a.rounds = p.tile_rounds;
  a.bins = 1 << p.bits;
  a.status = c.status;
  const int64_t out_bytes = c.vocab * c.width * (c.weight_type == kFp32 ? 4 : 2);
  for (int pass = 0; pass < p.passes; ++pass) {
    a.shift = pass * p.bits;
    a.keys_out = reinterpret_cast<uint32_t*>(workspace + p.keys[pass & 1]);
    a.order_out = reinterpret_cast<uint32_t*>(workspace + p.order[pass & 1]);
    int clear = 0;
    if (pass == 0) {
      a.zero = static_cast<uint4*>(c.out);
      a.zero_vectors = out_bytes / 16;
      a.zero_tail = static_cast<uint8_t*>(c.out) + out_bytes / 16 * 16;
      a.zero_tail_bytes = static_cast<int>(out_bytes % 16);
      const int64_t need = (a.zero_vectors + 4 * kThreads - 1) / (4 * kThreads) + 1;
      clear = static_cast<int>(need < 4 * sm_count ? need : 4 * sm_count);
    }
    {
      LaunchScope scope("embedding_sort_count", stream);
      launch_pdl(sort_count_kernel, static_cast<unsigned>(p.blocks + clear), kThreads, 0, stream, a);
    }
    {
      LaunchScope scope("embedding_sort_scan", stream);
      launch_pdl(sort_scan_kernel, static_cast<unsigned>((a.bins + kWarps - 1) / kWarps), kThreads, 0, stream, a.counts,
                 a.totals, p.blocks, a.bins);
    }
    {
      LaunchScope scope("embedding_sort_scatter", stream);
      launch_pdl(sort_scatter_kernel, static_cast<unsigned>(p.blocks), kThreads, 0, stream, a);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    a.keys_in = a.keys_out;
    a.order_in = a.order_out;
  }
  SumArgs s{};
  s.keys = a.keys_in;
  s.order = a.order_in;
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
  return by_type(c.out_type, [&](auto o) {
    return by_type(c.weight_type, [&](auto w) { return launch_sum_types<decltype(o), decltype(w)>(s, stream); });
  });
}

}  // namespace lsso
