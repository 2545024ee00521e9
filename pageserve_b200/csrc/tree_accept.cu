// Acceptance of a verified tree of drafted tokens, and the move of the accepted
// tokens' keys and values to the places they keep in the cache (the batched,
// device-side step after server.py:47-51's argmax when several tokens of a
// sequence were verified at once; slots by engine/paged_attention.py:74-77).
//
// Node i's mask row holds its ancestors and itself, so with parent(i) the
// highest bit below i: ok(0) = true, ok(i) = token(i) == target(parent(i)),
// accepted(i) = every bit of the row is ok. The path is the row of the
// accepted node with most bits (the lowest such node); its k-th node moves
// from cache position start + path(k) to start + k. path(k) >= k, so moving
// in ascending order never overwrites a row that is still to be read, and a
// thread that owns one 16-byte column of one layer can do it without any
// other thread. The cache ends (start_out) before the first node of the path
// whose row, or whose place, lies in no block of the pool.
//
// Bound by latency for few requests (a chain of five dependent loads), by the
// move for many: 32 requests moving 6 tokens of 64 layers x 2 x 2 KB rows read
// and write 101 MB in 18.2 us back to back, most of it in L2, and in 26.6 from
// HBM (3.8 TB/s, the chain included). Every CTA of a request finds the path
// again (at most 256 nodes, four barriers), which is cheaper than a second launch.
#include "common.cuh"

namespace {

using namespace ps;

constexpr int kThreads = 256;
constexpr int kMaxNodes = 256;
constexpr int kMaxWords = kMaxNodes / 64;
constexpr int kBatch = 8;  // rows a thread has in flight
constexpr int kCtas = 8 * 148;  // two rounds of what the SMs hold at once

struct AcceptParams {
  int32_t* num;
  int32_t* nodes;
  int32_t* out_tokens;
  int32_t* start_out;
  const long long* tokens;
  const int32_t* targets;
  const unsigned long long* mask;
  const int32_t* cu_q;
  const int32_t* start_pos;
  uint4* k_cache;
  uint4* v_cache;
  const int32_t* tables;
  int* status;
  int total_tokens;
  int max_q_len;
  int words;
  int max_blocks;
  int num_blocks;
  int block_size;
  int num_layers;
  int row_units;          // 16-byte units of one token's row in one layer
  long long layer_units;
};

__global__ void __launch_bounds__(kThreads) accept_trees_kernel(const AcceptParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t s_ok[kMaxNodes / 32];
  __shared__ int s_best;
  __shared__ int s_kept;  // path nodes before the first without a block
  __shared__ unsigned long long s_row[kMaxWords];
  __shared__ long long s_src[kMaxNodes], s_dst[kMaxNodes];  // unit offsets in a layer; src < 0: stays
  const int b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31;
  const int q0 = p.cu_q[b];
  const long long rows = static_cast<long long>(p.cu_q[b + 1]) - q0;  // of any 32-bit numbers
  const int start = p.start_pos[b];
  const bool lead = blockIdx.x == 0;
  const bool bad = rows < 0 || rows > p.max_q_len || q0 < 0 || start < 0 || q0 + rows > p.total_tokens ||
                   start + rows > INT32_MAX;
  const int n = bad ? 0 : static_cast<int>(rows);
  if (n == 0) {
    if (lead) {
      if (tid == 0) {
        p.num[b] = 0;
        p.start_out[b] = start;
        if (bad) record_error(p.status, kErrShape);
      }
      for (int i = tid; i < p.max_q_len; i += kThreads) {
        p.nodes[static_cast<long long>(b) * p.max_q_len + i] = -1;
        p.out_tokens[static_cast<long long>(b) * p.max_q_len + i] = -1;
      }
    }
    return;
  }
  // this thread's node: its mask row (bits past the tree dropped) and parent
  unsigned long long m[kMaxWords];
  int parent = -1, depth = 0;
#pragma unroll
  for (int w = 0; w < kMaxWords; ++w) {
    m[w] = 0;
    if (tid < n && w < p.words) {
      m[w] = p.mask[static_cast<long long>(q0 + tid) * p.words + w];
      if (64 * (w + 1) > n) m[w] &= n > 64 * w ? (~0ull >> (64 * (w + 1) - n)) : 0ull;
      const unsigned long long below = 64 * w + 63 < tid ? ~0ull : (tid > 64 * w ? (1ull << (tid - 64 * w)) - 1 : 0ull);
      if (m[w] & below) parent = 64 * w + 63 - __clzll(m[w] & below);
      depth += __popcll(m[w]);
    }
  }
  bool ok = tid == 0;
  if (tid > 0 && tid < n && parent >= 0) ok = p.tokens[q0 + tid] == p.targets[q0 + parent];
  const uint32_t bits = __ballot_sync(0xffffffffu, ok);
  if (lane == 0) s_ok[tid >> 5] = bits;
  if (tid == 0) {
    s_best = 0;
    s_kept = kMaxNodes;
  }
  __syncthreads();
  bool whole = tid < n && ok;
#pragma unroll
  for (int w = 0; w < kMaxWords; ++w) {
    const unsigned long long okw = s_ok[2 * w] | static_cast<unsigned long long>(s_ok[2 * w + 1]) << 32;
    if (m[w] & ~okw) whole = false;
  }
  // deepest first, then the lowest node (node 0 alone always qualifies)
  int key = whole ? depth * kMaxNodes + (kMaxNodes - 1 - tid) : 0;
  key = __reduce_max_sync(0xffffffffu, key);
  if (lane == 0 && key) atomicMax(&s_best, key);
  __syncthreads();
  const int best = s_best ? kMaxNodes - 1 - (s_best % kMaxNodes) : 0;
  if (tid == best) {
#pragma unroll
    for (int w = 0; w < kMaxWords; ++w) s_row[w] = m[w];
  }
  __syncthreads();
  int rank = 0, count = 0;
  bool on_path = false;
#pragma unroll
  for (int w = 0; w < kMaxWords; ++w) {
    const unsigned long long r = s_row[w];
    count += __popcll(r);
    if (64 * w + 63 < tid) rank += __popcll(r);
    else if (64 * w <= tid) {
      rank += __popcll(r & ((1ull << (tid - 64 * w)) - 1));
      on_path = (r >> (tid - 64 * w)) & 1;
    }
  }
  if (lead) {
    if (tid == 0) {
      p.num[b] = count;
      if (!p.k_cache) p.start_out[b] = start + count;
    }
    const long long o = static_cast<long long>(b) * p.max_q_len;
    if (on_path) {
      p.nodes[o + rank] = tid;
      p.out_tokens[o + rank] = p.targets[q0 + tid];
    }
    for (int i = count + tid; i < p.max_q_len; i += kThreads) {
      p.nodes[o + i] = -1;
      p.out_tokens[o + i] = -1;
    }
  }
  if (!p.k_cache) return;
  if (on_path) {
    const int32_t* table = p.tables + static_cast<long long>(b) * p.max_blocks;
    const long long ps = static_cast<long long>(start) + tid, pd = static_cast<long long>(start) + rank;
    const long long js = ps / p.block_size, jd = pd / p.block_size;
    long long src = -1, dst = -1;
    bool stored = false;
    if (js >= p.max_blocks) {
      record_error(p.status, kErrShape);
    } else {
      const int is = table[js], id = table[jd];
      stored = is >= 0 && is < p.num_blocks && id >= 0 && id < p.num_blocks;
      if (!stored) {
        record_error(p.status, kErrBlockId);
      } else if (tid != rank) {
        src = (static_cast<long long>(is) * p.block_size + ps % p.block_size) * p.row_units;
        dst = (static_cast<long long>(id) * p.block_size + pd % p.block_size) * p.row_units;
      }
    }
    if (!stored) atomicMin(&s_kept, rank);
    s_src[rank] = src;
    s_dst[rank] = dst;
  }
  __syncthreads();
  count = min(count, s_kept);
  if (lead && tid == 0) p.start_out[b] = start + count;
  const long long per_tensor = static_cast<long long>(p.num_layers) * p.row_units;
  for (long long u = blockIdx.x * static_cast<long long>(kThreads) + tid; u < 2 * per_tensor;
       u += static_cast<long long>(gridDim.x) * kThreads) {
    const bool is_v = u >= per_tensor;
    const long long r = is_v ? u - per_tensor : u;
    const long long layer = r / p.row_units;
    uint4* c = (is_v ? p.v_cache : p.k_cache) + layer * p.layer_units + (r - layer * p.row_units);
    // a batch's loads go out before its stores; later batches read positions
    // at or behind their own index, which no earlier batch wrote
    for (int i0 = 1; i0 < count; i0 += kBatch) {
      uint4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j < count && s_src[i0 + j] >= 0) v[j] = c[s_src[i0 + j]];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j < count && s_src[i0 + j] >= 0) c[s_dst[i0 + j]] = v[j];
    }
  }
}

}  // namespace

extern "C" int ps_accept_trees(int32_t* num, int32_t* nodes, int32_t* out_tokens, int32_t* start_out,
                               const int64_t* tokens, const int32_t* targets, const int64_t* tree_mask,
                               const int32_t* cu_q, const int32_t* start_pos, int num_seqs, int total_tokens,
                               int max_q_len, void* k_cache, void* v_cache, const int32_t* tables, int max_blocks,
                               int num_layers, int num_blocks, int block_size, int num_kv_heads, int head_dim,
                               int dtype, ps_stream_t stream) {
  if (num_seqs <= 0 || total_tokens < 0 || max_q_len <= 0) {
    ps_host::set_error("accept_trees: invalid sizes (seqs %d, tokens %d, max_q_len %d)", num_seqs, total_tokens,
                       max_q_len);
    return PS_ERR_INVALID;
  }
  if (max_q_len > kMaxNodes || num_seqs > 65535) {
    ps_host::set_error("accept_trees: trees of up to %d nodes, up to 65535 requests (max_q_len %d, seqs %d)",
                       kMaxNodes, max_q_len, num_seqs);
    return PS_ERR_UNSUPPORTED;
  }
  if (!num || !nodes || !out_tokens || !start_out || !cu_q || !start_pos ||
      (total_tokens > 0 && (!tokens || !targets || !tree_mask))) {
    ps_host::set_error("accept_trees: null pointer");
    return PS_ERR_INVALID;
  }
  AcceptParams p{};
  int slices = 1;
  if (k_cache || v_cache) {
    const int es = dtype == PS_F32 ? 4 : (dtype == PS_BF16 || dtype == PS_F16) ? 2 : 0;
    if (!es) {
      ps_host::set_error("accept_trees: unsupported dtype %d", dtype);
      return PS_ERR_UNSUPPORTED;
    }
    if (!k_cache || !v_cache || !tables || num_layers <= 0 || num_blocks <= 0 || block_size <= 0 ||
        max_blocks <= 0 || num_kv_heads <= 0 || head_dim <= 0) {
      ps_host::set_error("accept_trees: invalid cache (both caches, a table and positive sizes are needed)");
      return PS_ERR_INVALID;
    }
    const long long row_bytes = static_cast<long long>(num_kv_heads) * head_dim * es;
    if (row_bytes % 16 != 0 || !ps_host::aligned(k_cache, 16) || !ps_host::aligned(v_cache, 16)) {
      ps_host::set_error("accept_trees: cache rows must be whole 16-byte units and the caches 16-byte aligned");
      return PS_ERR_INVALID;
    }
    const uintptr_t k_at = reinterpret_cast<uintptr_t>(k_cache), v_at = reinterpret_cast<uintptr_t>(v_cache);
    const uintptr_t span = static_cast<uintptr_t>(num_layers) * num_blocks * block_size * row_bytes;
    if (k_at < v_at + span && v_at < k_at + span) {
      ps_host::set_error("accept_trees: the caches overlap; their rows are moved at the same time");
      return PS_ERR_INVALID;
    }
    p.row_units = static_cast<int>(row_bytes / 16);
    p.layer_units = static_cast<long long>(num_blocks) * block_size * p.row_units;
    // One unit per thread, unless that is more than kCtas CTAs, whose finding of
    // the path would then cost more than their loads overlap: 32 trees of 61 nodes
    // over 64 layers x 2 x 2 KB rows took 22.0 us as 2048 CTAs, 18.0 as 1184 and
    // 20.2 as 296 (back to back, in L2; 31.6, 28.7 and 28.7 from HBM).
    const long long want = (2LL * num_layers * p.row_units + kThreads - 1) / kThreads;
    const long long most = (kCtas + num_seqs - 1) / num_seqs;
    slices = static_cast<int>(want < most ? want : most);
  }
  // a request's first block writes its outputs while the others read all inputs
  const uintptr_t b4 = 4ull * num_seqs, t4 = 4ull * total_tokens;
  const ps_host::Range ins[] = {{tokens, 2 * t4}, {targets, t4}, {tree_mask, 2 * t4 * ((max_q_len + 63) / 64)},
                                {cu_q, b4 + 4}, {start_pos, b4}, {k_cache ? tables : nullptr, b4 * max_blocks}};
  const ps_host::Range outs[] = {{num, b4}, {nodes, b4 * max_q_len}, {out_tokens, b4 * max_q_len}, {start_out, b4}};
  for (const auto& out : outs)
    for (const auto& in : ins)
      if (ps_host::overlap(out, in)) {
        ps_host::set_error("accept_trees: an output overlaps an input that other blocks still read");
        return PS_ERR_INVALID;
      }
  p.num = num;
  p.nodes = nodes;
  p.out_tokens = out_tokens;
  p.start_out = start_out;
  p.tokens = reinterpret_cast<const long long*>(tokens);
  p.targets = targets;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  p.cu_q = cu_q;
  p.start_pos = start_pos;
  p.k_cache = static_cast<uint4*>(k_cache);
  p.v_cache = static_cast<uint4*>(v_cache);
  p.tables = tables;
  p.status = ps_host::status_word(PS_TU_TREE);
  p.total_tokens = total_tokens;
  p.max_q_len = max_q_len;
  p.words = (max_q_len + 63) / 64;
  p.max_blocks = max_blocks;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.num_layers = num_layers;
  ps_host::launch(accept_trees_kernel, dim3(slices, num_seqs), kThreads, 0, reinterpret_cast<cudaStream_t>(stream),
                  p);
  ps_host::count_launch();
  return ps_host::check_launch("accept_trees");
}
