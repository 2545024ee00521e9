// A step's block tables, positions, KV slots and ancestor masks, from lengths
// that live on the device (engine/scheduler.py's block bookkeeping and the slot
// formula of engine/paged_attention.py:74-77, without the host).
//
// For request b with seq cached and q new tokens:
//   need = ceil((seq + q) / bs), take = max(0, need - held)
//   first_b = sum of take over the requests before b
//   table[j] = old (j < held) | free[first_b + j - held] (j < need) | -1
//   slot(i)  = table[(seq + i) / bs] * bs + (seq + i) % bs
//   anc(i)   = {i} + anc(parent(i)),  position(i) = seq + |anc(i)| - 1
// A tree's rows from the first one on that has no slot get an empty mask, and so
// do all rows of a request whose context passes the table or the caller's bound:
// the keys of the first are stored nowhere, the second has no attention, and a node whose mask row is
// empty is never accepted, nor is one behind it.
//
// Bound by latency (captured: 2.9 us for one request, 4.3 for 64 trees of up to 16
// nodes, 6.1 for 513 requests with tables of 2049 entries, whose 4.2 MB would take
// 1.0 us): the bytes are a few kilobytes to a few megabytes. One
// launch, one CTA per request; each CTA sums take and q over the requests
// before its own, which costs 3 coalesced loads per 256 requests from L2 and
// needs no second pass, no atomics and no order between CTAs. What does not
// depend on that sum (the old entries, the -1 behind the last) is written
// before it.
#include "common.cuh"

namespace {

using namespace ps;

constexpr int kThreads = 256;
constexpr int kMaxNodes = 256;  // tree nodes per request
constexpr int kMaxWords = kMaxNodes / 64;

struct TablesParams {
  int32_t* tables;
  int32_t* held_out;
  int32_t* cu_q;
  int32_t* positions;
  int32_t* slots;
  unsigned long long* mask;
  int32_t* free_used;
  const int32_t* tables_in;
  const int32_t* held_in;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  const int32_t* free_blocks;
  const int32_t* parents;
  int* status;
  long long max_ctx;  // cached and new tokens of a request
  int num_seqs;
  int total_tokens;
  int max_q_len;
  int words;
  int max_blocks;
  int num_free;
  int num_blocks;
  int block_size;
};

struct Span {
  int seq, q, held, need;  // need: entries the request has after the step
};

PS_DEVICE Span span_of(const TablesParams& p, int b) {
  Span s;
  s.seq = max(p.seq_lens[b], 0);
  s.q = max(p.q_lens[b], 0);
  s.held = min(max(p.held_in[b], 0), p.max_blocks);
  const long long ctx = static_cast<long long>(s.seq) + s.q;
  const long long need = (ctx + p.block_size - 1) / p.block_size;
  s.need = max(s.held, static_cast<int>(need < p.max_blocks ? need : p.max_blocks));
  return s;
}

PS_DEVICE long long warp_sum_ll(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(kThreads) step_tables_kernel(const TablesParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ long long s_sum[kThreads / 32][2];
  __shared__ int s_ptr[kMaxNodes];
  __shared__ unsigned long long s_mask[kMaxNodes][kMaxWords];
  __shared__ int s_seen;  // nodes whose masks are kept
  const int b = blockIdx.x;
  const int tid = threadIdx.x;
  const Span s = span_of(p, b);
  const long long row = static_cast<long long>(b) * p.max_blocks;
  const int32_t* old = p.tables_in + row;
  int32_t* tab = p.tables + row;

  // take and q of the requests before this one
  long long take_before = 0, q_before = 0;
  for (int i = tid; i < b; i += kThreads) {
    const Span o = span_of(p, i);
    take_before += o.need - o.held;
    q_before += o.q;
  }
  // old entries and the -1 behind the last (in place: the old ones stay)
  if (tab != old)
    for (int j = tid; j < s.held; j += kThreads) tab[j] = old[j];
  for (int j = s.need + tid; j < p.max_blocks; j += kThreads) tab[j] = -1;

  take_before = warp_sum_ll(take_before);
  q_before = warp_sum_ll(q_before);
  if ((tid & 31) == 0) {
    s_sum[tid >> 5][0] = take_before;
    s_sum[tid >> 5][1] = q_before;
  }
  bool fits = true;  // of thread 0
  if (tid == 0) {
    fits = static_cast<long long>(s.seq) + s.q <= p.max_ctx;
    s_seen = fits ? kMaxNodes : 0;
  }
  __syncthreads();
  long long first = 0, cu = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    first += s_sum[w][0];
    cu += s_sum[w][1];
  }
  const int take = s.need - s.held;
  const long long left = first < p.num_free ? p.num_free - first : 0;
  const int given = static_cast<int>(left < take ? left : take);
  const int T = p.total_tokens;
  const int row0 = static_cast<int>(cu < T ? cu : T);
  const long long cu_next = cu + s.q;
  const int row1 = static_cast<int>(cu_next < T ? cu_next : T);

  for (int j = tid; j < take; j += kThreads) tab[s.held + j] = j < given ? p.free_blocks[first + j] : -1;
  if (tid == 0) {
    p.held_out[b] = s.held + given;
    p.cu_q[b] = row0;
    int err = kErrNone;
    if (p.seq_lens[b] < 0 || p.q_lens[b] < 0 || p.held_in[b] < 0 || p.held_in[b] > p.max_blocks ||
        cu_next > T || (p.parents && s.q > p.max_q_len) || !fits)
      err = kErrShape;
    else if (given < take)
      err = kErrNoBlocks;
    if (err) record_error(p.status, err);
    if (b == p.num_seqs - 1) {
      p.cu_q[p.num_seqs] = row1;
      const long long used = first + take;
      *p.free_used = static_cast<int32_t>(used < INT32_MAX ? used : INT32_MAX);
    }
  }

  // slots (and a chunk's positions): every new token's place in the cache
  for (int i = tid; i < row1 - row0; i += kThreads) {
    const long long at = static_cast<long long>(s.seq) + i;
    const long long j = at / p.block_size;
    int id = -1;
    if (j < s.held) id = old[j];
    else if (j < s.held + given) id = p.free_blocks[first + (j - s.held)];
    int slot = -1;
    if (id >= 0 && id < p.num_blocks) slot = id * p.block_size + static_cast<int>(at % p.block_size);
    else {
      record_error(p.status, j < s.held + given ? kErrBlockId : (j < s.need ? kErrNoBlocks : kErrShape));
      if (p.parents) atomicMin(&s_seen, i);
    }
    p.slots[row0 + i] = slot;
    if (!p.parents) p.positions[row0 + i] = static_cast<int32_t>(at < INT32_MAX ? at : INT32_MAX);
  }

  if (p.parents) {
    // ancestor masks by pointer doubling: after k rounds mask(i) holds the
    // ancestors less than 2^k generations away and ptr(i) the one 2^k away
    const int n = min(row1 - row0, p.max_q_len);
    const bool node = tid < n;
    int ptr = -1;
    if (node) {
      ptr = p.parents[row0 + tid];
      if (ptr < -1 || ptr >= tid) {
        record_error(p.status, kErrShape);
        ptr = -1;
      }
    }
    unsigned long long m[kMaxWords];
#pragma unroll
    for (int w = 0; w < kMaxWords; ++w) m[w] = (tid >> 6) == w ? 1ull << (tid & 63) : 0ull;
    while (true) {
      s_ptr[tid] = ptr;
#pragma unroll
      for (int w = 0; w < kMaxWords; ++w) s_mask[tid][w] = m[w];
      if (!__syncthreads_or(ptr >= 0)) break;
      if (ptr >= 0) {
#pragma unroll
        for (int w = 0; w < kMaxWords; ++w) m[w] |= s_mask[ptr][w];
        ptr = s_ptr[ptr];
      }
      __syncthreads();
    }
    if (node) {
      int depth = -1;
#pragma unroll
      for (int w = 0; w < kMaxWords; ++w) depth += __popcll(m[w]);
      const long long at = static_cast<long long>(s.seq) + depth;
      p.positions[row0 + tid] = static_cast<int32_t>(at < INT32_MAX ? at : INT32_MAX);
      const bool kept = tid < s_seen;  // (complete before the barriers above)
#pragma unroll
      for (int w = 0; w < kMaxWords; ++w)
        if (w < p.words) p.mask[static_cast<long long>(row0 + tid) * p.words + w] = kept ? m[w] : 0ull;
    }
    // nodes past the limit see nothing and are written nowhere (recorded above)
    for (int i = n + tid; i < row1 - row0; i += kThreads) {
      p.positions[row0 + i] = s.seq;
      p.slots[row0 + i] = -1;
      for (int w = 0; w < p.words; ++w) p.mask[static_cast<long long>(row0 + i) * p.words + w] = 0;
    }
  }

  if (b == p.num_seqs - 1) {  // rows behind the last request
    for (int t = row1 + tid; t < T; t += kThreads) {
      p.positions[t] = 0;
      p.slots[t] = -1;
      if (p.parents)
        for (int w = 0; w < p.words; ++w) p.mask[static_cast<long long>(t) * p.words + w] = 0;
    }
  }
}

}  // namespace

extern "C" {

int ps_build_step_tables(int32_t* tables, int32_t* held_out, int32_t* cu_q, int32_t* positions, int32_t* slots,
                         int64_t* tree_mask, int32_t* free_used, const int32_t* tables_in, const int32_t* held,
                         const int32_t* seq_lens, const int32_t* q_lens, const int32_t* free_blocks,
                         const int32_t* parents, int num_seqs, int total_tokens, int max_q_len, int max_blocks,
                         int num_free, int num_blocks, int block_size, ps_stream_t stream) {
  return ps_build_step_tables_bounded(tables, held_out, cu_q, positions, slots, tree_mask, free_used, tables_in, held,
                                      seq_lens, q_lens, free_blocks, parents, num_seqs, total_tokens, max_q_len,
                                      max_blocks, num_free, num_blocks, block_size, INT32_MAX, stream);
}

int ps_build_step_tables_bounded(int32_t* tables, int32_t* held_out, int32_t* cu_q, int32_t* positions,
                                 int32_t* slots, int64_t* tree_mask, int32_t* free_used, const int32_t* tables_in,
                                 const int32_t* held, const int32_t* seq_lens, const int32_t* q_lens,
                                 const int32_t* free_blocks, const int32_t* parents, int num_seqs, int total_tokens,
                                 int max_q_len, int max_blocks, int num_free, int num_blocks, int block_size,
                                 int max_ctx, ps_stream_t stream) {
  if (num_seqs <= 0 || total_tokens < 0 || max_blocks <= 0 || num_free < 0 || num_blocks <= 0 || block_size <= 0 ||
      max_ctx < 0) {
    ps_host::set_error("build_step_tables: invalid sizes (seqs %d, tokens %d, table width %d, free %d, pool %d x %d)",
                       num_seqs, total_tokens, max_blocks, num_free, num_blocks, block_size);
    return PS_ERR_INVALID;
  }
  if (static_cast<long long>(num_blocks) * block_size > INT32_MAX) {
    ps_host::set_error("build_step_tables: %d blocks of %d have slots past 32 bits", num_blocks, block_size);
    return PS_ERR_INVALID;
  }
  if (!tables || !held_out || !cu_q || !free_used || !tables_in || !held || !seq_lens || !q_lens ||
      (num_free > 0 && !free_blocks) || (total_tokens > 0 && (!positions || !slots)) ||
      (parents && total_tokens > 0 && !tree_mask)) {
    ps_host::set_error("build_step_tables: null pointer");
    return PS_ERR_INVALID;
  }
  if (parents && (max_q_len <= 0 || max_q_len > kMaxNodes)) {
    ps_host::set_error("build_step_tables: trees of 1 to %d nodes per request (max_q_len %d)", kMaxNodes, max_q_len);
    return max_q_len <= 0 ? PS_ERR_INVALID : PS_ERR_UNSUPPORTED;
  }
  // A request's outputs are written while others still read their inputs; tables
  // in place are the exception, for a request reads its own row alone.
  const uintptr_t b4 = 4ull * num_seqs, t4 = 4ull * total_tokens, w4 = b4 * max_blocks;
  const uintptr_t mask_bytes = parents ? 2 * t4 * ((max_q_len + 63) / 64) : 0;
  const ps_host::Range ins[] = {{tables_in, w4}, {held, b4}, {seq_lens, b4}, {q_lens, b4},
                                {free_blocks, 4ull * num_free}, {parents, t4}};
  const ps_host::Range outs[] = {{tables, w4}, {held_out, b4}, {cu_q, b4 + 4}, {positions, t4}, {slots, t4},
                                 {parents ? tree_mask : nullptr, mask_bytes}, {free_used, 4}};
  for (const auto& out : outs)
    for (const auto& in : ins)
      if (ps_host::overlap(out, in) && !(out.at == tables && in.at == tables_in && tables == tables_in)) {
        ps_host::set_error("build_step_tables: an output overlaps an input that other requests still read "
                           "(tables may be tables_in itself, nothing else)");
        return PS_ERR_INVALID;
      }
  TablesParams p{};
  p.tables = tables;
  p.held_out = held_out;
  p.cu_q = cu_q;
  p.positions = positions;
  p.slots = slots;
  p.mask = reinterpret_cast<unsigned long long*>(tree_mask);
  p.free_used = free_used;
  p.tables_in = tables_in;
  p.held_in = held;
  p.seq_lens = seq_lens;
  p.q_lens = q_lens;
  p.free_blocks = free_blocks;
  p.parents = parents;
  p.status = ps_host::status_word(PS_TU_TREE);
  const long long capacity = static_cast<long long>(max_blocks) * block_size;
  p.max_ctx = max_ctx < capacity ? max_ctx : capacity;
  p.num_seqs = num_seqs;
  p.total_tokens = total_tokens;
  p.max_q_len = max_q_len;
  p.words = (max_q_len + 63) / 64;
  p.max_blocks = max_blocks;
  p.num_free = num_free;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  ps_host::launch(step_tables_kernel, num_seqs, kThreads, 0, reinterpret_cast<cudaStream_t>(stream), p);
  ps_host::count_launch();
  return ps_host::check_launch("build_step_tables");
}

}  // extern "C"
