// Attention of a tree of drafted tokens over the paged cache: node i of request
// b sees the request's cached keys [0, start) and the drafted nodes whose bit
// is set in its mask row (itself and its ancestors),
//   o_i = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j,  0 where it sees nothing
// (engine/paged_attention.py:16-50, 82-99, 117-132 with the causal rule of the
// new tokens replaced by the tree's).
//
// Rows are (node, q head of the kv head's group) pairs, row r = node * G + g,
// so that a K/V tile is read once for the whole group. The work of a call is
// the list of (sequence, kv head, row tile, key tile) in that order; its length
// is known on the device only, and each CTA takes an equal, contiguous share of
// it. A row tile whose key tiles fall into several shares leaves (o, max, sum)
// partials in the workspace (at most two per CTA, whatever the contexts), and
// a second kernel joins them in order: no atomics, the same bits every time.
//
// What a node does not see does not reach it, NaN and infinities included:
// masked scores are replaced before the softmax, rows past the context are
// zero-filled, and a drafted V row with a value that is not finite is cleared
// from the tile and added back only to the rows that see it.
#include <cfloat>
#include <climits>
#include <cstdlib>

#include "common.cuh"

namespace {

using namespace ps;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxNodes = 256;

struct TreeParams {
  void* out;
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const int32_t* tables;
  const int32_t* cu_q;
  const int32_t* start_pos;
  const unsigned long long* mask;
  float* part;          // [CTA][2][rows][D] of o, then [CTA][2][rows][2] of (max, sum)
  float* part_ml;
  long long* seq_base;  // [num_seqs + 1] first work item of each sequence
  long long* share;     // work items per CTA
  int* status;
  int total_q;
  int words;
  int max_blocks;
  int num_blocks;
  int block_size;
  int Hq, Hkv, G;
  int max_q_len;
  int max_ctx;
  int num_seqs;
  int num_ctas;
  int min_share;        // fewest key tiles worth a CTA
  float scale_log2;
};

// ------------------------------------------------------- division of work --
struct Seq {
  int q0, n, start, row_tiles, key_tiles;
};

template <int ROWS, int KEYS>
PS_DEVICE Seq seq_of(const TreeParams& p, int b, bool record) {
  Seq s;
  s.q0 = p.cu_q[b];
  s.n = p.cu_q[b + 1] - s.q0;
  s.start = p.start_pos[b];
  s.row_tiles = s.key_tiles = 0;
  const long long ctx = static_cast<long long>(s.start) + s.n;
  if (s.n == 0) return s;
  if (s.n < 0 || s.n > p.max_q_len || s.q0 < 0 || s.q0 + s.n > p.total_q || s.start < 0 || ctx > p.max_ctx ||
      ctx > static_cast<long long>(p.max_blocks) * p.block_size) {
    if (record) record_error(p.status, kErrShape);
    s.n = 0;
    return s;
  }
  s.row_tiles = (s.n * p.G + ROWS - 1) / ROWS;
  s.key_tiles = (static_cast<int>(ctx) + KEYS - 1) / KEYS;
  return s;
}

template <int ROWS, int KEYS>
PS_DEVICE long long items_of(const TreeParams& p, int b, bool record) {
  const Seq s = seq_of<ROWS, KEYS>(p, b, record);
  return static_cast<long long>(p.Hkv) * s.row_tiles * s.key_tiles;
}

// By one whole warp: this CTA's share [*begin, *end) of the work, the sequence
// that holds *begin and that sequence's first item. CTA 0 also writes the
// sequences' first items for the joining kernel.
template <int ROWS, int KEYS>
PS_DEVICE void find_share(const TreeParams& p, int lane, long long* begin, long long* end, int* b_out,
                          long long* base_out) {
  const bool lead = blockIdx.x == 0;
  long long total = 0;
  for (int b = lane; b < p.num_seqs; b += 32) total += items_of<ROWS, KEYS>(p, b, lead);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  long long per = (total + p.num_ctas - 1) / p.num_ctas;
  if (per < p.min_share) per = p.min_share;
  const long long lo = per * blockIdx.x;
  *begin = lo < total ? lo : total;
  *end = lo + per < total ? lo + per : total;
  *b_out = p.num_seqs;
  *base_out = total;
  if (lead && lane == 0) {
    *p.share = per;
    p.seq_base[p.num_seqs] = total;
  }
  if (*begin >= *end && !lead) return;
  long long run = 0;
  bool found = false;
  for (int b0 = 0; b0 < p.num_seqs; b0 += 32) {
    const int b = b0 + lane;
    const long long n = b < p.num_seqs ? items_of<ROWS, KEYS>(p, b, false) : 0;
    long long incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const long long first = run + incl - n;
    if (lead && b < p.num_seqs) p.seq_base[b] = first;
    const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && *begin >= first && *begin < first + n);
    if (hit && !found) {
      const int src = __ffs(hit) - 1;
      *b_out = b0 + src;
      *base_out = __shfl_sync(0xffffffffu, first, src);
      found = true;
      if (!lead) return;
    }
    run += __shfl_sync(0xffffffffu, incl, 31);
  }
}

// Walk over the segments (one row tile's key tiles) of a share.
template <int ROWS, int KEYS>
struct Segment {
  long long cur, end, base;  // next item, share's end, first item of sequence b
  int b;
  Seq s;
  int h, row0, tile0, tile1;

  PS_DEVICE void init(const TreeParams& p, long long begin, long long end_, int b_, long long base_) {
    cur = begin;
    end = end_;
    b = b_;
    base = base_;
    if (cur < end) s = seq_of<ROWS, KEYS>(p, b, false);
  }
  PS_DEVICE bool next(const TreeParams& p) {
    if (cur >= end) return false;
    long long items = static_cast<long long>(p.Hkv) * s.row_tiles * s.key_tiles;
    while (cur >= base + items) {
      base += items;
      s = seq_of<ROWS, KEYS>(p, ++b, false);
      items = static_cast<long long>(p.Hkv) * s.row_tiles * s.key_tiles;
    }
    const long long at = cur - base;
    const long long pair = at / s.key_tiles;
    tile0 = static_cast<int>(at - pair * s.key_tiles);
    h = static_cast<int>(pair / s.row_tiles);
    row0 = static_cast<int>(pair - static_cast<long long>(h) * s.row_tiles) * ROWS;
    const long long left = end - cur;
    tile1 = left < s.key_tiles - tile0 ? tile0 + static_cast<int>(left) : s.key_tiles;
    cur += tile1 - tile0;
    return true;
  }
  PS_DEVICE bool whole() const { return tile0 == 0 && tile1 == s.key_tiles; }
  // a row tile's first part is the last segment of its CTA, the others the first
  PS_DEVICE int slot() const { return tile0 > 0 ? 0 : 1; }
};

// Bits of the 64 keys from tree index `off` on (keys before the tree are seen
// by every node, keys behind it by none).
PS_DEVICE unsigned long long seen64(const unsigned long long* row, int words, int off, int n) {
  if (off <= -64) return ~0ull;
  if (off >= n) return 0ull;
  unsigned long long v;
  if (off < 0) {
    v = (row[0] << -off) | ((1ull << -off) - 1);
  } else {
    const int w = off >> 6, sh = off & 63;
    v = row[w] >> sh;
    if (sh && w + 1 < words) v |= row[w + 1] << (64 - sh);
  }
  const int keep = n - off;  // keys of the tile that exist
  if (keep < 64) v &= (1ull << keep) - 1;
  return v;
}

template <typename T>
PS_DEVICE bool finite16(uint16_t x) {
  return std::is_same<T, __half>::value ? (x & 0x7C00u) != 0x7C00u : (x & 0x7F80u) != 0x7F80u;
}

// --------------------------------------------------------- mma.sync kernel --
// Any block size, head_dim 64 or 128: 64 rows per CTA (16 per warp), 64-key
// tiles through a 3-stage ring of 16-byte cp.async.
constexpr int kThreads = 128;
constexpr int kRows = 64;
constexpr int kKeys = 64;
constexpr int kStages = 3;

PS_DEVICE uint32_t swz(int row, int chunk, int row_bytes) {
  return static_cast<uint32_t>(row * row_bytes + ((chunk ^ (row & 7)) << 4));
}

template <typename T, int D>
PS_DEVICE void load_keys(const TreeParams& p, const int32_t* table, int h, int t0, int ctx, uint32_t ks,
                         uint32_t vs) {
  constexpr int kChunks = D / 8;
#pragma unroll
  for (int i = 0; i < kKeys * kChunks / kThreads; ++i) {
    const int id = threadIdx.x + i * kThreads;
    const int r = id / kChunks, c = id % kChunks;
    const int key = t0 + r;
    int bytes = 0;
    long long off = 0;
    if (key < ctx) {
      const int phys = table[key / p.block_size];
      if (phys >= 0 && phys < p.num_blocks) {
        off = ((static_cast<long long>(phys) * p.block_size + key % p.block_size) * p.Hkv + h) * D + c * 8;
        bytes = 16;
      } else {
        record_error(p.status, kErrBlockId);
      }
    }
    const uint32_t so = swz(r, c, D * 2);
    cp_async16(ks + so, static_cast<const T*>(p.k_cache) + off, bytes);
    cp_async16(vs + so, static_cast<const T*>(p.v_cache) + off, bytes);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) tree_mma_kernel(const TreeParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kTile = kKeys * D * 2;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_share[3];
  __shared__ int s_b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    long long begin, end, base;
    int b;
    find_share<kRows, kKeys>(p, lane, &begin, &end, &b, &base);
    if (lane == 0) {
      s_share[0] = begin;
      s_share[1] = end;
      s_share[2] = base;
      s_b = b;
    }
  }
  __syncthreads();
  Segment<kRows, kKeys> sg;
  sg.init(p, s_share[0], s_share[1], s_b, s_share[2]);
  const uint32_t base = smem_u32(smem);
  const int mat = lane >> 3;
  while (sg.next(p)) {
    const int ctx = sg.s.start + sg.s.n;
    const int R = sg.s.n * p.G;
    const int32_t* table = p.tables + static_cast<long long>(sg.b) * p.max_blocks;
    const int ntiles = sg.tile1 - sg.tile0;
    const int first_key = sg.tile0 * kKeys;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      const uint32_t st = base + s * 2 * kTile;
      if (s < ntiles) load_keys<T, D>(p, table, sg.h, first_key + s * kKeys, ctx, st, st + kTile);
      cp_async_commit();
    }
    // this warp's 16 rows: A fragments of Q, and the two rows this thread masks
    const int wrow = sg.row0 + warp * 16;
    uint32_t qa[D / 16][4];
    int node[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = wrow + (lane >> 2) + hf * 8;
      const bool ok = r < R;
      node[hf] = ok ? r / p.G : -1;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          static_cast<const T*>(p.q) +
          (static_cast<long long>(sg.s.q0 + (ok ? r / p.G : 0)) * p.Hq + sg.h * p.G + (ok ? r % p.G : 0)) * D);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qa[ks][hf] = ok ? src[ks * 8 + (lane & 3)] : 0u;
        qa[ks][hf + 2] = ok ? src[ks * 8 + (lane & 3) + 4] : 0u;
      }
    }
    const bool warp_on = wrow < R;
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.f, 0.f};
    bool odd_values = false;  // a drafted V row of this segment is not finite
    for (int j = 0; j < ntiles; ++j) {
      cp_async_wait<kStages - 2>();
      __syncthreads();
      {
        const int jn = j + kStages - 1;
        const uint32_t st = base + (jn % kStages) * 2 * kTile;
        if (jn < ntiles) load_keys<T, D>(p, table, sg.h, first_key + jn * kKeys, ctx, st, st + kTile);
        cp_async_commit();
      }
      const uint32_t ks = base + (j % kStages) * 2 * kTile;
      const uint32_t vs = ks + kTile;
      const int t0 = first_key + j * kKeys;
      const bool tail = t0 + kKeys > sg.s.start;  // drafted keys (or the end) in this tile
      if (tail) {
        // clear drafted V values that are not finite: 0 * inf would reach rows that do not see them
        bool bad = false;
        uint16_t* vt = reinterpret_cast<uint16_t*>(smem + (vs - base));
        for (int i = threadIdx.x; i < kKeys * D; i += kThreads) {
          const int r = i / D, c = i % D;
          if (t0 + r < sg.s.start || t0 + r >= ctx) continue;
          uint16_t* x = vt + swz(r, c >> 3, D * 2) / 2 + (c & 7);
          if (!finite16<T>(*x)) {
            bad = true;
            *x = 0;
          }
        }
        odd_values |= __syncthreads_or(bad) != 0;
      }
      if (!warp_on) continue;
      unsigned long long vis[2] = {~0ull, ~0ull};
      if (tail) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          vis[hf] = node[hf] < 0 ? 0ull
                                 : seen64(p.mask + static_cast<long long>(sg.s.q0 + node[hf]) * p.words, p.words,
                                          t0 - sg.s.start, sg.s.n);
      }
      float s[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int np = 0; np < 4; ++np) {
          uint32_t f[4];
          const int krow = np * 16 + ((mat >> 1) << 3) + (lane & 7);
          ldmatrix_x4(ks + swz(krow, 2 * k + (mat & 1), D * 2), f[0], f[1], f[2], f[3]);
          mma_16816<T>(s[2 * np], qa[k], f);
          mma_16816<T>(s[2 * np + 1], qa[k], f + 2);
        }
      float mt[2] = {-FLT_MAX, -FLT_MAX};
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kk = n * 8 + 2 * (lane & 3) + (e & 1);
          s[n][e] = (vis[e >> 1] >> kk) & 1 ? s[n][e] * p.scale_log2 : -INFINITY;
          mt[e >> 1] = fmaxf(mt[e >> 1], s[n][e]);
        }
      float corr[2];
#pragma unroll
      for (int ri = 0; ri < 2; ++ri) {
        mt[ri] = fmaxf(mt[ri], __shfl_xor_sync(0xffffffffu, mt[ri], 1));
        mt[ri] = fmaxf(mt[ri], __shfl_xor_sync(0xffffffffu, mt[ri], 2));
        const float mn = fmaxf(m[ri], mt[ri]);
        corr[ri] = exp2f(m[ri] - mn);  // m starts finite: a tile that shows nothing leaves it alone
        m[ri] = mn;
      }
      float rs[2] = {0.f, 0.f};
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = exp2f(s[n][e] - m[e >> 1]);
          rs[e >> 1] += s[n][e];
        }
#pragma unroll
      for (int ri = 0; ri < 2; ++ri) l[ri] = l[ri] * corr[ri] + rs[ri];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= corr[0];
        o[i][1] *= corr[0];
        o[i][2] *= corr[1];
        o[i][3] *= corr[1];
      }
      // P is rounded to the cache's type for the matrix unit: relative 2^-9
      // (bf16) or 2^-12 (f16) a term, below the rounding of the output
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t pa[4];
        pa[0] = pack2<T>(s[2 * kk][0], s[2 * kk][1]);
        pa[1] = pack2<T>(s[2 * kk][2], s[2 * kk][3]);
        pa[2] = pack2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
        pa[3] = pack2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
        const int vrow = kk * 16 + ((mat & 1) << 3) + (lane & 7);
#pragma unroll
        for (int dp = 0; dp < D / 16; ++dp) {
          uint32_t f[4];
          ldmatrix_x4_trans(vs + swz(vrow, 2 * dp + (mat >> 1), D * 2), f[0], f[1], f[2], f[3]);
          mma_16816<T>(o[2 * dp], pa, f);
          mma_16816<T>(o[2 * dp + 1], pa, f + 2);
        }
      }
    }
    cp_async_wait<0>();
    __syncthreads();  // the ring is free for the next segment
    if (!warp_on) continue;
#pragma unroll
    for (int ri = 0; ri < 2; ++ri) {
      l[ri] += __shfl_xor_sync(0xffffffffu, l[ri], 1);
      l[ri] += __shfl_xor_sync(0xffffffffu, l[ri], 2);
    }
    if (odd_values) {
      // add the cleared values to the rows that see them
      const int k0 = max(first_key, sg.s.start), k1 = min(sg.tile1 * kKeys, ctx);
      for (int key = k0; key < k1; ++key) {
        const int phys = table[key / p.block_size];
        if (phys < 0 || phys >= p.num_blocks) continue;
        const T* vr = static_cast<const T*>(p.v_cache) +
                      ((static_cast<long long>(phys) * p.block_size + key % p.block_size) * p.Hkv + sg.h) * D;
        const int jn = key - sg.s.start;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (node[hf] < 0 ||
              !((p.mask[static_cast<long long>(sg.s.q0 + node[hf]) * p.words + (jn >> 6)] >> (jn & 63)) & 1))
            continue;
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const T x = vr[i * 8 + 2 * (lane & 3) + e];
              if (!finite16<T>(*reinterpret_cast<const uint16_t*>(&x))) o[i][2 * hf + e] += to_f32(x);
            }
        }
      }
    }
    const bool whole = sg.whole();
    const long long pslot = (static_cast<long long>(blockIdx.x) * 2 + sg.slot()) * kRows;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = wrow + (lane >> 2) + hf * 8;
      if (r >= R) continue;
      if (whole) {
        const float inv = l[hf] == 0.f ? 0.f : 1.f / l[hf];
        T* dst = static_cast<T*>(p.out) +
                 (static_cast<long long>(sg.s.q0 + r / p.G) * p.Hq + sg.h * p.G + r % p.G) * D + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<uint32_t*>(dst + i * 8) = pack2<T>(o[i][2 * hf] * inv, o[i][2 * hf + 1] * inv);
      } else {
        const long long pr = pslot + r - sg.row0;
        float* dst = p.part + pr * D + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[i][2 * hf], o[i][2 * hf + 1]);
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(p.part_ml + pr * 2) = make_float2(m[hf], l[hf]);
      }
    }
  }
}

// -------------------------------------------------------------- the joining --
// One CTA column per boundary between two shares; the first boundary inside a
// row tile joins all its parts, one warp per row.
template <typename T, int D, int ROWS, int KEYS>
__global__ void __launch_bounds__(128) tree_join_kernel(const TreeParams p) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long per = *p.share;
  const long long total = p.seq_base[p.num_seqs];
  const long long x = per * (blockIdx.x + 1);
  if (x >= total) return;
  // the sequence of item x: the last with seq_base <= x (empty ones share a
  // base with the next and are passed over)
  int lo = 0, hi = p.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.seq_base[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  const int b = lo;
  const Seq s = seq_of<ROWS, KEYS>(p, b, false);
  if (s.key_tiles == 0) return;
  const long long at = x - p.seq_base[b];
  const long long pair = at / s.key_tiles;
  const long long first = p.seq_base[b] + pair * s.key_tiles, last = first + s.key_tiles - 1;
  const int c0 = static_cast<int>(first / per), c1 = static_cast<int>(last / per);
  if (first == x || c0 != static_cast<int>(blockIdx.x)) return;
  const int h = static_cast<int>(pair / s.row_tiles);
  const int row0 = static_cast<int>(pair - static_cast<long long>(h) * s.row_tiles) * ROWS;
  const int r = blockIdx.y * 4 + warp;
  if (row0 + r >= s.n * p.G) return;
  constexpr int DPL = D / 32;
  float mx = -FLT_MAX;
  for (int c = c0 + lane; c <= c1; c += 32)
    mx = fmaxf(mx, p.part_ml[((static_cast<long long>(c) * 2 + (c == c0)) * ROWS + r) * 2]);
  mx = warp_max(mx);
  float acc[DPL], l = 0.f;
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const long long pr = (static_cast<long long>(c) * 2 + (c == c0)) * ROWS + r;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + pr * 2);
    const float w = exp2f(ml.x - mx);
    l += w * ml.y;
    const float* o = p.part + pr * D + lane * DPL;
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[i] += w * o[i];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int row = row0 + r;
  T* dst = static_cast<T*>(p.out) + (static_cast<long long>(s.q0 + row / p.G) * p.Hq + h * p.G + row % p.G) * D +
           lane * DPL;
#pragma unroll
  for (int i = 0; i < DPL; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack2<T>(acc[i] * inv, acc[i + 1] * inv);
}

// ------------------------------------------------------------------- host --
struct Plan {
  int rows, keys, ctas, min_share;
  size_t bytes;
};

Plan plan_for(int num_seqs, int max_q_len, int max_ctx, int Hq, int Hkv, int D) {
  Plan pl{};
  pl.rows = kRows;
  pl.keys = kKeys;
  pl.min_share = 4;
  const long long rt = (static_cast<long long>(max_q_len) * (Hq / Hkv) + pl.rows - 1) / pl.rows;
  const long long kt = (static_cast<long long>(max_ctx) + pl.keys - 1) / pl.keys;
  const double items = static_cast<double>(num_seqs) * Hkv * rt * kt;
  long long ctas = 148 * 2;
  const double most = (items + pl.min_share - 1) / pl.min_share;
  if (most < ctas) ctas = static_cast<long long>(most);
  if (ctas < 1) ctas = 1;
  pl.ctas = static_cast<int>(ctas);
  const size_t parts = static_cast<size_t>(pl.ctas) * 2 * pl.rows;
  pl.bytes = 256 + parts * (D + 2) * sizeof(float) + (static_cast<size_t>(num_seqs) + 2) * sizeof(long long);
  return pl;
}

template <typename T, int D>
int launch_mma(TreeParams& p, cudaStream_t s) {
  auto kern = tree_mma_kernel<T, D>;
  const int smem = kStages * 2 * kKeys * D * 2;
  static std::atomic<uint64_t> done{0};
  if (!ps_host::reserve_smem(reinterpret_cast<const void*>(kern), smem, &done)) {
    ps_host::set_error("tree_attention: cannot reserve %d bytes of shared memory", smem);
    return PS_ERR_CUDA;
  }
  ps_host::launch(kern, p.num_ctas, kThreads, smem, s, p);
  ps_host::count_launch();
  int rc = ps_host::check_launch("tree_attention");
  if (rc != PS_OK || p.num_ctas == 1) return rc;
  auto join = tree_join_kernel<T, D, kRows, kKeys>;
  ps_host::launch(join, dim3(p.num_ctas - 1, kRows / 4), 128, 0, s, p);
  ps_host::count_launch();
  return ps_host::check_launch("tree_attention(join)");
}

}  // namespace

extern "C" {

size_t ps_tree_attention_workspace_size(int num_seqs, int max_q_len, int max_ctx, int Hq, int Hkv, int D) {
  if (num_seqs <= 0 || max_q_len <= 0 || max_q_len > kMaxNodes || max_ctx < max_q_len || Hq <= 0 || Hkv <= 0 ||
      Hq % Hkv != 0 || (D != 64 && D != 128))
    return 0;
  return plan_for(num_seqs, max_q_len, max_ctx, Hq, Hkv, D).bytes;
}

int ps_tree_attention(void* out, const void* q, const void* k_cache, const void* v_cache, const int32_t* tables,
                      int max_blocks, const int32_t* cu_q, const int32_t* start_pos, const int64_t* tree_mask,
                      int num_seqs, int total_q, int max_q_len, int max_ctx, int num_blocks, int block_size, int Hq,
                      int Hkv, int D, int dtype, void* workspace, size_t workspace_bytes, ps_stream_t stream) {
  if (num_seqs <= 0 || total_q < 0 || max_q_len <= 0 || max_ctx < max_q_len || block_size <= 0 || num_blocks <= 0 ||
      max_blocks <= 0 || Hq <= 0 || Hkv <= 0) {
    ps_host::set_error("tree_attention: invalid sizes (seqs %d, max_q %d, max_ctx %d)", num_seqs, max_q_len, max_ctx);
    return PS_ERR_INVALID;
  }
  if (Hq % Hkv != 0) {
    ps_host::set_error("tree_attention: %d q heads not divisible by %d kv heads", Hq, Hkv);
    return PS_ERR_INVALID;
  }
  if (max_q_len > kMaxNodes) {
    ps_host::set_error("tree_attention: trees of up to %d nodes per request (max_q_len %d)", kMaxNodes, max_q_len);
    return PS_ERR_UNSUPPORTED;
  }
  if (max_ctx > static_cast<long long>(max_blocks) * block_size) {
    ps_host::set_error("tree_attention: context %d needs %lld table entries, table has %d", max_ctx,
                       (static_cast<long long>(max_ctx) + block_size - 1) / block_size, max_blocks);
    return PS_ERR_INDEX;
  }
  if (max_ctx > INT32_MAX - 256) {
    ps_host::set_error("tree_attention: context %d too long", max_ctx);
    return PS_ERR_UNSUPPORTED;
  }
  if (total_q == 0) return PS_OK;
  if (!out || !q || !k_cache || !v_cache || !tables || !cu_q || !start_pos || !tree_mask) {
    ps_host::set_error("tree_attention: null pointer");
    return PS_ERR_INVALID;
  }
  if (!ps_host::aligned(k_cache, 16) || !ps_host::aligned(v_cache, 16) || !ps_host::aligned(q, 16) ||
      !ps_host::aligned(out, 16) || !ps_host::aligned(workspace, 16)) {
    ps_host::set_error("tree_attention: q, out, the caches and the workspace need 16-byte alignment");
    return PS_ERR_INVALID;
  }
  if (D != 64 && D != 128) {
    ps_host::set_error("tree_attention: head_dim %d unsupported (64, 128)", D);
    return PS_ERR_UNSUPPORTED;
  }
  if (dtype != PS_BF16 && dtype != PS_F16) {
    ps_host::set_error("tree_attention: dtype must be bf16 or f16");
    return PS_ERR_UNSUPPORTED;
  }
  const Plan pl = plan_for(num_seqs, max_q_len, max_ctx, Hq, Hkv, D);
  if (!workspace || workspace_bytes < pl.bytes) {
    ps_host::set_error("tree_attention: workspace of %zu bytes needed, %zu given", pl.bytes, workspace_bytes);
    return PS_ERR_INVALID;
  }
  TreeParams p{};
  p.out = out;
  p.q = q;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.tables = tables;
  p.cu_q = cu_q;
  p.start_pos = start_pos;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  const uintptr_t w = (reinterpret_cast<uintptr_t>(workspace) + 127) & ~static_cast<uintptr_t>(127);
  const size_t parts = static_cast<size_t>(pl.ctas) * 2 * pl.rows;
  p.part = reinterpret_cast<float*>(w);
  p.part_ml = p.part + parts * D;
  p.seq_base = reinterpret_cast<long long*>(p.part_ml + parts * 2);
  p.share = p.seq_base + num_seqs + 1;
  p.status = ps_host::status_word(PS_TU_TREE);
  p.total_q = total_q;
  p.words = (max_q_len + 63) / 64;
  p.max_blocks = max_blocks;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.max_q_len = max_q_len;
  p.max_ctx = max_ctx;
  p.num_seqs = num_seqs;
  p.num_ctas = pl.ctas;
  p.min_share = pl.min_share;
  p.scale_log2 = (1.0f / sqrtf(static_cast<float>(D))) * kLog2e;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == PS_BF16)
    return D == 128 ? launch_mma<__nv_bfloat16, 128>(p, s) : launch_mma<__nv_bfloat16, 64>(p, s);
  return D == 128 ? launch_mma<__half, 128>(p, s) : launch_mma<__half, 64>(p, s);
}

}  // extern "C"
