// Attention of a tree of drafted tokens over the paged cache: node i of request
// b sees the request's cached keys [0, start) and the drafted nodes whose bit
// is set in its mask row (itself and its ancestors),
//   o_i = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j,  0 where it sees nothing
// (engine/paged_attention.py:16-50, 82-99, 117-132 with the causal rule of the
// new tokens replaced by the tree's).
//
// Rows are (node, q head of the kv head's group) pairs, row r = node * G + g,
// so that a K/V tile is read once for the whole group. The work of a call is
// the list of (sequence, kv head, row group, key tile) in that order; its length
// is known on the device only, and each CTA takes an equal, contiguous share of
// it. A row group whose key tiles fall into several shares leaves (o, max, sum)
// partials in the workspace (at most two per CTA, whatever the contexts), and
// a second kernel joins them in order: no atomics, the same bits every time.
//
// What a node does not see does not reach it, NaN and infinities included:
// masked scores are replaced before the softmax, rows past the context are
// zero-filled, and a drafted V row with a value that is not finite is cleared
// from the tile and given back only to the rows that see it. What a node does
// see reaches it with a weight above 0, so an infinity is one in the output too:
// rounded or scaled to 0 a weight would make NaN of it (0 * inf). A row whose
// output is not finite although its sum is has its V columns looked at again
// (OddColumns).
#include <cfloat>
#include <climits>
#include <cstdlib>

#include "tc_ptx.cuh"

namespace {

using namespace ps;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxNodes = 256;

struct Part {  // the split row group whose later part (slot 0) a CTA holds; c0 < 0: none
  int q0, h, row0, rows, c0, c1;  // rows to store; CTAs c0 (slot 1) .. c1 (slot 0) hold its parts
  int pad[2];
};

struct TreeParams {
  void* out;
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const int32_t* tables;
  const int32_t* cu_q;
  const int32_t* start_pos;
  const unsigned long long* mask;
  float* part;     // [CTA][2 slots][D / 8][group_rows][8] of o
  float* part_ml;  // [CTA][2 slots][group_rows][2] of (max, sum)
  Part* parts;     // [CTA]
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
  int never_cut;   // by the call's bounds no row group is cut: there is nothing to join
  int group_rows;  // query rows per work item
  uint32_t rg_mul, rg_add, rg_magic, rg_shift;  // row groups of n nodes: ((n * mul + add) * magic) >> shift
  int box_shift;   // log2 of the keys per TMA box
  int block_shift; // log2 of the block size, or -1
  int out32;       // out is 32-byte aligned
  float scale_log2;
};

// ------------------------------------------------------- division of work --
// The work items of sequence b are (kv head, row group, key tile), key tile
// fastest; the host has checked that a call's items fit 31 bits.
struct Seq {
  int q0, n, start, row_groups, key_tiles;
  PS_DEVICE int items(int Hkv) const { return Hkv * row_groups * key_tiles; }
};

// From the raw lengths; a sequence that breaks the call's bounds has no work.
template <int KEYS>
PS_DEVICE Seq make_seq(const TreeParams& p, int q0, int q1, int start, bool* bad) {
  Seq s;
  s.q0 = q0;
  s.start = start;
  const long long n = static_cast<long long>(q1) - q0;  // of any 32-bit numbers
  const long long ctx = start + n;
  *bad = n != 0 && (n < 0 || n > p.max_q_len || q0 < 0 || q1 > p.total_q || start < 0 || ctx > p.max_ctx);
  s.n = *bad ? 0 : static_cast<int>(n);
  s.row_groups = ((s.n * p.rg_mul + p.rg_add) * p.rg_magic) >> p.rg_shift;
  s.key_tiles = s.n ? (static_cast<int>(ctx) + KEYS - 1) / KEYS : 0;
  return s;
}
template <int KEYS>
PS_DEVICE Seq seq_of(const TreeParams& p, int b) {
  bool bad;
  return make_seq<KEYS>(p, p.cu_q[b], p.cu_q[b + 1], p.start_pos[b], &bad);
}

// A CTA's share of the work, as segments (one row group's key tiles). Equal
// shares cut row groups, which then have to be joined; where whole row groups,
// an equal number per CTA, take at most kJoinCost key tiles longer, they are not
// cut (64 sequences x 2 heads at equal contexts: 17 key tiles per CTA against 15
// and a joining of about 6 us; a key tile takes 1.3 us; that case has doubled rows,
// and the bound serves the other forms too, unmeasured there). A share may be a single
// key tile: of at least 4, one request of 64 nodes at context 2000 (16 / 2 heads)
// took 15.3 us instead of 12.9, four of up to 40 nodes at 300 to 2000 20.9 instead
// of 15.4.
constexpr int kJoinCost = 4;

struct Cut {  // one segment
  int b, q0, n, start;   // sequence, its first row, nodes and context
  int h, row0, rows;     // kv head, rows [row0, row0 + rows) of the (node, head) rows
  int tile0, nt, whole;  // key tiles [tile0, tile0 + nt); all of them
};

template <int KEYS>
struct Share {
  int quota, unit, per, b, pair, tile0;  // quota: row groups (unit 1) or key tiles (unit 0) left
  Seq s;

  // By one whole warp; `kept` is shared memory for the sequences' sizes between
  // the sums and the search (of the first `room`; the others are read again).
  PS_DEVICE void find(const TreeParams& p, int lane, Seq* kept, int room) {
    int total = 0, groups = 0, longest = 0;
    bool any_bad = false;
#pragma unroll 1
    for (int b0 = lane; b0 < p.num_seqs; b0 += 128) {  // the loads of 128 sequences are out at once
      int q0[4], q1[4], st[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(b0 + 32 * u, p.num_seqs - 1);
        q0[u] = p.cu_q[i];
        q1[u] = p.cu_q[i + 1];
        st[u] = p.start_pos[i];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = b0 + 32 * u;
        if (i >= p.num_seqs) break;
        bool bad;
        const Seq q = make_seq<KEYS>(p, q0[u], q1[u], st[u], &bad);
        if (i < room) kept[i] = q;
        groups += p.Hkv * q.row_groups;
        total += q.items(p.Hkv);
        longest = max(longest, q.key_tiles);
        any_bad |= bad;
      }
    }
    if (any_bad && blockIdx.x == 0) record_error(p.status, kErrShape);
    total = __reduce_add_sync(0xffffffffu, total);
    groups = __reduce_add_sync(0xffffffffu, groups);
    longest = __reduce_max_sync(0xffffffffu, longest);
    per = max((total + p.num_ctas - 1) / p.num_ctas, 1);
    const int whole = (groups + p.num_ctas - 1) / p.num_ctas;
    unit = static_cast<long long>(whole) * longest <= per + kJoinCost;
    const long long lo = static_cast<long long>(unit ? whole : per) * blockIdx.x;
    const int all = unit ? groups : total;
    const int begin = static_cast<int>(lo < all ? lo : all);
    quota = min(unit ? whole : per, all - begin);
    if (quota <= 0) return;
    __syncwarp();
    int run = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.num_seqs; b0 += 32) {
      const int i = b0 + lane;
      Seq q{};
      if (i < p.num_seqs) q = i < room ? kept[i] : seq_of<KEYS>(p, i);
      const int n = unit ? p.Hkv * q.row_groups : q.items(p.Hkv);
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const int first = run + incl - n;
      const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && begin >= first && begin < first + n);
      if (hit) {
        const int src = __ffs(hit) - 1;
        b = b0 + src;
        pair = begin - __shfl_sync(0xffffffffu, first, src);  // items for now
        s.q0 = __shfl_sync(0xffffffffu, q.q0, src);
        s.n = __shfl_sync(0xffffffffu, q.n, src);
        s.start = __shfl_sync(0xffffffffu, q.start, src);
        s.row_groups = __shfl_sync(0xffffffffu, q.row_groups, src);
        s.key_tiles = __shfl_sync(0xffffffffu, q.key_tiles, src);
        break;
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    tile0 = 0;
    if (!unit) {
      const int items = pair;
      pair = items / s.key_tiles;
      tile0 = items - pair * s.key_tiles;
    }
  }

  PS_DEVICE bool next(const TreeParams& p, Cut& c) {
    if (quota <= 0) return false;
    while (pair >= p.Hkv * s.row_groups) {  // the next sequence with work
      s = seq_of<KEYS>(p, ++b);
      pair = 0;
    }
    c.b = b;
    c.q0 = s.q0;
    c.n = s.n;
    c.start = s.start;
    c.h = pair / s.row_groups;
    c.row0 = (pair - c.h * s.row_groups) * p.group_rows;
    c.rows = min(p.group_rows, s.n * p.G - c.row0);
    c.tile0 = tile0;
    c.nt = unit ? s.key_tiles : min(s.key_tiles - tile0, quota);
    c.whole = c.nt == s.key_tiles;
    quota -= unit ? 1 : c.nt;
    tile0 += c.nt;
    if (tile0 == s.key_tiles) {
      tile0 = 0;
      ++pair;
    }
    return true;
  }
  // Where the parts of a cut row group lie that began in an earlier CTA (c.tile0 > 0)
  PS_DEVICE Part part(const Cut& c) const {
    const int first = per * static_cast<int>(blockIdx.x) - c.tile0;  // the row group's first item
    return Part{c.q0, c.h, c.row0, c.rows, first / per, (first + s.key_tiles - 1) / per, {0, 0}};
  }
};
// a row group's first part is the last segment of its CTA, the others the first
PS_DEVICE int part_slot(const Cut& c) { return c.tile0 > 0 ? 0 : 1; }
// Partial o of (CTA, slot): 8-column chunks of all rows, so that a warp whose
// lanes hold a row each writes whole lines.
PS_DEVICE float* part_o(const TreeParams& p, int cta, int slot, int row, int chunk, int D) {
  return p.part + (static_cast<long long>(cta * 2 + slot) * (D / 8) + chunk) * p.group_rows * 8 + row * 8;
}
PS_DEVICE float2* part_ml(const TreeParams& p, int cta, int slot, int row) {
  return reinterpret_cast<float2*>(p.part_ml) + static_cast<long long>(cta * 2 + slot) * p.group_rows + row;
}

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

// Clears the values of 8 that are not finite; true if there were any.
template <typename T>
PS_DEVICE bool clear_odd(uint4& x) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&x);
  bool hit = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = (w[i] & kExp) == kExp, hi = (w[i] & (kExp << 16)) == (kExp << 16);
    hit |= lo | hi;
    if (lo) w[i] &= 0xFFFF0000u;
    if (hi) w[i] &= 0x0000FFFFu;
  }
  return hit;
}

// Which of a thread's N columns of V have values that are not finite in the rows
// that a query row sees, and what their sum is: with weights above 0 and a finite
// rest the output's value. Only looked for where a tile or an output has shown
// such a value.
// Cached keys are seen by all rows alike, so a warp's lanes share them out: with
// an infinity in every request 128 x 16 nodes at 4096 take 2.3 ms (0.39 without;
// 131 when each lane went over all keys).
struct OddColumns {
  unsigned long long plus = 0, minus = 0, nan = 0;
  template <typename T>
  PS_DEVICE void add(int column, uint16_t x) {
    if (finite16<T>(x)) return;
    const unsigned long long bit = 1ull << column;
    if (x & (std::is_same<T, __half>::value ? 0x03FF : 0x007F)) nan |= bit;
    else if (x & 0x8000) minus |= bit;
    else plus |= bit;
  }
  template <typename T>
  PS_DEVICE void add2(int column, uint32_t x) {
    add<T>(column, static_cast<uint16_t>(x));
    add<T>(column + 1, static_cast<uint16_t>(x >> 16));
  }
  // of the lanes that differ in the bits of `lanes`
  PS_DEVICE void join(int lanes) {
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      if (!(lanes & o)) continue;
      plus |= __shfl_xor_sync(0xffffffffu, plus, o);
      minus |= __shfl_xor_sync(0xffffffffu, minus, o);
      nan |= __shfl_xor_sync(0xffffffffu, nan, o);
    }
  }
  PS_DEVICE bool any(int column) const { return ((plus | minus | nan) >> column) & 1; }
  PS_DEVICE float value(int column) const {
    if (((nan | (plus & minus)) >> column) & 1) return NAN;
    return (plus >> column) & 1 ? INFINITY : -INFINITY;
  }
};
// A finite sum of weights: the row's scores are in order, and a value of its
// output that is not finite comes from V.
PS_DEVICE bool finite_sum(float l) { return fabsf(l) <= FLT_MAX; }

// --------------------------------------------------------- mma.sync kernel --
// Any block size and group: 64 rows per CTA (16 per warp), 64-key tiles through a
// 3-stage ring of 16-byte cp.async. Bound by its copies' addresses and the MMA
// chain of four warps: with blocks of 8, which both kernels can read, 64 requests
// x 8 nodes at 2048 took 85 us (tcgen05: 46, cold L2) and 128 x 16 nodes at 4096
// with 40 heads 1694 us (370), so it has only what the other cannot take.
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
  __shared__ Share<kKeys> s_share;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    Share<kKeys> sh;
    sh.find(p, lane, reinterpret_cast<Seq*>(smem), kStages * 2 * kTile / static_cast<int>(sizeof(Seq)));
    if (lane == 0) {
      s_share = sh;
      p.parts[blockIdx.x].c0 = -1;
    }
  }
  __syncthreads();
  Share<kKeys> share = s_share;
  Cut sg;
  const uint32_t base = smem_u32(smem);
  const int mat = lane >> 3;
  while (share.next(p, sg)) {
    const int ctx = sg.start + sg.n;
    const int R = sg.n * p.G;
    const int32_t* table = p.tables + static_cast<long long>(sg.b) * p.max_blocks;
    const int ntiles = sg.nt;
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
          (static_cast<long long>(sg.q0 + (ok ? r / p.G : 0)) * p.Hq + sg.h * p.G + (ok ? r % p.G : 0)) * D);
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
      const bool tail = t0 + kKeys > sg.start;  // drafted keys (or the end) in this tile
      if (tail) {
        // clear drafted V values that are not finite: 0 * inf would reach rows that do not see them
        bool bad = false;
        uint16_t* vt = reinterpret_cast<uint16_t*>(smem + (vs - base));
        for (int i = threadIdx.x; i < kKeys * D; i += kThreads) {
          const int r = i / D, c = i % D;
          if (t0 + r < sg.start || t0 + r >= ctx) continue;
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
                                 : seen64(p.mask + static_cast<long long>(sg.q0 + node[hf]) * p.words, p.words,
                                          t0 - sg.start, sg.n);
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
      // P is rounded to the cache's type for the matrix unit: relative 2^-8
      // (bf16) or 2^-11 (f16) a term, as the rounding of the output
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
    bool in_order[2], all = false;  // rows whose outputs are to be finite; one is not
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      in_order[hf] = node[hf] >= 0 && finite_sum(l[hf]);
      float zero = 0.f;  // NaN if a value of this row is not finite
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) zero = fmaf(o[i][2 * hf + e], 0.f, zero);
      all |= in_order[hf] && zero != 0.f;
    }
    all = __any_sync(0xffffffffu, all);
    if (odd_values || all) {
      const int k1 = min((sg.tile0 + sg.nt) * kKeys, ctx);
      auto add_key = [&](OddColumns& odd, int key) {
        const int phys = table[key / p.block_size];
        if (phys < 0 || phys >= p.num_blocks) return;
        const T* vr = static_cast<const T*>(p.v_cache) +
                      ((static_cast<long long>(phys) * p.block_size + key % p.block_size) * p.Hkv + sg.h) * D +
                      2 * (lane & 3);
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) odd.add2<T>(2 * i, *reinterpret_cast<const uint32_t*>(vr + i * 8));
      };
      OddColumns cached;
      if (all) {
#pragma unroll 1
        for (int key = first_key + (lane >> 2); key < min(k1, sg.start); key += 8) add_key(cached, key);
        __syncwarp();
        cached.join(4 + 8 + 16);
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        if (!in_order[hf]) continue;
        const unsigned long long* mrow = p.mask + static_cast<long long>(sg.q0 + node[hf]) * p.words;
        OddColumns odd = cached;
#pragma unroll 1
        for (int key = max(first_key, sg.start); key < k1; ++key) {
          const int jn = key - sg.start;
          if ((mrow[jn >> 6] >> (jn & 63)) & 1) add_key(odd, key);
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (odd.any(2 * i + e)) o[i][2 * hf + e] = odd.value(2 * i + e);
      }
    }
    const int slot = part_slot(sg);
    if (sg.tile0 > 0 && threadIdx.x == 0) p.parts[blockIdx.x] = share.part(sg);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = wrow + (lane >> 2) + hf * 8;
      if (r >= R) continue;
      if (sg.whole) {
        const float inv = l[hf] == 0.f ? 0.f : 1.f / l[hf];
        T* dst = static_cast<T*>(p.out) +
                 (static_cast<long long>(sg.q0 + r / p.G) * p.Hq + sg.h * p.G + r % p.G) * D + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<uint32_t*>(dst + i * 8) = pack2<T>(o[i][2 * hf] * inv, o[i][2 * hf + 1] * inv);
      } else {
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<float2*>(part_o(p, blockIdx.x, slot, r - sg.row0, i, D) + 2 * (lane & 3)) =
              make_float2(o[i][2 * hf], o[i][2 * hf + 1]);
        if ((lane & 3) == 0) *part_ml(p, blockIdx.x, slot, r - sg.row0) = make_float2(m[hf], l[hf]);
      }
    }
  }
}

// ----------------------------------------------------------- tcgen05 kernel --
// Block sizes of whole 8-key groups (the serving layouts). One CTA per SM, 128
// query rows, 128-key tiles:
//   warps 0, 3 TMA producers of K and of V: tiles go through one ring of equal
//              slots in the order that the MMAs read them (K0 K1 V0 K2 V1 ...),
//              as boxes of up to 128 keys of one block, one lane a box; keys past
//              the context or outside the pool are loads past the end of the tensor,
//              which fill zeros. A warp issues boxes at a bounded rate (2 KB ones
//              alone streamed 4.9 TB/s from HBM with one warp, 5.95 with two), so
//              a box carries both 64-dim panels of its keys
//   warp 2     walks the CTA's share and hands its segments to the other roles
//   warp 1     TMEM, the Q tile (128 / G nodes x the G heads of the group, one box
//              per 64 dims) and the MMAs: S_w = Q K_j^T (both operands in shared
//              memory), O += P_w V_j (P from TMEM, V read MN-major), all by one thread
//   warps 4-11 softmax, two threads per row (DUP: four): warps 4-7 the first 64
//              keys of a tile, warps 8-11 the others; a pair of warps exchanges its
//              rows' maxima, so that both halves of P refer to the same one
// Step t is a key tile: QK(t), softmax(t), PV(t). The MMA thread issues PV(t)
// QK(t + 2) under softmax(t + 1), with one commit: what a commit costs the pipe is
// about one MMA, so ring slots are given back by a softmax thread, for which S(t)
// complete says that K of step t and V of step t - 2 have been read (MMAs complete
// in order).
// A step lasts about 2300 clocks of the softmax warps (200 the largest scores, 200
// their exchange, 1430 exponentials and P, of which the special-function unit
// takes 1024), under which lie 1420 of the matrix unit. One thread per row and
// two groups of warps on alternate steps took 2500; looking for step t + 1's
// largest scores under step t's exponentials was no faster, for S(t + 1) is not
// there yet. Two row tiles that share each loaded key tile (128 x 2 rows, two O)
// were slower wherever they applied, for the partials of cut row groups doubled:
// 8 requests of up to 64 nodes 32.7 against 27.2 us, one of 33 nodes at context
// 32717 63.1 against 58.4, 64 of up to 64 nodes at 4096 148 against 138; the
// second reader of a key tile finds it in L2.
// DUP: calls whose row groups have at most 64 rows by their bounds load them into
// both halves of the tile, lanes r and r + 64. Of every 64 keys lane r's P has the
// first 32 and zeros, lane r + 64's the others: four threads per row, each with a
// quarter of its keys. The two lanes are two shares of the softmax with a maximum,
// a sum and an O each, joined when the row group's keys are done. One node at
// context 128: 9.0 -> 8.3 us, 5 requests x 7 nodes 10.6 -> 9.5, 64 x 8 nodes at 2048
// 35.6 -> 33.6 (copies of K and V alone at this pattern and these CTAs: within 10%).
// A softmax thread reads its scores from TMEM 32 at a time: holding them would
// need more than the 168 registers that 12 warps leave a thread.
// TMEM: S0 | S1 | O, 128 columns each; the halves of P overwrite the first 32
// columns of the halves of S.
// The ring and the barriers run on over the segments of a CTA's share: the next
// segment's tiles load while the last one's output is stored.
constexpr int kTcRows = 128;
constexpr int kTcKeys = 128;
constexpr int kTcThreads = 384;
constexpr int kTcCtas = 148;

template <int D, bool DUP>
struct Tc {
  static constexpr int kPanels = D / 64;                // 64-column panels of 128 rows x 128 bytes
  static constexpr int kGroup = kPanels * 1024;         // 8 keys of a K or V tile: panel after panel
  static constexpr int kSlot = kTcKeys * D * 2;         // one K or V tile
  static constexpr int kQ = kTcRows * D * 2;
  static constexpr int kQs = DUP ? 2 * kQ : kQ;         // (and what DUP's lanes exchange)
  static constexpr int kSlots = (224 * 1024 - kQs) / kSlot;  // 5 or 6 (D = 128), 12 or 13 (D = 64)
  static constexpr int kSmem = kQs + kSlots * kSlot + 3 * 1024 /* barriers, (max, sum), flags */;
};

// 128B-swizzled descriptor of a K or V tile: groups of 8 keys sbo bytes apart,
// panels of 64 dims (read MN-major) lbo bytes.
PS_DEVICE uint64_t tile_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | static_cast<uint64_t>(lbo >> 4) << 16 |
         static_cast<uint64_t>(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// B read MN-major ([k][n] rows of the V tile)
__host__ __device__ constexpr uint32_t idesc_bmn(bool bf16, int m, int n) {
  return instr_desc(bf16, m, n) | (1u << 16);
}

PS_DEVICE void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int group, int head) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %3, %4, %5}], "
      "[%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(group), "r"(head)
      : "memory");
}
PS_DEVICE void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// 32 columns of this warp's lanes, not waited for (tmem_ready orders the uses)
PS_DEVICE void tmem_ld32_issue(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
PS_DEVICE void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
PS_DEVICE void tmem_ready(float* v) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));
}
PS_DEVICE void st_global_32(void* p, const uint32_t* v) {  // 32 bytes, 32-byte aligned
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
PS_DEVICE float ex2_approx(float x) {  // relative error about 2^-22, 0 for -inf; far below P's rounding to 16 bits
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in one register pair, for the packed FMA pipe.
typedef unsigned long long f32x2;
PS_DEVICE f32x2 pack_f2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
PS_DEVICE void unpack_f2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
PS_DEVICE f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
PS_DEVICE f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
PS_DEVICE float max3_nan(float a, float b, float c) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The max that P, O and the sum refer to stays until a row's scores pass it by
// more than kSlack (log2): P <= 2^8 is well inside the 16-bit types. The new one
// is rounded up, so that O and the sum are scaled by a power of two, exactly.
constexpr float kSlack = 8.f;
// 2^-up for a whole number up >= 0 (0 when it is tiny, NaN when up is).
PS_DEVICE float pow2_down(float up) {
  return up <= 126.f ? __uint_as_float(static_cast<uint32_t>(127.f - up) << 23) : (up != up ? NAN : 0.f);
}
// n x 32 columns of this thread's O row times alpha.
PS_DEVICE void scale_o(uint32_t t_o, int n, float alpha) {
#pragma unroll 1
  for (int c = 0; c < n; ++c) {
    float v[32];
    tmem_ld32(t_o + c * 32, v);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= alpha;
    tmem_st16(t_o + c * 32, reinterpret_cast<const uint32_t*>(v));
    tmem_st16(t_o + c * 32 + 16, reinterpret_cast<const uint32_t*>(v) + 16);
  }
  tmem_wait_st();
}

// The largest of N of this thread's scores (in the log2 domain; NaN if one is).
// TAIL: bit i of v1:v0 says that the row sees key i.
template <int N, bool TAIL>
PS_DEVICE float top_score(uint32_t t_s, uint32_t v0, uint32_t v1, float scale) {
  float sv[N];
#pragma unroll
  for (int c = 0; c < N; c += 32) tmem_ld32_issue(t_s + c, sv + c);
  tmem_wait_ld();
#pragma unroll
  for (int c = 0; c < N; c += 32) tmem_ready(sv + c);
  auto seen = [&](int i) { return !TAIL || (((i < 32 ? v0 : v1) >> (i & 31)) & 1); };
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < N; i += 2)
    mx[(i >> 1) & 3] =
        max3_nan(mx[(i >> 1) & 3], seen(i) ? sv[i] : -INFINITY, seen(i + 1) ? sv[i + 1] : -INFINITY);
  return max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * scale;
}
// N of this thread's scores become P against the row's reference max, 32 at a time
// (16-bit columns 16 c .. lie below the scores still to be read); returns the sum
// of P. The loop stays rolled: longer bodies ran slower, from beyond the
// first-level instruction cache. (Taking 3 of 8 exponentials to the FMA pipe by a
// polynomial was no faster: the loop is bound by latency and issue, not by the
// special-function unit.)
template <typename T, int N, bool TAIL>
PS_DEVICE float softmax_part(uint32_t t_s, uint32_t t_p, uint32_t v0, uint32_t v1, float scale, float m_ref) {
  float sv[32];
  f32x2 sum[4] = {0, 0, 0, 0};
  const f32x2 scale2 = pack_f2(scale, scale), neg_m = pack_f2(-m_ref, -m_ref);
  tmem_ld32_issue(t_s, sv);
#pragma unroll 1
  for (int c = 0; c < N / 32; ++c) {
    const uint32_t vc = c ? v1 : v0;
    auto seen = [&](int i) { return !TAIL || ((vc >> i) & 1); };
    tmem_wait_ld();
    tmem_ready(sv);
    f32x2 x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = fma2(pack_f2(sv[2 * i], sv[2 * i + 1]), scale2, neg_m);
    if (N > 32 && c == 0) tmem_ld32_issue(t_s + 32, sv);  // under this group's exponentials
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x0, x1;
      unpack_f2(x[i], x0, x1);
      float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
      if (TAIL) {
        p0 = seen(2 * i) ? p0 : 0.f;
        p1 = seen(2 * i + 1) ? p1 : 0.f;
      }
      sum[i & 3] = add2(sum[i & 3], pack_f2(p0, p1));  // four chains: one would bound the loop by its latency
      // P rounded to 16 bits for the matrix unit: 2^-8 (bf16) or 2^-11 (f16) of a
      // term, as the output's own rounding
      pk[i] = pack2<T>(p0, p1);
    }
    tmem_st16(t_p + c * 16, pk);
  }
  float s0, s1;
  unpack_f2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
  return s0 + s1;
}

// A position of a ring of N slots: slot and phase parity.
template <int N>
struct Slot {
  int i;
  uint32_t phase;
  PS_DEVICE void advance(int n) {
    i += n;
    if (i >= 2 * N) {  // n may be a segment's whole length
      const int turns = i / N;
      i -= turns * N;
      phase ^= turns & 1;
    } else if (i >= N) {
      i -= N;
      phase ^= 1;
    }
  }
};

// After a wait gave up: let the copies or MMAs in flight end (bounded too).
PS_DEVICE void drain_wait(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - t0 < kWaitCycles) {
  }
}

// Order of a segment's loads, K_j and V_j among its 2 * nt tiles: as the MMAs
// read them, QK two steps ahead of PV.
PS_DEVICE int k_pos(int j) { return j < 2 ? j : 2 * j - 1; }
PS_DEVICE int v_pos(int j, int nt) { return min(nt, j + 2) + j; }

// A segment as the roles read it.
struct Seg {
  int b, q0, n, start, h, row0, rows, tile0, nt;
  int flags;
};
enum SegFlags : int { kSegStop = 1, kSegWhole = 2 };
constexpr int kSegRing = 4;
constexpr int kSegReaders = 11;  // two producers, the MMA thread, eight softmax warps

PS_DEVICE uint32_t mbar_test(uint32_t bar, uint32_t parity) {  // a try_wait may suspend the thread, this does not
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
// Bounded wait of one thread (see warp_wait).
PS_DEVICE bool thread_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitCycles) {
      *abort_flag = 1;
      record_error(status, kErrTimeout);
      return false;
    }
  }
  return true;
}

template <typename T, int D, bool DUP>
__global__ void __launch_bounds__(kTcThreads, 1) tree_tc_kernel(const __grid_constant__ CUtensorMap qmap,
                                                                const __grid_constant__ CUtensorMap kmap,
                                                                const __grid_constant__ CUtensorMap vmap,
                                                                const TreeParams p) {
  pdl_trigger();
  using C = Tc<D, DUP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kNS = C::kSlots;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t q_sa = smem_u32(smem_raw);
  unsigned char* gbase = smem_raw;
  if (q_sa & 1023) {  // the swizzle needs the declared alignment
    pdl_wait();
    if (threadIdx.x == 0) record_error(p.status, kErrShape);
    return;
  }
  const uint32_t ring = q_sa + C::kQs;
  const uint32_t bars = ring + kNS * C::kSlot;
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (kNS + s); };
  auto s_full = [&](int w) { return bars + 8 * (2 * kNS + w); };
  auto p_full = [&](int w) { return bars + 8 * (2 * kNS + 2 + w); };
  const uint32_t q_full = bars + 8 * (2 * kNS + 4);
  const uint32_t o_free = bars + 8 * (2 * kNS + 5);
  const uint32_t drained = bars + 8 * (2 * kNS + 6);
  auto pair = [&](int quarter) { return bars + 8 * (2 * kNS + 7 + quarter); };
  auto seg_full = [&](int i) { return bars + 8 * (2 * kNS + 11 + i); };
  auto seg_empty = [&](int i) { return bars + 8 * (2 * kNS + 11 + kSegRing + i); };
  auto cross = [&](int i) { return bars + 8 * (2 * kNS + 11 + 2 * kSegRing + i); };
  unsigned char* misc = gbase + C::kQs + kNS * C::kSlot + 8 * (2 * kNS + 14 + 2 * kSegRing);
  float* s_swap = reinterpret_cast<float*>(misc);  // [2][2 halves][128 rows]
  Seg* s_seg = reinterpret_cast<Seg*>(misc + 2 * 128 * 8);  // [kSegRing]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(s_seg + kSegRing);
  volatile int* s_odd = abort_flag + 1;  // [3], by segment mod 3
  uint32_t* tmem_slot = const_cast<uint32_t*>(reinterpret_cast<volatile uint32_t*>(abort_flag + 4));
  volatile uint32_t* s_at = tmem_slot + 1;  // [kNS] the tile last loaded into each slot

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (threadIdx.x == 0) {
    *abort_flag = 0;
    s_odd[0] = s_odd[1] = s_odd[2] = 0;
    for (int s = 0; s < kNS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
      s_at[s] = ~0u;
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(s_full(w), 1);
      mbar_init(p_full(w), 8);
    }
    mbar_init(q_full, 1);
    mbar_init(o_free, 8);
    for (int i = 0; i < 4; ++i) mbar_init(pair(i), 2);
    for (int i = 0; i < 2; ++i) mbar_init(cross(i), 4);
    mbar_init(drained, 1);
    for (int i = 0; i < kSegRing; ++i) {
      mbar_init(seg_full(i), 1);
      mbar_init(seg_empty(i), kSegReaders);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  } else if (threadIdx.x == 96) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qmap)) : "memory");
  }
  pdl_wait();  // barriers, TMEM and descriptors are ready before the kernel ahead ends
  Share<kTcKeys> share;
  if (warp == 2) {
    share.find(p, lane, reinterpret_cast<Seq*>(gbase + C::kQs), kNS * C::kSlot / static_cast<int>(sizeof(Seq)));
    fence_proxy_async();  // the ring is TMA's from here on
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // segment i for a reading warp; false: there is none, or a wait gave up
  auto read_seg = [&](uint32_t i, Seg& sg) {
    if (!warp_wait(seg_full(i % kSegRing), (i / kSegRing) & 1, abort_flag, p.status)) return false;
    sg = s_seg[i % kSegRing];
    __syncwarp();
    if (lane == 0) mbar_arrive(seg_empty(i % kSegRing));
    return !(sg.flags & kSegStop);
  };

  if (warp == 2) {
    // ----------------------------------------------------------- planner --
    if (lane == 0) p.parts[blockIdx.x].c0 = -1;
    bool more = true, ok = true;
    for (uint32_t i = 0; ok && more; ++i) {
      Cut c;
      more = share.next(p, c);
      if (i >= kSegRing) ok = warp_wait(seg_empty(i % kSegRing), ((i / kSegRing) - 1) & 1, abort_flag, p.status);
      if (ok && lane == 0) {
        Seg sg{};
        sg.flags = kSegStop;
        if (more) {
          sg = Seg{c.b, c.q0, c.n, c.start, c.h, c.row0, c.rows, c.tile0, c.nt, 0};
          if (c.whole) sg.flags |= kSegWhole;
          if (c.tile0 > 0) p.parts[blockIdx.x] = share.part(c);
        }
        s_seg[i % kSegRing] = sg;
        mbar_arrive(seg_full(i % kSegRing));
      }
      __syncwarp();
    }
  } else if (warp == 0 || warp == 3) {
    // ---------------------------------------------------- K, V producers --
    const bool is_v = warp == 3;
    const CUtensorMap* map = is_v ? &vmap : &kmap;
    const bool mine = lane < kTcKeys >> p.box_shift;  // this lane's box of a tile
    const int grp = lane;
    const uint32_t dst = ring + ((grp << p.box_shift) >> 3) * C::kGroup;
    const int past = p.num_blocks * p.block_size;  // a row behind the tensor: zeros
    uint32_t at = 0;  // position in the ring
    bool ok = true;
    Seg sg;
    for (uint32_t i = 0; ok && read_seg(i, sg); ++i) {
      const int nt = sg.nt;
      const int ctx = sg.start + sg.n;
      const int32_t* table = p.tables + static_cast<long long>(sg.b) * p.max_blocks;
      // row of this lane's box of tile j
      auto row_of = [&](int j) {
        const int key = (sg.tile0 + j) * kTcKeys + (grp << p.box_shift);
        if (!mine || j >= nt || key >= ctx) return past;
        const int entry = p.block_shift >= 0 ? key >> p.block_shift : key / p.block_size;
        const int phys = table[entry];
        if (phys < 0 || phys >= p.num_blocks) {
          record_error(p.status, kErrBlockId);
          return past;
        }
        return phys * p.block_size + key - entry * p.block_size;
      };
      // Both producers walk all positions of the ring, so that neither is ever
      // two phases away from a slot's barrier; each issues its own tensor's.
      auto turn = [&](bool v, int row) {
        const int s = static_cast<int>(at % kNS);
        if (at >= kNS && !warp_wait(empty(s), ((at / kNS) - 1) & 1, abort_flag, p.status)) {
          ok = false;
          return;
        }
        if (v == is_v) {
          if (lane == 0) {
            mbar_expect_tx(full(s), C::kSlot);
            s_at[s] = at;
          }
          __syncwarp();
          if (mine) tma_load_5d(dst + s * C::kSlot, map, full(s), row >> 3, sg.h);
        }
        ++at;
      };
      // K_0 [K_1] V_0 K_2 V_1 ...; rows are looked up about two tiles ahead of their loads
      int row0 = row_of(0), row1 = row_of(1), row2 = row_of(2);  // of the tiles j, j + 1, j + 2
      turn(false, row0);
      if (ok && nt > 1) turn(false, row1);
      for (int j = 0; ok && j < nt; ++j) {
        const int next = row_of(j + 3);
        turn(true, row0);
        if (ok && j + 2 < nt) turn(false, row2);
        row0 = row1;
        row1 = row2;
        row2 = next;
      }
    }
    if (*abort_flag)
      for (int s = 0; s < kNS; ++s)
        if (s_at[s] != ~0u) drain_wait(full(s), (s_at[s] / kNS) & 1);
  } else if (warp == 1) {
    // --------------------------------------------------------------- MMA --
    if (lane == 0) {
      constexpr uint32_t id_qk = instr_desc(kBf16, 128, kTcKeys);
      constexpr uint32_t id_pv = idesc_bmn(kBf16, 128, D);
      uint32_t seg = 0, q_loads = 0;
      Slot<kNS> base{0, 0};  // the segment's first ring position
      uint32_t tiles[2] = {0, 0};  // P tiles consumed of each group
      bool ok = true;
      Seg nx;
      auto take = [&](uint32_t i) {  // segment i into nx
        if (!thread_wait(seg_full(i % kSegRing), (i / kSegRing) & 1, abort_flag, p.status)) return false;
        nx = s_seg[i % kSegRing];
        mbar_arrive(seg_empty(i % kSegRing));
        return !(nx.flags & kSegStop);
      };
      auto load_q = [&] {  // of nx
        const int node = nx.q0 + nx.row0 / p.G;
        mbar_expect_tx(q_full, (DUP ? 2 : 1) * C::kPanels * p.group_rows * 128);
        for (int i = 0; i < (DUP ? 2 : 1); ++i)
          for (int pn = 0; pn < C::kPanels; ++pn)
            tma_load_3d(q_sa + i * (64 * 128) + pn * (kTcRows * 128), &qmap, q_full, pn * 64, nx.h * p.G, node);
        ++q_loads;
      };
      bool have = take(0);
      if (have) load_q();
      while (ok && have) {
        const int nt = nx.nt;
        ok = thread_wait(q_full, seg & 1, abort_flag, p.status);
        // ring slots of the next K (0 1 3 5 ..) and V (2 4 .., 1 apart at the end)
        Slot<kNS> vs = base, ks = base;
        vs.advance(v_pos(0, nt));
        auto qk = [&](int w) {
          const uint32_t k = ring + ks.i * C::kSlot;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            mma_f16(tmem + w * 128, smem_desc_sw128(q_sa + (kk >> 2) * (kTcRows * 128) + (kk & 3) * 32),
                    tile_desc(k + (kk >> 2) * 1024 + (kk & 3) * 32, 0, C::kGroup), id_qk, kk > 0 ? 1u : 0u);
          }
        };
        for (int t = 0; ok && t < 2; ++t) {
          if (t < nt) {
            ok = thread_wait(full(ks.i), ks.phase, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            qk(t);
            ks.advance(1 + t);
          }
          if (seg == 0) mma_commit(s_full(t));
        }
        if (ok && seg > 0) {
          // The softmax warps are done with the last segment's O and its two last S
          // phases: a commit before that could put a warp two phases behind.
          ok = thread_wait(o_free, (seg - 1) & 1, abort_flag, p.status);
          if (!ok) break;
          mma_commit(s_full(0));
          mma_commit(s_full(1));
        }
#pragma unroll 1
        for (int t = 0; ok && t < nt; ++t) {
          const int w = t & 1;
          const bool more = t + 2 < nt;
          const uint32_t bv = full(vs.i), bk = more ? full(ks.i) : bv, bp = p_full(w), pp = tiles[w] & 1;
          const uint32_t pk = more ? ks.phase : vs.phase;
          // usually all are complete: one round of tests
          if (!(mbar_test(bv, vs.phase) & mbar_test(bk, pk) & mbar_test(bp, pp))) {
            ok = thread_wait(bv, vs.phase, abort_flag, p.status) && thread_wait(bk, pk, abort_flag, p.status) &&
                 thread_wait(bp, pp, abort_flag, p.status);
            if (!ok) break;
          }
          ++tiles[w];
          tc_fence_after();
          const uint32_t v = ring + vs.i * C::kSlot;
          const uint32_t acc = t == 0 ? 0u : 1u;
#pragma unroll
          for (int kk = 0; kk < kTcKeys / 16; ++kk)
            mma_ts(tmem + 256, tmem + w * 128 + (kk >> 2) * 64 + (kk & 3) * 8,
                   tile_desc(v + kk * 2 * C::kGroup, 1024, C::kGroup), id_pv, kk > 0 ? 1u : acc);
          if (more) qk(w);
          mma_commit(s_full(w));  // S(t + 2), and in any case: PV(t) is done
          ks.advance(2);
          vs.advance(t < nt - 2 ? 2 : 1);
        }
        if (!ok) break;
        base.advance(2 * nt);
        ++seg;
        // the last P was there, so every QK of this segment is done with Q
        have = take(seg);
        if (have) load_q();
      }
      if (*abort_flag) {
        mma_commit(drained);
        drain_wait(drained, 0);
        if (q_loads) drain_wait(q_full, (q_loads - 1) & 1);
      }
    }
    __syncwarp();
  } else {
    // ----------------------------------------------------------- softmax --
    const int half = (warp - 4) >> 2;   // which 64 keys of a tile
    const int quarter = warp & 3;
    const int side = DUP ? quarter >> 1 : 0;
    const int t_lane = quarter * 32 + lane;   // this thread's TMEM lane
    const int r = DUP ? t_lane & 63 : t_lane;  // and the row of a tile in it
    const int first_row = r - lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const int r_node = r / p.G, r_head = r - r_node * p.G;
    const bool gives = threadIdx.x == 128;  // gives back the ring slots
    uint32_t seq = 0, swaps = 0, crosses = 0;
    uint32_t phase[2] = {0, 0};  // completed S waits of each buffer before this segment
    bool ok = true;
    // the value of this row's other thread; both warps of a pair make the same calls
    auto swap = [&](float v) {
      float* at = s_swap + (swaps & 1) * 256;
      at[half * 128 + t_lane] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(pair(quarter));
      ok = ok && warp_wait(pair(quarter), swaps & 1, abort_flag, p.status);
      ++swaps;
      return at[(half ^ 1) * 128 + t_lane];
    };
    Seg sg;
    for (uint32_t seg = 0; ok && read_seg(seg, sg); ++seg) {
      const int nt = sg.nt;
      const int n = sg.n, start = sg.start, ctx = start + n;
      const int node = sg.row0 / p.G + r_node;
      const bool row_on = r < sg.rows;
      auto give = [&](uint32_t at) { mbar_arrive(empty(static_cast<int>(at % kNS))); };
      // S(x) complete (x < nt + 2; from nt on: PV(x - 2) alone)
      auto wait_s = [&](int x) {
        return warp_wait(s_full(x & 1), (phase[x & 1] + (x >> 1)) & 1, abort_flag, p.status);
      };
      auto give_of = [&](int x) {  // what S(x) says has been read
        if (!gives) return;
        if (x < nt) give(seq + k_pos(x));
        if (x >= 2) give(seq + v_pos(x - 2, nt));
      };
      // s_odd of the next segment: last read two segments ago, next written after this segment's PVs
      if (gives) s_odd[(seg + 1) % 3] = 0;
      // a row of one mask word is fetched before it is needed
      const bool in_tree = (sg.tile0 + nt) * kTcKeys > start;
      auto mask_row = [&](int node) { return p.mask + static_cast<long long>(sg.q0 + node) * p.words; };
      const unsigned long long mword = in_tree && row_on ? mask_row(node)[0] : 0ull;
      float m_ref = -FLT_MAX, l = 0.f;  // the reference max (log2 domain) and the sum of this row
      for (int t = 0; t < nt; ++t) {
        const int w = t & 1;
        const int key0 = (sg.tile0 + t) * kTcKeys;
        const bool tail = key0 + kTcKeys > start;
        ok = wait_s(t);
        if (!ok) break;
        give_of(t);
        if (tail) {
          // V rows past the context hold anything, and a drafted row's values
          // that are not finite would reach rows that do not see it: clear them.
          // (S(t) is there, so the slot's last tile has been read and the wait
          // below is for this V's phase and no earlier one.)
          const uint32_t at = seq + v_pos(t, nt);
          const int s = static_cast<int>(at % kNS);
          ok = warp_wait(full(s), (at / kNS) & 1, abort_flag, p.status);
          if (!ok) break;
          const int row = t_lane, key = key0 + row;
          if (key >= start) {
            bool bad = false;
            unsigned char* line = gbase + C::kQs + s * C::kSlot + (row >> 3) * C::kGroup + (row & 7) * 128;
            constexpr int kChunks = 8 * C::kPanels / 2;  // 16-byte chunks for each of a row's threads
#pragma unroll 1
            for (int k = 0; k < kChunks; ++k) {
              // the lanes' lines share their banks: each starts at another chunk
              const int i = half * kChunks + ((k ^ row) & (kChunks < 8 ? kChunks - 1 : 7));
              uint4* at16 = reinterpret_cast<uint4*>(line + (i >> 3) * 1024 + ((i & 7) << 4));
              uint4 x = key < ctx ? *at16 : make_uint4(0, 0, 0, 0);
              const bool hit = clear_odd<T>(x);
              bad |= hit;
              if (hit || key >= ctx) *at16 = x;
            }
            if (bad) s_odd[seg % 3] = 1;
          }
          fence_proxy_async();
        }
        tc_fence_after();
        if (first_row < sg.rows) {
          const uint32_t t_s = tmem + w * 128 + half * 64 + lane_off;
          uint32_t v0 = 0, v1 = 0;
          if (tail) {
            const int off = key0 + half * 64 - start;
            const unsigned long long v =
                !row_on ? 0ull
                        : (p.words == 1 ? seen64(&mword, 1, off, n)
                                        : seen64(mask_row(node), p.words, off, n));
            v0 = static_cast<uint32_t>(v);
            v1 = static_cast<uint32_t>(v >> 32);
          }
          // DUP: the 32 keys of this side, and zeros in P for the other's
          constexpr int kN = DUP ? 32 : 64;
          const uint32_t t_n = t_s + side * 32, t_p = t_s + side * 16;
          if (DUP && side) v0 = v1;
          float top = tail ? top_score<kN, true>(t_n, v0, v1, p.scale_log2)
                           : top_score<kN, false>(t_n, 0, 0, p.scale_log2);
          // (exchanging under the exponentials instead, with the rare correction
          // after them, made the loop longer and slower)
          top = max3_nan(top, swap(top), -INFINITY);
          if (!ok) break;
          const bool moved = row_on && !(top <= m_ref + kSlack);
          if (__any_sync(0xffffffffu, moved)) {
            // infinite or NaN scores make the reference NaN and with it the row, as the formula does
            const float m_new = !moved ? m_ref : (top <= FLT_MAX ? ceilf(top) : NAN);
            const float a = pow2_down(m_new - m_ref);
            l *= a;
            m_ref = m_new;
            if (t > 0) {
              ok = wait_s(t + 1);  // PV(t - 1) may still be adding to O: S(t + 1) comes after it
              if (!ok) break;
              tc_fence_after();
              scale_o(tmem + 256 + half * (D / 2) + lane_off, D / 64, a);
            }
          }
          l += tail ? softmax_part<T, kN, true>(t_n, t_p, v0, v1, p.scale_log2, m_ref)
                    : softmax_part<T, kN, false>(t_n, t_p, 0, 0, p.scale_log2, m_ref);
          if (DUP) {
            const uint32_t zero[16] = {};
            tmem_st16(t_s + (side ^ 1) * 16, zero);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(w));
      }
      if (!ok) break;
      ok = wait_s(nt);
      if (!ok) break;
      give_of(nt);
      ok = wait_s(nt + 1);
      if (!ok) break;
      give_of(nt + 1);
      phase[0] += (nt + 3) >> 1;
      phase[1] += (nt + 2) >> 1;
      tc_fence_after();
      const bool whole = sg.flags & kSegWhole;
      const int slot = sg.tile0 > 0 ? 0 : 1;
      if (first_row < sg.rows) {  // this thread's half (DUP: quarter) of its row's columns
        float m = m_ref, lt = l + swap(l);
        if (!ok) break;
        constexpr int kCols = DUP ? D / 4 : D / 2;  // it stores, kChunk at a time
        constexpr int kChunk = kCols < 32 ? kCols : 32;
        const int col0 = half * (D / 2) + side * (D / 4);
        const uint32_t t_o = tmem + 256 + lane_off;
        float o[32], f = 1.f;
        if (DUP) {
          // Both sides' sums and half of each side's O change hands through the
          // room behind Q; the next segment's S comes after everyone's o_free.
          float* x = reinterpret_cast<float*>(gbase + C::kQ) + ((half * 2 + side) * kCols) * 64 + r;
          tmem_ld32(t_o + half * (D / 2) + (D == 128 ? (side ^ 1) * 32 : 0), o);
#pragma unroll
          for (int i = 0; i < kCols; ++i) x[i * 64] = D == 128 ? o[i] : (side ? o[i] : o[i + 32 - kCols]);
          float* at = s_swap + (swaps & 1) * 256 + t_lane;  // (the pair's next buffer)
          at[half * 128] = half ? lt : m;
          __syncwarp();
          if (lane == 0) mbar_arrive(cross(quarter & 1));
          ok = warp_wait(cross(quarter & 1), crosses++ & 1, abort_flag, p.status);
          if (!ok) break;
          const float* other = s_swap + (swaps & 1) * 256 + (t_lane ^ 64);
          const float m2 = other[0], l2 = other[128];
          const float m1 = m;
          m = fmaxf(m1, m2);
          f = exp2f(m1 - m);  // NaN if a max is
          const float f2 = exp2f(m2 - m);
          lt = lt * f + l2 * f2;
          if (D == 128) tmem_ld32(t_o + col0, o);
          const float* y = reinterpret_cast<float*>(gbase + C::kQ) + ((half * 2 + (side ^ 1)) * kCols) * 64 + r;
#pragma unroll
          for (int i = 0; i < kCols; ++i)
            o[i] = (D == 128 ? o[i] : (side ? o[i + 32 - kCols] : o[i])) * f + y[i * 64] * f2;
          f = 1.f;
        }
        if (whole) f = lt == 0.f ? 0.f : 1.f / lt;
        float zero = 0.f;  // NaN if one of its values is not finite
        T* dst = static_cast<T*>(p.out) +
                 (static_cast<long long>(sg.q0 + node) * p.Hq + sg.h * p.G + r_head) * D + col0;
#pragma unroll 1
        for (int c = 0; c < kCols / kChunk; ++c) {
          if (!DUP) tmem_ld32(t_o + col0 + c * 32, o);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) o[i] *= f;
#pragma unroll
          for (int i = 0; i < kChunk; ++i) zero = fmaf(o[i], 0.f, zero);
          if (row_on) {
            // a store of a warp's 32 rows to out touches a line each: the wider the better
            if (!whole) {
#pragma unroll
              for (int i = 0; i < kChunk / 8; ++i)
                st_global_32(part_o(p, blockIdx.x, slot, r, (col0 >> 3) + c * 4 + i, D),
                             reinterpret_cast<const uint32_t*>(o + 8 * i));
            } else if (p.out32) {
#pragma unroll
              for (int i = 0; i < kChunk; i += 16) {
                uint32_t v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = pack2<T>(o[i + 2 * e], o[i + 2 * e + 1]);
                st_global_32(dst + c * 32 + i, v);
              }
            } else {
#pragma unroll
              for (int i = 0; i < kChunk; i += 8) *reinterpret_cast<uint4*>(dst + c * 32 + i) = pack8<T>(o + i);
            }
          }
        }
        if (!whole && row_on && half == 0 && side == 0) *part_ml(p, blockIdx.x, slot, r) = make_float2(m, lt);
        const bool in_order = row_on && finite_sum(lt);  // its outputs are to be finite
        const bool all = __any_sync(0xffffffffu, in_order && zero != 0.f);  // one is not
        if (all || s_odd[seg % 3] != 0) {
          const int32_t* table = p.tables + static_cast<long long>(sg.b) * p.max_blocks;
          const int k0 = sg.tile0 * kTcKeys, k1 = min((sg.tile0 + nt) * kTcKeys, ctx);
          auto add_key = [&](OddColumns& odd, int key) {
            const int phys = table[key / p.block_size];
            if (phys < 0 || phys >= p.num_blocks) return;
            const uint4* vr = reinterpret_cast<const uint4*>(
                static_cast<const T*>(p.v_cache) +
                ((static_cast<long long>(phys) * p.block_size + key % p.block_size) * p.Hkv + sg.h) * D + col0);
#pragma unroll 1
            for (int i = 0; i < kCols / 8; ++i) {
              uint4 x = vr[i], y = x;
              if (!clear_odd<T>(y)) continue;
              odd.add2<T>(8 * i, x.x);
              odd.add2<T>(8 * i + 2, x.y);
              odd.add2<T>(8 * i + 4, x.z);
              odd.add2<T>(8 * i + 6, x.w);
            }
          };
          OddColumns odd;
          if (all) {
#pragma unroll 1
            for (int key = k0 + lane; key < min(k1, start); key += 32) add_key(odd, key);
            __syncwarp();
            odd.join(31);
          }
          if (in_order) {
            const unsigned long long* mrow = mask_row(node);
#pragma unroll 1
            for (int key = max(k0, start); key < k1; ++key) {
              const int jn = key - start;
              if ((mrow[jn >> 6] >> (jn & 63)) & 1) add_key(odd, key);
            }
#pragma unroll 1
            for (int i = 0; i < kCols; ++i) {  // over what this thread has stored
              if (!odd.any(i)) continue;
              if (whole) dst[i] = from_f32<T>(odd.value(i));
              else part_o(p, blockIdx.x, slot, r, (col0 + i) >> 3, D)[(col0 + i) & 7] = odd.value(i);
            }
          }
          __syncwarp();
        }
      }
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      seq += 2 * nt;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// -------------------------------------------------------------- the joining --
// A split row group's parts lie in the CTAs c0 (slot 1) and c0 + 1 .. c1 (slot
// 0); the block columns c0 + 1 .. c1 join its rows, an equal number each, so the
// work is even whatever the number of parts. Few parts: a warp per row; many, or
// no rows for the other warps: a row's parts are dealt to the warps of the block
// and summed in warp order. 16 row groups of 10 parts (33 nodes at context 32717):
// the whole call 58.5 us dealt, 57.0 not; 2 of 12 parts and 8 rows: 15.1 and 16.6.
constexpr int kJoinWarps = 8;
// Blocks of the grid, 4 to 16 per column: with 4 throughout, one request of 64
// nodes at 2000 (33 CTAs) took 16.5 us instead of 15.5.
constexpr int kJoinBlocks = 4 * 148;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) tree_join_kernel(const TreeParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int DPL = D / 32;
  __shared__ __align__(16) float s_acc[kJoinWarps][D];
  __shared__ float2 s_ml[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x + 1;
  const Part pt = p.parts[c];
  if (pt.c0 < 0) return;
  const int helpers = pt.c1 - pt.c0, parts = helpers + 1;
  const int units = helpers * gridDim.y;  // blocks that share this row group
  const int unit = (c - pt.c0 - 1) * gridDim.y + blockIdx.y;
  const int r_begin = pt.rows * unit / units, r_end = pt.rows * (unit + 1) / units;
  // deal a row's parts to the warps
  const bool deal = parts > 2 * kJoinWarps || (parts > kJoinWarps && r_end - r_begin <= 1);
  for (int r0 = r_begin; r0 < r_end; r0 += deal ? 1 : kJoinWarps) {
    const int r = deal ? r0 : r0 + warp;
    const bool on = r < r_end;
    float acc[DPL], l = 0.f, m = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[i] = 0.f;
    // (max, sum, o) of one more part; the loads of kAhead parts are out at once
    auto add = [&](float pm, float pl, const float* po) {
      const float mn = fmaxf(m, pm);
      const float a = exp2f(m - mn), w = exp2f(pm - mn);
      m = mn;
      l = l * a + w * pl;
#pragma unroll
      for (int i = 0; i < DPL; ++i) acc[i] = acc[i] * a + w * po[i];
    };
    if (on) {
      constexpr int kAhead = 4;
      const int step = deal ? kJoinWarps : 1;
      for (int k0 = deal ? warp : 0; k0 < parts; k0 += kAhead * step) {
        float2 ml[kAhead];
        float o[kAhead][DPL];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int k = k0 + j * step;
          if (k < parts) {
            ml[j] = *part_ml(p, pt.c0 + k, k == 0, r);
            const float* src = part_o(p, pt.c0 + k, k == 0, r, lane * DPL / 8, D) + lane * DPL % 8;
            if (DPL == 4) {
              *reinterpret_cast<float4*>(o[j]) = *reinterpret_cast<const float4*>(src);
            } else {
              *reinterpret_cast<float2*>(o[j]) = *reinterpret_cast<const float2*>(src);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
          if (k0 + j * step < parts) add(ml[j].x, ml[j].y, o[j]);
      }
    }
    if (deal) {
#pragma unroll
      for (int i = 0; i < DPL; ++i) s_acc[warp][lane * DPL + i] = acc[i];
      if (lane == 0) s_ml[warp] = make_float2(m, l);
      __syncthreads();
      if (warp == 0)
        for (int w = 1; w < kJoinWarps; ++w) add(s_ml[w].x, s_ml[w].y, &s_acc[w][lane * DPL]);
      __syncthreads();
    }
    if (on && (!deal || warp == 0)) {
      bool nan = false;
#pragma unroll
      for (int i = 0; i < DPL; ++i) nan |= acc[i] != acc[i];
      if (nan && finite_sum(l)) {
        // An infinity of a part whose weight underflowed became NaN: the value is
        // the sum of the parts' values that are not finite.
        float odd[DPL];
#pragma unroll
        for (int i = 0; i < DPL; ++i) odd[i] = 0.f;
#pragma unroll 1
        for (int k = 0; k < parts; ++k) {
          const float* src = part_o(p, pt.c0 + k, k == 0, r, lane * DPL / 8, D) + lane * DPL % 8;
#pragma unroll
          for (int i = 0; i < DPL; ++i)
            if (!(fabsf(src[i]) <= FLT_MAX)) odd[i] += src[i];
        }
#pragma unroll
        for (int i = 0; i < DPL; ++i)
          if (acc[i] != acc[i] && odd[i] != 0.f) acc[i] = odd[i];
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int row = pt.row0 + r;
      T* dst = static_cast<T*>(p.out) +
               (static_cast<long long>(pt.q0 + row / p.G) * p.Hq + pt.h * p.G + row % p.G) * D + lane * DPL;
#pragma unroll
      for (int i = 0; i < DPL; i += 2)
        *reinterpret_cast<uint32_t*>(dst + i) = pack2<T>(acc[i] * inv, acc[i + 1] * inv);
    }
  }
}

// ------------------------------------------------------------------- host --
struct Plan {
  bool tc, dup, never_cut;
  int group_rows, ctas;
  double items;  // bound of the call's work items
  size_t bytes;
};

// The tcgen05 kernel takes blocks of whole 8-key groups (the matrix unit's and its
// copies' unit) at 32-bit rows and the heads of a group in one tile.
bool tc_layout(int num_blocks, int block_size, int G) {
  return block_size % 8 == 0 && (static_cast<long long>(num_blocks) + 1) * block_size < INT32_MAX && G <= kTcRows;
}

Plan plan_for(bool tc, int num_seqs, int max_q_len, int max_ctx, int Hq, int Hkv, int D) {
  Plan pl{};
  const int G = Hq / Hkv, keys = tc ? kTcKeys : kKeys;
  pl.tc = tc;
  pl.dup = tc && static_cast<long long>(max_q_len) * G <= kTcRows / 2;
  pl.group_rows = tc ? (pl.dup ? kTcRows / 2 : kTcRows) / G * G : kRows;
  const int key_tiles = (max_ctx + keys - 1) / keys;
  const int row_groups = pl.group_rows ? (max_q_len * G + pl.group_rows - 1) / pl.group_rows : 1;
  pl.items = static_cast<double>(num_seqs) * Hkv * row_groups * key_tiles;
  const int ctas = tc ? kTcCtas : 2 * kTcCtas;
  pl.ctas = pl.items < ctas ? static_cast<int>(pl.items) : ctas;
  // Share::find takes whole row groups if their longest are within kJoinCost of a share
  pl.never_cut = static_cast<double>(num_seqs) * Hkv * row_groups <= pl.ctas && key_tiles <= 1 + kJoinCost;
  const size_t per_cta = 2 * static_cast<size_t>(pl.group_rows) * (D + 2) * sizeof(float) + sizeof(Part);
  pl.bytes = 256 + static_cast<size_t>(pl.ctas) * per_cta;
  return pl;
}

template <typename T, int D>
int launch_join(const TreeParams& p, cudaStream_t s) {
  if (p.num_ctas == 1 || p.never_cut) return PS_OK;
  const int y = kJoinBlocks / p.num_ctas;
  ps_host::launch(tree_join_kernel<T, D>, dim3(p.num_ctas - 1, y < 4 ? 4 : (y > 16 ? 16 : y)), kJoinWarps * 32, 0, s,
                  p);
  ps_host::count_launch();
  return ps_host::check_launch("tree_attention(join)");
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
  const int rc = ps_host::check_launch("tree_attention");
  return rc == PS_OK ? launch_join<T, D>(p, s) : rc;
}

// [rows][heads][D] of 16-bit values in boxes of box_rows x box_heads x 64 dims,
// 128-byte swizzle: q (the nodes of a tile, the heads of a group).
bool make_rows_map(CUtensorMap* map, const void* base, bool bf16, long long rows, int heads, int D, int box_heads,
                   int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(heads) * D * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// One layer's cache in boxes of box_keys keys of one head, as groups of 8 keys x
// panels of 64 dims: one copy writes both panels, in the matrix unit's order.
bool make_cache_map(CUtensorMap* map, const void* base, bool bf16, long long rows, int heads, int D, int box_keys) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t pitch = static_cast<cuuint64_t>(heads) * D * 2;
  cuuint64_t dims[5] = {64, 8, static_cast<cuuint64_t>(D / 64), static_cast<cuuint64_t>(rows / 8),
                        static_cast<cuuint64_t>(heads)};
  cuuint64_t strides[4] = {pitch, 128, 8 * pitch, static_cast<cuuint64_t>(D) * 2};
  cuuint32_t box[5] = {64, 8, static_cast<cuuint32_t>(D / 64), static_cast<cuuint32_t>(box_keys / 8), 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool DUP>
int launch_tc(TreeParams& p, cudaStream_t s) {
  CUtensorMap qm, km, vm;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const long long rows = static_cast<long long>(p.num_blocks) * p.block_size;
  p.box_shift = 3;  // the largest power of two of keys that lie together in a block, at most a tile
  while (p.box_shift < 7 && p.block_size % (2 << p.box_shift) == 0) ++p.box_shift;
  p.block_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (p.block_size == 1 << i) p.block_shift = i;
  p.out32 = ps_host::aligned(p.out, 32);
  if (!make_rows_map(&qm, p.q, bf16, p.total_q, p.Hq, D, p.G, p.group_rows / p.G) ||
      !make_cache_map(&km, p.k_cache, bf16, rows, p.Hkv, D, 1 << p.box_shift) ||
      !make_cache_map(&vm, p.v_cache, bf16, rows, p.Hkv, D, 1 << p.box_shift)) {
    ps_host::set_error("tree_attention: cuTensorMapEncodeTiled failed");
    return PS_ERR_CUDA;
  }
  auto kern = tree_tc_kernel<T, D, DUP>;
  static std::atomic<uint64_t> done{0};
  if (!ps_host::reserve_smem(reinterpret_cast<const void*>(kern), Tc<D, DUP>::kSmem, &done)) {
    ps_host::set_error("tree_attention: cannot reserve %d bytes of shared memory", Tc<D, DUP>::kSmem);
    return PS_ERR_CUDA;
  }
  ps_host::launch(kern, p.num_ctas, kTcThreads, Tc<D, DUP>::kSmem, s, qm, km, vm, p);
  ps_host::count_launch();
  const int rc = ps_host::check_launch("tree_attention");
  return rc == PS_OK ? launch_join<T, D>(p, s) : rc;
}

template <typename T, int D>
int launch_tc(TreeParams& p, cudaStream_t s, bool dup) {
  return dup ? launch_tc<T, D, true>(p, s) : launch_tc<T, D, false>(p, s);
}

}  // namespace

extern "C" {

size_t ps_tree_attention_workspace_size(int num_seqs, int max_q_len, int max_ctx, int Hq, int Hkv, int D) {
  if (num_seqs <= 0 || max_q_len <= 0 || max_q_len > kMaxNodes || max_ctx < max_q_len || Hq <= 0 || Hkv <= 0 ||
      Hq % Hkv != 0 || (D != 64 && D != 128))
    return 0;
  const size_t a = plan_for(true, num_seqs, max_q_len, max_ctx, Hq, Hkv, D).bytes;
  const size_t b = plan_for(false, num_seqs, max_q_len, max_ctx, Hq, Hkv, D).bytes;
  return a > b ? a : b;
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
  const Plan pl = plan_for(tc_layout(num_blocks, block_size, Hq / Hkv), num_seqs, max_q_len, max_ctx, Hq, Hkv, D);
  if (pl.items > INT32_MAX - 1024) {
    ps_host::set_error("tree_attention: %d sequences at context %d are more work items than 32 bits count", num_seqs,
                       max_ctx);
    return PS_ERR_UNSUPPORTED;
  }
  if (!workspace || workspace_bytes < pl.bytes) {
    ps_host::set_error("tree_attention: workspace of %zu bytes needed, %zu given", pl.bytes, workspace_bytes);
    return PS_ERR_INVALID;
  }
  const uintptr_t rows = static_cast<uintptr_t>(total_q) * Hq * D * 2, b4 = 4ull * num_seqs;
  const uintptr_t cache = static_cast<uintptr_t>(num_blocks) * block_size * Hkv * D * 2;
  const ps_host::Range ins[] = {{q, rows}, {k_cache, cache}, {v_cache, cache}, {tables, b4 * max_blocks},
                                {cu_q, b4 + 4}, {start_pos, b4},
                                {tree_mask, 8ull * total_q * ((max_q_len + 63) / 64)}};
  const ps_host::Range outs[] = {{out, rows}, {workspace, pl.bytes}};
  bool shared = ps_host::overlap(outs[0], outs[1]);
  for (const auto& o : outs)
    for (const auto& in : ins) shared |= ps_host::overlap(o, in);
  if (shared) {
    ps_host::set_error("tree_attention: out or the workspace overlaps q, another input that blocks may still read, "
                       "or the other");
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
  const size_t parts = static_cast<size_t>(pl.ctas) * 2 * pl.group_rows;
  p.part = reinterpret_cast<float*>(w);
  p.part_ml = p.part + parts * D;
  p.parts = reinterpret_cast<Part*>(p.part_ml + parts * 2);
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
  p.never_cut = pl.never_cut;
  p.group_rows = pl.group_rows;
  if (pl.tc) {
    // ceil(n / t), t = group_rows / G <= 128 nodes: exact, since (n + t - 1) * t < 2^20 for n <= 256
    const uint32_t t = pl.group_rows / p.G;
    p.rg_mul = 1;
    p.rg_add = t - 1;
    p.rg_shift = 20;
    p.rg_magic = ((1u << 20) + t - 1) / t;
  } else {  // ceil(n * G / 64)
    p.rg_mul = p.G;
    p.rg_add = kRows - 1;
    p.rg_shift = 6;
    p.rg_magic = 1;
  }
  p.scale_log2 = (1.0f / sqrtf(static_cast<float>(D))) * kLog2e;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (pl.tc) {
    if (dtype == PS_BF16)
      return D == 128 ? launch_tc<__nv_bfloat16, 128>(p, s, pl.dup) : launch_tc<__nv_bfloat16, 64>(p, s, pl.dup);
    return D == 128 ? launch_tc<__half, 128>(p, s, pl.dup) : launch_tc<__half, 64>(p, s, pl.dup);
  }
  if (dtype == PS_BF16)
    return D == 128 ? launch_mma<__nv_bfloat16, 128>(p, s) : launch_mma<__nv_bfloat16, 64>(p, s);
  return D == 128 ? launch_mma<__half, 128>(p, s) : launch_mma<__half, 64>(p, s);
}

}  // extern "C"
