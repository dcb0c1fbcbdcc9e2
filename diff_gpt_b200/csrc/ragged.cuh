// Attention over sequences whose lengths lie on the device: packed prompts and trees of drafted tokens.
//
// Both are rows of queries against the keys of one sequence and one key/value head,
//   o_r = sum_j p_rj v_j,   p_r = softmax_j(q_r . k_j * scale) over the keys that row r sees,
// and differ in which rows lie side by side, where keys lie and which of them a row sees.  A problem struct answers these for the
// kernels (ragged_simt.cu on the CUDA cores, ragged_tc.cu on the tensor cores): `item` turns a work item's number into the rows
// and keys of one tile, `q_row`, `k_row`, `v_row` give addresses, `sees` the mask, `out_row` and `head` where a tree's row goes.
#pragma once

#include "common.cuh"

namespace dgpt {

// Rows and keys are counted in 32 bits, with room behind the last one for a tile.
constexpr long long kRgMost = 0x7fffff00ll;

// One tile of up to BM rows against keys [key0, key1) of a sequence.
struct RaggedItem {
  int rows;        // rows of the tile that exist
  int seq, g, h;   // sequence, key/value head, query head of the tile (packed) or first query head of its group (tree)
  int row0;        // first row: token (packed), node * group + head in group (tree)
  int key0, key1;  // keys of this item; the sequence's first `clear` keys are seen by every row
  int clear;
  int last0;       // packed: the last key that the tile's first row sees (negative: none); row r sees r more
  int split;       // tree: which share of the keys
  int kbase;       // packed: row of the sequence's key 0
  int held;        // packed: the sequence's keys
  int gap0, gap1;  // tree: slots [gap0, gap1) before the drafts hold nothing
};

// ---- packed prompts ---------------------------------------------------------------------------------------------
// Sequence s owns query rows [q_starts[s], q_starts[s + 1]) and key rows [k_starts[s], k_starts[s + 1]); its last query sees all of
// its keys, the one before all but the last, and so on.
//
// Tiles of BM rows start at a sequence's first row, so their number follows from all lengths, which the host does not know.
// Without a pass that counts them: sequence s takes the tile slots from base(s) = q_starts[s] / BM + s on.  A sequence of n rows has
// ceil(n / BM) tiles, and base(s + 1) - base(s) is never less than that, so no two tiles share a slot; at most one slot a sequence stays
// empty, and a binary search over base() finds a slot's sequence.
struct PackedProblem {
  const void *q, *k, *v;
  long long q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, o_rs, o_hs;
  void* o;
  float* lse;  // [n_rows, H] or NULL
  const int *q_starts, *k_starts;
  int n_seq, n_rows, n_keys, H, G;
  float scale_log2;
  int* status;
  long long wait_limit;  // of the tensor-core kernel's waits, clock cycles

  __host__ __device__ long long slots(int bm) const { return (long long)n_rows / bm + n_seq; }
  // A start is taken into the tensor's rows: wrong numbers give wrong rows, never an access outside.
  __device__ int q_start(int s) const { return min(max(q_starts[s], 0), n_rows); }
  __device__ int k_start(int s) const { return min(max(k_starts[s], 0), n_keys); }
  // The last sequence whose base is not behind the slot: 32 at a time, for a whole warp.
  __device__ int find(int slot, int bm, int lane) const {
    int lo = 0, n = n_seq;
    while (n > 1) {
      const int step = (n + 31) >> 5, s = lo + lane * step;
      const bool before = lane * step < n && q_start(s) / bm + s <= slot;
      const int last = 31 - __clz(__ballot_sync(0xffffffffu, before) | 1u);
      lo += last * step;
      n = min(step, n - last * step);
    }
    return lo;
  }
  // A sequence and what is known of it.
  struct Cursor {
    int seq = 0, first = 0, end = 0, kb = 0, nk = 0, slot0 = 0, slot1 = 0;  // it has slots [slot0, slot1)
  };
  __device__ void load(int s, int bm, Cursor& c) const {
    c.seq = s;
    c.first = q_start(s);
    c.end = q_start(s + 1);
    c.kb = k_start(s);
    c.nk = max(0, k_start(s + 1) - c.kb);
    c.slot0 = c.first / bm + s;
    c.slot1 = c.end / bm + s + 1;
  }
  __device__ void seek(int slot, int bm, int lane, Cursor& c) const {
    if (slot < c.slot0 || slot >= c.slot1) load(find(slot, bm, lane), bm, c);
  }
  __device__ bool item(int slot, const Cursor& c, int h, int bm, RaggedItem& it) const {
    const int first = c.first, end = c.end, lo = c.seq;
    const int tile = slot - first / bm - lo;
    if (tile < 0 || (long long)first + (long long)tile * bm >= end) return false;
    const int row0 = first + tile * bm;
    it.seq = lo;
    it.h = h;
    it.g = h / (H / G);
    it.row0 = row0;
    it.rows = min(bm, end - row0);
    const int kb = c.kb, nk = c.nk;
    const long long behind = (long long)nk - (end - first) + (row0 - first);  // keys before the one of the tile's first row
    it.key0 = 0;
    it.last0 = (int)behind;
    it.key1 = (int)max(0ll, min((long long)nk, behind + it.rows));
    it.clear = (int)max(0ll, min((long long)nk, behind + 1));
    it.split = 0;
    it.kbase = kb;
    it.held = nk;
    it.gap0 = it.gap1 = 0;
    return true;
  }
  __device__ bool sees(const RaggedItem& it, int r, int j) const { return j < it.key1 && j <= it.last0 + r; }
  template <typename T>
  __device__ const T* q_row(const RaggedItem& it, int r) const {
    return static_cast<const T*>(q) + (long long)(it.row0 + r) * q_rs + (long long)it.h * q_hs;
  }
  template <typename T>
  __device__ const T* k_row(const RaggedItem& it, int j) const {
    return static_cast<const T*>(k) + (long long)(it.kbase + j) * k_rs + (long long)it.g * k_hs;
  }
  template <typename T>
  __device__ const T* v_row(const RaggedItem& it, int j) const {
    return static_cast<const T*>(v) + (long long)(it.kbase + j) * v_rs + (long long)it.g * v_hs;
  }
  // Whoever has the launch's first item looks at all starts.
  __device__ void check(bool first, int thread, int threads) const {
    if (!first || status == nullptr) return;
    bool bad = false;
    for (int s = thread; s <= n_seq; s += threads) {
      const int a = q_starts[s], b = k_starts[s];
      bad |= a < 0 || a > n_rows || b < 0 || b > n_keys;
      if (s > 0) bad |= a < q_starts[s - 1] || b < k_starts[s - 1];
    }
    if (bad) atomicOr(status, 1);
  }
};

// ---- trees of drafted tokens ------------------------------------------------------------------------------------
// Node t < n_nodes[s] of sequence s sits in cache slot ctx[s] + t and sees slots [0, ctx[s]), but for a gap [gap_start[s], gap_end[s]) (what a prompt
// leaves free of its last page), and those nodes j of its own sequence whose bit is set: word j / 64, bit j % 64 of ancestors[s][t].  The rows of one key/value head are its T * (H / G) pairs of node and
// query head, node-major, so that K and V are read once for all of them.
struct TreeProblem {
  static constexpr int kSorted = 64;  // sequences, at most, that are taken from the longest to the shortest
  const void* q;
  long long q_rs;
  KvView kv;
  const int* ctx;
  const int *gap_start, *gap_end;      // both NULL: no gaps
  const int* n_nodes;                  // NULL: T everywhere
  const unsigned long long* ancestors; // [B][T][words]
  int words;
  void* o;
  long long o_rs;
  float* part_o;    // [n_splits][B * T * H][D] and their sums' logarithms (base 2) [n_splits][B * T * H]; n_splits == 1: unused
  float* part_lse;
  int n_splits, B, T, H, G, D, group, rows_per_tile, tiles;  // group = H / G
  int tile_keys;  // keys of a tile, as the pass that joins the splits counts them
  float scale_log2;
  int* status;
  long long wait_limit;  // of the tensor-core kernel's waits, clock cycles

  __host__ __device__ long long items() const { return (long long)B * G * tiles * n_splits; }  // below 2^31 (the entry point sees to it)
  __device__ long long room() const { return min((long long)(kv.page_table ? kv.max_pages : 1) * kv.page_tokens, kRgMost); }
  // Keys [0, keys) of a sequence, of which the last `nodes` are drafts.  What does not fit the layout is left out.
  __device__ void lengths(int s, int& context, int& nodes) const {
    const long long room = this->room();
    context = (int)min((long long)max(ctx[s], 0), room);
    nodes = n_nodes ? min(max(n_nodes[s], 0), T) : T;
    nodes = (int)min((long long)nodes, room - context);
  }
  // Splits share the key tiles of `bn` keys evenly; where there are fewer tiles, the splits behind them get none.
  __device__ bool item(unsigned i, int bn, RaggedItem& it, const int* order = nullptr) const {
    const unsigned a = i / (unsigned)n_splits, b = a / (unsigned)tiles, c = b / (unsigned)G;
    it.split = (int)(i - a * (unsigned)n_splits);
    const int tile = (int)(a - b * (unsigned)tiles);
    it.g = (int)(b - c * (unsigned)G);
    it.seq = order ? order[c] : (int)c;
    it.h = it.g * group;
    int context, nodes;
    lengths(it.seq, context, nodes);
    const int n = n_nodes ? min(max(n_nodes[it.seq], 0), T) : T;
    it.row0 = tile * rows_per_tile;
    it.rows = min(rows_per_tile, n * group - it.row0);
    if (it.rows <= 0) return false;
    const int keys = context + nodes, n_tiles = (keys + bn - 1) / bn;
    const int per = n_tiles / n_splits, more = n_tiles - per * n_splits;  // the first `more` splits take one tile more
    const int t0 = it.split * per + min(it.split, more), t1 = t0 + per + (it.split < more ? 1 : 0);
    it.key0 = min(keys, t0 * bn);
    it.key1 = min(keys, t1 * bn);
    it.clear = context;
    it.last0 = 0;
    it.kbase = it.held = 0;
    it.gap0 = it.gap1 = 0;
    if (gap_start) {
      it.gap1 = min(max(gap_end[it.seq], 0), context);
      it.gap0 = min(max(gap_start[it.seq], 0), it.gap1);
    }
    return true;
  }
  // order[i]: the i-th longest sequence (B <= kSorted; for a whole warp).
  __device__ void sort(int* order, int lane) const {
    int c[2], r[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      c[u] = lane + 32 * u < B ? ctx[lane + 32 * u] : -1;
      r[u] = 0;
    }
    for (int j = 0; j < B; ++j) {
      const int o = __shfl_sync(0xffffffffu, j < 32 ? c[0] : c[1], j & 31);
#pragma unroll
      for (int u = 0; u < 2; ++u) r[u] += o > c[u] || (o == c[u] && j < lane + 32 * u);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (lane + 32 * u < B) order[r[u]] = lane + 32 * u;
    __syncwarp();
  }
  __device__ const unsigned long long* mask_row(const RaggedItem& it, int r) const {
    return ancestors + ((long long)it.seq * T + (it.row0 + r) / group) * words;
  }
  __device__ bool sees(const RaggedItem& it, int r, int j) const {
    if (j < it.clear) return j < it.gap0 || j >= it.gap1;
    const int d = j - it.clear;
    return (mask_row(it, r)[d >> 6] >> (d & 63)) & 1ull;
  }
  __device__ long long out_row(const RaggedItem& it, int r) const { return (long long)it.seq * T + (it.row0 + r) / group; }
  __device__ int head(const RaggedItem& it, int r) const { return it.h + (it.row0 + r) % group; }
  template <typename E>
  __device__ const E* q_row(const RaggedItem& it, int r) const {
    return static_cast<const E*>(q) + out_row(it, r) * q_rs + (long long)head(it, r) * D;
  }
  // Offset of key j; -1 in the gap, and where the page table names no page: there key and value count as zeros, as in the tensor-core kernel.
  __device__ long long key_offset(const RaggedItem& it, int j) const {
    if (j >= it.gap0 && j < it.gap1) return -1;
    const int lp = j / kv.page_tokens, in = j - lp * kv.page_tokens;
    const long long pg = kv.page_table ? (long long)kv.page_table[(long long)it.seq * kv.max_pages + lp] : it.seq;
    if (pg < 0 || (kv.n_pages > 0 && pg >= kv.n_pages)) return -1;
    return pg * kv.page_stride + (long long)it.g * kv.head_stride + (long long)in * kv.token_stride;
  }
  // Whoever has the launch's first item looks at all lengths.
  __device__ void check(bool first, int thread, int threads) const {
    if (!first || status == nullptr) return;
    for (int s = thread; s < B; s += threads) {
      const int n = n_nodes ? n_nodes[s] : T;
      bool bad = ctx[s] < 0 || n < 0 || n > T || (long long)ctx[s] + n > room();
      if (gap_start) bad |= gap_start[s] < 0 || gap_end[s] < gap_start[s] || gap_end[s] > ctx[s];
      if (bad) atomicOr(status, 1);
    }
  }
};

// ragged_simt.cu: any dtype, head_dim 8, 16, 32, 64 or 128
int packed_simt(const PackedProblem& p, int D, int dtype, cudaStream_t st);
int tree_simt(const TreeProblem& p, int dtype, cudaStream_t st);
// ragged_tc.cu: bf16, head_dim 32, 64 or 128
bool packed_tc_supported(const PackedProblem& p, int D, int dtype);
int packed_tc(const PackedProblem& p, int D, cudaStream_t st, long long wait_limit = 0);  // limit 0: the library's
bool tree_tc_supported(const TreeProblem& p, int dtype);
int tree_tc(const TreeProblem& p, cudaStream_t st);
// n_splits partials of every row into one (ragged_simt.cu)
int tree_merge(const TreeProblem& p, int tile_keys, int dtype, cudaStream_t st);

}  // namespace dgpt
