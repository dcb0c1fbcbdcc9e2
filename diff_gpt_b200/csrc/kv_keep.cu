// Rows of accepted drafts move to where they belong in the cache: for every sequence s, layer, head, and for keys and values alike,
//   slot dst[s] + i  <-  slot src[s] + path[s][i],   i < count[s].
// A copy of rows, bound by memory or, where few rows move, by the launch and the loads that depend on one another: count and path, page, row.
// A CTA owns 256 columns of 16 bytes of one sequence and all of its rows, a thread a column; the CTA works out once where the rows lie.  Eight rows
// at a time are read into registers before the first of them is written.  That is all the care that source and target need to overlap in any
// way, unless a row of a later round comes from a slot that an earlier round writes (it cannot where a path's rows only move down or away);
// then 32 threads share a column, and read all of its rows before they write one.
// (192 sequences, 12 layers, 12 heads of 64, 5 rows each: 95 us with 32 threads per column throughout, each finding its rows' places itself, 22 with
// 16 rows in registers and two CTAs an SM, 14 to 15 so; reading and writing them takes 12.)
#include "common.cuh"

namespace dgpt {

struct KeepParams {
  KvView kv;
  const int *src, *dst, *path, *count;
  long long layer_bytes, page_bytes, head_bytes, token_bytes;
  int B, T, H, kinds, vecs;  // kinds: 2 = keys and values, 1 = one storage; vecs: 16-byte columns of a row of one head
  long long columns;         // of a sequence: layers * kinds * H * vecs
  int* status;
};

constexpr int kKeepCols = 256, kKeepRound = 8, kKeepMost = 256;  // columns of a CTA, rows of a round, rows of a sequence

// MOST: rows of a sequence.  (Up to 64: the shared path's rows then take fewer registers of everyone; 8 drafts of 192 sequences 9.8 us for 10.5.)
template <int MOST>
__global__ void __launch_bounds__(kKeepCols) kv_keep_kernel(const KeepParams p, const unsigned blocks_per_seq) {
  __shared__ long long from[MOST], to[MOST];  // bytes from a column's base, or -1
  const int s = (int)(blockIdx.x / blocks_per_seq), tid = threadIdx.x;
  const unsigned block = blockIdx.x - (unsigned)s * blocks_per_seq;
  const int asked = p.count[s], src = p.src[s], dst = p.dst[s], node = tid < p.T ? p.path[(long long)s * p.T + tid] : 0;
  const int n = min(max(asked, 0), p.T);
  const int* table = p.kv.page_table ? p.kv.page_table + (long long)s * p.kv.max_pages : nullptr;
  bool bad = asked != n, later = false;
  if (tid < n) {
    const long long room = (long long)(table ? p.kv.max_pages : 1) * p.kv.page_tokens;
    auto place = [&](long long slot) -> long long {  // -1: no such slot, or its page is none
      if (slot < 0 || slot >= room) return -1;
      const unsigned lp = (unsigned)slot / (unsigned)p.kv.page_tokens, in = (unsigned)slot - lp * (unsigned)p.kv.page_tokens;
      const long long pg = table ? (long long)table[lp] : s;
      if (pg < 0 || (p.kv.n_pages > 0 && pg >= p.kv.n_pages)) return -1;
      return pg * p.page_bytes + (long long)in * p.token_bytes;
    };
    const long long a = node < 0 ? -1 : place((long long)src + node), b = place((long long)dst + tid);
    from[tid] = a < 0 || b < 0 ? -1 : a;
    to[tid] = b;
    bad |= a < 0 || b < 0;
    const long long ahead = (long long)src + node - dst;  // the row whose target is this one's source
    later = ahead >= 0 && ahead < (tid & ~(kKeepRound - 1));
  }
  if (bad && block == 0 && p.status) atomicOr(p.status, 1);
  const bool shared = __syncthreads_or(later) != 0;
  auto base = [&](long long col) -> char* {
    const unsigned c = (unsigned)col, lkh = c / (unsigned)p.vecs, lk = lkh / (unsigned)p.H;
    return static_cast<char*>(p.kinds > 1 && (lk & 1u) ? p.kv.v : p.kv.k) + (long long)(p.kinds > 1 ? lk >> 1 : lk) * p.layer_bytes +
           (long long)(lkh - lk * (unsigned)p.H) * p.head_bytes + (long long)(c - lkh * (unsigned)p.vecs) * 16;
  };
  const long long col0 = (long long)block * kKeepCols;
  if (!shared) {
    if (col0 + tid >= p.columns) return;
    char* at = base(col0 + tid);
    for (int i0 = 0; i0 < n; i0 += kKeepRound) {
      uint4 x[kKeepRound];
#pragma unroll
      for (int i = 0; i < kKeepRound; ++i)
        if (i0 + i < n && from[i0 + i] >= 0) x[i] = *reinterpret_cast<const uint4*>(at + from[i0 + i]);
#pragma unroll
      for (int i = 0; i < kKeepRound; ++i)
        if (i0 + i < n && from[i0 + i] >= 0) *reinterpret_cast<uint4*>(at + to[i0 + i]) = x[i];
    }
    return;
  }
  constexpr int kRows = (MOST + 31) / 32;
  const int row0 = tid >> 3;
  for (int c = 0; c < kKeepCols && col0 + c < p.columns; c += 8) {
    const long long col = col0 + c + (tid & 7);
    const bool on = col < p.columns;
    char* at = on ? base(col) : nullptr;
    uint4 x[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = row0 + i * 32;
      if (on && row < n && from[row] >= 0) x[i] = *reinterpret_cast<const uint4*>(at + from[row]);
    }
    __syncthreads();  // every row of these columns has been read
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = row0 + i * 32;
      if (on && row < n && from[row] >= 0) *reinterpret_cast<uint4*>(at + to[row]) = x[i];
    }
  }
}

}  // namespace dgpt

using namespace dgpt;

extern "C" int dgpt_kv_keep(const dgpt_kv_layout* kv, int64_t kv_token_stride, const int32_t* src_start, const int32_t* dst_start,
                            const int32_t* path, const int32_t* count, int32_t n_layer, int64_t layer_stride, int32_t B, int32_t T, int32_t H,
                            int32_t D, int32_t dtype, int32_t* status, void* stream) {
  DGPT_REQUIRE(B >= 0 && T >= 0 && n_layer > 0 && H > 0 && D > 0, "kv_keep: bad sizes");
  DGPT_REQUIRE(T <= kKeepMost, "kv_keep: at most 256 rows per sequence, got %d", T);
  if (dtype != DGPT_F32 && dtype != DGPT_BF16) {
    set_error("kv_keep: unknown dtype %d", dtype);
    return DGPT_E_UNSUPPORTED;
  }
  const int size = dtype == DGPT_F32 ? 4 : 2;
  DGPT_REQUIRE((int64_t)D * size % 16 == 0, "kv_keep: a head's row must be a multiple of 16 bytes");
  if (B == 0 || T == 0) return DGPT_OK;
  DGPT_REQUIRE(src_start && dst_start && path && count, "kv_keep: NULL pointer");
  if (int e = validate_kv(kv, D)) return e;
  DGPT_REQUIRE(kv_token_stride >= D && kv_token_stride % 8 == 0 && layer_stride % 8 == 0, "kv_keep: strides must be multiples of 8 elements");
  DGPT_REQUIRE(kv->n_pages >= 0, "kv_keep: pages must not be negative");
  DGPT_REQUIRE(kv->page_table || kv->n_pages == 0 || B <= kv->n_pages, "kv_keep: %d sequences in a cache of %lld", B, (long long)kv->n_pages);
  DGPT_REQUIRE((H == 1 || kv->head_stride >= D) && (n_layer == 1 || layer_stride != 0), "kv_keep: heads and layers must lie apart");
  KeepParams p;
  p.kv = make_view(kv);
  p.src = src_start;
  p.dst = dst_start;
  p.path = path;
  p.count = count;
  p.layer_bytes = layer_stride * size;
  p.page_bytes = kv->page_stride * size;
  p.head_bytes = kv->head_stride * size;
  p.token_bytes = kv_token_stride * size;
  p.B = B;
  p.T = T;
  p.H = H;
  p.kinds = kv->k_base == kv->v_base ? 1 : 2;
  p.vecs = D * size / 16;
  p.columns = (long long)n_layer * p.kinds * H * p.vecs;
  p.status = status;
  const long long per = (p.columns + kKeepCols - 1) / kKeepCols, blocks = per * B;
  DGPT_REQUIRE(blocks <= 0x7fffffffll && p.columns <= 0x7fffffffll, "kv_keep: too many rows");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T <= 64) kv_keep_kernel<64><<<(unsigned)blocks, kKeepCols, 0, st>>>(p, (unsigned)per);
  else kv_keep_kernel<kKeepMost><<<(unsigned)blocks, kKeepCols, 0, st>>>(p, (unsigned)per);
  return launch_status("kv_keep");
}
