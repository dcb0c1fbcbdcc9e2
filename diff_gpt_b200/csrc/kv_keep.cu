// Rows of accepted drafts move to where they belong in the cache: for every sequence s, layer, head, and for keys and values alike,
//   slot dst[s] + i  <-  slot src[s] + path[s][i],   i < count[s].
// A copy of rows, bound by memory or, where few rows move, by the launch.  A CTA owns 32 columns of 16 bytes of one sequence and all of
// its rows, reads every row before it writes the first, and columns do not mix: source and target may overlap in any way.  A thread
// keeps its rows in registers (up to 2, 8 or 32 of them, by the most rows that a sequence may move).
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

constexpr int kKeepCols = 32, kKeepRows = 8;

template <int RPT>
__global__ void __launch_bounds__(kKeepCols * kKeepRows) kv_keep_kernel(const KeepParams p, const unsigned blocks_per_seq) {
  const int s = (int)(blockIdx.x / blocks_per_seq);
  const long long col = (long long)(blockIdx.x % blocks_per_seq) * kKeepCols + (threadIdx.x & 31);
  const int row0 = threadIdx.x >> 5;
  const int asked = p.count[s], n = min(max(asked, 0), p.T);
  bool bad = asked != n;
  const bool on = col < p.columns;
  const int vec = (int)(col % p.vecs);
  const long long lkh = col / p.vecs, lk = lkh / p.H;
  const int h = (int)(lkh - lk * p.H), kind = (int)(lk % p.kinds);
  char* base = static_cast<char*>(kind == 0 ? p.kv.k : p.kv.v) + (lk / p.kinds) * p.layer_bytes + (long long)h * p.head_bytes + (long long)vec * 16;
  const int* table = p.kv.page_table ? p.kv.page_table + (long long)s * p.kv.max_pages : nullptr;
  const long long room = (long long)(table ? p.kv.max_pages : 1) * p.kv.page_tokens;
  auto place = [&](long long slot, char*& at) {  // false: no such slot, or its page is none
    if (slot < 0 || slot >= room) return false;
    const int lp = (int)(slot / p.kv.page_tokens), in = (int)(slot - (long long)lp * p.kv.page_tokens);
    const long long pg = table ? (long long)table[lp] : s;
    if (pg < 0 || (p.kv.n_pages > 0 && pg >= p.kv.n_pages)) return false;
    at = base + pg * p.page_bytes + (long long)in * p.token_bytes;
    return true;
  };
  const int* path = p.path + (long long)s * p.T;
  uint4 x[RPT];
  char* to[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int row = row0 + i * kKeepRows;
    to[i] = nullptr;
    if (row < n) {
      char *from, *at;
      const int node = path[row];
      if (node >= 0 && place((long long)p.src[s] + node, from) && place((long long)p.dst[s] + row, at)) {
        if (on) {
          x[i] = *reinterpret_cast<const uint4*>(from);
          to[i] = at;
        }
      } else {
        bad = true;
      }
    }
  }
  __syncthreads();  // every row of these columns has been read
#pragma unroll
  for (int i = 0; i < RPT; ++i)
    if (to[i]) *reinterpret_cast<uint4*>(to[i]) = x[i];
  if (bad && p.status && (threadIdx.x & 31) == 0) atomicOr(p.status, 1);
}

}  // namespace dgpt

using namespace dgpt;

extern "C" int dgpt_kv_keep(const dgpt_kv_layout* kv, int64_t kv_token_stride, const int32_t* src_start, const int32_t* dst_start,
                            const int32_t* path, const int32_t* count, int32_t n_layer, int64_t layer_stride, int32_t B, int32_t T, int32_t H,
                            int32_t D, int32_t dtype, int32_t* status, void* stream) {
  DGPT_REQUIRE(B >= 0 && T >= 0 && n_layer > 0 && H > 0 && D > 0, "kv_keep: bad sizes");
  DGPT_REQUIRE(T <= 256, "kv_keep: at most 256 rows per sequence, got %d", T);
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
  DGPT_REQUIRE(blocks <= 0x7fffffffll, "kv_keep: too many rows");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)blocks), block(kKeepCols * kKeepRows);
  if (T <= 2 * kKeepRows) kv_keep_kernel<2><<<grid, block, 0, st>>>(p, (unsigned)per);
  else if (T <= 8 * kKeepRows) kv_keep_kernel<8><<<grid, block, 0, st>>>(p, (unsigned)per);
  else kv_keep_kernel<32><<<grid, block, 0, st>>>(p, (unsigned)per);
  return launch_status("kv_keep");
}
