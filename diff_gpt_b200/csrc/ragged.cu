// Entry points of attention over packed prompts and over trees of drafted tokens: checks, and which kernel takes a call.
#include "ragged.cuh"

using namespace dgpt;

static bool head_dim_ok(int D) { return D == 8 || D == 16 || D == 32 || D == 64 || D == 128; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

extern "C" int dgpt_fmha_packed(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k, int64_t k_row_stride,
                                int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride, void* o,
                                int64_t o_row_stride, int64_t o_head_stride, float* lse, const int32_t* seq_starts,
                                const int32_t* key_starts, int32_t n_seq, int32_t n_rows, int32_t n_keys, int32_t H, int32_t G, int32_t D,
                                float scale, int32_t dtype, int32_t impl, int32_t* status, void* stream) {
  DGPT_REQUIRE(n_seq >= 0 && n_rows >= 0 && n_keys >= 0 && H > 0 && G > 0 && H % G == 0, "fmha_packed: bad sizes");
  DGPT_REQUIRE(n_rows <= kRgMost && n_keys <= kRgMost, "fmha_packed: too many rows");
  DGPT_REQUIRE(key_starts || n_keys == n_rows, "fmha_packed: without starts of their own the keys are as many as the queries");
  DGPT_REQUIRE(scale > 0.f, "fmha_packed: the scale must be positive");
  DGPT_REQUIRE(impl >= 0 && impl <= 2, "fmha_packed: impl must be 0 (choose), 1 (CUDA cores) or 2 (tensor cores)");
  if (dtype != DGPT_F32 && dtype != DGPT_BF16) {
    set_error("fmha_packed: unknown dtype %d", dtype);
    return DGPT_E_UNSUPPORTED;
  }
  if (!head_dim_ok(D)) {
    set_error("fmha_packed: head_dim %d is not built", D);
    return DGPT_E_UNSUPPORTED;
  }
  if (n_seq == 0 || n_rows == 0) return DGPT_OK;
  DGPT_REQUIRE(q && o && seq_starts && (n_keys == 0 || (k && v)), "fmha_packed: NULL pointer");
  DGPT_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o), "fmha_packed: pointers must be 16-byte aligned");
  const int64_t strides[8] = {q_row_stride, q_head_stride, k_row_stride, k_head_stride, v_row_stride, v_head_stride, o_row_stride, o_head_stride};
  for (int64_t s : strides) DGPT_REQUIRE(s >= D && s % 8 == 0, "fmha_packed: strides must be multiples of 8 elements, and rows and heads apart");
  PackedProblem p;
  p.q = q; p.k = k; p.v = v; p.o = o;
  p.q_rs = q_row_stride; p.q_hs = q_head_stride;
  p.k_rs = k_row_stride; p.k_hs = k_head_stride;
  p.v_rs = v_row_stride; p.v_hs = v_head_stride;
  p.o_rs = o_row_stride; p.o_hs = o_head_stride;
  p.lse = lse;
  p.q_starts = seq_starts;
  p.k_starts = key_starts ? key_starts : seq_starts;
  p.n_seq = n_seq; p.n_rows = n_rows; p.n_keys = n_keys; p.H = H; p.G = G;
  p.scale_log2 = scale * kLog2e;
  p.status = status;
  p.wait_limit = 0;
  const bool tensor = packed_tc_supported(p, D, dtype);
  if (tensor && impl != 1) return packed_tc(p, D, static_cast<cudaStream_t>(stream));
  if (impl == 2) {
    set_error("fmha_packed: the tensor-core kernel does not cover dtype %d, head_dim %d", dtype, D);
    return DGPT_E_UNSUPPORTED;
  }
  return packed_simt(p, D, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int dgpt_packed_wait_probe(int64_t limit_cycles, const void* x, void* o, const int32_t* seq_starts, int32_t n_seq, int32_t n_rows, int32_t H,
                                      int32_t D, int32_t* status, void* stream) {
  DGPT_REQUIRE(limit_cycles > 0 && limit_cycles <= 2000000000ll, "packed_wait_probe: limit must be in (0, 2e9] cycles");
  DGPT_REQUIRE(x && o && seq_starts && status && aligned16(x) && aligned16(o), "packed_wait_probe: NULL or unaligned pointer");
  DGPT_REQUIRE(n_seq > 0 && n_rows > 0 && n_rows <= 1 << 20 && H > 0, "packed_wait_probe: bad sizes");
  PackedProblem p = {};
  p.q = p.k = p.v = x;
  p.o = o;
  p.q_rs = p.k_rs = p.v_rs = p.o_rs = (long long)H * D;
  p.q_hs = p.k_hs = p.v_hs = p.o_hs = D;
  p.q_starts = p.k_starts = seq_starts;
  p.n_seq = n_seq; p.n_rows = p.n_keys = n_rows; p.H = p.G = H;
  p.scale_log2 = kLog2e / (float)D;
  p.status = status;
  if (!packed_tc_supported(p, D, DGPT_BF16)) {
    set_error("packed_wait_probe: the tensor-core kernel does not cover head_dim %d", D);
    return DGPT_E_UNSUPPORTED;
  }
  return packed_tc(p, D, static_cast<cudaStream_t>(stream), limit_cycles);
}

// One round of CTAs: a share is as long as its sequences allow.  The tensor-core kernel takes 128 rows an item and one CTA an SM; shares of its below two tiles
// of 128 keys, or beyond one round, write, read and join partial rows for nothing.  On the CUDA cores a tile of 64 keys takes so long that tiles of 16 rows are worth
// a share each (four CTAs an SM), and tiles of 64 rows two (two CTAs an SM); up to 128 keys the second pass costs what it saves.
// (us, bf16: 3 sequences of 40000 to 65000 keys, 64 drafts, 1 share 495, 6 as chosen 99, 8 134; 48 of 300 to 4000, 1 as chosen 53, 2 75; 8 of them 46, 4 as chosen 24, 8
// 28; one draft behind 2000 keys 26, 8 as chosen 13.4.  fp32, heads of 16: 24 sequences of 30 to 500 keys, 13 drafts, 1 share 12.2, 2 11.0, 6 as chosen 9.5; 2000 keys, 150
// drafts, 1 83, 17 as chosen 19, 24 15, 32 20; heads of 64: 1500 keys, one draft, 1 64, 6 15, 24 as chosen 8.5.  Where the number of shares and of tiles just miss one
// another the rule is up to a quarter behind the best number: 24 above, or 4 sequences of 800 keys, 40 drafts, heads of 32, 6 as chosen 13.1, 7 11.1; 64 of 1000, 4 drafts, heads of
// 128, 2 as chosen 77, 4 69.  It sees sizes only: a bf16 layout that the tensor-core kernel does not cover gets its number all the same.)
extern "C" int32_t dgpt_tree_attn_splits(int32_t B, int32_t T, int32_t H, int32_t G, int32_t D, int32_t max_keys, int32_t dtype) {
  if (B <= 0 || T <= 0 || H <= 0 || G <= 0 || H % G != 0 || max_keys <= 0) return 1;
  const bool tensor = dtype == DGPT_BF16 && D >= 32;
  const long long group = H / G, rows = T * group;
  long long tiles, ctas, least;
  if (tensor) {
    const long long nodes = group < 128 ? 128 / group : 1;
    tiles = (T + nodes - 1) / nodes;
    ctas = 148;
    least = 256;
  } else {
    tiles = rows <= 16 ? 1 : (rows + 63) / 64;
    ctas = (rows <= 16 ? 4 : 2) * 148;
    least = rows <= 16 ? 64 : 128;
  }
  const long long items = (long long)B * G * tiles, fit = ctas / items, most = max_keys <= 128 ? 1 : ((long long)max_keys + least - 1) / least;
  const long long n = fit < most ? fit : most;
  return (int32_t)(n < 1 ? 1 : n > 256 ? 256 : n);
}

extern "C" size_t dgpt_tree_attn_workspace_bytes(int32_t B, int32_t T, int32_t H, int32_t D, int32_t n_splits) {
  if (B <= 0 || T <= 0 || H <= 0 || D <= 0 || n_splits <= 1) return 0;
  return ((size_t)B * T * H * n_splits * (D + 1) * sizeof(float) + 15) / 16 * 16;
}

extern "C" int dgpt_tree_attn(const void* q, int64_t q_row_stride, const dgpt_kv_layout* kv, int64_t kv_token_stride, const int32_t* ctx_len,
                              const int32_t* gap_start, const int32_t* gap_end, const int32_t* n_nodes, const uint64_t* ancestors, int32_t words, void* out, int64_t out_row_stride,
                              void* workspace, size_t workspace_bytes, int32_t n_splits, int32_t B, int32_t T, int32_t H, int32_t G, int32_t D,
                              float scale, int32_t dtype, int32_t impl, int32_t* status, void* stream) {
  DGPT_REQUIRE(B >= 0 && T >= 0 && H > 0 && G > 0 && H % G == 0, "tree_attn: bad sizes");
  DGPT_REQUIRE(T <= 256, "tree_attn: at most 256 drafted tokens per sequence, got %d", T);
  DGPT_REQUIRE((long long)words * 64 >= T && words <= 4, "tree_attn: %d words of ancestors do not hold %d nodes", words, T);
  DGPT_REQUIRE(scale > 0.f, "tree_attn: the scale must be positive");
  DGPT_REQUIRE(impl >= 0 && impl <= 2, "tree_attn: impl must be 0 (choose), 1 (CUDA cores) or 2 (tensor cores)");
  DGPT_REQUIRE(n_splits >= 1 && n_splits <= 256, "tree_attn: n_splits must be 1 to 256");
  if (dtype != DGPT_F32 && dtype != DGPT_BF16) {
    set_error("tree_attn: unknown dtype %d", dtype);
    return DGPT_E_UNSUPPORTED;
  }
  if (!head_dim_ok(D)) {
    set_error("tree_attn: head_dim %d is not built", D);
    return DGPT_E_UNSUPPORTED;
  }
  if (B == 0 || T == 0) return DGPT_OK;
  DGPT_REQUIRE(q && ctx_len && ancestors && out, "tree_attn: NULL pointer");
  DGPT_REQUIRE((gap_start == nullptr) == (gap_end == nullptr), "tree_attn: a gap has a start and an end");
  if (int e = validate_kv(kv, D)) return e;
  DGPT_REQUIRE(kv->page_table || kv->n_pages <= 0 || B <= kv->n_pages, "tree_attn: %d sequences in a cache of %lld", B, (long long)kv->n_pages);
  DGPT_REQUIRE(aligned16(q) && aligned16(out), "tree_attn: pointers must be 16-byte aligned");
  DGPT_REQUIRE(q_row_stride >= (int64_t)H * D && out_row_stride >= (int64_t)H * D && q_row_stride % 8 == 0 && out_row_stride % 8 == 0,
               "tree_attn: row strides must be multiples of 8 elements that hold a row");
  DGPT_REQUIRE(kv_token_stride >= D && kv_token_stride % 8 == 0, "tree_attn: the token stride must be a multiple of 8 elements that holds a head");
  DGPT_REQUIRE(kv->head_stride >= 0 && kv->page_stride >= 0 && kv->n_pages >= 0, "tree_attn: strides and pages must not be negative");
  const size_t need = dgpt_tree_attn_workspace_bytes(B, T, H, D, n_splits);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    set_error("tree_attn: workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    return DGPT_E_WORKSPACE;
  }
  DGPT_REQUIRE(aligned16(workspace), "tree_attn: the workspace must be 16-byte aligned");
  TreeProblem p;
  p.q = q;
  p.q_rs = q_row_stride;
  p.kv = make_view(kv);
  p.kv.token_stride = kv_token_stride;
  p.ctx = ctx_len;
  p.gap_start = gap_start;
  p.gap_end = gap_end;
  p.n_nodes = n_nodes;
  p.ancestors = reinterpret_cast<const unsigned long long*>(ancestors);
  p.words = words;
  p.o = out;
  p.o_rs = out_row_stride;
  p.part_o = static_cast<float*>(workspace);
  p.part_lse = n_splits > 1 ? p.part_o + (size_t)B * T * H * n_splits * D : nullptr;
  p.n_splits = n_splits;
  p.B = B; p.T = T; p.H = H; p.G = G; p.D = D;
  p.group = H / G;
  p.rows_per_tile = p.tiles = p.tile_keys = 0;
  p.scale_log2 = scale * kLog2e;
  p.status = status;
  p.wait_limit = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool tensor = tree_tc_supported(p, dtype);
  if (impl == 2 && !tensor) {
    set_error("tree_attn: the tensor-core kernel does not cover dtype %d, head_dim %d with this layout", dtype, D);
    return DGPT_E_UNSUPPORTED;
  }
  const bool tc = tensor && impl != 1;
  const int rc = tc ? tree_tc(p, st) : tree_simt(p, dtype, st);
  if (rc != DGPT_OK || n_splits == 1) return rc;
  return tree_merge(p, tc ? 128 : 64, dtype, st);
}
