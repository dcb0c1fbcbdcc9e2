// Attention of packed prompts and of trees of drafted tokens on the CUDA cores: fp32, heads of 8 and 16, and layouts whose pages the
// tensor-core kernel cannot tile.
//
// A CTA of 256 threads owns a tile of BM rows and walks through its keys 64 at a time with the running maximum and sum of a softmax.
// Q, K, V and the probabilities of a step lie in shared memory as fp32; a row belongs to 16 or 32 threads of one warp, each with 4 or 2 rows, its share of
// a step's scores and of the output's columns, so that a number fetched from shared memory feeds several products and no barrier stands between the two products.
// fp32 products stay on the FMA units, whose rate is the floor (three bf16 parts per operand on the tensor cores would come close to 24 bits: not tried).  What bounds it: reads of shared memory and the softmax's shuffles
// between the products (8 prompts of 700, 8 heads of 64, 171 us, 54 at the FMA rate), and for small ones the chain of a CTA's few steps (32 of 20 to 140, 4
// heads of 16, 14 us).  Trees of up to 16 rows take tiles of 16 (24 trees of 13 drafts behind 30 to 500 keys in one share 12.2 us, with 64 rows 18.2; in six, as chosen, 9.5 and 15.2).
#include "ragged.cuh"

namespace dgpt {

// 2^x within 2 units of the last place; -inf gives 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int kRgThreads = 256;
constexpr int kRgBN = 64;

template <typename T, int D, int BM, class P, bool TREE>
__global__ void __launch_bounds__(kRgThreads) ragged_simt_kernel(const P p) {
  // Threads that share a row.  (16 and 32, us: tiles of 16 rows, heads of 64, 8 drafts behind 2000 keys 97 and 81, one behind 1500 75 and 64; tiles of 64, 8 prompts
  // of 700 171 and 199, 32 of 80 with heads of 16 7.1 and 8.3.)
  constexpr int LX = BM == 16 ? 32 : 16;
  constexpr int RM = BM * LX / kRgThreads;     // rows per thread
  constexpr int KC = kRgBN / LX;               // score columns per thread
  constexpr int CO = D >= LX ? D / LX : 1;     // output columns per thread
  constexpr int CV = CO < 4 ? CO : 4;          // of which lie side by side, so that a row's threads read neighbouring pieces of a value's row
  constexpr int KG = D >= LX ? 1 : LX / D;     // threads that share a step's keys of an output column
  constexpr int VEC = Io<T>::kVec16, VPR = D / VEC;
  constexpr int PITCH = D + 4, PPITCH = kRgBN + 4;
  extern __shared__ __align__(16) float sm[];
  float* Qs = sm;                      // [BM][PITCH]
  float* Ks = Qs + BM * PITCH;         // [64][PITCH]
  float* Vs = Ks + kRgBN * PITCH;      // [64][PITCH]
  float* Ps = Vs + kRgBN * PITCH;      // [BM][PPITCH]

  const int tid = threadIdx.x, tx = tid % LX, row0 = tid / LX * RM, group = tx / (LX / KG);
  auto column = [&](int c) { return c / CV * LX * CV + tx % (LX / KG) * CV + c % CV; };
  p.check(blockIdx.x == 0, tid, kRgThreads);
  RaggedItem it;
  if constexpr (TREE) {
    if (!p.item(blockIdx.x, kRgBN, it) || (p.n_splits > 1 && it.key0 >= it.key1)) return;
  } else {
    const unsigned slot = blockIdx.x / (unsigned)p.H;
    typename P::Cursor cur;
    p.load(p.find((int)slot, BM, tid & 31), BM, cur);
    if (!p.item((int)slot, cur, (int)(blockIdx.x - slot * (unsigned)p.H), BM, it)) return;
  }
  for (int i = tid; i < BM * VPR; i += kRgThreads) {
    const int r = i / VPR, c = i - r * VPR;
    float t[VEC];
    if (r < it.rows) {
      ld16<T>(p.template q_row<T>(it, r) + c * VEC, t);
#pragma unroll
      for (int x = 0; x < VEC; ++x) t[x] *= p.scale_log2;
    } else {
#pragma unroll
      for (int x = 0; x < VEC; ++x) t[x] = 0.f;
    }
#pragma unroll
    for (int x = 0; x < VEC; x += 4) *reinterpret_cast<float4*>(&Qs[r * PITCH + c * VEC + x]) = make_float4(t[x], t[x + 1], t[x + 2], t[x + 3]);
  }
  float m[RM], l[RM], acc[RM][CO];  // l: of this thread's keys
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < CO; ++c) acc[i][c] = 0.f;
  }
  // A step's keys and values are on their way in registers while the step before is worked on.
  constexpr int NV = (kRgBN * VPR + kRgThreads - 1) / kRgThreads;
  uint4 kr[NV], vr[NV];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = tid + u * kRgThreads, jj = i / VPR, c = i - jj * VPR, j = j0 + jj;
      kr[u] = vr[u] = make_uint4(0u, 0u, 0u, 0u);
      if (jj < kRgBN && j < it.key1) {
        if constexpr (TREE) {
          const long long off = p.key_offset(it, j);
          if (off >= 0) {
            kr[u] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.kv.k) + off + c * VEC));
            vr[u] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.kv.v) + off + c * VEC));
          }
        } else {
          kr[u] = __ldg(reinterpret_cast<const uint4*>(p.template k_row<T>(it, j) + c * VEC));
          vr[u] = __ldg(reinterpret_cast<const uint4*>(p.template v_row<T>(it, j) + c * VEC));
        }
      }
    }
  };
  fetch(it.key0);
  for (int j0 = it.key0; j0 < it.key1; j0 += kRgBN) {
    __syncthreads();  // Q is in place; the last step's K, V and P have been read
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = tid + u * kRgThreads, jj = i / VPR, c = i - jj * VPR;
      if (jj >= kRgBN) continue;
      float kf[VEC], vf[VEC];
      unpack16<T>(kr[u], kf);
      unpack16<T>(vr[u], vf);
#pragma unroll
      for (int x = 0; x < VEC; x += 4) {
        *reinterpret_cast<float4*>(&Ks[jj * PITCH + c * VEC + x]) = make_float4(kf[x], kf[x + 1], kf[x + 2], kf[x + 3]);
        *reinterpret_cast<float4*>(&Vs[jj * PITCH + c * VEC + x]) = make_float4(vf[x], vf[x + 1], vf[x + 2], vf[x + 3]);
      }
    }
    __syncthreads();
    if (j0 + kRgBN < it.key1) fetch(j0 + kRgBN);
    if (tid / 32 * 32 / LX * RM >= it.rows) continue;  // none of this warp's rows exists
    // scores: rows row0 + i, keys tx + LX j
    float s[RM][KC];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < KC; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 a[RM], b[KC];
#pragma unroll
      for (int i = 0; i < RM; ++i) a[i] = *reinterpret_cast<const float4*>(&Qs[(row0 + i) * PITCH + d]);
#pragma unroll
      for (int j = 0; j < KC; ++j) b[j] = *reinterpret_cast<const float4*>(&Ks[(tx + LX * j) * PITCH + d]);
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < KC; ++j) s[i][j] = fmaf(a[i].w, b[j].w, fmaf(a[i].z, b[j].z, fmaf(a[i].y, b[j].y, fmaf(a[i].x, b[j].x, s[i][j]))));
    }
    const bool masked = j0 + kRgBN > it.clear || j0 + kRgBN > it.key1 || (j0 < it.gap1 && j0 + kRgBN > it.gap0);
    if (masked) {
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          const int key = j0 + tx + LX * j;
          if (row0 + i >= it.rows || key >= it.key1 || !p.sees(it, row0 + i, key)) s[i][j] = -INFINITY;
        }
    }
    float top[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      top[i] = s[i][0];
#pragma unroll
      for (int j = 1; j < KC; ++j) top[i] = fmaxf(top[i], s[i][j]);
    }
#pragma unroll
    for (int x = LX / 2; x > 0; x >>= 1)
#pragma unroll
      for (int i = 0; i < RM; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], x));
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const float mn = fmaxf(m[i], top[i]), ref = mn == -INFINITY ? 0.f : mn;
      const float f = ex2(m[i] - ref);  // m = -inf: 0
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const float e = ex2(s[i][j] - ref);
        sum += e;
        Ps[(row0 + i) * PPITCH + tx + LX * j] = e;
      }
      m[i] = mn;
      l[i] = fmaf(l[i], f, sum);
#pragma unroll
      for (int c = 0; c < CO; ++c) acc[i][c] *= f;
    }
    __syncwarp();
    // output: the same rows (a row's threads are of one warp), columns column(c), every KG-th four keys
#pragma unroll 2
    for (int j = group * 4; j < kRgBN; j += 4 * KG) {
      float4 w[RM];
#pragma unroll
      for (int i = 0; i < RM; ++i) w[i] = *reinterpret_cast<const float4*>(&Ps[(row0 + i) * PPITCH + j]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        alignas(16) float b[CO];
#pragma unroll
        for (int c = 0; c < CO; c += CV) {
          const float* from = &Vs[(j + x) * PITCH + column(c)];
          if constexpr (CV == 4) *reinterpret_cast<float4*>(&b[c]) = *reinterpret_cast<const float4*>(from);
          else if constexpr (CV == 2) *reinterpret_cast<float2*>(&b[c]) = *reinterpret_cast<const float2*>(from);
          else b[c] = *from;
        }
#pragma unroll
        for (int i = 0; i < RM; ++i) {
          const float e = x == 0 ? w[i].x : x == 1 ? w[i].y : x == 2 ? w[i].z : w[i].w;
#pragma unroll
          for (int c = 0; c < CO; ++c) acc[i][c] = fmaf(e, b[c], acc[i][c]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int r = row0 + i;
#pragma unroll
    for (int x = LX / 2; x > 0; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
#pragma unroll
    for (int x = LX / KG; x < LX; x <<= 1)
#pragma unroll
      for (int c = 0; c < CO; ++c) acc[i][c] += __shfl_xor_sync(0xffffffffu, acc[i][c], x);
    if (r >= it.rows) continue;
    // !(l <= 0): a row with a key that is not a number keeps saying so
    const bool any = !(l[i] <= 0.f);
    const float inv = any ? 1.f / l[i] : 0.f;
    if constexpr (TREE) {
      const long long row = p.out_row(it, r);
      const int h = p.head(it, r);
      if (p.n_splits > 1) {
        const long long at = ((long long)it.split * p.B * p.T + row) * p.H + h;
        if (group == 0) {
#pragma unroll
          for (int c = 0; c < CO; ++c) p.part_o[at * D + column(c)] = any ? acc[i][c] * inv : 0.f;
        }
        if (tx == 0) p.part_lse[at] = any ? m[i] + log2f(l[i]) : -INFINITY;
        continue;
      }
      if (group == 0) {
        T* o = static_cast<T*>(p.o) + row * p.o_rs + (long long)h * D;
#pragma unroll
        for (int c = 0; c < CO; ++c) Io<T>::st(o + column(c), any ? acc[i][c] * inv : 0.f);
      }
    } else {
      if (group == 0) {
        T* o = static_cast<T*>(p.o) + (long long)(it.row0 + r) * p.o_rs + (long long)it.h * p.o_hs;
#pragma unroll
        for (int c = 0; c < CO; ++c) Io<T>::st(o + column(c), any ? acc[i][c] * inv : 0.f);
      }
      if (tx == 0 && p.lse) p.lse[(long long)(it.row0 + r) * p.H + it.h] = any ? (m[i] + log2f(l[i])) * kLn2 : -INFINITY;
    }
  }
}

template <typename T, int D, int BM, class P, bool TREE>
static int ragged_simt_go(const P& p, long long ctas, cudaStream_t st) {
  constexpr size_t smem = ((size_t)(BM + 2 * kRgBN) * (D + 4) + (size_t)BM * (kRgBN + 4)) * sizeof(float);
  auto kernel = ragged_simt_kernel<T, D, BM, P, TREE>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) {
    set_error("ragged attention: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    return DGPT_E_CUDA;
  }
  kernel<<<(unsigned)ctas, kRgThreads, smem, st>>>(p);
  return launch_status("ragged attention");
}

#define DGPT_BY_TYPE(GO)                                        \
  do {                                                          \
    if (dtype == DGPT_F32) {                                    \
      switch (D) {                                              \
        case 8: GO(float, 8);                                   \
        case 16: GO(float, 16);                                 \
        case 32: GO(float, 32);                                 \
        case 64: GO(float, 64);                                 \
        case 128: GO(float, 128);                               \
      }                                                         \
    } else if (dtype == DGPT_BF16) {                            \
      switch (D) {                                              \
        case 8: GO(__nv_bfloat16, 8);                           \
        case 16: GO(__nv_bfloat16, 16);                         \
        case 32: GO(__nv_bfloat16, 32);                         \
        case 64: GO(__nv_bfloat16, 64);                         \
        case 128: GO(__nv_bfloat16, 128);                       \
      }                                                         \
    }                                                           \
    set_error("ragged attention: dtype %d with head_dim %d is not built", dtype, D); \
    return DGPT_E_UNSUPPORTED;                                  \
  } while (0)

int packed_simt(const PackedProblem& p, int D, int dtype, cudaStream_t st) {
  const long long ctas = p.slots(64) * p.H;
  DGPT_REQUIRE(ctas <= 0x7fffffffll, "fmha_packed: too many rows");
#define DGPT_GO(T, DD) return ragged_simt_go<T, DD, 64, PackedProblem, false>(p, ctas, st)
  DGPT_BY_TYPE(DGPT_GO);
#undef DGPT_GO
}

int tree_simt(const TreeProblem& full, int dtype, cudaStream_t st) {
  TreeProblem p = full;
  const int D = p.D, rows = p.T * p.group, bm = rows <= 16 ? 16 : 64;
  p.rows_per_tile = bm;
  p.tiles = (rows + bm - 1) / bm;
  const long long ctas = p.items();
  DGPT_REQUIRE(ctas <= 0x7fffffffll, "tree_attn: too many rows");
#define DGPT_GO(T, DD)                                                                   \
  return bm == 16 ? ragged_simt_go<T, DD, 16, TreeProblem, true>(p, ctas, st)           \
                  : ragged_simt_go<T, DD, 64, TreeProblem, true>(p, ctas, st)
  DGPT_BY_TYPE(DGPT_GO);
#undef DGPT_GO
}

// ---- partials of a tree's rows into one -------------------------------------------------------------------------
// One warp per (row, head): y = sum_s 2^(lse_s - m) o_s / sum_s 2^(lse_s - m), with the running maximum m, STEP shares at a time.  Their loads, and
// those of the lengths that say how many shares there are, do not wait for one another (what is read of shares that were not written counts for nothing).
template <typename T, int STEP>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeProblem p) {
  dep_wait();
  const long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), n = (long long)p.B * p.T * p.H;
  if (at >= n) return;
  const int lane = threadIdx.x & 31, h = (int)(at % p.H);
  const long long row = at / p.H;
  const int s = (int)(row / p.T), t = (int)(row - (long long)s * p.T);
  const bool mine = lane * 4 < p.D;  // columns lane * 4 .. (D <= 128)
  int splits = p.n_splits;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, total = 0.f, m = -INFINITY;
  for (int i0 = 0; i0 < splits; i0 += STEP) {
    float lse[STEP];
    float4 v[STEP];
#pragma unroll
    for (int u = 0; u < STEP; ++u) {
      const long long slot = min(i0 + u, p.n_splits - 1) * n + at;
      lse[u] = p.part_lse[slot];
      v[u] = mine ? *reinterpret_cast<const float4*>(p.part_o + slot * p.D + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (i0 == 0) {
      if (p.n_nodes && t >= p.n_nodes[s]) return;
      int context, nodes;
      p.lengths(s, context, nodes);
      splits = min(p.n_splits, (context + nodes + p.tile_keys - 1) / p.tile_keys);  // the ones behind have no keys
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < STEP; ++u) {
      if (i0 + u >= splits) lse[u] = -INFINITY;
      top = fmaxf(top, lse[u]);
    }
    const float ref = top == -INFINITY ? 0.f : top, f = ex2(m - ref);
    m = top;
    total *= f;
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] *= f;
#pragma unroll
    for (int u = 0; u < STEP; ++u) {
      if (lse[u] == -INFINITY) continue;  // no key of this share is seen
      const float w = ex2(lse[u] - ref);
      total += w;
      acc[0] = fmaf(w, v[u].x, acc[0]);
      acc[1] = fmaf(w, v[u].y, acc[1]);
      acc[2] = fmaf(w, v[u].z, acc[2]);
      acc[3] = fmaf(w, v[u].w, acc[3]);
    }
  }
  if (!mine) return;
  const bool any = !(total <= 0.f);
  const float inv = any ? 1.f / total : 0.f;
  T* o = static_cast<T*>(p.o) + row * p.o_rs + (long long)h * p.D + lane * 4;
#pragma unroll
  for (int c = 0; c < 4; ++c) Io<T>::st(o + c, any ? acc[c] * inv : 0.f);
}

int tree_merge(const TreeProblem& full, int tile_keys, int dtype, cudaStream_t st) {
  TreeProblem p = full;
  p.tile_keys = tile_keys;
  const long long rows = (long long)p.B * p.T * p.H;
  const dim3 grid((unsigned)((rows + 7) / 8));
  // Eight shares at a time where there are more than four (one sequence of 30000 keys in 37: 25.9 us in fours, 24.5 so; 16 sequences in two: 31.2 and 33.0).
  const bool many = p.n_splits > 4;
  if (dtype == DGPT_F32) launch_few(true, many ? tree_merge_kernel<float, 8> : tree_merge_kernel<float, 4>, grid, dim3(256), 0, st, p);
  else launch_few(true, many ? tree_merge_kernel<__nv_bfloat16, 8> : tree_merge_kernel<__nv_bfloat16, 4>, grid, dim3(256), 0, st, p);
  return launch_status("tree_attn");
}

}  // namespace dgpt
