// Log probability of a given token per row of logits, the entropy of the row's distribution, and its most probable tokens.
//   z = logits / temperature,  lse = log sum_j e^(z_j):   logprob = z_target - lse,   entropy = lse - sum_j p_j z_j,   p_j = e^(z_j - lse)
// in one pass over the row.  With x_j = (logit_j - m) c, m the running maximum and c = log2(e) / temperature, a thread carries s = sum 2^x
// and w = sum x 2^x; then lse = m / temperature + ln s and entropy = (log2 s - w / s) ln 2, and when m moves, by d = (old - new) c, s <- s 2^d and
// w <- (w + d s) 2^d.  (The difference first, then the factor: m c alone would be rounded, which logits of the type's lowest value turn into more than
// any exponent holds.)
//
// The top tokens come from the same pass.  A token's key is its logit, made an unsigned number of the same order, above the
// complement of its index: keys differ, and ties go to the lower index.  Each thread knows the vector with its largest logit; the k-th
// largest of 32 maxima over groups of threads is a key that at least k tokens reach, so the top k lie among the tokens that reach it:
// a few dozen, all read by the few threads whose own maximum reaches it.  Those threads' vectors are read again (from L2, one in twenty or so of the row)
// and the tokens found are ranked by counting.
//
// A cluster of 1 to 8 CTAs shares a row where rows are few; its first CTA joins the others' sums and lists through distributed shared memory.
// What bounds it: one read of the logits.
#include "common.cuh"

namespace dgpt {

constexpr int kLpMost = 32;       // most top tokens
constexpr float kLpFar = -1e4f;  // an exponent whose power is 0: keeps 0 times infinity out of the sums
constexpr int kLpFound = 1024;    // tokens found above the bound that are ranked at once

__device__ __forceinline__ uint32_t lp_order(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 is 0
  if (v != v) return 0u;                        // not a number: behind everything
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t k) {
  return k == 0u ? __int_as_float(0x7fc00000) : __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long lp_key(float v, int index) {
  return ((unsigned long long)lp_order(v) << 32) | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ uint32_t lp_map(const void* p, uint32_t rank) {  // a shared address of another CTA of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float lp_ld_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ unsigned long long lp_ld_u64(uint32_t a) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void lp_cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct LpStat {  // sums against the largest logit m met; -inf: nothing yet
  float m, s, w;
};
__device__ __forceinline__ LpStat lp_join(const LpStat& a, const LpStat& b, float c) {
  LpStat r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  const float da = fmaxf((a.m - ref) * c, kLpFar), db = fmaxf((b.m - ref) * c, kLpFar);  // m = -inf: the sums are 0 (or not numbers)
  const float fa = lp_exp2(da), fb = lp_exp2(db);
  r.s = a.s * fa + b.s * fb;
  r.w = (a.w + a.s * da) * fa + (b.w + b.s * db) * fb;
  return r;
}

struct LpParams {
  const void* logits;
  long long stride;
  const int* targets;
  float *logprob, *entropy, *top_logprobs;
  int* top_ids;
  int R, V, k;
  float c, inv_t;  // log2(e) / temperature, 1 / temperature
  int* status;
};

// A row as vectors of 16 bytes from the boundary at or before its first element; vector 0 and the last may be partly outside.
template <typename T>
struct LpRow {
  static constexpr int VEC = Io<T>::kVec16;
  const T* row;
  int off, V, n;  // elements between the boundary and the row, vectors
  __device__ LpRow(const T* r, int v) : row(r), V(v) {
    off = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    n = (off + V + VEC - 1) / VEC;
  }
  __device__ int first(int vec) const { return vec * VEC - off; }  // index of a vector's first element
  __device__ bool whole(int vec) const { return first(vec) >= 0 && first(vec) + VEC <= V; }
  __device__ void load(int vec, float (&x)[VEC]) const {
    if (whole(vec)) {
      unpack16<T>(__ldg(reinterpret_cast<const uint4*>(row + first(vec))), x);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int j = first(vec) + i;
        x[i] = j >= 0 && j < V ? Io<T>::ld(row + j) : -INFINITY;  // adds nothing to the sums
      }
    }
  }
};

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(const LpParams p, const int cluster) {
  constexpr int VEC = Io<T>::kVec16, WARPS = THREADS / 32, UNROLL = 4;
  __shared__ unsigned long long bound[WARPS][32];
  __shared__ unsigned long long found[kLpFound];
  __shared__ unsigned long long best[8 * kLpMost];  // this CTA's top k in order; in the first CTA then those of all
  __shared__ unsigned long long limit;
  __shared__ int n_found, n_owners;
  __shared__ short owners[THREADS];
  __shared__ float stat[WARPS][3];
  __shared__ float mine[3];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = (int)(blockIdx.x / (unsigned)cluster), rank = (int)(blockIdx.x % (unsigned)cluster);
  const LpRow<T> row(static_cast<const T*>(p.logits) + (long long)r * p.stride, p.V);
  const int v0 = (int)((long long)row.n * rank / cluster), v1 = (int)((long long)row.n * (rank + 1) / cluster);

  float top = -INFINITY;  // this thread's largest logit, and the vector it was first met in
  int top_vec = -1;
  LpStat a = {-INFINITY, 0.f, 0.f};
  for (int base = v0 + tid; base < v1; base += THREADS * UNROLL) {
    float x[UNROLL][VEC];
    float vm[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int vec = base + u * THREADS;
      if (vec < v1) {
        row.load(vec, x[u]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[u][i] = -INFINITY;
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      vm[u] = x[u][0];
#pragma unroll
      for (int i = 1; i < VEC; ++i) vm[u] = fmaxf(vm[u], x[u][i]);
      const int vec = base + u * THREADS;
      if (vec < v1 && vm[u] == vm[u] && (vm[u] > top || top_vec < 0)) {  // the first of equal ones stays
        top = vm[u];
        top_vec = vec;
      }
    }
    if (top > a.m) {
      const float d = fmaxf((a.m - top) * p.c, kLpFar), f = lp_exp2(d);
      a.w = (a.w + a.s * d) * f;
      a.s *= f;
      a.m = top;
    }
    const float ref = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float y = (x[u][i] - ref) * p.c, e = lp_exp2(y);
        a.s += e;
        a.w = fmaf(e, fmaxf(y, kLpFar), a.w);
      }
  }
  // ---- the sums of the CTA ----
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpStat b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
    a = lane & o ? lp_join(b, a, p.c) : lp_join(a, b, p.c);  // the same sum in both lanes
  }
  if (lane == 0) {
    stat[warp][0] = a.m;
    stat[warp][1] = a.s;
    stat[warp][2] = a.w;
  }
  // ---- its top k ----
  if (p.k > 0) {
    // The key of this thread's largest logit lies between these two, by its vector's first and last element.
    const unsigned long long low = top_vec < 0 ? 0ull : lp_key(top, min(row.first(top_vec) + VEC - 1, p.V - 1));
    const unsigned long long high = top_vec < 0 ? 0ull : lp_key(top, max(row.first(top_vec), 0));
    bound[warp][lane] = low;
    if (tid == 0) n_found = n_owners = 0;
    __syncthreads();
    if (warp == 0) {
      unsigned long long g = 0ull;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) g = max(g, bound[w][lane]);
      int above = 0;
      for (int i = 0; i < 32; ++i) {
        const unsigned long long o = __shfl_sync(0xffffffffu, g, i);
        above += o > g || (o == g && i < lane);
      }
      if (above == p.k - 1) limit = g;
    }
    __syncthreads();
    unsigned long long lim = limit;
    if (high >= lim) owners[atomicAdd(&n_owners, 1)] = (short)tid;  // (bound 0: fewer maxima than k, everything is looked at)
    __syncthreads();
    const int per = (v1 - v0 + THREADS - 1) / THREADS;  // vectors of a thread
    const long long todo = (long long)n_owners * per;
    for (;;) {
      for (long long i = tid; i < todo; i += THREADS) {
        const int vec = v0 + owners[i / per] + (int)(i % per) * THREADS;
        if (vec >= v1) continue;
        float x[VEC];
        row.load(vec, x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int j = row.first(vec) + e;
          if (j < 0 || j >= p.V) continue;
          const unsigned long long key = lp_key(x[e], j);
          if (key >= lim) {
            const int at = atomicAdd(&n_found, 1);
            if (at < kLpFound) found[at] = key;
          }
        }
      }
      __syncthreads();
      const int n = min(n_found, kLpFound);
      const bool again = n_found > kLpFound;
      if (tid < p.k) best[tid] = 0ull;
      __syncthreads();
      for (int i = tid; i < n; i += THREADS) {
        const unsigned long long key = found[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += found[j] > key;
        if (above < p.k) best[above] = key;
      }
      __syncthreads();
      if (!again) break;
      // More tokens reach the bound than there is room for: the k-th of those that were kept is a higher one.
      lim = best[p.k - 1];
      if (tid == 0) n_found = 0;
      __syncthreads();
    }
  } else {
    __syncthreads();
  }
  if (warp == 0) {
    LpStat b = {-INFINITY, 0.f, 0.f};
    for (int w = 0; w < WARPS; ++w) b = lp_join(b, LpStat{stat[w][0], stat[w][1], stat[w][2]}, p.c);
    a = b;
    if (lane == 0) {
      mine[0] = a.m;
      mine[1] = a.s;
      mine[2] = a.w;
    }
  }
  if (cluster > 1) {
    __syncthreads();
    lp_cluster_sync();
    unsigned long long key = 0ull;
    if (rank == 0) {
      if (warp == 0) {
        a = LpStat{-INFINITY, 0.f, 0.f};
        for (int c = 0; c < cluster; ++c)
          a = lp_join(a, LpStat{lp_ld_f32(lp_map(&mine[0], c)), lp_ld_f32(lp_map(&mine[1], c)), lp_ld_f32(lp_map(&mine[2], c))}, p.c);
      }
      if (tid < cluster * p.k) key = lp_ld_u64(lp_map(&best[tid % p.k], tid / p.k));
    }
    lp_cluster_sync();  // the others may leave
    if (rank != 0) return;
    if (p.k > 0) {
      if (tid < cluster * p.k) found[tid] = key;
      __syncthreads();
      if (tid < cluster * p.k) {
        int above = 0;
        for (int j = 0; j < cluster * p.k; ++j) above += found[j] > key || (found[j] == key && j < tid);
        if (above < p.k) best[above] = key;
      }
      __syncthreads();
    }
  }
  if (warp == 0) {
    const float log_s = log2f(a.s);
    // nothing but -inf, or something that is not a number or +inf: no distribution
    const bool none = !(a.s > 0.f) || !(a.m < INFINITY);
    const float nan = __int_as_float(0x7fc00000);
    auto logprob = [&](float z) { return none ? nan : fmaf(z - a.m, p.inv_t, -log_s * kLn2); };
    if (lane == 0) {
      const int t = p.targets[r];
      const bool ok = t >= 0 && t < p.V;
      if (!ok && p.status) atomicOr(p.status, 4);
      p.logprob[r] = ok ? logprob(Io<T>::ld(row.row + t)) : nan;
      p.entropy[r] = none ? nan : fmaxf((log_s - a.w / a.s) * kLn2, 0.f);
    }
    if (lane < p.k) {
      const unsigned long long key = best[lane];
      p.top_ids[(long long)r * p.k + lane] = (int)(0xffffffffu - (uint32_t)key);
      p.top_logprobs[(long long)r * p.k + lane] = logprob(lp_value((uint32_t)(key >> 32)));
    }
  }
}

template <typename T>
static int logprobs_launch(const LpParams& p, cudaStream_t st) {
  constexpr int THREADS = 256;
  int cluster = 1;
  // one row's vectors over more CTAs while there are SMs without one and each thread keeps a vector
  while (cluster < 8 && (long long)p.R * cluster * 2 <= 296 && p.V / (Io<T>::kVec16 * THREADS) >= cluster * 2) cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.R * cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, THREADS>, p, cluster);
  return launch_status("token_logprobs");
}

}  // namespace dgpt

using namespace dgpt;

extern "C" int dgpt_token_logprobs(const void* logits, int64_t logits_row_stride, const int32_t* targets, float temperature, float* logprob,
                                   float* entropy, int32_t* top_ids, float* top_logprobs, int32_t top_k, int32_t R, int32_t V, int32_t dtype,
                                   int32_t* status, void* stream) {
  DGPT_REQUIRE(R >= 0 && V > 0 && V <= 0x7fffff00, "token_logprobs: bad sizes");
  DGPT_REQUIRE(top_k >= 0 && top_k <= kLpMost && top_k <= V, "token_logprobs: top_k must be 0 to %d and at most the vocabulary, got %d", kLpMost, top_k);
  DGPT_REQUIRE(temperature > 0.f && temperature < INFINITY, "token_logprobs: the temperature must be positive and finite");
  DGPT_REQUIRE(R <= 0x0fffffff, "token_logprobs: too many rows");
  if (dtype != DGPT_F32 && dtype != DGPT_BF16) {
    set_error("token_logprobs: unknown dtype %d", dtype);
    return DGPT_E_UNSUPPORTED;
  }
  if (R == 0) return DGPT_OK;
  DGPT_REQUIRE(logits && targets && logprob && entropy && (top_k == 0 || (top_ids && top_logprobs)), "token_logprobs: NULL pointer");
  DGPT_REQUIRE(logits_row_stride >= V || R == 1, "token_logprobs: rows overlap");
  DGPT_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == DGPT_F32 ? 4 : 2) == 0, "token_logprobs: logits are not aligned to their type");
  LpParams p = {logits, R == 1 ? (int64_t)V : logits_row_stride, targets, logprob, entropy, top_logprobs, top_ids, R, V, top_k, kLog2e / temperature, 1.f / temperature, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DGPT_F32 ? logprobs_launch<float>(p, st) : logprobs_launch<__nv_bfloat16>(p, st);
}
