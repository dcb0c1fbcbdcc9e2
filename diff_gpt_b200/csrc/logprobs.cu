// Log probability of a given token per row of logits, the entropy of the row's distribution, and its most probable tokens.
//   z = logits / temperature,  lse = log sum_j e^(z_j):   logprob = z_target - lse,   entropy = lse - sum_j p_j z_j,   p_j = e^(z_j - lse)
// in one pass over the row.  With c = log2(e) / temperature, M = m c rounded, m the running maximum, and x_j = logit_j c - M (one fma), a thread
// carries s = sum 2^x and w = sum x 2^x; then lse = (M + log2 s) ln 2 and entropy = (log2 s - w / s) ln 2, and when M moves by d = old - new,
// s <- s 2^d and w <- (w + d s) 2^d.  How M was rounded cancels out, unless it is so large that the rounding itself outgrows an exponent (logits of
// the type's lowest value throughout, temperatures next to 0): M is kept within 2^30, and a row whose maximum lies beyond is summed once more as
// (logit / 2 - m / 2) 2 c, two roundings that need no M (halves, since the difference of two fp32 numbers may have none).  So is every row at a temperature
// above 1.4e20: -inf is raised to -1e30 in the sums, which is nothing only while 1e30 c is far above 2^30.
//
// The top tokens come from the same pass.  A token's key is its logit, made an unsigned number of the same order, above the
// complement of its index: keys differ, and ties go to the lower index.  Each thread knows the vector with its largest logit; the k-th
// largest of 32 maxima over groups of threads is a key that at least k tokens reach, so the top k lie among the tokens that reach it:
// a few dozen.  A thread also keeps the largest logit of every fourth round; the rounds whose largest reaches the bound are read again (from L1 or L2, one
// vector in thirty of the row; all rounds of such threads, one in eight, 93 us for 84 with 20 of 32001)
// and the tokens found are ranked by counting.
//
// Eight warps of a CTA stream a row, a ninth finishes it (sums, top tokens, outputs) while they are at the next one; rows are handed over through
// two buffers.  A cluster of 1 to 8 CTAs shares a row where rows are few; its first CTA joins the others' sums and lists through distributed shared memory.
// What bounds it: one read of the logits, then the exponentials (16 a clock and SM: three quarters of a read's time in bf16) and the instructions
// around them, which is why pairs share them (fma, add, max) and the next vectors are on their way while these are worked on.  4096 rows of
// 32001 bf16 logits: 61 us without top tokens, 76 with 5, 84 with 20; their reading alone takes 40.5.  (A CTA of 256 threads per row whose every warp goes through
// every phase: 132 with 20.)
#include "common.cuh"

namespace dgpt {

constexpr int kLpMost = 32;       // most top tokens
constexpr int kLpStream = 256;    // threads that stream a row; a warp more finishes it
constexpr int kLpCtas = 4;        // of an SM
constexpr float kLpBig = 1073741824.f;  // 2^30: M is kept within it
constexpr float kLpCold = 1.17549435e-38f;  // lowest temperature, the smallest normal number: its reciprocal, and that times log2(e), are finite
constexpr float kLpHot = 1e-20f;  // least c of the sums in one pass: 1e30 c is then 1e10, so what was raised to -1e30 has the power 0 against every M
constexpr float kLpFar = -1e4f;  // an exponent whose power is 0: keeps 0 times infinity out of the sums
constexpr int kLpFound = 512;     // tokens found above the bound that are ranked at once

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
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}
__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct LpStat {  // largest logit m, sums against M (lp_ref(m)); m = -inf: nothing yet
  float m, M, s, w;
};
__device__ __forceinline__ float lp_ref(float m, float c) { return fminf(fmaxf(m * c, -kLpBig), kLpBig); }
// All lanes' sums, the same in every lane: over to the largest maximum, then added.
__device__ __forceinline__ LpStat lp_warp_join(const LpStat& a) {
  LpStat r;
  r.m = warp_max(a.m);
  r.M = warp_max(a.M);
  const float d = fmaxf(a.M - r.M, kLpFar), f = lp_exp2(d);
  r.s = warp_sum(a.s * f);
  r.w = warp_sum((a.w + a.s * d) * f);
  return r;
}
__device__ __forceinline__ uint64_t lp_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void lp_unpack(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t lp_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t lp_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

struct LpParams {
  const void* logits;
  long long stride;
  const int* targets;
  float *logprob, *entropy, *top_logprobs;
  int* top_ids;
  int R, V, k;
  float c, c2, inv2;  // log2(e), 2 log2(e) and 2, each / temperature
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
  // Vectors [whole0(), whole1()) lie in the row from end to end; of the others, at most one on either side, `edge` gives the ones that are.
  __device__ int whole0() const { return off > 0 ? 1 : 0; }
  __device__ int whole1() const { return max((off + V) / VEC, whole0()); }
  __device__ bool edge(int side, int& vec) const {
    vec = side == 0 ? 0 : n - 1;
    return side == 0 ? off > 0 : (off + V) % VEC != 0 && !(n == 1 && off > 0);
  }
  __device__ uint4 inner(int vec) const { return __ldg(reinterpret_cast<const uint4*>(row - off) + vec); }
  static constexpr uint32_t kNothing = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf: adds nothing to the sums
  // Any vector, with nothing where it is outside the row.  (It is read whole: memory is allocated in larger pieces than 16 bytes.  Element by element
  // the two edges of a row of 32001 cost a tenth of its time.)
  __device__ uint4 raw(int vec) const {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row - off) + vec);
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int j = first(vec) + i;
      if (j >= 0 && j < V) continue;
      if constexpr (sizeof(T) == 2) {
        w[i >> 1] = (i & 1) ? (w[i >> 1] & 0xffffu) | (kNothing << 16) : (w[i >> 1] & 0xffff0000u) | (kNothing & 0xffffu);
      } else {
        w[i] = kNothing;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Largest number of some vectors (NaN only where there is nothing else).
template <int N>
__device__ __forceinline__ float lp_top(const uint4 (&v)[N], __nv_bfloat16) {
  auto h = [](uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  };
  uint32_t m = h(h(v[0].x, v[0].y), h(v[0].z, v[0].w));
#pragma unroll
  for (int i = 1; i < N; ++i) m = h(m, h(h(v[i].x, v[i].y), h(v[i].z, v[i].w)));
  return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}
template <int N>
__device__ __forceinline__ float lp_top(const uint4 (&v)[N], float) {
  float m = __uint_as_float(v[0].x);
#pragma unroll
  for (int i = 0; i < N; ++i)
    m = fmaxf(fmaxf(fmaxf(m, __uint_as_float(v[i].x)), __uint_as_float(v[i].y)), fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w)));
  return m;
}
// Pairs of a vector, raised to -1e30 (a -inf times its power 0 is not a number).
__device__ __forceinline__ void lp_pairs(const uint4& v, uint64_t (&p)[4], __nv_bfloat16) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w[i]), "r"(0xf149f149u));  // -9.95e29 twice
    p[i] = lp_pack(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
  }
}
__device__ __forceinline__ void lp_pairs(const uint4& v, uint64_t (&p)[2], float) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("max.NaN.f32 %0, %1, %2;" : "=f"(x[i]) : "f"(__uint_as_float(w[i])), "f"(-1e30f));
  p[0] = lp_pack(x[0], x[1]);
  p[1] = lp_pack(x[2], x[3]);
}

// The k largest of n keys (all different, n <= kLpFound) in order, for one warp: a key's place is the number of larger ones.
__device__ __forceinline__ void lp_rank(unsigned long long* keys, int n, unsigned long long* best, int k, int lane) {
  if (lane < 8) keys[n + lane] = 0ull;  // up to whole rounds
  if (lane < k) best[lane] = 0ull;
  __syncwarp();
  for (int i0 = 0; i0 < n; i0 += 32) {
    const unsigned long long a = i0 + lane < n ? keys[i0 + lane] : 0ull;
    int over = 0;
    for (int j = 0; j < n; j += 8) {
#pragma unroll
      for (int u = 0; u < 8; u += 2) {
        const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(keys + j + u);
        over += (o.x > a) + (o.y > a);
      }
    }
    if (a != 0ull && over < k) best[over] = a;
  }
  __syncwarp();
}

template <int BAR>
__device__ __forceinline__ void lp_bar_sync(int which) { asm volatile("bar.sync %0, %1;" ::"r"(BAR + which), "n"(kLpStream + 32) : "memory"); }
template <int BAR>
__device__ __forceinline__ void lp_bar_arrive(int which) { asm volatile("bar.arrive %0, %1;" ::"r"(BAR + which), "n"(kLpStream + 32) : "memory"); }

template <typename T, int UNROLL>
__global__ void __launch_bounds__(kLpStream + 32, kLpCtas) token_logprobs_kernel(const LpParams p, const int log_cluster) {
  constexpr int VEC = Io<T>::kVec16, STREAM = kLpStream, WARPS = STREAM / 32;
  constexpr int PARTS = UNROLL > 1 ? 4 : 1;  // of a thread's rounds, looked at again one by one (in short rows all together)
  constexpr int kFull = 1, kFree = 3;  // named barriers, one per buffer
  constexpr int kStream = 5;
  __shared__ unsigned long long lows[2][STREAM];                        // what the key of each streaming thread's largest logit is at least
  __shared__ __align__(16) unsigned long long groups[32];
  __shared__ unsigned char owners[WARPS][32 * PARTS];                   // threads and parts of their rounds
  __shared__ __align__(16) unsigned long long founds[2][kLpFound + 8];  // tokens that reach the bound
  __shared__ int mets[2];                                               // how many do (there may be more than there is room for)
  __shared__ unsigned long long limits[2];                              // the bound
  __shared__ unsigned long long bests[2][kLpMost];                      // the top k in order
  __shared__ LpStat stat[2][WARPS], mine;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cluster = 1 << log_cluster;
  const int rank = (int)(blockIdx.x & (unsigned)(cluster - 1)), step = (int)(gridDim.x >> log_cluster), row0 = (int)(blockIdx.x >> log_cluster);
  auto row_of = [&](int r) { return LpRow<T>(static_cast<const T*>(p.logits) + (long long)r * p.stride, p.V); };
  // Whole vectors [part(rank), part(rank + 1)) are this CTA's; the row's partial ones are the first and the last CTA's (threads 0 and 1).
  auto part = [&](const LpRow<T>& w, int i) { return w.whole0() + (int)(((unsigned)(w.whole1() - w.whole0()) * (unsigned)i) >> log_cluster); };

  // A lane's vector: its tokens that reach the bound (`least`: the bound's logit, NaN for a bound of 0: nothing is below it).
  auto look = [&](const LpRow<T>& row, int vec, const uint4& v, unsigned long long lim, float least, int b) {
    float x[VEC];
    unpack16<T>(v, x);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (x[e] < least) continue;
      const int j = row.first(vec) + e;
      if (j < 0 || j >= p.V) continue;
      const unsigned long long key = lp_key(x[e], j);
      if (key < lim) continue;
      const int place = atomicAdd(&mets[b], 1);
      if (place < kLpFound) founds[b][place] = key;
    }
  };
  if (tid < 2) mets[tid] = 0;
  __syncthreads();
  if (warp < WARPS) {
    // ================= streaming warps: the sums, and the tokens that may be among the top k =================
    const uint64_t c2 = lp_pack(p.c, p.c);
    uint4 now[UNROLL];
    auto fetch = [&](const LpRow<T>& w, int base, int v1, uint4 (&to)[UNROLL]) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) to[u] = w.inner(min(base + u * STREAM, v1 - 1));  // (what lies behind is replaced when it is its turn)
    };
    auto begin = [&](int r) {  // the first vectors of a row
      const LpRow<T> w = row_of(r);
      const int v0 = part(w, rank), v1 = part(w, rank + 1);
      if (v1 > v0) fetch(w, v0 + tid, v1, now);
    };
    begin(row0);
    // (more than one row only without a cluster; a row's first vectors are on their way while the one before is finished)
    int n = 0;
    for (int r = row0; r < p.R; r += step, ++n) {
      const LpRow<T> row = row_of(r);
      const int v0 = part(row, rank), v1 = part(row, rank + 1);
      int top_vec = -1;
      // Largest logits of rounds r, r + 4, ..: the upper halves of their numbers, the last round's lowest
      uint32_t part_lo = 0xff80ff80u, part_hi = 0xff80ff80u;
      LpStat a = {-INFINITY, -kLpBig, 0.f, 0.f};
      auto meet = [&](float vm, int vec) {
        if (vm > a.m || (top_vec < 0 && vm == vm)) {  // the first of equal ones stays
          a.m = vm;
          top_vec = vec;
        }
      };
      auto refer = [&]() {  // sums go over to the new maximum
        const float M = lp_ref(a.m, p.c), d = fmaxf(a.M - M, kLpFar), f = lp_exp2(d);
        a.w = (a.w + a.s * d) * f;
        a.s *= f;
        a.M = M;
      };
      auto sum = [&](const uint4& v, uint64_t& s2, uint64_t& w2) {
        const uint64_t ref2 = lp_pack(-a.M, -a.M);
        uint64_t x2[VEC / 2];
        lp_pairs(v, x2, T{});
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const uint64_t y2 = lp_fma2(x2[i], c2, ref2);
          float y0, y1;
          lp_unpack(y2, y0, y1);
          const uint64_t e2 = lp_pack(lp_exp2(y0), lp_exp2(y1));
          s2 = lp_add2(s2, e2);
          w2 = lp_fma2(e2, y2, w2);
        }
      };
      auto add = [&](uint64_t s2, uint64_t w2) {
        float s0, s1, w0, w1;
        lp_unpack(s2, s0, s1);
        lp_unpack(w2, w0, w1);
        a.s += s0 + s1;
        a.w += w0 + w1;
      };
      auto take_edge = [&](int vec) {  // (its missing elements are -inf to the sums and nothing to the maximum)
        const uint4 v = row.raw(vec);
        float x[VEC], vm = __int_as_float(0x7fc00000);
        unpack16<T>(v, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int j = row.first(vec) + i;
          if (j >= 0 && j < p.V) vm = fmaxf(vm, x[i]);
        }
        meet(vm, vec);
        refer();
        uint64_t s2 = 0ull, w2 = 0ull;
        sum(v, s2, w2);
        add(s2, w2);
      };
      int edge_vec = 0;
      const bool edge = tid < 2 && rank == (tid == 0 ? 0 : cluster - 1) && row.edge(tid, edge_vec);
      if (edge && tid == 0) take_edge(edge_vec);
      for (int base = v0 + tid; base < v1; base += STREAM * UNROLL) {
        uint4 next[UNROLL];
        fetch(row, base + UNROLL * STREAM, v1, next);
        if (UNROLL > 1 && base + (UNROLL - 1) * STREAM >= v1) {  // the last round
#pragma unroll
          for (int u = 1; u < UNROLL; ++u)
            if (base + u * STREAM >= v1) now[u] = make_uint4(row.kNothing, row.kNothing, row.kNothing, row.kNothing);
        }
        const float round_top = lp_top(now, T{});
        if (PARTS > 1 && p.k > 0) {
          uint32_t most;  // (in its upper half)
          asm("max.bf16x2 %0, %1, %2;" : "=r"(most) : "r"(part_hi), "r"(__float_as_uint(round_top)));
          part_hi = __funnelshift_l(part_lo, part_hi, 16);
          part_lo = (part_lo << 16) | (most >> 16);
        }
        if (round_top > a.m || top_vec < 0) {
#pragma unroll
          for (int u = 0; u < UNROLL; ++u)
            if (u == 0 || base + u * STREAM < v1) meet(lp_top<1>({now[u]}, T{}), base + u * STREAM);
          refer();
        }
        uint64_t s2 = 0ull, w2 = 0ull;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          sum(now[u], s2, w2);
          now[u] = next[u];
        }
        add(s2, w2);
      }
      if (edge && tid == 1) take_edge(edge_vec);
      if (r + step < p.R) begin(r + step);
      const int b = n & 1;
      if (n >= 2) lp_bar_sync<kFree>(b);  // the row before last has been read
      if (p.k > 0) {
        lows[b][tid] = top_vec < 0 ? 0ull : lp_key(a.m, min(row.first(top_vec) + VEC - 1, p.V - 1));
        asm volatile("bar.sync %0, %1;" ::"n"(kStream), "n"(STREAM) : "memory");
        if (warp == 0) {
          unsigned long long g = 0ull;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) g = max(g, lows[b][w * 32 + lane]);
          groups[lane] = g;
          __syncwarp();
          int above = 0;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&groups[i]);
            above += (o.x > g || (o.x == g && i < lane)) + (o.y > g || (o.y == g && i + 1 < lane));
          }
          if (above == p.k - 1) limits[b] = g;  // 0: fewer maxima than k, everything is looked at
        }
        asm volatile("bar.sync %0, %1;" ::"n"(kStream), "n"(STREAM) : "memory");
        const unsigned long long lim = limits[b];
        const float least = lp_value((uint32_t)(lim >> 32));
        if (edge) look(row, edge_vec, row.raw(edge_vec), lim, least, b);
        const uint32_t lim_half = (uint32_t)(lim >> 48);
        const int rounds = (max(v1 - v0 - tid, 0) + STREAM * UNROLL - 1) / (STREAM * UNROLL);  // of this thread
        unsigned some = 0u;
        if constexpr (PARTS == 1) {
          part_lo = __float_as_uint(a.m) >> 16;
        }
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const uint32_t half = ((i & 2 ? part_hi : part_lo) >> (16 * (i & 1))) & 0xffffu;
          const bool reaches = lp_order(__uint_as_float(half << 16)) >> 16 >= lim_half;
          const unsigned who = __ballot_sync(0xffffffffu, reaches);
          if (reaches) owners[warp][some + __popc(who & ((1u << lane) - 1u))] = (unsigned char)(lane | ((rounds - 1 - i) & (PARTS - 1)) << 5);
          some += __popc(who);
        }
        __syncwarp();
        const unsigned per = (unsigned)((v1 - v0 + PARTS * STREAM * UNROLL - 1) / (PARTS * STREAM * UNROLL)) * UNROLL;  // vectors of a part
        const unsigned todo = some * per;
        auto vector_of = [&](unsigned i) -> int {
          const unsigned o = i / per, j = i - o * per, owner = owners[warp][o];
          return v0 + warp * 32 + (int)(owner & 31u) + (int)((owner >> 5) * UNROLL + j / UNROLL * (PARTS * UNROLL) + j % UNROLL) * STREAM;
        };
        for (unsigned i = lane; i < todo; i += 64u) {
          const int vec0 = vector_of(i), vec1 = i + 32u < todo ? vector_of(i + 32u) : v1;
          const uint4 x0 = row.inner(min(vec0, v1 - 1)), x1 = row.inner(min(vec1, v1 - 1));
          if (vec0 < v1) look(row, vec0, x0, lim, least, b);
          if (vec1 < v1) look(row, vec1, x1, lim, least, b);
        }
        __syncwarp();
      }
      a = lp_warp_join(a);
      if (lane == 0) stat[b][warp] = a;
      lp_bar_arrive<kFull>(b);
    }
    if (n >= 2) lp_bar_sync<kFree>(n & 1);  // the last two rows' signals are taken too
    if (n >= 1) lp_bar_sync<kFree>((n - 1) & 1);
    if (cluster > 1) {
      lp_cluster_sync();
      lp_cluster_sync();
    }
    return;
  }
  // ================= the last warp: a row's numbers, while the others are at the next one =================
  int n = 0;
  for (int r = row0; r < p.R; r += step, ++n) {
    const int b = n & 1;
    unsigned long long *found = founds[b], *best = bests[b];
    const LpRow<T> row = row_of(r);
    const int v0 = part(row, rank), v1 = part(row, rank + 1);
    const int target = p.targets[r];
    const bool target_ok = target >= 0 && target < p.V;
    const float target_logit = target_ok ? Io<T>::ld(row.row + target) : 0.f;
    lp_bar_sync<kFull>(b);
    LpStat a = lp_warp_join(lane < WARPS ? stat[b][lane] : LpStat{-INFINITY, -kLpBig, 0.f, 0.f});
    unsigned long long top = 0ull;  // lane i: key of the i-th of the top k
    if (p.k > 0) {
      unsigned long long lim = limits[b];
      for (;;) {
        const int n_found = mets[b];
        __syncwarp();
        if (lane == 0) mets[b] = 0;
        lp_rank(found, min(n_found, kLpFound), best, p.k, lane);
        // More tokens reach the bound than there is room for: the k-th of those that were kept is a higher one.  Fewer than k (a thread whose
        // bound was not a number's): everything is looked at.  Either way this warp goes through the CTA's vectors by itself.
        const unsigned long long kth = best[p.k - 1];
        const bool again = n_found > kLpFound;
        if (!again && (kth != 0ull || lim == 0ull)) break;
        lim = again ? kth : 0ull;
        const float least = lp_value((uint32_t)(lim >> 32));
        __syncwarp();
        for (int vec = v0 + lane; vec < v1; vec += 32) look(row, vec, row.inner(vec), lim, least, b);
        int edge_vec = 0;
        if (lane < 2 && rank == (lane == 0 ? 0 : cluster - 1) && row.edge(lane, edge_vec)) look(row, edge_vec, row.raw(edge_vec), lim, least, b);
        __syncwarp();
      }
      if (lane < p.k) top = best[lane];
    }
    __syncwarp();
    lp_bar_arrive<kFree>(b);
    if (cluster > 1) {  // one row: the first CTA joins
      if (lane == 0) mine = a;
      lp_cluster_sync();
      if (rank == 0) {
        LpStat other = {-INFINITY, -kLpBig, 0.f, 0.f};
        if (lane < cluster) {
          other.m = lp_ld_f32(lp_map(&mine.m, lane));
          other.M = lp_ld_f32(lp_map(&mine.M, lane));
          other.s = lp_ld_f32(lp_map(&mine.s, lane));
          other.w = lp_ld_f32(lp_map(&mine.w, lane));
        }
        a = lp_warp_join(other);
        if (lane < p.k)
          for (int c = 0; c < cluster; ++c) found[c * p.k + lane] = lp_ld_u64(lp_map(&best[lane], c));
      }
      lp_cluster_sync();  // the others may leave
      if (rank != 0) return;
      // lists of k in order: a key's place is the sum of its places in all of them
      const int all = cluster * p.k;
      if (lane < p.k) best[lane] = 0ull;
      __syncwarp();
      for (int i = lane; i < all; i += 32) {
        const unsigned long long key = found[i];
        if (key == 0ull) continue;
        int over = 0;
        for (int c = 0; c < cluster; ++c) {
          const unsigned long long* list = found + c * p.k;
          int at = 0;
#pragma unroll
          for (int half = 32; half > 0; half >>= 1)
            if (at + half <= p.k && list[at + half - 1] > key) at += half;
          over += at;
        }
        if (over < p.k) best[over] = key;
      }
      __syncwarp();
      if (lane < p.k) top = best[lane];
    }
    // A row beyond M's range, or at a temperature beyond that of one pass: once more, by this warp alone.
    const float m = a.m;
    const bool far = m < INFINITY && m > -INFINITY && (!(fabsf(m * p.c) < kLpBig) || p.c > 1e7f || p.c < kLpHot);
    if (far) {
      float s = 0.f, w = 0.f;
      for (int vec = lane; vec < row.n; vec += 32) {
        float x[VEC];
        unpack16<T>(row.raw(vec), x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float y = fmaf(x[i], 0.5f, -0.5f * m) * p.c2, e = lp_exp2(y);
          s += e;
          w = fmaf(e, fmaxf(y, kLpFar), w);
        }
      }
      a.s = warp_sum(s);
      a.w = warp_sum(w);
    }
    const float log_s = log2f(a.s);
    // nothing but -inf, or something that is not a number or +inf: no distribution
    const bool none = !(a.s > 0.f) || !(m < INFINITY) || m == -INFINITY;
    const float nan = __int_as_float(0x7fc00000);
    auto logprob = [&](float z) {
      if (none) return nan;
      if (far || z * p.c < -1e30f) return fmaf(fmaf(z, 0.5f, -0.5f * m), p.inv2, -log_s * kLn2);
      return (fmaf(z, p.c, -a.M) - log_s) * kLn2;
    };
    if (lane == 0) {
      if (!target_ok && p.status) atomicOr(p.status, 4);
      p.logprob[r] = target_ok ? logprob(target_logit) : nan;
      p.entropy[r] = none ? nan : fmaxf((log_s - a.w / a.s) * kLn2, 0.f);
    }
    if (lane < p.k) {
      p.top_ids[(long long)r * p.k + lane] = (int)(0xffffffffu - (uint32_t)top);
      p.top_logprobs[(long long)r * p.k + lane] = logprob(lp_value((uint32_t)(top >> 32)));
    }
  }
}

template <typename T, int UNROLL>
static int logprobs_go(const LpParams& p, int log_cluster, cudaStream_t st) {
  const int cluster = 1 << log_cluster;
  const long long most = 148 * kLpCtas;  // resident CTAs: the rows behind them follow in the same CTAs
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(cluster > 1 ? (long long)p.R * cluster : p.R < most ? p.R : most));
  cfg.blockDim = dim3(kLpStream + 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, UNROLL>, p, log_cluster);
  return launch_status("token_logprobs");
}

template <typename T>
static int logprobs_launch(const LpParams& p, cudaStream_t st) {
  const int vecs = p.V / (Io<T>::kVec16 * kLpStream);  // of a thread, with one CTA a row
  // One row's vectors over more CTAs while there are SMs for them and the row is long enough for what a cluster costs, its two barriers and with top
  // tokens the lists that are joined.  (13 rows of bf16, top 5, us with 1, 2, 4 and 8 CTAs a row: V = 16384 5.8 6.4 6.7 8.2, 32768 7.3 7.1 7.0 8.3, 65536
  // 10.1 8.9 7.7 8.9; without top tokens 4.0 4.2 4.0 3.8, 5.2 5.0 4.2 4.1, 7.7 6.3 5.0 4.4.)
  int log = 0;
  while (log < (p.k > 0 ? 2 : 3) && ((long long)p.R << (log + 1)) <= 296 && vecs >= (p.k > 0 ? 16 : 12) << log) ++log;
  // Four vectors a thread on their way, or one where rows are short and the last of a row would mostly be waited for in vain.  (4096 rows of bf16, top 5, us
  // with four and one: V = 4096 36.6 29.6, 12288 47.6 42.2, 16384 49.1 50.5, 32768 72.1 79.6; one of 128000 fp32 19.1 26.3.)
  return vecs >> log >= 8 ? logprobs_go<T, 4>(p, log, st) : logprobs_go<T, 1>(p, log, st);
}

}  // namespace dgpt

using namespace dgpt;

extern "C" int dgpt_token_logprobs(const void* logits, int64_t logits_row_stride, const int32_t* targets, float temperature, float* logprob,
                                   float* entropy, int32_t* top_ids, float* top_logprobs, int32_t top_k, int32_t R, int32_t V, int32_t dtype,
                                   int32_t* status, void* stream) {
  DGPT_REQUIRE(R >= 0 && V > 0 && V <= 0x7fffff00, "token_logprobs: bad sizes");
  DGPT_REQUIRE(top_k >= 0 && top_k <= kLpMost && top_k <= V, "token_logprobs: top_k must be 0 to %d and at most the vocabulary, got %d", kLpMost, top_k);
  DGPT_REQUIRE(temperature >= kLpCold && temperature < INFINITY, "token_logprobs: the temperature must be finite and at least %g", (double)kLpCold);
  DGPT_REQUIRE(R <= 0x0fffffff, "token_logprobs: too many rows");
  if (dtype != DGPT_F32 && dtype != DGPT_BF16) {
    set_error("token_logprobs: unknown dtype %d", dtype);
    return DGPT_E_UNSUPPORTED;
  }
  if (R == 0) return DGPT_OK;
  DGPT_REQUIRE(logits && targets && logprob && entropy && (top_k == 0 || (top_ids && top_logprobs)), "token_logprobs: NULL pointer");
  DGPT_REQUIRE(logits_row_stride >= V || R == 1, "token_logprobs: rows overlap");
  DGPT_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == DGPT_F32 ? 4 : 2) == 0, "token_logprobs: logits are not aligned to their type");
  LpParams p = {logits, R == 1 ? (int64_t)V : logits_row_stride, targets, logprob, entropy, top_logprobs, top_ids, R, V, top_k, kLog2e / temperature, 2.f * kLog2e / temperature, 2.f / temperature, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DGPT_F32 ? logprobs_launch<float>(p, st) : logprobs_launch<__nv_bfloat16>(p, st);
}
