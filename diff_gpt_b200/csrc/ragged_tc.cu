// Attention of packed prompts and of trees of drafted tokens on the tcgen05 tensor cores (sm_100a, bf16, head_dim 64 or 128; 32 rides on
// the 64-wide kernel: TMA boxes reach past the tensor and arrive as zeros).
//
// A persistent CTA of 512 threads per SM walks through work items: 128 query rows against a run of key tiles of 128.  Lengths lie on the
// device, so a warp of its own works out the items' rows and keys (ragged.cuh) and hands them to the others through a ring in shared memory.
// Sequences are short as often as long, which is why nothing stops between items: score products run two key tiles ahead of the
// probabilities whatever item they belong to, loads run ahead of those, and a warpgroup of its own takes a finished item's output out
// of TMEM while the softmax threads are at the next one.
//   warp 14          items
//   warp 13          loader: TMA loads of Q, K and V tiles into two slots of each (128-byte swizzle, one box per page and 64-wide
//                    half of the head); page numbers are fetched 32 at a time
//   warp 12, lane 0  issuer: S_g = Q K_g^T into one of two score buffers, O += P_g V_g with P from TMEM.  P V of tile g goes before S of tile
//                    g + 2, so that the arrival of those scores also says that P_g has been read
//   warps 0-7        softmax, 16 rows a warp and four threads a row (tcgen05.ld.16x256b): probabilities against the running maximum in one sweep
//                    that finds the tile's own maximum too; only where a score exceeds the running one by more than 2^8 is O rescaled and the tile
//                    redone.  (Two threads per row in different warps, each with half of a tile's columns and its maximum handed over through
//                    shared memory: 8 x 16 heads of 128 x 4096 631 us, so 588; of 64 614 and 520; 40 mixed prompts 102 and 95.)
//   warps 8-11       output: row sums from shared memory, O from TMEM (a row per thread), rows through shared memory so that a row's bytes leave together
// What bounds it is the softmax: 8 x 16 heads of 128 x 4096 causal 575 us = 956 TFLOP/s, 0.57 of the measured product rate, with the tensor pipe and the
// exponentials each busy 41 to 45 % of the time; long caches 1.35 us a tile of 128 x 128, prompts of 17 to 1000 tokens 1.7 (starts and masked ends).
// (Two CTAs an SM for heads of 64, each with one score buffer, its softmax threads storing the output: 512 prompts of 128 143 us instead of 161, 40 mixed
// ones 106 instead of 102, 8 of 4096 597 instead of 615; not kept.)
// TMEM columns: S0 [0,128)  S1 [128,256)  P0 [256,320)  P1 [320,384)  O [384, 384 + D).
// No cluster launch and no multicast.  Every wait is bounded in clock cycles; one that runs out raises the CTA's abort flag, on which the other
// roles stop too, and sets bit 1 of the status word.  However the CTA ends, copies and products that were issued are waited for (with a limit) before it frees its
// TMEM and returns.
#include <type_traits>

#include "ragged.cuh"
#include "tcgen05.cuh"

namespace dgpt {
namespace tc {

constexpr int kRtThreads = 512;
// Registers per thread: the launch's, and a softmax and a helper thread's after the warpgroups have traded them (an output thread keeps the launch's).
constexpr int kRtRegs = 128, kRtSoftmaxRegs = 152, kRtHelperRegs = 80;
static_assert(2 * kRtSoftmaxRegs + kRtRegs + kRtHelperRegs == 4 * kRtRegs, "the warpgroups share what the launch has");
constexpr int kRtLead = 3;                                                    // key tiles still to be loaded when the next item is asked for
// Limit of the waits that may last a whole item, 3 x 10^9 keys here, in limits of the others, which last a tile or two, run out first and raise the abort flag.
constexpr int kRtItemWaits = 16;
constexpr int kRtRing = 8;                                                    // items between the warp that finds them and the last role that reads them

struct RtItem {
  RaggedItem it;
  int tile0, n;  // key tiles tile0 .. tile0 + n - 1; n < 0: no more items
};
static_assert(sizeof(RtItem) % 4 == 0 && sizeof(RtItem) <= 64, "a ring slot is 64 bytes");

// A warp's 16 rows in the registers of four lanes each: lane t holds of every 8 columns the two from 2 (t % 4) on, of row t / 4 in registers 4 j and
// 4 j + 1 and of row t / 4 + 8 in 4 j + 2 and 4 j + 3.  A row's maximum and sum are then two shuffles away.
__device__ __forceinline__ void rows16_ld(uint32_t addr, float (&v)[32]) {  // 64 columns
  uint32_t r[32];
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr)
               : "memory");
  tc_wait_ld();
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void rows16_ld(uint32_t addr, float (&v)[16]) {  // 32 columns
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr)
               : "memory");
  tc_wait_ld();
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void rows16_ld(uint32_t addr, float (&v)[4]) {  // 8 columns
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  tc_wait_ld();
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void rows16_st(uint32_t addr, const float (&v)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
// The same rows' columns as pairs of bf16: word t % 4 of every 4, of row t / 4 in register 2 j and of row t / 4 + 8 in 2 j + 1.  32 words.
__device__ __forceinline__ void rows16_st_pairs(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

// Items are dealt at run time: the grid has a CTA for each, one per SM is resident, and a resident CTA that wants more work cancels one that
// has not been launched and takes its number (cluster launch control).  Numbers run from a prompt's last rows, which see the most keys, to its
// first ones, prompt by prompt, so that the CTAs at work share a prompt's K and V in L2 and the last items are the shortest.  (Dealt in fixed rounds, the
// busiest SM had 1.25 times the mean of 2 x 16 heads of 128 x 4096; 16 on 4 heads, 4 prompts of 2678 to 3455: 228 us so, 214 dealt at run time.)
__device__ __forceinline__ void ask_for_cta(uint32_t answer, uint32_t bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ bool cta_answer(uint32_t answer, unsigned& cta) {
  uint32_t ok, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .b64 lo, hi;\n\t.reg .pred p;\n\t"
      "ld.shared.v2.b64 {lo, hi}, [%2];\n\tmov.b128 h, {lo, hi};\n\tmov.u32 %1, 0;\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(ok), "=&r"(x)
      : "r"(answer)
      : "memory");
  cta = x;
  return ok != 0;
}

// The items of a launch by their numbers, for a whole warp.  Prompts: a tile's sequence is mostly that of the tile before.  Trees: from the longest
// sequence to the shortest where they are few enough to be sorted, so that the last items are short ones (48 trees behind 300 to 4000 keys 54 us, in the
// sequences' order 63).
struct PackedItems {
  const PackedProblem& p;
  PackedProblem::Cursor cur;
  __device__ PackedItems(const PackedProblem& q, int*, int) : p(q) {}
  __device__ bool get(unsigned i, RaggedItem& it, int lane) {
    const unsigned j = gridDim.x - 1u - i, slot = j / (unsigned)p.H;
    p.seek((int)slot, kBM, lane, cur);
    return p.item((int)slot, cur, (int)(j - slot * (unsigned)p.H), kBM, it);
  }
};
struct TreeItems {
  const TreeProblem& p;
  const int* order = nullptr;
  __device__ TreeItems(const TreeProblem& q, int* room, int lane) : p(q) {
    if (p.B > 1 && p.B <= TreeProblem::kSorted && p.items() > 148) {
      p.sort(room, lane);
      order = room;
    }
  }
  __device__ bool get(unsigned i, RaggedItem& it, int) { return p.item(i, kBN, it, order); }
};

// The rows of an item without keys: zeros.  (A share without keys of a tree's rows is left out by the pass that joins the shares.)
template <class P, bool TREE>
__device__ __forceinline__ void no_keys(const P& p, const RaggedItem& it, int d_head, int lane) {
  if constexpr (TREE)
    if (p.n_splits > 1) return;
#pragma unroll 1
  for (int r = 0; r < it.rows; ++r) {
    __nv_bfloat16* o;
    if constexpr (TREE) {
      o = static_cast<__nv_bfloat16*>(p.o) + p.out_row(it, r) * p.o_rs + (long long)p.head(it, r) * d_head;
    } else {
      o = static_cast<__nv_bfloat16*>(p.o) + (long long)(it.row0 + r) * p.o_rs + (long long)it.h * p.o_hs;
      if (p.lse && lane == 0) p.lse[(long long)(it.row0 + r) * p.H + it.h] = -INFINITY;
    }
    if (lane * 8 < d_head) *reinterpret_cast<uint4*>(o + lane * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int D, class P, bool TREE>
__global__ void __launch_bounds__(kRtThreads, 1)
ragged_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                 const P p, const int d_head) {
  constexpr int kSub = D / 64;
  constexpr uint32_t kSubBytes = kBN * 128;
  constexpr uint32_t kTileBytes = kSub * kSubBytes;
  constexpr uint32_t kIdescS = instr_desc(kBN, false);
  constexpr uint32_t kIdescPV = instr_desc(D, true);
  constexpr uint32_t kPCol = 256, kOCol = 384;
  constexpr uint32_t kTmem = 512;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sV = smem + 4 * kTileBytes;  // Q0 Q1 | K0 K1 | V0 V1 | barriers | row sums | items | output | order
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 6 * kTileBytes);
  constexpr int iQ = 0, iQF = 2, iK = 4, iKF = 6, iV = 8, iS = 10, iP = 12, iO = 14, iOF = 16, iL = 17, iLF = 19, iR = 21, iRF = iR + kRtRing,
                iC = iRF + kRtRing, iD = iC + 1, nBars = iD + 1;
  static_assert(nBars <= 43, "barriers, an answer of 16 bytes and three words in 48 words");
  uint64_t* answer = bars + 44;  // 16-byte aligned
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 43);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile unsigned* loaded = reinterpret_cast<volatile unsigned*>(bars + 46);  // K tiles asked for
  float* sums = reinterpret_cast<float*>(bars + 48);        // [2 items][l | m][128 rows]
  uint8_t* ring = reinterpret_cast<uint8_t*>(sums + 2 * 2 * kBM);                                // [kRtRing] items
  const uint32_t aQ = smem_u32(smem), aK = aQ + 2 * kTileBytes, aV = aQ + 4 * kTileBytes, bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    *abort_flag = 0;
    *loaded = 0u;
    for (int i = 0; i < nBars; ++i)
      mbar_init(bar(i), (i == iP || i == iP + 1 || i == iL || i == iL + 1) ? 2 * kBM : (i == iOF || i == iLF || i == iLF + 1) ? kBM : i >= iRF && i < iC ? 14 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if constexpr (TREE) {  // rows of Q that no load reaches: level scores keep their warp on the short path
    for (int i = p.rows_per_tile * 8 + tid; i < kBM * 8; i += kRtThreads)
#pragma unroll
      for (int s = 0; s < 2 * kSub; ++s) reinterpret_cast<uint4*>(smem + s * kSubBytes)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_async_smem();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  RtItem x;
  // A role's place in the ring.  `take` waits for the next item and reads it (every lane that calls gets it); false at the end or after a
  // wait that ran out (`ok` tells).  A slot is free when the loader, the issuer and every softmax and output warp have said `done`.
  auto wait_tile = [&](int b, unsigned parity) { return wait_or_abort(bar(b), parity, abort_flag, 2, p.wait_limit); };
  // (Output and item warps wait for thousands of cycles at a time: they sleep between looks, so that their polling takes no issue slots from
  // the softmax warps that share their schedulers.)
  auto wait_asleep = [&](int b, unsigned parity) -> bool {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar(b), parity)) {
      if (*abort_flag) return false;
      if (clock64() - t0 > kRtItemWaits * p.wait_limit) {
        *abort_flag = 2;
        return false;
      }
      __nanosleep(100);
    }
    return true;
  };
  unsigned taken = 0u;
  auto take = [&](RtItem& y, unsigned at, bool& ok) -> bool {
    ok = wait_tile(iR + (int)(at % kRtRing), (at / kRtRing) & 1u);
    if (!ok) return false;
    y = *reinterpret_cast<const RtItem*>(ring + (at % kRtRing) * 64);
    return y.n >= 0;
  };
  auto done = [&](unsigned at) { mbar_arrive(bar(iRF + (int)(at % kRtRing))); };

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRtHelperRegs));
    if (warp == 13) {
      // ================= loader =================
      if (lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mq)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mk)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mv)) : "memory");
      }
      unsigned items = 0u, kn = 0u, vn = 0u;  // loads issued: Q, K tiles, V tiles
      bool ok = true;
      auto wait = [&](int b, unsigned parity) { return __all_sync(0xffffffffu, wait_tile(b, parity)) != 0; };
      // tree: this lane holds the numbers of pages page0 + lane and page0 + 32 + lane of sequence page_seq, the latter on their way while the
      // former are used, and those of page `lane` of the last two K tiles, of which one is the next V tile
      int page0 = 0, page_seq = -1, page_id = 0, page_next = 0, newer = 0, older = 0;
      int pt = 0, max_pages = 0;  // pt 0: a dense run per sequence
      const int* tables = nullptr;
      if constexpr (TREE) {
        tables = p.kv.page_table;
        max_pages = p.kv.max_pages;
        pt = tables ? p.kv.page_tokens : 0;
      }
      const bool dense = pt == 0;
      const int per = dense || pt >= kBN ? 1 : kBN / pt;  // pages of a tile
      auto find_pages = [&](const RtItem& w, int t) {
        older = newer;
        if (dense) {
          newer = w.it.seq;
          return;
        }
        const int first = t * kBN / pt;
        if (page_seq != w.it.seq || first < page0 || first + per > page0 + 32) {
          const int* table = tables + (long long)w.it.seq * max_pages;
          auto fetch = [&](int lp) { return table[min(lp + lane, max_pages - 1)]; };
          // (32 pages hold a whole number of tiles, so a tile's pages end where a block of 32 ends)
          page_id = page_seq == w.it.seq && first == page0 + 32 ? page_next : fetch(first);
          page_seq = w.it.seq;
          page0 = first;
          page_next = fetch(first + 32);
        }
        newer = __shfl_sync(0xffffffffu, page_id, (first - page0 + lane) & 31);
      };
      auto load_tile = [&](const CUtensorMap* map, uint32_t dst, uint32_t full, const RtItem& w, int t, int pages) {
        const int t0 = t * kBN;
        if constexpr (!TREE) {
          if (lane == 0) {
            mbar_expect_tx(full, kTileBytes);
#pragma unroll
            for (int s = 0; s < kSub; ++s) tma_load_4d(dst + s * kSubBytes, map, full, s * 64, w.it.g, w.it.kbase + t0, 0);
          }
        } else {
          const int valid = per == 1 ? 1 : min(per, (w.it.key1 - t0 + pt - 1) / pt);
          const int in = per > 1 ? 0 : dense ? t0 : t0 % pt;
          if (lane == 0) mbar_expect_tx(full, per == 1 ? kTileBytes : (uint32_t)valid * pt * 128u * kSub);
          __syncwarp();
          // a lane per page
          if (lane < valid) {
#pragma unroll
            for (int s = 0; s < kSub; ++s) tma_load_4d(dst + s * kSubBytes + lane * pt * 128, map, full, s * 64, in, w.it.g, pages);
          }
        }
      };
      auto take_all = [&](RtItem& y, unsigned& at) -> bool {  // the next item, for the whole warp
        bool fine;
        const bool there = take(y, at, fine);
        ok = __all_sync(0xffffffffu, fine) != 0;
        ++at;
        return ok && there;
      };
      // K runs one tile ahead of V, across items too
      RtItem y;  // item of the K cursor
      unsigned ahead = 0u;
      int kj = 0;
      bool more = take_all(y, ahead);
      auto load_k = [&]() {
        if (kj == 0) {
          const unsigned qs = items & 1u;
          if (items >= 2) ok = wait(iQF + (int)qs, ((items - 2) >> 1) & 1u);  // the last S of the item before last is done
          if (!ok) return;
          if (lane == 0) {
            const uint32_t full = bar(iQ + (int)qs), to = aQ + qs * kTileBytes;
            if constexpr (TREE) {
              mbar_expect_tx(full, (uint32_t)(p.rows_per_tile * 128 * kSub));
#pragma unroll
              for (int s = 0; s < kSub; ++s) tma_load_4d(to + s * kSubBytes, &mq, full, s * 64, y.it.h, y.it.row0 / p.group, y.it.seq);
            } else {
              mbar_expect_tx(full, kTileBytes);
#pragma unroll
              for (int s = 0; s < kSub; ++s) tma_load_4d(to + s * kSubBytes, &mq, full, s * 64, y.it.h, y.it.row0, 0);
            }
          }
          ++items;
        }
        const unsigned ks = kn & 1u, ku = kn >> 1;
        if (ku > 0) ok = wait(iKF + (int)ks, (ku - 1) & 1u);
        if (!ok) return;
        if constexpr (TREE) find_pages(y, y.tile0 + kj);
        load_tile(&mk, aK + ks * kTileBytes, bar(iK + (int)ks), y, y.tile0 + kj, newer);
        ++kn;
        if (lane == 0) *loaded = kn;
        if (++kj == y.n) {
          kj = 0;
          more = take_all(y, ahead);
        }
      };
      if (more) load_k();
      while (ok && take_all(x, taken)) {
        for (int j = 0; ok && j < x.n; ++j) {
          if (more) load_k();
          if (!ok) break;
          const unsigned vs = vn & 1u;
          if (vn >= 2) ok = wait(iO + (int)vs, ((vn - 2) >> 1) & 1u);
          if (!ok) break;
          load_tile(&mv, aV + vs * kTileBytes, bar(iV + (int)vs), x, x.tile0 + j, kn == vn + 1u ? newer : older);
          ++vn;
        }
        __syncwarp();
        if (lane == 0) done(taken - 1);
      }
      if ((!ok || *abort_flag) && lane == 0 && p.status) atomicOr(p.status, 2);
      // Copies still in flight write shared memory.  (Another role may give up after the last of them was asked for, so they are waited for in any case; at a
      // usual end the products have.)
      for (unsigned i = 0; i < 2u && i < items; ++i) mbar_wait(bar(iQ + (int)((items - 1 - i) & 1u)), ((items - 1 - i) >> 1) & 1u);
      for (unsigned i = 0; i < 2u && i < kn; ++i) mbar_wait(bar(iK + (int)((kn - 1 - i) & 1u)), ((kn - 1 - i) >> 1) & 1u);
      for (unsigned i = 0; i < 2u && i < vn; ++i) mbar_wait(bar(iV + (int)((vn - 1 - i) & 1u)), ((vn - 1 - i) >> 1) & 1u);
    } else if (warp == 12) {
      // ================= MMA issuer (one lane) =================
      if (lane == 0) {
        const uint64_t dQK = smem_desc(0, 16, 1024), dV = smem_desc(0, kSubBytes, 1024);
        RtItem y;  // item of the score cursor
        int sj = 0;
        unsigned items = 0u, sg = 0u, g = 0u, ahead = 0u;
        bool ok = true;
        auto take_one = [&](RtItem& z, unsigned& at) -> bool { return take(z, at++, ok); };
        bool more = take_one(y, ahead);
        auto issue_s = [&]() {  // S(sg & 1) = Q K(sg & 1)^T
          if (sj == 0) {
            ok = wait_tile(iQ + (int)(items & 1u), (items >> 1) & 1u);
            ++items;
          }
          const unsigned qs = (items - 1u) & 1u, buf = sg & 1u;
          ok = ok && wait_tile(iK + (int)buf, (sg >> 1) & 1u);
          if (!ok) return;
          tc_fence_after();
          umma_ss_chain<D / 16>(tmem + buf * 128, dQK + ((aQ + qs * kTileBytes) >> 4), dQK + ((aK + buf * kTileBytes) >> 4), kIdescS, kSubBytes >> 4);
          umma_commit(bar(iS + (int)buf));
          umma_commit(bar(iKF + (int)buf));
          ++sg;
          if (++sj == y.n) {
            umma_commit(bar(iQF + (int)qs));  // Q may be overwritten
            sj = 0;
            more = take_one(y, ahead);
          }
        };
        for (int i = 0; i < 2 && ok && more; ++i) issue_s();
        unsigned outs = 0u;  // items whose first P V has been issued
        while (ok && take_one(x, taken)) {
          for (int j = 0; ok && j < x.n; ++j, ++g) {
            const unsigned buf = g & 1u, ph = (g >> 1) & 1u;
            // P_g is complete when every row has arrived; by then every row has also consumed S_g
            ok = wait_tile(iP + (int)buf, ph) && wait_tile(iV + (int)buf, ph);
            if (ok && j == 0) {
              if (outs > 0) ok = wait_tile(iOF, (outs - 1) & 1u);  // O of the item before has been read
              ++outs;
            }
            if (!ok) break;
            tc_fence_after();
            umma_ts_chain<kBN / 16>(tmem + kOCol, tmem + kPCol + buf * 64, dV + ((aV + buf * kTileBytes) >> 4), kIdescPV, j > 0 ? 1u : 0u);
            umma_commit(bar(iO + (int)buf));
            if (more) issue_s();
          }
          if (ok) done(taken - 1);
        }
        if (!ok) {
          if (!*abort_flag) *abort_flag = 2;
          if (p.status) atomicOr(p.status, 2);
        }
        // Products still in flight read shared memory, write TMEM and arrive on barriers.  (At a usual end they are done: the output warps have waited for them.)
        if (sg > 0u) {
          umma_commit(bar(iD));
          if (!mbar_wait(bar(iD), 0u) && p.status) atomicOr(p.status, 2);
        }
      }
    } else if (warp == 14) {
      // ================= items =================
      // An item is asked for when it will be wanted soon and not before, so that none waits behind a long one while another SM idles: when no more
      // than kRtLead key tiles are left to load.  (The issuer's score cursor and the loader's K cursor wait for the next item before they go on with what
      // they have; both have passed the last tile's K by then, so the next item is always on its way.  Items without a key never get here.  48 trees
      // of up to 32 drafts behind 300 to 4000 keys: the first SM done at 32, the last at 74 us with an item in store from the start; all of it 53 instead of 69.)
      std::conditional_t<TREE, TreeItems, PackedItems> items(p, reinterpret_cast<int*>(ring + kRtRing * 64 + 4 * 4096), lane);
      unsigned at = 0u, freed = 0u, asked = 0u, cta = blockIdx.x;  // items handed out, items finished
      unsigned handed = 0u;                                        // key tiles of the items handed out
      bool ok = true, more = true, first = false;  // first: item 0 is this CTA's
      auto push = [&]() {
        if (at - freed >= (unsigned)kRtRing) {
          ok = __all_sync(0xffffffffu, wait_asleep(iRF + (int)(freed % kRtRing), (freed / kRtRing) & 1u)) != 0;
          ++freed;
        }
        if (!ok) return;
        if (lane == 0) {
          *reinterpret_cast<RtItem*>(ring + (at % kRtRing) * 64) = x;
          mbar_arrive(bar(iR + (int)(at % kRtRing)));
        }
        __syncwarp();
        handed += (unsigned)x.n;
        ++at;
      };
      auto wanted = [&]() -> bool {  // whether the next item was wanted before the time ran out
        const long long t0 = clock64();
        while (handed - *loaded > (unsigned)kRtLead) {
          if (*abort_flag) return false;
          if (clock64() - t0 > kRtItemWaits * p.wait_limit) {
            *abort_flag = 2;
            return false;
          }
          __nanosleep(100);
        }
        return true;
      };
      while (ok && more) {
        first = first || cta == 0u;
        if (items.get(cta, x.it, lane)) {
          x.tile0 = x.it.key0 / kBN;
          x.n = (x.it.key1 - x.it.key0 + kBN - 1) / kBN;
          if (x.n > 0) push();
          else no_keys<P, TREE>(p, x.it, d_head, lane);
        }
        ok = __all_sync(0xffffffffu, wanted()) != 0;
        if (!ok) break;
        if (lane == 0) ask_for_cta(smem_u32(answer), bar(iC));
        if (!__all_sync(0xffffffffu, mbar_wait(bar(iC), asked & 1u))) {
          *abort_flag = 2;
          ok = false;
          break;
        }
        ++asked;
        more = cta_answer(smem_u32(answer), cta);
        fence_async_smem();  // read here before the next answer is written
        __syncwarp();
      }
      if (ok) {
        x.n = -1;
        push();
      }
      if (!ok && lane == 0 && p.status) atomicOr(p.status, 2);
      p.check(first, lane, 32);  // (CTA 0 itself may never be launched, its number being another's)
    }
  } else if (warp >= 8) {
    // ================= output =================
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t o_addr = tmem + ((uint32_t)(quarter * 32) << 16) + kOCol;
    uint8_t* stage = ring + kRtRing * 64 + quarter * 4096;
    unsigned items = 0u, g = 0u;
    bool ok = true;
    for (;; ++taken) {
      bool fine;
      const bool there = take(x, taken, fine);
      ok = __all_sync(0xffffffffu, fine) != 0;
      if (!ok || !there) break;
      __syncwarp();
      if (lane == 0) done(taken);
      const int rows = min(max(x.it.rows - quarter * 32, 0), 32);  // of this warp
      char* mine = nullptr;                                         // where this thread's row goes
      float* mine_lse = nullptr;
      bool part = false;
      if constexpr (TREE) part = p.n_splits > 1;
      if (lane < rows) {
        if constexpr (TREE) {
          const long long at = p.out_row(x.it, row);
          const int h = p.head(x.it, row);
          if (part) {
            const long long slot = ((long long)x.it.split * p.B * p.T + at) * p.H + h;
            mine = reinterpret_cast<char*>(p.part_o + slot * d_head);
            mine_lse = p.part_lse + slot;
          } else {
            mine = reinterpret_cast<char*>(static_cast<__nv_bfloat16*>(p.o) + at * p.o_rs + (long long)h * d_head);
          }
        } else {
          const long long at = x.it.row0 + row;
          mine = reinterpret_cast<char*>(static_cast<__nv_bfloat16*>(p.o) + at * p.o_rs + (long long)x.it.h * p.o_hs);
          if (p.lse) mine_lse = p.lse + at * p.H + x.it.h;
        }
      }
      const int slot = (int)(items & 1u);
      ok = __all_sync(0xffffffffu, wait_asleep(iL + slot, (items >> 1) & 1u)) != 0;
      if (!ok) break;
      const float l = sums[slot * 2 * kBM + row], m = sums[(slot * 2 + 1) * kBM + row];
      mbar_arrive(bar(iLF + slot));
      const unsigned last = g + (unsigned)x.n - 1u;
      ok = __all_sync(0xffffffffu, wait_tile(iO + (int)(last & 1u), (last >> 1) & 1u)) != 0;
      if (!ok) break;
      tc_fence_after();
      g += (unsigned)x.n;
      ++items;
      const bool any = !(l <= 0.f);  // a row with a score that is not a number keeps saying so
      const float inv = any ? 1.f / l : 0.f;
      // 128 bytes of every row at a time go through shared memory, so that eight lanes store a row's 128 bytes and not each lane 16 of its own
      // (an item of 128 rows of 128 bf16 numbers: 4000 cycles so, 1000 now)
      auto store = [&](const uint32_t* w, int col, int bytes) {  // w: this row's words; col, bytes: where they go in the row
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3), c = lane & 7;
          char* to = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), r));
          const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
          if (r < rows && c * 16 < bytes) *reinterpret_cast<uint4*>(to + col + c * 16) = v;
        }
      };
      if (rows > 0) {  // warp-uniform
        const int passes = part ? d_head / 32 : (d_head + 63) / 64;
#pragma unroll 1
        for (int c = 0; c < passes; ++c) {
          uint32_t w[32];
          float v[32];
          if (part) {
            tmem_ld32(o_addr + c * 32, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = any ? __float_as_uint(v[i] * inv) : 0u;
          } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              tmem_ld32(o_addr + c * 64 + u * 32, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i] * inv, v[2 * i + 1] * inv);
                w[u * 16 + i] = any ? *reinterpret_cast<const uint32_t*>(&h) : 0u;
              }
            }
          }
          if (c == passes - 1) {
            tc_fence_before();
            mbar_arrive(bar(iOF));
          }
          store(w, c * 128, part ? 128 : min(128, d_head * 2 - c * 128));
        }
        if (mine_lse) {
          const float base2 = m + log2f(l);
          *mine_lse = !any ? -INFINITY : TREE ? base2 : base2 * kLn2;
        }
      } else {
        mbar_arrive(bar(iOF));
      }
    }
    if (!ok && lane == 0 && p.status) atomicOr(p.status, 2);
  } else {
    // ================= softmax: 16 rows a warp =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRtSoftmaxRegs));
    const int quarter = warp & 3, half = warp >> 2, row0 = quarter * 32 + half * 16;
    const int row_of[2] = {row0 + (lane >> 2), row0 + (lane >> 2) + 8}, col = 2 * (lane & 3);  // this thread's rows, its first column of every 8
    const uint32_t lane_addr = tmem + ((uint32_t)row0 << 16);
    const float scale_log2 = p.scale_log2;
    unsigned g = 0u, items = 0u;
    bool fail = false;
    for (;; ++taken) {
      bool fine;
      const bool there = take(x, taken, fine);
      fail = !__all_sync(0xffffffffu, fine);
      if (fail || !there) break;
      __syncwarp();
      if (lane == 0) done(taken);
      const int n = x.n, rows = x.it.rows, clear = x.it.clear, gap0 = x.it.gap0, gap1 = x.it.gap1;
      // Key from which value rows may hold anything: the end of the sequence's keys.
      const int held_end = TREE ? x.it.key1 : x.it.held;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // l: of this thread's columns
      int t0 = x.tile0 * kBN;
      for (int j = 0; j < n; ++j, ++g, t0 += kBN) {
        const unsigned buf = g & 1u, ph = (g >> 1) & 1u;
        // exits are taken by whole warps (the vote makes the decision uniform), never by single lanes
        if (!__all_sync(0xffffffffu, wait_tile(iS + (int)buf, ph))) {
          fail = true;
          break;
        }
        tc_fence_after();
        const bool in_gap = TREE && t0 < gap1 && t0 + kBN > gap0;
        if (__builtin_expect(t0 + kBN > held_end || in_gap, 0)) {  // clear those rows so that 0 * x stays 0
          if (!__all_sync(0xffffffffu, wait_tile(iV + (int)buf, ph))) {
            fail = true;
            break;
          }
          const int vr = quarter * 32 + lane, key = t0 + vr;
          if (half == 0 && (key >= held_end || (in_gap && key >= gap0 && key < gap1))) {
#pragma unroll
            for (int s = 0; s < kSub; ++s) {
              uint4* vrow = reinterpret_cast<uint4*>(sV + buf * kTileBytes + s * kSubBytes + vr * 128);
#pragma unroll
              for (int c = 0; c < 8; ++c) vrow[c] = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async_smem();
          }
        }
        if (__builtin_expect(row0 >= rows, 0)) {  // none of this warp's rows exists: what it leaves in P reaches no other row
          tc_fence_before();
          mbar_arrive(bar(iP + (int)buf));
          continue;
        }
        // What a row sees of the tile, from this thread's first column on.  Prompts: the last column.  Trees: seen[r][c], a bit for each of the
        // columns from 64 c on.
        const bool masked = t0 + kBN > clear || in_gap;
        int last[2];
        unsigned long long seen[2][2];
        int halves = 2;  // of the tile that one of this warp's rows sees something of (8 x 16 heads of 128 x 4096 590 us with all of it, 575 so)
        if (__builtin_expect(masked, 0)) {
          if ((TREE ? x.it.key1 - 1 : min(x.it.last0 + row0 + 15, x.it.key1 - 1)) - t0 < 64) halves = 1;
          if constexpr (!TREE) {
            // (what Q holds behind the last row is anything; its scores stay as they are)
#pragma unroll
            for (int r = 0; r < 2; ++r) last[r] = row_of[r] < rows ? min(x.it.last0 + row_of[r], x.it.key1 - 1) - t0 - col : kBN;
          } else {
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              const int c0 = t0 + c * 64;
              unsigned long long both = ~0ull;  // what neither row sees is cleared
              const int a = max(gap0 - c0, 0), b = min(gap1 - c0, 64);  // the gap's columns
              if (in_gap && a < b) both &= ~((b < 64 ? (1ull << b) - 1ull : ~0ull) & ~((1ull << a) - 1ull));
              const int left = x.it.key1 - c0;
              if (left < 64) both = left > 0 ? both & ((1ull << left) - 1ull) : 0ull;
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                unsigned long long bits = ~0ull;
                const int d0 = c0 - clear;
                if (d0 > -64 && row_of[r] < rows) {
                  const unsigned long long* words = p.mask_row(x.it, row_of[r]);
                  auto word = [&](int w) { return w < p.words ? words[w] : 0ull; };
                  if (d0 < 0) {
                    bits = (word(0) << -d0) | ((1ull << -d0) - 1ull);
                  } else {
                    const int w = d0 >> 6, s = d0 & 63;
                    bits = word(w) >> s;
                    if (s) bits |= word(w + 1) << (64 - s);
                  }
                }
                bits = (bits & both) >> col;
                if (c == 0) seen[r][0] = bits;
                else seen[r][1] = bits;
              }
            }
          }
        }
        // 64 columns at a time, in loops that stay loops: with all of a tile's scores in registers at once, and the code for them, the softmax
        // warps waited for instructions (40 prompts of 17 to 1000, 12 heads of 64, 110 us so, 102 in this form)
        auto scores = [&](int c, float (&sv)[32]) {
          rows16_ld(lane_addr + buf * 128 + c * 64, sv);
          if (__builtin_expect(masked, 0)) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int end = TREE ? 0 : last[r] - c * 64;
              const unsigned long long bits = !TREE ? 0ull : c ? seen[r][1] : seen[r][0];
              const uint32_t w[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
#pragma unroll
              for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const bool sees = TREE ? ((w[i >> 2] >> (8 * (i & 3) + e)) & 1u) != 0u : 8 * i + e <= end;
                  sv[4 * i + 2 * r + e] = sees ? sv[4 * i + 2 * r + e] : -INFINITY;
                }
            }
          }
        };
        // One sweep turns this thread's scores into probabilities against references (log2 domain), writes them as packed bf16 and gives
        // their sums, and the largest exponents met, of its two rows.
        float sum[2], top[2];
        auto sweep = [&](float ref0, float ref1) {
          const uint64_t scale2 = pack2(scale_log2, scale_log2), neg2[2] = {pack2(-ref0, -ref0), pack2(-ref1, -ref1)};
          uint64_t rs2[4] = {0ull, 0ull, 0ull, 0ull};
          float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t packed[16];
            if (__builtin_expect(c >= halves, 0)) {
#pragma unroll
              for (int i = 0; i < 16; ++i) packed[i] = 0u;
              rows16_st_pairs(lane_addr + kPCol + buf * 64 + c * 32, packed);
              break;
            }
            float sv[32];
            scores(c, sv);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const int k = 2 * r + (i & 1);
                float x0, x1;
                unpack2(fma2(pack2(sv[4 * i + 2 * r], sv[4 * i + 2 * r + 1]), scale2, neg2[r]), x0, x1);
                tops[k] = max3(tops[k], x0, x1);
                // Probabilities go to the second product in bf16, since kind::f16 multiplies numbers of one type and that is the values': off by 2^-8 of
                // each at most, which averages out over a row's keys.  Their sum is taken before the rounding, in fp32.
                const float p0 = ex2(x0), p1 = ex2(x1);  // -inf -> 0
                rs2[k] = add2(rs2[k], pack2(p0, p1));
                const __nv_bfloat162 pk = __floats2bfloat162_rn(p0, p1);
                packed[2 * i + r] = *reinterpret_cast<const uint32_t*>(&pk);
              }
            }
            rows16_st_pairs(lane_addr + kPCol + buf * 64 + c * 32, packed);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float a, b;
            unpack2(add2(rs2[2 * r], rs2[2 * r + 1]), a, b);
            sum[r] = a + b;
            top[r] = fmaxf(tops[2 * r], tops[2 * r + 1]);
          }
        };
        auto quad_max = [](float v) {
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
        };
        // The running maximum is almost always good enough (it has to be within 2^8 of the true one), so the probabilities are taken against it at
        // once and the tile's maximum is found on the way.  In an item's first tile the largest of the first 8 scores stands in for it.
        if (__builtin_expect(!__all_sync(0xffffffffu, m[0] != -INFINITY && m[1] != -INFINITY), 0)) {
          float v[4];
          rows16_ld(lane_addr + buf * 128, v);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const bool sees0 = !masked || (TREE ? (seen[r][0] & 1ull) != 0ull : 0 <= last[r]), sees1 = !masked || (TREE ? (seen[r][0] & 2ull) != 0ull : 1 <= last[r]);
            const float first = quad_max(fmaxf(sees0 ? v[2 * r] : -INFINITY, sees1 ? v[2 * r + 1] : -INFINITY)) * scale_log2;
            if (m[r] == -INFINITY) m[r] = first;  // (nothing has been added to the row: no product to rescale)
          }
        }
        bool settled = false;
        float mx2[2];
        if (__builtin_expect(__all_sync(0xffffffffu, m[0] != -INFINITY && m[1] != -INFINITY), 1)) {
          sweep(m[0], m[1]);
          settled = !__any_sync(0xffffffffu, fmaxf(top[0], top[1]) > 8.f);
          if (settled) {
            l[0] += sum[0];
            l[1] += sum[1];
          } else {
            mx2[0] = quad_max(top[0]) + m[0];  // exponents were taken against m
            mx2[1] = quad_max(top[1]) + m[1];
          }
        } else {
          mx2[0] = mx2[1] = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            float sv[32];
            scores(c, sv);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float a = -INFINITY, b = -INFINITY;
#pragma unroll
              for (int i = 0; i < 8; i += 2) {
                a = max3(a, sv[4 * i + 2 * r], sv[4 * i + 2 * r + 1]);
                b = max3(b, sv[4 * i + 4 + 2 * r], sv[4 * i + 4 + 2 * r + 1]);
              }
              mx2[r] = max3(mx2[r], a, b);
            }
          }
          mx2[0] = quad_max(mx2[0]) * scale_log2;
          mx2[1] = quad_max(mx2[1]) * scale_log2;
        }
        if (__builtin_expect(!settled, 0)) {
          float alpha[2] = {1.f, 1.f};
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (mx2[r] > m[r] + 8.f || m[r] == -INFINITY) {
              alpha[r] = m[r] == -INFINITY ? 0.f : ex2(m[r] - mx2[r]);
              m[r] = mx2[r];
            }
          if (j > 0 && __any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
            // O may only be touched when no product into it is in flight: that of the tile before must be done (this tile's waits for these rows)
            if (!__all_sync(0xffffffffu, wait_tile(iO + (int)(buf ^ 1u), ((g - 1) >> 1) & 1u))) {
              fail = true;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float v[16];
              rows16_ld(lane_addr + kOCol + c * 32, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] *= alpha[(i >> 1) & 1];
              rows16_st(lane_addr + kOCol + c * 32, v);
            }
          }
          sweep(m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]);
          l[0] = l[0] * alpha[0] + sum[0];
          l[1] = l[1] * alpha[1] + sum[1];
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(bar(iP + (int)buf));
      }
      if (fail) break;
      // the item's sums go to the output threads
      const int slot = (int)(items & 1u);
      if (items >= 2 && !__all_sync(0xffffffffu, wait_tile(iLF + slot, ((items - 2) >> 1) & 1u))) {
        fail = true;
        break;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float t = l[r] + __shfl_xor_sync(0xffffffffu, l[r], 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        if ((lane & 3) == 0) {
          sums[slot * 2 * kBM + row_of[r]] = t;
          sums[(slot * 2 + 1) * kBM + row_of[r]] = m[r];
        }
      }
      mbar_arrive(bar(iL + slot));
      ++items;
    }
    if (fail) {
      tc_wait_st();  // probabilities of a tile that was given up
      if (p.status) atomicOr(p.status, 2);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, kTmem);
}

}  // namespace tc

constexpr size_t ragged_smem(int D) {
  const size_t smem = (size_t)6 * (D / 64) * tc::kBN * 128 + 48 * 8 + 4 * tc::kBM * 4 + tc::kRtRing * 64 + 4 * 4096 + TreeProblem::kSorted * 4 + 1024;
  return smem < 120 * 1024 ? 120 * 1024 : smem;  // one CTA owns an SM: it takes all 512 TMEM columns
}

// Whether the kernel can run on the current device: setmaxnreg would wait for registers that a launch with fewer a thread does not have.
// (A compiler that gives it another number leaves the calls to the CUDA cores.)
template <int D, class P, bool TREE>
static bool ragged_tc_ready() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  static signed char known[64] = {};  // 1: yes, -1: no; both are a device's for good
  if (known[dev] == 0) {
    auto kernel = tc::ragged_tc_kernel<D, P, TREE>;
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess) return false;
    if (attr.numRegs == tc::kRtRegs && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ragged_smem(D)) != cudaSuccess) return false;
    known[dev] = attr.numRegs == tc::kRtRegs ? 1 : -1;
  }
  return known[dev] > 0;
}

template <int D, class P, bool TREE>
static int ragged_tc_go(const TcMaps& maps, const P& p, long long items, int d_head, cudaStream_t st) {
  if (items > 0x7fffffffll) {
    set_error("ragged attention: too many rows");
    return DGPT_E_ARG;
  }
  tc::ragged_tc_kernel<D, P, TREE><<<(unsigned)items, tc::kRtThreads, ragged_smem(D), st>>>(maps.q, maps.k, maps.v, p, d_head);
  return launch_status("ragged attention");
}

template <class P, bool TREE>
static bool tc_type(int D, int dtype) {
  return dtype == DGPT_BF16 && (D == 32 || D == 64 || D == 128) && tc::device_is_sm100() && tc::encode_fn() != nullptr &&
         (D == 128 ? ragged_tc_ready<128, P, TREE>() : ragged_tc_ready<64, P, TREE>());
}

bool packed_tc_supported(const PackedProblem& p, int D, int dtype) { return p.n_keys > 0 && tc_type<PackedProblem, false>(D, dtype); }

int packed_tc(const PackedProblem& full, int D, cudaStream_t st, long long wait_limit) {
  using namespace tc;
  PackedProblem p = full;
  p.wait_limit = wait_limit > 0 ? wait_limit : kWaitLimitCycles;
  TcMaps maps;
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)kBM, 1};
  auto map = [&](CUtensorMap* m, const void* base, int heads, int rows, long long rs, long long hs) {
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows, 1};
    const cuuint64_t strides[3] = {(cuuint64_t)hs * 2, (cuuint64_t)rs * 2, (cuuint64_t)rs * 2};
    return encode_map(m, base, dims, strides, box);
  };
  if (!map(&maps.q, p.q, p.H, p.n_rows, p.q_rs, p.q_hs) || !map(&maps.k, p.k, p.G, p.n_keys, p.k_rs, p.k_hs) ||
      !map(&maps.v, p.v, p.G, p.n_keys, p.v_rs, p.v_hs))
    return DGPT_E_CUDA;
  const long long items = p.slots(kBM) * p.H;
  return D == 128 ? ragged_tc_go<128, PackedProblem, false>(maps, p, items, D, st) : ragged_tc_go<64, PackedProblem, false>(maps, p, items, D, st);
}

// Pages must make up whole key tiles, or be made up by them; one dense run per sequence may have any length: a tile never leaves the
// run's tensor, and what the box covers past its end arrives as zeros.
bool tree_tc_supported(const TreeProblem& p, int dtype) {
  const int pt = p.kv.page_tokens;
  if (!tc_type<TreeProblem, true>(p.D, dtype) || p.group > tc::kBM) return false;
  if (p.kv.head_stride <= 0 || p.kv.page_stride <= 0) return false;
  return p.kv.page_table == nullptr || (pt >= tc::kBN ? pt % tc::kBN == 0 : pt >= 8 && tc::kBN % pt == 0);
}

int tree_tc(const TreeProblem& full, cudaStream_t st) {
  using namespace tc;
  TreeProblem p = full;
  p.wait_limit = kWaitLimitCycles;
  const int nodes = kBM / p.group < p.T ? kBM / p.group : p.T;  // drafts of a tile, with all heads of a group
  p.rows_per_tile = nodes * p.group;
  p.tiles = (p.T + nodes - 1) / nodes;
  const int D = p.D, pt = p.kv.page_tokens;
  TcMaps maps;
  {
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)p.H, (cuuint64_t)p.T, (cuuint64_t)p.B};
    const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)p.q_rs * 2, (cuuint64_t)p.q_rs * p.T * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)p.group, (cuuint32_t)nodes, 1};
    if (!encode_map(&maps.q, p.q, dims, strides, box)) return DGPT_E_CUDA;
  }
  const bool dense = p.kv.page_table == nullptr;
  const cuuint64_t n_pages = dense ? (cuuint64_t)p.B : p.kv.n_pages > 0 ? (cuuint64_t)p.kv.n_pages : (cuuint64_t)1 << 24;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)pt, (cuuint64_t)p.G, n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)p.kv.token_stride * 2, (cuuint64_t)p.kv.head_stride * 2, (cuuint64_t)p.kv.page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)(!dense && pt < kBN ? pt : kBN), 1, 1};
  if (!encode_map(&maps.k, p.kv.k, dims, strides, box) || !encode_map(&maps.v, p.kv.v, dims, strides, box)) return DGPT_E_CUDA;
  return D == 128 ? ragged_tc_go<128, TreeProblem, true>(maps, p, p.items(), D, st) : ragged_tc_go<64, TreeProblem, true>(maps, p, p.items(), D, st);
}

}  // namespace dgpt
