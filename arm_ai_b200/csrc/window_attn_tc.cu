// window_attn_tc.cu — window attention of many queries on the 5th-generation
// tensor cores (f16 and bf16, head width up to 128: 64 or 128 columns, those
// behind the head zero-filled by TMA).
//
//   S = Q K^T, P = exp2(scale S - m), O += P V, over the visible key tiles
//
// A CTA has two tiles of 128 query rows of one key / value head; a row is a
// (token, query head) pair, the heads of a power-of-two part of the group
// inside the token, so that grouped heads share the keys they read and a tile
// spans few tokens: little of a window's edge tiles is masked away. One thread
// streams 64-key tiles of K and V by TMA straight from the cache into a ring; a
// warp per query tile issues its MMAs: S into one of the tile's two 64-column
// score buffers in tensor memory, then O += P V with P (16-bit, written back
// over S) as the A operand from tensor memory and V as the transposed (N-major)
// B operand from the rows as they lie in the cache. Four warps per query tile,
// a thread per row, do its softmax. The tensor cores turn one buffer round (P V
// of a key tile, S of the next but one) while the softmax works on the other.
//
// 8192 tokens, window 4096, 32 / 8 heads of 128, bf16: 355 us = 1160 TFLOP/s of
// the visible pairs. An MMA of 128 x N x 16 with both operands in shared memory
// takes 62 cycles for N = 64 as for N = 128, so S costs what a tile of 128 keys
// would, and the tensor cores are busy for 1540 of a key tile's 1650 cycles;
// the exponentials take 1020. Tiles of 128 keys leave room for one score buffer
// per query tile only, and the wait from P V to the S that overwrites its
// weights then shows: 418 us. Eight warps on one query tile, clusters of three,
// exponentials by polynomial and CTAs that go on to the next tiles were no
// faster. Small calls wait: five prompts of 37 to 1021 tokens, window 256, 32 / 4
// heads of 64 34 us, where a CTA takes 18000 cycles, 8000 of them before its first
// and after its last key tile.
//
// With few query tiles the key tiles are divided over the CTAs of a cluster,
// whose parts are joined through distributed shared memory in rank order
// (chunks of 33 to 61 tokens behind a window of 2048, 64 / 8 heads of 128: 45 ->
// 27.6 us).
//
// Rounding: scores, weights and sums f32; the weights rounded once to the
// tensors' type for P V (wa_weight_shift), the output once at the end.
// Every wait is bounded. What a softmax warp needs comes to it through the warp
// that issues its products: the loader's or the cleaning warp's wait that gives up
// makes a later wait of that warp give up. So an issuing warp that has given up
// says so before it hands over anything more, and the rows of the CTA (with
// divided keys of its cluster) are written as NaN; the device's error word tells
// the host (armai_dev_window_attention_status).
#include <cooperative_groups.h>
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "tcgen05.cuh"
#include "window_attn.cuh"

namespace cg = cooperative_groups;

namespace armai {
namespace {

constexpr int WT_KT = 64;                      // keys per tile
constexpr int WT_ROWS = 128;                   // query rows per tile, two tiles per CTA
constexpr int WT_LOAD = 8, WT_MMA = 9, WT_CLEAN = 11;  // warps 0-3, 4-7: softmax of query tile 0, 1; 9, 10: its MMAs
constexpr int WT_THREADS = 384;

template <int HD>
struct WtLayout {
  static constexpr uint32_t Q = 128u * HD * 2u;     // a query tile: HD / 64 blocks of 128 rows x 128 B
  static constexpr uint32_t KV = WT_KT * HD * 2u;   // a key tile of K or V: HD / 64 blocks of 64 rows x 128 B
  // the first two K tiles, then slots of V of a key tile and K of the next but
  // one: they are used, and given back, together
  static constexpr int SLOTS = 4;
  static constexpr uint32_t K0 = 2 * Q, RING = K0 + 2 * KV;
  static constexpr uint32_t BAR = RING + SLOTS * 2 * KV;
  // More than half of the SM's, so that two CTAs never share one: the second
  // would wait for tensor memory, and in a cluster the first for the second's
  // other ranks.
  static constexpr uint32_t SMEM = 1024 + BAR + 512 > 116u * 1024 ? 1024 + BAR + 512 : 116u * 1024;
};

// tcgen05.ld / st of 32 columns of this warp's 32 lanes; the caller waits.
__device__ __forceinline__ void wt_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Waits for the loads; the values pass through it, so that no use of them is
// moved ahead of it.
__device__ __forceinline__ void wt_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void wt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wt_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ float wt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 operations per instruction.
__device__ __forceinline__ uint64_t wt_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void wt_unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t wt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t wt_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float wt_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T>
__device__ __forceinline__ uint32_t wt_pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t wt_pack<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t wt_pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The weights exp2(scale s - base) of N scores, times the type's factor, as pairs
// of T in w[0 .. N/2 - 1] (which may be the start of s); returns their f32 sum (of
// the unrounded values).
template <typename T, int N>
__device__ __forceinline__ float wt_weights(const uint32_t* s, uint32_t* w, float sl, float base) {
  const float nb = wa_weight_shift<T>() - base;
  const uint64_t sl2 = wt_pair(sl, sl), nb2 = wt_pair(nb, nb);
  uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
  for (int c = 0; c < N / 2; c++) {
    float e0, e1;
    wt_unpair(wt_fma2(wt_pair(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), sl2, nb2), e0, e1);
    e0 = wt_exp2(e0);
    e1 = wt_exp2(e1);
    sum[c & 1] = wt_add2(sum[c & 1], wt_pair(e0, e1));
    w[c] = wt_pack<T>(e0, e1);
  }
  float e0, e1;
  wt_unpair(wt_add2(sum[0], sum[1]), e0, e1);
  return e0 + e1;
}

__device__ __forceinline__ void wt_tma3(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void wt_tma4(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// The CTA's work, the same for every thread: its tokens, each query tile's
// positions, the runs and their tiles.
struct WtWork {
  WaSeq sq;
  int vh, kvh, i0, nt;
  int qlo[2], qhi[2];  // positions of a query tile's first and last token; qhi < qlo: no token

  // whether any row of query tile h sees a key of the tile
  __device__ __forceinline__ bool needs(const WaParams& p, int h, const WaTile& x) const {
    const int lo = h ? qlo[1] : qlo[0], hi = h ? qhi[1] : qhi[0];
    return lo <= hi && x.pos <= hi && (lo - (x.pos + x.n - 1) < p.window || x.pos < p.n_sink);
  }
};

// Waits of a converged warp: one look, and the bounded loop only where that
// was not enough. After a wait that gave up (ok false) no further one waits,
// so the role runs to its end. `failed` (of the CTA, in shared memory) is set by
// the wait that gives up, before the caller commits a product or arrives
// anywhere again.
__device__ __forceinline__ bool wt_wait_slow(uint64_t* bar, uint32_t parity, bool ok, uint32_t* err, uint32_t* failed) {
  if (!ok) return false;
  ok = qg_wait_warp(bar, parity, err);
  if (!ok && failed) {
    *static_cast<volatile uint32_t*>(failed) = 1u;
    __threadfence_block();
  }
  return ok;
}
__device__ __forceinline__ void wt_wait(uint64_t* bar, uint32_t parity, bool& ok, uint32_t* err,
                                        uint32_t* failed = nullptr) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (!__all_sync(0xffffffffu, done)) ok = wt_wait_slow(bar, parity, ok, err, failed);
}

// One lane of a converged warp.
__device__ __forceinline__ bool wt_elect() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e != 0;
}

// The key tiles one after another.
struct WtIter {
  WaTile x;
  int run, left;
  // runs: rows, positions and lengths of the three runs, in shared memory (the
  // roles' loops have no registers to spare)
  __device__ __forceinline__ void enter(const int* runs) {
    x.row = runs[run];
    x.pos = runs[3 + run];
    left = runs[6 + run];
    x.n = min(left, WT_KT);
  }
  __device__ __forceinline__ explicit WtIter(const int* runs) : run(0) { enter(runs); }
  __device__ __forceinline__ void next(const int* runs) {
    x.row += WT_KT;
    x.pos += WT_KT;
    left -= WT_KT;
    x.n = min(left, WT_KT);
    if (left <= 0 && run < 2) {
      run++;
      enter(runs);
    }
  }
};

// The share of a run's tiles that lie in [a, b) of all tiles, t0 of them before it.
__device__ __forceinline__ void wt_share(int& row, int& pos, int& len, int& t0, int a, int b) {
  const int n = (len + WT_KT - 1) / WT_KT;
  const int lo = min(max(a - t0, 0), n), hi = min(max(b - t0, 0), n);
  row += lo * WT_KT;
  pos += lo * WT_KT;
  len = max(min(len, hi * WT_KT) - lo * WT_KT, 0);
  t0 += n;
}

// Place in a ring of N slots: the slot and how often it has been used before.
template <int N>
struct WtSlot {
  int s = 0;
  uint32_t turn = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      turn++;
    }
  }
};

// The parts of an operand descriptor that a kernel's tiles share, and the
// descriptor at an address.
constexpr uint32_t WT_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8-row groups 1024 B apart, 128-B swizzle
__device__ __forceinline__ uint64_t wt_desc(uint32_t lo) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(WT_DESC_HI));
  return d;
}
__device__ __forceinline__ uint32_t wt_desc_lo(uint32_t saddr, uint32_t lead) {
  return ((saddr >> 4) & 0x3FFFu) | (lead >> 4) << 16;
}

template <typename T, int HD>
__global__ void __launch_bounds__(WT_THREADS, 1)
    k_wa_tc(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
            const __grid_constant__ CUtensorMap mv, const WaParams p, int lpack, int lranks) {
  using L = WtLayout<HD>;
  const int pack = 1 << lpack, ranks = 1 << lranks;  // heads per token in a query tile; CTAs per cluster
  extern __shared__ uint8_t wt_raw[];
  const uint32_t raw = smem_u32(wt_raw);
  uint8_t* smem = wt_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* qs = smem;                  // two query tiles
  uint8_t* k0 = smem + L::K0;          // the first two K tiles
  uint8_t* ring = smem + L::RING;      // SLOTS x (V, K of the next key tile but one)
  uint64_t* qfull = reinterpret_cast<uint64_t*>(smem + L::BAR);  // the query tiles and the first K tiles
  uint64_t* full = qfull + 1;          // [SLOTS]
  uint64_t* empty = full + L::SLOTS;   // [SLOTS] both query tiles' products done
  uint64_t* sfull = empty + L::SLOTS;  // [2][2] S of query tile h in its buffer b written
  uint64_t* pready = sfull + 4;        // [2][2] P in place
  uint64_t* pvdone = pready + 4;       // [2][2] P V added
  uint64_t* vclean = pvdone + 4;       // [3] rows behind a short tile of V zeroed (a run has one at most)
  uint64_t* vgo = vclean + 3;          // [3] that tile has landed
  uint64_t* fin = vgo + 3;             // [2] every product done
  uint32_t* tslot = reinterpret_cast<uint32_t*>(fin + 2);
  uint32_t* info = tslot + 1;          // [SLOTS] of a slot's K tile: its keys, and the query tiles that need it
  int* runs = reinterpret_cast<int*>(info + L::SLOTS);  // [9]
  uint32_t* failed = reinterpret_cast<uint32_t*>(runs + 9);  // an issuing warp's wait gave up
  // over the operands, once they are done with: every rank's part of the rows
  // that this rank joins
  cg::cluster_group cluster = cg::this_cluster();
  const int lshare = 8 - lranks, share = 1 << lshare;   // rows: 256 / ranks
  float4* part_o = reinterpret_cast<float4*>(smem);     // [ranks][HD / 4][share]
  float2* part_s = reinterpret_cast<float2*>(smem + 2 * WT_ROWS * HD * 4);  // [ranks][share] maximum, sum

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == WT_MMA * 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  }
  WtWork w;
  w.sq = wa_seq(p, blockIdx.z);
  const int tokens = WT_ROWS >> lpack;  // per query tile
  const int rank = blockIdx.x & (ranks - 1);
  w.i0 = (int)((gridDim.x - 1 - blockIdx.x) >> lranks) * 2 * tokens;  // the longest causal rows first
  if (w.i0 >= w.sq.n) return;          // the whole cluster
  w.vh = blockIdx.y;
  w.kvh = w.vh * pack / p.group;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int t0 = w.i0 + h * tokens;  // behind the last token there may be no position in 32 bits
    w.qlo[h] = t0 < w.sq.n ? w.sq.pos0 + t0 : INT32_MAX;
    w.qhi[h] = t0 < w.sq.n ? w.sq.pos0 + min(w.sq.n, t0 + tokens) - 1 : INT32_MIN;
  }
  {
    WaRuns r = wa_runs(p, w.qlo[0], max(w.qhi[0], w.qhi[1]));
    w.nt = wa_tiles<WT_KT>(r);
    if (ranks > 1) {  // this rank's share
      const int lo = w.nt * rank / ranks, hi = w.nt * (rank + 1) / ranks;
      int t0 = 0;
#pragma unroll
      for (int i = 0; i < 3; i++) wt_share(r.row[i], r.pos[i], r.len[i], t0, lo, hi);
      w.nt = hi - lo;
    }
    if (warp == WT_LOAD) {
      // a lane per barrier
      const int nb = (int)(reinterpret_cast<uint64_t*>(tslot) - qfull);
      if (lane < nb) {
        const uint64_t* b = qfull + lane;
        mbar_init(qfull + lane, b >= empty && b < sfull ? 2 : b >= pready && b < pvdone ? 4 : b >= vgo && b < fin ? 2 : 1);
      }
      fence_mbar_init();
      __syncwarp();
    }
    if (tid == WT_LOAD * 32) {
      *failed = 0u;
      // without the empty runs: a loop goes from one to the next
      int k = 0;
#pragma unroll
      for (int i = 0; i < 3; i++) {
        if (r.len[i] > 0) {
          runs[k] = r.row[i];
          runs[3 + k] = r.pos[i];
          runs[6 + k] = r.len[i];
          k++;
        }
      }
      for (; k < 3; k++) runs[k] = runs[3 + k] = runs[6 + k] = 0;
      // the query tiles and the first K tiles are on their way before the CTA meets
      mbar_arrive_tx(qfull, 2 * L::Q + (uint32_t)min(w.nt, 2) * L::KV);
      for (int h = 0; h < 2; h++)
        for (int kb = 0; kb < HD / 64; kb++)
          wt_tma3(qs + h * L::Q + kb * 16384, &mq, 64 * kb, w.vh * pack, w.sq.q0 + w.i0 + h * tokens, qfull);
      WtIter it(runs);
      for (int t = 0; t < min(w.nt, 2); t++, it.next(runs))
        for (int kb = 0; kb < HD / 64; kb++)
          wt_tma4(k0 + t * L::KV + kb * 8192, &mk, 64 * kb, it.x.row, w.kvh, w.sq.slot, qfull);
    }
  }
  if (warp == WT_MMA) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // The whole of tensor memory, so from column 0 on: S of query tile h, buffer
  // b from 128 h + 64 b (P over the first half of it), O of query tile h from
  // 256 + 128 h.
  constexpr uint32_t tmem = 0;

  if (warp < WT_LOAD) {
    // ---- softmax: thread = query row ----
    const int h = warp >> 2, row = tid & 127;
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t to = tmem + lane_base + 256u + 128u * (uint32_t)h;
    const int tok = w.i0 + h * tokens + (row >> lpack), head = w.vh * pack + (row & (pack - 1));
    const int qpos = w.sq.pos0 + min(tok, w.sq.n - 1);  // rows behind the last token: as that, not written
    const float sl = p.scale_log2;
    float m = -INFINITY, l = 0.f;
    int n = 0;
    bool ok = true;
    // waits for the last product issued for these rows
    auto products = [&]() { wt_wait(&pvdone[2 * h + ((n - 1) & 1)], (uint32_t)((n - 1) >> 1 & 1), ok, p.err); };
    WtIter it(runs);
#pragma unroll 1
    for (int t = 0; t < w.nt; t++, it.next(runs)) {
      const WaTile x = it.x;
      if (!w.needs(p, h, x)) continue;
      const uint32_t ts = tmem + lane_base + 128u * (uint32_t)h + 64u * (uint32_t)(n & 1);
      // columns first .. last are seen, and those before `sink`
      const int last = min(x.n - 1, qpos - x.pos), first = qpos - x.pos - p.window + 1, sink = p.n_sink - x.pos;
      const bool all = __all_sync(0xffffffffu, last == WT_KT - 1 && (first <= 0 || sink >= WT_KT));
      // the maximum is raised to a larger score: the sum and the output so far follow
      auto raise = [&](float top) {
        if (__any_sync(0xffffffffu, top > m + WA_SLACK)) {
          const float nm = fmaxf(m, top);
          const float f = nm == -INFINITY ? 1.f : wt_exp2(m - nm);
          m = nm;
          l *= f;
          if (n > 0) {
            products();
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              wt_ld32(to + c, o);
              wt_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              wt_st32(to + c, o);
            }
          }
        }
      };
      wt_wait(&sfull[2 * h + (n & 1)], (uint32_t)(n >> 1 & 1), ok, p.err);
      tc_fence_after();
      if (all) {
        uint32_t s[64];
        wt_ld32(ts, s);
        wt_ld32(ts + 32u, s + 32);
        wt_wait_ld(s);
        wt_wait_ld(s + 32);
        float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; c += 8)
#pragma unroll
          for (int k = 0; k < 4; k++)
            a[k] = wt_max3(a[k], __uint_as_float(s[c + 2 * k]), __uint_as_float(s[c + 2 * k + 1]));
        raise(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])) * sl);
        l += wt_weights<T, 64>(s, s, sl, m == -INFINITY ? 0.f : m);
        wt_st32(ts, s);
      } else {
        // an edge tile, 32 columns at a time and twice over (few instructions:
        // seldom run, they are never in the instruction cache); P of a block
        // overwrites scores that have been read
        auto seen = [&](int c) {
          const int le = last - c + 1, ge = first - c, si = sink - c;
          const uint32_t ml = le >= 32 ? 0xffffffffu : le <= 0 ? 0u : (1u << le) - 1u;
          const uint32_t mg = ge >= 32 ? 0u : ge <= 0 ? 0xffffffffu : 0xffffffffu << ge;
          const uint32_t ms = si >= 32 ? 0xffffffffu : si <= 0 ? 0u : (1u << si) - 1u;
          return ml & (mg | ms);
        };
        auto load = [&](int c, uint32_t mask, uint32_t (&r)[32]) {
          wt_ld32(ts + c, r);
          wt_wait_ld(r);
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (!(mask >> e & 1)) r[e] = 0xff800000u;  // -inf
        };
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < x.n; c += 32) {
          const uint32_t mask = seen(c);
          if (!__any_sync(0xffffffffu, mask)) continue;
          uint32_t r[32];
          load(c, mask, r);
#pragma unroll
          for (int e = 0; e < 32; e += 2) top = wt_max3(top, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
        }
        raise(top * sl);
#pragma unroll 1
        for (int c = 0; c < x.n; c += 32) {
          const uint32_t mask = seen(c);
          uint32_t w16[16];
          if (__any_sync(0xffffffffu, mask)) {
            uint32_t r[32];
            load(c, mask, r);
            l += wt_weights<T, 32>(r, w16, sl, m == -INFINITY ? 0.f : m);
          } else {
#pragma unroll
            for (int e = 0; e < 16; e++) w16[e] = 0u;
          }
          qg_tmem_st16(ts + (c >> 1), w16);
        }
      }
      wt_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive1(&pready[2 * h + (n & 1)]);
      n++;
    }
    if (n > 0) {
      products();
      ok = ok && !*static_cast<volatile uint32_t*>(failed);
    }
    tc_fence_after();
    if (ranks == 1) {
      const bool none = n == 0 || l == 0.f;  // no key seen
      const float inv = ok ? 1.0f / l : __int_as_float(0x7fc00000);
      T* out = static_cast<T*>(p.out) + (int64_t)(w.sq.q0 + tok) * p.o_token + (int64_t)head * p.o_head;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        wt_ld32(to + c, o);
        wt_wait_ld(o);
        if (tok < w.sq.n) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
              v[k] = ok && none ? 0u
                                : wt_pack<T>(__uint_as_float(o[e + 2 * k]) * inv, __uint_as_float(o[e + 2 * k + 1]) * inv);
            if (c + e < p.head_dim) *reinterpret_cast<uint4*>(out + c + e) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    } else {
      // Each row's part goes to the rank that joins the row (remote stores: no
      // latency to wait for), once every rank is done with its operands.
      cluster.sync();
      const int r = tid, owner = r >> lshare;
      float4* to_o = cluster.map_shared_rank(part_o, owner) + rank * (HD / 4) * share + (r & (share - 1));
      float2* to_s = cluster.map_shared_rank(part_s, owner) + rank * share + (r & (share - 1));
      *to_s = make_float2(m, ok ? l : __int_as_float(0x7fc00000));
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        wt_ld32(to + c, o);
        wt_wait_ld(o);
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          to_o[(c + e) / 4 * share] =
              n == 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                     : make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                                   __uint_as_float(o[e + 3]));
      }
    }
  } else if (warp == WT_LOAD) {
    if (lane == 0) {
      WtIter iv(runs), ik(runs);  // the key tiles whose V, whose K comes next
      ik.next(runs);
      ik.next(runs);
      WtSlot<L::SLOTS> slot;
      int issued = 0;
      bool ok = true;
      for (int t = 0; t < w.nt; t++) {
        const bool more = t + 2 < w.nt;
        if (slot.turn) ok = qg_wait(&empty[slot.s], (slot.turn - 1) & 1, p.err);
        if (!ok) break;
        // what the issuing warps have to know of the slot's K tile
        info[slot.s] =
            more ? (uint32_t)ik.x.n | (uint32_t)w.needs(p, 0, ik.x) << 8 | (uint32_t)w.needs(p, 1, ik.x) << 9 : 0u;
        uint8_t* dst = ring + slot.s * 2 * L::KV;
        mbar_arrive_tx(&full[slot.s], (more ? 2 : 1) * L::KV);
        for (int kb = 0; kb < HD / 64; kb++)
          wt_tma4(dst + kb * 8192, &mv, 64 * kb, iv.x.row, w.kvh, w.sq.slot, &full[slot.s]);
        if (more)
          for (int kb = 0; kb < HD / 64; kb++)
            wt_tma4(dst + L::KV + kb * 8192, &mk, 64 * kb, ik.x.row, w.kvh, w.sq.slot, &full[slot.s]);
        slot.next();
        iv.next(runs);
        ik.next(runs);
        issued = t + 1;
      }
      // every requested box has landed before the CTA may end
      qg_wait(qfull, 0, p.err);
      for (int t = issued > L::SLOTS ? issued - L::SLOTS : 0; t < issued; t++)
        qg_wait(&full[t % L::SLOTS], (uint32_t)((t / L::SLOTS) & 1), p.err);
    }
  } else if (warp < WT_CLEAN) {
    // ---- products of query tile h. The whole warp walks the loop, so that the
    // operands' descriptors stay in uniform registers; one elected lane issues.
    const int h = warp - WT_MMA;
    constexpr uint32_t TY = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t BASE = (1u << 4) | (TY << 7) | (TY << 10) | ((uint32_t)(WT_ROWS >> 4) << 24);
    constexpr uint32_t PV = BASE | (1u << 16) | ((uint32_t)(HD >> 3) << 17);  // B transposed
    const uint32_t qa = wt_desc_lo(smem_u32(qs), 16) + (uint32_t)h * (L::Q >> 4);
    const uint32_t klo = wt_desc_lo(smem_u32(k0), 16), rlo = wt_desc_lo(smem_u32(ring), 16);
    const uint32_t ts = tmem + 128u * (uint32_t)h, to = tmem + 256u + 128u * (uint32_t)h;
    bool ok = true;
    uint32_t cleaned = 0;
    int nq = 0, np = 0;  // products S and P V issued
    auto qk = [&](int keys, uint32_t ka) {
      const int b = nq & 1;
      // its buffer held P of the key tile two before
      if (nq >= 2) wt_wait(&pvdone[2 * h + b], (uint32_t)((nq >> 1) - 1) & 1, ok, p.err, failed);
      tc_fence_after();
      const uint32_t idesc = BASE | ((uint32_t)((keys + 15) >> 4) << 18);  // N: the tile's keys, in steps of 16
      if (wt_elect()) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++)
          tc_mma_ss(ts + 64u * (uint32_t)b, wt_desc(qa + (uint32_t)(kk >> 2) * 1024u + 2u * (uint32_t)(kk & 3)),
                    wt_desc(ka + (uint32_t)(kk >> 2) * 512u + 2u * (uint32_t)(kk & 3)), idesc, kk > 0);
        qg_commit(&sfull[2 * h + b]);
      }
      __syncwarp();
      nq++;
    };
    // of the key tiles now, next and next but one: keys | whether this query tile needs them << 8
    uint32_t now = 0, next = 0;
    wt_wait(qfull, 0, ok, p.err, failed);
    {
      WtIter it(runs);
      if (w.nt > 0) now = (uint32_t)it.x.n | (uint32_t)w.needs(p, h, it.x) << 8;
      it.next(runs);
      if (w.nt > 1) next = (uint32_t)it.x.n | (uint32_t)w.needs(p, h, it.x) << 8;
      if (now >> 8) qk((int)(now & 255u), klo);
      if (next >> 8) qk((int)(next & 255u), klo + (L::KV >> 4));
    }
    WtSlot<L::SLOTS> slot;
    uint32_t word = 0;
    // the slot's tiles have landed, rows behind a short V tile are zeroed
    auto arrived = [&](int keys) {
      wt_wait(&full[slot.s], slot.turn & 1, ok, p.err, failed);
      word = info[slot.s];
      if (keys & 15) {
        if (lane == 0) mbar_arrive1(&vgo[cleaned]);
        wt_wait(&vclean[cleaned++], 0, ok, p.err, failed);
      }
    };
    if (w.nt > 0) arrived((int)(now & 255u));
    // The schedulers are busy with the softmax, and every step from a weight to
    // the next score but one is waited for: what can be done while P V runs
    // (looking after the next slot) is done there.
#pragma unroll 1
    for (int t = 0; t < w.nt; t++) {
      const uint32_t after = (word & 255u) | (word >> (8 + h) & 1) << 8;
      const int keys = (int)(now & 255u), s = slot.s;
      const uint32_t base = rlo + (uint32_t)s * (2 * L::KV >> 4);
      if (now >> 8) {
        const int b = np & 1;
        const uint32_t va = base + ((8192u - 16u) >> 4 << 16);  // 64-wide blocks of the row 8 KB apart
        wt_wait(&pready[2 * h + b], (uint32_t)(np >> 1) & 1, ok, p.err, failed);
        tc_fence_after();
        if (wt_elect()) {
#pragma unroll
          for (int kk = 0; kk < WT_KT / 16; kk++)
            if (16 * kk < keys)
              qg_mma_ts(to, ts + 64u * (uint32_t)b + 8u * kk, wt_desc(va + 128u * kk), PV, kk > 0 ? 1u : np > 0);
          qg_commit(&pvdone[2 * h + b]);
        }
        __syncwarp();
        np++;
      }
      now = next;
      next = after;
      slot.next();
      if (t + 1 < w.nt) arrived((int)(now & 255u));
      if (after >> 8) qk((int)(after & 255u), base + (L::KV >> 4));
      if (wt_elect()) qg_commit(&empty[s]);
      __syncwarp();
    }
    // no product is in flight when tensor memory is given back, failed waits or not
    if (wt_elect()) qg_commit(&fin[h]);
    __syncwarp();
    ok = true;
    wt_wait(&fin[h], 0, ok, p.err, failed);
  } else {
    // the last product of 16 keys of a short tile also reads rows behind the
    // tile's: zero them (their weights are zero, but the rows may hold anything)
    WtIter it(runs);
    WtSlot<L::SLOTS> slot;
    int cleaned = 0;
    for (int t = 0; t < w.nt; t++) {
      if (it.x.n & 15) {
        if (!qg_wait_warp(&vgo[cleaned], 0, p.err)) break;
        const int rows = 16 - (it.x.n & 15);
        for (int e = lane; e < rows * (HD / 8); e += 32)
          *reinterpret_cast<uint4*>(ring + slot.s * 2 * L::KV + (e & 7) * 16 + (it.x.n + (e >> 3) % rows) * 128 +
                                    ((e >> 3) / rows) * 8192) = make_uint4(0u, 0u, 0u, 0u);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive1(&vclean[cleaned]);
        cleaned++;
      }
      slot.next();
      it.next(runs);
    }
  }
  if (ranks > 1 && warp >= WT_LOAD) {
    __syncwarp();
    cluster.sync();  // the softmax warps' first
  }
  tc_fence_before();
  __syncthreads();
  if (warp == WT_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (ranks > 1) {
    cluster.sync();  // the parts of this rank's rows have come
    // 256 threads, so that a thread keeps its row where a share is at most 256
    // rows: the weights of the ranks' parts are made once per row
    if (warp < WT_LOAD) {
      const int i = tid & (share - 1), r = rank * share + i;
      const int tok = w.i0 + (r >> lpack), head = w.vh * pack + (r & (pack - 1));  // query tile 1 follows tile 0
      float m = -INFINITY, l = 0.f, f[8];
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (k < ranks) m = fmaxf(m, part_s[k * share + i].x);
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        f[k] = 0.f;
        if (k < ranks) {
          const float2 st = part_s[k * share + i];
          f[k] = wt_exp2(st.x - base);
          l += f[k] * st.y;
        }
      }
      const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key seen: 0 * 0
#pragma unroll
      for (int k = 0; k < 8; k++) f[k] *= inv;
      T* out = static_cast<T*>(p.out) + (int64_t)(w.sq.q0 + tok) * p.o_token + (int64_t)head * p.o_head;
      if (tok < w.sq.n) {
        // eight columns at a time
        for (int c = 2 * (tid >> lshare); c < HD / 4; c += 2 * (256 >> lshare)) {
          float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 8; k++)
            if (k < ranks) {
              const float4 v = part_o[(k * (HD / 4) + c) * share + i], u = part_o[(k * (HD / 4) + c + 1) * share + i];
              o[0] += f[k] * v.x, o[1] += f[k] * v.y, o[2] += f[k] * v.z, o[3] += f[k] * v.w;
              o[4] += f[k] * u.x, o[5] += f[k] * u.y, o[6] += f[k] * u.z, o[7] += f[k] * u.w;
            }
          if (4 * c < p.head_dim)
            *reinterpret_cast<uint4*>(out + 4 * c) = make_uint4(wt_pack<T>(o[0], o[1]), wt_pack<T>(o[2], o[3]),
                                                                wt_pack<T>(o[4], o[5]), wt_pack<T>(o[6], o[7]));
        }
      }
    }
  }
}

PFN_cuTensorMapEncodeTiled_v12000 wt_encoder() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

bool wt_map(CUtensorMap* map, int dtype, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box) {
  const auto enc = wt_encoder();
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return enc &&
         enc(map, dtype == ARMAI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank,
             const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Error word of this kernel's bounded waits (one per device that loads the
// library); read and cleared by armai_dev_window_attention_status.
__device__ uint32_t g_wt_err;

template <typename T, int HD>
int wt_launch(const WaParams& in, int dtype, cudaStream_t s, bool* fits) {
  WaParams p = in;
  const int n_kv = p.n_q_heads / p.group;
  int lpack = 0;  // heads per token in a query tile: the power of two in the group
  while (lpack < 7 && p.group % (2 << lpack) == 0) lpack++;
  const int pack = 1 << lpack;
  CUtensorMap mq, mk, mv;
  const cuuint64_t qd[3] = {(cuuint64_t)p.head_dim, (cuuint64_t)p.n_q_heads, (cuuint64_t)p.n_tokens};
  const cuuint64_t qst[2] = {(cuuint64_t)p.q_head * 2, (cuuint64_t)p.q_token * 2};
  const cuuint32_t qb[3] = {64, (cuuint32_t)pack, (cuuint32_t)(WT_ROWS / pack)};
  const cuuint64_t kd[4] = {(cuuint64_t)p.head_dim, (cuuint64_t)p.kv_rows, (cuuint64_t)n_kv, (cuuint64_t)p.n_slots};
  const cuuint64_t kst[3] = {(cuuint64_t)p.kv_row * 2, (cuuint64_t)p.kv_head * 2, (cuuint64_t)p.kv_slot * 2};
  const cuuint32_t kb[4] = {64, WT_KT, 1, 1};
  *fits = wt_map(&mq, dtype, 3, p.q, qd, qst, qb) && wt_map(&mk, dtype, 4, p.k, kd, kst, kb) &&
          wt_map(&mv, dtype, 4, p.v, kd, kst, kb);
  if (!*fits) return ARMAI_OK;
  ARMAI_CUDA(cudaGetSymbolAddress((void**)&p.err, g_wt_err));
  ARMAI_CUDA(cudaFuncSetAttribute(k_wa_tc<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WtLayout<HD>::SMEM));
  const int tokens = 2 * WT_ROWS / pack;
  const int64_t blocks = (p.max_q + tokens - 1) / tokens, ctas = blocks * (p.n_q_heads / pack) * p.n_seq;
  // The keys divided over clusters, as long as these run all at once and four
  // key tiles at least are left for each CTA (4100 visible keys, heads of 128: 64
  // or 72 CTAs by two 41 against 66 us; 32 by four 26.8 against 39.6 by two; 80,
  // which do not fit twice, 66.7).
  const int64_t keys = std::min<int64_t>(p.kv_rows, (int64_t)p.window + p.n_sink + tokens);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)(p.n_q_heads / pack), (unsigned)p.n_seq);
  cfg.blockDim = dim3(WT_THREADS);
  cfg.dynamicSmemBytes = WtLayout<HD>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int lranks = 0;
  for (int log2 = 1; log2 <= 3 && keys >= (int64_t)4 * WT_KT << log2 && ctas << log2 <= sm_count(); log2++) {
    cfg.gridDim.x = (unsigned)(blocks << log2);
    attr[0].val.clusterDim.x = 1u << log2;
    if (ctas > wa_clusters<k_wa_tc<T, HD>>(log2, cfg)) break;
    lranks = log2;
  }
  const int ranks = 1 << lranks;
  cfg.gridDim.x = (unsigned)(blocks * ranks);
  attr[0].val.clusterDim.x = (unsigned)ranks;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  ARMAI_CUDA(cudaLaunchKernelEx(&cfg, k_wa_tc<T, HD>, mq, mk, mv, p, lpack, lranks));
  return ARMAI_OK;
}

}  // namespace

int wa_tc_launch(const WaParams& p, int dtype, cudaStream_t s, bool* fits) {
  *fits = dtype != ARMAI_F32 && p.head_dim <= 128 && p.head_dim % 8 == 0 && p.scale_log2 > 0.f;
  if (!*fits) return ARMAI_OK;
  const bool narrow = p.head_dim <= 64;
  if (dtype == ARMAI_F16) return narrow ? wt_launch<__half, 64>(p, dtype, s, fits) : wt_launch<__half, 128>(p, dtype, s, fits);
  return narrow ? wt_launch<__nv_bfloat16, 64>(p, dtype, s, fits) : wt_launch<__nv_bfloat16, 128>(p, dtype, s, fits);
}

}  // namespace armai

extern "C" int armai_dev_window_attention_status(void) {
  using namespace armai;
  uint32_t e = 0;
  ARMAI_CUDA(cudaMemcpyFromSymbol(&e, g_wt_err, sizeof e));
  if (!e) return ARMAI_OK;
  const uint32_t zero = 0;
  ARMAI_CUDA(cudaMemcpyToSymbol(g_wt_err, &zero, sizeof zero));
  return fail(ARMAI_E_DEVICE, "window_attn: a wait of the tensor-core kernel gave up (error word " + std::to_string(e) +
                                  "); its rows are NaN");
}
