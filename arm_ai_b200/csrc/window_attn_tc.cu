// window_attn_tc.cu — window attention of many queries on the 5th-generation
// tensor cores (f16 and bf16, head width 64 or 128).
//
//   S = Q K^T, P = exp2(scale S - m), O += P V, over the visible key tiles
//
// A CTA has two tiles of 128 query rows of one key / value head; a row is a
// (token, query head) pair, the heads of a power-of-two part of the group
// inside the token, so that grouped heads share the keys they read and a tile
// spans few tokens: little of a window's edge tiles is masked away. One thread
// streams 128-key tiles of K and V by TMA straight from the cache into a ring;
// one thread issues the MMAs: S of each query tile into its 128 columns of
// tensor memory, then O += P V with P (16-bit, written back over S) as the A
// operand from tensor memory and V as the transposed (N-major) B operand from
// the rows as they lie in the cache. Four warps per query tile, one thread
// per row, do the softmax: no exchange between threads. While one tile's
// softmax runs, the tensor cores work on the other's products.
//
// The row's maximum is raised, and its output in tensor memory rescaled, only
// when a score exceeds it by more than 2^8: then weights stay below 2^8, sums
// far inside f32, and most tiles need no pass over the output.
//
// Rounding: scores, weights and sums f32; the weights rounded once to the
// tensors' type for P V (half a step each), the output once at the end.
// Every wait is bounded; rows whose wait gave up are written as NaN.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "tcgen05.cuh"
#include "window_attn.cuh"

namespace armai {
namespace {

constexpr int WT_KT = 128;                     // keys per tile
constexpr int WT_ROWS = 128;                   // query rows per tile, two tiles per CTA
constexpr int WT_LOAD = 8, WT_MMA = 9, WT_CLEAN = 10;  // warps 0-3, 4-7: softmax of tile 0, 1
constexpr int WT_THREADS = 384;                // warp 11 only completes the warp group
// Registers: 384 x 168 at launch; the loading group gives up what the softmax
// threads (128 scores each) need: 256 x 200 + 128 x 104 = 384 x 168.
constexpr int WT_REGS = 168, WT_REGS_SOFTMAX = 200, WT_REGS_LOAD = 104;
static_assert(256 * WT_REGS_SOFTMAX + 128 * WT_REGS_LOAD <= WT_THREADS * WT_REGS, "register split");
constexpr float WT_SLACK = 8.f;

template <int HD>
struct WtLayout {
  static constexpr uint32_t TILE = 128u * HD * 2u;       // one operand tile: HD / 64 blocks of 128 rows x 128 B
  static constexpr int SLOTS = HD == 128 ? 5 : 8;        // K and V tiles in turn
  static constexpr uint32_t BAR = (2 + SLOTS) * TILE;
  static constexpr uint32_t SMEM = 1024 + BAR + 512;
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

// The weights exp2(scale s - base) of N scores, as pairs of T in w[0 .. N/2 - 1]
// (which may be the start of s); returns their f32 sum (of the unrounded values).
template <typename T, int N>
__device__ __forceinline__ float wt_weights(const uint32_t* s, uint32_t* w, float sl, float base) {
  const uint64_t sl2 = wt_pair(sl, sl), nb2 = wt_pair(-base, -base);
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
// so the role runs to its end.
__device__ __forceinline__ bool wt_wait_slow(uint64_t* bar, uint32_t parity, bool ok, uint32_t* err) {
  return ok && qg_wait_warp(bar, parity, err);
}
__device__ __forceinline__ void wt_wait(uint64_t* bar, uint32_t parity, bool& ok, uint32_t* err) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (!__all_sync(0xffffffffu, done)) ok = wt_wait_slow(bar, parity, ok, err);
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
            const __grid_constant__ CUtensorMap mv, const WaParams p, int pack) {
  using L = WtLayout<HD>;
  extern __shared__ uint8_t wt_raw[];
  const uint32_t raw = smem_u32(wt_raw);
  uint8_t* smem = wt_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* qs = smem;                  // two query tiles
  uint8_t* ring = smem + 2 * L::TILE;  // SLOTS tiles: K of a key tile, then V
  uint64_t* qfull = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* full = qfull + 1;          // [SLOTS]
  uint64_t* empty = full + L::SLOTS;   // [SLOTS]
  uint64_t* sfull = empty + L::SLOTS;  // [2] S of query tile h written
  uint64_t* pready = sfull + 2;        // [2] P of query tile h in place
  uint64_t* pvdone = pready + 2;       // [2] P V of query tile h added
  uint64_t* vclean = pvdone + 2;       // [3] rows behind a short tile of V zeroed (a run has one at most)
  uint64_t* vgo = vclean + 3;          // [3] that tile has landed
  uint64_t* fin = vgo + 3;             // every product done
  uint32_t* tslot = reinterpret_cast<uint32_t*>(fin + 1);  // two words, then the runs (9)

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  WtWork w;
  w.sq = wa_seq(p, blockIdx.z);
  const int tokens = WT_ROWS / pack;   // per query tile
  w.i0 = (int)(gridDim.x - 1 - blockIdx.x) * 2 * tokens;  // the longest causal rows first
  if (w.i0 >= w.sq.n) return;
  w.vh = blockIdx.y;
  w.kvh = w.vh * pack / p.group;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    w.qlo[h] = w.sq.pos0 + w.i0 + h * tokens;
    w.qhi[h] = w.sq.pos0 + min(w.sq.n, w.i0 + (h + 1) * tokens) - 1;
  }
  int* runs = reinterpret_cast<int*>(fin + 2);
  {
    const WaRuns r = wa_runs(p, w.qlo[0], max(w.qhi[0], w.qhi[1]));
    w.nt = wa_tiles<WT_KT>(r);
    if (tid == 0) {
#pragma unroll
      for (int i = 0; i < 3; i++) {
        runs[i] = r.row[i];
        runs[3 + i] = r.pos[i];
        runs[6 + i] = r.len[i];
      }
    }
  }

  if (tid == 0) {
    mbar_init(qfull, 1);
    mbar_init(fin, 1);
    for (int i = 0; i < 3; i++) {
      mbar_init(&vclean[i], 1);
      mbar_init(&vgo[i], 1);
    }
    for (int i = 0; i < L::SLOTS; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int h = 0; h < 2; h++) {
      mbar_init(&sfull[h], 1);
      mbar_init(&pready[h], 4);
      mbar_init(&pvdone[h], 1);
    }
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // the whole of tensor memory, so from column 0 on: S 0 in 0-127, S 1 in 128-255, O 0 from 256, O 1 from 384
  constexpr uint32_t tmem = 0;

  if (warp < WT_LOAD) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(WT_REGS_SOFTMAX));
    // ---- softmax: thread = query row ----
    const int h = warp >> 2, row = tid & 127;
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lane_base + 128u * (uint32_t)h, to = ts + 256u;
    const int tok = w.i0 + h * tokens + row / pack, head = w.vh * pack + row % pack;
    const int qpos = w.sq.pos0 + tok;
    const float sl = p.scale_log2;
    float m = -INFINITY, l = 0.f;
    int n = 0;
    bool ok = true;
    WtIter it(runs);
    for (int t = 0; t < w.nt; t++, it.next(runs)) {
      const WaTile x = it.x;
      if (!w.needs(p, h, x)) continue;
      wt_wait(&sfull[h], (uint32_t)(n & 1), ok, p.err);
      tc_fence_after();
      // columns first .. last are seen, and those before `sink`
      const int last = min(x.n - 1, qpos - x.pos), first = qpos - x.pos - p.window + 1, sink = p.n_sink - x.pos;
      const bool all = last == WT_KT - 1 && (first <= 0 || sink >= WT_KT);
      float sum = 0.f;
      // the maximum is raised to a larger score: the sum and the output so far follow
      auto raise = [&](float top) {
        if (__any_sync(0xffffffffu, top > m + WT_SLACK)) {
          const float nm = fmaxf(m, top);
          const float f = nm == -INFINITY ? 1.f : wt_exp2(m - nm);
          m = nm;
          l *= f;
          if (n > 0) {
            wt_wait(&pvdone[h], (uint32_t)((n - 1) & 1), ok, p.err);
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
      if (__all_sync(0xffffffffu, all)) {
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 4; c++) wt_ld32(ts + 32u * c, s + 32 * c);
#pragma unroll
        for (int c = 0; c < 4; c++) wt_wait_ld(s + 32 * c);
        float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; c += 8)
#pragma unroll
          for (int k = 0; k < 4; k++)
            a[k] = wt_max3(a[k], __uint_as_float(s[c + 2 * k]), __uint_as_float(s[c + 2 * k + 1]));
        raise(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])) * sl);
        sum = wt_weights<T, 128>(s, s, sl, m == -INFINITY ? 0.f : m);
        wt_st32(ts, s);
        wt_st32(ts + 32u, s + 32);
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
            sum += wt_weights<T, 32>(r, w16, sl, m == -INFINITY ? 0.f : m);
          } else {
#pragma unroll
            for (int e = 0; e < 16; e++) w16[e] = 0u;
          }
          qg_tmem_st16(ts + (c >> 1), w16);
        }
      }
      l += sum;
      wt_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive1(&pready[h]);
      n++;
    }
    if (n > 0) wt_wait(&pvdone[h], (uint32_t)((n - 1) & 1), ok, p.err);
    tc_fence_after();
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
          *reinterpret_cast<uint4*>(out + c + e) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(WT_REGS_LOAD));
    if (warp == WT_LOAD) {
      if (lane == 0) {
        mbar_arrive_tx(qfull, 2 * L::TILE);
        for (int h = 0; h < 2; h++)
          for (int kb = 0; kb < HD / 64; kb++)
            wt_tma3(qs + h * L::TILE + kb * 16384, &mq, 64 * kb, w.vh * pack, w.sq.q0 + w.i0 + h * tokens, qfull);
        WtIter it(runs);
        WtSlot<L::SLOTS> slot;
        int issued = 0;
        bool ok = true;
        for (int j = 0; j < 2 * w.nt; j++) {
          if (slot.turn) ok = qg_wait(&empty[slot.s], (slot.turn - 1) & 1, p.err);
          if (!ok) break;
          mbar_arrive_tx(&full[slot.s], L::TILE);
          for (int kb = 0; kb < HD / 64; kb++)
            wt_tma4(ring + slot.s * L::TILE + kb * 16384, (j & 1) ? &mv : &mk, 64 * kb, it.x.row, w.kvh, w.sq.slot,
                    &full[slot.s]);
          slot.next();
          issued = j + 1;
          if (j & 1) it.next(runs);
        }
        // every requested box has landed before the CTA may end
        qg_wait(qfull, 0, p.err);
        for (int j = issued > L::SLOTS ? issued - L::SLOTS : 0; j < issued; j++)
          qg_wait(&full[j % L::SLOTS], (uint32_t)((j / L::SLOTS) & 1), p.err);
      }
    } else if (warp == WT_MMA) {
      // The whole warp walks the loop, so that the operands' descriptors stay in
      // uniform registers; one elected lane issues.
      constexpr uint32_t TY = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t BASE = (1u << 4) | (TY << 7) | (TY << 10) | ((uint32_t)(WT_ROWS >> 4) << 24);
      constexpr uint32_t PV = BASE | (1u << 16) | ((uint32_t)(HD >> 3) << 17);  // B transposed
      const uint32_t qlo = wt_desc_lo(smem_u32(qs), 16), rlo = wt_desc_lo(smem_u32(ring), 16);
      bool ok = true;
      wt_wait(qfull, 0, ok, p.err);
      WtIter it(runs);
      WtSlot<L::SLOTS> slot;
      uint32_t cleaned = 0;
      // bit h: query tile h takes part in the key tile; has had a product P V; the parity of their number
      uint32_t need = 0, begun = 0, par = 0;
      // S of query tile h with the K tile in slot s
      auto qk = [&](int h, const WaTile& x, int s) {
        // its columns held P of the tile before
        if (begun >> h & 1) wt_wait(&pvdone[h], (par >> h & 1) ^ 1, ok, p.err);
        tc_fence_after();
        const uint32_t idesc = BASE | ((uint32_t)((x.n + 15) >> 4) << 18);  // N: the tile's keys, in steps of 16
        const uint32_t qa = qlo + (uint32_t)h * (L::TILE >> 4), ka = rlo + (uint32_t)s * (L::TILE >> 4);
        if (wt_elect()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; kk++) {
            const uint32_t off = (uint32_t)(kk >> 2) * 1024u + 2u * (uint32_t)(kk & 3);
            tc_mma_ss(tmem + 128u * (uint32_t)h, wt_desc(qa + off), wt_desc(ka + off), idesc, kk > 0);
          }
          qg_commit(&sfull[h]);
        }
        __syncwarp();
      };
      if (w.nt > 0) {
        need = w.needs(p, 0, it.x) | w.needs(p, 1, it.x) << 1;
        wt_wait(&full[0], 0, ok, p.err);
#pragma unroll 1
        for (int h = 0; h < 2; h++)
          if (need >> h & 1) qk(h, it.x, 0);
        if (wt_elect()) qg_commit(&empty[0]);
        __syncwarp();
      }
      // Every step of this loop lies on the path between a weight and the next
      // score, and its code is refetched each time (the softmax's fills the
      // instruction caches): one copy for both query tiles, few branches.
#pragma unroll 1
      for (int t = 0; t < w.nt; t++) {
        const WaTile x = it.x;
        slot.next();
        const WtSlot<L::SLOTS> v = slot;
        slot.next();
        it.next(runs);
        const bool more = t + 1 < w.nt;
        const uint32_t next = more ? w.needs(p, 0, it.x) | w.needs(p, 1, it.x) << 1 : 0;
        wt_wait(&full[v.s], v.turn & 1, ok, p.err);
        if (more) wt_wait(&full[slot.s], slot.turn & 1, ok, p.err);
        if (x.n & 15) {
          if (lane == 0) mbar_arrive1(&vgo[cleaned]);
          wt_wait(&vclean[cleaned++], 0, ok, p.err);
        }
        // 64-wide blocks of the row 16 KB apart
        const uint32_t va = rlo + (uint32_t)v.s * (L::TILE >> 4) + ((16384u - 16u) >> 4 << 16);
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
          if (need >> h & 1) {
            const uint32_t o = tmem + 256u + 128u * (uint32_t)h, pa = tmem + 128u * (uint32_t)h;
            wt_wait(&pready[h], par >> h & 1, ok, p.err);
            tc_fence_after();
            if (wt_elect()) {
#pragma unroll
              for (int kk = 0; kk < WT_KT / 16; kk++)
                if (16 * kk < x.n)
                  qg_mma_ts(o, pa + 8u * kk, wt_desc(va + 128u * kk), PV, kk > 0 ? 1u : begun >> h & 1);
              qg_commit(&pvdone[h]);
            }
            __syncwarp();
            begun |= 1u << h;
            par ^= 1u << h;
          }
          if (next >> h & 1) qk(h, it.x, slot.s);
        }
        if (wt_elect()) {
          qg_commit(&empty[v.s]);
          if (more) qg_commit(&empty[slot.s]);
        }
        __syncwarp();
        need = next;
      }
      // no product is in flight when tensor memory is given back, failed waits or not
      if (wt_elect()) qg_commit(fin);
      __syncwarp();
      ok = true;
      wt_wait(fin, 0, ok, p.err);
    } else if (warp == WT_CLEAN) {
      // the last product of 16 keys of a short tile also reads rows behind the
      // tile's: zero them (their weights are zero, but the rows may hold anything)
      WtIter it(runs);
      WtSlot<L::SLOTS> slot;
      int cleaned = 0;
      for (int t = 0; t < w.nt; t++) {
        slot.next();
        if (it.x.n & 15) {
          if (!qg_wait_warp(&vgo[cleaned], 0, p.err)) break;
          const int rows = 16 - (it.x.n & 15);
          for (int e = lane; e < rows * (HD / 8); e += 32)
            *reinterpret_cast<uint4*>(ring + slot.s * L::TILE + (e & 7) * 16 + (it.x.n + (e >> 3) % rows) * 128 +
                                      ((e >> 3) / rows) * 16384) = make_uint4(0u, 0u, 0u, 0u);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive1(&vclean[cleaned]);
          cleaned++;
        }
        slot.next();
        it.next(runs);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
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

__device__ uint32_t g_wt_err;

template <typename T, int HD>
int wt_launch(const WaParams& in, int dtype, cudaStream_t s, bool* fits) {
  WaParams p = in;
  const int n_kv = p.n_q_heads / p.group;
  int pack = 1;  // heads per token in a tile: the power of two in the group
  while (pack < 128 && p.group % (2 * pack) == 0) pack *= 2;
  CUtensorMap mq, mk, mv;
  const cuuint64_t qd[3] = {(cuuint64_t)HD, (cuuint64_t)p.n_q_heads, (cuuint64_t)p.n_tokens};
  const cuuint64_t qst[2] = {(cuuint64_t)p.q_head * 2, (cuuint64_t)p.q_token * 2};
  const cuuint32_t qb[3] = {64, (cuuint32_t)pack, (cuuint32_t)(WT_ROWS / pack)};
  const cuuint64_t kd[4] = {(cuuint64_t)HD, (cuuint64_t)p.kv_rows, (cuuint64_t)n_kv, (cuuint64_t)p.n_slots};
  const cuuint64_t kst[3] = {(cuuint64_t)p.kv_row * 2, (cuuint64_t)p.kv_head * 2, (cuuint64_t)p.kv_slot * 2};
  const cuuint32_t kb[4] = {64, WT_KT, 1, 1};
  *fits = wt_map(&mq, dtype, 3, p.q, qd, qst, qb) && wt_map(&mk, dtype, 4, p.k, kd, kst, kb) &&
          wt_map(&mv, dtype, 4, p.v, kd, kst, kb);
  if (!*fits) return ARMAI_OK;
  ARMAI_CUDA(cudaGetSymbolAddress((void**)&p.err, g_wt_err));
  // the register split waits for registers that a smaller launch would not have
  static thread_local int regs = 0;
  if (!regs) {
    cudaFuncAttributes fa;
    ARMAI_CUDA(cudaFuncGetAttributes(&fa, k_wa_tc<T, HD>));
    regs = fa.numRegs;
  }
  if (regs != WT_REGS) return fail(ARMAI_E_INVALID, "window_attn: the tensor-core kernel was built with " + std::to_string(regs) + " registers");
  ARMAI_CUDA(cudaFuncSetAttribute(k_wa_tc<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WtLayout<HD>::SMEM));
  const int tokens = 2 * WT_ROWS / pack;
  const dim3 grid((unsigned)((p.max_q + tokens - 1) / tokens), (unsigned)(p.n_q_heads / pack), (unsigned)p.n_seq);
  k_wa_tc<T, HD><<<grid, WT_THREADS, WtLayout<HD>::SMEM, s>>>(mq, mk, mv, p, pack);
  ARMAI_CUDA(cudaGetLastError());
  return ARMAI_OK;
}

}  // namespace

int wa_tc_launch(const WaParams& p, int dtype, cudaStream_t s, bool* fits) {
  *fits = dtype != ARMAI_F32 && (p.head_dim == 64 || p.head_dim == 128) && p.scale_log2 > 0.f;
  if (!*fits) return ARMAI_OK;
  if (dtype == ARMAI_F16) return p.head_dim == 64 ? wt_launch<__half, 64>(p, dtype, s, fits) : wt_launch<__half, 128>(p, dtype, s, fits);
  return p.head_dim == 64 ? wt_launch<__nv_bfloat16, 64>(p, dtype, s, fits) : wt_launch<__nv_bfloat16, 128>(p, dtype, s, fits);
}

}  // namespace armai
