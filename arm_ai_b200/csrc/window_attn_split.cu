// window_attn_split.cu — window attention of few queries per sequence (single
// tokens, short chunks): the visible keys are split over the warps of a
// thread-block cluster and the parts joined through distributed shared memory.
//
// Bound by the bytes of the visible keys and values. A warp takes tiles of 16
// keys in turn with the cluster's other warps and keeps its own running
// maximum, sum and output, so no warp waits for another until the end. Its
// tiles arrive by asynchronous 16-byte copies (4-byte ones where rows do not
// start on 16 bytes), whole lines at a time, into a two-deep ring of its own. The order of the values within a row is free in
// both products, as long as q and k (or p and v) agree, so each lane's operands
// are whole 16-byte chunks.
//   16-bit types: m16n8k16 tensor instructions, 16 rows = (token, query head)
//   pairs of one key / value head, so a key is read once for all of them.
//   f32: products on the CUDA cores, 8 lanes per key. One stream of 4096 keys,
//   8 heads of 256: 15.7 us; 12 streams, 16 heads of 128: 139 us = 5.8 TB/s.
// Where the 5th-generation tensor cores cannot take 16-bit tensors, many queries
// come here too, in blocks of 16 rows that each read their keys, from L2 for the
// most part (4096 tokens, 32 / 8 heads of 128, a negative scale: 0.84 ms = 164
// TFLOP/s).
// The cluster's parts are joined in rank order: results do not depend on
// timing, no workspace, one launch.
#include <cooperative_groups.h>

#include <algorithm>

#include "llama_kernels.cuh"
#include "window_attn.cuh"

namespace cg = cooperative_groups;

namespace armai {
namespace {

// Warps per CTA by (padded) head width: beyond 128 a ring fills half an SM's
// shared memory, so that one CTA has to do; its warps are as many as their
// rings leave room for.
__host__ __device__ constexpr int sp_warps(int dt) { return dt > 128 ? 6 : 4; }
constexpr int SP_STAGES = 2;
constexpr int SP_MAX_SPLIT = 16;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4_or_zero(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float sp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a CTA works on: rows f0 .. f0 + nr - 1 of the (token, query head of
// the group) pairs of one sequence and key / value head.
struct SpBlock {
  WaSeq sq;
  int kvh, f0, nr;
  int qmin, qmax;  // positions of its first and last token
  WaRuns runs;
};
template <int R>
__device__ __forceinline__ bool sp_block(const WaParams& p, int split, SpBlock& b) {
  // blockIdx.x: rank of 2^split in the cluster, key / value head, block of rows (one, for single tokens)
  const int block = (int)blockIdx.x >> split, rb = (int)gridDim.x >> split == p.n_kv ? 0 : block / p.n_kv;
  b.kvh = block - rb * p.n_kv;
  b.f0 = rb * R;
  b.sq = wa_seq(p, blockIdx.y);
  b.nr = min(R, b.sq.n * p.group - b.f0);
  if (b.nr <= 0) return false;  // the same for the whole cluster
  b.qmin = b.sq.pos0 + wa_token(p, b.f0);
  b.qmax = b.sq.pos0 + wa_token(p, b.f0 + b.nr - 1);
  b.runs = wa_runs(p, b.qmin, b.qmax);
  return true;
}

// A warp's tiles, every step-th of KT keys through the runs.
template <int KT>
struct SpCursor {
  int run, off, row, pos, len;  // the run, the tile's place in it, and the run's own
  __device__ __forceinline__ void enter(const WaRuns& r) {
    row = run == 0 ? r.row[0] : run == 1 ? r.row[1] : r.row[2];
    pos = run == 0 ? r.pos[0] : run == 1 ? r.pos[1] : r.pos[2];
    len = run == 0 ? r.len[0] : run == 1 ? r.len[1] : r.len[2];
  }
  __device__ __forceinline__ SpCursor(const WaRuns& r, int tile) : run(0) {
    enter(r);
    off = 0;
    advance(r, tile);
  }
  __device__ __forceinline__ void advance(const WaRuns& r, int tiles) {
    off += tiles * KT;
    while (off >= len && run < 3) {  // into the next run: its tiles start where this one's ended
      off -= (len + KT - 1) / KT * KT;
      run++;
      if (run < 3) enter(r);
    }
  }
  __device__ __forceinline__ bool valid() const { return run < 3; }
  __device__ __forceinline__ int first_row() const { return row + off; }
  __device__ __forceinline__ int first_pos() const { return pos + off; }
  __device__ __forceinline__ int keys() const { return min(KT, len - off); }
};

__device__ __forceinline__ void sp_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void sp_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// What the ranks of a cluster send one another: the outputs of the values
// (rows x DT / 4 vectors) that a rank joins, from every rank, and all rows'
// maxima and sums. Behind the ring, which may still be in use.
template <int R, int DT>
struct SpMail {
  float4 o[R * DT / 4 + SP_MAX_SPLIT];
  float2 s[SP_MAX_SPLIT][R];
};

// Joins the warps' parts ([warp][R][DT] unnormalised outputs, [warp][R] maxima
// and sums in shared memory) within the CTA, then over the cluster, and writes
// the rows. Every rank joins a share of the values; the others send it theirs
// (remote stores: no latency to wait for). The caller has arrived at the
// cluster's barrier before, so that every rank's mail box is there.
template <typename T, int R, int DT, int CB>
__device__ __forceinline__ void sp_join(const WaParams& p, int split, const SpBlock& b, const float* part,
                                        const float* wm, const float* wl, SpMail<R, DT>* mail) {
  constexpr int WARPS = sp_warps(DT);
  const int tid = threadIdx.x, items = b.nr * (DT / 4);
  const int ranks = 1 << split, rank = (int)blockIdx.x & (ranks - 1), per = (items + ranks - 1) / ranks;
  auto write = [&](int r, int d, const float4& acc, float l) {
    if (d >= p.head_dim) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;  // an empty row: 0 * 0; NaN kept
    const int f = b.f0 + r, tok = wa_token(p, f);
    T* o = static_cast<T*>(p.out) + (int64_t)(b.sq.q0 + tok) * p.o_token +
           (int64_t)(b.kvh * p.group + f - tok * p.group) * p.o_head + d;
    if constexpr (CB < 16) {
      const float x[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
      for (int e = 0; e < 4; e += 4 / (int)sizeof(T)) {
        if (d + e >= p.head_dim) return;
        if constexpr (sizeof(T) == 4)
          o[e] = x[e];
        else
          *reinterpret_cast<uint32_t*>(o + e) = pack2<T>(x[e], x[e + 1]);
      }
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(o) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    } else {
      *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
    }
  };
  cg::cluster_group cluster = cg::this_cluster();
  __syncthreads();
  if (ranks > 1) sp_cluster_wait();
  for (int e = tid; e < items; e += 32 * WARPS) {
    const int r = e / (DT / 4), d = (e % (DT / 4)) * 4;
    float m = wm[r], l = 0.f;
#pragma unroll
    for (int w = 1; w < WARPS; w++) m = fmaxf(m, wm[w * R + r]);
    const float base = m == -INFINITY ? 0.f : m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f = sp_exp2(wm[w * R + r] - base);
      const float4 v = *reinterpret_cast<const float4*>(part + (w * R + r) * DT + d);
      l += f * wl[w * R + r];
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    if (ranks == 1) {
      write(r, d, acc, l);
    } else {
      const int owner = e / per;
      *cluster.map_shared_rank(&mail->o[rank * per + e - owner * per], owner) = acc;
      if (d / 4 < ranks) *cluster.map_shared_rank(&mail->s[rank][r], d / 4) = make_float2(m, l);  // DT / 4 >= 8 ranks
      if (DT / 4 < SP_MAX_SPLIT && d / 4 + DT / 4 < ranks)
        *cluster.map_shared_rank(&mail->s[rank][r], d / 4 + DT / 4) = make_float2(m, l);
    }
  }
  if (ranks == 1) return;
  sp_cluster_arrive();
  sp_cluster_wait();
  for (int e = rank * per + tid; e < min(items, (rank + 1) * per); e += 32 * WARPS) {
    const int r = e / (DT / 4), i = e - rank * per;
    float m = -INFINITY, l = 0.f;
    for (int k = 0; k < ranks; k++) m = fmaxf(m, mail->s[k][r].x);
    const float base = m == -INFINITY ? 0.f : m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < ranks; k++) {
      const float2 st = mail->s[k][r];
      const float4 v = mail->o[k * per + i];
      const float f = sp_exp2(st.x - base);
      l += f * st.y;
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    write(r, (e % (DT / 4)) * 4, acc, l);
  }
}

// ---------------------------------------------------------------------------
// 16-bit types. DT: head width, padded to 64, 128 or 256 (chunks beyond
// head_dim are zero-filled). Lane (g = lane / 4, c = lane % 4).
//   S = Q K^T: step s = 2 i + h of 16 takes the d = 8 (c + 4 i) + 4 h .. + 3
//   of lane c, for q and k alike.
//   O = P V: lane holds, for the tile's keys 2c, 2c+1, 2c+8, 2c+9, the
//   d = 64 b + 8 g .. + 7; product (b, e) has d = 64 b + 8 n + e as column n,
//   so a lane's outputs are the 16 values from 64 b + 16 c on.
// ---------------------------------------------------------------------------
constexpr int SP_ROWS = 16, SP_KT = 16;

// The eight lanes of one shared-memory access read, of K, four chunks of two
// consecutive keys; of V, two chunks of four keys two apart.
__device__ __forceinline__ int sp_swz_k(int key) { return (key & 1) << 2; }
__device__ __forceinline__ int sp_swz_v(int key) { return key & 6; }

template <typename T, int DT>
__host__ __device__ constexpr size_t sp_smem() {
  const size_t ring = (size_t)sp_warps(DT) * SP_STAGES * 2 * SP_KT * DT * 2;
  const size_t join = (size_t)sp_warps(DT) * SP_ROWS * (DT + 2) * 4;
  return ring > join ? ring : join;  // one after the other
}

// CB: bytes of a copy, 16 or (rows that do not start on 16 bytes, head widths
// of no whole 16 bytes) 4.
template <typename T, int DT, int CB>
__global__ void __launch_bounds__(32 * sp_warps(DT)) k_wa_split(const WaParams p, int split) {
  constexpr int WARPS = sp_warps(DT);
  constexpr int KC = DT / 32, VB = DT / 64;       // k chunks per key and lane; 64-wide blocks of v
  constexpr uint32_t TILE = SP_KT * DT * 2;       // a tile of K or V
  extern __shared__ __align__(16) uint8_t sm[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  SpBlock b;
  if (!sp_block<SP_ROWS>(p, split, b)) return;
  if (split) sp_cluster_arrive();
  const int chunks = p.head_dim >> 3;             // valid 16-byte chunks of a row
  const bool whole = p.head_dim == DT;
  // copies: 16-byte chunk cc of key ck + RPC i, consecutive lanes consecutive
  // chunks (requests of whole lines: half lines cost a third of the bandwidth);
  // chunk x of a row lies at x ^ swizzle of the key, so that the reads below
  // are free of bank conflicts
  constexpr int RC = DT / 8, RPC = 32 / RC;       // chunks per row, rows per copy instruction
  const int ck = lane / RC, cc = lane % RC;
  const int64_t kv_off = (int64_t)b.sq.slot * p.kv_slot + (int64_t)b.kvh * p.kv_head;
  const int64_t row = p.kv_row, tile_stride = (int64_t)(WARPS * SP_KT << split) * row;
  const T* kb = static_cast<const T*>(p.k) + kv_off + (CB == 16 ? ck * row + 8 * cc : 2 * lane);
  const T* vb = static_cast<const T*>(p.v) + kv_off + (CB == 16 ? ck * row + 8 * cc : 2 * lane);
  const uint8_t* ring = sm + warp * (SP_STAGES * 2 * TILE);
  const uint32_t ring32 = smem_u32(ring);
  const int step = WARPS << split, first = ((int)blockIdx.x & ((1 << split) - 1)) * WARPS + warp;

  SpCursor<SP_KT> cur(b.runs, first), ahead = cur;
  int64_t at = (int64_t)ahead.first_row() * row;  // of the loads' tile, in values from kb and vb
  auto load = [&](uint32_t dst) {
    if (ahead.valid()) {
      const int n = ahead.keys();
      const T* k = kb + at;
      const T* v = vb + at;
      if constexpr (CB == 16) {
#pragma unroll
        for (int i = 0; i < SP_KT / RPC; i++) {
          const int key = ck + RPC * i;
          const uint32_t dk = dst + key * (RC * 16) + ((cc ^ sp_swz_k(key)) << 4);
          const uint32_t dv = dst + TILE + key * (RC * 16) + ((cc ^ sp_swz_v(key)) << 4);
          if (whole && n == SP_KT) {
            cp16(dk, k + RPC * i * row);
            cp16(dv, v + RPC * i * row);
          } else {  // keys behind a short tile's end and chunks behind the head are zero
            const bool ok = key < n && cc < chunks;
            cp16_or_zero(dk, ok ? k + RPC * i * row : static_cast<const T*>(p.k), ok);
            cp16_or_zero(dv, ok ? v + RPC * i * row : static_cast<const T*>(p.v), ok);
          }
        }
      } else {
        // words lane + 32 i of a row, consecutive lanes consecutive words
#pragma unroll 4
        for (int key = 0; key < SP_KT; key++)
#pragma unroll
          for (int i = 0; i < DT / 64; i++) {
            const int word = lane + 32 * i, x = word >> 2;
            const bool ok = key < n && 2 * word < p.head_dim;
            const uint32_t at = dst + key * (RC * 16) + (word & 3) * 4;
            cp4_or_zero(at + ((x ^ sp_swz_k(key)) << 4), ok ? k + key * row + 64 * i : static_cast<const T*>(p.k), ok);
            cp4_or_zero(at + TILE + ((x ^ sp_swz_v(key)) << 4), ok ? v + key * row + 64 * i : static_cast<const T*>(p.v), ok);
          }
      }
      const int run = ahead.run;
      ahead.advance(b.runs, step);
      at = ahead.run == run ? at + tile_stride : (int64_t)ahead.first_row() * row;
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < SP_STAGES; s++) load(ring32 + s * 2 * TILE);

  // q rows g and g + 8; rows beyond the block are zero. A negative scale turns
  // q's signs instead, so that larger products always mean larger scores.
  uint32_t qa[KC][2][4];
  int qpos[2];
  const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
  const float sl = fabsf(p.scale_log2);
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int r = g + 8 * j, f = b.f0 + (r < b.nr ? r : 0);
    const int tok = wa_token(p, f);
    qpos[j] = b.sq.pos0 + tok;
    const T* src = static_cast<const T*>(p.q) + (int64_t)(b.sq.q0 + tok) * p.q_token +
                   (int64_t)(b.kvh * p.group + f - tok * p.group) * p.q_head;
#pragma unroll
    for (int i = 0; i < KC; i++) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (CB == 16) {
        if (r < b.nr && c + 4 * i < chunks) v = *reinterpret_cast<const uint4*>(src + 8 * (c + 4 * i));
      } else {
        const auto word = [&](int d) {
          return r < b.nr && d < p.head_dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
        };
        const int d = 8 * (c + 4 * i);
        v = make_uint4(word(d), word(d + 2), word(d + 4), word(d + 6));
      }
      qa[i][0][j] = v.x ^ flip;
      qa[i][0][2 + j] = v.y ^ flip;
      qa[i][1][j] = v.z ^ flip;
      qa[i][1][2 + j] = v.w ^ flip;
    }
  }
  const int qmin = b.qmin, qmax = b.qmax;

  float o[VB][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < VB; i++)
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int k = 0; k < 4; k++) o[i][e][k] = 0.f;

  // the lane's operands in a tile: K chunk c + 4 i of keys g and g + 8; V chunk
  // g + 8 i of keys 2c, 2c + 1, 2c + 8, 2c + 9 (one swizzle for the four)
  const uint32_t flipped = 64u * (g & 1);  // odd keys: the chunks of even and odd i change places
  const uint32_t kread[2] = {g * (RC * 16) + 16 * c + flipped, g * (RC * 16) + 16 * c - flipped};
  const uint32_t vread = TILE + 2 * c * (RC * 16) + ((g ^ sp_swz_v(2 * c)) << 4);
  int slot = 0;
#pragma unroll 1
  while (cur.valid()) {
    const uint8_t* src = ring + slot * 2 * TILE;
    cp_wait<SP_STAGES - 1>();
    __syncwarp();
    // s[j][0, 1]: row g, keys 8 j + 2 c, + 1; s[j][2, 3]: row g + 8. Two sums
    // each, for shorter chains (one at a width of 256, for its registers).
    constexpr bool TWO = DT < 256;
    float s[2][4], s2[TWO ? 2 : 1][4];
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int k = 0; k < 4; k++) s[j][k] = s2[TWO ? j : 0][k] = 0.f;
#pragma unroll
    for (int i = 0; i < KC; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint4 v = *reinterpret_cast<const uint4*>(src + kread[i & 1] + j * 8 * (RC * 16) + i * 64);
        mma16816<T>(s[j], qa[i][0], v.x, v.y);
        mma16816<T>(TWO ? s2[TWO ? j : 0] : s[j], qa[i][1], v.z, v.w);
      }
    const int pos = cur.first_pos(), n = cur.keys();
    cur.advance(b.runs, step);
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int k = 0; k < 4; k++) s[j][k] += TWO ? s2[TWO ? j : 0][k] : 0.f;
    if (!(n == SP_KT && pos + SP_KT - 1 <= qmin && (qmax - pos < p.window || pos + SP_KT - 1 < p.n_sink))) {
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int key = 8 * j + 2 * c + (k & 1);
          if (key >= n || !wa_sees(p, qpos[k >> 1], pos + key)) s[j][k] = -INFINITY;
        }
    }
    const float top[2] = {fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])) * sl,
                          fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])) * sl};
    if (__any_sync(0xffffffffu, top[0] > m[0] + WA_SLACK || top[1] > m[1] + WA_SLACK)) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        float y = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 1));
        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
        const float nm = fmaxf(m[j], y);
        const float f = nm == -INFINITY ? 1.f : sp_exp2(m[j] - nm);
        m[j] = nm;
        l[j] *= f;
#pragma unroll
        for (int i = 0; i < VB; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            o[i][e][2 * j] *= f;
            o[i][e][2 * j + 1] *= f;
          }
      }
    }
    uint32_t pa[4];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float base = (m[j] == -INFINITY ? 0.f : m[j]) - wa_weight_shift<T>();
      const float p0 = sp_exp2(fmaf(s[0][2 * j], sl, -base)), p1 = sp_exp2(fmaf(s[0][2 * j + 1], sl, -base));
      const float p2 = sp_exp2(fmaf(s[1][2 * j], sl, -base)), p3 = sp_exp2(fmaf(s[1][2 * j + 1], sl, -base));
      l[j] += (p0 + p1) + (p2 + p3);
      pa[j] = pack2<T>(p0, p1);      // rounded to T for the product, see wa_weight_shift
      pa[2 + j] = pack2<T>(p2, p3);
    }
#pragma unroll
    for (int i = 0; i < VB; i++) {
      const uint8_t* vs = src + vread + i * 128;
      const uint4 v0 = *reinterpret_cast<const uint4*>(vs), v1 = *reinterpret_cast<const uint4*>(vs + RC * 16);
      const uint4 v2 = *reinterpret_cast<const uint4*>(vs + 8 * RC * 16), v3 = *reinterpret_cast<const uint4*>(vs + 9 * RC * 16);
      const uint32_t a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
      const uint32_t a2[4] = {v2.x, v2.y, v2.z, v2.w}, a3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        mma16816<T>(o[i][2 * e], pa, __byte_perm(a0[e], a1[e], 0x5410), __byte_perm(a2[e], a3[e], 0x5410));
        mma16816<T>(o[i][2 * e + 1], pa, __byte_perm(a0[e], a1[e], 0x7632), __byte_perm(a2[e], a3[e], 0x7632));
      }
    }
    __syncwarp();  // every lane has read what the slot held
    load(ring32 + slot * 2 * TILE);
    slot = slot + 1 == SP_STAGES ? 0 : slot + 1;
  }
  cp_wait<0>();
  __syncthreads();  // the ring becomes the join area
  float* part = reinterpret_cast<float*>(sm);
  float* wm = part + WARPS * SP_ROWS * DT;
  float* wl = wm + WARPS * SP_ROWS;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
    l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
    const int r = g + 8 * j;
    if (c == 0) {
      wm[warp * SP_ROWS + r] = m[j];
      wl[warp * SP_ROWS + r] = l[j];
    }
#pragma unroll
    for (int i = 0; i < VB; i++)
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4*>(part + (warp * SP_ROWS + r) * DT + 64 * i + 16 * c + 8 * n + e) =
              make_float4(o[i][e][2 * j + n], o[i][e + 1][2 * j + n], o[i][e + 2][2 * j + n], o[i][e + 3][2 * j + n]);
  }
  sp_join<T, SP_ROWS, DT, CB>(p, split, b, part, wm, wl, reinterpret_cast<SpMail<SP_ROWS, DT>*>(sm + sp_smem<T, DT>()));
}

// ---------------------------------------------------------------------------
// f32: R rows (1, 2, 4 or 8), 8 lanes per key, lane x of them the chunks
// x + 8 i of 4 values; 4 keys at once, 8 per stage. The R partial dots are
// exchanged so that a lane ends with one row's whole score (R = 8: 7 shuffles
// for 8 rows), makes that row's weight, and hands it back to the 8 lanes.
// ---------------------------------------------------------------------------
constexpr int SF_KT = 8;

template <int CH>
__host__ __device__ constexpr size_t sf_smem(int rows) {
  const size_t ring = (size_t)sp_warps(32 * CH) * SP_STAGES * 2 * SF_KT * CH * 32 * 4;
  const size_t join = (size_t)sp_warps(32 * CH) * rows * (CH * 32 + 2) * 4;
  return ring > join ? ring : join;  // one after the other
}

template <int R, int CH, int CB>
__global__ void __launch_bounds__(32 * sp_warps(32 * CH)) k_wa_split_f32(const WaParams p, int split) {
  constexpr int DT = 32 * CH, WARPS = sp_warps(DT);
  constexpr int SH = R == 8 ? 0 : R == 4 ? 1 : R == 2 ? 2 : 3;  // lanes per row of the 8: 2^SH
  extern __shared__ __align__(16) uint8_t sm[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kg = lane >> 3, x8 = lane & 7;
  SpBlock b;
  if (!sp_block<R>(p, split, b)) return;
  if (split) sp_cluster_arrive();
  const int chunks = p.head_dim >> 2;
  const int64_t kv_off = (int64_t)b.sq.slot * p.kv_slot + (int64_t)b.kvh * p.kv_head;
  const float* kb = static_cast<const float*>(p.k) + kv_off;
  const float* vb = static_cast<const float*>(p.v) + kv_off;
  float4* ring = reinterpret_cast<float4*>(sm) + warp * (SP_STAGES * 4 * CH * 32) + lane;
  const int step = WARPS << split, first = ((int)blockIdx.x & ((1 << split) - 1)) * WARPS + warp;
  const int nt = wa_tiles<SF_KT>(b.runs);

  auto load = [&](int t, int slot) {
    if (t < nt) {
      const WaTile x = wa_tile<SF_KT>(b.runs, t);
      float4* dst = ring + slot * 4 * CH * 32;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int key = kg + 4 * j;
        const int64_t off = (int64_t)(x.row + (key < x.n ? key : 0)) * p.kv_row;
#pragma unroll
        for (int i = 0; i < CH; i++) {
          if constexpr (CB == 16) {
            const bool ok = key < x.n && x8 + 8 * i < chunks;
            cp16_or_zero(smem_u32(dst + (j * CH + i) * 32), kb + off + (ok ? 4 * (x8 + 8 * i) : 0), ok);
            cp16_or_zero(smem_u32(dst + ((2 + j) * CH + i) * 32), vb + off + (ok ? 4 * (x8 + 8 * i) : 0), ok);
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int d = 4 * (x8 + 8 * i) + e;
              const bool ok = key < x.n && d < p.head_dim;
              cp4_or_zero(smem_u32(dst + (j * CH + i) * 32) + 4 * e, kb + off + (ok ? d : 0), ok);
              cp4_or_zero(smem_u32(dst + ((2 + j) * CH + i) * 32) + 4 * e, vb + off + (ok ? d : 0), ok);
            }
          }
        }
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < SP_STAGES; s++) load(first + s * step, s);

  float4 q[R][CH], o[R][CH];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int f = b.f0 + (r < b.nr ? r : 0);
    const int tok = wa_token(p, f);
    const float* src = static_cast<const float*>(p.q) + (int64_t)(b.sq.q0 + tok) * p.q_token +
                       (int64_t)(b.kvh * p.group + f - tok * p.group) * p.q_head;
#pragma unroll
    for (int i = 0; i < CH; i++) {
      o[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      q[r][i] = o[r][i];
      const int d = 4 * (x8 + 8 * i);
      if (r < b.nr && (CB == 16 ? x8 + 8 * i < chunks : d < p.head_dim)) {
        float4 v;
        if constexpr (CB == 16)
          v = *reinterpret_cast<const float4*>(src + d);
        else
          v = make_float4(src[d], d + 1 < p.head_dim ? src[d + 1] : 0.f, d + 2 < p.head_dim ? src[d + 2] : 0.f,
                          d + 3 < p.head_dim ? src[d + 3] : 0.f);
        q[r][i] = make_float4(v.x * p.scale_log2, v.y * p.scale_log2, v.z * p.scale_log2, v.w * p.scale_log2);
      }
    }
  }
  const int mine = x8 >> SH;  // the row whose scores this lane ends with
  const int qpos = b.sq.pos0 + wa_token(p, b.f0 + min(mine, b.nr - 1));
  float m = -INFINITY, l = 0.f;

  int slot = 0;
#pragma unroll 1
  for (int t = first; t < nt; t += step) {
    const WaTile x = wa_tile<SF_KT>(b.runs, t);
    cp_wait<SP_STAGES - 1>();
    const float4* src = ring + slot * 4 * CH * 32;
    float s[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      float d[R];
#pragma unroll
      for (int r = 0; r < R; r++) d[r] = 0.f;
#pragma unroll
      for (int i = 0; i < CH; i++) {
        const float4 k = src[(j * CH + i) * 32];
#pragma unroll
        for (int r = 0; r < R; r++)
          d[r] += q[r][i].x * k.x + q[r][i].y * k.y + q[r][i].z * k.z + q[r][i].w * k.w;
      }
      int nr = R;
#pragma unroll
      for (int w = 4; w >= 1; w >>= 1) {
        if (nr > 1) {
          nr >>= 1;
#pragma unroll
          for (int r = 0; r < R / 2; r++)
            if (r < nr) {
              const bool up = (lane & w) != 0;
              const float send = up ? d[r] : d[r + nr], keep = up ? d[r + nr] : d[r];
              d[r] = keep + __shfl_xor_sync(0xffffffffu, send, w);
            }
        } else {
          d[0] += __shfl_xor_sync(0xffffffffu, d[0], w);
        }
      }
      const int key = kg + 4 * j;
      s[j] = key < x.n && wa_sees(p, qpos, x.pos + key) ? d[0] : -INFINITY;
    }
    const float top = fmaxf(s[0], s[1]);
    if (__any_sync(0xffffffffu, top > m + WA_SLACK)) {
      float y = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
      const float nm = fmaxf(m, y);
      const float f = nm == -INFINITY ? 1.f : exp2f(m - nm);
      m = nm;
      l *= f;
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float fr = __shfl_sync(0xffffffffu, f, (lane & 24) | (r << SH));
#pragma unroll
        for (int i = 0; i < CH; i++)
          o[r][i] = make_float4(o[r][i].x * fr, o[r][i].y * fr, o[r][i].z * fr, o[r][i].w * fr);
      }
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float e = exp2f(s[j] - base);
      l += e;
      float w[R];
#pragma unroll
      for (int r = 0; r < R; r++) w[r] = __shfl_sync(0xffffffffu, e, (lane & 24) | (r << SH));
#pragma unroll
      for (int i = 0; i < CH; i++) {
        const float4 v = src[((2 + j) * CH + i) * 32];
#pragma unroll
        for (int r = 0; r < R; r++) {
          o[r][i].x += w[r] * v.x;
          o[r][i].y += w[r] * v.y;
          o[r][i].z += w[r] * v.z;
          o[r][i].w += w[r] * v.w;
        }
      }
    }
    load(t + SP_STAGES * step, slot);
    slot = slot + 1 == SP_STAGES ? 0 : slot + 1;
  }
  cp_wait<0>();
  __syncthreads();
  // the warp's four key groups added up (they share the row's maximum)
  l += __shfl_xor_sync(0xffffffffu, l, 8);
  l += __shfl_xor_sync(0xffffffffu, l, 16);
  float* part = reinterpret_cast<float*>(sm);
  float* wm = part + WARPS * R * DT;
  float* wl = wm + WARPS * R;
  if (kg == 0 && (x8 & ((1 << SH) - 1)) == 0) {
    wm[warp * R + mine] = m;
    wl[warp * R + mine] = l;
  }
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int i = 0; i < CH; i++) {
      float4 v = o[r][i];
#pragma unroll
      for (int w = 8; w <= 16; w <<= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, w);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, w);
        v.z += __shfl_xor_sync(0xffffffffu, v.z, w);
        v.w += __shfl_xor_sync(0xffffffffu, v.w, w);
      }
      if (kg == 0) *reinterpret_cast<float4*>(part + (warp * R + r) * DT + 4 * (x8 + 8 * i)) = v;
    }
  sp_join<float, R, DT, CB>(p, split, b, part, wm, wl, reinterpret_cast<SpMail<R, DT>*>(sm + sf_smem<CH>(R)));
}

// A sequence and head's keys are split over as many CTAs as run at once, but
// no warp goes without a tile. A cluster left over would take as long again as
// the others (one stream, 4096 keys, width 256: 8 heads over 16 CTAs each 23.7
// us, over 8 each 18.1; 7 heads over 16 each 12.6), unless it is one in fifteen
// and SMs hold several CTAs (48 heads and streams of 4096 keys, width 128: over
// 8 CTAs each 18.3 us, 45 clusters at once; over 4 each 23.9).
// Narrow heads leave room for more, but four CTAs per SM are enough (single heads
// of 64, bf16, 4096 keys: 75 streams over 4 CTAs each 18.1 us, over 8 20.2; 300
// over 1 58.3, over 2 66.8; f32 of 32: 148 over 4 29.6, over 8 35.2, but 75 over 4
// 21.0, over 8 15.4).
// 32 streams of 4100 visible keys, 8 heads of 128, bf16: 82.4 us = 6.53 TB/s.
template <auto K>
int sp_launch(size_t smem, const WaParams& p, int rows, int kt, int warps, cudaStream_t s) {
  const int64_t pairs = (int64_t)p.max_q * p.group, rb = (pairs + rows - 1) / rows;
  const int64_t blocks = rb * p.n_kv;
  const int64_t span = std::min<int64_t>(p.max_q, (rows + p.group - 1) / p.group + 1);
  const int64_t keys = std::min<int64_t>(p.kv_rows, (int64_t)p.window + p.n_sink + span);
  ARMAI_CUDA(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(SP_MAX_SPLIT * blocks), (unsigned)p.n_seq);
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int split = 0;
  for (int log2 = 1; 1 << log2 <= SP_MAX_SPLIT; log2++) {
    const int n = 1 << log2;
    const int64_t clusters = blocks * p.n_seq;
    if ((int64_t)n * warps * kt > keys || clusters * n > 4 * (int64_t)sm_count()) break;
    if (n > 8) ARMAI_CUDA(cudaFuncSetAttribute(K, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr[0].val.clusterDim.x = (unsigned)n;
    const int active = wa_clusters<K>(log2, cfg);
    const bool several = active * n > sm_count();
    if (several ? clusters * 15 > (int64_t)active * 16 : clusters > active) break;
    split = log2;
  }
  cfg.gridDim.x = (unsigned)(blocks << split);
  attr[0].val.clusterDim.x = 1u << split;
  ARMAI_CUDA(cudaLaunchKernelEx(&cfg, K, p, split));
  return ARMAI_OK;
}

template <typename T, int DT, int CB>
int sp_width(const WaParams& p, cudaStream_t s) {
  return sp_launch<k_wa_split<T, DT, CB>>(sp_smem<T, DT>() + sizeof(SpMail<SP_ROWS, DT>), p, SP_ROWS, SP_KT, sp_warps(DT),
                                          s);
}
template <typename T, int CB>
int sp_half(const WaParams& p, cudaStream_t s) {
  if (p.head_dim <= 64) return sp_width<T, 64, CB>(p, s);
  if (p.head_dim <= 128) return sp_width<T, 128, CB>(p, s);
  return sp_width<T, 256, CB>(p, s);
}

template <int R, int CH, int CB>
int sp_f32(const WaParams& p, cudaStream_t s) {
  return sp_launch<k_wa_split_f32<R, CH, CB>>(sf_smem<CH>(R) + sizeof(SpMail<R, 32 * CH>), p, R, SF_KT, sp_warps(32 * CH),
                                              s);
}
// Rows per CTA as many as there are, up to eight; four or two at the widths
// where more rows of q and of the output would not fit the registers.
int sf_rows(int head_dim) { return head_dim <= 64 ? 8 : head_dim <= 128 ? 4 : 2; }
template <int CH, int CB>
int sp_f32_rows(const WaParams& p, cudaStream_t s) {
  const int64_t pairs = (int64_t)p.max_q * p.group;
  if (pairs <= 1) return sp_f32<1, CH, CB>(p, s);
  if constexpr (CH <= 4) {
    if (pairs > 2 && (CH > 2 || pairs <= 4)) return sp_f32<4, CH, CB>(p, s);
  }
  if constexpr (CH <= 2) {
    if (pairs > 4) return sp_f32<8, CH, CB>(p, s);
  }
  return sp_f32<2, CH, CB>(p, s);
}
template <int CB>
int sp_launch_by_type(const WaParams& p, int dtype, cudaStream_t s) {
  if (dtype == ARMAI_F16) return sp_half<__half, CB>(p, s);
  if (dtype == ARMAI_BF16) return sp_half<__nv_bfloat16, CB>(p, s);
  switch ((p.head_dim + 31) / 32) {
    case 1: return sp_f32_rows<1, CB>(p, s);
    case 2: return sp_f32_rows<2, CB>(p, s);
    case 3: return sp_f32_rows<3, CB>(p, s);
    case 4: return sp_f32_rows<4, CB>(p, s);
    case 5:
    case 6: return sp_f32_rows<6, CB>(p, s);
    default: return sp_f32_rows<8, CB>(p, s);
  }
}

}  // namespace

// Tensors of whole 16-byte vectors or 4-byte words, and heads that fit the grid.
bool wa_split_fits(const WaParams& p, int dtype) {
  const int rows = dtype == ARMAI_F32 ? sf_rows(p.head_dim) : SP_ROWS;
  const int64_t pairs = (int64_t)p.max_q * p.group;
  return wa_aligned(p, dtype, 4) && p.scale_log2 != 0.f && p.scale_log2 == p.scale_log2 &&
         pairs * p.group < int64_t(1) << 32 && (pairs + rows - 1) / rows * p.n_kv * SP_MAX_SPLIT <= 0x7fffffff;
}

int wa_split_launch(const WaParams& p, int dtype, cudaStream_t s) {
  return wa_aligned(p, dtype, 16) ? sp_launch_by_type<16>(p, dtype, s) : sp_launch_by_type<4>(p, dtype, s);
}

}  // namespace armai
