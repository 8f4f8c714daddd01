// window_attn.cuh — what the window-attention kernels share: the call's
// parameters, a sequence's place in the call, and the cache rows that a run
// of queries can see.
//
// Query at position i sees key position j iff j <= i and (j > i - W or j < S)
// (W: window, S: first positions that stay visible). The keys that queries
// plo .. phi see together are [0, S) and [plo - W + 1, phi], one range where
// the two touch; in a ring cache the second range may wrap once. So at most
// three runs of consecutive cache rows with consecutive positions, and a
// kernel walks their tiles.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "dev_call.cuh"

namespace armai {

struct WaParams {
  const void *q, *k, *v;
  void* out;
  const int32_t *q_start, *kv_len, *slots;
  int64_t q_token, q_head, o_token, o_head;
  int64_t kv_slot, kv_head, kv_row;
  int n_seq, max_q, n_tokens, n_q_heads, group, head_dim, n_slots, kv_rows;
  int window, n_sink, ring;  // ring: rows of the ring, 0 for a linear cache
  int n_kv;                  // key / value heads
  uint32_t group_mul;        // ceil(2^32 / group), see wa_token
  float scale_log2;          // scale * log2(e): the kernels use exp2
  uint32_t* err;             // bounded waits that ran out
};

// Token of (token, query head of the group) pair f, exact for f < 2^32 / group
// (group_mul exceeds 2^32 / group by less than 1): a product instead of a
// division.
__device__ __forceinline__ int wa_token(const WaParams& p, int f) {
  return p.group == 1 ? f : (int)__umulhi((uint32_t)f, p.group_mul);
}

// A sequence's queries: rows q0 .. q0 + n - 1 of q, the i-th at position
// pos0 + i.
struct WaSeq {
  int q0, n, pos0, slot;
};
__device__ __forceinline__ WaSeq wa_seq(const WaParams& p, int s) {
  WaSeq r;
  int len;
  if (p.q_start) {
    r.q0 = min(max(p.q_start[s], 0), p.n_tokens);
    len = min(max(p.q_start[s + 1], r.q0), p.n_tokens) - r.q0;
  } else {
    r.q0 = (int)min((int64_t)s * p.max_q, (int64_t)p.n_tokens);
    len = min(p.max_q, p.n_tokens - r.q0);
  }
  r.n = min(len, p.max_q);
  r.slot = p.slots ? p.slots[s] : s;
  const int kv = r.slot >= 0 && r.slot < p.n_slots ? max(p.kv_len[s], 0) : 0;
  r.pos0 = kv - len;
  return r;
}

struct WaRuns {
  int row[3], pos[3], len[3];
  int n;
  __device__ __forceinline__ void add(int r, int p, int l) {
    if (l <= 0) return;
    // n is 0, 1 or 2 here: written by comparison, so that the arrays stay in registers
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (n == i) {
        row[i] = r;
        pos[i] = p;
        len[i] = l;
      }
    n++;
  }
  // key range [a, b] at or behind the first positions, in a ring of R rows
  __device__ __forceinline__ void add_range(const WaParams& p, int a, int b) {
    if (a > b) return;
    if (!p.ring) {
      add(a, a, min(b, p.kv_rows - 1) - a + 1);
      return;
    }
    const int at = (a - p.n_sink) % p.ring;
    const int len = min(b - a + 1, p.ring), first = min(len, p.ring - at);
    add(p.n_sink + at, a, first);
    add(p.n_sink, a + first, len - first);
  }
};
// The cache rows that queries at positions plo .. phi see (a hull: tiles
// still need the mask).
__device__ __forceinline__ WaRuns wa_runs(const WaParams& p, int plo, int phi) {
  WaRuns r;
  r.n = 0;
#pragma unroll
  for (int i = 0; i < 3; i++) r.row[i] = r.pos[i] = r.len[i] = 0;
  if (phi < 0) return r;
  const int64_t lo64 = (int64_t)plo - p.window + 1;
  const int lo = lo64 > 0 ? (int)lo64 : 0;
  if (lo <= p.n_sink) {  // one range from the first position on; in a ring it has not wrapped
    r.add(0, 0, min(phi, p.kv_rows - 1) + 1);
  } else {
    r.add(0, 0, min(p.n_sink, p.kv_rows));
    r.add_range(p, lo, phi);
  }
  return r;
}

__device__ __forceinline__ bool wa_sees(const WaParams& p, int qpos, int kpos) {
  return kpos <= qpos && (qpos - kpos < p.window || kpos < p.n_sink);
}

// The running maximum is raised (and the output rescaled) only when a score
// exceeds it by more than this many powers of two: the weights stay below 2^8
// times their largest and their sum far inside f32, and most tiles need no pass
// over the output.
constexpr float WA_SLACK = 8.f;
// The weights of 16-bit tensors are exp2(score - maximum + this), rounded to
// the tensors' type for P V; the f32 sum has the same factor, which cancels. f16
// runs out of exponents: from 2^-14 down a weight loses bits. Seven powers of two
// up its largest is 2^15 (with the slack; f16 ends below 2^16), and a weight is
// rounded to half a step, 2^-11 of itself, down to 2^-21 of the row's largest, and
// to 2^-32 of the largest below. (Keys 17 nats below a first token whose value is
// 0: with no factor an output 44 % off, the weights being rounded to 2^-24 or 0.)
// bf16 has f32's exponents.
template <typename T>
__host__ __device__ constexpr float wa_weight_shift() { return std::is_same<T, __half>::value ? 7.f : 0.f; }

// Tile t of KT keys of the runs: its first cache row, first position and keys.
struct WaTile {
  int row, pos, n;
};
template <int KT>
__device__ __forceinline__ WaTile wa_tile(const WaRuns& r, int t) {
  const int c0 = (r.len[0] + KT - 1) / KT, c1 = (r.len[1] + KT - 1) / KT;
  const int s = t < c0 ? 0 : t < c0 + c1 ? 1 : 2;
  const int o = (s == 0 ? t : s == 1 ? t - c0 : t - c0 - c1) * KT;
  WaTile x;
  x.row = (s == 0 ? r.row[0] : s == 1 ? r.row[1] : r.row[2]) + o;
  x.pos = (s == 0 ? r.pos[0] : s == 1 ? r.pos[1] : r.pos[2]) + o;
  x.n = min(KT, (s == 0 ? r.len[0] : s == 1 ? r.len[1] : r.len[2]) - o);
  return x;
}
template <int KT>
__device__ __forceinline__ int wa_tiles(const WaRuns& r) {
  return (r.len[0] + KT - 1) / KT + (r.len[1] + KT - 1) / KT + (r.len[2] + KT - 1) / KT;
}

// Clusters of 2^log2 CTAs of a kernel that the device holds at once (with one CTA
// per SM 33 of 4, 15 of 8 and 7 of 16: what is left of a die's groups of SMs stays
// empty), asked for once per kernel, size and device. 0: it has no such. A
// question that fails is none for this call alone (no division over such
// clusters) and is asked again at the next.
template <auto K>
int wa_clusters(int log2, const cudaLaunchConfig_t& cfg) {
  constexpr int DEVICES = 32;
  static std::atomic<int> known[DEVICES][5];  // and one more: 0 is not known
  int dev = 0, active = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const int k = dev < DEVICES ? known[dev][log2].load(std::memory_order_relaxed) : 0;
  if (k) return k - 1;
  if (cudaOccupancyMaxActiveClusters(&active, K, &cfg) != cudaSuccess) {
    cudaGetLastError();  // not a failure of the call
    return 0;
  }
  if (dev < DEVICES) known[dev][log2].store(active + 1, std::memory_order_relaxed);
  return active;
}

// Every pointer, stride and the head a whole number of so many bytes.
bool wa_aligned(const WaParams& p, int dtype, int bytes);

int wa_simt_launch(const WaParams& p, int dtype, cudaStream_t s);
bool wa_split_fits(const WaParams& p, int dtype);
int wa_split_launch(const WaParams& p, int dtype, cudaStream_t s);
// Of aligned tensors; *fits false (and nothing launched): not this form's types,
// widths, scale or strides.
int wa_tc_launch(const WaParams& p, int dtype, cudaStream_t s, bool* fits);

}  // namespace armai
