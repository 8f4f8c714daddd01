// window_attn.cu — attention with a sliding window and first tokens that stay
// visible: the entry point, its checks and the choice of kernel, and the form
// on the CUDA cores.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i)
//   over the visible j, in one pass with a running maximum m and sum
//
// k_wa_simt takes every type, head width up to 256, alignment and stride. It
// is bound by f32 arithmetic: a CTA has 64 queries of one head and walks the
// visible keys in tiles of 64; 256 threads, each 4 queries x 4 keys of the
// scores and 4 queries x (width / 16) of the output, so that a float4 of q, k
// or v read from shared memory feeds four to sixteen products.
#include <algorithm>
#include <string>

#include "window_attn.cuh"

namespace armai {
namespace {

constexpr int WS_Q = 64, WS_K = 64, WS_THREADS = 256;
constexpr int WS_PP = WS_K + 4;  // row of P, padded

template <int DM>
constexpr size_t ws_smem() {
  return ((size_t)3 * WS_Q * (DM + 4) + WS_Q * WS_PP) * 4;
}

template <typename T, int DM>
__global__ void __launch_bounds__(WS_THREADS, 1) k_wa_simt(const WaParams p) {
  constexpr int DP = DM + 4;
  constexpr int OJ = DM / 64;  // float4 columns of the output per thread
  extern __shared__ float ws[];
  float* Qs = ws;
  float* Ks = Qs + WS_Q * DP;
  float* Vs = Ks + WS_K * DP;
  float* Ps = Vs + WS_K * DP;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, tx = tid & 15, ty = tid >> 4;
  const int h = blockIdx.y;
  const WaSeq sq = wa_seq(p, blockIdx.z);
  const int i0 = blockIdx.x * WS_Q;
  if (i0 >= sq.n) return;
  const int rows = min(WS_Q, sq.n - i0);
  const int64_t kv_off = (int64_t)sq.slot * p.kv_slot + (int64_t)(h / p.group) * p.kv_head;
  const T* qb = static_cast<const T*>(p.q) + (int64_t)(sq.q0 + i0) * p.q_token + (int64_t)h * p.q_head;
  const int D = p.head_dim;

  for (int r = warp; r < WS_Q; r += WS_THREADS / 32)
    for (int d = lane; d < DM; d += 32)
      Qs[r * DP + d] = r < rows && d < D ? to_f32(qb[(int64_t)r * p.q_token + d]) * p.scale_log2 : 0.f;

  float o[4][OJ * 4], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < OJ * 4; j++) o[i][j] = 0.f;
  }
  const int qpos0 = sq.pos0 + i0 + ty * 4;  // of this thread's first query
  const WaRuns runs = wa_runs(p, sq.pos0 + i0, sq.pos0 + i0 + rows - 1);
#pragma unroll 1
  for (int s = 0; s < runs.n; s++) {
    const int row0 = s == 0 ? runs.row[0] : s == 1 ? runs.row[1] : runs.row[2];
    const int pos0 = s == 0 ? runs.pos[0] : s == 1 ? runs.pos[1] : runs.pos[2];
    const int len = s == 0 ? runs.len[0] : s == 1 ? runs.len[1] : runs.len[2];
#pragma unroll 1
    for (int t0 = 0; t0 < len; t0 += WS_K) {
      const int nk = min(WS_K, len - t0);
      __syncthreads();
      for (int r = warp; r < WS_K; r += WS_THREADS / 32) {
        const int64_t off = kv_off + (int64_t)(row0 + t0 + r) * p.kv_row;
        const T* kr = static_cast<const T*>(p.k) + off;
        const T* vr = static_cast<const T*>(p.v) + off;
        for (int d = lane; d < DM; d += 32) {
          const bool ok = r < nk && d < D;
          Ks[r * DP + d] = ok ? to_f32(kr[d]) : 0.f;
          Vs[r * DP + d] = ok ? to_f32(vr[d]) : 0.f;
        }
      }
      __syncthreads();
      float acc[4][4];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = 0.f;
#pragma unroll 2
      for (int d = 0; d < DM; d += 4) {
        float4 a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = *reinterpret_cast<const float4*>(Qs + (ty * 4 + i) * DP + d);
#pragma unroll
        for (int j = 0; j < 4; j++) b[j] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * j) * DP + d);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            acc[i][j] += a[i].x * b[j].x + a[i].y * b[j].y + a[i].z * b[j].z + a[i].w * b[j].w;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float mt = m[i];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int kk = tx + 16 * j;
          if (kk >= nk || !wa_sees(p, qpos0 + i, pos0 + t0 + kk)) acc[i][j] = -INFINITY;
          mt = fmaxf(mt, acc[i][j]);
        }
#pragma unroll
        for (int x = 8; x >= 1; x >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
        const float base = mt == -INFINITY ? 0.f : mt;  // nothing seen yet: every p is exp2(-inf) = 0
        const float corr = exp2f(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float e = exp2f(acc[i][j] - base);
          sum += e;
          Ps[(ty * 4 + i) * WS_PP + tx + 16 * j] = e;
        }
#pragma unroll
        for (int x = 8; x >= 1; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        l[i] = l[i] * corr + sum;
        m[i] = mt;
#pragma unroll
        for (int j = 0; j < OJ * 4; j++) o[i][j] *= corr;
      }
      __syncwarp();  // a query's row of P is written and read by one half-warp
#pragma unroll 2
      for (int c = 0; c < WS_K; c += 4) {
        float4 a[4];
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = *reinterpret_cast<const float4*>(Ps + (ty * 4 + i) * WS_PP + c);
#pragma unroll
        for (int cc = 0; cc < 4; cc++)
#pragma unroll
          for (int j = 0; j < OJ; j++) {
            const float4 b = *reinterpret_cast<const float4*>(Vs + (c + cc) * DP + tx * 4 + 64 * j);
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float w = cc == 0 ? a[i].x : cc == 1 ? a[i].y : cc == 2 ? a[i].z : a[i].w;
              o[i][4 * j] += w * b.x;
              o[i][4 * j + 1] += w * b.y;
              o[i][4 * j + 2] += w * b.z;
              o[i][4 * j + 3] += w * b.w;
            }
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = ty * 4 + i;
    if (r >= rows) continue;
    T* ob = static_cast<T*>(p.out) + (int64_t)(sq.q0 + i0 + r) * p.o_token + (int64_t)h * p.o_head;
    const float inv = l[i] > 0.f ? 1.0f / l[i] : l[i];  // 0 for an empty row, NaN kept
#pragma unroll
    for (int j = 0; j < OJ * 4; j++) {
      const int d = tx * 4 + 64 * (j >> 2) + (j & 3);
      if (d < D) ob[d] = from_f32<T>(l[i] == 0.f ? 0.f : o[i][j] * inv);
    }
  }
}

template <typename T, int DM>
int ws_launch(const WaParams& p, cudaStream_t s) {
  ARMAI_CUDA(cudaFuncSetAttribute(k_wa_simt<T, DM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ws_smem<DM>()));
  const dim3 grid((unsigned)((p.max_q + WS_Q - 1) / WS_Q), (unsigned)p.n_q_heads, (unsigned)p.n_seq);
  k_wa_simt<T, DM><<<grid, WS_THREADS, ws_smem<DM>(), s>>>(p);
  ARMAI_CUDA(cudaGetLastError());
  return ARMAI_OK;
}
template <typename T>
int ws_dim(const WaParams& p, cudaStream_t s) {
  return p.head_dim <= 64 ? ws_launch<T, 64>(p, s) : p.head_dim <= 128 ? ws_launch<T, 128>(p, s) : ws_launch<T, 256>(p, s);
}

}  // namespace

bool wa_vectors(const WaParams& p, int dtype) {
  const int64_t es = dtype_size(dtype);
  const auto ok = [&](int64_t stride) { return stride * es % 16 == 0; };
  return (reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
          reinterpret_cast<uintptr_t>(p.out)) % 16 == 0 &&
         ok(p.q_token) && ok(p.q_head) && ok(p.o_token) && ok(p.o_head) && ok(p.kv_slot) && ok(p.kv_head) &&
         ok(p.kv_row);
}

int wa_simt_launch(const WaParams& p, int dtype, cudaStream_t s) {
  if (dtype == ARMAI_F32) return ws_dim<float>(p, s);
  if (dtype == ARMAI_F16) return ws_dim<__half>(p, s);
  return ws_dim<__nv_bfloat16>(p, s);
}

}  // namespace armai

using namespace armai;

extern "C" int armai_dev_window_attention(const armai_window_attention_args* a, void* stream) {
  if (!a) return fail(ARMAI_E_INVALID, "window_attn: args is NULL");
  const auto bad = [](const std::string& m) { return fail(ARMAI_E_INVALID, "window_attn: " + m); };
  if (!dtype_ok(a->dtype)) return bad("unknown dtype " + std::to_string(a->dtype));
  if (a->n_seq < 0 || a->n_seq > 65535) return bad("n_seq " + std::to_string(a->n_seq) + " is not in 0 .. 65535");
  if (a->max_q < 0 || a->max_q > 0x3fffffff || a->n_tokens < 0 || a->n_tokens > 0x3fffffff)
    return bad("max_q and n_tokens must be in 0 .. 2^30 - 1");
  if (a->n_q_heads < 0 || a->n_q_heads > 65535) return bad("n_q_heads is not in 0 .. 65535");
  if (!a->n_seq || !a->max_q || !a->n_tokens || !a->n_q_heads) return ARMAI_OK;
  if (a->n_kv_heads < 1 || a->n_q_heads % a->n_kv_heads)
    return bad("n_q_heads " + std::to_string(a->n_q_heads) + " must be a multiple of n_kv_heads " +
               std::to_string(a->n_kv_heads));
  if (a->head_dim < 1 || a->head_dim > 256) return bad("head_dim " + std::to_string(a->head_dim) + " is not in 1 .. 256");
  if (a->window < 1) return bad("window must be at least 1");
  if (a->n_sink < 0) return bad("n_sink is negative");
  if (a->n_slots < 1 || a->n_slots > 0x3fffffff || a->kv_rows < 1 || a->kv_rows > 0x3fffffff)
    return bad("n_slots and kv_rows must be in 1 .. 2^30 - 1");
  if (a->ring != 0 && a->ring != 1) return bad("ring must be 0 or 1");
  // a window beyond every position is no window
  const int64_t window = std::min<int64_t>(a->window, 0x7fffffff), sink = std::min<int64_t>(a->n_sink, 0x7fffffff);
  if (a->ring && (sink >= a->kv_rows || a->kv_rows - sink < window + a->max_q - 1))
    return bad("a ring needs kv_rows - n_sink >= window + max_q - 1 = " + std::to_string(window + a->max_q - 1) +
               ", got " + std::to_string(a->kv_rows - sink));
  DeviceScope dev("window_attn");
  ARMAI_TRY(dev.check("q", a->q));
  ARMAI_TRY(dev.check("k", a->k));
  ARMAI_TRY(dev.check("v", a->v));
  ARMAI_TRY(dev.check("out", a->out));
  ARMAI_TRY(dev.check("kv_len", a->kv_len));
  if (a->q_start) ARMAI_TRY(dev.check("q_start", a->q_start));
  if (a->slots) ARMAI_TRY(dev.check("slots", a->slots));
  WaParams p{};
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.q_start = a->q_start;
  p.kv_len = a->kv_len;
  p.slots = a->slots;
  p.q_token = a->q_token_stride;
  p.q_head = a->q_head_stride;
  p.o_token = a->out_token_stride;
  p.o_head = a->out_head_stride;
  p.kv_slot = a->kv_slot_stride;
  p.kv_head = a->kv_head_stride;
  p.kv_row = a->kv_row_stride;
  p.n_seq = (int)a->n_seq;
  p.max_q = (int)std::min(a->max_q, a->n_tokens);
  p.n_tokens = (int)a->n_tokens;
  p.n_q_heads = (int)a->n_q_heads;
  p.group = (int)(a->n_q_heads / a->n_kv_heads);
  p.head_dim = (int)a->head_dim;
  p.n_slots = (int)a->n_slots;
  p.kv_rows = (int)a->kv_rows;
  p.window = (int)window;
  p.n_sink = (int)sink;
  p.ring = a->ring ? (int)(a->kv_rows - sink) : 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  const cudaStream_t s = (cudaStream_t)stream;
  // Few query rows per key / value head: bound by the keys, split over the device.
  if (wa_vectors(p, a->dtype)) {
    if (wa_split_fits(p, a->dtype) && (int64_t)p.max_q * p.group <= 64) return wa_split_launch(p, a->dtype, s);
    bool fits = false;
    ARMAI_TRY(wa_tc_launch(p, a->dtype, s, &fits));
    if (fits) return ARMAI_OK;
  }
  return wa_simt_launch(p, a->dtype, s);
}
