// window_attn.cu — attention with a sliding window and first tokens that stay
// visible: the entry point, its checks and the choice of kernel, and the form
// on the CUDA cores.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i)
//   over the visible j, in one pass with a running maximum m and sum
//
// k_wa_simt takes every type, head width up to 256, alignment and stride. A CTA
// has 64 queries of one head (32, where 64 would leave SMs empty) and walks the
// visible keys in tiles of 64; a thread has 4 queries x 4 keys of the scores and
// 4 queries x (width / 16) of the output, so that a vector of q, k or v read
// from shared memory feeds eight to sixteen products, two to an instruction. Up
// to a width of 96 two or three CTAs share an SM.
// 4096 tokens, 32 / 8 heads of 128, f32: 4.1 ms = 33 TFLOP/s of the visible
// pairs; two prompts of 333 to 1000 tokens, window 300, 8 / 2 heads of 80: 77.5
// us, where FMA and shared-memory pipes are half busy each: 2 or 3 CTAs of four
// warps per SM leave them idle between dependent steps, and some SMs have one
// CTA more than others. Eight queries per thread halve the shared-memory reads
// but leave too few warps (no faster). Three tf32 tensor products per f32 product
// (71 us) turn an infinite key into NaN, so they are not used.
#include <algorithm>
#include <string>

#include "window_attn.cuh"

namespace armai {
namespace {

constexpr int WS_K = 64;        // keys per tile; queries: Q, 64 or 32, with 4 Q threads
constexpr int WS_PP = WS_K + 4;  // row of P, padded

template <int DM, int Q>
constexpr size_t ws_smem() {
  return ((size_t)(Q + 2 * WS_K) * (DM + 4) + Q * WS_PP) * 4;
}

// Two f32 products and sums per instruction.
__device__ __forceinline__ void ws_fma2(float2& c, float2 a, float2 b) {
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%0, %1};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "+f"(c.x), "+f"(c.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}

// n rows of head_dim values into shared rows of DM f32 (zeros behind them), f32
// copied asynchronously; `vec`: rows of whole 16-byte vectors.
template <typename T, int DM, int ROWS, int THREADS>
__device__ __forceinline__ void ws_rows(float* dst, const T* src, int64_t stride, int n, int D, bool vec) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (sizeof(T) == 4 && vec) {
    for (int e = threadIdx.x; e < ROWS * (DM / 4); e += THREADS) {
      const int r = e / (DM / 4), d = e % (DM / 4) * 4;
      const bool ok = r < n && d < D;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       (uint32_t)__cvta_generic_to_shared(dst + r * (DM + 4) + d)),
                   "l"(ok ? src + r * stride + d : src), "r"(ok ? 16 : 0)
                   : "memory");
    }
    return;
  }
  if constexpr (sizeof(T) == 4) {  // a value at a time, asynchronously all the same
    for (int r = warp; r < ROWS; r += THREADS / 32)
      for (int d = lane; d < DM; d += 32) {
        const bool ok = r < n && d < D;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                         (uint32_t)__cvta_generic_to_shared(dst + r * (DM + 4) + d)),
                     "l"(ok ? src + r * stride + d : src), "r"(ok ? 4 : 0)
                     : "memory");
      }
  } else {
#pragma unroll 4
    for (int r = warp; r < ROWS; r += THREADS / 32)
#pragma unroll
      for (int d = lane; d < DM; d += 32) dst[r * (DM + 4) + d] = r < n && d < D ? to_f32(src[r * stride + d]) : 0.f;
  }
}

template <typename T, int DM, int Q>
__global__ void __launch_bounds__(4 * Q, DM > 96 ? 1 : Q == 64 ? 2 : 3) k_wa_simt(const WaParams p, int vec) {
  constexpr int DP = DM + 4;
  constexpr int OJ = DM / 32;  // pairs of output columns per thread: 2 tx + 32 j
  extern __shared__ __align__(16) float ws[];
  float* Qs = ws;
  float* Ks = Qs + Q * DP;
  float* Vs = Ks + WS_K * DP;
  float* Ps = Vs + WS_K * DP;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int h = blockIdx.y;
  const WaSeq sq = wa_seq(p, blockIdx.z);
  const int i0 = blockIdx.x * Q;
  if (i0 >= sq.n) return;
  const int rows = min(Q, sq.n - i0);
  const int64_t kv_off = (int64_t)sq.slot * p.kv_slot + (int64_t)(h / p.group) * p.kv_head;
  const T* kb = static_cast<const T*>(p.k) + kv_off;
  const T* vb = static_cast<const T*>(p.v) + kv_off;
  const int D = p.head_dim;
  ws_rows<T, DM, Q, 4 * Q>(Qs, static_cast<const T*>(p.q) + (int64_t)(sq.q0 + i0) * p.q_token + (int64_t)h * p.q_head, p.q_token,
                 rows, D, vec);

  float m[4], l[4];
  float2 o[4][OJ];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < OJ; j++) o[i][j] = make_float2(0.f, 0.f);
  }
  const int qpos0 = sq.pos0 + i0 + ty * 4;  // of this thread's first query
  const int qlo = sq.pos0 + i0, qhi = qlo + rows - 1;
  const WaRuns runs = wa_runs(p, qlo, qhi);
  const int nt = wa_tiles<WS_K>(runs), dq = (D + 3) & ~3;
  // V of a key tile is copied while its scores are worked out, K of the next
  // one during the softmax and P V.
  WaTile x = wa_tile<WS_K>(runs, 0);
  if (nt > 0) ws_rows<T, DM, WS_K, 4 * Q>(Ks, kb + (int64_t)x.row * p.kv_row, p.kv_row, x.n, D, vec);
#pragma unroll 1
  for (int t = 0; t < nt; t++) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // K is here, V of the tile before is done with
    ws_rows<T, DM, WS_K, 4 * Q>(Vs, vb + (int64_t)x.row * p.kv_row, p.kv_row, x.n, D, vec);
    float acc[4][4];
    float2 part[4][4];  // of even and of odd values
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) part[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int d = 0; d < dq; d += 4) {
      float4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) a[i] = *reinterpret_cast<const float4*>(Qs + (ty * 4 + i) * DP + d);
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * j) * DP + d);
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          ws_fma2(part[i][j], make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y));
          ws_fma2(part[i][j], make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w));
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // V is here, K is done with
    const WaTile y = wa_tile<WS_K>(runs, min(t + 1, nt - 1));
    if (t + 1 < nt) ws_rows<T, DM, WS_K, 4 * Q>(Ks, kb + (int64_t)y.row * p.kv_row, p.kv_row, y.n, D, vec);
    const bool full = x.n == WS_K && x.pos + WS_K - 1 <= qlo && (qhi - x.pos < p.window || x.pos + WS_K - 1 < p.n_sink);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float mt = m[i];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int kk = tx + 16 * j;
        acc[i][j] = (part[i][j].x + part[i][j].y) * p.scale_log2;
        if (!full && (kk >= x.n || !wa_sees(p, qpos0 + i, x.pos + kk))) acc[i][j] = -INFINITY;
        mt = fmaxf(mt, acc[i][j]);
      }
#pragma unroll
      for (int w = 8; w >= 1; w >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, w));
      const float base = mt == -INFINITY ? 0.f : mt;  // nothing seen yet: every weight is exp2(-inf) = 0
      const float corr = exp2f(m[i] - base);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float e = exp2f(acc[i][j] - base);
        sum += e;
        Ps[(ty * 4 + i) * WS_PP + tx + 16 * j] = e;
      }
      l[i] = l[i] * corr + sum;  // this thread's keys; its sixteen are added up at the end
      m[i] = mt;
#pragma unroll
      for (int j = 0; j < OJ; j++) {
        o[i][j].x *= corr;
        o[i][j].y *= corr;
      }
    }
    __syncwarp();  // a query's row of P is written and read by one half-warp
#pragma unroll 2
    for (int c = 0; c < x.n; c += 4) {
      float4 a[4];
#pragma unroll
      for (int i = 0; i < 4; i++) a[i] = *reinterpret_cast<const float4*>(Ps + (ty * 4 + i) * WS_PP + c);
#pragma unroll
      for (int cc = 0; cc < 4; cc++)
#pragma unroll
        for (int j = 0; j < OJ; j++) {
          const float2 b = *reinterpret_cast<const float2*>(Vs + (c + cc) * DP + tx * 2 + 32 * j);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float w = cc == 0 ? a[i].x : cc == 1 ? a[i].y : cc == 2 ? a[i].z : a[i].w;
            ws_fma2(o[i][j], make_float2(w, w), b);
          }
        }
    }
    x = y;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // of the queries, where there was no key tile
#pragma unroll
  for (int i = 0; i < 4; i++) {
#pragma unroll
    for (int w = 8; w >= 1; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    const int r = ty * 4 + i;
    if (r >= rows) continue;
    T* ob = static_cast<T*>(p.out) + (int64_t)(sq.q0 + i0 + r) * p.o_token + (int64_t)h * p.o_head;
    const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];  // 0 for an empty row
#pragma unroll
    for (int j = 0; j < OJ; j++) {
      const int d = tx * 2 + 32 * j;
      if (d < D) ob[d] = from_f32<T>(o[i][j].x * inv);
      if (d + 1 < D) ob[d + 1] = from_f32<T>(o[i][j].y * inv);
    }
  }
}

template <typename T, int DM, int Q>
int ws_launch(const WaParams& p, int vec, cudaStream_t s) {
  constexpr size_t smem = ws_smem<DM, Q>();
  ARMAI_CUDA(cudaFuncSetAttribute(k_wa_simt<T, DM, Q>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const dim3 grid((unsigned)((p.max_q + Q - 1) / Q), (unsigned)p.n_q_heads, (unsigned)p.n_seq);
  k_wa_simt<T, DM, Q><<<grid, 4 * Q, smem, s>>>(p, vec);
  ARMAI_CUDA(cudaGetLastError());
  return ARMAI_OK;
}
// 32 queries per CTA where 64 would leave the SMs unevenly filled: up to four CTAs
// of 64 per SM (f32, 2 x 8 heads of 80, no window: 256 CTAs of 64 187 us, their
// halves 146; 640: 738 against 688; 1184: 2020 against 2023; 1808: 3492 against
// 3597; 32 / 8 heads of 64, window 300, 896: 178 against 184). Beyond a width of
// 128 an SM has room for one CTA of either kind: up to two (8 heads of 256: 256
// CTAs 535 against 520, 448: 803 against 974, 888: 1602 against 2011).
template <typename T, int DM>
int ws_rows_per_cta(const WaParams& p, int vec, cudaStream_t s) {
  const int64_t ctas = (int64_t)p.n_seq * p.n_q_heads * ((p.max_q + 63) / 64);
  return ctas > (DM > 128 ? 2 : 4) * (int64_t)sm_count() ? ws_launch<T, DM, 64>(p, vec, s) : ws_launch<T, DM, 32>(p, vec, s);
}
template <typename T>
int ws_dim(const WaParams& p, int vec, cudaStream_t s) {
  if (p.head_dim <= 64) return ws_rows_per_cta<T, 64>(p, vec, s);
  if (p.head_dim <= 96) return ws_rows_per_cta<T, 96>(p, vec, s);
  return p.head_dim <= 128 ? ws_rows_per_cta<T, 128>(p, vec, s) : ws_rows_per_cta<T, 256>(p, vec, s);
}

}  // namespace

bool wa_aligned(const WaParams& p, int dtype, int bytes) {
  const int64_t es = dtype_size(dtype);
  const auto ok = [&](int64_t values) { return values * es % bytes == 0; };
  return (reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
          reinterpret_cast<uintptr_t>(p.out)) % bytes == 0 &&
         ok(p.head_dim) && ok(p.q_token) && ok(p.q_head) && ok(p.o_token) && ok(p.o_head) && ok(p.kv_slot) &&
         ok(p.kv_head) && ok(p.kv_row);
}

namespace {

// Whether the split form is the faster one. It reads the keys once for each
// block of 16 rows (16-bit types) and never waits for full tiles of queries.
// 16-bit: with one block of rows always (32 streams of one token, window 512,
// 8 heads of 128: 15 us against 24 in tiles of 256 rows); with more as long as
// its reads stay below 80 MB (4096 keys x 8 heads of 128: 64 rows 16.1 against
// 15.2 us, 128 rows 24.6 against 15.2, 32 rows 13.6 against 15.4; 8 streams of
// 2048 keys: 32 rows 25.6 against 28.3, 64 rows 41 against 28.5).
// f32: a row costs it what 1.8 rows of a full 64-row tile cost on the CUDA
// cores, whose CTAs fill the SMs one by one: as long as there are fewer than 36
// rows per SM for each round of tiles (8 streams of 2048 keys, 8 heads of 128:
// 64 rows 250 against 308 us, 128 rows 476 against 308).
// Wider heads leave it two rows at once: 10 rows per SM (8 streams of 1024
// keys, 8 heads of 256: 16 rows 122 against 173 us, 64 rows 422 against 174;
// one stream of 4096 keys: 1 row 15.7 against 625, 128 rows 436 against 636).
bool wa_split_better(const WaParams& p, int dtype) {
  const int64_t pairs = (int64_t)p.max_q * p.group, heads = (int64_t)p.n_seq * p.n_kv;
  if (dtype != ARMAI_F32) {
    const int64_t keys = std::min<int64_t>(p.kv_rows, (int64_t)p.window + p.n_sink + p.max_q);
    return pairs <= 16 || heads * ((pairs + 15) / 16) * keys * 4 * p.head_dim <= 80 * 1000 * 1000;
  }
  const int64_t r = p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? 4 : 2, rows = heads * ((pairs + r - 1) / r) * r;
  const int64_t tiles = (int64_t)p.n_seq * p.n_q_heads * ((p.max_q + 63) / 64), sms = sm_count();
  return rows <= (p.head_dim <= 128 ? 36 : 10) * sms * ((tiles + sms - 1) / sms);
}

}  // namespace

int wa_simt_launch(const WaParams& p, int dtype, cudaStream_t s) {
  if (dtype == ARMAI_F32) return ws_dim<float>(p, wa_aligned(p, dtype, 16), s);
  if (dtype == ARMAI_F16) return ws_dim<__half>(p, 0, s);
  return ws_dim<__nv_bfloat16>(p, 0, s);
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
  const int es = dtype_size(a->dtype);
  ARMAI_TRY(dev.check("q", a->q, es));
  ARMAI_TRY(dev.check("k", a->k, es));
  ARMAI_TRY(dev.check("v", a->v, es));
  ARMAI_TRY(dev.check("out", a->out, es));
  ARMAI_TRY(dev.check("kv_len", a->kv_len, 4));
  if (a->q_start) ARMAI_TRY(dev.check("q_start", a->q_start, 4));
  if (a->slots) ARMAI_TRY(dev.check("slots", a->slots, 4));
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
  p.n_kv = (int)a->n_kv_heads;
  p.group_mul = (uint32_t)(((1ull << 32) + p.group - 1) / p.group);
  p.head_dim = (int)a->head_dim;
  p.n_slots = (int)a->n_slots;
  p.kv_rows = (int)a->kv_rows;
  p.window = (int)window;
  p.n_sink = (int)sink;
  p.ring = a->ring ? (int)(a->kv_rows - sink) : 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  const cudaStream_t s = (cudaStream_t)stream;
  const bool split = wa_split_fits(p, a->dtype);
  if (split && wa_split_better(p, a->dtype)) return wa_split_launch(p, a->dtype, s);
  bool fits = false;
  if (wa_aligned(p, a->dtype, 16)) ARMAI_TRY(wa_tc_launch(p, a->dtype, s, &fits));
  if (fits) return ARMAI_OK;
  // 16-bit tensors that the 5th-generation tensor cores cannot take (heads
  // wider than 128, strides of 0 or no 16 bytes, a negative scale): reading the
  // keys for every 16 rows is still faster than products on the CUDA cores (1024
  // tokens, 8 heads of 256, bf16: 72 us against 535; 8192 rows of 4 heads on
  // 4096 keys of 256: 2.7 ms against 10.3)
  if (split && a->dtype != ARMAI_F32) return wa_split_launch(p, a->dtype, s);
  return wa_simt_launch(p, a->dtype, s);
}
