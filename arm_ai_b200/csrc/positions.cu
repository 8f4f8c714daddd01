// positions.cu — rotary positions (both pair layouts, part of the head,
// scaled frequencies) and the per-head norms of q and k fused with the
// rotation and the append to the key / value cache.
//
//   pair i of a head:  a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t),
//   t = position * inv_freq[i], pairs (2i, 2i+1) or (i, i + rot/2)
//   norm (before the rotation): x * 1/sqrt(mean(x^2) + eps) * gamma
//
// Bound by memory: every value is read once and written once, with a handful
// of operations between. A CTA takes the heads of one token: its first
// threads make the token's cos / sin table in shared memory (one f64
// reduction and one sincospi per pair, instead of one per pair and head)
// while the heads' loads are in flight; each head then is a power-of-two
// group of lanes with one 16-byte vector each, so the norm's sum is a few
// shuffles and the partner of a half-layout pair one more.
#include <algorithm>
#include <cmath>

#include "dev_call.cuh"

namespace armai {
namespace {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_DIM = 256;

struct RotTensor {
  const void* src;
  void* dst;
  const float* gamma;          // null: no norm
  int64_t src_token, src_head, dst_token, dst_head;
  int heads;
};

struct RotParams {
  RotTensor t[3];              // q, k, v (or x alone); heads numbered through
  const int64_t* positions;
  const float* inv_freq;
  const int64_t* kv_rows;      // rows of t[1], t[2] in their destination
  int64_t n_rows;
  int dim, rot, heads;         // heads: of all tensors
  float eps, mscale;
};

// cos and sin of pos * f, times m. The product is exact in f64 (24 + 29
// bits; a position beyond 2^29 rounds it to 2^-53), reduced to half turns
// there, and only the remainder rounded to f32: 2^-24 of at most one half
// turn, 2e-7 absolute, at any position.
__device__ __forceinline__ float2 rot_angle(int64_t pos, float f, float m) {
  double t = (double)pos * (double)f * 0.15915494309189533577;  // turns
  t -= rint(t);
  float s, c;
  sincospif((float)(2.0 * t), &s, &c);
  return make_float2(c * m, s * m);
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// Which tensor and head the h-th head of a token is, and whether it is rotated.
__device__ __forceinline__ int rot_locate(const RotParams& p, int h, int& head) {
  int i = 0;
  head = h;
  if (head >= p.t[0].heads) {
    head -= p.t[0].heads;
    i = 1;
    if (head >= p.t[1].heads) {
      head -= p.t[1].heads;
      i = 2;
    }
  }
  return i;
}

// Destination row of a token in tensor i, or -1.
__device__ __forceinline__ int64_t rot_row(const RotParams& p, int i, int64_t token) {
  if (i == 0 || !p.kv_rows) return i == 0 || token < p.n_rows ? token : -1;
  const int64_t r = p.kv_rows[token];
  return r >= 0 && r < p.n_rows ? r : -1;
}

// Vector form: head_dim a multiple of the 16-byte vector, every head's start
// 16-byte aligned, pairs of the half layout a whole number of vectors apart.
// A group of HL lanes (power of two, at least head_dim / VEC) holds a head;
// a warp has 32 / HL heads at once and U such passes in flight.
template <typename T, typename KV, int U>
__global__ void __launch_bounds__(ROT_THREADS) k_rotate_vec(const RotParams p, int hl, int layout) {
  constexpr int VEC = 16 / (int)sizeof(T);
  __shared__ float2 cs[ROT_MAX_DIM / 2];
  const int64_t token = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_warp = 32 / hl, sub = lane / hl, l = lane % hl, d0 = l * VEC;
  const int per_pass = per_warp * (ROT_THREADS / 32);
  const int h0 = blockIdx.y * per_pass * U + warp * per_warp + sub;
  Vec<T, VEC> raw[U];
  int which[U], head[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int h = h0 + u * per_pass;
    which[u] = -1;
    if (h < p.heads && d0 < p.dim) {
      which[u] = rot_locate(p, h, head[u]);
      const RotTensor& t = p.t[which[u]];
      raw[u] = *reinterpret_cast<const Vec<T, VEC>*>(static_cast<const T*>(t.src) + token * t.src_token +
                                                     head[u] * t.src_head + d0);
    }
  }
  const int half = p.rot >> 1;
  if ((int)threadIdx.x < half) cs[threadIdx.x] = rot_angle(p.positions[token], p.inv_freq[threadIdx.x], p.mscale);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; u++) {
    float x[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) x[e] = which[u] >= 0 ? to_f32(raw[u].v[e]) : 0.f;
    const float* gamma = which[u] >= 0 ? p.t[which[u]].gamma : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; e++) ss += x[e] * x[e];
    for (int o = hl >> 1; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (gamma) {
      const float inv = 1.0f / sqrtf(ss / (float)p.dim + p.eps);
#pragma unroll
      for (int e = 0; e < VEC; e++) x[e] = x[e] * inv * gamma[d0 + e];
    }
    if (layout == ARMAI_ROPE_INTERLEAVED) {
      if (which[u] < 2) {
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          if (d0 + e < p.rot) {
            const float2 c = cs[(d0 + e) >> 1];
            const float a = x[e], b = x[e + 1];
            x[e] = a * c.x - b * c.y;
            x[e + 1] = a * c.y + b * c.x;
          }
        }
      }
    } else {
      // the partner vector: half / VEC lanes up (first half) or down
      const bool low = d0 < half;
      const int other = d0 < p.rot ? lane + (low ? half : -half) / VEC : lane;
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const float y = __shfl_sync(0xffffffffu, x[e], other);
        if (which[u] < 2 && d0 < p.rot) {
          const float2 c = cs[low ? d0 + e : d0 + e - half];
          x[e] = low ? x[e] * c.x - y * c.y : y * c.y + x[e] * c.x;
        }
      }
    }
    if (which[u] < 0) continue;
    const RotTensor& t = p.t[which[u]];
    const int64_t row = rot_row(p, which[u], token);
    if (row < 0) continue;
    const int64_t off = row * t.dst_token + head[u] * t.dst_head + d0;
    if (which[u] == 0) {
      Vec<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; e++) o.v[e] = from_f32<T>(x[e]);
      *reinterpret_cast<Vec<T, VEC>*>(static_cast<T*>(t.dst) + off) = o;
    } else {
      Vec<KV, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; e++) o.v[e] = from_f32<KV>(x[e]);
      *reinterpret_cast<Vec<KV, VEC>*>(static_cast<KV*>(t.dst) + off) = o;
    }
  }
}

// Any head_dim, alignment and pairing: a warp per head, one value per lane
// and 32 columns. Values and partners are all read before the first write,
// so a head may be rotated in place.
template <typename T, typename KV>
__global__ void __launch_bounds__(ROT_THREADS) k_rotate_any(const RotParams p, int layout) {
  __shared__ float2 cs[ROT_MAX_DIM / 2];
  const int64_t token = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = p.rot >> 1;
  if ((int)threadIdx.x < half) cs[threadIdx.x] = rot_angle(p.positions[token], p.inv_freq[threadIdx.x], p.mscale);
  __syncthreads();
  for (int h = blockIdx.y * (ROT_THREADS / 32) + warp; h < p.heads; h += gridDim.y * (ROT_THREADS / 32)) {
    int head;
    const int i = rot_locate(p, h, head);
    const RotTensor& t = p.t[i];
    const T* src = static_cast<const T*>(t.src) + token * t.src_token + head * t.src_head;
    float x[ROT_MAX_DIM / 32], y[ROT_MAX_DIM / 32], ss = 0.f;
#pragma unroll
    for (int j = 0; j < ROT_MAX_DIM / 32; j++) {
      const int d = lane + 32 * j;
      x[j] = y[j] = 0.f;
      if (d >= p.dim) continue;
      x[j] = to_f32(src[d]);
      ss += x[j] * x[j];
      if (i < 2 && d < p.rot)
        y[j] = to_f32(src[layout == ARMAI_ROPE_INTERLEAVED ? (d ^ 1) : d < half ? d + half : d - half]);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = t.gamma ? 1.0f / sqrtf(ss / (float)p.dim + p.eps) : 1.f;
    const int64_t row = rot_row(p, i, token);
    if (row < 0) continue;  // the whole warp
    const int64_t off = row * t.dst_token + head * t.dst_head;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < ROT_MAX_DIM / 32; j++) {
      const int d = lane + 32 * j;
      if (d >= p.dim) continue;
      float v = t.gamma ? x[j] * inv * t.gamma[d] : x[j];
      if (i < 2 && d < p.rot) {
        const bool il = layout == ARMAI_ROPE_INTERLEAVED;
        const int pd = il ? (d ^ 1) : d < half ? d + half : d - half;
        const bool first = il ? !(d & 1) : d < half;
        const float w = t.gamma ? y[j] * inv * t.gamma[pd] : y[j];
        const float2 c = cs[il ? d >> 1 : first ? d : pd];
        v = first ? v * c.x - w * c.y : w * c.y + v * c.x;
      }
      if (i == 0)
        static_cast<T*>(t.dst)[off + d] = from_f32<T>(v);
      else
        static_cast<KV*>(t.dst)[off + d] = from_f32<KV>(v);
    }
  }
}

bool aligned16(const RotTensor& t, int es, int des) {
  if (!t.heads) return true;
  return reinterpret_cast<uintptr_t>(t.src) % 16 == 0 && (t.src_token * es) % 16 == 0 && (t.src_head * es) % 16 == 0 &&
         // a destination vector is 16 bytes of the source type, so 8 where the cache is narrower
         reinterpret_cast<uintptr_t>(t.dst) % (16 * des / es) == 0 && (t.dst_token * des) % (16 * des / es) == 0 &&
         (t.dst_head * des) % (16 * des / es) == 0;
}

template <typename T, typename KV>
int rotate_launch(const RotParams& p, int64_t n_tokens, int layout, cudaStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  bool vec = p.dim % VEC == 0 && p.dim / VEC <= 32 &&
             (layout == ARMAI_ROPE_INTERLEAVED || (p.rot >> 1) % VEC == 0);
  for (int i = 0; i < 3; i++) vec = vec && aligned16(p.t[i], sizeof(T), i ? sizeof(KV) : sizeof(T));
  if (!vec) {
    const dim3 grid((unsigned)n_tokens, (unsigned)std::min<int64_t>((p.heads + 7) / 8, n_tokens < 64 ? 64 : 1));
    k_rotate_any<T, KV><<<grid, ROT_THREADS, 0, s>>>(p, layout);
    ARMAI_CUDA(cudaGetLastError());
    return ARMAI_OK;
  }
  int hl = 1;
  while (hl < p.dim / VEC) hl <<= 1;
  const int per_pass = (32 / hl) * (ROT_THREADS / 32);
  const int passes = (p.heads + per_pass - 1) / per_pass;
  // Few tokens: one pass per CTA, the heads spread over the SMs (latency).
  // Many: four passes per CTA, so that four loads per thread are in flight
  // and the token's angles are made once.
  if (n_tokens * passes <= 8 * (int64_t)sm_count()) {
    k_rotate_vec<T, KV, 1><<<dim3((unsigned)n_tokens, (unsigned)passes), ROT_THREADS, 0, s>>>(p, hl, layout);
  } else {
    k_rotate_vec<T, KV, 4><<<dim3((unsigned)n_tokens, (unsigned)((passes + 3) / 4)), ROT_THREADS, 0, s>>>(p, hl,
                                                                                                       layout);
  }
  ARMAI_CUDA(cudaGetLastError());
  return ARMAI_OK;
}

int rotate_dispatch(const RotParams& p, int64_t n_tokens, int dtype, int kv_dtype, int layout, cudaStream_t s) {
  if (dtype == ARMAI_F16) return rotate_launch<__half, __half>(p, n_tokens, layout, s);
  if (dtype == ARMAI_BF16) return rotate_launch<__nv_bfloat16, __nv_bfloat16>(p, n_tokens, layout, s);
  if (kv_dtype == ARMAI_F16) return rotate_launch<float, __half>(p, n_tokens, layout, s);
  if (kv_dtype == ARMAI_BF16) return rotate_launch<float, __nv_bfloat16>(p, n_tokens, layout, s);
  return rotate_launch<float, float>(p, n_tokens, layout, s);
}

// What both entry points ask of their common arguments.
int rot_checks(const std::string& op, int64_t n_tokens, int64_t heads, int64_t dim, int64_t rot, int dtype, int layout) {
  if (!dtype_ok(dtype)) return fail(ARMAI_E_INVALID, op + ": unknown dtype " + std::to_string(dtype));
  if (layout != ARMAI_ROPE_INTERLEAVED && layout != ARMAI_ROPE_HALF)
    return fail(ARMAI_E_INVALID, op + ": unknown layout " + std::to_string(layout));
  if (n_tokens < 0 || n_tokens > 0x7fffffff)
    return fail(ARMAI_E_INVALID, op + ": n_tokens " + std::to_string(n_tokens) + " is not in 0 .. 2^31 - 1");
  if (heads < 0 || heads > 65535)
    return fail(ARMAI_E_INVALID, op + ": " + std::to_string(heads) + " heads are not in 0 .. 65535");
  if (dim < 1 || dim > ROT_MAX_DIM)
    return fail(ARMAI_E_INVALID, op + ": head_dim " + std::to_string(dim) + " is not in 1 .. 256");
  if (rot < 0 || rot > dim || rot % 2)
    return fail(ARMAI_E_INVALID, op + ": rot_dim " + std::to_string(rot) + " must be even and at most head_dim " +
                                     std::to_string(dim));
  return ARMAI_OK;
}

}  // namespace
}  // namespace armai

using namespace armai;

extern "C" int armai_rope_frequencies(size_t rot_dim, double base, int scaling, double factor, double orig_ctx,
                                      double low, double high, float* inv_freq, size_t inv_freq_len) {
  if (rot_dim % 2) return fail(ARMAI_E_INVALID, "rope_frequencies: rot_dim " + std::to_string(rot_dim) + " must be even");
  if (inv_freq_len != rot_dim / 2)
    return fail(ARMAI_E_INVALID, "rope_frequencies: inv_freq len " + std::to_string(inv_freq_len) +
                                     " != rot_dim/2 = " + std::to_string(rot_dim / 2));
  if (!(base > 0.0) || !std::isfinite(base)) return fail(ARMAI_E_INVALID, "rope_frequencies: base must be positive");
  if (scaling < ARMAI_ROPE_SCALE_NONE || scaling > ARMAI_ROPE_SCALE_TURNS)
    return fail(ARMAI_E_INVALID, "rope_frequencies: unknown scaling " + std::to_string(scaling));
  if (scaling != ARMAI_ROPE_SCALE_NONE && (!(factor > 0.0) || !std::isfinite(factor)))
    return fail(ARMAI_E_INVALID, "rope_frequencies: factor must be positive");
  if (scaling == ARMAI_ROPE_SCALE_BASE && rot_dim == 2)
    return fail(ARMAI_E_INVALID, "rope_frequencies: scaling the base needs rot_dim above 2");
  if (scaling == ARMAI_ROPE_SCALE_TURNS && (!(orig_ctx > 0.0) || !(low < high)))
    return fail(ARMAI_E_INVALID, "rope_frequencies: scaling by turns needs orig_ctx > 0 and low < high");
  if (rot_dim && !inv_freq) return fail(ARMAI_E_INVALID, "rope_frequencies: inv_freq is NULL");
  const double n = (double)rot_dim;
  if (scaling == ARMAI_ROPE_SCALE_BASE) base *= std::pow(factor, n / (n - 2.0));
  for (size_t i = 0; i < rot_dim / 2; i++) {
    double f = std::pow(base, -2.0 * (double)i / n);
    if (scaling == ARMAI_ROPE_SCALE_LINEAR) f /= factor;
    if (scaling == ARMAI_ROPE_SCALE_TURNS) {
      const double turns = orig_ctx * f * 0.15915494309189533577;
      const double g = std::fmin(std::fmax((turns - low) / (high - low), 0.0), 1.0);
      f = (1.0 - g) * f / factor + g * f;
    }
    inv_freq[i] = (float)f;
  }
  return ARMAI_OK;
}

extern "C" int armai_dev_rope(const armai_rope_args* a, void* stream) {
  if (!a) return fail(ARMAI_E_INVALID, "rope: args is NULL");
  ARMAI_TRY(rot_checks("rope", a->n_tokens, a->n_heads, a->head_dim, a->rot_dim, a->dtype, a->layout));
  if (!a->n_tokens || !a->n_heads) return ARMAI_OK;
  if (a->x == a->out && (a->x_token_stride != a->out_token_stride || a->x_head_stride != a->out_head_stride))
    return fail(ARMAI_E_INVALID, "rope: in place, x and out must have the same strides");
  DeviceScope dev("rope");
  ARMAI_TRY(dev.check("x", a->x));
  ARMAI_TRY(dev.check("out", a->out));
  if (a->rot_dim) {
    ARMAI_TRY(dev.check("positions", a->positions));
    ARMAI_TRY(dev.check("inv_freq", a->inv_freq));
  }
  RotParams p{};
  p.t[0] = {a->x, a->out, nullptr, a->x_token_stride, a->x_head_stride, a->out_token_stride, a->out_head_stride,
            (int)a->n_heads};
  p.positions = a->positions;
  p.inv_freq = a->inv_freq;
  p.dim = (int)a->head_dim;
  p.rot = (int)a->rot_dim;
  p.heads = (int)a->n_heads;
  p.mscale = a->mscale;
  return rotate_dispatch(p, a->n_tokens, a->dtype, a->dtype, a->layout, (cudaStream_t)stream);
}

extern "C" int armai_dev_qk_norm_rope(const armai_qk_norm_rope_args* a, void* stream) {
  if (!a) return fail(ARMAI_E_INVALID, "qk_norm_rope: args is NULL");
  if (a->n_q_heads < 0 || a->n_kv_heads < 0 || a->n_q_heads > 65535 || a->n_kv_heads > 65535)
    return fail(ARMAI_E_INVALID, "qk_norm_rope: head counts are not in 0 .. 65535");
  ARMAI_TRY(rot_checks("qk_norm_rope", a->n_tokens, a->n_q_heads + 2 * a->n_kv_heads, a->head_dim, a->rot_dim,
                       a->dtype, a->layout));
  if (!dtype_ok(a->kv_dtype) || (a->kv_dtype != a->dtype && a->dtype != ARMAI_F32))
    return fail(ARMAI_E_INVALID, "qk_norm_rope: kv_dtype " + std::to_string(a->kv_dtype) +
                                     " must be dtype, or f16 / bf16 for f32 inputs");
  if (!a->n_tokens || !(a->n_q_heads + a->n_kv_heads)) return ARMAI_OK;
  if (a->n_q_heads && a->q == a->q_out &&
      (a->token_stride != a->q_out_token_stride || a->head_stride != a->q_out_head_stride))
    return fail(ARMAI_E_INVALID, "qk_norm_rope: in place, q and q_out must have the same strides");
  if (a->n_kv_heads && (a->k == a->k_out || (a->v && a->v == a->v_out)) &&
      (a->token_stride != a->kv_row_stride || a->head_stride != a->kv_head_stride || a->kv_rows ||
       a->kv_dtype != a->dtype))
    return fail(ARMAI_E_INVALID, "qk_norm_rope: in place, k and v must have the strides and type of k_out and v_out "
                                 "and no kv_rows");
  if (a->n_rows < 0) return fail(ARMAI_E_INVALID, "qk_norm_rope: n_rows is negative");
  DeviceScope dev("qk_norm_rope");
  if (a->n_q_heads) {
    ARMAI_TRY(dev.check("q", a->q));
    ARMAI_TRY(dev.check("q_out", a->q_out));
    if (a->q_gamma) ARMAI_TRY(dev.check("q_gamma", a->q_gamma));
  }
  if (a->n_kv_heads) {
    ARMAI_TRY(dev.check("k", a->k));
    ARMAI_TRY(dev.check("k_out", a->k_out));
    if (a->k_gamma) ARMAI_TRY(dev.check("k_gamma", a->k_gamma));
    if (a->kv_rows) ARMAI_TRY(dev.check("kv_rows", a->kv_rows));
    if (a->v) {
      ARMAI_TRY(dev.check("v", a->v));
      ARMAI_TRY(dev.check("v_out", a->v_out));
    }
  }
  if (a->rot_dim) {
    ARMAI_TRY(dev.check("positions", a->positions));
    ARMAI_TRY(dev.check("inv_freq", a->inv_freq));
  }
  RotParams p{};
  p.t[0] = {a->q, a->q_out, a->q_gamma, a->token_stride, a->head_stride, a->q_out_token_stride, a->q_out_head_stride,
            (int)a->n_q_heads};
  p.t[1] = {a->k, a->k_out, a->k_gamma, a->token_stride, a->head_stride, a->kv_row_stride, a->kv_head_stride,
            (int)a->n_kv_heads};
  p.t[2] = {a->v, a->v_out, nullptr, a->token_stride, a->head_stride, a->kv_row_stride, a->kv_head_stride,
            a->v ? (int)a->n_kv_heads : 0};
  p.positions = a->positions;
  p.inv_freq = a->inv_freq;
  p.kv_rows = a->kv_rows;
  p.n_rows = a->n_rows;
  p.dim = (int)a->head_dim;
  p.rot = (int)a->rot_dim;
  p.heads = p.t[0].heads + p.t[1].heads + p.t[2].heads;
  p.eps = a->eps;
  p.mscale = a->mscale;
  return rotate_dispatch(p, a->n_tokens, a->dtype, a->kv_dtype, a->layout, (cudaStream_t)stream);
}
