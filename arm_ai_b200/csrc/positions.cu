// positions.cu — rotary positions (both pair layouts, part of the head,
// scaled frequencies) and the per-head norms of q and k fused with the
// rotation and the append to the key / value cache.
//
//   pair i of a head:  a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t),
//   t = position * inv_freq[i], pairs (2i, 2i+1) or (i, i + rot/2)
//   norm (before the rotation): x * 1/sqrt(mean(x^2) + eps) * gamma
//
// Bound by memory: every value is read once and written once, with a handful
// of operations between. A warp has a token at a time: it makes the token's
// cosines and sines once (instead of once per head), and a lane keeps its own,
// and its gains, in registers for all heads. A power-of-two group of lanes holds a
// head; a lane has both members of its pairs (two vectors), so the
// rotation needs no exchange and the norm's sum a few shuffles per head.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dev_call.cuh"

namespace armai {
namespace {

constexpr int ROT_THREADS = 128;
constexpr int ROT_MAX_DIM = 256;
constexpr int ROT_WARPS = ROT_THREADS / 32;
// Items in flight per warp, and CTAs per SM: 20 warps with four items of 1 KB
// each. 16381 tokens of 32 + 8 + 8 heads of 128, bf16: 71.8 us = 5.61 TB/s (with
// addresses made anew for each item 85; six to eight CTAs or stages a tenth
// more; two heads per lane in registers and no ring 132; the cosines and sines
// of several tokens shared by a CTA 262).
constexpr int ROT_STAGES = 4;
constexpr int ROT_CTAS = 5;

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

// Turns per position of frequency f, as a 64-bit fraction of a turn. Times a
// position it wraps modulo one turn by itself (negative positions too). f / 2 pi
// is made as a sum of two f64 (1 / 2 pi as two, the first product's rounding by
// FMA: a product alone is off by 2^-53 of itself, 1e-4 rad at position 2^40), so
// that the fraction is off by less than two of its own steps for f below 2^10.
__device__ __forceinline__ uint64_t rot_turns(float f) {
  const double hi = 0.15915494309189535, lo = -9.839338337591243e-18;
  const double x = f, t = x * hi, rest = fma(x, hi, -t) + x * lo;
  return __double2ull_rz((t - floor(t)) * 18446744073709551616.0) +
         (uint64_t)__double2ll_rd(rest * 18446744073709551616.0);
}
// cos and sin of position * f, times m. The remainder, below half a turn, is
// rounded to f32: 2e-7, and 2^-60 per position of the fraction's steps (2e-7
// more at position 2^38). A frequency that is no finite number has no fraction
// of a turn: NaN.
__device__ __forceinline__ float2 rot_angle(int64_t pos, float f, float m) {
  const int32_t r = (int32_t)(((uint64_t)pos * rot_turns(f)) >> 32);  // signed, in 2^-32 turns
  float s, c;
  sincospif((float)r * 4.656612873077392578125e-10f, &s, &c);  // half turns: 2^-31
  m += f - f;
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

template <int BYTES>
__device__ __forceinline__ void rot_copy(void* dst, const void* src) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}

// Destination row of a token in tensor i, or -1.
__device__ __forceinline__ int64_t rot_row(const RotParams& p, int i, int64_t token) {
  if (i == 0 || !p.kv_rows) return i == 0 || token < p.n_rows ? token : -1;
  const int64_t r = p.kv_rows[token];
  return r >= 0 && r < p.n_rows ? r : -1;
}

// Vector form: vectors of VEC values (16, 8 or 4 bytes, the widest that fits),
// every head's start and the second vectors aligned to them.
// Lane l of a head's HL lanes (power of two) has the VEC pairs from l * VEC on:
//   half layout: the vectors at l * VEC and rot / 2 + l * VEC; the lanes behind
//   rot / 2 one of each half of what is not rotated
//   interleaved: the two vectors at 2 l * VEC
// A warp goes through a stream of items, one item being 32 / HL heads of a
// tensor of one token: all items of the tokens w, w + warps, ... (splits 1), or
// one item (splits: the items of a token). The stream's loads run ROT_STAGES
// items ahead, as asynchronous copies into a ring in which a lane reads back
// only what it copied itself: enough bytes in flight for the memory, whatever
// the registers hold.
template <typename T, typename KV, bool IL, int VEC>
__global__ void __launch_bounds__(ROT_THREADS) k_rotate_vec(const RotParams p, int hl, int64_t n_tokens, int splits,
                                                            float inv_dim) {
  __shared__ float2 table[ROT_WARPS][ROT_MAX_DIM / 2];
  __shared__ Vec<T, VEC> ring_[ROT_WARPS][ROT_STAGES][2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t unit = (int64_t)blockIdx.x * ROT_WARPS + warp;
  int64_t token = unit / splits;
  if (token >= n_tokens) return;
  const int64_t step = (int64_t)gridDim.x * ROT_WARPS;  // tokens between a warp's tokens (splits 1)
  const int half = p.rot >> 1, hpw = 32 / hl, sub = lane / hl, l = lane % hl, p0 = l * VEC;
  const int da = IL ? 2 * p0 : p0 < half ? p0 : half + p0;
  const int db = IL ? da + VEC : p0 < half ? p0 + half : da + (p.dim - p.rot) / 2;
  const bool mine = 2 * p0 < p.dim;

  // splits: the one item, as tensor and first head
  int only = 0, h0 = 0;
  if (splits > 1) {
    h0 = (int)(unit % splits) * hpw;
    for (; only < 2; only++) {
      const int padded = (p.t[only].heads + hpw - 1) / hpw * hpw;
      if (h0 < padded) break;
      h0 -= padded;
    }
  }
  // the loads' place in the stream: token, tensor, this lane's head in the item, its address
  Vec<T, VEC>(*ring)[2][32] = ring_[warp];
  int64_t ahead = token, ahead_step = 0;
  int ahead_i = only, ahead_h = h0 + sub, put = 0;
  const T* ahead_src = nullptr;
  auto enter = [&]() {  // the address, at a tensor's start; skips tensors without heads
    while (ahead < n_tokens) {
      const RotTensor& t = p.t[ahead_i];
      if (ahead_h - sub < t.heads) {
        ahead_src = static_cast<const T*>(t.src) + ahead * t.src_token + ahead_h * t.src_head;
        ahead_step = hpw * t.src_head;
        return;
      }
      ahead_h = sub;
      if (++ahead_i == 3) {
        ahead_i = 0;
        ahead += step;
      }
      if (splits > 1) ahead = n_tokens;
    }
  };
  enter();
  auto load = [&]() {
    if (ahead < n_tokens) {
      const int heads = p.t[ahead_i].heads;
      if (mine && ahead_h < heads) {
        rot_copy<VEC * (int)sizeof(T)>(&ring[put][0][lane], ahead_src + da);
        rot_copy<VEC * (int)sizeof(T)>(&ring[put][1][lane], ahead_src + db);
      }
      ahead_h += hpw;
      ahead_src += ahead_step;
      if (splits > 1)
        ahead = n_tokens;
      else if (ahead_h - sub >= heads)
        enter();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    put = put + 1 == ROT_STAGES ? 0 : put + 1;
  };
#pragma unroll
  for (int i = 0; i < ROT_STAGES; i++) load();

  int get = 0;
  float2* cs = table[warp];
  float c[VEC], s[VEC], ga[VEC], gb[VEC];
  for (; token < n_tokens; token += step) {
    __syncwarp();
    if (half) {
      const int64_t pos = p.positions[token];
      for (int i = lane; i < half; i += 32) cs[i] = rot_angle(pos, p.inv_freq[i], p.mscale);
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      const float2 v = p0 + e < half ? cs[p0 + e] : make_float2(1.f, 0.f);
      c[e] = v.x;
      s[e] = v.y;
    }
    for (int i = only; i < 3; i++) {
      const RotTensor& t = p.t[i];
      const bool norm = t.gamma != nullptr;
      if (norm && mine) {
        if constexpr (VEC >= 4) {
#pragma unroll
          for (int e = 0; e < VEC; e += 4) {
            const float4 x = *reinterpret_cast<const float4*>(t.gamma + (IL ? da + 2 * e : da + e));
            const float4 y = *reinterpret_cast<const float4*>(t.gamma + (IL ? da + 2 * e + 4 : db + e));
            if (IL) {
              ga[e] = x.x, gb[e] = x.y, ga[e + 1] = x.z, gb[e + 1] = x.w;
              ga[e + 2] = y.x, gb[e + 2] = y.y, ga[e + 3] = y.z, gb[e + 3] = y.w;
            } else {
              ga[e] = x.x, ga[e + 1] = x.y, ga[e + 2] = x.z, ga[e + 3] = x.w;
              gb[e] = y.x, gb[e + 1] = y.y, gb[e + 2] = y.z, gb[e + 3] = y.w;
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            ga[e] = t.gamma[IL ? da + 2 * e : da + e];
            gb[e] = t.gamma[IL ? da + 2 * e + 1 : db + e];
          }
        }
      }
      const int64_t row = rot_row(p, i, token);
      const int heads = t.heads;
      int64_t off = row * t.dst_token + (h0 + sub) * t.dst_head;
      const int64_t off_step = hpw * t.dst_head;
#pragma unroll 1
      for (int h = h0 + sub; h - sub < heads; h += hpw, off += off_step) {
        const bool on = mine && h < heads;
        asm volatile("cp.async.wait_group %0;" ::"n"(ROT_STAGES - 1) : "memory");
        const Vec<T, VEC> ra = ring[get][0][lane], rb = ring[get][1][lane];
        get = get + 1 == ROT_STAGES ? 0 : get + 1;
        float a[VEC], b[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          // interleaved: values 2e and 2e + 1 of the 2 VEC
          a[e] = to_f32(!IL ? ra.v[e] : 2 * e < VEC ? ra.v[(2 * e) % VEC] : rb.v[(2 * e) % VEC]);
          b[e] = to_f32(!IL ? rb.v[e] : 2 * e < VEC ? ra.v[(2 * e + 1) % VEC] : rb.v[(2 * e + 1) % VEC]);
        }
        load();  // this lane has read what the slot held
        if (norm) {
          float ss = 0.f;
          if (on) {
#pragma unroll
            for (int e = 0; e < VEC; e++) ss += a[e] * a[e] + b[e] * b[e];
          }
          for (int o = hl >> 1; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float inv = rsqrtf(ss * inv_dim + p.eps);
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            a[e] *= inv * ga[e];
            b[e] *= inv * gb[e];
          }
        }
        if (i < 2 && p0 < half) {
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            // where a lane's pairs end before its vectors, the others have cosine 1 and sine 0; a
            // selection, not a product, keeps infinities of one out of the other
            const float x = a[e], y = b[e];
            const bool in = !IL || p0 + e < half;
            a[e] = in ? x * c[e] - y * s[e] : x;
            b[e] = in ? x * s[e] + y * c[e] : y;
          }
        }
        if (on && row >= 0) {
          auto store = [&](auto* base) {
            using O = std::remove_reference_t<decltype(*base)>;
            Vec<O, VEC> oa, ob;
#pragma unroll
            for (int e = 0; e < VEC; e++) {
              if (IL) {
                Vec<O, VEC>& o = 2 * e < VEC ? oa : ob;
                o.v[(2 * e) % VEC] = from_f32<O>(a[e]);
                o.v[(2 * e + 1) % VEC] = from_f32<O>(b[e]);
              } else {
                oa.v[e] = from_f32<O>(a[e]);
                ob.v[e] = from_f32<O>(b[e]);
              }
            }
            *reinterpret_cast<Vec<O, VEC>*>(base + off + da) = oa;
            *reinterpret_cast<Vec<O, VEC>*>(base + off + db) = ob;
          };
          if (i == 0) store(static_cast<T*>(t.dst)); else store(static_cast<KV*>(t.dst));
        }
        if (splits > 1) break;
      }
      if (splits > 1) break;
    }
    if (splits > 1) break;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
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
  for (int i = threadIdx.x; i < half; i += ROT_THREADS)
    cs[i] = rot_angle(p.positions[token], p.inv_freq[i], p.mscale);
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

// Whether a tensor's heads are whole vectors of `vec` values of es bytes (des
// in the destination).
bool rot_aligned(const RotTensor& t, int vec, int es, int des) {
  if (!t.heads) return true;
  const auto ok = [vec](const void* base, int64_t token, int64_t head, int size) {
    return reinterpret_cast<uintptr_t>(base) % (vec * size) == 0 && token % vec == 0 && head % vec == 0;
  };
  return (vec < 4 || reinterpret_cast<uintptr_t>(t.gamma) % 16 == 0) && ok(t.src, t.src_token, t.src_head, es) &&
         ok(t.dst, t.dst_token, t.dst_head, des);
}

template <typename T, typename KV, int VEC>
int rotate_vectors(const RotParams& p, int64_t n_tokens, int layout, cudaStream_t s) {
  int hl = 1;
  while (hl * 2 * VEC < p.dim) hl <<= 1;
  const int hpw = 32 / hl;
  int64_t items = 0;
  for (int i = 0; i < 3; i++) items += (p.t[i].heads + hpw - 1) / hpw;
  // Few tokens: every item has a warp of its own (latency). Many: the warps
  // that fit the device at once share the tokens. 16 items per SM (40 bf16 heads
  // of 128, ten items a token: 32 tokens 2.9 against 5.8 us, 236 tokens, the limit,
  // 3.9 against 6.0, 400 tokens 6.0 against 5.9, 1200 tokens 12.3 against 7.5; f32:
  // 400 tokens 6.8 against 8.1, 600 tokens 9.2 against 8.7).
  const bool few = n_tokens * items <= 16 * (int64_t)sm_count();
  const int splits = few ? (int)items : 1;
  const int64_t ctas = std::min<int64_t>((n_tokens * splits + ROT_WARPS - 1) / ROT_WARPS,
                                         few ? INT32_MAX : ROT_CTAS * (int64_t)sm_count());
  const float inv = 1.0f / (float)p.dim;
  if (layout == ARMAI_ROPE_INTERLEAVED)
    k_rotate_vec<T, KV, true, VEC><<<(unsigned)ctas, ROT_THREADS, 0, s>>>(p, hl, n_tokens, splits, inv);
  else
    k_rotate_vec<T, KV, false, VEC><<<(unsigned)ctas, ROT_THREADS, 0, s>>>(p, hl, n_tokens, splits, inv);
  ARMAI_CUDA(cudaGetLastError());
  return ARMAI_OK;
}

// The widest vectors that the head, its rotated part and the tensors' alignment
// allow, a value at a time where none does (8191 tokens of 40 bf16 heads of 80,
// half of each rotated by halves, so vectors of 4: 32 us against 143).
template <typename T, typename KV, int VEC = 16 / (int)sizeof(T)>
int rotate_launch(const RotParams& p, int64_t n_tokens, int layout, cudaStream_t s) {
  const int half = p.rot >> 1;
  bool fits = p.dim % (2 * VEC) == 0 && p.dim <= 64 * VEC &&
              (layout == ARMAI_ROPE_INTERLEAVED || (half % VEC == 0 && (p.dim - p.rot) % (2 * VEC) == 0));
  for (int i = 0; i < 3; i++) fits = fits && rot_aligned(p.t[i], VEC, sizeof(T), i ? sizeof(KV) : sizeof(T));
  if (fits) return rotate_vectors<T, KV, VEC>(p, n_tokens, layout, s);
  if constexpr (VEC > 2) {
    return rotate_launch<T, KV, VEC / 2>(p, n_tokens, layout, s);
  } else {
    // a token's heads over several CTAs, up to 16 per SM (40 bf16 heads of 33: 64
    // tokens in ten CTAs each 3.0 us, in one 12.2; 800 tokens 14.6 against 13.9;
    // 2400 tokens 39.4 against 30.7)
    const int64_t y = std::max<int64_t>(16 * (int64_t)sm_count() / n_tokens, 1);
    const dim3 grid((unsigned)n_tokens, (unsigned)std::min<int64_t>((p.heads + ROT_WARPS - 1) / ROT_WARPS, y));
    k_rotate_any<T, KV><<<grid, ROT_THREADS, 0, s>>>(p, layout);
    ARMAI_CUDA(cudaGetLastError());
    return ARMAI_OK;
  }
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
  const int es = dtype_size(a->dtype);
  ARMAI_TRY(dev.check("x", a->x, es));
  ARMAI_TRY(dev.check("out", a->out, es));
  if (a->rot_dim) {
    ARMAI_TRY(dev.check("positions", a->positions, 8));
    ARMAI_TRY(dev.check("inv_freq", a->inv_freq, 4));
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
  const int es = dtype_size(a->dtype), kv = dtype_size(a->kv_dtype);
  if (a->n_q_heads) {
    ARMAI_TRY(dev.check("q", a->q, es));
    ARMAI_TRY(dev.check("q_out", a->q_out, es));
    if (a->q_gamma) ARMAI_TRY(dev.check("q_gamma", a->q_gamma, 4));
  }
  if (a->n_kv_heads) {
    ARMAI_TRY(dev.check("k", a->k, es));
    ARMAI_TRY(dev.check("k_out", a->k_out, kv));
    if (a->k_gamma) ARMAI_TRY(dev.check("k_gamma", a->k_gamma, 4));
    if (a->kv_rows) ARMAI_TRY(dev.check("kv_rows", a->kv_rows, 8));
    if (a->v) {
      ARMAI_TRY(dev.check("v", a->v, es));
      ARMAI_TRY(dev.check("v_out", a->v_out, kv));
    }
  }
  if (a->rot_dim) {
    ARMAI_TRY(dev.check("positions", a->positions, 8));
    ARMAI_TRY(dev.check("inv_freq", a->inv_freq, 4));
  }
  // Of a tensor without heads no pointer has been checked, and none goes
  // further: the kernel reads gains and cache rows before it looks at the heads.
  RotParams p{};
  if (a->n_q_heads)
    p.t[0] = {a->q, a->q_out, a->q_gamma, a->token_stride, a->head_stride, a->q_out_token_stride,
              a->q_out_head_stride, (int)a->n_q_heads};
  if (a->n_kv_heads) {
    p.t[1] = {a->k, a->k_out, a->k_gamma, a->token_stride, a->head_stride, a->kv_row_stride, a->kv_head_stride,
              (int)a->n_kv_heads};
    if (a->v)
      p.t[2] = {a->v, a->v_out, nullptr, a->token_stride, a->head_stride, a->kv_row_stride, a->kv_head_stride,
                (int)a->n_kv_heads};
    p.kv_rows = a->kv_rows;
    p.n_rows = a->n_rows;
  }
  p.positions = a->positions;
  p.inv_freq = a->inv_freq;
  p.dim = (int)a->head_dim;
  p.rot = (int)a->rot_dim;
  p.heads = p.t[0].heads + p.t[1].heads + p.t[2].heads;
  p.eps = a->eps;
  p.mscale = a->mscale;
  return rotate_dispatch(p, a->n_tokens, a->dtype, a->kv_dtype, a->layout, (cudaStream_t)stream);
}
