// Rotary positions of queries and keys in one launch (rbln_rotary), forward
// or transposed (the gradient).
//
// Bound by HBM: every element is read once and written once, and three
// operations an element are nothing beside it. What could cost more is the
// angle, so a CTA takes `tpb` tokens, finds each token's R/2 (cos, sin)
// once, in shared memory, one per thread, and applies them to all heads of q
// and k: a thread keeps the pairs of its (token, item) in registers and walks
// the heads with two 16-byte loads and stores each. Forward and gradient of 4
// sequences of 4096 tokens, 32 + 8 heads of 128 in bf16, take 122 us: 5.5 TB/s,
// 84 % of the copy rate. CTAs of 128 threads, six an SM, so that one's angles
// run under others' copies (256 threads, three: 135; 128, seven: 126; three
// heads a step and fewer CTAs: 141).

#include "rotary.cuh"

namespace rbln {
namespace {

constexpr int kRotThreads = 128;

struct RotaryArgs {
  const char* q;
  char* qo;
  const char* k;
  char* ko;
  int64_t qs[3], qos[3], ks[3], kos[3];  // elements: b, h, s
  const void* pos;
  int pos_dtype;
  int64_t pos_b, pos_s;
  const float* inv_freq;
  int64_t tokens;  // B * S
  int S, H, heads;  // heads = H + Hkv
  int D, R, items;  // items per row (vector path)
  int tpb, hp;      // tokens a CTA, heads side by side
  bool interleaved;
  float mscale, sin_sign;
};

template <typename T>
struct Vec;  // conversions of one 16-byte vector
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(uint4 w, float* x) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 store(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <bool BF16>
struct Vec16 {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(uint4 w, float* x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<BF16>(u[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 store(const float* x) {
    return make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]),
                      pack2<BF16>(x[6], x[7]));
  }
};
template <>
struct Vec<__nv_bfloat16> : Vec16<true> {};
template <>
struct Vec<__half> : Vec16<false> {};

__device__ __forceinline__ double position(const RotaryArgs& a, int b, int s) {
  return (double)load_index(a.pos, a.pos_dtype, b * a.pos_b + s * a.pos_s);
}

// grid (ceil(tokens / tpb), head groups), 128 threads: thread = (token,
// item, head lane), item fastest, so that 8 neighbours cover a 256-byte row.
// The first heads' loads are issued before the angles are found, and each
// step's next ones before its own are turned.
template <typename T>
__global__ void __launch_bounds__(kRotThreads, 6) rotary_vec_kernel(const RotaryArgs a) {
  constexpr int V = Vec<T>::N;
  extern __shared__ float2 table[];  // [tpb][R/2]
  const int half = a.R / 2;
  const int64_t tok0 = (int64_t)blockIdx.x * a.tpb;
  const int c = threadIdx.x % a.items;
  const int rest = threadIdx.x / a.items;
  const int t = rest % a.tpb, hl = rest / a.tpb;
  const bool live = hl < a.hp && tok0 + t < a.tokens;
  const int b = live ? (int)((tok0 + t) / a.S) : 0, s = live ? (int)(tok0 + t - (int64_t)b * a.S) : 0;
  const RotaryItem it = rotary_item(c, V, a.R, a.interleaved);
  const int step = a.hp * (int)gridDim.y, first = live ? blockIdx.y * a.hp + hl : a.heads;
  const T* qb = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + s * a.qs[2];
  const T* kb = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + s * a.ks[2];
  T* qo = reinterpret_cast<T*>(a.qo) + b * a.qos[0] + s * a.qos[2];
  T* ko = reinterpret_cast<T*>(a.ko) + b * a.kos[0] + s * a.kos[2];
  constexpr int U = 2;  // heads a step
  struct Heads {
    uint4 w[U][2];
  };
  auto load = [&](int h0, Heads& x) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * step;
      if (h >= a.heads) break;
      const T* src = h < a.H ? qb + h * a.qs[1] : kb + (h - a.H) * a.ks[1];
      x.w[u][0] = *reinterpret_cast<const uint4*>(src + it.e0);
      x.w[u][1] = *reinterpret_cast<const uint4*>(src + it.e1);
    }
  };
  Heads now, next;
  load(first, now);

  for (int i = threadIdx.x; i < a.tpb * half; i += kRotThreads) {
    const int r = i / half, p = i - r * half;
    if (tok0 + r >= a.tokens) break;
    const int rb = (int)((tok0 + r) / a.S), rs = (int)(tok0 + r - (int64_t)rb * a.S);
    float2 cs = rotary_cos_sin(position(a, rb, rs), a.inv_freq[p], a.mscale);
    cs.y *= a.sin_sign;
    table[i] = cs;
  }
  __syncthreads();
  float2 cs[V];
  if (it.turned) {
#pragma unroll
    for (int i = 0; i < V; ++i) cs[i] = table[t * half + c * V + i];
  }
  for (int h0 = first; h0 < a.heads; h0 += U * step) {
    load(h0 + U * step, next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * step;
      if (h >= a.heads) break;
      T* dst = h < a.H ? qo + h * a.qos[1] : ko + (h - a.H) * a.kos[1];
      if (it.turned) {
        float x[2 * V];
        Vec<T>::load(now.w[u][0], x);
        Vec<T>::load(now.w[u][1], x + V);
        rotary_turn<V>(x, cs, a.interleaved);
        now.w[u][0] = Vec<T>::store(x);
        now.w[u][1] = Vec<T>::store(x + V);
      }
      *reinterpret_cast<uint4*>(dst + it.e0) = now.w[u][0];
      *reinterpret_cast<uint4*>(dst + it.e1) = now.w[u][1];
    }
    now = next;
  }
}

// Any head dimension, R, stride and alignment: one thread per (token, pair or
// passed dimension), walking the heads one element pair at a time.
template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_scalar_kernel(const RotaryArgs a) {
  const int half = a.R / 2, slots = half + (a.D - a.R);
  const int64_t i = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  if (i >= a.tokens * slots) return;
  const int64_t tok = i / slots;
  const int p = (int)(i - tok * slots);
  const int b = (int)(tok / a.S), s = (int)(tok - (int64_t)b * a.S);
  const bool turned = p < half;
  const int e0 = !turned ? a.R + p - half : a.interleaved ? 2 * p : p;
  const int e1 = a.interleaved ? 2 * p + 1 : p + half;
  float2 cs = make_float2(1.f, 0.f);
  if (turned) {
    cs = rotary_cos_sin(position(a, b, s), a.inv_freq[p], a.mscale);
    cs.y *= a.sin_sign;
  }
  for (int h = blockIdx.y; h < a.heads; h += gridDim.y) {
    const T* src = h < a.H ? reinterpret_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[1] + s * a.qs[2]
                           : reinterpret_cast<const T*>(a.k) + b * a.ks[0] + (h - a.H) * a.ks[1] + s * a.ks[2];
    T* dst = h < a.H ? reinterpret_cast<T*>(a.qo) + b * a.qos[0] + h * a.qos[1] + s * a.qos[2]
                     : reinterpret_cast<T*>(a.ko) + b * a.kos[0] + (h - a.H) * a.kos[1] + s * a.kos[2];
    if (turned) {
      const float x0 = (float)src[e0], x1 = (float)src[e1];
      dst[e0] = (T)(x0 * cs.x - x1 * cs.y);
      dst[e1] = (T)(x1 * cs.x + x0 * cs.y);
    } else {
      dst[e0] = src[e0];
    }
  }
}

template <typename T>
int launch_rotary(RotaryArgs a, bool vec, cudaStream_t st) {
  constexpr int V = Vec<T>::N;
  if (vec) {
    a.items = a.D / (2 * V);
    // Tokens of a CTA share the latency of its angles, where there are enough
    // to fill the GPU; with fewer, one token a CTA and its heads spread over
    // CTAs, so that every thread has one head. 32 + 8 heads of 128, one, two,
    // four tokens a CTA: 8.2, 10.2, 12.3 us at 148 tokens, 10.2, 10.2, 12.3 at
    // 296, 12.3, 10.2, 12.3 at 592, 18.4, 14.4, 14.3 at 1184, 29, 18, 17 at
    // 2368, 145, 72, 66 at 16384 (eight: 68).
    a.tpb = a.tokens >= 8 * 148 ? 4 : a.tokens >= 2 * 148 ? 2 : 1;
    while (a.tpb > 1 && a.tpb * a.items > kRotThreads) a.tpb /= 2;
    a.hp = kRotThreads / (a.tpb * a.items);
    const int64_t gx = (a.tokens + a.tpb - 1) / a.tpb;
    const int gy = a.tpb == 1 ? (a.heads + a.hp - 1) / a.hp : 1;
    rotary_vec_kernel<T><<<dim3((unsigned)gx, (unsigned)gy), kRotThreads, a.tpb * (a.R / 2) * sizeof(float2), st>>>(a);
  } else {
    const int64_t n = a.tokens * (a.R / 2 + a.D - a.R);
    const int64_t gx = (n + kRotThreads - 1) / kRotThreads;
    if (gx > INT32_MAX) return RBLN_ERR_UNSUPPORTED;
    const int gy = gx >= 148 * 8 ? 1 : a.heads < 64 ? a.heads : 64;
    rotary_scalar_kernel<T><<<dim3((unsigned)gx, (unsigned)gy), kRotThreads, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? RBLN_OK : RBLN_ERR_LAUNCH;
}

}  // namespace
}  // namespace rbln

extern "C" size_t rbln_rotary_params_sizeof(void) { return sizeof(rbln_rotary_params_t); }

extern "C" int rbln_rotary(const rbln_rotary_params_t* p, cudaStream_t stream) {
  using namespace rbln;
  if (!p || p->batch < 0 || p->seq_len < 0 || p->q_heads < 0 || p->k_heads < 0 || p->head_dim <= 0 ||
      p->rotary_dim <= 0 || p->rotary_dim > p->head_dim || p->rotary_dim % 2)
    return RBLN_ERR_INVALID_ARGUMENT;
  if (p->dtype != RBLN_DT_F32 && p->dtype != RBLN_DT_F16 && p->dtype != RBLN_DT_BF16) return RBLN_ERR_UNSUPPORTED;
  if (p->positions_dtype != RBLN_DT_I32 && p->positions_dtype != RBLN_DT_I64) return RBLN_ERR_UNSUPPORTED;
  if (p->head_dim > 1024) return RBLN_ERR_UNSUPPORTED;
  const int64_t tokens = (int64_t)p->batch * p->seq_len;
  const int64_t heads = (int64_t)p->q_heads + p->k_heads;
  if (tokens == 0 || heads == 0) return RBLN_OK;
  if (tokens > INT32_MAX || heads > 65535) return RBLN_ERR_UNSUPPORTED;
  if (!p->positions || !p->inv_freq || (p->q_heads && (!p->q || !p->q_out)) || (p->k_heads && (!p->k || !p->k_out)))
    return RBLN_ERR_INVALID_ARGUMENT;
  RotaryArgs a{};
  a.q = static_cast<const char*>(p->q);
  a.qo = static_cast<char*>(p->q_out);
  a.k = static_cast<const char*>(p->k);
  a.ko = static_cast<char*>(p->k_out);
  const int size = p->dtype == RBLN_DT_F32 ? 4 : 2;
  const int V = 16 / size;
  bool vec = p->head_dim % (2 * V) == 0 && p->rotary_dim % (2 * V) == 0;
  auto check = [&](const void* t, const int64_t* s, int64_t* to) {
    vec = vec && (reinterpret_cast<uintptr_t>(t) & 15u) == 0;
    for (int i = 0; i < 3; ++i) {
      to[i] = s[i];
      vec = vec && s[i] % V == 0;
    }
  };
  if (p->q_heads) check(p->q, p->q_stride, a.qs), check(p->q_out, p->q_out_stride, a.qos);
  if (p->k_heads) check(p->k, p->k_stride, a.ks), check(p->k_out, p->k_out_stride, a.kos);
  a.pos = p->positions;
  a.pos_dtype = p->positions_dtype;
  a.pos_b = p->positions_stride[0];
  a.pos_s = p->positions_stride[1];
  a.inv_freq = p->inv_freq;
  a.tokens = tokens;
  a.S = p->seq_len;
  a.H = p->q_heads;
  a.heads = (int)heads;
  a.D = p->head_dim;
  a.R = p->rotary_dim;
  a.interleaved = p->interleaved != 0;
  a.mscale = p->mscale;
  a.sin_sign = p->inverse ? -1.f : 1.f;
  if (p->dtype == RBLN_DT_F32) return launch_rotary<float>(a, vec, stream);
  if (p->dtype == RBLN_DT_BF16) return launch_rotary<__nv_bfloat16>(a, vec, stream);
  return launch_rotary<__half>(a, vec, stream);
}
