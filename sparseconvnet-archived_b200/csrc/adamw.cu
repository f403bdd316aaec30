// AdamW over a list of tensors in one launch, with 32-bit or 8-bit moments; the norm of all gradients.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "scn_types.cuh"

namespace scn {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, BLOCK = SCN_ADAMW_BLOCK;
constexpr int CHUNK = WARPS * BLOCK; // values a CTA takes at a time: one block of 8-bit states a warp
constexpr float TOP_M = 127.f * 127.f, TOP_V = 4228250624.f; // the largest codes' values over the scale: 127^2, 255^4 in 32 bits

// The list as the kernel takes it, by value: nothing has to be copied to the device before the launch, and a captured
// launch keeps it.
struct Tensor {
  float *w;
  const void *g;
  void *m, *v;
  float *ms, *vs;
  void *w16;
  long long n;
  unsigned long long block; // blocks of BLOCK values in front of this tensor in the call's whole list
  float decay, least;
  int chunk;           // this tensor's first chunk in the launch
  short gtype, w16type;
  int wide;            // every array is aligned for eight values at once
};
template <int CAP> struct List {
  static constexpr int capacity = CAP;
  int count, chunks;
  Tensor t[CAP];
};
constexpr int CAP_SMALL = 16, CAP_LARGE = SCN_ADAMW_MAX_TENSORS;
static_assert(sizeof(List<CAP_LARGE>) <= 32000, "a launch takes at most 32764 bytes of parameters");

// The tensor that owns a chunk (tensors without values own none).
template <int CAP> __device__ __forceinline__ int owner(const List<CAP> &l, int chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.t[mid].chunk <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ float load_typed(const void *p, int type, long long i) {
  if (type == SCN_BF16) return to_float(((const __nv_bfloat16 *)p)[i]);
  if (type == SCN_F16) return to_float(((const __half *)p)[i]);
  return ((const float *)p)[i];
}
__device__ __forceinline__ void load8_typed(const void *p, int type, long long i, float (&x)[8]) {
  if (type == SCN_BF16) load8_16((const __nv_bfloat16 *)p + i, x);
  else if (type == SCN_F16) load8_16((const __half *)p + i, x);
  else load8((const float *)p + i, x);
}
__device__ __forceinline__ void store8_typed(void *p, int type, long long i, const float (&x)[8]) {
  if (type == SCN_BF16) store8_16((__nv_bfloat16 *)p + i, x);
  else store8_16((__half *)p + i, x);
}
__device__ __forceinline__ void store_16(void *p, int type, long long i, float v) {
  if (type == SCN_BF16) ((__nv_bfloat16 *)p)[i] = from_float<__nv_bfloat16>(v);
  else ((__half *)p)[i] = from_float<__half>(v);
}

// ------------------------------------------------------------------ norm
template <int CAP> __global__ void __launch_bounds__(THREADS) k_grad_norm_partial(const __grid_constant__ List<CAP> l, double *partial) {
  wait_for_prior_grids();
  double sum = 0;
  for (int chunk = blockIdx.x; chunk < l.chunks; chunk += gridDim.x) {
    const Tensor &t = l.t[owner(l, chunk)];
    const long long first = (long long)(chunk - t.chunk) * CHUNK;
    if (t.wide && first + CHUNK <= t.n) {
      float g[8];
      load8_typed(t.g, t.gtype, first + threadIdx.x * 8, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += (double)g[k] * g[k];
      continue;
    }
    for (int j = threadIdx.x; j < CHUNK && first + j < t.n; j += THREADS) {
      const double g = load_typed(t.g, t.gtype, first + j);
      sum += g * g;
    }
  }
  dependents_may_launch();
  __shared__ double warpSum[WARPS];
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if ((threadIdx.x & 31) == 0) warpSum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < WARPS; ++w) sum += warpSum[w];
    partial[blockIdx.x] = sum;
  }
}
__global__ void __launch_bounds__(THREADS) k_grad_norm_finish(const double *partial, int n, float *norm) {
  wait_for_prior_grids();
  double sum = 0;
  for (int i = threadIdx.x; i < n; i += THREADS) sum += partial[i];
  __shared__ double warpSum[WARPS];
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if ((threadIdx.x & 31) == 0) warpSum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < WARPS; ++w) sum += warpSum[w];
    *norm = (float)sqrt(sum);
  }
}

// ------------------------------------------------------------------ step
// What scales the gradients, or NaN if the norm is not finite: then nothing is changed.
__device__ __forceinline__ float gradient_scale(const scn_adamw_scalars_t &h, const float *norm) {
  if (!norm) return h.grad_scale;
  const float total = *norm * fabsf(h.grad_scale);
  if (!(total <= 3.402823466e38f)) return __int_as_float(0x7fffffff);
  const float clip = h.max_norm > 0.f && total > h.max_norm ? __fdiv_rn(h.max_norm, total) : 1.f;
  return __fmul_rn(h.grad_scale, clip);
}
// The moments.  Every operation is one rounding (no fused multiply-add), so that the 8-bit codes, which are compared
// against these values, come out the same in any program that computes the formula in 32 bits.
__device__ __forceinline__ void moments(const scn_adamw_scalars_t &h, float g, float &m, float &v) {
  m = __fadd_rn(__fmul_rn(m, h.beta1), __fmul_rn(g, h.one_minus_beta1));
  v = __fadd_rn(__fmul_rn(v, h.beta2), __fmul_rn(__fmul_rn(g, g), h.one_minus_beta2));
}
// The parameter's step may use the hardware's approximate root and quotient (an ulp or two of 32 bits): unlike the states it
// is compared with nothing.  max.NaN keeps a NaN.
__device__ __forceinline__ float updated(const scn_adamw_scalars_t &h, float w, float m, float v, float decay, float least) {
  float root, to;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
  const float step = fmaf(decay, w, __fdividef(m * h.bias1, fmaf(root, h.bias2, h.eps)));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(to) : "f"(fmaf(-h.lr, step, w)), "f"(least));
  return to;
}
// A CTA takes one chunk, a thread eight values of it: everything it reads is on its way before the first is used.
template <int CAP>
__global__ void __launch_bounds__(THREADS) k_adamw_32(const __grid_constant__ List<CAP> l, scn_adamw_scalars_t h, const scn_adamw_scalars_t *dh, const float *norm) {
  const Tensor &t = l.t[owner(l, blockIdx.x)];
  const long long first = (long long)((int)blockIdx.x - t.chunk) * CHUNK;
  float *ms = (float *)t.m, *vs = (float *)t.v;
  wait_for_prior_grids();
  if (dh) h = *dh;
  const float gs = gradient_scale(h, norm);
  if (gs != gs) return;
  if (t.wide && first + CHUNK <= t.n) {
    const long long i = first + threadIdx.x * 8;
    float w[8], g[8], m[8], v[8];
    load8_typed(t.g, t.gtype, i, g);
    load8(ms + i, m);
    load8(vs + i, v);
    load8(t.w + i, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      moments(h, __fmul_rn(g[k], gs), m[k], v[k]);
      w[k] = updated(h, w[k], m[k], v[k], t.decay, t.least);
    }
    store8(ms + i, m);
    store8(vs + i, v);
    store8(t.w + i, w);
    if (t.w16) store8_typed(t.w16, t.w16type, i, w);
    return;
  }
  for (int j = threadIdx.x; j < CHUNK && first + j < t.n; j += THREADS) {
    const long long i = first + j;
    float m = ms[i], v = vs[i];
    moments(h, __fmul_rn(load_typed(t.g, t.gtype, i), gs), m, v);
    const float w = updated(h, t.w[i], m, v, t.decay, t.least);
    ms[i] = m; vs[i] = v; t.w[i] = w;
    if (t.w16) store_16(t.w16, t.w16type, i, w);
  }
}

// 8-bit states.  A first moment is q |q| s with q in -127..127, a second one q^4 s with q in 0..255, s = 2^e the smallest
// power of two (e >= -126) that the block's largest value needs.  Squares and fourth powers put the codes where small
// values lie: the smallest is 1.6e4 (4.2e9) times below the largest, m / sqrt(v) of a value that just rounds to the smallest
// code stays bounded by the block's own.
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int scale_exponent(float most, float top, int bits) {
  int e = ((__float_as_int(most) >> 23) & 255) - 127 - bits;
  e = max(e, -126);
  return most > top * power_of_two(e) ? e + 1 : e;
}
__device__ __forceinline__ float square(float q) { return __fmul_rn(q, q); }
__device__ __forceinline__ float fourth(float q) { return square(square(q)); }
__device__ __forceinline__ float root(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// floor(r) for 0 <= r < 2^22, of an r made a little smaller first, so that an approximate root never comes out too large:
// adding 2^23 with rounding down leaves the whole part.
__device__ __forceinline__ float floor_below(float r) { return __fadd_rd(r * (1.f - 0x1p-20f), 8388608.f) - 8388608.f; }
// Largest whole q with power(q) <= x (the comparison decides; floor_below is right or one too small), then one more where
// the dither says so.
__device__ __forceinline__ float code_m(float x, float u) {
  float q = floor_below(root(x));
  if (square(q + 1.f) <= x) q += 1.f;
  return __fsub_rn(x, square(q)) > __fmul_rn(u, 2.f * q + 1.f) ? q + 1.f : q;
}
__device__ __forceinline__ float code_v(float y, float u) {
  float q = floor_below(root(root(y)));
  if (fourth(q + 1.f) <= y) q += 1.f;
  const float low = fourth(q);
  return __fsub_rn(y, low) > __fmul_rn(u, __fsub_rn(fourth(q + 1.f), low)) ? q + 1.f : q;
}
// A 32-bit mix of a position and the seed: multiplications by odd numbers (the fractional bits of the square roots of 2, 3,
// 5 and 7) between shifts that bring the high bits down.
__device__ __forceinline__ unsigned mix(unsigned at, unsigned key) {
  unsigned h = at * 0x6A09E667u + key;
  h ^= h >> 16;
  h *= 0xBB67AE85u;
  h ^= h >> 15;
  h *= 0x3C6EF373u;
  return h ^ h >> 16;
}
// (b + 1/2) / 2^16 of the 16 bits at bit 7 of x: they become the upper bits of a fraction of 1.
__device__ __forceinline__ float dither(unsigned x) { return __uint_as_float((x & 0x7FFF80u) | 0x3F800000u) - (1.f - 0x1p-17f); }
__device__ __forceinline__ float decode_m(int q, float s) { return __fmul_rn((float)(q * abs(q)), s); }
__device__ __forceinline__ float decode_v(int q, float s) { return __fmul_rn(fourth((float)q), s); }
// Byte k of a word as a float: the byte in the low bits of 2^23, less 2^23.
template <int K> __device__ __forceinline__ float byte_of(unsigned word) { return __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7650 + K)) - 8388608.f; }
template <int K> __device__ __forceinline__ float signed_byte_of(unsigned word) { // word: with every sign bit turned over
  return __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7650 + K)) - 8388736.f;
}
template <int K> __device__ __forceinline__ void decode4(unsigned mq, unsigned vq, float sm, float sv, float *m, float *v) {
  const float a = signed_byte_of<K>(mq), b = byte_of<K>(vq);
  m[K] = __fmul_rn(__fmul_rn(a, fabsf(a)), sm);
  v[K] = __fmul_rn(fourth(b), sv);
}

// A warp takes one block, a lane eight consecutive values of it.  Values behind the end of the tensor count as zeros.
// The largest |m| and v are found as whole numbers: the bits of floats that are not negative are in the floats' order, and what
// is not finite lies above all of them.
constexpr unsigned NOT_FINITE = 0x7F800000u;
template <int CAP>
__global__ void __launch_bounds__(THREADS) k_adamw_8(const __grid_constant__ List<CAP> l, scn_adamw_scalars_t h, const scn_adamw_scalars_t *dh, const float *norm) {
  const Tensor &t = l.t[owner(l, blockIdx.x)];
  const int lane = threadIdx.x & 31;
  const long long block = (long long)((int)blockIdx.x - t.chunk) * WARPS + (threadIdx.x >> 5), i = block * BLOCK + lane * 8;
  if (block * BLOCK >= t.n) return;
  signed char *mq = (signed char *)t.m;
  unsigned char *vq = (unsigned char *)t.v;
  wait_for_prior_grids();
  if (dh) h = *dh;
  const float gs = gradient_scale(h, norm);
  if (gs != gs) return;
  const bool wide = t.wide && (block + 1) * BLOCK <= t.n;
  float w[8], g[8], m[8], v[8];
  uint2 mw = {0, 0}, vw = {0, 0};
  const float sm = t.ms[block], sv = t.vs[block];
  if (wide) {
    load8_typed(t.g, t.gtype, i, g);
    mw = *(const uint2 *)(mq + i);
    vw = *(const uint2 *)(vq + i);
    load8(t.w + i, w);
  } else {
    unsigned mb[8], vb[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool in = i + k < t.n;
      g[k] = in ? load_typed(t.g, t.gtype, i + k) : 0.f;
      w[k] = in ? t.w[i + k] : 0.f;
      mb[k] = in ? (unsigned char)mq[i + k] : 0u;
      vb[k] = in ? vq[i + k] : 0u;
    }
    mw = make_uint2(mb[0] | mb[1] << 8 | mb[2] << 16 | mb[3] << 24, mb[4] | mb[5] << 8 | mb[6] << 16 | mb[7] << 24);
    vw = make_uint2(vb[0] | vb[1] << 8 | vb[2] << 16 | vb[3] << 24, vb[4] | vb[5] << 8 | vb[6] << 16 | vb[7] << 24);
  }
  mw.x ^= 0x80808080u; mw.y ^= 0x80808080u;
  decode4<0>(mw.x, vw.x, sm, sv, m, v); decode4<1>(mw.x, vw.x, sm, sv, m, v);
  decode4<2>(mw.x, vw.x, sm, sv, m, v); decode4<3>(mw.x, vw.x, sm, sv, m, v);
  decode4<0>(mw.y, vw.y, sm, sv, m + 4, v + 4); decode4<1>(mw.y, vw.y, sm, sv, m + 4, v + 4);
  decode4<2>(mw.y, vw.y, sm, sv, m + 4, v + 4); decode4<3>(mw.y, vw.y, sm, sv, m + 4, v + 4);
  unsigned mostM = 0, mostV = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    moments(h, __fmul_rn(g[k], gs), m[k], v[k]);
    w[k] = updated(h, w[k], m[k], v[k], t.decay, t.least);
    if (wide || i + k < t.n) { // (a NaN scale would reach the values behind the end)
      mostM = max(mostM, __float_as_uint(fabsf(m[k])));
      mostV = max(mostV, __float_as_uint(v[k]));
    }
  }
  mostM = __reduce_max_sync(~0u, mostM);
  mostV = __reduce_max_sync(~0u, mostV);
  const bool lost = max(mostM, mostV) >= NOT_FINITE;
  const float topM = __uint_as_float(mostM), topV = __uint_as_float(mostV);
  const int em = lost ? 0 : scale_exponent(topM, TOP_M, 13), ev = lost ? 0 : scale_exponent(topV, TOP_V, 31);
  if (lane == 0) {
    t.ms[block] = lost ? __uint_as_float(0x7FFFFFFFu) : mostM ? power_of_two(em) : 0.f;
    t.vs[block] = lost ? __uint_as_float(0x7FFFFFFFu) : mostV ? power_of_two(ev) : 0.f;
  }
  const float im = power_of_two(-em), iv = power_of_two(-ev);
  const unsigned long long at0 = (t.block + block) * BLOCK;
  const unsigned at = (unsigned)at0 + lane * 8, key = h.seed * 0xBB67AE85u + (unsigned)(at0 >> 32) * 0xA54FF53Bu;
  unsigned mb[8], vb[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const unsigned r = mix(at + k, key);
    float qm = code_m(__fmul_rn(fabsf(m[k]), im), dither(r << 7)), qv = code_v(__fmul_rn(v[k], iv), dither(r >> 9));
    if (v[k] > 0.f) qv = fmaxf(qv, 1.f);
    qm = m[k] < 0.f ? -qm : qm;
    mb[k] = __float_as_uint(qm + 8388736.f) ^ 0x80u; // the byte in the low bits again
    vb[k] = __float_as_uint(qv + 8388608.f);
  }
  if (lost) {
#pragma unroll
    for (int k = 0; k < 8; ++k) mb[k] = vb[k] = 0;
  }
  if (wide) {
    const auto pack = [](const unsigned *b) { return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410); };
    store8(t.w + i, w);
    if (t.w16) store8_typed(t.w16, t.w16type, i, w);
    *(uint2 *)(mq + i) = make_uint2(pack(mb), pack(mb + 4));
    *(uint2 *)(vq + i) = make_uint2(pack(vb), pack(vb + 4));
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (i + k >= t.n) break;
    t.w[i + k] = w[k];
    if (t.w16) store_16(t.w16, t.w16type, i + k, w[k]);
    mq[i + k] = (signed char)mb[k];
    vq[i + k] = (unsigned char)vb[k];
  }
}
// Four codes a thread where the arrays are aligned for it (`wide`: so many values are), then one by one.
__global__ void __launch_bounds__(THREADS) k_adamw_decode(const unsigned char *codes, const float *scale, long long n, long long wide, int second, float *out) {
  const long long step = (long long)gridDim.x * THREADS, self = blockIdx.x * (long long)THREADS + threadIdx.x;
  for (long long j = self; j < wide / 4; j += step) {
    const unsigned q = ((const unsigned *)codes)[j];
    const float s = scale[j / (BLOCK / 4)];
    float4 o;
    if (second) {
      o = make_float4(__fmul_rn(fourth(byte_of<0>(q)), s), __fmul_rn(fourth(byte_of<1>(q)), s), __fmul_rn(fourth(byte_of<2>(q)), s), __fmul_rn(fourth(byte_of<3>(q)), s));
    } else {
      const unsigned t = q ^ 0x80808080u;
      const float a = signed_byte_of<0>(t), b = signed_byte_of<1>(t), c = signed_byte_of<2>(t), d = signed_byte_of<3>(t);
      o = make_float4(__fmul_rn(a * fabsf(a), s), __fmul_rn(b * fabsf(b), s), __fmul_rn(c * fabsf(c), s), __fmul_rn(d * fabsf(d), s));
    }
    ((float4 *)out)[j] = o;
  }
  for (long long i = wide + self; i < n; i += step)
    out[i] = second ? decode_v(codes[i], scale[i / BLOCK]) : decode_m(((const signed char *)codes)[i], scale[i / BLOCK]);
}

// ------------------------------------------------------------------ host side
const char *wrong_list(const scn_adamw_tensor_t *t, int count, bool step) {
  if (count < 0 || (count && !t)) return "AdamW: bad list";
  for (int i = 0; i < count; ++i) {
    if (t[i].n < 0 || t[i].n > (1ll << 40)) return "AdamW: bad number of values";
    if (!type_known(t[i].g_type)) return "AdamW: unknown gradient type";
    if (t[i].n && !t[i].d_g) return "null pointer";
    if (!step) continue;
    if (t[i].n && (!t[i].d_w || !t[i].d_m || !t[i].d_v)) return "null pointer";
    if (!t[i].d_m_scale != !t[i].d_v_scale) return "AdamW: 8-bit states need both scales";
    if (t[i].d_w16 && t[i].w16_type != SCN_BF16 && t[i].w16_type != SCN_F16) return "AdamW: the 16-bit copy's type must be SCN_BF16 or SCN_F16";
    if (!std::isfinite(t[i].weight_decay)) return "AdamW: the weight decay must be finite";
    if (t[i].w_min != t[i].w_min) return "AdamW: w_min must be a number";
    if (((uintptr_t)t[i].d_w | (uintptr_t)t[i].d_m_scale | (uintptr_t)t[i].d_v_scale) & 3) return "AdamW: misaligned pointer";
    if (!t[i].d_m_scale && (((uintptr_t)t[i].d_m | (uintptr_t)t[i].d_v) & 3)) return "AdamW: misaligned pointer";
    if ((uintptr_t)t[i].d_w16 & 1) return "AdamW: misaligned pointer";
  }
  for (int i = 0; i < count; ++i)
    if ((uintptr_t)t[i].d_g & (type_bytes(t[i].g_type) - 1)) return "AdamW: misaligned pointer";
  return nullptr;
}
bool wide(const scn_adamw_tensor_t &t) {
  const uintptr_t states = (uintptr_t)t.d_m | (uintptr_t)t.d_v;
  return !((uintptr_t)t.d_w & 31) && !((uintptr_t)t.d_g & (8 * type_bytes(t.g_type) - 1)) && !((uintptr_t)t.d_w16 & 15) && !(states & (t.d_m_scale ? 7 : 31));
}
// LAUNCH(list) for the tensors that `take` accepts, CAP at a time; blocks are counted over the whole list.
template <int CAP, class Take, class Launch> int for_lists(const scn_adamw_tensor_t *t, int count, Take take, Launch launch) {
  List<CAP> l;
  l.count = l.chunks = 0;
  unsigned long long block = 0;
  auto flush = [&]() -> int {
    const int rc = l.count ? launch(l) : (int)SCN_OK;
    l.count = l.chunks = 0;
    return rc;
  };
  for (int i = 0; i < count; ++i) {
    const long long blocks = (t[i].n + BLOCK - 1) / BLOCK, chunks = (t[i].n + CHUNK - 1) / CHUNK;
    if (t[i].n > 0 && take(t[i])) {
      if (l.count == CAP || l.chunks + chunks > 0x7fffffffll) {
        const int rc = flush();
        if (rc != SCN_OK) return rc;
      }
      l.t[l.count++] = Tensor{t[i].d_w, t[i].d_g, t[i].d_m, t[i].d_v, t[i].d_m_scale, t[i].d_v_scale, t[i].d_w16, t[i].n, block,
                              t[i].weight_decay, t[i].w_min, l.chunks, (short)t[i].g_type, (short)t[i].w16_type, wide(t[i])};
      l.chunks += (int)chunks;
    }
    block += blocks;
  }
  return flush();
}
template <class Take, class Launch> int for_lists(const scn_adamw_tensor_t *t, int count, Take take, Launch launch) {
  return count <= CAP_SMALL ? for_lists<CAP_SMALL>(t, count, take, launch) : for_lists<CAP_LARGE>(t, count, take, launch);
}
int norm_ctas() { return 4 * sm_count(); }

} // namespace
} // namespace scn

using namespace scn;

extern "C" int scn_adamw_scalars(const scn_adamw_t *h, scn_adamw_scalars_t *out) {
  clear_error();
  if (!h || !out) return fail(SCN_ERR_INVALID, "null pointer");
  if (!(h->beta1 >= 0 && h->beta1 < 1 && h->beta2 >= 0 && h->beta2 < 1)) return fail(SCN_ERR_INVALID, "AdamW: beta1 and beta2 must be in [0, 1)");
  if (!std::isfinite(h->lr) || !std::isfinite(h->grad_scale)) return fail(SCN_ERR_INVALID, "AdamW: lr and grad_scale must be finite");
  if (!(std::isfinite(h->eps) && (float)h->eps > 0.f)) return fail(SCN_ERR_INVALID, "AdamW: eps must be positive in 32 bits");
  if (!(std::isfinite(h->max_norm) && h->max_norm >= 0)) return fail(SCN_ERR_INVALID, "AdamW: max_norm must be finite and not negative");
  if (h->step < 1) return fail(SCN_ERR_INVALID, "AdamW: steps count from 1");
  out->lr = (float)h->lr;
  out->beta1 = (float)h->beta1;
  out->beta2 = (float)h->beta2;
  out->one_minus_beta1 = (float)(1.0 - h->beta1);
  out->one_minus_beta2 = (float)(1.0 - h->beta2);
  out->eps = (float)h->eps;
  out->bias1 = (float)(1.0 / (1.0 - std::pow(h->beta1, (double)h->step)));
  out->bias2 = (float)(1.0 / std::sqrt(1.0 - std::pow(h->beta2, (double)h->step)));
  out->grad_scale = (float)h->grad_scale;
  out->max_norm = (float)h->max_norm;
  out->seed = h->seed;
  out->reserved = 0;
  return SCN_OK;
}

extern "C" size_t scn_grad_norm_workspace_bytes(void) { return sizeof(double) * 4 * 1024; }

extern "C" int scn_grad_norm(const scn_adamw_tensor_t *tensors, int count, float *d_norm, void *d_workspace, size_t workspace_bytes, scn_stream_t stream) {
  clear_error();
  if (const char *why = wrong_list(tensors, count, false)) return fail(SCN_ERR_INVALID, why);
  if (!d_norm || !d_workspace) return fail(SCN_ERR_INVALID, "null pointer");
  if (workspace_bytes < scn_grad_norm_workspace_bytes()) return fail(SCN_ERR_WORKSPACE, "workspace smaller than scn_grad_norm_workspace_bytes()");
  if ((uintptr_t)d_workspace & 7) return fail(SCN_ERR_INVALID, "AdamW: the workspace must be 8-byte aligned");
  cudaStream_t s = (cudaStream_t)stream;
  double *partial = (double *)d_workspace;
  const int most = (int)(scn_grad_norm_workspace_bytes() / sizeof(double));
  int used = 0, launches = (count + (count <= CAP_SMALL ? CAP_SMALL : CAP_LARGE) - 1) / (count <= CAP_SMALL ? CAP_SMALL : CAP_LARGE);
  if (launches > most) return fail(SCN_ERR_UNSUPPORTED, "AdamW: list too long");
  const int each = std::min(norm_ctas(), most / std::max(launches, 1));
  const int rc = for_lists(tensors, count, [](const scn_adamw_tensor_t &) { return true; }, [&](const auto &l) -> int {
    const int grid = std::min(l.chunks, each);
    SCN_CUDA_TRY(launch_dependent(k_grad_norm_partial<std::decay_t<decltype(l)>::capacity>, dim3(grid), dim3(THREADS), 0, s, l, partial + used));
    SCN_LAUNCH_CHECK("k_grad_norm_partial");
    used += grid;
    return SCN_OK;
  });
  if (rc != SCN_OK) return rc;
  SCN_CUDA_TRY(launch_dependent(k_grad_norm_finish, dim3(1), dim3(THREADS), 0, s, partial, used, d_norm));
  SCN_LAUNCH_CHECK("k_grad_norm_finish");
  return SCN_OK;
}

extern "C" int scn_adamw_step(const scn_adamw_tensor_t *tensors, int count, const scn_adamw_t *h, const scn_adamw_scalars_t *d_scalars, const float *d_norm,
                              scn_stream_t stream) {
  clear_error();
  if (const char *why = wrong_list(tensors, count, true)) return fail(SCN_ERR_INVALID, why);
  scn_adamw_scalars_t scalars = {};
  if (!d_scalars) {
    const int rc = scn_adamw_scalars(h, &scalars);
    if (rc != SCN_OK) return rc;
    if (h->max_norm > 0 && !d_norm) return fail(SCN_ERR_INVALID, "AdamW: clipping needs the gradients' norm");
  }
  cudaStream_t s = (cudaStream_t)stream;
  const auto eight = [](const scn_adamw_tensor_t &t) { return t.d_m_scale != nullptr; };
  int rc = for_lists(tensors, count, [&](const scn_adamw_tensor_t &t) { return !eight(t); }, [&](const auto &l) -> int {
    SCN_CUDA_TRY(launch_dependent(k_adamw_32<std::decay_t<decltype(l)>::capacity>, dim3(l.chunks), dim3(THREADS), 0, s, l, scalars, d_scalars, d_norm));
    SCN_LAUNCH_CHECK("k_adamw_32");
    return SCN_OK;
  });
  if (rc != SCN_OK) return rc;
  return for_lists(tensors, count, eight, [&](const auto &l) -> int {
    SCN_CUDA_TRY(launch_dependent(k_adamw_8<std::decay_t<decltype(l)>::capacity>, dim3(l.chunks), dim3(THREADS), 0, s, l, scalars, d_scalars, d_norm));
    SCN_LAUNCH_CHECK("k_adamw_8");
    return SCN_OK;
  });
}

extern "C" int scn_adamw_decode(const void *d_codes, const float *d_scale, long long n, int second, float *d_out, scn_stream_t stream) {
  clear_error();
  if (n < 0) return fail(SCN_ERR_INVALID, "bad size");
  if (n == 0) return SCN_OK;
  if (!d_codes || !d_scale || !d_out) return fail(SCN_ERR_INVALID, "null pointer");
  const long long wide = (((uintptr_t)d_codes & 3) | ((uintptr_t)d_out & 15)) == 0 ? n / 4 * 4 : 0;
  k_adamw_decode<<<grid_for((n + 3) / 4, THREADS, 32), THREADS, 0, (cudaStream_t)stream>>>((const unsigned char *)d_codes, d_scale, n, wide, second, d_out);
  SCN_LAUNCH_CHECK("k_adamw_decode");
  return SCN_OK;
}
