// AdamW over a list of tensors in one launch, with 32-bit or 8-bit moments; the norm of all gradients.  With 32-bit moments the
// step is bound by memory (28 bytes a value with 32-bit gradients), with 8-bit ones (16 bytes a value with 16-bit gradients and
// a 16-bit copy) about equally by the instructions that decode and code them; small lists by the launch.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "scn_types.cuh"

namespace scn {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, BLOCK = SCN_ADAMW_BLOCK;
constexpr int TURN = WARPS * BLOCK; // values a CTA takes at a time: eight a thread, one block of 8-bit states a warp
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
  short gtype, w16type;
  int wide;            // every array that the launch touches is aligned for eight values at once
};
template <int CAP> struct List {
  static constexpr int capacity = CAP;
  int count, chunks;
  int turns;      // of a chunk: its CTA takes turns * TURN values
  int first[CAP]; // each tensor's first chunk in the launch (apart from the tensors: the search touches few lines)
  Tensor t[CAP];
};
constexpr int CAP_SMALL = 16, CAP_MEDIUM = 64, CAP_LARGE = SCN_ADAMW_MAX_TENSORS;
static_assert(sizeof(List<CAP_LARGE>) <= 32000, "a launch takes at most 32764 bytes of parameters");

// The tensor that owns a chunk (tensors without values own none): for a short list without a chain of dependent reads.
template <int CAP> __device__ __forceinline__ int owner(const List<CAP> &l, int chunk) {
  if (CAP <= CAP_SMALL) {
    int at = 0;
#pragma unroll
    for (int i = 1; i < CAP; ++i) at += i < l.count && l.first[i] <= chunk;
    return at;
  }
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= chunk) lo = mid; else hi = mid - 1;
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
// Squares are added up in 64 bits: nothing overflows, and the result does not depend on how many CTAs there are by more than
// its last rounding.  A CTA a chunk leaves its sum, one CTA adds them up in a fixed order.  2.8 M values, from memory: 9 + 2 us (launches
// overlap); 30 M values of 32 bits 34 us, 3.5 TB/s, of 16 bits 29 us: half the bytes are hardly faster, so it is the conversions and sums in 64 bits
// that bound it there.
template <int CAP> __global__ void __launch_bounds__(THREADS) k_grad_norm_partial(const __grid_constant__ List<CAP> l, double *partial) {
  wait_for_prior_grids();
  double sum = 0;
  for (int chunk = blockIdx.x; chunk < l.chunks; chunk += gridDim.x) {
    const int at = owner(l, chunk);
    const Tensor &t = l.t[at];
    long long first = (long long)(chunk - l.first[at]) * l.turns * TURN;
    for (int turn = 0; turn < l.turns && first < t.n; ++turn, first += TURN) {
      if (t.wide && first + TURN <= t.n) {
        float g[8];
        load8_typed(t.g, t.gtype, first + threadIdx.x * 8, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += (double)g[k] * g[k];
        continue;
      }
      for (int j = threadIdx.x; j < TURN && first + j < t.n; j += THREADS) {
        const double g = load_typed(t.g, t.gtype, first + j);
        sum += g * g;
      }
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
constexpr int FINISH = 1024;
__global__ void __launch_bounds__(FINISH) k_grad_norm_finish(const double *partial, int n, float *norm) {
  wait_for_prior_grids();
  double sum = 0;
  for (int i = threadIdx.x; i < n; i += FINISH) sum += partial[i];
  __shared__ double warpSum[FINISH / 32];
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if ((threadIdx.x & 31) == 0) warpSum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = warpSum[threadIdx.x];
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (threadIdx.x == 0) *norm = (float)sqrt(sum);
  }
}

// ------------------------------------------------------------------ step
// What scales the gradients, or NaN if the norm is not finite: then nothing is changed.  Clipped it is grad_scale max_norm / (norm
// |grad_scale|), whose factors can leave 32 bits where the result does not: then it is taken as max_norm / norm with grad_scale's sign.
__device__ __forceinline__ float gradient_scale(const scn_adamw_scalars_t &h, const float *norm) {
  if (!norm) return h.grad_scale;
  if (!isfinite(*norm)) return __int_as_float(0x7fffffff);
  const float total = *norm * fabsf(h.grad_scale);
  if (!(h.max_norm > 0.f && total > h.max_norm)) return h.grad_scale;
  const float clip = __fdiv_rn(h.max_norm, total);
  return clip >= 0x1p-126f ? __fmul_rn(h.grad_scale, clip) : copysignf(__fdiv_rn(h.max_norm, *norm), h.grad_scale);
}
// Two values in one instruction each, as far as there is one: the 8-bit step is bound by the instructions it issues.
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); } // of nothing that mul() gave
// A sum that a product goes into, where both roundings count.  (A paired product and the paired sum behind it come out as one fused
// operation, also where PTX names the rounding of each; the tests that count codes show it.  So the sum is written as a fused operation
// itself, a 1 + b with a 1 that only the launch knows: one rounding, and nothing left to fuse.  150 M values with decodes: 713 -> 708 us.  The 32-bit
// step, which waits for memory, adds single values.)
struct Ones {
  float2 plus, minus; // 1 and -1
};
__device__ __forceinline__ float2 plus(const Ones &one, float2 a, float2 b) { return __ffma2_rn(a, one.plus, b); }
struct Singly {};
__device__ __forceinline__ float2 plus(Singly, float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); }
__device__ __forceinline__ float2 minus(const Ones &one, float2 a, float2 b) { return __ffma2_rn(b, one.minus, a); }
__device__ __forceinline__ float root(float x) { // an ulp or so off; 0 below 2^-126
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float any_root(float x) { return x < 0x1p-64f ? root(x * 0x1p64f) * 0x1p-32f : root(x); } // below 2^-126 too
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) { // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The moments.  Every operation is one rounding (no fused multiply-add), so that the 8-bit codes, which are compared
// against these values, come out the same in any program that computes the formula in 32 bits.
template <class Sum> __device__ __forceinline__ void moments(const Sum &one, const scn_adamw_scalars_t &h, float gs, float2 g, float2 &m, float2 &v) {
  g = mul(g, both(gs));
  m = plus(one, mul(m, both(h.beta1)), mul(g, both(h.one_minus_beta1)));
  v = plus(one, mul(v, both(h.beta2)), mul(mul(g, g), both(h.one_minus_beta2)));
}
// The parameter's step may use the hardware's approximate root and reciprocal (an ulp or two of 32 bits): unlike the states it
// is compared with nothing.
// That root is 0 for v below 2^-126.  exact_roots: whether eps is so small beside 2^-63 bias2, the largest root lost, that it would
// show; the values then take any_root.  (Asked once for eight values.  150 M values with 8-bit moments and decodes take 716 us with the
// question, 713 without; 32-bit moments wait for memory and take no longer.)
__device__ __forceinline__ bool exact_roots(const scn_adamw_scalars_t &h) { return !(h.eps >= 0x1p-39f * h.bias2); }
template <bool EXACT> __device__ __forceinline__ float2 updated(const scn_adamw_scalars_t &h, float2 w, float2 m, float2 v, float decay, float least) {
  const float2 r = EXACT ? make_float2(any_root(v.x), any_root(v.y)) : make_float2(root(v.x), root(v.y));
  const float2 den = __ffma2_rn(r, both(h.bias2), both(h.eps));
  const float2 hat = mul(mul(m, both(h.bias1)), make_float2(reciprocal(den.x), reciprocal(den.y)));
  w = __ffma2_rn(both(-h.lr), __ffma2_rn(both(decay), w, hat), w);
  return make_float2(max_nan(w.x, least), max_nan(w.y, least));
}
// A CTA takes one chunk, a thread eight values a turn: everything it reads is on its way before the first is used.  150 M values
// with 16-bit gradients and a 16-bit copy (28 bytes a value): 615 us, 6.8 TB/s, 104 % of a plain copy's rate; one value a thread at
// a time took 1455 us, four turns a CTA 634 us.  2.8 M values, from memory: 16 us (4.9 TB/s): two waves of CTAs, mostly their latency.
template <int CAP>
__global__ void __launch_bounds__(THREADS) k_adamw_32(const __grid_constant__ List<CAP> l, scn_adamw_scalars_t h, const scn_adamw_scalars_t *dh, const float *norm) {
  const int at = owner(l, blockIdx.x);
  const Tensor &t = l.t[at];
  const long long first = (long long)((int)blockIdx.x - l.first[at]) * TURN; // (chunks of one turn)
  float *ms = (float *)t.m, *vs = (float *)t.v;
  wait_for_prior_grids();
  if (dh) h = *dh;
  const float gs = gradient_scale(h, norm);
  if (gs != gs) return;
  const bool exactRoots = exact_roots(h);
  if (t.wide && first + TURN <= t.n) {
    const long long i = first + threadIdx.x * 8;
    float w[8], g[8], m[8], v[8];
    load8_typed(t.g, t.gtype, i, g);
    load8(ms + i, m);
    load8(vs + i, v);
    load8(t.w + i, w);
    const auto update = [&](auto exact) {
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        float2 m2 = make_float2(m[k], m[k + 1]), v2 = make_float2(v[k], v[k + 1]);
        moments(Singly(), h, gs, make_float2(g[k], g[k + 1]), m2, v2);
        const float2 w2 = updated<exact>(h, make_float2(w[k], w[k + 1]), m2, v2, t.decay, t.least);
        m[k] = m2.x; m[k + 1] = m2.y;
        v[k] = v2.x; v[k + 1] = v2.y;
        w[k] = w2.x; w[k + 1] = w2.y;
      }
    };
    if (exactRoots) update(std::true_type()); else update(std::false_type());
    store8(ms + i, m);
    store8(vs + i, v);
    store8(t.w + i, w);
    if (t.w16) store8_typed(t.w16, t.w16type, i, w);
    return;
  }
  for (int j = threadIdx.x; j < TURN && first + j < t.n; j += THREADS) {
    const long long i = first + j;
    float2 m = both(ms[i]), v = both(vs[i]);
    moments(Singly(), h, gs, both(load_typed(t.g, t.gtype, i)), m, v);
    const float2 w1 = both(t.w[i]);
    const float w = (exactRoots ? updated<true>(h, w1, m, v, t.decay, t.least) : updated<false>(h, w1, m, v, t.decay, t.least)).x;
    ms[i] = m.x; vs[i] = v.x; t.w[i] = w;
    if (t.w16) store_16(t.w16, t.w16type, i, w);
  }
}

// 8-bit states.  A first moment is q |q| s with q in -127..127, a second one q^4 s with q in 0..255, s = 2^e the smallest
// power of two (e >= -126) that the block's largest value needs.  Squares and fourth powers put the codes where small
// values lie: the smallest is 1.6e4 (4.2e9) times below the largest, m / sqrt(v) of a value that just rounds to the smallest
// code stays bounded by the block's own.  (Rounded to nearest, a moving average with 1 - beta2 = 1e-3 would never leave its code:
// one step moves it by a fraction of a code.  The dither makes the mean of what is stored the value.)
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int scale_exponent(float most, float top, int bits) {
  int e = ((__float_as_int(most) >> 23) & 255) - 127 - bits;
  e = max(e, -126);
  return most > top * power_of_two(e) ? e + 1 : e;
}
// 1 where x is above 0, else 0, for an x that is 0 or at least 2^-50 away from it.
__device__ __forceinline__ float2 positive(float2 x) { return make_float2(__saturatef(x.x * 0x1p60f), __saturatef(x.y * 0x1p60f)); }
__device__ __forceinline__ float2 nearest(float2 r) { return add(add(r, both(8388608.f)), both(-8388608.f)); } // 0 <= r < 2^22
// The largest whole q with q^2 <= x, then one more where x lies further above q^2 than u times the step to (q + 1)^2.  The
// whole number nearest to an approximate root is q or q + 1; which one, and what the dither decides, comes from differences
// that are 0 or at least 2^-41 (u is no smaller than 2^-17), so a multiplication that saturates tells their signs.
// (x - q^2 and 2 q + 1 are exact.)
__device__ __forceinline__ float2 code_m(const Ones &one, float2 x, float2 u) {
  float2 q = nearest(make_float2(root(x.x), root(x.y)));
  q = minus(one, q, positive(__ffma2_rn(q, q, make_float2(-x.x, -x.y))));
  const float2 over = __ffma2_rn(q, make_float2(-q.x, -q.y), x), limit = mul(u, __ffma2_rn(q, both(2.f), both(1.f)));
  return plus(one, q, positive(minus(one, over, limit)));
}
__device__ __forceinline__ float2 fourth(float2 q) { q = mul(q, q); return mul(q, q); }
__device__ __forceinline__ float2 code_v(const Ones &one, float2 y, float2 u) {
  float2 q = nearest(make_float2(root(root(y.x)), root(root(y.y))));
  q = minus(one, q, positive(minus(one, fourth(q), y)));
  const float2 low = fourth(q), limit = mul(u, minus(one, fourth(add(q, both(1.f))), low));
  return plus(one, q, positive(minus(one, minus(one, y, low), limit)));
}
// A 32-bit mix of a position and the seed: multiplications by odd numbers (the fractional bits of the square roots of 2, 3,
// 5 and 7) between shifts that bring the high bits down.  Its two halves, the lower one with the upper one mixed in once more,
// become (b + 1/2) / 2^16 each: the bits lie in the upper places of a fraction of 1.
__device__ __forceinline__ void dither(unsigned at, unsigned key, float &um, float &uv) {
  unsigned h = at * 0x6A09E667u + key;
  h ^= h >> 16;
  h *= 0xBB67AE85u;
  h ^= h >> 15;
  h *= 0x3C6EF373u;
  const unsigned upper = ((h >> 9) & 0x7FFF80u) | 0x3F800000u;
  uv = __uint_as_float(upper);
  um = __uint_as_float(((h << 7) & 0x7FFF80u) ^ upper);
}
constexpr float DITHER = 0x1p-17f - 1.f; // to be added to both
__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Bytes K and K + 1 of a word as floats: the byte in the low bits of 2^23, less 2^23 (less 2^23 + 128 where every sign bit
// has been turned over).
template <int K> __device__ __forceinline__ float2 bytes_of(unsigned word, float base) {
  return add(make_float2(__uint_as_float(__byte_perm(word, 0x4B000000u, 0x7650 + K)), __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7651 + K))), both(-base));
}
constexpr float UNSIGNED = 8388608.f, SIGNED = 8388736.f;
template <int K> __device__ __forceinline__ float2 decode_m(unsigned word, float s) {
  const float2 q = bytes_of<K>(word, SIGNED);
  return mul(make_float2(__fmul_rn(q.x, fabsf(q.x)), __fmul_rn(q.y, fabsf(q.y))), both(s));
}
template <int K> __device__ __forceinline__ float2 decode_v(unsigned word, float s) { return mul(fourth(bytes_of<K>(word, UNSIGNED)), both(s)); }

// A warp takes one block, a lane eight consecutive values of it.  Values behind the end of the tensor count as zeros.
// The largest |m| and v of the lanes are compared as whole numbers: the bits of floats that are not negative are in the floats' order,
// and what is not finite lies above all of them.
constexpr unsigned NOT_FINITE = 0x7F800000u;
// A block's share of everything, on its way to a warp while it works on the block before: the step issues instructions for
// most of the time that its memory needs, so a warp cannot do without either.  150 M values with 16-bit gradients and a 16-bit
// copy: 460 us, 5.2 TB/s of 16 bytes a value (80 % of a plain copy's rate; 80 % of the issue slots are taken); up to 500 us once the power cap
// has brought the clock from 1965 to some 1850 MHz.  Loads straight into
// registers took 485 us with five CTAs an SM, 510 with four; the next block's loads into registers 515; one value in an
// instruction 690; conversions and correctly rounded roots instead of the tricks below 2130.
struct Incoming {
  float w[BLOCK];
  float g[BLOCK]; // (of the gradient's type)
  unsigned char m[BLOCK], v[BLOCK];
};
template <int BYTES> __device__ __forceinline__ void copy_async(void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], %2;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void ask(const Tensor &t, long long block, int lane, Incoming &in) {
  const long long i = block * BLOCK;
  const int bytes = t.gtype == SCN_F32 ? 4 : 2;
#pragma unroll
  for (int k = 0; k < 2; ++k) copy_async<16>(in.w + (k * 32 + lane) * 4, t.w + i + (k * 32 + lane) * 4);
  copy_async<16>((char *)in.g + lane * 16, (const char *)t.g + i * bytes + lane * 16);
  if (bytes == 4) copy_async<16>((char *)in.g + 512 + lane * 16, (const char *)t.g + i * 4 + 512 + lane * 16);
  if (lane < 16) copy_async<16>(in.m + lane * 16, (const unsigned char *)t.m + i + lane * 16);
  else copy_async<16>(in.v + (lane - 16) * 16, (const unsigned char *)t.v + i + (lane - 16) * 16);
}
template <int CAP>
__global__ void __launch_bounds__(THREADS, 4) k_adamw_8(const __grid_constant__ List<CAP> l, scn_adamw_scalars_t h, const scn_adamw_scalars_t *dh, const float *norm, const Ones one) {
  __shared__ __align__(16) Incoming incoming[2][WARPS];
  const int own = owner(l, blockIdx.x);
  const Tensor &t = l.t[own];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long block = (long long)((int)blockIdx.x - l.first[own]) * l.turns * WARPS + warp;
  signed char *mq = (signed char *)t.m;
  unsigned char *vq = (unsigned char *)t.v;
  wait_for_prior_grids();
  if (dh) h = *dh;
  const float gs = gradient_scale(h, norm);
  if (gs != gs) return;
  const bool exactRoots = exact_roots(h);
  const auto whole = [&](long long b) { return t.wide && (b + 1) * BLOCK <= t.n; };
  if (whole(block)) ask(t, block, lane, incoming[0][warp]);
  asm volatile("cp.async.commit_group;" ::: "memory");
  for (int turn = 0; turn < l.turns && block * BLOCK < t.n; ++turn, block += WARPS) {
    const long long i = block * BLOCK + lane * 8;
    const bool wide = whole(block);
    float w[8], g[8];
    unsigned mw[2], vw[2];
    const float sm = t.ms[block], sv = t.vs[block];
    __syncwarp(); // (every lane has read what this turn's copies overwrite)
    if (turn + 1 < l.turns && whole(block + WARPS)) ask(t, block + WARPS, lane, incoming[(turn + 1) & 1][warp]);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (wide) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      const Incoming &in = incoming[turn & 1][warp];
      const uint2 a = ((const uint2 *)in.m)[lane], b = ((const uint2 *)in.v)[lane];
      mw[0] = a.x; mw[1] = a.y; vw[0] = b.x; vw[1] = b.y;
#pragma unroll
      for (int k = 0; k < 8; k += 4) *(float4 *)(w + k) = *(const float4 *)(in.w + lane * 8 + k);
      if (t.gtype == SCN_F32) {
#pragma unroll
        for (int k = 0; k < 8; k += 4) *(float4 *)(g + k) = *(const float4 *)(in.g + lane * 8 + k);
      } else if (t.gtype == SCN_BF16) load8_16((const __nv_bfloat16 *)in.g + lane * 8, g);
      else load8_16((const __half *)in.g + lane * 8, g);
    } else {
      mw[0] = mw[1] = vw[0] = vw[1] = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = i + k < t.n;
        g[k] = in ? load_typed(t.g, t.gtype, i + k) : 0.f;
        w[k] = in ? t.w[i + k] : 0.f;
        mw[k / 4] |= (in ? (unsigned)(unsigned char)mq[i + k] : 0u) << (k % 4 * 8);
        vw[k / 4] |= (in ? (unsigned)vq[i + k] : 0u) << (k % 4 * 8);
      }
    }
    float2 m[4], v[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const unsigned turned = mw[k] ^ 0x80808080u;
      m[2 * k] = decode_m<0>(turned, sm); m[2 * k + 1] = decode_m<2>(turned, sm);
      v[2 * k] = decode_v<0>(vw[k], sv); v[2 * k + 1] = decode_v<2>(vw[k], sv);
    }
    float topM = 0.f, topV = 0.f;
    const auto update = [&](auto exact) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        moments(one, h, gs, make_float2(g[2 * k], g[2 * k + 1]), m[k], v[k]);
        const float2 to = updated<exact>(h, make_float2(w[2 * k], w[2 * k + 1]), m[k], v[k], t.decay, t.least);
        w[2 * k] = to.x; w[2 * k + 1] = to.y;
      }
    };
    if (exactRoots) update(std::true_type()); else update(std::false_type());
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!wide) { // (a NaN scale would reach the values behind the end)
        if (i + 2 * k >= t.n) m[k].x = v[k].x = 0.f;
        if (i + 2 * k + 1 >= t.n) m[k].y = v[k].y = 0.f;
      }
      topM = max_abs_nan(topM, m[k].x, m[k].y);
      topV = max_abs_nan(topV, v[k].x, v[k].y);
    }
    if (wide) {
      store8(t.w + i, w);
      if (t.w16) store8_typed(t.w16, t.w16type, i, w);
    }
    const unsigned mostM = __reduce_max_sync(~0u, __float_as_uint(topM)), mostV = __reduce_max_sync(~0u, __float_as_uint(topV));
    const bool lost = max(mostM, mostV) >= NOT_FINITE;
    const int em = lost ? 0 : scale_exponent(__uint_as_float(mostM), TOP_M, 13), ev = lost ? 0 : scale_exponent(__uint_as_float(mostV), TOP_V, 31);
    if (lane == 0) {
      t.ms[block] = lost ? __uint_as_float(0x7FFFFFFFu) : mostM ? power_of_two(em) : 0.f;
      t.vs[block] = lost ? __uint_as_float(0x7FFFFFFFu) : mostV ? power_of_two(ev) : 0.f;
    }
    const float im = power_of_two(-em), iv = power_of_two(-ev);
    const unsigned long long at0 = (t.block + block) * BLOCK;
    const unsigned at = (unsigned)at0 + lane * 8, key = h.seed * 0xBB67AE85u + (unsigned)(at0 >> 32) * 0xA54FF53Bu;
    float2 qv[4], product = both(1.f);
    unsigned mb[8], vb[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 um, uv;
      dither(at + 2 * k, key, um.x, uv.x);
      dither(at + 2 * k + 1, key, um.y, uv.y);
      const float2 qm = code_m(one, make_float2(__fmul_rn(fabsf(m[k].x), im), __fmul_rn(fabsf(m[k].y), im)), add(um, both(DITHER)));
      qv[k] = code_v(one, mul(v[k], both(iv)), add(uv, both(DITHER)));
      product = mul(product, qv[k]);
      const float2 bytes = add(make_float2(copysignf(qm.x, m[k].x), copysignf(qm.y, m[k].y)), both(SIGNED)); // the bytes in the low bits again
      mb[2 * k] = __float_as_uint(bytes.x); mb[2 * k + 1] = __float_as_uint(bytes.y);
    }
    if (product.x * product.y == 0.f) { // a second moment's code is 0: only if it is 0 itself
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (v[k].x > 0.f) qv[k].x = fmaxf(qv[k].x, 1.f);
        if (v[k].y > 0.f) qv[k].y = fmaxf(qv[k].y, 1.f);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 bytes = add(qv[k], both(UNSIGNED));
      vb[2 * k] = __float_as_uint(bytes.x); vb[2 * k + 1] = __float_as_uint(bytes.y);
    }
    const auto pack = [](const unsigned *b) { return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410); };
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      mw[k] = lost ? 0u : pack(mb + 4 * k) ^ 0x80808080u;
      vw[k] = lost ? 0u : pack(vb + 4 * k);
    }
    if (wide) {
      *(uint2 *)(mq + i) = make_uint2(mw[0], mw[1]);
      *(uint2 *)(vq + i) = make_uint2(vw[0], vw[1]);
      continue;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (i + k >= t.n) break;
      t.w[i + k] = w[k];
      if (t.w16) store_16(t.w16, t.w16type, i + k, w[k]);
      mq[i + k] = (signed char)(mw[k / 4] >> (k % 4 * 8));
      vq[i + k] = (unsigned char)(vw[k / 4] >> (k % 4 * 8));
    }
  }
}
// What the codes stand for, bound by the 32-bit values written: 150 M codes in 123 us, 6.1 TB/s.
// Eight codes a thread where the arrays are aligned for it (`wide`: so many values are), then one by one.
__global__ void __launch_bounds__(THREADS) k_adamw_decode(const unsigned char *codes, const float *scale, long long n, long long wide, int second, float *out) {
  const long long step = (long long)gridDim.x * THREADS, self = blockIdx.x * (long long)THREADS + threadIdx.x;
  for (long long j = self; j < wide / 8; j += step) {
    const uint2 q = ((const uint2 *)codes)[j];
    const float s = scale[j / (BLOCK / 8)];
    float2 x[4];
    if (second) { x[0] = decode_v<0>(q.x, s); x[1] = decode_v<2>(q.x, s); x[2] = decode_v<0>(q.y, s); x[3] = decode_v<2>(q.y, s); }
    else {
      const unsigned a = q.x ^ 0x80808080u, b = q.y ^ 0x80808080u;
      x[0] = decode_m<0>(a, s); x[1] = decode_m<2>(a, s); x[2] = decode_m<0>(b, s); x[3] = decode_m<2>(b, s);
    }
    const float o[8] = {x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
    store8(out + 8 * j, o);
  }
  for (long long i = wide + self; i < n; i += step)
    out[i] = second ? decode_v<0>(codes[i], scale[i / BLOCK]).x : decode_m<0>(codes[i] ^ 0x80u, scale[i / BLOCK]).x;
}

// ------------------------------------------------------------------ host side
const char *wrong_list(const scn_adamw_tensor_t *t, int count, bool step) {
  if (count < 0 || (count && !t)) return "AdamW: bad list";
  long long all = 0;
  for (int i = 0; i < count; ++i) {
    if (t[i].n < 0 || t[i].n > (1ll << 40)) return "AdamW: bad number of values";
    all += t[i].n;
    // (chunks count in 32 bits: so many fit one launch for each SCN_ADAMW_MAX_TENSORS, which the norm's workspace expects)
    if (all > (1ll << 43)) return "AdamW: bad number of values";
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
bool wide_gradient(const scn_adamw_tensor_t &t) { return !((uintptr_t)t.d_g & (8 * type_bytes(t.g_type) - 1)); }
bool wide_step(const scn_adamw_tensor_t &t) {
  const uintptr_t states = (uintptr_t)t.d_m | (uintptr_t)t.d_v;
  return wide_gradient(t) && !((uintptr_t)t.d_w & 31) && !((uintptr_t)t.d_w16 & 15) && !(states & (t.d_m_scale ? 15 : 31));
}
// launch(list) for the tensors that `take` accepts, CAP at a time; blocks are counted over the whole list.  Where one turn a
// chunk gives more CTAs than an SM holds in a dozen waves, a CTA takes `most`: it finds its tensor once for all of them.  (150 M values: norm and
// 32-bit step 687 us with four turns in the norm, 717 with one; 8-bit step with decodes 770 us with one turn, 720 with four, 715 with eight, 720 with 16.)
template <int CAP, class Take, class Wide, class Launch> int for_lists(const scn_adamw_tensor_t *t, int count, int most, Take take, Wide wide, Launch launch) {
  List<CAP> l;
  long long all = 0;
  for (int i = 0; i < count; ++i) all += take(t[i]) ? (t[i].n + TURN - 1) / TURN : 0;
  l.turns = all > 100ll * 148 ? most : 1;
  const long long size = (long long)l.turns * TURN;
  l.count = l.chunks = 0;
  unsigned long long block = 0;
  for (int i = 0; i < count; ++i) {
    const long long blocks = (t[i].n + BLOCK - 1) / BLOCK, chunks = (t[i].n + size - 1) / size;
    if (t[i].n > 0 && take(t[i])) {
      if (l.count == CAP || l.chunks + chunks > 0x7fffffffll) {
        const int rc = launch(l);
        if (rc != SCN_OK) return rc;
        l.count = l.chunks = 0;
      }
      l.first[l.count] = l.chunks;
      l.t[l.count++] = Tensor{t[i].d_w, t[i].d_g, t[i].d_m, t[i].d_v, t[i].d_m_scale, t[i].d_v_scale, t[i].d_w16, t[i].n, block,
                              t[i].weight_decay, t[i].w_min, (short)t[i].g_type, (short)t[i].w16_type, wide(t[i])};
      l.chunks += (int)chunks;
    }
    block += blocks;
  }
  return l.count ? launch(l) : (int)SCN_OK;
}
// The parameters' bytes are copied at every launch: the smallest list that holds them all.  (A step over 12 tensors: 5.3 us, with the medium list 5.5, with
// the large one 7.1.)
template <class Take, class Wide, class Launch> int for_lists(const scn_adamw_tensor_t *t, int count, int most, Take take, Wide wide, Launch launch) {
  if (count <= CAP_SMALL) return for_lists<CAP_SMALL>(t, count, most, take, wide, launch);
  if (count <= CAP_MEDIUM) return for_lists<CAP_MEDIUM>(t, count, most, take, wide, launch);
  return for_lists<CAP_LARGE>(t, count, most, take, wide, launch);
}

} // namespace
} // namespace scn

using namespace scn;

extern "C" int scn_adamw_scalars(const scn_adamw_t *h, scn_adamw_scalars_t *out) {
  clear_error();
  if (!h || !out) return fail(SCN_ERR_INVALID, "null pointer");
  if (!(h->beta1 >= 0 && h->beta1 < 1 && h->beta2 >= 0 && h->beta2 < 1)) return fail(SCN_ERR_INVALID, "AdamW: beta1 and beta2 must be in [0, 1)");
  if (!std::isfinite((float)h->lr) || !std::isfinite((float)h->grad_scale)) return fail(SCN_ERR_INVALID, "AdamW: lr and grad_scale must be finite");
  if (!(std::isfinite(h->eps) && (float)h->eps >= 1.17549435e-38f)) return fail(SCN_ERR_INVALID, "AdamW: eps must be a positive normal 32-bit number");
  if (!(std::isfinite(h->max_norm) && h->max_norm >= 0)) return fail(SCN_ERR_INVALID, "AdamW: max_norm must be finite and not negative");
  if (h->max_norm > 0 && (float)h->max_norm == 0.f) return fail(SCN_ERR_INVALID, "AdamW: max_norm is 0 in 32 bits, which would not clip at all");
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
  if ((uintptr_t)d_norm & 3) return fail(SCN_ERR_INVALID, "AdamW: misaligned pointer");
  cudaStream_t s = (cudaStream_t)stream;
  double *partial = (double *)d_workspace;
  const int most = (int)(scn_grad_norm_workspace_bytes() / sizeof(double));
  int used = 0, launches = (count + CAP_LARGE - 1) / CAP_LARGE;
  if (launches > most) return fail(SCN_ERR_UNSUPPORTED, "AdamW: list too long");
  const int each = most / std::max(launches, 1); // a CTA a chunk as far as there are places for their sums
  const int rc = for_lists(tensors, count, 4, [](const scn_adamw_tensor_t &) { return true; }, wide_gradient, [&](const auto &l) -> int {
    const int grid = std::min(l.chunks, each);
    SCN_CUDA_TRY(launch_dependent(k_grad_norm_partial<std::decay_t<decltype(l)>::capacity>, dim3(grid), dim3(THREADS), 0, s, l, partial + used));
    SCN_LAUNCH_CHECK("k_grad_norm_partial");
    used += grid;
    return SCN_OK;
  });
  if (rc != SCN_OK) return rc;
  SCN_CUDA_TRY(launch_dependent(k_grad_norm_finish, dim3(1), dim3(FINISH), 0, s, partial, used, d_norm));
  SCN_LAUNCH_CHECK("k_grad_norm_finish");
  return SCN_OK;
}

extern "C" int scn_adamw_step(const scn_adamw_tensor_t *tensors, int count, const scn_adamw_t *h, const scn_adamw_scalars_t *d_scalars, const float *d_norm,
                              scn_stream_t stream) {
  clear_error();
  if (const char *why = wrong_list(tensors, count, true)) return fail(SCN_ERR_INVALID, why);
  if (((uintptr_t)d_scalars | (uintptr_t)d_norm) & 3) return fail(SCN_ERR_INVALID, "AdamW: misaligned pointer");
  scn_adamw_scalars_t scalars = {};
  if (!d_scalars) {
    const int rc = scn_adamw_scalars(h, &scalars);
    if (rc != SCN_OK) return rc;
    if (h->max_norm > 0 && !d_norm) return fail(SCN_ERR_INVALID, "AdamW: clipping needs the gradients' norm");
  }
  cudaStream_t s = (cudaStream_t)stream;
  const Ones ones = {make_float2(1.f, 1.f), make_float2(-1.f, -1.f)};
  const auto eight = [](const scn_adamw_tensor_t &t) { return t.d_m_scale != nullptr; };
  int rc = for_lists(tensors, count, 1, [&](const scn_adamw_tensor_t &t) { return !eight(t); }, wide_step, [&](const auto &l) -> int {
    SCN_CUDA_TRY(launch_dependent(k_adamw_32<std::decay_t<decltype(l)>::capacity>, dim3(l.chunks), dim3(THREADS), 0, s, l, scalars, d_scalars, d_norm));
    SCN_LAUNCH_CHECK("k_adamw_32");
    return SCN_OK;
  });
  if (rc != SCN_OK) return rc;
  return for_lists(tensors, count, 8, eight, wide_step, [&](const auto &l) -> int {
    SCN_CUDA_TRY(launch_dependent(k_adamw_8<std::decay_t<decltype(l)>::capacity>, dim3(l.chunks), dim3(THREADS), 0, s, l, scalars, d_scalars, d_norm, ones));
    SCN_LAUNCH_CHECK("k_adamw_8");
    return SCN_OK;
  });
}

extern "C" int scn_adamw_decode(const void *d_codes, const float *d_scale, long long n, int second, float *d_out, scn_stream_t stream) {
  clear_error();
  if (n < 0) return fail(SCN_ERR_INVALID, "bad size");
  if (n == 0) return SCN_OK;
  if (!d_codes || !d_scale || !d_out) return fail(SCN_ERR_INVALID, "null pointer");
  if (((uintptr_t)d_scale | (uintptr_t)d_out) & 3) return fail(SCN_ERR_INVALID, "AdamW: misaligned pointer");
  const long long wide = (((uintptr_t)d_codes & 7) | ((uintptr_t)d_out & 31)) == 0 ? n / 8 * 8 : 0;
  k_adamw_decode<<<grid_for((n + 7) / 8, THREADS, 32), THREADS, 0, (cudaStream_t)stream>>>((const unsigned char *)d_codes, d_scale, n, wide, second, d_out);
  SCN_LAUNCH_CHECK("k_adamw_decode");
  return SCN_OK;
}
