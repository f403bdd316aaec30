// Embedding table in front of the first layer: rows by token, and the table's gradient by sorted tokens.
#include <algorithm>
#include "scn_types.cuh"

namespace scn {
namespace {

// out[i][c] = scale * table[tokens[i]][c]; no row for a token outside [0, vocab).
template <class T, class O>
__global__ void k_embedding_forward(const T *table, int vocab, int C, const int *tokens, long long n, float scale, O *out, long long stride, int *errors) {
  const long long total = n * C;
  for (long long e = blockIdx.x * (long long)blockDim.x + threadIdx.x; e < total; e += (long long)gridDim.x * blockDim.x) {
    const long long i = e / C;
    const int c = (int)(e - i * C), t = tokens[i];
    float v = 0.f;
    if (t >= 0 && t < vocab) v = to_float(table[(long long)t * C + c]) * scale;
    else if (t >= vocab && errors && c == 0) atomicOr(errors, SCN_DEV_ERR_KEY);
    out[i * stride + c] = from_float<O>(v);
  }
}

// ------------------------------------------------------------------ stable radix sort of (token, row)
// Digits of at most MAX_DIGIT bits, least significant first; per pass: digit counts of each tile, their running sums
// over the tiles, and the scatter.  A tile is TILE consecutive entries, a warp of it WARP_ITEMS consecutive ones.
constexpr int THREADS = 256, WARPS = THREADS / 32, ROUNDS = 16, TILE = THREADS * ROUNDS, WARP_ITEMS = 32 * ROUNDS, MAX_DIGIT = 10;

struct Pass {
  const int *tokens;         // first pass: the caller's tokens (row = index), else null
  const unsigned *keys, *rows;
  unsigned *keysOut, *rowsOut;
  int n, vocab, tiles, shift, bits;
  unsigned *counts;          // [2^bits][tiles]
  unsigned *totals;          // [2^bits]
  int *errors;
};
// The token, or vocab (sorted behind all tokens) where it names no row.
__device__ __forceinline__ unsigned key_of(const Pass &p, int i) {
  if (!p.tokens) return p.keys[i];
  const int t = p.tokens[i];
  return t >= 0 && t < p.vocab ? (unsigned)t : (unsigned)p.vocab;
}
__global__ void __launch_bounds__(THREADS) k_radix_count(const Pass p) {
  extern __shared__ unsigned hist[];
  const int digits = 1 << p.bits;
  for (int d = threadIdx.x; d < digits; d += THREADS) hist[d] = 0;
  __syncthreads();
  const int first = blockIdx.x * TILE, last = min(p.n - first, TILE);
  for (int j = threadIdx.x; j < last; j += THREADS) {
    if (p.tokens && p.errors && p.tokens[first + j] >= p.vocab) atomicOr(p.errors, SCN_DEV_ERR_KEY);
    atomicAdd(&hist[(key_of(p, first + j) >> p.shift) & (digits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += THREADS) p.counts[(long long)d * p.tiles + blockIdx.x] = hist[d];
}
// One CTA a digit: counts[d][*] becomes its exclusive running sum, totals[d] its sum.
__global__ void __launch_bounds__(THREADS) k_radix_scan(const Pass p) {
  __shared__ unsigned warpSum[WARPS];
  unsigned *row = p.counts + (long long)blockIdx.x * p.tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned before = 0;
  for (int base = 0; base < p.tiles; base += THREADS) {
    const int j = base + threadIdx.x;
    const unsigned own = j < p.tiles ? row[j] : 0u;
    unsigned sum = own;
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) warpSum[warp] = sum;
    __syncthreads();
    unsigned all = 0, mine = 0;
    for (int w = 0; w < WARPS; ++w) { if (w == warp) mine = all; all += warpSum[w]; }
    if (j < p.tiles) row[j] = before + mine + sum - own;
    before += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.totals[blockIdx.x] = before;
}
__global__ void __launch_bounds__(THREADS) k_radix_scatter(const Pass p) {
  extern __shared__ unsigned mem[];
  const int digits = 1 << p.bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned *count = mem; // [warp][digit]
  __shared__ unsigned warpSum[WARPS];
  for (int d = threadIdx.x; d < WARPS * digits; d += THREADS) count[d] = 0;
  __syncthreads();
  const int first = blockIdx.x * TILE + warp * WARP_ITEMS;
  unsigned key[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = first + r * 32 + lane;
    const bool in = i < p.n;
    key[r] = in ? key_of(p, i) : 0u;
    const unsigned d = (key[r] >> p.shift) & (digits - 1);
    const unsigned peers = __match_any_sync(~0u, in ? d : (unsigned)digits);
    if (in) rank[r] = count[warp * digits + d] + __popc(peers & ((1u << lane) - 1));
    __syncwarp();
    if (in && (peers >> lane) == 1u) count[warp * digits + d] += __popc(peers); // the group's last lane
    __syncwarp();
  }
  __syncthreads();
  // count becomes each warp's own start: behind the smaller digits, this digit in earlier tiles and in earlier warps
  const int per = (digits + THREADS - 1) / THREADS, d0 = threadIdx.x * per;
  unsigned own = 0;
  for (int d = d0; d < min(digits, d0 + per); ++d) own += p.totals[d];
  unsigned sum = own;
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned v = __shfl_up_sync(~0u, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) warpSum[warp] = sum;
  __syncthreads();
  unsigned at = sum - own;
  for (int w = 0; w < warp; ++w) at += warpSum[w];
  for (int d = d0; d < min(digits, d0 + per); ++d) {
    unsigned s = at + p.counts[(long long)d * p.tiles + blockIdx.x];
    at += p.totals[d];
    for (int w = 0; w < WARPS; ++w) { const unsigned c = count[w * digits + d]; count[w * digits + d] = s; s += c; }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = first + r * 32 + lane;
    if (i >= p.n) continue;
    const unsigned dst = count[warp * digits + ((key[r] >> p.shift) & (digits - 1))] + rank[r];
    p.keysOut[dst] = key[r];
    p.rowsOut[dst] = p.tokens ? (unsigned)i : p.rows[i];
  }
}

// One warp a table row: its tokens' rows lie together in the sorted order.
__device__ __forceinline__ int lower_bound(const unsigned *keys, int n, unsigned t) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (keys[mid] < t) lo = mid + 1; else hi = mid;
  }
  return lo;
}
template <class T>
__global__ void __launch_bounds__(THREADS) k_embedding_backward(const unsigned *keys, const unsigned *rows, int n, const T *dout, long long stride, int vocab,
                                                                int C, float scale, int accumulate, float *dtable) {
  const int t = blockIdx.x * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= vocab) return;
  const int first = lower_bound(keys, n, t), last = lower_bound(keys, n, t + 1u);
  if (accumulate && first == last) return;
  for (int c = lane; c < C; c += 32) {
    float sum = 0.f;
    for (int i = first; i < last; ++i) sum += to_float(dout[rows[i] * stride + c]);
    float *to = dtable + (long long)t * C + c;
    *to = accumulate ? *to + scale * sum : scale * sum;
  }
}

struct SortPlan {
  int tiles, passes, digit;           // digit: bits a pass (the last one may have fewer)
  size_t array, counts, totals, total; // bytes
};
SortPlan plan_sort(long long n, int vocab) {
  SortPlan p;
  int bits = 1;
  while (bits < 31 && ((long long)vocab >> bits) > 0) ++bits; // keys 0..vocab
  p.passes = (bits + MAX_DIGIT - 1) / MAX_DIGIT;
  p.digit = (bits + p.passes - 1) / p.passes;
  p.tiles = (int)((n + TILE - 1) / TILE);
  p.array = align_up(sizeof(unsigned) * (size_t)n, 256);
  p.counts = align_up(sizeof(unsigned) * ((size_t)p.tiles << p.digit), 256);
  p.totals = align_up(sizeof(unsigned) << p.digit, 256);
  p.total = 4 * p.array + p.counts + p.totals + 256;
  return p;
}

} // namespace
} // namespace scn

using namespace scn;

extern "C" int scn_embedding_forward(const void *d_table, int table_type, int vocab, int C, const int *d_tokens, long long n, float scale, void *d_out,
                                     int out_type, long long out_stride, int *d_errors, scn_stream_t stream) {
  clear_error();
  if (vocab < 1 || C < 1 || n < 0 || n > 0x7fffffffll) return fail(SCN_ERR_INVALID, "bad embedding sizes");
  if (out_stride < C) return fail(SCN_ERR_INVALID, "embedding: the output's row stride is below the number of features");
  if (!type_known(table_type) || !type_known(out_type)) return fail(SCN_ERR_INVALID, "embedding: unknown type");
  if (n == 0) return SCN_OK;
  if (!d_table || !d_tokens || !d_out) return fail(SCN_ERR_INVALID, "null pointer");
  const int grid = grid_for(n * C, 256);
  SCN_DISPATCH_TYPE(table_type, T, SCN_DISPATCH_TYPE(out_type, O, (k_embedding_forward<T, O><<<grid, 256, 0, (cudaStream_t)stream>>>(
                    (const T *)d_table, vocab, C, d_tokens, n, scale, (O *)d_out, out_stride, d_errors))));
  SCN_LAUNCH_CHECK("k_embedding_forward");
  return SCN_OK;
}

extern "C" size_t scn_embedding_backward_workspace_bytes(long long n, int vocab, int C) {
  if (n < 0 || n > 0x7fffffffll - TILE || vocab < 1 || C < 1) return 0;
  return plan_sort(n, vocab).total;
}

extern "C" int scn_embedding_backward(const int *d_tokens, long long n, const void *d_dout, int dout_type, long long dout_stride, int vocab, int C,
                                      float scale, int accumulate, float *d_dtable, int *d_errors, void *d_workspace, size_t workspace_bytes,
                                      scn_stream_t stream) {
  clear_error();
  if (vocab < 1 || C < 1 || n < 0 || n > 0x7fffffffll - TILE) return fail(SCN_ERR_INVALID, "bad embedding sizes");
  if (dout_stride < C) return fail(SCN_ERR_INVALID, "embedding: the gradient's row stride is below the number of features");
  if (!type_known(dout_type)) return fail(SCN_ERR_INVALID, "embedding: unknown type");
  if (!d_dtable || !d_workspace) return fail(SCN_ERR_INVALID, "null pointer");
  if (n && (!d_tokens || !d_dout)) return fail(SCN_ERR_INVALID, "null pointer");
  const SortPlan sp = plan_sort(n, vocab);
  if (workspace_bytes < sp.total) return fail(SCN_ERR_WORKSPACE, "workspace smaller than scn_embedding_backward_workspace_bytes()");
  if ((uintptr_t)d_workspace & 15) return fail(SCN_ERR_INVALID, "embedding: the workspace must be 16-byte aligned");
  cudaStream_t s = (cudaStream_t)stream;
  if (n == 0) {
    if (!accumulate) SCN_CUDA_TRY(cudaMemsetAsync(d_dtable, 0, sizeof(float) * (size_t)vocab * C, s));
    return SCN_OK;
  }
  char *w = (char *)d_workspace;
  unsigned *array[4];
  for (int i = 0; i < 4; ++i) array[i] = (unsigned *)(w + i * sp.array);
  Pass p = {};
  p.n = (int)n; p.vocab = vocab; p.tiles = sp.tiles; p.bits = sp.digit;
  p.counts = (unsigned *)(w + 4 * sp.array);
  p.totals = (unsigned *)(w + 4 * sp.array + sp.counts);
  p.errors = d_errors;
  for (int k = 0; k < sp.passes; ++k) {
    p.tokens = k == 0 ? d_tokens : nullptr;
    p.keys = array[2 * ((k + 1) & 1)]; p.rows = array[2 * ((k + 1) & 1) + 1];
    p.keysOut = array[2 * (k & 1)]; p.rowsOut = array[2 * (k & 1) + 1];
    p.shift = k * sp.digit;
    const int digits = 1 << p.bits;
    k_radix_count<<<p.tiles, THREADS, sizeof(unsigned) * digits, s>>>(p);
    SCN_LAUNCH_CHECK("k_radix_count");
    k_radix_scan<<<digits, THREADS, 0, s>>>(p);
    SCN_LAUNCH_CHECK("k_radix_scan");
    k_radix_scatter<<<p.tiles, THREADS, sizeof(unsigned) * digits * WARPS, s>>>(p);
    SCN_LAUNCH_CHECK("k_radix_scatter");
  }
  SCN_DISPATCH_TYPE(dout_type, T, (k_embedding_backward<T><<<(vocab + WARPS - 1) / WARPS, THREADS, 0, s>>>(p.keysOut, p.rowsOut, (int)n, (const T *)d_dout,
                    dout_stride, vocab, C, scale, accumulate, d_dtable)));
  SCN_LAUNCH_CHECK("k_embedding_backward");
  return SCN_OK;
}
