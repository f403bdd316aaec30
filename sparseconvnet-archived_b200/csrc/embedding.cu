// Embedding table in front of the first layer: rows by token, and the table's gradient by sorted tokens.
#include <algorithm>
#include "scn_types.cuh"

namespace scn {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, MAX_LANES = 64;

// out[i][c] = scale * table[tokens[i]][c]; a zero row for a token outside [0, vocab).  Groups of `lanes` threads take a row, W
// columns a thread at a time, LOOKUP_ROWS rows at once so that as many table rows are on their way; the output, which is
// not read again here, is stored past the caches' reach of the table.
constexpr int LOOKUP_ROWS = 4;
template <class T, class O, int W>
__global__ void __launch_bounds__(THREADS) k_embedding_forward(const T *__restrict__ table, int vocab, int C, const int *__restrict__ tokens, long long n, float scale,
                                                               O *__restrict__ out, long long stride, int lanes, int groups, int *errors) {
  constexpr int V = W * sizeof(O) > 16 ? 16 / (int)sizeof(O) : W; // values a store
  const int group = threadIdx.x / lanes, lane = threadIdx.x - group * lanes, vectors = C / W;
  if (group >= groups) return;
  const long long step = (long long)gridDim.x * groups * LOOKUP_ROWS;
  for (long long i = (long long)blockIdx.x * groups * LOOKUP_ROWS + group; i < n; i += step) {
    int t[LOOKUP_ROWS];
#pragma unroll
    for (int u = 0; u < LOOKUP_ROWS; ++u) {
      t[u] = i + u * groups < n ? __ldg(tokens + i + u * groups) : -1;
      if (t[u] >= vocab) {
        if (lane == 0 && errors) atomicOr(errors, SCN_DEV_ERR_KEY);
        t[u] = -1;
      }
    }
    for (int v = lane; v < vectors; v += lanes) {
      Pack<T, W> from[LOOKUP_ROWS];
#pragma unroll
      for (int u = 0; u < LOOKUP_ROWS; ++u)
        if (t[u] >= 0) from[u] = load_pack<T, W>(table + (long long)t[u] * C + v * W);
#pragma unroll
      for (int u = 0; u < LOOKUP_ROWS; ++u) {
        if (i + u * groups >= n) break;
        O *to = out + (i + u * groups) * stride + v * W;
#pragma unroll
        for (int w = 0; w < W; w += V) {
          Pack<O, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) o.v[k] = from_float<O>(t[u] >= 0 ? to_float(from[u].v[w + k]) * scale : 0.f);
          __stcs((typename Raw<V * (int)sizeof(O)>::type *)(to + w), o.raw);
        }
      }
    }
  }
}
// Threads of a group for rows of so many W-value pieces: all of them at once up to MAX_LANES, else in equal turns.
int lanes_for(int vectors) {
  const int turns = (vectors + MAX_LANES - 1) / MAX_LANES;
  return (vectors + turns - 1) / turns;
}
template <class T, class O> void launch_forward(const T *table, int vocab, int C, const int *tokens, long long n, float scale, O *out, long long stride,
                                                int *errors, cudaStream_t s) {
  // the widest access that addresses, width and stride allow: at most 16 bytes of the table
  constexpr int MOST = 16 / (int)sizeof(T);
  int W = MOST;
  while (W > 1 && !(C % W == 0 && stride % W == 0 && (uintptr_t)table % (W * sizeof(T)) == 0 && (uintptr_t)out % std::min<size_t>(16, W * sizeof(O)) == 0)) W /= 2;
  const int lanes = lanes_for(C / W), groups = THREADS / lanes;
  const long long rows = (long long)groups * LOOKUP_ROWS;
  const int grid = (int)std::min((n + rows - 1) / rows, 64ll * sm_count());
  if (W == MOST) k_embedding_forward<T, O, MOST><<<grid, THREADS, 0, s>>>(table, vocab, C, tokens, n, scale, out, stride, lanes, groups, errors);
  else if (W == 1) k_embedding_forward<T, O, 1><<<grid, THREADS, 0, s>>>(table, vocab, C, tokens, n, scale, out, stride, lanes, groups, errors);
  else if (W == MOST / 2) k_embedding_forward<T, O, MOST / 2><<<grid, THREADS, 0, s>>>(table, vocab, C, tokens, n, scale, out, stride, lanes, groups, errors);
  else k_embedding_forward<T, O, 2><<<grid, THREADS, 0, s>>>(table, vocab, C, tokens, n, scale, out, stride, lanes, groups, errors);
}

// ------------------------------------------------------------------ stable radix sort of (token, row)
// Digits of at most MAX_DIGIT bits, least significant first; per pass: digit counts of each tile, their running sums
// over the tiles, and the scatter.  A tile is TILE consecutive entries, a warp of it WARP_ITEMS consecutive ones.
constexpr int ROUNDS = 16, TILE = THREADS * ROUNDS, WARP_ITEMS = 32 * ROUNDS, MAX_DIGIT = 10;

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

// ------------------------------------------------------------------ sums of the sorted rows
// A tile of the sorted entries goes to one CTA (times column slabs): groups of `lanes` threads, W columns a thread, take
// equal runs of it one after the other and add the rows up in registers.  A run's tokens that lie between its first and
// its last are complete and go straight to the table; what is left of its first and last token is joined over the CTA in
// shared memory, and what is left of the tile's first and last token over the tiles by k_embedding_join.  So a token's
// rows are added in an order that depends on the sorted tokens alone, a token on most of the rows costs no more than
// others, and each table row is written once.
constexpr int SUM_UNROLL = 8, MAX_TILE = 2048;
struct Sums {
  const unsigned *keys, *rows; // sorted
  int n, vocab, C, tile;       // tile: entries a CTA
  long long stride;            // of dout's rows
  int lanes, groups;           // threads of a group, groups of a CTA; a slab is lanes * W columns
  float scale;
  int accumulate;
  float *dtable;
  float *head, *tail;          // [tiles][C]: the part of a tile's first (last) token, where that began (goes on) in another tile
};
template <int W> __device__ __forceinline__ void write_row(const Sums &p, unsigned key, int c, const float (&sum)[W]) {
  float *to = p.dtable + (long long)key * p.C + c;
#pragma unroll
  for (int w = 0; w < W; w += (W < 4 ? W : 4)) {
    constexpr int V = W < 4 ? W : 4;
    Pack<float, V> o;
    if (p.accumulate) o.raw = *(typename Raw<V * 4>::type *)(to + w);
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = p.accumulate ? o.v[k] + p.scale * sum[w + k] : p.scale * sum[w + k];
    *(typename Raw<V * 4>::type *)(to + w) = o.raw;
  }
}
template <class T, int W> __global__ void __launch_bounds__(THREADS) k_embedding_sums(const Sums p, const T *dout) {
  extern __shared__ unsigned mem[];
  unsigned *key = mem, *row = key + p.tile, *itemKey = row + p.tile; // items: each group's first and last token's sums
  float *item = (float *)(itemKey + 2 * p.groups);
  const int first = blockIdx.x * p.tile, count = min(p.tile, p.n - first), width = p.lanes * W, column0 = blockIdx.y * width;
  for (int i = threadIdx.x; i < count; i += THREADS) { key[i] = p.keys[first + i]; row[i] = p.rows[first + i]; }
  const unsigned none = p.vocab; // the key of rows without a token: behind all others
  for (int i = threadIdx.x; i < 2 * p.groups; i += THREADS) itemKey[i] = none;
  __syncthreads();
  const int group = threadIdx.x / p.lanes, lane = threadIdx.x - group * p.lanes, c = column0 + lane * W;
  if (group < p.groups && c < p.C) {
    const int each = (count + p.groups - 1) / p.groups, begin = min(group * each, count), end = min(begin + each, count);
    float sum[W];
    unsigned now = begin < end ? key[begin] : none;
    bool atHead = true;
#pragma unroll
    for (int w = 0; w < W; ++w) sum[w] = 0.f;
    for (int i = begin; i < end && key[i] != none; i += SUM_UNROLL) {
      Pack<T, W> v[SUM_UNROLL];
      unsigned k[SUM_UNROLL];
#pragma unroll
      for (int u = 0; u < SUM_UNROLL; ++u) {
        k[u] = i + u < end ? key[i + u] : none;
        if (k[u] != none) v[u] = load_pack<T, W>(dout + row[i + u] * p.stride + c);
      }
#pragma unroll
      for (int u = 0; u < SUM_UNROLL; ++u) {
        if (k[u] == none) break;
        if (k[u] != now) {
          if (atHead) {
#pragma unroll
            for (int w = 0; w < W; ++w) item[2 * group * width + lane * W + w] = sum[w];
            if (lane == 0) itemKey[2 * group] = now;
            atHead = false;
          } else write_row<W>(p, now, c, sum);
          now = k[u];
#pragma unroll
          for (int w = 0; w < W; ++w) sum[w] = 0.f;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) sum[w] += to_float(v[u].v[w]);
      }
    }
    if (now != none) {
      const int at = 2 * group + (atHead ? 0 : 1);
#pragma unroll
      for (int w = 0; w < W; ++w) item[at * width + lane * W + w] = sum[w];
      if (lane == 0) itemKey[at] = now;
    }
  }
  __syncthreads();
  if (count <= 0) return;
  const unsigned before = first > 0 ? p.keys[first - 1] : none, after = first + count < p.n ? p.keys[first + count] : none;
  for (int x = threadIdx.x; x < width && column0 + x < p.C; x += THREADS) {
    unsigned now = none;
    float sum[1] = {0.f};
    for (int j = 0; j <= 2 * p.groups; ++j) {
      const unsigned k = j < 2 * p.groups ? itemKey[j] : none;
      if (k == none && j < 2 * p.groups) continue;
      if (k != now) {
        if (now != none) {
          if (now == before) p.head[(long long)blockIdx.x * p.C + column0 + x] = sum[0];
          else if (now == after) p.tail[(long long)blockIdx.x * p.C + column0 + x] = sum[0];
          else write_row<1>(p, now, column0 + x, sum);
        }
        now = k;
        sum[0] = 0.f;
      }
      if (j < 2 * p.groups) sum[0] += item[j * width + x];
    }
  }
}
// One CTA a tile (times 32-column slabs): if the tile's last token begins in it and goes on, its parts are added up, every
// WARPS-th one by a warp, then over the warps.
__global__ void __launch_bounds__(THREADS) k_embedding_join(const Sums p, int tiles) {
  const int b = blockIdx.x, first = b * p.tile, end = first + p.tile;
  if (end >= p.n) return;
  const unsigned k = p.keys[end - 1];
  if (k == (unsigned)p.vocab || p.keys[end] != k || (first > 0 && p.keys[first - 1] == k)) return;
  __shared__ float part[WARPS][32];
  int last = b + 1; // the first tile behind that does not begin with k
  for (;;) {
    const int t = last + threadIdx.x;
    const int off = __syncthreads_count(t < tiles && p.keys[(long long)t * p.tile] == k);
    last += off;
    if (off < THREADS) break;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int c0 = blockIdx.y * 32; c0 < p.C; c0 += gridDim.y * 32) {
    float sum[1] = {0.f};
    if (c0 + lane < p.C) {
#pragma unroll 8
      for (int t = b + warp; t < last; t += WARPS) sum[0] += (t == b ? p.tail : p.head)[(long long)t * p.C + c0 + lane];
    }
    part[warp][lane] = sum[0];
    __syncthreads();
    if (warp == 0 && c0 + lane < p.C) {
      for (int w = 1; w < WARPS; ++w) sum[0] += part[w][lane];
      write_row<1>(p, k, c0 + lane, sum);
    }
    __syncthreads();
  }
}

// Values a thread takes at once: what the addresses, widths and strides of dout and the table allow, up to 16 bytes of dout.
int pack_width(int type, const void *dout, long long stride, const float *dtable, int C) {
  const int size = type_bytes(type);
  for (int W = 16 / size; W > 1; W /= 2)
    if (C % W == 0 && stride % W == 0 && (uintptr_t)dout % (W * size) == 0 && (uintptr_t)dtable % (4 * std::min(W, 4)) == 0) return W;
  return 1;
}
// Entries a CTA sums: MAX_TILE, fewer (a power of two) where that would leave SMs with less than four CTAs each.
int sum_tile(long long n) {
  int tile = MAX_TILE;
  while (tile > 64 && n / tile < 4 * 148) tile /= 2;
  return tile;
}

struct SortPlan {
  int tiles, passes, digit;           // digit: bits a pass (the last one may have fewer)
  size_t array, counts, totals, parts, total; // bytes
};
SortPlan plan_sort(long long n, int vocab, int C) {
  SortPlan p;
  int bits = 1;
  while (bits < 31 && ((long long)vocab >> bits) > 0) ++bits; // keys 0..vocab
  p.passes = (bits + MAX_DIGIT - 1) / MAX_DIGIT;
  p.digit = (bits + p.passes - 1) / p.passes;
  p.tiles = (int)((n + TILE - 1) / TILE);
  p.array = align_up(sizeof(unsigned) * (size_t)n, 256);
  p.counts = align_up(sizeof(unsigned) * ((size_t)p.tiles << p.digit), 256);
  p.totals = align_up(sizeof(unsigned) << p.digit, 256);
  p.parts = align_up(sizeof(float) * (size_t)((n + sum_tile(n) - 1) / sum_tile(n)) * (size_t)C, 256); // of each tile's first and last token
  p.total = 4 * p.array + p.counts + p.totals + 2 * p.parts + 256;
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
  SCN_DISPATCH_TYPE(table_type, T, SCN_DISPATCH_TYPE(out_type, O, launch_forward((const T *)d_table, vocab, C, d_tokens, n, scale, (O *)d_out, out_stride,
                                                                                 d_errors, (cudaStream_t)stream)));
  SCN_LAUNCH_CHECK("k_embedding_forward");
  return SCN_OK;
}

extern "C" size_t scn_embedding_backward_workspace_bytes(long long n, int vocab, int C) {
  if (n < 0 || n > 0x7fffffffll - TILE || vocab < 1 || C < 1) return 0;
  return plan_sort(n, vocab, C).total;
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
  const SortPlan sp = plan_sort(n, vocab, C);
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
  const int W = pack_width(dout_type, d_dout, dout_stride, d_dtable, C), vectors = C / W, slabs = (vectors + MAX_LANES - 1) / MAX_LANES;
  Sums q = {};
  q.keys = p.keysOut; q.rows = p.rowsOut;
  q.n = (int)n; q.vocab = vocab; q.C = C; q.stride = dout_stride;
  q.lanes = lanes_for(vectors);
  q.groups = THREADS / q.lanes;
  q.tile = sum_tile(n);
  q.scale = scale; q.accumulate = accumulate; q.dtable = d_dtable;
  q.head = (float *)(w + 4 * sp.array + sp.counts + sp.totals);
  q.tail = (float *)(w + 4 * sp.array + sp.counts + sp.totals + sp.parts);
  const int tiles = (int)((n + q.tile - 1) / q.tile);
  if (!accumulate) SCN_CUDA_TRY(cudaMemsetAsync(d_dtable, 0, sizeof(float) * (size_t)vocab * C, s));
  const size_t smem = 4ull * (2 * q.tile + 2 * q.groups) + 4ull * 2 * q.groups * q.lanes * W;
  const dim3 grid(tiles, slabs);
  SCN_DISPATCH_TYPE(dout_type, T, {
    constexpr int MOST = 16 / (int)sizeof(T);
    const T *from = (const T *)d_dout;
    if (W == MOST) k_embedding_sums<T, MOST><<<grid, THREADS, smem, s>>>(q, from);
    else if (W == MOST / 2) k_embedding_sums<T, MOST / 2><<<grid, THREADS, smem, s>>>(q, from);
    else if (W == 1) k_embedding_sums<T, 1><<<grid, THREADS, smem, s>>>(q, from);
    else k_embedding_sums<T, 2><<<grid, THREADS, smem, s>>>(q, from);
  });
  SCN_LAUNCH_CHECK("k_embedding_sums");
  if (tiles > 1) {
    k_embedding_join<<<dim3(tiles, std::min((C + 31) / 32, 8)), THREADS, 0, s>>>(q, tiles);
    SCN_LAUNCH_CHECK("k_embedding_join");
  }
  return SCN_OK;
}
