// Embedding table in front of the first layer: rows by token, and the table's gradient by sorted tokens.
#include <algorithm>
#include "scn_types.cuh"

namespace scn {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, MAX_LANES = 64;

// out[i][c] = scale * table[tokens[i]][c]; a zero row for a token outside [0, vocab).  Groups of `lanes` threads take a row, W
// columns a thread at a time, LOOKUP_ROWS rows at once so that as many table rows are on their way; the output, which is
// not read again here, is stored past the caches' reach of the table.
template <class T, class O, int W, int ROWS>
__global__ void __launch_bounds__(THREADS) k_embedding_forward(const T *__restrict__ table, int vocab, int C, const int *__restrict__ tokens, long long n, float scale,
                                                               O *__restrict__ out, long long stride, int lanes, int groups, int *errors) {
  constexpr int V = W * sizeof(O) > 16 ? 16 / (int)sizeof(O) : W; // values a store
  const int group = threadIdx.x / lanes, lane = threadIdx.x - group * lanes, vectors = C / W;
  if (group >= groups) return;
  const long long step = (long long)gridDim.x * groups * ROWS;
  long long i = (long long)blockIdx.x * groups * ROWS + group;
  int next[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) next[u] = i + u * groups < n ? __ldg(tokens + i + u * groups) : -1;
  for (; i < n; i += step) {
    int t[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      t[u] = next[u];
      if (t[u] >= vocab) {
        if (lane == 0 && errors) atomicOr(errors, SCN_DEV_ERR_KEY);
        t[u] = -1;
      }
      next[u] = i + step + u * groups < n ? __ldg(tokens + i + step + u * groups) : -1; // the next turn's, while this one's rows travel
    }
    for (int v = lane; v < vectors; v += lanes) {
      Pack<T, W> from[ROWS];
#pragma unroll
      for (int u = 0; u < ROWS; ++u)
        if (t[u] >= 0) from[u] = load_pack<T, W>(table + (long long)t[u] * C + v * W);
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
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
  const auto launch = [&](auto kernel, int rows) {
    const int grid = (int)std::min((n + groups * rows - 1) / (groups * rows), 16ll * sm_count());
    kernel<<<grid, THREADS, 0, s>>>(table, vocab, C, tokens, n, scale, out, stride, lanes, groups, errors);
  };
  // narrow accesses: more rows at once, for as many bytes on their way
  if (W == MOST) launch(k_embedding_forward<T, O, MOST, 4>, 4);
  else if (W == 1) launch(k_embedding_forward<T, O, 1, 8>, 8);
  else if (W == MOST / 2) launch(k_embedding_forward<T, O, MOST / 2, 4>, 4);
  else launch(k_embedding_forward<T, O, 2, 8>, 8);
}

// ------------------------------------------------------------------ stable radix sort of (token, row)
// Digits of at most MAX_DIGIT bits, least significant first; per pass: digit counts of each tile, their running sums
// over the tiles, and the scatter.  A tile is THREADS * ROUNDS consecutive entries, a warp of it 32 * ROUNDS consecutive ones.
constexpr int MAX_DIGIT = 9;
struct Pass {
  const int *tokens;  // first pass: the caller's tokens (row = index), else null
  const uint2 *in;    // (key, row)
  uint2 *out;
  int n, vocab, tiles, shift, bits;
  unsigned *counts;   // [2^bits][tiles]
  unsigned *totals;   // [2^bits]
  int *errors;
  float *clear;       // first pass: clearN values to set to zero on the side, or null
  long long clearN;
};
// The token, or vocab (sorted behind all tokens) where it names no row.
__device__ __forceinline__ unsigned key_of(int token, int vocab) { return token >= 0 && token < vocab ? (unsigned)token : (unsigned)vocab; }
__device__ void clear_floats(float *p, long long n, long long self, long long step) {
  const long long before = min(n, (long long)(((16 - ((uintptr_t)p & 15)) & 15) / 4)), whole = (n - before) / 4;
  for (long long i = self; i < whole; i += step) ((float4 *)(p + before))[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (long long i = self; i < n; i += step)
    if (i >= before && i < before + 4 * whole) i += (before + 4 * whole - i - 1) / step * step; // (only the ends are left)
    else p[i] = 0.f;
}
template <int ROUNDS> __global__ void __launch_bounds__(THREADS) k_radix_count(const Pass p) {
  extern __shared__ unsigned hist[];
  wait_for_prior_grids();
  dependents_may_launch();
  if ((int)blockIdx.x >= p.tiles) { // the table's zeros, written while the sort's kernels wait for one another
    clear_floats(p.clear, p.clearN, (long long)(blockIdx.x - p.tiles) * THREADS + threadIdx.x, (long long)(gridDim.x - p.tiles) * THREADS);
    return;
  }
  const int digits = 1 << p.bits;
  const long long first = (long long)blockIdx.x * (THREADS * ROUNDS);
  unsigned key[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const long long i = first + r * THREADS + threadIdx.x;
    key[r] = i >= p.n ? 0u : p.tokens ? (unsigned)p.tokens[i] : p.in[i].x;
  }
  for (int d = threadIdx.x; d < digits; d += THREADS) hist[d] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (first + r * THREADS + threadIdx.x >= p.n) break;
    if (p.tokens) {
      if (p.errors && (int)key[r] >= p.vocab) atomicOr(p.errors, SCN_DEV_ERR_KEY);
      key[r] = key_of((int)key[r], p.vocab);
    }
    atomicAdd(&hist[(key[r] >> p.shift) & (digits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += THREADS) p.counts[(long long)d * p.tiles + blockIdx.x] = hist[d];
}
// Running sum over the CTA's threads: what the threads before this one hold; `all`: what all of them hold.
__device__ __forceinline__ unsigned sum_before(unsigned own, unsigned *warpSum, unsigned &all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned sum = own;
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned v = __shfl_up_sync(~0u, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) warpSum[warp] = sum;
  __syncthreads();
  unsigned before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) { if (w == warp) before = all; all += warpSum[w]; }
  __syncthreads();
  return before + sum - own;
}
// One CTA a digit: counts[d][*] becomes its exclusive running sum, totals[d] its sum.
__global__ void __launch_bounds__(THREADS) k_radix_scan(const Pass p) {
  __shared__ unsigned warpSum[WARPS];
  wait_for_prior_grids();
  dependents_may_launch();
  unsigned *row = p.counts + (long long)blockIdx.x * p.tiles;
  unsigned before = 0, all;
  for (int base = 0; base < p.tiles; base += THREADS) {
    const int j = base + threadIdx.x;
    const unsigned own = j < p.tiles ? row[j] : 0u, at = sum_before(own, warpSum, all);
    if (j < p.tiles) row[j] = before + at;
    before += all;
  }
  if (threadIdx.x == 0) p.totals[blockIdx.x] = before;
}
// Places of a tile's entries in its order by digit: place[r] of the entry that this thread holds in round r (a warp's entries
// lie one after the other, a round's in the order of the lanes).  count[WARPS][digits]: scratch; start(d, at, n) is called once
// for each digit with the place `at` of its first entry and their number n.  Ranks within a round come from one ballot a bit.
template <int ROUNDS, class Start>
__device__ __forceinline__ void places_by_digit(const unsigned (&key)[ROUNDS], int inTile, int shift, int bits, unsigned short *count, unsigned *warpSum,
                                                unsigned (&place)[ROUNDS], Start start) {
  const int digits = 1 << bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < WARPS * digits / 2; d += THREADS) ((unsigned *)count)[d] = 0;
  __syncthreads();
  unsigned short *own = count + warp * digits;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool in = (warp * ROUNDS + r) * 32 + lane < inTile;
    const unsigned d = (key[r] >> shift) & (digits - 1);
    unsigned peers = __ballot_sync(~0u, in);
    for (int b = 0; b < bits; ++b) {
      const bool set = d >> b & 1;
      const unsigned votes = __ballot_sync(~0u, set);
      peers &= set ? votes : ~votes;
    }
    if (in) {
      const unsigned n = own[d];
      place[r] = n + __popc(peers & ((1u << lane) - 1));
      __syncwarp(peers);
      if (peers >> lane == 1u) own[d] = (unsigned short)(n + __popc(peers)); // the last of the lanes with this digit
    }
    __syncwarp();
  }
  __syncthreads();
  const int per = (digits + THREADS - 1) / THREADS, d0 = threadIdx.x * per, d1 = min(digits, d0 + per);
  unsigned sum = 0, all;
  for (int d = d0; d < d1; ++d)
    for (int w = 0; w < WARPS; ++w) sum += count[w * digits + d];
  unsigned at = sum_before(sum, warpSum, all);
  for (int d = d0; d < d1; ++d) {
    const unsigned first = at;
    for (int w = 0; w < WARPS; ++w) {
      const unsigned n = count[w * digits + d];
      count[w * digits + d] = (unsigned short)at;
      at += n;
    }
    start(d, first, at - first);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if ((warp * ROUNDS + r) * 32 + lane < inTile) place[r] += own[(key[r] >> shift) & (digits - 1)];
}
// A tile is put in order in shared memory first, so that entries of one digit leave side by side.
template <int ROUNDS> __global__ void __launch_bounds__(THREADS) k_radix_scatter(const Pass p) {
  extern __shared__ uint2 stage[];
  constexpr int TILE = THREADS * ROUNDS;
  const int digits = 1 << p.bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned *shift = (unsigned *)(stage + TILE); // [digits]: place in the output less place in the tile
  unsigned short *count = (unsigned short *)(shift + digits);
  __shared__ unsigned warpSum[WARPS];
  wait_for_prior_grids();
  dependents_may_launch();
  const long long first = (long long)blockIdx.x * TILE;
  const int inTile = (int)min((long long)TILE, p.n - first);
  unsigned key[ROUNDS], row[ROUNDS], place[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int j = (warp * ROUNDS + r) * 32 + lane;
    key[r] = 0; row[r] = (unsigned)(first + j);
    if (j < inTile) {
      if (p.tokens) key[r] = key_of(p.tokens[first + j], p.vocab);
      else { const uint2 e = p.in[first + j]; key[r] = e.x; row[r] = e.y; }
    }
  }
  // entries of smaller digits, plus those of the digit in earlier tiles
  const int per = (digits + THREADS - 1) / THREADS, d0 = threadIdx.x * per, d1 = min(digits, d0 + per);
  unsigned sum = 0, all;
  for (int d = d0; d < d1; ++d) sum += p.totals[d];
  unsigned at = sum_before(sum, warpSum, all);
  for (int d = d0; d < d1; ++d) {
    shift[d] = at + p.counts[(long long)d * p.tiles + blockIdx.x];
    at += p.totals[d];
  }
  places_by_digit<ROUNDS>(key, inTile, p.shift, p.bits, count, warpSum, place, [&](int d, unsigned start, unsigned) { shift[d] -= start; });
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if ((warp * ROUNDS + r) * 32 + lane < inTile) stage[place[r]] = make_uint2(key[r], row[r]);
  __syncthreads();
  for (int j = threadIdx.x; j < inTile; j += THREADS) {
    const uint2 e = stage[j];
    p.out[shift[(e.x >> p.shift) & (digits - 1)] + j] = e;
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
  const uint2 *entries;        // (token, row), sorted
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
// The sums of `count` sorted entries in shared memory; before, after: the tokens around them.  items: 2 * groups keys and as
// many rows of a slab's width.
template <class T, int W>
__device__ __forceinline__ void sum_entries(const Sums &p, const T *dout, const uint2 *entry, int count, unsigned before, unsigned after, unsigned *itemKey, float *item) {
  const unsigned none = p.vocab; // the key of rows without a token: behind all others
  const int width = p.lanes * W, column0 = blockIdx.y * width, group = threadIdx.x / p.lanes, lane = threadIdx.x - group * p.lanes, c = column0 + lane * W;
  for (int i = threadIdx.x; i < 2 * p.groups; i += THREADS) itemKey[i] = none;
  __syncthreads();
  if (group < p.groups && c < p.C) {
    const int each = (count + p.groups - 1) / p.groups, begin = min(group * each, count), end = min(begin + each, count);
    float sum[W];
    unsigned now = begin < end ? entry[begin].x : none;
    bool atHead = true;
#pragma unroll
    for (int w = 0; w < W; ++w) sum[w] = 0.f;
    for (int i = begin; i < end && entry[i].x != none; i += SUM_UNROLL) {
      Pack<T, W> v[SUM_UNROLL];
      unsigned k[SUM_UNROLL];
#pragma unroll
      for (int u = 0; u < SUM_UNROLL; ++u) {
        const uint2 e = i + u < end ? entry[i + u] : make_uint2(none, 0u);
        k[u] = e.x;
        if (k[u] != none) v[u] = load_pack<T, W>(dout + e.y * p.stride + c);
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
template <class T, int W> __global__ void __launch_bounds__(THREADS) k_embedding_sums(const Sums p, const T *dout) {
  extern __shared__ uint2 entry[];
  unsigned *itemKey = (unsigned *)(entry + p.tile);
  wait_for_prior_grids();
  dependents_may_launch();
  const long long first = (long long)blockIdx.x * p.tile;
  const int count = (int)min((long long)p.tile, p.n - first);
  for (int i = threadIdx.x; i < count; i += THREADS) entry[i] = p.entries[first + i];
  const unsigned none = p.vocab;
  const unsigned before = first > 0 ? p.entries[first - 1].x : none, after = first + count < p.n ? p.entries[first + count].x : none;
  sum_entries<T, W>(p, dout, entry, count, before, after, itemKey, (float *)(itemKey + 2 * p.groups));
}
// The whole gradient of at most SMALL rows in one launch: the first CTAs (one a slab) sort the entries in shared memory and
// add them up; the others write the zeros of the rows that no token names, each for a range of `range` rows.
constexpr int SMALL_ROUNDS = 4, SMALL = THREADS * SMALL_ROUNDS, SMALL_DIGIT = 8, MOST_RANGE = 16384;
template <class T, int W>
__global__ void __launch_bounds__(THREADS) k_embedding_backward_small(const Sums p, const T *dout, const int *tokens, int bits, int range, int *errors) {
  extern __shared__ uint2 entry[]; // two copies of SMALL entries, then the items; the digit counts lie where the items go
  __shared__ unsigned warpSum[WARPS], named[MOST_RANGE / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_prior_grids();
  dependents_may_launch();
  if (blockIdx.x > 0) {
    if (blockIdx.y > 0) return;
    const int first = (int)(blockIdx.x - 1) * range, rows = min(range, p.vocab - first);
    for (int i = threadIdx.x; i < (rows + 31) / 32; i += THREADS) named[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.n; i += THREADS) {
      const int t = tokens[i] - first;
      if (tokens[i] >= first && t < rows) atomicOr(&named[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
    for (int r = warp; r < rows; r += WARPS)
      if (!(named[r >> 5] >> (r & 31) & 1)) clear_floats(p.dtable + (long long)(first + r) * p.C, p.C, lane, 32);
    return;
  }
  uint2 *now = entry, *other = entry + SMALL;
  unsigned *itemKey = (unsigned *)(entry + 2 * SMALL);
  for (int i = threadIdx.x; i < p.n; i += THREADS) {
    const int t = tokens[i];
    if (t >= p.vocab && errors && blockIdx.y == 0) atomicOr(errors, SCN_DEV_ERR_KEY);
    now[i] = make_uint2(key_of(t, p.vocab), i);
  }
  __syncthreads();
  const int passes = (bits + SMALL_DIGIT - 1) / SMALL_DIGIT, each = (bits + passes - 1) / passes;
  for (int k = 0; k < passes; ++k) {
    unsigned key[SMALL_ROUNDS], row[SMALL_ROUNDS], place[SMALL_ROUNDS];
#pragma unroll
    for (int r = 0; r < SMALL_ROUNDS; ++r) {
      const int j = (warp * SMALL_ROUNDS + r) * 32 + lane;
      const uint2 e = j < p.n ? now[j] : make_uint2(0u, 0u);
      key[r] = e.x; row[r] = e.y;
    }
    places_by_digit<SMALL_ROUNDS>(key, p.n, k * each, each, (unsigned short *)itemKey, warpSum, place, [](int, unsigned, unsigned) {});
#pragma unroll
    for (int r = 0; r < SMALL_ROUNDS; ++r)
      if ((warp * SMALL_ROUNDS + r) * 32 + lane < p.n) other[place[r]] = make_uint2(key[r], row[r]);
    __syncthreads();
    uint2 *t = now; now = other; other = t;
  }
  const unsigned none = p.vocab;
  sum_entries<T, W>(p, dout, now, p.n, none, none, itemKey, (float *)(itemKey + 2 * p.groups));
}
// One CTA a tile (times 32-column slabs): if the tile's last token begins in it and goes on, its parts are added up, every
// WARPS-th one by a warp, then over the warps.
__global__ void __launch_bounds__(THREADS) k_embedding_join(const Sums p, int tiles) {
  wait_for_prior_grids();
  dependents_may_launch();
  const int b = blockIdx.x;
  const long long first = (long long)b * p.tile, end = first + p.tile;
  if (end >= p.n) return;
  const unsigned k = p.entries[end - 1].x, after = p.entries[end].x, before = first > 0 ? p.entries[first - 1].x : (unsigned)p.vocab;
  if (k == (unsigned)p.vocab || after != k || before == k) return;
  __shared__ float part[WARPS][32];
  int last = b + 1; // the first tile behind that does not begin with k
  for (;;) {
    const int t = last + threadIdx.x;
    const int off = __syncthreads_count(t < tiles && p.entries[(long long)t * p.tile].x == k);
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

int sort_rounds(long long n) { return n > (1 << 20) ? 16 : 4; } // large tiles: longer runs of a digit; small ones: work for every SM
struct SortPlan {
  int tiles, passes, bits, digit;            // digit: bits a pass
  size_t array, counts, totals, parts, total; // bytes
};
SortPlan plan_sort(long long n, int vocab, int C) {
  SortPlan p;
  p.bits = 1;
  while (p.bits < 31 && ((long long)vocab >> p.bits) > 0) ++p.bits; // keys 0..vocab
  p.passes = (p.bits + MAX_DIGIT - 1) / MAX_DIGIT;
  p.digit = (p.bits + p.passes - 1) / p.passes;
  const long long tile = THREADS * sort_rounds(n);
  p.tiles = (int)((n + tile - 1) / tile);
  p.array = align_up(sizeof(uint2) * (size_t)n, 256);
  p.counts = align_up(sizeof(unsigned) * ((size_t)p.tiles << p.digit), 256);
  p.totals = align_up(sizeof(unsigned) << p.digit, 256);
  p.parts = align_up(sizeof(float) * (size_t)((n + sum_tile(n) - 1) / sum_tile(n)) * (size_t)C, 256); // of each tile's first and last token
  p.total = 2 * p.array + p.counts + p.totals + 2 * p.parts + 256;
  return p;
}
template <int ROUNDS> int sort_pass(const Pass &p, cudaStream_t s) {
  const int digits = 1 << p.bits, clearing = p.clear ? 2 * sm_count() : 0;
  SCN_CUDA_TRY(launch_dependent(k_radix_count<ROUNDS>, dim3(p.tiles + clearing), dim3(THREADS), sizeof(unsigned) * digits, s, p));
  SCN_LAUNCH_CHECK("k_radix_count");
  SCN_CUDA_TRY(launch_dependent(k_radix_scan, dim3(digits), dim3(THREADS), 0, s, p));
  SCN_LAUNCH_CHECK("k_radix_scan");
  const size_t smem = sizeof(uint2) * THREADS * ROUNDS + sizeof(unsigned) * digits + sizeof(unsigned short) * WARPS * digits;
  SCN_CUDA_TRY(launch_dependent(k_radix_scatter<ROUNDS>, dim3(p.tiles), dim3(THREADS), smem, s, p));
  SCN_LAUNCH_CHECK("k_radix_scatter");
  return SCN_OK;
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
  if (n < 0 || n > 0x7fff0000ll || vocab < 1 || C < 1) return 0;
  return plan_sort(n, vocab, C).total;
}

extern "C" int scn_embedding_backward(const int *d_tokens, long long n, const void *d_dout, int dout_type, long long dout_stride, int vocab, int C,
                                      float scale, int accumulate, float *d_dtable, int *d_errors, void *d_workspace, size_t workspace_bytes,
                                      scn_stream_t stream) {
  clear_error();
  if (vocab < 1 || C < 1 || n < 0 || n > 0x7fff0000ll) return fail(SCN_ERR_INVALID, "bad embedding sizes");
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
  const int W = pack_width(dout_type, d_dout, dout_stride, d_dtable, C), vectors = C / W, slabs = (vectors + MAX_LANES - 1) / MAX_LANES;
  Sums q = {};
  q.n = (int)n; q.vocab = vocab; q.C = C; q.stride = dout_stride;
  q.lanes = lanes_for(vectors);
  q.groups = THREADS / q.lanes;
  q.tile = sum_tile(n);
  q.scale = scale; q.accumulate = accumulate; q.dtable = d_dtable;
  q.head = (float *)(w + 2 * sp.array + sp.counts + sp.totals);
  q.tail = (float *)(w + 2 * sp.array + sp.counts + sp.totals + sp.parts);
  const size_t items = 4ull * 2 * q.groups * (1 + q.lanes * W);
  // F<T, W> for dout's type and the width
#define SCN_SUMS(F, ...)                                                                                              \
  SCN_DISPATCH_TYPE(dout_type, T, {                                                                                   \
    constexpr int MOST = 16 / (int)sizeof(T);                                                                         \
    if (W == MOST) SCN_CUDA_TRY(launch_dependent(F<T, MOST>, __VA_ARGS__));                                           \
    else if (W == MOST / 2) SCN_CUDA_TRY(launch_dependent(F<T, MOST / 2>, __VA_ARGS__));                              \
    else if (W == 1) SCN_CUDA_TRY(launch_dependent(F<T, 1>, __VA_ARGS__));                                            \
    else SCN_CUDA_TRY(launch_dependent(F<T, 2>, __VA_ARGS__));                                                        \
  })
  if (n <= SMALL) {
    const size_t counts = sizeof(unsigned short) * WARPS << SMALL_DIGIT;
    const int range = std::max(32, std::min(MOST_RANGE, (vocab + 4 * sm_count() - 1) / (4 * sm_count()))), clearing = accumulate ? 0 : (vocab + range - 1) / range;
    SCN_SUMS(k_embedding_backward_small, dim3(1 + clearing, slabs), dim3(THREADS), sizeof(uint2) * 2 * SMALL + std::max(items, counts), s, q, (const T *)d_dout,
             d_tokens, sp.bits, range, d_errors);
    SCN_LAUNCH_CHECK("k_embedding_backward_small");
    return SCN_OK;
  }
  uint2 *const array[2] = {(uint2 *)w, (uint2 *)(w + sp.array)};
  Pass p = {};
  p.n = (int)n; p.vocab = vocab; p.tiles = sp.tiles; p.bits = sp.digit;
  p.counts = (unsigned *)(w + 2 * sp.array);
  p.totals = (unsigned *)(w + 2 * sp.array + sp.counts);
  p.errors = d_errors;
  for (int k = 0; k < sp.passes; ++k) {
    p.tokens = k == 0 ? d_tokens : nullptr;
    p.in = array[(k + 1) & 1];
    p.out = array[k & 1];
    p.shift = k * sp.digit;
    p.clear = k == 0 && !accumulate ? d_dtable : nullptr;
    p.clearN = (long long)vocab * C;
    const int rc = sort_rounds(n) == 16 ? sort_pass<16>(p, s) : sort_pass<4>(p, s);
    if (rc != SCN_OK) return rc;
  }
  q.entries = p.out;
  const int tiles = (int)((n + q.tile - 1) / q.tile);
  SCN_SUMS(k_embedding_sums, dim3(tiles, slabs), dim3(THREADS), sizeof(uint2) * q.tile + items, s, q, (const T *)d_dout);
#undef SCN_SUMS
  SCN_LAUNCH_CHECK("k_embedding_sums");
  if (tiles > 1) {
    SCN_CUDA_TRY(launch_dependent(k_embedding_join, dim3(tiles, std::min((C + 31) / 32, 8)), dim3(THREADS), 0, s, q, tiles));
    SCN_LAUNCH_CHECK("k_embedding_join");
  }
  return SCN_OK;
}
