// Embedding table in front of the first layer: rows by token, out[i] = scale * table[tokens[i]], and the table's gradient,
// dtable[t] = scale * sum of dout[i] over tokens[i] == t, by sorted tokens.  Both are bound by memory: the lookup by its
// output (and the table rows, which mostly come out of the caches), the gradient by one read of dout and one write of the
// table, next to which the sort moves 8 bytes a row four times.
#include <algorithm>
#include "scn_types.cuh"

namespace scn {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, MAX_LANES = 64;

// out[i][c] = scale * table[tokens[i]][c]; a zero row for a token outside [0, vocab).  Groups of `lanes` threads take a row, W
// columns a thread at a time, ROWS rows at once so that as many table rows are on their way, with the tokens of the next turn
// already asked for; the output, which is not read again here, is stored so that it leaves the caches to the table.
// 3.4 M rows of 64 floats from a table of 65536: 160 us, 5.6 TB/s of the 889 MB it cannot do without (85 % of a plain copy's rate); 169 us
// once the power cap has brought the clock from 1965 to some 1800 MHz.
// Rows that end or begin inside a 32-byte sector next to bytes that nobody writes cost the memory a read of the sector each:
// the same rows 16 bytes apart take 350 us, 32 bytes apart 162 us.
struct Lookup {
  const char *table;
  const int *tokens;
  char *out;
  unsigned n, stride;     // stride: bytes from row to row of the output
  unsigned rowBytes;      // of the table
  int vocab, C;
  float scale;
  int *errors;
};
// The token, or -1 where it names no row.
__device__ __forceinline__ int row_of(const Lookup &p, unsigned i) {
  int t = i < p.n ? __ldg(p.tokens + i) : -1;
  if (t >= p.vocab) {
    if (p.errors) atomicOr(p.errors, SCN_DEV_ERR_KEY);
    t = -1;
  }
  return t;
}
template <class P> __device__ __forceinline__ P *at_row(P *base, unsigned row, unsigned bytes) { return base + (unsigned long long)row * bytes; }
template <class T, class O, int W, int ROWS> __global__ void __launch_bounds__(THREADS) k_embedding_forward(const Lookup p, unsigned lanes, unsigned groups) {
  constexpr int V = W * sizeof(O) > 16 ? 16 / (int)sizeof(O) : W; // values a store
  const unsigned group = threadIdx.x / lanes, lane = threadIdx.x - group * lanes, vectors = p.C / W;
  if (group >= groups) return;
  wait_for_prior_grids();
  dependents_may_launch();
  const unsigned step = gridDim.x * groups * ROWS;
  unsigned i = blockIdx.x * groups * ROWS + group;
  int next[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) next[u] = row_of(p, i + u * groups);
  for (; i < p.n; i += step) {
    int t[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) t[u] = next[u];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) next[u] = row_of(p, i + step + u * groups); // the next turn's, while this one's rows travel
    for (unsigned v = lane; v < vectors; v += lanes) {
      const char *column = p.table + v * (W * (unsigned)sizeof(T));
      Pack<T, W> from[ROWS];
#pragma unroll
      for (int u = 0; u < ROWS; ++u) from[u] = load_pack<T, W>((const T *)at_row(column, max(t[u], 0), p.rowBytes));
      char *to = p.out + v * (W * (unsigned)sizeof(O));
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        if (u > 0 && i + u * groups >= p.n) break;
        O *row = (O *)at_row(to, i + u * groups, p.stride);
#pragma unroll
        for (int w = 0; w < W; w += V) {
          Pack<O, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) o.v[k] = from_float<O>(t[u] >= 0 ? to_float(from[u].v[w + k]) * p.scale : 0.f);
          __stcs((typename Raw<V * (int)sizeof(O)>::type *)(row + w), o.raw);
        }
      }
    }
  }
}
// The same value by value, for widths, strides and addresses that allow no more: a warp takes ROWS rows and 32 * COLS columns at
// once.  224 k rows of 96 from a 16-bit table into rows of 99 floats: 26 us (a plain fill of as many bytes takes 14.5 us);
// groups of 48 threads with two turns a row took 39 us.
template <class T, class O, int ROWS, int COLS> __global__ void __launch_bounds__(THREADS) k_embedding_forward_single(const Lookup p) {
  const int lane = threadIdx.x & 31;
  const unsigned i = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * ROWS;
  if (i >= p.n) return;
  wait_for_prior_grids();
  dependents_may_launch();
  const int mine = row_of(p, lane < ROWS ? i + lane : p.n);
  for (int c = lane; c - lane < p.C; c += 32 * COLS) {
    const char *column = p.table + c * (int)sizeof(T);
    T v[ROWS][COLS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const T *row = (const T *)at_row(column, max(__shfl_sync(~0u, mine, u), 0), p.rowBytes);
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (c + 32 * j < p.C) v[u][j] = __ldg(row + 32 * j);
    }
    char *to = p.out + c * (int)sizeof(O);
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const bool named = __shfl_sync(~0u, mine, u) >= 0;
      if (u > 0 && i + u >= p.n) break;
      O *row = (O *)at_row(to, i + u, p.stride);
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (c + 32 * j < p.C) __stcs(row + 32 * j, from_float<O>(named ? to_float(v[u][j]) * p.scale : 0.f));
    }
  }
}
// Threads of a group for rows of so many W-value pieces: all of them at once up to MAX_LANES, else in equal turns.
int lanes_for(int vectors) {
  const int turns = (vectors + MAX_LANES - 1) / MAX_LANES;
  return (vectors + turns - 1) / turns;
}
template <class T, class O> cudaError_t launch_forward(const Lookup &p, cudaStream_t s) {
  // the widest access that addresses, width and stride allow: at most 16 bytes of the table
  constexpr int MOST = 16 / (int)sizeof(T);
  int W = MOST;
  while (W > 1 && !(p.C % W == 0 && (uintptr_t)p.table % (W * sizeof(T)) == 0 && ((uintptr_t)p.out | (uintptr_t)p.stride) % std::min<size_t>(16, W * sizeof(O)) == 0)) W /= 2;
  if (W == 1 && p.C > 16) {
    const auto single = [&](auto kernel, unsigned rows) { return launch_dependent(kernel, dim3((p.n + WARPS * rows - 1) / (WARPS * rows)), dim3(THREADS), 0, s, p); };
    // Rows of up to 32 values sixteen at a time, of up to 96 three, longer ones two, so that few lanes idle in a row's last columns.  224 k rows
    // three values apart, us with (16, 1), (3, 3), (2, 4): 20 columns 8.7, 13.1, 16.1; 32: 10.3, 13.1, 16.2; 48: 20.7, 15.8, 17.8; 64: 27.3, 18.6, 19.5;
    // 96: 41.5, 26.5, 26.2; 128: 53.8, 37.9, 33.1; 515: 243, 141, 124.  (8, 2) is no better than (3, 3) anywhere: 48: 16.1; 64: 19.7.
    if (p.C <= 32) return single(k_embedding_forward_single<T, O, 16, 1>, 16);
    if (p.C <= 96) return single(k_embedding_forward_single<T, O, 3, 3>, 3);
    return single(k_embedding_forward_single<T, O, 2, 4>, 2);
  }
  const unsigned lanes = lanes_for(p.C / W), groups = THREADS / lanes;
  const auto launch = [&](auto kernel, unsigned rows) {
    const unsigned grid = std::min((p.n + groups * rows - 1) / (groups * rows), 64u * sm_count());
    return launch_dependent(kernel, dim3(grid), dim3(THREADS), 0, s, p, lanes, groups);
  };
  // Two rows at once, four of half-width accesses.  us with two, four and eight rows: 3.4 M rows of 64 floats (16 bytes an access) 160, 188, 252; of
  // 30 (8 bytes) 119, 115, 192; of 15 (4 bytes) 99, 118, 168; 1 M rows of 98 16-bit values (4 bytes) 87, 88, 113.
  if (W == MOST / 2) return launch(k_embedding_forward<T, O, MOST / 2, 4>, 4);
  if (W == MOST) return launch(k_embedding_forward<T, O, MOST, 2>, 2);
  if constexpr (MOST == 8) // (a 16-bit table: 8, 4, 2, 1; floats: 4, 2, 1)
    if (W == 2) return launch(k_embedding_forward<T, O, 2, 2>, 2);
  return launch(k_embedding_forward<T, O, 1, 2>, 2);
}

// ------------------------------------------------------------------ stable radix sort of (token, row)
// Digits of at most MAX_DIGIT bits, least significant first; per pass: digit counts of each tile, their running sums
// over the tiles, and the scatter.  A tile is THREADS * ROUNDS consecutive entries, a warp of it 32 * ROUNDS consecutive ones.
// 3.4 M rows, 18-bit keys: 75 us for both passes (counts 12 + 5, running sums 6 + 5, scatters 24 + 21, overlapped launches
// included; the table's 33 MB of zeros are written beside the first counts).  It is bound by the latency of its short kernels
// and the scatter by the instructions that rank entries within a warp; wider digits (10 bits) and larger tiles (15 rounds: 219 us for the
// whole gradient, 8 rounds: 199, 4 rounds: 212) did not help.
constexpr int MAX_DIGIT = 9;
struct Pass {
  const int *tokens;  // first pass: the caller's tokens (row = index), else null
  const uint2 *in;    // (key, row)
  uint2 *out;
  int n, vocab, tiles, shift, bits;
  unsigned *counts;   // [tiles][2^bits]
  unsigned *totals;   // [2^bits], or null: counts as k_radix_count left them
  int *errors;
  float *clear;       // first pass: clearN values to set to zero on the side, or null
  long long clearN;
  unsigned *arrived;  // first pass: the sums' counters to set to zero (see join_group), or null
  long long arrivedN;
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
  for (long long i = blockIdx.x * (long long)THREADS + threadIdx.x; i < p.arrivedN; i += (long long)p.tiles * THREADS) p.arrived[i] = 0;
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
  for (int d = threadIdx.x; d < digits; d += THREADS) p.counts[(long long)blockIdx.x * digits + d] = hist[d];
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
// One CTA for SCAN_DIGITS digits (half a sector of each tile's counts, so that more SMs share the work): counts[*][d] becomes its exclusive running sum over the
// tiles, totals[d] its sum.  A thread takes one digit of a run of the tiles: it adds them up, learns what the runs before hold,
// and writes the running sums.  HELD: counts that stay in its registers in between, or 0 (reading them again
// took 3.4 M rows' gradient 187 us in place of 180).
constexpr int SCAN_DIGITS = 4, SCAN_THREADS = 1024, SCAN_RUNS = SCAN_THREADS / SCAN_DIGITS;
template <int HELD> __global__ void __launch_bounds__(SCAN_THREADS) k_radix_scan(const Pass p) {
  __shared__ unsigned runSum[SCAN_RUNS][SCAN_DIGITS];
  wait_for_prior_grids();
  dependents_may_launch();
  const int digits = 1 << p.bits, d = threadIdx.x % SCAN_DIGITS, run = threadIdx.x / SCAN_DIGITS;
  const int each = (p.tiles + SCAN_RUNS - 1) / SCAN_RUNS, begin = min(run * each, p.tiles), end = min(begin + each, p.tiles);
  unsigned *column = p.counts + blockIdx.x * SCAN_DIGITS + d;
  unsigned sum = 0, held[HELD > 0 ? HELD : 1];
  if constexpr (HELD > 0) {
#pragma unroll
    for (int u = 0; u < HELD; ++u) held[u] = begin + u < end ? column[(long long)(begin + u) * digits] : 0u;
#pragma unroll
    for (int u = 0; u < HELD; ++u) sum += held[u];
  } else {
#pragma unroll 8
    for (int t = begin; t < end; ++t) sum += column[(long long)t * digits];
  }
  runSum[run][d] = sum;
  __syncthreads();
  if (threadIdx.x < 32 * SCAN_DIGITS) { // a warp a digit: running sums over the runs
    const int lane = threadIdx.x & 31, digit = threadIdx.x >> 5;
    unsigned own[SCAN_RUNS / 32], all = 0;
#pragma unroll
    for (int r = 0; r < SCAN_RUNS / 32; ++r) { own[r] = runSum[lane * (SCAN_RUNS / 32) + r][digit]; all += own[r]; }
    unsigned at = all;
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(~0u, at, o);
      if (lane >= o) at += v;
    }
    if (lane == 31) p.totals[blockIdx.x * SCAN_DIGITS + digit] = at;
    at -= all;
#pragma unroll
    for (int r = 0; r < SCAN_RUNS / 32; ++r) { runSum[lane * (SCAN_RUNS / 32) + r][digit] = at; at += own[r]; }
  }
  __syncthreads();
  unsigned before = runSum[run][d];
  constexpr int TURN = HELD > 0 ? HELD : 8;
  for (int t0 = begin; t0 < end; t0 += TURN) {
    unsigned n[TURN];
#pragma unroll
    for (int u = 0; u < TURN; ++u) n[u] = HELD > 0 ? held[HELD > 0 ? u : 0] : t0 + u < end ? column[(long long)(t0 + u) * digits] : 0u;
#pragma unroll
    for (int u = 0; u < TURN; ++u) {
      if (t0 + u < end) column[(long long)(t0 + u) * digits] = before;
      before += n[u];
    }
  }
}
// Places of a tile's entries in its order by digit: place[r] of the entry that this thread holds in round r (a warp's entries
// lie one after the other, a round's in the order of the lanes).  count[WARPS][digits]: scratch, 4-byte aligned; start(d, at) is
// called once for each digit with the place of its first entry.  Ranks within a round come from one ballot a bit.
template <int ROUNDS, int BITS, class Start>
__device__ __forceinline__ void places_by_digit(const unsigned (&key)[ROUNDS], int inTile, int shift, unsigned short *count, unsigned *warpSum,
                                                unsigned (&place)[ROUNDS], Start start) {
  constexpr int DIGITS = 1 << BITS, PAIRS = DIGITS / 2;
  static_assert(PAIRS <= THREADS, "a thread takes a pair of digits");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned *pair = (unsigned *)count; // two digits' counts in a word: both stay below 2^16
  for (int d = threadIdx.x; d < WARPS * PAIRS; d += THREADS) pair[d] = 0;
  __syncthreads();
  unsigned short *own = count + warp * DIGITS;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool in = (warp * ROUNDS + r) * 32 + lane < inTile;
    const unsigned d = (key[r] >> shift) & (DIGITS - 1);
    unsigned peers = __ballot_sync(~0u, in);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
      const unsigned votes = __ballot_sync(~0u, d >> b & 1), other = (d >> b & 1) - 1u;
      peers &= votes ^ other;
    }
    const unsigned n = in ? own[d] : 0u;
    place[r] = n + __popc(peers & ((1u << lane) - 1));
    __syncwarp(); // (of the whole warp: lanes that waited for those with their digit alone would go on one digit after the other)
    if (in && peers >> lane == 1u) own[d] = (unsigned short)(n + __popc(peers)); // the last of the lanes with this digit
    __syncwarp();
  }
  __syncthreads();
  unsigned sum = 0, all; // counts become each warp's own start
  if (threadIdx.x < PAIRS)
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += pair[w * PAIRS + threadIdx.x];
  unsigned at = sum_before((sum & 0xffffu) + (sum >> 16), warpSum, all);
  if (threadIdx.x < PAIRS) {
    start(2 * threadIdx.x, at);
    start(2 * threadIdx.x + 1, at + (sum & 0xffffu));
    at |= (at + (sum & 0xffffu)) << 16;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const unsigned n = pair[w * PAIRS + threadIdx.x];
      pair[w * PAIRS + threadIdx.x] = at;
      at += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if ((warp * ROUNDS + r) * 32 + lane < inTile) place[r] += own[(key[r] >> shift) & (DIGITS - 1)];
}
// A tile is put in order in shared memory first, so that entries of one digit leave side by side.
template <int ROUNDS, int BITS> __global__ void __launch_bounds__(THREADS) k_radix_scatter(const Pass p) {
  constexpr int TILE = THREADS * ROUNDS, DIGITS = 1 << BITS, PAIRS = DIGITS / 2;
  __shared__ uint2 stage[TILE];
  __shared__ unsigned shift[DIGITS], warpSum[WARPS]; // shift: place in the output less place in the tile
  __shared__ __align__(4) unsigned short count[WARPS * DIGITS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
  unsigned all, low = 0, high = 0, lowBefore = 0, highBefore = 0;
  if (p.totals && threadIdx.x < PAIRS) {
    const uint2 total = ((const uint2 *)p.totals)[threadIdx.x], before = ((const uint2 *)p.counts)[(long long)blockIdx.x * PAIRS + threadIdx.x];
    low = total.x; high = total.y; lowBefore = before.x; highBefore = before.y;
  }
  if (!p.totals && threadIdx.x < PAIRS) { // few tiles: added up here, without k_radix_scan
#pragma unroll 16
    for (int t = 0; t < p.tiles; ++t) {
      const uint2 n = ((const uint2 *)p.counts)[t * PAIRS + threadIdx.x];
      if (t == (int)blockIdx.x) { lowBefore = low; highBefore = high; }
      low += n.x; high += n.y;
    }
  }
  const unsigned at = sum_before(low + high, warpSum, all);
  if (threadIdx.x < PAIRS) {
    shift[2 * threadIdx.x] = at + lowBefore;
    shift[2 * threadIdx.x + 1] = at + low + highBefore;
  }
  places_by_digit<ROUNDS, BITS>(key, inTile, p.shift, count, warpSum, place, [&](int d, unsigned start) { shift[d] -= start; });
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if ((warp * ROUNDS + r) * 32 + lane < inTile) stage[place[r]] = make_uint2(key[r], row[r]);
  __syncthreads();
  for (int j = threadIdx.x; j < inTile; j += THREADS) {
    const uint2 e = stage[j];
    p.out[shift[(e.x >> p.shift) & (DIGITS - 1)] + j] = e;
  }
}

// ------------------------------------------------------------------ sums of the sorted rows
// A tile of the sorted entries goes to one warp (times column slabs): groups of `lanes` threads, W columns a thread, take
// equal runs of it one after the other and add the rows up in registers.  A run's tokens that lie between its first and
// its last are complete and go straight to the table; what is left of its first and last token is joined over the warp in
// shared memory, and what is left of the tile's first and last token over the tiles by k_embedding_join.  So a token's
// rows are added in an order that depends on the sorted tokens alone, a token on most of the rows costs no more than
// others, and each table row is written once.  Warps wait for no other warp: a CTA whose warps met at its end would stand
// idle while its last rows arrive (that cost 22 of 129 us).  3.4 M rows of 64 16-bit values, 131072 tokens, the k-th in
// frequency about 1 / k: 97 us, 4.8 TB/s of the 463 MB read and written; reading rows of 128 bytes in that order and adding them up
// takes 78 us at best.  Tiles of 2048 entries a CTA took 120 us, a ring of asynchronous copies in front of the registers 130 us,
// rows interleaved over a warp's groups with a sum over the warp at each change of token 156 us.
constexpr int SUM_ROWS = 8, MAX_TILE = 256, MIN_TILE = 64; // rows a thread asks for at once
struct Sums {
  const uint2 *entries;        // (token, row), sorted
  int n, vocab, C, tile;       // tile: entries a warp
  unsigned stride;             // of dout's rows, in bytes
  int lanes;                   // threads of a group in the last slab (32 in the others); a slab is lanes * W columns (times J)
  float scale;
  int accumulate;
  float *dtable;
  float *head, *tail;          // [tiles][C]: the part of a tile's first (last) token, where that began (goes on) in another tile
  uint2 *ends;                 // [tiles]: each tile's first and last token
  unsigned *arrived;           // [slabs][tiles / 32], or null: see join_group
};
// The running sums of W columns.
template <int W> struct Columns {
  float2 v[W / 2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) v[i] = make_float2(0.f, 0.f);
  }
  template <class T> __device__ __forceinline__ void add(const Pack<T, W> &p) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) v[i] = __fadd2_rn(v[i], pair_of(p, i));
  }
  __device__ __forceinline__ float at(int w) const { return w & 1 ? v[w / 2].y : v[w / 2].x; }
};
template <> struct Columns<1> {
  float v;
  __device__ __forceinline__ void clear() { v = 0.f; }
  template <class T> __device__ __forceinline__ void add(const Pack<T, 1> &p) { v += to_float(p.v[0]); }
  __device__ __forceinline__ float at(int) const { return v; }
};
template <int W> __device__ __forceinline__ void write_row(const Sums &p, unsigned key, int c, const Columns<W> &sum) {
  float *to = p.dtable + (long long)key * p.C + c;
  constexpr int V = W < 4 ? W : 4;
#pragma unroll
  for (int w = 0; w < W; w += V) {
    Pack<float, V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = p.scale * sum.at(w + k);
    if (!p.accumulate) *(typename Raw<V * 4>::type *)(to + w) = o.raw;
    else if constexpr (V == 4) atomicAdd((float4 *)(to + w), make_float4(o.v[0], o.v[1], o.v[2], o.v[3])); // (not waited for; no other
    else if constexpr (V == 2) atomicAdd((float2 *)(to + w), make_float2(o.v[0], o.v[1]));                  //  thread adds to this row)
    else atomicAdd(to + w, o.v[0]);
  }
}
// The sums of a warp's `count` sorted entries in shared memory, all of them of tokens, with SUM_ROWS more entries behind them that
// name any row of dout; before, after: the tokens around them.  A slab is J pieces of lanes * W columns side by side (J > 1: for
// single values, with 32 lanes), a thread takes W columns of each.  item[2 g], item[2 g + 1]: what group g's run holds of its
// first and last token (0 for the last one where the run holds one token only), so that the items' tokens ascend.  head, tail:
// where the parts go that other warps have to do with.
template <int W, int J> struct Items {
  unsigned key[J > 1 ? 2 : 64];
  float sum[64 * W * J];
};
template <class T, int W, int J>
__device__ __forceinline__ void warp_sums(const Sums &p, const T *dout, const uint2 *entry, int count, unsigned before, unsigned after, Items<W, J> &items, float *head,
                                          float *tail) {
  const unsigned none = p.vocab;
  const int lanes = J > 1 || blockIdx.y + 1 < gridDim.y ? 32 : p.lanes, groups = J > 1 ? 1 : 32 / lanes, width = lanes * W * J, column0 = blockIdx.y * 32 * W * J;
  const int lane = threadIdx.x & 31, group = lane / lanes, column = (lane - group * lanes) * W, c = column0 + column;
  const int each = (count + groups - 1) / groups, begin = min(group * each, count), end = group < groups && c < p.C ? min(begin + each, count) : begin;
  Columns<W> sum[J];
#pragma unroll
  for (int j = 0; j < J; ++j) sum[j].clear();
  unsigned now = begin < end ? entry[begin].x : none;
  bool atHead = true;
  const auto to_item = [&](int at) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int w = 0; w < W; ++w) items.sum[at * width + column + 32 * W * j + w] = sum[j].at(w);
    if (column == 0) items.key[at] = now;
  };
  const char *from = (const char *)(dout + c);
  for (int s = 0; s < each; s += SUM_ROWS) {
    __syncwarp(); // the groups part where their tokens change, and ask for their next rows together
    const int i = begin + s;
    if (i >= end) continue;
    Pack<T, W> v[SUM_ROWS][J];
#pragma unroll
    for (int u = 0; u < SUM_ROWS; ++u) {
      const T *row = (const T *)(from + (unsigned long long)entry[i + u].y * p.stride);
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (j == 0 || c + 32 * W * j < p.C) v[u][j] = load_pack<T, W>(row + 32 * W * j);
    }
    if (i + SUM_ROWS <= end && entry[i + SUM_ROWS - 1].x == now) { // one token all along
#pragma unroll
      for (int u = 0; u < SUM_ROWS; ++u)
#pragma unroll
        for (int j = 0; j < J; ++j) sum[j].add(v[u][j]);
      continue;
    }
#pragma unroll
    for (int u = 0; u < SUM_ROWS; ++u) {
      if (i + u < end) {
        const unsigned k = entry[i + u].x;
        if (k != now) {
          if (atHead) to_item(2 * group);
          else {
#pragma unroll
            for (int j = 0; j < J; ++j)
              if (j == 0 || c + 32 * W * j < p.C) write_row<W>(p, now, c + 32 * W * j, sum[j]);
          }
          atHead = false;
          now = k;
#pragma unroll
          for (int j = 0; j < J; ++j) sum[j].clear();
        }
#pragma unroll
        for (int j = 0; j < J; ++j) sum[j].add(v[u][j]);
      }
    }
  }
  if (group < groups) {
    to_item(2 * group + (atHead ? 0 : 1));
    if (atHead) {
#pragma unroll
      for (int j = 0; j < J; ++j) sum[j].clear();
      to_item(2 * group + 1);
    }
  }
  __syncwarp();
  for (int x = lane; x < width && column0 + x < p.C; x += 32) {
    Columns<1> total;
    total.clear();
    now = none;
    for (int j = 0; j <= 2 * groups; ++j) {
      const unsigned k = j < 2 * groups ? items.key[j] : none;
      if (k != now) {
        if (now == none) ;
        else if (now == before) head[column0 + x] = total.v;
        else if (now == after) tail[column0 + x] = total.v;
        else write_row<1>(p, now, column0 + x, total);
        now = k;
        total.clear();
      }
      if (k != none) total.v += items.sum[j * width + x];
    }
  }
}
// A token that begins in one tile and goes on in others has its parts added up, in two steps so that one on most of the rows
// does not keep a single CTA busy (one CTA for each token: 62 us for a third of 224 k rows on one token).  First 32 tiles (from a
// multiple of 32 on) that all begin with a token from further in front become one part, in the place of the first: the last of
// their warps adds them up, so that nothing is launched for it (224 k rows: 49.5 -> 45 us for the whole gradient).  Where there are
// 2048 tiles or fewer, the second step's CTA takes them by itself: faster where no token is hot (rows of 33 floats added on: 50 k rows 28 us against 33,
// 100 k 33 against 35, 160 k, 2500 tiles, 40 against 41), slower with a third of the rows on one (96 floats: 50 k rows 35 against 31, 100 k 47
// against 37, 160 k 60 against 39, 224 k 73 against 44).
__device__ __forceinline__ void join_group(const Sums &p, long long tile, unsigned key, int first, int columns) {
  const int lane = threadIdx.x & 31;
  const long long t0 = tile / 32 * 32, tiles = (p.n + p.tile - 1ll) / p.tile;
  if (t0 == 0 || t0 + 32 > tiles || p.entries[t0 * p.tile - 1].x != key) return;
  unsigned before = 0;
  __syncwarp();
  if (lane == 0) {
    __threadfence();
    before = atomicAdd(p.arrived + blockIdx.y * (tiles / 32) + tile / 32, 1u);
    __threadfence();
  }
  __syncwarp();
  if (__shfl_sync(~0u, before, 0) != 31) return;
  float *at = p.head + t0 * p.C + first;
  for (int c = lane; c < columns; c += 32) {
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 32; ++t) sum += __ldcg(at + (long long)t * p.C + c);
    at[c] = sum;
  }
}
// GROUPS: whether tiles are joined by 32 (the code for it, unused, costs narrow types registers: 50 k rows of 33 floats 28 -> 32 us).
template <class T, int W, int J, bool GROUPS> __global__ void __launch_bounds__(THREADS, 4) k_embedding_sums(const Sums p, const T *dout) {
  __shared__ uint2 entries[WARPS][MAX_TILE + SUM_ROWS];
  __shared__ Items<W, J> items[WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_prior_grids();
  dependents_may_launch();
  const long long tile = (long long)blockIdx.x * WARPS + warp, first = tile * p.tile;
  if (first >= p.n) return;
  uint2 *entry = entries[warp];
  const unsigned none = p.vocab;
  const int most = (int)min((long long)p.tile, p.n - first);
  const unsigned before = first > 0 ? p.entries[first - 1].x : none, next = first + most < p.n ? p.entries[first + most].x : none;
  uint2 e[MAX_TILE / 32];
#pragma unroll
  for (int r = 0; r < MAX_TILE / 32; ++r) e[r] = r * 32 + lane < most ? p.entries[first + r * 32 + lane] : make_uint2(none, 0u);
  int count = 0; // entries with a token: they come first
#pragma unroll
  for (int r = 0; r < MAX_TILE / 32; ++r) {
    if (r * 32 + lane < most) entry[r * 32 + lane] = e[r];
    count += __popc(__ballot_sync(~0u, e[r].x != none));
  }
  __syncwarp();
  if (lane == 0 && blockIdx.y == 0) p.ends[tile] = make_uint2(e[0].x, entry[most - 1].x);
  if (count == 0) return;
  const unsigned any = entry[count - 1].y;
  __syncwarp();
  if (lane < SUM_ROWS) entry[count + lane] = make_uint2(none, any);
  __syncwarp();
  warp_sums<T, W, J>(p, dout, entry, count, before, count == most ? next : none, items[warp], p.head + tile * p.C, p.tail + tile * p.C);
  if constexpr (GROUPS) {
    const unsigned key = entry[0].x; // (all the tile's, or the last tile's of 32: the others cannot be part of 32 that begin alike)
    if (key == before && (entry[count - 1].x == key || (tile & 31) == 31)) {
      const int column0 = blockIdx.y * 32 * W * J;
      join_group(p, tile, key, column0, min(p.C - column0, 32 * W * J));
    }
  }
}
// The whole gradient of at most SMALL rows in one launch (203 rows of 32: 5.5 us on the GPU, where the launches of the
// general form take 22 us): the first CTAs (one a slab) sort the entries in shared memory and add them up; the others write the
// zeros of the rows that no token names, each for a range of `range` rows.
constexpr int SMALL_ROUNDS = 4, SMALL = THREADS * SMALL_ROUNDS, SMALL_DIGIT = 8, MOST_RANGE = 16384;
template <class T, int W, int J>
__global__ void __launch_bounds__(THREADS) k_embedding_backward_small(const Sums p, const T *dout, const int *tokens, int bits, int range, int *errors) {
  __shared__ uint2 entries[2][SMALL + SUM_ROWS];
  __shared__ union {
    unsigned present[MOST_RANGE / 32];             // (the CTAs that write zeros)
    unsigned short count[WARPS << SMALL_DIGIT];    // (while sorting)
    Items<W, J> items[WARPS];
  } sh;
  __shared__ unsigned warpSum[WARPS], all;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_prior_grids();
  dependents_may_launch();
  if (blockIdx.x > 0) {
    if (blockIdx.y > 0) return;
    const int first = (int)(blockIdx.x - 1) * range, rows = min(range, p.vocab - first);
    for (int i = threadIdx.x; i < (rows + 31) / 32; i += THREADS) sh.present[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.n; i += THREADS) {
      const int t = tokens[i];
      if (t >= first && t - first < rows) atomicOr(&sh.present[(t - first) >> 5], 1u << ((t - first) & 31));
    }
    __syncthreads();
    for (int r = warp; r < rows; r += WARPS)
      if (!(sh.present[r >> 5] >> (r & 31) & 1)) clear_floats(p.dtable + (long long)(first + r) * p.C, p.C, lane, 32);
    return;
  }
  uint2 *now = entries[0], *other = entries[1];
  const unsigned none = p.vocab;
  if (threadIdx.x == 0) all = 0;
  __syncthreads();
  int named = 0; // entries with a token: they come first in the end
  for (int i = threadIdx.x; i < p.n; i += THREADS) {
    const int t = tokens[i];
    if (t >= p.vocab && errors && blockIdx.y == 0) atomicOr(errors, SCN_DEV_ERR_KEY);
    now[i] = make_uint2(key_of(t, p.vocab), i);
    named += now[i].x != none;
  }
  named = __reduce_add_sync(~0u, named);
  if (lane == 0) atomicAdd(&all, (unsigned)named);
  __syncthreads();
  const int count = (int)all;
  if (count == 0) return;
  const int passes = (bits + SMALL_DIGIT - 1) / SMALL_DIGIT;
  for (int k = 0; k < passes; ++k) {
    unsigned key[SMALL_ROUNDS], row[SMALL_ROUNDS], place[SMALL_ROUNDS];
#pragma unroll
    for (int r = 0; r < SMALL_ROUNDS; ++r) {
      const int j = (warp * SMALL_ROUNDS + r) * 32 + lane;
      const uint2 e = j < p.n ? now[j] : make_uint2(0u, 0u);
      key[r] = e.x; row[r] = e.y;
    }
    places_by_digit<SMALL_ROUNDS, SMALL_DIGIT>(key, p.n, k * SMALL_DIGIT, sh.count, warpSum, place, [](int, unsigned) {});
#pragma unroll
    for (int r = 0; r < SMALL_ROUNDS; ++r)
      if ((warp * SMALL_ROUNDS + r) * 32 + lane < p.n) other[place[r]] = make_uint2(key[r], row[r]);
    __syncthreads();
    uint2 *t = now; now = other; other = t;
  }
  const unsigned any = now[count - 1].y;
  __syncthreads();
  if (threadIdx.x < SUM_ROWS) now[count + threadIdx.x] = make_uint2(none, any);
  __syncthreads();
  const int tile = (count + WARPS - 1) / WARPS, first = min(warp * tile, count), end = min(first + tile, count), column0 = blockIdx.y * 32 * W * J;
  const int width = (J > 1 || blockIdx.y + 1 < gridDim.y ? 32 : p.lanes) * W * J;
  const auto key_at = [&](int i) { return i >= 0 && i < count ? now[i].x : none; };
  if (first < end) // (a warp's head and tail take the places of its first two items, read by then)
    warp_sums<T, W, J>(p, dout, now + first, end - first, key_at(first - 1), key_at(end), sh.items[warp], sh.items[warp].sum - column0,
                    sh.items[warp].sum + width - column0);
  __syncthreads();
  if (first >= end) return;
  const unsigned last = now[end - 1].x; // as in k_embedding_join
  if (key_at(end) != last || key_at(first - 1) == last) return;
  for (int x = lane; x < width && column0 + x < p.C; x += 32) {
    Columns<1> sum;
    sum.v = sh.items[warp].sum[width + x];
    for (int w = warp + 1; w < WARPS && key_at(w * tile) == last; ++w) sum.v += sh.items[w].sum[x];
    write_row<1>(p, last, column0 + x, sum);
  }
}
// Then a warp looks at one tile after the other and adds up a token that begins in it and goes on in fewer than 32 more; a longer
// one is left for the whole CTA, whose warps take every JOIN_WARPS-th part and add up what they have.
constexpr int JOIN_THREADS = 256, JOIN_WARPS = JOIN_THREADS / 32, JOIN_COLUMNS = 4; // columns of a thread at once
__global__ void __launch_bounds__(JOIN_THREADS) k_embedding_join(const Sums p, int tiles) {
  __shared__ float share[JOIN_WARPS][32 * JOIN_COLUMNS];
  __shared__ int longOnes[JOIN_WARPS], found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned none = p.vocab;
  wait_for_prior_grids();
  dependents_may_launch();
  const auto first_token = [&](long long t) { return t < tiles ? p.ends[t].x : none; };
  // columns c, c + 32, ... of parts begin, begin + step, ...: added to sum
  const auto add_parts = [&](float (&sum)[JOIN_COLUMNS], int c, int begin, int end, int step, auto row_of) {
#pragma unroll 4
    for (int i = begin; i < end; i += step) {
      const float *part = row_of(i) + c;
#pragma unroll
      for (int j = 0; j < JOIN_COLUMNS; ++j) sum[j] += c + 32 * j < p.C ? part[32 * j] : 0.f;
    }
  };
  for (int base = blockIdx.x * JOIN_WARPS; base < tiles; base += gridDim.x * JOIN_WARPS) {
    const int b = base + warp;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    if (b + 1 < tiles) {
      const unsigned k = p.ends[b].y, before = b > 0 ? p.ends[b - 1].y : none;
      const unsigned follows = first_token((long long)b + 1 + lane); // the tokens that the next tiles begin with
      const unsigned same = __ballot_sync(~0u, follows == k);
      if (k != none && (same & 1) && before != k) {
        if (same == ~0u) {
          if (lane == 0) longOnes[atomicAdd(&found, 1)] = b;
        } else {
          for (int c = lane; c - lane < p.C; c += 32 * JOIN_COLUMNS) {
            float sum[JOIN_COLUMNS] = {};
            add_parts(sum, c, 0, __ffs(~same), 1, [&](int i) { return (i == 0 ? p.tail : p.head) + (long long)(b + i) * p.C; });
#pragma unroll
            for (int j = 0; j < JOIN_COLUMNS; ++j)
              if (c + 32 * j < p.C) write_row<1>(p, k, c + 32 * j, Columns<1>{sum[j]});
          }
        }
      }
    }
    __syncthreads();
    for (int l = 0; l < found; ++l) {
      const int t0 = longOnes[l];
      const unsigned k = p.ends[t0].y;
      int last = t0 + 1, beyond = tiles; // the last tile that begins with k: `last` does, `beyond` does not
      while (beyond - last > 1) {
        const int step = (beyond - last + JOIN_THREADS - 1) / JOIN_THREADS;
        const int with = __syncthreads_count(first_token((long long)last + (long long)threadIdx.x * step) == k);
        last += (with - 1) * step;
        beyond = (int)min((long long)beyond, (long long)last + step);
      }
      ++last;
      // the parts: t0's tail, single tiles, 32 tiles at a time where they have been joined, single tiles
      const int from = min(last, p.arrived ? (t0 + 32) / 32 * 32 : last), to = max(from, last / 32 * 32);
      const int singles = from - t0, both = singles + (to - from) / 32, parts = both + max(0, last - to);
      const auto row_of = [&](int i) {
        const int t = i < singles ? t0 + i : i < both ? from + 32 * (i - singles) : to + i - both;
        return (i == 0 ? p.tail : p.head) + (long long)t * p.C;
      };
      for (int c = lane; c - lane < p.C; c += 32 * JOIN_COLUMNS) {
        float sum[JOIN_COLUMNS] = {};
        add_parts(sum, c, warp, parts, JOIN_WARPS, row_of);
#pragma unroll
        for (int j = 0; j < JOIN_COLUMNS; ++j) share[warp][32 * j + lane] = sum[j];
        __syncthreads();
        const int column = c - lane + threadIdx.x;
        if (threadIdx.x < 32 * JOIN_COLUMNS && column < p.C) {
          Columns<1> total;
          total.clear();
#pragma unroll
          for (int w = 0; w < JOIN_WARPS; ++w) total.v += share[w][threadIdx.x];
          write_row<1>(p, k, column, total);
        }
        __syncthreads();
      }
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
// Entries a warp sums: MAX_TILE, fewer (a power of two) where that would leave SMs with less than 16 warps each.  us with 64, 128, 256: 50 k rows of
// 33 floats 28, 32, 44; 224 k of 96 44, 63, 70; 700 k of 96 94, 91, 83; 3.4 M 16-bit rows of 64 207, 189, 182.
int sum_tile(long long n) {
  int tile = MAX_TILE;
  while (tile > MIN_TILE && n < 16ll * 148 * tile) tile /= 2;
  return tile;
}

constexpr int LARGE_ROUNDS = 8, LEAST_DIGIT = 6;
// Up to so many tiles every scatter adds the tiles' counts up itself, which saves a launch: 5 k rows 23 us, 28 with k_radix_scan; 98 tiles 47 us with
// it, 52 without.
constexpr int FEW_TILES = 64;
// Large tiles: longer runs of a digit; small ones: work for every SM.  us with small and large ones: 100 k rows 47, 49; 1 M 87, 89; 1.5 M 114, 113;
// 3.4 M 195, 182.
int sort_rounds(long long n) { return n > (1 << 20) ? LARGE_ROUNDS : 4; }
struct SortPlan {
  int tiles, passes, bits, digit;            // digit: bits a pass
  int sumTile;
  long long sumTiles;
  size_t array, counts, totals, parts, ends, arrived, total; // bytes
};
SortPlan plan_sort(long long n, int vocab, int C) {
  SortPlan p;
  p.bits = 1;
  while (p.bits < 31 && ((long long)vocab >> p.bits) > 0) ++p.bits; // keys 0..vocab
  p.passes = (p.bits + MAX_DIGIT - 1) / MAX_DIGIT;
  p.digit = std::max(LEAST_DIGIT, (p.bits + p.passes - 1) / p.passes);
  const long long tile = THREADS * sort_rounds(n);
  p.tiles = (int)((n + tile - 1) / tile);
  p.array = align_up(sizeof(uint2) * (size_t)n, 256);
  p.counts = align_up(sizeof(unsigned) * ((size_t)p.tiles << p.digit), 256);
  p.totals = align_up(sizeof(unsigned) << p.digit, 256);
  p.sumTile = sum_tile(n);
  p.sumTiles = (n + p.sumTile - 1) / p.sumTile;
  p.parts = align_up(sizeof(float) * (size_t)p.sumTiles * (size_t)C, 256); // of each tile's first and last token
  p.ends = align_up(sizeof(uint2) * (size_t)p.sumTiles, 256);
  p.arrived = align_up(sizeof(unsigned) * (size_t)(p.sumTiles / 32) * (size_t)((C + 63) / 64), 256);
  p.total = 2 * p.array + p.counts + p.totals + 2 * p.parts + p.ends + p.arrived + 256;
  return p;
}
template <int ROUNDS> int sort_pass(const Pass &p, cudaStream_t s) {
  const int digits = 1 << p.bits, clearing = p.clear ? 2 * sm_count() : 0;
  SCN_CUDA_TRY(launch_dependent(k_radix_count<ROUNDS>, dim3(p.tiles + clearing), dim3(THREADS), sizeof(unsigned) * digits, s, p));
  SCN_LAUNCH_CHECK("k_radix_count");
  const int each = (p.tiles + SCAN_RUNS - 1) / SCAN_RUNS;
  const auto scan = each <= 2 ? k_radix_scan<2> : each <= 8 ? k_radix_scan<8> : each <= 24 ? k_radix_scan<24> : k_radix_scan<0>;
  if (p.totals) SCN_CUDA_TRY(launch_dependent(scan, dim3(digits / SCAN_DIGITS), dim3(SCAN_THREADS), 0, s, p));
  if (p.totals) SCN_LAUNCH_CHECK("k_radix_scan");
  switch (p.bits) {
  case 6: SCN_CUDA_TRY(launch_dependent(k_radix_scatter<ROUNDS, 6>, dim3(p.tiles), dim3(THREADS), 0, s, p)); break;
  case 7: SCN_CUDA_TRY(launch_dependent(k_radix_scatter<ROUNDS, 7>, dim3(p.tiles), dim3(THREADS), 0, s, p)); break;
  case 8: SCN_CUDA_TRY(launch_dependent(k_radix_scatter<ROUNDS, 8>, dim3(p.tiles), dim3(THREADS), 0, s, p)); break;
  default: SCN_CUDA_TRY(launch_dependent(k_radix_scatter<ROUNDS, 9>, dim3(p.tiles), dim3(THREADS), 0, s, p)); break;
  }
  SCN_LAUNCH_CHECK("k_radix_scatter");
  return SCN_OK;
}

} // namespace
} // namespace scn

using namespace scn;
static constexpr int MOST_COLUMNS = 1 << 28; // (a row's bytes fit 32 bits)
static constexpr int MOST_GRADIENT_COLUMNS = 65535 * 64; // (slabs of at least 64 columns are a grid's second dimension)

extern "C" int scn_embedding_forward(const void *d_table, int table_type, int vocab, int C, const int *d_tokens, long long n, float scale, void *d_out,
                                     int out_type, long long out_stride, int *d_errors, scn_stream_t stream) {
  clear_error();
  if (vocab < 1 || C < 1 || C > MOST_COLUMNS || n < 0 || n > 0x7fffffffll) return fail(SCN_ERR_INVALID, "bad embedding sizes");
  if (out_stride < C) return fail(SCN_ERR_INVALID, "embedding: the output's row stride is below the number of features");
  if (!type_known(table_type) || !type_known(out_type)) return fail(SCN_ERR_INVALID, "embedding: unknown type");
  if (out_stride > 0xffffffffll / type_bytes(out_type)) return fail(SCN_ERR_UNSUPPORTED, "embedding: the output's rows lie 4 GiB apart or more");
  if (n == 0) return SCN_OK;
  if (!d_table || !d_tokens || !d_out) return fail(SCN_ERR_INVALID, "null pointer");
  if (((uintptr_t)d_table & (type_bytes(table_type) - 1)) | ((uintptr_t)d_out & (type_bytes(out_type) - 1)) | (((uintptr_t)d_tokens | (uintptr_t)d_errors) & 3))
    return fail(SCN_ERR_INVALID, "embedding: misaligned pointer");
  const Lookup p = {(const char *)d_table, d_tokens, (char *)d_out, (unsigned)n, (unsigned)(out_stride * type_bytes(out_type)), (unsigned)C * type_bytes(table_type), vocab, C, scale, d_errors};
  SCN_DISPATCH_TYPE(table_type, T, SCN_DISPATCH_TYPE(out_type, O, SCN_CUDA_TRY((launch_forward<T, O>(p, (cudaStream_t)stream)))));
  SCN_LAUNCH_CHECK("k_embedding_forward");
  return SCN_OK;
}

extern "C" size_t scn_embedding_backward_workspace_bytes(long long n, int vocab, int C) {
  if (n < 0 || n > 0x7fff0000ll || vocab < 1 || C < 1 || C > MOST_GRADIENT_COLUMNS) return 0;
  return plan_sort(n, vocab, C).total;
}

extern "C" int scn_embedding_backward(const int *d_tokens, long long n, const void *d_dout, int dout_type, long long dout_stride, int vocab, int C,
                                      float scale, int accumulate, float *d_dtable, int *d_errors, void *d_workspace, size_t workspace_bytes,
                                      scn_stream_t stream) {
  clear_error();
  if (vocab < 1 || C < 1 || C > MOST_COLUMNS || n < 0 || n > 0x7fff0000ll) return fail(SCN_ERR_INVALID, "bad embedding sizes");
  if (dout_stride < C) return fail(SCN_ERR_INVALID, "embedding: the gradient's row stride is below the number of features");
  if (!type_known(dout_type)) return fail(SCN_ERR_INVALID, "embedding: unknown type");
  if (C > MOST_GRADIENT_COLUMNS) return fail(SCN_ERR_UNSUPPORTED, "embedding: a gradient has at most 4194240 features");
  if (dout_stride > 0xffffffffll / type_bytes(dout_type)) return fail(SCN_ERR_UNSUPPORTED, "embedding: the gradient's rows lie 4 GiB apart or more");
  if (!d_dtable || !d_workspace) return fail(SCN_ERR_INVALID, "null pointer");
  if (n && (!d_tokens || !d_dout)) return fail(SCN_ERR_INVALID, "null pointer");
  if (((uintptr_t)d_dout & (type_bytes(dout_type) - 1)) | (((uintptr_t)d_tokens | (uintptr_t)d_dtable | (uintptr_t)d_errors) & 3))
    return fail(SCN_ERR_INVALID, "embedding: misaligned pointer");
  const SortPlan sp = plan_sort(n, vocab, C);
  if (workspace_bytes < sp.total) return fail(SCN_ERR_WORKSPACE, "workspace smaller than scn_embedding_backward_workspace_bytes()");
  if ((uintptr_t)d_workspace & 15) return fail(SCN_ERR_INVALID, "embedding: the workspace must be 16-byte aligned");
  cudaStream_t s = (cudaStream_t)stream;
  if (n == 0) {
    if (!accumulate) SCN_CUDA_TRY(cudaMemsetAsync(d_dtable, 0, sizeof(float) * (size_t)vocab * C, s));
    return SCN_OK;
  }
  char *w = (char *)d_workspace;
  const int W = pack_width(dout_type, d_dout, dout_stride, d_dtable, C), vectors = C / W;
  const int J = W > 1 || C <= 32 ? 1 : C <= 64 ? 2 : 4, slabs = (vectors + 32 * J - 1) / (32 * J); // (see warp_sums)
  Sums q = {};
  q.n = (int)n; q.vocab = vocab; q.C = C; q.stride = (unsigned)(dout_stride * type_bytes(dout_type));
  q.lanes = J > 1 ? 32 : vectors - (slabs - 1) * 32;
  q.tile = sp.sumTile;
  q.scale = scale; q.accumulate = accumulate; q.dtable = d_dtable;
  q.head = (float *)(w + 2 * sp.array + sp.counts + sp.totals);
  q.tail = (float *)(w + 2 * sp.array + sp.counts + sp.totals + sp.parts);
  q.ends = (uint2 *)(w + 2 * sp.array + sp.counts + sp.totals + 2 * sp.parts);
  // F(T, W, J) for dout's type, the width and the pieces
#define SCN_SUMS(F, ...)                                                                                              \
  SCN_DISPATCH_TYPE(dout_type, T, {                                                                                   \
    constexpr int MOST = 16 / (int)sizeof(T);                                                                         \
    if (W == MOST) SCN_CUDA_TRY(launch_dependent(F(T, MOST, 1), __VA_ARGS__));                                        \
    else if (W == MOST / 2) SCN_CUDA_TRY(launch_dependent(F(T, MOST / 2, 1), __VA_ARGS__));                           \
    else if (W == 2) SCN_CUDA_TRY(launch_dependent(F(T, 2, 1), __VA_ARGS__));                                         \
    else if (J == 1) SCN_CUDA_TRY(launch_dependent(F(T, 1, 1), __VA_ARGS__));                                         \
    else if (J == 2) SCN_CUDA_TRY(launch_dependent(F(T, 1, 2), __VA_ARGS__));                                         \
    else SCN_CUDA_TRY(launch_dependent(F(T, 1, 4), __VA_ARGS__));                                                     \
  })
  if (n <= SMALL) {
    const long long share = (vocab - 1ll) / (4 * sm_count()) + 1; // (in 64 bits: vocab goes up to 2^31 - 1)
    const int range = (int)std::max(32ll, std::min((long long)MOST_RANGE, share)), clearing = accumulate ? 0 : (int)((vocab - 1ll) / range + 1);
#define SCN_SMALL(T, W, J) (k_embedding_backward_small<T, W, J>)
    SCN_SUMS(SCN_SMALL, dim3(1 + clearing, slabs), dim3(THREADS), 0, s, q, (const T *)d_dout, d_tokens, sp.bits, range, d_errors);
    SCN_LAUNCH_CHECK("k_embedding_backward_small");
    return SCN_OK;
  }
  uint2 *const array[2] = {(uint2 *)w, (uint2 *)(w + sp.array)};
  Pass p = {};
  p.n = (int)n; p.vocab = vocab; p.tiles = sp.tiles; p.bits = sp.digit;
  p.counts = (unsigned *)(w + 2 * sp.array);
  p.totals = sp.tiles > FEW_TILES ? (unsigned *)(w + 2 * sp.array + sp.counts) : nullptr;
  p.errors = d_errors;
  const int tiles = (int)sp.sumTiles;
  if (tiles > 2048) q.arrived = (unsigned *)(w + 2 * sp.array + sp.counts + sp.totals + 2 * sp.parts + sp.ends);
  for (int k = 0; k < sp.passes; ++k) {
    p.tokens = k == 0 ? d_tokens : nullptr;
    p.in = array[(k + 1) & 1];
    p.out = array[k & 1];
    p.shift = k * sp.digit;
    p.clear = k == 0 && !accumulate ? d_dtable : nullptr;
    p.clearN = (long long)vocab * C;
    p.arrived = q.arrived;
    p.arrivedN = k == 0 && q.arrived ? (long long)tiles / 32 * slabs : 0;
    const int rc = sort_rounds(n) == 4 ? sort_pass<4>(p, s) : sort_pass<LARGE_ROUNDS>(p, s);
    if (rc != SCN_OK) return rc;
  }
  q.entries = p.out;
#define SCN_TILES(T, W, J) (q.arrived ? k_embedding_sums<T, W, J, true> : k_embedding_sums<T, W, J, false>)
  SCN_SUMS(SCN_TILES, dim3((tiles + WARPS - 1) / WARPS, slabs), dim3(THREADS), 0, s, q, (const T *)d_dout);
#undef SCN_SUMS
#undef SCN_SMALL
#undef SCN_TILES
  SCN_LAUNCH_CHECK("k_embedding_sums");
  if (tiles > 1) {
    SCN_CUDA_TRY(launch_dependent(k_embedding_join, dim3(std::min((tiles + JOIN_WARPS - 1) / JOIN_WARPS, 8 * sm_count())), dim3(JOIN_THREADS), 0, s, q, tiles));
    SCN_LAUNCH_CHECK("k_embedding_join");
  }
  return SCN_OK;
}
