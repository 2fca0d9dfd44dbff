// Token embedding with scaling, and its gradient by sorted tokens, gfx950.
//
//   out[i]    = scale * W[t_i]
//   dW[v]     = scale * sum over the i with t_i = v of dout[i]
//               (zero for v = padding_idx, and for every v not in t)
//
// Both are bound by memory. The forward pass reads and writes N rows. The
// gradient reads N rows and writes V; adding rows to dW as they come would
// take atomics, whose order changes the sums from run to run, so the
// tokens are sorted first, stably, and each run of one token is added up
// in 32 bits, in an order that its positions alone decide (one after the
// other, or by parts where it is long), and rounded once.
//
// Up to 1024 tokens, owned_rows_kernel does all of it in one launch, unless
// they are more than two for each row of the table. Otherwise:
//
//   1. sort. Up to 16384 tokens one block sorts them in LDS (a stable
//      radix sort, at most 8 bits a pass), while the launch's other blocks
//      clear dW: 16381 tokens take 27 us, and clearing 60001 x 2048 16-bit
//      values 37, so that the sort costs nothing. More tokens take
//      histogram, scan and scatter launches for each digit.
//   2. sum_runs_kernel: each wave takes a chunk of the sorted positions and
//      64 vectors of columns, and writes the runs that lie within the
//      chunk; of a run that goes on beyond it, what it has is left in a
//      workspace. So the work is even however often a token occurs.
//   3. join_runs_kernel adds up the pieces of such runs, in order.
//
// Measured, 16381 tokens and 60001 x 2048 bf16: gather 25 us (5.3 TB/s),
// sort and clearing 37 (6.6 TB/s of stores), sums 23, join 5. 700 tokens and
// 10000 x 1500 float32: gather 4 us, owned rows 13 (60 MB written), against
// 19 by way of the sort. What bounds the large case is the dense gradient's
// 246 MB; the small ones are bound by launches and torch's autograd engine.
//
// A token outside [0, V) is never used as an index: its output is NaN, and
// it has no gradient.
#include <hip/hip_runtime.h>

#include "lm_common.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <vector>

namespace mgx {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ long token_at(const void* p, bool wide, long i) {
  return wide ? static_cast<const long*>(p)[i]
              : static_cast<long>(static_cast<const int*>(p)[i]);
}

// The first `cols` elements of a vector; the rest is zero.
template <typename T, bool PAST = false>
__device__ __forceinline__ u32x4 load_cols(const T* p, int cols) {
  constexpr int V = Elem<T>::kVec;
  if (cols >= V) return PAST ? load16_past(p) : load16(p);
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = j < cols ? Elem<T>::up(p[j]) : 0.f;
  return Elem<T>::pack(f);
}
template <typename T>
__device__ __forceinline__ void store_cols(T* p, int cols, const float* f) {
  constexpr int V = Elem<T>::kVec;
  if (cols >= V) {
    store16(p, Elem<T>::pack(f));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < cols) p[j] = Elem<T>::down(f[j]);
  }
}

// ------------------------------------------------------------- forward ---
// The output as rows of `vecs` vectors, the last of which may be short;
// each thread takes U vectors that lie 256 apart.
template <typename T, int U>
__global__ __launch_bounds__(kThreads) void gather_rows_kernel(
    const void* __restrict__ tokens, bool wide, long n,
    const T* __restrict__ weight, long row_stride, long vocab, int dim,
    unsigned vecs, float scale, T* __restrict__ out) {
  constexpr int V = Elem<T>::kVec;
  const long first = (long)blockIdx.x * (kThreads * U);
  const long row0 = first / vecs;
  const unsigned off0 = (unsigned)(first - row0 * vecs);
  u32x4 f[U];
  long row[U];
  int col[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned at = off0 + u * kThreads + threadIdx.x;
    row[u] = row0 + at / vecs;
    col[u] = (int)(at % vecs) * V;
    if (row[u] < n) {
      const long t = token_at(tokens, wide, row[u]);
      if (t >= 0 && t < vocab) {
        f[u] = load_cols(weight + t * row_stride + col[u], dim - col[u]);
      } else {
        float nan[V];
#pragma unroll
        for (int j = 0; j < V; ++j) nan[j] = __builtin_nanf("");
        f[u] = Elem<T>::pack(nan);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (row[u] < n) {
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = Elem<T>::get(f[u], j) * scale;
      store_cols(out + row[u] * dim + col[u], dim - col[u], y);
    }
}

// ---------------------------------------------------------------- sort ---
constexpr int kDigits = 256;

// Tokens that have no gradient (padding, outside the table) sort last.
__device__ __forceinline__ uint32_t sort_key(const void* tokens, bool wide,
                                             long i, long vocab,
                                             long padding) {
  const long t = token_at(tokens, wide, i);
  return t >= 0 && t < vocab && t != padding ? (uint32_t)t : (uint32_t)vocab;
}

__device__ __forceinline__ void wave_fence() {
  // orders one wave's LDS accesses, which the hardware keeps in order
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// For each of IPT items (item j of a lane stands 64 after item j - 1 in the
// wave's share) its rank among the wave's items of the same digit that
// stand before it; counts[] becomes the wave's histogram.
template <typename I, int IPT>
__device__ __forceinline__ void wave_ranks(const I (&item)[IPT], int shift,
                                           int bits, int* counts,
                                           int (&rank)[IPT]) {
  const unsigned long long below = (1ull << (threadIdx.x & 63)) - 1;
  const unsigned mask = (1u << bits) - 1;
#pragma unroll
  for (int j = 0; j < IPT; ++j) {
    const unsigned d = (unsigned)(item[j] >> shift) & mask;
    unsigned long long same = ~0ull;
    for (int b = 0; b < bits; ++b) {
      const bool one = (d >> b) & 1;
      const unsigned long long ones = __ballot(one);
      same &= one ? ones : ~ones;
    }
    const int before = __popcll(same & below);
    const int base = counts[d];
    wave_fence();
    rank[j] = base + before;
    if (before == 0) counts[d] = base + __popcll(same);
    wave_fence();
  }
}

// Exclusive sums over 256 threads; `lds` holds 4 ints.
__device__ __forceinline__ int exclusive_256(int x, int* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(s, off, 64);
    if (lane >= off) s += o;
  }
  if (wave < 4 && lane == 63) lds[wave] = s;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < 4; ++w) before += w < wave ? lds[w] : 0;
  return before + s - x;
}

// dW cleared by blocks `block` of `blocks`, 1024 threads each.
__device__ __forceinline__ void clear_bytes(char* p, long bytes, long block,
                                            long blocks) {
  const long whole = bytes & ~15L;
  const long step = blocks * blockDim.x * 16;
  for (long i = (block * blockDim.x + threadIdx.x) * 16; i < whole; i += step)
    store16(p + i, u32x4{0, 0, 0, 0});
  if (block == 0 && whole + (long)threadIdx.x < bytes)
    p[whole + threadIdx.x] = 0;
}

// Block 0 sorts up to 1024 * IPT tokens; the others clear dW. An item is
// the key above the position, in one word of `I`; the words behind the
// last token are all ones and stay last in every pass.
template <typename I, int IPT>
__global__ __launch_bounds__(1024) void sort_and_clear_kernel(
    const void* __restrict__ tokens, bool wide, int n, long vocab,
    long padding, int pos_bits, int key_bits, uint32_t* __restrict__ keys,
    uint32_t* __restrict__ positions, char* __restrict__ grad, long bytes) {
  if (blockIdx.x != 0) {
    clear_bytes(grad, bytes, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  constexpr int kWaves = 16;
  extern __shared__ __align__(16) char lds[];
  I* items = reinterpret_cast<I*>(lds);
  int* counts = reinterpret_cast<int*>(lds + sizeof(I) * 1024 * IPT);
  int* start = counts + kWaves * kDigits;
  int* sums = start + kDigits;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int mine = wave * 64 * IPT + lane;
  I item[IPT];
#pragma unroll
  for (int j = 0; j < IPT; ++j) {
    const int i = mine + 64 * j;
    item[j] = i < n
        ? ((I)sort_key(tokens, wide, i, vocab, padding) << pos_bits) | (I)i
        : ~(I)0;
  }
  const int passes = (key_bits + 7) / 8;
  const int width = (key_bits + passes - 1) / passes;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pos_bits + pass * width;
    for (int i = tid; i < kWaves * kDigits; i += 1024) counts[i] = 0;
    __syncthreads();
    int rank[IPT];
    wave_ranks<I, IPT>(item, shift, width, counts + wave * kDigits, rank);
    __syncthreads();
    int total = 0;
    if (tid < kDigits)
      for (int w = 0; w < kWaves; ++w) {
        const int c = counts[w * kDigits + tid];
        counts[w * kDigits + tid] = total;
        total += c;
      }
    const int before = exclusive_256(total, sums);
    if (tid < kDigits) start[tid] = before;
    __syncthreads();
    const unsigned mask = (1u << width) - 1;
#pragma unroll
    for (int j = 0; j < IPT; ++j) {
      const unsigned d = (unsigned)(item[j] >> shift) & mask;
      items[start[d] + counts[wave * kDigits + d] + rank[j]] = item[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < IPT; ++j) item[j] = items[mine + 64 * j];
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < IPT; ++j) {
    const int i = mine + 64 * j;
    if (i < n) {
      keys[i] = (uint32_t)(item[j] >> pos_bits);
      positions[i] = (uint32_t)(item[j] & (((I)1 << pos_bits) - 1));
    }
  }
}

// More tokens: for each digit of 8 bits or less, counts by tile, their
// exclusive sums for each digit over the tiles, and a stable scatter. A
// pass over 131072 tokens takes 20 us with dW's clearing and 18 without.
constexpr int kTileItems = 8;
constexpr int kTile = kThreads * kTileItems;

struct SortIn {            // the tokens, or what the last pass wrote
  const void* tokens;
  bool wide;
  long vocab, padding;
  const uint32_t* keys;
  const uint32_t* positions;
};

__device__ __forceinline__ uint32_t key_in(const SortIn& in, long i) {
  return in.keys != nullptr
      ? in.keys[i]
      : sort_key(in.tokens, in.wide, i, in.vocab, in.padding);
}

// Blocks behind the tiles clear dW (in the first pass).
__global__ __launch_bounds__(kThreads) void tile_counts_kernel(
    SortIn in, long n, int tiles, int shift, int bits,
    int* __restrict__ counts, char* __restrict__ grad, long bytes) {
  if ((int)blockIdx.x >= tiles) {
    clear_bytes(grad, bytes, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  __shared__ int mine[kDigits];
  mine[threadIdx.x] = 0;
  __syncthreads();
  const long from = (long)blockIdx.x * kTile;
  const unsigned mask = (1u << bits) - 1;
#pragma unroll 4
  for (int j = 0; j < kTileItems; ++j) {
    const long i = from + j * kThreads + threadIdx.x;
    if (i < n) atomicAdd(&mine[(key_in(in, i) >> shift) & mask], 1);
  }
  __syncthreads();
  counts[(long)threadIdx.x * tiles + blockIdx.x] = mine[threadIdx.x];
}

// Block d: the exclusive sums of digit d's counts over the tiles, and their
// total.
__global__ __launch_bounds__(kThreads) void scan_counts_kernel(
    int* __restrict__ counts, int tiles, int* __restrict__ totals) {
  __shared__ int sums[4];
  __shared__ int last;
  int* __restrict__ mine = counts + (long)blockIdx.x * tiles;
  int before = 0;
  for (int from = 0; from < tiles; from += kThreads) {
    const int i = from + threadIdx.x;
    const int c = i < tiles ? mine[i] : 0;
    const int at = before + exclusive_256(c, sums);
    if (i < tiles) mine[i] = at;
    if (threadIdx.x == kThreads - 1) last = at + c;
    __syncthreads();
    before = last;
    __syncthreads();                   // sums and last are free again
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

__global__ __launch_bounds__(kThreads) void tile_scatter_kernel(
    SortIn in, long n, int tiles, int shift, int bits,
    const int* __restrict__ counts, const int* __restrict__ totals,
    uint32_t* __restrict__ keys, uint32_t* __restrict__ positions) {
  constexpr int kWaves = kThreads / 64;
  __shared__ int mine[kWaves * kDigits];
  __shared__ int sums[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < kWaves * kDigits; i += kThreads) mine[i] = 0;
  __syncthreads();
  const long from =
      (long)blockIdx.x * kTile + wave * 64 * kTileItems + lane;
  uint32_t item[kTileItems];
#pragma unroll
  for (int j = 0; j < kTileItems; ++j) {
    const long i = from + 64 * j;
    item[j] = i < n ? key_in(in, i) : ~0u;   // last of the last tile
  }
  int rank[kTileItems];
  wave_ranks<uint32_t, kTileItems>(item, shift, bits, mine + wave * kDigits,
                                   rank);
  // what stands before this tile's share of digit threadIdx.x: the lower
  // digits, and the same digit in the tiles before (the sum's barrier also
  // orders the ranks)
  int at = exclusive_256(totals[threadIdx.x], sums) +
      counts[(long)threadIdx.x * tiles + blockIdx.x];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int c = mine[w * kDigits + threadIdx.x];
    mine[w * kDigits + threadIdx.x] = at;
    at += c;
  }
  __syncthreads();
  const unsigned mask = (1u << bits) - 1;
#pragma unroll
  for (int j = 0; j < kTileItems; ++j) {
    const long i = from + 64 * j;
    if (i < n) {
      const unsigned d = (item[j] >> shift) & mask;
      const long to = mine[wave * kDigits + d] + rank[j];
      keys[to] = item[j];
      positions[to] = in.positions != nullptr ? in.positions[i] : (uint32_t)i;
    }
  }
}

// ---------------------------------------------------------------- sums ---
// Few tokens: one launch, no sort. A block owns kOwned rows of dW, far
// apart (frequent tokens are often neighbours), and 64 vectors of columns;
// it looks through all the tokens for those rows, keeping the order of
// their positions, and writes each row's sum, or zeros. Each wave takes the
// rows that are its own; a row with many tokens is taken by the whole
// block, a quarter of the positions in each wave.
constexpr int kOwned = 16;
constexpr int kOwnedTokens = 1024;
constexpr int kMany = 16;

template <typename T>
__global__ __launch_bounds__(kThreads) void owned_rows_kernel(
    const void* __restrict__ tokens, bool wide, int n, long vocab,
    long padding, int dim, int slices, float scale,
    const T* __restrict__ dout, long row_stride, T* __restrict__ grad) {
  constexpr int V = Elem<T>::kVec;
  constexpr int kWaves = kThreads / 64;
  constexpr int kEach = kOwnedTokens / kWaves / 64;  // of a lane
  __shared__ uint16_t found[kWaves][kOwnedTokens / kWaves];
  __shared__ int length[kWaves];
  __shared__ int count[kOwned];
  __shared__ float part[kWaves][64][V];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned stride = (unsigned)((vocab + kOwned - 1) / kOwned);
  const unsigned row0 = blockIdx.x / slices;     // and row0 + stride, ...
  const int rows = (int)((vocab - row0 + stride - 1) / stride);
  const int col = ((int)(blockIdx.x % slices) * 64 + lane) * V;
  const int cols = dim - col;            // may be none
  if (threadIdx.x < kOwned) count[threadIdx.x] = 0;
  __syncthreads();

  const int quarter = (n + kThreads - 1) / kThreads * 64;
  const unsigned long long below = (1ull << lane) - 1;
  long token[kEach];
#pragma unroll
  for (int g = 0; g < kEach; ++g) {
    const int i = wave * quarter + g * 64 + lane;
    token[g] = g * 64 < quarter && i < n ? token_at(tokens, wide, i) : -1;
  }
  int mine = 0;
#pragma unroll
  for (int g = 0; g < kEach; ++g) {
    const unsigned t = (unsigned)token[g];
    const unsigned r = t / stride;
    const bool hit = token[g] >= 0 && token[g] < vocab &&
        token[g] != padding && t - r * stride == row0;
    const unsigned long long hits = __ballot(hit);
    if (hit) {
      const int i = wave * quarter + g * 64 + lane;
      found[wave][mine + __popcll(hits & below)] = (uint16_t)(i << 4 | r);
      atomicAdd(&count[r], 1);
    }
    mine += __popcll(hits);
  }
  if (lane == 0) length[wave] = mine;
  __syncthreads();

  float acc[V];
  // adds a wave's finds for row r, in order
  const auto add = [&](int w, int r) {
    const int len = length[w];
    for (int from = 0; from < len; from += 64) {
      const int f = from + lane < len ? found[w][from + lane] : 0xffffffff;
      unsigned long long left = __ballot(f >= 0 && (f & (kOwned - 1)) == r);
      while (left) {
        u32x4 v[8];
        int have = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (left) {
            const int at = __ffsll(left) - 1;
            left &= left - 1;
            const int pos = __builtin_amdgcn_readlane(f, at) >> 4;
            if (cols > 0)
              v[u] = load_cols(dout + pos * row_stride + col, cols);
            have = u + 1;
          }
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (u < have) {
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += Elem<T>::get(v[u], j);
          }
      }
    }
  };
  const auto write = [&](int r) {
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] *= scale;
    if (cols > 0)
      store_cols(grad + (row0 + (long)r * stride) * dim + col, cols, acc);
  };
  const int counts = lane < rows ? count[lane] : 0;
  const unsigned some = (unsigned)__ballot(counts > 0);
  unsigned many = (unsigned)__ballot(counts > kMany);
  // the rows without a token first: nothing waits for their stores
  for (int r = wave; r < rows; r += kWaves)
    if (!(some >> r & 1)) {
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = 0.f;
      write(r);
    }
  for (int r = wave; r < rows; r += kWaves)
    if ((some & ~many) >> r & 1) {
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = 0.f;
      for (int w = 0; w < kWaves; ++w) add(w, r);
      write(r);
    }
  for (; many; many &= many - 1) {
    const int r = __ffs(many) - 1;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    add(wave, r);
#pragma unroll
    for (int j = 0; j < V; ++j) part[wave][lane][j] = acc[j];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += part[w][lane][j];
      write(r);
    }
    __syncthreads();
  }
}

struct Runs {
  const uint32_t* keys;
  const uint32_t* positions;
  int n;
  int per;              // positions of a chunk: 8 to 64
  int chunks;
  int slices;           // of 64 vectors of columns
  uint32_t vocab;
  int dim;
  float scale;
};

// One wave: one chunk and one slice. Of a run that began before the chunk,
// the sum goes to pieces[chunk][0]; of one that begins here and goes on
// behind it, to pieces[chunk][1].
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_runs_kernel(
    Runs r, const T* __restrict__ dout, long row_stride, T* __restrict__ grad,
    float* __restrict__ pieces) {
  constexpr int V = Elem<T>::kVec;
  const int lane = threadIdx.x & 63;
  const long work = (long)blockIdx.x * (kThreads / 64) +
      __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (work >= (long)r.chunks * r.slices) return;
  const int chunk = (int)(work / r.slices);
  const int slice = (int)(work % r.slices);
  const int from = chunk * r.per;
  const int n = min(r.per, r.n - from);
  const int col = (slice * 64 + lane) * V;
  const int cols = r.dim - col;          // may be none

  const int i = from + lane;
  const uint32_t key = lane < n ? r.keys[i] : ~0u;
  const uint32_t pos = lane < n ? r.positions[i] : 0u;
  const uint32_t last_key = from > 0 ? r.keys[from - 1] : ~0u;
  const uint32_t next_key = from + n < r.n ? r.keys[from + n] : ~0u;

  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  const auto leave = [&](uint32_t k, bool before, bool behind) {
    if (cols <= 0) return;
    if (before || behind) {
      float* p = pieces +
          (((long)chunk * 2 + (before ? 0 : 1)) * r.slices * 64 +
           slice * 64 + lane) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) p[j] = acc[j];
    } else {
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = acc[j] * r.scale;
      store_cols(grad + (long)k * r.dim + col, cols, f);
    }
  };
  constexpr int U = 8;
  bool first = true;                     // the run at hand is the chunk's first
  for (int j0 = 0; j0 < n; j0 += U) {
    u32x4 f[U];
    uint32_t ks[U + 1];
#pragma unroll
    for (int u = 0; u <= U; ++u)
      ks[u] = j0 + u < n ? __builtin_amdgcn_readlane(key, min(j0 + u, 63))
                         : (j0 + u == n ? next_key : ~0u);
    if (ks[0] >= r.vocab) break;         // from here on nothing has a gradient
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + u < n && cols > 0) {
        const uint32_t p = __builtin_amdgcn_readlane(pos, min(j0 + u, 63));
        f[u] = load_cols<T, true>(dout + (long)p * row_stride + col, cols);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + u < n && ks[u] < r.vocab) {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += Elem<T>::get(f[u], j);
        const bool end = j0 + u == n - 1;
        if (end || ks[u + 1] != ks[u]) {
          leave(ks[u], first && from > 0 && last_key == ks[u],
                end && next_key == ks[u]);
          first = false;
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] = 0.f;
        }
      }
  }
}

// One block for each chunk and slice; those whose last run begins there
// and goes on behind add up its pieces, a quarter of them in each wave.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_runs_kernel(
    Runs r, const float* __restrict__ pieces, T* __restrict__ grad) {
  constexpr int V = Elem<T>::kVec;
  constexpr int kWaves = kThreads / 64;
  __shared__ float part[kWaves][64][V];
  const int chunk = (int)(blockIdx.x / r.slices);
  const int slice = (int)(blockIdx.x % r.slices);
  const int from = chunk * r.per, to = from + r.per;
  if (to >= r.n) return;
  const uint32_t key = r.keys[to - 1];
  if (key >= r.vocab || r.keys[to] != key) return;
  if (from > 0 && r.keys[from - 1] == key) return;   // it began before
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // chunks that begin with this key: the run's others
  int more = 0;
  for (;;) {
    const long c = (long)chunk + 1 + more + lane;
    const bool same = c < r.chunks && r.keys[c * r.per] == key;
    const int have = __popcll(__ballot(same));
    more += have;
    if (have < 64) break;
  }
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  const long row = (long)r.slices * 64 * V;
  const float* p = pieces + ((long)slice * 64 + lane) * V;
  // piece 0 is the run's beginning, piece i the first of chunk + i; four of
  // them under way at once
  const auto piece = [&](int i) {
    return p + (i == 0 ? (long)chunk * 2 + 1 : ((long)chunk + i) * 2) * row;
  };
  int i = wave;
  for (; i + 3 * kWaves <= more; i += 4 * kWaves) {
    float f[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* q = piece(i + u * kWaves);
#pragma unroll
      for (int j = 0; j < V; ++j) f[u][j] = q[j];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += f[u][j];
  }
  for (; i <= more; i += kWaves) {
    const float* q = piece(i);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] += q[j];
  }
#pragma unroll
  for (int j = 0; j < V; ++j) part[wave][lane][j] = acc[j];
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += part[w][lane][j];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] *= r.scale;
    const int col = (slice * 64 + lane) * V;
    if (col < r.dim)
      store_cols(grad + (long)key * r.dim + col, r.dim - col, acc);
  }
}

// ---------------------------------------------------------------- host ---
long ceil_div(long a, long b) { return (a + b - 1) / b; }

int bits_for(unsigned long most) {       // to hold 0..most
  int b = 1;
  while (b < 64 && (most >> b) != 0) ++b;
  return b;
}

bool is_wide(const torch::Tensor& t) { return t.scalar_type() == at::kLong; }

torch::Tensor gather_rows(const torch::Tensor& weight,
                          const torch::Tensor& tokens, float scale) {
  const long n = tokens.numel();
  const long dim = weight.size(1);
  auto out = torch::empty({n, dim}, weight.options());
  if (n == 0 || dim == 0) return out;
  const auto stream = current_stream();
  with_elem(weight.scalar_type(), "the embedding weight", [&](auto z) {
    using T = decltype(z);
    const long vecs = ceil_div(dim, Elem<T>::kVec);
    // four vectors a thread once they still fill the card
    const bool four = n * vecs >= 4L * kThreads * 1024;
    const long blocks = ceil_div(n * vecs, kThreads * (four ? 4 : 1));
    const dim3 grid = grid_of(blocks, kThreads, "tokens");
    const auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream,
                         tokens.data_ptr(), is_wide(tokens), n,
                         static_cast<const T*>(weight.data_ptr()),
                         (long)weight.stride(0), (long)weight.size(0),
                         (int)dim, (unsigned)vecs, scale,
                         static_cast<T*>(out.data_ptr()));
    };
    if (four) go(gather_rows_kernel<T, 4>); else go(gather_rows_kernel<T, 1>);
    CHECK_HIP(hipGetLastError());
  });
  return out;
}

template <typename I, int IPT>
void launch_sort(const torch::Tensor& tokens, long vocab, long padding,
                 int pos_bits, int key_bits, torch::Tensor& keys,
                 torch::Tensor& positions, torch::Tensor& grad) {
  const long bytes = grad.numel() * grad.element_size();
  const int clear = (int)std::min(512L, std::max(1L, bytes / 65536));
  const size_t lds = sizeof(I) * 1024 * IPT +
      sizeof(int) * (16 * kDigits + kDigits + 4);
  auto kernel = sort_and_clear_kernel<I, IPT>;
  if (lds > 65536)
    CHECK_HIP(hipFuncSetAttribute(
        reinterpret_cast<const void*>(kernel),
        hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(kernel, dim3(1 + clear), dim3(1024), lds,
                     current_stream(), tokens.data_ptr(), is_wide(tokens),
                     (int)tokens.numel(), vocab, padding, pos_bits, key_bits,
                     reinterpret_cast<uint32_t*>(keys.data_ptr<int>()),
                     reinterpret_cast<uint32_t*>(positions.data_ptr<int>()),
                     static_cast<char*>(grad.data_ptr()), bytes);
  CHECK_HIP(hipGetLastError());
}

void launch_big_sort(const torch::Tensor& tokens, long vocab, long padding,
                     int key_bits, torch::Tensor& keys,
                     torch::Tensor& positions, torch::Tensor& grad) {
  const long n = tokens.numel();
  const long bytes = grad.numel() * grad.element_size();
  const int tiles = (int)ceil_div(n, kTile);
  const int clear = (int)std::min(1024L, std::max(1L, bytes / 16384));
  auto counts = torch::empty({(long)kDigits * (tiles + 1)}, keys.options());
  int* totals = counts.data_ptr<int>() + (long)kDigits * tiles;
  auto keys2 = torch::empty_like(keys);
  auto positions2 = torch::empty_like(positions);
  const int passes = (key_bits + 7) / 8;
  const int width = (key_bits + passes - 1) / passes;
  const auto stream = current_stream();
  SortIn in{tokens.data_ptr(), is_wide(tokens), vocab, padding, nullptr,
            nullptr};
  for (int pass = 0; pass < passes; ++pass) {
    hipLaunchKernelGGL(tile_counts_kernel,
                       dim3(tiles + (pass == 0 ? clear : 0)), dim3(kThreads),
                       0, stream, in, n, tiles, pass * width, width,
                       counts.data_ptr<int>(),
                       static_cast<char*>(grad.data_ptr()), bytes);
    CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL(scan_counts_kernel, dim3(kDigits), dim3(kThreads), 0,
                       stream, counts.data_ptr<int>(), tiles, totals);
    CHECK_HIP(hipGetLastError());
    auto* k = reinterpret_cast<uint32_t*>(keys2.data_ptr<int>());
    auto* p = reinterpret_cast<uint32_t*>(positions2.data_ptr<int>());
    hipLaunchKernelGGL(tile_scatter_kernel, dim3(tiles), dim3(kThreads), 0,
                       stream, in, n, tiles, pass * width, width,
                       counts.data_ptr<int>(), totals, k, p);
    CHECK_HIP(hipGetLastError());
    in.keys = k;
    in.positions = p;
    std::swap(keys, keys2);
    std::swap(positions, positions2);
  }
}

torch::Tensor weight_grad(const torch::Tensor& tokens,
                          const torch::Tensor& dout, long vocab, long dim,
                          float scale, long padding) {
  const long n = tokens.numel();
  auto grad = torch::empty({vocab, dim}, dout.options());
  if (grad.numel() == 0) return grad;
  if (n == 0) return grad.zero_();
  // Without a sort while the tokens are few and their rows mostly have one
  // or none: each block then looks through all of them.
  if (n <= kOwnedTokens && n <= 2 * vocab) {
    with_elem(dout.scalar_type(), "the embedding gradient", [&](auto z) {
      using T = decltype(z);
      const long slices = ceil_div(dim, 64L * Elem<T>::kVec);
      const long blocks = ceil_div(vocab, kOwned) * slices;
      hipLaunchKernelGGL(owned_rows_kernel<T>,
                         grid_of(blocks, kThreads, "rows of the table"),
                         dim3(kThreads), 0, current_stream(), tokens.data_ptr(),
                         is_wide(tokens), (int)n, vocab, padding, (int)dim,
                         (int)slices, scale,
                         static_cast<const T*>(dout.data_ptr()),
                         (long)dout.stride(0),
                         static_cast<T*>(grad.data_ptr()));
      CHECK_HIP(hipGetLastError());
    });
    return grad;
  }
  const auto ints = tokens.options().dtype(torch::kInt);
  auto keys = torch::empty({n}, ints);
  auto positions = torch::empty({n}, ints);
  const int key_bits = bits_for(vocab);   // the key of no gradient is vocab
  const int pos_bits = bits_for(n - 1);
  if (n > 16384) {
    launch_big_sort(tokens, vocab, padding, key_bits, keys, positions, grad);
  } else {
    const bool narrow = key_bits + pos_bits <= 32;
#define SORT(I, IPT)                                                      \
  launch_sort<I, IPT>(tokens, vocab, padding, pos_bits, key_bits, keys,   \
                      positions, grad)
    if (n <= 1024) {                  // and more than two for each row of dW
      SORT(uint32_t, 1);
    } else if (n <= 4096) {
      if (narrow) SORT(uint32_t, 4); else SORT(uint64_t, 4);
    } else {
      if (narrow) SORT(uint32_t, 16); else SORT(uint64_t, 16);
    }
#undef SORT
  }
  with_elem(dout.scalar_type(), "the embedding gradient", [&](auto z) {
    using T = decltype(z);
    Runs r;
    r.keys = reinterpret_cast<const uint32_t*>(keys.data_ptr<int>());
    r.positions = reinterpret_cast<const uint32_t*>(positions.data_ptr<int>());
    r.n = (int)n;
    r.slices = (int)ceil_div(dim, 64L * Elem<T>::kVec);
    // long chunks leave fewer pieces, short ones make more waves: as long
    // as they still give each CU eight
    r.per = 64;
    while (r.per > 8 && ceil_div(n, r.per) * r.slices < 2048) r.per /= 2;
    r.chunks = (int)ceil_div(n, r.per);
    r.vocab = (uint32_t)vocab;
    r.dim = (int)dim;
    r.scale = scale;
    const long waves = (long)r.chunks * r.slices;
    const dim3 joins = grid_of(waves, kThreads, "tokens");
    auto pieces = torch::empty(
        {r.chunks > 1 ? waves * 2 * 64 * Elem<T>::kVec : 1},
        dout.options().dtype(torch::kFloat));
    T* pg = static_cast<T*>(grad.data_ptr());
    float* pp = static_cast<float*>(pieces.data_ptr());
    const auto stream = current_stream();
    hipLaunchKernelGGL(sum_runs_kernel<T>,
                       dim3(ceil_div(waves, kThreads / 64)), dim3(kThreads),
                       0, stream, r, static_cast<const T*>(dout.data_ptr()),
                       (long)dout.stride(0), pg, pp);
    CHECK_HIP(hipGetLastError());
    if (r.chunks > 1) {
      hipLaunchKernelGGL(join_runs_kernel<T>, joins, dim3(kThreads), 0,
                         stream, r, pp, pg);
      CHECK_HIP(hipGetLastError());
    }
  });
  return grad;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

torch::Tensor grad_rows(const torch::Tensor& tokens, torch::Tensor dout,
                        int64_t vocab, double scale, int64_t padding) {
  c10::DeviceGuard guard(tokens.device());
  if (dout.size(1) > 1 && dout.stride(1) != 1) dout = dout.contiguous();
  return weight_grad(tokens, dout, vocab, dout.size(1), (float)scale,
                     padding);
}

// `twice`: the backward pass may itself be differentiated. The rows' sums
// are linear in dout, and their own gradient is a gather again, of zeros
// for tokens that have no gradient.
struct Embedding : torch::autograd::Function<Embedding> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor weight,
                               torch::Tensor tokens, double scale,
                               int64_t padding, bool twice) {
    c10::DeviceGuard guard(weight.device());
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["twice"] = twice;
    return gather_rows(weight, tokens, (float)scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor dout,
                               torch::Tensor tokens, int64_t vocab,
                               double scale, int64_t padding) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = vocab;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return grad_rows(tokens, dout, vocab, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto tokens = ctx->get_saved_variables()[0];
    const int64_t padding = ctx->saved_data["padding"].toInt();
    const auto g = grads[0].size(1) < 2 || grads[0].stride(1) == 1
        ? grads[0] : grads[0].contiguous();
    const auto out = Embedding::apply(
        g, tokens, ctx->saved_data["scale"].toDouble(), padding, true);
    const auto none = tokens.eq(padding)
                          .logical_or(tokens.lt(0))
                          .logical_or(
                              tokens.ge(ctx->saved_data["vocab"].toInt()));
    return {out.masked_fill(none.unsqueeze(1), 0), torch::Tensor(),
            torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

variable_list Embedding::backward(AutogradContext* ctx, variable_list grads) {
  const auto tokens = ctx->get_saved_variables()[0];
  const int64_t vocab = ctx->saved_data["vocab"].toInt();
  const double scale = ctx->saved_data["scale"].toDouble();
  const int64_t padding = ctx->saved_data["padding"].toInt();
  torch::Tensor grad;
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK(ctx->saved_data["twice"].toBool(),
                "the embedding has no second derivative: it cannot be "
                "differentiated with create_graph=True");
    grad = EmbeddingGrad::apply(grads[0], tokens, vocab, scale, padding);
  } else {
    grad = grad_rows(tokens, grads[0], vocab, scale, padding);
  }
  return {grad, torch::Tensor(), torch::Tensor(), torch::Tensor(),
          torch::Tensor()};
}

}  // namespace

// padding: a row that gets no gradient, or -1.
torch::Tensor embedding(const torch::Tensor& tokens,
                        const torch::Tensor& weight, double scale,
                        int64_t padding, bool twice) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(),
              "the embedding kernel cannot be traced");
  TORCH_CHECK_VALUE(weight.is_cuda() && weight.dim() == 2,
                    "the embedding weight must be a matrix on a GPU");
  TORCH_CHECK_VALUE(weight.size(0) < (1L << 31) - 1 &&
                        weight.size(1) < (1L << 30),
                    "the embedding weight is too large");
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong ||
                       tokens.scalar_type() == at::kInt,
                   "tokens must be int64 or int32, not ",
                   tokens.scalar_type());
  TORCH_CHECK_VALUE(tokens.device() == weight.device(),
                    "tokens must be on the weight's device");
  TORCH_CHECK_VALUE(tokens.numel() < (1L << 31) - 4096, "too many tokens");
  TORCH_CHECK_VALUE(padding >= -1 && padding < weight.size(0),
                    "padding_idx must be a row of the weight: ", padding);
  with_elem(weight.scalar_type(), "the embedding weight", [](auto) {});
  c10::DeviceGuard guard(weight.device());
  const auto w = weight.size(1) < 2 || weight.stride(1) == 1
      ? weight : weight.contiguous();
  auto out = Embedding::apply(w, tokens.reshape({-1}).contiguous(), scale,
                              padding, twice);
  if (tokens.dim() == 1) return out;
  auto shape = tokens.sizes().vec();
  shape.push_back(weight.size(1));
  return out.view(shape);
}

}  // namespace mgx
