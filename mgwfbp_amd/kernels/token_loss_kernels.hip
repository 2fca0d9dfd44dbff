// Cross entropy with its gradient, and log probabilities of given tokens
// with the row's entropy and its best alternatives, gfx950.
//
// For a row x of V logits and any reference r near its maximum, with
// t_j = (x_j - r) log2 e, s = sum 2^t_j and u = sum 2^t_j t_j:
//
//   log p_j = ln 2 (t_j - log2 s)        entropy H = ln 2 (log2 s - u / s)
//   d log p_t / d x_j = [j = t] - p_j    d H / d x_j = -p_j (log p_j + H)
//
// The reference has to be near for the differences' sake: one that is d
// binary orders below the maximum leaves both sides of them near d, and a
// log probability or an entropy near 0 is then off by d roundings. So it is
// the maximum of what is held or has streamed past so far; only the loss,
// which needs no u, takes one from a part of the row and the target, see
// row_loss_kernel. What the last rounding leaves on the wrong side of 0 is
// set to 0.
//
// All of it is bound by memory: a row is read once for s and u (in 32
// bits), and a gradient is one more read and a write. Where the loss is to
// be differentiated its gradient leaves the forward pass, from a row that
// is still in registers, so that the logits are read once in all; see
// row_loss_kernel.
//
// Next to memory comes the arithmetic: at 6 TB/s of 16-bit logits a CU has
// some 13 lane-cycles for an element, of which 2^t takes 4. So t is one
// fused multiply-add, x log2 e - K, whose only rounding is that of the
// result; K, the reference in these units, is held within +-kFar, where
// that is exact enough, and nothing is tested for each element. A row
// whose s does not come out sane (a NaN, an infinity, nothing but -inf, or
// logits beyond kFar, such as a row masked with the type's lowest value) is
// done again by slow_row, which subtracts first and takes every case; its
// stats are told apart by a negative s.
//
// Measured: 8190 x 50001 bf16, loss and gradient 304 us, of which 299 (5.5
// TB/s) in row_loss_kernel; 4095 x 32768 bf16, log probabilities with
// entropy 52 us (5.1 TB/s) and their gradient 87 (6.1 TB/s); 700 x 10000
// float32 with the best five 10 us; 4 x 50001 bf16 with the best eight 10.
//
// A logit of -inf has p = 0 and adds nothing anywhere (t is held at kFloor
// where it is a factor, so that no 0 * inf arises). A row with a NaN, a
// +inf or nothing but -inf has no distribution and gives NaN, as torch's
// log_softmax does. A target outside [0, V) that is not ignore_index is
// never read: it gives NaN, in the value and the gradient.
#include <hip/hip_runtime.h>

#include "lm_common.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <limits>
#include <tuple>
#include <vector>

namespace mgx {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -300.f;       // 2^kFloor is 0 in float32
constexpr float kFar = 4194304.f;      // 2^22
constexpr float kInf = __builtin_inff();
constexpr int kThreads = 256;
constexpr int kMaxTop = 64;
constexpr int kGroups = 256;           // of maxima, in the search for the best
constexpr int kCandidates = 512;       // that the search holds
constexpr int kJoin = 1024;            // keys that the join of a row takes
constexpr int kMaxSplits = 64;

__device__ __forceinline__ float exp2_(float t) {
  return __builtin_amdgcn_exp2f(t);
}

__device__ __forceinline__ long target_at(const void* p, bool wide, long i) {
  return wide ? static_cast<const long*>(p)[i]
              : static_cast<long>(static_cast<const int*>(p)[i]);
}

// s and u of part of a row, against reference k.
struct Stat {
  float k = -kFar, s = 0.f, u = 0.f;

  static __device__ __forceinline__ float ref(float max) {
    return fminf(fmaxf(max * kLog2e, -kFar), kFar);
  }
  // against reference `to`, which is no lower
  __device__ __forceinline__ void raise(float to) {
    const float d = k - to;
    const float f = exp2_(d);
    u = fmaf(s, d, u) * f;
    s *= f;
    k = to;
  }
  template <bool ENT>
  __device__ __forceinline__ void add(float x) {
    const float t = fmaf(x, kLog2e, -k);
    const float e = exp2_(t);
    s += e;
    if (ENT) u = fmaf(e, fmaxf(t, kFloor), u);
  }
  // N more elements, whose maximum is the result: the reference is raised
  // to it first where it is lower.
  template <int N, typename F>
  __device__ __forceinline__ float add_all(F&& x) {
    float m = -kInf;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x(i));
    const float to = ref(m);
    if (to > k) raise(to);
#pragma unroll
    for (int i = 0; i < N; ++i) add<true>(x(i));
    return m;
  }
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// The same for every lane: the reference first, then plain sums.
template <bool ENT>
__device__ __forceinline__ void wave_merge(Stat& a) {
  a.raise(wave_max(a.k));
  a.s = wave_sum(a.s);
  if (ENT) a.u = wave_sum(a.u);
}

// And for every thread of the block; `lds` holds 3 floats for each wave
// and is free again after the caller's next barrier.
template <bool ENT, int BLOCK>
__device__ __forceinline__ void block_merge(Stat& a, float* lds) {
  constexpr int kWaves = BLOCK / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  wave_merge<ENT>(a);
  if (lane == 0) {
    lds[wave] = a.k;
    lds[kWaves + wave] = a.s;
    if (ENT) lds[2 * kWaves + wave] = a.u;
  }
  __syncthreads();
  a = Stat();
  if (lane < kWaves) {
    a.k = lds[lane];
    a.s = lds[kWaves + lane];
    if (ENT) a.u = lds[2 * kWaves + lane];
  }
  wave_merge<ENT>(a);
}

// A row's stats as they are stored: reference and s; with s negated where
// the reference is in the logits' own units, and NaN where there is no
// distribution.
struct Row {
  float ref, s, log2s;
  bool slow;

  __device__ __forceinline__ Row(float r, float signed_s)
      : ref(r), s(fabsf(signed_s)), log2s(log2f(fabsf(signed_s))),
        slow(signed_s < 0.f) {}
  template <bool SLOW>
  __device__ __forceinline__ float t(float x) const {
    return SLOW ? (x - ref) * kLog2e : fmaf(x, kLog2e, -ref);
  }
  // a NaN stays one
  __device__ __forceinline__ float log_prob(float x) const {
    const float lp = kLn2 * ((slow ? t<true>(x) : t<false>(x)) - log2s);
    return lp > 0.f ? 0.f : lp;
  }
  __device__ __forceinline__ float entropy(float u) const {
    const float h = kLn2 * (log2s - u / s);
    return h < 0.f ? 0.f : h;
  }
};

// Whether the fast way has given a sum to go on with. Against its maximum,
// or kLower below, a row of n logits has one between 1 and n, or 2^kLower
// times that; not so where the reference was held at +-kFar, or where
// something is not finite.
constexpr float kLower = 17.f;
__device__ __forceinline__ bool sane(float s, int n) {
  return s > 0.25f && s < 262144.f * (float)n;
}

// Every case, by the whole block, from memory: the maximum, then sums of
// what is left when it is subtracted. Returns s as it is stored; ref and u
// besides.
template <typename T, int BLOCK>
__device__ __forceinline__ float slow_row(const T* x, int n, float* lds,
                                          float& ref, float& u) {
  constexpr int kWaves = BLOCK / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float m = -kInf;
#pragma unroll 1
  for (int j = threadIdx.x; j < n; j += BLOCK)
    m = fmaxf(m, Elem<T>::up(x[j]));
  m = wave_max(m);
  __syncthreads();                     // lds may still be read
  if (lane == 0) lds[wave] = m;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, lds[w]);
  float s = 0.f, v = 0.f;
#pragma unroll 1
  for (int j = threadIdx.x; j < n; j += BLOCK) {
    const float t = (Elem<T>::up(x[j]) - m) * kLog2e;
    const float e = exp2_(t);
    s += e;
    v = fmaf(e, fmaxf(t, kFloor), v);
  }
  s = wave_sum(s);
  v = wave_sum(v);
  __syncthreads();
  if (lane == 0) {
    lds[wave] = s;
    lds[kWaves + wave] = v;
  }
  __syncthreads();
  s = v = 0.f;
  for (int w = 0; w < kWaves; ++w) {
    s += lds[w];
    v += lds[kWaves + w];
  }
  ref = m;
  u = v;
  return s > 0.f && s < kInf ? -s : __builtin_nanf("");
}

// A stretch of a row as its vectors: whole ones that begin at multiples of
// 16 bytes, and the up to 2 V - 2 elements before and behind them, one for
// a thread. Rows of an odd width begin anywhere, and 8190 rows of 50001
// 16-bit logits take a quarter less time this way than by vectors that
// begin where the row does, each of which lies in two lines.
struct Parts {
  int head, vecs, edges;       // edges: elements before and behind

  template <typename T>
  static __device__ __forceinline__ Parts of(const T* x, int n) {
    constexpr int V = Elem<T>::kVec;
    Parts p;
    p.head = min(n, (int)((0u - (unsigned)(uintptr_t)x) % 16u) /
                        (int)sizeof(T));
    p.vecs = (n - p.head) / V;
    p.edges = n - p.vecs * V;
    return p;
  }
  // the element of thread (or edge) i, i < edges
  template <int V>
  __device__ __forceinline__ int edge(int i) const {
    return i < head ? i : i + vecs * V;
  }
  // the thread of a block of BLOCK that has element j
  template <int V, int BLOCK>
  __device__ __forceinline__ int owner(int j) const {
    if (j < head) return j;
    const int v = (j - head) / V;
    return v < vecs ? v % BLOCK : j - vecs * V;
  }
};

// A slice of a row in the registers of a block: NV vectors of each thread,
// 16 bytes each, and one element of what is left of a vector.
//
// Every load is made, of the last vector where there is none for it: so many
// loads are under way for certain, and the compiler can wait for the first
// alone and start on it while the others come. What is too much counts as
// -inf where it would matter.
template <typename T, int BLOCK, int NV>
struct Held {
  static constexpr int V = Elem<T>::kVec;
  u32x4 r[NV];
  T last;
  Parts p;

  // Where the slice has no whole vector, the 16 bytes before the first
  // one's place are read instead; the host sees to it that they are the
  // row's (kHeldLeast).
  __device__ __forceinline__ void load(const T* x, int n) {
    p = Parts::of(x, n);
    const int mine = p.edge<V>((int)threadIdx.x);
    last = x[(int)threadIdx.x < p.edges ? mine : 0];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      r[i] = load16_past(
          x + p.head + min((int)threadIdx.x + i * BLOCK, p.vecs - 1) * V);
  }
  // vector i, and the element besides the vectors
  __device__ __forceinline__ u32x4 vec(int i) const {
    return (int)threadIdx.x + i * BLOCK < p.vecs ? r[i]
                                                 : Elem<T>::minus_inf();
  }
  __device__ __forceinline__ float rest() const {
    return (int)threadIdx.x < p.edges ? Elem<T>::up(last) : -kInf;
  }
  __device__ __forceinline__ float max() const {
    float m = rest();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const u32x4 q = vec(i);
#pragma unroll
      for (int j = 0; j < V; ++j) m = fmaxf(m, Elem<T>::get(q, j));
    }
    return m;
  }
  template <bool ENT>
  __device__ __forceinline__ Stat stat(float max) const {
    Stat a;
    a.k = Stat::ref(max);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const u32x4 q = vec(i);
#pragma unroll
      for (int j = 0; j < V; ++j)
        a.template add<ENT>(Elem<T>::get(q, j));
    }
    a.template add<ENT>(rest());
    return a;
  }
  // A reference for the thread's share: the maximum of its first vector, or
  // of all where that one is masked. It serves for s alone, and where it
  // turns out to be no more than kLower below the row's maximum.
  __device__ __forceinline__ float guess() const {
    const u32x4 q = vec(0);
    float m = -kInf;
#pragma unroll
    for (int j = 0; j < V; ++j) m = fmaxf(m, Elem<T>::get(q, j));
    if (!(m > -64.f)) m = max();
    return m;
  }
  // f(value, index) for the elements that are not below tau
  template <typename F>
  __device__ __forceinline__ void each_from(float tau, F&& f) const {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = tid + i * BLOCK;
      bool any = false;
#pragma unroll
      for (int j = 0; j < V; ++j) any |= !(Elem<T>::get(r[i], j) < tau);
      if (any && at < p.vecs) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float x = Elem<T>::get(r[i], j);
          if (!(x < tau)) f(x, p.head + at * V + j);
        }
      }
    }
    const float x = Elem<T>::up(last);
    if (tid < p.edges && !(x < tau)) f(x, p.edge<V>(tid));
  }
  // Keeps the compiler from carrying what it has unpacked from one use of
  // the slice to the next, which takes up to four times the registers.
  __device__ __forceinline__ void unpack_again() {
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(r[i]));
  }
};

// -------------------------------------------------------- best of a row --
// A value's place in the order: larger is better, NaN best of all, both
// zeros the same. With the index below it, keys are distinct, and of equal
// values the lowest index is best.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t key_of(float x, int j) {
  return (static_cast<uint64_t>(order_of(x)) << 32) |
         static_cast<uint32_t>(~j);
}

struct Best {
  uint32_t group[kGroups];
  uint64_t found[kCandidates];
  uint64_t wave[16];
  uint32_t least;
  int count;
};

// The k best keys of a slice, handed to put(rank, key), best first; key 0
// where there are fewer. `top` is the largest value of this thread's share
// (a NaN is passed over). The k-th largest of 256 shares' maxima is at most
// the k-th largest value, so everything from there up is gathered (about k
// values unless many are equal) and ranked. Where they do not fit, k
// rounds over x[0..n) take the best below the last one. `each_from(tau, f)`
// calls f(value, index) for this thread's elements that are not below tau;
// `base` is added to the indices.
template <typename T, int BLOCK, typename E, typename F>
__device__ __forceinline__ void best_of(const T* x, int n, E&& each_from,
                                        int base, int k, float top, Best& b,
                                        F&& put) {
  // the lowest bit of the order that the threshold is worked out to; bits
  // that are left out only lower it
  constexpr int KLAST = sizeof(T) == 2 ? 13 : 8;
  constexpr int kShare = BLOCK / kGroups;  // threads of a group
  static_assert(kShare * kGroups == BLOCK && (kShare & (kShare - 1)) == 0,
                "neighbouring threads make up a group");
  const int tid = threadIdx.x;
#pragma unroll
  for (int off = 1; off < kShare; off <<= 1)
    top = fmaxf(top, __shfl_xor(top, off, 64));
  if (tid % kShare == 0) b.group[tid / kShare] = order_of(top);
  if (tid == 0) b.count = 0;
  __syncthreads();
  if (tid < 64) {
    uint32_t g[kGroups / 64];
#pragma unroll
    for (int i = 0; i < kGroups / 64; ++i) g[i] = b.group[tid + 64 * i];
    uint32_t least = 0;
    for (int bit = 31; bit >= KLAST; --bit) {
      const uint32_t c = least | (1u << bit);
      int have = 0;
#pragma unroll
      for (int i = 0; i < kGroups / 64; ++i)
        have += __popcll(__ballot(g[i] >= c));
      if (have >= k) least = c;
    }
    if (tid == 0) b.least = least;
  }
  __syncthreads();
  // as a value: below it nothing can be among the best; a NaN is not below
  const uint32_t least = b.least;
  const float tau = least <= order_of(-kInf) ? -kInf : value_of(least);
  each_from(tau, [&](float v, int j) {
    const int at = atomicAdd(&b.count, 1);
    if (at < kCandidates) b.found[at] = key_of(v, base + j);
  });
  __syncthreads();
  const int count = b.count;
  if (count <= kCandidates) {
    for (int c = tid; c < count; c += BLOCK) {
      const uint64_t key = b.found[c];
      int rank = 0;
#pragma unroll 8
      for (int o = 0; o < count; ++o) rank += b.found[o] > key;
      if (rank < k) put(rank, key);
    }
    for (int r = count + tid; r < k; r += BLOCK) put(r, 0);
    return;
  }
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
#pragma unroll 1
    for (int j = tid; j < n; j += BLOCK) {
      const uint64_t key = key_of(Elem<T>::up(x[j]), base + j);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)best, off, 64);
      best = o > best ? o : best;
    }
    if ((tid & 63) == 0) b.wave[tid >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w)
      best = b.wave[w] > best ? b.wave[w] : best;
    __syncthreads();
    if (tid == 0) put(r, best);
    last = best;
  }
}

// ------------------------------------------------------------- forward ---
struct RowOut {
  float2* stats;       // m and s of each row
  float* log_probs;    // of the target; or its negative, for a loss
  float* entropy;      // may be null
  float* top_values;   // [rows, k]
  long* top_ids;
  float sign;          // -1 for a loss
};

__device__ __forceinline__ void finish_row(const Row& a, float u, long row,
                                           int vocab, float x_target,
                                           long target, long ignore,
                                           const RowOut& out) {
  float lp = 0.f;
  if (target != ignore)
    lp = out.sign * (target < 0 || target >= vocab
                         ? __builtin_nanf("") : a.log_prob(x_target));
  out.log_probs[row] = lp;
  out.stats[row] = make_float2(a.ref, a.slow ? -a.s : a.s);
  if (out.entropy != nullptr) out.entropy[row] = a.entropy(u);
}

struct Where {                 // a launch's rows
  long row_stride;
  int vocab;
  int splits;                  // blocks of a row ...
  int slice;                   // ... and the elements that each takes
  const void* targets;
  bool wide;
  long ignore;
  int k;
};

// A row's target and its logit, asked for early: at the end they would be
// two latencies, one after the other, with nothing beside them.
struct Target {
  long id;
  float x;

  template <typename T>
  static __device__ __forceinline__ Target of(const T* row_x, long row,
                                              const Where& w) {
    Target t;
    t.id = target_at(w.targets, w.wide, row);
    t.x = Elem<T>::up(row_x[t.id >= 0 && t.id < w.vocab ? t.id : 0]);
    return t;
  }
  // The same where the block takes the row whole, as a scalar load of the
  // word that the logit lies in: what waits for it need not wait for the
  // row, as it would behind vector loads, which come back in order.
  template <typename T>
  static __device__ __forceinline__ Target of_row(const T* row_x, long row,
                                                  const Where& w) {
    typedef const __attribute__((address_space(4))) uint32_t* Word;
    Target t;
    t.id = target_at(w.targets, w.wide, row);
    const auto at = reinterpret_cast<uintptr_t>(
        row_x + (t.id >= 0 && t.id < w.vocab ? t.id : 0));
    const uint32_t word = *(Word)(at & ~(uintptr_t)3);
    t.x = Elem<T>::get(u32x4{word, 0u, 0u, 0u},
                       (int)(at & 3) / (int)sizeof(T));
    return t;
  }
};

// What a block found of its slice: the row's outputs where it is the whole
// row, else pieces for join_rows_kernel. Returns the row's stats for the
// former.
template <typename T, int BLOCK>
__device__ __forceinline__ Row finish_slice(const T* x, const Target& t,
                                            Stat a, long row, int part,
                                            const Where& w,
                                            const RowOut& out, float* lds,
                                            float* part_stats) {
  float ref = a.k, s = a.s, u = a.u;
  if (w.splits > 1) {
    if (threadIdx.x == 0) {
      float* p = part_stats + 3 * (row * w.splits + part);
      p[0] = ref; p[1] = s; p[2] = u;
    }
    return Row(0.f, 1.f);
  }
  if (!sane(s, w.vocab)) s = slow_row<T, BLOCK>(x, w.vocab, lds, ref, u);
  const Row r(ref, s);
  if (threadIdx.x == 0)
    finish_row(r, u, row, w.vocab, t.x, t.id, w.ignore, out);
  return r;
}

template <typename F>
__device__ __forceinline__ void put_best(const Row& r, const Where& w,
                                         long row, int part,
                                         const RowOut& out,
                                         uint64_t* part_keys, F&& search) {
  if (w.splits > 1) {
    uint64_t* keys = part_keys + (row * w.splits + part) * w.k;
    search([&](int rank, uint64_t key) { keys[rank] = key; });
  } else {
    search([&](int rank, uint64_t key) {
      out.top_ids[row * w.k + rank] = static_cast<int>(~(uint32_t)key);
      out.top_values[row * w.k + rank] = r.log_prob(value_of(key >> 32));
    });
  }
}

// One block a row, or, for rows that one block cannot hold, `splits` of
// them that each leave what they found of their slice for
// join_rows_kernel. This one takes slices too long for held_stats_kernel:
// they stream past, and with TOP are read a second time.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void row_stats_kernel(
    const T* __restrict__ logits, Where w, RowOut out,
    float* __restrict__ part_stats, uint64_t* __restrict__ part_keys) {
  constexpr int V = Elem<T>::kVec;
  constexpr int U = 4;
  __shared__ float lds[3 * kThreads / 64];
  __shared__ typename std::conditional<TOP, Best, int>::type best;
  const long row = blockIdx.x / w.splits;
  const int part = blockIdx.x % w.splits;
  const int from = part * w.slice;
  const int n = min(w.slice, w.vocab - from);
  const T* __restrict__ x = logits + row * w.row_stride + from;
  const int tid = threadIdx.x;
  const Target target = Target::of(x - from, row, w);

  Stat a;
  float top = -kInf;
  const Parts p = Parts::of(x, n);
  const T* __restrict__ xv = x + p.head;
  int i = tid;
  for (; i + (U - 1) * kThreads < p.vecs; i += U * kThreads) {
    u32x4 r[U];
#pragma unroll
    for (int q = 0; q < U; ++q)
      r[q] = load16_past(xv + (i + q * kThreads) * V);
    const auto get = [&](int e) { return Elem<T>::get(r[e / V], e % V); };
    top = fmaxf(top, a.template add_all<U * V>(get));
  }
  for (; i < p.vecs; i += kThreads) {
    const u32x4 r = load16_past(xv + i * V);
    const auto get = [&](int e) { return Elem<T>::get(r, e); };
    top = fmaxf(top, a.template add_all<V>(get));
  }
  if (tid < p.edges) {
    const float v = Elem<T>::up(x[p.edge<V>(tid)]);
    top = fmaxf(top, a.template add_all<1>([&](int) { return v; }));
  }
  block_merge<true, kThreads>(a, lds);
  const Row r =
      finish_slice<T, kThreads>(x, target, a, row, part, w, out, lds,
                                part_stats);
  if constexpr (TOP)
    put_best(r, w, row, part, out, part_keys, [&](auto put) {
      best_of<T, kThreads>(
          x, n,
          [&](float tau, auto f) {
#pragma unroll 4
            for (int j = tid; j < n; j += kThreads) {
              const float v = Elem<T>::up(x[j]);
              if (!(v < tau)) f(v, j);
            }
          },
          from, w.k, top, best, put);
    });
}

// Waves on each SIMD that a block of NV vectors a thread leaves registers
// for: two blocks or more on a CU, so that one's loads run beside another's
// arithmetic, but for the longest slices.
constexpr int waves_for(int block, int nv, bool top = false) {
  return nv <= 4 ? 8 : block == 1024 ? 4 : top ? 5 : 6;
}

// The same for a slice that fits the registers of a block: all its loads
// are under way at once, and what comes after reads no memory.
template <typename T, int BLOCK, int NV, bool TOP>
__global__ __launch_bounds__(
    BLOCK, waves_for(BLOCK, NV, TOP)) void held_stats_kernel(
    const T* __restrict__ logits, Where w, RowOut out,
    float* __restrict__ part_stats, uint64_t* __restrict__ part_keys) {
  __shared__ float lds[3 * BLOCK / 64];
  __shared__ typename std::conditional<TOP, Best, int>::type best;
  const long row = blockIdx.x / w.splits;
  const int part = blockIdx.x % w.splits;
  const int from = part * w.slice;
  const int n = min(w.slice, w.vocab - from);
  const T* __restrict__ x = logits + row * w.row_stride + from;
  const Target target = Target::of(x - from, row, w);
  Held<T, BLOCK, NV> held;
  held.load(x, n);
  const float top = held.max();
  held.unpack_again();
  Stat a = held.template stat<true>(top);
  block_merge<true, BLOCK>(a, lds);
  const Row r = finish_slice<T, BLOCK>(x, target, a, row, part, w, out, lds,
                                       part_stats);
  if constexpr (TOP) {
    held.unpack_again();
    put_best(r, w, row, part, out, part_keys, [&](auto put) {
      best_of<T, BLOCK>(
          x, n, [&](float tau, auto f) { held.each_from(tau, f); }, from,
          w.k, top, best, put);
    });
  }
}

template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void join_rows_kernel(
    const T* __restrict__ logits, Where w, RowOut out,
    const float* __restrict__ part_stats,
    const uint64_t* __restrict__ part_keys) {
  __shared__ uint64_t keys[TOP ? kJoin : 1];
  __shared__ float lds[3 * kThreads / 64];
  const long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const T* __restrict__ x = logits + row * w.row_stride;
  const Target target = Target::of(x, row, w);
  const int count = TOP ? w.splits * w.k : 0;    // at most kJoin
  for (int i = tid; i < count; i += kThreads)
    keys[i] = part_keys[row * count + i];
  Stat a;
  if (lane < w.splits) {
    const float* p = part_stats + 3 * (row * w.splits + lane);
    a.k = p[0]; a.s = p[1]; a.u = p[2];
  }
  wave_merge<true>(a);
  w.splits = 1;
  const Row r = finish_slice<T, kThreads>(x, target, a, row, 0, w, out, lds,
                                          (float*)nullptr);
  if constexpr (TOP) {
    __syncthreads();
    for (int i = tid; i < count; i += kThreads) {
      const uint64_t key = keys[i];
      int rank = 0;
#pragma unroll 8
      for (int o = 0; o < count; ++o) rank += keys[o] > key;
      if (key != 0 && rank < w.k) {
        out.top_ids[row * w.k + rank] = static_cast<int>(~(uint32_t)key);
        out.top_values[row * w.k + rank] = r.log_prob(value_of(key >> 32));
      }
    }
  }
}

// Rows that are not ignored; what a mean is divided by.
__global__ __launch_bounds__(1024) void count_kept_kernel(
    const void* __restrict__ targets, bool wide, long ignore, long rows,
    float* __restrict__ share) {
  __shared__ int waves[16];
  int c = 0;
#pragma unroll 4
  for (long i = threadIdx.x; i < rows; i += 1024)
    c += target_at(targets, wide, i) != ignore;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) c += __shfl_xor(c, off, 64);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    c = 0;
    for (int w = 0; w < 16; ++w) c += waves[w];
    *share = 1.f / (float)c;
  }
}

// The loss of a row and its gradient, from one read: the row is held in
// the block's registers, 4 to 64 of them for a thread, while its sums are
// worked out. The gradient is that of the summed loss, times *share if
// given, times one; what comes in for it in the backward pass is nearly
// always that, and rescale_rows_kernel sees to the rest. Up to kCountHere
// rows the block counts the rows that are kept itself, which costs less
// than a launch.
//
// The reference is the maximum of the threads' first vectors, so that the
// exponentials begin when those have come, and of the target, beside which
// the loss may be small. A logit that is far above both shows in s: then
// the row's maximum is looked for, and if it is more than kLower above, the
// sums are taken once more, from the registers. 2^kLower is as many classes
// as a row here has, so that an even row need not be looked through:
// 8190 x 50001 bf16 nearly even logits take 310 us like others, and 348
// with a kLower of 10. (All rows with a logit of 30 in the last place, not
// the target: 353.) An exponent of 17 is off by 2^-20 at most, and so far
// from the others' is then the probability of such a logit.
constexpr int kCountHere = 1024;

template <typename T, int BLOCK, int NV>
__global__ __launch_bounds__(BLOCK, waves_for(BLOCK, NV)) void row_loss_kernel(
    const T* __restrict__ logits, Where w, RowOut out, long rows, bool mean,
    const float* __restrict__ share, T* __restrict__ grad) {
  constexpr int V = Elem<T>::kVec;
  constexpr int kWaves = BLOCK / 64;
  __shared__ float lds[3 * kWaves];
  __shared__ int kept[kWaves];
  const long row = blockIdx.x;
  const int n = w.vocab;
  const T* __restrict__ x = logits + row * w.row_stride;
  const Target target = Target::of_row(x, row, w);
  Held<T, BLOCK, NV> held;
  held.load(x, n);
  int c = 0;
  if (mean && share == nullptr) {
    for (int i = threadIdx.x; i < (int)rows; i += BLOCK)
      c += target_at(w.targets, w.wide, i) != w.ignore;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) c += __shfl_xor(c, off, 64);
    if ((threadIdx.x & 63) == 0) kept[threadIdx.x >> 6] = c;
  }
  Stat a = held.template stat<false>(fmaxf(held.guess(), target.x));
  block_merge<false, BLOCK>(a, lds);    // a barrier: kept is there too
  if (!(a.s <= 131072.f)) {             // 2^kLower
    held.unpack_again();
    const float top = held.max();
    if (__syncthreads_or(Stat::ref(top) > a.k + kLower)) {
      held.unpack_again();
      a = held.template stat<false>(top);
      block_merge<false, BLOCK>(a, lds);
    }
  }
  float by = 1.f;
  if (mean) {
    if (share != nullptr) {
      by = *share;
    } else {
      c = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) c += kept[i];
      by = 1.f / (float)c;
    }
  }
  const Row r = finish_slice<T, BLOCK>(x, target, a, row, 0, w, out, lds,
                                       (float*)nullptr);
  held.unpack_again();
  T* __restrict__ y = grad + row * n;
  const Parts& p = held.p;
  int tid = threadIdx.x;               // worked out again: see unpack_again
  asm volatile("" : "+v"(tid));
  const auto write = [&](auto of) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = tid + i * BLOCK;
      if (at < p.vecs) {
        float f[V];
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = of(Elem<T>::get(held.r[i], j));
        store16_past(y + p.head + at * V, Elem<T>::pack(f));
      }
    }
    if (tid < p.edges)
      y[p.edge<V>(tid)] = Elem<T>::down(of(Elem<T>::up(held.last)));
  };
  if (target.id == w.ignore) {
    // zero, even where the row is not finite
    write([](float) { return 0.f; });
    return;
  }
  const bool there = target.id >= 0 && target.id < n;
  if (!there) by = __builtin_nanf("");
  const float scale = by / r.s;
  if (r.slow)
    write([&](float v) { return exp2_(r.template t<true>(v)) * scale; });
  else
    write([&](float v) { return exp2_(r.template t<false>(v)) * scale; });
  // The target's place once more, by the thread that has just written it.
  if (there && p.owner<V, BLOCK>((int)target.id) == tid) {
    const float t = r.slow ? r.template t<true>(target.x)
                           : r.template t<false>(target.x);
    y[target.id] = Elem<T>::down(fmaf(exp2_(t), scale, -by));
  }
}

// Sum, or mean over the rows that are not ignored, of the rows' losses, in
// 64 bits and in a fixed order; and what each row's gradient is divided
// by.
__global__ __launch_bounds__(1024) void reduce_loss_kernel(
    const float* __restrict__ each, const void* __restrict__ targets,
    bool wide, long ignore, long rows, bool mean, float* __restrict__ loss,
    float* __restrict__ share) {
  __shared__ double sums[16];
  __shared__ double kept[16];
  double s = 0., c = 0.;
#pragma unroll 4
  for (long i = threadIdx.x; i < rows; i += 1024) {
    s += each[i];
    c += target_at(targets, wide, i) != ignore ? 1. : 0.;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    s += __shfl_xor(s, off, 64);
    c += __shfl_xor(c, off, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6] = s;
    kept[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = c = 0.;
    for (int w = 0; w < 16; ++w) {
      s += sums[w];
      c += kept[w];
    }
    *loss = (float)(mean ? s / c : s);
    *share = mean ? (float)(1. / c) : 1.f;
  }
}

// ------------------------------------------------------------- backward --
struct GradIn {
  const float2* stats;
  const float* entropy;     // of the rows, where grad_entropy is given
  const void* targets;
  bool wide;
  long ignore;
  const float* grad;        // for the log probability (or the loss) ...
  long grad_stride;         // ... of each row, or 0: one for all
  const float* share;       // times this, if given
  float sign;               // -1 for a loss
  const float* grad_entropy;
  long grad_entropy_stride;
};

// out_j = p_j (a + b log p_j) + c [j = t], for `n` elements of a row from
// `from` on.
template <typename T, bool ENT>
__device__ __forceinline__ void grad_slice(const T* __restrict__ x,
                                           T* __restrict__ y, long row,
                                           int vocab, int from, int n,
                                           const GradIn& in) {
  constexpr int V = Elem<T>::kVec;
  constexpr int U = 4;
  const int tid = threadIdx.x;
  const long t = target_at(in.targets, in.wide, row);
  const float2 st = in.stats[row];
  const Row r(st.x, st.y);
  float g = 0.f;
  if (t != in.ignore) {
    if (in.grad != nullptr) g = in.sign * in.grad[row * in.grad_stride];
    if (in.share != nullptr) g *= *in.share;
    if (t < 0 || t >= vocab) g = __builtin_nanf("");
  }
  float a = -g, b = 0.f;
  if (ENT) {
    b = -in.grad_entropy[row * in.grad_entropy_stride];
    a = fmaf(b, in.entropy[row], a);
    b *= kLn2;
  }
  const float inv = 1.f / r.s;
  a *= inv;
  b *= inv;
  const Parts p = Parts::of(x, n);
  const auto run = [&](auto one) {
    const auto vec = [&](u32x4 q, int i) {
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = one(Elem<T>::get(q, j));
      store16_past(y + p.head + i * V, Elem<T>::pack(f));
    };
    const T* __restrict__ xv = x + p.head;
    int i = tid;
    for (; i + (U - 1) * kThreads < p.vecs; i += U * kThreads) {
      u32x4 q[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        q[k] = load16_past(xv + (i + k * kThreads) * V);
#pragma unroll
      for (int k = 0; k < U; ++k) vec(q[k], i + k * kThreads);
    }
    for (; i < p.vecs; i += kThreads) vec(load16_past(xv + i * V), i);
    if (tid < p.edges) {
      const int j = p.edge<V>(tid);
      y[j] = Elem<T>::down(one(Elem<T>::up(x[j])));
    }
  };
  const auto from_t = [&](float e) {
    return ENT ? exp2_(e) * fmaf(b, fmaxf(e, kFloor) - r.log2s, a)
               : exp2_(e) * a;
  };
  if (t == in.ignore && !(ENT && b != 0.f)) {
    // zero, even where the row is not finite
    run([](float) { return 0.f; });
    return;
  }
  if (r.slow)
    run([&](float v) { return from_t(r.template t<true>(v)); });
  else
    run([&](float v) { return from_t(r.template t<false>(v)); });
  // The target's place once more, by the thread that has just written it.
  if (t >= from && t < (long)from + n) {
    const int hit = (int)(t - from);
    if (p.owner<V, kThreads>(hit) == tid) {
      const float v = Elem<T>::up(x[hit]);
      y[hit] = Elem<T>::down(
          from_t(r.slow ? r.template t<true>(v) : r.template t<false>(v)) +
          g);
    }
  }
}

// Each block takes `slice` elements of a row; nothing is shared between
// blocks, so a long row with few beside it is spread like any other.
template <typename T, bool ENT>
__global__ __launch_bounds__(kThreads) void row_grad_kernel(
    const T* __restrict__ logits, long row_stride, int vocab, int parts,
    int slice, GradIn in, T* __restrict__ out) {
  const long row = blockIdx.x / parts;
  const int from = (int)(blockIdx.x % parts) * slice;
  grad_slice<T, ENT>(logits + row * row_stride + from,
                     out + row * vocab + from, row, vocab, from,
                     min(slice, vocab - from), in);
}

// `out` holds the gradient for an incoming one of 1, and stays so if that
// is what came in; else the rows are worked out once more, so that they
// are rounded once.
template <typename T>
__global__ __launch_bounds__(kThreads) void rescale_rows_kernel(
    const T* __restrict__ logits, long row_stride, int vocab, int parts,
    int slice, long work, GradIn in, T* __restrict__ out) {
  if (*in.grad == 1.f) return;
  for (long i = blockIdx.x; i < work; i += gridDim.x) {
    const long row = i / parts;
    const int from = (int)(i % parts) * slice;
    grad_slice<T, false>(logits + row * row_stride + from,
                         out + row * vocab + from, row, vocab, from,
                         min(slice, vocab - from), in);
  }
}

// ---------------------------------------------------------------- host ---
bool is_wide(const torch::Tensor& targets) {
  return targets.scalar_type() == at::kLong;
}

long ceil_div(long a, long b) { return (a + b - 1) / b; }

// Logits as rows whose elements lie next to one another.
torch::Tensor as_rows(const torch::Tensor& logits) {
  auto x = logits.dim() == 2 ? logits
                             : logits.reshape({-1, logits.size(-1)});
  return x.size(1) == 1 || x.stride(1) == 1 ? x : x.contiguous();
}

void check_inputs(const torch::Tensor& logits, const torch::Tensor& targets) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(),
              "the token loss kernels cannot be traced");
  TORCH_CHECK_VALUE(logits.is_cuda(), "logits must be on a GPU");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 &&
                        logits.size(-1) < (1L << 30),
                    "logits need a last dimension of 1 to 2^30 - 1 classes");
  TORCH_CHECK_TYPE(targets.scalar_type() == at::kLong ||
                       targets.scalar_type() == at::kInt,
                   "targets must be int64 or int32, not ",
                   targets.scalar_type());
  TORCH_CHECK_VALUE(targets.device() == logits.device(),
                    "targets must be on the logits' device");
  TORCH_CHECK_VALUE(
      targets.sizes() == logits.sizes().slice(0, logits.dim() - 1),
      "targets must have the logits' shape without the last dimension: ",
      targets.sizes(), " for logits ", logits.sizes());
}

// A block and its registers for `vecs` vectors of a row or of a slice: the
// smallest that holds them; f gets BLOCK and NV as constants. False if none
// does.
//
// With many blocks a slice is one that leaves room for a second on the CU;
// with no more of them than CUs it is twice that, since a second launch to
// join slices costs more than it gives: best eight of 4 x 50001 bf16 10.2 us
// against 12.1 by 25 slices, 4 x 20000 float32 8.5 against 12.0; but 1024 x
// 20000 float32 32.6 against 24.0 us, 256 x 131072 41.9 against 31.8.
constexpr long kFewBlocks = 256;
constexpr long kHeldSlice = 4096;
constexpr long kHeldFew = 8192;
constexpr long kHeldLeast = 16;   // elements: a whole vector for certain

template <typename F>
bool with_shared(long vecs, F&& f) {
  using std::integral_constant;
  if (vecs <= 256)
    f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (vecs <= 1024)
    f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else if (vecs <= 2560)
    // every place costs, used or not: 700 rows of 2500 vectors and their
    // best five take 11.7 us with 8 to a thread, 10.4 us with 5
    f(integral_constant<int, 512>{}, integral_constant<int, 5>{});
  else if (vecs <= kHeldSlice)
    f(integral_constant<int, 512>{}, integral_constant<int, 8>{});
  else
    return false;
  return true;
}

template <typename F>
bool with_slice(long vecs, bool few, F&& f) {
  using std::integral_constant;
  if (with_shared(vecs, f)) return true;
  if (!few || vecs > kHeldFew) return false;
  f(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
  return true;
}

// A whole row, which cannot be split where its gradient leaves with it.
template <typename F>
bool with_row(long vecs, F&& f) {
  using std::integral_constant;
  if (with_shared(vecs, f)) return true;
  if (vecs <= 9216)
    f(integral_constant<int, 768>{}, integral_constant<int, 12>{});
  else if (vecs <= 16384)
    f(integral_constant<int, 1024>{}, integral_constant<int, 16>{});
  else
    return false;
  return true;
}

Where where(const torch::Tensor& x, const torch::Tensor& targets,
            long ignore, int k) {
  return Where{(long)x.stride(0), (int)x.size(1), 1, (int)x.size(1),
               targets.data_ptr(), is_wide(targets), ignore, k};
}

template <typename T, bool TOP>
void launch_stats(const torch::Tensor& x, const torch::Tensor& targets,
                  long ignore, int k, const RowOut& out) {
  const long rows = x.size(0);
  const int vocab = (int)x.size(1);
  const int step = kThreads * Elem<T>::kVec;
  const bool few =
      rows * ceil_div(vocab, kHeldFew * Elem<T>::kVec) <= kFewBlocks;
  const long most = TOP ? std::min(kJoin / k, kMaxSplits) : kMaxSplits;
  long splits = std::min(
      ceil_div(vocab, (few ? kHeldFew : kHeldSlice) * Elem<T>::kVec), most);
  Where w = where(x, targets, ignore, k);
  if (splits > 1)
    w.slice = (int)(ceil_div(ceil_div(vocab, splits), step) * step);
  splits = ceil_div(vocab, w.slice);
  w.splits = (int)splits;
  const auto stream = current_stream();
  const auto opts = torch::TensorOptions().device(x.device());
  torch::Tensor stats, keys;
  if (splits > 1) {
    stats = torch::empty({rows * splits * 3}, opts.dtype(torch::kFloat));
    if (TOP)
      keys = torch::empty({rows * splits * k}, opts.dtype(torch::kLong));
  }
  float* ps = splits > 1 ? stats.data_ptr<float>() : nullptr;
  auto* pk = splits > 1 && TOP
      ? reinterpret_cast<uint64_t*>(keys.data_ptr<int64_t>()) : nullptr;
  const T* px = static_cast<const T*>(x.data_ptr());
  const bool held = vocab >= kHeldLeast &&
      with_slice(w.slice / Elem<T>::kVec, few, [&](auto block, auto nv) {
        hipLaunchKernelGGL((held_stats_kernel<T, block.value, nv.value, TOP>),
                           grid_of(rows * splits, block.value, "rows"),
                           dim3(block.value), 0, stream, px, w, out, ps, pk);
      });
  if (!held)
    hipLaunchKernelGGL((row_stats_kernel<T, TOP>),
                       grid_of(rows * splits, kThreads, "rows"),
                       dim3(kThreads), 0, stream, px, w, out, ps, pk);
  CHECK_HIP(hipGetLastError());
  if (splits > 1) {
    hipLaunchKernelGGL((join_rows_kernel<T, TOP>),
                       grid_of(rows, kThreads, "rows"), dim3(kThreads), 0,
                       stream, px, w, out, ps, pk);
    CHECK_HIP(hipGetLastError());
  }
}

void stats_of(const torch::Tensor& x, const torch::Tensor& targets,
              long ignore, int k, const RowOut& out) {
  if (x.size(0) == 0) return;
  with_elem(x.scalar_type(), "logits", [&](auto z) {
    using T = decltype(z);
    if (k > 0)
      launch_stats<T, true>(x, targets, ignore, k, out);
    else
      launch_stats<T, false>(x, targets, ignore, 1, out);
  });
}

// The rows' losses and their gradient in one, if a row fits the registers
// of a block; else an undefined tensor, and nothing done.
torch::Tensor loss_and_grad(const torch::Tensor& x,
                            const torch::Tensor& targets, long ignore,
                            bool mean, float* share, const RowOut& out) {
  torch::Tensor grad;
  const long rows = x.size(0);
  if (rows == 0 || x.size(1) < kHeldLeast) return grad;
  const auto stream = current_stream();
  with_elem(x.scalar_type(), "logits", [&](auto z) {
    using T = decltype(z);
    const Where w = where(x, targets, ignore, 1);
    with_row(w.vocab / Elem<T>::kVec, [&](auto block, auto nv) {
      const bool count = mean && rows > kCountHere;
      if (count) {
        hipLaunchKernelGGL(count_kept_kernel, dim3(1), dim3(1024), 0, stream,
                           w.targets, w.wide, ignore, rows, share);
        CHECK_HIP(hipGetLastError());
      }
      grad = torch::empty({rows, x.size(1)}, x.options());
      hipLaunchKernelGGL((row_loss_kernel<T, block.value, nv.value>),
                         grid_of(rows, block.value, "rows"),
                         dim3(block.value), 0, stream,
                         static_cast<const T*>(x.data_ptr()), w, out, rows,
                         mean, count ? share : nullptr,
                         static_cast<T*>(grad.data_ptr()));
      CHECK_HIP(hipGetLastError());
    });
  });
  return grad;
}

// The gradient of x's rows. `ready`, if defined, has it for an incoming
// gradient of 1, and is what is returned.
torch::Tensor grad_of(const torch::Tensor& x, const GradIn& in,
                      torch::Tensor ready = torch::Tensor()) {
  const long rows = x.size(0);
  auto out = ready.defined()
      ? ready : torch::empty({rows, x.size(1)}, x.options());
  if (rows == 0) return out;
  const int vocab = (int)x.size(1);
  with_elem(x.scalar_type(), "logits", [&](auto z) {
    using T = decltype(z);
    // blocks that stay take longer slices: what comes before a slice's first
    // load is a latency of its own
    const int slice = (ready.defined() ? 32 : 4) * kThreads * Elem<T>::kVec;
    const long parts = ceil_div(vocab, slice);
    const T* px = static_cast<const T*>(x.data_ptr());
    T* py = static_cast<T*>(out.data_ptr());
    const auto stream = current_stream();
    if (ready.defined()) {
      hipLaunchKernelGGL(rescale_rows_kernel<T>,
                         dim3(std::min(rows * parts, 2048L)), dim3(kThreads),
                         0, stream, px, (long)x.stride(0), vocab, (int)parts,
                         slice, rows * parts, in, py);
    } else {
      const dim3 grid = grid_of(rows * parts, kThreads, "rows");
      if (in.grad_entropy != nullptr)
        hipLaunchKernelGGL((row_grad_kernel<T, true>), grid, dim3(kThreads),
                           0, stream, px, (long)x.stride(0), vocab,
                           (int)parts, slice, in, py);
      else
        hipLaunchKernelGGL((row_grad_kernel<T, false>), grid, dim3(kThreads),
                           0, stream, px, (long)x.stride(0), vocab,
                           (int)parts, slice, in, py);
    }
    CHECK_HIP(hipGetLastError());
  });
  return out;
}

// The number of the capture that the stream is in; 0 for none.
unsigned long long capture_id() {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  CHECK_HIP(hipStreamGetCaptureInfo(current_stream(), &status, &id));
  return status == hipStreamCaptureStatusActive ? id + 1 : 0;
}

// A gradient that comes back from autograd: float32, and how far apart its
// elements are (an expanded one has stride 0).
torch::Tensor flat_grad(const torch::Tensor& g) {
  auto f = g.scalar_type() == at::kFloat ? g : g.to(at::kFloat);
  return f.dim() <= 1 ? f : f.reshape({-1});
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

enum Reduction { kNone = 0, kMean = 1, kSum = 2 };

void refuse_second_order() {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "the token loss has no second derivative: it cannot be "
              "differentiated with create_graph=True");
}

GradIn loss_grad_in(const torch::Tensor& g, const torch::Tensor& targets,
                    const torch::Tensor& work, long rows, long ignore,
                    bool none) {
  const float* w = work.data_ptr<float>();
  return GradIn{reinterpret_cast<const float2*>(w), nullptr,
                targets.data_ptr(), is_wide(targets), ignore,
                g.data_ptr<float>(), none ? (long)g.stride(0) : 0L,
                none ? nullptr : w + 3 * rows, -1.f, nullptr, 0L};
}

// The loss's gradient as a function of the logits and of the gradient g
// that comes in, d_j = c (p_j - [j = t]) with c = g, times a mean's share.
// For a gradient e of d that comes in in turn, with m = sum_j p_j e_j:
//
//   of x_j: c p_j (e_j - m)        of g: share (m - e_t), summed over the
//                                  rows where g is one for all
//
// This is rare, and made of torch's own operations, which can be
// differentiated further.
struct CrossEntropyGrad : torch::autograd::Function<CrossEntropyGrad> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor x,
                               torch::Tensor grad, torch::Tensor targets,
                               torch::Tensor work, int64_t ignore,
                               bool none) {
    c10::DeviceGuard guard(x.device());
    ctx->save_for_backward({x, grad, targets, work});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["none"] = none;
    const auto g = flat_grad(grad);
    return grad_of(x, loss_grad_in(g, targets, work, x.size(0), ignore,
                                   none));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto& x = saved[0];
    const auto& targets = saved[2];
    const bool none = ctx->saved_data["none"].toBool();
    c10::DeviceGuard guard(x.device());
    const auto kept = targets.ne(ctx->saved_data["ignore"].toInt());
    const auto there = targets.ge(0).logical_and(targets.lt(x.size(1)));
    // a row that takes no part may be anything; it is left out first
    const auto p = x.to(at::kFloat)
                       .masked_fill(kept.logical_not().unsqueeze(1), 0)
                       .softmax(1);
    const auto e = grads[0].to(at::kFloat);
    const auto m = (p * e).sum(1, true);
    auto c = kept.logical_and(there).to(at::kFloat);
    c = c.masked_fill(kept.logical_and(there.logical_not()),
                      std::numeric_limits<float>::quiet_NaN());
    if (!none) c = c * saved[3][3 * x.size(0)];
    const auto g = saved[1].to(at::kFloat);
    const auto at = targets.to(at::kLong)
                        .masked_fill(there.logical_not(), 0).unsqueeze(1);
    auto dg = (c.unsqueeze(1) * (m - e.gather(1, at))).squeeze(1)
                  .masked_fill(kept.logical_not(), 0);
    if (!none) dg = dg.sum();
    const auto dx = ((c * g).unsqueeze(1) * p * (e - m))
                        .masked_fill(kept.logical_not().unsqueeze(1), 0);
    return {dx.to(x.scalar_type()), dg.to(saved[1].scalar_type()),
            torch::Tensor(), torch::Tensor(), torch::Tensor(),
            torch::Tensor()};
  }
};

// The forward pass leaves the gradient for an incoming 1, and the first
// backward pass hands it on. A second one works it out again, since by then
// it is the caller's own; so does one that is captured into another graph
// than the forward pass, which may be replayed alone.
//
// `twice`: the backward pass may itself be differentiated; it is then a
// function of its own.
struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor x,
                               torch::Tensor targets, int64_t ignore,
                               int64_t reduction, bool with_grad,
                               bool twice) {
    c10::DeviceGuard guard(x.device());
    const long rows = x.size(0);
    const auto f32 = x.options().dtype(torch::kFloat);
    // stats of each row, each row's loss, and what a mean multiplies by
    auto work = torch::empty({3 * rows + 1}, f32);
    auto* stats = reinterpret_cast<float2*>(work.data_ptr<float>());
    float* each = work.data_ptr<float>() + 2 * rows;
    float* share = each + rows;
    torch::Tensor loss;
    if (reduction == kNone) {
      loss = torch::empty({rows}, f32);
      each = loss.data_ptr<float>();
    } else {
      loss = torch::empty({}, f32);
    }
    RowOut out{stats, each, nullptr, nullptr, nullptr, -1.f};
    torch::Tensor ready;
    if (with_grad && reduction != kNone)
      ready = loss_and_grad(x, targets, ignore, reduction == kMean, share,
                            out);
    if (!ready.defined()) stats_of(x, targets, ignore, 0, out);
    if (reduction != kNone) {
      hipLaunchKernelGGL(reduce_loss_kernel, dim3(1), dim3(1024), 0,
                         current_stream(), each, targets.data_ptr(),
                         is_wide(targets), (long)ignore, rows,
                         reduction == kMean, loss.data_ptr<float>(), share);
      CHECK_HIP(hipGetLastError());
    }
    ctx->save_for_backward({x, targets, work});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["twice"] = twice;
    if (ready.defined()) {
      ctx->saved_data["capture"] = (int64_t)capture_id();
      ctx->saved_data["ready"] = ready;
    }
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto& x = saved[0];
    const bool none = ctx->saved_data["reduction"].toInt() == kNone;
    const int64_t ignore = ctx->saved_data["ignore"].toInt();
    if (at::GradMode::is_enabled()) {
      if (!ctx->saved_data["twice"].toBool()) refuse_second_order();
      return {CrossEntropyGrad::apply(x, grads[0], saved[1], saved[2], ignore,
                                      none),
              torch::Tensor(), torch::Tensor(), torch::Tensor(),
              torch::Tensor(), torch::Tensor()};
    }
    c10::DeviceGuard guard(x.device());
    const auto g = flat_grad(grads[0]);
    const GradIn in = loss_grad_in(g, saved[1], saved[2], x.size(0), ignore,
                                   none);
    torch::Tensor ready;
    const auto at = ctx->saved_data.find("ready");
    if (at != ctx->saved_data.end() &&
        ctx->saved_data["capture"].toInt() == (int64_t)capture_id()) {
      ready = at->second.toTensor();
      ctx->saved_data.erase("ready");
    }
    return {grad_of(x, in, ready), torch::Tensor(), torch::Tensor(),
            torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, torch::Tensor x,
                               torch::Tensor targets, int64_t k,
                               int64_t ignore) {
    c10::DeviceGuard guard(x.device());
    const long rows = x.size(0);
    const auto f32 = x.options().dtype(torch::kFloat);
    auto stats = torch::empty({rows, 2}, f32);
    auto lp = torch::empty({rows}, f32);
    auto entropy = torch::empty({rows}, f32);
    auto values = torch::empty({rows, k}, f32);
    auto ids = torch::empty({rows, k}, x.options().dtype(torch::kLong));
    RowOut out{reinterpret_cast<float2*>(stats.data_ptr<float>()),
               lp.data_ptr<float>(), entropy.data_ptr<float>(),
               values.data_ptr<float>(), ids.data_ptr<int64_t>(), 1.f};
    stats_of(x, targets, ignore, (int)k, out);
    ctx->save_for_backward({x, targets, stats, entropy});
    ctx->saved_data["ignore"] = ignore;
    ctx->mark_non_differentiable({values, ids});
    ctx->set_materialize_grads(false);
    return {lp, entropy, values, ids};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_second_order();
    const auto saved = ctx->get_saved_variables();
    const auto& x = saved[0];
    c10::DeviceGuard guard(x.device());
    torch::Tensor gl, ge;
    if (grads[0].defined()) gl = flat_grad(grads[0]);
    if (grads[1].defined()) ge = flat_grad(grads[1]);
    GradIn in{reinterpret_cast<const float2*>(saved[2].data_ptr<float>()),
              saved[3].data_ptr<float>(), saved[1].data_ptr(),
              is_wide(saved[1]), (long)ctx->saved_data["ignore"].toInt(),
              gl.defined() ? gl.data_ptr<float>() : nullptr,
              gl.defined() ? (long)gl.stride(0) : 0L, nullptr, 1.f,
              ge.defined() ? ge.data_ptr<float>() : nullptr,
              ge.defined() ? (long)ge.stride(0) : 0L};
    return {grad_of(x, in), torch::Tensor(), torch::Tensor(),
            torch::Tensor()};
  }
};

}  // namespace

torch::Tensor cross_entropy(const torch::Tensor& logits,
                            const torch::Tensor& targets, int64_t ignore,
                            int64_t reduction, bool scaled, bool twice) {
  check_inputs(logits, targets);
  TORCH_CHECK_VALUE(reduction >= kNone && reduction <= kSum,
                    "unknown reduction ", reduction);
  with_elem(logits.scalar_type(), "logits", [](auto) {});
  c10::DeviceGuard guard(logits.device());
  auto loss = CrossEntropy::apply(
      as_rows(logits), targets.reshape({-1}).contiguous(), ignore, reduction,
      !scaled && at::GradMode::is_enabled() && logits.requires_grad(), twice);
  return reduction == kNone && targets.dim() != 1
      ? loss.view(targets.sizes()) : loss;
}

std::vector<torch::Tensor> token_log_probs(const torch::Tensor& logits,
                                           const torch::Tensor& targets,
                                           int64_t k, int64_t ignore) {
  check_inputs(logits, targets);
  TORCH_CHECK_VALUE(k >= 0 && k <= kMaxTop && k <= logits.size(-1),
                    "top_k must be between 0 and the number of classes, at "
                    "most ", kMaxTop, ": ", k);
  with_elem(logits.scalar_type(), "logits", [](auto) {});
  c10::DeviceGuard guard(logits.device());
  auto r = TokenLogProbs::apply(
      as_rows(logits), targets.reshape({-1}).contiguous(), k, ignore);
  if (targets.dim() != 1) {
    auto shape = targets.sizes().vec();
    r[0] = r[0].view(shape);
    r[1] = r[1].view(shape);
    shape.push_back(k);
    r[2] = r[2].view(shape);
    r[3] = r[3].view(shape);
  }
  return r;
}

}  // namespace mgx
