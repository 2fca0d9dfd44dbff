// Cross entropy with its gradient, and log probabilities of given tokens
// with the row's entropy and its best alternatives, gfx950.
//
// For a row x of V logits, with m = max x, s = sum e^(x_j - m) and
// u = sum e^(x_j - m) (x_j - m):
//
//   log p_j = (x_j - m) - log s          entropy H = log s - u / s
//   d log p_t / d x_j = [j = t] - p_j    d H / d x_j = -p_j (log p_j + H)
//
// All of it is bound by memory: a row is read once for m, s and u (kept
// running, in 32 bits, by rescaling when the maximum grows), and a
// gradient is one more read and a write. Where the loss is to be
// differentiated its gradient leaves the forward pass, from a row that is
// still in registers, so that the logits are read once in all; see
// loss_grad_kernel.
//
// A logit of -inf has p = 0 and adds nothing anywhere (x - m is held at
// kFloor, where e^ is an exact 0, so that no 0 * inf arises). A row with
// a NaN, a +inf or nothing but -inf has no distribution and gives NaN, as
// torch's log_softmax does. A target outside [0, V) that is not
// ignore_index is never read: it gives NaN, in the value and the gradient.
#include <hip/hip_runtime.h>

#include "lm_common.h"

#include <torch/csrc/autograd/custom_function.h>

#include <algorithm>
#include <tuple>
#include <vector>

namespace mgx {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kFloor = -200.f;       // 2^(kFloor * log2 e) is 0 in float32
constexpr float kInf = __builtin_inff();
constexpr int kThreads = 256;
constexpr int kMaxTop = 64;
constexpr int kCandidates = 512;       // of one block's search for the best
constexpr int kJoin = 1024;            // keys that the join of a row takes
constexpr int kMaxSplits = 64;

__device__ __forceinline__ float exp_diff(float d) {
  d = d < kFloor ? kFloor : d;         // a NaN stays one
  return __builtin_amdgcn_exp2f(d * kLog2e);
}

__device__ __forceinline__ long target_at(const void* p, bool wide, long i) {
  return wide ? static_cast<const long*>(p)[i]
              : static_cast<long>(static_cast<const int*>(p)[i]);
}

// Running maximum and sums of part of a row. m is -inf where nothing
// finite was seen; the sums are then taken against 0 and are 0 (or NaN).
struct Stat {
  float m = -kInf, s = 0.f, u = 0.f;

  __device__ __forceinline__ void raise(float to) {
    if (to > m) {
      if (s != 0.f) {
        const float d = m - to;
        const float f = exp_diff(d);
        u = f == 0.f ? 0.f * s : (u + s * d) * f;   // a NaN in s stays
        s *= f;
      }
      m = to;
    }
  }
  template <bool ENT>
  __device__ __forceinline__ void add(float x) {
    float d = x - (m == -kInf ? 0.f : m);
    d = d < kFloor ? kFloor : d;
    const float e = __builtin_amdgcn_exp2f(d * kLog2e);
    s += e;
    if (ENT) u = fmaf(e, d, u);
  }
  __device__ __forceinline__ void merge(float bm, float bs, float bu) {
    Stat b;
    b.m = bm; b.s = bs; b.u = bu;
    const float to = fmaxf(m, bm);
    raise(to);
    b.raise(to);
    s += b.s;
    u += b.u;
  }
};

template <bool ENT>
__device__ __forceinline__ void wave_merge(Stat& a) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float m = __shfl_xor(a.m, off, 64);
    const float s = __shfl_xor(a.s, off, 64);
    const float u = ENT ? __shfl_xor(a.u, off, 64) : 0.f;
    a.merge(m, s, u);
  }
}

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
  uint32_t group[kThreads];
  uint64_t found[kCandidates];
  uint64_t wave[kThreads / 64];
  uint32_t least;
  int count;
};

// The k best keys of x[0..n), written to out[0..k) best first, zeros where
// n < k. `top` is the largest value that this thread has seen in its share
// of the row. The k-th largest of the 256 threads' maxima is at most the
// k-th largest value, so everything from there up is gathered (about k
// values unless many are equal) and ranked; if they do not fit, k rounds
// over the row take the best below the last one. `base` is added to the
// indices.
template <typename T, typename F>
__device__ void best_of(const T* __restrict__ x, int n, int base, int k,
                        float top, Best& b, F&& put) {
  constexpr int V = Elem<T>::kVec;
  const int tid = threadIdx.x;
  b.group[tid] = order_of(top);
  if (tid == 0) b.count = 0;
  __syncthreads();
  if (tid < 64) {
    uint32_t g[kThreads / 64];
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) g[i] = b.group[tid + 64 * i];
    // highest threshold that k of the groups reach, bit by bit; the bits
    // that are left out only lower it
    uint32_t least = 0;
    constexpr int kLast = sizeof(T) == 2 ? 13 : 8;
    for (int bit = 31; bit >= kLast; --bit) {
      const uint32_t c = least | (1u << bit);
      int have = 0;
#pragma unroll
      for (int i = 0; i < kThreads / 64; ++i)
        have += __popcll(__ballot(g[i] >= c));
      if (have >= k) least = c;
    }
    if (tid == 0) b.least = least;
  }
  __syncthreads();
  const uint32_t least = b.least;
  const auto gather = [&](float v, int j) {
    if (order_of(v) >= least) {
      const int at = atomicAdd(&b.count, 1);
      if (at < kCandidates) b.found[at] = key_of(v, base + j);
    }
  };
  const int whole = n / V * V;
  int i = tid * V;
  for (; i + 3 * kThreads * V < whole; i += 4 * kThreads * V) {
    u32x4 r[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) r[w] = load16(x + i + w * kThreads * V);
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j)
        gather(Elem<T>::get(r[w], j), i + w * kThreads * V + j);
  }
  for (; i < whole; i += kThreads * V) {
    const u32x4 r = load16(x + i);
#pragma unroll
    for (int j = 0; j < V; ++j) gather(Elem<T>::get(r, j), i + j);
  }
  if (whole + tid < n) gather(Elem<T>::up(x[whole + tid]), whole + tid);
  __syncthreads();
  const int count = b.count;
  if (count <= kCandidates) {
    for (int c = tid; c < count; c += kThreads) {
      const uint64_t key = b.found[c];
      int rank = 0;
      for (int o = 0; o < count; ++o) rank += b.found[o] > key;
      if (rank < k) put(rank, key);
    }
    for (int r = count + tid; r < k; r += kThreads) put(r, 0);
    return;
  }
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    for (int j = tid; j < n; j += kThreads) {
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
    for (int w = 0; w < kThreads / 64; ++w)
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

__device__ __forceinline__ void finish_row(const Stat& a, long row, int vocab,
                                           float x_target, long target,
                                           long ignore, const RowOut& out) {
  const float log_s = logf(a.s);
  float lp;
  if (target == ignore)
    lp = 0.f;
  else if (target < 0 || target >= vocab)
    lp = __builtin_nanf("");
  else
    lp = (x_target - a.m) - log_s;
  out.log_probs[row] = target == ignore ? 0.f : out.sign * lp;
  out.stats[row] = make_float2(a.m, a.s);
  if (out.entropy != nullptr) out.entropy[row] = log_s - a.u / a.s;
}

// One block a row, or `splits` blocks a row that each leave what they
// found of their slice for join_rows_kernel: with few rows one block
// cannot draw the bandwidth of the card.
template <typename T, bool ENT, bool TOP>
__global__ __launch_bounds__(kThreads) void row_stats_kernel(
    const T* __restrict__ logits, long row_stride, int vocab, int splits,
    int slice, const void* __restrict__ targets, bool wide, long ignore,
    int k, RowOut out, float* __restrict__ part_stats,
    uint64_t* __restrict__ part_keys) {
  constexpr int V = Elem<T>::kVec;
  __shared__ float waves[kThreads / 64][3];
  __shared__ typename std::conditional<TOP, Best, int>::type best;
  const long row = blockIdx.x / splits;
  const int part = blockIdx.x % splits;
  const int from = part * slice;
  const int n = min(slice, vocab - from);
  const T* __restrict__ x = logits + row * row_stride + from;
  const int tid = threadIdx.x;

  Stat a;
  float top = -kInf;
  const int whole = n / V * V;
  int i = tid * V;
  for (; i + 3 * kThreads * V < whole; i += 4 * kThreads * V) {
    u32x4 r[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) r[w] = load16(x + i + w * kThreads * V);
    float c = -kInf;
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j) c = fmaxf(c, Elem<T>::get(r[w], j));
    a.raise(c);
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j) a.template add<ENT>(Elem<T>::get(r[w], j));
  }
  for (; i < whole; i += kThreads * V) {
    const u32x4 r = load16(x + i);
    float c = -kInf;
#pragma unroll
    for (int j = 0; j < V; ++j) c = fmaxf(c, Elem<T>::get(r, j));
    a.raise(c);
#pragma unroll
    for (int j = 0; j < V; ++j) a.template add<ENT>(Elem<T>::get(r, j));
  }
  if (whole + tid < n) {
    const float v = Elem<T>::up(x[whole + tid]);
    a.raise(fmaxf(v, -kInf));
    a.template add<ENT>(v);
  }
  top = a.m;
  wave_merge<ENT>(a);
  if ((tid & 63) == 0) {
    float* w = waves[tid >> 6];
    w[0] = a.m; w[1] = a.s; w[2] = a.u;
  }
  __syncthreads();
  a = Stat();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w)
    a.merge(waves[w][0], waves[w][1], waves[w][2]);

  if (tid == 0) {
    if (splits == 1) {
      const long t = target_at(targets, wide, row);
      const float xt =
          t >= 0 && t < vocab ? Elem<T>::up(x[t]) : 0.f;
      finish_row(a, row, vocab, xt, t, ignore, out);
    } else {
      float* p = part_stats + 3 * (row * splits + part);
      p[0] = a.m; p[1] = a.s; p[2] = a.u;
    }
  }
  if constexpr (TOP) {
    if (splits == 1) {
      const float m = a.m, log_s = logf(a.s);
      best_of<T>(x, n, 0, k, top, best, [&](int r, uint64_t key) {
        out.top_ids[row * k + r] = static_cast<int>(~(uint32_t)key);
        out.top_values[row * k + r] = (value_of(key >> 32) - m) - log_s;
      });
    } else {
      uint64_t* keys = part_keys + (row * splits + part) * k;
      best_of<T>(x, n, from, k, top, best,
                 [&](int r, uint64_t key) { keys[r] = key; });
    }
  }
}

template <typename T, bool ENT, bool TOP>
__global__ __launch_bounds__(kThreads) void join_rows_kernel(
    const T* __restrict__ logits, long row_stride, int vocab, int splits,
    const void* __restrict__ targets, bool wide, long ignore, int k,
    RowOut out, const float* __restrict__ part_stats,
    const uint64_t* __restrict__ part_keys) {
  __shared__ uint64_t keys[TOP ? kJoin : 1];
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  Stat a;
  const int lane = tid & 63;
  if (lane < splits) {
    const float* p = part_stats + 3 * (row * splits + lane);
    a.m = p[0]; a.s = p[1]; a.u = p[2];
  }
  wave_merge<ENT>(a);
  if (tid == 0) {
    const long t = target_at(targets, wide, row);
    const float xt = t >= 0 && t < vocab
        ? Elem<T>::up(logits[row * row_stride + t]) : 0.f;
    finish_row(a, row, vocab, xt, t, ignore, out);
  }
  if constexpr (TOP) {
    const int count = splits * k;      // at most kJoin, by the host
    for (int i = tid; i < count; i += kThreads)
      keys[i] = part_keys[row * count + i];
    __syncthreads();
    const float log_s = logf(a.s);
    for (int i = tid; i < count; i += kThreads) {
      const uint64_t key = keys[i];
      if (key == 0) continue;
      int rank = 0;
      for (int o = 0; o < count && rank < k; ++o) rank += keys[o] > key;
      if (rank < k) {
        out.top_ids[row * k + rank] = static_cast<int>(~(uint32_t)key);
        out.top_values[row * k + rank] = (value_of(key >> 32) - a.m) - log_s;
      }
    }
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

// out_j = p_j (a + b log p_j) + c [j = t]. Each block takes `slice`
// elements of a row; nothing is shared between blocks, so a long row with
// few beside it is spread like any other.
template <typename T, bool ENT>
__global__ __launch_bounds__(kThreads) void row_grad_kernel(
    const T* __restrict__ logits, long row_stride, int vocab, int parts,
    int slice, GradIn in, T* __restrict__ out) {
  constexpr int V = Elem<T>::kVec;
  const long row = blockIdx.x / parts;
  const int from = (int)(blockIdx.x % parts) * slice;
  const int n = min(slice, vocab - from);
  const T* __restrict__ x = logits + row * row_stride + from;
  T* __restrict__ y = out + row * vocab + from;
  const int tid = threadIdx.x;

  const long t = target_at(in.targets, in.wide, row);
  const float2 st = in.stats[row];
  float g = 0.f;
  if (t != in.ignore) {
    if (in.grad != nullptr) g = in.sign * in.grad[row * in.grad_stride];
    if (in.share != nullptr) g *= *in.share;
    if (t < 0 || t >= vocab) g = __builtin_nanf("");
  }
  const float inv = 1.f / st.y, log_s = logf(st.y), m = st.x;
  float a = -g, b = 0.f;
  if (ENT) {
    b = -in.grad_entropy[row * in.grad_entropy_stride];
    a = fmaf(b, in.entropy[row], a);
  }
  // an ignored row's gradient is zero, even where the row is not finite
  const bool nothing = t == in.ignore && !(ENT && b != 0.f);
  a *= inv;
  b *= inv;
  const int hit = (t >= from && t < (long)from + n) ? (int)(t - from) : -1;
  const auto one = [&](float v, int j) {
    float d = v - m;
    d = d < kFloor ? kFloor : d;
    const float e = __builtin_amdgcn_exp2f(d * kLog2e);
    float r = ENT ? e * fmaf(b, d - log_s, a) : e * a;
    if (j == hit) r += g;
    return nothing ? 0.f : r;
  };
  const int whole = n / V * V;
  int i = tid * V;
  for (; i + 3 * kThreads * V < whole; i += 4 * kThreads * V) {
    u32x4 r[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) r[w] = load16(x + i + w * kThreads * V);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j)
        f[j] = one(Elem<T>::get(r[w], j), i + w * kThreads * V + j);
      store16(y + i + w * kThreads * V, Elem<T>::pack(f));
    }
  }
  for (; i < whole; i += kThreads * V) {
    const u32x4 r = load16(x + i);
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = one(Elem<T>::get(r, j), i + j);
    store16(y + i, Elem<T>::pack(f));
  }
  if (whole + tid < n)
    y[whole + tid] =
        Elem<T>::down(one(Elem<T>::up(x[whole + tid]), whole + tid));
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

template <typename T, bool ENT, bool TOP>
void launch_stats(const torch::Tensor& x, const torch::Tensor& targets,
                  long ignore, int k, const RowOut& out) {
  const long rows = x.size(0);
  const int vocab = (int)x.size(1);
  const int step = kThreads * Elem<T>::kVec;
  // Blocks enough for the card, and a slice that is worth a block.
  long splits = std::min({ceil_div(512, rows), ceil_div(vocab, 4L * step),
                          (long)kMaxSplits});
  if (TOP) splits = std::min(splits, (long)(kJoin / k));
  splits = std::max(splits, 1L);
  const int slice = splits == 1
      ? vocab : (int)(ceil_div(ceil_div(vocab, splits), step) * step);
  splits = ceil_div(vocab, slice);
  TORCH_CHECK_VALUE(rows * splits < (1L << 31), "too many rows");
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
  hipLaunchKernelGGL((row_stats_kernel<T, ENT, TOP>), dim3(rows * splits),
                     dim3(kThreads), 0, stream, px, (long)x.stride(0), vocab,
                     (int)splits, slice, targets.data_ptr(),
                     is_wide(targets), ignore, k, out, ps, pk);
  CHECK_HIP(hipGetLastError());
  if (splits > 1) {
    hipLaunchKernelGGL((join_rows_kernel<T, ENT, TOP>), dim3(rows),
                       dim3(kThreads), 0, stream, px, (long)x.stride(0),
                       vocab, (int)splits, targets.data_ptr(),
                       is_wide(targets), ignore, k, out, ps, pk);
    CHECK_HIP(hipGetLastError());
  }
}

void stats_of(const torch::Tensor& x, const torch::Tensor& targets,
              long ignore, int k, const RowOut& out) {
  if (x.size(0) == 0) return;
  with_elem(x.scalar_type(), "logits", [&](auto z) {
    using T = decltype(z);
    if (k > 0)
      launch_stats<T, true, true>(x, targets, ignore, k, out);
    else if (out.entropy != nullptr)
      launch_stats<T, true, false>(x, targets, ignore, 1, out);
    else
      launch_stats<T, false, false>(x, targets, ignore, 1, out);
  });
}

torch::Tensor grad_of(const torch::Tensor& x, const GradIn& in) {
  auto out = torch::empty({x.size(0), x.size(1)}, x.options());
  const long rows = x.size(0);
  if (rows == 0) return out;
  const int vocab = (int)x.size(1);
  with_elem(x.scalar_type(), "logits", [&](auto z) {
    using T = decltype(z);
    const int step = kThreads * Elem<T>::kVec;
    const long parts = ceil_div(vocab, 4L * step);
    const int slice = 4 * step;
    TORCH_CHECK_VALUE(rows * parts < (1L << 31), "too many rows");
    const T* px = static_cast<const T*>(x.data_ptr());
    T* py = static_cast<T*>(out.data_ptr());
    const auto stream = current_stream();
    if (in.grad_entropy != nullptr)
      hipLaunchKernelGGL((row_grad_kernel<T, true>), dim3(rows * parts),
                         dim3(kThreads), 0, stream, px, (long)x.stride(0),
                         vocab, (int)parts, slice, in, py);
    else
      hipLaunchKernelGGL((row_grad_kernel<T, false>), dim3(rows * parts),
                         dim3(kThreads), 0, stream, px, (long)x.stride(0),
                         vocab, (int)parts, slice, in, py);
    CHECK_HIP(hipGetLastError());
  });
  return out;
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

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor x,
                               torch::Tensor targets, int64_t ignore,
                               int64_t reduction) {
    c10::DeviceGuard guard(x.device());
    const auto f32 = x.options().dtype(torch::kFloat);
    auto stats = torch::empty({x.size(0), 2}, f32);
    auto each = torch::empty({x.size(0)}, f32);
    RowOut out{reinterpret_cast<float2*>(stats.data_ptr<float>()),
               each.data_ptr<float>(), nullptr, nullptr, nullptr, -1.f};
    stats_of(x, targets, ignore, 0, out);
    torch::Tensor share;
    torch::Tensor loss = each;
    if (reduction != kNone) {
      loss = torch::empty({}, f32);
      share = torch::empty({}, f32);
      hipLaunchKernelGGL(reduce_loss_kernel, dim3(1), dim3(1024), 0,
                         current_stream(), each.data_ptr<float>(),
                         targets.data_ptr(), is_wide(targets), (long)ignore,
                         (long)x.size(0), reduction == kMean,
                         loss.data_ptr<float>(), share.data_ptr<float>());
      CHECK_HIP(hipGetLastError());
    }
    ctx->save_for_backward({x, targets, stats, share});
    ctx->saved_data["ignore"] = ignore;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_second_order();
    const auto saved = ctx->get_saved_variables();
    const auto& x = saved[0];
    c10::DeviceGuard guard(x.device());
    const auto g = flat_grad(grads[0]);
    const auto& share = saved[3];
    GradIn in{reinterpret_cast<const float2*>(saved[2].data_ptr<float>()),
              nullptr, saved[1].data_ptr(), is_wide(saved[1]),
              (long)ctx->saved_data["ignore"].toInt(),
              g.data_ptr<float>(),
              share.defined() ? 0L : (long)g.stride(0),
              share.defined() ? share.data_ptr<float>() : nullptr, -1.f,
              nullptr, 0L};
    return {grad_of(x, in), torch::Tensor(), torch::Tensor(),
            torch::Tensor()};
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
                            int64_t reduction) {
  check_inputs(logits, targets);
  TORCH_CHECK_VALUE(reduction >= kNone && reduction <= kSum,
                    "unknown reduction ", reduction);
  with_elem(logits.scalar_type(), "logits", [](auto) {});
  c10::DeviceGuard guard(logits.device());
  auto loss = CrossEntropy::apply(
      as_rows(logits), targets.reshape({-1}).contiguous(), ignore, reduction);
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
