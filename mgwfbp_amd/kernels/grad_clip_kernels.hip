// Global gradient norm over many tensors, and clipping by it, gfx950.
//
//   norm = sqrt(sum over all tensors of sum g^2)
//   y    = g * min(1, max_norm / (norm + eps))
//
// Bound by memory: one read for the norm, one read and one write for the
// scaling. Two launches for up to kMaxTensors tensors: the tensors'
// addresses travel as kernel arguments, so there is no table to build,
// copy or go stale, and a captured graph keeps what it needs. Squares are
// summed in 64 bits, which costs nothing beside the loads and neither
// overflows nor loses squares of small gradients; each block leaves one
// partial sum and every block of the second launch adds the partial sums
// up in the same order, so the result has no atomics in it and is the
// same on every run. Measured, 300M elements, 16-bit matrices and 32-bit
// vectors: norm 90 us (6.7 TB/s), scaling into new tensors 200 us (6.0 TB/s).
#include <hip/hip_runtime.h>

#include "lm_common.h"

#include <algorithm>
#include <tuple>
#include <vector>

namespace mgx {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTensors = 120;       // their addresses fit 4 KB of arguments
constexpr int kChunk = 16384;          // elements of one block's turn
constexpr int kMaxBlocks = 1024;       // that leave a partial sum
constexpr int kMaxScaleBlocks = 2048;  // that stay and take several chunks

struct TensorList {
  const void* src[kMaxTensors];
  void* dst[kMaxTensors];              // of the second launch
  long numel[kMaxTensors];
  int first[kMaxTensors + 1];          // each tensor's first chunk
  unsigned char type[kMaxTensors];     // 0 float32, 1 bfloat16, 2 float16
  int count;
};
static_assert(sizeof(TensorList) <= 3600, "kernel arguments");

// The tensor that a chunk lies in. `chunk` is the same for the whole
// block, so these are scalar loads and branches.
__device__ __forceinline__ int tensor_of(const TensorList& l, int chunk) {
  int lo = 0, hi = l.count;            // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// Together larger than this, the gradients go past the 256 MB cache both
// times; below, the second pass finds them there. Three passes over 64 and
// 256 MB of gradients that were not there before: 36 and 159 us through the
// cache, 40 and 137 us past it.
constexpr long kPastBytes = 128L << 20;

template <bool PAST>
__device__ __forceinline__ u32x4 load_(const void* p) {
  return PAST ? load16_past(p) : load16(p);
}
template <bool PAST>
__device__ __forceinline__ void store_(void* p, u32x4 v) {
  if (PAST) store16_past(p, v); else store16(p, v);
}

template <bool PAST, typename T>
__device__ __forceinline__ double squares(const T* __restrict__ p, int n) {
  constexpr int V = Elem<T>::kVec;
  constexpr int kStep = kThreads * V;
  double a0 = 0., a1 = 0.;
  const int whole = n / V * V;
  int i = threadIdx.x * V;
  for (; i + 3 * kStep < whole; i += 4 * kStep) {
    u32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = load_<PAST>(p + i + u * kStep);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const double x = Elem<T>::get(v[u], j);
        const double y = Elem<T>::get(v[u], j + 1);
        a0 = fma(x, x, a0);
        a1 = fma(y, y, a1);
      }
  }
  for (; i < whole; i += kStep) {
    const u32x4 v = load_<PAST>(p + i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double x = Elem<T>::get(v, j);
      a0 = fma(x, x, a0);
    }
  }
  if (whole + (int)threadIdx.x < n) {
    const double x = Elem<T>::up(p[whole + threadIdx.x]);
    a1 = fma(x, x, a1);
  }
  return a0 + a1;
}

__device__ __forceinline__ double block_sum(double x, double* lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0.;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) s += lds[w];
  return s;
}

template <bool PAST>
__global__ __launch_bounds__(kThreads) void norm_partials_kernel(
    const TensorList l, double* __restrict__ partials) {
  __shared__ double lds[kThreads / 64];
  const int chunks = l.first[l.count];
  double acc = 0.;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    const long start = (long)(c - l.first[t]) * kChunk;
    const int n = (int)min((long)kChunk, l.numel[t] - start);
    switch (l.type[t]) {
      case 0:
        acc += squares<PAST>(static_cast<const float*>(l.src[t]) + start, n);
        break;
      case 1:
        acc += squares<PAST>(
            static_cast<const __hip_bfloat16*>(l.src[t]) + start, n);
        break;
      default:
        acc += squares<PAST>(static_cast<const __half*>(l.src[t]) + start, n);
    }
  }
  const double s = block_sum(acc, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

template <bool PAST, typename T>
__device__ __forceinline__ void scaled(const T* p, T* q, int n, float f) {
  constexpr int V = Elem<T>::kVec;
  constexpr int kStep = kThreads * V;
  const int whole = n / V * V;
  int i = threadIdx.x * V;
  for (; i + 3 * kStep < whole; i += 4 * kStep) {
    u32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = load_<PAST>(p + i + u * kStep);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float x[V];
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = Elem<T>::get(v[u], j) * f;
      store_<PAST>(q + i + u * kStep, Elem<T>::pack(x));
    }
  }
  for (; i < whole; i += kStep) {
    const u32x4 v = load_<PAST>(p + i);
    float x[V];
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = Elem<T>::get(v, j) * f;
    store_<PAST>(q + i, Elem<T>::pack(x));
  }
  if (whole + (int)threadIdx.x < n)
    q[whole + threadIdx.x] =
        Elem<T>::down(Elem<T>::up(p[whole + threadIdx.x]) * f);
}

// Also the whole of the norm alone, with no tensors in the list.
template <bool PAST>
__global__ __launch_bounds__(kThreads) void clip_scale_list_kernel(
    const TensorList l, const double* __restrict__ partials, int npartials,
    double max_norm, double eps, float* __restrict__ norm_out) {
  __shared__ double lds[kThreads / 64];
  double acc = 0.;
  for (int i = threadIdx.x; i < npartials; i += kThreads) acc += partials[i];
  const double norm = sqrt(block_sum(acc, lds));
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0)
    *norm_out = (float)norm;
  const double c = max_norm / (norm + eps);
  const float f = c >= 1. ? 1.f : (float)c;   // a NaN stays one
  const int chunks = l.first[l.count];
  // From the last chunk back: what the first launch read last is still in
  // the 256 MB cache. Past the cache in order, and a block for each chunk:
  // 300M elements take 311 us by 2048 blocks from the back, 295 us so.
  for (int k = blockIdx.x; k < chunks; k += gridDim.x) {
    const int c = PAST ? k : chunks - 1 - k;
    const int t = tensor_of(l, c);
    if (f == 1.f && l.src[t] == l.dst[t]) continue;
    const long start = (long)(c - l.first[t]) * kChunk;
    const int n = (int)min((long)kChunk, l.numel[t] - start);
    switch (l.type[t]) {
      case 0:
        scaled<PAST>(static_cast<const float*>(l.src[t]) + start,
               static_cast<float*>(l.dst[t]) + start, n, f);
        break;
      case 1:
        scaled<PAST>(static_cast<const __hip_bfloat16*>(l.src[t]) + start,
               static_cast<__hip_bfloat16*>(l.dst[t]) + start, n, f);
        break;
      default:
        scaled<PAST>(static_cast<const __half*>(l.src[t]) + start,
               static_cast<__half*>(l.dst[t]) + start, n, f);
    }
  }
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      TORCH_CHECK_TYPE(false, "gradients must be float32, bfloat16 or "
                       "float16, not ", t);
  }
}

// The gradients as the kernels take them: on one GPU, of a known type, and
// dense in some order (a copy where they are not).
std::vector<torch::Tensor> as_dense(const std::vector<torch::Tensor>& ts) {
  std::vector<torch::Tensor> out;
  out.reserve(ts.size());
  for (const auto& t : ts) {
    TORCH_CHECK_TYPE(t.defined() && t.layout() == at::kStrided,
                     "gradients must be dense tensors");
    TORCH_CHECK_VALUE(t.is_cuda() && t.device() == ts[0].device(),
                      "gradients must be on one GPU");
    type_code(t.scalar_type());
    out.push_back(t.is_non_overlapping_and_dense() ? t : t.contiguous());
  }
  return out;
}

// Two gradients that share memory would be scaled twice, by two blocks at
// once.
void check_apart(const std::vector<torch::Tensor>& ts) {
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  spans.reserve(ts.size());
  for (const auto& t : ts)
    if (t.numel() > 0) {
      const auto p = reinterpret_cast<uintptr_t>(t.data_ptr());
      spans.emplace_back(p, p + t.numel() * t.element_size());
    }
  if (!std::is_sorted(spans.begin(), spans.end()))
    std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    TORCH_CHECK_VALUE(spans[i].first >= spans[i - 1].second,
                      "two of the gradients share memory");
}

// Norm of `src` (dense), and src times the clip factor in `dst` where dst
// is not empty: the same tensors, or others of the same types and strides.
torch::Tensor clip_list(const std::vector<torch::Tensor>& src,
                        const std::vector<torch::Tensor>& dst,
                        double max_norm, double eps) {
  const auto device = src[0].device();
  const auto stream = current_stream();

  std::vector<TensorList> lists;
  long bytes = 0;
  for (size_t i = 0; i < src.size(); ++i) {
    if (src[i].numel() == 0) continue;
    bytes += src[i].numel() * src[i].element_size();
    const long chunks = (src[i].numel() + kChunk - 1) / kChunk;
    if (lists.empty() || lists.back().count == kMaxTensors) {
      lists.emplace_back();
      lists.back().count = 0;
      lists.back().first[0] = 0;
    }
    TensorList& l = lists.back();
    grid_of(l.first[l.count] + chunks, kThreads, "gradients");
    l.src[l.count] = src[i].data_ptr();
    l.dst[l.count] = dst.empty() ? nullptr : dst[i].data_ptr();
    l.numel[l.count] = src[i].numel();
    l.type[l.count] = type_code(src[i].scalar_type());
    l.first[l.count + 1] = l.first[l.count] + (int)chunks;
    ++l.count;
  }
  const auto opts = torch::TensorOptions().device(device);
  auto norm = torch::empty({}, opts.dtype(torch::kFloat));
  std::vector<int> at(1, 0);
  for (const auto& l : lists)
    at.push_back(at.back() + std::min(l.first[l.count], kMaxBlocks));
  auto partials =
      torch::empty({std::max(at.back(), 1)}, opts.dtype(torch::kDouble));
  double* pp = partials.data_ptr<double>();
  const bool past = bytes >= kPastBytes;
  for (size_t i = 0; i < lists.size(); ++i) {
    const auto kernel =
        past ? norm_partials_kernel<true> : norm_partials_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(at[i + 1] - at[i]), dim3(kThreads), 0,
                       stream, lists[i], pp + at[i]);
    CHECK_HIP(hipGetLastError());
  }
  if (dst.empty() || lists.empty()) {
    lists.resize(1);
    lists[0].count = 0;
    lists[0].first[0] = 0;
  }
  for (size_t i = lists.size(); i-- > 0;) {
    const int chunks = lists[i].first[lists[i].count];
    const auto kernel =
        past ? clip_scale_list_kernel<true> : clip_scale_list_kernel<false>;
    hipLaunchKernelGGL(kernel,
                       dim3(std::max(1, past ? chunks
                                         : std::min(chunks, kMaxScaleBlocks))),
                       dim3(kThreads), 0, stream, lists[i], pp, at.back(),
                       max_norm, eps,
                       i == 0 ? norm.data_ptr<float>() : nullptr);
    CHECK_HIP(hipGetLastError());
  }
  return norm;
}

}  // namespace

torch::Tensor grad_norm(const std::vector<torch::Tensor>& grads) {
  TORCH_CHECK(!grads.empty(), "no gradients");
  c10::DeviceGuard guard(grads[0].device());
  return clip_list(as_dense(grads), {}, 0., 0.);
}

std::tuple<std::vector<torch::Tensor>, torch::Tensor> clip_grads(
    const std::vector<torch::Tensor>& grads, double max_norm, double eps) {
  TORCH_CHECK(!grads.empty(), "no gradients");
  c10::DeviceGuard guard(grads[0].device());
  const auto src = as_dense(grads);
  // One buffer for all of them, each at a multiple of 256 bytes: an
  // allocation for each costs as much host time as all the rest.
  std::vector<long> at(1, 0);
  for (const auto& t : src)
    at.push_back((at.back() + t.numel() * (long)t.element_size() + 255) &
                 ~255L);
  const auto buffer = torch::empty(
      {at.back()}, torch::TensorOptions().device(src[0].device()).dtype(
                       torch::kByte));
  std::vector<torch::Tensor> dst;
  dst.reserve(src.size());
  for (size_t i = 0; i < src.size(); ++i) {
    auto t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(buffer.storage()), buffer.key_set(), src[i].dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(
        at[i] / (long)src[i].element_size());
    t.unsafeGetTensorImpl()->set_sizes_and_strides(src[i].sizes(),
                                                   src[i].strides());
    dst.push_back(std::move(t));
  }
  auto norm = clip_list(src, dst, max_norm, eps);
  return {std::move(dst), std::move(norm)};
}

torch::Tensor clip_grads_(const std::vector<torch::Tensor>& grads,
                          double max_norm, double eps) {
  TORCH_CHECK(!grads.empty(), "no gradients");
  c10::DeviceGuard guard(grads[0].device());
  const auto work = as_dense(grads);
  for (size_t i = 0; i < grads.size(); ++i)
    if (!work[i].is_same(grads[i]))
      for (int64_t d = 0; d < grads[i].dim(); ++d)
        TORCH_CHECK_VALUE(grads[i].stride(d) != 0 || grads[i].size(d) < 2,
                          "an expanded gradient cannot be clipped in place");
  check_apart(work);
  auto norm = clip_list(work, work, max_norm, eps);
  for (size_t i = 0; i < grads.size(); ++i)
    if (!work[i].is_same(grads[i]))
      grads[i].copy_(work[i]);
    else
      grads[i].unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace mgx
