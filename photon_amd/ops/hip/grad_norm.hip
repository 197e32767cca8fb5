// Norms of many tensors in one sweep, and clipping by their global norm.
//
//   s_t = sum g^2,  norm_t = sqrt(s_t),  total = sqrt(sum_t s_t)
//   c = max_norm / (total + 1e-6);  g = round(c * g)  where c < 1
//
// Bound by memory: one read for the norms, one more read and one write where
// the gradients are clipped. The tensors may differ in length and in type;
// their addresses travel in the kernel's arguments, BATCH of them a launch,
// so nothing is copied to the device and a call can be captured in a graph.
//
// Measured: the 3B configuration's gradients, 5.3 GB in bf16 and fp32, are
// read at 5.8 TB/s (0.92 ms); the 1B configuration's 5.3 GB in fp32 take 0.92
// ms and another 2.06 ms to be clipped, 10.5 GB at 5.1 TB/s (a large copy
// moves 4.7). 58 MB in 27 tensors: 12 + 4 + 20 us, mostly out of the caches.
// Stores that bypass the caches change neither.
//
// Squares are summed in 64 bits: a square leaves the range of fp32 at
// 1.8e19 and loses its bits below 1e-19, the sum over 10^9 elements
// needs more than 24 bits, and the fp64 pipe has room while memory is waited
// for. Every element belongs to a chunk of fixed size, every chunk to a block,
// and the chunks are added in order: the result does not change from run to
// run.

#include "host_common.h"

#include <algorithm>
#include <vector>

namespace photon_hip {

namespace {

constexpr int GN_BLOCK = 256;
constexpr int BATCH = 160;  // tensors a launch; 4 KiB of arguments at most
constexpr long MIN_CHUNK = 8192;
constexpr long MAX_CHUNKS = 8192;  // aim, without the tensors' last chunks

struct TensorList {
  void* p[BATCH];
  long n[BATCH];         // elements * 2 + (1 if bf16)
  int first[BATCH + 1];  // first chunk of each tensor in this launch
  int count;
  int chunk0;  // first chunk of this launch among all
  int tensor0;
  long chunk;  // elements a chunk
};
static_assert(sizeof(TensorList) <= 3968, "kernel arguments");

// The block's piece of a tensor.
struct Piece {
  char* p;
  long n;
  bool bf16;
  int tensor;
};

DEV_INLINE Piece find_piece(const TensorList& list, int c) {
  int lo = 0, hi = list.count - 1;  // last tensor that begins at or before c
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (list.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  const long n = list.n[lo] >> 1;
  const bool bf16 = list.n[lo] & 1;
  const long at = (long)(c - list.first[lo]) * list.chunk;
  return {(char*)list.p[lo] + at * (bf16 ? 2 : 4), min(list.chunk, n - at),
          bf16, lo};
}

// f(pointer, count of elements) over a piece: VEC-element accesses of 16
// bytes between the unaligned ends.
template <typename T, typename Wide, typename One>
DEV_INLINE void sweep(T* p, long n, Wide wide, One one) {
  constexpr int VEC = 16 / sizeof(T);
  const long head =
      min(n, (long)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T)));
  if (threadIdx.x < head) one(p + threadIdx.x);
  T* body = p + head;
  const long nv = (n - head) / VEC;
#pragma unroll 4
  for (long i = threadIdx.x; i < nv; i += GN_BLOCK) wide(body + i * VEC);
  const long done = head + nv * VEC;
  if (done + threadIdx.x < n) one(p + done + threadIdx.x);
}

DEV_INLINE double square(float x) { return (double)x * (double)x; }

DEV_INLINE double block_sum(double v, double* scratch) {
  for (int off = WAVE / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
  const int waves = blockDim.x / WAVE;
  if ((threadIdx.x & (WAVE - 1)) == 0) scratch[threadIdx.x / WAVE] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < waves; ++w) s += scratch[w];
  return s;
}

__global__ __launch_bounds__(GN_BLOCK) void sum_squares_kernel(
    const TensorList list, double* __restrict__ partials,
    int* __restrict__ firsts) {
  __shared__ double scratch[GN_BLOCK / WAVE];
  const int c = blockIdx.x;
  const Piece q = find_piece(list, c);
  double s = 0.0;
  if (q.bf16) {
    sweep(
        (const unsigned short*)q.p, q.n,
        [&](const unsigned short* p) {
          const shortx8 v = *(const shortx8*)p;
#pragma unroll
          for (int j = 0; j < 8; ++j) s += square(bf16_to_f32((unsigned short)v[j]));
        },
        [&](const unsigned short* p) { s += square(bf16_to_f32(*p)); });
  } else {
    sweep(
        (const float*)q.p, q.n,
        [&](const float* p) {
          const floatx4 v = *(const floatx4*)p;
#pragma unroll
          for (int j = 0; j < 4; ++j) s += square(v[j]);
        },
        [&](const float* p) { s += square(*p); });
  }
  s = block_sum(s, scratch);
  if (threadIdx.x == 0) {
    partials[list.chunk0 + c] = s;
    if (c == list.first[q.tensor])
      firsts[list.tensor0 + q.tensor] = list.chunk0 + c;
  }
}

// Block 0 adds all chunks, the other blocks a tensor's each.
constexpr int FIN_BLOCK = 512;
__global__ __launch_bounds__(FIN_BLOCK) void finish_norms_kernel(
    const double* __restrict__ partials, const int* __restrict__ firsts,
    int chunks, int tensors, float* __restrict__ total,
    float* __restrict__ norms) {
  __shared__ double scratch[FIN_BLOCK / WAVE];
  const int t = (int)blockIdx.x - 1;
  const int from = t < 0 ? 0 : firsts[t];
  const int to = t < 0 || t + 1 == tensors ? chunks : firsts[t + 1];
  double s = 0.0;
#pragma unroll 4
  for (int i = from + threadIdx.x; i < to; i += FIN_BLOCK) s += partials[i];
  s = block_sum(s, scratch);
  if (threadIdx.x == 0) (t < 0 ? total[0] : norms[t]) = (float)sqrt(s);
}

// From the last chunk to the first: the end of the list is what the norms'
// sweep left in the caches.
__global__ __launch_bounds__(GN_BLOCK) void clip_kernel(
    const TensorList list, const float* __restrict__ total, float max_norm) {
  const float scale = max_norm / (total[0] + 1e-6f);
  if (scale >= 1.f) return;  // a NaN goes on, and into every gradient
  const Piece q = find_piece(list, (int)(gridDim.x - 1 - blockIdx.x));
  if (q.bf16) {
    sweep(
        (unsigned short*)q.p, q.n,
        [&](unsigned short* p) {
          union { shortx8 s; __bf16 b[8]; } r;
          const shortx8 v = *(const shortx8*)p;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            r.b[j] = (__bf16)(bf16_to_f32((unsigned short)v[j]) * scale);
          *(shortx8*)p = r.s;
        },
        [&](unsigned short* p) {
          *(__bf16*)p = (__bf16)(bf16_to_f32(*p) * scale);
        });
  } else {
    sweep(
        (float*)q.p, q.n,
        [&](float* p) {
          floatx4 v = *(const floatx4*)p;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] *= scale;
          *(floatx4*)p = v;
        },
        [&](float* p) { *p *= scale; });
  }
}

struct Plan {
  std::vector<torch::Tensor> t;  // dense; a copy where the caller's is not
  std::vector<char> copied;
  std::vector<TensorList> lists;
  std::vector<int> grids;
  int chunks = 0;
};

Plan make_plan(const std::vector<torch::Tensor>& ts, const char* name) {
  TORCH_CHECK(!ts.empty(), name, ": empty list of tensors");
  Plan plan;
  long all = 0;
  for (const auto& t : ts) {
    TORCH_CHECK(t.layout() == at::kStrided && t.is_cuda() &&
                    t.device() == ts[0].device(),
                name, ": the tensors must be strided and on one GPU");
    TORCH_CHECK(t.scalar_type() == at::kFloat ||
                    t.scalar_type() == at::kBFloat16,
                name, ": unsupported dtype ", t.dtype());
    const bool dense = t.is_non_overlapping_and_dense();
    plan.t.push_back(dense ? t : t.contiguous());
    plan.copied.push_back(!dense);
    all += t.numel();
  }
  const long quantum = 4 * GN_BLOCK * 8;  // whole unrolled rounds of a block
  long chunk = std::max(MIN_CHUNK, (all + MAX_CHUNKS - 1) / MAX_CHUNKS);
  chunk = (chunk + quantum - 1) / quantum * quantum;
  for (size_t s = 0; s < ts.size(); s += BATCH) {
    TensorList list{};
    list.count = (int)std::min((size_t)BATCH, ts.size() - s);
    list.chunk0 = plan.chunks;
    list.tensor0 = (int)s;
    list.chunk = chunk;
    long at = 0;
    for (int i = 0; i < list.count; ++i) {
      const auto& t = plan.t[s + i];
      list.p[i] = t.data_ptr();
      list.n[i] = t.numel() * 2 + (t.scalar_type() == at::kBFloat16 ? 1 : 0);
      list.first[i] = (int)at;
      at += std::max(1L, (t.numel() + chunk - 1) / chunk);
    }
    list.first[list.count] = (int)at;
    plan.chunks += (int)at;
    plan.lists.push_back(list);
    plan.grids.push_back((int)at);
  }
  return plan;
}

std::vector<torch::Tensor> run_norms(const Plan& plan) {
  const auto opt = plan.t[0].options();
  const int tensors = (int)plan.t.size();
  auto partials = torch::empty({plan.chunks}, opt.dtype(at::kDouble));
  auto firsts = torch::empty({tensors}, opt.dtype(at::kInt));
  auto total = torch::empty({}, opt.dtype(at::kFloat));
  auto norms = torch::empty({tensors}, opt.dtype(at::kFloat));
  for (size_t i = 0; i < plan.lists.size(); ++i)
    hipLaunchKernelGGL(sum_squares_kernel, dim3(plan.grids[i]), dim3(GN_BLOCK),
                       0, cur_stream(), plan.lists[i],
                       partials.data_ptr<double>(), firsts.data_ptr<int>());
  hipLaunchKernelGGL(finish_norms_kernel, dim3(1 + tensors), dim3(FIN_BLOCK),
                     0, cur_stream(), partials.data_ptr<double>(),
                     firsts.data_ptr<int>(), plan.chunks, tensors,
                     total.data_ptr<float>(), norms.data_ptr<float>());
  return {total, norms};
}

}  // namespace

std::vector<torch::Tensor> tensor_norms(std::vector<torch::Tensor> ts) {
  TORCH_CHECK(!ts.empty(), "tensor_norms: empty list of tensors");
  const c10::DeviceGuard guard(ts[0].device());
  return run_norms(make_plan(ts, "tensor_norms"));
}

std::vector<torch::Tensor> clip_grads(std::vector<torch::Tensor> gs,
                                      double max_norm) {
  TORCH_CHECK(!gs.empty(), "clip_grads: empty list of tensors");
  const c10::DeviceGuard guard(gs[0].device());
  // A gradient that is there twice would be counted and scaled twice, or half
  // of it. Of a strided one, whose gaps may hold others, the first element.
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  for (const auto& g : gs) {
    TORCH_CHECK(g.layout() == at::kStrided, "clip_grads: strided tensors only");
    check_writable(g, "clip_grads", "a gradient");
    check_no_tangent(g, "clip_grads");
    if (g.numel() == 0) continue;
    long span = 1;
    for (int d = 0; d < g.dim(); ++d) {
      const long reach = (g.size(d) - 1) * g.stride(d);
      span += reach;
      TORCH_CHECK(g.size(d) == 1 || g.stride(d) != 0,
                  "clip_grads: a gradient shares elements with itself");
    }
    const auto p = (uintptr_t)g.data_ptr();
    if (!g.is_non_overlapping_and_dense()) span = 1;
    spans.emplace_back(p, p + span * g.element_size());
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    TORCH_CHECK(spans[i].first >= spans[i - 1].second,
                "clip_grads: two gradients share memory");
  const Plan plan = make_plan(gs, "clip_grads");
  auto result = run_norms(plan);
  for (size_t i = plan.lists.size(); i-- > 0;)
    hipLaunchKernelGGL(clip_kernel, dim3(plan.grids[i]), dim3(GN_BLOCK), 0,
                       cur_stream(), plan.lists[i],
                       result[0].data_ptr<float>(), (float)max_norm);
  for (size_t i = 0; i < gs.size(); ++i) {
    if (plan.copied[i])
      gs[i].copy_(plan.t[i]);
    else
      gs[i].unsafeGetTensorImpl()->bump_version();  // written in place
  }
  return result;
}

}  // namespace photon_hip
