// Fused multi-tensor AdamW / ADOPT kernels for CDNA4.
//
// Replaces torch's _fused_adamw multi-tensor-apply + the reference "adopt"
// optimizer. Tensors are batched into a struct
// passed by kernarg (up to MT_CHUNK tensors per launch); each block
// grid-strides over one tensor's elements (block -> tensor mapping by
// cumulative block counts). All state math in fp32; params may be fp32 or
// bf16.

#include "host_common.h"

#include <vector>

namespace photon_hip {

constexpr int MT_CHUNK = 8;

template <typename T>
struct TensorBatch {
  T* p[MT_CHUNK];
  T* g[MT_CHUNK];
  float* m[MT_CHUNK];
  float* v[MT_CHUNK];
  float* w[MT_CHUNK];  // fp32 master weights (null = p IS the master)
  long n[MT_CHUNK];
  int count;
};

// blocks are distributed proportionally: block b handles tensor
// b % count, striding with gridDim.x/count-ish. Simpler: each block picks
// tensor (b % count) and strides by the number of blocks assigned to it.
template <typename T, int BLOCK>
__global__ void adamw_kernel(TensorBatch<T> batch, float lr, float b1,
                             float b2, float eps, float wd, float bc1,
                             float bc2) {
  const int t = blockIdx.x % batch.count;
  const int nb = (gridDim.x + batch.count - 1 - t) / batch.count;  // blocks on t
  const int bi = blockIdx.x / batch.count;
  T* p = batch.p[t];
  T* g = batch.g[t];
  float* m = batch.m[t];
  float* v = batch.v[t];
  float* w = batch.w[t];  // fp32 master (PURE mixed precision), or null
  const long n = batch.n[t];
  const float decay = 1.f - lr * wd;
  for (long i = (long)(bi * BLOCK + threadIdx.x); i < n; i += (long)nb * BLOCK) {
    float gf = load_f32<T>(g, i);
    float mi = m[i] = b1 * m[i] + (1.f - b1) * gf;
    float vi = v[i] = b2 * v[i] + (1.f - b2) * gf * gf;
    float pv = w ? w[i] : load_f32<T>(p, i);
    if (wd != 0.f) pv *= decay;
    pv -= lr * (mi / bc1) / (sqrtf(vi / bc2) + eps);
    if (w) w[i] = pv;
    store_f32<T>(p, i, pv);
  }
}

template <typename T, int BLOCK>
__global__ void adopt_kernel(TensorBatch<T> batch, float lr, float b1,
                             float b2, float eps, float wd, float clip,
                             int step) {
  const int t = blockIdx.x % batch.count;
  const int nb = (gridDim.x + batch.count - 1 - t) / batch.count;
  const int bi = blockIdx.x / batch.count;
  T* p = batch.p[t];
  T* g = batch.g[t];
  float* m = batch.m[t];
  float* v = batch.v[t];
  float* w = batch.w[t];
  const long n = batch.n[t];
  const float decay = 1.f - lr * wd;
  for (long i = (long)(bi * BLOCK + threadIdx.x); i < n; i += (long)nb * BLOCK) {
    float gf = load_f32<T>(g, i);
    if (step == 1) {
      v[i] = gf * gf;  // v0 init; no param update
      continue;
    }
    float c = gf / fmaxf(sqrtf(v[i]), eps);
    c = fminf(fmaxf(c, -clip), clip);
    float mi = m[i] = b1 * m[i] + (1.f - b1) * c;
    float pv = w ? w[i] : load_f32<T>(p, i);
    if (wd != 0.f) pv *= decay;
    pv -= lr * mi;
    if (w) w[i] = pv;
    store_f32<T>(p, i, pv);
    v[i] = b2 * v[i] + (1.f - b2) * gf * gf;
  }
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
namespace {
constexpr int OPT_BLOCK = 256;

template <typename T>
TensorBatch<T> make_batch(const std::vector<torch::Tensor>* ps,
                          const std::vector<torch::Tensor>& gs,
                          const std::vector<torch::Tensor>* ms,
                          const std::vector<torch::Tensor>* vs, size_t start,
                          size_t count,
                          const std::vector<torch::Tensor>* ws = nullptr) {
  TensorBatch<T> b{};
  b.count = (int)count;
  for (size_t i = 0; i < count; ++i) {
    b.p[i] = ps ? (T*)(*ps)[start + i].data_ptr() : nullptr;
    b.g[i] = (T*)gs[start + i].data_ptr();
    b.m[i] = ms ? (*ms)[start + i].data_ptr<float>() : nullptr;
    b.v[i] = vs ? (*vs)[start + i].data_ptr<float>() : nullptr;
    b.w[i] = (ws && !ws->empty()) ? (*ws)[start + i].data_ptr<float>()
                                  : nullptr;
    b.n[i] = gs[start + i].numel();
  }
  return b;
}
}  // namespace

void adamw_step(std::vector<torch::Tensor> ps, std::vector<torch::Tensor> gs,
                std::vector<torch::Tensor> ms, std::vector<torch::Tensor> vs,
                double lr, double b1, double b2, double eps, double wd,
                double bc1, double bc2,
                std::vector<torch::Tensor> masters = {}) {
  const int GRID = 1024;
  for (size_t s = 0; s < ps.size(); s += MT_CHUNK) {
    size_t c = std::min((size_t)MT_CHUNK, ps.size() - s);
    DISPATCH_DTYPE(ps[s], "adamw_step", {
      auto batch = make_batch<scalar_t>(&ps, gs, &ms, &vs, s, c, &masters);
      hipLaunchKernelGGL((adamw_kernel<scalar_t, OPT_BLOCK>), dim3(GRID),
                         dim3(OPT_BLOCK), 0, cur_stream(), batch, (float)lr,
                         (float)b1, (float)b2, (float)eps, (float)wd,
                         (float)bc1, (float)bc2);
    });
  }
}

void adopt_step(std::vector<torch::Tensor> ps, std::vector<torch::Tensor> gs,
                std::vector<torch::Tensor> ms, std::vector<torch::Tensor> vs,
                double lr, double b1, double b2, double eps, double wd,
                double clip, long step,
                std::vector<torch::Tensor> masters = {}) {
  const int GRID = 1024;
  for (size_t s = 0; s < ps.size(); s += MT_CHUNK) {
    size_t c = std::min((size_t)MT_CHUNK, ps.size() - s);
    DISPATCH_DTYPE(ps[s], "adopt_step", {
      auto batch = make_batch<scalar_t>(&ps, gs, &ms, &vs, s, c, &masters);
      hipLaunchKernelGGL((adopt_kernel<scalar_t, OPT_BLOCK>), dim3(GRID),
                         dim3(OPT_BLOCK), 0, cur_stream(), batch, (float)lr,
                         (float)b1, (float)b2, (float)eps, (float)wd,
                         (float)clip, (int)step);
    });
  }
}

}  // namespace photon_hip
