// Host side of the attention over a shared prefix (device code and its
// reasons in prefix_attn_kernels.h).

#include "host_common.h"
#include "prefix_attn_kernels.h"

#include <algorithm>

namespace photon_hip {

namespace {

// How a call is cut into workgroups: items of `rows` query rows of one head,
// the last `rest` of them split `splits` times along the keys.
struct Cut {
  int waves;  // of 32 rows each
  int rows, items, full, rest, splits;
  int groups() const { return full + rest * splits; }
  long partial_rows() const { return (long)rest * splits * rows; }
};

// Whole rounds of items fill the chip by themselves; what is left over is
// split until it does, but not below two key tiles each. `always`: every item
// leaves partial rows.
Cut cut(long T, int H, int D, int key_tiles, bool always) {
  Cut c;
  c.waves = T <= 32 ? 1 : T <= 64 ? 2 : 4;
  c.rows = c.waves * QB;
  const long items = (T + c.rows - 1) / c.rows * H;
  TORCH_CHECK(items < (1L << 22), "prefix attention: too many rows");
  c.items = (int)items;
  // a CU holds two workgroups of four waves (three with short heads), or one
  // with four buffers
  const int at_once = c.waves < 4 ? 256 : D == 64 ? 768 : 512;
  c.full = always ? 0 : c.items / at_once * at_once;
  c.rest = c.items - c.full;
  c.splits = 1;
  if (c.rest > 0 && c.rest < at_once)
    c.splits = std::max(1, std::min((at_once + c.rest / 2) / c.rest, key_tiles / 2));
  if (c.splits == 1 && !always) {
    c.full = c.items;
    c.rest = 0;
  }
  return c;
}

template <bool DECODE>
void launch(const torch::Tensor& qkv, const torch::Tensor& prefix, int H,
            int D, const torch::Tensor& slopes, const torch::Tensor& info,
            __bf16* out, float* part_o, float* part_ml, int T, int P,
            const Cut& c) {
  const __bf16* pre = (const __bf16*)prefix.data_ptr();
  const __bf16* pk = pre + (long)H * D;
  const __bf16* pv = pre + 2L * H * D;
#define ARGS                                                                 \
  cur_stream(), (const __bf16*)qkv.data_ptr(), qkv.stride(0), pk, pv,        \
      prefix.stride(0), slopes.data_ptr<float>(), info.data_ptr<int>(), out, \
      part_o, part_ml, T, P, H, c.full, c.splits
#define LAUNCH(DD, NW, BUFS)                                                 \
  hipLaunchKernelGGL((prefix_attn_kernel<DD, NW, BUFS, DECODE>),             \
                     dim3(c.groups()), dim3(64 * NW),                        \
                     lds_bytes(DD, NW, BUFS), ARGS)
#define LAUNCH_D(DD)                                                         \
  if (c.waves == 1) { LAUNCH(DD, 1, 4); }                                    \
  else if (c.waves == 2) { LAUNCH(DD, 2, 4); }                               \
  else if (c.groups() <= 256) { LAUNCH(DD, 4, 4); }                          \
  else { LAUNCH(DD, 4, 2); }
  if (D == 64) {
    LAUNCH_D(64)
  } else {
    LAUNCH_D(128)
  }
#undef LAUNCH_D
#undef LAUNCH
#undef ARGS
}

// Rows of [q | k | v], 16-byte accesses allowed.
torch::Tensor checked_rows(const torch::Tensor& t, long width,
                           const torch::Device& dev, const char* what) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kBFloat16,
              "prefix attention: ", what, " must be bf16 on ", dev);
  TORCH_CHECK(t.dim() == 2 && t.size(1) == width, "prefix attention: ", what,
              " must be [rows, ", width, "], got ", t.sizes());
  TORCH_CHECK(t.size(0) < (1L << 30), "prefix attention: too many rows");
  // a tile of 64 rows is addressed with 32-bit byte offsets
  const bool fits = t.size(0) <= 1 || (t.stride(0) >= width &&
                                       t.stride(0) < (1L << 23) &&
                                       t.stride(0) % 8 == 0);
  const bool ok = t.stride(1) == 1 && fits && ((uintptr_t)t.data_ptr() % 16) == 0;
  return ok ? t : t.contiguous().clone();
}

struct Args {
  torch::Tensor qkv, prefix, slopes, info;
  int T, P, H, D;
};

Args check(const torch::Tensor& qkv, const torch::Tensor& prefix, long H,
           const torch::Tensor& slopes, const torch::Tensor& info) {
  TORCH_CHECK(qkv.is_cuda() && qkv.dim() == 2 && H > 0 && H < 65536 &&
                  qkv.size(1) % (3 * H) == 0,
              "prefix attention: qkv must be a GPU tensor [rows, 3 * heads * d]");
  const long D = qkv.size(1) / (3 * H);
  TORCH_CHECK(D == 64 || D == 128,
              "prefix attention: d_head must be 64 or 128, got ", D);
  TORCH_CHECK(qkv.size(1) < (1L << 23), "prefix attention: rows too long");
  const auto dev = qkv.device();
  Args a;
  a.qkv = checked_rows(qkv, qkv.size(1), dev, "qkv");
  a.prefix = checked_rows(prefix, qkv.size(1), dev, "prefix");
  a.T = (int)qkv.size(0);
  a.P = (int)prefix.size(0);
  a.H = (int)H;
  a.D = (int)D;
  TORCH_CHECK(slopes.dim() == 1 && slopes.size(0) == H,
              "prefix attention: one slope for each head");
  a.slopes = slopes.to(dev, at::kFloat).contiguous();
  TORCH_CHECK(info.device() == dev && info.scalar_type() == at::kInt &&
                  info.dim() == 1 && info.size(0) == a.T,
              "prefix attention: one int32 for each row of qkv, on its device");
  a.info = info.contiguous();
  return a;
}

}  // namespace

torch::Tensor prefix_attention(torch::Tensor qkv, torch::Tensor prefix, long H,
                               torch::Tensor slopes, torch::Tensor starts) {
  const c10::DeviceGuard guard(qkv.device());
  const Args a = check(qkv, prefix, H, slopes, starts);
  auto out = torch::empty({(long)a.T, (long)a.H * a.D}, qkv.options());
  if (a.T == 0) return out;
  const Cut c = cut(a.T, a.H, a.D, (a.P + PKB - 1) / PKB + 1, false);
  torch::Tensor po, pm;
  if (c.rest) {
    auto f = qkv.options().dtype(at::kFloat);
    po = torch::empty({c.partial_rows() * a.D}, f);
    pm = torch::empty({c.partial_rows() * 2}, f);
  }
  launch<false>(a.qkv, a.prefix, a.H, a.D, a.slopes, a.info,
                (__bf16*)out.data_ptr(),
                c.rest ? po.data_ptr<float>() : nullptr,
                c.rest ? pm.data_ptr<float>() : nullptr, a.T, a.P, c);
  if (c.rest) {
    const long threads = (long)c.rest * c.rows * a.D / 4;
    auto join = a.D == 64 ? prefix_join_kernel<64> : prefix_join_kernel<128>;
    hipLaunchKernelGGL(join, dim3((unsigned)((threads + 255) / 256)),
                       dim3(256), 0, cur_stream(), po.data_ptr<float>(),
                       pm.data_ptr<float>(), (__bf16*)out.data_ptr(), a.T, a.H,
                       c.rows, c.full, c.rest, c.splits);
  }
  return out;
}

torch::Tensor prefix_attention_decode(torch::Tensor qkv, torch::Tensor prefix,
                                      long H, torch::Tensor slopes,
                                      torch::Tensor cache, torch::Tensor held) {
  const c10::DeviceGuard guard(qkv.device());
  const Args a = check(qkv, prefix, H, slopes, held);
  const long B = a.T;
  TORCH_CHECK(cache.device() == qkv.device() &&
                  cache.scalar_type() == at::kBFloat16 && cache.dim() == 5 &&
                  cache.size(0) == B && cache.size(2) == 2 &&
                  cache.size(3) == H && cache.size(4) == a.D,
              "prefix attention: cache must be bf16 [", B, ", slots, 2, ", H,
              ", ", a.D, "], got ", cache.sizes());
  TORCH_CHECK(cache.size(1) < (1L << 30), "prefix attention: too many slots");
  bool fits = cache.stride(4) == 1 && ((uintptr_t)cache.data_ptr() % 16) == 0;
  for (int d = 0; d < 4; ++d)
    fits = fits && cache.stride(d) % 8 == 0 &&
           (cache.size(d) <= 1 || cache.stride(d) != 0);
  TORCH_CHECK(fits,
              "prefix attention: the cache's last dimension must be contiguous "
              "and its rows aligned to 16 bytes");
  TORCH_CHECK(B < 65536, "prefix attention: too many sequences");
  auto out = torch::empty({B, (long)a.H * a.D}, qkv.options());
  if (B == 0) return out;
  Cut c{};
  torch::Tensor po, pm;
  if (a.P > 0) {
    c = cut(B, a.H, a.D, (a.P + PKB - 1) / PKB, true);
    auto f = qkv.options().dtype(at::kFloat);
    po = torch::empty({c.partial_rows() * a.D}, f);
    pm = torch::empty({c.partial_rows() * 2}, f);
    launch<true>(a.qkv, a.prefix, a.H, a.D, a.slopes, a.info, nullptr,
                 po.data_ptr<float>(), pm.data_ptr<float>(), a.T, a.P, c);
  }
  const dim3 grid(a.H, (unsigned)B);
  const float* pop = c.splits ? po.data_ptr<float>() : nullptr;
  const float* pmp = c.splits ? pm.data_ptr<float>() : nullptr;
#define LAUNCH_OWN(DD)                                                        \
  hipLaunchKernelGGL((decode_own_kernel<DD>), grid, dim3(OWN_BLOCK), 0,       \
                     cur_stream(), (const __bf16*)a.qkv.data_ptr(),           \
                     a.qkv.stride(0), (__bf16*)cache.data_ptr(),              \
                     cache.stride(0), cache.stride(1), cache.stride(2),       \
                     cache.stride(3), a.slopes.data_ptr<float>(),             \
                     a.info.data_ptr<int>(), pop, pmp,                        \
                     (__bf16*)out.data_ptr(), a.H, (int)cache.size(1),        \
                     std::max(1, c.rows), c.items, c.splits)
  if (a.D == 64) {
    LAUNCH_OWN(64);
  } else {
    LAUNCH_OWN(128);
  }
#undef LAUNCH_OWN
  return out;
}

}  // namespace photon_hip
