// Host side of the attention over a shared prefix (device code and its
// reasons in prefix_attn_kernels.h).

#include "host_common.h"
#include "prefix_attn_kernels.h"

#include <algorithm>

namespace photon_hip {

namespace {

// How a call is cut into workgroups: items of `rows` query rows of one head,
// `rest` of them, from `first_split` on, split `splits` times along the keys.
struct Cut {
  bool few;  // few rows: waves share the keys, not the rows
  int rows, items, first_split, rest, splits;
  int groups() const { return items + rest * (splits - 1); }
  long partial_rows() const { return (long)rest * splits * rows; }
};

template <int D>
using FewRows = Shape<D, 1, 4>;
template <int D>
using ManyRows = Shape<D, 4, 1>;
// Few rows are 128 items of 32 rows at most: half the chip, so that the keys
// can be split at least once more. 16 heads of 128 over 1507 keys, 160 rows (80
// items): 17 us, and 25 with tiles of 128 rows; 32 heads over 3900 keys, 160
// rows (160 items): 54 us, and 36.
constexpr long FEW_ITEMS = 128;

// Whole rounds of items fill the chip by themselves; what is left over is
// split until it does, but not below some keys each. The split ones come right
// after the first round, where heads that see the whole prefix are still on:
// the short ones that follow fill the gaps (4416 rows over 3901 keys, 32 heads of
// 128: 261 us with the split ones last, 232 so). With many rows these are
// two tiles. With few rows a split call is bound by the host's two launches,
// 10 us: 20 rows of 12 heads of 64 over 701 keys take 8.7 us whole and 10.0 in
// two, 96 rows of 16 heads of 128 over 1507 keys 20.7 whole and 15.4 in four.
// `always` (the decode form, which joins anyway): every item leaves partial
// rows. 64 sequences of 12 heads of 64 over 2000 keys take 18.4 us with 128
// keys a split at least, 13.7 with 256 and 13.4 with 384; 16 sequences of 32
// heads of 128 over 700 keys 14.0, 13.6 and 15.8.
Cut cut(long T, int H, int D, long keys, bool always) {
  Cut c;
  c.few = (T + FewRows<64>::ROWS - 1) / FewRows<64>::ROWS * H <= FEW_ITEMS;
  c.rows = c.few ? FewRows<64>::ROWS : ManyRows<64>::ROWS;
  const long items = (T + c.rows - 1) / c.rows * H;
  TORCH_CHECK(items < (1L << 22), "prefix attention: too many rows");
  c.items = (int)items;
  // workgroups that are on the chip together, by their registers and LDS
  const int at_once = c.few ? (D == 64 ? 512 : 256) : (D == 64 ? 768 : 512);
  c.rest = always ? c.items : c.items % at_once;
  c.first_split = c.items > c.rest ? at_once : 0;
  c.splits = 1;
  if (c.rest > 0 && c.rest < at_once)
    c.splits = (int)std::max(
        1L, std::min<long>(at_once / c.rest,
                           keys / (!c.few ? 128 : always ? 256 : 384)));
  if (c.splits == 1 && !always) c.rest = 0;
  return c;
}

template <bool DECODE>
void launch(const torch::Tensor& qkv, const torch::Tensor& prefix, int H,
            int D, const torch::Tensor& slopes, const torch::Tensor& info,
            const float* norms, __bf16* out, float* part_o, float* part_ml, int T, int P,
            const Cut& c) {
  const __bf16* pre = (const __bf16*)prefix.data_ptr();
  const __bf16* pk = pre + (long)H * D;
  const __bf16* pv = pre + 2L * H * D;
#define ARGS                                                                 \
  cur_stream(), (const __bf16*)qkv.data_ptr(), qkv.stride(0), pk, pv,        \
      prefix.stride(0), slopes.data_ptr<float>(), info.data_ptr<int>(),      \
      norms, out, part_o, part_ml, T, P, H, c.first_split, c.rest,                  \
      c.splits
#define LAUNCH(SHAPE)                                                        \
  hipLaunchKernelGGL((prefix_attn_kernel<SHAPE, DECODE>), dim3(c.groups()),  \
                     dim3(SHAPE::THREADS), SHAPE::BYTES, ARGS)
  if (D == 64) {
    if (c.few) { LAUNCH(FewRows<64>); } else { LAUNCH(ManyRows<64>); }
  } else {
    if (c.few) { LAUNCH(FewRows<128>); } else { LAUNCH(ManyRows<128>); }
  }
#undef LAUNCH
#undef ARGS
}

// Rows of [q | k | v], 16-byte accesses allowed.
torch::Tensor rows_of(const torch::Tensor& t, long width) {
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

Args check(const char* name, const torch::Tensor& qkv,
           const torch::Tensor& prefix, long H, const torch::Tensor& slopes,
           const torch::Tensor& info, const char* info_name) {
  TORCH_CHECK(!at::GradMode::is_enabled() ||
                  !(qkv.requires_grad() || prefix.requires_grad() ||
                    slopes.requires_grad()),
              name, ": no backward pass; call it under torch.no_grad()");
  TORCH_CHECK_VALUE(H > 0 && H < 65536 && qkv.dim() == 2 &&
                        qkv.size(1) % (3 * H) == 0,
                    name, ": qkv must be [rows, 3 * n_heads * d], got ",
                    qkv.sizes(), " for ", H, " heads");
  for (const auto* t : {&qkv, &prefix, &slopes}) check_no_tangent(*t, name);
  const long width = qkv.size(1), D = width / (3 * H);
  TORCH_CHECK_VALUE(prefix.dim() == 2 && prefix.size(1) == width, name,
                    ": prefix_qkv must be [P, ", width, "], got ",
                    prefix.sizes());
  const auto dev = qkv.device();
  TORCH_CHECK_VALUE(prefix.scalar_type() == qkv.scalar_type() &&
                        prefix.device() == dev,
                    name, ": prefix_qkv must have qkv's dtype and device");
  TORCH_CHECK_VALUE(slopes.dim() == 1 && slopes.size(0) == H, name,
                    ": slopes must be [", H, "], got ", slopes.sizes());
  TORCH_CHECK_VALUE(info.scalar_type() == at::kInt && info.dim() == 1 &&
                        info.size(0) == qkv.size(0),
                    name, ": ", info_name, " must be int32 [", qkv.size(0),
                    "], got ", info.dtype(), " ", info.sizes());
  TORCH_CHECK_VALUE(info.device() == dev, name, ": ", info_name,
                    " must be on ", dev);
  TORCH_CHECK(qkv.is_cuda() && qkv.scalar_type() == at::kBFloat16, name,
              ": qkv must be bf16 on a GPU (impl=\"torch\" takes others)");
  TORCH_CHECK(D == 64 || D == 128, name, ": d_head must be 64 or 128, got ", D);
  TORCH_CHECK(qkv.size(0) < (1L << 30) && prefix.size(0) < (1L << 30) &&
                  width < (1L << 23),
              name, ": too many rows, or too long ones");
  Args a;
  a.qkv = rows_of(qkv, width);
  a.prefix = rows_of(prefix, width);
  a.T = (int)qkv.size(0);
  a.P = (int)prefix.size(0);
  a.H = (int)H;
  a.D = (int)D;
  a.slopes = slopes.device() == dev && slopes.scalar_type() == at::kFloat
                 ? slopes.contiguous()
                 : slopes.to(dev, at::kFloat).contiguous();
  a.info = info.contiguous();
  return a;
}

// The splits' partial rows, and behind them their maxima and sums.
struct Partial {
  torch::Tensor t;
  float *o = nullptr, *ml = nullptr;
  Partial() = default;
  Partial(const Cut& c, int D, const torch::Tensor& like) {
    if (c.rest == 0) return;
    t = torch::empty({c.partial_rows() * (D + 2)},
                     like.options().dtype(at::kFloat));
    o = t.data_ptr<float>();
    ml = o + c.partial_rows() * D;
  }
};

}  // namespace

torch::Tensor prefix_attention(torch::Tensor qkv, torch::Tensor prefix, long H,
                               torch::Tensor slopes, torch::Tensor starts) {
  const c10::DeviceGuard guard(qkv.device());
  const Args a = check("prefix_attention_qkv", qkv, prefix, H, slopes, starts,
                       "starts");
  auto out = torch::empty({(long)a.T, (long)a.H * a.D}, qkv.options());
  if (a.T == 0) return out;
  const Cut c = cut(a.T, a.H, a.D, (long)a.P + 64, false);
  const Partial part(c, a.D, qkv);
  torch::Tensor norms;
  // The keys' lengths, by which far tiles are left out, where that is worth the
  // pass: more than one round of workgroups (in one, the flattest head's take as
  // long as before) over a long prefix. 32 heads of 128, 4000 rows: 237 us
  // without and 195 with over 4000 keys, 145 and 143 over 2000, 93 and 94 over
  // 1000; 2000 rows (one round) over 4000 keys 121 and 120.
  if (c.first_split > 0 && a.P >= 2500 && a.P < (1 << 28)) {  // (grid.x)
    const int tiles = (a.P + NORM_KEYS - 1) / NORM_KEYS;
    norms = torch::empty({(long)a.H * tiles}, qkv.options().dtype(at::kFloat));
    auto fn = a.D == 64 ? key_norms_kernel<64> : key_norms_kernel<128>;
    hipLaunchKernelGGL(fn, dim3(tiles, a.H), dim3(256), 0, cur_stream(),
                       (const __bf16*)a.prefix.data_ptr() + (long)a.H * a.D,
                       a.prefix.stride(0), norms.data_ptr<float>(), a.P);
  }
  launch<false>(a.qkv, a.prefix, a.H, a.D, a.slopes, a.info,
                norms.defined() ? norms.data_ptr<float>() : nullptr,
                (__bf16*)out.data_ptr(), part.o, part.ml, a.T, a.P, c);
  if (c.rest) {
    const long threads = (long)c.rest * c.rows * a.D / 4;
    auto join = a.D == 64 ? prefix_join_kernel<64> : prefix_join_kernel<128>;
    hipLaunchKernelGGL(join, dim3((unsigned)((threads + 255) / 256)),
                       dim3(256), 0, cur_stream(), part.o, part.ml,
                       (__bf16*)out.data_ptr(), a.T, a.H, c.rows, c.first_split,
                       c.rest, c.splits, !c.few && a.H % 8 == 0);
  }
  return out;
}

torch::Tensor prefix_attention_decode(torch::Tensor qkv, torch::Tensor prefix,
                                      long H, torch::Tensor slopes,
                                      torch::Tensor cache, torch::Tensor held) {
  const char* name = "prefix_attention_decode";
  const c10::DeviceGuard guard(qkv.device());
  const Args a = check(name, qkv, prefix, H, slopes, held, "held");
  const long B = a.T;
  TORCH_CHECK_VALUE(cache.dim() == 5 && cache.size(0) == B &&
                        cache.size(2) == 2 && cache.size(3) == H &&
                        cache.size(4) == a.D,
                    name, ": cache must be [", B, ", slots, 2, ", H, ", ", a.D,
                    "], got ", cache.sizes());
  TORCH_CHECK_VALUE(cache.scalar_type() == qkv.scalar_type() &&
                        cache.device() == qkv.device(),
                    name, ": cache must have qkv's dtype and device");
  bool fits = cache.stride(4) == 1 && ((uintptr_t)cache.data_ptr() % 16) == 0;
  for (int d = 0; d < 4; ++d)
    fits = fits && cache.stride(d) % 8 == 0 &&
           (cache.size(d) <= 1 || cache.stride(d) != 0);
  TORCH_CHECK(fits, name,
              ": the cache's last dimension must be contiguous and its rows "
              "aligned to 16 bytes");
  TORCH_CHECK(B < 65536 && cache.size(1) < (1L << 30), name,
              ": too many sequences or slots");
  check_writable(cache, name, "the cache");
  check_no_tangent(cache, name);
  auto out = torch::empty({B, (long)a.H * a.D}, qkv.options());
  if (B == 0) return out;
  Cut c{};
  c.rows = 1;
  // Up to a workgroup a CU each is a large one, which also attends a short
  // prefix by itself: there is next to nothing to share, and one kernel is the
  // shorter chain. 12 heads of 64 over 700 keys, 1 to 16 sequences: 7.4 us, and
  // 10.6 in two kernels; 32 heads of 128, 1 to 4 sequences, over 1000 keys 10.2
  // and 13.6, over 2000 keys 17 and 16; 16 sequences of them over 700 keys 16.9
  // and 13.8. Caches of 4000 own keys, 32 heads of 128: 30 us, and 71 in small
  // workgroups.
  const bool large = B * a.H <= 256;
  const bool direct = large && a.P > 0 && (long)a.P * a.D <= 160000;
  if (a.P > 0 && !direct) c = cut(B, a.H, a.D, a.P, true);
  const Partial part(c, a.D, qkv);
  if (a.P > 0 && !direct)
    launch<true>(a.qkv, a.prefix, a.H, a.D, a.slopes, a.info, nullptr,
                 nullptr, part.o,
                 part.ml, a.T, a.P, c);
  const __bf16* pk = (const __bf16*)a.prefix.data_ptr() + (long)a.H * a.D;
  auto own = large ? (a.D == 64 ? decode_own_kernel<64, LARGE_BLOCK>
                                : decode_own_kernel<128, LARGE_BLOCK>)
                   : (a.D == 64 ? decode_own_kernel<64, OWN_BLOCK>
                                : decode_own_kernel<128, OWN_BLOCK>);
  hipLaunchKernelGGL(own, dim3(a.H, (unsigned)B),
                     dim3(large ? LARGE_BLOCK : OWN_BLOCK), 0,
                     cur_stream(), (const __bf16*)a.qkv.data_ptr(),
                     a.qkv.stride(0), (__bf16*)cache.data_ptr(),
                     cache.stride(0), cache.stride(1), cache.stride(2),
                     cache.stride(3), a.slopes.data_ptr<float>(),
                     a.info.data_ptr<int>(), pk, pk + (long)a.H * a.D,
                     a.prefix.stride(0), direct ? a.P : 0, part.o, part.ml,
                     (__bf16*)out.data_ptr(), a.H, (int)cache.size(1), c.rows,
                     c.items, c.splits);
  cache.unsafeGetTensorImpl()->bump_version();  // written in place
  return out;
}

}  // namespace photon_hip
