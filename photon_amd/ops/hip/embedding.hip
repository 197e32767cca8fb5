// Embedding lookup with scaling, and its gradient by sorted tokens (CDNA4).
//
//   forward:  y[n, :]  = round(scale * W[ids[n], :])
//   backward: dW[v, :] = round(scale * sum over {n: ids[n] = v} of dy[n, :])
//
// Both only move memory. The gradient is a dense [V, D] tensor, so most of
// what it writes are the zero rows of the tokens that did not occur.
//
// Bound by memory. 65536 ids of a text, 50368 x 768 fp32, bf16 out (135 us):
// the lookup takes 43 us (106 MB fetched, 98 MB written), clearing the
// gradient beside the sort 42 (155 MB; the sort alone takes 20), the sums 43
// (131 + 54 MB), the join 8. A large copy moves 4.7 TB/s on this card.
//
// The sum is deterministic: positions are sorted by (token, position) with a
// stable radix sort, every wave adds up the rows of CHUNK sorted positions,
// and a token whose positions spread over several chunks is joined from the
// chunks' partial rows in their order. Floating-point atomics would be
// shorter, but their order changes from run to run, and the frequent tokens
// of a text serialise on their rows. Sums are held in fp32 and rounded once.
//
// Ids outside [0, V) read as NaN rows and have no gradient.

#include "host_common.h"


namespace photon_hip {

namespace {

constexpr int EMB_BLOCK = 256;
constexpr long MAX_GRID = 1L << 23;  // blocks; a grid has < 2^32 threads

// VEC elements of a row, widened to fp32
template <int VEC, typename T>
DEV_INLINE void load_vec(const T* p, float* f) {
  if constexpr (VEC == 1) {
    f[0] = load_f32<T>(p, 0);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const floatx4 v = load4<T>(p + i);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
  }
}

DEV_INLINE unsigned short round_bf16(float f) {
  union { __bf16 b; unsigned short u; } r;
  r.b = (__bf16)f;  // nearest even, NaN stays NaN
  return r.u;
}

template <int VEC, typename T>
DEV_INLINE void store_vec(T* p, const float* f) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (VEC == 1) {
      p[0] = f[0];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 4)
        *reinterpret_cast<floatx4*>(p + i) =
            floatx4{f[i], f[i + 1], f[i + 2], f[i + 3]};
    }
  } else {
    if constexpr (VEC == 1) {
      p[0] = round_bf16(f[0]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        shortx4 r;
        r.x = (short)round_bf16(f[i]);
        r.y = (short)round_bf16(f[i + 1]);
        r.z = (short)round_bf16(f[i + 2]);
        r.w = (short)round_bf16(f[i + 3]);
        *reinterpret_cast<shortx4*>(p + i) = r;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Forward: a block copies `rows` rows, a thread VEC columns at a time.
// ---------------------------------------------------------------------------
template <typename I, typename TW, typename TO, int VEC>
__global__ __launch_bounds__(EMB_BLOCK) void embed_fwd_kernel(
    const I* __restrict__ ids, const TW* __restrict__ w, long w_rs,
    TO* __restrict__ out, long N, int D, long V, float scale, int rows) {
  const int cpr = D / VEC;
  for (long row0 = (long)blockIdx.x * rows; row0 < N;
       row0 += (long)gridDim.x * rows) {
    const int items = (int)min((long)rows, N - row0) * cpr;
#pragma unroll 4
    for (int i = threadIdx.x; i < items; i += EMB_BLOCK) {
      const int r = i / cpr;
      const int c = (i - r * cpr) * VEC;
      const long id = (long)ids[row0 + r];
      float f[VEC];
      if (id >= 0 && id < V) {
        load_vec<VEC, TW>(w + id * w_rs + c, f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] *= scale;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = __builtin_nanf("");
      }
      store_vec<VEC, TO>(out + (row0 + r) * (long)D + c, f);
    }
  }
}

// ---------------------------------------------------------------------------
// Backward, step 1: stable radix sort of (token, position), 8 bits a pass.
//
// A block owns `rounds` * SORT_TILE consecutive items. A pass counts digits a
// block and then scatters; every scatter block derives its places from all
// blocks' counts, which stands for a scan kernel in between. At most
// SORT_BLOCKS blocks, so that these counts stay at 128 KiB. (Counting the next
// pass's digits with atomics while scattering saves a launch and took 8 us
// more than it at 65536 positions.)
//
// The sort is bound by latencies and leaves the memory idle; the blocks behind
// the sorting ones use that time to clear the gradient, a share in each kernel
// (a row that has tokens is written again by step 2).
// ---------------------------------------------------------------------------
constexpr int SORT_BLOCKS = 128;
constexpr int ITEMS = 4;  // a lane and round
constexpr int SORT_TILE = EMB_BLOCK * ITEMS;
constexpr int DIGITS = 256;
constexpr int SORT_WAVES = EMB_BLOCK / WAVE;

struct Fill {
  uint4* p;   // aligned to 16 bytes
  long n;     // 16-byte words
  int first;  // first block that clears
};

DEV_INLINE void clear(const Fill& f) {
  const long step = (long)(gridDim.x - f.first) * EMB_BLOCK;
#pragma unroll 4
  for (long i = (long)(blockIdx.x - f.first) * EMB_BLOCK + threadIdx.x; i < f.n;
       i += step)
    f.p[i] = uint4{0, 0, 0, 0};
}

template <typename I>
DEV_INLINE unsigned token_key(const I* ids, long i, long V) {
  const long id = (long)ids[i];
  return (id >= 0 && id < V) ? (unsigned)id : (unsigned)V;  // sorted last
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(EMB_BLOCK) void sort_count_kernel(
    const I* __restrict__ ids, const unsigned* __restrict__ keys, int N, long V,
    int rounds, int shift, unsigned* __restrict__ counts, const Fill fill) {
  if ((int)blockIdx.x >= fill.first) return clear(fill);
  __shared__ unsigned hist[DIGITS];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const long tile = (long)rounds * SORT_TILE;
  const long b0 = blockIdx.x * tile;
  const long b1 = min(b0 + tile, (long)N);
#pragma unroll 4
  for (long i = b0 + threadIdx.x; i < b1; i += EMB_BLOCK) {
    const unsigned k = FIRST ? token_key(ids, i, V) : keys[i];
    atomicAdd(&hist[(k >> shift) & 255u], 1u);
  }
  __syncthreads();
  counts[blockIdx.x * DIGITS + threadIdx.x] = hist[threadIdx.x];
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(EMB_BLOCK) void sort_scatter_kernel(
    const I* __restrict__ ids, const unsigned* __restrict__ keys_in,
    const unsigned* __restrict__ pos_in, unsigned* __restrict__ keys_out,
    unsigned* __restrict__ pos_out, int N, long V, int rounds, int shift,
    const unsigned* __restrict__ counts, const Fill fill) {
  if ((int)blockIdx.x >= fill.first) return clear(fill);
  __shared__ unsigned offs[SORT_WAVES][DIGITS];
  __shared__ unsigned wave_totals[SORT_WAVES];
  const int tid = threadIdx.x;
  const int lane = tid & (WAVE - 1);
  const int wid = tid / WAVE;
  const int nblk = fill.first;
  const long tile = (long)rounds * SORT_TILE;

  // a wave owns a quarter of the tile, in order; a round's items are loaded
  // together
  const long per_wave = tile / SORT_WAVES;
  const long w0 = blockIdx.x * tile + wid * per_wave;
  const long w1 = min(w0 + per_wave, (long)N);
  unsigned key[ITEMS], pos[ITEMS];
  auto load = [&](int round) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const long i = w0 + ((long)round * ITEMS + j) * WAVE + lane;
      key[j] = pos[j] = 0;
      if (i < w1) {
        key[j] = FIRST ? token_key(ids, i, V) : keys_in[i];
        pos[j] = FIRST ? (unsigned)i : pos_in[i];
      }
    }
  };
  load(0);

  // this thread's digit: items in earlier blocks, and in all blocks
  unsigned before = 0, total = 0;
#pragma unroll 32
  for (int b = 0; b < nblk; ++b) {
    const unsigned c = counts[b * DIGITS + tid];
    total += c;
    before += b < (int)blockIdx.x ? c : 0u;
  }
#pragma unroll
  for (int w = 0; w < SORT_WAVES; ++w) offs[w][tid] = 0;
  unsigned scan = total;  // inclusive, over the wave's digits
#pragma unroll
  for (int d = 1; d < WAVE; d <<= 1) {
    const unsigned x = __shfl_up(scan, d, WAVE);
    if (lane >= d) scan += x;
  }
  if (lane == WAVE - 1) wave_totals[wid] = scan;
  __syncthreads();
  unsigned base = scan - total + before;
  for (int w = 0; w < wid; ++w) base += wave_totals[w];

  for (int r = 0; r < rounds; ++r) {
    if (r > 0) load(r);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (w0 + ((long)r * ITEMS + j) * WAVE + lane < w1)
        atomicAdd(&offs[wid][(key[j] >> shift) & 255u], 1u);
  }
  __syncthreads();
  unsigned run = base;
#pragma unroll
  for (int w = 0; w < SORT_WAVES; ++w) {
    const unsigned c = offs[w][tid];
    offs[w][tid] = run;
    run += c;
  }
  __syncthreads();
  volatile unsigned* mine = offs[wid];
  for (int r = 0; r < rounds; ++r) {
    if (rounds > 1) load(r);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const bool live = w0 + ((long)r * ITEMS + j) * WAVE + lane < w1;
      const unsigned k = key[j];
      const unsigned digit = (k >> shift) & 255u;
      unsigned long long same = __ballot(live);
#pragma unroll
      for (int bit = 0; bit < 8; ++bit) {
        const unsigned long long one = __ballot((digit >> bit) & 1u);
        same &= ((digit >> bit) & 1u) ? one : ~one;
      }
      if (live) {
        const int rank = __popcll(same & ((1ull << lane) - 1ull));
        const unsigned at = mine[digit];
        __builtin_amdgcn_wave_barrier();
        if (rank == 0) mine[digit] = at + (unsigned)__popcll(same);
        const unsigned dst = at + rank;
        keys_out[dst] = k;
        pos_out[dst] = pos[j];
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// Up to ONE_BLOCK_IDS positions: all passes in one workgroup, the items in
// registers and one exchange through LDS a pass, beside the blocks that clear
// the gradient. Every launch costs the host 3 to 4 us, and four of them are
// longer than the sort.
constexpr int ONE_BLOCK = 1024;
constexpr int ONE_WAVES = ONE_BLOCK / WAVE;
constexpr long ONE_BLOCK_IDS = ONE_BLOCK * 16;

template <typename I, int ONE_ITEMS>
__global__ __launch_bounds__(ONE_BLOCK) void sort_one_block_kernel(
    const I* __restrict__ ids, unsigned* __restrict__ keys_out,
    unsigned* __restrict__ pos_out, int N, long V, int passes,
    const Fill fill) {
  if ((int)blockIdx.x >= fill.first) {
    const long step = (long)(gridDim.x - fill.first) * ONE_BLOCK;
#pragma unroll 4
    for (long i = (long)(blockIdx.x - fill.first) * ONE_BLOCK + threadIdx.x;
         i < fill.n; i += step)
      fill.p[i] = uint4{0, 0, 0, 0};
    return;
  }
  __shared__ unsigned s_key[ONE_BLOCK * ONE_ITEMS];
  __shared__ unsigned s_pos[ONE_BLOCK * ONE_ITEMS];
  __shared__ unsigned offs[ONE_WAVES][DIGITS];
  __shared__ unsigned wave_totals[SORT_WAVES];
  const int tid = threadIdx.x;
  const int lane = tid & (WAVE - 1);
  const int wid = tid / WAVE;
  const int i0 = wid * (WAVE * ONE_ITEMS) + lane;  // a wave's items are in order
  unsigned key[ONE_ITEMS], pos[ONE_ITEMS];
#pragma unroll
  for (int j = 0; j < ONE_ITEMS; ++j) {
    const int i = i0 + j * WAVE;
    key[j] = i < N ? token_key(ids, i, V) : 0u;
    pos[j] = (unsigned)i;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = 8 * p;
    for (int i = tid; i < ONE_WAVES * DIGITS; i += ONE_BLOCK)
      (&offs[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ONE_ITEMS; ++j)
      if (i0 + j * WAVE < N) atomicAdd(&offs[wid][(key[j] >> shift) & 255u], 1u);
    __syncthreads();
    unsigned total = 0, scan = 0;
    if (tid < DIGITS) {
#pragma unroll
      for (int w = 0; w < ONE_WAVES; ++w) total += offs[w][tid];
      scan = total;
#pragma unroll
      for (int d = 1; d < WAVE; d <<= 1) {
        const unsigned x = __shfl_up(scan, d, WAVE);
        if (lane >= d) scan += x;
      }
      if (lane == WAVE - 1) wave_totals[wid] = scan;
    }
    __syncthreads();
    if (tid < DIGITS) {
      unsigned run = scan - total;
      for (int w = 0; w < wid; ++w) run += wave_totals[w];
#pragma unroll
      for (int w = 0; w < ONE_WAVES; ++w) {
        const unsigned c = offs[w][tid];
        offs[w][tid] = run;
        run += c;
      }
    }
    __syncthreads();
    volatile unsigned* mine = offs[wid];
#pragma unroll
    for (int j = 0; j < ONE_ITEMS; ++j) {
      const bool live = i0 + j * WAVE < N;
      const unsigned digit = (key[j] >> shift) & 255u;
      unsigned long long same = __ballot(live);
#pragma unroll
      for (int bit = 0; bit < 8; ++bit) {
        const unsigned long long one = __ballot((digit >> bit) & 1u);
        same &= ((digit >> bit) & 1u) ? one : ~one;
      }
      if (live) {
        const int rank = __popcll(same & ((1ull << lane) - 1ull));
        const unsigned at = mine[digit];
        __builtin_amdgcn_wave_barrier();
        if (rank == 0) mine[digit] = at + (unsigned)__popcll(same);
        s_key[at + rank] = key[j];
        s_pos[at + rank] = pos[j];
      }
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ONE_ITEMS; ++j) {
      const int i = i0 + j * WAVE;
      if (i < N) {
        key[j] = s_key[i];
        pos[j] = s_pos[i];
      }
    }
    // (the next pass's two barriers stand between these reads and its writes)
  }
#pragma unroll
  for (int j = 0; j < ONE_ITEMS; ++j) {
    const int i = i0 + j * WAVE;
    if (i < N) {
      keys_out[i] = key[j];
      pos_out[i] = pos[j];
    }
  }
}

// ---------------------------------------------------------------------------
// Backward, step 2: sums over CHUNK sorted positions, COLS columns a wave.
// A segment (one token's positions) inside its chunk is final; one that came
// from the chunk before goes to head[chunk], one that goes on to the next
// (and began here) to tail[chunk].
// ---------------------------------------------------------------------------
constexpr int CHUNK = 32;

template <typename TG, typename TW, int VEC>
__global__ __launch_bounds__(EMB_BLOCK) void embed_sum_kernel(
    const TG* __restrict__ dy, const unsigned* __restrict__ keys,
    const unsigned* __restrict__ pos, TW* __restrict__ dw,
    float* __restrict__ head, float* __restrict__ tail, int N, int D, long V,
    float scale) {
  constexpr int COLS = WAVE * VEC;
  const int lane = threadIdx.x & (WAVE - 1);
  const int wid = threadIdx.x / WAVE;
  const int tiles = (D + COLS - 1) / COLS;
  const long item = (long)blockIdx.x * SORT_WAVES + wid;
  const long chunk = item / tiles;
  const int c = (int)(item - chunk * tiles) * COLS + lane * VEC;
  const long first = chunk * CHUNK;
  if (first >= N) return;
  const int count = (int)min((long)CHUNK, N - first);
  const bool in = c < D;
  // lane i holds sorted position first + i; lane CHUNK looks one further
  const long mine = first + lane;
  const unsigned key = (lane <= count && mine < N) ? keys[mine] : 0xffffffffu;
  const unsigned p = (lane < count) ? pos[mine] : 0u;
  const unsigned last = first > 0 ? keys[first - 1] : 0xffffffffu;
  bool from_before = (unsigned)__builtin_amdgcn_readlane(key, 0) == last;

  float acc[VEC] = {};
  // Rows in flight: 8 take 43 us at 65536 x 768; 16 and 32 cost the registers
  // of other waves and take 65 and 108.
  constexpr int U = 8;
  for (int i0 = 0; i0 < count; i0 += U) {
    float f[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned row = __builtin_amdgcn_readlane(p, i0 + u);
      if (in) load_vec<VEC, TG>(dy + (long)row * D + c, f[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i < count) {
        const unsigned k = __builtin_amdgcn_readlane(key, i);
        const unsigned next = __builtin_amdgcn_readlane(key, i + 1);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += f[u][j];
        const bool ends = i + 1 == count || next != k;
        if (ends) {
          const bool goes_on = i + 1 == count && next == k;
          if (in && k < (unsigned)V) {
            if (from_before) {
              store_vec<VEC, float>(head + chunk * D + c, acc);
            } else if (goes_on) {
              store_vec<VEC, float>(tail + chunk * D + c, acc);
            } else {
#pragma unroll
              for (int j = 0; j < VEC; ++j) acc[j] *= scale;
              store_vec<VEC, TW>(dw + (long)k * D + c, acc);
            }
          }
          from_before = false;
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        }
      }
    }
  }
}

// Step 3: a token that leaves the chunk it began in is that chunk's tail and
// the heads of the chunks up to the one that holds its last position. The
// block's waves take every eighth of them and are added in order. One block
// for each chunk and column tile; most find nothing to join. Bound by the
// latencies of the most frequent token: 8 us at 65536 positions of a text,
// also where eight chunks share a block.
constexpr int JOIN_BLOCK = 512;
constexpr int JOIN_WAVES = JOIN_BLOCK / WAVE;
template <typename TW, int VEC>
__global__ __launch_bounds__(JOIN_BLOCK) void embed_join_kernel(
    const unsigned* __restrict__ keys, const float* __restrict__ head,
    const float* __restrict__ tail, TW* __restrict__ dw, int N, int D, long V,
    float scale) {
  constexpr int COLS = WAVE * VEC;
  __shared__ float sums[JOIN_WAVES][COLS];
  const int lane = threadIdx.x & (WAVE - 1);
  const int wid = threadIdx.x / WAVE;
  const long chunk = blockIdx.x;
  const long first = chunk * CHUNK;
  const long end = first + CHUNK;  // first position of the next chunk
  if (end >= N) return;
  const unsigned k = keys[end - 1];
  const unsigned k_next = keys[end];
  const unsigned k_first = keys[first];
  const unsigned k_before = keys[max(first - 1, 0L)];
  const unsigned k_far = keys[min(end + CHUNK, (long)N) - 1];
  if (k_next != k || k >= (unsigned)V) return;
  if (first > 0 && k_first == k && k_before == k) return;
  long last = chunk + 1;  // heads chunk + 1 .. last
  if (k_far == k) {
    // last position of the token, 64 probes at a time
    long lo = end, n = N - end;  // keys[lo] is the token's, lo + n is behind
    while (n > 1) {
      const long step = (n + WAVE - 1) / WAVE;
      const long at = lo + lane * step;
      const bool mine = at < lo + n && keys[at] == k;
      const int found = __popcll(__ballot(mine));  // lanes 0 .. found - 1
      n = min(step, n - (found - 1) * step);
      lo += (found - 1) * step;
    }
    last = lo / CHUNK;
  }
  const int c = blockIdx.y * COLS + lane * VEC;
  float acc[VEC] = {};
  if (c < D) {
    if (wid == 0) load_vec<VEC, float>(tail + chunk * D + c, acc);
#pragma unroll 8
    for (long h = chunk + 1 + wid; h <= last; h += JOIN_WAVES) {
      float f[VEC];
      load_vec<VEC, float>(head + h * D + c, f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += f[j];
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) sums[wid][lane * VEC + j] = acc[j];
  __syncthreads();
  if (wid == 0 && c < D) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float s = sums[0][lane * VEC + j];
#pragma unroll
      for (int w = 1; w < JOIN_WAVES; ++w) s += sums[w][lane * VEC + j];
      acc[j] = s * scale;
    }
    store_vec<VEC, TW>(dw + (long)k * D + c, acc);
  }
}

bool aligned(const void* p, int bytes) { return ((uintptr_t)p % bytes) == 0; }

}  // namespace

#define DISPATCH_IDS(TENSOR, ...)                                        \
  if ((TENSOR).scalar_type() == at::kLong) {                             \
    using id_t = long;                                                   \
    __VA_ARGS__;                                                         \
  } else {                                                               \
    using id_t = int;                                                    \
    __VA_ARGS__;                                                         \
  }

// Two tensors' types at once; TORCH_CHECKed by embedding().
#define DISPATCH_TWO(A, B, ...)                                          \
  if ((A) == at::kBFloat16 && (B) == at::kBFloat16) {                    \
    using a_t = unsigned short; using b_t = unsigned short;              \
    __VA_ARGS__;                                                         \
  } else if ((A) == at::kBFloat16) {                                     \
    using a_t = unsigned short; using b_t = float;                       \
    __VA_ARGS__;                                                         \
  } else if ((B) == at::kBFloat16) {                                     \
    using a_t = float; using b_t = unsigned short;                       \
    __VA_ARGS__;                                                         \
  } else {                                                               \
    using a_t = float; using b_t = float;                                \
    __VA_ARGS__;                                                         \
  }

torch::Tensor embedding_fwd(const torch::Tensor& ids_in,
                            const torch::Tensor& w, double scale,
                            at::ScalarType out_dtype) {
  const c10::DeviceGuard guard(w.device());
  auto ids = ids_in.contiguous();
  const long N = ids.numel(), V = w.size(0);
  const int D = (int)w.size(1);
  auto sizes = ids.sizes().vec();
  sizes.push_back(D);
  auto out = torch::empty(sizes, w.options().dtype(out_dtype));
  if (N == 0 || D == 0) return out;
  const long rs = w.stride(0);
  const bool wide = D % 4 == 0 && rs % 4 == 0 &&
                    aligned(w.data_ptr(), 4 * (int)w.element_size());
  const bool wider = wide && D % 8 == 0 && rs % 8 == 0 &&
                     aligned(w.data_ptr(), 16);
  // Four vectors a thread, as wide as D allows: 65536 rows of 768 fp32 take 43
  // us with vectors of 8 and 53 with 4 (106 MB fetched, 98 MB written).
  const int vec = wider ? 8 : wide ? 4 : 1;
  const int rows = std::max(1, 4 * EMB_BLOCK / std::max(1, D / vec));
  const long blocks = std::min<long>((N + rows - 1) / rows, MAX_GRID);
  DISPATCH_IDS(ids, DISPATCH_TWO(w.scalar_type(), out_dtype, {
    auto kernel = vec == 8   ? embed_fwd_kernel<id_t, a_t, b_t, 8>
                  : vec == 4 ? embed_fwd_kernel<id_t, a_t, b_t, 4>
                             : embed_fwd_kernel<id_t, a_t, b_t, 1>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(EMB_BLOCK), 0, cur_stream(),
                       (const id_t*)ids.data_ptr(), (const a_t*)w.data_ptr(),
                       rs, (b_t*)out.data_ptr(), N, D, V, (float)scale, rows);
  }));
  return out;
}

torch::Tensor embedding_bwd(const torch::Tensor& dy_in,
                            const torch::Tensor& ids_in, long V, double scale,
                            at::ScalarType w_dtype) {
  const c10::DeviceGuard guard(dy_in.device());
  auto dy = dy_in.contiguous();
  auto ids = ids_in.contiguous();
  const long N = ids.numel();
  const int D = (int)dy.size(-1);
  TORCH_CHECK(N < (1L << 31) - CHUNK, "embedding: too many ids for a gradient");
  auto dw = torch::empty({V, (long)D}, dy.options().dtype(w_dtype));
  if (V == 0 || D == 0) return dw;
  if (N == 0) return dw.zero_();
  int passes = 1;
  while (passes < 4 && (V >> (8 * passes)) != 0) ++passes;
  const int rounds =
      (int)((N + (long)SORT_TILE * SORT_BLOCKS - 1) / ((long)SORT_TILE * SORT_BLOCKS));
  const long tile = (long)rounds * SORT_TILE;
  const bool one_block = N <= ONE_BLOCK_IDS;
  const int nblk = one_block ? 1 : (int)((N + tile - 1) / tile);
  const long chunks = (N + CHUNK - 1) / CHUNK;

  // One workspace: heads and tails, the sorted (key, position) pairs twice,
  // the counts.
  const long parts = 2 * chunks * D, sorted = one_block ? 2 * N : 4 * N;
  auto space = torch::empty({parts + sorted + (long)nblk * DIGITS},
                            dy.options().dtype(at::kFloat));
  float* head = space.data_ptr<float>();
  float* tail = head + chunks * D;
  unsigned* sp = (unsigned*)(head + parts);
  unsigned* cp = sp + sorted;
  const auto stream = cur_stream();
  // The gradient's 16-byte words in shares: one for each counting kernel, two
  // for each (longer) scatter kernel. Its last bytes are cleared by themselves.
  const long bytes = dw.numel() * (long)dw.element_size();
  const long words = bytes / 16;
  if (bytes % 16 != 0)
    dw.flatten().slice(0, words * 16 / (long)dw.element_size()).zero_();
  const int shares = one_block ? 1 : 3 * passes;
  auto share = [&](int from, int to) {
    const long a = words * from / shares, b = words * to / shares;
    return Fill{(uint4*)dw.data_ptr() + a, b - a, nblk};
  };
  // four stores a thread, 4096 blocks of 256 at most
  auto blocks = [&](const Fill& f, int threads) {
    return dim3(nblk + (unsigned)std::min<long>((f.n + 4 * threads - 1) / (4 * threads),
                                                4096 * EMB_BLOCK / threads));
  };
  int at_pair = 0;
  DISPATCH_IDS(ids, {
    const id_t* ip = (const id_t*)ids.data_ptr();
    if (one_block) {
      const Fill f = share(0, 1);
      auto sort = N <= 4 * ONE_BLOCK ? sort_one_block_kernel<id_t, 4>
                                     : sort_one_block_kernel<id_t, 16>;
      hipLaunchKernelGGL(sort, blocks(f, ONE_BLOCK), dim3(ONE_BLOCK), 0, stream,
                         ip, sp, sp + N, (int)N, V, passes, f);
      at_pair = 1;
    }
    for (int p = 0; !one_block && p < passes; ++p) {
      unsigned* in = sp + (long)(1 - at_pair) * 2 * N;
      unsigned* to = sp + (long)at_pair * 2 * N;
      const Fill f0 = share(3 * p, 3 * p + 1), f1 = share(3 * p + 1, 3 * p + 3);
      auto count = p == 0 ? sort_count_kernel<id_t, true>
                          : sort_count_kernel<id_t, false>;
      hipLaunchKernelGGL(count, blocks(f0, EMB_BLOCK), dim3(EMB_BLOCK), 0,
                         stream, ip, in, (int)N, V, rounds, 8 * p, cp, f0);
      auto scatter = p == 0 ? sort_scatter_kernel<id_t, true>
                            : sort_scatter_kernel<id_t, false>;
      hipLaunchKernelGGL(scatter, blocks(f1, EMB_BLOCK), dim3(EMB_BLOCK), 0,
                         stream, ip, in, in + N, to, to + N, (int)N, V, rounds,
                         8 * p, cp, f1);
      at_pair = 1 - at_pair;
    }
  });
  const unsigned* keys = sp + (long)(1 - at_pair) * 2 * N;
  const unsigned* pos = keys + N;
  const bool wide = D % 4 == 0 && aligned(dy.data_ptr(), 4 * (int)dy.element_size());
  const bool wider = wide && dy.element_size() == 2 && D % 8 == 0 &&
                     aligned(dy.data_ptr(), 16);
  const int vec = wider ? 8 : wide ? 4 : 1;
  const int cols = WAVE * vec;
  const long items = chunks * ((D + cols - 1) / cols);
  const long sum_blocks = (items + SORT_WAVES - 1) / SORT_WAVES;
  const long col_tiles = (D + cols - 1) / cols;
  TORCH_CHECK(sum_blocks < MAX_GRID && chunks < MAX_GRID && col_tiles < 65536,
              "embedding: gradient too large");
  DISPATCH_TWO(dy.scalar_type(), w_dtype, {
    auto sum = vec == 8   ? embed_sum_kernel<a_t, b_t, 8>
               : vec == 4 ? embed_sum_kernel<a_t, b_t, 4>
                          : embed_sum_kernel<a_t, b_t, 1>;
    hipLaunchKernelGGL(sum, dim3(sum_blocks), dim3(EMB_BLOCK), 0, stream,
                       (const a_t*)dy.data_ptr(), keys, pos,
                       (b_t*)dw.data_ptr(), head, tail, (int)N, D, V,
                       (float)scale);
    auto join = vec == 8   ? embed_join_kernel<b_t, 8>
                : vec == 4 ? embed_join_kernel<b_t, 4>
                           : embed_join_kernel<b_t, 1>;
    if (chunks > 1)
      hipLaunchKernelGGL(join, dim3(chunks - 1, col_tiles), dim3(JOIN_BLOCK), 0,
                         stream, keys, head, tail, (b_t*)dw.data_ptr(), (int)N, D, V,
                         (float)scale);
  });
  return dw;
}

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

class EmbeddingFn : public torch::autograd::Function<EmbeddingFn> {
 public:
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor w,
                               torch::Tensor ids, double scale,
                               int64_t out_dtype) {
    at::AutoDispatchBelowADInplaceOrView g;
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["dtype"] = (int64_t)w.scalar_type();
    return embedding_fwd(ids, w, scale, (at::ScalarType)out_dtype);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "embedding: a second derivative is not supported "
                "(create_graph=True)");
    check_no_tangent(grads[0], "embedding");
    auto ids = ctx->get_saved_variables()[0];
    auto dw = embedding_bwd(grads[0], ids, ctx->saved_data["rows"].toInt(),
                            ctx->saved_data["scale"].toDouble(),
                            (at::ScalarType)ctx->saved_data["dtype"].toInt());
    return {dw, torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

bool known_dtype(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16;
}

}  // namespace

torch::Tensor embedding(torch::Tensor ids, torch::Tensor w, double scale,
                        at::ScalarType out_dtype) {
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong ||
                       ids.scalar_type() == at::kInt,
                   "embedding: ids must be int64 or int32, got ", ids.dtype());
  TORCH_CHECK_VALUE(w.dim() == 2, "embedding: table must be [V, D], got ",
                    w.sizes());
  TORCH_CHECK(w.is_cuda() && known_dtype(w.scalar_type()),
              "embedding: the table must be fp32 or bf16 on a GPU");
  TORCH_CHECK(w.size(1) < (1L << 30) && w.size(0) < (1L << 31),
              "embedding: table too large");
  TORCH_CHECK(w.size(1) <= 1 || w.stride(1) == 1,
              "embedding: a table row must be contiguous");
  TORCH_CHECK(ids.device() == w.device(), "embedding: ids on ", ids.device(),
              ", table on ", w.device());
  TORCH_CHECK(known_dtype(out_dtype), "embedding: output must be fp32 or bf16");
  check_no_tangent(w, "embedding");
  if (w.requires_grad() && at::GradMode::is_enabled())
    return EmbeddingFn::apply(w, ids, scale, (int64_t)out_dtype);
  return embedding_fwd(ids, w, scale, out_dtype);
}

}  // namespace photon_hip
