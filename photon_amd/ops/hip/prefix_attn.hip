// Attention of a batch of sequences that share a long prefix (ALiBi, CDNA4).
//
// Sequence b continues the same P tokens with its own ones. Its query at own
// position i (position P + i of the text) sees all P keys of the prefix and
// its own keys 0..i:
//
//   w = q . k / sqrt(d) - slope_h * (P + i - pos_k),  o = softmax(w) v
//
// The prefix is the same for every row of every sequence, so the rows of all
// sequences are stacked into the query tiles of ONE attention over it: a key
// tile is read once for 32 * NW rows, whatever sequence they belong to, where
// attention per sequence would read the prefix once per sequence. Behind the
// prefix come the packed rows themselves, masked to a block diagonal.
//
// The key axis can be split over workgroups: each leaves (m, l, o) with
// m = max w, l = sum e^(w - m), o = sum e^(w - m) v, and
//   M = max m_i,  o = sum e^(m_i - M) o_i / sum e^(m_i - M) l_i
// joins them. Statistics and sums are fp32; the probabilities are rounded to
// bf16 for the second matrix product, as the values they weigh are.

#include "host_common.h"
#include "attn_kernels.h"

#include <algorithm>

namespace photon_hip {

namespace {

constexpr int PKB = 64;  // keys a tile

// LDS: two buffers of a key and a value image (or, at the end, the fp32 rows
// of all waves), and a word for each wave.
constexpr int lds_images(int D, int nw) {
  const int images = 4 * PKB * D * 2, rows = nw * 32 * D * 4;
  return images > rows ? images : rows;
}
constexpr int lds_bytes(int D, int nw) { return lds_images(D, nw) + 64; }

// Swapped product (keys x queries): lane holds query lane & 31, its 16
// registers the keys (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5) of 32.
//
// `info` is each row's first own row (packed form) or, in the decode form, how
// many own keys the row's sequence holds; there the kernel covers the prefix
// only.
template <int D, int NW, bool DECODE>
__global__ __launch_bounds__(64 * NW, 2) void prefix_attn_kernel(
    const __bf16* __restrict__ qkv, long q_rs, const __bf16* __restrict__ pk,
    const __bf16* __restrict__ pv, long p_rs,
    const float* __restrict__ slopes, const int* __restrict__ info,
    __bf16* __restrict__ out, float* __restrict__ part_o,
    float* __restrict__ part_ml, int T, int P, int H, int splits) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int IMG = PKB * D * 2;  // bytes of a [64][D] image
  constexpr bool D64 = D == 64;

  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int hi = lane >> 5;
  const int lq = lane & 31;
  const int h = blockIdx.x;
  const int split = blockIdx.y % splits;
  const int q0_block = (blockIdx.y / splits) * (NW * QB);
  const int my_q = q0_block + wave * QB + lq;
  const int row = min(my_q, T - 1);

  const float scale2 = rsqrtf((float)D) * LOG2E;
  const float slope2 = slopes[h] * LOG2E;

  const __bf16* q = qkv + (long)h * D;
  const __bf16* k = q + (long)H * D;
  const __bf16* v = k + (long)H * D;
  pk += (long)h * D;
  pv += (long)h * D;

  bf16x8 qfrag[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    qfrag[kk] = *(const bf16x8*)(q + row * q_rs + kk * 16 + 8 * hi);

  // own position of this lane's row, and the first packed row it may see
  int first = 0, own = 0;
  if (DECODE) {
    own = max(info[row], 0);
  } else {
    first = min(max(info[row], 0), row);
    own = row - first;
  }

  // key tiles: the prefix's, then the packed rows lo..hi_row of this block
  const int n_pre = (P + PKB - 1) / PKB;
  int lo = 0, n_own = 0, end_row = 0;
  if (!DECODE) {
    lo = __builtin_amdgcn_readfirstlane(
        min(max(info[q0_block], 0), q0_block));
    end_row = min(q0_block + NW * QB, T);
    n_own = (end_row - lo + PKB - 1) / PKB;
  }
  const int n_all = n_pre + n_own;
  const int t0 = (int)((long)n_all * split / splits);
  const int t1 = (int)((long)n_all * (split + 1) / splits);

  float m_run = -1e30f;  // finite: exp2(-huge) == 0 and no NaN from inf - inf
  float l_run = 0.f;
  f32x16 o_acc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) o_acc[db] = f32x16{};

  float alibi2[16];
#pragma unroll
  for (int r = 0; r < 16; ++r)
    alibi2[r] = slope2 * (float)((r & 3) + 8 * (r >> 2) + 4 * hi);

  // Staging: a wave-instruction moves 1 KiB to LDS, lane by lane in order;
  // the swizzle is applied to the source. The descriptor starts at the tile
  // (64-bit base), so a prefix of any length keeps 32-bit offsets, and ends
  // with its last row: what lies behind reads as zeros.
  constexpr int NWIN = IMG / 1024 / NW;
  int dma_row[NWIN], dma_col[NWIN];
#pragma unroll
  for (int i = 0; i < NWIN; ++i) {
    const int dest = (wave * NWIN + i) * 1024 + lane * 16;
    const int r = dest / (D * 2);
    dma_row[i] = r;
    dma_col[i] =
        (dest ^ (int)(swz_field((unsigned)r & 15u, D64) << 4)) % (D * 2);
  }
  auto stage = [&](int t, int b) {
    const bool pre = t < n_pre;
    const long rs = pre ? p_rs : q_rs;
    const long at = pre ? (long)t * PKB : (long)lo + (long)(t - n_pre) * PKB;
    const int rows = min(PKB, (pre ? P : end_row) - (int)at);
    const long bytes = ((long)(rows - 1) * rs + D) * 2;
    const auto krs = make_rsrc((pre ? pk : k) + at * rs, bytes);
    const auto vrs = make_rsrc((pre ? pv : v) + at * rs, bytes);
    const int rs2 = (int)(rs * 2);
    char* dst = smem + b * 2 * IMG;
#pragma unroll
    for (int i = 0; i < NWIN; ++i) {
      const int win = (wave * NWIN + i) * 1024;
      const int off = dma_row[i] * rs2 + dma_col[i];
      lds_dma16(krs, dst + win, off, 0);
      lds_dma16(vrs, dst + IMG + win, off, 0);
    }
  };

  // LDS read addresses (see the swizzle's row rule in attn_kernels.h)
  unsigned qk_addr[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    qk_addr[kk] = swz((unsigned)(lq * (D * 2) + kk * 32 + hi * 16), lq, D64);
  const int tj = lane & 15;
  const int tg = (lane >> 4) & 1;
  unsigned pv_addr[2][D / 32];
#pragma unroll
  for (int rd = 0; rd < 2; ++rd) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      const int key0 = 8 * hi + 4 * rd + (tj >> 2);
      const int dh = db * 32 + 16 * tg + 4 * (tj & 3);
      pv_addr[rd][db] = swz((unsigned)(key0 * (D * 2) + dh * 2), key0, D64);
    }
  }
  auto scores = [&](int b, int sub) {
    f32x16 s = f32x16{};
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const bf16x8 a = *(const bf16x8*)(smem + qk_addr[kk] + b * 2 * IMG +
                                        sub * 32 * (D * 2));
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qfrag[kk], s, 0, 0, 0);
    }
    return s;
  };
  auto add_values = [&](const float* p, int b, int sub) {
#pragma unroll
    for (int s16 = 0; s16 < 2; ++s16) {
      const bf16x8 pf = pack_bfrag(p, 8 * s16);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        union { bf16x4 half[2]; bf16x8 all; } a;
#pragma unroll
        for (int rd = 0; rd < 2; ++rd)
          a.half[rd] = lds_tr16((const __bf16*)(smem + IMG),
                                pv_addr[rd][db] + b * 2 * IMG +
                                    sub * 32 * (D * 2) + s16 * 16 * (D * 2));
        o_acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.all, pf,
                                                            o_acc[db], 0, 0, 0);
      }
    }
  };
  // Rescale only when a row's maximum grew by more than 2^8: until then the
  // weights stay below 2^8 and the sums in range.
  auto raise = [&](float top) {
    if (!__all(top - m_run <= 8.f)) {
      const float m_new = fmaxf(m_run, top);
      const float a = exp2_fast(m_run - m_new);
      l_run *= a;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o_acc[db][r] *= a;
      m_run = m_new;
    }
  };

  // A weight of zero does not hide an infinity or NaN among the values it is
  // multiplied with. Prefix tiles hold nothing that a row may not see; in the
  // packed rows a value belongs to other sequences or later rows as well. So
  // values that are not finite are taken out of such a tile (returns whether
  // there were any) and added by add_bad() where they are seen.
  int* bad_words = (int*)(smem + lds_images(D, NW));
  auto take_out_bad = [&](int b) {
    unsigned* img = (unsigned*)(smem + b * 2 * IMG + IMG);
    auto bad_half = [](unsigned w, unsigned mask) { return (w & mask) == mask; };
    bool bad = false;
    for (int i = threadIdx.x; i < IMG / 4; i += 64 * NW)
      bad |= bad_half(img[i], 0x7f800000u) || bad_half(img[i], 0x7f80u);
    const bool wave_bad = __any(bad);
    if (lane == 0) bad_words[wave] = wave_bad;
    __syncthreads();
    bool any = false;
#pragma unroll
    for (int w = 0; w < NW; ++w) any |= bad_words[w] != 0;
    if (!any) return false;
    for (int i = threadIdx.x; i < IMG / 4; i += 64 * NW) {
      if (bad_half(img[i], 0x7f800000u)) img[i] &= 0xffffu;
      if (bad_half(img[i], 0x7f80u)) img[i] &= 0xffff0000u;
    }
    __syncthreads();
    return true;
  };
  auto add_bad = [&](int kv0) {
    const int end = min(kv0 + PKB, end_row);
#pragma unroll 1
    for (int key = kv0; key < end; ++key) {
      const bool seen = key >= first && key <= row;
      const __bf16* x = v + (long)key * q_rs;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float f = (float)x[db * 32 + (r & 3) + 8 * (r >> 2) + 4 * hi];
          if (seen && !(fabsf(f) < INFINITY)) o_acc[db][r] += f;
        }
    }
  };

  if (t0 < t1) stage(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int b = (t - t0) & 1;
    vm_wait0();
    __syncthreads();  // tile b is there; all reads of the other one are done
    if (t + 1 < t1) stage(t + 1, 1 - b);
    const bool pre = t < n_pre;
    if (pre && (t + 1) * PKB <= P) {  // a whole tile that every row sees
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const f32x16 s = scores(b, sub);
        float p[16], top = -1e30f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = fmaf(s[r], scale2, alibi2[r]);
          top = fmaxf(top, p[r]);
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float b2 = slope2 * (float)(t * PKB + sub * 32 - P - own);
        raise(top + b2);
        const float shift = m_run - b2;
        float l_add = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = exp2_fast(p[r] - shift);
          l_add += p[r];
        }
        l_run += l_add + __shfl_xor(l_add, 32, 64);
        add_values(p, b, sub);
      }
    } else {
      const int kv0 = pre ? t * PKB : lo + (t - n_pre) * PKB;
      const int me = pre ? P + own : row;  // position on the tile's axis
      const int from = pre ? 0 : first;
      const int to = pre ? P - 1 : row;
      const bool bad = pre ? false : take_out_bad(b);
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const int kv = kv0 + sub * 32;
        if (!__any(kv + 31 >= from && kv <= to)) continue;
        const f32x16 s = scores(b, sub);
        const float b2 = slope2 * (float)(kv - me);
        float p[16], top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kv + (r & 3) + 8 * (r >> 2) + 4 * hi;
          const float w = fmaf(s[r], scale2, alibi2[r] + b2);
          p[r] = (key >= from && key <= to) ? w : -INFINITY;
          top = fmaxf(top, p[r]);
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        raise(top);
        float l_add = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = exp2_fast(p[r] - m_run);  // exp2(-inf) == 0: m is finite
          l_add += p[r];
        }
        l_run += l_add + __shfl_xor(l_add, 32, 64);
        add_values(p, b, sub);
      }
      if (bad) add_bad(kv0);
    }
  }
  __syncthreads();  // the images are free

  // Through LDS to whole rows. A wave has the 32 x D values of its own rows.
  if (splits == 1 && !DECODE) {
    __bf16* o_img = (__bf16*)smem + wave * 32 * D;
    const float inv = l_run > 0.f ? 1.f / l_run : 0.f;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        o_img[lq * D + db * 32 + (r & 3) + 8 * (r >> 2) + 4 * hi] =
            (__bf16)(o_acc[db][r] * inv);
    __syncthreads();
    for (int c = lane; c < 32 * D / 8; c += 64) {
      const int r = q0_block + wave * QB + c / (D / 8);
      const int col = (c % (D / 8)) * 8;
      if (r < T)
        *(bf16x8*)(out + (long)r * H * D + (long)h * D + col) =
            *(const bf16x8*)(o_img + c * 8);
    }
  } else {
    float* o_img = (float*)smem + wave * 32 * D;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(f32x4*)(o_img + lq * D + db * 32 + 2 * r + 4 * hi) =
            f32x4{o_acc[db][r], o_acc[db][r + 1], o_acc[db][r + 2],
                  o_acc[db][r + 3]};
    __syncthreads();
    const long base = ((long)split * H + h) * T;
    for (int c = lane; c < 32 * D / 4; c += 64) {
      const int r = q0_block + wave * QB + c / (D / 4);
      if (r < T)
        *(f32x4*)(part_o + (base + r) * D + (c % (D / 4)) * 4) =
            *(const f32x4*)(o_img + c * 4);
    }
    if (hi == 0 && my_q < T) {
      part_ml[(base + my_q) * 2] = m_run;
      part_ml[(base + my_q) * 2 + 1] = l_run;
    }
  }
}

// Joins the splits: a thread has four columns of a row.
template <int D>
__global__ __launch_bounds__(256) void prefix_join_kernel(
    const float* __restrict__ part_o, const float* __restrict__ part_ml,
    __bf16* __restrict__ out, int T, int H, int splits) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long rh = i / (D / 4);  // row of the [H, T] rows
  const int col = (int)(i % (D / 4)) * 4;
  if (rh >= (long)H * T) return;
  const long stride = (long)H * T;
  float M = -1e30f;
  for (int s = 0; s < splits; ++s)
    M = fmaxf(M, part_ml[(s * stride + rh) * 2]);
  float l = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float w = exp2_fast(part_ml[(s * stride + rh) * 2] - M);
    l += w * part_ml[(s * stride + rh) * 2 + 1];
    const f32x4 x = *(const f32x4*)(part_o + (s * stride + rh) * D + col);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += w * x[j];
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const long h = rh / T, t = rh - h * T;
  bf16x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = (__bf16)(o[j] * inv);
  *(bf16x4*)(out + (t * H + h) * D + col) = r;
}

// Decode: one workgroup per (sequence, head) writes the new key and value to
// the cache, attends the sequence's own keys and joins what the prefix gave.
// D / 8 lanes hold a key's 8 columns each, all groups of the block stride
// over the keys with a running maximum and sum of their own.
constexpr int OWN_BLOCK = 256;
template <int D>
__global__ __launch_bounds__(OWN_BLOCK) void decode_own_kernel(
    const __bf16* __restrict__ qkv, long q_rs, __bf16* __restrict__ cache,
    long c_bs, long c_ss, long c_ks, long c_hs,
    const float* __restrict__ slopes, const int* __restrict__ held,
    const float* __restrict__ part_o, const float* __restrict__ part_ml,
    __bf16* __restrict__ out, int B, int H, int slots, int splits) {
  constexpr int L = D / 8;               // lanes a key
  constexpr int G = OWN_BLOCK / L;       // keys at a time
  __shared__ float s_o[OWN_BLOCK / 64][D];
  __shared__ float s_m[OWN_BLOCK / 64], s_l[OWN_BLOCK / 64];
  const int h = blockIdx.x;
  const int b = blockIdx.y;
  const int tid = threadIdx.x;
  const int g = tid / L;
  const int c = (tid % L) * 8;
  const __bf16* q = qkv + b * q_rs + (long)h * D;
  const int n = held[b];
  __bf16* o_row = out + ((long)b * H + h) * D;
  if (n < 0 || n >= slots) {  // no room for the new key: say so
    if (tid < D) o_row[tid] = (__bf16)__builtin_nanf("");
    return;
  }
  __bf16* ck = cache + b * c_bs + (long)h * c_hs;
  __bf16* cv = ck + c_ks;
  const bf16x8 new_k = *(const bf16x8*)(q + (long)H * D + c);
  const bf16x8 new_v = *(const bf16x8*)(q + 2L * H * D + c);
  if (g == 0) {
    *(bf16x8*)(ck + (long)n * c_ss + c) = new_k;
    *(bf16x8*)(cv + (long)n * c_ss + c) = new_v;
  }
  float qf[8];
  const bf16x8 qv = *(const bf16x8*)(q + c);
  const float scale2 = rsqrtf((float)D) * LOG2E;
  const float slope2 = slopes[h] * LOG2E;
#pragma unroll
  for (int j = 0; j < 8; ++j) qf[j] = (float)qv[j] * scale2;
  float m = -1e30f, l = 0.f, o[8] = {};
  for (int i = g; i <= n; i += G) {
    bf16x8 kv = new_k, vv = new_v;  // the new ones from registers
    if (i < n) {
      kv = *(const bf16x8*)(ck + (long)i * c_ss + c);
      vv = *(const bf16x8*)(cv + (long)i * c_ss + c);
    }
    float w = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) w = fmaf(qf[j], (float)kv[j], w);
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) w += __shfl_xor(w, off, WAVE);
    w -= slope2 * (float)(n - i);
    const float m_new = fmaxf(m, w);
    const float a = exp2_fast(m - m_new);
    const float p = exp2_fast(w - m_new);
    m = m_new;
    l = l * a + p;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = fmaf(p, (float)vv[j], o[j] * a);
  }
  // the wave's groups, then the block's waves
#pragma unroll
  for (int off = L; off < WAVE; off <<= 1) {
    const float m2 = __shfl_xor(m, off, WAVE);
    const float l2 = __shfl_xor(l, off, WAVE);
    const float M = fmaxf(m, m2);
    const float a = exp2_fast(m - M), a2 = exp2_fast(m2 - M);
    m = M;
    l = l * a + l2 * a2;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = o[j] * a + __shfl_xor(o[j], off, WAVE) * a2;
  }
  const int wave = tid >> 6;
  if ((tid & 63) < L) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s_o[wave][c + j] = o[j];
    if ((tid & 63) == 0) {
      s_m[wave] = m;
      s_l[wave] = l;
    }
  }
  __syncthreads();
  if (tid >= D) return;
  const long stride = (long)H * B;
  const long rh = (long)h * B + b;
  float M = -1e30f;
  for (int s = 0; s < splits; ++s)
    M = fmaxf(M, part_ml[(s * stride + rh) * 2]);
#pragma unroll
  for (int w = 0; w < OWN_BLOCK / 64; ++w) M = fmaxf(M, s_m[w]);
  float sum = 0.f, acc = 0.f;
#pragma unroll
  for (int w = 0; w < OWN_BLOCK / 64; ++w) {
    const float a = exp2_fast(s_m[w] - M);
    sum += a * s_l[w];
    acc += a * s_o[w][tid];
  }
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float a = exp2_fast(part_ml[(s * stride + rh) * 2] - M);
    sum += a * part_ml[(s * stride + rh) * 2 + 1];
    acc += a * part_o[(s * stride + rh) * D + tid];
  }
  o_row[tid] = (__bf16)(acc / sum);
}

// A workgroup takes 32 rows a wave; fewer waves where there are few rows.
int waves_for(int T) { return T <= 32 ? 1 : T <= 64 ? 2 : 4; }

// The key axis is split until the chip has workgroups to choose from, but
// not below two key tiles each.
int splits_for(long groups, int tiles) {
  const long want = (512 + groups - 1) / groups;
  return (int)std::max(1L, std::min<long>(want, tiles / 2));
}

template <bool DECODE>
void launch(const torch::Tensor& qkv, const torch::Tensor& prefix, int H,
            int D, const torch::Tensor& slopes, const torch::Tensor& info,
            __bf16* out, float* part_o, float* part_ml, int T, int P,
            int splits) {
  const __bf16* pre = (const __bf16*)prefix.data_ptr();
  const __bf16* pk = pre + (long)H * D;
  const __bf16* pv = pre + 2L * H * D;
  const int nw = waves_for(T);
  const long tiles = (T + nw * QB - 1) / (nw * QB);
  const dim3 grid(H, (unsigned)(tiles * splits));
#define LAUNCH(DD, NW)                                                       \
  hipLaunchKernelGGL((prefix_attn_kernel<DD, NW, DECODE>), grid,             \
                     dim3(64 * NW), lds_bytes(DD, NW), cur_stream(),         \
                     (const __bf16*)qkv.data_ptr(), qkv.stride(0), pk, pv,   \
                     prefix.stride(0), slopes.data_ptr<float>(),             \
                     info.data_ptr<int>(), out, part_o, part_ml, T, P, H,    \
                     splits)
  if (D == 64) {
    if (nw == 1) { LAUNCH(64, 1); } else if (nw == 2) { LAUNCH(64, 2); } else { LAUNCH(64, 4); }
  } else {
    if (nw == 1) { LAUNCH(128, 1); } else if (nw == 2) { LAUNCH(128, 2); } else { LAUNCH(128, 4); }
  }
#undef LAUNCH
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
  const int rows = waves_for(a.T) * QB;
  const long groups = (long)a.H * ((a.T + rows - 1) / rows);
  const int splits = splits_for(groups, (a.P + PKB - 1) / PKB + 1);
  TORCH_CHECK(groups / a.H * splits < 65536, "prefix attention: too many rows");
  torch::Tensor po, pm;
  if (splits > 1) {
    auto f = qkv.options().dtype(at::kFloat);
    po = torch::empty({(long)splits * a.H * a.T * a.D}, f);
    pm = torch::empty({(long)splits * a.H * a.T * 2}, f);
  }
  launch<false>(a.qkv, a.prefix, a.H, a.D, a.slopes, a.info,
                (__bf16*)out.data_ptr(),
                splits > 1 ? po.data_ptr<float>() : nullptr,
                splits > 1 ? pm.data_ptr<float>() : nullptr, a.T, a.P, splits);
  if (splits > 1) {
    const long threads = (long)a.H * a.T * a.D / 4;
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (a.D == 64)
      hipLaunchKernelGGL((prefix_join_kernel<64>), grid, dim3(256), 0,
                         cur_stream(), po.data_ptr<float>(),
                         pm.data_ptr<float>(), (__bf16*)out.data_ptr(), a.T,
                         a.H, splits);
    else
      hipLaunchKernelGGL((prefix_join_kernel<128>), grid, dim3(256), 0,
                         cur_stream(), po.data_ptr<float>(),
                         pm.data_ptr<float>(), (__bf16*)out.data_ptr(), a.T,
                         a.H, splits);
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
  int splits = 0;
  torch::Tensor po, pm;
  auto f = qkv.options().dtype(at::kFloat);
  if (a.P > 0) {
    const int rows = waves_for(a.T) * QB;
    const long groups = (long)a.H * ((a.T + rows - 1) / rows);
    splits = splits_for(groups, (a.P + PKB - 1) / PKB);
    po = torch::empty({(long)splits * a.H * B * a.D}, f);
    pm = torch::empty({(long)splits * a.H * B * 2}, f);
    launch<true>(a.qkv, a.prefix, a.H, a.D, a.slopes, a.info, nullptr,
                 po.data_ptr<float>(), pm.data_ptr<float>(), a.T, a.P, splits);
  }
  const dim3 grid(a.H, (unsigned)B);
  const float* pop = splits ? po.data_ptr<float>() : nullptr;
  const float* pmp = splits ? pm.data_ptr<float>() : nullptr;
#define LAUNCH_OWN(DD)                                                        \
  hipLaunchKernelGGL((decode_own_kernel<DD>), grid, dim3(OWN_BLOCK), 0,       \
                     cur_stream(), (const __bf16*)a.qkv.data_ptr(),           \
                     a.qkv.stride(0), (__bf16*)cache.data_ptr(),              \
                     cache.stride(0), cache.stride(1), cache.stride(2),       \
                     cache.stride(3), a.slopes.data_ptr<float>(),             \
                     a.info.data_ptr<int>(), pop, pmp,                        \
                     (__bf16*)out.data_ptr(), (int)B, a.H,                    \
                     (int)cache.size(1), splits)
  if (a.D == 64) {
    LAUNCH_OWN(64);
  } else {
    LAUNCH_OWN(128);
  }
#undef LAUNCH_OWN
  return out;
}

}  // namespace photon_hip
