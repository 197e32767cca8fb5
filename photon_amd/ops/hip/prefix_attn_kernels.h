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
// joins them. Statistics and sums are fp32; the weights are rounded to bf16 for
// the second matrix product, as the values they weigh are (2^-8 of each weight
// at most, and the result's own rounding is as large).
//
// Below 2^-150 of a row's maximum a weight is zero in fp32, and ALiBi makes most
// far keys of a steep head that: their tiles are left out after the first product
// (the scores say so) or, with many rows over a long prefix, before they are
// loaded (Cauchy and Schwarz: q . k <= |q| max |k|, see key_norms_kernel).
//
// Measured on an MI355X. Many rows (4416 over 3901 shared keys, 32 heads of
// 128): 234 us, of which 8 go to the keys' lengths and 8 to the join; 290 GFLOP
// by the formula, 174 computed. Of the SIMDs' cycles matrix instructions take
// 32% and vector instructions 38% with little overlap, LDS accesses 22% of the
// CUs'; the rest is waiting, at 1.6 waves a SIMD of 2. Few rows (93 over 1507, 16
// heads of 128): 12 us and 4 for the join, a chain of latencies. One new token
// for each of 64 sequences over 3967 keys and caches of 512, 32 heads of 128: 20
// us for the prefix (66 MB) and 60 for the caches (267 MB, 4.4 TB/s); for one
// sequence over 701 keys, 12 heads of 64, 7 us.

#pragma once

#include "attn_kernels.h"

namespace photon_hip {

// A workgroup is NW x KW waves: NW of 32 query rows each that share their key
// tiles (64 keys), or, where there are few rows, KW that take every KW-th key
// tile (32 keys) of the same rows and are joined at the end. For each, one tile
// is in LDS and the next on its way.
template <int D_, int NW_, int KW_>
struct Shape {
  static constexpr int D = D_, NW = NW_, KW = KW_;
  static constexpr int SUBS = KW == 1 ? 2 : 1;  // subtiles of 32 keys
  static constexpr int KEYS = 32 * SUBS;
  static constexpr int IMG = KEYS * D * 2;      // bytes of a [KEYS][D] image
  static constexpr int THREADS = 64 * NW * KW;
  static constexpr int ROWS = 32 * NW;
  // LDS: the images (or, at the end, the waves' fp32 rows), then each wave's
  // maxima and sums; a word a wave for the search of bad values
  static constexpr int IMAGES = KW * 2 * 2 * IMG;
  static constexpr int FP32_ROWS = NW * KW * 32 * D * 4;
  static constexpr int STATS = IMAGES > FP32_ROWS ? IMAGES : FP32_ROWS;
  static constexpr int BYTES = STATS + NW * KW * 32 * 8;
};

// Buffer descriptor of `bytes` from `base` as four words (flags: a valid
// format, see make_rsrc), and a copy of 16 bytes a lane to LDS through it.
//
// The builtin for this copy makes the compiler wait for ALL copies in flight
// before a transposing LDS read, which it takes for a possible reader of the
// tile that is still on its way: a stall of a memory latency every tile. The
// copies written here are invisible to it and waited for by vm_wait0(). They
// write no register; the wait states stand between a descriptor word that a
// vector instruction wrote and its use.
typedef __attribute__((ext_vector_type(4))) unsigned desc_t;
DEV_INLINE desc_t make_desc(const __bf16* base, long bytes) {
  const unsigned long a = (unsigned long)base;
  return desc_t{(unsigned)a, (unsigned)(a >> 32) & 0xffffu, (unsigned)bytes,
                0x27FACu};
}
DEV_INLINE unsigned lds_base(const char* smem) {
  typedef __attribute__((address_space(3))) const char* lds_cp;
  return __builtin_amdgcn_readfirstlane((unsigned)(size_t)(lds_cp)smem);
}
DEV_INLINE void copy16_to_lds(desc_t desc, unsigned lds, int offset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 4\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(offset), "s"(desc)
      : "memory", "m0");
}

// Until this wave's LDS accesses are done.
DEV_INLINE void lds_wait0() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// The larger of a row's two halves (lanes l and l + 32); NaN if one is.
DEV_INLINE float swap_max(float x) {
  union { float f; unsigned u; } a, b;
  a.f = x;
  const auto r = __builtin_amdgcn_permlane32_swap(a.u, a.u, false, false);
  a.u = r[0];
  b.u = r[1];
  return __builtin_elementwise_maximum(a.f, b.f);
}

// Eight weights (rows of the score tile) as a fragment of the next product,
// see pack_bfrag; the compiler places the conversions.
DEV_INLINE bf16x8 pack_weights(const float* p) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  union { bf16x2 v; unsigned u; } d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    d[i].v[0] = (__bf16)p[2 * i];
    d[i].v[1] = (__bf16)p[2 * i + 1];
  }
  const auto a = __builtin_amdgcn_permlane32_swap(d[0].u, d[2].u, false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(d[1].u, d[3].u, false, false);
  union { unsigned u[4]; bf16x8 v; } out;
  out.u[0] = a[0];
  out.u[1] = b[0];
  out.u[2] = a[1];
  out.u[3] = b[1];
  return out.v;
}

// The largest |k|^2 of each head and NORM_KEYS keys of the prefix, [H][tiles];
// NaN if one of them is. A workgroup reads these keys of one head, D / 8 lanes
// each. Bound by memory: 32 MB (3901 keys, 32 heads of 128) in 8 us.
constexpr int NORM_KEYS = 64;
DEV_INLINE int norm_tiles(int P) { return (P + NORM_KEYS - 1) / NORM_KEYS; }
template <int D>
__global__ __launch_bounds__(256) void key_norms_kernel(
    const __bf16* __restrict__ pk, long p_rs, float* __restrict__ norms,
    int P) {
  constexpr int L = D / 8, G = 256 / L;
  __shared__ float s_max[4];
  const int tile = blockIdx.x, h = blockIdx.y;
  const int g = threadIdx.x / L, c = threadIdx.x % L * 8;
  const __bf16* at = pk + (long)h * D + c;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < NORM_KEYS / G; ++i) {
    const int key = tile * NORM_KEYS + i * G + g;
    float sum = 0.f;
    if (key < P) {
      const bf16x8 x = *(const bf16x8*)(at + (long)key * p_rs);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf((float)x[j], (float)x[j], sum);
    }
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, WAVE);
    top = __builtin_elementwise_maximum(top, sum);  // NaN stays
  }
#pragma unroll
  for (int off = 32; off >= L; off >>= 1)
    top = __builtin_elementwise_maximum(top, __shfl_xor(top, off, WAVE));
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 4; ++w)
      top = __builtin_elementwise_maximum(top, s_max[w]);
    norms[(long)h * gridDim.x + tile] = top;
  }
}

// Which query tile and head an item is. `by_head` (many rows, a multiple of 8
// heads): workgroup i runs on XCD i % 8, so each XCD takes one of every 8 heads,
// in turn from below and from above, and its tiles one head after the other, the
// flattest first: where slopes fall with the head's number, as ALiBi's do, what
// comes last is short (294 -> 275 us at the many rows above). Otherwise tile by
// tile.
DEV_INLINE void place(int item, int H, int tiles, bool by_head, int& tile,
                      int& h) {
  if (by_head) {
    const int x = item & 7, j = item >> 3;
    const int g = H / 8 - 1 - j / tiles;
    tile = j % tiles;
    h = 8 * g + (g & 1 ? 7 - x : x);
  } else {
    tile = item / H;
    h = item % H;
  }
}

// Swapped product (keys x queries): lane holds query lane & 31, its 16
// registers the keys (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5) of 32.
//
// `info` is each row's first own row (packed form) or, in the decode form, how
// many own keys the row's sequence holds; there the kernel covers the prefix
// only.
template <typename S, bool DECODE>
__global__ __launch_bounds__(S::THREADS, S::D == 64 ? 3 : 2) void prefix_attn_kernel(
    const __bf16* __restrict__ qkv, long q_rs, const __bf16* __restrict__ pk,
    const __bf16* __restrict__ pv, long p_rs,
    const float* __restrict__ slopes, const int* __restrict__ info,
    const float* __restrict__ norms, __bf16* __restrict__ out,
    float* __restrict__ part_o, float* __restrict__ part_ml, int T, int P,
    int H, int first_split, int rest, int splits) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int D = S::D, NW = S::NW, KW = S::KW;
  constexpr int SUBS = S::SUBS, KEYS = S::KEYS, IMG = S::IMG;
  constexpr bool D64 = D == 64;
  constexpr bool STOPS = KW == 1 && !DECODE;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % NW, kw = wave / NW;  // rows, keys of this wave
  const int hi = lane >> 5;
  const int lq = lane & 31;
  // `rest` items from `first_split` on are split, the others whole
  int item = blockIdx.x, split = 0, parts = 1;
  if (item >= first_split + rest * splits) {
    item -= rest * (splits - 1);
  } else if (item >= first_split) {
    const int i = item - first_split;
    split = KW == 1 ? i / rest : i % splits;  // many rows: on its head's XCD
    item = first_split + (KW == 1 ? i % rest : i / splits);
    parts = splits;
  }
  int tile, h;
  place(item, H, (T + S::ROWS - 1) / S::ROWS, !DECODE && KW == 1 && H % 8 == 0,
        tile, h);
  const int q0_block = tile * S::ROWS;
  const int my_q = q0_block + rw * QB + lq;
  const int row = min(my_q, T - 1);

  const __bf16* q = qkv + (long)h * D;
  const __bf16* k = q + (long)H * D;
  const __bf16* v = k + (long)H * D;
  pk += (long)h * D;
  pv += (long)h * D;

  // own position of this lane's row, and the first packed row it may see
  int first = 0, own = 0;
  if (DECODE) {
    own = min(max(info[row], 0), 1 << 30);
  } else {
    first = min(max(info[row], 0), row);
    own = row - first;
  }

  // key tiles: the prefix's, then the packed rows lo .. end_row - 1
  const int n_pre = (P + KEYS - 1) / KEYS;
  int lo = 0, n_own = 0, end_row = 0;
  if (!DECODE) {
    lo = __builtin_amdgcn_readfirstlane(
        min(max(info[q0_block], 0), q0_block));
    end_row = min(q0_block + NW * QB, T);
    n_own = (end_row - lo + KEYS - 1) / KEYS;
  }
  const int n_all = n_pre + n_own;
  const int each = n_all / parts, more = n_all - each * parts;
  const int t0 = split * each + min(split, more);
  const int t1 = t0 + each + (split < more ? 1 : 0);

  // Staging: a wave-instruction moves 1 KiB to LDS, lane by lane in order;
  // the swizzle is applied to the source. The descriptor starts at the tile
  // (64-bit base), so a prefix of any length keeps 32-bit offsets, and ends
  // with its last row: what lies behind reads as zeros.
  constexpr int NWIN = IMG / 1024 / NW;
  int dma_row[NWIN], dma_col[NWIN];
#pragma unroll
  for (int i = 0; i < NWIN; ++i) {
    const int dest = (rw * NWIN + i) * 1024 + lane * 16;
    const int r = dest / (D * 2);
    dma_row[i] = r;
    dma_col[i] =
        (dest ^ (int)(swz_field((unsigned)r & 15u, D64) << 4)) % (D * 2);
  }
  char* const images = smem + kw * (2 * 2 * IMG);
  const unsigned wave_win = __builtin_amdgcn_readfirstlane(
      lds_base(smem) + kw * (2 * 2 * IMG) + rw * (NWIN * 1024));
  auto stage = [&](int t, int b) {
    const bool pre = t < n_pre;
    const long rs = pre ? p_rs : q_rs;
    const long at = pre ? (long)t * KEYS : (long)lo + (long)(t - n_pre) * KEYS;
    const int rows = min(KEYS, (pre ? P : end_row) - (int)at);
    const long bytes = ((long)(rows - 1) * rs + D) * 2;
    const desc_t krs = make_desc((pre ? pk : k) + at * rs, bytes);
    const desc_t vrs = make_desc((pre ? pv : v) + at * rs, bytes);
    const int rs2 = (int)(rs * 2);
    const unsigned dst = wave_win + b * 2 * IMG;
#pragma unroll
    for (int i = 0; i < NWIN; ++i) {
      const int off = dma_row[i] * rs2 + dma_col[i];
      copy16_to_lds(krs, dst + i * 1024, off);
      copy16_to_lds(vrs, dst + IMG + i * 1024, off);
    }
  };

  // From the nearest keys to the farthest: ALiBi makes the weights fall on
  // the way, so the first tiles set the maximum and the sums are hardly ever
  // rescaled (forwards, a steep head's maximum rises with every tile). With
  // few rows, where the whole call is one chain of latencies, the first copies
  // leave before anything else is loaded.
  const int last = t1 - 1 - kw;
  auto first_copies = [&]() {
    if (last >= t0) stage(last, 0);
  };
  if constexpr (KW > 1) first_copies();

  const float scale2 = rsqrtf((float)D) * LOG2E;
  const float slope2 = slopes[h] * LOG2E;
  bf16x8 qfrag[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    qfrag[kk] = *(const bf16x8*)(q + row * q_rs + kk * 16 + 8 * hi);

  float m_run = -1e30f;  // finite: exp2(-huge) == 0 and no NaN from inf - inf
  float l_run = 0.f;      // this half's share of the sum
  f32x16 o_acc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) o_acc[db] = f32x16{};

  // What no score with a key of the prefix exceeds: |q| times the longest key
  // (the factor is for the rounding of both). The row's score with its own key
  // is a bound from below of its maximum, also where the keys are split.
  float bound = INFINITY;
  if (STOPS && norms != nullptr) {
    float longest = 0.f, qq = 0.f, self = 0.f;
    for (int i = lane; i < norm_tiles(P); i += 64)
      longest = __builtin_elementwise_maximum(longest,
                                              norms[(long)h * norm_tiles(P) + i]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
      longest = __builtin_elementwise_maximum(
          longest, __shfl_xor(longest, off, WAVE));
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const bf16x8 own_k = *(const bf16x8*)(k + row * q_rs + kk * 16 + 8 * hi);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = (float)qfrag[kk][j];
        qq = fmaf(x, x, qq);
        self = fmaf(x, (float)own_k[j], self);
      }
    }
    qq += __shfl_xor(qq, 32, WAVE);
    self += __shfl_xor(self, 32, WAVE);
    bound = sqrtf(qq * longest) * scale2 * 1.001f;
    m_run = fmaxf(m_run, self * scale2);
  }

  // The accumulators of the scores begin at slope * sqrt(d) * (key within the
  // subtile); the rest of the bias is a constant of row and subtile that joins
  // the maximum's subtraction.
  f32x16 alibi;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    alibi[r] = slopes[h] * sqrtf((float)D) *
               (float)((r & 3) + 8 * (r >> 2) + 4 * hi);

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
  // The tile's scores. All fragments are read before the products: left to
  // itself the compiler reads each into the same registers and waits.
  auto scores = [&](int b, f32x16 (&s)[SUBS]) {
    bf16x8 a[SUBS][D / 16];
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        a[sub][kk] = *(const bf16x8*)(images + qk_addr[kk] + b * 2 * IMG +
                                      sub * 32 * (D * 2));
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      s[sub] = alibi;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        s[sub] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[sub][kk], qfrag[kk],
                                                         s[sub], 0, 0, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, SUBS * D / 16, 0);  // LDS reads
    __builtin_amdgcn_sched_group_barrier(0x008, SUBS * D / 16, 0);  // products
  };
  auto add_values = [&](const float* p, int b, int sub) {
#pragma unroll
    for (int s16 = 0; s16 < 2; ++s16) {
      const bf16x8 pf = pack_weights(p + 8 * s16);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        union { bf16x4 half[2]; bf16x8 all; } a;
#pragma unroll
        for (int rd = 0; rd < 2; ++rd)
          a.half[rd] = lds_tr16((const __bf16*)(images + IMG),
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
  int* bad_words = (int*)(smem + S::STATS);
  auto take_out_bad = [&](int b) {
    uint4* img = (uint4*)(images + b * 2 * IMG + IMG);
    constexpr int STEP = 64 * NW, EACH = IMG / 16 / STEP;
    const int me = rw * 64 + lane;
    auto bad_half = [](unsigned w, unsigned mask) { return (w & mask) == mask; };
    auto bad_word = [&](unsigned w) {
      return bad_half(w, 0x7f800000u) | bad_half(w, 0x7f80u);
    };
    uint4 w[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) w[i] = img[me + i * STEP];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      bad |= bad_word(w[i].x) | bad_word(w[i].y) | bad_word(w[i].z) |
             bad_word(w[i].w);
    bool any = __any(bad);
    if (KW == 1) {
      if (lane == 0) bad_words[wave] = any;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) any |= bad_words[w] != 0;
    }
    if (!any) return false;
    unsigned* words = (unsigned*)img;
#pragma unroll 1
    for (int i = me; i < IMG / 4; i += STEP) {
      if (bad_half(words[i], 0x7f800000u)) words[i] &= 0xffffu;
      if (bad_half(words[i], 0x7f80u)) words[i] &= 0xffff0000u;
    }
    if (KW == 1)
      __syncthreads();
    else
      lds_wait0();
    return true;
  };
  auto add_bad = [&](int kv0) {
    const int end = min(kv0 + KEYS, end_row);
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

  // All loads so far (vmcnt 0; a wait that the compiler knows of): otherwise it
  // waits for the query's inside the loop, and with them for the next tile.
  __builtin_amdgcn_s_waitcnt(0x0F70);
  if constexpr (KW == 1) first_copies();
  int b = 1;
  for (int t = last; t >= t0; t -= KW) {
    b ^= 1;
    vm_wait0();
    // tile t is there, and the reads of the one before are done
    const bool look = STOPS && norms != nullptr && (t & 3) == 0 && t < n_pre;
    int* const done = bad_words + NW;  // read long before the next is written
    if (look) {
      // ALiBi takes this much, or more, from the tiles up to t
      const float most = bound + slope2 * (float)((t + 1) * KEYS - 1 - P - own);
      const bool all = __all(most - m_run < -150.f) && slope2 >= 0.f;
      if (lane == 0) done[rw] = all;
    }
    if (KW == 1)
      __syncthreads();
    else
      lds_wait0();
    if (look) {
      bool all = true;
#pragma unroll
      for (int w = 0; w < NW; ++w) all &= done[w] != 0;
      if (all) break;  // nothing is on its way
    }
    if (t - KW >= t0) stage(t - KW, b ^ 1);
    const bool pre = t < n_pre;
    const int kv0 = pre ? t * KEYS : lo + (t - n_pre) * KEYS;
    const bool masked = !pre || (t + 1) * KEYS > P;
    const bool bad = pre ? false : take_out_bad(b);
    f32x16 s[SUBS];
    scores(b, s);
    if (masked) {
      // keys from .. from + span of this row, counted from the lane's first
      const int from = (pre ? 0 : first) - (kv0 + 4 * hi);
      const unsigned span = pre ? P - 1 : row - first;
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = sub * 32 + (r & 3) + 8 * (r >> 2);
          if ((unsigned)(key - from) > span) s[sub][r] = -INFINITY;
        }
    }
    const float c = slope2 * (float)(kv0 - (pre ? P + own : row));
    float top[SUBS];
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      top[sub] = s[sub][0];
#pragma unroll
      for (int r = 1; r < 16; ++r)
        top[sub] = __builtin_elementwise_maximum(top[sub], s[sub][r]);
      top[sub] = fmaf(top[sub], scale2, c + (float)(32 * sub) * slope2);
    }
    const float highest = swap_max(
        __builtin_elementwise_maximum(top[0], top[SUBS - 1]));
    // Below 2^-150 of the maximum a weight is zero in fp32: a tile of such
    // weights (far keys of a steep head, other sequences' rows) adds nothing.
    // A NaN among the scores makes the comparison false; one among a prefix
    // tile's values is not looked for under weights that are all zero.
    if (!bad && __all(highest - m_run < -150.f)) continue;
    raise(highest);
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      const float shift = c + (float)(32 * sub) * slope2 - m_run;
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = exp2_fast(fmaf(s[sub][r], scale2, shift));
        l_run += p[r];
      }
      add_values(p, b, sub);
    }
    if (bad) add_bad(kv0);
  }
  l_run += __shfl_xor(l_run, 32, 64);
  __syncthreads();  // the images are free

  // Through LDS to whole rows.
  // partial rows: [split][item - first_split][row of the item]
  const long base = ((long)split * rest + item - first_split) * S::ROWS;
  const bool whole = parts == 1 && !DECODE;
  if (KW == 1 && whole) {
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
      const int r = q0_block + rw * QB + c / (D / 8);
      const int col = (c % (D / 8)) * 8;
      if (r < T)
        *(bf16x8*)(out + (long)r * H * D + (long)h * D + col) =
            *(const bf16x8*)(o_img + c * 8);
    }
    return;
  }
  float* o_img = (float*)smem + wave * 32 * D;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *(f32x4*)(o_img + lq * D + db * 32 + 2 * r + 4 * hi) =
          f32x4{o_acc[db][r], o_acc[db][r + 1], o_acc[db][r + 2],
                o_acc[db][r + 3]};
  if (KW == 1) {
    __syncthreads();
    for (int c = lane; c < 32 * D / 4; c += 64)
      *(f32x4*)(part_o + (base + rw * QB) * D + c * 4) =
          *(const f32x4*)(o_img + c * 4);
    if (hi == 0) {
      part_ml[(base + rw * QB + lq) * 2] = m_run;
      part_ml[(base + rw * QB + lq) * 2 + 1] = l_run;
    }
  } else {
    float* stats = (float*)(smem + S::STATS);  // [wave][row]: maximum, sum
    if (hi == 0) {
      stats[(wave * 32 + lq) * 2] = m_run;
      stats[(wave * 32 + lq) * 2 + 1] = l_run;
    }
    __syncthreads();
    // a row's key waves: EACH threads a row, four columns at a time
    constexpr int EACH = S::THREADS / 32;
    const int r = threadIdx.x / EACH;
    float M = -1e30f, l = 0.f, a[KW];
#pragma unroll
    for (int w = 0; w < KW; ++w) M = fmaxf(M, stats[(w * 32 + r) * 2]);
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      a[w] = exp2_fast(stats[(w * 32 + r) * 2] - M);
      l += a[w] * stats[(w * 32 + r) * 2 + 1];
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int q_row = q0_block + r;
    for (int c = (threadIdx.x % EACH) * 4; c < D; c += EACH * 4) {
      f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const f32x4 x = *(const f32x4*)((float*)smem + (w * 32 + r) * D + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += a[w] * x[j];
      }
      if (whole) {
        bf16x4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = (__bf16)(o[j] * inv);
        if (q_row < T)
          *(bf16x4*)(out + (long)q_row * H * D + (long)h * D + c) = y;
      } else {
        *(f32x4*)(part_o + (base + r) * D + c) = o;
      }
    }
    if (!whole && threadIdx.x % EACH == 0) {
      part_ml[(base + r) * 2] = M;
      part_ml[(base + r) * 2 + 1] = l;
    }
  }
}

// Joins the splits: a thread has four columns of a row.
// An item is `rows` rows of one head; `rest` items were split.
template <int D>
__global__ __launch_bounds__(256) void prefix_join_kernel(
    const float* __restrict__ part_o, const float* __restrict__ part_ml,
    __bf16* __restrict__ out, int T, int H, int rows, int first_split, int rest,
    int splits, bool by_head) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long pr = i / (D / 4);  // partial row: [item - first_split][row]
  const int col = (int)(i % (D / 4)) * 4;
  if (pr >= (long)rest * rows) return;
  const int item = first_split + (int)(pr / rows);
  int tile, h;
  place(item, H, (T + rows - 1) / rows, by_head, tile, h);
  const long t = (long)tile * rows + pr % rows;
  if (t >= T) return;
  const long stride = (long)rest * rows;
  float M = -1e30f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s)
    M = fmaxf(M, part_ml[(s * stride + pr) * 2]);
  float l = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const float w = exp2_fast(part_ml[(s * stride + pr) * 2] - M);
    l += w * part_ml[(s * stride + pr) * 2 + 1];
    const f32x4 x = *(const f32x4*)(part_o + (s * stride + pr) * D + col);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += w * x[j];
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  bf16x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = (__bf16)(o[j] * inv);
  *(bf16x4*)(out + (t * H + h) * D + col) = r;
}

// Decode: one workgroup per (sequence, head) writes the new key and value to
// the cache, attends the sequence's own keys and joins what the prefix gave.
// D / 8 lanes hold a key's 8 columns each, all groups of the block stride
// over the keys with a running maximum and sum of their own.
// Where there are few workgroups each is a large one, and may attend `direct`
// keys of the prefix as well (all of them; no partial rows then).
constexpr int OWN_BLOCK = 256;
constexpr int LARGE_BLOCK = 1024;
template <int D, int BLOCK>
__global__ __launch_bounds__(BLOCK) void decode_own_kernel(
    const __bf16* __restrict__ qkv, long q_rs, __bf16* __restrict__ cache,
    long c_bs, long c_ss, long c_ks, long c_hs,
    const float* __restrict__ slopes, const int* __restrict__ held,
    const __bf16* __restrict__ pk, const __bf16* __restrict__ pv, long p_rs,
    int direct, const float* __restrict__ part_o,
    const float* __restrict__ part_ml, __bf16* __restrict__ out, int H,
    int slots, int rows, int items, int splits) {
  constexpr int L = D / 8;               // lanes a key
  constexpr int G = BLOCK / L;           // keys at a time
  __shared__ float s_o[BLOCK / 64][D];
  __shared__ float s_m[BLOCK / 64], s_l[BLOCK / 64];
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
  // The first of the prefix's partial rows are asked for before the sequence's
  // own keys: their way from memory is not on the chain behind them.
  constexpr int EARLY = 8;
  const long stride = (long)items * rows;
  const long pr = ((long)(b / rows) * H + h) * rows + b % rows;
  float pm[EARLY], pl[EARLY], po[EARLY];
#pragma unroll
  for (int s = 0; s < EARLY; ++s) {
    pm[s] = -1e30f;
    pl[s] = po[s] = 0.f;
    if (s < splits && tid < D) {
      pm[s] = part_ml[(s * stride + pr) * 2];
      pl[s] = part_ml[(s * stride + pr) * 2 + 1];
      po[s] = part_o[(s * stride + pr) * D + tid];
    }
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
  // U keys at a time, all their loads in flight together and one rescaling
  constexpr int U = 4;
  // keys 0 .. count - 1, which lie `stored` rows of stride `rs` behind k0 and
  // v0; the rest (the new one) come from registers. Key i is gap - i away.
  auto attend = [&](int count, int stored, const __bf16* k0, const __bf16* v0,
                    long rs, int gap) {
    for (int i0 = g; i0 < count; i0 += U * G) {
      bf16x8 kv[U], vv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * G;
        kv[u] = new_k;
        vv[u] = new_v;
        if (i < stored) {
          kv[u] = *(const bf16x8*)(k0 + (long)i * rs + c);
          vv[u] = *(const bf16x8*)(v0 + (long)i * rs + c);
        }
      }
      float w[U];
      float m_new = m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) x = fmaf(qf[j], (float)kv[u][j], x);
#pragma unroll
        for (int off = L / 2; off > 0; off >>= 1) x += __shfl_xor(x, off, WAVE);
        const int i = i0 + u * G;
        w[u] = i < count ? x - slope2 * (float)(gap - i) : -INFINITY;
        m_new = fmaxf(m_new, w[u]);
      }
      const float a = exp2_fast(m - m_new);
      m = m_new;
      l *= a;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= a;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + u * G < count) {  // a value behind the last is not touched
          const float p = exp2_fast(w[u] - m);
          l += p;
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = fmaf(p, (float)vv[u][j], o[j]);
        }
      }
    }
  };
  if (direct > 0)
    attend(direct, direct, pk + (long)h * D, pv + (long)h * D, p_rs, direct + n);
  attend(n + 1, n, ck, cv, c_ss, n);
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
  float M = -1e30f;
#pragma unroll
  for (int s = 0; s < EARLY; ++s) M = fmaxf(M, pm[s]);
#pragma unroll 8
  for (int s = EARLY; s < splits; ++s)
    M = fmaxf(M, part_ml[(s * stride + pr) * 2]);
#pragma unroll
  for (int w = 0; w < BLOCK / 64; ++w) M = fmaxf(M, s_m[w]);
  float sum = 0.f, acc = 0.f;
#pragma unroll
  for (int w = 0; w < BLOCK / 64; ++w) {
    const float a = exp2_fast(s_m[w] - M);
    sum += a * s_l[w];
    acc += a * s_o[w][tid];
  }
#pragma unroll
  for (int s = 0; s < EARLY; ++s) {
    const float a = exp2_fast(pm[s] - M);
    sum += a * pl[s];
    acc += a * po[s];
  }
#pragma unroll 8
  for (int s = EARLY; s < splits; ++s) {
    const float a = exp2_fast(part_ml[(s * stride + pr) * 2] - M);
    sum += a * part_ml[(s * stride + pr) * 2 + 1];
    acc += a * part_o[(s * stride + pr) * D + tid];
  }
  o_row[tid] = (__bf16)(acc / sum);
}

}  // namespace photon_hip
