// Attention of query rows over key rows with shared key heads and ragged lengths, forward and backward.
//
//   s = scale q k^T (key j takes part if j < k_len[b], query t if t < q_len[b])     p = softmax(s)     o = p v
//   delta = sum_d go o      gv = p^T go      ds = p (go v^T - delta)      gq = scale ds k      gk = scale ds^T q
//
// One pass over the keys with the running maximum and sum of the softmax; nothing of size Tq x Tk is ever stored. The
// backward pass rebuilds p = exp(s - lse) from the row's log-sum.
//
// Rows. The G = Hq / Hk query heads of a key head and its Tq queries are the R = Tq G rows of one problem (b, hk), row
// r = t G + g: keys and values are read once for the whole group, the gradients of a shared head are sums over rows of
// the same problem (no atomics, a fixed order), and a single query still fills G rows of a tile.
//
// Layout of the products. Every product is taken transposed or not so that its result feeds the next one from the
// registers it lies in. A 32 x 32 product leaves lane (c, h) = (lane % 32, lane / 32) with column c and the 16 rows
// 8 (i / 4) + 4 h + i % 4. The forward pass takes S^T = K Q^T (column = query), so a lane owns 16 keys of one query: the
// softmax needs one exchange between lanes c and c + 32, and the probabilities are the B operand of O^T = V^T P^T as
// they are, if the keys of a k-slice are numbered in the order in which the lane holds them - which only says which
// rows of V the A operand reads. bf16 reads them with the transposing LDS load (4 keys of one column per lane), f32 with
// 4-byte loads. Queries' gradients use the same shape; the gradients of keys and values its mirror image (column = key).
//
// Bound by the SIMDs: the vector instructions of the softmax (one exponential, two to four others an element) add to the
// matrix instructions instead of hiding under them, so heads of 128 come nearer the matrix rate than heads of 64. Measured
// in loops of calls, bf16: 8192 queries and keys, 2 x 16 query and 4 key heads of 128 ("the long case" below) forward 1.15 ms
// (0.96 PFLOP/s; a library product of 8192^3 reaches 1.28), backward 3.51 ms (0.78 on its five products, 1.10 with the two
// that both walks rebuild); 1024 queries and keys, 8 x 16 heads of 64 51 and 145 us (0.67 and 0.59 PFLOP/s).
#include <float.h>
#include <math.h>

#include "token_common.h"

namespace {

constexpr int kWaves = 4;
constexpr int kTileRows = 32 * kWaves;     // rows (forward, queries' gradient) or keys (keys' gradient) of a block

struct AttnParams {
  vg_attention_geom g;
  const void *q, *k, *v, *o, *go;
  void *out, *gq, *gk, *gv;
  __bf16* low;               // bf16: what the rounding of o left, dense (written forward, read for delta); null: not wanted
  const float *lse_in, *delta;
  float* lse;
  const int *q_len, *k_len;
  float* part;               // split walks over keys: f32 partial rows
  float* part_ml;            // forward: running maximum and sum of every row and split
  float* part_kv;            // split walks over rows: f32 partial gradients of keys, then of values
  int G, R;
  int splits, chunk;         // walks over keys (forward, queries' gradient): how many, keys of each
  int r_splits, r_chunk;     // walks over rows (keys' gradient)
  int gkv_blocks;            // backward: blocks of the keys' gradient, ahead of those of the queries'
  unsigned g_magic;          // ceil(2^32 / G)
  int row_tiles, key_tiles;
  float cs;                  // scale * log2(e)
};

__device__ __forceinline__ int row_query(const AttnParams& p, int r) { return p.G == 1 ? r : (int)__umulhi((unsigned)r, p.g_magic); }

template <class T>
__device__ __forceinline__ const T* row_at(const void* base, const vg_heads_layout& l, const AttnParams& p, int b, int hk, int r) {
  const int t = row_query(p, r), g = r - t * p.G;
  return (const T*)base + b * l.sb + t * l.st + (int64_t)(hk * p.G + g) * l.sh;
}

__device__ __forceinline__ int clamped(const int* len, int b, int most) {
  if (!len) return most;
  const int n = len[b];
  return n < 0 ? 0 : n > most ? most : n;
}

// ---- fragments ------------------------------------------------------------------------------------------------------
// An LDS tile of rows of DP elements. A fragment of rows is read 16 bytes a lane, rows 0..15 side by side: padded by 16
// bytes, they start on different banks. The transposing load (TR tiles, bf16) reads 64 bytes of four rows side by
// side: its rows are 16 banks apart (mod 64), and to keep the first kind of read apart as well the four 16-byte pieces of
// every 64 bytes change places by bits 2-3 of the row. (Padded by 16 bytes alone, half the LDS cycles of these
// kernels were bank conflicts of the transposing loads, ten cycles each instead of four.) f32 columns are read 4 bytes
// a lane, side by side.
template <class T, int DP, bool TR>
struct Tile {
  static constexpr int V = TokNum<T>::V;
  static constexpr bool SWAP = TR && sizeof(T) == 2;
  static constexpr int LD = SWAP ? (DP == 32 ? 32 : DP + 32) : DP + V;
  // element index of a 16-byte piece that starts at column d
  static __device__ __forceinline__ int at(int row, int d) { return row * LD + (SWAP ? d ^ (((row >> 2) & 3) * 8) : d); }
};

// Registers of a 32-row operand whose contraction index is d: bf16 holds 8 d of each 16 (8 h ..), f32 4 of each 8.
template <class T, int DP>
struct RowFrag;
template <int DP>
struct RowFrag<__bf16, DP> {
  bf16x8 f[DP / 16];
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) f[s] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, f[s]) ^ 0x80008000u);
  }
  __device__ __forceinline__ void load(const __bf16* row, int D, int h, bool ok) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * h;
      const u32x4 raw = ok && d < D ? *reinterpret_cast<const u32x4*>(row + d) : u32x4{0, 0, 0, 0};
      f[s] = __builtin_bit_cast(bf16x8, raw);
    }
  }
};
template <int DP>
struct RowFrag<float, DP> {
  f32x4 f[DP / 8];
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int s = 0; s < DP / 8; ++s) f[s] = -f[s];
  }
  __device__ __forceinline__ void load(const float* row, int D, int h, bool ok) {
#pragma unroll
    for (int s = 0; s < DP / 8; ++s) {
      const int d = 8 * s + 4 * h;
      f[s] = ok && d < D ? *reinterpret_cast<const f32x4*>(row + d) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
};

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// C[row of the LDS tile][column] = acc + sum_d tile[row0 + row][d] * frag(column)[d]
template <int DP, bool TR>
__device__ __forceinline__ f32x16 mul_rows(const __bf16* tile, const RowFrag<__bf16, DP>& b, int row0, int c, int h, f32x16 acc = zero16()) {
  const __bf16 *even = tile + Tile<__bf16, DP, TR>::at(row0 + c, 8 * h), *odd = tile + Tile<__bf16, DP, TR>::at(row0 + c, 16 + 8 * h);
#pragma unroll
  for (int s = 0; s < DP / 16; ++s)
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>((s % 2 ? odd : even) + s / 2 * 32), b.f[s], acc, 0, 0, 0);
  return acc;
}
template <int DP, bool TR>
__device__ __forceinline__ f32x16 mul_rows(const float* tile, const RowFrag<float, DP>& b, int row0, int c, int h, f32x16 acc = zero16()) {
  const float* a = tile + Tile<float, DP, TR>::at(row0 + c, 4 * h);
#pragma unroll
  for (int s = 0; s < DP / 8; ++s) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(a + 8 * s);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], b.f[s][e], acc, 0, 0, 0);
  }
  return acc;
}
// the same with both operands in LDS (rows of a plain tile as columns)
template <int DP, bool TR>
__device__ __forceinline__ f32x16 mul_tiles(const __bf16* tile, const __bf16* cols, int row0, int col0, int c, int h, f32x16 acc) {
  const __bf16 *even = tile + Tile<__bf16, DP, TR>::at(row0 + c, 8 * h), *odd = tile + Tile<__bf16, DP, TR>::at(row0 + c, 16 + 8 * h);
  const __bf16* b = cols + Tile<__bf16, DP, false>::at(col0 + c, 8 * h);
#pragma unroll
  for (int s = 0; s < DP / 16; ++s)
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>((s % 2 ? odd : even) + s / 2 * 32),
                                                  *reinterpret_cast<const bf16x8*>(b + 16 * s), acc, 0, 0, 0);
  return acc;
}

// acc[j] (rows d = 32 j + row) += sum over the 32 rows k0.. of a TR tile of tile[k][d] * w[k][column], w as a product left it.
// bf16: w (probabilities, ds) is rounded to bf16 for this; FINE: taken as two bf16 terms, i.e. to 2^-17. `total` (not with
// FINE): every element += the sum over the 32 rows of the rounded w[column].
template <int DP, bool FINE>
__device__ __forceinline__ void mul_cols(const __bf16* tile, const f32x16& w, int k0, int lane, f32x16 (&acc)[DP / 32], f32x16* total = nullptr) {
  using L = Tile<__bf16, DP, true>;
  const int h = lane >> 5, q = (lane & 15) >> 2, col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  // rows k0 + 16 s + 4 h + q and 8 further: bits 2-3 of the row are h and 2 + h
  const __bf16 *a = tile + (k0 + 4 * h + q) * L::LD + (col ^ (8 * h)), *b = tile + (k0 + 8 + 4 * h + q) * L::LD + (col ^ (8 * (2 + h)));
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float left[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) left[i] = w[8 * s + i];
    const bf16x8 x = __builtin_bit_cast(bf16x8, tok_narrow(left));
    [[maybe_unused]] bf16x8 x2;
    if constexpr (FINE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) left[i] -= (float)x[i];
      x2 = __builtin_bit_cast(bf16x8, tok_narrow(left));
    } else if (total) {
      const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
      *total = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ones, x, *total, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) {
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 16 * s * L::LD + 32 * j));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(b + 16 * s * L::LD + 32 * j));
      const s16x8 y = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if constexpr (FINE) acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, y), x2, acc[j], 0, 0, 0);
      acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, y), x, acc[j], 0, 0, 0);
    }
  }
}
template <int DP, bool>
__device__ __forceinline__ void mul_cols(const float* tile, const f32x16& w, int k0, int lane, f32x16 (&acc)[DP / 32], f32x16* = nullptr) {
  constexpr int LD = Tile<float, DP, true>::LD;
  const int h = lane >> 5, c = lane & 31;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float* a = tile + (k0 + 8 * (i / 4) + 4 * h + i % 4) * LD + c;
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[32 * j], w[i], acc[j], 0, 0, 0);
  }
}

// Stages ROWS rows of up to DP elements in registers on their way to an LDS tile; what is out of range becomes zero.
// A thread's byte offsets from the tile's first row are the same in every tile, so a tile costs one scalar addition to
// the base and the range-checked loads themselves (vector instructions do not overlap the matrix instructions of a
// SIMD: the address arithmetic of pointers, five instructions a vector, took a fifth of the forward kernel).
constexpr int kOutside = 0x7fffffff, kRange = 0x7ffffff0;
template <class T, int DP, int ROWS, bool TR>
struct Stage {
  static constexpr int V = TokNum<T>::V, VPR = DP / V, N = ROWS * VPR / (64 * kWaves);
  static_assert(ROWS * VPR % (64 * kWaves) == 0, "whole vectors per thread");
  u32x4 r[N];
  int off[N];
  template <class At>
  __device__ __forceinline__ void place(int D, At at) {     // at(row) -> its byte offset from the tile's first row
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = threadIdx.x + i * 64 * kWaves, row = id / VPR, d = (id % VPR) * V;
      off[i] = d < D ? at(row) + d * (int)sizeof(T) : kOutside;
    }
  }
  __device__ __forceinline__ void load(const T* base, int rows) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, kRange, 0x00020000);
    if (rows >= ROWS) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off[i], 0, 0));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = (threadIdx.x + i * 64 * kWaves) / VPR;
        r[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, row < rows ? off[i] : kOutside, 0, 0));
      }
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = threadIdx.x + i * 64 * kWaves, row = id / VPR, d = (id % VPR) * V;
      *reinterpret_cast<u32x4*>(tile + Tile<T, DP, TR>::at(row, d)) = r[i];
    }
  }
};

// keys (rows) of a staged tile: two buffers of two tiles fit the 160 KB of a CU
template <class T, int DP>
constexpr int tile_len() {
  return sizeof(T) == 2 ? 64 : DP >= 128 ? 32 : 64;
}

// What rounding four values to bf16 leaves of them, rounded itself (2^-17 of the value). delta = go o is a small difference's
// worth in ds = p (go v^T - delta) where a row has few keys: taken from the rounded o alone it would carry more error than
// all other roundings together.
__device__ __forceinline__ float left_over(float x) { return x - (float)(__bf16)x; }
__device__ __forceinline__ void store_low(__bf16* p, float a, float b, float c, float d) {
  tok_store4(p, left_over(a), left_over(b), left_over(c), left_over(d));
}
__device__ __forceinline__ size_t low_at(const AttnParams& p, int b, int hk, int r) {
  const int t = row_query(p, r), h = hk * p.G + r - t * p.G;
  return (((size_t)b * p.g.Tq + t) * p.g.Hq + h) * p.g.D;
}

template <class T>
__device__ __forceinline__ void store_cols(T* row, const f32x16& a, int j, int h, int D, float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = 32 * j + 8 * i + 4 * h;
    if (d < D) tok_store4(row + d, a[4 * i] * f, a[4 * i + 1] * f, a[4 * i + 2] * f, a[4 * i + 3] * f);
  }
}

// ---- forward --------------------------------------------------------------------------------------------------------
// Grid: (row tile, split, problem), the row tiles of a problem on one XCD. SPLIT: every split leaves its unnormalised
// rows, maximum and sum for the joining kernel.
template <class T, int DP, bool SPLIT, bool FINE>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) attn_fwd_kernel(const AttnParams p) {
  constexpr int KT = tile_len<T, DP>();
  __shared__ __attribute__((aligned(16))) T ktile[2][KT * Tile<T, DP, false>::LD];
  __shared__ __attribute__((aligned(16))) T vtile[2][KT * Tile<T, DP, true>::LD];
  const vg_attention_geom& g = p.g;
  const int id = tok_xcd_order(blockIdx.x, gridDim.x);
  const int rt = id % p.row_tiles, sp = (id / p.row_tiles) % p.splits, prob = id / (p.row_tiles * p.splits);
  const int b = prob / g.Hk, hk = prob - b * g.Hk;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int rows = clamped(p.q_len, b, g.Tq) * p.G;
  const int kl = clamped(p.k_len, b, g.Tk);
  const int r = rt * kTileRows + wid * 32 + c;
  const int kbeg = sp * p.chunk, kend = rt * kTileRows < rows ? min(kl, kbeg + p.chunk) : 0;

  RowFrag<T, DP> qf;
  qf.load(row_at<T>(p.q, g.q, p, b, hk, r < rows ? r : 0), g.D, h, r < rows);
  if (p.cs < 0.f) qf.negate();             // the largest score is then the largest product
  const float cs = fabsf(p.cs);
  const T* kb = (const T*)p.k + b * g.k.sb + hk * g.k.sh;
  const T* vb = (const T*)p.v + b * g.v.sb + hk * g.v.sh;
  Stage<T, DP, KT, false> sk;
  Stage<T, DP, KT, true> sv;
  sk.place(g.D, [&](int row) { return row * (int)(g.k.st * sizeof(T)); });
  sv.place(g.D, [&](int row) { return row * (int)(g.v.st * sizeof(T)); });
  auto fetch = [&](int j) {
    sk.load(kb + j * g.k.st, kend - j);
    sv.load(vb + j * g.v.st, kend - j);
  };
  f32x16 o[DP / 32];
#pragma unroll
  for (int j = 0; j < DP / 32; ++j) o[j] = zero16();
  float m = -FLT_MAX, l = 0.f;       // finite: a row whose scores are all -inf sums to zero, not to NaN
  // Probabilities of one bf16 term are divided by the sum of what they were rounded to, not of what they were: their roundings
  // then only move o among the values, and nothing of the values' common part reaches delta = go o, in which it would be
  // many times the scores' gradients (values, keys and output gradients of mean 3 and deviation 1: queries' gradient off by
  // 9 to 11 % so, 0.7 % here). The matrix cores form that sum (any element of `total`, over both lane halves) in little more
  // time than the additions would take: the long case 1.12 -> 1.15 ms, the other 49.5 -> 51.2 us.
  constexpr bool kRounded = sizeof(T) == 2 && !FINE;
  f32x16 total = zero16();
  // Split walks have few rows: a wave without any only loads (16 problems of 8 rows on 16384 keys of 64, bf16: 16.5 -> 13.6 us
  // where calls repeat on keys and values that stay in the last-level cache in part; 16.4, 4.1 TB/s, where they change). f32:
  // 45.8 us either way, 2.9 TB/s; the one wave with rows takes 8192 cycles of f32 products for 64 keys of 64, most of them
  // for empty rows of the 32.
  const bool idle = SPLIT && rt * kTileRows + __builtin_amdgcn_readfirstlane(wid) * 32 >= rows;
  int buf = 0;
  if (kbeg < kend) {
    fetch(kbeg);
    sk.store(ktile[0]);
    sv.store(vtile[0]);
  }
  __syncthreads();
  for (int j = kbeg; j < kend; j += KT) {
    const bool more = j + KT < kend;
    if (idle) {
      if (more) fetch(j + KT);
    } else {
      f32x16 s[KT / 32];
#pragma unroll
      for (int kk = 0; kk < KT / 32; ++kk) s[kk] = mul_rows<DP, false>(ktile[buf], qf, 32 * kk, c, h);
      if (more) fetch(j + KT);          // (behind the products: at the top of the loop 3 to 6 % slower)
      if (j + KT > kend) {
#pragma unroll
        for (int kk = 0; kk < KT / 32; ++kk)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (j + 32 * kk + 8 * (i / 4) + 4 * h + i % 4 >= kend) s[kk][i] = -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int kk = 0; kk < KT / 32; ++kk)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kk][i]);
      top = fmaxf(top, __shfl_xor(top, 32, 64)) * cs;
      // the rows' scale follows a maximum that grows by more than 2^8 only: that seldom happens after the first tile, and up to
      // 2^8 the f32 sums and the relative roundings of the probabilities lose nothing
      if (__any(top > m + 8.f)) {
        top = fmaxf(top, m);
        const float alpha = __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= alpha;
        total[0] *= alpha;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
      }
#pragma unroll
      for (int kk = 0; kk < KT / 32; ++kk)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[kk][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk][i], cs, -m));
          if (!kRounded) l += s[kk][i];
        }
#pragma unroll
      for (int kk = 0; kk < KT / 32; ++kk) mul_cols<DP, FINE>(vtile[buf], s[kk], 32 * kk, lane, o, kRounded ? &total : nullptr);
    }
    if (more) {
      sk.store(ktile[buf ^ 1]);
      sv.store(vtile[buf ^ 1]);
    }
    __syncthreads();
    buf ^= 1;
  }
  l = kRounded ? total[0] : l + __shfl_xor(l, 32, 64);
  if (r >= rows) l = 0.f;       // (took part as a row of zeros)
  if (r >= p.R) return;
  if constexpr (SPLIT) {
    const size_t at = ((size_t)prob * p.splits + sp) * p.R + r;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) store_cols(p.part + at * DP, r < rows ? o[d] : zero16(), d, h, DP, 1.f);
    if (h == 0) {
      p.part_ml[2 * at] = m;
      p.part_ml[2 * at + 1] = l;
    }
  } else {
    const float f = l > 0.f || l != l ? 1.f / l : 0.f;
    T* out = const_cast<T*>(row_at<T>(p.out, g.o, p, b, hk, r));
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) store_cols(out, r < rows ? o[d] : zero16(), d, h, g.D, f);
    if constexpr (sizeof(T) == 2) {
      if (p.low && r < rows) {           // (other rows' are not read)
        __bf16* low = p.low + low_at(p, b, hk, r);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            if (32 * d + 2 * i + 4 * h < g.D)
              store_low(low + 32 * d + 2 * i + 4 * h, o[d][i] * f, o[d][i + 1] * f, o[d][i + 2] * f, o[d][i + 3] * f);
      }
    }
    // a row without keys: +inf, so that the backward pass finds p = exp(s - inf) = 0
    if (h == 0 && p.lse) p.lse[(size_t)prob * p.R + r] = f != 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY;
  }
}

// Joins the splits of a row: DP / 4 lanes of 4 elements side by side, the row's splits dealt to `per_row` such groups of lanes.
template <class T, int DP>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnParams p, int per_row) {
  constexpr int LPR = DP / 4, GROUPS = 256 / LPR;
  __shared__ float red[GROUPS][DP + 4];
  __shared__ float tops[GROUPS], sums[GROUPS];
  const vg_attention_geom& g = p.g;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, share = group % per_row;
  const long long row = (long long)blockIdx.x * (GROUPS / per_row) + group / per_row;
  const bool in = row < (long long)g.B * g.Hk * p.R;
  const int prob = (int)(row / p.R), r = (int)(row - (long long)prob * p.R);
  const int b = prob / g.Hk, hk = prob - b * g.Hk;
  const size_t first = (size_t)prob * p.splits * p.R + r;
  float m = -FLT_MAX, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = in ? share : p.splits; s < p.splits; s += per_row) {
    const size_t at = first + (size_t)s * p.R;
    const float ms = p.part_ml[2 * at], ls = p.part_ml[2 * at + 1];
    const f32x4 x = *reinterpret_cast<const f32x4*>(p.part + at * DP + 4 * lane);
    const float top = fmaxf(m, ms), a = __builtin_amdgcn_exp2f(m - top), f = __builtin_amdgcn_exp2f(ms - top);
    m = top;
    l = l * a + f * ls;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * a + f * x[e];
  }
  *reinterpret_cast<f32x4*>(&red[group][4 * lane]) = o;
  if (lane == 0) {
    tops[group] = m;
    sums[group] = l;
  }
  __syncthreads();
  if (share || !in) return;
  for (int s = group + 1; s < group + per_row; ++s) {
    const float ms = tops[s], top = fmaxf(m, ms), a = __builtin_amdgcn_exp2f(m - top), f = __builtin_amdgcn_exp2f(ms - top);
    m = top;
    l = l * a + f * sums[s];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * a + f * red[s][4 * lane + e];
  }
  const float f = l > 0.f || l != l ? 1.f / l : 0.f;
  const int d = 4 * lane;
  if (d < g.D) tok_store4(const_cast<T*>(row_at<T>(p.out, g.o, p, b, hk, r)) + d, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
  if (sizeof(T) == 2 && p.low && d < g.D) store_low(p.low + low_at(p, b, hk, r) + d, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
  if (d == 0 && p.lse) p.lse[row] = f != 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY;
}

// ---- backward -------------------------------------------------------------------------------------------------------
// delta[row] = sum_d go o: eight lanes a row
template <class T>
__global__ void __launch_bounds__(256) attn_delta_kernel(const AttnParams p, float* delta) {
  constexpr int V = TokNum<T>::V;
  const vg_attention_geom& g = p.g;
  const long long row = (long long)blockIdx.x * 32 + threadIdx.x / 8;
  float sum = 0.f;
  if (row < (long long)g.B * g.Hk * p.R) {
    const int prob = (int)(row / p.R), r = (int)(row - (long long)prob * p.R);
    const int b = prob / g.Hk, hk = prob - b * g.Hk;
    if (r < clamped(p.q_len, b, g.Tq) * p.G) {
      const T* go = row_at<T>(p.go, g.go, p, b, hk, r);
      const T* o = row_at<T>(p.o, g.o, p, b, hk, r);
      for (int d = (threadIdx.x % 8) * V; d < g.D; d += 8 * V) {
        float x[V], y[V];
        tok_widen(*reinterpret_cast<const u32x4*>(go + d), x);
        tok_widen(*reinterpret_cast<const u32x4*>(o + d), y);
        if constexpr (sizeof(T) == 2) {
          if (p.low) {
            float z[V];
            tok_widen(*reinterpret_cast<const u32x4*>(p.low + low_at(p, b, hk, r) + d), z);
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] += z[e];
          }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) sum = __builtin_fmaf(x[e], y[e], sum);
      }
    }
  }
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (threadIdx.x % 8 == 0 && row < (long long)g.B * g.Hk * p.R) delta[row] = sum;
}

// Queries' gradient: the forward kernel's walk with p rebuilt from lse. Heads of 128 take their keys 32 at a time (fewer
// staging registers: at 64 the kernel spills).
template <class T, int DP>
struct GqTiles {
  static constexpr int KT = DP >= 128 ? 32 : tile_len<T, DP>();
  T k[2][KT * Tile<T, DP, true>::LD];
  T v[2][KT * Tile<T, DP, false>::LD];
};
template <class T, int DP, bool FINE>
__device__ __forceinline__ void queries_gradient(const AttnParams& p, int id, GqTiles<T, DP>& tiles) {
  constexpr int KT = GqTiles<T, DP>::KT;
  auto& ktile = tiles.k;
  auto& vtile = tiles.v;
  const vg_attention_geom& g = p.g;
  const int rt = id % p.row_tiles, sp = (id / p.row_tiles) % p.splits, prob = id / (p.row_tiles * p.splits);
  const int b = prob / g.Hk, hk = prob - b * g.Hk;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int rows = clamped(p.q_len, b, g.Tq) * p.G;
  const int kl = clamped(p.k_len, b, g.Tk);
  const int r = rt * kTileRows + wid * 32 + c;
  const int kbeg = sp * p.chunk, kend = rt * kTileRows < rows ? min(kl, kbeg + p.chunk) : 0;

  RowFrag<T, DP> qf, gf;
  qf.load(row_at<T>(p.q, g.q, p, b, hk, r < rows ? r : 0), g.D, h, r < rows);
  gf.load(row_at<T>(p.go, g.go, p, b, hk, r < rows ? r : 0), g.D, h, r < rows);
  const float lse = r < rows ? p.lse_in[(size_t)prob * p.R + r] : INFINITY;
  f32x16 less;               // -delta: what the product go v^T starts from
  {
    const float delta = r < rows ? p.delta[(size_t)prob * p.R + r] : 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) less[i] = -delta;
  }
  const T* kb = (const T*)p.k + b * g.k.sb + hk * g.k.sh;
  const T* vb = (const T*)p.v + b * g.v.sb + hk * g.v.sh;
  Stage<T, DP, KT, true> sk;
  Stage<T, DP, KT, false> sv;
  sk.place(g.D, [&](int row) { return row * (int)(g.k.st * sizeof(T)); });
  sv.place(g.D, [&](int row) { return row * (int)(g.v.st * sizeof(T)); });
  auto fetch = [&](int j) {
    sk.load(kb + j * g.k.st, kend - j);
    sv.load(vb + j * g.v.st, kend - j);
  };
  f32x16 acc[DP / 32];
#pragma unroll
  for (int j = 0; j < DP / 32; ++j) acc[j] = zero16();
  int buf = 0;
  if (kbeg < kend) {
    fetch(kbeg);
    sk.store(ktile[0]);
    sv.store(vtile[0]);
  }
  __syncthreads();
  for (int j = kbeg; j < kend; j += KT) {
    const bool more = j + KT < kend;
#pragma unroll
    for (int kk = 0; kk < KT / 32; ++kk) {
      f32x16 s = mul_rows<DP, true>(ktile[buf], qf, 32 * kk, c, h);
      if (kk == 0 && more) fetch(j + KT);
      f32x16 dp = mul_rows<DP, false>(vtile[buf], gf, 32 * kk, c, h, less);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], p.cs, -lse));
      if (j + KT > kend) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (j + 32 * kk + 8 * (i / 4) + 4 * h + i % 4 >= kend) s[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] *= s[i];
      mul_cols<DP, FINE>(ktile[buf], dp, 32 * kk, lane, acc);
    }
    if (more) {
      sk.store(ktile[buf ^ 1]);
      sv.store(vtile[buf ^ 1]);
    }
    __syncthreads();
    buf ^= 1;
  }
  if (r >= p.R) return;
  if (kl == 1) {               // the softmax of one key is constant
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = zero16();
  }
  if (p.splits > 1) {
    float* out = p.part + (((size_t)prob * p.splits + sp) * p.R + r) * DP;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) store_cols(out, acc[d], d, h, DP, 1.f);
  } else {
    T* out = const_cast<T*>(row_at<T>(p.gq, g.gq, p, b, hk, r));
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) store_cols(out, acc[d], d, h, g.D, g.scale);
  }
}

// Gradients of keys and values: a block owns kTileRows keys (32 a wave, in registers) and walks the problem's rows. bf16
// heads of 128: the values of the block's keys stay in LDS instead and the rows come 32 at a time, which brings the kernel
// under 256 registers, i.e. to two waves a SIMD (this walk of the long case: 3138 us with
// all in registers, 2350 so).
template <class T, int DP>
constexpr int row_len() {
  return sizeof(T) == 2 && DP < 128 ? 64 : 32;
}
template <class T, int DP>
struct GkvTiles {
  static constexpr int RT = row_len<T, DP>();
  static constexpr bool kValues = sizeof(T) == 2 && DP == 128;
  T rows[2][2][RT * Tile<T, DP, true>::LD];              // [buffer][queries, their output gradients]
  T v[kValues ? kTileRows * Tile<T, DP, false>::LD : 8];
  float stat[2][2][RT];                                  // [buffer][row sums' logarithms, -delta]
};
template <class T, int DP, bool FINE>
__device__ __forceinline__ void keys_gradient(const AttnParams& p, int id, GkvTiles<T, DP>& tiles) {
  constexpr int RT = GkvTiles<T, DP>::RT;
  constexpr bool kValuesInLds = GkvTiles<T, DP>::kValues;
  using Plain = Tile<T, DP, false>;
  auto& smem = tiles.rows;
  auto& vtile = tiles.v;
  auto& stat = tiles.stat;
  const vg_attention_geom& g = p.g;
  const int kt = id % p.key_tiles, sp = (id / p.key_tiles) % p.r_splits, prob = id / (p.key_tiles * p.r_splits);
  const int b = prob / g.Hk, hk = prob - b * g.Hk;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int rows = clamped(p.q_len, b, g.Tq) * p.G;
  const int kl = clamped(p.k_len, b, g.Tk);
  const int key = kt * kTileRows + wid * 32 + c;
  const int rbeg = sp * p.r_chunk, rend = kt * kTileRows < kl ? min(rows, rbeg + p.r_chunk) : 0;

  RowFrag<T, DP> kf, vf;
  kf.load((const T*)p.k + b * g.k.sb + hk * g.k.sh + (int64_t)(key < kl ? key : 0) * g.k.st, g.D, h, key < kl);
  if constexpr (kValuesInLds) {
    constexpr int V = TokNum<T>::V;
    for (int id = threadIdx.x; id < kTileRows * DP / V; id += 64 * kWaves) {
      const int row = id / (DP / V), d = id % (DP / V) * V, j = kt * kTileRows + row;
      const T* src = (const T*)p.v + b * g.v.sb + hk * g.v.sh + (int64_t)j * g.v.st + d;
      *reinterpret_cast<u32x4*>(vtile + Plain::at(row, d)) = j < kl && d < g.D ? *reinterpret_cast<const u32x4*>(src) : u32x4{0, 0, 0, 0};
    }
  } else {
    vf.load((const T*)p.v + b * g.v.sb + hk * g.v.sh + (int64_t)(key < kl ? key : 0) * g.v.st, g.D, h, key < kl);
  }
  Stage<T, DP, RT, true> sq, sg;
  float st_l = INFINITY, st_d = 0.f;
  auto place = [&](int j) {        // rows of a tile are whole queries where G divides RT: the same offsets in every tile
    const int t0 = row_query(p, j);
    auto at = [&](int row, const vg_heads_layout& l) {
      const int r = j + row, t = row_query(p, r);
      return (int)(((t - t0) * l.st + (r - t * p.G) * l.sh) * (int64_t)sizeof(T));
    };
    sq.place(g.D, [&](int row) { return at(row, g.q); });
    sg.place(g.D, [&](int row) { return at(row, g.go); });
  };
  place(rbeg);
  const T* qb = (const T*)p.q + b * g.q.sb + (int64_t)hk * p.G * g.q.sh;
  const T* gb = (const T*)p.go + b * g.go.sb + (int64_t)hk * p.G * g.go.sh;
  const bool whole = RT % p.G == 0;
  auto fetch = [&](int j) {
    if (!whole) place(j);
    const int t0 = row_query(p, j);
    sq.load(qb + t0 * g.q.st, rend - j);
    sg.load(gb + t0 * g.go.st, rend - j);
    if (threadIdx.x < RT) {
      const bool ok = j + (int)threadIdx.x < rend;
      st_l = ok ? p.lse_in[(size_t)prob * p.R + j + threadIdx.x] : INFINITY;
      st_d = ok ? p.delta[(size_t)prob * p.R + j + threadIdx.x] : 0.f;
    }
  };
  auto put = [&](int buf) {
    sq.store(smem[buf][0]);
    sg.store(smem[buf][1]);
    if (threadIdx.x < RT) {
      stat[buf][0][threadIdx.x] = st_l;
      stat[buf][1][threadIdx.x] = -st_d;
    }
  };
  f32x16 gk[DP / 32], gv[DP / 32];
#pragma unroll
  for (int j = 0; j < DP / 32; ++j) gk[j] = gv[j] = zero16();
  int buf = 0;
  if (rbeg < rend) {
    fetch(rbeg);
    put(0);
  }
  __syncthreads();
  for (int j = rbeg; j < rend; j += RT) {
    const bool more = j + RT < rend;
#pragma unroll
    for (int rr = 0; rr < RT / 32; ++rr) {
      f32x16 w = mul_rows<DP, true>(smem[buf][0], kf, 32 * rr, c, h), dp;
      if (rr == 0 && more) fetch(j + RT);
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {      // go v^T starts from -delta
        const f32x4 lse = *reinterpret_cast<const f32x4*>(&stat[buf][0][32 * rr + 8 * i4 + 4 * h]);
        const f32x4 less = *reinterpret_cast<const f32x4*>(&stat[buf][1][32 * rr + 8 * i4 + 4 * h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[4 * i4 + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[4 * i4 + e], p.cs, -lse[e]));
          dp[4 * i4 + e] = less[e];
        }
      }
      if constexpr (kValuesInLds)
        dp = mul_tiles<DP, true>(smem[buf][1], vtile, 32 * rr, 32 * wid, c, h, dp);
      else
        dp = mul_rows<DP, true>(smem[buf][1], vf, 32 * rr, c, h, dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] *= w[i];
      mul_cols<DP, FINE>(smem[buf][1], w, 32 * rr, lane, gv);
      __builtin_amdgcn_sched_barrier(0);     // (reads hoisted across this line spill)
      mul_cols<DP, FINE>(smem[buf][0], dp, 32 * rr, lane, gk);
    }
    if (more) put(buf ^ 1);
    __syncthreads();
    buf ^= 1;
  }
  if (key >= g.Tk) return;
  // keys that take no part went through the products as zeros: their columns are not used
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) {
    if (key >= kl) gk[d] = gv[d] = zero16();
    if (kl == 1) gk[d] = zero16();         // (the softmax of one key is constant)
    if (p.r_splits > 1) {
      const size_t at = (((size_t)prob * p.r_splits + sp) * g.Tk + key) * DP;
      const size_t half = (size_t)g.B * g.Hk * p.r_splits * g.Tk * DP;
      store_cols(p.part_kv + at, gk[d], d, h, DP, 1.f);
      store_cols(p.part_kv + half + at, gv[d], d, h, DP, 1.f);
    } else {
      store_cols((T*)p.gk + b * g.gk.sb + hk * g.gk.sh + (int64_t)key * g.gk.st, gk[d], d, h, g.D, g.scale);
      store_cols((T*)p.gv + b * g.gv.sb + hk * g.gv.sh + (int64_t)key * g.gv.st, gv[d], d, h, g.D, 1.f);
    }
  }
}

// Both in one launch, so that neither waits for the other's last blocks: those of the keys' gradient, which take longer, first.
template <class T, int DP, bool FINE>
__global__ void __launch_bounds__(256, sizeof(T) == 2 || DP <= 64 ? 2 : 1) attn_bwd_kernel(const AttnParams p) {
  __shared__ __attribute__((aligned(16))) union {
    unsigned char keys[sizeof(GkvTiles<T, DP>)];
    unsigned char queries[sizeof(GqTiles<T, DP>)];
  } smem;
  const int id = blockIdx.x - p.gkv_blocks;
  if (id < 0)
    keys_gradient<T, DP, FINE>(p, tok_xcd_order(blockIdx.x, p.gkv_blocks), *reinterpret_cast<GkvTiles<T, DP>*>(smem.keys));
  else
    queries_gradient<T, DP, FINE>(p, tok_xcd_order(id, gridDim.x - p.gkv_blocks), *reinterpret_cast<GqTiles<T, DP>*>(smem.queries));
}

// The split walks' results: queries' rows (if split), keys, values (if split), each the sum over its splits in order, times
// scale (values: 1).
template <class T, int DP>
__global__ void __launch_bounds__(256) attn_sum_kernel(const AttnParams p) {
  constexpr int LPR = DP / 4;
  const vg_attention_geom& g = p.g;
  const long long nq = p.splits > 1 ? (long long)g.B * g.Hk * p.R : 0, nk = p.r_splits > 1 ? (long long)g.B * g.Hk * g.Tk : 0;
  long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int d = (threadIdx.x % LPR) * 4;
  if (row >= nq + 2 * nk || d >= g.D) return;
  const int which = row < nq ? 0 : row < nq + nk ? 1 : 2;
  row -= which == 0 ? 0 : which == 1 ? nq : nq + nk;
  const int n = which == 0 ? p.R : g.Tk, splits = which == 0 ? p.splits : p.r_splits;
  const float* part = which == 0 ? p.part : p.part_kv + (which == 2 ? (size_t)nk * splits * DP : 0);
  const int prob = (int)(row / n), r = (int)(row - (long long)prob * n);
  const int b = prob / g.Hk, hk = prob - b * g.Hk;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  part += ((size_t)prob * splits * n + r) * DP + d;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(part + (size_t)s * n * DP);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += x[e];
  }
  const float f = which == 2 ? 1.f : g.scale;
  T* out = which == 0   ? const_cast<T*>(row_at<T>(p.gq, g.gq, p, b, hk, r))
           : which == 1 ? (T*)p.gk + b * g.gk.sb + hk * g.gk.sh + (int64_t)r * g.gk.st
                        : (T*)p.gv + b * g.gv.sb + hk * g.gv.sh + (int64_t)r * g.gv.st;
  tok_store4(out + d, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
}

// ---- host -----------------------------------------------------------------------------------------------------------
// Heads are worked on at the next width of these (zeros behind their own elements): 72 and 96 cost what 128 does (4 x 8 heads,
// 2048 queries and keys, bf16: 86 us forward, 238 backward; 64: 61 and 137).
int padded_width(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

int check_geom(const vg_attention_geom* g) {
  VG_REQUIRE(g, "attention: null geometry");
  VG_REQUIRE(g->B >= 0 && g->Tq >= 0 && g->Tk >= 0 && g->Hq >= 1 && g->Hk >= 1, "attention: bad sizes B=%d Tq=%d Tk=%d Hq=%d Hk=%d", g->B,
             g->Tq, g->Tk, g->Hq, g->Hk);
  VG_REQUIRE(g->Hq % g->Hk == 0, "attention: %d query heads are not a multiple of %d key heads", g->Hq, g->Hk);
  VG_REQUIRE(g->D >= 8 && g->D <= 128 && g->D % 8 == 0, "attention: head width %d is not a multiple of 8 from 8 to 128", g->D);
  const long long G = g->Hq / g->Hk, R = (long long)g->Tq * G;
  // r / G by a 32-bit product; block counts of 31 bits
  VG_REQUIRE((R + kTileRows) * G < (1ll << 32) && R < (1ll << 30) && g->Tk < (1 << 30), "attention: %d queries of %lld heads a group are too many",
             g->Tq, G);
  VG_REQUIRE(((R + kTileRows - 1) / kTileRows + 1) * g->B * (long long)g->Hk < (1ll << 31) / 64 &&
                 (((long long)g->Tk + kTileRows - 1) / kTileRows + 1) * g->B * (long long)g->Hk < (1ll << 31) / 64,
             "attention: too many blocks");
  VG_REQUIRE(isfinite(g->scale) && g->scale != 0.f, "attention: scale is zero or not finite");
  return VG_OK;
}

// byte offsets inside a tile of 64 rows are 31-bit
template <class T>
bool strides_ok(const vg_heads_layout& l, int tokens, int heads) {
  const int64_t most = kRange / 2 / (int64_t)sizeof(T);
  return (tokens <= 1 || (l.st >= 0 && l.st < most / 66)) && (heads <= 1 || (l.sh >= 0 && l.sh < most / heads));
}
template <class T>
int check_strides(const vg_attention_geom* g, bool backward) {
  const int G = g->Hq / g->Hk;
  VG_REQUIRE(strides_ok<T>(g->q, g->Tq, G) && (!backward || strides_ok<T>(g->go, g->Tq, G)) && strides_ok<T>(g->k, g->Tk, 1) &&
                 strides_ok<T>(g->v, g->Tk, 1),
             "attention: a stride between tokens or heads is too large");
  return VG_OK;
}

// A walk over `len` (keys, or rows) is split where the blocks alone leave compute units idle: towards 512 blocks (two
// for each of the 256), but into no more than len / 128 splits (f32, whose products take eight times as long: len / 64),
// beyond which a split's own start and its partial results cost more than the walk it saves. The splits' length is then
// rounded up to whole tiles of 64 (chunk_of), so the last splits of some lengths are empty: of the 8 over 517 f32 keys, 128
// each, three are. They write zeros, which the joining kernel adds like the others.
template <class T>
int splits_for(long long blocks, long long len) {
  if (blocks >= 256 || blocks == 0) return 1;
  long long s = 512 / blocks, most = len / (sizeof(T) == 2 ? 128 : 64);
  if (s > most) s = most;
  return s < 1 ? 1 : (int)s;
}

struct Plan {
  int G, R, row_tiles, key_tiles, probs, fwd_splits, gkv_splits;
};
template <class T>
Plan plan_of(const vg_attention_geom* g) {
  Plan q;
  q.G = g->Hq / g->Hk;
  q.R = g->Tq * q.G;
  q.probs = g->B * g->Hk;
  q.row_tiles = ceil_div(q.R, kTileRows);
  q.key_tiles = ceil_div(g->Tk, kTileRows);
  q.fwd_splits = splits_for<T>((long long)q.row_tiles * q.probs, g->Tk);
  q.gkv_splits = splits_for<T>((long long)q.key_tiles * q.probs, q.R);
  return q;
}
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t fwd_bytes(const vg_attention_geom* g, const Plan& q) {
  if (q.fwd_splits == 1) return 0;
  const size_t rows = (size_t)q.probs * q.fwd_splits * q.R;
  return align256(rows * padded_width(g->D) * 4) + rows * 8;
}
// delta, partial queries' rows, partial keys and values
size_t gq_bytes(const vg_attention_geom* g, const Plan& q) {
  return q.fwd_splits == 1 ? 0 : align256((size_t)q.probs * q.fwd_splits * q.R * padded_width(g->D) * 4);
}
size_t bwd_bytes(const vg_attention_geom* g, const Plan& q) {
  const size_t kv = q.gkv_splits == 1 ? 0 : 2 * (size_t)q.probs * q.gkv_splits * g->Tk * padded_width(g->D) * 4;
  return align256((size_t)q.probs * q.R * 4) + gq_bytes(g, q) + kv;
}

AttnParams params_of(const vg_attention_geom* g, const Plan& q) {
  AttnParams p = {};
  p.g = *g;
  p.G = q.G;
  p.R = q.R;
  p.g_magic = (unsigned)(((1ull << 32) + q.G - 1) / q.G);
  p.row_tiles = q.row_tiles;
  p.key_tiles = q.key_tiles;
  p.cs = g->scale * 1.44269504088896341f;
  return p;
}
int chunk_of(int len, int splits) { return ((len + splits - 1) / splits + 63) & ~63; }

// bf16: probabilities and ds go into their products rounded to bf16. That costs a result up to 0.4 of its own rounding,
// whatever the number of terms (l2 against 64 bits, heads of 64, 2 to 512 keys: o 1.8 to 2.3e-3, gradients 2.3 to 2.5e-3, the
// results' rounding alone 1.7e-3), and the queries' gradient more where the keys have a part in common: ds sums to zero and
// cancels it, the rounded ds do not (keys, values and output gradients of deviation 1 and mean 1: 3.2 to 3.6e-3, mean 3: 6.4
// to 7.3e-3). Calls of under 2^20 scores take both as two bf16 terms (2^-17) and come out at the results' rounding alone in
// all of these; there the products take a few microseconds. In larger calls the second term would cost up to a fifth (64 x
// 16 heads of 128 of one query on 2048 keys: forward 49 -> 60 us). The size is that of the whole call, so a batch element's
// last bits depend on the batch it is in.
template <class T>
bool fine(const vg_attention_geom& g) {
  return sizeof(T) == 2 && (double)g.B * g.Hq * g.Tq * g.Tk < (double)(1 << 20);
}
template <class T, int DP, bool FINE>
void launch_fwd_of(AttnParams& p, const Plan& q, hipStream_t st) {
  p.splits = q.fwd_splits;
  p.chunk = chunk_of(p.g.Tk, p.splits);
  const int grid = q.row_tiles * p.splits * q.probs;
  if (p.splits == 1) {
    attn_fwd_kernel<T, DP, false, FINE><<<grid, 256, 0, st>>>(p);
  } else {
    attn_fwd_kernel<T, DP, true, FINE><<<grid, 256, 0, st>>>(p);
    int per_row = 1;           // four splits a group of lanes
    while (per_row < 256 / (DP / 4) && per_row * 4 < p.splits) per_row *= 2;
    attn_join_kernel<T, DP><<<ceil_div((long long)q.probs * q.R * per_row, 256 / (DP / 4)), 256, 0, st>>>(p, per_row);
  }
}
template <class T, int DP>
void launch_fwd(AttnParams& p, const Plan& q, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (fine<T>(p.g)) return launch_fwd_of<T, DP, true>(p, q, st);
  launch_fwd_of<T, DP, false>(p, q, st);
}
template <class T, int DP>
void launch_bwd(AttnParams& p, const Plan& q, float* delta, hipStream_t st) {
  if (q.R > 0) attn_delta_kernel<T><<<ceil_div((long long)q.probs * q.R, 32), 256, 0, st>>>(p, delta);
  p.splits = p.gq ? q.fwd_splits : 1;
  p.chunk = chunk_of(p.g.Tk, p.splits);
  p.r_splits = p.gk ? q.gkv_splits : 1;
  p.r_chunk = chunk_of(q.R, p.r_splits);
  p.gkv_blocks = p.gk ? q.key_tiles * p.r_splits * q.probs : 0;
  const int gq_blocks = p.gq ? q.row_tiles * p.splits * q.probs : 0;
  if (p.gkv_blocks + gq_blocks > 0) {
    auto kernel = attn_bwd_kernel<T, DP, false>;
    if constexpr (sizeof(T) == 2)
      if (fine<T>(p.g)) kernel = attn_bwd_kernel<T, DP, true>;
    kernel<<<p.gkv_blocks + gq_blocks, 256, 0, st>>>(p);
  }
  const long long rows = (p.splits > 1 ? (long long)q.probs * q.R : 0) + (p.r_splits > 1 ? 2ll * q.probs * p.g.Tk : 0);
  if (rows > 0) attn_sum_kernel<T, DP><<<ceil_div(rows, 256 / (DP / 4)), 256, 0, st>>>(p);
}

template <class T>
int attention_fwd(const vg_attention_geom* g, const void* q, const void* k, const void* v, const int32_t* q_len, const int32_t* k_len,
                  void* o, void* low, float* lse, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_geom(g);
  if (rc) return rc;
  const Plan pl = plan_of<T>(g);
  if (pl.probs == 0 || pl.R == 0) return VG_OK;
  VG_REQUIRE(q && o && (g->Tk == 0 || (k && v)), "attention: null tensor");
  VG_REQUIRE(tok_layout_ok<T>(g->q, q, g->B, g->Tq, g->Hq) && tok_layout_ok<T>(g->o, o, g->B, g->Tq, g->Hq) &&
                 tok_layout_ok<T>(g->k, k, g->B, g->Tk, g->Hk) && tok_layout_ok<T>(g->v, v, g->B, g->Tk, g->Hk),
             "attention: a head does not start on a 16-byte border");
  const int sc = check_strides<T>(g, false);
  if (sc) return sc;
  const size_t need = fwd_bytes(g, pl);
  if (need && (!ws || ws_bytes < need)) return vg_fail(VG_ERR_WORKSPACE, "attention: workspace of %zu bytes, %zu are needed", ws_bytes, need);
  VG_REQUIRE(!need || vg_aligned16(ws), "attention: workspace is not 16-byte aligned");
  AttnParams p = params_of(g, pl);
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = o;
  p.low = (__bf16*)low;
  p.lse = lse;
  p.q_len = q_len;
  p.k_len = k_len;
  p.part = (float*)ws;
  if (need) p.part_ml = (float*)((char*)ws + align256((size_t)pl.probs * pl.fwd_splits * pl.R * padded_width(g->D) * 4));
  hipStream_t st = (hipStream_t)stream;
  switch (padded_width(g->D)) {
    case 32: launch_fwd<T, 32>(p, pl, st); break;
    case 64: launch_fwd<T, 64>(p, pl, st); break;
    default: launch_fwd<T, 128>(p, pl, st);
  }
  VG_CHECK_LAUNCH("attention");
  return VG_OK;
}

template <class T>
int attention_bwd(const vg_attention_geom* g, const void* q, const void* k, const void* v, const void* o, const void* low,
                  const float* lse, const void* go, const int32_t* q_len, const int32_t* k_len, void* gq, void* gk, void* gv, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_geom(g);
  if (rc) return rc;
  const Plan pl = plan_of<T>(g);
  if (pl.probs == 0 || (pl.R == 0 && g->Tk == 0)) return VG_OK;
  VG_REQUIRE((pl.R == 0 || (q && o && lse && go)) && (g->Tk == 0 || (k && v)) && !gk == !gv, "attention backward: null tensor");
  VG_REQUIRE(tok_layout_ok<T>(g->q, q, g->B, g->Tq, g->Hq) && tok_layout_ok<T>(g->o, o, g->B, g->Tq, g->Hq) &&
                 tok_layout_ok<T>(g->go, go, g->B, g->Tq, g->Hq) && tok_layout_ok<T>(g->gq, gq, g->B, g->Tq, g->Hq) &&
                 tok_layout_ok<T>(g->k, k, g->B, g->Tk, g->Hk) && tok_layout_ok<T>(g->v, v, g->B, g->Tk, g->Hk) &&
                 tok_layout_ok<T>(g->gk, gk, g->B, g->Tk, g->Hk) && tok_layout_ok<T>(g->gv, gv, g->B, g->Tk, g->Hk),
             "attention backward: a head does not start on a 16-byte border");
  const int sc = check_strides<T>(g, true);
  if (sc) return sc;
  const size_t need = bwd_bytes(g, pl);
  if (need && (!ws || ws_bytes < need))
    return vg_fail(VG_ERR_WORKSPACE, "attention backward: workspace of %zu bytes, %zu are needed", ws_bytes, need);
  VG_REQUIRE(!need || vg_aligned16(ws), "attention backward: workspace is not 16-byte aligned");
  AttnParams p = params_of(g, pl);
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = o;
  p.go = go;
  p.low = (__bf16*)const_cast<void*>(low);
  p.lse_in = lse;
  p.q_len = q_len;
  p.k_len = k_len;
  p.gq = gq;
  p.gk = gk;
  p.gv = gv;
  float* delta = (float*)ws;
  p.delta = delta;
  p.part = (float*)((char*)ws + align256((size_t)pl.probs * pl.R * 4));
  p.part_kv = (float*)((char*)p.part + gq_bytes(g, pl));
  hipStream_t st = (hipStream_t)stream;
  switch (padded_width(g->D)) {
    case 32: launch_bwd<T, 32>(p, pl, delta, st); break;
    case 64: launch_bwd<T, 64>(p, pl, delta, st); break;
    default: launch_bwd<T, 128>(p, pl, delta, st);
  }
  VG_CHECK_LAUNCH("attention backward");
  return VG_OK;
}

}  // namespace

extern "C" {

size_t vg_attention_workspace_bytes(const vg_attention_geom* g, int backward, int half) {
  if (check_geom(g)) return 0;
  const Plan q = half ? plan_of<__bf16>(g) : plan_of<float>(g);
  if (q.probs == 0) return 0;
  return backward ? bwd_bytes(g, q) : fwd_bytes(g, q);
}
int vg_attention_fwd(const vg_attention_geom* g, const float* q, const float* k, const float* v, const int32_t* q_len, const int32_t* k_len,
                     float* o, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return attention_fwd<float>(g, q, k, v, q_len, k_len, o, nullptr, lse, workspace, workspace_bytes, stream);
}
int vg_attention_fwd_h(const vg_attention_geom* g, const void* q, const void* k, const void* v, const int32_t* q_len, const int32_t* k_len,
                       void* o, void* o_low, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  VG_REQUIRE(vg_aligned16(o_low), "attention: a tensor does not start on a 16-byte border");
  return attention_fwd<__bf16>(g, q, k, v, q_len, k_len, o, o_low, lse, workspace, workspace_bytes, stream);
}
int vg_attention_bwd(const vg_attention_geom* g, const float* q, const float* k, const float* v, const float* o, const float* lse,
                     const float* go, const int32_t* q_len, const int32_t* k_len, float* gq, float* gk, float* gv, void* workspace,
                     size_t workspace_bytes, void* stream) {
  return attention_bwd<float>(g, q, k, v, o, nullptr, lse, go, q_len, k_len, gq, gk, gv, workspace, workspace_bytes, stream);
}
int vg_attention_bwd_h(const vg_attention_geom* g, const void* q, const void* k, const void* v, const void* o, const void* o_low,
                       const float* lse, const void* go, const int32_t* q_len, const int32_t* k_len, void* gq, void* gk, void* gv,
                       void* workspace, size_t workspace_bytes, void* stream) {
  VG_REQUIRE(vg_aligned16(o_low), "attention backward: a tensor does not start on a 16-byte border");
  return attention_bwd<__bf16>(g, q, k, v, o, o_low, lse, go, q_len, k_len, gq, gk, gv, workspace, workspace_bytes, stream);
}

}  // extern "C"
