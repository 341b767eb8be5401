// Tile product of the gated linear layer on the matrix cores: acc[m][n] = sum over k of A[m][k] B[n][k] for a BM x BN tile,
// f32 accumulators, bf16 operands on v_mfma_f32_32x32x16_bf16 and f32 operands on v_mfma_f32_32x32x2_f32.
//
// An operand is contiguous along k (KC: element (row, k) at row * ld + k) or along its row index (RC: at k * ld + row).
// Tiles go global -> registers -> LDS in 16-byte vectors, two LDS buffers, one barrier per k-step, the next k-step's
// loads in flight under the products. KC tiles are kept [row][k] with 16 bytes of padding (a lane's 8 k are one
// ds_read_b128); RC tiles are kept [k][row] as loaded and read with the transposing LDS load, which hands a lane 4
// consecutive k of its row (f32: 4-byte loads). Operands whose rows do not start on 16-byte borders are loaded element by element
// (ALIGNED = false): same tiles, same results.
#pragma once
#include "token_common.h"

template <class T>
struct TokOperand {
  const T* p;
  int64_t ld;
  int rows;     // valid row indices
  int split;    // KC with two interleaved halves (gate and value weights): rows of the second half start here; 0: plain
};

template <class T, bool RC, int ROWS, int BK, int NT, bool ALIGNED>
struct TokStage {
  static constexpr int V = TokNum<T>::V;
  static constexpr int LD = RC ? ROWS + 32 : BK + V;                   // elements of an LDS row
  static constexpr int ELEMS = RC ? BK * LD : ROWS * LD;
  static constexpr int VPR = (RC ? ROWS : BK) / V;                     // vectors of an LDS row
  static constexpr int N = ROWS * BK / V / NT;
  static_assert(ROWS * BK / V % NT == 0, "whole vectors per thread");
  u32x4 r[N];

  static __device__ __forceinline__ u32x4 vec(const T* p, int left) {   // `left` elements of the vector are inside
    if constexpr (ALIGNED) {
      return left > 0 ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
    } else {
      u32x4 out = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (sizeof(T) == 4) {
          if (e < left) out[e] = *reinterpret_cast<const unsigned*>(p + e);
        } else {
          if (e < left) out[e / 2] |= (unsigned)*reinterpret_cast<const unsigned short*>(p + e) << (16 * (e % 2));
        }
      }
      return out;
    }
  }
  // rows row0.. of the operand, k from k0, nothing at or past kend
  __device__ __forceinline__ void load(const TokOperand<T>& a, int row0, int k0, int kend) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = threadIdx.x + i * NT, lr = id / VPR, lv = (id % VPR) * V;
      if constexpr (RC) {
        const int k = k0 + lr, row = row0 + lv;
        r[i] = vec(a.p + k * a.ld + row, k < kend ? a.rows - row : 0);
      } else {
        int row = row0 + lr;
        bool ok = row < a.rows;
        if (a.split) {       // 32 rows of the first half, the matching 32 of the second, ...
          const int f = (row >> 6) * 32 + (row & 31);
          ok = f < a.split;
          row = f + ((row >> 5) & 1) * a.split;
        }
        r[i] = vec(a.p + row * a.ld + k0 + lv, ok ? kend - k0 - lv : 0);
      }
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = threadIdx.x + i * NT;
      *reinterpret_cast<u32x4*>(tile + (id / VPR) * LD + (id % VPR) * V) = r[i];
    }
  }
  // fragment of 32 rows from row0, 16 k (bf16) from 16 s, or 8 k (f32; lane half h holds 4 of them) from 8 s
  static __device__ __forceinline__ bf16x8 frag(const __bf16* tile, int row0, int s, int lane) {
    const int c = lane & 31, h = lane >> 5;
    if constexpr (!RC) {
      return *reinterpret_cast<const bf16x8*>(tile + (row0 + c) * LD + 16 * s + 8 * h);
    } else {
      const __bf16* a = tile + (16 * s + 8 * h + ((lane & 15) >> 2)) * LD + row0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 4 * LD));
      const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(bf16x8, v);
    }
  }
  static __device__ __forceinline__ f32x4 frag(const float* tile, int row0, int s, int lane) {
    const int c = lane & 31, h = lane >> 5;
    if constexpr (!RC) {
      return *reinterpret_cast<const f32x4*>(tile + (row0 + c) * LD + 8 * s + 4 * h);
    } else {
      const float* a = tile + (8 * s + 4 * h) * LD + row0 + c;
      return f32x4{a[0], a[LD], a[2 * LD], a[3 * LD]};
    }
  }
};

__device__ __forceinline__ f32x16 tok_mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 tok_mma(f32x4 a, f32x4 b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

template <class T, bool ARC, bool BRC, int BM, int BN, int WM, int WN, bool ALIGNED>
struct TokGemm {
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int BK = sizeof(T) == 2 ? 64 : 32;
  static constexpr int TM = BM / (32 * WM), TN = BN / (32 * WN);
  static constexpr int KS = sizeof(T) == 2 ? 16 : 8;        // k of one fragment
  using SA = TokStage<T, ARC, BM, BK, NT, ALIGNED>;
  using SB = TokStage<T, BRC, BN, BK, NT, ALIGNED>;
  static constexpr int BUF = SA::ELEMS + SB::ELEMS;
  static constexpr int LDS_BYTES = 2 * BUF * (int)sizeof(T);

  // acc over k in [kbeg, kend); smem holds LDS_BYTES. All threads of the block call it.
  static __device__ __forceinline__ void run(const TokOperand<T>& A, const TokOperand<T>& B, int m0, int n0, int kbeg, int kend, T* smem,
                                             f32x16 (&acc)[TM][TN]) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int mw = (wid / WN) * TM * 32, nw = (wid % WN) * TN * 32;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    SA sa;
    SB sb;
    int buf = 0;
    if (kbeg < kend) {
      sa.load(A, m0, kbeg, kend);
      sb.load(B, n0, kbeg, kend);
      sa.store(smem);
      sb.store(smem + SA::ELEMS);
    }
    __syncthreads();
    for (int k = kbeg; k < kend; k += BK) {
      const bool more = k + BK < kend;
      if (more) {
        sa.load(A, m0, k + BK, kend);
        sb.load(B, n0, k + BK, kend);
      }
      const T* ta = smem + buf * BUF;
      const T* tb = ta + SA::ELEMS;
#pragma unroll
      for (int s = 0; s < BK / KS; ++s) {
        decltype(SA::frag(ta, 0, 0, 0)) fa[TM], fb[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[i] = SA::frag(ta, mw + 32 * i, s, lane);
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[j] = SB::frag(tb, nw + 32 * j, s, lane);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = tok_mma(fa[i], fb[j], acc[i][j]);
      }
      if (more) {
        sa.store(smem + (buf ^ 1) * BUF);
        sb.store(smem + (buf ^ 1) * BUF + SA::ELEMS);
      }
      __syncthreads();
      buf ^= 1;
    }
  }
};
