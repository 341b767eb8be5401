// Tile product of the gated linear layer on the matrix cores: acc[m][n] = sum over k of A[m][k] B[n][k] for a BM x BN tile,
// f32 accumulators, bf16 operands on v_mfma_f32_32x32x16_bf16 and f32 operands on v_mfma_f32_32x32x2_f32.
//
// An operand is contiguous along k (KC: element (row, k) at row * ld + k) or along its row index (RC: at k * ld + row).
// Tiles go global -> registers -> LDS in 16-byte vectors, two LDS buffers, one barrier per k-step, the next k-step's
// loads in flight under the products. KC tiles are kept [row][k] with 16 bytes of padding (a lane's 8 k are one
// ds_read_b128); RC tiles are kept [k][row] as loaded and read with the transposing LDS load, which hands a lane 4
// consecutive k of its row (f32: 4-byte loads). A thread's offsets from the tile's first element are the same in every
// k-step; only the uniform base moves. Row indices past the operand are clamped to its last row (what they produce is
// not stored); k past the end becomes zero, in the last k-step only. The vector loads need no alignment beyond an
// element's, so odd leading dimensions take the same path.
#pragma once
#include "token_common.h"

template <class T>
struct TokOperand {
  const T* p;
  int64_t ld;
  int rows;     // valid row indices
  int split;    // KC, two interleaved halves (gate and value weights): rows of the second half start here; 0: plain
};

// Order of the 32 rows of a block of an interleaved operand: a product leaves lane half h the rows 8 (i / 4) + 4 h + i % 4 of
// its column; with this order those are the operand's rows 16 h + i, sixteen in a row that leave as one piece.
__device__ __forceinline__ int tok_split_row(int r) { return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3); }

template <class T, bool RC, int ROWS, int BK, int NT>
struct TokStage {
  static constexpr int V = TokNum<T>::V;
  static constexpr int LD = RC ? ROWS + 32 : BK + V;                   // elements of an LDS row
  static constexpr int ELEMS = RC ? BK * LD : ROWS * LD;
  static constexpr int VPR = (RC ? ROWS : BK) / V;                     // vectors of an LDS row
  static constexpr int N = ROWS * BK / V / NT;
  static_assert(ROWS * BK / V % NT == 0, "whole vectors per thread");
  u32x4 r[N];
  unsigned off[N];      // bytes from the base: inside the tile, i.e. at most 256 rows (k) of the operand
  const char* base;     // first row of the tile at the current k (interleaved: the first of vector 0's half)
  int64_t half;         // interleaved: bytes from one half of the operand to the other where a thread's vectors alternate
  bool edge;            // RC: vectors of the tile cross the operand's last row

  static __device__ __forceinline__ u32x4 whole(const char* p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
  }
  static __device__ __forceinline__ u32x4 part(const char* p, int left) {   // the first `left` elements, then zeros
    u32x4 out = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (sizeof(T) == 4) {
        if (e < left) out[e] = *reinterpret_cast<const unsigned*>(p + 4 * e);
      } else {
        if (e < left) out[e / 2] |= (unsigned)*reinterpret_cast<const unsigned short*>(p + 2 * e) << (16 * (e % 2));
      }
    }
    return out;
  }
  // An interleaved tile lies in two runs of rows, up to 2^40 bytes apart, so the way from one to the other is not part of
  // the 32-bit offsets: 32 rows of one half are followed by 32 of the other, and a block's threads cover RPV rows with one
  // vector each. Where that is 32 a thread's vectors alternate between the halves; where it is a multiple of 64 they all lie
  // in one half, the same for a whole wave.
  static constexpr int RPV = RC ? 64 : NT / VPR;
  static_assert(RPV == 32 || RPV % 64 == 0, "a thread's vectors alternate between the halves or stay in one");
  __device__ __forceinline__ const char* at(int i) const { return (RPV == 32 && i % 2 ? base + half : base) + off[i]; }
  // rows row0.. of the operand, from k
  __device__ __forceinline__ void place(const TokOperand<T>& a, int row0, int k) {
    half = a.split * a.ld * (int64_t)sizeof(T);
    base = reinterpret_cast<const char*>(a.p + (RC ? k * a.ld + row0 : k + (a.split ? row0 / 2 : row0) * a.ld));
    if (!RC && RPV != 32 && (__builtin_amdgcn_readfirstlane(threadIdx.x) / VPR >> 5) % 2) base += half;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = threadIdx.x + i * NT, lr = id / VPR, lv = (id % VPR) * V;
      if constexpr (RC) {
        const int left = a.rows - row0 - lv;
        off[i] = (unsigned)(((int64_t)lr * a.ld + (left > 0 ? lv : 0)) * (int)sizeof(T));
      } else {
        int row = lr;
        if (a.split) {       // 32 rows of the first half, the matching 32 of the second, ... (tok_split_row)
          const int f = (lr >> 6) * 32 + tok_split_row(lr & 31), last = a.split - 1 - row0 / 2;
          row = f < last ? f : last;
        } else if (row0 + row >= a.rows) {
          row = a.rows - 1 - row0;
        }
        off[i] = (unsigned)(((int64_t)row * a.ld + lv) * (int)sizeof(T));
      }
    }
    edge = RC && row0 + ROWS > a.rows && a.rows % V != 0;
  }
  // the k-step at the base, all of it inside the operand; then on to the next
  __device__ __forceinline__ void load_inside(const TokOperand<T>& a) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = whole(at(i));
    base += (RC ? BK * a.ld : BK) * (int64_t)sizeof(T);
  }
  // The first `left` elements at p, zeros behind them: the 16 bytes that end with them, shifted down (`left` may be
  // negative: zeros; the V elements before p + left are readable).
  static __device__ __forceinline__ u32x4 first(const char* p, int left) {
    const int s = left >= V ? 0 : left <= 0 ? V : V - left;
    u32x4 w = whole(p + (left < V ? left - V : 0) * (int)sizeof(T));
    const int bytes = s * (int)sizeof(T);
    if (bytes & 4) w = u32x4{w[1], w[2], w[3], 0u};
    if (bytes & 8) w = u32x4{w[2], w[3], 0u, 0u};
    if (sizeof(T) == 2 && (bytes & 2))
      w = u32x4{__builtin_amdgcn_alignbyte(w[1], w[0], 2), __builtin_amdgcn_alignbyte(w[2], w[1], 2), __builtin_amdgcn_alignbyte(w[3], w[2], 2),
                w[3] >> 16};
    return bytes >= 16 ? u32x4{0, 0, 0, 0} : w;
  }
  // the k-step that starts at k, whatever lies outside
  __device__ __forceinline__ void load(const TokOperand<T>& a, int row0, int k, int kend) {
    if (k + BK <= kend && !edge) {
      load_inside(a);
      return;
    }
    const bool roomy = RC ? a.rows >= V : kend >= V;       // a row has the 16 bytes that first() reads
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = threadIdx.x + i * NT, lr = id / VPR, lv = (id % VPR) * V;
      if constexpr (RC) {
        // (past the last row: what lies at the clamped offset, it is not used)
        const int inside = a.rows - row0 - lv, left = k + lr < kend ? (inside > 0 ? inside : a.rows - row0) : 0;
        if (left <= 0)
          r[i] = u32x4{0, 0, 0, 0};
        else
          r[i] = roomy ? first(at(i), left) : part(at(i), left);
      } else {
        const int left = kend - k - lv;
        r[i] = roomy ? first(at(i), left) : part(at(i), left);
      }
    }
    base += (RC ? BK * a.ld : BK) * (int64_t)sizeof(T);
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

// One product of two fragments is kParts matrix instructions (f32: a fragment's 4 k, two at a time over the lane halves).
template <class T>
constexpr int tok_parts() { return sizeof(T) == 2 ? 1 : 4; }
__device__ __forceinline__ f32x16 tok_mma(bf16x8 a, bf16x8 b, f32x16 c, int) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 tok_mma(f32x4 a, f32x4 b, f32x16 c, int e) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
}

template <class T, bool ARC, bool BRC, int BM, int BN, int WM, int WN>
struct TokGemm {
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int BK = sizeof(T) == 2 ? 64 : 32;
  static constexpr int TM = BM / (32 * WM), TN = BN / (32 * WN);
  static constexpr int KS = sizeof(T) == 2 ? 16 : 8;        // k of one fragment
  using SA = TokStage<T, ARC, BM, BK, NT>;
  using SB = TokStage<T, BRC, BN, BK, NT>;
  static constexpr int BUF = SA::ELEMS + SB::ELEMS;
  static constexpr int LDS_BYTES = 2 * BUF * (int)sizeof(T);

  // acc over k in [kbeg, kend); smem holds LDS_BYTES. All threads of the block call it; both operands have rows.
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
    sa.place(A, m0, kbeg);
    sb.place(B, n0, kbeg);
    using FA = decltype(SA::frag(smem, 0, 0, 0));
    constexpr int S = BK / KS;
    int buf = 0;
    // One k-step on buffer `buf`. The registers hold the next one: it goes to the other buffer under the products, and
    // the one behind it is requested then, a whole k-step before its own turn.
    auto step = [&](auto inside, int k) {
      const T* ta = smem + buf * BUF;
      const T* tb = ta + SA::ELEMS;
      FA fa[2][TM], fb[2][TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[0][i] = SA::frag(ta, mw + 32 * i, 0, lane);
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[0][j] = SB::frag(tb, nw + 32 * j, 0, lane);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (s + 1 < S) {
#pragma unroll
          for (int i = 0; i < TM; ++i) fa[(s + 1) & 1][i] = SA::frag(ta, mw + 32 * i, s + 1, lane);
#pragma unroll
          for (int j = 0; j < TN; ++j) fb[(s + 1) & 1][j] = SB::frag(tb, nw + 32 * j, s + 1, lane);
        }
#pragma unroll
        for (int e = 0; e < tok_parts<T>(); ++e)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = tok_mma(fa[s & 1][i], fb[s & 1][j], acc[i][j], e);
        if (s == 0) {
          T* next = smem + (buf ^ 1) * BUF;
          if constexpr (decltype(inside)::value) {
            sa.store(next);
            sb.store(next + SA::ELEMS);
            sa.load_inside(A);
            sb.load_inside(B);
          } else if (k + BK < kend) {
            sa.store(next);
            sb.store(next + SA::ELEMS);
            if (k + 2 * BK < kend) {
              sa.load(A, m0, k + 2 * BK, kend);
              sb.load(B, n0, k + 2 * BK, kend);
            }
          }
        }
      }
      __syncthreads();
      buf ^= 1;
    };
    if (kbeg < kend) {
      sa.load(A, m0, kbeg, kend);
      sb.load(B, n0, kbeg, kend);
      sa.store(smem);
      sb.store(smem + SA::ELEMS);
      if (kbeg + BK < kend) {
        sa.load(A, m0, kbeg + BK, kend);
        sb.load(B, n0, kbeg + BK, kend);
      }
    }
    __syncthreads();
    int k = kbeg;
    if (!sa.edge && !sb.edge)
      for (; k + 3 * BK <= kend; k += BK) step(std::true_type{}, k);
    for (; k < kend; k += BK) step(std::false_type{}, k);
  }
};
