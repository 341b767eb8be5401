// Gated linear layer h = act(g) * u, g = x Wg^T + bg, u = x Wu^T + bu, both projections, the activation and the product
// in one kernel, with its backward pass.
//
//   gg = gh u act'(g)     gu = gh act(g)     gx = [gg gu] [Wg; Wu]     gW = [gg gu]^T x     gb = column sums of [gg gu]
//
// The weights lie as one [2F][C] matrix (gate rows first). A block's weight tile takes 32 gate rows, the matching 32
// value rows, the next 32 gate rows, ...: gate and value of one output element end in the same lane's accumulators and
// the epilogue is private to the lane. Bound by the matrix cores (4 M C F flops forward, twice that backward).
//
// What the backward pass needs of g and u is either written by the forward pass in f32 (z) or, with bf16 operands and
// few input features, computed again: a product of C terms per element against 8 bytes written and read. z is never
// rounded to bf16: the two gradients would carry its error and their own.
#include "token_gemm.h"

namespace {

struct GatedParams {
  const void *x, *w;
  const float* bias;     // [2F] or null
  void* h;               // forward: [M][F]
  float* z;              // forward: [M][2F] or null
  const void* gh;        // recomputing backward: [M][F]
  void* gz;              // [M][2F]
  float* gb_part;        // [row tiles][2F] or null
  int M, C, F, act, row_tiles, col_tiles;
};

__device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + expf(-g)); }

__device__ __forceinline__ float gate(float g, int act) {
  switch (act) {
    case VG_GATE_SIGMOID: return sigmoid(g);
    case VG_GATE_RELU: return g > 0.f ? g : (g != g ? g : 0.f);
    case VG_GATE_GELU: return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
    default: return g * sigmoid(g);
  }
}
// act(g) and act'(g)
__device__ __forceinline__ void gate_both(float g, int act, float& a, float& d) {
  switch (act) {
    case VG_GATE_SIGMOID: {
      a = sigmoid(g);
      d = a * (1.f - a);
      break;
    }
    case VG_GATE_RELU: {
      a = g > 0.f ? g : (g != g ? g : 0.f);
      d = g > 0.f ? 1.f : 0.f;
      break;
    }
    case VG_GATE_GELU: {
      const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
      a = g * cdf;
      d = __builtin_fmaf(g * 0.3989422804014327f, expf(-0.5f * g * g), cdf);
      break;
    }
    default: {
      const float s = sigmoid(g);
      a = g * s;
      d = __builtin_fmaf(a, 1.f - s, s);
    }
  }
}

template <class T>
__device__ __forceinline__ float load1(const T* p) { return (float)*p; }

// BWD: the epilogue turns gh into [gg gu] instead of writing h
template <class T, int BM, int BN, int WM, int WN, bool ALIGNED, bool BWD>
__global__ void __launch_bounds__(64 * WM * WN, 1) gated_kernel(const GatedParams p) {
  using G = TokGemm<T, false, false, BM, BN, WM, WN, ALIGNED>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  T* smem = reinterpret_cast<T*>(smem_raw);
  const int id = tok_xcd_order(blockIdx.x, gridDim.x);
  const int mt = id / p.col_tiles, nt = id - mt * p.col_tiles;
  const int m0 = mt * BM, n0 = nt * BN;
  f32x16 acc[G::TM][G::TN];
  const TokOperand<T> A = {(const T*)p.x, p.C, p.M, 0}, B = {(const T*)p.w, p.C, 2 * p.F, p.F};
  G::run(A, B, m0, n0, 0, p.C, smem, acc);

  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int wm = wid / WN, wn = wid % WN;
  float sums[G::TN];
#pragma unroll
  for (int j = 0; j < G::TN; j += 2) {
    const int f = n0 / 2 + wn * G::TN * 16 + j * 16 + c;
    const bool in = f < p.F;
    const float bg = in && p.bias ? p.bias[f] : 0.f, bu = in && p.bias ? p.bias[p.F + f] : 0.f;
    float sg = 0.f, su = 0.f;
#pragma unroll
    for (int i = 0; i < G::TM; ++i) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int m = m0 + (wm * G::TM + i) * 32 + 8 * (e / 4) + 4 * h + e % 4;
        if (!in || m >= p.M) continue;
        const float g = acc[i][j][e] + bg, u = acc[i][j + 1][e] + bu;
        if constexpr (!BWD) {
          ((T*)p.h)[(size_t)m * p.F + f] = (T)(gate(g, p.act) * u);
          if (p.z) {
            p.z[(size_t)m * 2 * p.F + f] = g;
            p.z[(size_t)m * 2 * p.F + p.F + f] = u;
          }
        } else {
          float a, d;
          gate_both(g, p.act, a, d);
          const float gh = load1((const T*)p.gh + (size_t)m * p.F + f);
          const float gg = gh * u * d, gu = gh * a;
          sg += gg;
          su += gu;
          ((T*)p.gz)[(size_t)m * 2 * p.F + f] = (T)gg;
          ((T*)p.gz)[(size_t)m * 2 * p.F + p.F + f] = (T)gu;
        }
      }
    }
    sums[j] = sg;
    sums[j + 1] = su;
  }
  if constexpr (BWD) {
    if (!p.gb_part) return;
    // column sums of the block's rows: lane halves, then the row waves, in a fixed order
    float* red = reinterpret_cast<float*>(smem_raw);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < G::TN; ++j) {
      const float v = sums[j] + __shfl_xor(sums[j], 32, 64);
      if (h == 0) red[wm * BN + (wn * G::TN + j) * 32 + c] = v;
    }
    __syncthreads();
    for (int n = threadIdx.x; n < BN; n += G::NT) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WM; ++w) v += red[w * BN + n];
      const int f = n0 / 2 + (n >> 6) * 32 + (n & 31);
      if (f < p.F) p.gb_part[(size_t)mt * 2 * p.F + ((n >> 5) & 1) * p.F + f] = v;
    }
  }
}

// [gg gu] from z and gh, elementwise; a block covers 256 columns (4 a thread, V = 4; 1 a thread: 64) and kRowsBlock rows
constexpr int kRowsBlock = 64;
template <class T, int V>
__global__ void __launch_bounds__(256) gated_bwd_kernel(const GatedParams p) {
  const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6;
  const int f = (blockIdx.y * 64 + cl) * V;
  const int r0 = blockIdx.x * kRowsBlock, r1 = min(p.M, r0 + kRowsBlock);
  float sg[V], su[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sg[e] = su[e] = 0.f;
  if (f < p.F) {
    for (int m = r0 + rl; m < r1; m += 4) {
      const float* zg = p.z + (size_t)m * 2 * p.F + f;
      const T* gh = (const T*)p.gh + (size_t)m * p.F + f;
      float g[V], u[V], x[V], gg[V], gu[V];
      if constexpr (V == 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(zg), b = *reinterpret_cast<const f32x4*>(zg + p.F);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] = a[e];
          u[e] = b[e];
        }
        if constexpr (sizeof(T) == 4) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(gh);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = y[e];
        } else {
          const u32x2 y = *reinterpret_cast<const u32x2*>(gh);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = __builtin_bit_cast(float, (unsigned)(e % 2 ? y[e / 2] & 0xffff0000u : y[e / 2] << 16));
        }
      } else {
        g[0] = zg[0];
        u[0] = zg[p.F];
        x[0] = load1(gh);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float a, d;
        gate_both(g[e], p.act, a, d);
        gg[e] = x[e] * u[e] * d;
        gu[e] = x[e] * a;
        sg[e] += gg[e];
        su[e] += gu[e];
      }
      T* out = (T*)p.gz + (size_t)m * 2 * p.F + f;
      if constexpr (V == 4) {
        tok_store4(out, gg[0], gg[1], gg[2], gg[3]);
        tok_store4(out + p.F, gu[0], gu[1], gu[2], gu[3]);
      } else {
        out[0] = (T)gg[0];
        out[p.F] = (T)gu[0];
      }
    }
  }
  if (!p.gb_part) return;
  __shared__ float red[2][4][64 * V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    red[0][rl][cl * V + e] = sg[e];
    red[1][rl][cl * V + e] = su[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * V; i += 256) {
    const int which = i / (64 * V), col = i % (64 * V), ff = blockIdx.y * 64 * V + col;
    if (ff < p.F)
      p.gb_part[(size_t)blockIdx.x * 2 * p.F + which * p.F + ff] =
          (red[which][0][col] + red[which][1][col]) + (red[which][2][col] + red[which][3][col]);
  }
}

// ---- products of the backward pass -----------------------------------------------------------------------------
struct ProductParams {
  const void *a, *b;
  int64_t lda, ldb;
  int M, N, K;
  void* out;            // [M][N], or splits slabs of it (f32)
  int out_f32, col_tiles, tiles, splits, chunk;
};
template <class T, bool ARC, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ void __launch_bounds__(64 * WM * WN, 1) product_kernel(const ProductParams p) {
  using G = TokGemm<T, ARC, true, BM, BN, WM, WN, ALIGNED>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  const int id = tok_xcd_order(blockIdx.x, gridDim.x);
  const int sp = id / p.tiles, t = id - sp * p.tiles;
  const int mt = t / p.col_tiles, nt = t - mt * p.col_tiles;
  const int m0 = mt * BM, n0 = nt * BN, kbeg = sp * p.chunk, kend = min(p.K, kbeg + p.chunk);
  f32x16 acc[G::TM][G::TN];
  const TokOperand<T> A = {(const T*)p.a, p.lda, p.M, 0}, B = {(const T*)p.b, p.ldb, p.N, 0};
  G::run(A, B, m0, n0, kbeg, kend, reinterpret_cast<T*>(smem_raw), acc);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int wm = wid / WN, wn = wid % WN;
  const size_t slab = (size_t)sp * p.M * p.N;
#pragma unroll
  for (int j = 0; j < G::TN; ++j) {
    const int n = n0 + (wn * G::TN + j) * 32 + c;
    if (n >= p.N) continue;
#pragma unroll
    for (int i = 0; i < G::TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int m = m0 + (wm * G::TM + i) * 32 + 8 * (e / 4) + 4 * h + e % 4;
        if (m >= p.M) continue;
        if (p.out_f32)
          ((float*)p.out)[slab + (size_t)m * p.N + n] = acc[i][j][e];
        else
          ((__bf16*)p.out)[(size_t)m * p.N + n] = (__bf16)acc[i][j][e];
      }
  }
}
// out = sum of the slabs in order
template <class O>
__global__ void __launch_bounds__(256) slab_sum_kernel(const float* slabs, int splits, size_t n, O* out) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    float v = slabs[i];
    for (int s = 1; s < splits; ++s) v += slabs[(size_t)s * n + i];
    out[i] = (O)v;
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
constexpr int kBM = 128, kBN = 128;

template <class K>
int allow_lds(K kernel, int bytes) {
  if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
    (void)hipGetLastError();
    return vg_fail(VG_ERR_LAUNCH, "gated: %d bytes of LDS refused", bytes);
  }
  return VG_OK;
}

int check_sizes(int M, int C, int F, int act) {
  VG_REQUIRE(M >= 0 && C >= 1 && F >= 1, "gated: bad sizes rows=%d in=%d out=%d", M, C, F);
  VG_REQUIRE(act >= VG_GATE_SIGMOID && act <= VG_GATE_SILU, "gated: unknown activation %d", act);
  // tile counts and row indices of 31 bits (element offsets are 64-bit)
  VG_REQUIRE(M < (1 << 30) && C < (1 << 30) && F < (1 << 29) &&
                 ((long long)M / kBM + 1) * ((long long)F * 2 / kBN + 1) < (1ll << 31) && ((long long)M / kBM + 1) * ((long long)C / kBN + 1) < (1ll << 31) / 64 &&
                 ((long long)F * 2 / kBM + 1) * ((long long)C / kBN + 1) < (1ll << 31) / 64,
             "gated: too many tiles (rows=%d in=%d out=%d)", M, C, F);
  return VG_OK;
}

template <class T, bool BWD>
int launch_gated(GatedParams& p, hipStream_t st) {
  p.row_tiles = ceil_div(p.M, kBM);
  p.col_tiles = ceil_div(2ll * p.F, kBN);      // 64 output columns a tile
  const bool aligned = vg_aligned16(p.x) && vg_aligned16(p.w) && p.C % TokNum<T>::V == 0;
  const int grid = p.row_tiles * p.col_tiles;
  auto go = [&](auto kernel, int lds) {
    const int rc = allow_lds(kernel, lds);
    if (rc) return rc;
    kernel<<<grid, 256, lds, st>>>(p);
    return (int)VG_OK;
  };
  const int rc = aligned ? go(gated_kernel<T, kBM, kBN, 2, 2, true, BWD>, TokGemm<T, false, false, kBM, kBN, 2, 2, true>::LDS_BYTES)
                         : go(gated_kernel<T, kBM, kBN, 2, 2, false, BWD>, TokGemm<T, false, false, kBM, kBN, 2, 2, false>::LDS_BYTES);
  if (rc) return rc;
  VG_CHECK_LAUNCH("gated");
  return VG_OK;
}

template <class T>
int gated_fwd(int M, int C, int F, const void* x, const void* w, const float* bias, void* h, float* z, int act, void* stream) {
  const int rc = check_sizes(M, C, F, act);
  if (rc || M == 0) return rc;
  VG_REQUIRE(x && w && h, "gated: null tensor");
  GatedParams p = {};
  p.x = x;
  p.w = w;
  p.bias = bias;
  p.h = h;
  p.z = z;
  p.M = M;
  p.C = C;
  p.F = F;
  p.act = act;
  return launch_gated<T, false>(p, (hipStream_t)stream);
}

template <class T>
int gated_bwd_z(int M, int F, const float* z, const void* gh, void* gz, float* gb_part, int act, void* stream) {
  const int rc = check_sizes(M, 1, F, act);
  if (rc || M == 0) return rc;
  VG_REQUIRE(z && gh && gz, "gated backward: null tensor");
  VG_REQUIRE(ceil_div(F, 64) <= 65535, "gated backward: %d columns are too many", F);
  GatedParams p = {};
  p.z = const_cast<float*>(z);
  p.gh = gh;
  p.gz = gz;
  p.gb_part = gb_part;
  p.M = M;
  p.F = F;
  p.act = act;
  hipStream_t st = (hipStream_t)stream;
  const bool wide = F % 4 == 0 && vg_aligned16(z) && vg_aligned16(gh) && vg_aligned16(gz);
  const dim3 grid(ceil_div(M, kRowsBlock), ceil_div(F, wide ? 256 : 64));
  if (wide)
    gated_bwd_kernel<T, 4><<<grid, 256, 0, st>>>(p);
  else
    gated_bwd_kernel<T, 1><<<grid, 256, 0, st>>>(p);
  VG_CHECK_LAUNCH("gated backward");
  return VG_OK;
}

// A product with fewer tiles than compute units is split along k towards one block for each, no split under 4 k-steps.
int product_splits(int M, int N, int K) {
  const long long tiles = (long long)ceil_div(M, kBM) * ceil_div(N, kBN);
  if (tiles >= 192) return 1;
  long long s = 256 / tiles, most = K / 256;
  if (s > most) s = most;
  return s < 1 ? 1 : (int)s;
}
size_t product_bytes(int M, int N, int K) {
  const int s = product_splits(M, N, K);
  return s == 1 ? 0 : (size_t)s * M * N * 4;
}

template <class T, bool ARC>
int product(const void* a, int64_t lda, const void* b, int64_t ldb, int M, int N, int K, void* out, int out_f32, void* ws, size_t ws_bytes,
            hipStream_t st) {
  const size_t need = product_bytes(M, N, K);
  if (need && (!ws || ws_bytes < need)) return vg_fail(VG_ERR_WORKSPACE, "gated backward: workspace of %zu bytes, %zu are needed", ws_bytes, need);
  ProductParams p = {};
  p.a = a;
  p.b = b;
  p.lda = lda;
  p.ldb = ldb;
  p.M = M;
  p.N = N;
  p.K = K;
  p.splits = product_splits(M, N, K);
  p.chunk = ((K + p.splits - 1) / p.splits + 63) & ~63;
  p.out = p.splits > 1 ? ws : out;
  p.out_f32 = p.splits > 1 ? 1 : out_f32;
  p.col_tiles = ceil_div(N, kBN);
  p.tiles = ceil_div(M, kBM) * p.col_tiles;
  const bool aligned = vg_aligned16(a) && vg_aligned16(b) && lda % TokNum<T>::V == 0 && ldb % TokNum<T>::V == 0;
  const int grid = p.tiles * p.splits;
  auto go = [&](auto kernel, int lds) {
    const int rc = allow_lds(kernel, lds);
    if (rc) return rc;
    kernel<<<grid, 256, lds, st>>>(p);
    return (int)VG_OK;
  };
  const int rc = aligned ? go(product_kernel<T, ARC, kBM, kBN, 2, 2, true>, TokGemm<T, ARC, true, kBM, kBN, 2, 2, true>::LDS_BYTES)
                         : go(product_kernel<T, ARC, kBM, kBN, 2, 2, false>, TokGemm<T, ARC, true, kBM, kBN, 2, 2, false>::LDS_BYTES);
  if (rc) return rc;
  if (p.splits > 1) {
    const size_t n = (size_t)M * N;
    if (out_f32)
      slab_sum_kernel<float><<<vg_stream_grid(n, 256), 256, 0, st>>>((const float*)ws, p.splits, n, (float*)out);
    else
      slab_sum_kernel<__bf16><<<vg_stream_grid(n, 256), 256, 0, st>>>((const float*)ws, p.splits, n, (__bf16*)out);
  }
  VG_CHECK_LAUNCH("gated backward product");
  return VG_OK;
}

template <class T>
int gated_gx(int M, int C, int F, const void* gz, const void* w, void* gx, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_sizes(M, C, F, VG_GATE_SILU);
  if (rc || M == 0) return rc;
  VG_REQUIRE(gz && w && gx, "gated backward: null tensor");
  return product<T, false>(gz, 2 * (int64_t)F, w, C, M, C, 2 * F, gx, sizeof(T) == 4, ws, ws_bytes, (hipStream_t)stream);
}
template <class T>
int gated_gw(int M, int C, int F, const void* gz, const void* x, void* gw, int gw_f32, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_sizes(M, C, F, VG_GATE_SILU);
  if (rc) return rc;
  VG_REQUIRE(gw && (M == 0 || (gz && x)), "gated backward: null tensor");
  return product<T, true>(gz, 2 * (int64_t)F, x, C, 2 * F, C, M, gw, gw_f32, ws, ws_bytes, (hipStream_t)stream);
}

}  // namespace

extern "C" {

int vg_gated_linear_fwd(int M, int C, int F, const float* x, const float* w, const float* bias, float* h, float* z, int act, void* stream) {
  return gated_fwd<float>(M, C, F, x, w, bias, h, z, act, stream);
}
int vg_gated_linear_fwd_h(int M, int C, int F, const void* x, const void* w, const float* bias, void* h, float* z, int act, void* stream) {
  return gated_fwd<__bf16>(M, C, F, x, w, bias, h, z, act, stream);
}
int vg_gated_linear_bwd(int M, int F, const float* z, const float* gh, float* gz, float* gb_part, int act, void* stream) {
  return gated_bwd_z<float>(M, F, z, gh, gz, gb_part, act, stream);
}
int vg_gated_linear_bwd_h(int M, int F, const float* z, const void* gh, void* gz, float* gb_part, int act, void* stream) {
  return gated_bwd_z<__bf16>(M, F, z, gh, gz, gb_part, act, stream);
}
int vg_gated_linear_partial_rows(int M, int recompute) { return M < 1 ? 0 : ceil_div(M, recompute ? kBM : kRowsBlock); }
int vg_gated_linear_recomputes_h(int M, int C, int F) { return C <= 1024; }
int vg_gated_linear_rebwd_h(int M, int C, int F, const void* x, const void* w, const float* bias, const void* gh, void* gz, float* gb_part,
                            int act, void* stream) {
  const int rc = check_sizes(M, C, F, act);
  if (rc || M == 0) return rc;
  VG_REQUIRE(x && w && gh && gz, "gated backward: null tensor");
  GatedParams p = {};
  p.x = x;
  p.w = w;
  p.bias = bias;
  p.gh = gh;
  p.gz = gz;
  p.gb_part = gb_part;
  p.M = M;
  p.C = C;
  p.F = F;
  p.act = act;
  return launch_gated<__bf16, true>(p, (hipStream_t)stream);
}
size_t vg_gated_linear_gx_workspace_bytes(int M, int C, int F) {
  return check_sizes(M, C, F, VG_GATE_SILU) || M == 0 ? 0 : product_bytes(M, C, 2 * F);
}
size_t vg_gated_linear_gw_workspace_bytes(int M, int C, int F) {
  return check_sizes(M, C, F, VG_GATE_SILU) || M == 0 ? 0 : product_bytes(2 * F, C, M);
}
int vg_gated_linear_gx(int M, int C, int F, const float* gz, const float* w, float* gx, void* workspace, size_t workspace_bytes,
                       void* stream) {
  return gated_gx<float>(M, C, F, gz, w, gx, workspace, workspace_bytes, stream);
}
int vg_gated_linear_gx_h(int M, int C, int F, const void* gz, const void* w, void* gx, void* workspace, size_t workspace_bytes,
                         void* stream) {
  return gated_gx<__bf16>(M, C, F, gz, w, gx, workspace, workspace_bytes, stream);
}
int vg_gated_linear_gw(int M, int C, int F, const float* gz, const float* x, float* gw, void* workspace, size_t workspace_bytes,
                       void* stream) {
  return gated_gw<float>(M, C, F, gz, x, gw, 1, workspace, workspace_bytes, stream);
}
int vg_gated_linear_gw_h(int M, int C, int F, const void* gz, const void* x, void* gw, int gw_f32, void* workspace, size_t workspace_bytes,
                         void* stream) {
  return gated_gw<__bf16>(M, C, F, gz, x, gw, gw_f32, workspace, workspace_bytes, stream);
}

}  // extern "C"
