// Gated linear layer h = act(g) * u, g = x Wg^T + bg, u = x Wu^T + bu, both projections, the activation and the product
// in one kernel, with its backward pass.
//
//   gg = gh u act'(g)     gu = gh act(g)     gx = [gg gu] [Wg; Wu]     gW = [gg gu]^T x     gb = column sums of [gg gu]
//
// The weights lie as one [2F][C] matrix (gate rows first). They are the rows of the product and x its columns; a block's
// weight tile takes 32 gate rows, the matching 32 value rows, the next 32 gate rows, ...: gate and value of one output
// element end in the same lane's accumulators, sixteen neighbouring elements of one row of h a lane, so the epilogue
// needs no other lane's values. Bound by the matrix cores (4 M C F flops forward, twice that backward) and, behind them, by
// what is written. Measured in a loop of calls, bf16, 16384 x 1024 x 4096: forward 441 us where the pre-activations are kept
// (671 MB written), 308 where not (134 MB); backward 679, of which 187 are the elementwise pass with the bias gradient (939 MB)
// and 237 and 251 the products for the inputs' and the weights' gradients (1.16 and 1.10 PFLOP/s; library products of the same
// operand orders take 218 and 255). f32, 4096 x 512 x 1408: forward 108 us, backward 236 (library products: 108, 98 and 101).
// Launches under a profiler, with pauses between them, take up to a quarter longer.
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
  void* gz;              // [M][2F], two of them where `terms` is 2: the rounded gradient and what the rounding left
  float* gb_part;        // [row tiles][2F] or null
  int M, C, F, act, row_tiles, col_tiles, terms;
};

// The gates. f32 takes the library's exponential and error function. bf16 results keep 8 bits: the hardware's exponential
// and reciprocal (one unit in the last place of f32) and, for the normal distribution's tail, formula 7.1.26 of
// Abramowitz and Stegun, erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + p x), off by at most 1.5e-7 - the library's
// error function took longer than the products of a tile. Far in the tail that is no longer small beside the value: off by
// 0.05 % of it at g = -4, 0.3 % at -5.7, 1 % at -8, where gelu itself is -1e-4, -3e-8 and -5e-15 (half a step of bf16: 0.4 %).
template <bool FAST>
__device__ __forceinline__ float sigmoid(float g) {
  if constexpr (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g));
  return 1.f / (1.f + expf(-g));
}
// distribution and density of the standard normal
template <bool FAST>
__device__ __forceinline__ void normal(float g, float& cdf, float& pdf) {
  if constexpr (FAST) {
    const float e = __builtin_amdgcn_exp2f(-0.72134752044448170f * g * g);      // exp(-g^2 / 2)
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678118654752f, fabsf(g), 1.f));
    float q = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
    q = __builtin_fmaf(t, q, 1.421413741f);
    q = __builtin_fmaf(t, q, -0.284496736f);
    q = __builtin_fmaf(t, q, 0.254829592f);
    const float tail = 0.5f * t * q * e;
    cdf = g < 0.f ? tail : 1.f - tail;
    pdf = 0.3989422804014327f * e;
  } else {
    cdf = 0.5f * erfcf(-0.70710678118654752f * g);
    pdf = 0.3989422804014327f * expf(-0.5f * g * g);
  }
}
// act(g) and act'(g) (the caller's compiler drops what it does not use)
template <bool FAST>
__device__ __forceinline__ void gate_both(float g, int act, float& a, float& d) {
  switch (act) {
    case VG_GATE_SIGMOID: {
      a = sigmoid<FAST>(g);
      d = a * (1.f - a);
      break;
    }
    case VG_GATE_RELU: {
      a = g > 0.f ? g : (g != g ? g : 0.f);
      d = g > 0.f ? 1.f : 0.f;
      break;
    }
    case VG_GATE_GELU: {
      float pdf;
      normal<FAST>(g, d, pdf);
      a = g * d;
      d = __builtin_fmaf(g, pdf, d);
      break;
    }
    default: {
      const float s = sigmoid<FAST>(g);
      a = g * s;
      d = __builtin_fmaf(a, 1.f - s, s);
    }
  }
}

template <class T>
__device__ __forceinline__ float load1(const T* p) { return (float)*p; }

// Sixteen neighbouring elements, n of them inside the row; any alignment of an element.
template <class T>
__device__ __forceinline__ void load16(const T* p, int n, float (&v)[16]) {
  constexpr int V = TokNum<T>::V;
  if (n >= 16) {
#pragma unroll
    for (int i = 0; i < 16 / V; ++i) {
      u32x4 raw;
      __builtin_memcpy(&raw, p + i * V, 16);
      float f[V];
      tok_widen(raw, f);
#pragma unroll
      for (int e = 0; e < V; ++e) v[i * V + e] = f[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = e < n ? (float)p[e] : 0.f;
  }
}
// A 32 x 32 tile of a result, `rows` x `cols` of it inside. A lane holds 16 neighbouring columns of row lane % 32: stored
// from there, every lane of a 16-byte store would be in a line of its own. The wave turns the tile in LDS (its own kTurn
// floats) and stores whole runs of 128 bytes (f32) or 64 (bf16): 16384 x 1024 x 4096 with z (671 MB of results) 565 -> 490
// us, 4096 x 512 x 1408 in f32 132 -> 121.
constexpr int kTurnLd = 36, kTurn = 32 * kTurnLd;
template <class O>
__device__ __forceinline__ void store_tile(float* mine, O* out, size_t ld, int rows, int cols, const float (&v)[16], int lane) {
  constexpr int V = TokNum<O>::V, LANES = 32 / V;      // lanes of a row
#pragma unroll
  for (int e = 0; e < 16; e += 4)
    *reinterpret_cast<f32x4*>(mine + (lane & 31) * kTurnLd + 16 * (lane >> 5) + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const int r0 = lane / LANES, col = lane % LANES * V;
#pragma unroll
  for (int r = r0; r < 32 + r0; r += 64 / LANES) {
    float f[V];
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(mine + r * kTurnLd + col + e);
#pragma unroll
      for (int k = 0; k < 4; ++k) f[e + k] = a[k];
    }
    O* to = out + (size_t)r * ld + col;
    if (r < rows) {
      if (col + V <= cols) {
        const u32x4 raw = tok_narrow(f);
        __builtin_memcpy(to, &raw, 16);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (col + e < cols) to[e] = (O)f[e];
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Tile order: runs of kGroup row tiles walk the column tiles together, so that the tiles in flight on an XCD share rows of
// x and of the weights in its L2 (32 tiles at once: 8 + 4 operand tiles instead of 1 + 32).
constexpr int kGroup = 8;
__device__ __forceinline__ void tile_of(int id, int row_tiles, int col_tiles, int& mt, int& nt) {
  const int run = kGroup * col_tiles, first = id / run * kGroup, rest = id % run, wide = min(kGroup, row_tiles - first);
  mt = first + rest % wide;
  nt = rest / wide;
}

// BWD: the epilogue turns gh into [gg gu] instead of writing h. WM waves along the weights' rows, WN along the rows of x.
template <class T, int BF, int BM, int WM, int WN, bool BWD>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN / 4) gated_kernel(const GatedParams p) {
  using G = TokGemm<T, false, false, BF, BM, WM, WN>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  int mt, nt;
  tile_of(tok_xcd_order(blockIdx.x, gridDim.x), p.row_tiles, p.col_tiles, mt, nt);
  const int m0 = mt * BM, n0 = nt * BF;
  f32x16 acc[G::TM][G::TN];
  const TokOperand<T> A = {(const T*)p.w, p.C, 2 * p.F, p.F}, B = {(const T*)p.x, p.C, p.M, 0};
  G::run(A, B, n0, m0, 0, p.C, reinterpret_cast<T*>(smem_raw), acc);

  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int wm = wid / WN, wn = wid % WN;
  constexpr int LDR = 68;                                       // a lane column of partial sums, padded
  float* red = reinterpret_cast<float*>(smem_raw);              // [wave][32][LDR], then [WN][BF] sums behind it
  float* total = red + WM * WN * 32 * LDR;
  float* mine = red + wid * 32 * LDR;                           // the wave's own space: no barrier needed
  static_assert(kTurn <= 32 * LDR, "a tile to be turned fits it");
  static_assert((WM * WN * 32 * LDR + WN * BF) * 4 <= G::LDS_BYTES, "the sums fit the tiles' space");
#pragma unroll
  for (int i = 0; i < G::TM; i += 2) {
    const int f = n0 / 2 + (wm * G::TM + i) * 16 + 16 * h, left = p.F - f;
    float bg[16], bu[16], sg[16], su[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) sg[e] = su[e] = bg[e] = bu[e] = 0.f;
    if (p.bias) {
      load16(p.bias + f, left, bg);
      load16(p.bias + p.F + f, left, bu);
    }
#pragma unroll
    for (int j = 0; j < G::TN; ++j) {
      const int mt0 = m0 + (wn * G::TN + j) * 32, m = mt0 + c, ft = f - 16 * h, rows = p.M - mt0, cols = p.F - ft;
      if (rows <= 0 || cols <= 0) continue;      // uniform
      const bool ok = m < p.M && left > 0;
      float g[16], u[16], gg[16], gu[16];
      [[maybe_unused]] float x[16];
      const size_t at = (size_t)mt0 * p.F + ft, at2 = (size_t)mt0 * 2 * p.F + ft;
      if constexpr (BWD) load16((const T*)p.gh + (size_t)m * p.F + f, ok ? left : 0, x);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        g[e] = acc[i][j][e] + bg[e];
        u[e] = acc[i + 1][j][e] + bu[e];
        float a, d;
        gate_both<sizeof(T) == 2>(g[e], p.act, a, d);
        if constexpr (BWD) {
          gg[e] = x[e] * u[e] * d;
          gu[e] = x[e] * a;
          if (ok) {
            sg[e] += gg[e];
            su[e] += gu[e];
          }
        } else {
          gg[e] = a * u[e];
        }
      }
      if constexpr (BWD) {
        store_tile(mine, (T*)p.gz + at2, 2 * p.F, rows, cols, gg, lane);
        store_tile(mine, (T*)p.gz + at2 + p.F, 2 * p.F, rows, cols, gu, lane);
        if (sizeof(T) == 2 && p.terms == 2) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            gg[e] -= (float)(T)gg[e];
            gu[e] -= (float)(T)gu[e];
          }
          T* low = (T*)p.gz + (size_t)p.M * 2 * p.F + at2;
          store_tile(mine, low, 2 * p.F, rows, cols, gg, lane);
          store_tile(mine, low + p.F, 2 * p.F, rows, cols, gu, lane);
        }
      } else {
        store_tile(mine, (T*)p.h + at, p.F, rows, cols, gg, lane);
        if (p.z) {
          store_tile(mine, p.z + at2, 2 * p.F, rows, cols, g, lane);
          store_tile(mine, p.z + at2 + p.F, 2 * p.F, rows, cols, u, lane);
        }
      }
    }
    if constexpr (BWD) {
      if (p.gb_part) {       // column sums: the wave's 32 rows of x in a fixed order
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          *reinterpret_cast<f32x4*>(mine + c * LDR + 32 * h + e) = f32x4{sg[e], sg[e + 1], sg[e + 2], sg[e + 3]};
          *reinterpret_cast<f32x4*>(mine + c * LDR + 32 * h + 16 + e) = f32x4{su[e], su[e + 1], su[e + 2], su[e + 3]};
        }
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        float v = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) v += mine[r * LDR + lane];
        total[wn * BF + (wm * G::TM + i) * 32 + lane] = v;      // lane = 32 h + 16 (value) + element
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
  }
  if constexpr (BWD) {
    if (!p.gb_part) return;
    __syncthreads();
    for (int n = threadIdx.x; n < BF; n += G::NT) {             // n = 64 block + 32 h + 16 (value) + element
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WN; ++w) v += total[w * BF + n];
      const int f = n0 / 2 + (n >> 6) * 32 + ((n >> 5) & 1) * 16 + (n & 15);
      if (f < p.F) p.gb_part[(size_t)mt * 2 * p.F + ((n >> 4) & 1) * p.F + f] = v;
    }
  }
}

// Few rows of x (up to 64): all there is to read is the weights, once. A block takes 16 output columns, i.e. 16 gate and 16
// value rows as the 32 rows of a product tile whose columns are the rows of x, and its waves split the features. Weights
// and x go from memory into the operand registers: a lane reads 128 bytes of one row (the order of k inside a product does
// not matter, so its half of a block of k is contiguous), eight 16-byte loads in flight. The partial products of the waves
// meet in LDS. Tiles of rows 0..15 and 16..31 put gate and value of an element in one lane: registers i and i + 8.
constexpr int kFewRows = 64, kFewWaves = 8;
template <class T, int NB>
__global__ void __launch_bounds__(64 * kFewWaves) gated_few_kernel(const GatedParams p) {
  constexpr int V = TokNum<T>::V, HALF = 8 * V, KB = 2 * HALF;     // features a lane half, a wave takes at once
  using Frag = std::conditional_t<sizeof(T) == 2, bf16x8, f32x4>;
  __shared__ float red[kFewWaves][NB][16][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int f0 = blockIdx.x * 16;
  const int fr = min(f0 + (c & 15), p.F - 1);                      // clamped: what it gives is not stored
  const T* w = (const T*)p.w + (size_t)(fr + (c >> 4) * p.F) * p.C + h * HALF;
  const T* x[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) x[n] = (const T*)p.x + (size_t)min(n * 32 + c, p.M - 1) * p.C + h * HALF;
  f32x16 acc[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[n][e] = 0.f;
  using S = TokStage<T, false, 128, sizeof(T) == 2 ? 64 : 32, 256>;      // (its loads)
  for (int k = wid * KB; k < p.C; k += kFewWaves * KB) {
    u32x4 a[8], b[NB][8];
    if (k + KB <= p.C) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = S::whole(reinterpret_cast<const char*>(w + k + i * V));
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) b[n][i] = S::whole(reinterpret_cast<const char*>(x[n] + k + i * V));
    } else {
      auto first = [&](const T* at, int left) {
        const char* c = reinterpret_cast<const char*>(at);
        return p.C >= V ? S::first(c, left) : S::part(c, left);
      };
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int left = p.C - k - h * HALF - i * V;
        a[i] = first(w + k + i * V, left);
#pragma unroll
        for (int n = 0; n < NB; ++n) b[n][i] = first(x[n] + k + i * V, left);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < tok_parts<T>(); ++e)
          acc[n] = tok_mma(__builtin_bit_cast(Frag, a[i]), __builtin_bit_cast(Frag, b[n][i]), acc[n], e);
  }
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 16; ++e) red[wid][n][e][lane] = acc[n][e];
  __syncthreads();
  for (int id = threadIdx.x; id < NB * 8 * 64; id += 64 * kFewWaves) {
    const int l = id & 63, i = (id >> 6) & 7, n = id >> 9;
    const int f = f0 + 8 * (i / 4) + 4 * (l >> 5) + i % 4, m = n * 32 + (l & 31);
    if (f >= p.F || m >= p.M) continue;
    float g = p.bias ? p.bias[f] : 0.f, u = p.bias ? p.bias[p.F + f] : 0.f;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) {
      g += red[v][n][i][l];
      u += red[v][n][i + 8][l];
    }
    float a, d;
    gate_both<sizeof(T) == 2>(g, p.act, a, d);
    ((T*)p.h)[(size_t)m * p.F + f] = (T)(a * u);
    if (p.z) {
      p.z[(size_t)m * 2 * p.F + f] = g;
      p.z[(size_t)m * 2 * p.F + p.F + f] = u;
    }
  }
}

// [gg gu] from z and gh, elementwise: V neighbouring columns a thread (one 16-byte vector of T, or 1 where the rows do not
// start on 16-byte borders), 64 V columns and kRowsBlock rows a block. Bound by HBM: 8 + 3 sizeof(T) bytes an element.
// STREAM reads and writes past the caches, for calls whose bytes fill the 256 MB last-level cache anyhow: 16384 rows of 4096
// features in bf16 (939 MB) 238 -> 190 us, the two products that read gz unchanged. Below that the products find gz in the
// cache: 4096 rows of 704 features in f32 (58 MB) take 21 us so, 27 past the caches.
constexpr int kRowsBlock = 64;
constexpr size_t kStreamBytes = (size_t)256 << 20;
template <bool STREAM, class A>
__device__ __forceinline__ A get(const void* at) {
  if constexpr (STREAM)
    return __builtin_nontemporal_load(static_cast<const A*>(at));
  else
    return *static_cast<const A*>(at);
}
template <bool STREAM>
__device__ __forceinline__ void put(void* at, u32x4 v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, static_cast<u32x4*>(at));
  else
    *static_cast<u32x4*>(at) = v;
}
template <class T, int V, bool STREAM>
__global__ void __launch_bounds__(256) gated_bwd_kernel(const GatedParams p) {
  const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6;
  const int f = (blockIdx.y * 64 + cl) * V;
  const int r0 = blockIdx.x * kRowsBlock, r1 = min(p.M, r0 + kRowsBlock);
  float sg[V], su[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sg[e] = su[e] = 0.f;
  if (f < p.F) {
#pragma unroll 2
    for (int m = r0 + rl; m < r1; m += 4) {
      const float* zg = p.z + (size_t)m * 2 * p.F + f;
      const T* gh = (const T*)p.gh + (size_t)m * p.F + f;
      float g[V], u[V], x[V], gg[V], gu[V];
      if constexpr (V > 1) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          const f32x4 a = get<STREAM, f32x4>(zg + e), b = get<STREAM, f32x4>(zg + p.F + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            g[e + k] = a[k];
            u[e + k] = b[k];
          }
        }
        tok_widen(get<STREAM, u32x4>(gh), x);
      } else {
        g[0] = zg[0];
        u[0] = zg[p.F];
        x[0] = load1(gh);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float a, d;
        gate_both<sizeof(T) == 2>(g[e], p.act, a, d);
        gg[e] = x[e] * u[e] * d;
        gu[e] = x[e] * a;
        sg[e] += gg[e];
        su[e] += gu[e];
      }
      T* out = (T*)p.gz + (size_t)m * 2 * p.F + f;
      for (int t = 0; t < p.terms; ++t) {
        if constexpr (V > 1) {
          put<STREAM>(out, tok_narrow(gg));
          put<STREAM>(out + p.F, tok_narrow(gu));
        } else {
          out[0] = (T)gg[0];
          out[p.F] = (T)gu[0];
        }
        out += (size_t)p.M * 2 * p.F;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          gg[e] -= (float)(T)gg[e];
          gu[e] -= (float)(T)gu[e];
        }
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
  int64_t a_term;       // elements from the first term of a to the second
  int out_f32, col_tiles, tiles, splits, chunk;     // splits: of each term
};
template <class T, bool ARC, int BMN, int WM, int WN>
__device__ __forceinline__ void product_tile(const ProductParams& p, int id, T* smem) {
  using G = TokGemm<T, ARC, true, BMN, BMN, WM, WN>;
  constexpr int BM = BMN, BN = BMN;
  const int slab_id = id / p.tiles, t = id - slab_id * p.tiles, term = slab_id / p.splits, sp = slab_id - term * p.splits;
  const int mt = t / p.col_tiles, nt = t - mt * p.col_tiles;
  const int m0 = mt * BM, n0 = nt * BN, kbeg = sp * p.chunk, kend = min(p.K, kbeg + p.chunk);
  f32x16 acc[G::TM][G::TN];
  const TokOperand<T> A = {(const T*)p.a + term * p.a_term, p.lda, p.M, 0}, B = {(const T*)p.b, p.ldb, p.N, 0};
  G::run(A, B, m0, n0, kbeg, kend, smem, acc);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int wm = wid / WN, wn = wid % WN;
  const size_t slab = (size_t)slab_id * p.M * p.N;
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
// gx = [gg gu] w (the first blocks) and gw = [gg gu]^T x in one launch: neither waits for the other's last blocks (1001 rows,
// 333 x 777, bf16: 18 us, one after the other 17 + 17)
template <class T, int BMN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN / 4) products_kernel(const ProductParams gx, const ProductParams gw, int gx_blocks) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  const int id = (int)blockIdx.x - gx_blocks;
  if (id < 0)
    product_tile<T, false, BMN, WM, WN>(gx, tok_xcd_order(blockIdx.x, gx_blocks), reinterpret_cast<T*>(smem_raw));
  else
    product_tile<T, true, BMN, WM, WN>(gw, tok_xcd_order(id, gridDim.x - gx_blocks), reinterpret_cast<T*>(smem_raw));
}

// What is left to add up, in one launch: the slabs of gx and gw, elementwise and in order, and gb, the partial column sums'
// rows in a fixed order (32 columns and 32 row lanes a block).
struct SlabSum {
  const float* slabs;
  void* out;
  size_t n;
  int splits, out_f32, blocks;
};
__global__ void __launch_bounds__(1024) gated_sums_kernel(const SlabSum gx, const SlabSum gw, const float* part, int rows, int n, float* gb) {
  const int id = blockIdx.x;
  if (id < gx.blocks + gw.blocks) {
    const SlabSum& p = id < gx.blocks ? gx : gw;
    for (size_t i = (size_t)(id < gx.blocks ? id : id - gx.blocks) * 1024 + threadIdx.x; i < p.n; i += (size_t)p.blocks * 1024) {
      float v = p.slabs[i];
      for (int s = 1; s < p.splits; ++s) v += p.slabs[(size_t)s * p.n + i];
      if (p.out_f32)
        ((float*)p.out)[i] = v;
      else
        ((__bf16*)p.out)[i] = (__bf16)v;
    }
    return;
  }
  __shared__ float red[32][33];
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5, i = (id - gx.blocks - gw.blocks) * 32 + col;
  float v = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int r = row; r < rows; r += 32) v += part[(size_t)r * n + i];
  }
  red[row][col] = v;
  __syncthreads();
  if (row == 0 && i < n) {
#pragma unroll
    for (int r = 1; r < 32; ++r) v += red[r][col];
    gb[i] = v;
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

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
  // tile counts and row indices of 31 bits; byte offsets inside a tile (256 rows of C, 64 of 2F) of 32, all others of 64
  VG_REQUIRE(M < (1 << 30) && C < (1 << 21) && F < (1 << 20) &&
                 ((long long)M / 128 + 1) * ((long long)F * 2 / 128 + 1) < (1ll << 31) && ((long long)M / 128 + 1) * ((long long)C / 128 + 1) < (1ll << 31) / 64 &&
                 ((long long)F * 2 / 128 + 1) * ((long long)C / 128 + 1) < (1ll << 31) / 64,
             "gated: too many tiles (rows=%d in=%d out=%d)", M, C, F);
  return VG_OK;
}

// Products are cut into 256 x 256 tiles (bf16: eight waves of 128 x 64, one block a CU) or 128 x 128 (two blocks a CU). The
// large tile reads its operands half as often from the caches and takes 0.65 of the time of four small ones (16384 x 1024
// x 8192: 284 us against 416); the small one wins where too few large ones are there for 256 compute units. f32 products
// are bound by the matrix cores with either and take the small one, by eight waves of 64 x 32 (4096 x 512 x 2816: input
// gradient 110 us, with four waves of 64 x 64 121).
constexpr double kLarge = 4 * 0.65;
template <class T>
bool large_tiles(long long M, long long N) {
  const long long large = (long long)ceil_div(M, 256) * ceil_div(N, 256), small = (long long)ceil_div(M, 128) * ceil_div(N, 128);
  return sizeof(T) == 2 && ceil_div(large, 256) * kLarge < ceil_div(small, 256);
}
template <class T, int BMN, int WM, int WN, bool BWD>
int launch_gated_tiles(GatedParams& p, hipStream_t st) {
  p.row_tiles = ceil_div(p.M, BMN);
  p.col_tiles = ceil_div(2ll * p.F, BMN);      // BMN / 2 output columns a tile
  using G = TokGemm<T, false, false, BMN, BMN, WM, WN>;
  auto kernel = gated_kernel<T, BMN, BMN, WM, WN, BWD>;
  const int rc = allow_lds(kernel, G::LDS_BYTES);
  if (rc) return rc;
  kernel<<<p.row_tiles * p.col_tiles, G::NT, G::LDS_BYTES, st>>>(p);
  VG_CHECK_LAUNCH("gated");
  return VG_OK;
}
template <class T, bool BWD>
int launch_gated(GatedParams& p, hipStream_t st) {
  if constexpr (!BWD) {
    if (p.M <= kFewRows) {
      if (p.M <= 32)
        gated_few_kernel<T, 1><<<ceil_div(p.F, 16), 64 * kFewWaves, 0, st>>>(p);
      else
        gated_few_kernel<T, 2><<<ceil_div(p.F, 16), 64 * kFewWaves, 0, st>>>(p);
      VG_CHECK_LAUNCH("gated");
      return VG_OK;
    }
  }
  if constexpr (sizeof(T) == 2)
    if (large_tiles<T>(p.M, 2ll * p.F)) return launch_gated_tiles<T, 256, 2, 4, BWD>(p, st);
  return launch_gated_tiles<T, 128, 2, sizeof(T) == 4 ? 4 : 2, BWD>(p, st);
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

struct ProductPlan {
  int tile, splits, chunk;
};
// A product with few tiles is split along k, each split into a slab of its own (f32), summed in order. With n blocks on
// the busiest compute unit the time goes as n (K / splits + 128): 128 k for a block's start, its stores and its share of
// the slab sum. No split under 128 k (a block of few k is bound by the latency of its loads, one k-step after the other:
// 1554 x 333 x 1001 in splits of 334 k 22 us, of 167 17).
template <class T>
ProductPlan product_plan(int M, int N, int K) {
  ProductPlan best = {128, 1, K};
  double least = 1e30;
  for (int tile = 128; tile <= (sizeof(T) == 2 ? 256 : 128); tile *= 2) {
    const long long tiles = (long long)ceil_div(M, tile) * ceil_div(N, tile);
    if (tile == 256 && (M < 256 || N < 256)) break;
    for (int s = 1; s <= 64 && (s == 1 || K / s >= 128); ++s) {
      const long long n = (tiles * s + 255) / 256;
      const double t = (double)n * ((double)K / s + 128) * (tile == 256 ? kLarge : 1);
      if (t < least * (s > 1 ? 0.97 : 1.0)) {
        least = t;
        best = {tile, s, K};
      }
    }
  }
  best.chunk = ((K + best.splits - 1) / best.splits + 63) & ~63;
  return best;
}
template <class T>
size_t product_bytes(int M, int N, int K, int terms) {
  const int s = product_plan<T>(M, N, K).splits * terms;
  return s == 1 ? 0 : (size_t)s * M * N * 4;
}

// One of the two products: how it is cut, and its kernel's arguments.
struct Product {
  ProductPlan plan;
  ProductParams p;
  SlabSum sum;
  int blocks;
};
template <class T>
Product product(const void* a, int64_t lda, int terms, int64_t a_term, const void* b, int64_t ldb, int M, int N, int K, void* out, int out_f32,
                void* slabs) {
  Product q = {product_plan<T>(M, N, K)};
  const int count = q.plan.splits * terms;
  q.p.a = a;
  q.p.b = b;
  q.p.lda = lda;
  q.p.ldb = ldb;
  q.p.M = M;
  q.p.N = N;
  q.p.K = K;
  q.p.splits = q.plan.splits;
  q.p.chunk = q.plan.chunk;
  q.p.a_term = a_term;
  q.p.col_tiles = ceil_div(N, q.plan.tile);
  q.p.tiles = ceil_div(M, q.plan.tile) * q.p.col_tiles;
  q.p.out = count > 1 ? slabs : out;
  q.p.out_f32 = count > 1 ? 1 : out_f32;
  q.blocks = q.p.tiles * count;
  if (count > 1) q.sum = {(const float*)slabs, out, (size_t)M * N, count, out_f32, vg_stream_grid((size_t)M * N, 1024)};
  return q;
}
template <class T, int BMN, int WM, int WN>
int launch_products_of(const Product& gx, const Product& gw, hipStream_t st) {
  constexpr int A = TokGemm<T, false, true, BMN, BMN, WM, WN>::LDS_BYTES, B = TokGemm<T, true, true, BMN, BMN, WM, WN>::LDS_BYTES;
  auto kernel = products_kernel<T, BMN, WM, WN>;
  const int rc = allow_lds(kernel, A > B ? A : B);
  if (rc) return rc;
  kernel<<<gx.blocks + gw.blocks, 64 * WM * WN, A > B ? A : B, st>>>(gx.p, gw.p, gx.blocks);
  VG_CHECK_LAUNCH("gated backward products");
  return VG_OK;
}
// either may have no blocks
template <class T>
int launch_products(const Product& gx, const Product& gw, hipStream_t st) {
  if constexpr (sizeof(T) == 4) {
    return launch_products_of<T, 128, 2, 4>(gx, gw, st);
  } else {
    if (gx.blocks && gw.blocks && gx.plan.tile != gw.plan.tile) {
      const int rc = launch_products<T>(gx, Product{}, st);
      return rc ? rc : launch_products<T>(Product{}, gw, st);
    }
    return (gx.blocks ? gx : gw).plan.tile == 256 ? launch_products_of<T, 256, 2, 4>(gx, gw, st) : launch_products_of<T, 128, 2, 2>(gx, gw, st);
  }
}

// What the backward pass of these sizes runs on: pre-activations kept by the forward pass in f32 (8 bytes written and read
// an element), or, with bf16 operands, computed again. Forward and backward, again / kept: 16384 x C x 4096: C = 256 622 /
// 651 us, 512 814 / 782, 768 1168 / 1079, 1024 1242 / 1107; 16384 x C x 1024: 256 184 / 209, 512 236 / 256, 768 375 / 353,
// 1024 352 / 329. (Up to 64 rows the forward kernel has no backward twin.)
template <class T>
bool keeps_z(int M, int C) { return sizeof(T) == 4 || M <= kFewRows || C > 512; }

// Scratch of the backward pass, one piece after the other: [gg gu], partial column sums, slabs of the two products.
// bf16: [gg gu] is rounded to bf16 for the two products, which costs a result 0.4 of its own rounding. In a small call (under
// 2^19 of them) what the rounding left is multiplied too, as a second term, at no visible cost. The size is that of the
// whole call, so a row's last bits depend on how many others come with it.
template <class T>
int gz_terms(int M, int F) { return sizeof(T) == 2 && (long long)M * 2 * F < (1 << 19) ? 2 : 1; }

struct BwdSpace {
  size_t gz, part, gx_slabs, gw_slabs, total;
  int rows;          // of partial column sums
};
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
template <class T>
BwdSpace bwd_space(int M, int C, int F) {
  BwdSpace s;
  s.rows = ceil_div(M, keeps_z<T>(M, C) ? kRowsBlock : large_tiles<T>(M, 2ll * F) ? 256 : 128);
  s.gz = 0;
  s.part = align256((size_t)M * 2 * F * sizeof(T) * gz_terms<T>(M, F));
  const int terms = gz_terms<T>(M, F);
  s.gx_slabs = s.part + align256((size_t)s.rows * 2 * F * 4);
  s.gw_slabs = s.gx_slabs + align256(product_bytes<T>(M, C, 2 * F, terms));
  s.total = s.gw_slabs + product_bytes<T>(2 * F, C, M, terms);
  return s;
}

template <class T>
int gated_bwd(int M, int C, int F, const void* x, const void* w, const float* bias, const float* z, const void* gh, void* gx, void* gw,
              int gw_f32, float* gb, int act, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_sizes(M, C, F, act);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (M == 0) {        // sums over no rows
    if (gw) rc = launch_products<T>(Product{}, product<T>(gh, 2 * (int64_t)F, 1, 0, x, C, 2 * F, C, 0, gw, gw_f32, nullptr), st);
    if (!rc && gb) rc = vg_fill(gb, 0.f, 2 * (size_t)F, stream);
    return rc;
  }
  VG_REQUIRE(x && w && gh, "gated backward: null tensor");
  VG_REQUIRE(!keeps_z<T>(M, C) || z, "gated backward: these sizes need the pre-activations of the forward pass");
  const BwdSpace s = bwd_space<T>(M, C, F);
  if (!ws || ws_bytes < s.total) return vg_fail(VG_ERR_WORKSPACE, "gated backward: workspace of %zu bytes, %zu are needed", ws_bytes, s.total);
  VG_REQUIRE(vg_aligned16(ws), "gated backward: workspace is not 16-byte aligned");
  char* at = (char*)ws;
  GatedParams p = {};
  p.x = x;
  p.w = w;
  p.bias = bias;
  p.gh = gh;
  p.gz = at + s.gz;
  p.gb_part = gb ? (float*)(at + s.part) : nullptr;
  p.M = M;
  p.C = C;
  p.F = F;
  p.act = act;
  p.terms = gz_terms<T>(M, F);
  if (keeps_z<T>(M, C)) {
    p.z = const_cast<float*>(z);
    constexpr int V = TokNum<T>::V;
    const bool wide = F % V == 0 && vg_aligned16(z) && vg_aligned16(gh);
    const dim3 grid(ceil_div(M, kRowsBlock), ceil_div(F, wide ? 64 * V : 64));
    if (wide && (size_t)M * F * (8 + 3 * sizeof(T)) > kStreamBytes)
      gated_bwd_kernel<T, V, true><<<grid, 256, 0, st>>>(p);
    else if (wide)
      gated_bwd_kernel<T, V, false><<<grid, 256, 0, st>>>(p);
    else
      gated_bwd_kernel<T, 1, false><<<grid, 256, 0, st>>>(p);
    VG_CHECK_LAUNCH("gated backward");
  } else if constexpr (sizeof(T) == 2) {
    rc = launch_gated<T, true>(p, st);
    if (rc) return rc;
  }
  Product px = {}, pw = {};
  if (gx) px = product<T>(p.gz, 2 * (int64_t)F, p.terms, (int64_t)M * 2 * F, w, C, M, C, 2 * F, gx, sizeof(T) == 4, at + s.gx_slabs);
  if (gw) pw = product<T>(p.gz, 2 * (int64_t)F, p.terms, (int64_t)M * 2 * F, x, C, 2 * F, C, M, gw, gw_f32, at + s.gw_slabs);
  if (gx || gw) rc = launch_products<T>(px, pw, st);
  if (rc) return rc;
  const int sums = px.sum.blocks + pw.sum.blocks + (gb ? ceil_div(2ll * F, 32) : 0);
  if (sums) {
    gated_sums_kernel<<<sums, 1024, 0, st>>>(px.sum, pw.sum, p.gb_part, s.rows, 2 * F, gb);
    VG_CHECK_LAUNCH("gated backward sums");
  }
  return rc;
}

}  // namespace

extern "C" {

int vg_gated_linear_fwd(int M, int C, int F, const float* x, const float* w, const float* bias, float* h, float* z, int act, void* stream) {
  return gated_fwd<float>(M, C, F, x, w, bias, h, z, act, stream);
}
int vg_gated_linear_fwd_h(int M, int C, int F, const void* x, const void* w, const float* bias, void* h, float* z, int act, void* stream) {
  return gated_fwd<__bf16>(M, C, F, x, w, bias, h, z, act, stream);
}
int vg_gated_linear_keeps_z(int M, int C, int F, int half) { return half ? keeps_z<__bf16>(M, C) : keeps_z<float>(M, C); }
size_t vg_gated_linear_bwd_workspace_bytes(int M, int C, int F, int half) {
  if (check_sizes(M, C, F, VG_GATE_SILU) || M == 0) return 0;
  return half ? bwd_space<__bf16>(M, C, F).total : bwd_space<float>(M, C, F).total;
}
int vg_gated_linear_bwd(int M, int C, int F, const float* x, const float* w, const float* bias, const float* z, const float* gh, float* gx,
                        float* gw, int gw_f32, float* gb, int act, void* workspace, size_t workspace_bytes, void* stream) {
  VG_REQUIRE(gw_f32 || !gw, "gated backward: f32 tensors have an f32 weight gradient");
  return gated_bwd<float>(M, C, F, x, w, bias, z, gh, gx, gw, 1, gb, act, workspace, workspace_bytes, stream);
}
int vg_gated_linear_bwd_h(int M, int C, int F, const void* x, const void* w, const float* bias, const float* z, const void* gh, void* gx,
                          void* gw, int gw_f32, float* gb, int act, void* workspace, size_t workspace_bytes, void* stream) {
  return gated_bwd<__bf16>(M, C, F, x, w, bias, z, gh, gx, gw, gw_f32, gb, act, workspace, workspace_bytes, stream);
}

}  // extern "C"
