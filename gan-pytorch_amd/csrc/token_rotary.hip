// Per-head RMS norm of queries and keys and their rotation by positions on several axes, one pass over the data.
//
//   r = 1 / sqrt(mean(x^2) + eps)      n = x r w           (w null: n = x)
//   section a of a head (width[a] elements, pairs (2i, 2i+1)):  theta = pos[a] base^(-2i / width[a])
//   y0 = n0 cos - n1 sin    y1 = n0 sin + n1 cos           (elements behind the sections: y = n)
// backward:  gn = R^T gy     gw = sum gn x r     gx = r (w gn - x r mean(w gn x r))     (heads with gy = 0: nothing)
//
// Bound by HBM: one read and one write per element forward, two reads and one write backward. A thread holds one
// 16-byte vector of a head, a power of two of neighbouring lanes the head, and a wave one token (or several, where its
// heads do not fill it) whose heads it walks, queries, then keys: the angles depend on the token and the lane's place in
// the head only, so the sine and cosine are worked out once per token and thread, not per head, under the loads of the
// heads. The angle is formed in 64 bits, in turns, and reduced to half a turn before it becomes an f32, so far positions
// keep their accuracy.
#include <math.h>

#include "token_common.h"

namespace {

struct RotaryParams {
  vg_rotary_geom g;
  const void *q, *k, *gq, *gk;
  void *oq, *ok;
  const float *wq, *wk;
  const void* pos;
  float* part;            // backward: [blocks][2][D] partial sums of the weight gradients
  int lph, hps;           // lanes of a head, head slots of a wave's token group
  int wave_tokens;        // tokens a wave works on at once
  double decay[4];        // log2 of the ratio of neighbouring elements' frequencies on an axis
};

// Blocks of four waves: as many as run at once (registers: four waves a SIMD forward, three backward), so that a wave's
// start (frequencies in 64 bits) is spread over as many tokens as can be. Measured on 4 x 8192 tokens, 20 heads of 128, bf16
// (336 MB forward, 503 MB backward): forward 67 us (5.0 TB/s; half the blocks 94), backward 106 us (4.8 TB/s; half 163);
// twice the blocks take the same. The outputs are written past the caches, which leaves those to the reads: 70 and 119 us
// without; 3 x 777 tokens of 8 heads of 72 in f32 (27 MB both ways) take 8 + 11 us so, 10 + 12 without.
constexpr int kBlocks = 1024;
constexpr int kBwdBlocks = 768;     // rows of partial weight-gradient sums at most

template <int V>
__device__ __forceinline__ void angles(const RotaryParams& p, long long at, const double (&freq)[V / 2], const int (&axis)[V / 2],
                                       float (&c)[V / 2], float (&s)[V / 2]) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
    if (axis[i] >= 0) {
      const double x = p.g.pos_wide ? (double)((const long long*)p.pos)[at + axis[i]] : (double)((const int*)p.pos)[at + axis[i]];
      const double turn = x * freq[i];
      sincospif(2.f * (float)(turn - rint(turn)), &s[i], &c[i]);
    }
  }
}

// sum over the `lanes` (a power of two) neighbouring lanes of a head, in every one of them
template <int CTRL>
__device__ __forceinline__ float plus_lane(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float head_sum(float v, int lanes) {
  if (lanes >= 2) v = plus_lane<0xB1>(v);      // lane ^ 1
  if (lanes >= 4) v = plus_lane<0x4E>(v);      // lane ^ 2
  if (lanes >= 8) v = plus_lane<0x141>(v);     // mirrored in 8: the other four's sum
  if (lanes >= 16) v = plus_lane<0x140>(v);    // mirrored in 16
  if (lanes >= 32) v += __shfl_xor(v, 16, 64);
  if (lanes >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// Whether any of the head's gradients is not zero. A head without takes no part in the backward pass, whatever it holds: the
// padding of a batch may be NaN, and 0 NaN would reach the weights' gradients.
__device__ __forceinline__ bool head_any(u32x4 g, unsigned magnitude, int lane, int lanes) {
  const unsigned long long some = __ballot(((g[0] | g[1] | g[2] | g[3]) & magnitude) != 0);
  return (some >> (lane & -lanes) & (lanes == 64 ? ~0ull : (1ull << lanes) - 1)) != 0;
}

template <class T, bool BWD>
__global__ void __launch_bounds__(256, BWD ? 3 : 4) rotary_kernel(const RotaryParams p) {
  constexpr int V = TokNum<T>::V;
  constexpr int kUnroll = BWD ? 5 : 6;     // head steps whose loads are in flight together (what the registers hold)
  __shared__ float weight[2][256];
  const vg_rotary_geom& g = p.g;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int lh = lane & (p.lph - 1);                   // lane in the head
  const int slot = (lane / p.lph) & (p.hps - 1);       // head slot
  const int sub = lane / (p.lph * p.hps);              // token of the group
  const int d0 = lh * V;
  const bool in = d0 < g.D;

  // the lane's pairs: axis and frequency (in turns per position)
  double freq[V / 2];
  int axis[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    axis[i] = -1;
    int d = d0 + 2 * i;
    double e = 0.0;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (a < g.axes && axis[i] < 0) {
        if (d < g.width[a]) {
          axis[i] = a;
          e = (double)d * p.decay[a];
        }
        d -= g.width[a];
      }
    }
    freq[i] = g.axes ? exp2(e) * 0.15915494309189533577 : 0.0;
    if (!in) axis[i] = -1;
  }
  {
    const int d = threadIdx.x;
    weight[0][d] = d < g.D && p.wq ? p.wq[d] : 1.f;
    weight[1][d] = d < g.D && p.wk ? p.wk[d] : 1.f;
  }
  __syncthreads();
  float sq[V], sk[V];                                  // (backward) sums of the weights' gradients
#pragma unroll
  for (int e = 0; e < V; ++e) sq[e] = sk[e] = 0.f;
  const float inv_d = 1.f / (float)g.D;
  const unsigned tokens = (unsigned)g.B * (unsigned)g.T, stride = gridDim.x * 4 * p.wave_tokens;
  const int q_steps = (g.Hq + p.hps - 1) / p.hps, steps = q_steps + (g.Hk + p.hps - 1) / p.hps;
  for (unsigned base = (blockIdx.x * 4 + wid) * p.wave_tokens; base < tokens; base += stride) {
    const unsigned token = base + sub;
    const bool tok = token < tokens;
    const int b = tok ? (int)(token / (unsigned)g.T) : 0, t = tok ? (int)(token - (unsigned)b * g.T) : 0;
    float c[V / 2], s[V / 2];
    for (int s0 = 0; s0 < steps; s0 += kUnroll) {
      u32x4 rx[kUnroll], rg[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const bool isq = s0 + u < q_steps;                       // uniform
        const int h = (s0 + u - (isq ? 0 : q_steps)) * p.hps + slot;
        const bool ok = tok && in && s0 + u < steps && h < (isq ? g.Hq : g.Hk);
        const vg_heads_layout& lx = isq ? g.q : g.k;
        const T* x = (const T*)(isq ? p.q : p.k) + b * lx.sb + t * lx.st + h * lx.sh + d0;
        rx[u] = ok && (!BWD || (isq ? p.wq : p.wk)) ? *reinterpret_cast<const u32x4*>(x) : u32x4{0, 0, 0, 0};
        if constexpr (BWD) {
          const vg_heads_layout& lg = isq ? g.gq : g.gk;
          const T* gy = (const T*)(isq ? p.gq : p.gk) + b * lg.sb + t * lg.st + h * lg.sh + d0;
          rg[u] = ok ? *reinterpret_cast<const u32x4*>(gy) : u32x4{0, 0, 0, 0};
        }
      }
      if (s0 == 0) angles<V>(p, (long long)b * g.pos_sb + (long long)t * g.axes, freq, axis, c, s);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (s0 + u >= steps) break;          // uniform
        const bool isq = s0 + u < q_steps;
        const int h = (s0 + u - (isq ? 0 : q_steps)) * p.hps + slot;
        const bool ok = tok && in && h < (isq ? g.Hq : g.Hk);
        const vg_heads_layout& lo = isq ? g.oq : g.ok;
        T* out = (T*)(isq ? p.oq : p.ok) + b * lo.sb + t * lo.st + h * lo.sh + d0;
        auto one = [&](int which, bool normed, float (&sum)[V]) {
          float xv[V], y[V], w[V];
#pragma unroll
          for (int e = 0; e < V; ++e) w[e] = weight[which][d0 + e];
          tok_widen(rx[u], xv);
          float r = 1.f;
          if (normed) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) ss = __builtin_fmaf(xv[e], xv[e], ss);
            r = __builtin_amdgcn_rsqf(__builtin_fmaf(head_sum(ss, p.lph), inv_d, g.eps));
          }
          if constexpr (!BWD) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const float n0 = xv[2 * i] * r * w[2 * i], n1 = xv[2 * i + 1] * r * w[2 * i + 1];
              y[2 * i] = n0 * c[i] - n1 * s[i];
              y[2 * i + 1] = n0 * s[i] + n1 * c[i];
            }
          } else {
            float gv[V], inner = 0.f;
            tok_widen(rg[u], gv);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              y[2 * i] = gv[2 * i] * c[i] + gv[2 * i + 1] * s[i];
              y[2 * i + 1] = gv[2 * i + 1] * c[i] - gv[2 * i] * s[i];
            }
            if (normed) {
              const bool live = head_any(rg[u], sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu, lane, p.lph);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float xh = live ? xv[e] * r : 0.f, wg = w[e] * y[e];
                if (ok) sum[e] = __builtin_fmaf(y[e], xh, sum[e]);
                inner = __builtin_fmaf(wg, xh, inner);
                xv[e] = xh;
                y[e] = wg;
              }
              inner = head_sum(inner, p.lph) * inv_d;
#pragma unroll
              for (int e = 0; e < V; ++e) y[e] = live ? r * __builtin_fmaf(-xv[e], inner, y[e]) : 0.f;
            }
          }
          if (ok) __builtin_nontemporal_store(tok_narrow(y), reinterpret_cast<u32x4*>(out));
        };
        if (isq)
          one(0, p.wq != nullptr, sq);
        else
          one(1, p.wk != nullptr, sk);
      }
    }
  }
  if constexpr (BWD) {
    if (!p.part) return;
    // sums of the block's waves and of the lanes that hold the same elements, in a fixed order
    __shared__ float red[2][4][64][V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      red[0][wid][lane][e] = sq[e];
      red[1][wid][lane][e] = sk[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * g.D; i += 256) {
      const int which = i >= g.D, d = which ? i - g.D : i;
      float v = 0.f;
      for (int w = 0; w < 4; ++w)
        for (int l = d / V; l < 64; l += p.lph) v += red[which][w][l][d % V];
      p.part[(size_t)blockIdx.x * 2 * g.D + i] = v;
    }
  }
}

// gw[which][d] = sum over blocks of part[block][which][d]: 32 columns and 32 row lanes per workgroup, every lane's rows
// requested before the first is added
__global__ void __launch_bounds__(1024) rotary_weight_kernel(const float* part, int rows, int D, float* gwq, float* gwk) {
  __shared__ float red[32][33];
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + col;
  float got[kBwdBlocks / 32], v = 0.f;
#pragma unroll
  for (int r = 0; r < kBwdBlocks / 32; ++r) got[r] = i < 2 * D && row + 32 * r < rows ? part[(size_t)(row + 32 * r) * 2 * D + i] : 0.f;
#pragma unroll
  for (int r = 0; r < kBwdBlocks / 32; ++r) v += got[r];
  red[row][col] = v;
  __syncthreads();
  if (row == 0 && i < 2 * D) {
#pragma unroll
    for (int r = 1; r < 32; ++r) v += red[r][col];
    float* out = i < D ? gwq : gwk;
    if (out) out[i < D ? i : i - D] = v;
  }
}

int check_geom(const vg_rotary_geom* g, const void* pos) {
  VG_REQUIRE(g, "rotary: null geometry");
  VG_REQUIRE(g->B >= 0 && g->T >= 0 && g->Hq >= 1 && g->Hk >= 0, "rotary: bad sizes B=%d T=%d Hq=%d Hk=%d", g->B, g->T, g->Hq, g->Hk);
  VG_REQUIRE((long long)g->B * g->T < (1ll << 31), "rotary: %lld tokens are too many", (long long)g->B * g->T);
  VG_REQUIRE(g->D >= 8 && g->D <= 256 && g->D % 8 == 0, "rotary: head width %d is not a multiple of 8 from 8 to 256", g->D);
  VG_REQUIRE(g->axes >= 0 && g->axes <= 4, "rotary: %d axes, 0 to 4 are supported", g->axes);
  VG_REQUIRE(g->axes == 0 || pos || (long long)g->B * g->T == 0, "rotary: null positions");
  int64_t total = 0;
  for (int a = 0; a < g->axes; ++a) {
    VG_REQUIRE(g->width[a] >= 2 && g->width[a] % 2 == 0, "rotary: axis width %d is not even and positive", g->width[a]);
    total += g->width[a];
  }
  VG_REQUIRE(total <= g->D, "rotary: axis widths sum to %lld, more than the head width %d", (long long)total, g->D);
  VG_REQUIRE(g->axes == 0 || g->base > 0.0, "rotary: base must be positive");
  return VG_OK;
}

void plan(RotaryParams& p, int V) {
  auto pow2 = [](int n) {
    int r = 1;
    while (r < n) r *= 2;
    return r;
  };
  p.lph = pow2((p.g.D + V - 1) / V);
  const int heads = p.g.Hq > p.g.Hk ? p.g.Hq : p.g.Hk;
  p.hps = pow2(heads) < 64 / p.lph ? pow2(heads) : 64 / p.lph;
  p.wave_tokens = 64 / (p.lph * p.hps);
  for (int a = 0; a < p.g.axes; ++a) p.decay[a] = -log2(p.g.base) / p.g.width[a];
}

long long wave_groups(const RotaryParams& p) { return ((long long)p.g.B * p.g.T + p.wave_tokens - 1) / p.wave_tokens; }

template <class T>
int rotary_fwd(const vg_rotary_geom* g, const void* q, const void* k, const float* wq, const float* wk, const void* pos, void* yq,
               void* yk, void* stream) {
  const int rc = check_geom(g, pos);
  if (rc) return rc;
  if ((long long)g->B * g->T == 0) return VG_OK;
  VG_REQUIRE(q && yq && (g->Hk == 0 || (k && yk)), "rotary: null tensor");
  VG_REQUIRE(tok_layout_ok<T>(g->q, q, g->B, g->T, g->Hq) && tok_layout_ok<T>(g->oq, yq, g->B, g->T, g->Hq) &&
                 (g->Hk == 0 || (tok_layout_ok<T>(g->k, k, g->B, g->T, g->Hk) && tok_layout_ok<T>(g->ok, yk, g->B, g->T, g->Hk))),
             "rotary: a head does not start on a 16-byte border");
  RotaryParams p = {*g, q, k, nullptr, nullptr, yq, yk, wq, wk, pos};
  plan(p, TokNum<T>::V);
  long long blocks = (wave_groups(p) + 3) / 4;
  if (blocks > kBlocks) blocks = kBlocks;
  rotary_kernel<T, false><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(p);
  VG_CHECK_LAUNCH("rotary");
  return VG_OK;
}

int bwd_blocks(const RotaryParams& p) {
  const long long blocks = (wave_groups(p) + 3) / 4;
  return (int)(blocks < kBwdBlocks ? blocks : kBwdBlocks);
}

template <class T>
int rotary_bwd(const vg_rotary_geom* g, const void* q, const void* k, const float* wq, const float* wk, const void* pos,
               const void* gyq, const void* gyk, void* gq, void* gk, float* gwq, float* gwk, void* workspace, size_t workspace_bytes,
               void* stream) {
  const int rc = check_geom(g, pos);
  if (rc) return rc;
  VG_REQUIRE((!gwq || wq) && (!gwk || wk), "rotary: gradient of a weight that is not there");
  const bool sums = gwq || gwk;
  hipStream_t st = (hipStream_t)stream;
  RotaryParams p = {*g, q, k, gyq, gyk, gq, gk, wq, wk, pos};
  plan(p, TokNum<T>::V);
  int blocks = 0;
  if ((long long)g->B * g->T != 0) {
    VG_REQUIRE(gyq && gq && (g->Hk == 0 || (gyk && gk)) && (!wq || q) && (!wk || g->Hk == 0 || k), "rotary: null tensor");
    VG_REQUIRE(tok_layout_ok<T>(g->q, q, g->B, g->T, g->Hq) && tok_layout_ok<T>(g->gq, gyq, g->B, g->T, g->Hq) &&
                   tok_layout_ok<T>(g->oq, gq, g->B, g->T, g->Hq) &&
                   (g->Hk == 0 || (tok_layout_ok<T>(g->k, k, g->B, g->T, g->Hk) && tok_layout_ok<T>(g->gk, gyk, g->B, g->T, g->Hk) &&
                                   tok_layout_ok<T>(g->ok, gk, g->B, g->T, g->Hk))),
               "rotary: a head does not start on a 16-byte border");
    blocks = bwd_blocks(p);
    if (sums) {
      if (!workspace || workspace_bytes < (size_t)blocks * 2 * g->D * sizeof(float))
        return vg_fail(VG_ERR_WORKSPACE, "rotary: workspace of %zu bytes is too small", workspace_bytes);
      p.part = (float*)workspace;
    }
    rotary_kernel<T, true><<<blocks, 256, 0, st>>>(p);
    VG_CHECK_LAUNCH("rotary backward");
  }
  if (sums) {      // (no tokens: zeros)
    rotary_weight_kernel<<<(2 * g->D + 31) / 32, 1024, 0, st>>>(p.part, blocks, g->D, gwq, gwk);
    VG_CHECK_LAUNCH("rotary weight gradient");
  }
  return VG_OK;
}

}  // namespace

extern "C" {

size_t vg_qk_norm_rotary_workspace_bytes(const vg_rotary_geom* g) {
  if (check_geom(g, g)) return 0;
  return (size_t)kBwdBlocks * 2 * g->D * sizeof(float);
}
int vg_qk_norm_rotary_fwd(const vg_rotary_geom* g, const float* q, const float* k, const float* wq, const float* wk, const void* pos,
                          float* yq, float* yk, void* stream) {
  return rotary_fwd<float>(g, q, k, wq, wk, pos, yq, yk, stream);
}
int vg_qk_norm_rotary_fwd_h(const vg_rotary_geom* g, const void* q, const void* k, const float* wq, const float* wk, const void* pos,
                            void* yq, void* yk, void* stream) {
  return rotary_fwd<__bf16>(g, q, k, wq, wk, pos, yq, yk, stream);
}
int vg_qk_norm_rotary_bwd(const vg_rotary_geom* g, const float* q, const float* k, const float* wq, const float* wk, const void* pos,
                          const float* gyq, const float* gyk, float* gq, float* gk, float* gwq, float* gwk, void* workspace,
                          size_t workspace_bytes, void* stream) {
  return rotary_bwd<float>(g, q, k, wq, wk, pos, gyq, gyk, gq, gk, gwq, gwk, workspace, workspace_bytes, stream);
}
int vg_qk_norm_rotary_bwd_h(const vg_rotary_geom* g, const void* q, const void* k, const float* wq, const float* wk, const void* pos,
                            const void* gyq, const void* gyk, void* gq, void* gk, float* gwq, float* gwk, void* workspace,
                            size_t workspace_bytes, void* stream) {
  return rotary_bwd<__bf16>(g, q, k, wq, wk, pos, gyq, gyk, gq, gk, gwq, gwk, workspace, workspace_bytes, stream);
}

}  // extern "C"
