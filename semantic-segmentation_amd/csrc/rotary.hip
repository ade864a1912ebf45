// Root-mean-square norm of every query and key head and the rotation of its channel pairs by position angles, in one
// pass over the heads (several position axes: time, height, width), and its backward pass.
//   r = (mean_d x_d^2 + eps)^-1/2,  y = w x r,  pair c turned by t = position[axis of c] * inv_freq[c]:
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t)
// Memory-bound: every head is read once and written once (backward: x and dy read, dx written).  bf16, 16 maps of 65 x 65
// pixels with 16 + 16 heads of 64 channels: 116 us, 4.8 TB/s (a copy reaches 5.09); 16 maps of 33 x 33 with 16 + 16 heads of
// 128: forward 66 us, backward 100 us, 4.3 TB/s; one token 3.8 us, the launch.
#include "common.h"

namespace segk {

constexpr int ROT_THREADS = 256;
constexpr int ROT_UNROLL = 4;        // heads in flight per group of lanes (and as many asked for)
constexpr int ROT_MAX_BLOCKS = 2048; // of the backward pass: rows of weight-gradient partials

struct RotSide {   // queries or keys
  const char* x;
  long long xn, xl, xh;     // byte strides
  const char* dy;
  long long dn, dl, dh;
  char* y;                  // forward result / backward dx, contiguous
  const float* w;
  int heads;
};

struct RotDev {
  RotSide s[2];
  const char* pos;
  long long pn, pl, pa;     // element strides
  int pos_dtype, axes;
  int first[4];             // first pair of each axis
  const float* inv_freq;
  float eps;
  int norm, interleaved, pairs;
  int N, L, D;
  float inv_d;
  int heads_per, chunks;    // heads of one piece of work, pieces per token
  int work;                 // pieces in all
  float* part;              // [2 * D][blocks] weight-gradient partials
  int blocks;
};

// 4 channels as they lie in memory
template <typename T>
struct RotRaw;
template <>
struct RotRaw<bf16_t> {
  u32x2 v;
  __device__ __forceinline__ void to(float* x) const {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      x[2 * e] = __uint_as_float(v[e] << 16);
      x[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
    }
  }
};
template <>
struct RotRaw<float> {
  f32x4 v;
  __device__ __forceinline__ void to(float* x) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v[e];
  }
};

template <typename T>
__device__ __forceinline__ void rot_store4(char* p, const float* v);
template <>
__device__ __forceinline__ void rot_store4<bf16_t>(char* p, const float* v) {
  *reinterpret_cast<u32x2*>(p) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}
template <>
__device__ __forceinline__ void rot_store4<float>(char* p, const float* v) {
  *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
}

// A lane owns 4 pairs = 8 channels of a head, v[0 .. 3] and v[4 .. 7] from the runs of 4 channels at lo and hi.  INTER
// (neighbours are paired): one run of 8, pairs (v[2c], v[2c + 1]).  Else pairs (v[c], v[4 + c]): channel c of the first
// half and of the second half of the rotated channels, and then of the channels past them (which turn by nothing).
template <bool INTER>
struct RotLane {
  int lo, hi;
  bool live;
  float c[4], s[4];
  __device__ __forceinline__ RotLane(const RotDev& p, int j) {
    live = j * 8 < p.D;
    const bool turned = 4 * j < p.pairs;
    lo = INTER ? 8 * j : turned ? 4 * j : p.pairs + 4 * j;
    hi = INTER ? 8 * j + 4 : turned ? p.pairs + 4 * j : p.D / 2 + 4 * j;
    if (!live) lo = hi = 0;      // (never stored)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = 1.f, s[e] = 0.f;
  }
  __device__ __forceinline__ int channel(int e) const { return e < 4 ? lo + e : hi + e - 4; }
  // cos and sin of this lane's pairs.  The angle is formed and reduced to half turns in fp64 (a position in the hundred
  // thousands times a frequency loses its fraction in fp32), the rest in fp32.
  __device__ __forceinline__ void angles(const RotDev& p, int j, int n, int l) {
    if (4 * j >= p.pairs) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 4 * j + e;
      int axis = 0;
#pragma unroll
      for (int a = 1; a < 4; ++a) axis = a < p.axes && k >= p.first[a] ? a : axis;
      const long long at = n * p.pn + l * p.pl + axis * p.pa;
      double x;
      if (p.pos_dtype == 0) x = ((const int*)p.pos)[at];
      else if (p.pos_dtype == 1) x = (double)((const long long*)p.pos)[at];
      else x = ((const float*)p.pos)[at];
      const double half_turns = x * (double)p.inv_freq[k] * 0.31830988618379067154;
      const float f = (float)(half_turns - 2.0 * rint(half_turns * 0.5));
      sincospif(f, &s[e], &c[e]);
    }
  }
  // forward turn (sign +1) or its inverse (-1)
  __device__ __forceinline__ void turn(float sign, float* v) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float &a = v[INTER ? 2 * e : e], &b = v[INTER ? 2 * e + 1 : 4 + e];
      const float z = sign * s[e];
      const float x = a * c[e] - b * z, y = a * z + b * c[e];
      a = x;
      b = y;
    }
  }
  template <typename T>
  __device__ __forceinline__ void load_raw(const char* row, RotRaw<T>* x) const {
    x[0].v = *reinterpret_cast<const decltype(x[0].v)*>(row + lo * (int)sizeof(T));
    x[1].v = *reinterpret_cast<const decltype(x[0].v)*>(row + hi * (int)sizeof(T));
  }
  template <typename T>
  __device__ __forceinline__ void store(char* row, const float* v) const {
    rot_store4<T>(row + lo * (int)sizeof(T), v);
    rot_store4<T>(row + hi * (int)sizeof(T), v + 4);
  }
};

// Sum over a group of LPH neighbouring lanes, to every lane: exchanges inside 16 lanes are DPP operands.
template <int LPH>
__device__ __forceinline__ float group_sum(float v) {
#define ROT_DPP(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
  if (LPH >= 2) ROT_DPP(0xb1);    // lanes 1 0 3 2 of a quad
  if (LPH >= 4) ROT_DPP(0x4e);    // lanes 2 3 0 1 of a quad
  if (LPH >= 8) ROT_DPP(0x141);   // mirror of 8 lanes: the other quad
  if (LPH >= 16) ROT_DPP(0x140);  // mirror of 16 lanes: the other eight
#undef ROT_DPP
  if (LPH >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

// one head of the forward pass, from registers
template <typename T, int LPH, bool INTER>
__device__ __forceinline__ void rot_head(const RotDev& p, const RotLane<INTER>& t, const float* w, float* v, char* dst) {
  if (p.norm) {
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) q = fmaf(v[e], v[e], q);
    const float r = rsqrtf(fmaf(group_sum<LPH>(q), p.inv_d, p.eps));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= r * w[e];
  }
  t.turn(1.f, v);
  if (t.live) t.template store<T>(dst, v);
}

// A group of LPH lanes (D / 8 rounded up to a power of two) takes one token and `heads_per` of its heads (queries, then
// keys): the angles are computed once for all of them.
template <typename T, int LPH, bool INTER>
__global__ __launch_bounds__(ROT_THREADS) void qk_norm_rotary_kernel(const RotDev p) {
  const int j = threadIdx.x % LPH;
  const unsigned work = blockIdx.x * (ROT_THREADS / LPH) + threadIdx.x / LPH;
  if (work >= (unsigned)p.work) return;
  const unsigned nl = work / (unsigned)p.chunks;
  const int h0 = (int)(work - nl * (unsigned)p.chunks) * p.heads_per;
  const int n = (int)(nl / (unsigned)p.L), l = (int)(nl - (unsigned)n * (unsigned)p.L);
  RotLane<INTER> t(p, j);
  t.angles(p, j, n, l);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const RotSide& sd = p.s[q];
    const int shift = q ? p.s[0].heads : 0;
    const int a = max(h0 - shift, 0), b = min(h0 + p.heads_per - shift, sd.heads);
    if (a >= b) continue;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = t.live && sd.w ? sd.w[t.channel(e)] : 1.f;
    const char* src = sd.x + n * sd.xn + l * sd.xl;
    char* dst = sd.y + (long long)nl * sd.heads * p.D * (int)sizeof(T);
    // the next heads are asked for before these are worked on (lanes past D re-read channel 0 and count for nothing)
    RotRaw<T> raw[ROT_UNROLL][2];
    auto ask = [&](int hb) {
#pragma unroll
      for (int u = 0; u < ROT_UNROLL; ++u) t.template load_raw<T>(src + min(hb + u, b - 1) * sd.xh, raw[u]);
    };
    ask(a);
    for (int hb = a; hb < b; hb += ROT_UNROLL) {
      RotRaw<T> now[ROT_UNROLL][2];
#pragma unroll
      for (int u = 0; u < ROT_UNROLL; ++u) now[u][0] = raw[u][0], now[u][1] = raw[u][1];
      if (hb + ROT_UNROLL < b) ask(hb + ROT_UNROLL);
#pragma unroll
      for (int u = 0; u < ROT_UNROLL; ++u)
        if (hb + u < b) {
          float v[8];
          now[u][0].to(v);
          now[u][1].to(v + 4);
          if (!t.live) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
          }
          rot_head<T, LPH, INTER>(p, t, w, v, dst + (long long)(hb + u) * p.D * (int)sizeof(T));
        }
    }
  }
}

// Backward.  dn = dy turned back; dw = sum dn x r; g = w dn; dx = r (g - x r mean(g x r)).  Weight gradients: each lane
// sums its channels over its work in fp32, the groups of a workgroup are joined in LDS in order, one partial per
// workgroup and channel, joined in fp64 by the second kernel: no atomics, a fixed order.
template <typename T, int LPH, bool INTER>
__global__ __launch_bounds__(ROT_THREADS) void qk_norm_rotary_bwd_kernel(const RotDev p) {
  __shared__ float red[ROT_THREADS][17];   // (17: a column walk meets distinct banks)
  constexpr int GROUPS = ROT_THREADS / LPH;
  const int j = threadIdx.x % LPH;
  RotLane<INTER> t(p, j);
  float w[2][8], dw[2][8];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[q][e] = t.live && p.s[q].w ? p.s[q].w[t.channel(e)] : 1.f;
      dw[q][e] = 0.f;
    }
  for (unsigned work = blockIdx.x * GROUPS + threadIdx.x / LPH; work < (unsigned)p.work; work += gridDim.x * GROUPS) {
    const unsigned nl = work / (unsigned)p.chunks;
    const int h0 = (int)(work - nl * (unsigned)p.chunks) * p.heads_per;
    const int n = (int)(nl / (unsigned)p.L), l = (int)(nl - (unsigned)n * (unsigned)p.L);
    t.angles(p, j, n, l);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const RotSide& sd = p.s[q];
      const int shift = q ? p.s[0].heads : 0;
      const int a = max(h0 - shift, 0), b = min(h0 + p.heads_per - shift, sd.heads);
      if (a >= b) continue;
      const char* src = sd.x + n * sd.xn + l * sd.xl;
      const char* dys = sd.dy + n * sd.dn + l * sd.dl;
      char* dst = sd.y + (long long)nl * sd.heads * p.D * (int)sizeof(T);
      // (two heads in flight, two asked for, as in the forward kernel)
      RotRaw<T> raw[2][4];
      auto ask = [&](int hb) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int hh = min(hb + u, b - 1);
          t.template load_raw<T>(dys + hh * sd.dh, raw[u]);
          if (p.norm) t.template load_raw<T>(src + hh * sd.xh, raw[u] + 2);
        }
      };
      ask(a);
      for (int hb = a; hb < b; hb += 2) {
        float v[2][8], g[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          raw[u][0].to(g[u]);
          raw[u][1].to(g[u] + 4);
          if (p.norm) {
            raw[u][2].to(v[u]);
            raw[u][3].to(v[u] + 4);
          }
          if (!t.live) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] = g[u][e] = 0.f;
          }
        }
        if (hb + 2 < b) ask(hb + 2);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (hb + u >= b) break;
          t.turn(-1.f, g[u]);
          if (p.norm) {
            float z = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) z = fmaf(v[u][e], v[u][e], z);
            const float r = rsqrtf(fmaf(group_sum<LPH>(z), p.inv_d, p.eps));
            float dot = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              v[u][e] *= r;
              dw[q][e] = fmaf(g[u][e], v[u][e], dw[q][e]);
              g[u][e] *= w[q][e];
              dot = fmaf(g[u][e], v[u][e], dot);
            }
            dot = group_sum<LPH>(dot) * p.inv_d;
#pragma unroll
            for (int e = 0; e < 8; ++e) g[u][e] = r * (g[u][e] - v[u][e] * dot);
          }
          if (t.live) t.template store<T>(dst + (long long)(hb + u) * p.D * (int)sizeof(T), g[u]);
        }
      }
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) red[threadIdx.x][q * 8 + e] = dw[q][e];
  __syncthreads();
  for (int i = threadIdx.x; i < LPH * 16; i += ROT_THREADS) {
    const int jj = i % LPH, slot = i / LPH;
    float s = 0.f;
    for (int g = 0; g < GROUPS; ++g) s += red[g * LPH + jj][slot];
    const RotLane<INTER> o(p, jj);
    if (o.live) p.part[((long long)(slot >> 3) * p.D + o.channel(slot & 7)) * p.blocks + blockIdx.x] = s;
  }
}

// one wavefront per channel: dq_weight[0 .. D), dk_weight[0 .. D)
__global__ __launch_bounds__(64) void qk_norm_weight_grad_kernel(const float* __restrict__ part, int blocks, int D, float* __restrict__ dqw,
                                                                 float* __restrict__ dkw) {
  const int ch = blockIdx.x;
  double s = 0.0;
  for (int i = threadIdx.x; i < blocks; i += 64) s += (double)part[(long long)ch * blocks + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  float* dst = ch < D ? dqw : dkw;
  if (threadIdx.x == 0 && dst) dst[ch < D ? ch : ch - D] = (float)s;
}

static int rot_lanes(int D) {
  int l = 1;
  while (l * 8 < D) l *= 2;
  return l;
}

static int rot_fill(const segk_qk_norm_rotary_args* a, RotDev* p, bool backward) {
  SEGK_REQUIRE(a && valid_dtype(a->dtype), "qk_norm_rotary: null arguments or bad dtype");
  SEGK_REQUIRE(a->N > 0 && a->L > 0 && a->Hq > 0 && a->Hk >= 0 && (long long)a->N * a->L < 0x7fffffffLL,
               "qk_norm_rotary: bad shape N=%d L=%d Hq=%d Hk=%d", a->N, a->L, a->Hq, a->Hk);
  SEGK_UNSUPPORTED(a->D > 0 && a->D % 8 == 0 && a->D <= 256, "qk_norm_rotary: head size %d is not a multiple of 8 up to 256", a->D);
  SEGK_REQUIRE(a->axes >= 1 && a->axes <= 4 && a->positions && a->inv_freq && a->pos_dtype >= 0 && a->pos_dtype <= 2,
               "qk_norm_rotary: positions of 1 to 4 axes and their frequencies are needed");
  int pairs = 0;
  for (int i = 0; i < 4; ++i) {
    p->first[i] = pairs;
    if (i < a->axes) {
      SEGK_REQUIRE(a->section[i] >= 0 && a->section[i] <= 128, "qk_norm_rotary: section of %d pairs", a->section[i]);
      pairs += a->section[i];
    }
  }
  SEGK_UNSUPPORTED(pairs > 0 && pairs % 4 == 0 && 2 * pairs <= a->D,
                   "qk_norm_rotary: %d rotated pairs for a head size of %d (a multiple of 4 up to half of it)", pairs, a->D);
  SEGK_REQUIRE(!a->norm || a->eps >= 0.f, "qk_norm_rotary: negative eps");
  SEGK_REQUIRE(a->norm || (!a->q_weight && !a->k_weight), "qk_norm_rotary: weights belong to the norm");
  const int es = dtype_size(a->dtype), e8 = 16 / es;
  for (int i = 0; i < 2; ++i) {
    RotSide& s = p->s[i];
    const segk_attention_view& x = i ? a->k : a->q;
    const segk_attention_view& g = i ? a->dk : a->dq;
    s.heads = i ? a->Hk : a->Hq;
    s.x = (const char*)x.p, s.xn = x.n * es, s.xl = x.l * es, s.xh = x.h * es;
    s.dy = (const char*)g.p, s.dn = g.n * es, s.dl = g.l * es, s.dh = g.h * es;
    s.y = (char*)(i ? a->k_out : a->q_out);
    s.w = i ? a->k_weight : a->q_weight;
    if (s.heads == 0) continue;
    SEGK_REQUIRE(s.x && s.y && (!backward || s.dy), "qk_norm_rotary: null operand");
    SEGK_REQUIRE((((uintptr_t)s.x | (uintptr_t)s.y | (backward ? (uintptr_t)s.dy : 0)) & 15) == 0 && x.n % e8 == 0 && x.l % e8 == 0 &&
                     x.h % e8 == 0 && (!backward || (g.n % e8 == 0 && g.l % e8 == 0 && g.h % e8 == 0)),
                 "qk_norm_rotary: operands need 16-byte aligned pointers and strides that are multiples of 16 bytes");
  }
  p->pos = (const char*)a->positions, p->pn = a->pos_n, p->pl = a->pos_l, p->pa = a->pos_a;
  p->pos_dtype = a->pos_dtype, p->axes = a->axes, p->inv_freq = a->inv_freq;
  p->eps = a->eps, p->norm = a->norm != 0, p->interleaved = a->interleaved != 0, p->pairs = pairs;
  p->N = a->N, p->L = a->L, p->D = a->D;
  // Heads of a token that one group of lanes takes: all of them (the angles are computed once) as long as that leaves
  // 512 threads for every CU, else fewer, down to one.  One token of 20 heads: 3.8 us in 20 groups, 9.4 us in one.  fp32 clip
  // of 10890 tokens with 10 heads, forward and backward: 18 + 25 us in one group a token, 21 + 32 us in two, 43 + 47 us in ten.
  const int lanes = rot_lanes(a->D), total = a->Hq + a->Hk;
  const long long threads = (long long)a->N * a->L * total * lanes;
  long long per = threads / (256 * 512);
  per = per < 1 ? 1 : per > total ? total : per;
  if (per > 4) per = (per + 3) / 4 * 4;
  p->heads_per = (int)per;
  p->chunks = ceil_div(total, p->heads_per);
  const long long work = (long long)a->N * a->L * p->chunks;
  SEGK_UNSUPPORTED(work < 0x7f000000LL, "qk_norm_rotary: too many heads");
  p->work = (int)work;
  p->inv_d = 1.f / (float)a->D;
  p->part = nullptr;
  p->blocks = 0;
  return SEGK_OK;
}

static int rot_blocks(const RotDev& p) { return ceil_div(p.work, ROT_THREADS / rot_lanes(p.D)); }
static int rot_bwd_blocks(const RotDev& p) { return rot_blocks(p) < ROT_MAX_BLOCKS ? rot_blocks(p) : ROT_MAX_BLOCKS; }

}  // namespace segk

using namespace segk;

#define ROT_CASE(kernel, grid, LPH)                                              \
  case LPH:                                                                      \
    if (p.interleaved) kernel<T, LPH, true><<<(grid), ROT_THREADS, 0, st>>>(p);  \
    else kernel<T, LPH, false><<<(grid), ROT_THREADS, 0, st>>>(p);               \
    break;
#define ROT_LAUNCH(kernel, grid)                                                                     \
  switch (rot_lanes(p.D)) {                                                                          \
    ROT_CASE(kernel, grid, 1) ROT_CASE(kernel, grid, 2) ROT_CASE(kernel, grid, 4)                    \
    ROT_CASE(kernel, grid, 8) ROT_CASE(kernel, grid, 16) ROT_CASE(kernel, grid, 32)                  \
  }

extern "C" int segk_qk_norm_rotary(const segk_qk_norm_rotary_args* a, segk_stream_t stream) {
  RotDev p;
  const int rc = rot_fill(a, &p, false);
  if (rc != SEGK_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  SEGK_DISPATCH_DTYPE(a->dtype, T, ROT_LAUNCH(qk_norm_rotary_kernel, rot_blocks(p)));
  SEGK_CHECK_LAUNCH("qk_norm_rotary");
  return SEGK_OK;
}

extern "C" long long segk_qk_norm_rotary_bwd_workspace(const segk_qk_norm_rotary_args* a) {
  RotDev p;
  const int rc = rot_fill(a, &p, true);
  if (rc != SEGK_OK) return rc;
  return a->dq_weight || a->dk_weight ? (long long)rot_bwd_blocks(p) * 2 * p.D * 4 : 0;
}

extern "C" int segk_qk_norm_rotary_bwd(const segk_qk_norm_rotary_args* a, segk_stream_t stream) {
  RotDev p;
  const int rc = rot_fill(a, &p, true);
  if (rc != SEGK_OK) return rc;
  SEGK_REQUIRE(p.norm || (!a->dq_weight && !a->dk_weight), "qk_norm_rotary_bwd: weights belong to the norm");
  hipStream_t st = (hipStream_t)stream;
  p.blocks = rot_bwd_blocks(p);
  if (a->dq_weight || a->dk_weight) {
    SEGK_REQUIRE(a->workspace && ((uintptr_t)a->workspace & 15) == 0, "qk_norm_rotary_bwd: workspace missing or not 16-byte aligned");
    const long long need = (long long)p.blocks * 2 * p.D * 4;
    if (a->workspace_bytes < need) {
      set_error("qk_norm_rotary_bwd: workspace of %lld bytes, needs %lld", a->workspace_bytes, need);
      return SEGK_WORKSPACE_TOO_SMALL;
    }
    p.part = (float*)a->workspace;
  }
  SEGK_DISPATCH_DTYPE(a->dtype, T, ROT_LAUNCH(qk_norm_rotary_bwd_kernel, p.blocks));
  SEGK_CHECK_LAUNCH("qk_norm_rotary_bwd");
  if (p.part) {
    qk_norm_weight_grad_kernel<<<2 * p.D, 64, 0, st>>>(p.part, p.blocks, p.D, a->dq_weight, a->dk_weight);
    SEGK_CHECK_LAUNCH("qk_norm_rotary_bwd weights");
  }
  return SEGK_OK;
}
