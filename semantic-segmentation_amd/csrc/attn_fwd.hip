// Multi-head attention, forward: out = softmax(scale q k^T) v per head in one pass over the keys, with a running maximum
// and sum per row (fp32, base-2 exponents), and the host side of the attention entry points.
#include <math.h>

#include "attn.h"

namespace segk {

constexpr int KT = 64;   // keys per step

// One workgroup: 4 wavefronts of 32 * QB rows each; a loop over tiles of 64 keys.  Scores are computed transposed
// (S^T = K Q^T, a lane owns one query), so the row maximum is an in-lane reduction plus one exchange, the running
// statistics are one register, and S^T is the operand of O^T = V^T P^T as it lies (attn.h).
// MASKED: a pair mask and / or a key mask is read.
template <typename T, int DP, int QB, bool MASKED>
__global__ __launch_bounds__(ATTN_THREADS, (DP * QB * (int)sizeof(T) >= 512 ? 1 : 2)) void attn_fwd_kernel(const AttnDev p) {
  typedef AttnTile<T, DP> Tile;
  typedef AttnRead<T, DP> Rd;
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int TILE_B = KT * Tile::PITCH;
  constexpr int NP = TILE_B / 4096;       // 1-KiB pieces per wavefront and operand
  constexpr int RPW = 32 * QB, RPB = 4 * RPW;
  extern __shared__ __attribute__((aligned(1024))) char smem[];   // 2 x (K tile, V tile)

  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
  int w = xcd_contiguous(p.tiles * p.splits * p.N * p.Hk);
  if (w < 0) return;
  const int split = w % p.splits;
  w /= p.splits;
  const int tile = w % p.tiles;
  w /= p.tiles;
  const int hk = w % p.Hk, n = w / p.Hk;
  const int row0 = tile * RPB;

  // keys that some row of the workgroup may use
  const int last_row = min(row0 + RPB, p.R) - 1;
  int k_end = p.Lk;
  if (p.causal) k_end = max(0, min(k_end, div_g(p, last_row) + p.off + 1));
  const int all_steps = (k_end + KT - 1) / KT;
  const int per = (all_steps + p.splits - 1) / p.splits;
  const int t0 = min(split * per, all_steps), t1 = min(t0 + per, all_steps);

  AttnFrag<T> qf[QB][KS];
  int tok[QB], head[QB];
  bool row_ok[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = row0 + wave * RPW + qb * 32 + l31;
    row_ok[qb] = r < p.R;
    const int rr = row_ok[qb] ? r : 0;
    tok[qb] = div_g(p, rr);
    head[qb] = hk * p.G + rr - tok[qb] * p.G;
    const char* src = p.q.p + ((long long)n * p.q.n + (long long)tok[qb] * p.q.l + (long long)head[qb] * p.q.h) * (int)sizeof(T);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[qb][ks] = load_frag<T>(src, ks, h, p.D, row_ok[qb]);
  }
  const int wave_tok0 = __builtin_amdgcn_readfirstlane(div_g(p, min(row0 + wave * RPW, p.R - 1)));
  const unsigned char* mrow[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
    mrow[qb] = MASKED && p.mask ? p.mask + n * p.m_n + (long long)head[qb] * p.m_h + (long long)tok[qb] * p.m_q : nullptr;

  // staging: this lane's place in the pieces it loads
  const int lin = wave * 1024 + lane * 16;
  const int st_row = lin / Tile::PITCH;
  const int st_chunk = ((lin % Tile::PITCH) >> 4) ^ Tile::swz(st_row);     // (4096 / PITCH is a period of swz)
  const bool st_ok = st_chunk * 16 < p.D * (int)sizeof(T);
  const unsigned k_step_b = (unsigned)(p.k.l * (int)sizeof(T)), v_step_b = (unsigned)(p.v.l * (int)sizeof(T));
  const char* const kbase = p.k.p + ((long long)n * p.k.n + (long long)hk * p.k.h) * (int)sizeof(T);
  const char* const vbase = p.v.p + ((long long)n * p.v.n + (long long)hk * p.v.h) * (int)sizeof(T);
  const unsigned char* const kmask = MASKED && p.kmask ? p.kmask + n * p.km_n : nullptr;
  const unsigned lds0 = lds_addr(smem) + wave * 1024;
  auto stage = [&](int t, int buf) {
    const int key0 = t * KT;
    const u32x4 kr = buffer_of(kbase + (long long)key0 * k_step_b);
    const u32x4 vr = buffer_of(vbase + (long long)key0 * v_step_b);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int row = st_row + i * (4096 / Tile::PITCH);
      bool ok = st_ok && key0 + row < p.Lk;
      // a key that its mask closes is not read: whatever its memory holds, zeros arrive
      if (MASKED && kmask && ok) ok = kmask[(long long)(key0 + row) * p.km_k] != 0;
      const unsigned lds = lds0 + buf * (2 * TILE_B) + i * 4096;
      dma_1k(kr, lds, ok ? row * k_step_b + st_chunk * 16 : ATTN_OOB);
      dma_1k(vr, lds + TILE_B, ok ? row * v_step_b + st_chunk * 16 : ATTN_OOB);
    }
  };

  f32x16 o[QB][DB];
  float m[QB], l[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m[qb] = -INFINITY;
    l[qb] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[qb][db] = zero16();
  }

  if (t0 < t1) stage(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    tile_barrier();                       // tile t is here; every wavefront has left tile t - 1
    if (t + 1 < t1) stage(t + 1, buf ^ 1);
    const char* kt = smem + buf * (2 * TILE_B);
    const char* vt = kt + TILE_B;
    const int key0 = t * KT;

    f32x16 s[QB][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) s[qb][kb] = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const AttnFrag<T> a = Rd::rows(kt, kb * 32, ks, lane);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) mma32(s[qb][kb], a, qf[qb][ks]);
      }

    // closed pairs: past the last key, above the diagonal, masked
    const bool ragged = key0 + KT > p.Lk || (p.causal && key0 + KT - 1 > wave_tok0 + p.off);
    if (MASKED || ragged) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int lim = p.causal ? min(p.Lk - 1, tok[qb] + p.off) : p.Lk - 1;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = key0 + kb * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
            bool open = j <= lim;
            if (MASKED && open) {
              if (kmask) open = kmask[(long long)j * p.km_k] != 0;
              if (mrow[qb] && open) open = mrow[qb][(long long)j * p.m_k] != 0;
            }
            s[qb][kb][i] = open ? s[qb][kb][i] : -INFINITY;
          }
      }
    }

    AttnFrag<T> pf[QB][4];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float mx = s[qb][0][0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[qb][kb][i]);
      mx = pair_max(mx) * p.scale_log2;
      // The maximum in use may lag the true one by up to 8 (probabilities up to 2^8, harmless in fp32 and in the relative
      // precision of bf16): the accumulators are then rescaled a few times per row instead of once per tile.
      if (__any(mx > m[qb] + 8.f)) {
        const float nm = fmaxf(m[qb], mx);
        const float safe = nm == -INFINITY ? 0.f : nm;
        const float alpha = exp2_fast(m[qb] - safe);
        m[qb] = nm;
        l[qb] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[qb][db][i] *= alpha;
      }
      const float ms = m[qb] == -INFINITY ? 0.f : m[qb];
      float sum = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = exp2_fast(fmaf(s[qb][kb][i], p.scale_log2, -ms));
          s[qb][kb][i] = e;
          sum += e;
        }
      l[qb] += sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) pf[qb][j] = pack_frag<T>(s[qb][j >> 1], j & 1);
    }

#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const AttnFrag<T> a = Rd::cols(vt, j * 16, db * 32, lane);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) mma32(o[qb][db], a, pf[qb][j]);
      }
  }

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float lt = pair_sum(l[qb]);
    if (!row_ok[qb]) continue;
    if (p.splits == 1) {
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      char* dst = p.out + ((long long)n * p.o.n + (long long)tok[qb] * p.o.l + (long long)head[qb] * p.o.h) * (int)sizeof(T);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int d = db * 32 + 2 * i + 4 * h;
          if (d < p.D) store4<T>(dst, d, o[qb][db][i] * inv, o[qb][db][i + 1] * inv, o[qb][db][i + 2] * inv, o[qb][db][i + 3] * inv);
        }
      if (p.lse && h == 0)
        p.lse[((long long)n * p.Hq + head[qb]) * p.Lq + tok[qb]] = lt == 0.f ? -INFINITY : (m[qb] + log2f(lt)) * 0.6931471805599453f;
    } else {
      const long long r = ((long long)split * p.N * p.Hk + (long long)n * p.Hk + hk) * p.R + row0 + wave * RPW + qb * 32 + l31;
      float* dst = p.part + r * p.D;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int d = db * 32 + 2 * i + 4 * h;
          if (d < p.D) store4<float>((char*)dst, d, o[qb][db][i], o[qb][db][i + 1], o[qb][db][i + 2], o[qb][db][i + 3]);
        }
      if (h == 0) {
        p.part_ml[2 * r] = m[qb];
        p.part_ml[2 * r + 1] = lt;
      }
    }
  }
}

// Joins the parts of a split key axis, in part order: one wavefront per row.
template <typename T>
__global__ __launch_bounds__(ATTN_THREADS) void attn_join_kernel(const AttnDev p) {
  const int lane = threadIdx.x & 63;
  const long long rows = (long long)p.N * p.Hk * p.R;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_ml[2 * (s * rows + r)]);
  const float ms = m == -INFINITY ? 0.f : m;
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const long long at = s * rows + r;
    const float a = exp2_fast(p.part_ml[2 * at] - ms);
    l = fmaf(p.part_ml[2 * at + 1], a, l);
    if (lane < p.D) o0 = fmaf(p.part[at * p.D + lane], a, o0);
    if (lane + 64 < p.D) o1 = fmaf(p.part[at * p.D + lane + 64], a, o1);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int rr = (int)(r % p.R);
  const long long nh = r / p.R;
  const int hk = (int)(nh % p.Hk), n = (int)(nh / p.Hk);
  const int tok = div_g(p, rr), head = hk * p.G + rr - tok * p.G;
  T* dst = (T*)p.out + (long long)n * p.o.n + (long long)tok * p.o.l + (long long)head * p.o.h;
  if (lane < p.D) Elem<T>::store(dst + lane, o0 * inv);
  if (lane + 64 < p.D) Elem<T>::store(dst + lane + 64, o1 * inv);
  if (p.lse && lane == 0)
    p.lse[((long long)n * p.Hq + head) * p.Lq + tok] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Row statistics of the backward pass in packed row order: rowsum(dout * out) and the base-2 lse (+inf where a row has no
// open key and in the padding: its probabilities then come out as zeros).  D / 8 lanes (rounded up to a power of two)
// share a row.
template <typename T>
__global__ __launch_bounds__(ATTN_THREADS) void attn_row_stats_kernel(const AttnDev p, int lanes) {
  const int per = ATTN_THREADS / lanes;
  const long long rows = (long long)p.N * p.Hk * p.Rp;
  const long long r = (long long)blockIdx.x * per + threadIdx.x / lanes;
  const int c = threadIdx.x % lanes;
  if (r >= rows) return;
  const int rr = (int)(r % p.Rp);
  const long long nh = r / p.Rp;
  const int hk = (int)(nh % p.Hk), n = (int)(nh / p.Hk);
  float sum = 0.f, lse = INFINITY;
  if (rr < p.R) {
    const int tok = div_g(p, rr), head = hk * p.G + rr - tok * p.G;
    const float x = p.lse[((long long)n * p.Hq + head) * p.Lq + tok];
    lse = x == -INFINITY ? INFINITY : x * LOG2E;
    // (a row without an open key has no gradient, whatever arrives for it: its dout is not looked at)
    if (c * 8 < p.D && x != -INFINITY) {
      const AttnFrag<T> a = load_frag<T>(p.o.p + ((long long)n * p.o.n + (long long)tok * p.o.l + (long long)head * p.o.h) * (int)sizeof(T), c >> 1, c & 1, p.D, true);
      const AttnFrag<T> b = load_frag<T>(p.dout.p + ((long long)n * p.dout.n + (long long)tok * p.dout.l + (long long)head * p.dout.h) * (int)sizeof(T), c >> 1, c & 1, p.D, true);
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum = fmaf(__uint_as_float(a.v[e] << 16), __uint_as_float(b.v[e] << 16), sum);
          sum = fmaf(__uint_as_float(a.v[e] & 0xffff0000u), __uint_as_float(b.v[e] & 0xffff0000u), sum);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(a.v[e], b.v[e], sum);
      }
    }
  }
  for (int s = lanes >> 1; s > 0; s >>= 1) sum += __shfl_xor(sum, s, 64);
  if (c == 0) {
    p.row_lse2[r] = lse;
    p.row_delta[r] = sum;
  }
}

// ------------------------------------------------------------------ host ----
static int attn_dp(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }
static int attn_pitch(int D, int dtype) {
  const int b = attn_dp(D) * dtype_size(dtype);
  return b <= 64 ? 64 : b <= 128 ? 128 : b <= 256 ? 256 : 512;
}

static int fwd_rows_per_block(const AttnDev& p, int dtype) { return 128; }

static int fwd_splits(const AttnDev& p, int dtype) {
  const int rpb = fwd_rows_per_block(p, dtype);
  const long long blocks = (long long)ceil_div(p.R, rpb) * p.N * p.Hk;
  const int steps = ceil_div(p.Lk, KT);
  // Too few workgroups for 256 CUs: cut the key axis, at least 2 steps a part.
  if (blocks >= 256 || steps < 4) return 1;
  long long s = (512 + blocks - 1) / blocks;
  if (s > steps / 2) s = steps / 2;
  return s < 1 ? 1 : (int)s;
}

#define CHK_VIEW(v, name, L, H)                                                                                                   \
  SEGK_REQUIRE(a->v.p && ((uintptr_t)a->v.p & 15) == 0 && a->v.n % e8 == 0 && a->v.l % e8 == 0 && a->v.h % e8 == 0 &&            \
                   a->v.n >= 0 && a->v.l >= 0 && a->v.h >= 0,                                                                     \
               "attention: " name " needs a 16-byte aligned pointer and strides that are multiples of 16 bytes");                \
  SEGK_UNSUPPORTED((a->v.l * 64 + a->v.h * (H)) * (long long)dtype_size(a->dtype) < 0xf0000000LL,                                \
                   "attention: " name ": 64 tokens and the heads of a group must lie within 3.75 GiB")

int attn_check(const segk_attention_args* a, AttnDev* p, bool backward) {
  SEGK_REQUIRE(a, "attention: null arguments");
  SEGK_REQUIRE(valid_dtype(a->dtype), "attention: bad dtype %d", a->dtype);
  SEGK_REQUIRE(a->N > 0 && a->Lq > 0 && a->Lk >= 0 && a->Hq > 0 && a->Hk > 0 && a->Hq % a->Hk == 0,
               "attention: bad shape N=%d Lq=%d Lk=%d Hq=%d Hk=%d", a->N, a->Lq, a->Lk, a->Hq, a->Hk);
  SEGK_UNSUPPORTED(a->D > 0 && a->D <= 128 && a->D % 8 == 0, "attention: head size %d is not a multiple of 8 up to 128", a->D);
  SEGK_REQUIRE(a->scale > 0.f && a->scale < INFINITY, "attention: the scale must be positive and finite");
  const int e8 = 16 / dtype_size(a->dtype);
  const int G = a->Hq / a->Hk;
  CHK_VIEW(q, "q", a->Lq, G);
  CHK_VIEW(out, "out", a->Lq, G);
  if (a->Lk > 0) {
    CHK_VIEW(k, "k", a->Lk, 0);
    CHK_VIEW(v, "v", a->Lk, 0);
  }
  const long long R = (long long)a->Lq * G;
  SEGK_UNSUPPORTED(R * G < 0xffffffffLL && R <= 0x7fffff00LL && a->Lk <= 0x7fffff00,
                   "attention: Lq=%d with %d heads to a group is out of range", a->Lq, G);
  p->q = {(const char*)a->q.p, a->q.n, a->q.l, a->q.h};
  p->k = {(const char*)a->k.p, a->k.n, a->k.l, a->k.h};
  p->v = {(const char*)a->v.p, a->v.n, a->v.l, a->v.h};
  p->o = {(const char*)a->out.p, a->out.n, a->out.l, a->out.h};
  p->dout = {nullptr, 0, 0, 0};
  p->out = (char*)a->out.p;
  p->lse = a->lse;
  p->mask = (const unsigned char*)a->mask;
  p->m_n = a->mask_n, p->m_h = a->mask_h, p->m_q = a->mask_q, p->m_k = a->mask_k;
  p->kmask = (const unsigned char*)a->key_mask;
  p->km_n = a->key_mask_n, p->km_k = a->key_mask_k;
  p->N = a->N, p->Lq = a->Lq, p->Lk = a->Lk, p->Hq = a->Hq, p->Hk = a->Hk, p->G = G, p->D = a->D;
  p->R = (int)R;
  p->Rp = round_up((int)R, 64);
  p->g_magic = G > 1 ? (unsigned)((0x100000000ULL + G - 1) / G) : 0;
  p->causal = a->causal != 0;
  p->off = a->Lk - a->Lq;
  p->scale = a->scale;
  p->scale_log2 = a->scale * LOG2E;
  p->tiles = p->splits = 1;
  p->part = p->part_ml = nullptr;
  p->dq = p->dk = p->dv = nullptr;
  p->row_lse2 = p->row_delta = nullptr;
  if (backward) {
    CHK_VIEW(dout, "dout", a->Lq, G);
    p->dout = {(const char*)a->dout.p, a->dout.n, a->dout.l, a->dout.h};
    p->dq = (char*)a->dq, p->dk = (char*)a->dk, p->dv = (char*)a->dv;
    SEGK_REQUIRE(a->lse, "attention_bwd: the forward pass's lse is needed");
    SEGK_REQUIRE((p->dk != nullptr) == (p->dv != nullptr), "attention_bwd: dk and dv are computed together");
    SEGK_REQUIRE((((uintptr_t)p->dq | (uintptr_t)p->dk | (uintptr_t)p->dv) & 15) == 0, "attention_bwd: gradients must be 16-byte aligned");
  }
  return SEGK_OK;
}

template <typename T, int DP, int QB>
static int launch_fwd(const AttnDev& p, hipStream_t st) {
  const int lds = 4 * KT * AttnTile<T, DP>::PITCH;
  const long long blocks = (long long)p.tiles * p.splits * p.N * p.Hk;
  SEGK_UNSUPPORTED(blocks < 0x7ffffff0LL, "attention: too many workgroups");
  const unsigned grid = (unsigned)((blocks + 7) / 8 * 8);
  const bool masked = p.mask || p.kmask;
  auto kern = masked ? attn_fwd_kernel<T, DP, QB, true> : attn_fwd_kernel<T, DP, QB, false>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("attention: %s", hipGetErrorString(e));
      return SEGK_HIP_ERROR;
    }
  }
  kern<<<grid, ATTN_THREADS, lds, st>>>(p);
  SEGK_CHECK_LAUNCH("attention_fwd");
  return SEGK_OK;
}

template <typename T>
static int dispatch_fwd(const AttnDev& p, hipStream_t st) {
  switch (attn_dp(p.D)) {
    case 32: return launch_fwd<T, 32, 1>(p, st);
    case 64: return launch_fwd<T, 64, 1>(p, st);
    case 96: return launch_fwd<T, 96, 1>(p, st);
    default: return launch_fwd<T, 128, 1>(p, st);
  }
}

static long long fwd_part_floats(const AttnDev& p, int splits) {
  return splits > 1 ? (long long)splits * p.N * p.Hk * p.R * (p.D + 2) : 0;
}

}  // namespace segk

using namespace segk;

extern "C" long long segk_attention_workspace(const segk_attention_args* a, int backward) {
  AttnDev p;
  const int rc = attn_check(a, &p, backward != 0);
  if (rc != SEGK_OK) return rc;
  if (!backward) return fwd_part_floats(p, fwd_splits(p, a->dtype)) * 4;
  const long long stats = 2LL * p.N * p.Hk * p.Rp;
  long long part = 0;
  if (p.dk && p.Lk > 0) {
    const int s = attn_dkv_splits(p, a->dtype);
    if (s > 1) part = 2LL * s * p.N * p.Hk * p.Lk * p.D;
  }
  if (p.dq && p.Lk > 0) {
    const int s = attn_dq_splits(p, a->dtype);
    const long long x = s > 1 ? (long long)s * p.N * p.Hk * p.R * p.D : 0;
    if (x > part) part = x;
  }
  return (stats + part) * 4;
}

extern "C" int segk_attention_fwd(const segk_attention_args* a, segk_stream_t stream) {
  AttnDev p;
  const int rc = attn_check(a, &p, false);
  if (rc != SEGK_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  p.tiles = ceil_div(p.R, fwd_rows_per_block(p, a->dtype));
  p.splits = fwd_splits(p, a->dtype);
  const long long need = fwd_part_floats(p, p.splits) * 4;
  if (need > 0) {
    SEGK_REQUIRE(a->workspace && ((uintptr_t)a->workspace & 15) == 0, "attention_fwd: workspace missing or not 16-byte aligned");
    if (a->workspace_bytes < need) {
      set_error("attention_fwd: workspace of %lld bytes, needs %lld", a->workspace_bytes, need);
      return SEGK_WORKSPACE_TOO_SMALL;
    }
    p.part = (float*)a->workspace;
    p.part_ml = p.part + (long long)p.splits * p.N * p.Hk * p.R * p.D;
  }
  const int rc2 = a->dtype == SEGK_BF16 ? dispatch_fwd<bf16_t>(p, st) : dispatch_fwd<float>(p, st);
  if (rc2 != SEGK_OK || p.splits == 1) return rc2;
  const unsigned grid = (unsigned)(((long long)p.N * p.Hk * p.R + 3) / 4);
  SEGK_DISPATCH_DTYPE(a->dtype, T, (attn_join_kernel<T><<<grid, ATTN_THREADS, 0, st>>>(p)));
  SEGK_CHECK_LAUNCH("attention_fwd join");
  return SEGK_OK;
}

extern "C" int segk_attention_bwd(const segk_attention_args* a, segk_stream_t stream) {
  AttnDev p;
  const int rc = attn_check(a, &p, true);
  if (rc != SEGK_OK) return rc;
  SEGK_REQUIRE(p.Lk > 0, "attention_bwd: no keys");
  const long long need = segk_attention_workspace(a, 1);
  SEGK_REQUIRE(a->workspace && ((uintptr_t)a->workspace & 15) == 0, "attention_bwd: workspace missing or not 16-byte aligned");
  if (a->workspace_bytes < need) {
    set_error("attention_bwd: workspace of %lld bytes, needs %lld", a->workspace_bytes, need);
    return SEGK_WORKSPACE_TOO_SMALL;
  }
  hipStream_t st = (hipStream_t)stream;
  const long long rows = (long long)p.N * p.Hk * p.Rp;
  p.row_lse2 = (float*)a->workspace;
  p.row_delta = p.row_lse2 + rows;
  p.part = p.row_delta + rows;
  const int lanes = p.D <= 8 ? 1 : p.D <= 16 ? 2 : p.D <= 32 ? 4 : p.D <= 64 ? 8 : 16;
  const long long blocks = (rows * lanes + ATTN_THREADS - 1) / ATTN_THREADS;
  SEGK_UNSUPPORTED(blocks < 0x7fffffffLL, "attention_bwd: too many rows");
  SEGK_DISPATCH_DTYPE(a->dtype, T, (attn_row_stats_kernel<T><<<(unsigned)blocks, ATTN_THREADS, 0, st>>>(p, lanes)));
  SEGK_CHECK_LAUNCH("attention_bwd statistics");
  if (p.dk) {
    const int r = launch_attn_dkv(p, a->dtype, st);
    if (r != SEGK_OK) return r;
  }
  if (p.dq) return launch_attn_dq(p, a->dtype, st);
  return SEGK_OK;
}
