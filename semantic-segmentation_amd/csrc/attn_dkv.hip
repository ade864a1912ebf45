// Multi-head attention, backward: gradients of keys and values.  With p = exp(s - lse) computed again from q, k and lse:
//   dv_j = sum_i p_ij dout_i,   ds_ij = p_ij (dout_i . v_j - delta_i),   dk_j = scale sum_i ds_ij q_i.
// A workgroup owns 128 keys and walks over the packed rows (tokens x heads of the group): shared heads add up in its
// registers, nothing is added atomically, every sum has a fixed order.
#include "attn.h"

namespace segk {

constexpr int QT = 64;   // rows per step

// 4 wavefronts of 32 keys.  Scores are computed with queries as rows (a lane owns one key), so P and dS are the operands
// of dV^T = dO^T P and dK^T = Q^T dS as they lie; K and V of the wavefront's keys stay in registers, Q and dO tiles of 64
// rows are staged through LDS and read both along rows and along columns.
template <typename T, int DP, bool MASKED>
__global__ __launch_bounds__(ATTN_THREADS, (DP * (int)sizeof(T) >= 192 ? 1 : 2)) void attn_dkv_kernel(const AttnDev p) {
  typedef AttnTile<T, DP> Tile;
  typedef AttnRead<T, DP> Rd;
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int TILE_B = QT * Tile::PITCH;
  constexpr int NP = TILE_B / 4096;
  constexpr int STAGE_B = 2 * TILE_B + 512;      // Q tile, dO tile, 64 lse, 64 delta
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
  int w = xcd_contiguous(p.tiles * p.splits * p.N * p.Hk);
  if (w < 0) return;
  const int split = w % p.splits;
  w /= p.splits;
  const int tile = w % p.tiles;
  w /= p.tiles;
  const int hk = w % p.Hk, n = w / p.Hk;
  const int key_wg = tile * 128;
  const int key = key_wg + wave * 32 + l31;

  const int all_steps = p.Rp / QT;
  int first = 0;
  if (p.causal) first = min(all_steps, max(0, key_wg - p.off) >= p.Lq ? all_steps : max(0, key_wg - p.off) * p.G / QT);
  const int per = (all_steps - first + p.splits - 1) / p.splits;
  const int t0 = min(first + split * per, all_steps), t1 = min(t0 + per, all_steps);

  bool key_ok = key < p.Lk;
  if (MASKED && p.kmask && key_ok) key_ok = p.kmask[n * p.km_n + (long long)key * p.km_k] != 0;
  AttnFrag<T> kf[KS], vf[KS];
  {
    const long long kk = key_ok ? key : 0;
    const char* ks_ = p.k.p + ((long long)n * p.k.n + kk * p.k.l + (long long)hk * p.k.h) * (int)sizeof(T);
    const char* vs_ = p.v.p + ((long long)n * p.v.n + kk * p.v.l + (long long)hk * p.v.h) * (int)sizeof(T);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kf[ks] = load_frag<T>(ks_, ks, h, p.D, key_ok);
      vf[ks] = load_frag<T>(vs_, ks, h, p.D, key_ok);
    }
  }

  const int lin = wave * 1024 + lane * 16;
  const int st_row = lin / Tile::PITCH;
  const int st_chunk = ((lin % Tile::PITCH) >> 4) ^ Tile::swz(st_row);
  const bool st_ok = st_chunk * 16 < p.D * (int)sizeof(T);
  const char* const qbase = p.q.p + ((long long)n * p.q.n + (long long)hk * p.G * p.q.h) * (int)sizeof(T);
  const char* const gbase = p.dout.p + ((long long)n * p.dout.n + (long long)hk * p.G * p.dout.h) * (int)sizeof(T);
  const float* const lse2 = p.row_lse2 + ((long long)n * p.Hk + hk) * p.Rp;
  const float* const delta = p.row_delta + ((long long)n * p.Hk + hk) * p.Rp;
  const unsigned char* const mkey =
      MASKED && p.mask ? p.mask + n * p.m_n + (long long)hk * p.G * p.m_h + (long long)(key < p.Lk ? key : 0) * p.m_k : nullptr;
  // Rows without an open key exist under masks and where the diagonal starts above the keys: they are not read, so that
  // whatever their memory holds meets no product.
  const bool empty_rows = MASKED || (p.causal && p.off < 0);
  const unsigned lds0 = lds_addr(smem);
  auto stage = [&](int t, int buf) {
    const int row0 = t * QT;
    const int tok0 = __builtin_amdgcn_readfirstlane(div_g(p, row0));
    const u32x4 qr = buffer_of(qbase + (long long)tok0 * p.q.l * (int)sizeof(T));
    const u32x4 gr = buffer_of(gbase + (long long)tok0 * p.dout.l * (int)sizeof(T));
    const unsigned at = lds0 + buf * STAGE_B;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = row0 + st_row + i * (4096 / Tile::PITCH);
      bool ok = st_ok && r < p.R;
      if (empty_rows && ok) ok = lse2[r] != INFINITY;
      const int tok = div_g(p, r), hg = r - tok * p.G;
      const unsigned qo = (unsigned)(((tok - tok0) * p.q.l + hg * p.q.h) * (int)sizeof(T)) + st_chunk * 16;
      const unsigned go = (unsigned)(((tok - tok0) * p.dout.l + hg * p.dout.h) * (int)sizeof(T)) + st_chunk * 16;
      dma_1k(qr, at + wave * 1024 + i * 4096, ok ? qo : ATTN_OOB);
      dma_1k(gr, at + TILE_B + wave * 1024 + i * 4096, ok ? go : ATTN_OOB);
    }
    if (wave == 0) dma_256(buffer_of((const char*)(lse2 + row0)), at + 2 * TILE_B, lane * 4);
    if (wave == 1) dma_256(buffer_of((const char*)(delta + row0)), at + 2 * TILE_B + 256, lane * 4);
  };

  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dk[db] = dv[db] = zero16();

  if (t0 < t1) stage(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    tile_barrier();
    if (t + 1 < t1) stage(t + 1, buf ^ 1);
    const char* qt = smem + buf * STAGE_B;
    const char* gt = qt + TILE_B;
    const float* st = reinterpret_cast<const float*>(qt + 2 * TILE_B);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const int row0 = t * QT + rb * 32;
      if (row0 >= p.R) break;
      unsigned char open[16];
      if (MASKED && mkey) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = min(row0 + 8 * (i >> 2) + 4 * h + (i & 3), p.R - 1);
          const int tok = div_g(p, r);
          open[i] = mkey[(long long)(r - tok * p.G) * p.m_h + (long long)tok * p.m_q];
        }
      }
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma32(s, Rd::rows(qt, rb * 32, ks, lane), kf[ks]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma32(dp, Rd::rows(gt, rb * 32, ks, lane), vf[ks]);
      float ls[16], dl[16];
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(st + rb * 32 + 2 * i + 4 * h);
        const f32x4 b = *reinterpret_cast<const f32x4*>(st + 64 + rb * 32 + 2 * i + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ls[i + e] = a[e];
          dl[i + e] = b[e];
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = exp2_fast(fmaf(s[i], p.scale_log2, -ls[i]));
      // closed pairs (a closed key's products are those of zeros; the padding rows' lse is +inf)
      if (p.causal && key_wg + 127 > div_g(p, row0) + p.off) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = row0 + 8 * (i >> 2) + 4 * h + (i & 3);
          s[i] = key <= div_g(p, r) + p.off ? s[i] : 0.f;
        }
      }
      if (MASKED) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = key_ok && (!mkey || open[i] != 0) ? s[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = s[i] * (dp[i] - dl[i]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const AttnFrag<T> pf = pack_frag<T>(s, j), sf = pack_frag<T>(dp, j);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          mma32(dv[db], Rd::cols(gt, rb * 32 + j * 16, db * 32, lane), pf);
          mma32(dk[db], Rd::cols(qt, rb * 32 + j * 16, db * 32, lane), sf);
        }
      }
    }
  }

  if (key >= p.Lk) return;
  const long long at = (((long long)n * p.Lk + key) * p.Hk + hk) * p.D;
  if (p.splits == 1) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = db * 32 + 2 * i + 4 * h;
        if (d < p.D) {
          store4<T>(p.dk + at * (int)sizeof(T), d, dk[db][i] * p.scale, dk[db][i + 1] * p.scale, dk[db][i + 2] * p.scale, dk[db][i + 3] * p.scale);
          store4<T>(p.dv + at * (int)sizeof(T), d, dv[db][i], dv[db][i + 1], dv[db][i + 2], dv[db][i + 3]);
        }
      }
  } else {
    const long long all = (long long)p.N * p.Lk * p.Hk * p.D;
    char* pk = (char*)(p.part + (long long)split * 2 * all + at);
    char* pv = (char*)(p.part + (long long)split * 2 * all + all + at);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = db * 32 + 2 * i + 4 * h;
        if (d < p.D) {
          store4<float>(pk, d, dk[db][i], dk[db][i + 1], dk[db][i + 2], dk[db][i + 3]);
          store4<float>(pv, d, dv[db][i], dv[db][i + 1], dv[db][i + 2], dv[db][i + 3]);
        }
      }
  }
}

// out = scale * sum over the parts, in part order; 4 elements a thread (every length is a multiple of 8)
template <typename T>
__global__ __launch_bounds__(ATTN_THREADS) void attn_sum_kernel(const float* __restrict__ part, long long part_stride, int parts,
                                                                float scale, char* __restrict__ out, long long count) {
  const long long i = ((long long)blockIdx.x * ATTN_THREADS + threadIdx.x) * 4;
  if (i >= count) return;
  f32x4 v = *reinterpret_cast<const f32x4*>(part + i);
  for (int s = 1; s < parts; ++s) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(part + s * part_stride + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += x[e];
  }
  store4<T>(out + i * (int)sizeof(T), 0, v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
}

int launch_attn_sum(const float* part, long long part_stride, int parts, float scale, char* out, long long count, int dtype,
                    hipStream_t st) {
  const long long blocks = (count / 4 + ATTN_THREADS - 1) / ATTN_THREADS;
  SEGK_UNSUPPORTED(blocks < 0x7fffffffLL, "attention_bwd: too many elements");
  SEGK_DISPATCH_DTYPE(dtype, T, (attn_sum_kernel<T><<<(unsigned)blocks, ATTN_THREADS, 0, st>>>(part, part_stride, parts, scale, out, count)));
  SEGK_CHECK_LAUNCH("attention_bwd sum");
  return SEGK_OK;
}

int attn_dkv_splits(const AttnDev& p, int dtype) {
  const long long blocks = (long long)ceil_div(p.Lk, 128) * p.N * p.Hk;
  const int steps = p.Rp / QT;
  if (blocks >= 256 || steps < 4) return 1;
  long long s = (512 + blocks - 1) / blocks;
  if (s > steps / 2) s = steps / 2;
  return s < 1 ? 1 : (int)s;
}

template <typename T, int DP>
static int launch(const AttnDev& p, hipStream_t st) {
  const int lds = 2 * (2 * QT * AttnTile<T, DP>::PITCH + 512);
  const long long blocks = (long long)p.tiles * p.splits * p.N * p.Hk;
  SEGK_UNSUPPORTED(blocks < 0x7ffffff0LL, "attention_bwd: too many workgroups");
  auto kern = p.mask || p.kmask ? attn_dkv_kernel<T, DP, true> : attn_dkv_kernel<T, DP, false>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("attention_bwd: %s", hipGetErrorString(e));
      return SEGK_HIP_ERROR;
    }
  }
  kern<<<(unsigned)((blocks + 7) / 8 * 8), ATTN_THREADS, lds, st>>>(p);
  SEGK_CHECK_LAUNCH("attention_bwd keys");
  return SEGK_OK;
}

template <typename T>
static int dispatch(const AttnDev& p, hipStream_t st) {
  if (p.D <= 32) return launch<T, 32>(p, st);
  if (p.D <= 64) return launch<T, 64>(p, st);
  if (p.D <= 96) return launch<T, 96>(p, st);
  return launch<T, 128>(p, st);
}

int launch_attn_dkv(AttnDev p, int dtype, hipStream_t st) {
  p.tiles = ceil_div(p.Lk, 128);
  p.splits = attn_dkv_splits(p, dtype);
  const int rc = dtype == SEGK_BF16 ? dispatch<bf16_t>(p, st) : dispatch<float>(p, st);
  if (rc != SEGK_OK || p.splits == 1) return rc;
  const long long all = (long long)p.N * p.Lk * p.Hk * p.D;
  const int rk = launch_attn_sum(p.part, 2 * all, p.splits, p.scale, p.dk, all, dtype, st);
  if (rk != SEGK_OK) return rk;
  return launch_attn_sum(p.part + all, 2 * all, p.splits, 1.f, p.dv, all, dtype, st);
}

}  // namespace segk
