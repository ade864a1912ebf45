// Multi-head attention, backward: gradient of the queries, dq_i = scale sum_j ds_ij k_j with ds as in attn_dkv.hip.  The
// scores are computed a third time instead of adding dq up with atomics from the key-owning workgroups: two more products
// of seven in all, for sums whose order is fixed.
#include "attn.h"

namespace segk {

constexpr int DQ_KT = 64;

// As the forward kernel: 4 wavefronts of 32 packed rows, tiles of 64 keys, a lane owns one query.
//   S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T.
template <typename T, int DP, bool MASKED>
__global__ __launch_bounds__(ATTN_THREADS, (DP * (int)sizeof(T) >= 384 ? 1 : 2)) void attn_dq_kernel(const AttnDev p) {
  typedef AttnTile<T, DP> Tile;
  typedef AttnRead<T, DP> Rd;
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int TILE_B = DQ_KT * Tile::PITCH;
  constexpr int NP = TILE_B / 4096;
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
  const int row0 = tile * 128;

  const int last_row = min(row0 + 128, p.R) - 1;
  int k_end = p.Lk;
  if (p.causal) k_end = max(0, min(k_end, div_g(p, last_row) + p.off + 1));
  const int all_steps = (k_end + DQ_KT - 1) / DQ_KT;
  const int per = (all_steps + p.splits - 1) / p.splits;
  const int t0 = min(split * per, all_steps), t1 = min(t0 + per, all_steps);

  const int r = row0 + wave * 32 + l31;
  const bool row_in = r < p.R;
  const int rr = row_in ? r : 0;
  const int tok = div_g(p, rr), head = hk * p.G + rr - tok * p.G;
  const long long stat = ((long long)n * p.Hk + hk) * p.Rp + rr;
  const float lse2 = row_in ? p.row_lse2[stat] : INFINITY;
  const float delta = row_in ? p.row_delta[stat] : 0.f;
  const bool row_ok = lse2 != INFINITY;     // (rows without an open key are not read)
  AttnFrag<T> qf[KS], gf[KS];
  {
    const char* qs = p.q.p + ((long long)n * p.q.n + (long long)tok * p.q.l + (long long)head * p.q.h) * (int)sizeof(T);
    const char* gs = p.dout.p + ((long long)n * p.dout.n + (long long)tok * p.dout.l + (long long)head * p.dout.h) * (int)sizeof(T);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = load_frag<T>(qs, ks, h, p.D, row_ok);
      gf[ks] = load_frag<T>(gs, ks, h, p.D, row_ok);
    }
  }
  const int wave_tok0 = __builtin_amdgcn_readfirstlane(div_g(p, min(row0 + wave * 32, p.R - 1)));
  const unsigned char* const mrow =
      MASKED && p.mask ? p.mask + n * p.m_n + (long long)head * p.m_h + (long long)tok * p.m_q : nullptr;

  const int lin = wave * 1024 + lane * 16;
  const int st_row = lin / Tile::PITCH;
  const int st_chunk = ((lin % Tile::PITCH) >> 4) ^ Tile::swz(st_row);
  const bool st_ok = st_chunk * 16 < p.D * (int)sizeof(T);
  const unsigned k_step_b = (unsigned)(p.k.l * (int)sizeof(T)), v_step_b = (unsigned)(p.v.l * (int)sizeof(T));
  const char* const kbase = p.k.p + ((long long)n * p.k.n + (long long)hk * p.k.h) * (int)sizeof(T);
  const char* const vbase = p.v.p + ((long long)n * p.v.n + (long long)hk * p.v.h) * (int)sizeof(T);
  const unsigned char* const kmask = MASKED && p.kmask ? p.kmask + n * p.km_n : nullptr;
  const unsigned lds0 = lds_addr(smem) + wave * 1024;
  auto stage = [&](int t, int buf) {
    const int key0 = t * DQ_KT;
    const u32x4 kr = buffer_of(kbase + (long long)key0 * k_step_b);
    const u32x4 vr = buffer_of(vbase + (long long)key0 * v_step_b);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int row = st_row + i * (4096 / Tile::PITCH);
      bool ok = st_ok && key0 + row < p.Lk;
      if (MASKED && kmask && ok) ok = kmask[(long long)(key0 + row) * p.km_k] != 0;
      const unsigned lds = lds0 + buf * (2 * TILE_B) + i * 4096;
      dma_1k(kr, lds, ok ? row * k_step_b + st_chunk * 16 : ATTN_OOB);
      dma_1k(vr, lds + TILE_B, ok ? row * v_step_b + st_chunk * 16 : ATTN_OOB);
    }
  };

  f32x16 dq[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dq[db] = zero16();

  if (t0 < t1) stage(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    tile_barrier();
    if (t + 1 < t1) stage(t + 1, buf ^ 1);
    const char* kt = smem + buf * (2 * TILE_B);
    const char* vt = kt + TILE_B;
    const int key0 = t * DQ_KT;
    const bool ragged = key0 + DQ_KT > p.Lk || (p.causal && key0 + DQ_KT - 1 > wave_tok0 + p.off);
    const int lim = p.causal ? min(p.Lk - 1, tok + p.off) : p.Lk - 1;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma32(s, Rd::rows(kt, kb * 32, ks, lane), qf[ks]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma32(dp, Rd::rows(vt, kb * 32, ks, lane), gf[ks]);
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = exp2_fast(fmaf(s[i], p.scale_log2, -lse2)) * (dp[i] - delta);
      if (MASKED || ragged) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = key0 + kb * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
          bool open = j <= lim;
          if (MASKED && open) {
            if (kmask) open = kmask[(long long)j * p.km_k] != 0;
            if (mrow && open) open = mrow[(long long)j * p.m_k] != 0;
          }
          dp[i] = open ? dp[i] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const AttnFrag<T> sf = pack_frag<T>(dp, j);
#pragma unroll
        for (int db = 0; db < DB; ++db) mma32(dq[db], Rd::cols(kt, kb * 32 + j * 16, db * 32, lane), sf);
      }
    }
  }

  if (!row_in) return;
  const long long at = (((long long)n * p.Lq + tok) * p.Hq + head) * p.D;
  if (p.splits == 1) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = db * 32 + 2 * i + 4 * h;
        if (d < p.D)
          store4<T>(p.dq + at * (int)sizeof(T), d, dq[db][i] * p.scale, dq[db][i + 1] * p.scale, dq[db][i + 2] * p.scale, dq[db][i + 3] * p.scale);
      }
  } else {
    char* dst = (char*)(p.part + (long long)split * p.N * p.Lq * p.Hq * p.D + at);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = db * 32 + 2 * i + 4 * h;
        if (d < p.D) store4<float>(dst, d, dq[db][i], dq[db][i + 1], dq[db][i + 2], dq[db][i + 3]);
      }
  }
}

int attn_dq_splits(const AttnDev& p, int dtype) {
  const long long blocks = (long long)ceil_div(p.R, 128) * p.N * p.Hk;
  const int steps = ceil_div(p.Lk, DQ_KT);
  if (blocks >= 256 || steps < 4) return 1;
  long long s = (512 + blocks - 1) / blocks;
  if (s > steps / 2) s = steps / 2;
  return s < 1 ? 1 : (int)s;
}

template <typename T, int DP>
static int launch(const AttnDev& p, hipStream_t st) {
  const int lds = 4 * DQ_KT * AttnTile<T, DP>::PITCH;
  const long long blocks = (long long)p.tiles * p.splits * p.N * p.Hk;
  SEGK_UNSUPPORTED(blocks < 0x7ffffff0LL, "attention_bwd: too many workgroups");
  auto kern = p.mask || p.kmask ? attn_dq_kernel<T, DP, true> : attn_dq_kernel<T, DP, false>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("attention_bwd: %s", hipGetErrorString(e));
      return SEGK_HIP_ERROR;
    }
  }
  kern<<<(unsigned)((blocks + 7) / 8 * 8), ATTN_THREADS, lds, st>>>(p);
  SEGK_CHECK_LAUNCH("attention_bwd queries");
  return SEGK_OK;
}

template <typename T>
static int dispatch(const AttnDev& p, hipStream_t st) {
  if (p.D <= 32) return launch<T, 32>(p, st);
  if (p.D <= 64) return launch<T, 64>(p, st);
  if (p.D <= 96) return launch<T, 96>(p, st);
  return launch<T, 128>(p, st);
}

int launch_attn_dq(AttnDev p, int dtype, hipStream_t st) {
  p.tiles = ceil_div(p.R, 128);
  p.splits = attn_dq_splits(p, dtype);
  const int rc = dtype == SEGK_BF16 ? dispatch<bf16_t>(p, st) : dispatch<float>(p, st);
  if (rc != SEGK_OK || p.splits == 1) return rc;
  const long long all = (long long)p.N * p.Lq * p.Hq * p.D;
  return launch_attn_sum(p.part, all, p.splits, p.scale, p.dq, all, dtype, st);
}

}  // namespace segk
