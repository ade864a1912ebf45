// Multi-head attention, backward: gradient of the queries, dq_i = scale sum_j ds_ij k_j with ds as in attn_dkv.hip.  The
// scores are computed a third time instead of adding dq up with atomics from the key-owning workgroups: two more products
// of seven in all, for sums whose order is fixed.
#include <type_traits>

#include "attn.h"

namespace segk {

// As the forward kernel (attn_fwd.hip): a lane owns one query,
//   S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T.
// bf16: dS goes into its product as two operands, the rounded value and what the rounding left over.  A row's dS sum to zero,
// so that a query's gradient is a difference of large terms and would carry their roundings: rms error against 64 bits 0.0024
// (every pixel's own map) to 0.0027 (class queries under masks) of the gradient's size instead of 0.0017, the final
// rounding's alone.  It costs a fourth product in three: 100 -> 120 us (16 images of 961 tokens, 16 heads of 64 channels).
// Matrix-bound on long maps: 4 images of 4225 tokens, 16 heads over 4 of 128 channels: 0.96 ms, 1220 TFLOP/s with the fourth
// product, matrix cores busy 65 % of the cycles.
// Wavefronts to a SIMD: what is fastest.  At 64 channels under masks 3 of them spill 8 registers: 16 images of 961 tokens, 16
// heads 121 us, 2 without spills 136 us.
// What a row needs: its statistics and its query and output gradient in registers (zeros for a row that has no open key,
// whatever its memory holds).
template <typename T, int DP>
struct AttnGradRow {
  static constexpr int KS = DP / 16;
  int tok, head;
  float lse2, minus;     // base-2 lse, -delta
  AttnFrag<T> qf[KS], gf[KS];
  __device__ __forceinline__ AttnGradRow(const AttnDev& p, int n, int hk, int r, int h) {
    const bool in = r < p.R;
    const int rr = in ? r : 0;
    tok = div_g(p, rr);
    head = hk * p.G + rr - tok * p.G;
    const long long stat = ((long long)n * p.Hk + hk) * p.Rp + rr;
    lse2 = in ? p.row_lse2[stat] : INFINITY;
    minus = in ? p.minus_delta[stat] : 0.f;
    const char* qs = p.q.p + ((long long)n * p.q.n + (long long)tok * p.q.l + (long long)head * p.q.h) * (int)sizeof(T);
    const char* gs = p.dout.p + ((long long)n * p.dout.n + (long long)tok * p.dout.l + (long long)head * p.dout.h) * (int)sizeof(T);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = load_frag<T>(qs, ks, h, p.D, in);
      gf[ks] = load_frag<T>(gs, ks, h, p.D, in);
    }
    const bool live = lse2 != INFINITY;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (unsigned e = 0; e < sizeof(qf[0].v) / sizeof(qf[0].v[0]); ++e) {
        qf[ks].v[e] = live ? qf[ks].v[e] : 0;
        gf[ks].v[e] = live ? gf[ks].v[e] : 0;
      }
  }
};

template <typename T, int DP, bool MASKED>
__global__ __launch_bounds__(ATTN_THREADS, (DP * (int)sizeof(T) >= 384 ? 1 : DP * (int)sizeof(T) > 128 ? 2 : 3)) void attn_dq_kernel(const AttnDev p) {
  typedef AttnTile<T, DP> Tile;
  constexpr int KT = 64, KS = DP / 16, DB = DP / 32;
  constexpr int TILE_B = KT * Tile::PITCH;
  extern __shared__ __attribute__((aligned(1024))) char smem[];   // 2 x (K tile, V tile); MASKED: 2 x 64 starts

  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
  const AttnWork w = attn_work(p);
  if (w.n < 0) return;
  const int n = w.n, hk = w.hk;
  const int row0 = w.tile * 128 + wave * 32;

  const AttnStage<T, DP> st(p, n, hk, wave, lane, smem);
  const unsigned char* const kmask = MASKED && p.kmask ? p.kmask + n * p.km_n : nullptr;
  AttnKeyMask km(kmask, p.km_k, p.Lk, lane);
  char* const start0 = smem + 4 * TILE_B;

  const int last_row = min(w.tile * 128 + 128, p.R) - 1;
  int k_end = p.Lk;
  if (p.causal) k_end = max(0, min(k_end, div_g(p, last_row) + p.off + 1));
  if (MASKED && kmask) k_end = min(k_end, last_open_key(kmask, p.km_k, k_end, lane) + 1);
  const int all_steps = (k_end + KT - 1) / KT;
  const int per = (all_steps + w.parts - 1) / w.parts;
  const int t0 = min(w.part * per, all_steps), t1 = min(t0 + per, all_steps);
  auto stage = [&](int t, int buf) __attribute__((always_inline)) {
    unsigned long long bits = 0;
    if (MASKED) {
      bits = km.next();
      km.load((t + 1) * KT);
      if (wave == 0) write_start(start0 + buf * 256, bits, lane);
    }
    st.template both<MASKED>(p, t * KT, buf, bits);
  };
  if (t0 < t1) {               // the first tile is asked for before anything else
    if (MASKED) km.load(t0 * KT);
    stage(t0, 0);
  }

  const int r = row0 + l31;
  const AttnGradRow<T, DP> row(p, n, hk, r, h);
  const int wave_tok0 = __builtin_amdgcn_readfirstlane(div_g(p, min(row0, p.R - 1)));
  const int lim = (p.causal ? min(p.Lk - 1, row.tok + p.off) : p.Lk - 1) - 4 * h;
  const int ragged0 = p.causal ? min(p.Lk, wave_tok0 + p.off + 1) : p.Lk;
  AttnPairMask pm(MASKED && p.mask ? p.mask + n * p.m_n + (long long)row.head * p.m_h + (long long)row.tok * p.m_q : nullptr, p.m_k, p.Lk, h);
  if (MASKED && pm.row && t0 < t1) pm.load(t0 * KT);

  f32x16 dq[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dq[db] = zero16();
  // The score gradients' products start from -delta where 16 registers can be spared for it (64 channels: 105 -> 101 us).
  constexpr bool START = DP * (int)sizeof(T) <= 128;
  f32x16 start = zero16();
  if (START) {
#pragma unroll
    for (int i = 0; i < 16; ++i) start[i] = row.minus;
  }

  const AttnLane<T, DP> ln(smem, lane);
  const bool idle = row0 >= p.R;
  auto step = [&](int t, auto buf_) __attribute__((always_inline)) {
    constexpr int buf = buf_.value, kt = buf * 2 * TILE_B, vt = kt + TILE_B;
    tile_barrier();
    if (idle) {
      if (t + 1 < t1) stage(t + 1, buf ^ 1);
      return;
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int key0 = t * KT + kb * 32, at = kb * 32 * Tile::PITCH;
      f32x16 s = MASKED ? read_start(start0 + buf * 256 + kb * 128, h) : zero16(), dp = START ? start : zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma32(s, ln.rows(kt + at, ks), row.qf[ks]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma32(dp, ln.rows(vt + at, ks), row.gf[ks]);
      if (kb == 0 && t + 1 < t1) stage(t + 1, buf ^ 1);       // (behind the first LDS reads: see the forward kernel)
      if (key0 + 32 > ragged0) close_past(s, -INFINITY, lim - key0);
      if (MASKED && pm.row) {
        close_pairs(s, -INFINITY, pm.w);
        pm.load(key0 + 32);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = exp2_fast(fmaf(s[i], p.scale_log2, -row.lse2)) * (START ? dp[i] : dp[i] + row.minus);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const AttnFrag<T> sf = pack_frag<T>(dp, j);
        AttnFrag<T> rest;
        if constexpr (sizeof(T) == 2) rest = pack_rest(dp, j, sf);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const AttnFrag<T> kf = ln.cols(kt + at + j * 16 * Tile::PITCH, db);
          mma32(dq[db], kf, sf);
          if constexpr (sizeof(T) == 2) mma32(dq[db], kf, rest);
        }
      }
    }
  };
  constexpr std::integral_constant<int, 0> zero;
  constexpr std::integral_constant<int, 1> one;
  int t = t0;
  for (; t + 1 < t1; t += 2) {
    step(t, zero);
    step(t + 1, one);
  }
  if (t < t1) step(t, zero);

  if (r >= p.R) return;
  if (w.parts == 1) {
    const long long at = (((long long)n * p.Lq + row.tok) * p.Hq + row.head) * p.D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = db * 32 + 2 * i + 4 * h;
        if (d < p.D)
          store4<T>(p.dq + at * (int)sizeof(T), d, dq[db][i] * p.scale, dq[db][i + 1] * p.scale, dq[db][i + 2] * p.scale, dq[db][i + 3] * p.scale);
      }
  } else {
    char* dst = (char*)(p.part + (((long long)w.slot * p.parts + w.part) * p.tile_rows + wave * 32 + l31) * p.D);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = db * 32 + 2 * i + 4 * h;
        if (d < p.D) store4<float>(dst, d, dq[db][i], dq[db][i + 1], dq[db][i + 2], dq[db][i + 3]);
      }
  }
}

// Sums the parts of the tiles that were cut, in part order: 4 channels of one row a thread.
template <typename T>
__global__ __launch_bounds__(ATTN_THREADS) void attn_dq_sum_kernel(const AttnDev p) {
  const long long x = (long long)blockIdx.x * ATTN_THREADS + threadIdx.x;
  const int quads = p.D / 4;
  const long long line = x / quads;
  const int d = (int)(x - line * quads) * 4;
  if (line >= (long long)p.rest * p.tile_rows) return;
  const int slot = (int)(line / p.tile_rows), row = (int)(line - (long long)slot * p.tile_rows);
  AttnWork w;
  attn_decode_tile(p, p.whole + slot, &w);
  const int rr = w.tile * 128 + row, parts = attn_tile_parts(p, w.tile);
  if (rr >= p.R || parts == 1) return;       // (a tile in one part is finished)
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8      // (one part after the other: 9 -> 4 us where 21 class queries have 26 parts)
  for (int s = 0; s < parts; ++s) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(p.part + (((long long)slot * p.parts + s) * p.tile_rows + row) * p.D + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += y[e];
  }
  const int tok = div_g(p, rr), head = w.hk * p.G + rr - tok * p.G;
  store4<T>(p.dq + (((long long)w.n * p.Lq + tok) * p.Hq + head) * p.D * (int)sizeof(T), d, v[0] * p.scale, v[1] * p.scale,
            v[2] * p.scale, v[3] * p.scale);
}

template <typename T, int DP>
static int launch(AttnDev* p, bool plan_only, hipStream_t st) {
  static std::atomic<int> seen[2][ATTN_DEVICES];
  const bool masked = p->mask || p->kmask;
  const int lds = 4 * 64 * AttnTile<T, DP>::PITCH + (masked ? 512 : 0);
  void (*const kern)(const AttnDev) = masked ? attn_dq_kernel<T, DP, true> : attn_dq_kernel<T, DP, false>;
  const int per_cu = attn_occupancy((const void*)kern, lds, seen[masked]);
  if (per_cu < 0) return per_cu;
  p->tiles = ceil_div(p->R, 128);
  p->loop_rows = 0;
  SEGK_UNSUPPORTED((long long)p->tiles * p->N * p->Hk < 0x40000000LL, "attention_bwd: too many workgroups");
  const long long grid = attn_deal(p, per_cu, ceil_div(p->Lk, 64), 2);
  if (plan_only) return SEGK_OK;
  kern<<<(unsigned)grid, ATTN_THREADS, lds, st>>>(*p);
  SEGK_CHECK_LAUNCH("attention_bwd queries");
  if (p->parts > 1) {
    const long long blocks = ((long long)p->rest * p->tile_rows * (p->D / 4) + ATTN_THREADS - 1) / ATTN_THREADS;
    attn_dq_sum_kernel<T><<<(unsigned)blocks, ATTN_THREADS, 0, st>>>(*p);
    SEGK_CHECK_LAUNCH("attention_bwd queries' sum");
  }
  return SEGK_OK;
}

template <typename T>
static int dispatch(AttnDev* p, bool plan_only, hipStream_t st) {
  if (p->D <= 32) return launch<T, 32>(p, plan_only, st);
  if (p->D <= 64) return launch<T, 64>(p, plan_only, st);
  if (p->D <= 96) return launch<T, 96>(p, plan_only, st);
  return launch<T, 128>(p, plan_only, st);
}

int attn_dq(AttnDev* p, int dtype, bool plan_only, hipStream_t st) {
  return dtype == SEGK_BF16 ? dispatch<bf16_t>(p, plan_only, st) : dispatch<float>(p, plan_only, st);
}

}  // namespace segk
