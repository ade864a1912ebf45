// Multi-head attention, backward: gradients of keys and values.  With p = exp(s - lse) computed again from q, k and lse:
//   dv_j = sum_i p_ij dout_i,   ds_ij = p_ij (dout_i . v_j - delta_i),   dk_j = scale sum_i ds_ij q_i.
// A workgroup owns 128 keys and walks over the packed rows (tokens x heads of the group): shared heads add up in its
// registers, nothing is added atomically, every sum has a fixed order.
// bf16: P and dS are rounded to operands of their products, as the probabilities of the forward pass are: rms error against 64
// bits 0.0023 of the gradient's size, 0.0017 of it the final rounding.  Up to 64 rows they go in as two operands each, the rounded
// value and what the rounding left over: 0.0017.  A key's gradient is then a sum of few terms, often one, whose roundings nothing
// evens out (0.0024 and more for dk of class queries whose windows hold few keys, where plain fp32 has 0.0016), and the products
// are not what such a kernel waits for.
// Time of the two more products, 8 images of 4225 keys, 8 heads of 32 (pair mask) / 64 / 64 (key mask) / 128 channels:
//   21 rows 26.5 -> 28.0, 40 -> 42, 37 -> 40, 77 -> 78 us     64 rows 32 -> 35, 45 -> 47, 39 -> 45, 89 -> 92
//   256 rows 77 -> 87, 66 -> 78, 60 -> 83, 142 -> 156         1024 rows 254 -> 298, 170 -> 226, 145 -> 217, 354 -> 430
#include <type_traits>

#include "attn.h"

namespace segk {

// Rows of a tile: 32, or 64 where 32 are less than a KiB for every wavefront to stage (64 channels, bf16, 16 images of 961
// tokens, 16 heads: 159 us with 32, 170 us with 64).
template <typename T, int DP>
constexpr int dkv_rows() { return AttnTile<T, DP>::PITCH < 128 ? 64 : 32; }

// 4 wavefronts of 32 keys.  Scores are computed with queries as rows (a lane owns one key), so P and dS are the operands
// of dV^T = dO^T P and dK^T = Q^T dS as they lie.  K of the wavefront's keys stays in registers; Q and dO tiles of QT rows
// are staged through LDS and read both along rows and along columns.
// V lies in LDS, too: at 128 channels the registers it would take leave one wavefront to a SIMD instead of two, which cover
// each other's exponentials (2.49 -> 1.13 ms in the first case below); at 64 channels 165 -> 159 us (the second); at
// 32 it costs 1.5 % (class queries, 47.7 -> 48.5 us), which is not worth a second form.
// Wavefronts to a SIMD: what is fastest.  Registers spilled: 4 with a pair mask at 32 channels (3 wavefronts 49 us for class
// queries, 2 without spills 58, 4 wavefronts 64), 8 with a key mask at 128 channels (2 wavefronts 97 us for 4 images of 1089
// tokens, 1 129 us), 2 in fp32 with a pair mask at 64 channels (2 wavefronts 334 us, 1 388 us).  With a pair mask at 128 channels
// 2 wavefronts would spill 66: 4 images of 4225 tokens, 8 heads 1660 us, 1 wavefront 1366 us; 8 images of 1089 tokens, 16 heads
// over 4 587 and 375 us.
// Matrix-bound on long maps: 4 images of 4225 tokens, 16 heads over 4 of 128 channels: 1.05 to 1.13 ms for four products,
// 1060 TFLOP/s, matrix cores busy 56 % of the cycles.  16 images of 961 tokens under key masks, 16 heads of 64 channels:
// 155 us; a third of the tiles is padding and ends at once, so that 1.4 of 2 wavefronts to a SIMD are there on average.  A
// pipelined form (three blocks in flight, K and V in registers) took 155 us there, too, and 1.45 ms instead of 1.13 at 128
// channels.
// MASKS: 0 none, 1 a key mask, 2 a pair mask (and perhaps a key mask)
// REST: P and dS as two operands each (see above)
template <typename T, int DP, int MASKS, bool REST>
__global__ __launch_bounds__(ATTN_THREADS, (DP * (int)sizeof(T) >= 384 || (MASKS == 2 && DP >= 128) ? 1 : DP * (int)sizeof(T) > 64 ? 2 : 3)) void attn_dkv_kernel(const AttnDev p) {
  typedef AttnTile<T, DP> Tile;
  typedef AttnPiece<T, DP> Piece;
  constexpr int QT = dkv_rows<T, DP>();
  constexpr bool MASKED = MASKS != 0, PAIRS = MASKS == 2;
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int TILE_B = QT * Tile::PITCH;
  constexpr int STAGE_B = 2 * TILE_B + 512;      // Q tile, dO tile, lse, delta
  extern __shared__ __attribute__((aligned(1024))) char smem[];   // 2 stages, V

  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
  const AttnWork w = attn_work(p);
  if (w.n < 0) return;
  const int n = w.n, hk = w.hk;
  const int key_wg = w.tile * 128;
  const int key = key_wg + wave * 32 + l31;

  const int all_steps = (p.R + QT - 1) / QT;
  int first = 0;
  if (p.causal) first = max(0, key_wg - p.off) >= p.Lq ? all_steps : max(0, key_wg - p.off) * p.G / QT;
  const int per = (all_steps - first + w.parts - 1) / w.parts;
  const int t0 = min(first + w.part * per, all_steps);
  int t1 = min(t0 + per, all_steps);

  bool key_ok = key < p.Lk;
  if (MASKED && p.kmask && key_ok) key_ok = p.kmask[n * p.km_n + (long long)key * p.km_k] != 0;
  // (a tile without an open key has nothing to walk over: its gradients are zeros)
  if (MASKED && p.kmask && !any_open_key(p.kmask + n * p.km_n, p.km_k, key_wg, p.Lk, lane)) t1 = t0;

  const AttnLane<T, DP> ln(smem, lane);
  const AttnLane<T, DP> lv(smem + wave * 32 * Tile::PITCH, lane);     // this wavefront's rows of V
  const Piece pc(wave, lane);
  const int row_b = p.D * (int)sizeof(T);
  const char* const qbase = p.q.p + ((long long)n * p.q.n + (long long)hk * p.G * p.q.h) * (int)sizeof(T);
  const char* const gbase = p.dout.p + ((long long)n * p.dout.n + (long long)hk * p.G * p.dout.h) * (int)sizeof(T);
  const float* const lse2 = p.row_lse2 + ((long long)n * p.Hk + hk) * p.Rp;
  const float* const delta = p.minus_delta + ((long long)n * p.Hk + hk) * p.Rp;
  const unsigned char* const mkey =
      PAIRS ? p.mask + n * p.m_n + (long long)hk * p.G * p.m_h + (long long)(key < p.Lk ? key : 0) * p.m_k : nullptr;
  // Rows without an open key exist under masks and where the diagonal starts above the keys: they are not read, so that
  // whatever their memory holds meets no product.
  const bool empty_rows = MASKED || (p.causal && p.off < 0);
  // Where the group's heads divide a tile evenly, a lane's place relative to the tile's first token never changes.
  const bool even = QT % p.G == 0;
  constexpr int NPC = TILE_B / 4096;
  unsigned qo[NPC], go[NPC];
  auto place = [&](int r, int tok0, int c, const AttnView& x) {
    const int tok = div_g(p, r), hg = r - tok * p.G;
    return c < row_b ? (unsigned)(((tok - tok0) * x.l + hg * x.h) * (int)sizeof(T)) + c : ATTN_OOB;
  };
#pragma unroll
  for (int i = 0; i < NPC; ++i) {
    qo[i] = place(pc.row + i * Piece::STEP, 0, pc.chunk(i) * 16, p.q);
    go[i] = place(pc.row + i * Piece::STEP, 0, pc.chunk(i) * 16, p.dout);
  }
  // (their lse is asked for one tile ahead)
  float live[NPC];
  auto ask_live = [&](int t) {
#pragma unroll
    for (int i = 0; i < NPC; ++i) {
      const int r = t * QT + pc.row + i * Piece::STEP;
      live[i] = r < p.R ? lse2[r] : INFINITY;
    }
  };
  const unsigned lds0 = lds_addr(smem);
  auto stage = [&](int t, int buf) {
    const int row0 = t * QT;
    const int tok0 = __builtin_amdgcn_readfirstlane(div_g(p, row0));
    const u32x4 qr = buffer_of(qbase + (long long)tok0 * p.q.l * (int)sizeof(T));
    const u32x4 gr = buffer_of(gbase + (long long)tok0 * p.dout.l * (int)sizeof(T));
    const unsigned at = lds0 + buf * STAGE_B;
    static_assert(TILE_B % 4096 == 0, "every wavefront stages whole pieces");
    if (even && !empty_rows && row0 + QT <= p.R) {
#pragma unroll
      for (int i = 0; i < NPC; ++i) {
        dma_1k(qr, at + wave * 1024 + i * 4096, qo[i]);
        dma_1k(gr, at + TILE_B + wave * 1024 + i * 4096, go[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NPC; ++i) {
        const int r = row0 + pc.row + i * Piece::STEP;
        bool ok = r < p.R;
        if (empty_rows) ok = live[i] != INFINITY;
        const unsigned a = even ? qo[i] : place(r, tok0, pc.chunk(i) * 16, p.q);
        const unsigned b = even ? go[i] : place(r, tok0, pc.chunk(i) * 16, p.dout);
        dma_1k(qr, at + wave * 1024 + i * 4096, ok ? a : ATTN_OOB);
        dma_1k(gr, at + TILE_B + wave * 1024 + i * 4096, ok ? b : ATTN_OOB);
      }
    }
    if (empty_rows) ask_live(t + 1);
    // (the statistics are padded to 64 rows: of a tile of 32 the lanes past it are told to read nothing)
    const unsigned so = lane < QT ? lane * 4 : ATTN_OOB;
    if (wave == 0) dma_256(buffer_of((const char*)(lse2 + row0)), at + 2 * TILE_B, so);
    if (wave == 1) dma_256(buffer_of((const char*)(delta + row0)), at + 2 * TILE_B + 256, so);
  };

  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dk[db] = dv[db] = zero16();

  // The first tile of rows is asked for before the wavefront's own keys and values (of a closed key: zeros, whatever its
  // memory holds).
  if (t0 < t1) {
    if (empty_rows) ask_live(t0);
    stage(t0, 0);
  }
  AttnFrag<T> kf[KS];
  {
    const long long kk = key_ok ? key : 0;
    const char* ks_ = p.k.p + ((long long)n * p.k.n + kk * p.k.l + (long long)hk * p.k.h) * (int)sizeof(T);
    const char* vs_ = p.v.p + ((long long)n * p.v.n + kk * p.v.l + (long long)hk * p.v.h) * (int)sizeof(T);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = load_frag<T>(ks_, ks, h, p.D, key_ok);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) lv.write_rows(2 * STAGE_B, ks, load_frag<T>(vs_, ks, h, p.D, key_ok));
  }
  auto step = [&](int t, auto buf_) __attribute__((always_inline)) {
    constexpr int buf = buf_.value;
    tile_barrier();
    const int qt = buf * STAGE_B, gt = qt + TILE_B;
    const float* st = reinterpret_cast<const float*>(smem + qt + 2 * TILE_B);
#pragma unroll
    for (int rb = 0; rb < QT / 32; ++rb) {
      const int row0 = t * QT + rb * 32;
      if (rb > 0 && row0 >= p.R) return;
      unsigned char open[16];
      if (PAIRS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = min(row0 + 8 * (i >> 2) + 4 * h + (i & 3), p.R - 1);
          const int tok = div_g(p, r);
          open[i] = mkey[(long long)(r - tok * p.G) * p.m_h + (long long)tok * p.m_q];
        }
      }
      // the score gradients' products start from -delta
      f32x16 s = zero16(), dp;
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 dl = *reinterpret_cast<const f32x4*>(st + 64 + rb * 32 + 2 * i + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[i + e] = dl[e];
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma32(s, ln.rows(qt + rb * 32 * Tile::PITCH, ks), kf[ks]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma32(dp, ln.rows(gt + rb * 32 * Tile::PITCH, ks), lv.rows(2 * STAGE_B, ks));
      if (rb == 0 && t + 1 < t1) stage(t + 1, buf ^ 1);     // (behind the first LDS reads, as in the forward kernel)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(st + rb * 32 + 2 * i + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i + e] = exp2_fast(fmaf(s[i + e], p.scale_log2, -ls[e]));
      }
      // closed pairs (what a closed key's column holds is not stored; the padding rows' lse is +inf)
      if (p.causal && key_wg + 127 > div_g(p, row0) + p.off) {
        keep_branch();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = row0 + 8 * (i >> 2) + 4 * h + (i & 3);
          s[i] = key <= div_g(p, r) + p.off ? s[i] : 0.f;
        }
      }
      if (PAIRS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = open[i] != 0 ? s[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] *= s[i];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const AttnFrag<T> pf = pack_frag<T>(s, j), sf = pack_frag<T>(dp, j);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const AttnFrag<T> gc = ln.cols(gt + (rb * 32 + j * 16) * Tile::PITCH, db), qc = ln.cols(qt + (rb * 32 + j * 16) * Tile::PITCH, db);
          mma32(dv[db], gc, pf);
          mma32(dk[db], qc, sf);
          if constexpr (REST) {
            mma32(dv[db], gc, pack_rest(s, j, pf));
            mma32(dk[db], qc, pack_rest(dp, j, sf));
          }
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

  if (key >= p.Lk) return;
  if (MASKED && !key_ok) {
#pragma unroll
    for (int db = 0; db < DB; ++db) dk[db] = dv[db] = zero16();
  }
  const long long at = (((long long)n * p.Lk + key) * p.Hk + hk) * p.D;
  if (w.parts == 1) {
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
    float* const at0 = p.part + (((long long)w.slot * p.parts + w.part) * 256 + wave * 32 + l31) * p.D;
    char *const pk = (char*)at0, *const pv = (char*)(at0 + 128LL * p.D);
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

// Sums the parts of the tiles that were cut, in part order: 4 channels of one key a thread, dk and dv.
template <typename T>
__global__ __launch_bounds__(ATTN_THREADS) void attn_dkv_sum_kernel(const AttnDev p) {
  const long long x = (long long)blockIdx.x * ATTN_THREADS + threadIdx.x;
  const int quads = p.D / 4;
  const long long line = x / quads;           // [rest][dk, dv][128]
  const int d = (int)(x - line * quads) * 4;
  if (line >= (long long)p.rest * 256) return;
  const int slot = (int)(line >> 8), row = (int)(line & 127);
  const bool is_v = (line & 128) != 0;
  AttnWork w;
  attn_decode_tile(p, p.whole + slot, &w);
  const int key = w.tile * 128 + row, parts = attn_tile_parts(p, w.tile);
  if (key >= p.Lk || parts == 1) return;     // (a tile in one part is finished)
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < parts; ++s) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(p.part + (((long long)slot * p.parts + s) * 256 + (line & 255)) * p.D + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += y[e];
  }
  const float scale = is_v ? 1.f : p.scale;
  store4<T>((is_v ? p.dv : p.dk) + (((long long)w.n * p.Lk + key) * p.Hk + w.hk) * p.D * (int)sizeof(T), d, v[0] * scale, v[1] * scale,
            v[2] * scale, v[3] * scale);
}

template <typename T, int DP>
static int launch(AttnDev* p, bool plan_only, hipStream_t st) {
  constexpr int QT = dkv_rows<T, DP>();
  const int lds = 2 * (2 * QT * AttnTile<T, DP>::PITCH + 512) + 128 * AttnTile<T, DP>::PITCH;
  static std::atomic<int> seen[2][3][ATTN_DEVICES];
  const int masks = p->mask ? 2 : p->kmask ? 1 : 0;
  const bool rest = sizeof(T) == 2 && p->R <= 64;
  auto kern = p->mask ? attn_dkv_kernel<T, DP, 2, false> : p->kmask ? attn_dkv_kernel<T, DP, 1, false> : attn_dkv_kernel<T, DP, 0, false>;
  if constexpr (sizeof(T) == 2) {
    if (rest) kern = p->mask ? attn_dkv_kernel<T, DP, 2, true> : p->kmask ? attn_dkv_kernel<T, DP, 1, true> : attn_dkv_kernel<T, DP, 0, true>;
  }
  const int per_cu = attn_occupancy((const void*)kern, lds, seen[rest][masks]);
  if (per_cu < 0) return per_cu;
  p->tiles = ceil_div(p->Lk, 128);
  p->loop_rows = QT;
  SEGK_UNSUPPORTED((long long)p->tiles * p->N * p->Hk < 0x40000000LL, "attention_bwd: too many workgroups");
  const long long grid = attn_deal(p, per_cu, ceil_div(p->R, QT), 2);
  if (plan_only) return SEGK_OK;
  kern<<<(unsigned)grid, ATTN_THREADS, lds, st>>>(*p);
  SEGK_CHECK_LAUNCH("attention_bwd keys");
  if (p->parts > 1) {
    const long long blocks = ((long long)p->rest * 256 * (p->D / 4) + ATTN_THREADS - 1) / ATTN_THREADS;
    attn_dkv_sum_kernel<T><<<(unsigned)blocks, ATTN_THREADS, 0, st>>>(*p);
    SEGK_CHECK_LAUNCH("attention_bwd keys' sum");
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

int attn_dkv(AttnDev* p, int dtype, bool plan_only, hipStream_t st) {
  return dtype == SEGK_BF16 ? dispatch<bf16_t>(p, plan_only, st) : dispatch<float>(p, plan_only, st);
}

}  // namespace segk
