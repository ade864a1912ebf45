// Multi-head attention, forward: out = softmax(scale q k^T) v per head in one pass over the keys, with a running reference
// and sums per row (fp32, base-2 exponents), and the host side of the attention entry points.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "attn.h"

namespace segk {

// Scores are computed transposed (S^T = K Q^T, a lane owns one query), so the running statistics are one
// register and S^T is the operand of O^T = V^T P^T as it lies (attn.h).  Keys in blocks of 32.
//   p = exp2(s scale log2(e) - m) for a reference m that need not be the maximum: in floating point any m serves that
//   neither overflows nor loses the largest terms.  m starts as the lowest finite number, to which closed scores (-inf) still
//   add nothing and any score adds infinity, and is raised to a block's maximum (accumulators rescaled) only when a block's
//   sum passes 2^30: at the first open key, then hardly ever, so that the common block needs no maximum and a row without open
//   keys none at all.  (m = -inf would raise all of a wavefront's rows in every block until each has met an open key: 21 class
//   queries, one in ten of them empty, 16 images of 4225 keys 22.6 us instead of 20.2, 4 images of 16641 keys 25.2 and 21.4.)
//   Scores of +inf and NaN end up there, too.
// Two sums: l of p, for lse (LSE: training), and in bf16 lr of p as rounded for its product, by which out is divided.  Out is
// then the exact mean of v under weights off by their rounding; divided by l, the roundings of the few probabilities that carry
// a row would not cancel in delta = rowsum(dout out), next to which ds is small.  rms error of dq, of its size, at scores of
// standard deviation 1 / 3 / 5 / 8 (512 x 1024, 64 channels): divided by l, delta from out as rounded 0.0017 / 0.0027 / 0.0044 /
// 0.0054; by lr, out's own rounding carried (out_rest) 0.0017 / 0.0018 / 0.0019 / 0.0019; the final rounding alone 0.0017.
template <typename T, int DB, bool LSE>
struct AttnRow {
  static constexpr bool ROUNDED = sizeof(T) == 2, BOTH = ROUNDED && LSE;
  f32x16 o[DB];
  float m, l, lr;
  __device__ __forceinline__ AttnRow() : m(-FLT_MAX), l(0.f), lr(0.f) {
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = zero16();
  }
  // probabilities of a block as two operands; their sum (the rounded ones' where it is the only one)
  __device__ __forceinline__ float weigh(const f32x16& s, float scale_log2, float ref, AttnFrag<T>* pf) const {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = exp2_fast(fmaf(s[8 * j + i], scale_log2, -ref));
      if constexpr (ROUNDED && !LSE) {
        float unused = 0.f;
        pf[j] = pack_sum<T>(e, unused);
        sum += sum_frag(pf[j], 0.f);
      } else {
        pf[j] = pack_sum<T>(e, sum);
      }
    }
    return sum;
  }
  __device__ __forceinline__ bool fine(float sum) const { return __builtin_amdgcn_ballot_w64(!(sum < 1073741824.f)) == 0; }
  // raises m to the block's maximum and weighs it again
  __device__ __forceinline__ float raise(const f32x16& s, float scale_log2, AttnFrag<T>* pf) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    const float nm = fmaxf(m, pair_max(mx) * scale_log2);
    const float alpha = exp2_fast(m - nm);
    m = nm;
    l *= alpha;
    lr *= alpha;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
    return weigh(s, scale_log2, nm, pf);
  }
  __device__ __forceinline__ void add(float sum, const AttnFrag<T>* pf) {
    l += sum;
    if constexpr (BOTH) lr += sum_frag(pf[0], 0.f) + sum_frag(pf[1], 0.f);
  }
};

// Row tiles: 4 wavefronts of 32 rows, tiles of 64 keys shared through LDS.  A wavefront works on three blocks at a time:
// the scores of block b + 1 and the values of block b - 1 on the matrix cores while the exponentials of block b run on the
// vector unit: one wavefront keeps both busy, as independent instructions of one basic block.  LDS holds two K and two V
// tiles; K runs one tile ahead of V.  Wavefronts to a SIMD: 4 where a row of a tile has 64 bytes (class queries under masks, 32
// channels: 26.5 -> 22.3 us against 3, 20.2 now), 3 up to 128 bytes, 1 for fp32 heads over 96 channels (under masks over 64: 8
// images of 1089 tokens, 8 heads of 96 channels, key mask 573 -> 459 us; without a mask 2 take 410 and 1 takes 417), else 2.  At 32
// and 64 channels under masks one register is spilled (64 channels, training, with 2 wavefronts and no spill: 115 us instead of 99).
// Matrix-bound on long maps: 2 images of 16641 tokens, 8 heads over 2 of 128 channels, bf16: 2.06 to 2.12 ms, 1070 to 1100
// TFLOP/s (a large library product reaches 1164 here); the matrix cores are busy 60 % of the cycles, at 1.8 GHz.
// 16 images of 1089 tokens, 16 heads of 64 channels: 104 us, 747 TFLOP/s: half as many products to an exponential.
// Training (LSE) costs the second sum and out_rest's 2 bytes an element: 16 images of 961 tokens under key masks, 16 heads of
// 64 channels 87 -> 99 us (sum 4, out_rest 8), 4 images of 4225 tokens, 16 heads of 128 channels 551 -> 585 us (20 and 14).
// Few rows (one token, class queries) take one tile, whose wavefronts without rows only stage: 16641 keys of 4 heads in 7 us,
// 2.4 TB/s.  Kernels that dealt the keys of a tile to the four wavefronts and joined them in LDS measured 6.7 us there, 24 us
// against 23 for 21 class queries under masks, and 22 us against 19.5 in the gradient: not worth a second form.
template <typename T, int DP, bool MASKED, bool LSE>
__global__ __launch_bounds__(ATTN_THREADS, (DP * (int)sizeof(T) >= (MASKED ? 384 : 512) ? 1 : DP * (int)sizeof(T) > 128 ? 2 : DP * (int)sizeof(T) > 64 ? 3 : 4)) void attn_fwd_kernel(const AttnDev p) {
  typedef AttnTile<T, DP> Tile;
  constexpr int KT = 64, KS = DP / 16, DB = DP / 32;
  constexpr int TILE_B = KT * Tile::PITCH;
  extern __shared__ __attribute__((aligned(1024))) char smem[];   // K tiles 0, 1, V tiles 0, 1; MASKED: 2 x 64 starts

  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
  const AttnWork w = attn_work(p);
  if (w.n < 0) return;
  const int n = w.n, hk = w.hk;
  const int row0 = w.tile * 128 + wave * 32;

  const AttnStage<T, DP> st(p, n, hk, wave, lane, smem);
  const unsigned char* const kmask = MASKED && p.kmask ? p.kmask + n * p.km_n : nullptr;
  AttnKeyMask km(kmask, p.km_k, p.Lk, lane);
  unsigned long long bits_next = ~0ULL;      // open keys of the K tile last asked for: V follows

  // keys that some row of the workgroup may use
  const int last_row = min(w.tile * 128 + 128, p.R) - 1;
  int k_end = p.Lk;
  if (p.causal) k_end = max(0, min(k_end, div_g(p, last_row) + p.off + 1));
  if (MASKED && kmask) k_end = min(k_end, last_open_key(kmask, p.km_k, k_end, lane) + 1);
  const int all_steps = (k_end + KT - 1) / KT;
  const int per = (all_steps + w.parts - 1) / w.parts;
  const int t0 = min(w.part * per, all_steps), t1 = min(t0 + per, all_steps);
  const int last = t1 - t0 - 1;              // tiles are counted from t0: u = 0 .. last

  char* const start0 = smem + 4 * TILE_B;    // MASKED: what the scores of K tiles 0, 1 start from
  if (t0 < t1) {                             // the first tile is asked for before anything else
    if (MASKED) {
      km.load(t0 * KT);
      bits_next = km.next();
      km.load((t0 + 1) * KT);
      if (wave == 0) write_start(start0, bits_next, lane);
    }
    st.template one<MASKED>(p, st.kbase, st.k_step, t0 * KT, 0, bits_next);
    st.template one<MASKED>(p, st.vbase, st.v_step, t0 * KT, 2 * TILE_B, bits_next);
  }

  const int r = row0 + l31;
  const bool row_ok = r < p.R;
  const int rr = row_ok ? r : 0;
  const int tok = div_g(p, rr), head = hk * p.G + rr - tok * p.G;
  AttnFrag<T> qf[KS];
  {
    const char* src = p.q.p + ((long long)n * p.q.n + (long long)tok * p.q.l + (long long)head * p.q.h) * (int)sizeof(T);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load_frag<T>(src, ks, h, p.D, row_ok);
  }
  const int wave_tok0 = __builtin_amdgcn_readfirstlane(div_g(p, min(row0, p.R - 1)));
  // last key open to the lane's row, and the first key that is closed to some row of the wavefront
  const int lim = (p.causal ? min(p.Lk - 1, tok + p.off) : p.Lk - 1) - 4 * h;
  const int ragged0 = p.causal ? min(p.Lk, wave_tok0 + p.off + 1) : p.Lk;

  AttnPairMask pm(MASKED && p.mask ? p.mask + n * p.m_n + (long long)head * p.m_h + (long long)tok * p.m_q : nullptr, p.m_k, p.Lk, h);
  constexpr int key_b = 32 * Tile::PITCH;
  constexpr std::integral_constant<int, 0> zero, no;
  constexpr std::integral_constant<int, 1> one, yes;

  typedef AttnRow<T, DB, LSE> Row;
  Row row;
  bool odd = false;          // the row's query is not finite
  f32x16 s[2];
  AttnFrag<T> pf[2][2];

  const AttnLane<T, DP> ln(smem, lane);
  // scores and values of the block at LDS byte `at`; `half` of K tile `buf`
  auto scores = [&](f32x16& x, int at, int buf, int half) __attribute__((always_inline)) {
    if (MASKED) x = read_start(start0 + buf * 256 + half * 128, h);
    else x = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) mma32(x, ln.rows(at, ks), qf[ks]);
  };
  auto values = [&](const AttnFrag<T>* f, int at) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int db = 0; db < DB; ++db) mma32(row.o[db], ln.cols(at + j * 16 * Tile::PITCH, db), f[j]);
  };
  // block b of parity `odd`: its scores are in s[odd]; next_k: the K block after it (of tile buffer next_buf), last_v: the V
  // block before it
  auto block = [&](int key0, auto odd_, auto with_k, int next_k, int next_buf, auto with_v, int last_v) __attribute__((always_inline)) {
    constexpr int odd = odd_.value;
    if (key0 + 32 > ragged0) close_past(s[odd], -INFINITY, lim - key0);
    if (MASKED && pm.row) {
      close_pairs(s[odd], -INFINITY, pm.w);
      pm.load(key0 + 32);
    }
    if constexpr (with_k.value) scores(s[odd ^ 1], next_k, next_buf, odd ^ 1);
    float sum = row.weigh(s[odd], p.scale_log2, row.m, pf[odd]);
    if constexpr (with_v.value) values(pf[odd ^ 1], last_v);
    pin(pf[odd][0]);
    pin(pf[odd][1]);
    if (__builtin_expect(!row.fine(sum), 0)) sum = row.raise(s[odd], p.scale_log2, pf[odd]);
    row.add(sum, pf[odd]);
  };
  // at the barrier of turn u: K tile u + 1 and V tile u are here; every wavefront is done with K tile u and V tile u - 1
  auto stage = [&](int u, int here) __attribute__((always_inline)) {
    const int t = t0 + u, there = TILE_B - here;
    unsigned long long bits2 = ~0ULL;
    if (MASKED) {
      bits2 = km.next();
      km.load((t + 3) * KT);
      if (wave == 0) write_start(start0 + (here ? 256 : 0), bits2, lane);
    }
    if (u + 2 <= last) st.template one<MASKED>(p, st.kbase, st.k_step, (t + 2) * KT, here, bits2);
    st.template one<MASKED>(p, st.vbase, st.v_step, (t + 1) * KT, 2 * TILE_B + there, bits_next);
    if (MASKED) bits_next = bits2;
  };

  if (t0 < t1) {
    if (MASKED) {
      if (pm.row) pm.load(t0 * KT);
      bits_next = km.next();
      km.load((t0 + 2) * KT);
    }
    tile_barrier();
    if (last > 0) {
      st.template one<MASKED>(p, st.kbase, st.k_step, (t0 + 1) * KT, TILE_B, bits_next);
      if (MASKED && wave == 0) write_start(start0 + 256, bits_next, lane);
    }
    if (row0 >= p.R) {          // no rows: this wavefront only helps to stage the tiles
      for (int u = 0; u < last; ++u) {
        tile_barrier();
        stage(u, (u & 1) * TILE_B);
      }
      tile_barrier();
      return;
    }
    // A query that is not finite has a softmax of NaN over whatever keys are open to it.  Its scores do not tell (all -inf looks
    // like a row without an open key; a closed key's -inf + query * 0 is NaN): it is taken as zeros, and its row becomes NaN
    // below if it has met an open key.
    {
      float x = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) x += probe_frag(qf[ks]);
      odd = !(pair_sum(x) == 0.f);
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd) != 0, 0)) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (unsigned e = 0; e < sizeof(qf[0].v) / sizeof(qf[0].v[0]); ++e) qf[ks].v[e] = odd ? 0 : qf[ks].v[e];
      }
    }
    scores(s[0], 0, 0, 0);
    block(t0 * KT, zero, yes, key_b, 0, no, 0);
    // The second block of tile u and the first of tile u + 1; two turns to a round of the loop, so that the buffers are
    // constants of each.
    auto turn = [&](int u, auto even_) __attribute__((always_inline)) {
      constexpr int here = even_.value * TILE_B, there = TILE_B - here;
      tile_barrier();
      stage(u, here);
      const int key0 = (t0 + u) * KT + 32;
      block(key0, one, yes, there, even_.value ^ 1, yes, 2 * TILE_B + here);
      block(key0 + 32, zero, yes, there + key_b, even_.value ^ 1, yes, 2 * TILE_B + here + key_b);
    };
    int u = 0;
    for (; u + 1 < last; u += 2) {
      turn(u, zero);
      turn(u + 1, one);
    }
    if (u < last) turn(u, zero);
    tile_barrier();
    const int v = (2 + (last & 1)) * TILE_B, key0 = (t0 + last) * KT + 32;
    if (key0 < k_end) {
      block(key0, one, no, 0, 0, yes, v);
      values(pf[1], v + key_b);
    } else {
      values(pf[0], v);
    }
  }

  float lt = pair_sum(row.l), lrt = Row::BOTH ? pair_sum(row.lr) : lt;
  if (odd && lt != 0.f) lt = lrt = NAN;
  // (the row's place is worked out again: carried through the loop it costs the registers that 64 channels under masks lack)
  int out_row = l31;
  asm volatile("" : "+v"(out_row));
  out_row += row0;
  if (out_row >= p.R) return;
  const int out_tok = div_g(p, out_row), out_head = hk * p.G + out_row - out_tok * p.G;
  if (w.parts == 1) {
    const float inv = lt == 0.f ? 0.f : 1.f / lrt;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = db * 32 + 2 * i + 4 * h;
        if (d < p.D) store_out<T>(p, n, out_tok, out_head, d, row.o[db][i] * inv, row.o[db][i + 1] * inv, row.o[db][i + 2] * inv, row.o[db][i + 3] * inv);
      }
    if (LSE && p.lse && h == 0)
      p.lse[((long long)n * p.Hq + out_head) * p.Lq + out_tok] = lt == 0.f ? -INFINITY : (row.m + log2f(lt)) * 0.6931471805599453f;
  } else {
    const long long at = ((long long)w.slot * p.parts + w.part) * p.tile_rows + out_row - w.tile * 128;
    char* dst = (char*)(p.part + at * p.D);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = db * 32 + 2 * i + 4 * h;
        if (d < p.D) store4<float>(dst, d, row.o[db][i], row.o[db][i + 1], row.o[db][i + 2], row.o[db][i + 3]);
      }
    if (h == 0) {
      p.part_ml[3 * at] = row.m;
      p.part_ml[3 * at + 1] = lt;
      p.part_ml[3 * at + 2] = lrt;
    }
  }
}

// Joins the parts of the tiles that were cut.  `lanes` = D / 4 rounded up to a power of two threads walk a row's channels of
// every `groups`-th part (about four parts a thread); the groups of a row are joined in LDS in order.  4 heads of one token, 88
// parts each: 8 us, most of it the launch and two reads one after the other.
template <typename T>
__global__ __launch_bounds__(ATTN_THREADS) void attn_join_kernel(const AttnDev p, int lanes, int groups) {
  __shared__ f32x4 so[ATTN_THREADS];
  __shared__ float sl[ATTN_THREADS], sr[ATTN_THREADS], sm[ATTN_THREADS];
  const int c = threadIdx.x % lanes, g = threadIdx.x / lanes % groups, in = threadIdx.x / (lanes * groups);
  const long long line = (long long)blockIdx.x * (ATTN_THREADS / (lanes * groups)) + in;
  const int slot = (int)(line / p.tile_rows), row = (int)(line - (long long)slot * p.tile_rows);
  AttnWork w = {0, 0, 0, 0, 1, 0};
  int parts = 0;
  if (slot < p.rest) {
    attn_decode_tile(p, p.whole + slot, &w);
    parts = attn_tile_parts(p, w.tile);
  }
  const bool ok = parts > 1;       // (a tile in one part is finished)
  const long long first = ok ? (long long)slot * p.parts * p.tile_rows + row : 0;
  // every group looks at its own parts' maxima first, so that the sums are scaled once
  float m = -INFINITY, l = 0.f, lr = 0.f;
  if (ok)
    for (int s = g; s < parts; s += groups) m = fmaxf(m, p.part_ml[3 * (first + (long long)s * p.tile_rows)]);
  sm[threadIdx.x] = m;
  __syncthreads();
  for (int i = 0; i < groups; ++i) m = fmaxf(m, sm[(in * groups + i) * lanes + c]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (ok)
    for (int s = g; s < parts; s += groups) {
      const long long at = first + (long long)s * p.tile_rows;
      const float a = exp2_fast(p.part_ml[3 * at] - m);
      l = fmaf(p.part_ml[3 * at + 1], a, l);
      lr = fmaf(p.part_ml[3 * at + 2], a, lr);
      if (c * 4 < p.D) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(p.part + at * p.D + c * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], a, o[e]);
      }
    }
  so[threadIdx.x] = o;
  sl[threadIdx.x] = l;
  sr[threadIdx.x] = lr;
  __syncthreads();
  if (!ok || g != 0 || c * 4 >= p.D) return;
  const int rr = w.tile * 128 + row;
  if (rr >= p.R) return;
  for (int i = 1; i < groups; ++i) {
    const f32x4 x = so[threadIdx.x + i * lanes];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += x[e];
    l += sl[threadIdx.x + i * lanes];
    lr += sr[threadIdx.x + i * lanes];
  }
  const float inv = l == 0.f ? 0.f : 1.f / lr;
  const int n = w.n, tok = div_g(p, rr), head = w.hk * p.G + rr - tok * p.G;
  store_out<T>(p, n, tok, head, c * 4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (p.lse && c == 0)
    p.lse[((long long)n * p.Hq + head) * p.Lq + tok] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Row statistics of the backward pass in packed row order: -rowsum(dout * out) and the base-2 lse (+inf where a row has no
// open key and in the padding: its probabilities then come out as zeros).  D / 8 lanes (rounded up to a power of two)
// share a row.  bf16: out with what its rounding left over (see AttnRow); without that, as rounded for the caller.
// Memory-bound: 16 images of 961 tokens, 16 heads of 64 channels 17 us, 5.5 TB/s (14 us without out_rest).
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
    const float ln = p.lse[((long long)n * p.Hq + head) * p.Lq + tok];
    lse = ln == -INFINITY ? INFINITY : ln * LOG2E;
    // (a row without an open key has no gradient, whatever arrives for it: its dout is not looked at)
    if (c * 8 < p.D && ln != -INFINITY) {
      const AttnFrag<T> a = load_frag<T>(p.o.p + ((long long)n * p.o.n + (long long)tok * p.o.l + (long long)head * p.o.h) * (int)sizeof(T), c >> 1, c & 1, p.D, true);
      AttnFrag<T> x = {};
      if (sizeof(T) == 2 && p.out_rest)
        x = load_frag<T>(p.out_rest + (((long long)n * p.Lq + tok) * p.Hq + head) * p.D * (int)sizeof(T), c >> 1, c & 1, p.D, true);
      const AttnFrag<T> b = load_frag<T>(p.dout.p + ((long long)n * p.dout.n + (long long)tok * p.dout.l + (long long)head * p.dout.h) * (int)sizeof(T), c >> 1, c & 1, p.D, true);
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum = fmaf(__uint_as_float(a.v[e] << 16) + __uint_as_float(x.v[e] << 16), __uint_as_float(b.v[e] << 16), sum);
          sum = fmaf(__uint_as_float(a.v[e] & 0xffff0000u) + __uint_as_float(x.v[e] & 0xffff0000u), __uint_as_float(b.v[e] & 0xffff0000u), sum);
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
    p.minus_delta[r] = -sum;
  }
}

// ------------------------------------------------------------------ host ----
long long attn_deal(AttnDev* p, int per_cu, int steps, int min_steps) {
  const long long all = (long long)p->tiles * p->N * p->Hk;
  const long long round = 256LL * per_cu;      // workgroups that run at once
  p->even_steps = p->even_units = 0;
  if (p->causal && p->tiles > 1 && all < round) {
    // Fewer tiles than a round, of different lengths: parts of equal length, a round of them.  Against equal numbers of parts:
    // fp32, 2 images of 1089 tokens, 8 heads of 64 channels: forward 51.8 -> 50.8 us, keys 92 -> 71, queries 73 -> 55; bf16, one
    // image: 2048 tokens, 8 heads over 2 of 64 channels 20.1 -> 18.4, 29.2 -> 25.9, 25.0 -> 20.3; 16641 tokens, 2 heads of 64
    // channels 147 -> 116, 290 -> 220, 238 -> 179 (and 4 us more to join); 4225 tokens, 8 heads over 2 of 128 channels (264 tiles
    // of 512: equal numbers leave one part) 107 -> 66, 142 -> 138, 174 -> 100.  It loses a little where equal numbers fill the
    // round just so: 4096 tokens, 8 heads over 2 of 64 channels 34 -> 40, 72 -> 68, 52 -> 51.
    // Parts of half the length gain 5 us in the first forward kernel and lose them in the join; parts of twice the length take 59,
    // 98 and 81 us there.
    long long sum = 0;
    for (int t = 0; t < p->tiles; ++t) sum += attn_causal_steps(*p, t);
    long long per = (sum * p->N * p->Hk + round - 1) / round;
    p->even_steps = (int)(per < min_steps ? min_steps : per);
    int most = 1, units = 0;
    for (int t = 0; t < p->tiles; ++t) {
      const int n = attn_tile_parts(*p, t);
      units += n;
      if (n > most) most = n;
    }
    p->even_units = units;
    p->whole = 0, p->rest = (int)all, p->parts = most;
    p->rest_x = (int)(((long long)units * p->N * p->Hk + 7) / 8);
    return 8LL * p->rest_x;
  }
  // Under the diagonal tiles differ in length and even out by themselves once there are enough of them.
  long long whole = p->causal && all >= round ? all / 8 * 8 : all / round * round;
  // A last round that is not full is worth cutting up (and joining) only where a round is long: 18 steps of 64 keys gained
  // nothing, 67 steps 5 %, 261 steps 12 %.
  if (whole > 0 && steps < 64) whole = (all + 7) / 8 * 8;
  long long rest = all > whole ? all - whole : 0, parts = 1;
  if (rest > 0) {
    parts = round / rest;
    if (parts > steps / min_steps) parts = steps / min_steps;
    if (parts < 1) parts = 1;
    const long long per = (steps + parts - 1) / parts;   // as many as have work
    parts = per > 0 ? (steps + per - 1) / per : 1;
    if (parts < 1) parts = 1;
  }
  p->whole = (int)whole, p->rest = (int)rest, p->parts = (int)parts;
  p->rest_x = (int)((rest * parts + 7) / 8);
  return whole + 8LL * p->rest_x;
}

int attn_occupancy(const void* kernel, int lds, std::atomic<int>* seen) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= ATTN_DEVICES) {
    set_error("attention: no current device among the first %d", ATTN_DEVICES);
    return SEGK_HIP_ERROR;
  }
  const int known = seen[dev].load(std::memory_order_relaxed);
  if (known) return known;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("attention: %s", hipGetErrorString(e));
      return SEGK_HIP_ERROR;
    }
  }
  int n = 0;
  const hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, ATTN_THREADS, (size_t)lds);
  if (e != hipSuccess || n < 1) {
    set_error("attention: no workgroup fits a CU: %s", hipGetErrorString(e));
    return SEGK_HIP_ERROR;
  }
  seen[dev].store(n, std::memory_order_relaxed);
  return n;
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
  SEGK_REQUIRE(a->scale > 0.f && a->scale * LOG2E < INFINITY, "attention: the scale must be positive and finite");
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
  SEGK_REQUIRE(!a->out_rest || (a->dtype == SEGK_BF16 && ((uintptr_t)a->out_rest & 15) == 0),
               "attention: out_rest belongs to bf16 operands and must be 16-byte aligned");
  p->out_rest = (char*)a->out_rest;
  p->mask = (const unsigned char*)a->mask;
  p->m_n = a->mask_n, p->m_h = a->mask_h, p->m_q = a->mask_q, p->m_k = a->mask_k;
  p->kmask = (const unsigned char*)a->key_mask;
  p->km_n = a->key_mask_n, p->km_k = a->key_mask_k;
  p->N = a->N, p->Lq = a->Lq, p->Lk = a->Lk, p->Hq = a->Hq, p->Hk = a->Hk, p->G = G, p->D = a->D;
  p->R = (int)R;
  p->Rp = round_up((int)R, 64);
  p->tile_rows = R < 128 ? (int)R : 128;
  p->g_magic = G > 1 ? (unsigned)((0x100000000ULL + G - 1) / G) : 0;
  p->causal = a->causal != 0;
  p->off = a->Lk - a->Lq;
  p->scale = a->scale;
  p->scale_log2 = a->scale * LOG2E;
  p->tiles = p->whole = p->rest = p->parts = p->rest_x = 0;
  p->even_steps = p->even_units = p->loop_rows = 0;
  p->part = p->part_ml = nullptr;
  p->dq = p->dk = p->dv = nullptr;
  p->row_lse2 = p->minus_delta = nullptr;
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

template <typename T, int DP>
static int launch_fwd(AttnDev* p, bool plan_only, hipStream_t st) {
  static std::atomic<int> seen[2][2][ATTN_DEVICES];
  const bool masked = p->mask || p->kmask, lse = sizeof(T) == 4 || p->lse;     // (fp32: one form)
  const int lds = 4 * 64 * AttnTile<T, DP>::PITCH + (masked ? 512 : 0);
  void (*kern)(const AttnDev) = masked ? attn_fwd_kernel<T, DP, true, true> : attn_fwd_kernel<T, DP, false, true>;
  if constexpr (sizeof(T) == 2) {
    if (!lse) kern = masked ? attn_fwd_kernel<T, DP, true, false> : attn_fwd_kernel<T, DP, false, false>;
  }
  const int per_cu = attn_occupancy((const void*)kern, lds, seen[masked][lse]);
  if (per_cu < 0) return per_cu;
  p->tiles = ceil_div(p->R, 128);
  SEGK_UNSUPPORTED((long long)p->tiles * p->N * p->Hk < 0x40000000LL, "attention: too many workgroups");
  const long long grid = attn_deal(p, per_cu, ceil_div(p->Lk, 64), 2);
  if (plan_only) return SEGK_OK;
  kern<<<(unsigned)grid, ATTN_THREADS, lds, st>>>(*p);
  SEGK_CHECK_LAUNCH("attention_fwd");
  return SEGK_OK;
}

template <typename T>
static int dispatch_fwd(AttnDev* p, bool plan_only, hipStream_t st) {
  if (p->D <= 32) return launch_fwd<T, 32>(p, plan_only, st);
  if (p->D <= 64) return launch_fwd<T, 64>(p, plan_only, st);
  if (p->D <= 96) return launch_fwd<T, 96>(p, plan_only, st);
  return launch_fwd<T, 128>(p, plan_only, st);
}

// The deal of a forward pass.  Launches unless plan_only.
static int run_fwd(AttnDev* p, int dtype, bool plan_only, hipStream_t st) {
  return dtype == SEGK_BF16 ? dispatch_fwd<bf16_t>(p, plan_only, st) : dispatch_fwd<float>(p, plan_only, st);
}

// Floats of the backward pass's workspace: row statistics, then the partial results of whichever pass is running.
static int bwd_floats(AttnDev p, int dtype, long long* floats) {
  const long long stats = 2LL * p.N * p.Hk * p.Rp;
  long long part = 0;
  if (p.dk && p.Lk > 0) {
    const int rc = attn_dkv(&p, dtype, true, nullptr);
    if (rc != SEGK_OK) return rc;
    part = attn_part_floats(p, 128, 2 * p.D);
  }
  if (p.dq && p.Lk > 0) {
    const int rc = attn_dq(&p, dtype, true, nullptr);
    if (rc != SEGK_OK) return rc;
    const long long x = attn_part_floats(p, p.tile_rows, p.D);
    if (x > part) part = x;
  }
  *floats = stats + part;
  return SEGK_OK;
}

}  // namespace segk

using namespace segk;

extern "C" long long segk_attention_workspace(const segk_attention_args* a, int backward) {
  AttnDev p;
  int rc = attn_check(a, &p, backward != 0);
  if (rc != SEGK_OK) return rc;
  long long floats = 0;
  if (backward) {
    rc = bwd_floats(p, a->dtype, &floats);
  } else {
    rc = run_fwd(&p, a->dtype, true, nullptr);
    floats = attn_part_floats(p, p.tile_rows, p.D + 3);
  }
  return rc != SEGK_OK ? rc : floats * 4;
}

static int take_workspace(const segk_attention_args* a, long long need, const char* name) {
  SEGK_REQUIRE(a->workspace && ((uintptr_t)a->workspace & 15) == 0, "%s: workspace missing or not 16-byte aligned", name);
  if (a->workspace_bytes < need) {
    set_error("%s: workspace of %lld bytes, needs %lld", name, a->workspace_bytes, need);
    return SEGK_WORKSPACE_TOO_SMALL;
  }
  return SEGK_OK;
}

extern "C" int segk_attention_fwd(const segk_attention_args* a, segk_stream_t stream) {
  AttnDev p;
  int rc = attn_check(a, &p, false);
  if (rc != SEGK_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  rc = run_fwd(&p, a->dtype, true, st);
  if (rc != SEGK_OK) return rc;
  const long long floats = attn_part_floats(p, p.tile_rows, p.D + 3);
  if (floats > 0) {
    rc = take_workspace(a, floats * 4, "attention_fwd");
    if (rc != SEGK_OK) return rc;
    p.part = (float*)a->workspace;
    p.part_ml = p.part + attn_part_floats(p, p.tile_rows, p.D);
  }
  rc = run_fwd(&p, a->dtype, false, st);
  if (rc != SEGK_OK || p.parts == 1) return rc;
  const int lanes = p.D <= 8 ? 2 : p.D <= 16 ? 4 : p.D <= 32 ? 8 : p.D <= 64 ? 16 : 32;
  int groups = 1;
  while (groups * 4 < p.parts && groups * lanes < ATTN_THREADS) groups *= 2;     // about four parts a thread
  const int lines = ATTN_THREADS / (lanes * groups);
  const unsigned grid = (unsigned)ceil_div((long long)p.rest * p.tile_rows, lines);   // (rest is less than a round of workgroups)
  SEGK_DISPATCH_DTYPE(a->dtype, T, (attn_join_kernel<T><<<grid, ATTN_THREADS, 0, st>>>(p, lanes, groups)));
  SEGK_CHECK_LAUNCH("attention_fwd join");
  return SEGK_OK;
}

extern "C" int segk_attention_bwd(const segk_attention_args* a, segk_stream_t stream) {
  AttnDev p;
  int rc = attn_check(a, &p, true);
  if (rc != SEGK_OK) return rc;
  SEGK_REQUIRE(p.Lk > 0, "attention_bwd: no keys");
  long long floats = 0;
  rc = bwd_floats(p, a->dtype, &floats);
  if (rc != SEGK_OK) return rc;
  rc = take_workspace(a, floats * 4, "attention_bwd");
  if (rc != SEGK_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  const long long rows = (long long)p.N * p.Hk * p.Rp;
  p.row_lse2 = (float*)a->workspace;
  p.minus_delta = p.row_lse2 + rows;
  p.part = p.minus_delta + rows;
  const int lanes = p.D <= 8 ? 1 : p.D <= 16 ? 2 : p.D <= 32 ? 4 : p.D <= 64 ? 8 : 16;
  const long long blocks = (rows * lanes + ATTN_THREADS - 1) / ATTN_THREADS;
  SEGK_UNSUPPORTED(blocks < 0x7fffffffLL, "attention_bwd: too many rows");
  SEGK_DISPATCH_DTYPE(a->dtype, T, (attn_row_stats_kernel<T><<<(unsigned)blocks, ATTN_THREADS, 0, st>>>(p, lanes)));
  SEGK_CHECK_LAUNCH("attention_bwd statistics");
  if (p.dk) {
    rc = attn_dkv(&p, a->dtype, false, st);
    if (rc != SEGK_OK) return rc;
  }
  return p.dq ? attn_dq(&p, a->dtype, false, st) : SEGK_OK;
}
