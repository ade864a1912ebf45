// Shared pieces of the multi-head attention kernels (attn_fwd.hip, attn_dkv.hip, attn_dq.hip).
//
// Everything is built from 32 x 32 MFMA tiles whose contraction runs over 16 elements ("k-step"):
//   operand fragment  lane l holds row (or column) l & 31 and 8 of the 16 contracted elements; h = l >> 5 picks which
//   result tile       lane l holds column l & 31 and the 16 rows 8 * (i / 4) + 4 * h + i % 4, i = 0 .. 15
// The contracted elements may be dealt to the (h, e) slots in any order as long as both operands use the same one.  A
// result tile therefore IS the operand of the next product without any exchange between lanes: registers 8 s .. 8 s + 7
// of a tile of scores hold rows 16 s + 8 (e / 4) + 4 h + e % 4, and the other operand is read from LDS in that order
// (AttnLane::cols below).  So the probabilities never leave the registers of the lane that computed them.
//   bf16: v_mfma_f32_32x32x16_bf16; fp32: eight v_mfma_f32_32x32x2_f32 on the same fragments.
//
// Shared heads: the G = Hq / Hk query heads that read one key / value head are packed into the rows of one problem,
// row r = token r / G, head r % G of the group.  Keys and values are then read once for the group, and the gradient of a
// shared head is a sum over rows inside one workgroup.
#pragma once
#include <atomic>

#include "common.h"

namespace segk {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(8))) __bf16 attn_bf16x8;
typedef __attribute__((ext_vector_type(4))) short attn_s16x4;
typedef __attribute__((address_space(3))) void* attn_lds_ptr;

constexpr int ATTN_THREADS = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned ATTN_OOB = 0xfffffff0u;   // buffer offsets at or past this read as zeros and touch no memory

struct AttnView {   // element strides of a [N][L][heads][D] operand, unit stride over D
  const char* p;
  long long n, l, h;
};

struct AttnDev {
  AttnView q, k, v, o, dout;
  char *out, *dq, *dk, *dv;       // out: strides of `o`; gradients contiguous [N][L][heads][D]
  float* lse;                     // [N][Hq][Lq] natural log, or NULL
  char* out_rest;                 // [N][Lq][Hq][D] what the rounding of out left over, or NULL
  const unsigned char* mask;      // element strides below; NULL = all open
  long long m_n, m_h, m_q, m_k;
  const unsigned char* kmask;     // [N][Lk]
  long long km_n, km_k;
  int N, Lq, Lk, Hq, Hk, G, D;
  int R;                          // rows of one problem: Lq * G
  int Rp;                         // R rounded up to 64 (row statistics of the backward pass)
  unsigned g_magic;               // r / G = umulhi(r, g_magic) for G > 1
  int causal, off;                // key j is open to token i when j <= i + off, off = Lk - Lq
  float scale, scale_log2;
  int tiles;                      // workgroup tiles of one problem
  int whole, rest, parts, rest_x; // how the tiles are dealt out, see attn_work
  int even_steps, even_units;     // tiles of different lengths: steps of a part, parts of one problem (0: equal lengths)
  int loop_rows;                  // what a tile's loop runs over: 0 keys by 64, else packed rows by this many
  int tile_rows;                  // rows of a tile that exist: 128, of a shorter problem all of it
  float* part;                    // partial results: [rest][parts][tile_rows][D] (keys: [rest][parts][dk, dv][128][D])
  float* part_ml;                 // [rest][parts][tile_rows][3]: maxima and both sums of the forward pass
  float *row_lse2, *minus_delta;    // [N][Hk][Rp]: log2-domain lse (+inf: no open key) and -rowsum(dout * out)
};

__device__ __forceinline__ int div_g(const AttnDev& p, int r) { return p.G == 1 ? r : (int)__umulhi((unsigned)r, p.g_magic); }

// What a workgroup does.  The tiles of all problems (a problem: one image's key / value head) are numbered; the first
// `whole` of them (full rounds of the chip) go to one workgroup each, the `rest` that would leave most of the chip idle for
// a round are cut along their loop into `parts` parts, whose results another kernel joins in part order.  A problem with few
// tiles is all rest.  The tiles of one problem stay on one XCD (blockIdx % 8 in launch order): they share keys and values
// (rows, in the backward pass over keys) in its L2.  XCDs take runs of problems; under a key mask, whose images differ in
// length, problems are dealt to them in turns where their number allows.  16 images of 961 keys, a third of them padding:
// forward 90.5 -> 87, dq 108 -> 103 us; of equal images it costs 1.5 %
// (16 of 1089 tokens, 16 heads of 64 channels: 104.8 -> 106.2 us).  Tiles in plain launch order: 107.4 and, padded, 93.
struct AttnWork {
  int n, hk, tile;   // n < 0: nothing
  int part, parts;
  int slot;          // number among the tiles that are cut
};
// Tile number `tile` of a problem in launch order.
__device__ __forceinline__ int attn_tile(const AttnDev& p, int tile) {
  // Under the diagonal the longest tiles start first, of rows the last ones, of keys the first: keys of 2 images of 4225 tokens,
  // 16 heads of 64 channels 242 -> 202 us, 8 images, 8 heads over 4 of 128 channels 779 -> 730 us against the other order.
  // (Cut into equal parts they take the same time either way.)
  return p.causal && !p.loop_rows ? p.tiles - 1 - tile : tile;
}
__device__ __forceinline__ void attn_decode(const AttnDev& p, int problem, int tile, AttnWork* w) {
  w->tile = attn_tile(p, tile);
  w->hk = problem % p.Hk;
  w->n = problem / p.Hk;
}
// tile number g of all
__device__ __forceinline__ void attn_decode_tile(const AttnDev& p, int g, AttnWork* w) {
  if (p.kmask && ((p.N * p.Hk) & 7) == 0 && !p.even_steps) {
    const int whole_x = p.whole >> 3, rest_x = p.rest >> 3, s = g - p.whole;
    const int x = s < 0 ? g / whole_x : s / rest_x;
    const int i = s < 0 ? g - x * whole_x : whole_x + s - x * rest_x;
    attn_decode(p, x + 8 * (i / p.tiles), i % p.tiles, w);
  } else {
    attn_decode(p, g / p.tiles, g % p.tiles, w);
  }
}

// Steps of a tile's loop under the diagonal.
__host__ __device__ inline int attn_causal_steps(const AttnDev& p, int tile) {
  if (p.loop_rows) {           // keys tile * 128 .. : rows from the first token that may use one of them
    const int all = (p.R + p.loop_rows - 1) / p.loop_rows, tok = tile * 128 - p.off;
    return tok >= p.Lq ? 0 : all - (tok > 0 ? tok : 0) * p.G / p.loop_rows;
  }
  const int last = (tile * 128 + 128 < p.R ? tile * 128 + 128 : p.R) - 1;
  const int end = last / p.G + p.off + 1;
  return ((end < p.Lk ? (end > 0 ? end : 0) : p.Lk) + 63) / 64;
}
__host__ __device__ inline int attn_tile_parts(const AttnDev& p, int tile) {
  if (!p.even_steps) return p.parts;
  const int s = attn_causal_steps(p, tile);
  return s > p.even_steps ? (s + p.even_steps - 1) / p.even_steps : 1;
}
__device__ __forceinline__ AttnWork attn_work(const AttnDev& p) {
  AttnWork w = {-1, 0, 0, 0, 1, 0};
  const int x = (int)blockIdx.x & 7, i = (int)blockIdx.x >> 3, whole_x = p.whole >> 3;
  if (i < whole_x) {
    if (x * whole_x + i < p.tiles * p.N * p.Hk) attn_decode_tile(p, x * whole_x + i, &w);
    return w;
  }
  int u = x * p.rest_x + i - whole_x;
  if (p.even_steps) {          // tiles of different lengths: every part has about as many steps
    const int head = u / p.even_units;
    if (head >= p.N * p.Hk) return w;
    u -= head * p.even_units;
    // Lane t counts the parts of tile t; the tile of part u is the first whose running sum passes it.  (One tile after the
    // other: 0.3 us a tile, 1 image of 2048 tokens, 8 heads over 2 of 64 channels 36 us instead of 18.)
    const int lane = (int)threadIdx.x & 63;
    for (int t0 = 0; t0 < p.tiles; t0 += 64) {
      const int mine = t0 + lane < p.tiles ? attn_tile_parts(p, attn_tile(p, t0 + lane)) : 0;
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const int x = __shfl_up(sum, o, 64);
        sum += lane >= o ? x : 0;
      }
      const int all = __builtin_amdgcn_readlane(sum, 63);
      if (u < all) {
        const int t = __builtin_ctzll(__ballot(sum > u));
        w.parts = __builtin_amdgcn_readlane(mine, t);
        w.part = u - __builtin_amdgcn_readlane(sum, t) + w.parts;
        w.slot = head * p.tiles + t0 + t;
        attn_decode_tile(p, w.slot, &w);
        return w;
      }
      u -= all;
    }
    return w;
  }
  if (u >= p.rest * p.parts) return w;
  w.part = u / p.rest;
  w.parts = p.parts;
  w.slot = u - w.part * p.rest;
  attn_decode_tile(p, p.whole + w.slot, &w);
  return w;
}

template <typename T>
struct AttnFrag;
template <>
struct AttnFrag<bf16_t> {
  u32x4 v;
};
template <>
struct AttnFrag<float> {
  f32x8 v;
};

__device__ __forceinline__ void mma32(f32x16& c, const AttnFrag<bf16_t>& a, const AttnFrag<bf16_t>& b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(attn_bf16x8, a.v), __builtin_bit_cast(attn_bf16x8, b.v), c, 0, 0, 0);
}
__device__ __forceinline__ void mma32(f32x16& c, const AttnFrag<float>& a, const AttnFrag<float>& b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// registers 8 s .. 8 s + 7 of a result tile as an operand.  bf16: probabilities (and the score gradients) are rounded to
// the operand type here, as every bf16 product of the framework rounds its operands; sums and statistics stay fp32.
template <typename T>
__device__ __forceinline__ AttnFrag<T> pack_frag(const f32x16& s, int half);
template <>
__device__ __forceinline__ AttnFrag<bf16_t> pack_frag<bf16_t>(const f32x16& s, int half) {
  f32x8 x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = s[8 * half + j];
  AttnFrag<bf16_t> f;
  f.v = __builtin_bit_cast(u32x4, __builtin_convertvector(x, attn_bf16x8));   // (four v_cvt_pk_bf16_f32)
  return f;
}
template <>
__device__ __forceinline__ AttnFrag<float> pack_frag<float>(const f32x16& s, int half) {
  AttnFrag<float> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = s[8 * half + j];
  return f;
}

// What pack_frag's rounding left over, as a second operand.
__device__ __forceinline__ AttnFrag<bf16_t> pack_rest(const f32x16& s, int half, const AttnFrag<bf16_t>& f) {
  f32x16 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = s[8 * half + 2 * j] - __uint_as_float(f.v[j] << 16);
    x[2 * j + 1] = s[8 * half + 2 * j + 1] - __uint_as_float(f.v[j] & 0xffff0000u);
  }
  return pack_frag<bf16_t>(x, 0);
}

// 8 probabilities as an operand, and their sum added to `sum` (unrounded: lse is an fp32 statistic).
template <typename T>
__device__ __forceinline__ AttnFrag<T> pack_sum(const float* x, float& sum);
template <>
__device__ __forceinline__ AttnFrag<bf16_t> pack_sum<bf16_t>(const float* x, float& sum) {
  f32x8 y;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    y[j] = x[j];
    sum += x[j];
  }
  AttnFrag<bf16_t> f;
  f.v = __builtin_bit_cast(u32x4, __builtin_convertvector(y, attn_bf16x8));
  return f;
}
template <>
__device__ __forceinline__ AttnFrag<float> pack_sum<float>(const float* x, float& sum) {
  AttnFrag<float> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f.v[j] = x[j];
    sum += x[j];
  }
  return f;
}

// The sum of an operand's 8 probabilities as rounded, added to `sum` (four two-term products with ones).
__device__ __forceinline__ float sum_frag(const AttnFrag<bf16_t>& f, float sum) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned two = f.v[e];      // (a cast of f.v[e] itself takes element 0)
    sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
  }
  return sum;
}

// ---- tiles in LDS -------------------------------------------------------------------------------
// Rows of DP elements at a pitch of a power of two; the 16-byte chunks of a row are permuted by XOR with a function of
// the row.  LDS serves 256 bytes a clock: 16 lanes of a 16-byte read (AttnLane::rows: the same chunk of 16 neighbouring
// rows), 32 lanes of an 8-byte transposing read (cols in bf16: 64 bytes of four neighbouring rows) or 64 lanes of a 4-byte
// read (cols in fp32: 128 bytes of two rows, four apart).  swz() gives each of these groups distinct banks (fp32 columns of
// 128-byte rows excepted: both rows lie in the same half).
template <typename T, int DP>
struct AttnTile {
  static constexpr int ES = sizeof(T);
  static constexpr int PITCH = DP * ES <= 64 ? 64 : DP * ES <= 128 ? 128 : DP * ES <= 256 ? 256 : 512;
  static __device__ __forceinline__ int swz(int row) {
    if (PITCH == 64) return (row >> 2) & 3;
    if (PITCH == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    if (ES == 2) return ((row & 3) << 2) | ((row >> 2) & 3);
    return (((row >> 2) & 1) << 3) | ((row & 3) << 1) | ((row >> 3) & 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * PITCH + ((chunk ^ swz(row)) << 4); }
};

// One lane's share of staging a tile by LDS-DMA: the tile is cut into 1-KiB pieces, wavefront w takes pieces w, w + 4, ...;
// piece i of a wavefront holds rows row + i * STEP, and the lane fetches chunk(i) of its row (the DMA writes lanes in
// order, so the permutation is applied to what a lane reads).
template <typename T, int DP>
struct AttnPiece {
  typedef AttnTile<T, DP> Tile;
  static constexpr int STEP = 4096 / Tile::PITCH;
  int row, chunk0;
  __device__ __forceinline__ AttnPiece(int wave, int lane) {
    const int lin = wave * 1024 + lane * 16;
    row = lin / Tile::PITCH;
    chunk0 = ((lin % Tile::PITCH) >> 4) ^ Tile::swz(row);
  }
  // (STEP is a period of swz but for the 512-byte pitch, where every other piece flips its lowest bit)
  __device__ __forceinline__ int chunk(int i) const { return Tile::PITCH == 512 ? chunk0 ^ (i & 1) : chunk0; }
};

// One lane's reads of a tile in LDS, from byte addresses; `at`: LDS byte of the block of rows.
//   rows(): operand fragment contracted along the tile's rows in memory: lane (l & 31, h) reads elements 16 ks + 8 h .. + 7
//           of row l & 31.
//   cols(): operand fragment contracted over the tile's rows: lane (l & 31, h) gets column 32 db + (l & 31) of rows
//           8 (e / 4) + 4 h + e % 4, the order in which a result tile holds them.
//   write_rows(): stores what rows() reads.
// bf16: a lane's places differ between k-steps and columns by XORs that are kept in registers; what is added (tile, row
// block) is a constant of the instruction where the caller's is one.
template <typename T, int DP>
struct AttnLane;
template <int DP>
struct AttnLane<bf16_t, DP> {
  typedef AttnTile<bf16_t, DP> Tile;
  unsigned ra[DP / 16], ca[DP / 32][2];
  __device__ __forceinline__ AttnLane(const char* smem, int lane) {
    const unsigned base = (unsigned)(unsigned long long)(attn_lds_ptr)smem;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) ra[ks] = base + Tile::at(lane & 31, 2 * ks + (lane >> 5));
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // (a group of 16 lanes reads a block of 4 rows x 16 columns, 8 bytes a lane, and receives it transposed)
        const int row = 8 * j + 4 * (lane >> 5) + ((lane & 15) >> 2);
        ca[db][j] = base + Tile::at(row, db * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) + (lane & 1) * 8;
      }
  }
  __device__ __forceinline__ AttnFrag<bf16_t> rows(int at, int ks) const {
    AttnFrag<bf16_t> f;
    f.v = *(const __attribute__((address_space(3))) u32x4*)(size_t)(ra[ks] + at);
    return f;
  }
  __device__ __forceinline__ void write_rows(int at, int ks, const AttnFrag<bf16_t>& f) const {
    *(__attribute__((address_space(3))) u32x4*)(size_t)(ra[ks] + at) = f.v;
  }
  __device__ __forceinline__ AttnFrag<bf16_t> cols(int at, int db) const {
    AttnFrag<bf16_t> f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const attn_s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attn_s16x4*)(size_t)(ca[db][j] + at));
      const u32x2 u = __builtin_bit_cast(u32x2, t);
      f.v[2 * j] = u[0];
      f.v[2 * j + 1] = u[1];
    }
    return f;
  }
};
template <int DP>
struct AttnLane<float, DP> {
  typedef AttnTile<float, DP> Tile;
  char* smem;
  int lane;
  __device__ __forceinline__ AttnLane(char* s, int l) : smem(s), lane(l) {}
  __device__ __forceinline__ AttnFrag<float> rows(int at, int ks) const {
    AttnFrag<float> f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(smem + at + Tile::at(lane & 31, 4 * ks + 2 * (lane >> 5) + j));
#pragma unroll
      for (int e = 0; e < 4; ++e) f.v[4 * j + e] = t[e];
    }
    return f;
  }
  __device__ __forceinline__ void write_rows(int at, int ks, const AttnFrag<float>& f) const {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      *reinterpret_cast<f32x4*>(smem + at + Tile::at(lane & 31, 4 * ks + 2 * (lane >> 5) + j)) =
          f32x4{f.v[4 * j], f.v[4 * j + 1], f.v[4 * j + 2], f.v[4 * j + 3]};
  }
  __device__ __forceinline__ AttnFrag<float> cols(int at, int db) const {
    const int d = db * 32 + (lane & 31);
    AttnFrag<float> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int row = 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
      f.v[e] = *reinterpret_cast<const float*>(smem + at + Tile::at(row, d >> 2) + (d & 3) * 4);
    }
    return f;
  }
};

// Keeps an operand packed from here on (the compiler would carry the unpacked values to its use).
__device__ __forceinline__ void pin(AttnFrag<bf16_t>& f) { asm("" : "+v"(f.v)); }
__device__ __forceinline__ void pin(AttnFrag<float>&) {}

// Operand fragment straight from global memory: 8 elements from channel 16 ks + 8 h of one row (zeros past D and for
// ok == false).  D is a multiple of 8, so a fragment is whole or absent.
template <typename T>
__device__ __forceinline__ AttnFrag<T> load_frag(const char* row, int ks, int h, int D, bool ok);
template <>
__device__ __forceinline__ AttnFrag<bf16_t> load_frag<bf16_t>(const char* row, int ks, int h, int D, bool ok) {
  AttnFrag<bf16_t> f;
  f.v = u32x4{0, 0, 0, 0};
  const int d = 16 * ks + 8 * h;
  if (ok && d < D) f.v = *reinterpret_cast<const u32x4*>(row + d * 2);
  return f;
}
template <>
__device__ __forceinline__ AttnFrag<float> load_frag<float>(const char* row, int ks, int h, int D, bool ok) {
  AttnFrag<float> f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f.v[e] = 0.f;
  const int d = 16 * ks + 8 * h;
  if (ok && d < D) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(row + d * 4), b = *reinterpret_cast<const f32x4*>(row + d * 4 + 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f.v[e] = a[e];
      f.v[4 + e] = b[e];
    }
  }
  return f;
}

// Zero, or NaN if one of the fragment's elements is not finite.
__device__ __forceinline__ float probe_frag(const AttnFrag<bf16_t>& f) {
  float x = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) x = fmaf(__uint_as_float(f.v[e] << 16), 0.f, fmaf(__uint_as_float(f.v[e] & 0xffff0000u), 0.f, x));
  return x;
}
__device__ __forceinline__ float probe_frag(const AttnFrag<float>& f) {
  float x = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) x = fmaf(f.v[e], 0.f, x);
  return x;
}

// 4 consecutive channels of one row
template <typename T>
__device__ __forceinline__ void store4(char* row, int d, float a, float b, float c, float e);
template <>
__device__ __forceinline__ void store4<bf16_t>(char* row, int d, float a, float b, float c, float e) {
  *reinterpret_cast<u32x2*>(row + d * 2) = u32x2{pack_bf16x2(a, b), pack_bf16x2(c, e)};
}
template <>
__device__ __forceinline__ void store4<float>(char* row, int d, float a, float b, float c, float e) {
  *reinterpret_cast<f32x4*>(row + d * 4) = f32x4{a, b, c, e};
}

// out, 4 consecutive channels of one row (row, token and head give its place), and what its rounding left over
template <typename T>
__device__ __forceinline__ void store_out(const AttnDev& p, int n, int tok, int head, int d, float a, float b, float c, float e) {
  store4<T>(p.out + ((long long)n * p.o.n + (long long)tok * p.o.l + (long long)head * p.o.h) * (int)sizeof(T), d, a, b, c, e);
  if constexpr (sizeof(T) == 2) {
    if (p.out_rest) {
      const unsigned x = pack_bf16x2(a, b), y = pack_bf16x2(c, e);
      store4<T>(p.out_rest + (((long long)n * p.Lq + tok) * p.Hq + head) * p.D * (int)sizeof(T), d, a - __uint_as_float(x << 16),
                b - __uint_as_float(x & 0xffff0000u), c - __uint_as_float(y << 16), e - __uint_as_float(y & 0xffff0000u));
    }
  }
}

// ---- LDS-DMA ------------------------------------------------------------------------------------
// One 1-KiB piece: lane l's 16 bytes at buffer offset voff land at lds + 16 l; offsets from ATTN_OOB on write zeros.  In
// assembly because the compiler puts a wait for every LDS-DMA in flight before the next LDS read, which would empty the
// prefetch; the loops below wait themselves.  It has no register output.  s_nop 4: the resource may come from a
// v_readfirstlane, which needs five wait states before a buffer instruction reads it (s_mov_b32 is one of them).
__device__ __forceinline__ void dma_1k(const u32x4& rsrc, unsigned lds, unsigned voff) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 4\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(voff), "s"(rsrc)
      : "memory");
}
// the same with 4 bytes a lane (256 B)
__device__ __forceinline__ void dma_256(const u32x4& rsrc, unsigned lds, unsigned voff) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 4\n\t"
      "buffer_load_dword %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(voff), "s"(rsrc)
      : "memory");
}

__device__ __forceinline__ u32x4 buffer_of(const char* base) {
  const unsigned long long a = (unsigned long long)base;
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((unsigned)a);
  r[1] = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffffu);
  r[2] = ATTN_OOB;
  r[3] = 0x00020000u;
  return r;
}

__device__ __forceinline__ unsigned lds_addr(const char* p) {
  return (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(unsigned long long)(attn_lds_ptr)p);
}

// Every LDS-DMA of this wavefront has landed and every LDS read has returned; then all wavefronts meet.  (The bare
// barrier: the compiler's own would be the same here, the counts are spelled out because the DMA is in assembly.)
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Stages tiles of 64 keys and their values.
template <typename T, int DP>
struct AttnStage {
  typedef AttnTile<T, DP> Tile;
  typedef AttnPiece<T, DP> Piece;
  static constexpr int KT = 64, TILE_B = KT * Tile::PITCH;
  Piece pc;
  int row_b;               // bytes of a row that exist
  unsigned k_step, v_step, lds0;
  const char *kbase, *vbase;
  __device__ __forceinline__ AttnStage(const AttnDev& p, int n, int hk, int wave, int lane, const char* smem) : pc(wave, lane) {
    row_b = p.D * (int)sizeof(T);
    k_step = (unsigned)(p.k.l * (int)sizeof(T)), v_step = (unsigned)(p.v.l * (int)sizeof(T));
    kbase = p.k.p + ((long long)n * p.k.n + (long long)hk * p.k.h) * (int)sizeof(T);
    vbase = p.v.p + ((long long)n * p.v.n + (long long)hk * p.v.h) * (int)sizeof(T);
    lds0 = lds_addr(smem) + wave * 1024;
  }
  // One operand's tile at byte `at` of LDS.  bits: the tile's open keys (MASKED).  A closed key is not read: whatever its
  // memory holds, zeros arrive.
  template <bool MASKED>
  __device__ __forceinline__ void one(const AttnDev& p, const char* base, unsigned step, int key0, int at, unsigned long long bits) const {
    const u32x4 rsrc = buffer_of(base + (long long)key0 * step);
    const bool inside = !MASKED && key0 + KT <= p.Lk;
#pragma unroll
    for (int i = 0; i < TILE_B / 4096; ++i) {
      const int x = pc.row + i * Piece::STEP, c = pc.chunk(i) * 16;
      const unsigned off = c < row_b ? x * step + c : ATTN_OOB;
      if (inside) {
        dma_1k(rsrc, lds0 + at + i * 4096, off);
      } else {
        bool in = key0 + x < p.Lk;
        if (MASKED) in = in && ((bits >> x) & 1);
        dma_1k(rsrc, lds0 + at + i * 4096, in ? off : ATTN_OOB);
      }
    }
  }
  // both operands' tiles of buffer `buf`: K and V one after the other
  template <bool MASKED>
  __device__ __forceinline__ void both(const AttnDev& p, int key0, int buf, unsigned long long bits) const {
    one<MASKED>(p, kbase, k_step, key0, buf * 2 * TILE_B, bits);
    one<MASKED>(p, vbase, v_step, key0, buf * 2 * TILE_B + TILE_B, bits);
  }
};

// Keeps a rarely taken uniform branch a branch (the compiler would compute both sides and select).
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// Key mask of a tile of 64 keys as one bit per key, the same in every wavefront: load() asks for a tile's bytes, next()
// turns the bytes asked for last into bits.  Without a key mask (under a pair mask) a key's bit says whether the key exists.
struct AttnKeyMask {
  const unsigned char* mask;
  long long step;
  int Lk, lane;
  unsigned char raw;
  __device__ __forceinline__ AttnKeyMask(const unsigned char* m, long long s, int lk, int ln) : mask(m), step(s), Lk(lk), lane(ln) {}
  __device__ __forceinline__ void load(int key0) {
    const int j = key0 + lane;
    raw = j < Lk ? (mask ? mask[j * step] : 1) : 0;
  }
  __device__ __forceinline__ unsigned long long next() const { return __ballot(raw != 0); }
};

// The closed keys of a tile of 64 as what the products of its scores start from: 0 or -inf for every key, in LDS.
__device__ __forceinline__ void write_start(char* at, unsigned long long bits, int lane) {
  reinterpret_cast<float*>(at)[lane] = (bits >> lane) & 1 ? 0.f : -INFINITY;
}
__device__ __forceinline__ f32x16 read_start(const char* at, int h) {
  f32x16 x;
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const f32x4 y = reinterpret_cast<const f32x4*>(at)[i / 2 + h];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i + e] = y[e];
  }
  return x;
}

// The last of the first `keys` keys that the mask leaves open, -1 if none: a wavefront's answer, 256 keys at a time.
__device__ __forceinline__ int last_open_key(const unsigned char* mask, long long step, int keys, int lane) {
  for (int j0 = (keys - 1) / 256 * 256; j0 >= 0 && keys > 0; j0 -= 256) {
    unsigned char x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * 64 + lane;
      x[i] = j < keys ? mask[j * step] : 0;
    }
    for (int i = 3; i >= 0; --i) {
      const unsigned long long open = __ballot(x[i] != 0);
      if (open) return j0 + i * 64 + 63 - __builtin_clzll(open);
    }
  }
  return -1;
}

// Whether any of the 128 keys from key0 is open: the same answer in every wavefront.
__device__ __forceinline__ bool any_open_key(const unsigned char* mask, long long step, int key0, int Lk, int lane) {
  const int a = key0 + lane, b = a + 64;
  const unsigned char x = a < Lk ? mask[a * step] : 0, y = b < Lk ? mask[b * step] : 0;
  return __ballot((x | y) != 0) != 0;
}

// Pair mask of one row against a block of 32 keys: byte e of w[g] belongs to key 8 g + 4 h + e of the block, the order of a
// result tile's registers.
struct AttnPairMask {
  const unsigned char* row;
  long long step;
  int Lk, h4;
  unsigned w[4];
  __device__ __forceinline__ AttnPairMask(const unsigned char* m, long long s, int lk, int h) : row(m), step(s), Lk(lk), h4(4 * h) {}
  __device__ __forceinline__ void load(int key0) {
    if (!row) return;
    if (step == 1 && key0 + 32 <= Lk) {
#pragma unroll
      for (int g = 0; g < 4; ++g) __builtin_memcpy(&w[g], row + key0 + h4 + 8 * g, 4);
      return;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      unsigned x = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = key0 + h4 + 8 * g + e;
        if (j < Lk && row[j * step]) x |= 0xffu << (8 * e);
      }
      w[g] = x;
    }
  }
};

// Puts `closed` wherever a block's pair is closed: past `lim` (the last open key's place counted from the lane's first) ...
__device__ __forceinline__ void close_past(f32x16& s, float closed, int lim) {
  keep_branch();
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) <= lim ? s[i] : closed;
}
// ... by the pair mask.
__device__ __forceinline__ void close_pairs(f32x16& s, float closed, const unsigned* pair) {
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = pair[i >> 2] & (0xffu << (8 * (i & 3))) ? s[i] : closed;
}

// maximum and sum over the two lanes that share a result column (l and l ^ 32)
__device__ __forceinline__ float pair_max(float v) {
  const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- host side ----------------------------------------------------------------------------------
int attn_check(const segk_attention_args* a, AttnDev* p, bool backward);                 // attn_fwd.hip
// Deals p->tiles of every problem out to workgroups of which `per_cu` share a CU; `steps`: length of a tile's loop, of
// which a part takes at least min_steps.  Returns the grid.
long long attn_deal(AttnDev* p, int per_cu, int steps, int min_steps);
// Sets a kernel's LDS limit and returns how many of its workgroups share a CU (negative: status); `seen` keeps the answer
// for each device.
constexpr int ATTN_DEVICES = 64;
int attn_occupancy(const void* kernel, int lds, std::atomic<int>* seen);
// Each fills in the deal and, unless plan_only, launches.
int attn_dkv(AttnDev* p, int dtype, bool plan_only, hipStream_t st);                     // attn_dkv.hip
int attn_dq(AttnDev* p, int dtype, bool plan_only, hipStream_t st);                      // attn_dq.hip
static inline long long attn_part_floats(const AttnDev& p, int tile_rows, int floats_per_row) {
  return p.parts > 1 ? (long long)p.rest * p.parts * tile_rows * floats_per_row : 0;
}

}  // namespace segk
