// Newton-Schulz orthogonalisation of a stack of matrices, and the optimiser's step that uses it.
//
//   X_0 = X / (|X|_F + eps);   G = X X^T,   X <- a X + (b G + c G^2) X      once a step
//
// X is taken as [M, N] with M <= N (a tall matrix is transposed on its way in and out: the iteration commutes with it).  X is carried as two
// planes of half precision, high and low, 22 bits together (values below 2^-13 in steps of 2^-34), scaled by 2^10 so that the low plane keeps its bits: singular values
// stay near or below 1, so entries do not overflow.
//
// Products add up high x high, high x low and low x high planes, three multiplies for one, whatever the result's type.  (High planes alone, 11 bits, do not do for bfloat16 results either.  What X's rounding
// leaves out lands in weak directions too, and each of them grows by up to 3.4445 a step: in front of the last rounding, which is 1.7e-3 of the norm, emulated, 7e-4 for random matrices of 512 rows, but 8e-3 for
// 8 x 4096 of rank 4 over 0.3 % noise, 3e-2 for exactly low-rank ones after eight steps.  Both planes of X alone: 3e-3 for 512 x 2048 of which four rows are not zero.  Both planes of everything: 3e-5 at most in
// five steps.  What two planes leave out, and fp32 sums round, grows in a direction that is exactly zero as well, so that more steps of low-rank matrices leave more: 9e-4 after eight.)
// G and the polynomial enter products less their mean diagonal, whose part is exact, so that the rounding of near-identity matrices is that of what is left of them:
//   A = G - d I,   B = (b + 2 c d) A + c (A^2 - e I),   X <- (a + b d + c d^2 + c e) X + B X,   d = |X|^2 / M,   e = |A|^2 / M.
//
// A step of 64 matrices of 1536 x 2048 takes 1015 to 1044 us for G, 838 to 867 for the polynomial and 1595 to 1640 for the update; 17.5 to 18.1 ms in all, 1.0 PFLOP/s counting three products and half of a symmetric one.
// Between tiles eight waves store results and read what they add to (25 us a tile of 256, of 1.4 us a slab of 64), and 64 x 21 triangular tiles are 5.25 rounds of the chip.  What is small is bound by
// latency: 512 x 512, three kernels of 13.5 us a step.
//
// G and G^2 are symmetric: only tiles on and below the diagonal are computed, and stored twice.  No sum depends on the order of arrival: norms are
// summed per tile and the tiles' sums in order.

#include "launch.hpp"
#include "stream_gemm.hpp"

namespace tgg {

enum : int { NS_GRAM = 0, NS_POLY = 1, NS_UPDATE = 2, NS_LAST = 3 };  // NS_LAST: the last step's update, straight to the result

constexpr float kNsScale = 1024.f, kNsInv2 = 1.f / (1024.f * 1024.f);

// Where results go: out = v, or with `weight` out = keep out - step v.
struct NsTarget {
  void* out;
  int dt, weight;  // dt 0 bf16, 1 fp16, 2 fp32
  int whole;       // eight elements of a row are whole and aligned to 16 bytes
  float keep, step;
};

// One product for all matrices.  Planes: element (m, i, j) at m * stride + i * ld + j.
struct NsProduct {
  const uint16_t *a_hi, *a_lo, *b_hi, *b_lo;  // operands: GRAM X, X; POLY A, A; UPDATE B, X
  uint16_t *o_hi, *o_lo;                      // result's planes
  const uint16_t *c_hi, *c_lo;                // what the epilogue adds: POLY A, UPDATE X
  int64_t a_stride, b_stride, o_stride;       // per matrix, in elements
  int lda, ldb, ldo;
  int rows, cols, depth;                      // the result's size and the sum's length
  int batch;
  float ca, cb, cc;                           // the polynomial's coefficients
  const float *x_sums, *a_sums;               // |X|^2 and |A|^2 by tile, x_tiles and a_tiles a matrix
  float* o_sums;                              // the result's (GRAM, UPDATE)
  int x_tiles, a_tiles;                       // x_tiles 0: the first step, d = 1 / M
  NsTarget target;                            // LAST
  int tall;                                   // LAST: the result is the transposed matrix
};

namespace {

struct NsSplit { uint16_t hi, lo; };
TGG_DEV NsSplit ns_split(float v) {
  const _Float16 h = (_Float16)v;
  const _Float16 l = (_Float16)(v - (float)h);
  return {__builtin_bit_cast(uint16_t, h), __builtin_bit_cast(uint16_t, l)};
}
TGG_DEV float ns_f16(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }

TGG_DEV float ns_from16(uint16_t x, int dt) { return dt == 0 ? __builtin_bit_cast(float, (uint32_t)x << 16) : ns_f16(x); }
TGG_DEV uint16_t ns_to16(float x, int dt) { return dt == 0 ? Out16<DT_BF16>::cvt(x) : Out16<DT_F16>::cvt(x); }

// the n sums of a matrix, added by a wave: every lane gets the same bits, and every workgroup
TGG_DEV float ns_sum(const float* p, int n) {
  float s = 0.f;
  for (int i = lane_id(); i < n; i += 64) s += p[i];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d, 64);
  return s;
}

// n (up to 8) neighbouring values as fp32; VEC: all eight, in 16-byte loads
template <bool VEC> TGG_DEV void ns_load8(float (&v)[8], const void* p, int64_t i, int dt, int n) {
  if (VEC) {
    if (dt == 2) {
      const f32x4_t a = *(const f32x4_t*)((const float*)p + i), b = *(const f32x4_t*)((const float*)p + i + 4);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v[x] = a[x];
        v[4 + x] = b[x];
      }
    } else {
      const i32x4_t a = *(const i32x4_t*)((const uint16_t*)p + i);
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] = ns_from16((uint16_t)((uint32_t)a[x / 2] >> (16 * (x & 1))), dt);
    }
  } else {
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = x >= n ? 0.f : dt == 2 ? ((const float*)p)[i + x] : ns_from16(((const uint16_t*)p)[i + x], dt);
  }
}
template <bool VEC> TGG_DEV void ns_store8(void* p, int64_t i, int dt, const float (&v)[8], int n) {
  if (VEC) {
    if (dt == 2) {
      *(f32x4_t*)((float*)p + i) = f32x4_t{v[0], v[1], v[2], v[3]};
      *(f32x4_t*)((float*)p + i + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
    } else {
      i32x4_t a;
#pragma unroll
      for (int x = 0; x < 4; ++x) a[x] = (int)(dt == 0 ? pack2<DT_BF16>(v[2 * x], v[2 * x + 1]) : pack2<DT_F16>(v[2 * x], v[2 * x + 1]));
      *(i32x4_t*)((uint16_t*)p + i) = a;
    }
  } else {
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < n) {
        if (dt == 2) ((float*)p)[i + x] = v[x]; else ((uint16_t*)p)[i + x] = ns_to16(v[x], dt);
      }
  }
}
// Fused operations of steps are written out here and in ns_mix: which product the compiler fuses may differ between variants, and an unaligned matrix has to
// get an aligned one's bits.
TGG_DEV float ns_stepped(const NsTarget& t, float old, float v) { return __builtin_fmaf(-t.step, v, t.keep * old); }
// n (up to 8) neighbouring results at element o; v in the planes' scale.  whole: all eight, aligned
TGG_DEV void ns_store_result(const NsTarget& t, int64_t o, float (&v)[8], int n, bool whole) {
  float old[8];
  if (t.weight) whole ? ns_load8<true>(old, t.out, o, t.dt, 8) : ns_load8<false>(old, t.out, o, t.dt, n);
#pragma unroll
  for (int x = 0; x < 8; ++x) v[x] = t.weight ? ns_stepped(t, old[x], v[x] * (1.f / kNsScale)) : v[x] * (1.f / kNsScale);
  whole ? ns_store8<true>(t.out, o, t.dt, v, 8) : ns_store8<false>(t.out, o, t.dt, v, n);
}

typedef __amdgpu_buffer_rsrc_t rsrc_t;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;
TGG_DEV rsrc_t ns_window(const void* base, int64_t bytes) {
  bytes = bytes < 0 ? 0 : (bytes > 0x3fffffff ? 0x3fffffff : bytes);
  return __builtin_amdgcn_make_buffer_rsrc((void*)uniform64((uint64_t)base), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
constexpr int kNowhere = 0x40000000;  // beyond every window, also with a tile's rows added

template <class C, int MODE> struct NsProblem {
  static constexpr bool SYM = MODE <= NS_POLY, B_KMAJOR = SYM;
  static_assert(!SYM || C::BM == C::BN, "symmetric results have square tiles");
  // The epilogue takes pieces of 16 rows x HC columns of the wave's block through the wave's staging: a multiply leaves a lane four columns of one row, and
  // neighbouring lanes in different rows, of which every one is an access of its own (64 cycles an instruction; 256-row tiles spent 36 us there).  Staged, a lane has eight columns and
  // four lanes 64 bytes of a row.
  static constexpr int HC = C::TN >= 2 ? 32 : 16, PIECES = C::TN * 16 / HC, LPR = HC / 8;
  // Bytes between rows: fp32 (16-byte pieces swizzled by the row, no padding: two workgroups of 128-row tiles have to fit a compute unit), 16 bits, 16 bits transposed.
  static constexpr int PITCH = HC * 4, PITCH16 = HC * 2 + 16, PITCH_T = 48;
  static constexpr int STAGE_WAVE = 16 * PITCH > HC * PITCH_T ? 16 * PITCH : HC * PITCH_T;
  static constexpr int SMEM_BYTES = C::EPI_OFF + C::NWAVES * STAGE_WAVE;
  static_assert(STAGE_WAVE >= 16 * PITCH16 && (C::BM != 128 || 2 * SMEM_BYTES <= 160 * 1024), "the staging's size");
  static TGG_DEV int staged(int row, int piece) { return row * PITCH + ((piece ^ (row % (HC / 4))) << 4); }

  const NsProduct& p;
  StreamWalk walk;
  StreamCursor<C, B_KMAJOR> cur;
  int tiles_m, tiles_n, per_matrix, pos, pass;
  int64_t a_tile, b_tile;  // the tile's first bytes in the planes
  int a_rows, b_rows, b_skip;
  bool live;

  TGG_DEV NsProblem(const NsProduct& q, int tiles_m_, int tiles_n_)
      : p(q), walk(q.batch * (SYM ? tiles_m_ * (tiles_m_ + 1) / 2 : tiles_m_ * tiles_n_)), cur(q.lda * 2, q.ldb * 2, q.depth) {  // (planes are zero between the depth and the next multiple of 8)
    tiles_m = tiles_m_;
    tiles_n = tiles_n_;
    per_matrix = SYM ? tiles_m * (tiles_m + 1) / 2 : tiles_m * tiles_n;
    pos = -1;
  }
  TGG_DEV int tile_at(int q) const { return walk.at(q); }
  TGG_DEV int slabs(int) const { return 3 * cur.kt; }
  // id -> matrix, first row, first column
  struct Place { int m, row0, col0; };
  TGG_DEV Place locate(int id) const {
    const int m = id / per_matrix, t = id - m * per_matrix;
    int i, j;
    if (SYM) {
      i = (int)((__builtin_sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);  // (within one: t is exact)
      i -= i * (i + 1) / 2 > t;
      i += (i + 1) * (i + 2) / 2 <= t;
      j = t - i * (i + 1) / 2;
    } else {
      i = t / tiles_n;
      j = t - i * tiles_n;
    }
    return {__builtin_amdgcn_readfirstlane(m), __builtin_amdgcn_readfirstlane(i * C::BM), __builtin_amdgcn_readfirstlane(j * C::BN)};
  }
  // passes: high x high planes, high x low, low x high
  TGG_DEV void begin_pass() {
    const uint16_t* const a = pass == 2 ? p.a_lo : p.a_hi;
    const uint16_t* const b = pass == 1 ? p.b_lo : p.b_hi;
    cur.begin(live, (uint64_t)a + a_tile, (uint64_t)b + b_tile, a_rows, b_rows, b_skip);
  }
  TGG_DEV void seek(int id) {
    ++pos;
    pass = 0;
    live = id >= 0;
    const Place at = locate(live ? id : 0);
    a_tile = (at.m * p.a_stride + (int64_t)at.row0 * p.lda) * 2;
    b_tile = (at.m * p.b_stride + (B_KMAJOR ? (int64_t)at.col0 * p.ldb : (int64_t)at.col0)) * 2;
    a_rows = min(C::BM, p.rows - at.row0);
    b_rows = B_KMAJOR ? min(C::BN, p.cols - at.col0) : p.depth;
    b_skip = at.col0 * 2;
    begin_pass();
  }
  TGG_DEV void turn() {
    if (pass < 2) {
      ++pass;
      begin_pass();
    } else {
      seek(tile_at(pos + 1));
    }
  }
  TGG_DEV void begin(int, f32x4_t (&)[C::TM][C::TN], const StreamPlace<C>&) const {}

  // A piece of 16-bit values, eight columns of a row a lane, to out with rows and columns exchanged; row, col: the piece's first, `pitch` values between out's rows.  The
  // transposing read hands a lane four rows of a column; through LDS again, two lanes have a column's 16 rows.
  TGG_DEV void store_transposed(char* mine, const i32x4_t& v, uint16_t* out, int64_t pitch, int row, int col, int rows_end, int cols_end, int el) const {
    const int l16 = el & 15, lg = el >> 4;
    if (el < 16 * LPR) *(i32x4_t*)(mine + el / LPR * PITCH16 + el % LPR * 16) = v;
    asm volatile("" : : : "memory");  // read as another type, by other lanes of the wave; its LDS operations complete in order
    i16x4_t t[HC / 16];
#pragma unroll
    for (int j = 0; j < HC / 16; ++j) t[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr_t)(mine + (4 * lg + (l16 >> 2)) * PITCH16 + (16 * j + 4 * (l16 & 3)) * 2));
    asm volatile("" : : : "memory");
#pragma unroll
    for (int j = 0; j < HC / 16; ++j) *(i16x4_t*)(mine + (16 * j + l16) * PITCH_T + lg * 8) = t[j];
    asm volatile("" : : : "memory");
    const int c = el >> 1, r = (el & 1) * 8;
    if (c < HC && col + c < cols_end && row + r < rows_end) *(i32x4_t*)(out + (int64_t)(col + c) * pitch + row + r) = *(const i32x4_t*)(mine + c * PITCH_T + r * 2);
    asm volatile("" : : : "memory");
  }

  TGG_DEV void epilogue(int id, f32x4_t (&acc)[C::TM][C::TN], const StreamPlace<C>& at, char* stage) const {
    int el = at.lane;
    asm volatile("" : "+v"(el));  // (addresses are made afresh per tile instead of living across the multiplies)
    const int l16 = el & 15, lg = el >> 4;
    const Place tile = locate(id);
    const int m = tile.m;
    const int64_t base = m * p.o_stride;
    const int rbase = tile.row0 + at.wm0, cbase = tile.col0 + at.wn0;
    const int rl = el / LPR, cl = el % LPR * 8;  // the lane's row and first column of a piece
    const bool mine_too = LPR == 4 || el < 16 * LPR;
    // Planes are reached through windows that begin at the tile's first row (the mirrored tile's: its first column) and end with the matrix's last: what lies below reads as zeros and is not
    // written.  Columns to the right of a row are nowhere.
    auto rows_of = [&](const uint16_t* plane, int first, int rows) __attribute__((always_inline)) { return ns_window(plane + base + (int64_t)first * p.ldo, (int64_t)lesser(rows, p.rows - first) * p.ldo * 2); };
    const rsrc_t o_hi = rows_of(p.o_hi, tile.row0, C::BM), o_lo = rows_of(p.o_lo, tile.row0, C::BM);
    const rsrc_t c_hi_w = rows_of(p.c_hi, tile.row0, MODE != NS_GRAM ? C::BM : 0), c_lo_w = rows_of(p.c_lo, tile.row0, MODE != NS_GRAM ? C::BM : 0);
    const int pitch = p.ldo * 2;
    int lane_at[PIECES];
#pragma unroll
    for (int q = 0; q < PIECES; ++q) lane_at[q] = mine_too && cbase + q * HC + cl < p.ldo ? (at.wm0 + rl) * pitch + (cbase + q * HC + cl) * 2 : kNowhere;
    // what the result adds to, some pieces ahead of its use: a wait for it is one for the stores before it too
    constexpr int AHEAD = C::BM == 256 ? 4 : 2;
    i32x4_t c_hi[AHEAD], c_lo[AHEAD];
    auto fetch = [&](int n) __attribute__((always_inline)) {
      c_hi[n % AHEAD] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(c_hi_w, lane_at[n % PIECES] + n / PIECES * 16 * pitch, 0, 0));
      c_lo[n % AHEAD] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(c_lo_w, lane_at[n % PIECES] + n / PIECES * 16 * pitch, 0, 0));
    };
    if (MODE != NS_GRAM) {
#pragma unroll
      for (int n = 0; n < AHEAD && n < C::TM * PIECES; ++n) fetch(n);
    }
    const float inv_rows = 1.f / (float)p.rows;
    const float d = p.x_tiles ? ns_sum(p.x_sums + (int64_t)m * p.x_tiles, p.x_tiles) * inv_rows : inv_rows;
    const float e = MODE == NS_GRAM ? 0.f : ns_sum(p.a_sums + (int64_t)m * p.a_tiles, p.a_tiles) * inv_rows;
    // the result is f acc + g C, less h on the diagonal, all times kNsScale
    const float f = (MODE == NS_POLY ? p.cc : 1.f) * kNsInv2 * kNsScale;
    const float g = MODE == NS_POLY ? p.cb + 2.f * p.cc * d : !SYM ? p.ca + p.cb * d + p.cc * d * d + p.cc * e : 0.f;
    const float h = (MODE == NS_GRAM ? d : MODE == NS_POLY ? p.cc * e : 0.f) * kNsScale;
    const bool diagonal = SYM && tile.row0 == tile.col0, edge = tile.row0 + C::BM > p.rows || tile.col0 + C::BN > p.cols || LPR != 4;
    const rsrc_t m_hi = rows_of(p.o_hi, tile.col0, SYM ? C::BN : 0), m_lo = rows_of(p.o_lo, tile.col0, SYM ? C::BN : 0);
    const int c_row = el >> 1, r0 = (el & 1) * 8;  // of the mirrored piece
    const int mirror_at = c_row < HC ? (at.wn0 + c_row) * pitch + (rbase + r0) * 2 : kNowhere;
    char* const mine = stage + at.wave * STAGE_WAVE;
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < C::TM * PIECES; ++n) {
      const int i = n / PIECES, half = n % PIECES;
#pragma unroll
      for (int j = 0; j < HC / 16; ++j) *(f32x4_t*)(mine + staged(l16, 4 * j + lg)) = acc[i][half * (HC / 16) + j];
      asm volatile("" : : : "memory");
      const int row = rbase + 16 * i + rl, col = cbase + half * HC + cl;
      float v[8];
      {
        const f32x4_t a = *(const f32x4_t*)(mine + staged(rl % 16, cl / 4)), b = *(const f32x4_t*)(mine + staged(rl % 16, cl / 4 + 1));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          v[x] = f * a[x];
          v[4 + x] = f * b[x];
        }
      }
      asm volatile("" : : : "memory");
      if (MODE != NS_GRAM) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int h2 = c_hi[n % AHEAD][x / 2], l2 = c_lo[n % AHEAD][x / 2];  // (a bit cast of a vector's element takes the first one)
          const f16x2_t hi = __builtin_bit_cast(f16x2_t, h2), lo = __builtin_bit_cast(f16x2_t, l2);
          v[x] = __builtin_fmaf((float)lo[x & 1], g, v[x]);
          v[x] = __builtin_fmaf((float)hi[x & 1], g, v[x]);
        }
        if (n + AHEAD < C::TM * PIECES) fetch(n + AHEAD);
      }
      if (diagonal) {
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] -= row == col + x ? h : 0.f;
      }
      if (edge) {
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = mine_too && row < p.rows && col + x < p.cols ? v[x] : 0.f;  // (what lies beyond is a sum of whatever the operands' next rows hold)
      }
      if (MODE == NS_GRAM || MODE == NS_UPDATE) {
#pragma unroll
        for (int x = 0; x < 8; ++x) sum = __builtin_fmaf(v[x], v[x], sum);
      }
      if constexpr (MODE == NS_LAST) {
        const float by = 1.f / kNsScale;
        if (p.tall) {  // 16-bit results only
          i32x4_t w;
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = (int)(p.target.dt == 0 ? pack2<DT_BF16>(v[2 * x] * by, v[2 * x + 1] * by) : pack2<DT_F16>(v[2 * x] * by, v[2 * x + 1] * by));
          store_transposed(mine, w, (uint16_t*)p.target.out + (int64_t)m * p.rows * p.cols, p.rows, rbase + 16 * i, cbase + half * HC, p.rows, p.cols, el);
        } else if (mine_too && row < p.rows && col < p.cols) {
          ns_store_result(p.target, ((int64_t)m * p.rows + row) * p.cols + col, v, (int)lesser(8, p.cols - col), p.target.whole);
        }
      } else {
        i32x4_t hi, lo;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t q = pack2<DT_F16>(v[2 * x], v[2 * x + 1]);
          const f16x2_t r = __builtin_bit_cast(f16x2_t, q);
          hi[x] = (int)q;
          lo[x] = (int)pack2<DT_F16>(v[2 * x] - (float)r[0], v[2 * x + 1] - (float)r[1]);
        }
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, hi), o_hi, lane_at[half] + i * 16 * pitch, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, lo), o_lo, lane_at[half] + i * 16 * pitch, 0, 0);
        if (SYM && !diagonal) {  // the same with rows and columns exchanged: both planes of a value in a word, a lane reads eight rows of a column
          uint32_t w[8];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            w[2 * x] = ((uint32_t)hi[x] & 0xffffu) | (uint32_t)lo[x] << 16;
            w[2 * x + 1] = (uint32_t)hi[x] >> 16 | ((uint32_t)lo[x] & 0xffff0000u);
          }
          if (mine_too) {
            *(i32x4_t*)(mine + staged(rl, cl / 4)) = i32x4_t{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
            *(i32x4_t*)(mine + staged(rl, cl / 4 + 1)) = i32x4_t{(int)w[4], (int)w[5], (int)w[6], (int)w[7]};
          }
          asm volatile("" : : : "memory");
#pragma unroll
          for (int x = 0; x < 8; ++x) w[x] = *(const uint32_t*)(mine + staged(r0 + x, c_row % HC >> 2) + (c_row & 3) * 4);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            hi[x] = (int)((w[2 * x] & 0xffffu) | w[2 * x + 1] << 16);
            lo[x] = (int)(w[2 * x] >> 16 | (w[2 * x + 1] & 0xffff0000u));
          }
          const int o = rbase + 16 * i + r0 < p.ldo ? mirror_at + half * HC * pitch + i * 32 : kNowhere;
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, hi), m_hi, o, 0, 0);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, lo), m_lo, o, 0, 0);
          asm volatile("" : : : "memory");
        }
      }
    }
    if (MODE == NS_GRAM || MODE == NS_UPDATE) {
      if (SYM && !diagonal) sum *= 2.f;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
      if (el == 0) *(float*)mine = sum;  // (read before the next tile's epilogue: its slabs have barriers)
      __syncthreads();
      if (threadIdx.x == 0) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < C::NWAVES; ++w) s += *(const float*)(stage + w * STAGE_WAVE);
        p.o_sums[id] = s * kNsInv2;
      }
    }
  }
};

template <class C, int MODE> __global__ __launch_bounds__(C::THREADS) void ns_product_kernel(const NsProduct p, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  NsProblem<C, MODE> prob(p, tiles_m, tiles_n);
  stream_gemm<C, DT_F16, NsProblem<C, MODE>::B_KMAJOR>(prob, smem);
}

// ---- into the planes and out of them -------------------------------------------------------------------------------------

constexpr int kNsThreads = 256, kNsChunk = 16384;  // values of a workgroup's sum of squares

TGG_DEV void ns_store_planes(uint16_t* hi, uint16_t* lo, int64_t o, const float (&v)[8]) {
  i32x4_t a, b;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const NsSplit s0 = ns_split(v[2 * x]), s1 = ns_split(v[2 * x + 1]);
    a[x] = (int)((uint32_t)s0.hi | (uint32_t)s1.hi << 16);
    b[x] = (int)((uint32_t)s0.lo | (uint32_t)s1.lo << 16);
  }
  *(i32x4_t*)(hi + o) = a;
  *(i32x4_t*)(lo + o) = b;
}

// What is orthogonalised: x, or, with momentum, the momentum's value after this step and with Nesterov's look ahead.
struct NsSource {
  const void* x;   // the input or the gradient
  float* momentum; // or null
  float beta, keep;  // keep = 1 - beta, in 64 bits before its rounding (1 - 0.999f is 1.3e-5 of itself off)
  int nesterov, dt;
};
TGG_DEV float ns_mix(const NsSource& s, float m, float g) { return __builtin_fmaf(s.beta, m, s.keep * g); }
// eight values of the direction; `step`: the momentum takes its step
template <bool VEC> TGG_DEV void ns_direction(float (&v)[8], const NsSource& s, int64_t i, int n, bool step) {
  ns_load8<VEC>(v, s.x, i, s.dt, n);
  if (!s.momentum) return;
  float m[8];
  ns_load8<VEC>(m, s.momentum, i, 2, n);
  if (step) {
#pragma unroll
    for (int x = 0; x < 8; ++x) m[x] = ns_mix(s, m[x], v[x]);
    ns_store8<VEC>(s.momentum, i, 2, m, n);
  }
#pragma unroll
  for (int x = 0; x < 8; ++x) v[x] = s.nesterov ? ns_mix(s, m[x], v[x]) : m[x];
}

// Sums of squares of a matrix's chunks, in 64 bits (values far from 1 have no squares in fp32); with momentum, its step.  16 x 2048 x 768 with momentum 46 us for 252 MB, 64 x 1536 x 2048 76 us for 403 MB (5.3 TB/s).  VEC: matrices are multiples of eight values.
template <bool VEC> __global__ __launch_bounds__(kNsThreads) void ns_norm_kernel(const NsSource s, int64_t values, int chunks, double* sums) {
  const int m = blockIdx.x / chunks, c = blockIdx.x % chunks;
  const int64_t first = m * values + (int64_t)c * kNsChunk, end = lesser(first + kNsChunk, (m + 1) * values);
  double sum = 0.0;
#pragma unroll 2
  for (int64_t i = first + threadIdx.x * 8; i < end; i += kNsThreads * 8) {
    float v[8];
    ns_direction<VEC>(v, s, i, (int)lesser(8, end - i), true);
#pragma unroll
    for (int x = 0; x < 8; ++x) sum = __builtin_fma((double)v[x], (double)v[x], sum);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
  __shared__ double waves[kNsThreads / 64];
  if (lane_id() == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < kNsThreads / 64; ++w) t += waves[w];
    sums[blockIdx.x] = t;
  }
}

// Tiles of 64 x 64 into the planes, transposed where the matrix is tall.  64 x 1536 x 2048: 221 us for 1.2 GB (5.5 TB/s).  VEC: rows are multiples of eight values.
template <bool VEC> __global__ __launch_bounds__(kNsThreads) void ns_load_kernel(const NsSource s, int rows, int cols, int tall, int chunks, const double* sums, float eps, uint16_t* hi, uint16_t* lo, int64_t stride,
                                                                                 int ld, int tiles_r, int tiles_c) {
  __shared__ float tile[64][65];
  __shared__ double waves[kNsThreads / 64];
  const int per = tiles_r * tiles_c, m = blockIdx.x / per, t = blockIdx.x % per;
  const int r0 = t / tiles_c * 64, c0 = t % tiles_c * 64;
  const int y0 = threadIdx.x >> 3, x0 = (threadIdx.x & 7) * 8;  // two rows of 32 apart, eight values each
  float v[2][8];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r = r0 + y0 + 32 * q, n = r < rows ? min(8, cols - c0 - x0) : 0;
#pragma unroll
    for (int x = 0; x < 8; ++x) v[q][x] = 0.f;
    if (n > 0) ns_direction<VEC>(v[q], s, ((int64_t)m * rows + r) * cols + c0 + x0, n, false);
  }
  double sum = 0.0;
  for (int i = threadIdx.x; i < chunks; i += kNsThreads) sum += sums[(int64_t)m * chunks + i];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
  if (lane_id() == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kNsThreads / 64; ++w) sum += waves[w];
  const float inv = (float)((double)kNsScale / (sqrt(sum) + (double)eps));
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int x = 0; x < 8; ++x) v[q][x] *= inv;
  if (!tall) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (r0 + y0 + 32 * q < rows && c0 + x0 < ld) ns_store_planes(hi, lo, m * stride + (int64_t)(r0 + y0 + 32 * q) * ld + c0 + x0, v[q]);
    return;
  }
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int x = 0; x < 8; ++x) tile[y0 + 32 * q][x0 + x] = v[q][x];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r = c0 + y0 + 32 * q, c = r0 + x0;
#pragma unroll
    for (int x = 0; x < 8; ++x) v[q][x] = tile[x0 + x][y0 + 32 * q];
    if (r < cols && c < ld) ns_store_planes(hi, lo, m * stride + (int64_t)r * ld + c, v[q]);
  }
}

// Out of the planes where the last step's update cannot: transposed results of more than 16 bits or with weights, odd ones, and those of no steps at all.
template <bool VEC> __global__ __launch_bounds__(kNsThreads) void ns_store_kernel(const NsTarget o, int rows, int cols, int tall, const uint16_t* hi, const uint16_t* lo, int64_t stride, int ld, int tiles_r, int tiles_c) {
  __shared__ float tile[64][65];
  const int per = tiles_r * tiles_c, m = blockIdx.x / per, t = blockIdx.x % per;
  const int r0 = t / tiles_c * 64, c0 = t % tiles_c * 64;  // of the result
  const int p_rows = tall ? cols : rows, pr0 = tall ? c0 : r0, pc0 = tall ? r0 : c0;
  const int y0 = threadIdx.x >> 3, x0 = (threadIdx.x & 7) * 8;
  float v[2][8];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    i32x4_t a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    if (pr0 + y0 + 32 * q < p_rows && pc0 + x0 < ld) {
      const int64_t i = m * stride + (int64_t)(pr0 + y0 + 32 * q) * ld + pc0 + x0;
      a = *(const i32x4_t*)(hi + i);
      b = *(const i32x4_t*)(lo + i);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) v[q][x] = (ns_f16((uint16_t)((uint32_t)a[x / 2] >> (16 * (x & 1)))) + ns_f16((uint16_t)((uint32_t)b[x / 2] >> (16 * (x & 1))))) * (1.f / kNsScale);
  }
  if (tall) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int x = 0; x < 8; ++x) tile[y0 + 32 * q][x0 + x] = v[q][x];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int x = 0; x < 8; ++x) v[q][x] = tile[x0 + x][y0 + 32 * q];
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r = r0 + y0 + 32 * q, n = r < rows ? min(8, cols - c0 - x0) : 0;
    if (n <= 0) continue;
    const int64_t i = ((int64_t)m * rows + r) * cols + c0 + x0;
    if (o.weight) {
      float old[8];
      ns_load8<VEC>(old, o.out, i, o.dt, n);
#pragma unroll
      for (int x = 0; x < 8; ++x) v[q][x] = ns_stepped(o, old[x], v[q][x]);
    }
    ns_store8<VEC>(o.out, i, o.dt, v[q], n);
  }
}

typedef StreamCfg<256, 256, 2, 4> NsWide;
typedef StreamCfg<128, 128, 2, 4> NsNarrow;
typedef StreamCfg<64, 64, 2, 4, 8> NsSmall;

template <class C, int MODE> int ns_launch(const NsProduct& p, hipStream_t s) {
  typedef NsProblem<C, MODE> P;
  static bool attr_set[64] = {false};
  if (int e = stream_lds(ns_product_kernel<C, MODE>, P::SMEM_BYTES, attr_set)) return e;
  const int tm = (p.rows + C::BM - 1) / C::BM, tn = (p.cols + C::BN - 1) / C::BN;
  const int64_t tiles = (int64_t)p.batch * (P::SYM ? tm * (tm + 1) / 2 : tm * tn);
  const int slots = num_cus() * (int)(160 * 1024 / P::SMEM_BYTES);
  ns_product_kernel<C, MODE><<<dim3((unsigned)(tiles < slots ? tiles : slots)), dim3(C::THREADS), P::SMEM_BYTES, s>>>(p, tm, tn);
  return check_launch("ns_product");
}

template <int MODE> int ns_product(const NsProduct& p, int tile, hipStream_t s) { return tile == 64 ? ns_launch<NsSmall, MODE>(p, s) : tile == 256 ? ns_launch<NsWide, MODE>(p, s) : ns_launch<NsNarrow, MODE>(p, s); }

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int64_t ns_align(int64_t x) { return (x + 255) & ~(int64_t)255; }

// Where everything is in the workspace, and how the products are tiled.
struct NsPlan {
  int m, n, ldm, ldn, chunks;
  bool tall;
  int gram_tile, poly_tile, update_tile;
  int gram_tiles, update_tiles;
  int64_t x_plane, g_plane;  // elements of a plane of all matrices
  int64_t off_x, off_a, off_b, off_sums, off_xs[2], off_as, bytes;
};

// Tiles of 64, 128 or 256 for a product of `slabs` slabs of depth a tile: the estimated time in microseconds, from the rounds of workgroups and what a tile took.  A round of 256-row
// tiles: 1.65 a slab and 24 for results and start; of two 128-row tiles a compute unit 1.2 and 10, of one 0.8 and 8; of one 64-row tile, with eight slabs in flight, 0.38 and 1.  Measured for stacks of
// 1 to 64 matrices of 128 to 2048 rows, the choice was the fastest or within 3 % of it, but for 64 matrices of 256 x 512 and 512 x 512 (9 and 12 %); the other tiles took up to 3 times as long (five steps in tiles of 64, 128 and 256:
// 512 x 512 215, 307 and 594 us; 8 of 768 x 2048 1604, 919 and 1256; 64 of 1536 x 2048 52.2, 21.1 and 17.5 ms).
int ns_tile(int64_t batch, int rows, int cols, bool sym, int64_t slabs) {
  auto tiles = [&](int b) { const int64_t tm = (rows + b - 1) / b, tn = (cols + b - 1) / b; return batch * (sym ? tm * (tm + 1) / 2 : tm * tn); };
  const int64_t cus = num_cus(), full = tiles(128) / (2 * cus), rest = tiles(128) % (2 * cus);
  const double pair = 1.2 * slabs + 10;
  const double small = (tiles(64) + cus - 1) / cus * (0.38 * slabs + 1), wide = (tiles(256) + cus - 1) / cus * (1.65 * slabs + 24);
  const double narrow = full * pair + (rest == 0 ? 0 : rest <= cus ? 0.8 * slabs + 8 : pair);
  return small <= narrow && small <= wide ? 64 : narrow <= wide ? 128 : 256;
}

NsPlan ns_plan(int64_t batch, int rows, int cols) {
  NsPlan q;
  q.tall = rows > cols;
  q.m = q.tall ? cols : rows;
  q.n = q.tall ? rows : cols;
  q.ldm = (q.m + 7) & ~7;
  q.ldn = (q.n + 7) & ~7;
  q.chunks = (int)(((int64_t)rows * cols + kNsChunk - 1) / kNsChunk);
  const int deep = (q.n + 63) / 64 * 3, shallow = (q.m + 63) / 64 * 3;
  q.gram_tile = ns_tile(batch, q.m, q.m, true, deep);
  q.poly_tile = ns_tile(batch, q.m, q.m, true, shallow);
  q.update_tile = ns_tile(batch, q.m, q.n, false, shallow);
  const int bg = q.gram_tile, bu = q.update_tile;
  const int tg = (q.m + bg - 1) / bg;
  q.gram_tiles = tg * (tg + 1) / 2;
  q.update_tiles = ((q.m + bu - 1) / bu) * ((q.n + bu - 1) / bu);
  q.x_plane = batch * q.m * q.ldn;
  q.g_plane = batch * q.m * q.ldm;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t here = at; at += ns_align(bytes); return here; };
  q.off_x = take(0);
  for (int i = 0; i < 4; ++i) take(q.x_plane * 2);  // two X, two planes each; plane i at off_x + i * ns_align(x_plane * 2)
  q.off_a = take(0);
  for (int i = 0; i < 4; ++i) take(q.g_plane * 2);  // A and B
  q.off_b = q.off_a + 2 * ns_align(q.g_plane * 2);
  q.off_sums = take(batch * q.chunks * 8);
  for (int64_t& xs : q.off_xs) xs = take(batch * q.update_tiles * 4);  // (an update's tiles read the sums of the step before while others write)
  q.off_as = take(batch * q.gram_tiles * 4);
  q.bytes = at;
  return q;
}

}  // namespace

int64_t newton_schulz_workspace(int64_t batch, int rows, int cols) { return ns_plan(batch, rows, cols).bytes; }

// x -> out, or with momentum the weights' step on out.  dt: 0 bf16, 1 fp16, 2 fp32
int launch_newton_schulz(const void* x, int x_dt, float* momentum, double beta, int nesterov, void* out, int out_dt, int weight, float keep, float step, int64_t batch, int rows, int cols, int steps,
                         float ca, float cb, float cc, float eps, void* workspace, hipStream_t s) {
  const NsPlan q = ns_plan(batch, rows, cols);
  char* const ws = (char*)workspace;
  const int64_t xp = ns_align(q.x_plane * 2), gp = ns_align(q.g_plane * 2);
  uint16_t* xs[2][2] = {{(uint16_t*)(ws + q.off_x), (uint16_t*)(ws + q.off_x + xp)}, {(uint16_t*)(ws + q.off_x + 2 * xp), (uint16_t*)(ws + q.off_x + 3 * xp)}};
  uint16_t *a_hi = (uint16_t*)(ws + q.off_a), *a_lo = (uint16_t*)(ws + q.off_a + gp), *b_hi = (uint16_t*)(ws + q.off_b), *b_lo = (uint16_t*)(ws + q.off_b + gp);
  double* sums = (double*)(ws + q.off_sums);
  float* const x_sums[2] = {(float*)(ws + q.off_xs[0]), (float*)(ws + q.off_xs[1])};
  float* const a_sums = (float*)(ws + q.off_as);
  const NsSource src = {x, momentum, (float)beta, (float)(1.0 - beta), nesterov, x_dt};
  const bool vec_in = ((int64_t)rows * cols & 7) == 0 && aligned16(x) && aligned16(momentum), vec_rows = (cols & 7) == 0;
  const dim3 threads(kNsThreads), norm_grid((unsigned)(batch * q.chunks));
  if (vec_in) ns_norm_kernel<true><<<norm_grid, threads, 0, s>>>(src, (int64_t)rows * cols, q.chunks, sums);
  else ns_norm_kernel<false><<<norm_grid, threads, 0, s>>>(src, (int64_t)rows * cols, q.chunks, sums);
  if (int e = check_launch("ns_norm")) return e;
  // tiles cover the planes' padding too: columns up to a multiple of 8
  const int tr = ((q.tall ? q.ldn : rows) + 63) / 64, tc = ((q.tall ? cols : q.ldn) + 63) / 64;
  const dim3 load_grid((unsigned)(batch * tr * tc));
  if (vec_in && vec_rows) ns_load_kernel<true><<<load_grid, threads, 0, s>>>(src, rows, cols, q.tall, q.chunks, sums, eps, xs[0][0], xs[0][1], (int64_t)q.m * q.ldn, q.ldn, tr, tc);
  else ns_load_kernel<false><<<load_grid, threads, 0, s>>>(src, rows, cols, q.tall, q.chunks, sums, eps, xs[0][0], xs[0][1], (int64_t)q.m * q.ldn, q.ldn, tr, tc);
  if (int e = check_launch("ns_load")) return e;
  const NsTarget dst = {out, out_dt, weight, vec_rows && aligned16(out), keep, step};
  // the last step's update writes rows of the result; transposed ones if they are plain 16-bit values in whole eights
  const bool direct = steps > 0 && (q.tall ? !weight && out_dt != 2 && (q.m & 7) == 0 && aligned16(out) : true);
  const int64_t xstride = (int64_t)q.m * q.ldn, gstride = (int64_t)q.m * q.ldm;
  for (int i = 0; i < steps; ++i) {
    uint16_t **from = xs[i & 1], **to = xs[(i + 1) & 1];
    NsProduct p = {};
    p.batch = (int)batch;
    p.ca = ca; p.cb = cb; p.cc = cc;
    p.x_sums = x_sums[i & 1]; p.a_sums = a_sums;
    p.x_tiles = i ? q.update_tiles : 0;
    p.a_tiles = q.gram_tiles;
    p.rows = p.cols = q.m;
    p.depth = q.n;
    p.a_hi = p.b_hi = from[0]; p.a_lo = p.b_lo = from[1];
    p.lda = p.ldb = q.ldn; p.a_stride = p.b_stride = xstride;
    p.o_hi = a_hi; p.o_lo = a_lo; p.ldo = q.ldm; p.o_stride = gstride; p.o_sums = a_sums;
    if (int e = ns_product<NS_GRAM>(p, q.gram_tile, s)) return e;
    p.depth = q.m;
    p.a_hi = p.b_hi = p.c_hi = a_hi; p.a_lo = p.b_lo = p.c_lo = a_lo;
    p.lda = p.ldb = q.ldm; p.a_stride = p.b_stride = gstride;
    p.o_hi = b_hi; p.o_lo = b_lo; p.o_sums = nullptr;
    if (int e = ns_product<NS_POLY>(p, q.poly_tile, s)) return e;
    p.cols = q.n;
    p.a_hi = b_hi; p.a_lo = b_lo;
    p.b_hi = p.c_hi = from[0]; p.b_lo = p.c_lo = from[1]; p.ldb = q.ldn; p.b_stride = xstride;
    p.o_hi = to[0]; p.o_lo = to[1]; p.ldo = q.ldn; p.o_stride = xstride; p.o_sums = x_sums[(i + 1) & 1];
    p.target = dst;
    p.tall = q.tall;
    if (direct && i == steps - 1) return ns_product<NS_LAST>(p, q.update_tile, s);
    if (int e = ns_product<NS_UPDATE>(p, q.update_tile, s)) return e;
  }
  const int sr = (rows + 63) / 64, sc = (cols + 63) / 64;
  const dim3 store_grid((unsigned)(batch * sr * sc));
  if (dst.whole) ns_store_kernel<true><<<store_grid, threads, 0, s>>>(dst, rows, cols, q.tall, xs[steps & 1][0], xs[steps & 1][1], xstride, q.ldn, sr, sc);
  else ns_store_kernel<false><<<store_grid, threads, 0, s>>>(dst, rows, cols, q.tall, xs[steps & 1][0], xs[steps & 1][1], xstride, q.ldn, sr, sc);
  return check_launch("ns_store");
}

}  // namespace tgg
