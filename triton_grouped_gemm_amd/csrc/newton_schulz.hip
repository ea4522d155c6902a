// Newton-Schulz orthogonalisation of a stack of matrices, and the optimiser's step that uses it.
//
//   X_0 = X / (|X|_F + eps);   G = X X^T,   X <- a X + (b G + c G^2) X      once a step
//
// X is taken as [M, N] with M <= N (a tall matrix is transposed on its way in and out: the iteration commutes with it).  Every X and G is held as two
// planes of half precision, high and low, 22 bits together, scaled by 2^10 so that the low plane keeps its bits: singular values
// stay near or below 1, so entries do not overflow.
//
// Results in bfloat16 are multiplied from the high planes alone, 11 bits, with what the rounding would reach first taken out of the products:
// the sum that carries X over, a X, and the linear term of the polynomial use both planes, and G and the polynomial enter the products less their mean diagonal, whose part is
// exact:   A = G - d I,   B = (b + 2 c d) A + c (A^2 - e I),   X <- (a + b d + c d^2 + c e) X + B X,   d = |X|^2 / M,   e = |A|^2 / M.
// The rounding of near-identity matrices is then that of what is left of them.  Errors against 64 bits, before the last rounding (random and low-rank matrices of 256 to 768 rows): 2e-4 to 1.1e-3, where
// G and B with their diagonals give up to 2.6e-3 and bfloat16 operands 2e-2; the result's own rounding is 1.7e-3.  Results in half precision and fp32 add the products of
// high and low planes, three multiplies for one, and are as good as fp32 products.
//
// G and G^2 are symmetric: only tiles on and below the diagonal are computed, and stored twice.  No sum depends on the order of arrival: norms are
// summed per tile and the tiles' sums in order.
#include <type_traits>

#include "launch.hpp"
#include "stream_gemm.hpp"

namespace tgg {

enum : int { NS_GRAM = 0, NS_POLY = 1, NS_UPDATE = 2 };

constexpr float kNsScale = 1024.f, kNsInv2 = 1.f / (1024.f * 1024.f);

// One product for all matrices.  Planes: element (m, i, j) at m * stride + i * ld + j.
struct NsProduct {
  const uint16_t *a_hi, *a_lo, *b_hi, *b_lo;  // operands: GRAM X, X; POLY A, A; UPDATE B, X
  uint16_t *o_hi, *o_lo;                      // result's planes; o_lo may be null
  const uint16_t *c_hi, *c_lo;                // what the epilogue adds: POLY A, UPDATE X
  int64_t a_stride, b_stride, o_stride;       // per matrix, in elements
  int lda, ldb, ldo;
  int rows, cols, depth;                      // the result's size and the sum's length
  int batch;
  float ca, cb, cc;                           // the polynomial's coefficients
  const float *x_sums, *a_sums;               // |X|^2 and |A|^2 by tile, x_tiles and a_tiles a matrix
  float* o_sums;                              // the result's (GRAM, UPDATE)
  int x_tiles, a_tiles;                       // x_tiles 0: the first step, d = 1 / M
};

namespace {

struct NsSplit { uint16_t hi, lo; };
TGG_DEV NsSplit ns_split(float v) {
  const _Float16 h = (_Float16)v;
  const _Float16 l = (_Float16)(v - (float)h);
  return {__builtin_bit_cast(uint16_t, h), __builtin_bit_cast(uint16_t, l)};
}
TGG_DEV float ns_f16(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }

// the n sums of a matrix, added by a wave: every lane gets the same bits, and every workgroup
TGG_DEV float ns_sum(const float* p, int n) {
  float s = 0.f;
  for (int i = lane_id(); i < n; i += 64) s += p[i];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d, 64);
  return s;
}

template <class C, int MODE, bool PRECISE> struct NsProblem {
  static constexpr bool B_KMAJOR = MODE != NS_UPDATE, SYM = MODE != NS_UPDATE;
  static_assert(!SYM || C::BM == C::BN, "symmetric results have square tiles");
  static constexpr int PITCH = C::TN * 32 + 16;  // staged strip of 16 rows: bytes between rows
  static constexpr int STAGE_WAVE = 16 * PITCH;
  static constexpr int SUMS_OFF = C::NWAVES * STAGE_WAVE;
  static constexpr int SMEM_BYTES = C::EPI_OFF + SUMS_OFF + C::NWAVES * 4;

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
  TGG_DEV int slabs(int) const { return PRECISE ? 3 * cur.kt : cur.kt; }
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
    const uint16_t* const a = PRECISE && pass == 2 ? p.a_lo : p.a_hi;
    const uint16_t* const b = PRECISE && pass == 1 ? p.b_lo : p.b_hi;
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
    if (PRECISE && pass < 2) {
      ++pass;
      begin_pass();
    } else {
      seek(tile_at(pos + 1));
    }
  }
  TGG_DEV void begin(int, f32x4_t (&)[C::TM][C::TN], const StreamPlace<C>&) const {}

  TGG_DEV void epilogue(int id, f32x4_t (&acc)[C::TM][C::TN], const StreamPlace<C>& at, char* stage) const {
    int el = at.lane;
    asm volatile("" : "+v"(el));  // (addresses are made afresh per tile instead of living across the multiplies)
    const int l16 = el & 15, lg = el >> 4;
    const Place tile = locate(id);
    const int m = tile.m, row0 = tile.row0, col0 = tile.col0;
    const float inv_rows = 1.f / (float)p.rows;
    const float d = p.x_tiles ? ns_sum(p.x_sums + (int64_t)m * p.x_tiles, p.x_tiles) * inv_rows : inv_rows;
    const float e = MODE == NS_GRAM ? 0.f : ns_sum(p.a_sums + (int64_t)m * p.a_tiles, p.a_tiles) * inv_rows;
    // the result is f acc + g C, less h on the diagonal, all times kNsScale
    const float f = (MODE == NS_POLY ? p.cc : 1.f) * kNsInv2;
    const float g = MODE == NS_POLY ? p.cb + 2.f * p.cc * d : MODE == NS_UPDATE ? p.ca + p.cb * d + p.cc * d * d + p.cc * e : 0.f;
    const float h = MODE == NS_GRAM ? d : MODE == NS_POLY ? p.cc * e : 0.f;
    const int64_t base = m * p.o_stride;
    const int rbase = row0 + at.wm0, cbase = col0 + at.wn0;
    const bool mirror = SYM && row0 != col0;
    char* const mine = stage + at.wave * STAGE_WAVE;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
      const int row = rbase + 16 * i + l16;
      uint2 hi[C::TN], lo[C::TN];
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        const int col = cbase + 16 * j + 4 * lg;
        const bool there = row < p.rows && col < p.ldo;
        const int64_t o = base + (int64_t)row * p.ldo + col;
        uint2 ch = {0, 0}, cl = {0, 0};
        if (MODE != NS_GRAM && there) {
          ch = *(const uint2*)(p.c_hi + o);
          cl = *(const uint2*)(p.c_lo + o);
        }
        float v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float c = 0.f;
          if (MODE != NS_GRAM) {
            const uint32_t wh = x < 2 ? ch.x : ch.y, wl = x < 2 ? cl.x : cl.y;
            c = ns_f16((uint16_t)(wh >> (16 * (x & 1)))) + ns_f16((uint16_t)(wl >> (16 * (x & 1))));
          }
          const float r = f * kNsScale * acc[i][j][x] + g * c - (SYM && row == col + x ? h * kNsScale : 0.f);
          v[x] = row < p.rows && col + x < p.cols ? r : 0.f;  // (what lies beyond is a sum of whatever the operands' next rows hold)
          sum += v[x] * v[x];
        }
        uint16_t a[4], b[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const NsSplit s = ns_split(v[x]);
          a[x] = s.hi;
          b[x] = s.lo;
        }
        hi[j] = {(uint32_t)a[0] | (uint32_t)a[1] << 16, (uint32_t)a[2] | (uint32_t)a[3] << 16};
        lo[j] = {(uint32_t)b[0] | (uint32_t)b[1] << 16, (uint32_t)b[2] | (uint32_t)b[3] << 16};
        if (there) {
          *(uint2*)(p.o_hi + o) = hi[j];
          if (p.o_lo) *(uint2*)(p.o_lo + o) = lo[j];
        }
      }
      if (SYM && mirror) {
        // transposed through LDS: rows of the mirrored tile are this strip's columns, 16 values of each
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
          uint16_t* const out = plane ? p.o_lo : p.o_hi;
          if (out) {
#pragma unroll
            for (int j = 0; j < C::TN; ++j) *(uint2*)(mine + l16 * PITCH + (16 * j + 4 * lg) * 2) = plane ? lo[j] : hi[j];
            asm volatile("" : : : "memory");  // read as another type, by other lanes of the wave; its LDS operations complete in order
#pragma unroll
            for (int it = 0; it < (C::TN * 32 + 63) / 64; ++it) {
              const int idx = it * 64 + el, c = idx >> 1, r0 = (idx & 1) * 8;  // 8 rows of column c
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x)
                w[x] = (uint32_t)*(const uint16_t*)(mine + (r0 + 2 * x) * PITCH + c * 2) | (uint32_t)*(const uint16_t*)(mine + (r0 + 2 * x + 1) * PITCH + c * 2) << 16;
              const int orow = cbase + c, ocol = rbase + 16 * i + r0;
              if (orow < p.cols && ocol < p.ldo) {
                const i32x4_t q = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
                *(i32x4_t*)(out + base + (int64_t)orow * p.ldo + ocol) = q;
              }
            }
            asm volatile("" : : : "memory");
          }
        }
      }
    }
    if (MODE != NS_POLY) {
      if (mirror) sum *= 2.f;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
      float* const sums = (float*)(stage + SUMS_OFF);
      __syncthreads();  // the sums of the tile before have been read
      if (el == 0) sums[at.wave] = sum;
      __syncthreads();
      if (threadIdx.x == 0) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < C::NWAVES; ++w) s += sums[w];
        p.o_sums[id] = s * kNsInv2;
      }
    }
  }
};

template <class C, int MODE, bool PRECISE> __global__ __launch_bounds__(C::THREADS) void ns_product_kernel(const NsProduct p, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  NsProblem<C, MODE, PRECISE> prob(p, tiles_m, tiles_n);
  stream_gemm<C, DT_F16, NsProblem<C, MODE, PRECISE>::B_KMAJOR>(prob, smem);
}

// ---- into the planes and out of them -------------------------------------------------------------------------------------

constexpr int kNsThreads = 256, kNsChunk = 16384;  // values of a workgroup's sum of squares

TGG_DEV float ns_load(const void* p, int64_t i, int dt) {  // dt 0 bf16, 1 fp16, 2 fp32
  if (dt == 2) return ((const float*)p)[i];
  const uint16_t h = ((const uint16_t*)p)[i];
  return dt == 0 ? __builtin_bit_cast(float, (uint32_t)h << 16) : ns_f16(h);
}

// What is orthogonalised: x, or, with momentum, the momentum's value after this step and with Nesterov's look ahead.
struct NsSource {
  const void* x;   // the input or the gradient
  float* momentum; // or null
  float beta, keep;  // keep = 1 - beta
  int nesterov, dt;
};
TGG_DEV float ns_direction(const NsSource& s, int64_t i, float m) {
  const float x = ns_load(s.x, i, s.dt);
  if (!s.momentum) return x;
  return s.nesterov ? s.beta * m + s.keep * x : m;
}

// Sums of squares of a matrix's chunks; with momentum, its step.
__global__ __launch_bounds__(kNsThreads) void ns_norm_kernel(const NsSource s, int64_t values, int chunks, double* sums) {
  const int m = blockIdx.x / chunks, c = blockIdx.x % chunks;
  const int64_t first = m * values + (int64_t)c * kNsChunk, end = min(first + kNsChunk, (m + 1) * values);
  double sum = 0.0;
  for (int64_t i = first + threadIdx.x; i < end; i += kNsThreads) {
    float mom = 0.f;
    if (s.momentum) {
      mom = s.beta * s.momentum[i] + s.keep * ns_load(s.x, i, s.dt);
      s.momentum[i] = mom;
    }
    const double v = ns_direction(s, i, mom);
    sum += v * v;
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

// Tiles of 64 x 64 into the planes, transposed where the matrix is tall.
__global__ __launch_bounds__(kNsThreads) void ns_load_kernel(const NsSource s, int rows, int cols, int tall, int chunks, const double* sums, float eps, uint16_t* hi, uint16_t* lo, int64_t stride,
                                                             int ld, int tiles_r, int tiles_c) {
  __shared__ float tile[64][65];
  __shared__ double waves[kNsThreads / 64];
  const int per = tiles_r * tiles_c, m = blockIdx.x / per, t = blockIdx.x % per;
  const int r0 = t / tiles_c * 64, c0 = t % tiles_c * 64;
  double sum = 0.0;
  for (int i = threadIdx.x; i < chunks; i += kNsThreads) sum += sums[(int64_t)m * chunks + i];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
  if (lane_id() == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kNsThreads / 64; ++w) sum += waves[w];
  const float inv = (float)((double)kNsScale / (sqrt(sum) + (double)eps));
  const int x = threadIdx.x & 63;
  for (int y = threadIdx.x >> 6; y < 64; y += kNsThreads / 64) {
    float v = 0.f;
    if (r0 + y < rows && c0 + x < cols) {
      const int64_t i = ((int64_t)m * rows + r0 + y) * cols + c0 + x;
      v = ns_direction(s, i, s.momentum ? s.momentum[i] : 0.f) * inv;
    }
    tile[y][x] = v;
  }
  __syncthreads();
  const int o_rows = tall ? cols : rows, or0 = tall ? c0 : r0, oc0 = tall ? r0 : c0;
  for (int y = threadIdx.x >> 6; y < 64; y += kNsThreads / 64) {
    if (or0 + y < o_rows && oc0 + x < ld) {
      const NsSplit v = ns_split(tall ? tile[x][y] : tile[y][x]);
      const int64_t o = m * stride + (int64_t)(or0 + y) * ld + oc0 + x;
      hi[o] = v.hi;
      lo[o] = v.lo;
    }
  }
}

// Out of the planes: out = v, or with `weight` out = keep out - step v.
struct NsTarget {
  void* out;
  int dt, weight;
  float keep, step;
};
__global__ __launch_bounds__(kNsThreads) void ns_store_kernel(const NsTarget o, int rows, int cols, int tall, const uint16_t* hi, const uint16_t* lo, int64_t stride, int ld, int tiles_r, int tiles_c) {
  __shared__ float tile[64][65];
  const int per = tiles_r * tiles_c, m = blockIdx.x / per, t = blockIdx.x % per;
  const int r0 = t / tiles_c * 64, c0 = t % tiles_c * 64;  // of the result
  const int p_rows = tall ? cols : rows, p_cols = tall ? rows : cols, pr0 = tall ? c0 : r0, pc0 = tall ? r0 : c0;
  const int x = threadIdx.x & 63;
  for (int y = threadIdx.x >> 6; y < 64; y += kNsThreads / 64) {
    float v = 0.f;
    if (pr0 + y < p_rows && pc0 + x < p_cols) {
      const int64_t i = m * stride + (int64_t)(pr0 + y) * ld + pc0 + x;
      v = (ns_f16(hi[i]) + ns_f16(lo[i])) * (1.f / kNsScale);
    }
    if (tall) tile[x][y] = v; else tile[y][x] = v;
  }
  __syncthreads();
  for (int y = threadIdx.x >> 6; y < 64; y += kNsThreads / 64) {
    if (r0 + y >= rows || c0 + x >= cols) continue;
    const int64_t i = ((int64_t)m * rows + r0 + y) * cols + c0 + x;
    float v = tile[y][x];
    if (o.weight) v = o.keep * ns_load(o.out, i, o.dt) - o.step * v;
    if (o.dt == 2) ((float*)o.out)[i] = v;
    else ((uint16_t*)o.out)[i] = o.dt == 0 ? Out16<DT_BF16>::cvt(v) : Out16<DT_F16>::cvt(v);
  }
}

typedef StreamCfg<256, 256, 2, 4> NsWide;
typedef StreamCfg<128, 128, 2, 4> NsNarrow;

template <class C, int MODE, bool PRECISE> int ns_launch(const NsProduct& p, hipStream_t s) {
  typedef NsProblem<C, MODE, PRECISE> P;
  static bool attr_done = false;
  if (!attr_done) {
    if (hipFuncSetAttribute((const void*)ns_product_kernel<C, MODE, PRECISE>, hipFuncAttributeMaxDynamicSharedMemorySize, P::SMEM_BYTES) != hipSuccess) return check_launch("hipFuncSetAttribute(ns_product)");
    attr_done = true;
  }
  const int tm = (p.rows + C::BM - 1) / C::BM, tn = (p.cols + C::BN - 1) / C::BN;
  const int64_t tiles = (int64_t)p.batch * (P::SYM ? tm * (tm + 1) / 2 : tm * tn);
  const int slots = num_cus() * (C::BM == 128 ? 2 : 1);
  ns_product_kernel<C, MODE, PRECISE><<<dim3((unsigned)(tiles < slots ? tiles : slots)), dim3(C::THREADS), P::SMEM_BYTES, s>>>(p, tm, tn);
  return check_launch("ns_product");
}

template <int MODE> int ns_product(const NsProduct& p, bool wide, bool precise, hipStream_t s) {
  if (wide) return precise ? ns_launch<NsWide, MODE, true>(p, s) : ns_launch<NsWide, MODE, false>(p, s);
  return precise ? ns_launch<NsNarrow, MODE, true>(p, s) : ns_launch<NsNarrow, MODE, false>(p, s);
}

int64_t ns_align(int64_t x) { return (x + 255) & ~(int64_t)255; }

// Where everything is in the workspace, and how the products are tiled.
struct NsPlan {
  int m, n, ldm, ldn, chunks;
  bool tall, wide_gram, wide_poly, wide_update;
  int gram_tiles, update_tiles;
  int64_t x_plane, g_plane;  // elements of a plane of all matrices
  int64_t off_x, off_a, off_b, off_sums, off_xs[2], off_as, bytes;
};

// Tiles of 256 or of 128: rounds of the compute units (two workgroups of the narrow tiles share one).  A quarter of a wide tile's work takes a narrow one about a third of its time.
bool ns_wide(int64_t batch, int rows, int cols, bool sym) {
  auto tiles = [&](int b) { const int64_t tm = (rows + b - 1) / b, tn = (cols + b - 1) / b; return batch * (sym ? tm * (tm + 1) / 2 : tm * tn); };
  const int64_t cus = num_cus();
  const int64_t wide = (tiles(256) + cus - 1) / cus * 3, narrow = (tiles(128) + 2 * cus - 1) / (2 * cus) * 2;
  return wide <= narrow;
}

NsPlan ns_plan(int64_t batch, int rows, int cols) {
  NsPlan q;
  q.tall = rows > cols;
  q.m = q.tall ? cols : rows;
  q.n = q.tall ? rows : cols;
  q.ldm = (q.m + 7) & ~7;
  q.ldn = (q.n + 7) & ~7;
  q.chunks = (int)(((int64_t)rows * cols + kNsChunk - 1) / kNsChunk);
  q.wide_gram = q.wide_poly = ns_wide(batch, q.m, q.m, true);
  q.wide_update = ns_wide(batch, q.m, q.n, false);
  const int bg = q.wide_gram ? 256 : 128, bu = q.wide_update ? 256 : 128;
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
int launch_newton_schulz(const void* x, int x_dt, float* momentum, float beta, int nesterov, void* out, int out_dt, int weight, float keep, float step, int64_t batch, int rows, int cols, int steps,
                         float ca, float cb, float cc, float eps, void* workspace, hipStream_t s) {
  const NsPlan q = ns_plan(batch, rows, cols);
  char* const ws = (char*)workspace;
  const int64_t xp = ns_align(q.x_plane * 2), gp = ns_align(q.g_plane * 2);
  uint16_t* xs[2][2] = {{(uint16_t*)(ws + q.off_x), (uint16_t*)(ws + q.off_x + xp)}, {(uint16_t*)(ws + q.off_x + 2 * xp), (uint16_t*)(ws + q.off_x + 3 * xp)}};
  uint16_t *a_hi = (uint16_t*)(ws + q.off_a), *a_lo = (uint16_t*)(ws + q.off_a + gp), *b_hi = (uint16_t*)(ws + q.off_b), *b_lo = (uint16_t*)(ws + q.off_b + gp);
  double* sums = (double*)(ws + q.off_sums);
  float* const x_sums[2] = {(float*)(ws + q.off_xs[0]), (float*)(ws + q.off_xs[1])};
  float* const a_sums = (float*)(ws + q.off_as);
  const bool precise = out_dt != 0;  // results of more than 8 bits
  const NsSource src = {x, momentum, beta, 1.f - beta, nesterov, x_dt};
  ns_norm_kernel<<<dim3((unsigned)(batch * q.chunks)), dim3(kNsThreads), 0, s>>>(src, (int64_t)rows * cols, q.chunks, sums);
  if (int e = check_launch("ns_norm")) return e;
  // tiles cover the planes' padding too: columns up to a multiple of 8
  const int tr = ((q.tall ? q.ldn : rows) + 63) / 64, tc = ((q.tall ? cols : q.ldn) + 63) / 64;
  ns_load_kernel<<<dim3((unsigned)(batch * tr * tc)), dim3(kNsThreads), 0, s>>>(src, rows, cols, q.tall, q.chunks, sums, eps, xs[0][0], xs[0][1], (int64_t)q.m * q.ldn, q.ldn, tr, tc);
  if (int e = check_launch("ns_load")) return e;
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
    if (int e = ns_product<NS_GRAM>(p, q.wide_gram, precise, s)) return e;
    p.depth = q.m;
    p.a_hi = p.b_hi = p.c_hi = a_hi; p.a_lo = p.b_lo = p.c_lo = a_lo;
    p.lda = p.ldb = q.ldm; p.a_stride = p.b_stride = gstride;
    p.o_hi = b_hi; p.o_lo = precise ? b_lo : nullptr; p.o_sums = nullptr;
    if (int e = ns_product<NS_POLY>(p, q.wide_poly, precise, s)) return e;
    p.cols = q.n;
    p.a_hi = b_hi; p.a_lo = b_lo;
    p.b_hi = p.c_hi = from[0]; p.b_lo = p.c_lo = from[1]; p.ldb = q.ldn; p.b_stride = xstride;
    p.o_hi = to[0]; p.o_lo = to[1]; p.ldo = q.ldn; p.o_stride = xstride; p.o_sums = x_sums[(i + 1) & 1];
    if (int e = ns_product<NS_UPDATE>(p, q.wide_update, precise, s)) return e;
  }
  const NsTarget dst = {out, out_dt, weight, keep, step};
  const int sr = (rows + 63) / 64, sc = (cols + 63) / 64;
  ns_store_kernel<<<dim3((unsigned)(batch * sr * sc)), dim3(kNsThreads), 0, s>>>(dst, rows, cols, q.tall, xs[steps & 1][0], xs[steps & 1][1], xstride, q.ldn, sr, sc);
  return check_launch("ns_store");
}

}  // namespace tgg
