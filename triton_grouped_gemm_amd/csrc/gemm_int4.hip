// Grouped products with 4-bit weights and group scales, for the rows of a decode step:
//   out[r, n] = sum_k x[r, k] (q[n, k] - z[n, k / gs]) s[n, k / gs],   q in 0..15, z = 8 unless given,
// plain, or as a gated block (N = 2 F: out = act(first F) * last F).
//
// Few rows share a group's weights, so a launch is bound by reading the codes once: N K / 2 bytes per group with rows.  The codes are stored as the
// kernel reads them: blocks of 16 columns x 128 values, 1 KB each, of which lane (l16, lg) of a wave holds in 16 consecutive bytes what four
// 16x16x32 multiplies want from column l16: value 32 s + 8 lg + e of the block is nibble e (in the order 0 2 4 6 1 3 5 7) of word s.  A load instruction
// is one contiguous kilobyte, and every multiply covers 32 consecutive values, so scale groups of 32 need no other layout than those of 128.
//
// Codes become operands without arithmetic: in bfloat16 0x4300 | q is 128 + q (the nibble order makes a masked shift a pair of values), and the
// sum's surplus is in its first addend, a multiply of the same activations by the constant -(128 + 8): sums are fp32, so what this costs is a few
// times 2^-24 of 136 sum |x|, below a result's own rounding unless the sum cancels to a thousandth.  With zero points the bias is 144 and the code's
// difference is taken in integers, 0x4310 + q - z.  Half precision has a packed subtraction: 0x6400 | q is 1024 + q, less 1024 + z exactly.  A scale
// group's sum then enters the row's accumulator with its scale: weights are never rounded.
//
// A tile is up to 64 rows of a group x some blocks of columns.  The activations are the multiply's first operand, so a lane ends up with four rows of one
// column: it needs one scale (and zero point) of a scale group, not four.  What bounds a launch with small scale groups is the number of load instructions, 16
// cycles of the address unit each: with weights first and a load per scale group and block, 2047 rows over 64 groups, N = 1544, K = 2080, groups of 32 with zero points
// took 79 us; the lanes' four quarters now load four groups' scales at once and hand them round.  The tile's activations go through LDS in chunks of 32 KB (16 rows x 1024 values, 32 x 512 or 64 x 256), read whole rows at a time: a fragment
// read straight from memory touches sixteen rows, a cache line for every lane (that way, with the waves' sums joined in LDS, 128 groups of 64 rows, N = 4096,
// K = 1536: 604 us, this way 204-213 by run; 512 rows over 128 groups, N = 2048, K = 768: 46 and 23).  Two chunks alternate, one multiplied while the other is copied, straight to LDS (through
// registers 226 and 24.5 us, and scale groups of 32 spilled).  Codes go from memory to registers two or four blocks ahead.  The four waves
// of a workgroup take columns side by side, or, where there are too few tiles to go round, every fourth block along K, and add up in LDS, in order.
// All loads go through buffer descriptors, whose range check gives zeros for rows and values beyond the operands.
#include <type_traits>

#include "fast_common.hpp"
#include "gate.hpp"
#include "launch.hpp"

namespace tgg {

struct Int4Params {
  GemmParams g;  // the group table's part: sizes, G, m_total, N (of a gated block 2 F), K
  const void* x;
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;
  void* out;
  int scale_groups;  // per column: ceil(K / gs)
  int blocks_per_scale;  // gs / 128 where gs >= 128
};

namespace {

constexpr int kI4Threads = 256, kI4Waves = 4, kI4Rows = 64, kI4MaxGroups = 1024;
constexpr int kI4Chunk = 32 * 1024;  // bytes of a chunk of activations

// The groups' first rows and first row tiles.  (The shared table of sched.hpp keeps 64-bit rows; with it two workgroups do not fit a compute unit.)
struct Int4Table {
  int32_t row[kI4MaxGroups + 1], tile[kI4MaxGroups + 1];
  int32_t scan[2][kI4Waves];
};

// Built by the whole workgroup, four groups a thread; ends with a barrier.  Rows beyond m_total belong to no group.
TGG_DEV void int4_table(const GemmParams& g, Int4Table& t) {
  constexpr int PER = kI4MaxGroups / kI4Threads;
  const int lane = lane_id(), wave = threadIdx.x >> 6, per = (g.G + kI4Threads - 1) / kI4Threads, g0 = threadIdx.x * per;
  int64_t size[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    size[i] = i < per && g0 + i < g.G ? load_size(g.sizes, g.sizes_i64, g0 + i) : 0;
    size[i] = size[i] < g.m_total ? size[i] : g.m_total;
    sum += size[i];
  }
  // 1024 groups of at most m_total < 2^31 rows: the sum stays within 64 bits
  __shared__ int64_t wave_rows[kI4Waves];
  const int64_t rows_incl = sched_wave_scan(sum);
  if (lane == 63) wave_rows[wave] = rows_incl;
  __syncthreads();
  int64_t row = rows_incl - sum;
  for (int w = 0; w < wave; ++w) row += wave_rows[w];
  int32_t first[PER], tiles = 0, count[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t begin = row < g.m_total ? row : g.m_total, end = row + size[i] < g.m_total ? row + size[i] : g.m_total;
    first[i] = (int32_t)begin;
    count[i] = (int32_t)((end - begin + kI4Rows - 1) / kI4Rows);
    tiles += count[i];
    row += size[i];
  }
  const int32_t end_row = (int32_t)(row < g.m_total ? row : g.m_total);
  const int32_t tiles_incl = (int32_t)sched_wave_scan(tiles);
  if (lane == 63) t.scan[0][wave] = tiles_incl;
  __syncthreads();
  int32_t tile = tiles_incl - tiles;
  for (int w = 0; w < wave; ++w) tile += t.scan[0][w];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (i < per && g0 + i < g.G) {
      t.row[g0 + i] = first[i];
      t.tile[g0 + i] = tile;
      tile += count[i];
      if (g0 + i == g.G - 1) {
        t.row[g.G] = end_row;
        t.tile[g.G] = tile;
      }
    }
  __syncthreads();
}

struct Int4Tile { int g, row0, rows, nt; };
// Tile ids run over (row tile, column tile), columns innermost: what runs together shares activations, and a group's row tiles its weights.
TGG_DEV Int4Tile int4_tile_at(const Int4Table& t, int G, int id, int tiles_n) {
  Int4Tile r;
  const int mt = id / tiles_n;
  r.nt = id - mt * tiles_n;
  int lo = 0, hi = G;  // the last group with tile[g] <= mt
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.tile[mid] <= mt) lo = mid; else hi = mid;
  }
  r.g = __builtin_amdgcn_readfirstlane(lo);
  const int at = (mt - t.tile[lo]) * kI4Rows, left = t.row[lo + 1] - t.row[lo] - at;
  r.row0 = __builtin_amdgcn_readfirstlane(t.row[lo] + at);
  r.rows = __builtin_amdgcn_readfirstlane(left < kI4Rows ? left : kI4Rows);
  r.nt = __builtin_amdgcn_readfirstlane(r.nt);
  return r;
}

typedef __amdgpu_buffer_rsrc_t rsrc_t;
TGG_DEV rsrc_t window(const void* base, int64_t bytes) {
  bytes = bytes < 0 ? 0 : (bytes > 0x7fffffff ? 0x7fffffff : bytes);
  return __builtin_amdgcn_make_buffer_rsrc((void*)uniform64((uint64_t)base), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
constexpr int kNowhere = 0x7ffffff0;  // beyond every window

// c[row][column] += x[row][k] w[column][k]: the lane's rows 4 lg + (0..3) of column l16
template <int DT> TGG_DEV f32x4_t mma(const i32x4_t& x, const i32x4_t& w, const f32x4_t& c) {
  if constexpr (DT == DT_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), __builtin_bit_cast(bf16x8_t, w), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, x), __builtin_bit_cast(f16x8_t, w), c, 0, 0, 0);
}

template <int DT> TGG_DEV float scale_value(uint32_t bits) {
  if (DT == DT_BF16) return __builtin_bit_cast(float, bits << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// The eight values of a word of codes as a multiply's operand, plus 128 (or 144) in bfloat16.  zz: the zero point in both halves (bfloat16, ZEROS), or
// minus (1024 + zero point) as a pair of half precision values.
// mask and base are 0x000f000f and the exponents' bits, in registers: as literals the two would take an instruction each (the 64 rows of above: 204 us for 213).
template <int DT, bool ZEROS> TGG_DEV i32x4_t operand(uint32_t word, uint32_t zz, uint32_t mask, uint32_t base) {
  i32x4_t r;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t q = ((word >> (4 * t)) & mask) | base;
    if constexpr (DT == DT_BF16) {
      r[t] = (int)(ZEROS ? q - zz : q);
    } else {
      const f16x2_t v = __builtin_bit_cast(f16x2_t, q) + __builtin_bit_cast(f16x2_t, zz);
      r[t] = __builtin_bit_cast(int, v);
    }
  }
  return r;
}

// GPT: scale groups per 128 values (1 where a group is 128 or more).  RB: row blocks, CB: column blocks of a wave.  KSPLIT: the waves share the columns and
// take every fourth block along K.
template <int DT, bool GATED, bool ZEROS, int GPT, int RB, int CB, bool KSPLIT>
TGG_DEV void int4_tile(const Int4Params& p, const Int4Tile& t, char* buf0, char* buf1) {
  // (opaque, so that the lane's offsets are made afresh per tile: hoisted out of the tile loop, those of all variants would spill)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int N = p.g.N, K = p.g.K, F = N / 2;
  const int blocks_n = (N + 15) / 16, blocks_k = (K + 127) / 128;
  const int rows = t.rows;
  const int64_t row0 = t.row0;
  const int64_t scale_elems = (int64_t)p.scale_groups * N;
  const rsrc_t cw = window(p.codes + (int64_t)t.g * blocks_n * blocks_k * 1024, (int64_t)blocks_n * blocks_k * 1024);
  const rsrc_t xw = window((const char*)p.x + row0 * K * 2, (int64_t)rows * K * 2);
  const rsrc_t sw = window((const char*)p.scales + (int64_t)t.g * scale_elems * 2, scale_elems * 2);
  const rsrc_t zw = window(ZEROS ? p.zeros + (int64_t)t.g * scale_elems : nullptr, ZEROS ? scale_elems : 0);

  // first column of the wave's column block c: of a gated tile the first half are the gate's, the others the up projection's of the same outputs
  constexpr int OC = GATED ? CB / 2 : CB;  // column blocks of outputs
  const int out0 = (t.nt * (KSPLIT ? 1 : kI4Waves) + (KSPLIT ? 0 : wave)) * OC * 16;
  auto col_of = [&](int c) { return out0 + (c % OC) * 16 + (GATED && c >= OC ? F : 0); };
  const int out_n = GATED ? F : N;

  // ---- activations: chunks of 16 RB rows x KC values (32 KB, or 24 where RB = 3), 16-byte pieces of a row swizzled by the row's number (a fragment read touches 16 rows) ----
  constexpr int KC = RB == 1 ? 1024 : RB == 2 ? 512 : 256, PIECES = KC / 8, PER = 16 * RB * PIECES / kI4Threads, BLOCKS = KC / 128;
  static_assert(16 * RB * KC * 2 <= kI4Chunk, "a chunk's place");
  static_assert(PIECES % 16 == 0 && (KC == 256 || kI4Threads % PIECES == 0 || PIECES % kI4Threads == 0), "a thread keeps its place in a row");
  constexpr int TPR = PIECES < kI4Threads ? PIECES : kI4Threads, ROWS_PER = kI4Threads / TPR;  // threads of a row, rows of one go
  const int xt_row = tid / TPR, xt_piece = (tid % TPR) ^ (xt_row & 15);
  // straight to LDS: a wave's instruction fills a kilobyte in the lanes' order, so the swizzle is in which piece a lane fetches
  auto x_copy = [&](int chunk, char* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = chunk * KC + (xt_piece ^ (i * ROWS_PER & 15)) * 8;
      const uint32_t at = (k < K ? (uint32_t)((xt_row * K + k) * 2) : (uint32_t)kNowhere) + (uint32_t)(i * ROWS_PER * K * 2);  // (beyond every window also with 64 rows' distance added)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xw, (lds_ptr_t)(buf + wave * 1024 + i * (kI4Threads * 16)), 16, (int)at, 0, 0, 0);
    }
  };

  // the wave's own copies have landed, by a read behind them that the compiler waits for, and then everybody's
  auto x_landed = [&](const char* buf) __attribute__((always_inline)) {
    const int last = *(const int*)(buf + (PER - 1) * (kI4Threads * 16) + tid * 16);
    asm volatile("" : : "v"(last));
    __syncthreads();
  };

  struct Stage {
    i32x4_t code[CB];
    uint16_t scale[CB];  // of the lane's column in scale group lg mod GPT of the block
    uint8_t zero[ZEROS ? CB : 1];
  };
  auto load = [&](Stage& st, int kb) __attribute__((always_inline)) {
    const bool live = kb < blocks_k;
    const int sg = GPT == 1 ? (p.blocks_per_scale == 1 ? kb : kb / p.blocks_per_scale) : kb * GPT + (lg & (GPT - 1));
    const bool there = sg < p.scale_groups;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      const int block = col_of(c) >> 4, at = sg * N + col_of(c) + l16;
      st.code[c] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(cw, live && block < blocks_n ? (block * blocks_k + kb) * 1024 + lane * 16 : kNowhere, 0, 2));
      st.scale[c] = __builtin_amdgcn_raw_buffer_load_b16(sw, there ? at * 2 : kNowhere, 0, 0);
      if (ZEROS) st.zero[c] = __builtin_amdgcn_raw_buffer_load_b8(zw, there ? at : kNowhere, 0, 0);
    }
  };

  f32x4_t acc[CB][RB];
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[c][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int bias2 = ZEROS ? (int)0xc310c310u : (int)0xc308c308u;  // -144 or -136, twice
  uint32_t mask = 0x000f000fu, base = DT != DT_BF16 ? 0x64006400u : ZEROS ? 0x43104310u : 0x43004300u;
  asm volatile("" : "+s"(mask), "+v"(base));
  const i32x4_t bias = {bias2, bias2, bias2, bias2};

  // a block of K whose activations are block `at` of the chunk at xs
  auto compute = [&](const Stage& st, const char* xs, int at) __attribute__((always_inline)) {
    constexpr int SP = 4 / GPT;  // steps of 32 values per scale group
    uint32_t meta[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) meta[c] = st.scale[c] | (ZEROS ? (uint32_t)st.zero[c] << 16 : 0u);
#pragma unroll
    for (int j = 0; j < GPT; ++j) {
      i32x4_t x[RB][SP];
#pragma unroll
      for (int s = 0; s < SP; ++s)
#pragma unroll
        for (int b = 0; b < RB; ++b) x[b][s] = *(const i32x4_t*)(xs + (16 * b + l16) * (KC * 2) + at * 256 + (((4 * (j * SP + s) + lg) ^ l16) << 4));
      f32x4_t first[RB];
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        first[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if constexpr (DT == DT_BF16) {
#pragma unroll
          for (int s = 0; s < SP; ++s) first[b] = mma<DT>(x[b][s], bias, first[b]);
        }
      }
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const uint32_t m = GPT == 1 ? meta[c] : (uint32_t)__builtin_amdgcn_ds_bpermute((16 * j + l16) * 4, (int)meta[c]);
        uint32_t zz = 0;
        if constexpr (DT == DT_BF16) {
          if (ZEROS) zz = (m >> 16) * 0x00010001u;
        } else {  // minus (1024 + z): 0xe400 | z
          zz = ZEROS ? 0xe400e400u + (m >> 16) * 0x00010001u : 0xe408e408u;
        }
        i32x4_t w[SP];
#pragma unroll
        for (int s = 0; s < SP; ++s) w[s] = operand<DT, ZEROS>((uint32_t)st.code[c][j * SP + s], zz, mask, base);
        const float scale = scale_value<DT>(m & 0xffff);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          f32x4_t part = first[b];
#pragma unroll
          for (int s = 0; s < SP; ++s) part = mma<DT>(x[b][s], w[s], part);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[c][b][e] = __builtin_fmaf(part[e], scale, acc[c][b][e]);
        }
      }
      // Several scale groups' sums are added in time: all of them at once do not fit the registers.  (Where a block is one group this costs an
      // overlap of blocks: the 64 rows of above 226 us for 213.)
      if (GPT == 2 || (GPT == 4 && (j & 1))) {
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
          for (int b = 0; b < RB; ++b) asm volatile("" : "+v"(acc[c][b]));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  constexpr int STEP = KSPLIT ? kI4Waves : 1, OWN = BLOCKS / STEP;  // the wave's blocks of a chunk
  static_assert(OWN >= 1, "a chunk has a block for every wave");
  constexpr int D = !KSPLIT && CB == 2 && RB <= 2 ? 4 : 2;  // blocks in flight
  const int kb0 = KSPLIT ? wave : 0;
  Stage st[D];
#pragma unroll
  for (int i = 0; i < D; ++i) load(st[i], kb0 + i * STEP);
  __syncthreads();  // the tile before has been read
  x_copy(0, buf0);
  x_landed(buf0);
  const int chunks = (blocks_k + BLOCKS - 1) / BLOCKS;
  // Chunk q, in xs, whose first block is in stage S.  All but the last one have all their blocks: without branches around the loads the compiler
  // can tell how many of them are behind the copies it waits for.
  constexpr int RUN = OWN < D ? OWN : D;
  auto whole = [&](auto Sc, int q, const char* xs, char* next) __attribute__((always_inline)) {
    constexpr int S = decltype(Sc)::value;
    x_copy(q + 1, next);
#pragma unroll 1
    for (int i0 = 0; i0 < OWN; i0 += RUN) {
#pragma unroll
      for (int i = 0; i < RUN; ++i) {
        compute(st[(S + i) % D], xs, kb0 + (i0 + i) * STEP);
        load(st[(S + i) % D], q * BLOCKS + kb0 + (i0 + i + D) * STEP);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    x_landed(next);
  };
  auto last = [&](auto Sc, int q, const char* xs) __attribute__((always_inline)) {
    constexpr int S = decltype(Sc)::value;
    const int left = (blocks_k - q * BLOCKS - kb0 + STEP - 1) / STEP, n = left < OWN ? left : OWN;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += RUN) {
#pragma unroll
      for (int i = 0; i < RUN; ++i) {
        if (i == 0 || i0 + i < n) {
          compute(st[(S + i) % D], xs, kb0 + (i0 + i) * STEP);
          if (OWN > D) load(st[(S + i) % D], q * BLOCKS + kb0 + (i0 + i + D) * STEP);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  static_assert(2 * OWN % D == 0, "after two chunks the first block is in stage 0 again");
  typedef std::integral_constant<int, 0> Even;
  typedef std::integral_constant<int, OWN % D> Odd;
  int q = 0;
  while (q + 1 < chunks) {
    whole(Even(), q, buf0, buf1);
    if (++q + 1 == chunks) break;
    whole(Odd(), q, buf1, buf0);
    ++q;
  }
  if constexpr (OWN % D == 0) last(Even(), q, q & 1 ? buf1 : buf0);
  else if (q & 1) last(Odd(), q, buf1);
  else last(Even(), q, buf0);

  // Rows 4 lg + e of block b, column l16: neighbouring lanes exchange halves, so that a store is two columns of a row.
  auto put = [&](int c, int b, f32x4_t v, const f32x4_t& u) __attribute__((always_inline)) {
    if constexpr (GATED) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (p.g.act == GATE_SILU ? gate_act<GATE_SILU>(v[e]) : gate_act<GATE_GELU_TANH>(v[e])) * u[e];
    }
    const bool odd = l16 & 1;
    const int n = col_of(c) + (l16 & ~1), row = 16 * b + 4 * lg + (odd ? 2 : 0);
    char* const at = (char*)p.out + ((row0 + row) * out_n + n) * 2;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float give = odd ? v[e] : v[e + 2], keep = odd ? v[e + 2] : v[e];
      const float got = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, give), 0xB1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
      if (row + e < rows && n < out_n) *(uint32_t*)(at + (int64_t)e * out_n * 2) = odd ? pack2<DT>(got, keep) : pack2<DT>(keep, got);
    }
  };
  if constexpr (!KSPLIT) {
#pragma unroll
    for (int c = 0; c < OC; ++c)
#pragma unroll
      for (int b = 0; b < RB; ++b) put(c, b, acc[c][b], acc[GATED ? c + OC : c][b]);
  } else {  // the waves' sums, added in their order
    float4* const red = (float4*)buf0;  // [wave][column block][row block][lane]
    static_assert(kI4Waves * CB * RB * 1024 <= kI4Chunk, "the sums fit where the activations were");
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int b = 0; b < RB; ++b) red[((wave * CB + c) * RB + b) * 64 + lane] = __builtin_bit_cast(float4, acc[c][b]);
    __syncthreads();
    auto total = [&](int c, int b) __attribute__((always_inline)) {
      f32x4_t v = __builtin_bit_cast(f32x4_t, red[(c * RB + b) * 64 + lane]);
#pragma unroll
      for (int w = 1; w < kI4Waves; ++w) v += __builtin_bit_cast(f32x4_t, red[((w * CB + c) * RB + b) * 64 + lane]);
      return v;
    };
    for (int i = wave; i < OC * RB; i += kI4Waves) {
      const int c = i / RB, b = i % RB;
      put(c, b, total(c, b), total(GATED ? c + OC : c, b));
    }
  }
}

template <int DT, bool GATED, bool ZEROS, int GPT, int CB, bool KSPLIT>
TGG_DEV void int4_tiles(const Int4Params& p, const Int4Table& table, char* buf0, char* buf1) {
  constexpr int COLS = 16 * CB * (KSPLIT ? 1 : kI4Waves);
  const int tiles_n = (p.g.N + COLS - 1) / COLS;
  const TileWalk walk = sched_walk((int64_t)table.tile[p.g.G] * tiles_n, p.g.tile_split != 0);
  for (int64_t id = walk.first; id < walk.end; id += walk.stride) {
    const Int4Tile t = int4_tile_at(table, p.g.G, (int)id, tiles_n);
    if (t.rows <= 16) int4_tile<DT, GATED, ZEROS, GPT, 1, CB, KSPLIT>(p, t, buf0, buf1);
    else if (t.rows <= 32) int4_tile<DT, GATED, ZEROS, GPT, 2, CB, KSPLIT>(p, t, buf0, buf1);
    else if constexpr (!KSPLIT) {  // four column blocks of more rows do not fit the registers: two and two
      Int4Tile h = t;
#pragma unroll 1
      for (int half = 0; half < CB / 2; ++half) {
        h.nt = t.nt * (CB / 2) + half;
        if (t.rows <= 48) int4_tile<DT, GATED, ZEROS, GPT, 3, 2, false>(p, h, buf0, buf1);
        else int4_tile<DT, GATED, ZEROS, GPT, 4, 2, false>(p, h, buf0, buf1);
      }
    }
    else {  // a chunk of 64 rows has no block for every wave: the tile's halves in turn
      Int4Tile h = t;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        h.row0 = t.row0 + 32 * half;
        h.rows = half ? t.rows - 32 : 32;
        int4_tile<DT, GATED, ZEROS, GPT, 2, CB, true>(p, h, buf0, buf1);
      }
    }
  }
}

template <int DT, bool GATED, bool ZEROS, int GPT>
__global__ __launch_bounds__(kI4Threads, 2) void gemm_int4_kernel(const Int4Params p) {
  __shared__ Int4Table table;
  __shared__ __attribute__((aligned(1024))) char buf0[kI4Chunk];
  __shared__ __attribute__((aligned(1024))) char buf1[kI4Chunk];
  int4_table(p.g, table);
  // Wide tiles read an activation once for more columns; narrow ones where the wide ones are too few to go round.
  const int64_t row_tiles = table.tile[p.g.G];
  if (row_tiles * ((p.g.N + 255) / 256) >= (int64_t)gridDim.x) int4_tiles<DT, GATED, ZEROS, GPT, 4, false>(p, table, buf0, buf1);
  else if (row_tiles * ((p.g.N + 127) / 128) >= (int64_t)gridDim.x) int4_tiles<DT, GATED, ZEROS, GPT, 2, false>(p, table, buf0, buf1);
  else int4_tiles<DT, GATED, ZEROS, GPT, 2, true>(p, table, buf0, buf1);
}

template <int DT, bool GATED, bool ZEROS, int GPT>
int launch_int4_as(const Int4Params& p, hipStream_t s) {
  int grid = 2 * num_cus();  // two workgroups a compute unit
  if (p.g.grid_limit > 0 && p.g.grid_limit < grid) grid = p.g.grid_limit;
  hipLaunchKernelGGL((gemm_int4_kernel<DT, GATED, ZEROS, GPT>), dim3(grid), dim3(kI4Threads), 0, s, p);
  return check_launch("gemm_int4");
}

template <int DT, bool GATED, bool ZEROS>
int launch_int4_groups(const Int4Params& p, int gs, hipStream_t s) {
  if (gs == 32) return launch_int4_as<DT, GATED, ZEROS, 4>(p, s);
  if (gs == 64) return launch_int4_as<DT, GATED, ZEROS, 2>(p, s);
  return launch_int4_as<DT, GATED, ZEROS, 1>(p, s);
}

template <int DT>
int launch_int4_type(const Int4Params& p, int gs, bool gated, hipStream_t s) {
  if (gated) return p.zeros ? launch_int4_groups<DT, true, true>(p, gs, s) : launch_int4_groups<DT, true, false>(p, gs, s);
  return p.zeros ? launch_int4_groups<DT, false, true>(p, gs, s) : launch_int4_groups<DT, false, false>(p, gs, s);
}

}  // namespace

int launch_int4(const GemmParams& g, const void* x, const uint8_t* codes, const void* scales, const uint8_t* zeros, void* out, int gs, bool gated, int dt, hipStream_t s) {
  Int4Params p;
  p.g = g;
  p.x = x;
  p.codes = codes;
  p.scales = scales;
  p.zeros = zeros;
  p.out = out;
  p.scale_groups = (g.K + gs - 1) / gs;
  p.blocks_per_scale = gs >= 128 ? gs / 128 : 1;
  return dt == DT_BF16 ? launch_int4_type<DT_BF16>(p, gs, gated, s) : launch_int4_type<DT_F16>(p, gs, gated, s);
}

}  // namespace tgg
