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
// A tile is up to 64 rows of a group x CB blocks of columns (weights are the multiply's first operand: a lane ends up with four neighbouring columns of a
// row).  The four waves of a workgroup take every fourth block of 128 values along K and add up in LDS, in order; all loads go through buffer
// descriptors, whose range check gives zeros for rows and values beyond the operands, and run two blocks ahead.
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

constexpr int kI4Threads = 256, kI4Waves = 4, kI4Rows = 64;

typedef __amdgpu_buffer_rsrc_t rsrc_t;
TGG_DEV rsrc_t window(const void* base, int64_t bytes) {
  bytes = bytes < 0 ? 0 : (bytes > 0x7fffffff ? 0x7fffffff : bytes);
  return __builtin_amdgcn_make_buffer_rsrc((void*)uniform64((uint64_t)base), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
constexpr int kNowhere = 0x7ffffff0;  // beyond every window

template <int DT> TGG_DEV f32x4_t mma(const i32x4_t& w, const i32x4_t& x, const f32x4_t& c) {
  if constexpr (DT == DT_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), __builtin_bit_cast(bf16x8_t, x), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w), __builtin_bit_cast(f16x8_t, x), c, 0, 0, 0);
}

template <int DT> TGG_DEV float scale_value(uint32_t bits) {
  if (DT == DT_BF16) return __builtin_bit_cast(float, bits << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// The eight values of a word of codes as a multiply's operand, plus 128 (or 144) in bfloat16.  zz: the zero point in both halves (bfloat16, ZEROS), or
// minus (1024 + zero point) as a pair of half precision values.
template <int DT, bool ZEROS> TGG_DEV i32x4_t operand(uint32_t word, uint32_t zz) {
  i32x4_t r;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t q = (word >> (4 * t)) & 0x000f000fu;
    if constexpr (DT == DT_BF16) {
      r[t] = (int)(ZEROS ? (q | 0x43104310u) - zz : (q | 0x43004300u));
    } else {
      const f16x2_t v = __builtin_bit_cast(f16x2_t, q | 0x64006400u) + __builtin_bit_cast(f16x2_t, zz);
      r[t] = __builtin_bit_cast(int, v);
    }
  }
  return r;
}

// GPT: scale groups per 128 values (1 where a group is 128 or more)
template <int DT, bool GATED, bool ZEROS, int GPT, int RB, int CB>
TGG_DEV void int4_tile(const Int4Params& p, const Tile& t, float4* red) {
  const int lane = lane_id(), l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int N = p.g.N, K = p.g.K, F = N / 2;
  const int blocks_n = (N + 15) / 16, blocks_k = (K + 127) / 128;
  const int g = __builtin_amdgcn_readfirstlane(t.g), rows = __builtin_amdgcn_readfirstlane(t.rows), n0 = __builtin_amdgcn_readfirstlane(t.n0);
  const int64_t row0 = (int64_t)uniform64((uint64_t)t.row0);
  const int64_t scale_elems = (int64_t)p.scale_groups * N;
  const rsrc_t cw = window(p.codes + (int64_t)g * blocks_n * blocks_k * 1024, (int64_t)blocks_n * blocks_k * 1024);
  const rsrc_t xw = window((const char*)p.x + row0 * K * 2, (int64_t)rows * K * 2);
  const rsrc_t sw = window((const char*)p.scales + (int64_t)g * scale_elems * 2, scale_elems * 2);
  const rsrc_t zw = window(ZEROS ? p.zeros + (int64_t)g * scale_elems : nullptr, ZEROS ? scale_elems : 0);

  // first column of column block c: of a gated tile the first half are the gate's, the others the up projection's of the same outputs
  auto col_of = [&](int c) { return GATED ? n0 / 2 + (c % (CB / 2)) * 16 + (c >= CB / 2 ? F : 0) : n0 + c * 16; };

  struct Stage {
    i32x4_t code[CB];
    i32x4_t x[RB][4];
    uint2 scale[GPT][CB];
    uint8_t zero[ZEROS ? GPT : 1][CB];
  };
  auto load = [&](Stage& st, int kb) __attribute__((always_inline)) {
    const bool live = kb < blocks_k;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      const int block = col_of(c) >> 4;
      st.code[c] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(cw, live && block < blocks_n ? (block * blocks_k + kb) * 1024 + lane * 16 : kNowhere, 0, 2));
    }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int k = kb * 128 + 32 * s + 8 * lg;
        st.x[b][s] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(xw, k < K ? ((16 * b + l16) * K + k) * 2 : kNowhere, 0, 0));
      }
#pragma unroll
    for (int j = 0; j < GPT; ++j) {
      const int sg = GPT == 1 ? kb / p.blocks_per_scale : kb * GPT + j;
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const int n = col_of(c);
        const bool there = sg < p.scale_groups;
        st.scale[j][c] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(sw, there ? (sg * N + n + 4 * lg) * 2 : kNowhere, 0, 0));
        if (ZEROS) st.zero[j][c] = __builtin_amdgcn_raw_buffer_load_b8(zw, there ? sg * N + n + l16 : kNowhere, 0, 0);
      }
    }
  };

  f32x4_t acc[CB][RB];
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[c][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int bias2 = ZEROS ? (int)0xc310c310u : (int)0xc308c308u;  // -144 or -136, twice
  const i32x4_t bias = {bias2, bias2, bias2, bias2};

  auto compute = [&](const Stage& st) __attribute__((always_inline)) {
    constexpr int SP = 4 / GPT;  // steps of 32 values per scale group
#pragma unroll
    for (int j = 0; j < GPT; ++j) {
      f32x4_t first[RB];
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        first[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if constexpr (DT == DT_BF16) {
#pragma unroll
          for (int s = 0; s < SP; ++s) first[b] = mma<DT>(bias, st.x[b][j * SP + s], first[b]);
        }
      }
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        uint32_t zz = 0;
        if constexpr (DT == DT_BF16) {
          if (ZEROS) zz = st.zero[j][c] * 0x00010001u;
        } else {  // minus (1024 + z): 0xe400 | z
          zz = ZEROS ? 0xe400e400u + st.zero[j][c] * 0x00010001u : 0xe408e408u;
        }
        i32x4_t w[SP];
#pragma unroll
        for (int s = 0; s < SP; ++s) w[s] = operand<DT, ZEROS>((uint32_t)st.code[c][j * SP + s], zz);
        const float s4[4] = {scale_value<DT>(st.scale[j][c].x & 0xffff), scale_value<DT>(st.scale[j][c].x >> 16),
                             scale_value<DT>(st.scale[j][c].y & 0xffff), scale_value<DT>(st.scale[j][c].y >> 16)};
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          f32x4_t part = first[b];
#pragma unroll
          for (int s = 0; s < SP; ++s) part = mma<DT>(w[s], st.x[b][j * SP + s], part);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[c][b][e] = __builtin_fmaf(part[e], s4[e], acc[c][b][e]);
        }
      }
    }
  };

  Stage st[2];
  load(st[0], wave);
  load(st[1], wave + kI4Waves);
  for (int kb = wave; kb < blocks_k; kb += 2 * kI4Waves) {
    compute(st[0]);
    load(st[0], kb + 2 * kI4Waves);
    if (kb + kI4Waves < blocks_k) {
      compute(st[1]);
      load(st[1], kb + 3 * kI4Waves);
    }
  }

  // the waves' sums, added in their order, two row blocks at a time
  constexpr int OC = GATED ? CB / 2 : CB, HB = RB < 2 ? RB : 2;  // column blocks of outputs; row blocks at a time
  const int out_n = GATED ? F : N;
#pragma unroll
  for (int b0 = 0; b0 < RB; b0 += HB) {
    __syncthreads();  // what was there before has been read
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int b = 0; b < HB; ++b) red[((wave * CB + c) * HB + b) * 64 + lane] = __builtin_bit_cast(float4, acc[c][b0 + b]);
    __syncthreads();
    auto total = [&](int c, int b) __attribute__((always_inline)) {
      f32x4_t v = __builtin_bit_cast(f32x4_t, red[(c * HB + b) * 64 + lane]);
#pragma unroll
      for (int w = 1; w < kI4Waves; ++w) v += __builtin_bit_cast(f32x4_t, red[((w * CB + c) * HB + b) * 64 + lane]);
      return v;
    };
    for (int i = wave; i < OC * HB; i += kI4Waves) {
      const int c = i / HB, b = i % HB, row = 16 * (b0 + b) + l16, n = col_of(c) + 4 * lg;
      f32x4_t v = total(c, b);
      if constexpr (GATED) {
        const f32x4_t u = total(c + OC, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (p.g.act == GATE_SILU ? gate_act<GATE_SILU>(v[e]) : gate_act<GATE_GELU_TANH>(v[e])) * u[e];
      }
      if (row < rows && n < out_n) *(uint2*)((char*)p.out + ((row0 + row) * (int64_t)out_n + n) * 2) = pack4<DT>(v[0], v[1], v[2], v[3]);
    }
  }
}

template <int DT, bool GATED, bool ZEROS, int GPT, int CB>
TGG_DEV void int4_tiles(const Int4Params& p, const SchedTable& sched, float4* red) {
  const int64_t tiles = sched_num_tiles<kI4Rows, 16 * CB>(p.g, sched);
  const TileWalk walk = sched_walk(tiles, p.g.tile_split != 0);
  for (int64_t id = walk.first; id < walk.end; id += walk.stride) {
    const Tile t = sched_tile<kI4Rows, 16 * CB>(p.g, sched, id);
    const int rows = __builtin_amdgcn_readfirstlane(t.rows);
    if (rows <= 16) int4_tile<DT, GATED, ZEROS, GPT, 1, CB>(p, t, red);
    else if (rows <= 32) int4_tile<DT, GATED, ZEROS, GPT, 2, CB>(p, t, red);
    else int4_tile<DT, GATED, ZEROS, GPT, 4, CB>(p, t, red);
  }
}

template <int DT, bool GATED, bool ZEROS, int GPT>
__global__ __launch_bounds__(kI4Threads, 2) void gemm_int4_kernel(const Int4Params p) {
  __shared__ SchedTable sched;
  __shared__ __attribute__((aligned(16))) float4 red[kI4Waves * 4 * 2 * 64];  // [wave][column block][row block][lane]
  sched_init<kI4Rows>(p.g, sched);
  // Wide tiles read an activation once for twice the columns; narrow ones where the wide ones are too few to go round.
  if (sched_num_tiles<kI4Rows, 64>(p.g, sched) >= (int64_t)gridDim.x) int4_tiles<DT, GATED, ZEROS, GPT, 4>(p, sched, red);
  else int4_tiles<DT, GATED, ZEROS, GPT, 2>(p, sched, red);
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
