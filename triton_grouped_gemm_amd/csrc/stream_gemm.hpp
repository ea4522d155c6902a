// Main loop of the 16-bit products of newton_schulz.hip and lora.hip: a workgroup's tiles as one uninterrupted stream of 64-deep slabs.
//
// The scheme is that of the eight-wave kernels (gemm_fast.hip): eight waves, a ring of slab buffers in LDS (two, more for small tiles, whose slabs take less time than
// their copies) filled by direct copies that run that many slabs ahead across tile boundaries, fragment reads a K step ahead across the one barrier a slab, copies issued between multiplies.  What differs is
// who says what a slab is: a problem P hands out slabs one after another, so a tile may add up products of several pairs of operands
// (a matrix's two planes, a row's shared projection and its adapters), and takes a tile's sums.  P has
//
//   StreamCursor<C, B_KMAJOR> cur         where the copies are
//   int tile_at(int pos)                  id of the workgroup's pos-th tile, -1 past the last one
//   int slabs(int id)                     slabs of a tile, at least one
//   void seek(int id)                     begins the tile's slabs in `cur`; id -1: no more slabs
//   void turn()                           the slabs begun last have all been handed out: begins the tile's next ones, or seeks the next tile
//   void begin(id, acc, at)               the tile's sums before its first slab (they are zero)
//   void epilogue(id, acc, at, stage)     the tile's sums: acc[i][j][e] is row wm0 + 16 i + l16, column wn0 + 16 j + 4 lg + e
//
// A [rows, K] is K-contiguous; B is K-contiguous rows [columns, K] (B_KMAJOR) or token rows [K, columns].
#pragma once
#include "fast_common.hpp"
#include "launch.hpp"

namespace tgg {

// (min and max of two 64-bit numbers: the runtime's own are for 32-bit ones in host code and cut them off)
__host__ __device__ constexpr int64_t lesser(int64_t a, int64_t b) { return a < b ? a : b; }
__host__ __device__ constexpr int64_t larger(int64_t a, int64_t b) { return a < b ? b : a; }

// a kernel's dynamic LDS beyond the default limit: once for each device
template <class Kern> int stream_lds(Kern kern, int bytes, bool (&attr_set)[64]) {
  int dev = 0;
  (void)hipGetDevice(&dev);
  const bool listed = dev >= 0 && dev < 64;
  if (listed && attr_set[dev]) return 0;
  if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return check_launch("hipFuncSetAttribute(stream)");
  if (listed) attr_set[dev] = true;
  return 0;
}

template <int BM_, int BN_, int WM_, int WN_, int RING_ = 2> struct StreamCfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int RING = RING_;
  static constexpr int NWAVES = WM * WN, THREADS = NWAVES * 64;
  static constexpr int A_BYTES = BM * kSlabRowBytes, B_BYTES = BN * kSlabRowBytes, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int CA = A_BYTES / 1024 / NWAVES, CB = B_BYTES / 1024 / NWAVES, NC = CA + CB;  // copies of a wave and slab
  static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  static constexpr int EPI_OFF = RING * STAGE_BYTES;
  static_assert(CA * NWAVES * 1024 == A_BYTES && CB * NWAVES * 1024 == B_BYTES, "copies must divide evenly over waves");
  static_assert(NWAVES == 8, "a wave keeps one swizzle pattern for all its copies");
  static_assert(NC % 2 == 0 && TM % 2 == 0 && (TM * TN / 2) % (NC / 2) == 0, "a slab's copies are spread over the multiplies of two half K steps");
};

struct StreamSlab {
  i32x4_t ra, rb;
};

// The slabs of one pair of operands: descriptors that move on by 64 values of depth, and the lane's source offsets in the wave's copies, which stay the same but
// for a last slab that the depth cuts short.  32-bit bookkeeping keeps the scalar work per slab short (eight waves share the scalar unit).
template <class C, bool B_KMAJOR> struct StreamCursor {
  typedef Operand<C::BM, true> OpA;
  typedef Operand<C::BN, B_KMAJOR> OpB;
  int va[C::CA], vb[C::CB];
  int lda, ldb;            // bytes between rows
  int a_voff, b_voff;
  bool a_there, b_there;   // whether the lane fetches in a slab that is cut short
  int kt, tail;            // slabs; whether the last one is cut short
  uint64_t a_at, b_at;     // the next slab
  int a_rem, b_rem, b_skip;  // bytes left of the tile's rows; of token rows, how many are left, and the bytes in front of the tile's columns
  int run;                 // slabs until something changes
  bool in_tail;

  TGG_DEV StreamCursor(int lda_, int ldb_, int depth) : lda(lda_), ldb(ldb_) {
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    a_voff = OpA::lane_voff(lane, wave % OpA::NPAT, lda) + wave * OpA::RPI * lda;
    b_voff = OpB::lane_voff(lane, wave % OpB::NPAT, ldb) + wave * OpB::RPI * ldb;
    kt = (depth + 63) / 64;
    const int chunks = ((depth + 7) / 8) % 8;  // 16-byte pieces of a K-contiguous row in a slab that is cut short
    tail = chunks != 0;
    a_there = OpA::lane_chunk(lane, wave % OpA::NPAT) < chunks;
    b_there = !B_KMAJOR || OpB::lane_chunk(lane, wave % OpB::NPAT) < chunks;
  }
  TGG_DEV void offsets(bool whole) {
#pragma unroll
    for (int k = 0; k < C::CA; ++k) va[k] = whole || a_there ? a_voff + k * C::NWAVES * OpA::RPI * lda : kNoFetch;
#pragma unroll
    for (int k = 0; k < C::CB; ++k) vb[k] = whole || b_there ? b_voff + k * C::NWAVES * OpB::RPI * ldb : kNoFetch;
    in_tail = !whole;
    run = whole ? kt - tail : 1;
  }
  // a, b: the tile's first bytes; rows of A, and of B its columns' rows or (token rows) the depth.  live false: nothing, for good
  TGG_DEV void begin(bool live, uint64_t a, uint64_t b, int a_rows, int b_rows, int skip) {
    a_at = uniform64(a);
    b_at = uniform64(b);
    a_rem = __builtin_amdgcn_readfirstlane(live ? a_rows * lda : 0);
    b_rem = __builtin_amdgcn_readfirstlane(live ? (B_KMAJOR ? b_rows * ldb : b_rows) : 0);
    b_skip = skip;
    offsets(kt > tail);
    run = live ? run : 0x7fffffff;
  }
  TGG_DEV void next(StreamSlab& s) {
    s.ra = make_rsrc32(a_at, a_rem);
    s.rb = make_rsrc32(b_at, B_KMAJOR ? b_rem : min(64, b_rem) * ldb - b_skip);
    a_at += 128;
    a_rem -= 128;
    b_at += B_KMAJOR ? 128 : (uint64_t)(64 * ldb);
    b_rem -= B_KMAJOR ? 128 : 64;
    --run;
  }
};

// where a wave's block of the tile begins, and a lane's place in a 16 x 16 block
template <class C> struct StreamPlace {
  int lane, wave, wm0, wn0, l16, lg;
  TGG_DEV StreamPlace() {
    lane = lane_id();
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm0 = (wave / C::WN) * (C::BM / C::WM);
    wn0 = (wave % C::WN) * (C::BN / C::WN);
    l16 = lane & 15;
    lg = lane >> 4;
  }
};

// Which tiles a workgroup takes: workgroups are dealt round robin to the XCDs, and each XCD takes a contiguous range of ids, so that what
// runs together in front of one L2 shares operands.
struct StreamWalk {
  int first, stride, end;
  TGG_DEV explicit StreamWalk(int tiles) {
    const int grid = gridDim.x, id = blockIdx.x;
    if ((grid & 7) || tiles <= grid) {
      first = id;
      stride = grid;
      end = tiles;
    } else {
      const int xcd = id & 7;
      first = (int)((int64_t)tiles * xcd / 8) + (id >> 3);
      stride = grid >> 3;
      end = (int)((int64_t)tiles * (xcd + 1) / 8);
    }
  }
  TGG_DEV int at(int pos) const {
    const int64_t id = first + (int64_t)pos * stride;
    return id < end ? (int)id : -1;
  }
};

template <int DT> TGG_DEV f32x4_t stream_mma(const i32x4_t& w, const i32x4_t& x, const f32x4_t& c) {
  if constexpr (DT == DT_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), __builtin_bit_cast(bf16x8_t, x), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w), __builtin_bit_cast(f16x8_t, x), c, 0, 0, 0);
}

// The next slab.  All copies of the one before have been issued: offsets may change.  (A copy must not follow the vector instruction that wrote a scalar of its
// descriptor too closely, and the compiler does not look inside the copies.)
template <class P> TGG_DEV void stream_next(P& prob, StreamSlab& s) {
  if (__builtin_expect(prob.cur.run == 0, 0)) {
    if (prob.cur.tail && !prob.cur.in_tail) prob.cur.offsets(false); else prob.turn();
  }
  prob.cur.next(s);
  asm volatile("s_nop 4" : "+s"(s.ra), "+s"(s.rb));
}

template <class C, int DT, bool B_KMAJOR, class P> TGG_DEV void stream_gemm(P& prob, char* smem) {
  const StreamPlace<C> at;
  const uint32_t smem_addr = (uint32_t)(uintptr_t)(lds_ptr_t)smem;
  const int l16 = at.l16, lg = at.lg;

  // a lane's LDS offsets of the fragment reads, relative to the operand's slab (see gemm_fast.hip)
  int a_rd[2], b_rd[B_KMAJOR ? 2 : C::TN];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) a_rd[ks] = (at.wm0 + l16) * 128 + (((4 * ks + lg) ^ ((l16 / 2) % 8)) << 4);
  if (B_KMAJOR) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) b_rd[ks] = (at.wn0 + l16) * 128 + (((4 * ks + lg) ^ ((l16 / 2) % 8)) << 4);
  } else {
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const int e = l16 >> 2, c = l16 & 3;
      const int chunk = ((at.wn0 + 16 * j) / 8 + (c >> 1)) ^ Operand<C::BN, false>::token_swizzle(8 * (lg & 1) + e);
      b_rd[j] = (lg * 8 + e) * (C::BN * 2) + chunk * 16 + (c & 1) * 8;
    }
  }
  auto load_a = [&](const char* s, int ks, int i) __attribute__((always_inline)) -> i32x4_t { return *(const i32x4_t*)(s + a_rd[ks] + i * 16 * 128); };
  auto load_b = [&](const char* s, int ks, int j) __attribute__((always_inline)) -> i32x4_t {
    if (B_KMAJOR) return *(const i32x4_t*)(s + b_rd[ks] + j * 16 * 128);
    const char* q = s + b_rd[B_KMAJOR ? 0 : j] + ks * 32 * (C::BN * 2);
    const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr_t)q);
    // four token rows on: their swizzle is the same (it goes by k % 4 and k / 8, or, in rows of 128 bytes, by k / 2 % 2 and k / 8)
    const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr_t)(q + 4 * (C::BN * 2)));
    return __builtin_bit_cast(i32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  constexpr int SP2 = (C::TM * C::TN / 2) / (C::NC / 2), SP1 = 1;  // multiplies between copies, behind the barrier and in the half step after that
  StreamSlab sc, sc_next;
  uint32_t sc_base = 0, sc_next_base = 0;
  auto copy_k = [&](int k) __attribute__((always_inline)) {
    if (k < C::CA) {
      copy_b128_to_lds(sc.ra, __builtin_amdgcn_readfirstlane(sc_base + (at.wave + k * C::NWAVES) * 1024), prob.cur.va[k]);
    } else {
      copy_b128_to_lds(sc.rb, __builtin_amdgcn_readfirstlane(sc_base + C::A_BYTES + (at.wave + (k - C::CA) * C::NWAVES) * 1024), prob.cur.vb[k - C::CA]);
    }
  };

  prob.seek(prob.tile_at(0));
#pragma unroll
  for (int q = 0; q < C::RING - 1; ++q) {
    stream_next(prob, sc);
    sc_base = smem_addr + q * C::STAGE_BYTES;
#pragma unroll
    for (int k = 0; k < C::NC; ++k) copy_k(k);
  }
  wait_vmcnt<(C::RING - 2) * C::NC>();
  __syncthreads();
  stream_next(prob, sc);
  sc_base = smem_addr + (C::RING - 1) * C::STAGE_BYTES;
#pragma unroll
  for (int k = 0; k < C::NC / 2; ++k) copy_k(k);
  i32x4_t fa[C::TM - 1], fa_last[2], fb[2][C::TN];
  int ring = 0;  // the buffer of the slab that is multiplied

  f32x4_t acc[C::TM][C::TN];
  for (int pos = 0, id; (id = prob.tile_at(pos)) >= 0; ++pos) {
    const int slabs = __builtin_amdgcn_readfirstlane(prob.slabs(id));
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    prob.begin(id, acc, at);
    // The first slab's first fragments.  (The slab before has read them already, if this is not the first tile: read again, their registers are free for begin() and epilogue().)
    {
      const char* s = smem + ring * C::STAGE_BYTES;
#pragma unroll
      for (int i = 0; i < C::TM - 1; ++i) fa[i] = load_a(s, 0, i);
      fa_last[0] = load_a(s, 0, C::TM - 1);
#pragma unroll
      for (int j = 0; j < C::TN; ++j) fb[0][j] = load_b(s + C::A_BYTES, 0, j);
    }
    enum { READ_EARLY, READ_ROLL, READ_NONE, READ_CATCH_UP };  // as in gemm_fast.hip
    // (inlined before anything else: a lambda that is simplified by itself turns stores to the problem's members into stores through selected pointers, and the
    // members stay in memory)
    auto half = [&](int cur, int h, const char* s, int ks, int mode, int k0, bool prepare = false) __attribute__((always_inline)) {
      constexpr int HM = C::TM / 2;
#pragma unroll
      for (int ii = 0; ii < HM; ++ii) {
        const int i = h * HM + ii;
        const i32x4_t a = i == C::TM - 1 ? fa_last[cur] : fa[i < C::TM - 1 ? i : 0];
#pragma unroll
        for (int jj = 0; jj < C::TN; ++jj) {
          const int j = (i & 1) ? C::TN - 1 - jj : jj;
          acc[i][j] = stream_mma<DT>(fb[cur][j], a, acc[i][j]);
          const int n = ii * C::TN + jj;
          if (n == 0 && (mode == READ_EARLY || mode == READ_CATCH_UP)) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j2 = 0; j2 < C::TN; ++j2) fb[cur ^ 1][j2] = load_b(s + C::A_BYTES, ks, j2);
            fa_last[cur ^ 1] = load_a(s, ks, C::TM - 1);
            if (mode == READ_CATCH_UP) {
#pragma unroll
              for (int i2 = 0; i2 < HM; ++i2) fa[i2] = load_a(s, ks, i2);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if (prepare && n == (HM * C::TN > 1 ? 1 : 0)) {  // scalar work, under the multiplies just issued
            stream_next(prob, sc_next);
            sc_next_base = smem_addr + ring * C::STAGE_BYTES;
          }
          const int sp = k0 == 0 ? SP1 : SP2;
          if (k0 >= 0 && (n + 1) % sp == 0 && (n + 1) / sp <= C::NC / 2) {
            __builtin_amdgcn_sched_barrier(0);
            copy_k(k0 + (n + 1) / sp - 1);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        if (mode != READ_NONE && i < C::TM - 1) {
          __builtin_amdgcn_sched_barrier(0);
          fa[i < C::TM - 1 ? i : 0] = load_a(s, ks, i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int kt = 0; kt < slabs; ++kt) {
      const char* s = smem + ring * C::STAGE_BYTES;
      const int next = ring + 1 == C::RING ? 0 : ring + 1;
      const char* sn = smem + next * C::STAGE_BYTES;
      half(0, 0, s, 1, READ_EARLY, C::NC / 2);
      half(0, 1, s, 1, READ_ROLL, -1, true);
      half(1, 0, sn, 0, READ_NONE, -1);
      wait_vmcnt<(C::RING - 2) * C::NC>();  // the next slab is there; those behind it may be on their way
      __syncthreads();
      sc = sc_next;
      sc_base = sc_next_base;
      half(1, 1, sn, 0, READ_CATCH_UP, 0);
      ring = next;
    }
    prob.epilogue(id, acc, at, smem + C::EPI_OFF);
  }
  wait_vmcnt<0>();  // the trailing copies, which fetch nothing, still write LDS
}

}  // namespace tgg
