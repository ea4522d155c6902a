// Low-rank adapters of many requests beside a shared projection:
//   y[m] = W x[m] + s_l B_l (A_l x[m]),   l = the row's adapter, no second term where it has none
// with W [N, K], A [L, R, K], B [L, N, R], and the gradients of x, A and B:
//   h[m] = s_l A_l x[m],   dh[m] = s_l B_l^T g[m],   dx = W^T g + A_l^T dh,   dA_l = sum of dh[m] x[m]^T over l's rows,   dB_l = sum of g[m] h[m]^T
//
// Three kinds of kernel:
//   lora_down   h (or dh, from B transposed): few outputs, long sums.  A workgroup has 16 to 64 rows, its waves share the sum's length; the rows' distinct adapters
//               are taken in turn (rows of a request follow one another, so that is mostly one), and a row keeps the sums of its own.
//   lora_gemm   y and dx: the shared product, whose sums begin with the adapters' part: for every adapter of a wave's rows, R more values of depth, h (the rows
//               of other adapters as zeros) against B_l (A_l transposed), from memory to registers.  So the adapters enter the fp32 sums and there is one rounding.
//               h is fp32 and enters as two planes of bfloat16, high and low, 16 bits with fp32's range; against them half-precision adapters are split into two bfloat16
//               values without loss.  Infinities come out as the formulas have them: no part of a value that is zero, or of the other sign, meets one.
//   lora_outer  dA and dB: sums over an adapter's rows, which are gathered from wherever they stand.
// and lora_few, which streams W for the few rows of a decode step.
#include "launch.hpp"
#include "stream_gemm.hpp"

namespace tgg {

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
TGG_DEV rsrc_t window(const void* base, int64_t bytes) {
  bytes = bytes < 0 ? 0 : (bytes > 0x7fffffff ? 0x7fffffff : bytes);
  return __builtin_amdgcn_make_buffer_rsrc((void*)uniform64((uint64_t)base), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
constexpr int kNowhere = 0x7ffffff0;  // beyond every window

struct Ids {
  const void* p;
  int i64, L;
  // the row's adapter, -1 where it has none
  TGG_DEV int at(int64_t row) const {
    const int64_t v = i64 ? ((const int64_t*)p)[row] : ((const int32_t*)p)[row];
    return v >= 0 && v < L ? (int)v : -1;
  }
};

template <int DT> TGG_DEV float from_bits(uint16_t h) {
  if (DT == DT_BF16) return __builtin_bit_cast(float, (uint32_t)h << 16);
  return (float)__builtin_bit_cast(_Float16, h);
}
// two 16-bit values that add up to v but for 2^-17 (bf16) or 2^-22 of it (and what half precision's range cuts off)
// keep: a value below half precision's smallest step becomes one in the high part (and is taken back in the low one): what is not zero has no zero for a high part
template <int DT> TGG_DEV void split2(float v, uint16_t& hi, uint16_t& lo, bool keep = false) {
  hi = Out16<DT>::cvt(v);
  if (keep) hi |= v != 0.f && !(hi & 0x7fffu) ? 1 : 0;
  const float rest = v - from_bits<DT>(hi);
  lo = Out16<DT>::cvt(__builtin_isfinite(rest) ? rest : 0.f);  // an infinity stays one
}
// 2^e with |v| 2^e in [2^10, 2^11); 1 for zeros and what is not finite
TGG_DEV float row_scale(float v) {
  if (!(v > 0.f) || !__builtin_isfinite(v)) return 1.f;
  int e = (int)(__builtin_bit_cast(uint32_t, v) >> 23) - 127;
  e = 10 - (e < -110 ? -110 : e);
  return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
}

// Chunks of 256 values of depth of a few rows of two K-contiguous operands, through a ring in LDS; the eight waves share a chunk's depth, 32 values each.  (Fragments read
// straight from memory have every lane in another row than its neighbours, which takes the address unit 64 cycles instead of 16: 64 rows of x and 16 columns
// of W a workgroup, 4096 x 4096: 23 us; through the ring 14.)  Rows of 512 bytes, 16-byte pieces swizzled by the row.
template <int XB, int WB, int STAGES> struct ChunkRing {
  static constexpr int X_BYTES = XB * 16 * 512, STAGE_BYTES = X_BYTES + WB * 16 * 512, BYTES = STAGES * STAGE_BYTES, NC = XB + WB;  // NC: a wave's copies of a chunk
  static_assert(BYTES <= 160 * 1024 && (STAGES - 1) * NC < 64, "LDS, and copies that a wait can count");
  i32x4_t xr, wr;
  int voff, piece, pitch, depth, step, end;  // the lane's offset in a copy; chunks step ... end - 1
  uint32_t at;
  char* smem;

  TGG_DEV ChunkRing(char* smem_, const void* x, int64_t x_bytes, const void* w, int64_t w_bytes, int depth_, int first, int end_) : depth(depth_), step(first), end(end_), smem(smem_) {
    xr = make_rsrc((uint64_t)x, x_bytes);
    wr = make_rsrc((uint64_t)w, w_bytes);
    at = (uint32_t)(uintptr_t)(lds_ptr_t)smem;
    const int lane = lane_id(), wave = threadIdx.x >> 6, row = 2 * wave + (lane >> 5);  // of 16
    pitch = depth * 2;
    piece = (lane & 31) ^ row;
    voff = row * pitch + piece * 16;
  }
  TGG_DEV void copy(int chunk) {
    const bool there = chunk < end && chunk * 256 + piece * 8 < depth;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t to = at + chunk_buffer(chunk) * STAGE_BYTES + wave * 1024;
    asm volatile("s_nop 4" : "+s"(xr), "+s"(wr));
#pragma unroll
    for (int i = 0; i < XB; ++i) copy_b128_to_lds(xr, __builtin_amdgcn_readfirstlane(to + i * 8192), there ? voff + chunk * 512 + i * 16 * pitch : kNoFetch);
#pragma unroll
    for (int i = 0; i < WB; ++i) copy_b128_to_lds(wr, __builtin_amdgcn_readfirstlane(to + X_BYTES + i * 8192), there ? voff + chunk * 512 + i * 16 * pitch : kNoFetch);
  }
  TGG_DEV int chunk_buffer(int chunk) const { return (chunk - step) % STAGES; }
  // run(x fragments, w fragments) for every chunk, on the wave's 32 values of it
  template <class F> TGG_DEV void run(F&& f) {
    const int lane = lane_id(), l16 = lane & 15, lg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int frag = l16 * 512 + (((4 * wave + lg) ^ l16) << 4);
    for (int c = step; c < end; ++c) {
      wait_vmcnt<(STAGES - 2) * NC>();
      __syncthreads();  // the chunk is there, and the buffer of the one before has been read
      copy(c + STAGES - 1);
      const char* const s = smem + chunk_buffer(c) * STAGE_BYTES + frag;
      i32x4_t x[XB], w[WB];
#pragma unroll
      for (int i = 0; i < XB; ++i) x[i] = *(const i32x4_t*)(s + i * 8192);
#pragma unroll
      for (int i = 0; i < WB; ++i) w[i] = *(const i32x4_t*)(s + X_BYTES + i * 8192);
      f(x, w);
    }
    wait_vmcnt<0>();  // (the copies behind the last chunk fetch nothing, but write)
    __syncthreads();
  }
  TGG_DEV void start() {
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) copy(step + i);
  }
};

constexpr int kDownThreads = 512, kDownWaves = 8;
// chunks of `blocks` blocks of 16 rows (8 KB each) in the ring: two workgroups a compute unit where three chunks of each fit
constexpr int down_stages(int blocks) { return blocks <= 2 ? 5 : blocks <= 6 ? 3 : 2; }

struct DownParams {
  const void* x;     // [M, depth]
  const void* a;     // [L, R, depth]
  const float* scales;
  Ids ids;
  float* h;          // [parts, M, R]: the sums, part by part of the depth
  uint16_t* planes;  // [M, 2, R] bfloat16, or null
  int64_t M;
  int R, depth, parts;
};

// RB: blocks of 16 rows, RC: blocks of 16 of R (RC * 16 >= R).  blockIdx.x: rows; y: adapters in turn; z: part of the depth.  Bound by reading the rows (16384 x 4096, rank 16: 31 us, 4.3 TB/s)
// where they follow one another, by a ring's start for every adapter of 16 rows (and the adapters, from L2) where they are mixed: 2047 rows of 16 adapters, rank 32, depth 1536, 20 us.
template <int DT, int RB, int RC> __global__ __launch_bounds__(kDownThreads) void lora_down_kernel(const DownParams p) {
  constexpr int COLS = RC * 16, STAGES = down_stages(RB + RC);
  typedef ChunkRing<RB, RC, STAGES> Ring;
  static_assert(kDownWaves * 16 * COLS * 4 <= Ring::BYTES, "the waves' sums reuse the ring");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  float* const sums = (float*)smem;
  const int lane = lane_id(), l16 = lane & 15, lg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row0 = (int64_t)blockIdx.x * (16 * RB);
  const int rows = (int)lesser(16 * RB, p.M - row0);
  const int id = lane < rows ? p.ids.at(row0 + lane) : -1;
  // lanes whose row is the first of its adapter
  uint64_t firsts = 0;
#pragma unroll
  for (int i = 0; i < 16 * RB; ++i) {
    const int other = __builtin_amdgcn_readlane(id, i);
    const uint64_t same = __ballot(id == other);
    if (other >= 0 && (same & ((1ull << i) - 1)) == 0) firsts |= 1ull << i;
  }
  const int chunks = (p.depth + 255) / 256, first_chunk = (int)((int64_t)chunks * blockIdx.z / p.parts), end_chunk = (int)((int64_t)chunks * (blockIdx.z + 1) / p.parts);
  float* const h = p.h + (int64_t)blockIdx.z * p.M * p.R;
  if (blockIdx.y == 0) {  // rows without an adapter
    for (int i = threadIdx.x; i < rows * p.R; i += kDownThreads) {
      const int r = i / p.R, c = i - r * p.R;
      if (p.ids.at(row0 + r) < 0) {
        h[(row0 + r) * p.R + c] = 0.f;
        if (p.planes) p.planes[((row0 + r) * 2) * p.R + c] = p.planes[((row0 + r) * 2 + 1) * p.R + c] = 0;
      }
    }
  }
  uint64_t left = firsts;
  for (int turn = 0; left; ++turn, left &= left - 1) {
    if (turn % (int)gridDim.y != (int)blockIdx.y) continue;
    const int l = __builtin_amdgcn_readlane(id, __ffsll((unsigned long long)left) - 1);
    const uint64_t keep = __ballot(id == l);
    Ring ring(smem, (const uint16_t*)p.x + row0 * p.depth, (int64_t)rows * p.depth * 2, (const uint16_t*)p.a + (int64_t)l * p.R * p.depth, (int64_t)p.R * p.depth * 2, p.depth, first_chunk, end_chunk);
    f32x4_t acc[RB][RC];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int c = 0; c < RC; ++c) acc[b][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    ring.start();
    ring.run([&](const i32x4_t (&x)[RB], const i32x4_t (&a)[RC]) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int c = 0; c < RC; ++c) acc[b][c] = stream_mma<DT>(a[c], x[b], acc[b][c]);  // lane: row l16, columns 4 lg + (0..3)
    });
    const float scale = p.scales ? p.scales[l] : 1.f;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      if (b) __syncthreads();
#pragma unroll
      for (int c = 0; c < RC; ++c) *(f32x4_t*)&sums[(wave * 16 + l16) * COLS + 16 * c + 4 * lg] = acc[b][c];
      __syncthreads();
      // 32 threads a row
      const int r = threadIdx.x >> 5, row = b * 16 + r;
      const bool mine = row < rows && (keep >> row & 1);
#pragma unroll
      for (int i = 0; i < (COLS + 31) / 32; ++i) {
        const int c = (threadIdx.x & 31) + 32 * i;
        if (mine && c < p.R) {
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < kDownWaves; ++w) v += sums[(w * 16 + r) * COLS + c];
          v *= scale;
          h[(row0 + row) * p.R + c] = v;
          if (p.planes) {
            uint16_t hi, lo;
            split2<DT_BF16>(v, hi, lo);
            p.planes[((row0 + row) * 2) * p.R + c] = hi;
            p.planes[((row0 + row) * 2 + 1) * p.R + c] = lo;
          }
        }
      }
    }
    __syncthreads();  // the sums have been read: the ring's again
  }
}

// Two stacks of L matrices, transposed, for the backward pass, whose sums run along the other sides (8 adapters of 4096 + 4096 columns, rank 16: 8 us): [L, rows, cols] -> [L, cols, rows]
struct TransposeParams {
  struct { const uint16_t* in; uint16_t* out; int rows, cols, tiles_r, tiles_c; } s[2];
  int first;  // workgroups of the first stack
};
__global__ __launch_bounds__(256) void lora_transpose_kernel(const TransposeParams p) {
  __shared__ uint16_t tile[64][66];
  const int second = (int)blockIdx.x >= p.first, id = second ? blockIdx.x - p.first : blockIdx.x;
  const auto& q = p.s[second];
  const uint16_t* const in = q.in;
  uint16_t* const out = q.out;
  const int N = q.rows, R = q.cols;
  const int per = q.tiles_r * q.tiles_c, l = id / per, t = id % per, n0 = t / q.tiles_c * 64, r0 = t % q.tiles_c * 64, x = threadIdx.x & 63;
  for (int y = threadIdx.x >> 6; y < 64; y += 4)
    if (n0 + y < N && r0 + x < R) tile[y][x] = in[((int64_t)l * N + n0 + y) * R + r0 + x];
  __syncthreads();
  for (int y = threadIdx.x >> 6; y < 64; y += 4)
    if (r0 + y < R && n0 + x < N) out[((int64_t)l * R + r0 + y) * N + n0 + x] = tile[x][y];
}

// ---- the shared product with the adapters' depth added ---------------------------------------------------------------------
// 16384 rows, 4096 x 4096, rank 16: y 392 to 424 us, dx 402 to 431 (1.28 to 1.40 PFLOP/s, the matrix pipe 0.73 of the cycles; torch's library product of 8192 x 8192 x 8192 reaches 1.39).  Where a tile's rows are of many
// adapters every one of them is R more values of depth in two planes (and again two for the parts of half-precision adapters): 2047 rows of 16 adapters, rank 32, 1536 x 2048, 57 and 63 us, of which the
// adapters' part is more than half.

struct LoraGemm {
  const void* x;        // [M, depth]
  const void* w;        // NT [cols, depth], NN [depth, cols]
  const uint16_t* pair;    // [L, cols, R]: B, or A transposed
  const uint16_t* planes;  // [M, 2, R] bfloat16
  Ids ids;
  void* out;            // [M, cols]
  int64_t M;
  int cols, depth, R, tiles_m, tiles_n;
};

template <class C, int DT, bool NT> struct LoraProblem {
  static constexpr int PITCH = C::TN * 32 + 16, STAGE_WAVE = 16 * PITCH;
  static constexpr int SMEM_BYTES = C::EPI_OFF + C::NWAVES * STAGE_WAVE;
  static constexpr int CHUNK = 8;  // column tiles that are taken together
  static constexpr uint32_t EXPONENT = DT == DT_BF16 ? 0x7f80u : 0x7c00u, ONES = DT == DT_BF16 ? 0x3f803f80u : 0x3c003c00u;

  const LoraGemm& p;
  StreamWalk walk;
  StreamCursor<C, NT> cur;
  int pos;
  bool infinite;  // begin() has left something out

  TGG_DEV explicit LoraProblem(const LoraGemm& q) : p(q), walk(q.tiles_m * q.tiles_n), cur(q.depth * 2, (NT ? q.depth : q.cols) * 2, q.depth) { pos = -1; }
  TGG_DEV int tile_at(int q) const { return walk.at(q); }
  TGG_DEV int slabs(int) const { return cur.kt; }
  // chunks of column tiles, in them row tiles, in them columns: the workgroups of an XCD share rows and columns
  struct Place { int tm, tn; };
  TGG_DEV Place locate(int id) const {
    const int full = p.tiles_n / CHUNK * CHUNK, first = CHUNK * p.tiles_m;
    const int c = id / first, in = id - c * first, width = c * CHUNK < full ? CHUNK : p.tiles_n - full;
    const int tm = in / width;
    return {__builtin_amdgcn_readfirstlane(tm), __builtin_amdgcn_readfirstlane(c * CHUNK + in - tm * width)};
  }
  TGG_DEV void seek(int id) {
    ++pos;
    const bool live = id >= 0;
    const Place at = locate(live ? id : 0);
    const int64_t row0 = (int64_t)at.tm * C::BM, col0 = (int64_t)at.tn * C::BN;
    cur.begin(live, (uint64_t)p.x + row0 * p.depth * 2, (uint64_t)p.w + (NT ? col0 * p.depth : col0) * 2, (int)lesser(C::BM, p.M - row0), NT ? min(C::BN, p.cols - (int)col0) : p.depth, (int)col0 * 2);
  }
  TGG_DEV void turn() { seek(tile_at(pos + 1)); }

  // The adapters' part.  Rows of other adapters are zeros against an adapter, and zero times infinity or NaN is NaN: where a wave's rows do not all have the
  // adapter, what is not finite becomes a one of its sign (so that an infinite row stays infinite), and add_infinite() adds it to the rows that it belongs to.  The low plane of h meets ones
  // instead of what is not finite in any case: it may be zero or of the other sign, and the high plane's product is infinite, or NaN, by itself.
  TGG_DEV void begin(int id, f32x4_t (&acc)[C::TM][C::TN], const StreamPlace<C>& at) {
    const Place tile = locate(id);
    int el = at.lane;
    asm volatile("" : "+v"(el));  // (addresses are made afresh per tile instead of living across the multiplies)
    const int l16 = el & 15, lg = el >> 4;
    const int64_t row0 = (int64_t)tile.tm * C::BM + at.wm0;
    const int rows = (int)lesser(C::BM / C::WM, p.M - row0), col0 = tile.tn * C::BN + at.wn0;  // (rows may be negative)
    infinite = false;
    if (rows <= 0) return;
    int ids[C::TM];
#pragma unroll
    for (int i = 0; i < C::TM; ++i) ids[i] = 16 * i + l16 < rows ? p.ids.at(row0 + 16 * i + l16) : -1;
    const rsrc_t hw = window(p.planes + row0 * 2 * p.R, (int64_t)rows * p.R * 4);
    // Steps of 32 values of depth (the high plane, then the low one) of every adapter, in the order of their numbers.  Of narrow tiles a step's operands are under way while the
    // step before is multiplied (16 adapters in 64 rows, rank 32: the two steps of each took 1.25 us, the wait for memory).
    struct Step {
      int l, k0;
      bool mixed;
    };
    auto next_adapter = [&](int after) __attribute__((always_inline)) {
      uint32_t lowest = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < C::TM; ++i) lowest = ids[i] > after && (uint32_t)ids[i] < lowest ? (uint32_t)ids[i] : lowest;
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) {  // (all four groups of lanes hold the same rows)
        const uint32_t other = (uint32_t)__shfl_xor((int)lowest, d, 64);
        lowest = other < lowest ? other : lowest;
      }
      Step s;
      s.l = __builtin_amdgcn_readfirstlane((int)lowest);
      s.k0 = 0;
      bool all = true;
#pragma unroll
      for (int i = 0; i < C::TM; ++i) all = all && (ids[i] == s.l || 16 * i + l16 >= rows);
      s.mixed = __ballot(!all) != 0;
      return s;
    };
    auto advance = [&](const Step& s) __attribute__((always_inline)) {
      if (s.k0 + 32 < 2 * p.R) return Step{s.l, s.k0 + 32, s.mixed};
      return next_adapter(s.l);
    };
    auto load = [&](const Step& s, i32x4_t (&a)[C::TM], i32x4_t (&b)[C::TN]) __attribute__((always_inline)) {
      const rsrc_t bw = window(p.pair + ((int64_t)s.l * p.cols + col0) * p.R, (int64_t)min(C::BN / C::WN, p.cols - col0) * p.R * 2);
      const int k = s.k0 + 8 * lg, r = k < p.R ? k : k - p.R;
#pragma unroll
      for (int j = 0; j < C::TN; ++j) b[j] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(bw, k < 2 * p.R ? ((16 * j + l16) * p.R + r) * 2 : kNowhere, 0, 0));
#pragma unroll
      for (int i = 0; i < C::TM; ++i) a[i] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(hw, ids[i] == s.l && k < 2 * p.R ? ((16 * i + l16) * 2 * p.R + k) * 2 : kNowhere, 0, 0));
    };
    auto multiply = [&](const Step& s, const i32x4_t (&a)[C::TM], i32x4_t (&b)[C::TN]) __attribute__((always_inline)) {
      if (s.mixed || s.k0 + 32 > p.R) {
        const uint32_t replaced = s.mixed || s.k0 + 8 * lg >= p.R ? 0xffffffffu : 0u;
        uint32_t out = 0;
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t x = (uint32_t)b[j][w], bad = (((x & EXPONENT) == EXPONENT ? 0xffffu : 0u) | ((x >> 16 & EXPONENT) == EXPONENT ? 0xffff0000u : 0u)) & replaced;
            b[j][w] = (int)((x & ~bad) | (((x & 0x80008000u) | ONES) & bad));
            out |= bad;
          }
        }
        infinite = infinite || (s.mixed && __ballot(out != 0) != 0);
      }
      i32x4_t rest[C::TN];
      if (DT == DT_F16) {
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float v0 = from_bits<DT_F16>((uint16_t)b[j][w]), v1 = from_bits<DT_F16>((uint16_t)((uint32_t)b[j][w] >> 16));
            // the eight bits next to v on zero's side, and what is left (four bits): both have v's sign and neither is zero but for v = 0, so that they agree on an infinite h's product
            const uint32_t u0 = __builtin_bit_cast(uint32_t, v0), u1 = __builtin_bit_cast(uint32_t, v1);
            const uint32_t t0 = (u0 - (v0 != 0.f ? 1u : 0u)) & 0xffff0000u, t1 = (u1 - (v1 != 0.f ? 1u : 0u)) & 0xffff0000u;
            b[j][w] = (int)(t0 >> 16 | t1);
            rest[j][w] = (int)pack2<DT_BF16>(v0 - __builtin_bit_cast(float, t0), v1 - __builtin_bit_cast(float, t1));
          }
      }
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        if (__ballot(ids[i] == s.l) == 0) continue;
#pragma unroll
        for (int j = 0; j < C::TN; ++j) acc[i][j] = stream_mma<DT_BF16>(b[j], a[i], acc[i][j]);
        if (DT == DT_F16) {
#pragma unroll
          for (int j = 0; j < C::TN; ++j) acc[i][j] = stream_mma<DT_BF16>(rest[j], a[i], acc[i][j]);
        }
      }
    };
    i32x4_t a0[C::TM], b0[C::TN];
    if constexpr (C::TM == 4) {
      i32x4_t a1[C::TM], b1[C::TN];
      Step s = next_adapter(-1);
      if (s.l >= 0) load(s, a0, b0);
      while (s.l >= 0) {
        const Step t = advance(s);
        if (t.l >= 0) load(t, a1, b1);
        multiply(s, a0, b0);
        if (t.l < 0) break;
        s = advance(t);
        if (s.l >= 0) load(s, a0, b0);
        multiply(t, a1, b1);
      }
    } else {
      for (Step s = next_adapter(-1); s.l >= 0; s = advance(s)) {
        load(s, a0, b0);
        multiply(s, a0, b0);
      }
    }
  }
  // What begin() has taken out: an infinity or a NaN, whatever finite value or infinity of its sign it is added to, so it may as well be added to the stored outputs.
  TGG_DEV void add_infinite(int64_t row0, int col0, int lane) const {
    wait_vmcnt<0>();  // (the wave's own stores)
    const int col = col0 + lane;
    if (lane >= C::BN / C::WN || col >= p.cols) return;
#pragma unroll 1
    for (int64_t row = row0; row < lesser(row0 + C::BM / C::WM, p.M); ++row) {
      const int l = p.ids.at(row);
      if (l < 0) continue;
      const uint16_t* const b = p.pair + ((int64_t)l * p.cols + col) * p.R;
      float add = 0.f;
#pragma unroll 1
      for (int r = 0; r < p.R; ++r)
        if ((b[r] & EXPONENT) == EXPONENT) add += from_bits<DT>(b[r]) * (from_bits<DT_BF16>(p.planes[row * 2 * p.R + r]) + from_bits<DT_BF16>(p.planes[(row * 2 + 1) * p.R + r]));
      volatile uint16_t* const o = (volatile uint16_t*)p.out + row * p.cols + col;
      if (add != 0.f) *o = Out16<DT>::cvt(from_bits<DT>(*o) + add);
    }
  }

  TGG_DEV void epilogue(int id, f32x4_t (&acc)[C::TM][C::TN], const StreamPlace<C>& at, char* stage) const {
    int el = at.lane;
    asm volatile("" : "+v"(el));
    const int l16 = el & 15, lg = el >> 4;
    const Place tile = locate(id);
    char* const mine = stage + at.wave * STAGE_WAVE;
    const int cbase = tile.tn * C::BN + at.wn0;
    const int64_t rbase = (int64_t)tile.tm * C::BM + at.wm0;
    constexpr int CPS = 2 * C::TN, PASSES = 16 * CPS / 64;  // 16-byte pieces of a staged row, wave-wide reads of a strip
    static_assert(PASSES * 64 == 16 * CPS, "a strip is read back by whole waves");
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) *(uint2*)(mine + l16 * PITCH + (16 * j + 4 * lg) * 2) = pack4<DT>(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
      asm volatile("" : : : "memory");
#pragma unroll
      for (int it = 0; it < PASSES; ++it) {
        const int idx = it * 64 + el, r = idx / CPS, ch = idx % CPS;
        const i32x4_t v = *(const i32x4_t*)(mine + r * PITCH + ch * 16);
        const int64_t row = rbase + 16 * i + r;
        if (row < p.M && cbase + ch * 8 < p.cols) store_c((i32x4_t*)((uint16_t*)p.out + row * p.cols + cbase + ch * 8), v, 1);
      }
      asm volatile("" : : : "memory");
    }
    if (__builtin_expect(infinite, 0)) add_infinite(rbase, cbase, el);
  }
};

template <class C, int DT, bool NT> __global__ __launch_bounds__(C::THREADS, C::BM == 128 ? 4 : 2) void lora_gemm_kernel(const LoraGemm p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  LoraProblem<C, DT, NT> prob(p);
  stream_gemm<C, DT, NT>(prob, smem);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------

constexpr int kFewThreads = 512, kFewWaves = 8;

struct FewParams {
  const void *x, *w, *b;
  const float* h;  // [parts, M, R]
  Ids ids;
  void* out;
  int64_t M;
  int N, K, R, parts;
};

// RB blocks of 16 rows x 16 columns; the waves share the depth.  Bound by W: 64 rows, 4096 x 4096, 14.2 us for 34 MB of W (2.4 TB/s, every compute unit reads x's 512 KB besides, from L2); one row,
// 768 x 2048, 5.2 us, the latency of a ring's start, the adapters' part and the join of eight waves.
template <int DT, int RB> __global__ __launch_bounds__(kFewThreads) void lora_few_kernel(const FewParams p) {
  constexpr int ROWS = RB * 16, COLS = 16, QUADS = ROWS * COLS / 4;
  typedef ChunkRing<RB, 1, RB == 1 ? 6 : RB == 2 ? 5 : 3> Ring;
  static_assert(QUADS <= kFewThreads && kFewWaves * ROWS * COLS * 4 <= Ring::BYTES, "a thread has four outputs; the waves' sums reuse the ring");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  float* const sums = (float*)smem;
  const int lane = lane_id(), l16 = lane & 15, lg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * COLS;
  const int64_t row0 = (int64_t)blockIdx.y * ROWS;
  const int rows = (int)lesser(ROWS, p.M - row0);
  Ring ring(smem, (const uint16_t*)p.x + row0 * p.K, (int64_t)rows * p.K * 2, (const uint16_t*)p.w + (int64_t)n0 * p.K, (int64_t)lesser(COLS, p.N - n0) * p.K * 2, p.K, 0, (p.K + 255) / 256);
  ring.start();
  // the adapters' part of the thread's outputs, four columns of one row, while the first weights arrive
  float own[4] = {0.f, 0.f, 0.f, 0.f};
  const int r = threadIdx.x / (COLS / 4), c = threadIdx.x % (COLS / 4) * 4;
  const bool mine = r < rows && n0 + c < p.N;
  if (mine) {
    const int id = p.ids.at(row0 + r);
    if (id >= 0) {
      const uint16_t* const b = (const uint16_t*)p.b + ((int64_t)id * p.N + n0 + c) * p.R;
      for (int k = 0; k < p.R; k += 8) {
        float h[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int part = 0; part < p.parts; ++part) {
          const f32x4_t* const hp = (const f32x4_t*)(p.h + ((int64_t)part * p.M + row0 + r) * p.R + k);
          const f32x4_t h0 = hp[0], h1 = hp[1];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[e] += h0[e];
            h[4 + e] += h1[e];
          }
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const i32x4_t v = *(const i32x4_t*)(b + (int64_t)y * p.R + k);
#pragma unroll
          for (int e = 0; e < 8; ++e) own[y] = __builtin_fmaf(h[e], from_bits<DT>((uint16_t)((uint32_t)v[e / 2] >> (16 * (e & 1)))), own[y]);
        }
      }
    }
  }
  f32x4_t acc[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) acc[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  ring.run([&](const i32x4_t (&x)[RB], const i32x4_t (&w)[1]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[b] = stream_mma<DT>(w[0], x[b], acc[b]);
  });
#pragma unroll
  for (int b = 0; b < RB; ++b) *(f32x4_t*)&sums[(wave * ROWS + 16 * b + l16) * COLS + 4 * lg] = acc[b];
  __syncthreads();
  if (mine) {
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      const f32x4_t t = *(const f32x4_t*)&sums[(w * ROWS + r) * COLS + c];
#pragma unroll
      for (int e = 0; e < 4; ++e) own[e] += t[e];
    }
    *(uint2*)((uint16_t*)p.out + (row0 + r) * p.N + n0 + c) = pack4<DT>(own[0], own[1], own[2], own[3]);
  }
}

// ---- gradients of the adapters ------------------------------------------------------------------------------------------

constexpr int kOuterThreads = 256, kOuterWaves = 4, kOuterCols = 128, kOuterRows = 64, kOuterWindow = 4096;

struct OuterParams {
  const void *x, *g;       // [M, K], [M, N]
  const float *dh, *h;     // [M, R]
  Ids ids;
  void *da, *db;           // [L, R, K], [L, N, R]; either may be null
  float *part_a, *part_b;  // [parts, L, ...] where there are several parts
  int32_t* rows;           // [parts, L]: rows of each part
  int64_t M;
  int K, N, R, L, parts, blocks_a;
};

// blockIdx.x: 128 columns of K (dA), then of N (dB); y: adapter; z: part of the rows.  RC blocks of 16 of R.  Every workgroup lists its adapter's rows window by window, so that ids may stand in any
// order, and sums them in the order of their numbers.  Bound by reading x and g once: 16384 rows of 8 adapters, 4096 + 4096 columns, 85 to 91 us for 268 MB (3.0 TB/s); 2047 rows of 16, 14 us.
// (Every workgroup reads all ids: 1024 adapters of 16384 rows, 65536 workgroups, 4.3 GB of them, from L2.)
template <int DT, int RC> __global__ __launch_bounds__(kOuterThreads) void lora_outer_kernel(const OuterParams p) {
  typedef Operand<kOuterCols, false> OpZ;
  constexpr int Z_BYTES = OpZ::SLAB_BYTES, PP = RC * 32 + 16, P_BYTES = kOuterRows * PP;  // a plane of the P tile: 64 rows of RC * 16 values
  constexpr uint32_t EXPONENTS = DT == DT_BF16 ? 0x7f807f80u : 0x7c007c00u, EXPONENT_STEP = DT == DT_BF16 ? 0x00800080u : 0x04000400u;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  char* const zbuf = smem;                   // two tiles of 64 rows x 128 columns
  char* const pbuf = smem + 2 * Z_BYTES;     // high and low plane
  uint16_t* const list = (uint16_t*)(pbuf + 2 * P_BYTES);
  int32_t* const scan = (int32_t*)(list + kOuterWindow);
  float* const tops = (float*)(scan + kOuterWaves);
  const int lane = lane_id(), l16 = lane & 15, lg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool is_a = (int)blockIdx.x < p.blocks_a;
  const int l = blockIdx.y, cols = is_a ? p.K : p.N, col0 = (is_a ? blockIdx.x : blockIdx.x - p.blocks_a) * kOuterCols;
  const uint16_t* const z = (const uint16_t*)(is_a ? p.x : p.g);
  const float* const src = is_a ? p.dh : p.h;
  const int64_t begin = p.M * blockIdx.z / p.parts, end = p.M * (blockIdx.z + 1) / p.parts;
  const uint32_t smem_addr = (uint32_t)(uintptr_t)(lds_ptr_t)smem;

  f32x4_t acc[RC][2];
#pragma unroll
  for (int c = 0; c < RC; ++c) acc[c][0] = acc[c][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float unit = 0.f;  // fp16: what P is multiplied with, acc's values too (0: nothing so far)
  int total = 0;
  // the lane's place in a copy of four rows, and its chunk of the row
  const int z_row = lane / OpZ::CPR, z_chunk = (lane % OpZ::CPR) ^ OpZ::token_swizzle(wave * OpZ::RPI + z_row);
  const bool z_there = col0 + z_chunk * 8 < cols;

  for (int64_t w0 = begin; w0 < end; w0 += kOuterWindow) {
    // the window's rows of this adapter, in order
    constexpr int PER = kOuterWindow / kOuterThreads;
    const int n = (int)lesser(kOuterWindow, end - w0);
    int count = 0;
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = threadIdx.x * PER + i;
      if (r < n && p.ids.at(w0 + r) == l) {
        mine |= 1u << i;
        ++count;
      }
    }
    int incl = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d, 64);
      if (lane >= d) incl += o;
    }
    __syncthreads();  // the list and the scan of the window before have been read
    if (lane == 63) scan[wave] = incl;
    __syncthreads();
    int at = incl - count, all = 0;
    for (int w = 0; w < kOuterWaves; ++w) {
      if (w < wave) at += scan[w];
      all += scan[w];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (mine >> i & 1) list[at++] = (uint16_t)(threadIdx.x * PER + i);
    __syncthreads();
    all = __builtin_amdgcn_readfirstlane(all);
    if (!all) continue;
    total += all;
    const i32x4_t zr = make_rsrc((uint64_t)z + (uint64_t)(w0 * cols + col0) * 2, (n * (int64_t)cols - col0) * 2);
    auto copy = [&](int c, int buf) {
#pragma unroll
      for (int k = 0; k < OpZ::NI / kOuterWaves; ++k) {
        const int idx = wave + k * kOuterWaves, r = c * kOuterRows + idx * OpZ::RPI + z_row;
        const int voff = r < all && z_there ? (int)list[r < all ? r : 0] * cols * 2 + z_chunk * 16 : kNoFetch;
        copy_b128_to_lds(zr, __builtin_amdgcn_readfirstlane(smem_addr + buf * Z_BYTES + idx * 1024), voff);
      }
    };
    const int chunks = (all + kOuterRows - 1) / kOuterRows;
    copy(0, 0);
    for (int c = 0; c < chunks; ++c) {
      // P: 64 rows of R values in fp32, four threads a row
      constexpr int VALUES = RC * 4;
      const int pr = threadIdx.x >> 2, pc = (threadIdx.x & 3) * VALUES, r = c * kOuterRows + pr;
      float v[VALUES], top = 0.f;
      const float* const row = src + (w0 + list[r < all ? r : 0]) * p.R;
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        v[i] = r < all && pc + i < p.R ? row[pc + i] : 0.f;
        top = fmaxf(top, __builtin_isfinite(v[i]) ? fabsf(v[i]) : 0.f);  // (an infinity needs no scale and must not set the others')
      }
      if (DT == DT_F16) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        if (lane == 0) tops[wave] = top;
      }
      wait_vmcnt<0>();
      __syncthreads();  // this chunk's Z is there, the planes of the chunk before have been read
      if (DT == DT_F16) {
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const float want = row_scale(top);
        if (top > 0.f && (unit == 0.f || want < unit)) {  // larger values than before: the sums move to their scale
          const float by = unit == 0.f ? 0.f : fmaxf(want / unit, __FLT_MIN__);  // (zero would make NaN of infinite sums)
#pragma unroll
          for (int q = 0; q < RC; ++q)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[q][b][e] = unit == 0.f ? acc[q][b][e] : acc[q][b][e] * by;
          unit = want;
        }
      }
      const float by = DT == DT_F16 && unit != 0.f ? unit : 1.f;
#pragma unroll
      for (int i = 0; i < VALUES; i += 4) {
        uint16_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split2<DT>(v[i + e] * by, hi[e], lo[e], DT == DT_F16);
        *(uint2*)(pbuf + pr * PP + (pc + i) * 2) = {(uint32_t)hi[0] | (uint32_t)hi[1] << 16, (uint32_t)hi[2] | (uint32_t)hi[3] << 16};
        *(uint2*)(pbuf + P_BYTES + pr * PP + (pc + i) * 2) = {(uint32_t)lo[0] | (uint32_t)lo[1] << 16, (uint32_t)lo[2] | (uint32_t)lo[3] << 16};
      }
      __syncthreads();
      if (c + 1 < chunks) copy(c + 1, (c + 1) & 1);
      const char* const zs = zbuf + (c & 1) * Z_BYTES;
      const int e4 = l16 >> 2, c4 = l16 & 3;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        i32x4_t zf[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int chunk = ((wave * 32 + 16 * b) / 8 + (c4 >> 1)) ^ OpZ::token_swizzle(8 * (lg & 1) + e4);
          const char* const q = zs + (ks * 32 + lg * 8 + e4) * OpZ::ROW_BYTES + chunk * 16 + (c4 & 1) * 8;
          const i16x4_t lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr_t)q);
          const i16x4_t hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr_t)(q + 4 * OpZ::ROW_BYTES));
          zf[b] = __builtin_bit_cast(i32x4_t, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        // Z for the low plane of P, which may be zero or of the other sign: without infinities and NaN, whose products the high plane has.  (An exponent of ones carries into the sign's place)
        i32x4_t zl[2] = {zf[0], zf[1]};
        uint32_t ones = 0;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int w = 0; w < 4; ++w) ones |= ((uint32_t)zf[b][w] & EXPONENTS) + EXPONENT_STEP;
        if (__builtin_expect(__ballot((ones & 0x80008000u) != 0) != 0, 0)) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t at = (((uint32_t)zf[b][w] & EXPONENTS) + EXPONENT_STEP) & 0x80008000u;
              zl[b][w] = (int)((uint32_t)zf[b][w] & ~((at >> 15) * 0xffffu));
            }
        }
#pragma unroll
        for (int plane = 0; plane < 2; ++plane)
#pragma unroll
          for (int q = 0; q < RC; ++q) {
            const char* const s = pbuf + plane * P_BYTES + (ks * 32 + lg * 8 + e4) * PP + q * 32 + c4 * 8;
            const i16x4_t lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr_t)s);
            const i16x4_t hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr_t)(s + 4 * PP));
            const i32x4_t pf = __builtin_bit_cast(i32x4_t, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const i32x4_t& zv = plane ? zl[b] : zf[b];
              acc[q][b] = is_a ? stream_mma<DT>(zv, pf, acc[q][b]) : stream_mma<DT>(pf, zv, acc[q][b]);
            }
          }
      }
    }
  }
  if (p.parts > 1 && blockIdx.x == 0 && threadIdx.x == 0) p.rows[blockIdx.z * p.L + l] = total;
  if (p.parts > 1 && !total) return;
  const float back = DT == DT_F16 && unit != 0.f ? 1.f / unit : 1.f;
  // dA: lane has row 16 q + l16 of R, columns 16 b + 4 lg + (0..3); dB: row 16 b + l16 of N, columns 16 q + 4 lg + (0..3) of R
#pragma unroll
  for (int q = 0; q < RC; ++q)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int zc = col0 + wave * 32 + 16 * b, r = 16 * q + (is_a ? l16 : 4 * lg), c = zc + (is_a ? 4 * lg : l16);
      if (r >= p.R || c >= cols) continue;
      const f32x4_t v = {acc[q][b][0] * back, acc[q][b][1] * back, acc[q][b][2] * back, acc[q][b][3] * back};
      const int64_t o = is_a ? ((int64_t)l * p.R + r) * p.K + c : ((int64_t)l * p.N + c) * p.R + r;
      if (p.parts > 1) {
        float* const part = is_a ? p.part_a + (int64_t)blockIdx.z * p.L * p.R * p.K : p.part_b + (int64_t)blockIdx.z * p.L * p.R * p.N;
        *(f32x4_t*)(part + o) = v;
      } else {
        *(uint2*)((uint16_t*)(is_a ? p.da : p.db) + o) = pack4<DT>(v[0], v[1], v[2], v[3]);
      }
    }
}

// The parts' sums, in order.  Four values a thread; dA's values and then dB's.
template <int DT> __global__ __launch_bounds__(256) void lora_join_kernel(const OuterParams p) {
  const int64_t per_a = (int64_t)p.R * p.K, per_b = (int64_t)p.R * p.N, quads_a = p.da ? p.L * per_a / 4 : 0, quads_b = p.db ? p.L * per_b / 4 : 0;
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads_a + quads_b) return;
  const bool is_a = i < quads_a;
  if (!is_a) i -= quads_a;
  const int64_t per = is_a ? per_a : per_b, o = i * 4;
  const int l = (int)(o / per);
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.parts; ++s) {
    if (!p.rows[s * p.L + l]) continue;
    const f32x4_t t = *(const f32x4_t*)((is_a ? p.part_a : p.part_b) + s * p.L * per + o);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += t[e];
  }
  *(uint2*)((uint16_t*)(is_a ? p.da : p.db) + o) = pack4<DT>(v[0], v[1], v[2], v[3]);
}

// ---- launches ---------------------------------------------------------------------------------------------------------------

int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

template <class Kern, class P> int launch_smem(Kern kern, int smem, bool (&attr_set)[64], dim3 grid, int threads, const P& p, hipStream_t s, const char* what) {
  if (int e = stream_lds(kern, smem, attr_set)) return e;
  kern<<<grid, dim3(threads), smem, s>>>(p);
  return check_launch(what);
}

template <int DT, int RB, int RC> int down_launch(const DownParams& p, hipStream_t s) {
  static bool attr_set[64] = {false};
  constexpr int smem = ChunkRing<RB, RC, down_stages(RB + RC)>::BYTES;
  const int64_t blocks = (p.M + 16 * RB - 1) / (16 * RB);
  // few rows: their adapters side by side
  const int turns = RB > 1 || blocks >= 1024 ? 1 : (int)lesser(16, 1024 / blocks);
  return launch_smem(lora_down_kernel<DT, RB, RC>, smem, attr_set, dim3((unsigned)blocks, turns, p.parts), kDownThreads, p, s, "lora_down");
}

template <int DT> int launch_down(const DownParams& p, hipStream_t s) {
  const int rc = (p.R + 15) / 16;
  if (rc > 4) return down_launch<DT, 1, 8>(p, s);
  // 32 rows a workgroup read the adapter half as often, which pays where its chunks are the larger part and the chip is full anyway: depth 4096, rank 64, with the product behind it, 16384 rows
  // 117 us (16 rows: 126), 4096 rows 88 (87); rank 16, 16384 rows 95 (92).
  if (rc > 2) return p.M >= 8192 ? down_launch<DT, 2, 4>(p, s) : down_launch<DT, 1, 4>(p, s);
  return rc <= 1 ? down_launch<DT, 1, 1>(p, s) : down_launch<DT, 1, 2>(p, s);
}

typedef StreamCfg<256, 256, 2, 4> LoraWide;
typedef StreamCfg<128, 128, 2, 4> LoraNarrow;

template <class C, int DT, bool NT> int gemm_launch(const LoraGemm& p, hipStream_t s) {
  typedef LoraProblem<C, DT, NT> P;
  static bool attr_set[64] = {false};
  const int tiles = p.tiles_m * p.tiles_n, slots = num_cus() * (C::BM == 128 ? 2 : 1);
  return launch_smem(lora_gemm_kernel<C, DT, NT>, P::SMEM_BYTES, attr_set, dim3(tiles < slots ? tiles : slots), C::THREADS, p, s, "lora_gemm");
}

template <int DT, bool NT> int launch_gemm(LoraGemm p, int tile, hipStream_t s) {
  p.tiles_m = (int)((p.M + tile - 1) / tile);
  p.tiles_n = (p.cols + tile - 1) / tile;
  return tile == 256 ? gemm_launch<LoraWide, DT, NT>(p, s) : gemm_launch<LoraNarrow, DT, NT>(p, s);
}

// Tiles of 256 or of 128 for M x cols outputs: a round of 256-row tiles, one a compute unit, takes 1.5 times one of 128-row tiles, two a compute unit.  With the kernel in front, of 8 adapters, rank 16, in runs, in tiles of 128
// and 256: 2048 rows, 4096 x 4096, 78 and 91 us; 4096 rows 146 and 110; 6000 rows, 2568 columns x 4104, 170 and 221; 16384 rows 555 and 404; 16384 rows, 1024 x 1024, 55 and 49.  Rank 64, and 16 adapters in
// mixed rows, have the same faster side in all these (the choice within 5 %), so the rule leaves both out.
int tile_of(int64_t M, int cols) {
  auto tiles = [&](int b) { return (M + b - 1) / b * ((cols + b - 1) / b); };
  const int64_t cus = num_cus();
  return (tiles(256) + cus - 1) / cus * 3 <= (tiles(128) + 2 * cus - 1) / (2 * cus) * 2 ? 256 : 128;
}

// lora_few up to 128 rows.  It reads W once for 64 rows, and rows of many adapters cost it little; with the kernel in front, of 1, 16 and 128 adapters in mixed rows (lora_gemm in brackets), us:
//   columns x depth, rank   64 rows               128                   129                   256                    512
//   4096 x 4096, 16         19 20 21 (64 77 110)  31 32 33 (65 79 112)  41 42 45 (62 74 109)  57 58 61 (65 79 109)   103 108 115 (65 81 111)
//   8192 x 2048, 16         23 24 26 (36 49 83)   40 41 43 (38 50 78)   53 55 57 (35 48 83)   75 76 80 (38 51 85)    138 145 152 (39 54 84)
//   2048 x 1536, 32         13 14 15 (23 42 88)   14 15 16 (24 44 102)  20 21 24 (24 45 95)   23 25 29 (24 46 105)   38 45 52 (24 55 108)
// So up to 128 rows it is the faster one or within 7 %.  Beyond, a limit that looked at N and the number of adapters would gain up to 4 times; this one does not.
bool few_rows(int64_t M) { return M <= 128; }
constexpr int kFewParts = 2;  // parts of the depth in lora_down for few rows: more workgroups, 64 rows of 4096 25.9 us in 2 parts, 26.7 in 1 and 26.4 in 4

template <int DT, int RB> int few_launch(const FewParams& p, hipStream_t s) {
  static bool attr_set[64] = {false};
  constexpr int smem = ChunkRing<RB, 1, (RB == 1 ? 6 : RB == 2 ? 5 : 3)>::BYTES;
  return launch_smem(lora_few_kernel<DT, RB>, smem, attr_set, dim3((p.N + 15) / 16, (unsigned)((p.M + 16 * RB - 1) / (16 * RB))), kFewThreads, p, s, "lora_few");
}
template <int DT> int launch_few(const FewParams& p, hipStream_t s) { return p.M <= 16 ? few_launch<DT, 1>(p, s) : p.M <= 32 ? few_launch<DT, 2>(p, s) : few_launch<DT, 4>(p, s); }

template <int DT, int RC> int outer_launch(const OuterParams& p, dim3 grid, hipStream_t s) {
  constexpr int smem = 2 * kOuterRows * kOuterCols * 2 + 2 * kOuterRows * (RC * 32 + 16) + kOuterWindow * 2 + kOuterWaves * 8;
  static bool attr_set[64] = {false};
  return launch_smem(lora_outer_kernel<DT, RC>, smem, attr_set, grid, kOuterThreads, p, s, "lora_outer");
}

// Parts of the rows: 512 rows of an adapter a part on average, as adapters have unequal shares of the rows and the longest one's workgroups are waited for; adding the parts costs a pass
// over them.  Forward and backward passes, rows in unequal requests: 16384 rows of 8 adapters, 4096 x 4096, 990, 932, 926 and 943 us in 1, 2, 4 and 8 parts; 32768 of 4, 1024 x 1024, 325, 270, 238 and
// 241 in 4, 8, 16 and 32; 2047 of 16, 1536 x 2048, 179 and 191 in 1 and 2; 16384 of 32, 2048 x 2048, 337, 333 and 351 in 1, 2 and 8.
int outer_parts(int64_t M, int N, int K, int L) {
  const int64_t groups = (int64_t)L * ((N + kOuterCols - 1) / kOuterCols + (K + kOuterCols - 1) / kOuterCols);
  return (int)larger(1, lesser(64, lesser(8 * num_cus() / groups, M / (512 * (int64_t)L))));
}

struct LoraPlan {
  int tile, parts;
  int64_t h, planes, at, bt, rows, part_a, part_b, bytes;
};
LoraPlan lora_plan(bool backward, int64_t M, int N, int K, int R, int L) {
  LoraPlan q = {};
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t here = at; at += align256(bytes); return here; };
  q.tile = tile_of(M, backward ? K : N);
  q.h = take((!backward && few_rows(M) ? kFewParts : 1) * M * R * 4);
  q.planes = take(M * R * 4);
  if (backward) {
    q.parts = outer_parts(M, N, K, L);
    q.at = take((int64_t)L * K * R * 2);
    q.bt = take((int64_t)L * N * R * 2);
    q.rows = take((int64_t)q.parts * L * 4);
    if (q.parts > 1) {
      q.part_a = take((int64_t)q.parts * L * R * K * 4);
      q.part_b = take((int64_t)q.parts * L * R * N * 4);
    }
  }
  q.bytes = at;
  return q;
}

template <int DT> int forward(const void* x, const void* w, const void* a, const void* b, const Ids& ids, const float* scales, void* out, float* h, int64_t M, int N, int K, int R, char* ws, hipStream_t s) {
  const LoraPlan q = lora_plan(false, M, N, K, R, ids.L);
  const bool few = few_rows(M);
  DownParams d = {};
  d.x = x; d.a = a; d.scales = scales; d.ids = ids; d.M = M; d.R = R; d.depth = K;
  d.parts = few && !h ? kFewParts : 1;  // (what is kept for the backward pass is one sum)
  d.h = h ? h : (float*)(ws + q.h);
  if (!few) d.planes = (uint16_t*)(ws + q.planes);
  if (int e = launch_down<DT>(d, s)) return e;
  if (few) return launch_few<DT>({x, w, b, d.h, ids, out, M, N, K, R, d.parts}, s);
  LoraGemm g = {};
  g.x = x; g.w = w; g.pair = (const uint16_t*)b; g.planes = d.planes; g.ids = ids; g.out = out;
  g.M = M; g.cols = N; g.depth = K; g.R = R;
  return launch_gemm<DT, true>(g, q.tile, s);
}

template <int DT> int backward(const void* grad, const void* x, const void* w, const void* a, const void* b, const Ids& ids, const float* scales, const float* h, void* dx, void* da, void* db, int64_t M, int N,
                               int K, int R, char* ws, hipStream_t s) {
  const LoraPlan q = lora_plan(true, M, N, K, R, ids.L);
  if (dx || da) {
    TransposeParams t = {};
    const int tr = (R + 63) / 64, tn = (N + 63) / 64, tk = dx ? (K + 63) / 64 : 0;
    t.s[0] = {(const uint16_t*)b, (uint16_t*)(ws + q.bt), N, R, tn, tr};
    t.s[1] = {(const uint16_t*)a, (uint16_t*)(ws + q.at), R, K, tr, tk};
    t.first = ids.L * tn * tr;
    lora_transpose_kernel<<<dim3((unsigned)(t.first + ids.L * tk * tr)), dim3(256), 0, s>>>(t);
    if (int e = check_launch("lora_transpose")) return e;
    DownParams d = {};
    d.x = grad; d.a = ws + q.bt; d.scales = scales; d.ids = ids; d.M = M; d.R = R; d.depth = N; d.parts = 1;
    d.h = (float*)(ws + q.h);
    if (dx) d.planes = (uint16_t*)(ws + q.planes);
    if (int e = launch_down<DT>(d, s)) return e;
    if (dx) {
      LoraGemm g = {};
      g.x = grad; g.w = w; g.pair = (const uint16_t*)(ws + q.at); g.planes = d.planes; g.ids = ids; g.out = dx;
      g.M = M; g.cols = K; g.depth = N; g.R = R;
      if (int e = launch_gemm<DT, false>(g, q.tile, s)) return e;
    }
  }
  if (!da && !db) return 0;
  OuterParams o = {};
  o.x = x; o.g = grad; o.dh = (const float*)(ws + q.h); o.h = h; o.ids = ids; o.da = da; o.db = db;
  o.part_a = (float*)(ws + q.part_a); o.part_b = (float*)(ws + q.part_b); o.rows = (int32_t*)(ws + q.rows);
  o.M = M; o.K = K; o.N = N; o.R = R; o.L = ids.L; o.parts = q.parts;
  o.blocks_a = da ? (K + kOuterCols - 1) / kOuterCols : 0;
  const dim3 grid(o.blocks_a + (db ? (N + kOuterCols - 1) / kOuterCols : 0), ids.L, q.parts);
  const int rc = (R + 15) / 16;
  if (int e = rc <= 1 ? outer_launch<DT, 1>(o, grid, s) : rc <= 2 ? outer_launch<DT, 2>(o, grid, s) : rc <= 4 ? outer_launch<DT, 4>(o, grid, s) : outer_launch<DT, 8>(o, grid, s)) return e;
  if (q.parts == 1) return 0;
  const int64_t quads = ((da ? (int64_t)ids.L * R * K : 0) + (db ? (int64_t)ids.L * R * N : 0)) / 4;
  lora_join_kernel<DT><<<dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s>>>(o);
  return check_launch("lora_join");
}

}  // namespace

int64_t lora_workspace(int backward, int64_t M, int N, int K, int R, int L) { return lora_plan(backward != 0, M, N, K, R, L).bytes; }

int launch_lora(const void* x, const void* w, const void* a, const void* b, const void* ids, int ids_i64, const float* scales, void* out, float* h, int64_t M, int N, int K, int R, int L, int dt,
                void* ws, hipStream_t s) {
  const Ids i = {ids, ids_i64, L};
  return dt == DT_BF16 ? forward<DT_BF16>(x, w, a, b, i, scales, out, h, M, N, K, R, (char*)ws, s) : forward<DT_F16>(x, w, a, b, i, scales, out, h, M, N, K, R, (char*)ws, s);
}

int launch_lora_bwd(const void* grad, const void* x, const void* w, const void* a, const void* b, const void* ids, int ids_i64, const float* scales, const float* h, void* dx, void* da, void* db,
                    int64_t M, int N, int K, int R, int L, int dt, void* ws, hipStream_t s) {
  const Ids i = {ids, ids_i64, L};
  return dt == DT_BF16 ? backward<DT_BF16>(grad, x, w, a, b, i, scales, h, dx, da, db, M, N, K, R, (char*)ws, s)
                       : backward<DT_F16>(grad, x, w, a, b, i, scales, h, dx, da, db, M, N, K, R, (char*)ws, s);
}

}  // namespace tgg
