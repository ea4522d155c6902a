// The four-wave kernel's plain products (gemm_w4.hpp) and which launches it takes.
#include "gemm_w4.hpp"

namespace tgg {

// More than two rounds of 256x256 tiles whatever the group sizes turn out to be: at least ceil(m_total / 256) row tiles.
static bool w4_large(const GemmParams& p) {
  int grid = num_cus();
  if (p.grid_limit > 0 && p.grid_limit < grid) grid = p.grid_limit;
  return ((p.m_total + 255) / 256) * ((p.N + 127) / 128) > 4 * (int64_t)grid;
}

// Whether 256-row tiles pay depends on the group sizes, which only the device knows.  With 512 rows and more per group on
// average they do; a masked launch (counts anywhere up to its row stride), one with smaller groups or one of fewer rounds is
// enqueued together with the eight-wave kernel, and the two decide from the sizes which of them runs.  The average is that of the operand, whose rows the
// groups may own in part only (a buffer of fixed size, a padded layout of small groups).  Filled whole, launches of 200-511 rows a group take 0.95 of the
// eight-wave kernel's time by this kernel alone and 0.97 decided on the device; filled to a tenth and less 1.05-1.14 alone (15 random ones, up to
// 1.21).  Large ones of longer groups 0.93-0.98 alone, however much of them is filled (56 random ones, a fiftieth to the whole).
bool w4_decided_on_device(const GemmParams& p) {
  return p.mode == MODE_MASKED || p.m_total < 512 * (int64_t)p.G || !w4_large(p);
}

// The four-wave kernel takes large M-grouped and masked launches, and M-grouped ones of 128 rows and more per group whose likely tiles
// (every group's last one half full) cost two rounds of K = 2048 or more and would not be chosen for 128-row tiles
// (sched_wide_tiles_chosen).  Of 574 of those, drawn at random with operands in no cache, 554 were its by their sizes as well and
// took 0.91 of the eight-wave kernel's time (0.92 with a tail, 0.85-1.01; before half tiles) with the launch that returns in it; 20 were not and lost 4-6 us, 1.03.
// Large ones with a tail: 0.93.  32 groups of 1635 rows, N = 1536, K = 3208: 549 -> 487 us; 8 of 1700, N = 3296, K = 1256: 136 -> 123.
// Smaller launches stay with the eight-wave kernels, which choose narrower tiles on the device.
bool w4_supported(const GemmParams& p, int dt, int layout, bool any_size) {
  if (dt != DT_BF16 && dt != DT_F16) return false;
  if (layout != W4_NT && layout != W4_NN) return false;
  // NN: a group's B, with the rows that the tail may add, within 2 GiB
  if (layout == W4_NN && ((int64_t)p.K + 128) * p.N * 2 >= (1ll << 31)) return false;
  if (p.mode != MODE_MG && p.mode != MODE_MG_PAD && p.mode != MODE_MASKED) return false;
  // launches whose groups may be small are decided on the device (w4_decided_on_device), by a predicate that needs
  // one thread of this kernel per group; besides, with more groups than threads one of them makes the whole table, 0.12-0.2 us a group, which the eight-wave
  // kernels' 512 threads do together (367 groups of 256 rows, N = 512, K = 768: 106 us there, 171 here)
  if (w4_decided_on_device(p) && p.G > W4Cfg::THREADS) return false;
  if (p.q_fmt != 0 || p.G > kFastMaxGroups) return false;
  if ((p.N & 7) != 0 || p.K < 8 || (p.K & 7) != 0) return false;
  if ((int64_t)p.K * 2 * 256 >= (1ll << 30)) return false;
  if ((int64_t)p.N * 2 * 128 >= (1ll << 30)) return false;  // a wave's block of the output within the epilogue's 32-bit offsets, out-of-range marker included
  if (p.K < 192) return false;  // the first three slabs of a tile are whole
  // masked launches with a tail: the launch that returns costs more than this kernel gains (120 random ones from K = 776 on, counts up to 0.05-0.4 of the
  // slots 1.035 of the eight-wave kernels' time alone, up to 0.7 and all of them 0.995)
  if (p.mode == MODE_MASKED && needs_tail(p, layout)) return false;
  if (any_size) return true;
  // a short K spends more on the slab that makes the tail's number even than the eight-wave kernel loses (4 groups of 13000 rows, N = 3096,
  // K = 512, [K, N]: 195 us there, 202 here; 16 of 1200, N = 3072, K = 536: 79 and 81)
  if (needs_tail(p, layout) && p.K < 768) return false;
  // and so does, up to K = 1024, the launch that returns where only N is cut, whose slabs the eight-wave kernel has whole as well (17 random ones 1.014 of
  // its time alone, up to 1.07; K = 1152-1500 0.995; K no multiple of 128: 0.98)
  if (layout == W4_NN && p.K % 128 == 0 && p.K <= 1024 && needs_tail(p, layout) && w4_decided_on_device(p)) return false;
  if (w4_large(p)) return true;
  if (p.mode == MODE_MASKED || p.m_total < 128 * (int64_t)p.G) return false;
  int grid = num_cus();
  if (p.grid_limit > 0 && p.grid_limit < grid) grid = p.grid_limit;
  const int64_t tiles_n = (p.N + 255) / 256;
  const int64_t full_2 = (2 * ((p.m_total + 255) / 256) + p.G) * tiles_n, half_2 = (2 * ((p.m_total + 127) / 128) + p.G) * tiles_n;  // twice the likely tiles
  const int64_t rounds_full = (full_2 + 2 * grid - 1) / (2 * grid), rounds_half = (half_2 + 2 * grid - 1) / (2 * grid);
  // (Fewer rounds are no safe choice: launches of 256 rows a group and more take 0.91 of the eight-wave kernel's time from 1.15 rounds of likely tiles on
  // and from 0.7 to 0.9 of one where the groups fill the operand, but 1.03 with half of it filled, up to 1.24, and 1.1 with a tenth, up to 1.29: its narrower
  // tiles fit what is left.  Decided on the device they would pay 4 us for 30-100.)
  return full_2 * p.K >= 2 * 4096 * (int64_t)grid && rounds_half * 3 > rounds_full * 4;
}

template <int DT, int LAYOUT>
int launch_w4_layout(const GemmParams& p, hipStream_t s) {
  return needs_tail(p, LAYOUT) ? launch_w4<DT, LAYOUT, true>(p, s) : launch_w4<DT, LAYOUT, false>(p, s);
}

int launch_w4_16bit(const GemmParams& p, int dt, int layout, hipStream_t s) {
  if (layout == W4_NT) return dt == DT_BF16 ? launch_w4_layout<DT_BF16, W4_NT>(p, s) : launch_w4_layout<DT_F16, W4_NT>(p, s);
  return dt == DT_BF16 ? launch_w4_layout<DT_BF16, W4_NN>(p, s) : launch_w4_layout<DT_F16, W4_NN>(p, s);
}

}  // namespace tgg
