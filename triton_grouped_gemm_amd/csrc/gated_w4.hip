// The four-wave kernel's gated feed-forward blocks (gemm_w4.hpp), apart from the plain products because they take as long to compile.
#include "gemm_w4.hpp"

namespace tgg {

bool w4_supported(const GemmParams& p, int dt, int layout, bool any_size);

// The gated block: as the plain product (of N = 2 F columns) without a tail, with one window over a group's gate and up columns and projections within
// the epilogue's 32-bit offsets.
bool w4_gated_supported(const GemmParams& p, int dt, int layout, bool any_size) {
  return (p.N & 15) == 0 && (int64_t)p.N * p.K * 2 < (1ll << 30) && (int64_t)p.N * 4 * 128 < (1ll << 30) && !needs_tail(p, layout) && w4_supported(p, dt, layout, any_size);
}

template <int DT, int LAYOUT>
static int launch_w4_gated_as(const GemmParams& p, hipStream_t s) {
  if (p.act == GATE_SILU) return p.H ? launch_w4<DT, LAYOUT, false, GATE_SILU + 1, true>(p, s) : launch_w4<DT, LAYOUT, false, GATE_SILU + 1, false>(p, s);
  return p.H ? launch_w4<DT, LAYOUT, false, GATE_GELU_TANH + 1, true>(p, s) : launch_w4<DT, LAYOUT, false, GATE_GELU_TANH + 1, false>(p, s);
}

int launch_w4_gated(const GemmParams& p, int dt, int layout, hipStream_t s) {
  if (layout == W4_NT) return dt == DT_BF16 ? launch_w4_gated_as<DT_BF16, W4_NT>(p, s) : launch_w4_gated_as<DT_F16, W4_NT>(p, s);
  return dt == DT_BF16 ? launch_w4_gated_as<DT_BF16, W4_NN>(p, s) : launch_w4_gated_as<DT_F16, W4_NN>(p, s);
}

}  // namespace tgg
