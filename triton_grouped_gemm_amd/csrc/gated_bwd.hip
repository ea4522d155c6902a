// Backward pass of the gated feed-forward block between its two products: from the gradient d of out = act(gate) * up and the saved projections
// h = [gate | up], both [rows, F] halves of a row of 2 F values,
//   d gate = d up act'(gate),   d up = d act(gate)
// as one matrix dh [rows, 2 F], which the grouped products for the activations' and the weights' gradients then take.
//
// h is fp32: stored in 16 bits its rounding would be a third one in the gradients, beside dh's and their own (0.0030 of their norm in place of 0.0024 in
// bfloat16).  One pass: 10 F bytes of a row are read and 4 F written, 16 bytes a lane and access; fp32 between, one rounding.  Memory-bound.
#include "gate.hpp"
#include "launch.hpp"

namespace tgg {

namespace {

constexpr int kThreads = 256, kPer = 2;  // vectors (8 values) of a thread, loaded together before any is used

template <int DT> TGG_DEV float lo16(uint32_t w) {
  if (DT == DT_BF16) return __builtin_bit_cast(float, w << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
}
template <int DT> TGG_DEV float hi16(uint32_t w) {
  if (DT == DT_BF16) return __builtin_bit_cast(float, w & 0xffff0000u);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
}

// A workgroup takes kThreads * kPer consecutive vectors of the [rows, F / 8] matrix of vectors.
template <int DT, int ACT>
__global__ __launch_bounds__(kThreads) void gated_bwd_kernel(const i32x4_t* __restrict__ dout, const f32x4_t* __restrict__ h, i32x4_t* __restrict__ dh,
                                                             int64_t vectors, int per_row) {
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kPer);
  const int64_t row0 = first / per_row;  // the same in the whole workgroup
  const uint32_t col0 = (uint32_t)(first - row0 * per_row);
  i32x4_t d[kPer];
  f32x4_t g[kPer][2], u[kPer][2];
  int64_t at[kPer];
  bool live[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t off = threadIdx.x + i * kThreads, col = col0 + off, row = col / (uint32_t)per_row;
    live[i] = first + off < vectors;
    at[i] = (row0 + row) * (2 * (int64_t)per_row) + (col - row * (uint32_t)per_row);  // of the gate's vector in dh; two of h
    if (live[i]) {
      d[i] = __builtin_nontemporal_load(dout + first + off);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        g[i][q] = __builtin_nontemporal_load(h + 2 * at[i] + q);
        u[i][q] = __builtin_nontemporal_load(h + 2 * (at[i] + per_row) + q);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (!live[i]) continue;
    i32x4_t dg, du;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float a0, a1, s0, s1;
      gate_act_slope<ACT>(g[i][w / 2][w % 2 * 2], a0, s0);
      gate_act_slope<ACT>(g[i][w / 2][w % 2 * 2 + 1], a1, s1);
      const float d0 = lo16<DT>(d[i][w]), d1 = hi16<DT>(d[i][w]);
      dg[w] = (int)pack2<DT>(d0 * u[i][w / 2][w % 2 * 2] * s0, d1 * u[i][w / 2][w % 2 * 2 + 1] * s1);
      du[w] = (int)pack2<DT>(d0 * a0, d1 * a1);
    }
    dh[at[i]] = dg;
    dh[at[i] + per_row] = du;
  }
}

template <int DT, int ACT>
int launch_as(const void* dout, const void* h, void* dh, int64_t rows, int F, hipStream_t s) {
  const int64_t vectors = rows * (F / 8), blocks = (vectors + kThreads * kPer - 1) / (kThreads * kPer);
  if (blocks > 0x7fffffff) return set_error("gated backward pass over %lld rows of %d outputs: too many", (long long)rows, F);
  hipLaunchKernelGGL((gated_bwd_kernel<DT, ACT>), dim3((uint32_t)blocks), dim3(kThreads), 0, s, (const i32x4_t*)dout, (const f32x4_t*)h, (i32x4_t*)dh, vectors, F / 8);
  return check_launch("gated_bwd");
}

}  // namespace

int launch_gated_bwd(const void* dout, const void* h, void* dh, int64_t rows, int F, int act, int dt, hipStream_t s) {
  if (dt == DT_BF16) return act == GATE_SILU ? launch_as<DT_BF16, GATE_SILU>(dout, h, dh, rows, F, s) : launch_as<DT_BF16, GATE_GELU_TANH>(dout, h, dh, rows, F, s);
  return act == GATE_SILU ? launch_as<DT_F16, GATE_SILU>(dout, h, dh, rows, F, s) : launch_as<DT_F16, GATE_GELU_TANH>(dout, h, dh, rows, F, s);
}

}  // namespace tgg
