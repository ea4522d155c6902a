// Top-k router of a mixture-of-experts layer: the k largest of a token's E logits, their probabilities, and the gradient.
//
// Order of a row: larger logit first, equal ones (and -0 and +0) by index, NaN above every number.  A logit of -inf is a masked expert and never
// chosen: what is left of the k entries then has index -1 (an assignment that the token movement drops) and probability 0.
//   softmax   p_e = exp(l_e - max) / sum over all experts      sigmoid   p_e = 1 / (1 + exp(-l_e))
//   renormalised: q_k = p_k / sum of the chosen p.  For softmax that is the softmax over the chosen logits, for sigmoid the softmax over the
//   chosen log sigma(l): no quotient of vanishing numbers.
// Everything is fp32.
//
// LPT lanes work on a token, each on VPL neighbouring logits.  A lane's logits become integer keys that sort like them (for 16-bit logits with the
// index in the lower half: one 32-bit key says which, and no two are equal; 64 bits for fp32), sorted in registers once by a network; the k
// largest of the row are then k rounds of a maximum over the lanes' heads (moves between lanes inside the vector unit) after which the one lane that
// owns the maximum pops its list.  Lane t of a token keeps round t's result, so that probabilities and stores are one step for all of them.
#include "common.hpp"
#include "launch.hpp"

namespace tgg {

namespace {

enum : int { RT_BF16 = 0, RT_F16 = 1, RT_F32 = 2 };
enum : int { SCORE_SOFTMAX = 0, SCORE_SIGMOID = 1 };
constexpr int kRouterThreads = 256;

// Maximum / sum over the LPT lanes of a token, in every one of them.
template <int CTRL> TGG_DEV uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false); }
template <int LPT, class F> TGG_DEV uint32_t over_lanes(uint32_t v, const F& f) {
  v = f(v, dpp<0xB1>(v));   // quad_perm [1,0,3,2]
  v = f(v, dpp<0x4E>(v));   // quad_perm [2,3,0,1]
  v = f(v, dpp<0x141>(v));  // row_half_mirror: the other four of eight
  v = f(v, dpp<0x140>(v));  // row_mirror: the other eight of sixteen
  if (LPT > 16) v = f(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  if (LPT > 32) v = f(v, (uint32_t)__shfl_xor((int)v, 32, 64));
  return v;
}
template <int LPT> TGG_DEV uint32_t max_over(uint32_t v) { return over_lanes<LPT>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); }
template <int LPT> TGG_DEV uint64_t max_over(uint64_t v) {
  const uint32_t hi = max_over<LPT>((uint32_t)(v >> 32));
  const uint32_t lo = max_over<LPT>((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return ((uint64_t)hi << 32) | lo;
}
template <int LPT> TGG_DEV float sum_over(float v) {
  return __builtin_bit_cast(float, over_lanes<LPT>(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b)); }));
}

// A logit as it was read, in the upper bits of a word.
template <int RT> TGG_DEV float logit_value(uint32_t u) {
  if (RT == RT_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
  return __builtin_bit_cast(float, u);
}
// Its place in the order, as an unsigned integer above 0 (16-bit logits fill the upper 16 bits): the signed value of sign and magnitude, which is the same for
// -0 and +0, with the sign bit turned; NaN is the first magnitude behind infinity.
template <int RT> TGG_DEV uint32_t logit_order(uint32_t u) {
  constexpr uint32_t inf = RT == RT_F16 ? 0x7c000000u : 0x7f800000u, step = RT == RT_F32 ? 1u : 0x10000u;
  const uint32_t mag = u & 0x7fffffffu, sign = mag > inf ? 0u : (uint32_t)((int)u >> 31);
  return (((mag > inf ? inf + step : mag) ^ sign) - sign) ^ 0x80000000u;
}
// The same for two 16-bit logits at once, in packed 16-bit instructions (five a logit in place of nine).
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
typedef __attribute__((ext_vector_type(2))) short s16x2_t;
template <int RT> TGG_DEV uint32_t logit_order_pair(uint32_t w) {
  constexpr unsigned short inf = RT == RT_F16 ? 0x7c00 : 0x7f80;
  const u16x2_t infs = {inf, inf}, behind = {inf + 1, inf + 1}, one = {1, 1};
  const u16x2_t mag = __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu);
  const u16x2_t nan = (u16x2_t)0 - __builtin_elementwise_min(__builtin_elementwise_sub_sat(mag, infs), one);  // all ones where NaN
  const u16x2_t sign = __builtin_bit_cast(u16x2_t, (s16x2_t)(__builtin_bit_cast(s16x2_t, w) >> 15)) & ~nan;
  return __builtin_bit_cast(uint32_t, (u16x2_t)((__builtin_elementwise_min(mag, behind) ^ sign) - sign)) ^ 0x80008000u;
}
template <int RT> TGG_DEV uint32_t logit_of_order(uint32_t key) {
  const uint32_t value = key ^ 0x80000000u, sign = (uint32_t)((int)value >> 31);
  return ((value ^ sign) - sign) | (sign & 0x80000000u);
}

template <int RT> struct KeyOf { typedef uint32_t type; };
template <> struct KeyOf<RT_F32> { typedef uint64_t type; };
template <int RT> TGG_DEV uint32_t key_logit(typename KeyOf<RT>::type key) {
  if constexpr (RT == RT_F32) return logit_of_order<RT>((uint32_t)(key >> 32));
  else return logit_of_order<RT>(key & 0xffff0000u);
}
template <int RT> TGG_DEV int key_index(typename KeyOf<RT>::type key) {
  if constexpr (RT == RT_F32) return (int)(0xffffffffu - (uint32_t)key);
  else return (int)(0xffffu - (key & 0xffffu));
}

// Which logits a lane holds.  VEC: VPL neighbouring ones, read 16 bytes at a time (rows begin on 16 bytes and hold whole 16-byte pieces); otherwise
// every LPT-th one, so that a read instruction covers neighbouring logits (161 fp32 logits a row, 16383 rows: 22 -> 11.3 us forward, 14.3 -> 8.1 backward).
template <int LPT, int VPL, bool VEC> TGG_DEV int expert_of(int lane, int i) { return VEC ? lane * VPL + i : i * LPT + lane; }

// A lane's logits, in the upper bits; those beyond E are -inf.
template <int RT, int LPT, int VPL, bool VEC> TGG_DEV void load_logits(const void* row, int lane, int E, uint32_t (&u)[VPL]) {
  constexpr uint32_t masked = RT == RT_F16 ? 0xfc000000u : 0xff800000u;
  constexpr int ES = RT == RT_F32 ? 4 : 2, PER = 16 / ES;
  if constexpr (VEC) {
    static_assert(VPL % PER == 0, "whole 16-byte pieces");
#pragma unroll
    for (int c = 0; c < VPL / PER; ++c) {
      const int e = lane * VPL + c * PER;
      const uint32_t none = RT == RT_F32 ? masked : masked | (masked >> 16);
      uint4 w = {none, none, none, none};
      if (e < E) w = *(const uint4*)((const char*)row + (int64_t)e * ES);
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (RT == RT_F32) u[c * 4 + i] = x[i];
        else {
          u[c * 8 + 2 * i] = x[i] << 16;
          u[c * 8 + 2 * i + 1] = x[i] & 0xffff0000u;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = expert_of<LPT, VPL, VEC>(lane, i);
      u[i] = masked;
      if (e < E) u[i] = RT == RT_F32 ? ((const uint32_t*)row)[e] : (uint32_t)((const uint16_t*)row)[e] << 16;
    }
  }
}

// Descending order by a merge network of comparisons between fixed places.
template <int N, class K> TGG_DEV void sort_descending(K (&key)[N]) {
#pragma unroll
  for (int p = 1; p < N; p <<= 1)
#pragma unroll
    for (int q = p; q >= 1; q >>= 1)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const K a = key[i + j], b = key[i + j + q];
            key[i + j] = a > b ? a : b;
            key[i + j + q] = a > b ? b : a;
          }
}

TGG_DEV float log_sigmoid(float x) { return fminf(x, 0.f) - log1pf(expf(-fabsf(x))); }

// The row's largest logit for the exponentials; of a row without experts 0, so that every exp(l - max) is 0 there.
TGG_DEV float shift_of(float top) { return top == -__builtin_inff() ? 0.f : top; }

// m ? b : a, m all ones or zero.  (Written as a choice, the compiler makes the list below a choice of places: 80 instructions a round in place of 7.)
TGG_DEV uint32_t choose(uint32_t a, uint32_t b, uint32_t m) { return (b & m) | (a & ~m); }
TGG_DEV uint64_t choose(uint64_t a, uint64_t b, uint32_t m) {
  return ((uint64_t)choose((uint32_t)(a >> 32), (uint32_t)(b >> 32), m) << 32) | choose((uint32_t)a, (uint32_t)b, m);
}

template <int RT, int LPT, int VPL, bool VEC>
__global__ __launch_bounds__(kRouterThreads) void router_fwd_kernel(const char* __restrict__ logits, int64_t row_bytes, int64_t tokens, int E, int k,
                                                                    int scoring, int renorm, float* __restrict__ probs, int32_t* __restrict__ indices) {
  typedef typename KeyOf<RT>::type Key;
  const int lane = threadIdx.x % LPT;
  const int64_t token = (int64_t)blockIdx.x * (kRouterThreads / LPT) + threadIdx.x / LPT;
  const bool live = token < tokens;
  uint32_t u[VPL];
  load_logits<RT, LPT, VPL, VEC>(logits + token * row_bytes, lane, live ? E : 0, u);
  // (places beyond E hold -inf behind every real one: they are never chosen)
  Key key[VPL];
#pragma unroll
  for (int i = 0; i < VPL; i += 2) {
    const uint32_t e = (uint32_t)expert_of<LPT, VPL, VEC>(lane, i), f = (uint32_t)expert_of<LPT, VPL, VEC>(lane, i + 1);
    if constexpr (RT == RT_F32) {
      key[i] = ((uint64_t)logit_order<RT>(u[i]) << 32) | (0xffffffffu - e);
      key[i + 1] = ((uint64_t)logit_order<RT>(u[i + 1]) << 32) | (0xffffffffu - f);
    } else {
      const uint32_t both = logit_order_pair<RT>((u[i] >> 16) | u[i + 1]);
      key[i] = (both << 16) | (0xffffu - e);
      key[i + 1] = (both & 0xffff0000u) | (0xffffu - f);
    }
  }
  sort_descending(key);
  Key mine = 0;  // lane t: the t-th of the row
  Key first = 0;
  for (int t = 0; t < k; ++t) {
    const Key top = max_over<LPT>(key[0]);
    if (t == 0) first = top;
    if (lane == t) mine = top;
    const uint32_t own = key[0] == top ? 0xffffffffu : 0u;
#pragma unroll
    for (int i = 0; i + 1 < VPL; ++i) key[i] = choose(key[i], key[i + 1], own);
    key[VPL - 1] = choose(key[VPL - 1], Key(0), own);
  }
  const float x = logit_value<RT>(key_logit<RT>(mine));
  const bool chosen = lane < k && !(x == -__builtin_inff());
  const float top = shift_of(logit_value<RT>(key_logit<RT>(first)));
  float prob;
  if (scoring == SCORE_SOFTMAX) {
    const float e = chosen ? expf(x - top) : 0.f;
    float sum;
    if (renorm) {
      sum = sum_over<LPT>(e);
    } else {
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) part += expf(logit_value<RT>(u[i]) - top);  // those beyond E are -inf
      sum = sum_over<LPT>(part);
    }
    prob = e / sum;
  } else if (renorm) {  // log sigma rises with the logit: the first is the largest
    const float e = chosen ? expf(log_sigmoid(x) - log_sigmoid(top)) : 0.f;
    prob = e / sum_over<LPT>(e);
  } else {
    prob = 1.f / (1.f + expf(-x));
  }
  if (live && lane < k) {
    probs[token * k + lane] = chosen ? prob : 0.f;
    indices[token * k + lane] = chosen ? key_index<RT>(mine) : -1;
  }
}

template <int RT> TGG_DEV void store_logit(char* row, int e, float v) {
  if constexpr (RT == RT_F32) ((float*)row)[e] = v;
  else ((uint16_t*)row)[e] = Out16<RT>::cvt(v);
}

// Gradient of the logits.  What the chosen experts get, lane t of a token computes from round t's probability; through a row of LDS it reaches the lane
// that writes that expert's logit.
template <int RT, int LPT, int VPL, bool VEC>
__global__ __launch_bounds__(kRouterThreads) void router_bwd_kernel(const char* __restrict__ logits, int64_t row_bytes, const float* __restrict__ probs,
                                                                    const int32_t* __restrict__ indices, const float* __restrict__ grad, int64_t tokens, int E, int k,
                                                                    int scoring, int renorm, char* __restrict__ dlogits) {
  __shared__ __attribute__((aligned(16))) float part[kRouterThreads / LPT][LPT * VPL];
  constexpr int ES = RT == RT_F32 ? 4 : 2;
  const int lane = threadIdx.x % LPT, slot = threadIdx.x / LPT;
  const int64_t token = (int64_t)blockIdx.x * (kRouterThreads / LPT) + slot;
  const bool live = token < tokens;
  const char* const row = logits + token * row_bytes;
  int at = -1;
  float p = 0.f, d = 0.f, x = 0.f;
  if (live && lane < k) {
    at = indices[token * k + lane];
    if (at >= 0 && at < E) {
      p = probs[token * k + lane];
      d = grad[token * k + lane];
      if (scoring == SCORE_SIGMOID) x = RT == RT_F32 ? ((const float*)row)[at] : logit_value<RT>((uint32_t)((const uint16_t*)row)[at] << 16);
    } else {
      at = -1;
    }
  }
  const float pd = p * d, all = sum_over<LPT>(pd);
  float v = renorm ? p * (d - all) : pd;
  if (scoring == SCORE_SIGMOID) v *= 1.f / (1.f + expf(x));
  float* const mine = part[slot];
#pragma unroll
  for (int i = 0; i < VPL; ++i) mine[i * LPT + lane] = 0.f;
  if (at >= 0) mine[VEC ? at % VPL * LPT + at / VPL : at] = v;  // where the lane that holds this logit reads below
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // a token's lanes are of one wave: LDS serves them in order
  float g[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) g[i] = mine[i * LPT + lane];
  if (scoring == SCORE_SOFTMAX && !renorm) {  // every expert's probability took part in the sum
    uint32_t u[VPL];
    load_logits<RT, LPT, VPL, VEC>(row, lane, live ? E : 0, u);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const uint32_t o = logit_order<RT>(u[i]);
      most = o > most ? o : most;
    }
    const float top = shift_of(logit_value<RT>(logit_of_order<RT>(max_over<LPT>(most))));
    float e[VPL], sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum += e[i] = expf(logit_value<RT>(u[i]) - top);
    sum = sum_over<LPT>(sum);
    const float scale = sum > 0.f || sum != sum ? all / sum : 0.f;  // a row without experts has no gradient
#pragma unroll
    for (int i = 0; i < VPL; ++i) g[i] -= e[i] * scale;
  }
  if (!live) return;
  char* const out = dlogits + token * (int64_t)E * ES;
  if constexpr (VEC) {
    constexpr int PER = 16 / ES;
#pragma unroll
    for (int c = 0; c < VPL / PER; ++c) {
      const int e = lane * VPL + c * PER;
      if (e >= E) continue;
      if constexpr (RT == RT_F32) {
        *(float4*)(out + (int64_t)e * 4) = make_float4(g[4 * c], g[4 * c + 1], g[4 * c + 2], g[4 * c + 3]);
      } else {
        uint4 w;
        w.x = pack2<RT>(g[8 * c], g[8 * c + 1]);
        w.y = pack2<RT>(g[8 * c + 2], g[8 * c + 3]);
        w.z = pack2<RT>(g[8 * c + 4], g[8 * c + 5]);
        w.w = pack2<RT>(g[8 * c + 6], g[8 * c + 7]);
        *(uint4*)(out + (int64_t)e * 2) = w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = expert_of<LPT, VPL, VEC>(lane, i);
      if (e < E) store_logit<RT>(out, e, g[i]);
    }
  }
}

struct RouterArgs {
  const char* logits;
  int64_t row_bytes, tokens;
  int E, k, scoring, renorm;
  float* probs;         // forward: written; backward: read
  int32_t* indices;
  const float* grad;    // backward
  char* dlogits;
};

template <int RT, int LPT, int VPL, bool VEC, bool BWD>
int launch_router_kernel(const RouterArgs& a, hipStream_t s) {
  constexpr int PER = kRouterThreads / LPT;
  const int64_t blocks = (a.tokens + PER - 1) / PER;
  if (blocks > 0x7fffffff) return set_error("router over %lld tokens: too many", (long long)a.tokens);
  if constexpr (BWD) {
    hipLaunchKernelGGL((router_bwd_kernel<RT, LPT, VPL, VEC>), dim3((uint32_t)blocks), dim3(kRouterThreads), 0, s, a.logits, a.row_bytes, a.probs, a.indices, a.grad, a.tokens,
                       a.E, a.k, a.scoring, a.renorm, a.dlogits);
  } else {
    hipLaunchKernelGGL((router_fwd_kernel<RT, LPT, VPL, VEC>), dim3((uint32_t)blocks), dim3(kRouterThreads), 0, s, a.logits, a.row_bytes, a.tokens, a.E, a.k, a.scoring,
                       a.renorm, a.probs, a.indices);
  }
  return check_launch("moe_router");
}

template <int RT, int LPT, int VPL, bool BWD>
int launch_router_as(const RouterArgs& a, hipStream_t s) {
  constexpr int ES = RT == RT_F32 ? 4 : 2;
  if constexpr (VPL * ES >= 16) {
    const bool rows = ((uintptr_t)a.logits & 15) == 0 && (a.row_bytes & 15) == 0 && (a.E * ES & 15) == 0;
    if (rows && (!BWD || ((uintptr_t)a.dlogits & 15) == 0)) return launch_router_kernel<RT, LPT, VPL, true, BWD>(a, s);
  }
  return launch_router_kernel<RT, LPT, VPL, false, BWD>(a, s);
}

// As few lanes a token as its experts (eight logits a lane; two in rows of at most 32 experts, sixteen in rows of more than 512) and its k results need.
template <int RT, bool BWD>
int launch_router_type(const RouterArgs& a, hipStream_t s) {
  if (a.E <= 32 && a.k <= 16) return launch_router_as<RT, 16, 2, BWD>(a, s);
  if (a.E <= 128 && a.k <= 16) return launch_router_as<RT, 16, 8, BWD>(a, s);
  if (a.E <= 256 && a.k <= 32) return launch_router_as<RT, 32, 8, BWD>(a, s);
  if (a.E <= 512) return launch_router_as<RT, 64, 8, BWD>(a, s);
  return launch_router_as<RT, 64, 16, BWD>(a, s);
}

template <bool BWD>
int launch_router(const RouterArgs& a, int dt, hipStream_t s) {
  if (dt == RT_BF16) return launch_router_type<RT_BF16, BWD>(a, s);
  if (dt == RT_F16) return launch_router_type<RT_F16, BWD>(a, s);
  return launch_router_type<RT_F32, BWD>(a, s);
}

}  // namespace

int launch_moe_router(const void* logits, int64_t row_bytes, int64_t tokens, int E, int k, int scoring, int renorm, int dt, float* probs, int32_t* indices, hipStream_t s) {
  return launch_router<false>(RouterArgs{(const char*)logits, row_bytes, tokens, E, k, scoring, renorm, probs, indices, nullptr, nullptr}, dt, s);
}
int launch_moe_router_bwd(const void* logits, int64_t row_bytes, const float* probs, const int32_t* indices, const float* grad, int64_t tokens, int E, int k, int scoring,
                          int renorm, int dt, void* dlogits, hipStream_t s) {
  return launch_router<true>(RouterArgs{(const char*)logits, row_bytes, tokens, E, k, scoring, renorm, (float*)probs, (int32_t*)indices, grad, (char*)dlogits}, dt, s);
}

}  // namespace tgg
