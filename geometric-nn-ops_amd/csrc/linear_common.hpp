// What the linear layer's kernels share: activations and their slopes, the arguments, and the epilogue of 8
// consecutive outputs of a row.
#pragma once

#include "gnn_common.hpp"
#include "gnn_internal.hpp"

namespace gnn {
namespace lin {

typedef __attribute__((address_space(3))) void lds_void_t;

// Source of the chunks that a DMA fills with zeros
__device__ __attribute__((aligned(16))) const uint32_t zero_chunk[4] = {0u, 0u, 0u, 0u};

// ---- activations ------------------------------------------------------------------------
// 16-bit results: exp2 and rcp of the hardware (1 ulp each) and polynomials fitted to the normal distribution (in
// 64 bits, weighted least squares iterated to an even error). With m = |z|, Phi(-m) = 2^P(m), off by at most 2e-7 / m
// and by 1.5e-4 of itself to m = 7 (1.5 % at 8, half at 10, where gelu is -5e-15 and -8e-23 and only bf16 holds it);
// the slope's part Phi(-m) - m phi(m) = exp(-m^2 / 2) S(m), off by at most 4e-7 and from m = 2 to 4 by 3.2e-4 of
// itself. Beyond, S alone would be 15 % off at 5.5 and a cubic of its own takes over, 2.5e-4 off to the end of bf16's
// range (the slopes and both gradients of 147456 x 128 -> 512, bf16: 164 us, with S alone 158). Half a step of fp16
// is 2.4e-4 to 4.9e-4 of a value, of bf16 eight times that. Both vanish beyond m = 16. The vector unit's time, which the
// products and the stores hide only in part, is what the wide layers with an activation pay: 147456 x 128 -> 512
// in bf16 takes 40 us without one, 54 with silu, 77 with gelu (90 with Phi by one exponential and one reciprocal,
// Abramowitz and Stegun 7.1.26; dz and dx in one pass 122, with silu 101). fp32: the library's functions and full
// divisions.
template <bool F32>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (F32) return 1.0f / (1.0f + expf(-z));
  return __builtin_amdgcn_rcpf(1.0f + fast_exp2(-1.4426950408889634f * z));
}

template <bool F32>
__device__ __forceinline__ float gelu(float z) {
  if constexpr (F32) return z * (0.5f * erfcf(-0.7071067811865476f * z));
  const float m = __builtin_elementwise_minimum(fabsf(z), 16.f);  // NaN stays
  constexpr float P[] = {-0.999999166f, -1.15114188f, -0.45895192f, -0.0531633832f, 0.00789580215f,
                         -0.000686984218f, 1.0452366e-05f, 3.52678785e-06f, -2.20578514e-07f};
  float p = P[8];
#pragma unroll
  for (int k = 7; k >= 0; --k) p = fmaf(p, m, P[k]);
  return fmaf(-m, fast_exp2(p), fmaxf(z, 0.f));
}
template <bool F32>
__device__ __forceinline__ float gelu_slope(float z) {
  if constexpr (F32)
    return 0.5f * erfcf(-0.7071067811865476f * z) + z * 0.3989422804014327f * expf(-0.5f * z * z);
  const float m = __builtin_elementwise_minimum(fabsf(z), 16.f);  // NaN stays
  constexpr float S[] = {0.499999732f, -0.797864914f, 0.249752283f, -0.131772861f, 0.0594967604f,
                         -0.0222308412f, 0.00638278481f, -0.0012711552f, 0.000151940651f, -8.06298158e-06f};
  float s = S[9];
#pragma unroll
  for (int k = 8; k >= 0; --k) s = fmaf(s, m, S[k]);
  const float far = fmaf(fmaf(fmaf(-0.000113982198f, m, 0.00370404311f), m, -0.442016602f), m, 0.214368284f);
  s = (m > 4.f ? far : s) * fast_exp2(-0.7213475204444817f * m * m);
  return z < 0.f ? s : 1.0f - s;
}

template <bool F32, int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == GNN_ACT_RELU) return __builtin_elementwise_maximum(z, 0.f);  // NaN stays
  if constexpr (ACT == GNN_ACT_GELU) return gelu<F32>(z);
  if constexpr (ACT == GNN_ACT_SILU) return z * sigmoid<F32>(z);
  if constexpr (ACT == GNN_ACT_SIGMOID) return sigmoid<F32>(z);
  return z;
}
template <bool F32, int ACT>
__device__ __forceinline__ float slope(float z) {
  if constexpr (ACT == GNN_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
  if constexpr (ACT == GNN_ACT_GELU) return gelu_slope<F32>(z);
  if constexpr (ACT == GNN_ACT_SILU) {
    const float s = sigmoid<F32>(z);
    return s * (1.0f + z * (1.0f - s));
  }
  if constexpr (ACT == GNN_ACT_SIGMOID) {
    // e / (1 + e)^2 with e = exp(-|z|), which is even: s (1 - s) has no digits left where s rounds to 1
    const float e = F32 ? expf(-fabsf(z)) : fast_exp2(-1.4426950408889634f * fabsf(z));
    const float r = F32 ? 1.0f / (1.0f + e) : __builtin_amdgcn_rcpf(1.0f + e);
    return e * r * r;
  }
  return 1.f;
}

// A vector of values at once: one uniform branch (16 of them, one an element, took longer than the products)
template <bool F32, int ACT, typename V>
__device__ __forceinline__ void activate_all(V& z) {
#pragma unroll
  for (int e = 0; e < (int)(sizeof(V) / sizeof(float)); ++e) z[e] = activate<F32, ACT>(z[e]);
}
template <bool F32, typename V>
__device__ __forceinline__ void activate_all(int act, V& z) {
  switch (act) {
    case GNN_ACT_RELU: activate_all<F32, GNN_ACT_RELU>(z); break;
    case GNN_ACT_GELU: activate_all<F32, GNN_ACT_GELU>(z); break;
    case GNN_ACT_SILU: activate_all<F32, GNN_ACT_SILU>(z); break;
    case GNN_ACT_SIGMOID: activate_all<F32, GNN_ACT_SIGMOID>(z); break;
    default: break;
  }
}
template <bool F32, int ACT, typename V>
__device__ __forceinline__ void slope_all(V& z) {
#pragma unroll
  for (int e = 0; e < (int)(sizeof(V) / sizeof(float)); ++e) z[e] = slope<F32, ACT>(z[e]);
}
template <bool F32, typename V>
__device__ __forceinline__ void slope_all(int act, V& z) {
  switch (act) {
    case GNN_ACT_RELU: slope_all<F32, GNN_ACT_RELU>(z); break;
    case GNN_ACT_GELU: slope_all<F32, GNN_ACT_GELU>(z); break;
    case GNN_ACT_SILU: slope_all<F32, GNN_ACT_SILU>(z); break;
    case GNN_ACT_SIGMOID: slope_all<F32, GNN_ACT_SIGMOID>(z); break;
    default: slope_all<F32, GNN_ACT_NONE>(z); break;
  }
}

// ---- arguments and epilogue ---------------------------------------------------------------
struct LinArgs {
  const void* x;
  const void* w;
  const void* bias;
  const void* side;  // residual, or dy
  void* out;
  int64_t M;
  int64_t x_ld, w_ld, side_ld, out_ld;
  int I, O;      // contraction (a multiple of 8; 4 in fp32), outputs
  int out_cols;  // columns written, zeros from O on
  int act;
  bool dz;  // out = side * act'(z) instead of act(z) + side
  void* dx;  // with dz, or NULL: out W
  int64_t dx_ld;
};

// 8 consecutive elements at any element's address, the first `left` of them
template <typename T>
__device__ __forceinline__ f32x8 load8_any(const T* p, int left) {
  typedef typename TypeOps<T>::V8 V8;
  typedef V8 VU __attribute__((aligned(sizeof(T))));
  if (left >= 8) {
    const V8 v = *(const __attribute__((address_space(1))) VU*)p;
    return TypeOps<T>::to_f32(v);
  }
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < left ? (float)p[e] : 0.f;
  return v;
}
template <typename T>
__device__ __forceinline__ void store8_any(T* p, const f32x8& v, int left) {
  typedef typename TypeOps<T>::V8 V8;
  typedef V8 VU __attribute__((aligned(sizeof(T))));
  const V8 o = TypeOps<T>::from_f32(v);
  if (left >= 8) {
    *(__attribute__((address_space(1))) VU*)p = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) p[e] = o[e];
}

// The 32x32 accumulator has rows 8 q + 4 g + i (q = r / 4, i = r % 4) in a lane. Tile row r of the transposed
// product takes output tile_output(r), so that a lane's 8 registers 8 t .. 8 t + 7 are the 8 consecutive
// outputs 16 t + 8 g + (0 .. 7), and tile_row is the other way round. (Exchanging the halves of natural tiles
// with v_permlane32_swap took 8 more instructions a tile.)
__host__ __device__ constexpr int tile_output(int r) { return (r & 16) | (r & 4) << 1 | (r & 8) >> 1 | (r & 3); }
__host__ __device__ constexpr int tile_row(int n) { return (n & 16) | (n & 8) >> 1 | (n & 4) << 1 | (n & 3); }
__device__ __forceinline__ f32x8 outputs8(const f32x16& acc, int t) {
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = acc[8 * t + e];
  return v;
}

// Bias, activation and residual (or the slope of dy) on 8 outputs n .. n + 7 of row m, and their store
template <typename T>
__device__ __forceinline__ void finish8(const LinArgs& a, const f32x8& z0, const f32x8& b, int64_t m, int n) {
  constexpr bool F32 = sizeof(T) == 4;
  const int left = a.O - n;
  f32x8 z = z0 + b;
  if (a.dz) {
    slope_all<F32>(a.act, z);
    z *= load8_any((const T*)a.side + m * a.side_ld + n, left);
  } else {
    activate_all<F32>(a.act, z);
    if (a.side) z += load8_any((const T*)a.side + m * a.side_ld + n, left);
  }
  if (left < 8)
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = e < left ? z[e] : 0.f;
  store8_any((T*)a.out + m * a.out_ld + n, z, a.out_cols - n);
}

}  // namespace lin

// Kernels that keep the whole weight in LDS (16-bit types, many rows); false where a call is not theirs.
bool linear_resident_applicable(const gnn_linear_args& a);
bool linear_resident_takes_dx(const gnn_linear_args& a);
int linear_resident(const gnn_linear_args& a, hipStream_t stream);

}  // namespace gnn
