// A gated layer in one pass, y = act(x Wg^T + bg) (x Wu^T + bu) for rows x [M, I] and Wg, Wu [O, I], and of its
// backward the gradients that go into the products:
//   zg = x Wg^T + bg, zu = x Wu^T + bu,   dzg = dy zu act'(zg), dzu = dy act(zg),
//   dx = dzg Wg + dzu Wu,   dWg = dzg^T x, dWu = dzu^T x,   dbg, dbu = column sums of dzg, dzu.
//
// Neither zg nor zu nor act(zg) touches memory: both products of an output are formed in the same tile (a wave's 32
// outputs of the gate and the same 32 of the other projection), so that a lane holds both sums of its elements.
// The backward forms zg and zu again from x and the weights: kept in 16 bits they would round twice under every
// gradient, in fp32 they would move 8 M O bytes twice. dzg and dzu leave side by side as rows of 2 out_cols, rounded
// once to x's type (the operands of the products after them), so that dx is one product over both and the weights'
// gradients are one product too.
#include <algorithm>

#include "linear_tiles.hpp"

namespace gnn {

namespace {

using namespace lin;

struct GatedArgs {
  const void* x;
  const void* wg;
  const void* wu;
  const void* bg;
  const void* bu;
  const void* dy;  // NULL: forward
  void* out;
  int64_t M;
  int64_t x_ld, wg_ld, wu_ld, dy_ld, out_ld;
  int I, O, out_cols, act;
};

// act(z) and act'(z) of one value
template <bool F32, int ACT>
__device__ __forceinline__ void value_and_slope(float z, float& y, float& s) {
  if constexpr (ACT == GNN_ACT_SILU) {
    const float p = sigmoid<F32>(z);
    y = z * p, s = p * (1.0f + z * (1.0f - p));
  } else {
    y = activate<F32, ACT>(z), s = slope<F32, ACT>(z);
  }
}
// dzg, dzu from zg, zu and dy, in their places
template <bool F32, int ACT>
__device__ __forceinline__ void gradients(f32x8& zg, f32x8& zu, const f32x8& dy) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float y, s;
    value_and_slope<F32, ACT>(zg[e], y, s);
    zg[e] = dy[e] * zu[e] * s;
    zu[e] = dy[e] * y;
  }
}
template <bool F32>
__device__ __forceinline__ void gradients(int act, f32x8& zg, f32x8& zu, const f32x8& dy) {
  switch (act) {
    case GNN_ACT_RELU: gradients<F32, GNN_ACT_RELU>(zg, zu, dy); break;
    case GNN_ACT_GELU: gradients<F32, GNN_ACT_GELU>(zg, zu, dy); break;
    case GNN_ACT_SILU: gradients<F32, GNN_ACT_SILU>(zg, zu, dy); break;
    case GNN_ACT_SIGMOID: gradients<F32, GNN_ACT_SIGMOID>(zg, zu, dy); break;
    default: gradients<F32, GNN_ACT_NONE>(zg, zu, dy); break;
  }
}

template <typename T>
__device__ __forceinline__ f32x8 bias8(const void* b, int n, int O) {
  if (b && n < O) return load8_any((const T*)b + n, O - n);
  return f32x8{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}

// 8 outputs n .. n + 7 of row m from their two sums
template <typename T>
__device__ __forceinline__ void finish8(const GatedArgs& a, f32x8 zg, f32x8 zu, int64_t m, int n) {
  constexpr bool F32 = sizeof(T) == 4;
  const int left = a.O - n;
  T* out = (T*)a.out + m * a.out_ld + n;
  if (!a.dy) {
    activate_all<F32>(a.act, zg);
    store8_any(out, zg * zu, left);
    return;
  }
  gradients<F32>(a.act, zg, zu, load8_any((const T*)a.dy + m * a.dy_ld + n, left));
  if (left < 8)
#pragma unroll
    for (int e = 0; e < 8; ++e) zg[e] = e < left ? zg[e] : 0.f, zu[e] = e < left ? zu[e] : 0.f;
  store8_any(out, zg, 8);
  store8_any(out + a.out_cols, zu, 8);
}

// ---- tiles -----------------------------------------------------------------------------------
// A tile's weight rows are BN / 2 outputs of both matrices: a wave's first Y / 2 tiles of 32 the gate's, the others
// the other projection's of the same outputs.
constexpr int GROUP = 4;

template <typename T, int PREC, typename Cfg>
__global__ __launch_bounds__(Cfg::NT, Cfg::WGS * Cfg::NW / 4) void gated_kernel(const GatedArgs a) {
  constexpr int X = Cfg::X, Y = Cfg::Y, H = Y / 2, BO = Cfg::BN / 2;
  static_assert(Y % 2 == 0, "pairs of tiles");
  __shared__ __align__(16) unsigned char smem[Cfg::LDS];
  // as in linear_kernel: a block of GROUP tiles of rows before the next tiles of outputs
  const uint32_t ntn = (uint32_t)(a.O + BO - 1) / BO;
  const uint32_t w = xcd_remap(blockIdx.x, gridDim.x), group = w / (GROUP * ntn), rest = w % (GROUP * ntn);
  const uint32_t high = min((uint32_t)GROUP, gridDim.x / ntn - group * GROUP);
  const int n0 = (int)(rest / high) * BO;
  const int64_t m0 = (int64_t)(group * GROUP + rest % high) * Cfg::BM;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  const int wm = wave / Cfg::GN, wn = wave % Cfg::GN;

  // rows and outputs past the end repeat the last one (never stored)
  f32x16 acc[X][Y];
  tile_products<T, PREC, Cfg>(
      acc, smem, a.I, [&](int r) { return (const T*)a.x + min(m0 + r, a.M - 1) * a.x_ld; },
      [&](int r) {
        const int t = r >> 5, y = t % Y, n = n0 + 32 * (t / Y * H + y % H) + tile_output(r & 31);
        const int64_t at = min(n, a.O - 1);
        return y < H ? (const T*)a.wg + at * a.wg_ld : (const T*)a.wu + at * a.wu_ld;
      });

  // The sums turn through LDS as linear_kernel's do, the two tiles of an output side by side
  wait_vm_lgkm0<0>();
  asm volatile("s_barrier" ::: "memory");
  constexpr int PAIRS = X * H, FIT = Cfg::LDS / Cfg::NW / 8192, PASS = FIT < PAIRS ? FIT : PAIRS;
  static_assert(PASS >= 1 && PAIRS % PASS == 0, "passes");
  unsigned char* tiles = smem + wave * PASS * 8192;
  auto at = [&](int tile, int row, int chunk) {
    return reinterpret_cast<f32x4*>(tiles + tile * 4096 + row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4));
  };
#pragma unroll
  for (int p = 0; p < PAIRS; p += PASS) {
#pragma unroll
    for (int t = 0; t < 2 * PASS; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& v = acc[(p + t / 2) % X][(p + t / 2) / X + t % 2 * H];
        *at(t, l32, 4 * (q / 2) + 2 * g + q % 2) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      }
#pragma unroll 2
    for (int h = 0; h < 2 * PASS; ++h) {
      const int t = h >> 1, x = (p + t) % X, y = (p + t) / X;
      const int row = 16 * (h & 1) + (lane >> 2), n = n0 + 32 * (H * wn + y) + 8 * (lane & 3);
      const int64_t m = m0 + 32 * (X * wm + x) + row;
      f32x8 z[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const f32x4 lo = *at(2 * t + k, row, 2 * (lane & 3)), hi = *at(2 * t + k, row, 2 * (lane & 3) + 1);
        z[k] = f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      }
      if (m < a.M && n < a.O) finish8<T>(a, z[0] + bias8<T>(a.bg, n, a.O), z[1] + bias8<T>(a.bu, n, a.O), m, n);
    }
  }
}

template <typename Cfg>
int64_t tiles_of(const GatedArgs& a) {
  return (a.M + Cfg::BM - 1) / Cfg::BM * ((a.O + Cfg::BN / 2 - 1) / (Cfg::BN / 2));
}

template <typename T, int PREC, typename Cfg>
int launch(const GatedArgs& a, hipStream_t st) {
  const int64_t tiles = tiles_of<Cfg>(a);
  if (tiles >= ((int64_t)1 << 31)) return set_error(GNN_ERR_UNSUPPORTED, "gated_linear: grid too large");
  hipLaunchKernelGGL((gated_kernel<T, PREC, Cfg>), dim3((uint32_t)tiles), dim3(Cfg::NT), 0, st, a);
  return (int)hipGetLastError();
}

// ---- few tiles ------------------------------------------------------------------------------
// Single tokens and short sequences, as linear_few_kernel: 32 rows x 32 outputs of both products a workgroup, whose
// 8 waves split the contraction; the partial sums are added in wave order.
constexpr int GF_NW = 8, GF_NT = 64 * GF_NW, GF_AHEAD = 4;
constexpr int GF_LD = 20;  // floats a lane's 16 sums take in LDS: 4 more keep the lanes on different banks

template <typename T, int PREC>
__global__ __launch_bounds__(GF_NT, 2) void gated_few_kernel(const GatedArgs a) {
  typedef typename TypeOps<T>::V8 V8;
  __shared__ __align__(16) float part[2][GF_NW][64][GF_LD];
  const uint32_t ntn = (uint32_t)(a.O + 31) / 32;
  const int n0 = (int)(blockIdx.x % ntn) * 32;
  const int64_t m0 = (int64_t)(blockIdx.x / ntn) * 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l32 = lane & 31, g = lane >> 5;
  // rows past the end repeat the last one
  const int64_t n = min(n0 + tile_output(l32), a.O - 1);
  const T* src[3] = {(const T*)a.x + min(m0 + l32, a.M - 1) * a.x_ld + 8 * g, (const T*)a.wg + n * a.wg_ld + 8 * g,
                     (const T*)a.wu + n * a.wu_ld + 8 * g};
  const int steps = (a.I + 15) / 16, whole = a.I / 16, each = (steps + GF_NW - 1) / GF_NW;
  const int k0 = wave * each, k1 = min(whole, k0 + each);
  f32x16 acc[2];
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[0][r] = acc[1][r] = 0.f;
  // No load in a branch: a batch's last steps may be read again, and are not multiplied
  for (int k = k0; k < k1; k += GF_AHEAD) {
    V8 f[GF_AHEAD][3];
#pragma unroll
    for (int u = 0; u < GF_AHEAD; ++u)
#pragma unroll
      for (int i = 0; i < 3; ++i) f[u][i] = load8_global(src[i] + 16 * min(k + u, k1 - 1));
#pragma unroll
    for (int u = 0; u < GF_AHEAD; ++u)
      if (k + u < k1) {
        Mma<T, PREC>::step(acc[0], f[u][1], f[u][0]);
        Mma<T, PREC>::step(acc[1], f[u][2], f[u][0]);
      }
  }
  if (whole < steps && whole >= k0 && whole < k0 + each) {  // part of a step: what lies past the row's end is zero
    const int left = a.I - 16 * whole - 8 * g;  // of this lane's 8 elements
    V8 f[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      f[i] = zero8<T>();
      if (left >= 8) {
        f[i] = load8_global(src[i] + 16 * whole);
      } else if (sizeof(T) == 4 && left > 0) {  // fp32 rows of 16-byte chunks may end after 4
        const auto half = load4(src[i] + 16 * whole);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[i][e] = half[e];
      }
    }
    Mma<T, PREC>::step(acc[0], f[1], f[0]);
    Mma<T, PREC>::step(acc[1], f[2], f[0]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(&part[i][wave][lane][4 * q]) =
          f32x4{acc[i][4 * q], acc[i][4 * q + 1], acc[i][4 * q + 2], acc[i][4 * q + 3]};
  __syncthreads();
  if (threadIdx.x >= 128) return;
  // 8 outputs 16 t + 8 g of a row a thread
  const int t = threadIdx.x >> 6, o = n0 + 16 * t + 8 * g;
  const int64_t m = m0 + l32;
  if (m >= a.M || o >= a.O) return;
  f32x8 z[2] = {bias8<T>(a.bg, o, a.O), bias8<T>(a.bu, o, a.O)};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f32x8 s = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < GF_NW; ++k) s += *reinterpret_cast<const f32x8*>(&part[i][k][lane][8 * t]);
    z[i] += s;
  }
  finish8<T>(a, z[0], z[1], m, o);
}

template <typename T, int PREC>
int run(const GatedArgs& a, hipStream_t st) {
  const int64_t cus = compute_units();
  if constexpr (sizeof(T) == 4) {
    typedef Tile<T, 2, 2, 1, 2, 128, 2> Medium;
    if (tiles_of<Medium>(a) >= cus / 2) return launch<T, PREC, Medium>(a, st);
  } else {
    typedef Tile<T, 2, 4, 4, 2, 128, 2> Large;
    typedef Tile<T, 2, 2, 2, 2, 128, 2> Medium;
    typedef Tile<T, 2, 1, 1, 2, 128, 4> Small;
    if (tiles_of<Large>(a) >= cus) return launch<T, PREC, Large>(a, st);
    if (tiles_of<Medium>(a) >= cus) return launch<T, PREC, Medium>(a, st);
    if (tiles_of<Small>(a) >= cus / 2) return launch<T, PREC, Small>(a, st);
  }
  const int64_t few = (a.M + 31) / 32 * ((a.O + 31) / 32);
  if (few >= ((int64_t)1 << 31)) return set_error(GNN_ERR_UNSUPPORTED, "gated_linear: grid too large");
  hipLaunchKernelGGL((gated_few_kernel<T, PREC>), dim3((uint32_t)few), dim3(GF_NT), 0, st, a);
  return (int)hipGetLastError();
}

// ---- the weights as dx reads them ---------------------------------------------------------------
// dst[i] = column i of Wg and of Wu, out_cols elements each with zeros behind, in tiles of 64 x 64 through LDS
template <typename E>
__global__ __launch_bounds__(256) void gated_turn_kernel(const gnn_gated_turn_args a) {
  constexpr int N = 16 / (int)sizeof(E), B = 64;
  typedef E V __attribute__((ext_vector_type(N)));
  __shared__ E tile[B][B + 1];  // [output][column]
  const E* src = (const E*)(blockIdx.y ? a.wu : a.wg);
  const int64_t ld = blockIdx.y ? a.wu_ld : a.wg_ld;
  const uint32_t across = (uint32_t)((a.out_cols + B - 1) / B);
  const int64_t i0 = (int64_t)(blockIdx.x / across) * B, o0 = (int64_t)(blockIdx.x % across) * B;
  for (int k = threadIdx.x; k < B * B; k += 256) {
    const int64_t o = o0 + k / B, i = i0 + k % B;
    tile[k / B][k % B] = o < a.O && i < a.I ? src[o * ld + i] : (E)0;
  }
  __syncthreads();
  E* dst = (E*)a.dst + blockIdx.y * a.out_cols;
  for (int k = threadIdx.x; k < B * B / N; k += 256) {
    const int i = k / (B / N), o = k % (B / N) * N;
    V v;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = tile[o + e][i];
    if (i0 + i < a.I && o0 + o < a.out_cols) *reinterpret_cast<V*>(dst + (i0 + i) * 2 * a.out_cols + o0 + o) = v;
  }
}

}  // namespace

int gated_linear(const gnn_gated_linear_args& g, hipStream_t st) {
  GatedArgs a{};
  a.x = g.x, a.wg = g.wg, a.wu = g.wu, a.bg = g.bg, a.bu = g.bu, a.dy = g.dy, a.out = g.out;
  a.M = g.M, a.x_ld = g.x_ld, a.wg_ld = g.wg_ld, a.wu_ld = g.wu_ld, a.dy_ld = g.dy_ld, a.out_ld = g.out_ld;
  a.I = (int)g.I, a.O = (int)g.O, a.out_cols = (int)g.out_cols, a.act = g.activation;
  switch (g.dtype) {
    case GNN_BF16: return run<bf16, PREC_NATIVE>(a, st);
    case GNN_F16: return run<f16, PREC_NATIVE>(a, st);
    default: return g.precision == GNN_PREC_BF16X3 ? run<float, PREC_BF16X3>(a, st) : run<float, PREC_IEEE>(a, st);
  }
}

int gated_turn(const gnn_gated_turn_args& a, hipStream_t st) {
  const int64_t blocks = (a.I + 63) / 64 * ((a.out_cols + 63) / 64);
  if (blocks >= ((int64_t)1 << 31)) return set_error(GNN_ERR_UNSUPPORTED, "gated_linear: grid too large");
  const dim3 grid((uint32_t)blocks, 2);
  if (a.dtype == GNN_F32)
    hipLaunchKernelGGL(gated_turn_kernel<uint32_t>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(gated_turn_kernel<uint16_t>, grid, dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace gnn
