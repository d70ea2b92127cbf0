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

#include "linear_rows.hpp"
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

// ---- few tiles, fp32 ------------------------------------------------------------------------
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

// ---- many rows ------------------------------------------------------------------------------
// The gated layer of a pair transition, which HBM bounds (128 -> 512 over 384^2 rows, bf16: 189 MB against 39 GFLOP): as
// in linear_resident.hip a workgroup of 8 waves keeps weights in LDS and every wave walks over 32 rows at a time
// without a barrier. Both weights rarely fit: a workgroup holds `cols` outputs of both, tile y of the gate's 32 rows
// beside tile y of the other's, and the workgroups that share rows lie on one XCD, whose L2 they read them from.
constexpr int GR_NT = 512;

template <typename T, int KS, int ACT, bool BWD>
__global__ __launch_bounds__(GR_NT, GR_NT / 256) void gated_rows_kernel(const GatedArgs a, int cols, int parts) {
  typedef typename TypeOps<T>::V8 V8;
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int ROWB = 32 * KS, NW = GR_NT / 64;
  const int part = blockIdx.x / 8 % parts, n0 = part * cols, held = min(cols, a.O - n0);
  const int64_t worker = (int64_t)(blockIdx.x / 8 / parts) * 8 + blockIdx.x % 8, workers = gridDim.x / parts;
  const int nb = (held + 63) / 64 * 2;  // tiles of 32 outputs, by twos
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  unsigned char* const weight = smem + NW * TURN;
  float* const bias = (float*)(weight + 2 * 32 * nb * ROWB);
  // LDS row r: output n0 + 32 (r / 64) + tile_output(r % 32) of matrix r / 32 % 2, zeros past I and O
  for (int e0 = wave * 64; e0 < 64 * nb * 2 * KS; e0 += GR_NT) {  // 1 KB an instruction
    const uint32_t e = e0 + lane, r = e / (2 * KS), c = (e % (2 * KS)) ^ chunk_swizzle<ROWB>(r);
    const int n = n0 + 32 * (r / 64) + tile_output(r & 31);
    const T* row = r & 32 ? (const T*)a.wu + (int64_t)n * a.wu_ld : (const T*)a.wg + (int64_t)n * a.wg_ld;
    __builtin_amdgcn_global_load_lds(n < a.O && 8 * (int)c < a.I ? (const void*)(row + 8 * c) : (const void*)zero_chunk,
                                     (lds_void_t*)(weight + 16 * e0), 16, 0, 0);
  }
  for (int r = threadIdx.x; r < 64 * nb; r += GR_NT) {
    const int n = n0 + 32 * (r / 64) + (r & 31);
    const T* b = (const T*)(r & 32 ? a.bu : a.bg);
    bias[r] = b && n < a.O ? (float)b[n] : 0.f;
  }
  wait_vm_lgkm0<0>();
  __syncthreads();

  const Turn turn(smem + wave * TURN, lane);
  const MemOrder xm(a.x_ld, a.I, lane), dm(a.dy_ld, held, lane), om(a.out_ld, held, lane);
  const int64_t groups = (a.M + 31) / 32, step = workers * NW;
  auto load_rows = [&](u32x4_t (&x)[KS / 2][2], int64_t grp) {
    const auto r = rows_rsrc<T>(a.x, grp * 32, a.M, a.x_ld, a.I);
#pragma unroll
    for (int p = 0; p < KS / 2; ++p) xm.load(x[p], r, 32 * p);
  };
  const unsigned char* wrow[KS];
#pragma unroll
  for (int kk = 0; kk < KS; ++kk)
    wrow[kk] = weight + l32 * ROWB + (((2 * kk + g) ^ chunk_swizzle<ROWB>(l32)) << 4);
  // the backward's rows of 8 steps, beside twice the sums, are not loaded ahead
  constexpr bool AHEAD = KS <= (BWD ? 4 : 8);
  u32x4_t next[KS / 2][2], x[KS / 2][2];
  auto turn_rows = [&]() {
#pragma unroll
    for (int p = 0; p < KS / 2; ++p) {
      Turn::put(turn.to_mem, next[p]);
      Turn::get(turn.to_rows, x[p]);
    }
  };
  // Both sums of tile y; they run beside the epilogue of the tile before, of the last rows' last one at their end
  struct Sums {
    f32x16 gate, up;
  };
  auto tile = [&](int y) {
    Sums s = {bias_tile(bias + 64 * y, g), bias_tile(bias + 64 * y + 32, g)};
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const unsigned char* w = wrow[kk] + y * 64 * ROWB;
      const V8 xf = __builtin_bit_cast(V8, x[kk / 2][kk % 2]);
      Mma<T, PREC_NATIVE>::step(s.gate, *reinterpret_cast<const V8*>(w), xf);
      Mma<T, PREC_NATIVE>::step(s.up, *reinterpret_cast<const V8*>(w + 32 * ROWB), xf);
    }
    return s;
  };
  // 32 x 32 outputs in memory order: y, or dzg and dzu
  auto finish = [&](const Sums& s, const u32x4_t (&dy)[2], u32x4_t (&o)[BWD ? 2 : 1][2]) {
    u32x4_t d[2];
    if constexpr (BWD) {
      Turn::put(turn.to_mem, dy);
      Turn::get(turn.to_rows, d);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x8 zg = outputs8(s.gate, t), zu = outputs8(s.up, t);
      if constexpr (BWD) {
        gradients<false, ACT>(zg, zu, to8<T>(d[t]));
        o[BWD][t] = __builtin_bit_cast(u32x4_t, TypeOps<T>::from_f32(zu));
      } else {
        activate_all<false, ACT>(zg);
        zg *= zu;
      }
      o[0][t] = __builtin_bit_cast(u32x4_t, TypeOps<T>::from_f32(zg));
    }
#pragma unroll
    for (int k = 0; k < (BWD ? 2 : 1); ++k) {
      Turn::put(turn.to_rows, o[k]);
      Turn::get(turn.to_mem, o[k]);
    }
  };
  int64_t grp = worker * NW + wave;
  load_rows(next, grp);
  turn_rows();
  if (AHEAD) load_rows(next, grp + step);
  Sums now = tile(0);
  for (; grp < groups; grp += step) {
    const auto drs = rows_rsrc<T>((const T*)a.dy + (BWD ? n0 : 0), grp * 32, BWD ? a.M : 0, a.dy_ld, held);
    const auto grs = rows_rsrc<T>((const T*)a.out + n0, grp * 32, a.M, a.out_ld, held);
    const auto urs = rows_rsrc<T>((const T*)a.out + (BWD ? a.out_cols + n0 : 0), grp * 32, BWD ? a.M : 0, a.out_ld, held);
    u32x4_t dy[2][2];
    auto load_dy = [&](int y) {
      dm.load(dy[0], drs, 32 * y);
      dm.load(dy[1], drs, 32 * (y + 1));
    };
    if (BWD) load_dy(0);
    // tiles by twos, whose 128-byte lines are stored at once
    for (int y = 0; y < nb; y += 2) {
      u32x4_t o[2][BWD ? 2 : 1][2];
      Sums ahead = tile(y + 1);
      finish(now, dy[0], o[0]);
      now = ahead;
      if (y + 2 < nb) {
        ahead = tile(y + 2);
      } else {
        if (!AHEAD) load_rows(next, grp + step);
        turn_rows();
        if (AHEAD) load_rows(next, grp + 2 * step);
        ahead = tile(0);
      }
      finish(now, dy[1], o[1]);
      now = ahead;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        om.store(o[k][0], grs, 32 * (y + k));
        if (BWD) om.store(o[k][BWD], urs, 32 * (y + k));
      }
      if (BWD) load_dy(y + 2);
    }
  }
}

// Outputs of both weights that LDS holds beside the waves' turning tiles, and what they take; 0 where this is no form
// for the call
struct RowsForm {
  int ks, cols, parts;
  size_t lds;
};
// Rows of up to 128 inputs: of 256 half as many outputs fit, each workgroup's rows are read by twice as many, and tiles are
// as fast or faster (147456 x 256 -> 512, bf16: 119 us both, the backward's first kernel 225 here, 202 in tiles).
RowsForm rows_form(const GatedArgs& a, int bytes) {
  auto rows16 = [](const void* p, int64_t ld) { return ((uintptr_t)p % 16) == 0 && ld % 8 == 0 && ld < (1 << 24); };
  if (bytes != 2 || a.M < RS_MIN_ROWS || a.I > 128 || a.O % 8 || a.x_ld >= (1 << 24) || !rows16(a.out, a.out_ld) ||
      (a.dy && !rows16(a.dy, a.dy_ld)))
    return {};
  RowsForm f{};
  f.ks = a.I <= 64 ? 4 : 8;
  const int each = 2 * (32 * f.ks + 4), most = RS_LDS / each / 64 * 64;
  f.parts = (a.O + most - 1) / most;
  f.cols = ((a.O + f.parts - 1) / f.parts + 63) / 64 * 64;
  f.parts = (a.O + f.cols - 1) / f.cols;
  f.lds = (size_t)f.cols * each + GR_NT / 64 * TURN;
  return f;
}

template <typename T, int KS, bool BWD>
int launch_rows(const GatedArgs& a, const RowsForm& f, hipStream_t st) {
  int rc = 0;
  with_activation(a.act, [&](auto act) {
    auto fn = gated_rows_kernel<T, KS, decltype(act)::value, BWD>;
    if (f.lds > 64 * 1024)
      (void)hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)f.lds);
    // whole eights of workgroups for each part, so that a part's workgroups and those of the others meet on every XCD
    const int64_t groups = (a.M + 31) / 32, places = persistent_grid((const void*)fn, GR_NT, f.lds);
    const int64_t eights = std::max<int64_t>(1, std::min(places / 8 / f.parts, (groups + 63) / 64));
    hipLaunchKernelGGL(fn, dim3((uint32_t)(8 * eights * f.parts)), dim3(GR_NT), f.lds, st, a, f.cols, f.parts);
    rc = (int)hipGetLastError();
  });
  return rc;
}
template <typename T>
int launch_rows(const GatedArgs& a, const RowsForm& f, hipStream_t st) {
  if (f.ks == 4) return a.dy ? launch_rows<T, 4, true>(a, f, st) : launch_rows<T, 4, false>(a, f, st);
  return a.dy ? launch_rows<T, 8, true>(a, f, st) : launch_rows<T, 8, false>(a, f, st);
}

// The form of a call. Resident weights for many short rows, up to 4 parts of which read the same rows (262144 x 128 ->
// 1024, bf16: 223 us; 65536 rows 52, in tiles 83; 32768 x 128 -> 512 19.5 and 24.9, 16384 17.1 and 14.2).
// Tiles of 256 x 128 where they fill the CUs and leave no second round half empty (x 1024 -> 2048, 256 tiles 36 us, of
// 128 x 64 42; 288 tiles 62 and 54; 384 tiles 62 both; 512 tiles 69 and 82), of 128 x 64 where those fill them
// (1024 x 1024 -> 2048: 15.0 us, of 64 x 32 17.9; 1024 x 1024 -> 1024: 13.9 and 10.0). fp32: tiles of 128 x 64 where
// their last round is full enough (4099 x 336 -> 883, 0.9 of a round: 55 us, of 64 x 64 63; 3000 x 256 -> 2048, 1.5 rounds:
// 61 and 65; x 1024 -> 1024, 1.03 rounds: 207 and 178), of 64 x 64, and below half a tile of those a CU few rows' form (512 x
// 512 -> 512: 12 us, in tiles 24; 1024 x 512 -> 1024: 34 and 26).
template <typename T, int PREC>
int run(const GatedArgs& a, hipStream_t st) {
  const int64_t cus = compute_units();
  if constexpr (sizeof(T) == 4) {
    typedef Tile<T, 2, 2, 1, 2, 128, 2> Small;
    typedef Tile<T, 4, 2, 1, 2, 128, 2> Large;
    const int64_t large = tiles_of<Large>(a), rounds = (large + 2 * cus - 1) / (2 * cus);  // two workgroups a CU
    if (10 * large >= 7 * rounds * 2 * cus) return launch<T, PREC, Large>(a, st);
    if (tiles_of<Small>(a) >= cus / 2) return launch<T, PREC, Small>(a, st);
    const int64_t few = (a.M + 31) / 32 * ((a.O + 31) / 32);
    hipLaunchKernelGGL((gated_few_kernel<T, PREC>), dim3((uint32_t)few), dim3(GF_NT), 0, st, a);
    return (int)hipGetLastError();
  } else {
    const RowsForm f = rows_form(a, sizeof(T));
    if (f.parts && f.parts <= 4) return launch_rows<T>(a, f, st);
    typedef Tile<T, 2, 4, 4, 2, 128, 2> Large;
    typedef Tile<T, 2, 2, 2, 2, 128, 2> Medium;
    typedef Tile<T, 2, 1, 1, 2, 128, 4> Small;
    const int64_t large = tiles_of<Large>(a);
    if ((16 * large >= 15 * cus && large <= cus) || 2 * large >= 3 * cus) return launch<T, PREC, Large>(a, st);
    if (tiles_of<Medium>(a) >= cus) return launch<T, PREC, Medium>(a, st);
    return launch<T, PREC, Small>(a, st);
  }
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
  E v[B * B / 256];  // no load in a branch: past the end the last row or column, and then zero
#pragma unroll
  for (int k = 0; k < B * B / 256; ++k) {
    const int64_t o = o0 + threadIdx.x / B + k * (256 / B), i = i0 + threadIdx.x % B;
    v[k] = src[min(o, a.O - 1) * ld + min(i, a.I - 1)];
  }
#pragma unroll
  for (int k = 0; k < B * B / 256; ++k) {
    const int o = threadIdx.x / B + k * (256 / B);
    tile[o][threadIdx.x % B] = o0 + o < a.O ? v[k] : (E)0;
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
