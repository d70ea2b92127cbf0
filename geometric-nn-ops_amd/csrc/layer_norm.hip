// LayerNorm over the last dimension of rows of any width up to 16384, and its backward:
//   y  = (x - mean) rstd w + b,   rstd = 1 / sqrt(var + eps), var the mean of (x - mean)^2,
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),   g = dy w, xhat = (x - mean) rstd,
//   dw = sum over the rows of dy xhat,   db = sum over the rows of dy.
//
// Both are bound by HBM (one read of x and one write of y; x and dy in, dx out), so a row is read once
// and stays in registers, as it came: a team of lanes takes a row, each lane C chunks of 16 bytes, and
// the statistics are two sums over the team (the squared deviations from the mean that is already known:
// E[x^2] - mean^2 would lose the variance of rows with a large mean). Teams are 8 to 64 lanes of a wave for
// rows of up to 192 chunks (several rows a wave where they are short: sums by DPP and lane swaps, no LDS)
// and 4, 8 or 16 waves for wider ones. Workgroups stay and walk over the rows, so that a lane keeps its
// columns: their parameters are loaded once, and in the backward their sums of dy xhat and dy run in its
// registers until the workgroup leaves one fp32 row of partial sums (added in order by reduce_parts).
// The forward leaves mean and rstd of each row in fp32 where a backward will follow: 8 bytes a row
// instead of both sums over again, with their latency, in front of the backward's own.
// Kernel times, with the ordered sums: 147456 x 128 bf16 forward 14 us (5.4 TB/s), backward 26; 8192 x 5120 bf16 33
// and 60 (5.1, 4.2 TB/s); 8191 x 5003 fp16, rows at odd addresses, 40 and 70 (4.1, 3.5); 8192 x 3000 fp32 33 and 56.
// Rows of any alignment and width are read in the same 16-byte accesses (gfx950 takes them at any
// element's address); the last chunk of a width that is no multiple of 16 bytes goes by elements.
#include <algorithm>

#include "gnn_common.hpp"
#include "gnn_internal.hpp"

namespace gnn {

namespace {

constexpr int LN_MAX_K = 16384;

// Sum over groups of L consecutive lanes, in every lane. DPP within 16 lanes (xor 1, xor 2, the mirrors of 8
// and 16 lanes: each adds the other half's sum), lane swaps beyond.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float team_sum(float x) {
  static_assert(L == 8 || L == 16 || L == 32 || L == 64, "lanes of a team");
  x = dpp_add<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  x = dpp_add<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  x = dpp_add<0x141>(x);  // row_half_mirror
  if constexpr (L >= 16) x = dpp_add<0x140>(x);  // row_mirror
  if constexpr (L >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  if constexpr (L >= 64) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return x;
}

// 16 bytes of elements at any element's address, and their fp32 values
template <typename T> struct Chunk;
template <> struct Chunk<bf16> { typedef bf16x8 V; typedef f32x8 F; };
template <> struct Chunk<f16> { typedef f16x8 V; typedef f32x8 F; };
template <> struct Chunk<float> { typedef f32x4 V; typedef f32x4 F; };

template <typename T>
__device__ __forceinline__ typename Chunk<T>::V load_chunk(const T* p, int left) {
  typedef typename Chunk<T>::V V;
  constexpr int E = 16 / (int)sizeof(T);
  typedef V VU __attribute__((aligned(sizeof(T))));
  if (left >= E) return *(const __attribute__((address_space(1))) VU*)p;
  V v;
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = e < left ? p[e] : (T)0.f;
  return v;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const typename Chunk<T>::V& v, int left) {
  typedef typename Chunk<T>::V V;
  constexpr int E = 16 / (int)sizeof(T);
  typedef V VU __attribute__((aligned(sizeof(T))));
  if (left >= E) {
    *(__attribute__((address_space(1))) VU*)p = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < left) p[e] = v[e];
}
template <typename T>
__device__ __forceinline__ typename Chunk<T>::F chunk_f32(const typename Chunk<T>::V& v) {
  return __builtin_convertvector(v, typename Chunk<T>::F);
}
// The parameters of a chunk's columns, in the rows' type or fp32; `fill` where there are none
template <typename T>
__device__ __forceinline__ typename Chunk<T>::F load_param(const void* p, bool f32, int col, int left, float fill) {
  constexpr int E = 16 / (int)sizeof(T);
  typename Chunk<T>::F w;
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = fill;
  if (!p || left <= 0) return w;
  if (!f32) return chunk_f32<T>(load_chunk((const T*)p + col, left));
#pragma unroll
  for (int h = 0; h < E; h += 4) {
    const f32x4 v = load_chunk((const float*)p + col + h, left - h);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[h + e] = v[e];
  }
  return w;
}

struct Rows {  // address of a row: two levels of strides, in elements
  int64_t inner, outer_stride, inner_stride;
};
template <typename T>
__device__ __forceinline__ T* row_at(T* p, const Rows& r, int64_t row) {
  if (r.inner == 0) return p + row * r.inner_stride;
  const int64_t o = row / r.inner;
  return p + o * r.outer_stride + (row - o * r.inner) * r.inner_stride;
}

struct LnArgs {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  void* out;  // y or dx
  float* mean;
  float* rstd;
  float* partial;
  int64_t rows;
  int K;
  Rows xr, dyr;
  float eps;
  bool w_f32;
};

// A team's place: L lanes of a wave (NW = 1), or NW whole waves (L = 64). NT threads a workgroup.
template <int NT, int L, int NW>
struct Team {
  static constexpr int LANES = L * NW;
  static constexpr int N = NT / LANES;  // teams a workgroup
};

// Sum over a team of NW waves, through LDS: `slot` alternates, so that one barrier is enough
template <int NT, int L, int NW>
__device__ __forceinline__ float2 wide_sum(float2 s, float2 (*red)[16], int slot) {
  s.x = team_sum<L>(s.x);
  s.y = team_sum<L>(s.y);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x >> 6, first = wave / NW * NW;
    if ((threadIdx.x & 63) == 0) red[slot][wave] = s;
    __syncthreads();
    s = red[slot][first];
#pragma unroll
    for (int k = 1; k < NW; ++k) {
      s.x += red[slot][first + k].x;
      s.y += red[slot][first + k].y;
    }
  }
  return s;
}

template <typename T, int NT, int L, int NW, int C>
__global__ __launch_bounds__(NT) void layer_norm_fwd_kernel(const LnArgs a) {
  typedef Team<NT, L, NW> Tm;
  typedef typename Chunk<T>::V V;
  typedef typename Chunk<T>::F F;
  constexpr int E = 16 / (int)sizeof(T);
  __shared__ float2 red[2][16];
  const int team = threadIdx.x / Tm::LANES, lane = threadIdx.x % Tm::LANES;
  const int K = a.K;
  F w[C], b[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (lane + c * Tm::LANES) * E;
    w[c] = load_param<T>(a.w, a.w_f32, col, K - col, 1.f);
    b[c] = load_param<T>(a.b, a.w_f32, col, K - col, 0.f);
  }
  // every team of a workgroup takes the same number of turns (they meet at barriers)
  for (int64_t r0 = (int64_t)blockIdx.x * Tm::N; r0 < a.rows; r0 += (int64_t)gridDim.x * Tm::N) {
    const int64_t row = r0 + team;
    const bool live = row < a.rows;
    const T* x = row_at((const T*)a.x, a.xr, live ? row : a.rows - 1);
    V v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (lane + c * Tm::LANES) * E;
      v[c] = load_chunk(x + col, K - col);
    }
    float2 s = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const F f = chunk_f32<T>(v[c]);
      float t = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) t += f[e];
      s.x += t;
    }
    const float mean = wide_sum<NT, L, NW>(s, red, 0).x / (float)K;
    s.x = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int left = K - (lane + c * Tm::LANES) * E;
      const F f = chunk_f32<T>(v[c]) - mean;
      float t = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) t += e < left ? f[e] * f[e] : 0.f;
      s.x += t;
    }
    const float var = wide_sum<NT, L, NW>(s, red, 1).x / (float)K;
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (!live) continue;  // no barrier below
    T* y = (T*)a.out + row * K;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (lane + c * Tm::LANES) * E;
      const F f = (chunk_f32<T>(v[c]) - mean) * rstd * w[c] + b[c];
      store_chunk(y + col, __builtin_convertvector(f, V), K - col);
    }
    if (a.mean && lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T, int NT, int L, int NW, int C>
__global__ __launch_bounds__(NT) void layer_norm_bwd_kernel(const LnArgs a) {
  typedef Team<NT, L, NW> Tm;
  typedef typename Chunk<T>::V V;
  typedef typename Chunk<T>::F F;
  constexpr int E = 16 / (int)sizeof(T);
  __shared__ float2 red[2][16];
  const int team = threadIdx.x / Tm::LANES, lane = threadIdx.x % Tm::LANES;
  const int K = a.K;
  const float inv_k = 1.0f / (float)K;
  F w[C], dw[C], db[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (lane + c * Tm::LANES) * E;
    w[c] = load_param<T>(a.w, a.w_f32, col, K - col, 1.f);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[c][e] = db[c][e] = 0.f;
  }
  struct Row {
    V x[C], dy[C];
    float mean, rstd;
  };
  auto load = [&](Row& r, int64_t row) {
    row = min(row, a.rows - 1);
    const T* x = row_at((const T*)a.x, a.xr, row);
    const T* dy = row_at((const T*)a.dy, a.dyr, row);
    r.mean = a.mean[row], r.rstd = a.rstd[row];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (lane + c * Tm::LANES) * E;
      r.x[c] = load_chunk(x + col, K - col);
      r.dy[c] = load_chunk(dy + col, K - col);
    }
  };
  // Workgroups of 8 waves have a CU, and registers, to themselves: their next row is on its way while they are
  // at this one (8192 x 3000 fp32: 56 us, 61 without, 8191 x 5003 fp16: 70 and 72, with the sums of the parts; the
  // smaller teams hide it behind other workgroups)
  constexpr bool AHEAD = NW > 1 && NT <= 512;
  const int64_t step = (int64_t)gridDim.x * Tm::N;
  Row now, next;
  if (AHEAD) load(next, (int64_t)blockIdx.x * Tm::N + team);
  int slot = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * Tm::N; r0 < a.rows; r0 += step, slot ^= 1) {
    const bool live = r0 + team < a.rows;
    const int64_t row = live ? r0 + team : a.rows - 1;
    if (AHEAD) {
      now = next;
      if (r0 + step < a.rows) load(next, r0 + step + team);
    } else {
      load(now, row);
    }
    const V (&xv)[C] = now.x, (&gv)[C] = now.dy;
    const float mean = now.mean, rstd = now.rstd;
    float2 s = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      // columns past the end have dy = 0: they add nothing to any sum
      const F xh = (chunk_f32<T>(xv[c]) - mean) * rstd, d = chunk_f32<T>(gv[c]);
      const F g = d * w[c];
      float t = 0.f, u = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        t += g[e];
        u += g[e] * xh[e];
      }
      s.x += t;
      s.y += u;
      if (live) {
        dw[c] += d * xh;
        db[c] += d;
      }
    }
    s = wide_sum<NT, L, NW>(s, red, slot);
    if (!a.out || !live) continue;
    const float c1 = s.x * inv_k, c2 = s.y * inv_k;
    T* dx = (T*)a.out + row * K;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (lane + c * Tm::LANES) * E;
      const F xh = (chunk_f32<T>(xv[c]) - mean) * rstd, g = chunk_f32<T>(gv[c]) * w[c];
      store_chunk(dx + col, __builtin_convertvector((g - c1 - xh * c2) * rstd, V), K - col);
    }
  }
  if (!a.partial) return;
  // the teams' column sums meet in LDS, a chunk of each lane at a time, and are added in team order
  constexpr int TN = Tm::N;
  __shared__ __align__(16) float sum[2 * NT * E];
  float* out = a.partial + (int64_t)blockIdx.x * 2 * K;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      sum[e * NT + threadIdx.x] = dw[c][e];
      sum[(E + e) * NT + threadIdx.x] = db[c][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * E * Tm::LANES; i += NT) {
      const int ln = i / E % Tm::LANES, e = i % E, which = i / (E * Tm::LANES);
      const int col = (ln + c * Tm::LANES) * E + e;
      if (col >= K) continue;
      float t = 0.f;
#pragma unroll 8
      for (int k = 0; k < TN; ++k) t += sum[(which * E + e) * NT + k * Tm::LANES + ln];
      out[which * K + col] = t;
    }
  }
}

// The team for a width of n chunks of 16 bytes: short rows several to a wave, and C = 3 where the lanes of
// the next power of two would stand idle (a width of 384: 16 lanes of 3 chunks, not 48 lanes of 64). Three
// chunks of 16-bit elements and their sums take 143 registers in the backward: those teams come in workgroups
// of 8 waves, the other wide ones in 16 (at most 128).
struct Shape {
  int lanes, waves, chunks, threads;
};
Shape shape_for(int64_t K, int32_t dtype) {
  const int64_t e = dtype == GNN_F32 ? 4 : 8, n = (K + e - 1) / e;
  if (n <= 8) return {8, 1, 1, 256};
  if (n <= 16) return {16, 1, 1, 256};
  if (n <= 24) return {8, 1, 3, 256};
  if (n <= 32) return {32, 1, 1, 256};
  if (n <= 48) return {16, 1, 3, 256};
  if (n <= 64) return {64, 1, 1, 256};
  if (n <= 96) return {32, 1, 3, 256};
  if (n <= 128) return {64, 1, 2, 256};
  if (n <= 192) return {64, 1, 3, 256};
  // several waves a row: 64 lanes x waves x chunks
  if (n <= 64 * 4) return {64, 4, 1, 1024};
  if (n <= 64 * 4 * 2) return {64, 4, 2, 1024};
  if (n <= 64 * 4 * 3) return {64, 4, 3, 512};
  if (n <= 64 * 8 * 2) return {64, 8, 2, 1024};
  if (n <= 64 * 8 * 3) return {64, 8, 3, 512};
  if (n <= 64 * 16 * 2) return {64, 16, 2, 1024};
  if (n <= 64 * 16 * 3) return {64, 16, 3, 1024};
  return {64, 16, 4, 1024};
}

int64_t team_rows(const Shape& s) { return s.threads / (s.lanes * s.waves); }

// Workgroups: enough to fill the card, no more than there are rows for
int64_t fwd_grid(int64_t rows, const Shape& s) {
  const int64_t full = (int64_t)compute_units() * (2048 / s.threads);
  return std::max<int64_t>(1, std::min(full, (rows + team_rows(s) - 1) / team_rows(s)));
}
// ... and in the backward, each leaves a row of partial sums
int64_t bwd_grid(int64_t rows, const Shape& s) {
  const int64_t full = (int64_t)compute_units() * (s.threads >= 512 ? 1 : 6);
  return std::max<int64_t>(1, std::min(full, (rows + team_rows(s) - 1) / team_rows(s)));
}

template <typename T, int NT, int L, int NW, int C>
void launch(const LnArgs& a, bool backward, int64_t grid, hipStream_t st) {
  if (backward)
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, NT, L, NW, C>), dim3((uint32_t)grid), dim3(NT), 0, st, a);
  else
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, NT, L, NW, C>), dim3((uint32_t)grid), dim3(NT), 0, st, a);
}

template <typename T>
int dispatch(const LnArgs& a, const Shape& s, bool backward, int64_t grid, hipStream_t st) {
  const int key = s.waves * 1000 + s.lanes * 10 + s.chunks;
  switch (key) {
    case 1081: launch<T, 256, 8, 1, 1>(a, backward, grid, st); break;
    case 1161: launch<T, 256, 16, 1, 1>(a, backward, grid, st); break;
    case 1083: launch<T, 256, 8, 1, 3>(a, backward, grid, st); break;
    case 1321: launch<T, 256, 32, 1, 1>(a, backward, grid, st); break;
    case 1163: launch<T, 256, 16, 1, 3>(a, backward, grid, st); break;
    case 1641: launch<T, 256, 64, 1, 1>(a, backward, grid, st); break;
    case 1323: launch<T, 256, 32, 1, 3>(a, backward, grid, st); break;
    case 1642: launch<T, 256, 64, 1, 2>(a, backward, grid, st); break;
    case 1643: launch<T, 256, 64, 1, 3>(a, backward, grid, st); break;
    case 4641: launch<T, 1024, 64, 4, 1>(a, backward, grid, st); break;
    case 4642: launch<T, 1024, 64, 4, 2>(a, backward, grid, st); break;
    case 4643: launch<T, 512, 64, 4, 3>(a, backward, grid, st); break;
    case 8642: launch<T, 1024, 64, 8, 2>(a, backward, grid, st); break;
    case 8643: launch<T, 512, 64, 8, 3>(a, backward, grid, st); break;
    case 16642: launch<T, 1024, 64, 16, 2>(a, backward, grid, st); break;
    case 16643:
      if constexpr (sizeof(T) == 4) launch<T, 1024, 64, 16, 3>(a, backward, grid, st);
      break;
    default:
      if constexpr (sizeof(T) == 4) launch<T, 1024, 64, 16, 4>(a, backward, grid, st);
      break;
  }
  return (int)hipGetLastError();
}

int run(const LnArgs& a, const Shape& s, int32_t dtype, bool backward, int64_t grid, hipStream_t st) {
  switch (dtype) {
    case GNN_BF16: return dispatch<bf16>(a, s, backward, grid, st);
    case GNN_F16: return dispatch<f16>(a, s, backward, grid, st);
    default: return dispatch<float>(a, s, backward, grid, st);
  }
}

}  // namespace

int64_t layer_norm_bwd_parts(int64_t rows, int64_t K, int32_t dtype) {
  return bwd_grid(rows, shape_for(K, dtype));
}

int layer_norm_fwd(const gnn_layer_norm_fwd_args& a, hipStream_t st) {
  if (a.K > LN_MAX_K) return set_error(GNN_ERR_UNSUPPORTED, "layer_norm: rows wider than 16384");
  LnArgs k{};
  k.x = a.x, k.w = a.weight, k.b = a.bias, k.out = a.y, k.mean = a.mean, k.rstd = a.rstd;
  k.rows = a.rows, k.K = (int)a.K, k.eps = a.eps, k.w_f32 = a.param_dtype == GNN_F32;
  k.xr = {a.x_inner == a.rows ? 0 : a.x_inner, a.x_outer_stride, a.x_stride};
  const Shape s = shape_for(a.K, a.dtype);
  return run(k, s, a.dtype, false, fwd_grid(a.rows, s), st);
}

int layer_norm_bwd(const gnn_layer_norm_bwd_args& a, hipStream_t st) {
  if (a.K > LN_MAX_K) return set_error(GNN_ERR_UNSUPPORTED, "layer_norm backward: rows wider than 16384");
  LnArgs k{};
  k.x = a.x, k.dy = a.dy, k.w = a.weight, k.out = a.dx;
  k.mean = const_cast<float*>(a.mean), k.rstd = const_cast<float*>(a.rstd), k.partial = a.partial;
  k.rows = a.rows, k.K = (int)a.K, k.w_f32 = a.param_dtype == GNN_F32;
  k.xr = {a.x_inner == a.rows ? 0 : a.x_inner, a.x_outer_stride, a.x_stride};
  k.dyr = {a.dy_inner == a.rows ? 0 : a.dy_inner, a.dy_outer_stride, a.dy_stride};
  return run(k, shape_for(a.K, a.dtype), a.dtype, true, a.parts, st);
}

}  // namespace gnn
