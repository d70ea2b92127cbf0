// Norms of queries and keys for each head with the position rotation behind them, in one pass over both:
//   n = x / sqrt(mean(x^2) + eps) w,   y = R(pos) n,
// where R turns pair j of the first R elements by the angle pos f[j] (pairs j and j + R/2, or 2j and 2j + 1), and
//   g = R(pos)^T dy,  dw = sum over the rows of g x / rms,  dx = (g w - xh mean(g w xh)) / rms,  xh = x / rms.
//
// Bound by HBM: one read and one write of every row (two reads in the backward), no statistics kept: a row of a
// head is at most 256 elements, which a team of 1 to 32 lanes holds, 2 E elements a lane. A lane's elements are E
// whole pairs, so that the rotation needs no exchange, and behind the turned part the two halves of 2 E plain ones
// (angle 0). A team takes some heads of one token: a lane's E angles are the same for all of them and are made
// once. The product pos f is formed in 64 bits and reduced to a fraction of a turn there: at position 10^6 fp32
// would be 0.06 off. For 16-bit rows the hardware's sine and cosine take the turns, off by 2^-23 at most over half a turn
// to both sides (measured at 2^20 places), a two-thousandth of fp16's rounding; fp32 rows, whose rounding that is twice of,
// have polynomials of their own.
// Workgroups are the queries' or the keys'; in the backward they stay and walk over their tokens, and each leaves
// one fp32 row of its weight's gradient, added in order afterwards.
#include <algorithm>

#include "gnn_common.hpp"
#include "gnn_internal.hpp"

namespace gnn {

namespace {

constexpr int QR_NT = 256;
constexpr int QR_MAX_PAIRS = 128;

struct Side {
  const void* x;
  const void* dy;
  const void* w;
  const void* pos;
  void* out;
  float* partial;
  int64_t xs[3], ds[3], ps;  // strides: batch, token, head; positions' batch
  int64_t N, units;
  int H, heads, groups;  // heads a unit, units a token
  uint32_t blocks;
};
struct RotaryArgs {
  Side side[2];
  double turns[QR_MAX_PAIRS];  // of a pair, a position
  int D, R, log_l;
  float eps, inv_d;
  bool norm, pos64, w_f32;
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// Sum over a team of 2^log_l lanes, in every lane
__device__ __forceinline__ float team_sum(float x, int log_l) {
  if (log_l >= 1) x = dpp_add<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  if (log_l >= 2) x = dpp_add<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  if (log_l >= 3) x = dpp_add<0x141>(x);  // row_half_mirror
  if (log_l >= 4) x = dpp_add<0x140>(x);  // row_mirror
  if (log_l >= 5) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return x;
}

template <typename T, int E> struct Vec {
  typedef T V __attribute__((ext_vector_type(E)));
  typedef float F __attribute__((ext_vector_type(E)));
  typedef V VU __attribute__((aligned(sizeof(T))));  // rows at any element's address
  static __device__ __forceinline__ V load(const T* p) { return *(const __attribute__((address_space(1))) VU*)p; }
  static __device__ __forceinline__ void store(T* p, const F& v) {
    *(__attribute__((address_space(1))) VU*)p = __builtin_convertvector(v, V);
  }
};

// A lane's 2 E elements: as they lie (lo, hi), and as the first and second elements of its pairs
template <typename T, int E, bool NEIGHBOURS>
struct Pairs {
  typedef Vec<T, E> O;
  typedef typename O::F F;
  static __device__ __forceinline__ void split(const typename O::V& lo, const typename O::V& hi, F& a, F& c) {
    const F l = __builtin_convertvector(lo, F), h = __builtin_convertvector(hi, F);
    if constexpr (NEIGHBOURS) {
#pragma unroll
      for (int e = 0; e < E / 2; ++e)
        a[e] = l[2 * e], c[e] = l[2 * e + 1], a[E / 2 + e] = h[2 * e], c[E / 2 + e] = h[2 * e + 1];
    } else {
      a = l, c = h;
    }
  }
  static __device__ __forceinline__ void store(T* lo, T* hi, const F& a, const F& c) {
    if constexpr (NEIGHBOURS) {
      F l, h;
#pragma unroll
      for (int e = 0; e < E / 2; ++e)
        l[2 * e] = a[e], l[2 * e + 1] = c[e], h[2 * e] = a[E / 2 + e], h[2 * e + 1] = c[E / 2 + e];
      O::store(lo, l), O::store(hi, h);
    } else {
      O::store(lo, a), O::store(hi, c);
    }
  }
};

// Of a turn in -1/2 .. 1/2, which is (k + 4 f) quarters with |f| <= 1/8. fp32: sin(2 pi f) = f (2 pi + P(f^2)), cos(2 pi f)
// = 1 + f^2 Q(f^2) with polynomials fitted in 64 bits (even relative errors of 2^-28 and 2^-33), swapped and signed by
// k: off by 1.5 units of 2^-24 of themselves at most (3 10^6 places in fp32 arithmetic against 80 bits).
template <typename T>
__device__ __forceinline__ void sine_cosine(float turn, float& sn, float& cs) {
  if constexpr (sizeof(T) == 2) {
    sn = __builtin_amdgcn_sinf(turn), cs = __builtin_amdgcn_cosf(turn);
  } else {
    const float k = rintf(4.f * turn), f = __builtin_fmaf(-0.25f, k, turn), x = f * f;
    const float p = __builtin_fmaf(x, __builtin_fmaf(x, __builtin_fmaf(x, -75.39356f, 81.592354f), -41.341663f), -1.9519194e-07f);
    const float q = __builtin_fmaf(x, __builtin_fmaf(x, __builtin_fmaf(x, 59.229218f, -85.44324f), 64.93932f), -19.739208f);
    const float s = __builtin_fmaf(f, 6.2831855f, f * p), c = __builtin_fmaf(x, q, 1.f);
    const uint32_t quarter = (uint32_t)(int)k;
    const bool odd = quarter & 1;
    sn = __uint_as_float(__float_as_uint(odd ? c : s) ^ (quarter & 2) << 30);
    cs = __uint_as_float(__float_as_uint(odd ? s : c) ^ (quarter + 1 & 2) << 30);
  }
}

// The backward: three waves a SIMD. Of 169 registers, one more than these have, it took up to a fifth longer in fp32.
template <typename T, int E, bool NEIGHBOURS, bool BWD>
__global__ __launch_bounds__(QR_NT, BWD ? 3 : 1) void qk_norm_rotary_kernel(const RotaryArgs a) {
  typedef Vec<T, E> O;
  typedef typename O::V V;
  typedef typename O::F F;
  typedef Pairs<T, E, NEIGHBOURS> P;
  constexpr int AT_ONCE = BWD ? 2 : 4;  // heads whose loads are in flight
  const bool keys = blockIdx.x >= a.side[0].blocks;
  const Side& s = a.side[keys];
  const uint32_t block = blockIdx.x - (keys ? a.side[0].blocks : 0);
  const int L = 1 << a.log_l, teams = QR_NT >> a.log_l;
  const int team = threadIdx.x >> a.log_l, slot = threadIdx.x & (L - 1);
  const int turned = a.R / (2 * E);                 // slots of turned pairs
  const bool held = slot < a.D / (2 * E);           // lanes past the row read slot 0 and write nothing
  const int at = held ? slot : 0;
  const bool turns = at < turned && s.pos;
  const int lo = at >= turned || NEIGHBOURS ? 2 * E * at : E * at;
  const int hi = at >= turned || NEIGHBOURS ? lo + E : lo + a.R / 2;
  F wa, wc, dwa, dwc;
#pragma unroll
  for (int e = 0; e < E; ++e) wa[e] = wc[e] = 1.f, dwa[e] = dwc[e] = 0.f;
  if (s.w) {
    if (a.w_f32) {
      typedef Pairs<float, E, NEIGHBOURS> PW;
      PW::split(Vec<float, E>::load((const float*)s.w + lo), Vec<float, E>::load((const float*)s.w + hi), wa, wc);
    } else {
      P::split(O::load((const T*)s.w + lo), O::load((const T*)s.w + hi), wa, wc);
    }
  }
  // every team of a workgroup takes the same turns; the last ones repeat a unit and write nothing
  for (int64_t u0 = (int64_t)block * teams; u0 < s.units; u0 += (int64_t)s.blocks * teams) {
    const bool live = u0 + team < s.units;
    const int64_t unit = live ? u0 + team : s.units - 1, token = unit / s.groups;
    const int h0 = (int)(unit - token * s.groups) * s.heads;
    const int64_t b = token / s.N, n = token - b * s.N;
    F cosv, sinv;
#pragma unroll
    for (int e = 0; e < E; ++e) cosv[e] = 1.f, sinv[e] = 0.f;
    if (turns) {
      const int64_t place = b * s.ps + n;
      const double p = a.pos64 ? (double)((const int64_t*)s.pos)[place] : (double)((const int32_t*)s.pos)[place];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double t = p * a.turns[E * at + e];
        const float turn = (float)(t - rint(t));
        float sn, cs;
        sine_cosine<T>(turn, sn, cs);
        sinv[e] = sn, cosv[e] = cs;
      }
    }
    const T* x = (const T*)s.x + b * s.xs[0] + n * s.xs[1];
    const T* dy = BWD ? (const T*)s.dy + b * s.ds[0] + n * s.ds[1] : nullptr;
    for (int i = 0; i < s.heads; i += AT_ONCE) {
      V xl[AT_ONCE], xh[AT_ONCE], gl[AT_ONCE], gh[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int64_t h = min(h0 + i + k, s.H - 1);
        xl[k] = O::load(x + h * s.xs[2] + lo), xh[k] = O::load(x + h * s.xs[2] + hi);
        if constexpr (BWD) gl[k] = O::load(dy + h * s.ds[2] + lo), gh[k] = O::load(dy + h * s.ds[2] + hi);
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int h = h0 + i + k;
        const bool mine = live && held && i + k < s.heads && h < s.H;
        F xa, xc;
        P::split(xl[k], xh[k], xa, xc);
        T* out = s.out ? (T*)s.out + (token * s.H + min(h, s.H - 1)) * a.D : nullptr;
        if constexpr (!BWD) {
          if (a.norm) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) sum += xa[e] * xa[e] + xc[e] * xc[e];
            const float r = 1.0f / sqrtf(team_sum(held ? sum : 0.f, a.log_l) * a.inv_d + a.eps);
            xa = xa * r * wa, xc = xc * r * wc;
          }
          if (mine) P::store(out + lo, out + hi, xa * cosv - xc * sinv, xc * cosv + xa * sinv);
        } else {
          F da, dc;
          P::split(gl[k], gh[k], da, dc);
          F ga = da * cosv + dc * sinv, gc = dc * cosv - da * sinv;
          if (a.norm) {
            float sum = 0.f, dot = 0.f;
            const F va = ga * wa, vc = gc * wc;
#pragma unroll
            for (int e = 0; e < E; ++e) {
              sum += xa[e] * xa[e] + xc[e] * xc[e];
              dot += va[e] * xa[e] + vc[e] * xc[e];
            }
            sum = team_sum(held ? sum : 0.f, a.log_l), dot = team_sum(held ? dot : 0.f, a.log_l);
            const float r = 1.0f / sqrtf(sum * a.inv_d + a.eps), m = dot * r * a.inv_d;
            xa *= r, xc *= r;
            if (mine) dwa += ga * xa, dwc += gc * xc;
            ga = (va - xa * m) * r, gc = (vc - xc * m) * r;
          }
          if (mine && out) P::store(out + lo, out + hi, ga, gc);
        }
      }
    }
  }
  if constexpr (BWD) {
    if (!s.partial) return;
    // the teams' sums, in team order
    __shared__ float sum[2 * E][QR_NT];
    F first, second;  // as the columns lie
    if constexpr (NEIGHBOURS) {
#pragma unroll
      for (int e = 0; e < E / 2; ++e)
        first[2 * e] = dwa[e], first[2 * e + 1] = dwc[e], second[2 * e] = dwa[E / 2 + e], second[2 * e + 1] = dwc[E / 2 + e];
    } else {
      first = dwa, second = dwc;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e][threadIdx.x] = first[e], sum[E + e][threadIdx.x] = second[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * E * L; i += QR_NT) {
      const int sl = i & (L - 1), e = i >> a.log_l;
      if (sl >= a.D / (2 * E)) continue;
      float t = 0.f;
      for (int k = 0; k < teams; ++k) t += sum[e][(k << a.log_l) + sl];
      const bool plain = sl >= turned || NEIGHBOURS;
      const int col = (e < E ? (plain ? 2 * E * sl : E * sl) : (plain ? 2 * E * sl + E : E * sl + a.R / 2)) + e % E;
      s.partial[(int64_t)block * a.D + col] = t;
    }
  }
}

// Heads a unit: as many as leave 2 workgroups a CU, so that the angles of a token are made seldom (3 x 1021
// tokens, 25 heads of 80, fp16: 13 us, with 8 workgroups a CU 18; 2 x 4096 of 32 heads of 128, bf16: 25 and 29)
void divide(Side& s, int64_t B, int teams) {
  const int64_t want = (int64_t)compute_units() * 2 * teams, rows = B * s.N * s.H;
  s.heads = (int)std::min<int64_t>(s.H, std::max<int64_t>(1, rows / want));
  s.groups = (s.H + s.heads - 1) / s.heads;
  s.units = B * s.N * s.groups;
}

// Elements of each half of a lane's share
int share(const gnn_qk_rotary_args& g) { return g.D % 16 == 0 && g.R % 16 == 0 ? 8 : 4; }

int log_team(const gnn_qk_rotary_args& g) {
  const int slots = (int)g.D / (2 * share(g));
  int l = 0;
  while ((1 << l) < slots) ++l;
  return l;
}

template <typename T, int E, bool NEIGHBOURS>
int launch(const RotaryArgs& a, bool bwd, uint32_t blocks, hipStream_t st) {
  if (bwd)
    hipLaunchKernelGGL((qk_norm_rotary_kernel<T, E, NEIGHBOURS, true>), dim3(blocks), dim3(QR_NT), 0, st, a);
  else
    hipLaunchKernelGGL((qk_norm_rotary_kernel<T, E, NEIGHBOURS, false>), dim3(blocks), dim3(QR_NT), 0, st, a);
  return (int)hipGetLastError();
}
template <typename T>
int launch(const RotaryArgs& a, int e, bool neighbours, bool bwd, uint32_t blocks, hipStream_t st) {
  if (e == 8) return neighbours ? launch<T, 8, true>(a, bwd, blocks, st) : launch<T, 8, false>(a, bwd, blocks, st);
  return neighbours ? launch<T, 4, true>(a, bwd, blocks, st) : launch<T, 4, false>(a, bwd, blocks, st);
}

}  // namespace

int64_t qk_rotary_parts(const gnn_qk_rotary_args& g, int side) {
  Side s{};
  s.N = g.N[side], s.H = (int)g.H[side];
  const int teams = QR_NT >> log_team(g);
  divide(s, g.B, teams);
  return std::max<int64_t>(1, std::min<int64_t>((s.units + teams - 1) / teams, (int64_t)compute_units() * 4));
}

int qk_rotary(const gnn_qk_rotary_args& g, bool bwd, hipStream_t st) {
  RotaryArgs a{};
  a.D = (int)g.D, a.R = (int)g.R, a.log_l = log_team(g);
  a.eps = g.eps, a.inv_d = 1.0f / (float)g.D;
  a.norm = g.norm != 0, a.pos64 = g.pos_bytes == 8, a.w_f32 = g.param_dtype == GNN_F32;
  for (int j = 0; j < a.R / 2; ++j) a.turns[j] = g.frequencies[j] * 0.15915494309189533577;  // 1 / (2 pi)
  const int teams = QR_NT >> a.log_l;
  int64_t blocks = 0;
  float* partial = g.partial;
  for (int k = 0; k < 2; ++k) {
    Side& s = a.side[k];
    s.N = g.N[k], s.H = (int)g.H[k];
    s.x = g.x[k], s.dy = g.dy[k], s.w = g.weight[k], s.pos = g.pos[k], s.out = g.out[k], s.ps = g.pos_stride[k];
    for (int i = 0; i < 3; ++i) s.xs[i] = g.x_stride[k][i], s.ds[i] = g.dy_stride[k][i];
    if (!g.B || !s.N || !s.H || (bwd && !s.out && !g.dweight[k])) continue;
    divide(s, g.B, teams);
    const int64_t n = bwd ? g.parts[k] : (s.units + teams - 1) / teams;
    blocks += n;
    if (blocks >= ((int64_t)1 << 31)) return set_error(GNN_ERR_UNSUPPORTED, "qk_norm_rotary: grid too large");
    s.blocks = (uint32_t)n;
    if (bwd && g.dweight[k]) s.partial = partial, partial += n * g.D;
  }
  if (!blocks) return GNN_OK;
  const int e = share(g);
  const bool neighbours = g.interleaved != 0;
  switch (g.dtype) {
    case GNN_BF16: return launch<bf16>(a, e, neighbours, bwd, (uint32_t)blocks, st);
    case GNN_F16: return launch<f16>(a, e, neighbours, bwd, (uint32_t)blocks, st);
    default: return launch<float>(a, e, neighbours, bwd, (uint32_t)blocks, st);
  }
}

}  // namespace gnn
