// Attention of queries over the states of another sequence, forward:
//   o[b,u,h,:] = sum_j softmax_j(x_j) v[b,j,h/G,:],  x_j = scale q[b,u,h,:].k[b,j,h/G,:] + bias[b,h,u,j] over kept keys,
// zero where a row keeps no key. The rows of a workgroup are queries of all heads that share a key head
// (cross_common.hpp).
//
// One pass over the keys with a running maximum and sum. The scores are formed transposed, S^T = K Q^T on 32x32x16
// MFMA, so that a lane holds one row and 16 keys of a half tile: statistics are scalars of a lane, and the
// probabilities feed O^T = V^T P^T from the registers where they are, V being read turned from LDS. Without a bias the
// scores stay as they are and scale log2(e) enters the exponent's FMA; with one, logits are formed in natural units and
// the maximum is subtracted first, so that biases down to the type's lowest value stay logits like others. The maximum
// moves only where a tile raises it by more than 8 log2 units (p <= 2^8 then). p is rounded to the operands' type for
// the second product, the sum adds it before that.
//
// Masked keys are selected away (not added to), and their rows of V are zeros in LDS: what they hold, NaN too, reaches
// nothing. Tiles without a kept key are not visited.
//
// Two forms by the number of rows:
//   4 waves of 32 rows each, all walking over the same tiles of 64 keys;
//   up to 32 rows (a decoded token): 4 waves that share the 32 rows and take 32 keys each of tiles of 128; their
//   maxima, sums and outputs meet in LDS at the end.
// Where these leave CUs idle the keys are split over workgroups, whose fp32 outputs a second kernel joins.
#include <algorithm>

#include "cross_common.hpp"

namespace gnn {

namespace {

using namespace cross;

constexpr int NT = 256;
constexpr float RISE = 8.f;  // log2 units
// log2 units of a logit's unit, as the kernels hold it
template <bool BIAS> constexpr float unit() { return BIAS ? LOG2E : 1.f; }

struct FwdArgs {
  Shape s;
  const void* q;
  const void* k;
  const void* v;
  const void* bias;
  const uint8_t* mask;
  void* o;
  float* stats;    // [B][H][U][2]: the reference maximum (+inf where no key is kept) and the log2 of the sum; or NULL
  float* part_o;   // [splits][B][U][H][D]
  float* part_ml;  // [splits][B][H][U][2]
  int64_t qs[3], ks[3], vs[3], bs[3], ms[2];
  float scale;  // of the scores: with a bias the caller's, otherwise times log2(e)
  int splits, tiles_per_split;
};

// WK waves share rows and divide keys (1 or 4)
template <typename T, int DP, int WK>
struct Cfg {
  static constexpr int SUBS = WK == 1 ? 2 : 1;    // half tiles of 32 keys a wave
  static constexpr int KT = 32 * SUBS * WK;       // keys a tile
  static constexpr int ROWS = 128 / WK;           // rows a workgroup
  static constexpr int NBUF = sizeof(T) == 2 && WK == 1 ? 2 : 1;
  static constexpr int TILE = KT * RowTile<T, DP>::PITCH;
  static constexpr int MERGE = WK == 1 ? 0 : 4 * 64 * (16 * (DP / 32) + 4) * 4;  // of the waves' results
  static constexpr int LDS = NBUF * 2 * TILE > MERGE ? NBUF * 2 * TILE : MERGE;
};

template <typename T, int PREC, int DP, int WK, bool BIAS>
__global__ __launch_bounds__(NT, sizeof(T) == 4 && DP == 128 ? 1 : 2) void cross_fwd_kernel(const FwdArgs a) {
  typedef Cfg<T, DP, WK> C;
  typedef RowTile<T, DP> Tile;
  typedef typename TypeOps<T>::V8 V8;
  __shared__ __align__(16) unsigned char smem[C::LDS];
  __shared__ int found[2];
  const Shape& s = a.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;

  // blocks of rows fastest: those of one key head share its K and V in an XCD's L2
  const uint32_t nrb = (uint32_t)(s.rows + C::ROWS - 1) / C::ROWS;
  uint32_t w = xcd_remap(blockIdx.x, gridDim.x);
  const int rb = w % nrb;
  w /= nrb;
  const int split = w % a.splits;
  w /= a.splits;
  const int hk = w % s.Hk, b = w / s.Hk;

  const int row = rb * C::ROWS + (WK == 1 ? wave * 32 : 0) + l32;
  const bool row_ok = row < s.rows;
  const int safe = min(row, s.rows - 1), u = safe / s.G, h = hk * s.G + safe % s.G;
  const T* qp = (const T*)a.q + b * a.qs[0] + u * a.qs[1] + h * a.qs[2];
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  const T* bp = BIAS ? (const T*)a.bias + b * a.bs[0] + h * a.bs[1] + u * a.bs[2] : nullptr;
  const uint8_t* mask = a.mask ? a.mask + b * a.ms[0] : nullptr;

  int key_end = min(s.V, (split + 1) * a.tiles_per_split * C::KT), key0 = split * a.tiles_per_split * C::KT;
  if (mask) live_range<NT>(mask, a.ms[1], key0, key_end, found);
  const int t_end = key0 < key_end ? (key_end + C::KT - 1) / C::KT : 0;

  V8 qf[DP / 16];
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const int d = 16 * kk + 8 * g;
    qf[kk] = load8_at(qp + (d < s.D ? d : 0));
    if (d >= s.D) qf[kk] = zero8<T>();
  }
  f32x16 o[DP / 32];
#pragma unroll
  for (int cc = 0; cc < DP / 32; ++cc) clear(o[cc]);
  float m = -INFINITY, sum = 0.f;

  Staged<T, DP, C::KT, NT> kreg, vreg;
  uint64_t live[(C::KT + 63) / 64], next_live[(C::KT + 63) / 64];
  // the words of the next tile from t on that keeps a key; t_end where there is none
  auto seek = [&](int t, uint64_t (&words)[(C::KT + 63) / 64]) {
    for (; t < t_end; ++t) {
      uint64_t any = 0;
#pragma unroll
      for (int i = 0; i < (C::KT + 63) / 64; ++i) any |= words[i] = live_keys(mask, a.ms[1], t * C::KT + 64 * i, s.V);
      if (any) break;
    }
    return t;
  };
  auto load = [&](int t) {
    kreg.load_rows(kp, a.ks[1], t * C::KT, s.V, s.D);
    vreg.load_rows(vp, a.vs[1], t * C::KT, s.V, s.D);
  };
  auto put = [&](int buf, const uint64_t (&words)[(C::KT + 63) / 64]) {
    unsigned char* st = smem + buf * 2 * C::TILE;
    bool whole = s.D == DP;
#pragma unroll
    for (int i = 0; i < (C::KT + 63) / 64; ++i) whole = whole && words[i] == ~0ull;
    if (whole) {  // uniform
      kreg.store(st);
      vreg.store(st + C::TILE);
      return;
    }
    kreg.store(st, s.D, [](int) { return true; });
    vreg.store(st + C::TILE, s.D, [&](int r) { return (words[r / 64] >> (r & 63) & 1) != 0; });
  };

  int t = seek(key0 / C::KT, live);
  if (t < t_end) {
    load(t);
    put(0, live);
  }
  __syncthreads();
  for (int buf = 0; t < t_end; buf ^= C::NBUF - 1) {
    const int next = seek(t + 1, next_live);
    if (next < t_end) load(next);
    const unsigned char* ks = smem + buf * 2 * C::TILE;
    const unsigned char* vs = ks + C::TILE;
    const int r0 = WK == 1 ? 0 : 32 * wave;  // this wave's keys of the tile
    f32x16 sc[C::SUBS];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int sub = 0; sub < C::SUBS; ++sub) {
      clear(sc[sub]);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
        Mma<T, PREC>::step(sc[sub], Tile::row8(ks, r0 + 32 * sub + l32, kk, g), qf[kk]);
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (BIAS) {
#pragma unroll
      for (int sub = 0; sub < C::SUBS; ++sub)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int key = t * C::KT + r0 + 32 * sub + 8 * q + 4 * g;
          const f32x4 bv = key < s.V ? load4_at(bp + key, s.V - key) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[sub][4 * q + e] = __builtin_fmaf(sc[sub][4 * q + e], a.scale, bv[e]);
        }
    }
#pragma unroll
    for (int sub = 0; sub < C::SUBS; ++sub) {
      const int at = r0 + 32 * sub;
      const uint32_t word = (uint32_t)(live[at / 64] >> (at & 63));
      if (word != ~0u) {  // uniform
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[sub][i] = word >> acc_row(i, g) & 1 ? sc[sub][i] : -INFINITY;
      }
    }
    float top = sc[0][0];
#pragma unroll
    for (int sub = 0; sub < C::SUBS; ++sub)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[sub][i]);
    top = pair_top(top) * (BIAS ? 1.f : a.scale);
    if (__any(top > m + RISE / unit<BIAS>())) {
      const float mn = fmaxf(m, top);
      const float alpha = fast_exp2(mn == -INFINITY ? 0.f : (m - mn) * unit<BIAS>());
      m = mn;
      sum *= alpha;
#pragma unroll
      for (int cc = 0; cc < DP / 32; ++cc)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[cc][i] *= alpha;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int sub = 0; sub < C::SUBS; ++sub) {
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sc[sub][i] = fast_exp2(BIAS ? (sc[sub][i] - base) * LOG2E : __builtin_fmaf(sc[sub][i], a.scale, -base));
        part[i % 4] += sc[sub][i];
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const V8 p = acc_frag<T>(sc[sub], kk);
#pragma unroll
        for (int cc = 0; cc < DP / 32; ++cc)
          Mma<T, PREC>::step(o[cc], Tile::turned8(vs, r0 + 32 * sub, kk, cc, lane), p);
      }
    }
    if constexpr (C::NBUF == 1) __syncthreads();
    if (next < t_end) put(C::NBUF == 1 ? 0 : buf ^ 1, next_live);
    __syncthreads();
    t = next;
#pragma unroll
    for (int i = 0; i < (C::KT + 63) / 64; ++i) live[i] = next_live[i];
  }
  sum = pair_sum(sum);

  if constexpr (WK > 1) {  // the waves' results, in wave order
    constexpr int LD = 16 * (DP / 32) + 4;  // floats a lane: 4 more keep the lanes on different banks
    float* mine = (float*)smem + (wave * 64 + lane) * LD;
#pragma unroll
    for (int cc = 0; cc < DP / 32; ++cc)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(mine + 16 * cc + 4 * q) =
            f32x4{o[cc][4 * q], o[cc][4 * q + 1], o[cc][4 * q + 2], o[cc][4 * q + 3]};
    mine[LD - 4] = m, mine[LD - 3] = sum;
    __syncthreads();
    if (wave >= DP / 32) return;
    // wave cc joins the columns 32 cc ..
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, ((float*)smem)[(k * 64 + lane) * LD + LD - 4]);
    float total = 0.f;
    f32x16 joined;
    clear(joined);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* from = (const float*)smem + (k * 64 + lane) * LD;
      const float f = fast_exp2(top == -INFINITY ? 0.f : (from[LD - 4] - top) * unit<BIAS>());
      total += f * from[LD - 3];
#pragma unroll
      for (int i = 0; i < 16; ++i) joined[i] += f * from[16 * wave + i];
    }
    m = top, sum = total;
    o[0] = joined;
  }
  if (!row_ok) return;
  const int64_t head = ((int64_t)b * s.U + u) * s.H + h, stat = ((int64_t)b * s.H + h) * s.U + u;
  const bool first = g == 0 && (WK == 1 || wave == 0);
  const float inv = a.splits > 1 ? 1.f : sum > 0.f ? 1.0f / sum : sum == 0.f ? 0.f : sum;  // NaN stays
  if (a.splits > 1) {
    if (first) {
      float* ml = a.part_ml + (split * (int64_t)s.B * s.H * s.U + stat) * 2;
      ml[0] = m, ml[1] = sum;
    }
  } else if (first && a.stats) {
    a.stats[2 * stat] = sum == 0.f ? INFINITY : m, a.stats[2 * stat + 1] = sum == 0.f ? 0.f : log2f(sum);
  }
  const int64_t each = (int64_t)s.B * s.U * s.H * s.D;
#pragma unroll
  for (int k = 0; k < (WK == 1 ? DP / 32 : 1); ++k) {
    const int cc = WK == 1 ? k : wave;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * cc + 8 * q + 4 * g;
      if (d >= s.D) continue;
      const f32x4 x = f32x4{o[k][4 * q], o[k][4 * q + 1], o[k][4 * q + 2], o[k][4 * q + 3]} * inv;
      if (a.splits > 1)
        *reinterpret_cast<f32x4*>(a.part_o + split * each + head * s.D + d) = x;
      else
        store4((T*)a.o + head * s.D + d, TypeOps<T>::from_f32(x));
    }
  }
}

// The splits of a row: 4 consecutive elements a thread
template <typename T, bool BIAS>
__global__ __launch_bounds__(NT) void cross_join_kernel(const FwdArgs a) {
  const Shape& s = a.s;
  const int per = s.D / 4;
  const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x, heads = (int64_t)s.B * s.U * s.H;
  const int64_t head = i / per;
  if (head >= heads) return;
  const int d = (int)(i - head * per) * 4, h = (int)(head % s.H);
  const int64_t bu = head / s.H, b = bu / s.U, u = bu - b * s.U, stat = (b * s.H + h) * s.U + u;
  float m = -INFINITY;
  for (int k = 0; k < a.splits; ++k) m = fmaxf(m, a.part_ml[(k * heads + stat) * 2]);
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.splits; ++k) {
    const float* ml = a.part_ml + (k * heads + stat) * 2;
    const float f = fast_exp2(m == -INFINITY ? 0.f : (ml[0] - m) * unit<BIAS>());
    sum += f * ml[1];
    o += f * *reinterpret_cast<const f32x4*>(a.part_o + (k * heads + head) * s.D + d);
  }
  const float inv = sum > 0.f ? 1.0f / sum : sum == 0.f ? 0.f : sum;
  store4((T*)a.o + head * s.D + d, TypeOps<T>::from_f32(o * inv));
  if (a.stats && d == 0)
    a.stats[2 * stat] = sum == 0.f ? INFINITY : m, a.stats[2 * stat + 1] = sum == 0.f ? 0.f : log2f(sum);
}

struct Plan {
  bool few;  // up to 32 rows
  int64_t blocks, splits, tiles_per_split;
};
Plan plan(const gnn_cross_attn_args& g) {
  Plan p{};
  const int64_t rows = g.U * (g.H / g.Hk);
  p.few = rows <= 32;
  const int64_t base = (p.few ? 1 : (rows + 127) / 128) * g.B * g.Hk, kt = p.few ? 128 : 64, tiles = (g.V + kt - 1) / kt;
  // two workgroups a CU where the keys allow it, of 4 tiles at least
  const int64_t want = std::max<int64_t>(1, 2 * (int64_t)compute_units() / base);
  const int64_t most = std::max<int64_t>(1, tiles / 4);
  p.tiles_per_split = (tiles + std::min(want, most) - 1) / std::min(want, most);
  p.splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
  p.blocks = base * p.splits;
  return p;
}

template <typename T, int PREC, int DP>
int launch(const FwdArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((uint32_t)p.blocks), blk(NT);
  if (p.few) {
    if (a.bias)
      hipLaunchKernelGGL((cross_fwd_kernel<T, PREC, DP, 4, true>), grid, blk, 0, st, a);
    else
      hipLaunchKernelGGL((cross_fwd_kernel<T, PREC, DP, 4, false>), grid, blk, 0, st, a);
  } else {
    if (a.bias)
      hipLaunchKernelGGL((cross_fwd_kernel<T, PREC, DP, 1, true>), grid, blk, 0, st, a);
    else
      hipLaunchKernelGGL((cross_fwd_kernel<T, PREC, DP, 1, false>), grid, blk, 0, st, a);
  }
  int rc = (int)hipGetLastError();
  if (rc == 0 && a.splits > 1) {
    const int64_t threads = (int64_t)a.s.B * a.s.U * a.s.H * (a.s.D / 4);
    const dim3 join((uint32_t)((threads + NT - 1) / NT));
    if (a.bias)
      hipLaunchKernelGGL((cross_join_kernel<T, true>), join, blk, 0, st, a);
    else
      hipLaunchKernelGGL((cross_join_kernel<T, false>), join, blk, 0, st, a);
    rc = (int)hipGetLastError();
  }
  return rc;
}

template <typename T, int PREC>
int run(const FwdArgs& a, const Plan& p, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (a.s.D <= 32) return launch<T, PREC, 32>(a, p, st);
    if (a.s.D > 64 && a.s.D <= 96) return launch<T, PREC, 96>(a, p, st);
  }
  if (a.s.D <= 64) return launch<T, PREC, 64>(a, p, st);
  return launch<T, PREC, 128>(a, p, st);
}

}  // namespace

size_t cross_attn_workspace_bytes(const gnn_cross_attn_args& g) {
  const Plan p = plan(g);
  return p.splits > 1 ? (size_t)p.splits * g.B * g.U * g.H * (g.D + 2) * sizeof(float) : 0;
}

int cross_attn_fwd(const gnn_cross_attn_args& g, hipStream_t st) {
  const Plan p = plan(g);
  if (p.blocks >= ((int64_t)1 << 31) || g.B * g.U * g.H >= ((int64_t)1 << 31))
    return set_error(GNN_ERR_UNSUPPORTED, "cross_attention: grid too large");
  FwdArgs a{};
  a.s = {(int)g.B, (int)g.U, (int)g.V, (int)g.H, (int)g.Hk, (int)(g.H / g.Hk), (int)g.D, (int)(g.U * (g.H / g.Hk))};
  a.q = g.q, a.k = g.k, a.v = g.v, a.bias = g.bias, a.mask = g.mask, a.o = g.o, a.stats = g.stats;
  for (int i = 0; i < 3; ++i) a.qs[i] = g.q_stride[i], a.ks[i] = g.k_stride[i], a.vs[i] = g.v_stride[i], a.bs[i] = g.bias_stride[i];
  for (int i = 0; i < 2; ++i) a.ms[i] = g.mask_stride[i];
  a.scale = g.bias ? g.scale : g.scale * LOG2E;
  a.splits = (int)p.splits, a.tiles_per_split = (int)p.tiles_per_split;
  if (p.splits > 1) {
    if (!g.workspace || g.workspace_bytes < cross_attn_workspace_bytes(g))
      return set_error(GNN_ERR_WORKSPACE, "cross_attention: workspace missing or too small");
    a.part_o = (float*)g.workspace;
    a.part_ml = a.part_o + p.splits * g.B * g.U * g.H * g.D;
  }
  switch (g.dtype) {
    case GNN_BF16: return run<bf16, PREC_NATIVE>(a, p, st);
    case GNN_F16: return run<f16, PREC_NATIVE>(a, p, st);
    default: return g.precision == GNN_PREC_BF16X3 ? run<float, PREC_BF16X3>(a, p, st) : run<float, PREC_IEEE>(a, p, st);
  }
}

}  // namespace gnn
