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
// the second product (in two parts where keys or rows are few), the sum adds it before that.
//
// Masked keys are selected away (not added to), and their rows of V are zeros in LDS: what they hold, NaN too, reaches
// nothing. Tiles without a kept key are not visited.
//
// Two forms by the number of rows:
//   4 waves of 32 rows each, all walking over the same tiles of 64 keys;
//   up to 32 rows (a decoded token): 4 waves that share the 32 rows and take 32 keys each of tiles of 128; their
//   maxima, sums and outputs meet in LDS at the end.
// Where these leave CUs idle the keys are split over workgroups, whose fp32 outputs a second kernel joins.
//
// 4096 x 8192, 32 heads of 128, bf16: 574 us of 550 GFLOP (441 at a large product's rate), the softmax's vector work beside
// the products. One query of 8191 keys, 8 sequences, 32 heads of 128 over 8: 41 us, K and V at 5 TB/s, and 4 for the joining.
#include <algorithm>
#include <cmath>
#include <type_traits>

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
  void* o_low;     // dense like o, what o's rounding left; or NULL
  float* stats;    // [B][H][U][2], what store_stats leaves of a row; or NULL
  float* part_o;   // [splits][B][U][H][D]
  float* part_ml;  // [splits][B][H][U][2]
  int64_t qs[3], ks[3], vs[3], bs[3], ms[2];
  float scale;  // of the scores: with a bias the caller's, otherwise times log2(e)
  int splits, tiles_per_split;
  bool fine;  // p in two parts
};

// WK waves share rows and divide keys (1 or 4); a wave has QW times 32 rows
template <typename T, int DP, int WK, int QW>
struct Cfg {
  static constexpr int SUBS = WK == 1 ? 2 : 1;    // half tiles of 32 keys a wave
  static constexpr int KT = 32 * SUBS * WK;       // keys a tile
  static constexpr int WORDS = (KT + 63) / 64;
  static constexpr int ROWS = 128 / WK * QW;      // rows a workgroup
  static constexpr int NBUF = sizeof(T) == 2 && WK == 1 ? 2 : 1;
  typedef RowTile<T, DP, BY_ROWS> KTile;
  typedef RowTile<T, DP, BY_COLUMNS> VTile;
  static constexpr int KBYTES = KT * KTile::PITCH, TILE = KBYTES + KT * VTile::PITCH;
  static constexpr int MERGE = WK == 1 ? 0 : 4 * 64 * (16 * (DP / 32) + 4) * 4;  // of the waves' results
  static constexpr int LDS = NBUF * TILE > MERGE ? NBUF * TILE : MERGE;
  static constexpr int WGS = sizeof(T) == 4 && DP > 64 ? 1 : 2;  // workgroups a CU
};

template <typename T>
__device__ __forceinline__ void store_out(const FwdArgs& a, int64_t at, const f32x4& x) {
  const auto y = TypeOps<T>::from_f32(x);
  store4((T*)a.o + at, y);
  if constexpr (sizeof(T) == 2)
    if (a.o_low) store4((T*)a.o_low + at, TypeOps<T>::from_f32(x - TypeOps<T>::to_f32(y)));
}

// What the backward needs of a row whose probabilities sum to `sum` beside the maximum m: m and the log2 of the sum; +inf
// and 0 where nothing is left; NaN twice where the row holds one. Of one key, whose logit the backward does not
// form, 0 and 0.
__device__ __forceinline__ void store_stats(const FwdArgs& a, int64_t at, float m, float sum) {
  a.stats[2 * at] = sum > 0.f ? (a.s.V == 1 ? 0.f : m) : sum == 0.f ? INFINITY : sum;
  a.stats[2 * at + 1] = sum == 0.f ? 0.f : log2f(sum);
}

template <typename T, int PREC, int DP, int WK, int QW, bool BIAS>
__global__ __launch_bounds__(NT, (Cfg<T, DP, WK, QW>::WGS)) void cross_fwd_kernel(const FwdArgs a) {
  typedef Cfg<T, DP, WK, QW> C;
  typedef typename C::KTile KTile;
  typedef typename C::VTile VTile;
  typedef typename TypeOps<T>::V8 V8;
  constexpr bool FINER = sizeof(T) == 2 && QW == 1;
  __shared__ __align__(16) unsigned char smem[C::LDS];
  __shared__ int found[2];
  const Shape& s = a.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;

  // blocks of rows fastest: those of one key head share its K and V in an XCD's L2; then the sequences, whose lengths
  // differ, so that every XCD has some of each
  const uint32_t nrb = (uint32_t)(s.rows + C::ROWS - 1) / C::ROWS;
  uint32_t w = xcd_remap(blockIdx.x, gridDim.x);
  const int rb = w % nrb;
  w /= nrb;
  const int split = w % a.splits;
  w /= a.splits;
  const int b = w % s.B, hk = w / s.B;

  int u[QW], h[QW];
  const int row0 = rb * C::ROWS + (WK == 1 ? wave * 32 * QW : 0) + l32;
#pragma unroll
  for (int i = 0; i < QW; ++i) {
    const int row = min(row0 + 32 * i, s.rows - 1);
    u[i] = row / s.G, h[i] = hk * s.G + row % s.G;
  }
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  const uint8_t* mask = a.mask ? a.mask + b * a.ms[0] : nullptr;

  int key_end = min(s.V, (split + 1) * a.tiles_per_split * C::KT), key0 = split * a.tiles_per_split * C::KT;
  if (mask) live_range<NT>(mask, a.ms[1], key0, key_end, found);
  const int t_end = key0 < key_end ? (key_end + C::KT - 1) / C::KT : 0;

  V8 qf[QW][DP / 16];
  f32x16 o[QW][DP / 32];
  float m[QW], sum[QW];
  const T* bp[QW];
#pragma unroll
  for (int i = 0; i < QW; ++i) {
    const T* qp = (const T*)a.q + b * a.qs[0] + u[i] * a.qs[1] + h[i] * a.qs[2];
    bp[i] = BIAS ? (const T*)a.bias + b * a.bs[0] + h[i] * a.bs[1] + u[i] * a.bs[2] : nullptr;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const int d = 16 * kk + 8 * g;
      qf[i][kk] = load8_at(qp + (d < s.D ? d : 0));
      if (d >= s.D) qf[i][kk] = zero8<T>();
    }
#pragma unroll
    for (int cc = 0; cc < DP / 32; ++cc) clear(o[i][cc]);
    m[i] = -INFINITY, sum[i] = 0.f;
  }

  Staged<T, DP, C::KT, NT> kreg, vreg;
  uint64_t live[C::WORDS], next_live[C::WORDS];
  // the words of the next tile from t on that keeps a key; t_end where there is none
  auto seek = [&](int t, uint64_t (&words)[C::WORDS]) {
    for (; t < t_end; ++t) {
      uint64_t any = 0;
#pragma unroll
      for (int i = 0; i < C::WORDS; ++i) any |= words[i] = live_keys(mask, a.ms[1], t * C::KT + 64 * i, s.V);
      if (any) break;
    }
    return t;
  };
  auto load = [&](int t) {
    kreg.load_rows(kp, a.ks[1], t * C::KT, s.V, s.D);
    vreg.load_rows(vp, a.vs[1], t * C::KT, s.V, s.D);
  };
  auto put = [&](int buf, const uint64_t (&words)[C::WORDS]) {
    unsigned char* st = smem + buf * C::TILE;
    bool whole = s.D == DP;
#pragma unroll
    for (int i = 0; i < C::WORDS; ++i) whole = whole && words[i] == ~0ull;
    if (whole) {  // uniform
      kreg.template store<KTile>(st);
      vreg.template store<VTile>(st + C::KBYTES);
      return;
    }
    kreg.template store<KTile>(st, s.D, [](int) { return true; });
    vreg.template store<VTile>(st + C::KBYTES, s.D, [&](int r) { return (words[r / 64] >> (r & 63) & 1) != 0; });
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
    const unsigned char* ks = smem + buf * C::TILE;
    const unsigned char* vs = ks + C::KBYTES;
    const int r0 = WK == 1 ? 0 : 32 * wave;  // this wave's keys of the tile
    HalfBias<T> bias[BIAS ? C::SUBS : 1][BIAS ? QW : 1];
    if constexpr (BIAS)
#pragma unroll
      for (int sub = 0; sub < C::SUBS; ++sub)
#pragma unroll
        for (int i = 0; i < QW; ++i) bias[sub][i].template load<false>(bp[i], t * C::KT + r0 + 32 * sub, s.V, g);
    f32x16 sc[C::SUBS][QW];
#pragma unroll
    for (int sub = 0; sub < C::SUBS; ++sub) {
#pragma unroll
      for (int i = 0; i < QW; ++i) clear(sc[sub][i]);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const V8 kf = KTile::row8(ks, r0 + 32 * sub + l32, kk, g);
#pragma unroll
        for (int i = 0; i < QW; ++i) Mma<T, PREC>::step(sc[sub][i], kf, qf[i][kk]);
      }
    }
    if constexpr (BIAS) {
#pragma unroll
      for (int sub = 0; sub < C::SUBS; ++sub)
#pragma unroll
        for (int i = 0; i < QW; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 bv = bias[sub][i].at(q);
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[sub][i][4 * q + e] = __builtin_fmaf(sc[sub][i][4 * q + e], a.scale, bv[e]);
          }
    }
    bool whole = true;
#pragma unroll
    for (int i = 0; i < C::WORDS; ++i) whole = whole && live[i] == ~0ull;
    if (!whole) {  // uniform
#pragma unroll
      for (int sub = 0; sub < C::SUBS; ++sub) {
        const int at = r0 + 32 * sub;
        const uint32_t word = (uint32_t)(live[at / 64] >> (at & 63));
#pragma unroll
        for (int i = 0; i < QW; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[sub][i][e] = word >> acc_row(e, g) & 1 ? sc[sub][i][e] : -INFINITY;
      }
    }
    float top[QW];
    bool rises = false;
#pragma unroll
    for (int i = 0; i < QW; ++i) {
      top[i] = sc[0][i][0];
#pragma unroll
      for (int sub = 0; sub < C::SUBS; ++sub)
#pragma unroll
        for (int e = 0; e < 16; ++e) top[i] = fmaxf(top[i], sc[sub][i][e]);
      top[i] = pair_top(top[i]) * (BIAS ? 1.f : a.scale);
      rises = rises || top[i] > m[i] + RISE / unit<BIAS>();
    }
    if (__any(rises)) {
#pragma unroll
      for (int i = 0; i < QW; ++i) {
        const float mn = fmaxf(m[i], top[i]);
        const float alpha = fast_exp2(mn == -INFINITY ? 0.f : (m[i] - mn) * unit<BIAS>());
        m[i] = mn;
        sum[i] *= alpha;
#pragma unroll
        for (int cc = 0; cc < DP / 32; ++cc)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[i][cc][e] *= alpha;
      }
    }
#pragma unroll
    for (int sub = 0; sub < C::SUBS; ++sub) {
      V8 p[QW][2];
#pragma unroll
      for (int i = 0; i < QW; ++i) {
        const float base = m[i] == -INFINITY ? 0.f : m[i];
        f32x16& x = sc[sub][i];
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x[e] = fast_exp2(BIAS ? (x[e] - base) * LOG2E : __builtin_fmaf(x[e], a.scale, -base));
          part[e % 4] += x[e];
        }
        sum[i] += (part[0] + part[1]) + (part[2] + part[3]);
        p[i][0] = acc_frag<T>(x, 0), p[i][1] = acc_frag<T>(x, 1);
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int cc = 0; cc < DP / 32; ++cc) {
          const V8 vf = VTile::turned8(vs, r0 + 32 * sub, kk, cc, lane);
#pragma unroll
          for (int i = 0; i < QW; ++i) Mma<T, PREC>::step(o[i][cc], vf, p[i][kk]);
        }
      if constexpr (FINER)
        if (a.fine)  // uniform; behind the products, not among them: 4096 x 8192, 32 heads of 128, took 582 us then, 563 so
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            const V8 low = low_frag<T>(sc[sub][0], kk, p[0][kk]);
#pragma unroll
            for (int cc = 0; cc < DP / 32; ++cc)
              Mma<T, PREC>::step(o[0][cc], VTile::turned8(vs, r0 + 32 * sub, kk, cc, lane), low);
          }
    }
    if constexpr (C::NBUF == 1) __syncthreads();
    if (next < t_end) put(C::NBUF == 1 ? 0 : buf ^ 1, next_live);
    __syncthreads();
    t = next;
#pragma unroll
    for (int i = 0; i < C::WORDS; ++i) live[i] = next_live[i];
  }
#pragma unroll
  for (int i = 0; i < QW; ++i) sum[i] = pair_sum(sum[i]);

  if constexpr (WK > 1) {  // the waves' results, in wave order
    static_assert(QW == 1, "shared rows");
    constexpr int LD = 16 * (DP / 32) + 4;  // floats a lane: 4 more keep the lanes on different banks
    float* mine = (float*)smem + (wave * 64 + lane) * LD;
#pragma unroll
    for (int cc = 0; cc < DP / 32; ++cc)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(mine + 16 * cc + 4 * q) =
            f32x4{o[0][cc][4 * q], o[0][cc][4 * q + 1], o[0][cc][4 * q + 2], o[0][cc][4 * q + 3]};
    mine[LD - 4] = m[0], mine[LD - 3] = sum[0];
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
    m[0] = top, sum[0] = total;
    o[0][0] = joined;
  }
  const int64_t each = (int64_t)s.B * s.U * s.H * s.D;
#pragma unroll
  for (int i = 0; i < QW; ++i) {
    if (row0 + 32 * i >= s.rows) break;
    const int64_t head = ((int64_t)b * s.U + u[i]) * s.H + h[i], stat = ((int64_t)b * s.H + h[i]) * s.U + u[i];
    const bool first = g == 0 && (WK == 1 || wave == 0);
    const float inv = a.splits > 1 ? 1.f : sum[i] > 0.f ? 1.0f / sum[i] : sum[i] == 0.f ? 0.f : sum[i];  // NaN stays
    if (a.splits > 1) {
      if (first) {
        float* ml = a.part_ml + (split * (int64_t)s.B * s.H * s.U + stat) * 2;
        ml[0] = m[i], ml[1] = sum[i];
      }
    } else if (first && a.stats) {
      store_stats(a, stat, m[i], sum[i]);
    }
#pragma unroll
    for (int k = 0; k < (WK == 1 ? DP / 32 : 1); ++k) {
      const int cc = WK == 1 ? k : wave;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = 32 * cc + 8 * q + 4 * g;
        if (d >= s.D) continue;
        const f32x16& v = o[i][k];
        const f32x4 x = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]} * inv;
        if (a.splits > 1)
          *reinterpret_cast<f32x4*>(a.part_o + split * each + head * s.D + d) = x;
        else
          store_out<T>(a, head * s.D + d, x);
      }
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
  // 8 splits at a time, no load in a branch: past the last one its copies, with no weight
  float m = -INFINITY, sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < a.splits; k0 += 8) {
    float mk[8], lk[8];
    f32x4 ok[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = min(k0 + i, a.splits - 1);
      mk[i] = a.part_ml[(k * heads + stat) * 2], lk[i] = a.part_ml[(k * heads + stat) * 2 + 1];
      ok[i] = *reinterpret_cast<const f32x4*>(a.part_o + (k * heads + head) * s.D + d);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, mk[i]);
    const float old = fast_exp2(top == -INFINITY ? 0.f : (m - top) * unit<BIAS>());
    sum *= old, o *= old, m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = k0 + i < a.splits ? fast_exp2(top == -INFINITY ? 0.f : (mk[i] - top) * unit<BIAS>()) : 0.f;
      sum += f * lk[i];
      o += f * ok[i];
    }
  }
  const float inv = sum > 0.f ? 1.0f / sum : sum == 0.f ? 0.f : sum;
  store_out<T>(a, head * s.D + d, o * inv);
  if (a.stats && d == 0) store_stats(a, stat, m, sum);
}

// Few: up to 32 rows (8 x 1 x 4096, 32 heads of 64 over 8, bf16: 13.2 us, in the other form 19.0).
// Wide: 64 rows a wave, so that a fragment of K and V serves two products, where the registers hold them: up to 64 columns,
// with a bias 32 (4 x 2048 x 1400, 16 heads, bf16: of 64 59 us and 67, with a bias 112 and 107; of 32 46 and 47, with a bias
// 80 and 93; of 128 twice as long), and two workgroups a CU are left (half the batch of 64: 49 and 36).
struct Plan {
  bool few;
  bool wide;
  int64_t blocks, splits, tiles_per_split;
};
Plan plan(const gnn_cross_attn_args& g) {
  Plan p{};
  const int64_t rows = g.U * (g.H / g.Hk);
  p.few = rows <= 32;
  p.wide = g.dtype != GNN_F32 && g.D <= (g.bias ? 32 : 64) && g.V > FINE && (rows + 255) / 256 * g.B * g.Hk >= 2 * (int64_t)compute_units();
  const int64_t per = p.wide ? 256 : 128, base = (p.few ? 1 : (rows + per - 1) / per) * g.B * g.Hk, kt = p.few ? 128 : 64, tiles = (g.V + kt - 1) / kt;
  // The split of the keys that ends first, in us: rounds of workgroups (two a CU; in fp32 one where the products bound
  // it or LDS holds one), each a start and its tiles, and with several splits the second kernel, its launch and each
  // split's sums written and read. One query of 2048 keys, 2 sequences, 8 heads of 64, bf16: 8.9 us with two tiles a
  // split, with four 10.6; 300 queries of 8192 keys, 4 heads of 128: 25.2 with eight, with four 28.9.
  const bool f32 = g.dtype == GNN_F32;
  const int64_t places = (f32 && (!p.few || g.D > 64) ? 1 : 2) * (int64_t)compute_units();
  const double start = 3, tile = f32 ? 1.7 * ((g.D + 31) / 32) / (p.few ? 2 : 1) : 0.7, launch = 4;
  const double sums = 0.1 + (double)g.B * g.U * g.H * g.D * 8 / 5e6;
  // none, whole rounds, and where the tiles' and the sums' time are balanced
  const int64_t tries[] = {1, places / base, 2 * places / base, 3 * places / base, (int64_t)std::sqrt((double)tiles * tile / sums)};
  double best = 0;
  for (const int64_t want : tries) {
    const int64_t most = std::max<int64_t>(1, std::min(want, tiles));
    const int64_t each = (tiles + most - 1) / most, splits = (tiles + each - 1) / each;
    const double rounds = (double)((base * splits + places - 1) / places);
    const double time = rounds * (start + (double)each * tile) + (splits > 1 ? launch + (double)splits * sums : 0);
    if (best == 0 || time < best) best = time, p.splits = splits, p.tiles_per_split = each;
  }
  p.blocks = base * p.splits;
  return p;
}

template <typename T, int PREC, int DP>
int launch(const FwdArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((uint32_t)p.blocks), blk(NT);
  auto go = [&](auto bias) {
    constexpr bool BIAS = decltype(bias)::value;
    if (p.few) {
      hipLaunchKernelGGL((cross_fwd_kernel<T, PREC, DP, 4, 1, BIAS>), grid, blk, 0, st, a);
      return;
    }
    if constexpr (sizeof(T) == 2 && DP <= (BIAS ? 32 : 64))
      if (p.wide) {
        hipLaunchKernelGGL((cross_fwd_kernel<T, PREC, DP, 1, 2, BIAS>), grid, blk, 0, st, a);
        return;
      }
    hipLaunchKernelGGL((cross_fwd_kernel<T, PREC, DP, 1, 1, BIAS>), grid, blk, 0, st, a);
  };
  if (a.bias)
    go(std::true_type{});
  else
    go(std::false_type{});
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
  if (a.s.D <= 32) return launch<T, PREC, 32>(a, p, st);
  if (a.s.D <= 64) return launch<T, PREC, 64>(a, p, st);
  if (a.s.D <= 96) return launch<T, PREC, 96>(a, p, st);
  return launch<T, PREC, 128>(a, p, st);
}

}  // namespace

size_t cross_attn_workspace_bytes(const gnn_cross_attn_args& g) {
  const Plan p = plan(g);
  return p.splits > 1 ? (size_t)p.splits * g.B * g.U * g.H * (g.D + 2) * sizeof(float) : 0;
}

int cross_attn_fwd(const gnn_cross_attn_args& g, hipStream_t st) {
  const Plan p = plan(g);
  if (p.blocks >= ((int64_t)1 << 31))
    return set_error(GNN_ERR_UNSUPPORTED, "cross_attention: grid too large");
  FwdArgs a{};
  a.s = {(int)g.B, (int)g.U, (int)g.V, (int)g.H, (int)g.Hk, (int)(g.H / g.Hk), (int)g.D, (int)(g.U * (g.H / g.Hk))};
  a.q = g.q, a.k = g.k, a.v = g.v, a.bias = g.bias, a.mask = g.mask, a.o = g.o, a.o_low = g.o_low, a.stats = g.stats;
  for (int i = 0; i < 3; ++i) a.qs[i] = g.q_stride[i], a.ks[i] = g.k_stride[i], a.vs[i] = g.v_stride[i], a.bs[i] = g.bias_stride[i];
  for (int i = 0; i < 2; ++i) a.ms[i] = g.mask_stride[i];
  // One key has the weight 1 at any scale: at 1 its score less the maximum is an exact 0
  a.scale = g.bias ? g.scale : g.V == 1 ? 1.f : g.scale * LOG2E;
  // Few keys, and few rows, which the keys' bytes bound: 8 x 1 x 8191, 32 heads of 128 over 8, bf16: 45.4 us, with p in one
  // part 45.0, and the output 1.35 times as far off
  a.fine = g.V <= FINE || p.few;
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
