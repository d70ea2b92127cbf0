// Backward of attention over the states of another sequence (cross_fwd.hip). With x the logits, m and l the reference
// maximum and the log2 of the sum that the forward leaves of each row, and P = 2^((x - m) log2(e) - l) (as one number,
// m + l would lose l beside the lowest values of a type):
//   dV_j = sum_r P_rj dO_r,   dP_rj = dO_r . v_j,   Delta_r = dO_r . O_r,   dS_rj = P_rj (dP_rj - Delta_r),
//   dQ_r = scale sum_j dS_rj k_j,   dK_j = scale sum_r dS_rj q_r,   dbias = dS (summed over a batch that shares it).
// Rows r are the queries of all heads that share a key head, so that dK and dV of a shared head are one sum.
//
// Every sum has one owner and one order; S and dP are formed by each of the three that need them:
//   dq_block    the forward's layout (a lane holds a row and 16 keys): the dS^T accumulator is the operand of
//               dQ^T += K^T dS^T as it stands, K being read turned from LDS; it also writes dbias where every sequence
//               has its own.
//   dkdv_block  keys on the lanes, a wave 32 of them; tiles of 64 rows of Q and dO in LDS, read plain for S and dP and
//               turned for dV^T += dO^T P and dK^T += Q^T dS.
//   dbias_block a bias for all sequences: a tile of 128 rows x 64 keys of one head group walks over the batch.
// Delta comes from a kernel of its own, so that the three are workgroups of one launch (dk and dv, the longest, first)
// whose ends fill each other's: 16 heads, 4 x 2048 x 1400, 64 columns. In 16 bits and more columns dk and dv take all of a
// CU's registers and go alone, dQ after them. Where one of the first two leaves CUs idle its loop is split over workgroups,
// whose fp32 sums are added in order.
// P and dS are rounded to the operands' type for the products behind them (dS in two parts for dQ of few keys and short
// heads), and Delta takes what the rounding of O left with it.
//
// fp16's range: P is held 2^10 times as large for dV, or a row spread over 10^5 keys would fall below the normal range.
// dS falls sooner, with the output gradient, and as much above 1 it would leave the range upwards. |dS_rj| is at most
// 2 |dO_r| max_j |v_j|, and dS is held at the power of two that brings this bound into 2^14 .. 2^15: each row's own for dQ,
// where it goes into the exponent of P and out with the store, the largest of all rows for dK, whose sums go over rows.
// The lengths |dO_r| come with Delta, the longest v_j from further workgroups of that kernel. (16384 keys, dO of 2^-8: dQ is
// off by 4.1e-4, 5.4e-3 unscaled, the storing alone by 3.5e-4; one factor for all calls would overflow beside large
// gradients. 4 x 2048 x 1400, 16 heads of 64: 214 us, 205 unscaled.)
//
// 4 x 2048 x 1400, 16 heads of 64, bf16: 191 to 205 us (card by card) for five products of 19 GFLOP (77 at a large product's rate), of
// which S and dP are formed twice. The matrix units are busy 31% of the time, the vector units 41%, LDS 42%: 212 registers leave
// two waves a SIMD, too few to keep all three busy at once.
#include <algorithm>
#include <type_traits>

#include "cross_common.hpp"

namespace gnn {

namespace {

using namespace cross;

constexpr int NT = 256;
// Keys a tile (dQ, dbias), rows a tile (dK, dV). fp32 with more than 64 columns holds 128 registers of operands and 128 of
// sums a lane: of 64 rows, 64 more on their way to LDS were spilled.
constexpr int tile_of(bool f32, int D) { return f32 && D > 64 ? 32 : 64; }

struct BwdArgs {
  Shape s;
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  const void* o_low;  // dense, or NULL
  const void* dout;
  const void* bias;
  const uint8_t* mask;
  const float* stats;  // [B][H][U][2]
  float* delta;      // [B][H][U]
  float* length;     // fp16: |dO| of each row, [B][H][U]
  float* top;        // fp16: the longest kept v_j of each part of the keys, [B][Hk][v_parts]
  int v_parts;
  void* dq;
  void* dk;
  void* dv;
  void* dbias;       // [B or 1][H][U][V]
  float* part_q;     // [q_splits][B][U][H][D], or NULL
  float* part_k;     // [k_splits][2][B][V][Hk][D], or NULL
  int64_t qs[3], ks[3], vs[3], os[3], ds[3], bs[3], ms[2];
  float scale, logit_scale;  // the caller's; without a bias times log2(e)
  int q_splits, q_tiles;  // tiles of keys a split
  int k_splits, k_tiles;  // tiles of rows a split
  uint32_t delta_blocks, q_blocks, k_blocks, b_blocks;
  bool shared_bias;
  bool q_first;  // the workgroups of dQ before those of dK and dV
};

template <typename T> constexpr bool RANGED = false;  // operands held at powers of two
template <> constexpr bool RANGED<f16> = true;
constexpr int P_LOG = 10;  // of P in dV, where RANGED

// Of dS below `bound`; 0 where nothing or no number bounds it
__device__ __forceinline__ int ds_log(float bound) {
  return bound > 0.f && bound < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(bound) : 0;
}
__device__ __forceinline__ float wave_top(float x) {
#pragma unroll
  for (int k = 1; k < 64; k *= 2) x = fmaxf(x, __shfl_xor(x, k));
  return x;
}
// The longest v_j of a key head
__device__ __forceinline__ float longest_value(const BwdArgs& a, int b, int hk) {
  return wave_top(a.top[((int64_t)b * a.s.Hk + hk) * a.v_parts + min((int)(threadIdx.x & 63), a.v_parts - 1)]);
}

// Fragments of one row of a lane, zeros past D
template <typename T, int DP>
__device__ __forceinline__ void load_row(typename TypeOps<T>::V8 (&f)[DP / 16], const T* p, int D, int g) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const int d = 16 * kk + 8 * g;
    f[kk] = load8_at(p + (d < D ? d : 0));
    if (d >= D) f[kk] = zero8<T>();
  }
}

// A row's part of the exponent: with a bias m and l of 2^((score scale + bias - m) log2(e) - l), without one, where scale
// and m are in log2 units, their sum.
template <bool BIAS>
__device__ __forceinline__ float probability(float score, float scale, float bias, float m, float l) {
  if constexpr (BIAS) return fast_exp2(__builtin_fmaf(__builtin_fmaf(score, scale, bias) - m, LOG2E, -l));
  return fast_exp2(__builtin_fmaf(score, scale, -m));
}
template <bool BIAS>
__device__ __forceinline__ void row_stats(const float* stats, float& m, float& l) {
  m = stats[0], l = stats[1];
  if constexpr (!BIAS) m += l;
}

// dS^T = P (dP - Delta) of one half tile of 32 keys for the lane's row. `word`: the kept keys of the half tile; `dead`:
// some row of the wave has none (m is +inf): zeros there, whatever its output gradient holds.
template <typename T, int PREC, int DP, bool BIAS>
__device__ __forceinline__ void half_tile(f32x16& dp, const unsigned char* ks, const unsigned char* vs, int at,
                                          const typename TypeOps<T>::V8 (&qf)[DP / 16],
                                          const typename TypeOps<T>::V8 (&df)[DP / 16], const T* bias_row, int key0, int V,
                                          float scale, float m, float l, const f32x16& minus_delta, uint32_t word,
                                          bool dead) {
  typedef RowTile<T, DP> Tile;
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  HalfBias<T> bias;
  if constexpr (BIAS) bias.template load<false>(bias_row, key0, V, g);
  f32x16 sc;
  clear(sc);
  dp = minus_delta;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    Mma<T, PREC>::step(sc, Tile::row8(ks, at + l32, kk, g), qf[kk]);
    Mma<T, PREC>::step(dp, Tile::row8(vs, at + l32, kk, g), df[kk]);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f32x4 add = {0.f, 0.f, 0.f, 0.f};
    if constexpr (BIAS) add = bias.at(q);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * q + e;
      dp[i] *= probability<BIAS>(sc[i], scale, add[e], m, l);
    }
  }
  if (word != ~0u || dead) {  // uniform
    const uint32_t kept = m == INFINITY ? 0u : word;
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] = kept >> acc_row(i, g) & 1 ? dp[i] : 0.f;
  }
}

// ------------------------------------------------------------------------------------ Delta
__device__ __forceinline__ float sum8(const f32x8& x) { return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])); }

// The longest kept v_j of one part of a key head's keys; 2^LOG lanes of 8 elements a row
constexpr int KEYS_A_PART = 256, MAX_PARTS = 64;
template <typename T, int LOG>
__device__ __forceinline__ void longest_of_part(const BwdArgs& a, uint32_t block) {
  constexpr int AT_ONCE = 4, ROWS = NT >> LOG;
  __shared__ float tops[NT / 64];
  const Shape& s = a.s;
  const int part = block % a.v_parts, hk = block / a.v_parts % s.Hk, b = block / a.v_parts / s.Hk;
  const int each = (s.V + a.v_parts - 1) / a.v_parts, end = min(s.V, (part + 1) * each);
  const int d = (int)(threadIdx.x & ((1 << LOG) - 1)) * 8;
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2] + (d < s.D ? d : 0);
  const uint8_t* mask = a.mask ? a.mask + b * a.ms[0] : nullptr;
  float top = 0.f;
  for (int k0 = part * each + ((int)threadIdx.x >> LOG); k0 < end; k0 += AT_ONCE * ROWS) {
    f32x8 x[AT_ONCE];
    bool kept[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int64_t key = min(k0 + i * ROWS, end - 1);
      x[i] = TypeOps<T>::to_f32(load8_at(vp + key * a.vs[1]));
      kept[i] = !mask || mask[key * a.ms[1]] != 0;
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      float sum = d < s.D ? sum8(x[i] * x[i]) : 0.f;
#pragma unroll
      for (int k = 1; k < (1 << LOG); k *= 2) sum += __shfl_xor(sum, k);
      if (kept[i]) top = fmaxf(top, sum);
    }
  }
  top = wave_top(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) a.top[block] = sqrtf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
}

// 2^LOG lanes of 8 elements a row
template <typename T, int LOG>
__global__ __launch_bounds__(NT) void cross_delta_kernel(const BwdArgs a) {
  const Shape& s = a.s;
  if constexpr (RANGED<T>)
    if (blockIdx.x >= a.delta_blocks) return longest_of_part<T, LOG>(a, blockIdx.x - a.delta_blocks);
  const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x, heads = (int64_t)s.B * s.U * s.H;
  const int64_t head = min(i >> LOG, heads - 1);
  const int d = (int)(i & ((1 << LOG) - 1)) * 8, h = (int)(head % s.H);
  const int64_t bu = head / s.H, b = bu / s.U, u = bu - b * s.U;
  float sum = 0.f, square = 0.f;
  if (d < s.D) {
    f32x8 o = TypeOps<T>::to_f32(load8_at((const T*)a.o + b * a.os[0] + u * a.os[1] + h * a.os[2] + d));
    if (a.o_low) o += TypeOps<T>::to_f32(load8_at((const T*)a.o_low + head * s.D + d));
    const f32x8 x = TypeOps<T>::to_f32(load8_at((const T*)a.dout + b * a.ds[0] + u * a.ds[1] + h * a.ds[2] + d));
    sum = sum8(o * x);
    if constexpr (RANGED<T>) square = sum8(x * x);
  }
#pragma unroll
  for (int k = 1; k < (1 << LOG); k *= 2) {
    sum += __shfl_xor(sum, k);
    if constexpr (RANGED<T>) square += __shfl_xor(square, k);
  }
  if (d == 0 && i >> LOG < heads) {
    const int64_t stat = (b * s.H + h) * s.U + u;
    a.delta[stat] = sum;
    if constexpr (RANGED<T>) a.length[stat] = sqrtf(square);
  }
}

// LDS of a workgroup
template <typename T, int DP>
struct Lds {
  static constexpr int NBUF = sizeof(T) == 2 ? 2 : 1;
  static constexpr int KT = tile_of(sizeof(T) == 4, DP);
  static constexpr uint64_t ALL = KT == 64 ? ~0ull : ~0u;  // a tile's keys
  static constexpr int TILE = KT * RowTile<T, DP>::PITCH;
  __align__(16) unsigned char tile[NBUF * 2 * TILE];
  __align__(16) float m[NBUF][KT], l[NBUF][KT], minus_delta[NBUF][KT];
  int64_t bias_at[NBUF][KT];
  int found[2];
};

// -------------------------------------------------------------------------------------- dQ
// FINER: dS in two parts. 16 bits, 128 columns: the 256 registers of two waves a SIMD do not hold it all, 9 are kept in
// scratch, with a bias 45 (fp16: 10 and 55).
template <typename T, int PREC, int DP, bool BIAS, bool FINER>
__device__ __forceinline__ void dq_block(const BwdArgs& a, Lds<T, DP>& lds, uint32_t block) {
  typedef RowTile<T, DP> Tile;
  typedef typename TypeOps<T>::V8 V8;
  constexpr int TILE = Lds<T, DP>::TILE, NBUF = Lds<T, DP>::NBUF, KT = Lds<T, DP>::KT;
  unsigned char* smem = lds.tile;
  const Shape& s = a.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  const uint32_t nrb = (uint32_t)(s.rows + 127) / 128;
  uint32_t w = xcd_remap(block, a.q_blocks);
  const int rb = w % nrb;
  w /= nrb;
  const int split = w % a.q_splits;
  w /= a.q_splits;
  const int b = w % s.B, hk = w / s.B;
  const int row = rb * 128 + wave * 32 + l32;
  const bool row_ok = row < s.rows;
  const int safe = min(row, s.rows - 1), u = safe / s.G, h = hk * s.G + safe % s.G;
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  const T* bias_row = BIAS ? (const T*)a.bias + b * a.bs[0] + h * a.bs[1] + u * a.bs[2] : nullptr;
  const uint8_t* mask = a.mask ? a.mask + b * a.ms[0] : nullptr;
  const int64_t stat = ((int64_t)b * s.H + h) * s.U + u;

  V8 qf[DP / 16], df[DP / 16];
  load_row<T, DP>(qf, (const T*)a.q + b * a.qs[0] + u * a.qs[1] + h * a.qs[2], s.D, g);
  load_row<T, DP>(df, (const T*)a.dout + b * a.ds[0] + u * a.ds[1] + h * a.ds[2], s.D, g);
  float m, l;
  row_stats<BIAS>(a.stats + 2 * stat, m, l);
  const bool dead = __any(m == INFINITY);
  float undo = 1.f;  // of dS's power of two
  if constexpr (RANGED<T>) {
    const int log = ds_log(2.f * a.length[stat] * longest_value(a, b, hk));
    (BIAS ? l : m) -= (float)log;
    undo = ldexpf(1.f, -log);
  }
  f32x16 minus_delta;  // what the sums of dP start from
  fill(minus_delta, -a.delta[stat]);
  // own bias: every tile is visited, so that what no row keeps gets its zeros
  T* dbias = BIAS && a.dbias && !a.shared_bias ? (T*)a.dbias + stat * s.V : nullptr;
  int key_end = min(s.V, (split + 1) * a.q_tiles * KT), key0 = split * a.q_tiles * KT;
  if (mask && !dbias) live_range<NT>(mask, a.ms[1], key0, key_end, lds.found);
  const int t_end = key0 < key_end ? (key_end + KT - 1) / KT : 0;

  f32x16 dq[DP / 32];
#pragma unroll
  for (int cc = 0; cc < DP / 32; ++cc) clear(dq[cc]);
  Staged<T, DP, KT, NT> kreg, vreg;
  auto seek = [&](int t, uint64_t& word) {
    for (; t < t_end; ++t) {
      word = live_keys(mask, a.ms[1], t * KT, s.V) & Lds<T, DP>::ALL;
      if (word || dbias) break;
    }
    return t;
  };
  auto load = [&](int t) {
    kreg.load_rows(kp, a.ks[1], t * KT, s.V, s.D);
    vreg.load_rows(vp, a.vs[1], t * KT, s.V, s.D);
  };
  auto put = [&](int buf, uint64_t word) {  // what masked keys hold, NaN too, meets only zeros
    unsigned char* st = smem + buf * 2 * TILE;
    if (s.D == DP && word == Lds<T, DP>::ALL) {  // uniform
      kreg.store(st);
      vreg.store(st + TILE);
      return;
    }
    kreg.store(st, s.D, [&](int r) { return (word >> r & 1) != 0; });
    vreg.store(st + TILE, s.D, [&](int r) { return (word >> r & 1) != 0; });
  };
  uint64_t live = 0, next_live = 0;
  int t = seek(key0 / KT, live);
  if (t < t_end) {
    load(t);
    put(0, live);
  }
  __syncthreads();
  for (int buf = 0; t < t_end; buf ^= NBUF - 1) {
    const int next = seek(t + 1, next_live);
    if (next < t_end) load(next);
    const unsigned char* ks = smem + buf * 2 * TILE;
    if (sizeof(T) == 2 || rb * 128 + wave * 32 < s.rows)  // uniform; a wave without rows only stages (in 16 bits the branch costs more)
#pragma unroll
    for (int sub = 0; sub < KT / 32; ++sub) {
      f32x16 ds;
      half_tile<T, PREC, DP, BIAS>(ds, ks, ks + TILE, 32 * sub, qf, df, bias_row, t * KT + 32 * sub, s.V, a.logit_scale, m, l,
                                   minus_delta, (uint32_t)(live >> (32 * sub)), dead);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const V8 f = acc_frag<T>(ds, kk);
        V8 low;
        if constexpr (FINER) low = low_frag<T>(ds, kk, f);
#pragma unroll
        for (int cc = 0; cc < DP / 32; ++cc) {
          const V8 kf = Tile::turned8(ks, 32 * sub, kk, cc, lane);
          Mma<T, PREC>::step(dq[cc], kf, f);
          if constexpr (FINER) Mma<T, PREC>::step(dq[cc], kf, low);
        }
      }
      if constexpr (BIAS) {
        if (dbias && row_ok)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int key = t * KT + 32 * sub + 8 * q + 4 * g;
            if (key < s.V) store4_at(dbias + key, f32x4{ds[4 * q], ds[4 * q + 1], ds[4 * q + 2], ds[4 * q + 3]} * undo, s.V - key);
          }
      }
    }
    if constexpr (NBUF == 1) __syncthreads();
    if (next < t_end) put(NBUF == 1 ? 0 : buf ^ 1, next_live);
    __syncthreads();
    t = next, live = next_live;
  }
  if (!row_ok) return;
  const int64_t head = ((int64_t)b * s.U + u) * s.H + h, each = (int64_t)s.B * s.U * s.H * s.D;
#pragma unroll
  for (int cc = 0; cc < DP / 32; ++cc)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * cc + 8 * q + 4 * g;
      if (d >= s.D) continue;
      const f32x4 x = f32x4{dq[cc][4 * q], dq[cc][4 * q + 1], dq[cc][4 * q + 2], dq[cc][4 * q + 3]} * (a.scale * undo);
      if (a.part_q)
        *reinterpret_cast<f32x4*>(a.part_q + split * each + head * s.D + d) = x;
      else
        store4((T*)a.dq + head * s.D + d, TypeOps<T>::from_f32(x));
    }
}

// ---------------------------------------------------------------------------------- dK, dV
template <typename T, int PREC, int DP, bool BIAS>
__device__ __forceinline__ void dkdv_block(const BwdArgs& a, Lds<T, DP>& lds, uint32_t block) {
  typedef RowTile<T, DP> Tile;
  typedef typename TypeOps<T>::V8 V8;
  constexpr int TILE = Lds<T, DP>::TILE, NBUF = Lds<T, DP>::NBUF, KT = Lds<T, DP>::KT;
  unsigned char* smem = lds.tile;
  const Shape& s = a.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  const uint32_t nkb = (uint32_t)(s.V + 127) / 128;
  uint32_t w = xcd_remap(block, a.k_blocks);
  const int kb = w % nkb;
  w /= nkb;
  const int split = w % a.k_splits;
  w /= a.k_splits;
  const int b = w % s.B, hk = w / s.B;
  const int key = kb * 128 + wave * 32 + l32, safe = min(key, s.V - 1);
  const bool kept = key < s.V && (!a.mask || a.mask[b * a.ms[0] + (int64_t)safe * a.ms[1]] != 0);
  const bool all_kept = __all(kept), any_kept = __syncthreads_or(kept);
  const T* qp = (const T*)a.q + b * a.qs[0] + hk * s.G * a.qs[2];
  const T* dop = (const T*)a.dout + b * a.ds[0] + hk * s.G * a.ds[2];

  // what masked keys hold meets only zeros
  V8 kf[DP / 16], vf[DP / 16];
  load_row<T, DP>(kf, (const T*)a.k + b * a.ks[0] + (int64_t)safe * a.ks[1] + hk * a.ks[2], s.D, g);
  load_row<T, DP>(vf, (const T*)a.v + b * a.vs[0] + (int64_t)safe * a.vs[1] + hk * a.vs[2], s.D, g);
  if (!kept)
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) kf[kk] = vf[kk] = zero8<T>();
  const T* bias_key = BIAS ? (const T*)a.bias + b * a.bs[0] + safe : nullptr;

  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int cc = 0; cc < DP / 32; ++cc) clear(dk[cc]), clear(dv[cc]);
  const int tiles = (s.rows + KT - 1) / KT;
  const int t0 = split * a.k_tiles, t_end = any_kept ? min(tiles, t0 + a.k_tiles) : t0;
  float hold = 1.f, undo = 1.f;  // dS's power of two over P's, and what undoes it; the same in every split
  if constexpr (RANGED<T>) {
    constexpr int AT_ONCE = 8;
    const float* length = a.length + ((int64_t)b * s.H + hk * s.G) * s.U;  // of the key head's rows
    if (threadIdx.x == 0) lds.found[0] = 0;
    __syncthreads();
    float top = 0.f;
    for (int i = threadIdx.x; i < s.rows; i += AT_ONCE * NT)
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) top = fmaxf(top, length[min(i + k * NT, s.rows - 1)]);
    top = wave_top(top);
    if (lane == 0) atomicMax(&lds.found[0], __float_as_int(top));
    __syncthreads();
    const int log = __builtin_amdgcn_readfirstlane(ds_log(2.f * __int_as_float(lds.found[0]) * longest_value(a, b, hk)));
    hold = ldexpf(1.f, log - P_LOG), undo = ldexpf(1.f, -log);
  }
  Staged<T, DP, KT, NT> qreg, dreg;
  float next_m = 0.f, next_l = 0.f, next_delta = 0.f;
  int64_t next_bias = 0;
  auto load = [&](int t) {
    qreg.load_heads(qp, a.qs[1], a.qs[2], s.G, t * KT, s.rows, s.D);
    dreg.load_heads(dop, a.ds[1], a.ds[2], s.G, t * KT, s.rows, s.D);
    if (threadIdx.x < KT) {
      const int row = min(t * KT + (int)threadIdx.x, s.rows - 1), u = row / s.G, h = hk * s.G + row % s.G;
      const int64_t stat = ((int64_t)b * s.H + h) * s.U + u;
      row_stats<BIAS>(a.stats + 2 * stat, next_m, next_l);
      if constexpr (RANGED<T>) (BIAS ? next_l : next_m) -= (float)P_LOG;
      if (t * KT + (int)threadIdx.x >= s.rows) next_m = INFINITY;  // P = 2^-inf, and zeros of Q and dO
      next_delta = a.delta[stat];
      if constexpr (BIAS) next_bias = h * a.bs[1] + u * a.bs[2];
    }
  };
  auto put = [&](int t, int buf) {
    unsigned char* st = smem + buf * 2 * TILE;
    if (s.D == DP && (t + 1) * KT <= s.rows) {  // uniform
      qreg.store(st);
      dreg.store(st + TILE);
    } else {
      qreg.store(st, s.D, [&](int r) { return t * KT + r < s.rows; });
      dreg.store(st + TILE, s.D, [&](int r) { return t * KT + r < s.rows; });
    }
    if (threadIdx.x < KT) {
      lds.m[buf][threadIdx.x] = next_m;
      if constexpr (BIAS) lds.l[buf][threadIdx.x] = next_l;
      lds.minus_delta[buf][threadIdx.x] = -next_delta;
      if constexpr (BIAS) lds.bias_at[buf][threadIdx.x] = next_bias;
    }
  };
  if (t0 < t_end) {
    load(t0);
    put(t0, 0);
  }
  __syncthreads();
  int buf = 0;
  for (int t = t0; t < t_end; ++t, buf ^= NBUF - 1) {
    if (t + 1 < t_end) load(t + 1);
    const unsigned char* qs = smem + buf * 2 * TILE;
    const unsigned char* ds = qs + TILE;
#pragma unroll
    for (int sub = 0; sub < KT / 32; ++sub) {
      const int r0 = 32 * sub;
      // uniform: no row there (in 16 bits the products cost less than the branch between them: 195 us of 4 x 2048 x 1400,
      // 208 with it)
      if (sizeof(T) == 4 && t * KT + r0 >= s.rows) break;
      f32x16 p, dp;  // the sums of dP start from -Delta
      clear(p);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(&lds.minus_delta[buf][r0 + 8 * q + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * q + e] = d4[e];
      }
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        Mma<T, PREC>::step(p, Tile::row8(qs, r0 + l32, kk, g), kf[kk]);
        Mma<T, PREC>::step(dp, Tile::row8(ds, r0 + l32, kk, g), vf[kk]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 m4 = *reinterpret_cast<const f32x4*>(&lds.m[buf][r0 + 8 * q + 4 * g]);
        f32x4 l4 = {0.f, 0.f, 0.f, 0.f};
        if constexpr (BIAS) l4 = *reinterpret_cast<const f32x4*>(&lds.l[buf][r0 + 8 * q + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * q + e;
          float add = 0.f;
          if constexpr (BIAS) add = TypeOps<T>::to_f32(bias_key[lds.bias_at[buf][r0 + 8 * q + 4 * g + e]]);
          p[i] = probability<BIAS>(p[i], a.logit_scale, add, m4[e], l4[e]);
        }
      }
      if (!all_kept)  // uniform
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = kept ? p[i] : 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] *= p[i];
      if constexpr (RANGED<T>)
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] *= hold;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const V8 pf = acc_frag<T>(p, kk), sf = acc_frag<T>(dp, kk);
#pragma unroll
        for (int cc = 0; cc < DP / 32; ++cc) {
          Mma<T, PREC>::step(dv[cc], Tile::turned8(ds, r0, kk, cc, lane), pf);
          Mma<T, PREC>::step(dk[cc], Tile::turned8(qs, r0, kk, cc, lane), sf);
        }
      }
    }
    if constexpr (NBUF == 1) __syncthreads();
    if (t + 1 < t_end) put(t + 1, NBUF == 1 ? 0 : buf ^ 1);
    __syncthreads();
  }
  if (key >= s.V) return;
  const int64_t at = (((int64_t)b * s.V + key) * s.Hk + hk) * s.D, each = (int64_t)s.B * s.V * s.Hk * s.D;
#pragma unroll
  for (int cc = 0; cc < DP / 32; ++cc)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * cc + 8 * q + 4 * g;
      if (d >= s.D) continue;
      f32x4 x = f32x4{dk[cc][4 * q], dk[cc][4 * q + 1], dk[cc][4 * q + 2], dk[cc][4 * q + 3]} * (a.scale * undo);
      f32x4 y = f32x4{dv[cc][4 * q], dv[cc][4 * q + 1], dv[cc][4 * q + 2], dv[cc][4 * q + 3]} * (RANGED<T> ? 0x1p-10f : 1.f);
      if (!kept) x = y = f32x4{0.f, 0.f, 0.f, 0.f};  // zeros so far, but where Q or dO hold infinities or NaN
      if (a.part_k) {
        *reinterpret_cast<f32x4*>(a.part_k + 2 * split * each + at + d) = x;
        *reinterpret_cast<f32x4*>(a.part_k + (2 * split + 1) * each + at + d) = y;
      } else {
        store4((T*)a.dk + at + d, TypeOps<T>::from_f32(x));
        store4((T*)a.dv + at + d, TypeOps<T>::from_f32(y));
      }
    }
}

// ------------------------------------------------------------------- dbias of a shared bias
template <typename T, int PREC, int DP>
__device__ __forceinline__ void dbias_block(const BwdArgs& a, Lds<T, DP>& lds, uint32_t block) {
  typedef RowTile<T, DP> Tile;
  typedef typename TypeOps<T>::V8 V8;
  constexpr int TILE = Lds<T, DP>::TILE, KT = Lds<T, DP>::KT;
  unsigned char* smem = lds.tile;
  const Shape& s = a.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  const uint32_t nrb = (uint32_t)(s.rows + 127) / 128, nkb = (uint32_t)(s.V + KT - 1) / KT;
  uint32_t w = xcd_remap(block, a.b_blocks);
  const int rb = w % nrb;
  w /= nrb;
  const int kb = w % nkb, hk = w / nkb;
  const int row = rb * 128 + wave * 32 + l32;
  const int safe = min(row, s.rows - 1), u = safe / s.G, h = hk * s.G + safe % s.G;
  const T* bias_row = (const T*)a.bias + h * a.bs[1] + u * a.bs[2];
  f32x16 sum[KT / 32];
#pragma unroll
  for (int sub = 0; sub < KT / 32; ++sub) clear(sum[sub]);
  for (int b = 0; b < s.B; ++b) {
    const uint64_t live = live_keys(a.mask ? a.mask + b * a.ms[0] : nullptr, a.ms[1], kb * KT, s.V) & Lds<T, DP>::ALL;
    if (!live) continue;  // the same for the whole workgroup
    const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
    const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
    Staged<T, DP, KT, NT> kreg, vreg;
    kreg.load_rows(kp, a.ks[1], kb * KT, s.V, s.D);
    vreg.load_rows(vp, a.vs[1], kb * KT, s.V, s.D);
    V8 qf[DP / 16], df[DP / 16];
    load_row<T, DP>(qf, (const T*)a.q + b * a.qs[0] + u * a.qs[1] + h * a.qs[2], s.D, g);
    load_row<T, DP>(df, (const T*)a.dout + b * a.ds[0] + u * a.ds[1] + h * a.ds[2], s.D, g);
    const int64_t stat = ((int64_t)b * s.H + h) * s.U + u;
    float m, l;
    row_stats<true>(a.stats + 2 * stat, m, l);
    f32x16 minus_delta;
    fill(minus_delta, -a.delta[stat]);
    __syncthreads();  // the sequence before is done with
    kreg.store(smem, s.D, [&](int r) { return (live >> r & 1) != 0; });
    vreg.store(smem + TILE, s.D, [&](int r) { return (live >> r & 1) != 0; });
    __syncthreads();
#pragma unroll
    for (int sub = 0; sub < KT / 32; ++sub) {
      f32x16 ds;
      half_tile<T, PREC, DP, true>(ds, smem, smem + TILE, 32 * sub, qf, df, bias_row, kb * KT + 32 * sub, s.V, a.logit_scale,
                                   m, l, minus_delta, (uint32_t)(live >> (32 * sub)), __any(m == INFINITY));
      sum[sub] += ds;
    }
  }
  if (row >= s.rows) return;
  T* out = (T*)a.dbias + ((int64_t)h * s.U + u) * s.V;
#pragma unroll
  for (int sub = 0; sub < KT / 32; ++sub)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int key = kb * KT + 32 * sub + 8 * q + 4 * g;
      const f32x16& x = sum[sub];
      if (key < s.V) store4_at(out + key, f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]}, s.V - key);
    }
}

// The workgroups of DKDV and those of dQ, the longer walks first (24 rows of 7883 keys, 8 sequences, 4 heads of 64, fp32:
// 223 us, those of dQ last 294), then those of a shared dbias
template <typename T, int PREC, int DP, bool BIAS, bool DKDV, bool DQ, bool FINER>
__global__ __launch_bounds__(NT, sizeof(T) == 4 || (DKDV && DP > 64) ? 1 : 2) void cross_bwd_kernel(const BwdArgs a) {
  __shared__ Lds<T, DP> lds;
  uint32_t block = blockIdx.x;
  if (DKDV && DQ && a.q_first && block < a.k_blocks + a.q_blocks)
    block = block < a.q_blocks ? block + a.k_blocks : block - a.q_blocks;
  if constexpr (DKDV) {
    if (!DQ || block < a.k_blocks) return dkdv_block<T, PREC, DP, BIAS>(a, lds, block);
    block -= a.k_blocks;
  }
  if constexpr (DQ) {
    if (!BIAS || block < a.q_blocks) return dq_block<T, PREC, DP, BIAS, FINER>(a, lds, block);
    if constexpr (BIAS) dbias_block<T, PREC, DP>(a, lds, block - a.q_blocks);
  }
}

// dbias of one key, [B or 1][H][U]: 0, and NaN where a row's probability or output gradient has it
template <typename T>
__global__ __launch_bounds__(NT) void one_key_dbias_kernel(const BwdArgs a, T* dbias, int sequences) {
  const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x, each = (int64_t)a.s.H * a.s.U, n = a.s.B / sequences * each;
  if (i >= n) return;
  float sum = 0.f;
  for (int b = 0; b < sequences; ++b) {
    const int64_t stat = b * each + i;
    if (a.stats[2 * stat] != INFINITY) sum += 0.f * (a.stats[2 * stat + 1] + a.delta[stat]);
  }
  dbias[i] = (T)sum;
}

struct Plan {
  int64_t q_blocks, q_splits, q_tiles, k_blocks, k_splits, k_tiles;
};
// One workgroup of 4 waves a CU in fp32 and for the products of more than 64 columns, two otherwise. Those of dQ
// and of dK, dV are split so that none has more than about an equal part of all tiles (the queries of a few tokens walk
// over all keys, while each of many workgroups of dK and dV has one tile: 2 x 9 x 4391, 20 heads of 128 over 10, fp32:
// 178 us, 985 with dQ in one walk): a tile of dK and dV costs four products, one of dQ three.
// (The two launches of 16 bits above 64 columns each have the card to themselves and get a part of it: 1 x 1024 x 2048, 8
// heads of 128, bf16: 53 us on 128 workgroups of dK and dV, then 86 on 128 of dQ.)
Plan plan(const gnn_cross_attn_bwd_args& g) {
  Plan p{};
  const int KT = tile_of(g.dtype == GNN_F32, (int)g.D);
  const int64_t rows = g.U * (g.H / g.Hk), heads = g.B * g.Hk, cus = compute_units();
  const int64_t places = g.dtype == GNN_F32 || g.D > 64 ? cus : 2 * cus;
  const int64_t qb = (rows + 127) / 128 * heads, kb = g.dk ? (g.V + 127) / 128 * heads : 0;
  const int64_t qt = (g.V + KT - 1) / KT, kt = (rows + KT - 1) / KT;
  auto divide = [](int64_t tiles, int64_t most, int64_t& splits, int64_t& each) {
    splits = (tiles + most - 1) / most, each = (tiles + splits - 1) / splits;
  };
  int64_t part = (3 * qb * qt + 4 * kb * kt + places - 1) / places;
  const int64_t least = g.dtype == GNN_F32 ? 2 : 4;  // tiles a workgroup, beside its start and its sums
  for (;; part += part / 16 + 1) {  // until rounding up leaves no second round
    divide(qt, std::max(least, (part + 2) / 3), p.q_splits, p.q_tiles);
    divide(kt, std::max(least, (part + 3) / 4), p.k_splits, p.k_tiles);
    if (qb + kb >= places || qb * p.q_splits + kb * p.k_splits <= places || (p.q_splits == 1 && p.k_splits == 1)) break;
  }
  p.q_blocks = qb * p.q_splits;
  p.k_blocks = kb * p.k_splits;
  return p;
}

template <typename T, int LOG>
int delta(BwdArgs& a, hipStream_t st) {
  a.delta_blocks = (uint32_t)((((int64_t)a.s.B * a.s.U * a.s.H << LOG) + NT - 1) / NT);
  const uint32_t more = RANGED<T> ? (uint32_t)(a.s.B * a.s.Hk * a.v_parts) : 0;
  hipLaunchKernelGGL((cross_delta_kernel<T, LOG>), dim3(a.delta_blocks + more), dim3(NT), 0, st, a);
  return (int)hipGetLastError();
}

template <typename T, int PREC, int DP, bool BIAS>
int launch(BwdArgs& a, hipStream_t st) {
  constexpr int LOG = DP <= 32 ? 2 : DP <= 64 ? 3 : 4;
  if (int rc = delta<T, LOG>(a, st)) return rc;
  const uint32_t rest = a.q_blocks + a.b_blocks;
  auto go = [&](auto finer) {
    constexpr bool FINER = decltype(finer)::value;
    if constexpr (DP <= 64 || sizeof(T) == 4) {
      hipLaunchKernelGGL((cross_bwd_kernel<T, PREC, DP, BIAS, true, true, FINER>), dim3(a.k_blocks + rest), dim3(NT), 0, st, a);
    } else {
      if (a.k_blocks)
        hipLaunchKernelGGL((cross_bwd_kernel<T, PREC, DP, BIAS, true, false, false>), dim3(a.k_blocks), dim3(NT), 0, st, a);
      hipLaunchKernelGGL((cross_bwd_kernel<T, PREC, DP, BIAS, false, true, FINER>), dim3(rest), dim3(NT), 0, st, a);
    }
  };
  // dS in two parts: few keys, and heads so short that a query's pull on its keys shows in their sum: |K|^2 is D + 1 where
  // their spread is D. A variant of its own: a branch among the products cost 4 x 2048 x 1400 10% (209 us, 190 without).
  if constexpr (sizeof(T) == 4) {
    go(std::false_type{});
  } else if constexpr (DP == 32) {
    go(std::true_type{});
  } else {
    if (a.s.V <= FINE)
      go(std::true_type{});
    else
      go(std::false_type{});
  }
  return (int)hipGetLastError();
}

template <typename T, int PREC>
int run(BwdArgs& a, hipStream_t st) {
  auto go = [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    return a.bias ? launch<T, PREC, DP, true>(a, st) : launch<T, PREC, DP, false>(a, st);
  };
  if (a.s.D <= 32) return go(std::integral_constant<int, 32>{});
  if (a.s.D <= 64) return go(std::integral_constant<int, 64>{});
  if (a.s.D <= 96) return go(std::integral_constant<int, 96>{});
  return go(std::integral_constant<int, 128>{});
}

// The workspace: Delta, and in fp16 the rows' lengths and the parts' longest values, in whole 16 bytes each; then the fp32
// sums of the splits, dQ's, and behind them dK's and dV's
struct Heads {
  int64_t rows, tops, v_parts;
  int64_t floats() const { return rows + (tops ? rows + tops : 0); }
};
Heads heads_of(const gnn_cross_attn_bwd_args& g) {
  Heads h{};
  h.rows = (g.B * g.U * g.H + 3) / 4 * 4;
  if (g.dtype == GNN_F16) {
    h.v_parts = std::min<int64_t>(MAX_PARTS, (g.V + KEYS_A_PART - 1) / KEYS_A_PART);
    h.tops = (g.B * g.Hk * h.v_parts + 3) / 4 * 4;
  }
  return h;
}
void partial_sums(const gnn_cross_attn_bwd_args& g, const Plan& p, int64_t& q, int64_t& k) {
  q = p.q_splits > 1 ? p.q_splits * g.B * g.U * g.H * g.D : 0;
  k = p.k_splits > 1 && g.dk ? 2 * p.k_splits * g.B * g.V * g.Hk * g.D : 0;
}

}  // namespace

size_t cross_attn_bwd_workspace_bytes(const gnn_cross_attn_bwd_args& g) {
  int64_t q, k;
  partial_sums(g, plan(g), q, k);
  return (size_t)(heads_of(g).floats() + q + k) * sizeof(float);
}

int cross_attn_bwd(const gnn_cross_attn_bwd_args& g, hipStream_t st) {
  const Plan p = plan(g);
  const bool one_key = g.V == 1;
  const int KT = tile_of(g.dtype == GNN_F32, (int)g.D);
  const bool shared_bias = g.bias && g.shared_bias && g.B > 1;
  const int64_t rows = g.U * (g.H / g.Hk);
  const int64_t b_blocks = shared_bias && g.dbias && !one_key ? (rows + 127) / 128 * ((g.V + KT - 1) / KT) * g.Hk : 0;
  if (p.q_blocks + p.k_blocks + b_blocks >= ((int64_t)1 << 31))
    return set_error(GNN_ERR_UNSUPPORTED, "cross_attention: grid too large");
  if (!g.workspace || g.workspace_bytes < cross_attn_bwd_workspace_bytes(g))
    return set_error(GNN_ERR_WORKSPACE, "cross_attention: workspace missing or too small");
  BwdArgs a{};
  a.s = {(int)g.B, (int)g.U, (int)g.V, (int)g.H, (int)g.Hk, (int)(g.H / g.Hk), (int)g.D, (int)(g.U * (g.H / g.Hk))};
  a.q = g.q, a.k = g.k, a.v = g.v, a.o = g.o, a.o_low = g.o_low, a.dout = g.dout, a.bias = g.bias, a.mask = g.mask, a.stats = g.stats;
  a.dq = g.dq, a.dk = g.dk, a.dv = g.dv, a.dbias = g.dbias;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = g.q_stride[i], a.ks[i] = g.k_stride[i], a.vs[i] = g.v_stride[i];
    a.os[i] = g.o_stride[i], a.ds[i] = g.do_stride[i], a.bs[i] = g.bias_stride[i];
  }
  for (int i = 0; i < 2; ++i) a.ms[i] = g.mask_stride[i];
  a.scale = g.scale, a.logit_scale = g.bias ? g.scale : g.scale * LOG2E;
  // One key has probability 1, or 0 where its bias leaves nothing, whatever its logit: P comes from the row's statistics
  // alone (store_stats), and the logits' gradients are zeros, where P (dP - Delta) would leave the rounding errors of two
  // sums of the same products.
  if (one_key) a.scale = a.logit_scale = 0.f, a.bias = nullptr, a.dbias = nullptr;
  a.q_splits = (int)p.q_splits, a.q_tiles = (int)p.q_tiles, a.k_splits = (int)p.k_splits, a.k_tiles = (int)p.k_tiles;
  int64_t nq, nk;
  partial_sums(g, p, nq, nk);
  const Heads heads = heads_of(g);
  a.delta = (float*)g.workspace;
  if (heads.tops) a.length = a.delta + heads.rows, a.top = a.length + heads.rows, a.v_parts = (int)heads.v_parts;
  float* parts = a.delta + heads.floats();
  if (nq) a.part_q = parts;
  if (nk) a.part_k = parts + nq;
  a.q_blocks = (uint32_t)p.q_blocks, a.k_blocks = (uint32_t)p.k_blocks, a.b_blocks = (uint32_t)b_blocks;
  a.shared_bias = shared_bias;
  a.q_first = 3 * p.q_tiles > 4 * p.k_tiles;
  int rc;
  switch (g.dtype) {
    case GNN_BF16: rc = run<bf16, PREC_NATIVE>(a, st); break;
    case GNN_F16: rc = run<f16, PREC_NATIVE>(a, st); break;
    default: rc = g.precision == GNN_PREC_BF16X3 ? run<float, PREC_BF16X3>(a, st) : run<float, PREC_IEEE>(a, st);
  }
  if (rc == 0 && one_key && g.dbias) {
    const int sequences = g.shared_bias ? a.s.B : 1;  // summed
    const dim3 grid((uint32_t)((g.B / sequences * g.H * g.U + NT - 1) / NT));
    switch (g.dtype) {
      case GNN_BF16: hipLaunchKernelGGL(one_key_dbias_kernel<bf16>, grid, dim3(NT), 0, st, a, (bf16*)g.dbias, sequences); break;
      case GNN_F16: hipLaunchKernelGGL(one_key_dbias_kernel<f16>, grid, dim3(NT), 0, st, a, (f16*)g.dbias, sequences); break;
      default: hipLaunchKernelGGL(one_key_dbias_kernel<float>, grid, dim3(NT), 0, st, a, (float*)g.dbias, sequences);
    }
    rc = (int)hipGetLastError();
  }
  if (rc || (!nq && !nk)) return rc;
  gnn_reduce_args r{};
  if (nq) r.seg[r.count++] = {a.part_q, g.dq, p.q_splits, nq / p.q_splits, nq / p.q_splits, g.dtype, 0};
  if (nk) {
    const int64_t each = nk / p.k_splits / 2;
    r.seg[r.count++] = {a.part_k, g.dk, p.k_splits, 2 * each, each, g.dtype, 0};
    r.seg[r.count++] = {a.part_k + each, g.dv, p.k_splits, 2 * each, each, g.dtype, 0};
  }
  return reduce_parts(r, st);
}

}  // namespace gnn
