// The product of a tile of rows and a tile of a weight's rows, both contiguous along the contraction, as the linear
// layers' kernels form it.
#pragma once

#include "linear_common.hpp"

namespace gnn {
namespace lin {

// s_waitcnt vmcnt(VM) expcnt(7) lgkmcnt(0)
template <int VM>
__device__ __forceinline__ void wait_vm_lgkm0() {
  static_assert(VM >= 0 && VM < 64, "vmcnt immediate");
  __builtin_amdgcn_s_waitcnt(0x070 | (VM & 15) | ((VM >> 4) << 14));
}

// GM x GN waves of 32 X rows x 32 Y outputs; stages of ROWB bytes of a row
template <typename T, int GM_, int GN_, int X_, int Y_, int ROWB_, int STAGES_>
struct Tile {
  static constexpr int GM = GM_, GN = GN_, X = X_, Y = Y_, ROWB = ROWB_, STAGES = STAGES_;
  static constexpr int BM = 32 * GM * X, BN = 32 * GN * Y;
  static constexpr int NW = GM * GN, NT = 64 * NW;
  static constexpr int BK = ROWB / (int)sizeof(T);  // elements of a row a stage
  static constexpr int EPC = 16 / (int)sizeof(T);   // elements a chunk
  static constexpr int CPR = ROWB / 16, RPI = 1024 / ROWB;        // chunks a row, rows a DMA instruction
  static constexpr int QA = BM / RPI / NW, QB = BN / RPI / NW;    // DMA instructions a wave and stage
  static constexpr int QPS = QA + QB;
  static constexpr int STAGE = (BM + BN) * ROWB;
  static constexpr int LDS = STAGES * STAGE;
  static constexpr int WGS = (160 << 10) / LDS;  // workgroups a CU
  static_assert(ROWB == 64 || ROWB == 128, "swizzle");
  static_assert(QA * RPI * NW == BM && QB * RPI * NW == BN, "DMA split");
  static_assert(STAGES >= 2 && STAGES <= 4 && NW * 4096 <= LDS, "waits and the epilogue's tiles");
  static __device__ __forceinline__ int swz(int row, int chunk) { return chunk ^ chunk_swizzle<ROWB>(row); }
};

// acc[x][y] = rows 32 (X wm + x) .. of the weight's 32 (Y wn + y) .., transposed (a lane holds one row of x, and with
// the weight's rows in tile_output's order 8 consecutive outputs). xrow(r), wrow(r): the address of the tile's row r.
// Every wave of the workgroup calls it; LDS holds stages that DMA may still be writing when it returns.
template <typename T, int PREC, typename Cfg, typename XRow, typename WRow>
__device__ __forceinline__ void tile_products(f32x16 (&acc)[Cfg::X][Cfg::Y], unsigned char* smem, int I, XRow xrow,
                                              WRow wrow) {
  typedef typename TypeOps<T>::V8 V8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
  const int wm = wave / Cfg::GN, wn = wave % Cfg::GN;

  // DMA: an instruction moves RPI rows; lane -> row lane / CPR, stored chunk lane % CPR, which holds the row's
  // chunk swz(row, lane % CPR). Chunks past the contraction's end are zeros in both operands.
  const int drow = lane / Cfg::CPR, dpos = lane % Cfg::CPR;
  const T* xsrc[Cfg::QA];
  const T* wsrc[Cfg::QB];
#pragma unroll
  for (int q = 0; q < Cfg::QA; ++q) xsrc[q] = xrow(Cfg::RPI * (Cfg::QA * wave + q) + drow);
#pragma unroll
  for (int q = 0; q < Cfg::QB; ++q) wsrc[q] = wrow(Cfg::RPI * (Cfg::QB * wave + q) + drow);
  const int nkt = (I + Cfg::BK - 1) / Cfg::BK;
  // instructions [q0, q1) of a stage's QPS, x's first
  auto issue = [&](int kt, int q0, int q1) {
    unsigned char* st = smem + (kt % Cfg::STAGES) * Cfg::STAGE;
    const int k0 = kt * Cfg::BK;
#pragma unroll
    for (int q = q0; q < q1; ++q) {
      const bool is_x = q < Cfg::QA;
      const int at = is_x ? Cfg::QA * wave + q : Cfg::QB * wave + q - Cfg::QA;
      const T* src = is_x ? xsrc[is_x ? q : 0] : wsrc[is_x ? 0 : q - Cfg::QA];
      const int k = k0 + Cfg::swz(Cfg::RPI * at + drow, dpos) * Cfg::EPC;
      __builtin_amdgcn_global_load_lds(k < I ? (const void*)(src + k) : (const void*)zero_chunk,
                                       (lds_void_t*)(st + (is_x ? 0 : Cfg::BM * Cfg::ROWB) + at * 1024), 16, 0, 0);
    }
  };
  // 8 elements kk * 16 + 8 g of a row
  auto frag = [&](const unsigned char* base, int r, int kk) -> V8 {
    const unsigned char* row = base + r * Cfg::ROWB;
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const V8*>(row + (Cfg::swz(r, 2 * kk + g) << 4));
    } else {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(row + (Cfg::swz(r, 4 * kk + 2 * g) << 4));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(row + (Cfg::swz(r, 4 * kk + 2 * g + 1) << 4));
      return V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  };

#pragma unroll
  for (int x = 0; x < Cfg::X; ++x)
#pragma unroll
    for (int y = 0; y < Cfg::Y; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;

  // A stage's products go in steps of 16 elements; a step begins with the reads of the next step's fragments, over
  // the stage's end too. With three stages in flight the DMA of the stage after them goes in equal shares beside
  // the steps' products (4096 x 4096 -> 1024, bf16: 44 us; all at the stage's start 52). With two buffers it has
  // only until the stage's end to land and goes in the first two steps (4096^3: 142 us; in shares 149). Stages
  // past the end are zeros.
  constexpr int KS = Cfg::BK / 16, SHARE = Cfg::QPS / KS, FIRST = KS > 2 ? 2 : 1;
  constexpr bool SPREAD = Cfg::STAGES > 2;
  static_assert(KS % 2 == 0 && (!SPREAD || SHARE * KS == Cfg::QPS), "steps");
  V8 xf[2][Cfg::X], wf[2][Cfg::Y];
  auto load_frags = [&](int slot, int kt, int kk) {
    const unsigned char* sx = smem + (kt % Cfg::STAGES) * Cfg::STAGE;
    const unsigned char* sw = sx + Cfg::BM * Cfg::ROWB;
#pragma unroll
    for (int y = 0; y < Cfg::Y; ++y) wf[slot][y] = frag(sw, 32 * (Cfg::Y * wn + y) + l32, kk);
#pragma unroll
    for (int x = 0; x < Cfg::X; ++x) xf[slot][x] = frag(sx, 32 * (Cfg::X * wm + x) + l32, kk);
  };
  // This wave's DMA of a stage has landed (the later stages' may be in flight) and its reads so far have
  // returned; after the barrier every wave's have, and the buffer of the stage before is free.
  auto arrive = [&]() {
    wait_vm_lgkm0<(Cfg::STAGES - 2) * Cfg::QPS>();
    asm volatile("s_barrier" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < Cfg::STAGES - 1; ++s) issue(s, 0, Cfg::QPS);
  arrive();
  load_frags(0, 0, 0);
  if (SPREAD) issue(Cfg::STAGES - 1, 0, SHARE);
  for (int kt = 0; kt < nkt; ++kt) {
    const int next = kt + Cfg::STAGES - 1;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const bool last = kk + 1 == KS;
      if (last) arrive();
      load_frags((kk + 1) & 1, last ? kt + 1 : kt, last ? 0 : kk + 1);
      if (SPREAD)
        issue(last ? next + 1 : next, last ? 0 : (kk + 1) * SHARE, last ? SHARE : (kk + 2) * SHARE);
      else if (kk < FIRST)  // before the stage's last step, which waits for it
        issue(next, kk * Cfg::QPS / FIRST, (kk + 1) * Cfg::QPS / FIRST);
#pragma unroll
      for (int x = 0; x < Cfg::X; ++x)
#pragma unroll
        for (int y = 0; y < Cfg::Y; ++y) Mma<T, PREC>::step(acc[x][y], wf[kk & 1][y], xf[kk & 1][x]);
    }
  }
}

}  // namespace lin
}  // namespace gnn
