// A learned bias by buckets of the signed distance between a key and a query, and its gradient:
//   out[b, h, i, j] (or [b, i, j, h]) = table[bucket(key_pos[b, j] - query_pos[b, i])][h],
//   dtable[t][h] = sum over the (b, i, j) with bucket t of dout[b, h, i, j].
//
// Buckets. "Clip": the difference clamped to [-D, D] (two-sided: 2 D + 1 buckets), or how far the key lies
// behind, clamped to [0, D] (one-sided). "Log": of the n buckets of a side the first e = n / 2 hold one
// distance each, the other n - e widen geometrically up to D: bucket e + k starts at the least d with
// d >= e (D / e)^(k / (n - e)). Those borders are whole numbers that the host finds in exact integers and
// passes with the call; the kernel estimates k from log2(d) and corrects it against the borders, so no
// rounding decides a bucket.
// Every bucket is an interval of differences: where the smallest and the largest difference of a group of
// keys fall into one bucket, all of them do. That is the rule away from the diagonal.
//
// Forward: bound by the write of out. The table of a few heads lies in LDS in the output's type; heads first,
// a lane keeps 16 bytes of keys, works out their buckets once a query and writes them for every head;
// heads last, a lane writes 16 bytes of a pixel's heads.
// Backward: bound by the one read of dout. The sums are kept in fp32 and in a fixed order: every lane adds
// to bins of its own in LDS (heads first: [bucket][lane]; heads last: a wave's lanes own its channels,
// [bucket][channel]), and a wave leaves one row of partial sums, added in order by reduce_parts.
// 2048^2 x 16 heads, bf16, log, 134 MB: forward 29 us (4.6 TB/s), backward 51 (2.6: the blocks of keys
// across the diagonal, whose lanes look buckets up and add to bins, and each wave's set-up; the next loads issued a
// turn ahead 55, half or twice the waves 68 and 62); positions in random order, where every group straddles, 322.
// 509^2 x 128 channels, clip, 66 MB: 20 (3.3 TB/s, start and end of a short launch: 1018^2 takes 56, 4.7 TB/s) and 32
// (2.1: the chain of bins; half or twice the workgroups 47 and 45).
// More than 256 buckets (heads last 128) take a pass over dout for each 256 (128): 1024^2 x 16, 129, 257, 513 and 2049
// buckets 53, 101, 191 and 705 us (heads last 61, 120, 253 and 964).
#include <algorithm>

#include "gnn_common.hpp"
#include "gnn_internal.hpp"

namespace gnn {

namespace {

constexpr int RP_NT = 256;
constexpr int RP_MAX_BUCKETS = 4096;

template <typename T> struct Pack;  // 16 bytes of elements
template <> struct Pack<bf16> { typedef bf16x8 V; };
template <> struct Pack<f16> { typedef f16x8 V; };
template <> struct Pack<float> { typedef f32x4 V; };

struct Buckets {
  int n;     // log: buckets of a side
  int near;  // log: of them with one distance each
  int far;   // D
  int log, two_sided;
  float scale;  // log: (n - near) / log2(D / near)
  float log_near;
};

// The key's distance from the query, clamped to [-far, far]; positions may differ by more than 63 bits.
template <typename P>
__device__ __forceinline__ int ahead_of(P k, P q, int far) {
  if (sizeof(P) == 4) {
    const int64_t d = (int64_t)k - (int64_t)q;
    return (int)max<int64_t>(-far, min<int64_t>(far, d));
  }
  const uint64_t up = (uint64_t)k - (uint64_t)q, down = (uint64_t)q - (uint64_t)k;
  return k >= q ? (int)min<uint64_t>(up, (uint64_t)far) : -(int)min<uint64_t>(down, (uint64_t)far);
}

// `border[k]`, k = 0 .. n - near: the first distance of bucket near + k, border[0] = near and one past all
// distances at the end.
__device__ __forceinline__ int bucket_of(const Buckets& B, const int* border, int ahead) {
  if (!B.log) return B.two_sided ? ahead + B.far : max(-ahead, 0);
  const int d = B.two_sided ? abs(ahead) : max(-ahead, 0);
  int side = d;
  if (d >= B.near) {
    int k = (int)((__builtin_amdgcn_logf((float)d) - B.log_near) * B.scale);
    k = max(0, min(k, B.n - B.near - 1));
    while (d < border[k]) --k;       // border[0] = near <= d
    while (d >= border[k + 1]) ++k;  // border[n - near] > far >= d
    side = B.near + k;
  }
  return B.two_sided && ahead > 0 ? B.n + side : side;
}

// The differences that lie in bucket t, unclamped: from .. to
__device__ __forceinline__ void bucket_range(const Buckets& B, const int* border, int t, int& from, int& to) {
  constexpr int ALL = 0x7fffffff;
  if (!B.log) {
    if (B.two_sided) {
      from = t == 0 ? -ALL : t - B.far;
      to = t == 2 * B.far ? ALL : t - B.far;
    } else {
      to = t == 0 ? ALL : -t;
      from = t == B.far ? -ALL : -t;
    }
    return;
  }
  const bool up = B.two_sided && t >= B.n;
  const int side = up ? t - B.n : t;
  int d0 = side, d1 = side;  // distances d0 .. d1
  if (side >= B.near) {
    d0 = border[side - B.near];
    d1 = border[side - B.near + 1] - 1;  // beyond every distance for the last bucket
  }
  if (side == B.n - 1) d1 = ALL;
  if (up)
    from = d0, to = d1;
  else
    from = -d1, to = !B.two_sided && side == 0 ? ALL : -d0;
}

struct RpArgs {
  const void* table;  // [buckets][H]
  const void* qpos;
  const void* kpos;
  void* out;          // forward
  const void* dout;   // backward
  float* partial;     // backward
  int64_t q_bstride, k_bstride;
  int64_t sb, sh, si;  // strides of out / dout: heads first b, h, i; heads last b, -, i (rows of V * H)
  int B, U, V, H, buckets;
  int heads;  // heads first: per workgroup; heads last: whether the table goes to LDS
  int rows;   // queries per workgroup (forward) or wave (backward); heads last: groups of pixels per wave
  Buckets bk;
  int border[GNN_RELPOS_MAX_BORDERS + 2];
};

__device__ __forceinline__ void load_borders(const RpArgs& a, int* border) {
  if (a.bk.log)
    for (int i = threadIdx.x; i <= a.bk.n - a.bk.near; i += blockDim.x) border[i] = a.border[i];
}

template <typename T>
__device__ __forceinline__ void store_pack(T* p, const typename Pack<T>::V& v, int left) {
  typedef typename Pack<T>::V V;
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
__device__ __forceinline__ typename Pack<T>::V load_pack(const T* p, int left) {
  typedef typename Pack<T>::V V;
  constexpr int E = 16 / (int)sizeof(T);
  typedef V VU __attribute__((aligned(sizeof(T))));
  if (left >= E) return *(const __attribute__((address_space(1))) VU*)p;
  V v;
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = e < left ? p[e] : (T)0.f;
  return v;
}

// ---- heads first ------------------------------------------------------------------------
// Workgroup: 256 lanes of 16 bytes of keys x `rows` queries x `heads` heads of one sequence.
template <typename T, typename P>
__global__ __launch_bounds__(RP_NT) void relpos_fwd_kernel(const RpArgs a) {
  typedef typename Pack<T>::V V;
  constexpr int E = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned char smem[];
  T* table = (T*)smem;  // [heads][buckets]
  __shared__ int border[GNN_RELPOS_MAX_BORDERS + 2];
  const int nkey = (a.V + RP_NT * E - 1) / (RP_NT * E), nq = (a.U + a.rows - 1) / a.rows,
            nh = (a.H + a.heads - 1) / a.heads;
  uint32_t w = blockIdx.x;
  const int h0 = (int)(w % (uint32_t)nh) * a.heads;
  w /= (uint32_t)nh;
  const int j = ((int)(w % (uint32_t)nkey) * RP_NT + threadIdx.x) * E;
  w /= (uint32_t)nkey;
  const int i0 = (int)(w % (uint32_t)nq) * a.rows, b = (int)(w / (uint32_t)nq);
  const int heads = min(a.heads, a.H - h0);
  load_borders(a, border);
  for (int e = threadIdx.x; e < heads * a.buckets; e += RP_NT) {
    const int t = e / heads, h = e - t * heads;
    table[h * a.buckets + t] = ((const T*)a.table)[(int64_t)t * a.H + h0 + h];
  }
  __syncthreads();
  if (j >= a.V) return;
  const P* kp = (const P*)a.kpos + b * a.k_bstride;
  const P* qp = (const P*)a.qpos + b * a.q_bstride;
  P k[E];
#pragma unroll
  for (int e = 0; e < E; ++e) k[e] = kp[min(j + e, a.V - 1)];
  for (int i = i0; i < min(i0 + a.rows, a.U); ++i) {
    const P q = qp[i];
    int at[E];
#pragma unroll
    for (int e = 0; e < E; ++e) at[e] = bucket_of(a.bk, border, ahead_of(k[e], q, a.bk.far));
    T* out = (T*)a.out + b * a.sb + (int64_t)h0 * a.sh + i * a.si + j;
    for (int h = 0; h < heads; ++h, out += a.sh) {
      V v;
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = table[h * a.buckets + at[e]];
      store_pack(out, v, a.V - j);
    }
  }
}

// A wave takes one head and a range of queries; its bins are [buckets of this pass][64 lanes]. A lane keeps
// its 16 bytes of keys over the queries of a sequence, eight of which are read ahead. Away from the diagonal
// the group of keys stays in one bucket over many queries: the lane knows the differences that this bucket
// holds and adds in a register until it is left (4 instructions a query beside the sum; two bucket_of a query
// took 109 us of 134 MB). Where a group straddles buckets every key is looked up, in a table of all
// differences where they are few. Differences run in 32 bits from a base that follows the queries.
constexpr int RP_AHEAD = 8;
constexpr int RP_LUT_FAR = 1023;           // differences looked up: 2 far + 1 16-bit entries
constexpr int RP_FAR_BASE = 1 << 28;       // queries this far from the base move it
template <typename T, typename P>
__global__ __launch_bounds__(64) void relpos_bwd_kernel(const RpArgs a, int first, int count) {
  typedef typename Pack<T>::V V;
  constexpr int E = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned char smem[];
  float* bins = (float*)smem;
  uint16_t* lut = (uint16_t*)(bins + count * 64);
  __shared__ int border[GNN_RELPOS_MAX_BORDERS + 2];
  const int lane = threadIdx.x;
  const uint32_t h = blockIdx.x % (uint32_t)a.H, part = blockIdx.x / (uint32_t)a.H;
  const int far = a.bk.far;
  load_borders(a, border);
  for (int t = 0; t < count; ++t) bins[t * 64 + lane] = 0.f;
  __syncthreads();
  const bool looked_up = far <= RP_LUT_FAR;
  if (looked_up) {
    for (int d = lane; d <= 2 * far; d += 64) lut[d] = (uint16_t)bucket_of(a.bk, border, d - far);
    __syncthreads();
  }
  auto bucket = [&](int ahead) {
    const int d = max(-far, min(far, ahead));
    return looked_up ? (int)lut[d + far] : bucket_of(a.bk, border, d);
  };
  // one lane adds to a bin: the order is the program's
  auto add = [&](int t, float x) {
    t -= first;
    if ((unsigned)t < (unsigned)count)
      __hip_atomic_fetch_add(bins + t * 64 + lane, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  const int rows = a.B * a.U;
  const int r1 = min(rows, (int)(part + 1) * a.rows);
  for (int r0 = (int)part * a.rows; r0 < r1;) {
    const int b = r0 / a.U, i0 = r0 - b * a.U;
    const int i1 = min(a.U, i0 + (r1 - r0));
    r0 += i1 - i0;
    const P* kp = (const P*)a.kpos + b * a.k_bstride;
    const P* qp = (const P*)a.qpos + b * a.q_bstride;
    const T* src = (const T*)a.dout + b * a.sb + (int64_t)h * a.sh;
    for (int j = lane * E; j < a.V; j += 64 * E) {
      P base = qp[i0];
      int k[E], lo, hi;  // from the base, saturated beyond any bucket's border
      auto rebase = [&]() {
#pragma unroll
        for (int e = 0; e < E; ++e) k[e] = ahead_of(kp[min(j + e, a.V - 1)], base, 1 << 30);
        lo = hi = k[0];
#pragma unroll
        for (int e = 1; e < E; ++e) lo = min(lo, k[e]), hi = max(hi, k[e]);
      };
      rebase();
      int cur = 0, from = 1, to = 0;  // differences from .. to lie in bucket cur: none so far
      float sum = 0.f;
      for (int i = i0; i < i1; i += RP_AHEAD) {
        V v[RP_AHEAD];
#pragma unroll
        for (int u = 0; u < RP_AHEAD; ++u) v[u] = load_pack(src + min(i + u, i1 - 1) * a.si + j, a.V - j);
#pragma unroll
        for (int u = 0; u < RP_AHEAD; ++u) {
          if (i + u >= i1) break;
          const P q = qp[i + u];
          int dq = ahead_of(q, base, RP_FAR_BASE);
          if (abs(dq) == RP_FAR_BASE) {  // uniform
            base = q;
            dq = 0;
            rebase();
          }
          if (lo - dq < from || hi - dq > to) {
            const int t = bucket(lo - dq);
            if (cur != t || from > to) {
              if (sum != 0.f) add(cur, sum);
              sum = 0.f;
            }
            if (t == bucket(hi - dq)) {
              cur = t;
              bucket_range(a.bk, border, t, from, to);
            } else {
              if (sum != 0.f) add(cur, sum);
              sum = 0.f;
              from = 1, to = 0;
#pragma unroll
              for (int e = 0; e < E; ++e) add(bucket(k[e] - dq), (float)v[u][e]);
              continue;
            }
          }
          float s = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) s += (float)v[u][e];  // zeros past the last key
          sum += s;
        }
      }
      if (from <= to) add(cur, sum);
    }
  }
  __syncthreads();
  // partial[part][bucket][head]: the lanes' bins, each bucket's from another lane on (64 banks)
  for (int t = lane; t < count; t += 64) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int l = 0; l < 64; ++l) s[l % 4] += bins[t * 64 + ((l + lane) & 63)];
    a.partial[((int64_t)part * a.buckets + first + t) * a.H + h] = (s[0] + s[1]) + (s[2] + s[3]);
  }
}

// ---- heads last -------------------------------------------------------------------------
// out rows [V * H] of a query, 16 bytes a lane; a lane's elements lie in one pixel where H is a multiple of
// their number, otherwise each is looked up.
template <typename T, typename P>
__global__ __launch_bounds__(RP_NT) void relpos_last_fwd_kernel(const RpArgs a) {
  typedef typename Pack<T>::V V;
  constexpr int E = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned char smem[];
  T* table = (T*)smem;  // [buckets][H], where it fits
  const T* gtable = (const T*)a.table;
  __shared__ int border[GNN_RELPOS_MAX_BORDERS + 2];
  load_borders(a, border);
  if (a.heads)
    for (int e = threadIdx.x; e < a.buckets * a.H; e += RP_NT) table[e] = gtable[e];
  __syncthreads();
  const int len = a.V * a.H;  // below 2^31, as the number of items is
  const bool whole = a.H % E == 0;
  const uint32_t nseg = (uint32_t)(len + RP_NT * E - 1) / (RP_NT * E), items = (uint32_t)(a.B * a.U) * nseg;
  for (uint32_t w = blockIdx.x; w < items; w += gridDim.x) {
    const uint32_t r = w / nseg;
    const int x = (int)((w - r * nseg) * RP_NT + threadIdx.x) * E;
    if (x >= len) continue;
    const int b = (int)(r / (uint32_t)a.U), i = (int)(r - (uint32_t)b * (uint32_t)a.U);
    const P* kp = (const P*)a.kpos + b * a.k_bstride;
    const P q = ((const P*)a.qpos)[b * a.q_bstride + i];
    T* out = (T*)a.out + b * a.sb + i * a.si + x;
    V v;
    int j = (int)((uint32_t)x / (uint32_t)a.H), c = x - j * a.H;
    int t = bucket_of(a.bk, border, ahead_of(kp[j], q, a.bk.far));
    if (whole) {
      if (a.heads)
        v = *reinterpret_cast<const V*>(table + t * a.H + c);
      else
        v = load_pack(gtable + (int64_t)t * a.H + c, E);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = a.heads ? table[t * a.H + c] : gtable[(int64_t)t * a.H + c];
        if (x + e + 1 < len && ++c == a.H) {  // past the row's end the last element again, which is not stored
          c = 0;
          t = bucket_of(a.bk, border, ahead_of(kp[++j], q, a.bk.far));
        }
      }
    }
    store_pack(out, v, min(E, len - x));
  }
}

// A workgroup takes 128 channels, two a lane, and a range of groups of 64 pixels; each of its waves has bins
// [buckets of this pass][128] of its own, added in wave order at the end. The buckets of 64 pixels are worked
// out by the lanes at once and handed round as scalars; a run of pixels in one bucket adds in registers.
constexpr int RP_BATCH = 32;  // pixels in flight
template <typename T, typename P>
__global__ __launch_bounds__(256) void relpos_last_bwd_kernel(const RpArgs a, int first, int count) {
  typedef T V2 __attribute__((ext_vector_type(2)));
  typedef V2 V2U __attribute__((aligned(sizeof(T))));
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int border[GNN_RELPOS_MAX_BORDERS + 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int nc = (a.H + 127) / 128;
  const int c0 = (int)(blockIdx.x % (uint32_t)nc) * 128, part = blockIdx.x / (uint32_t)nc;
  float* bins = (float*)smem + wave * count * 128;
  load_borders(a, border);
  for (int t = 0; t < 2 * count; ++t) bins[t * 64 + lane] = 0.f;
  __syncthreads();
  // Two channels are there to be read for every lane: the last of an odd number comes with the one before it, and
  // lanes past the last channel read along (their bins are not)
  const int c = c0 + 2 * lane, read = min(c, a.H - 2);
  const bool second = c == a.H - 1;
  const uint32_t groups = (uint32_t)(a.V + 63) / 64, items = (uint32_t)(a.B * a.U) * groups;
  const uint32_t w0 = min(items, (uint32_t)(part * waves + wave) * (uint32_t)a.rows), w1 = min(items, w0 + (uint32_t)a.rows);
  float2* const mybins = (float2*)bins + lane;
  int cur = -1;
  float2 sum = {0.f, 0.f};
  for (uint32_t w = w0; w < w1; ++w) {
    const uint32_t r = w / groups;
    const int j0 = (int)(w - r * groups) * 64;
    const int b = (int)(r / (uint32_t)a.U), i = (int)(r - (uint32_t)b * (uint32_t)a.U);
    const P* kp = (const P*)a.kpos + b * a.k_bstride;
    const P q = ((const P*)a.qpos)[b * a.q_bstride + i];
    const T* src = (const T*)a.dout + b * a.sb + i * a.si + read;
    const int mine = bucket_of(a.bk, border, ahead_of(kp[min(j0 + lane, a.V - 1)], q, a.bk.far)) - first;
    const int n = min(64, a.V - j0);
    for (int p0 = 0; p0 < n; p0 += RP_BATCH) {
      V2 x[RP_BATCH];
#pragma unroll
      for (int p = 0; p < RP_BATCH; ++p) {
        x[p] = *(const __attribute__((address_space(1))) V2U*)(src + (int64_t)(j0 + min(p0 + p, n - 1)) * a.H);
      }
#pragma unroll
      for (int p = 0; p < RP_BATCH; ++p) {
        if (p0 + p >= n) break;
        const int t = __builtin_amdgcn_readlane(mine, p0 + p);
        if (t != cur) {  // uniform
          if ((unsigned)cur < (unsigned)count) mybins[cur * 64] = sum;
          if ((unsigned)t < (unsigned)count) sum = mybins[t * 64];
          cur = t;
        }
        sum.x += (float)(second ? x[p][1] : x[p][0]);
        sum.y += (float)x[p][1];
      }
    }
  }
  if ((unsigned)cur < (unsigned)count) mybins[cur * 64] = sum;
  __syncthreads();
  for (int e = threadIdx.x; e < count * 128; e += blockDim.x) {
    const int t = e >> 7, ch = c0 + (e & 127);
    if (ch >= a.H) continue;
    float s = 0.f;
    for (int k = 0; k < waves; ++k) s += ((const float*)smem)[k * count * 128 + e];
    a.partial[((int64_t)part * a.buckets + first + t) * a.H + ch] = s;
  }
}

// The same for 2 to 64 channels, where one pixel would leave most lanes idle: `lanes` (a power of two, two
// channels each) take a pixel and a wave 64 / lanes neighbouring ones at once, each group of lanes in bins of its
// own. The buckets of RP_PIXELS pixels pass through LDS. (2048^2 x 16
// channels, bf16: 50 us, a pixel a wave 470.)
constexpr int RP_PIXELS = 256;
template <typename T, typename P>
__global__ __launch_bounds__(256) void relpos_last_narrow_bwd_kernel(const RpArgs a, int first, int count, int lanes) {
  typedef T V2 __attribute__((ext_vector_type(2)));
  typedef V2 V2U __attribute__((aligned(sizeof(T))));
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int border[GNN_RELPOS_MAX_BORDERS + 2];
  __shared__ uint16_t buckets[4][RP_PIXELS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int at_once = 64 / lanes, sub = lane / lanes, c = 2 * (lane % lanes);
  float* bins = (float*)smem + wave * count * 128;
  load_borders(a, border);
  for (int t = 0; t < 2 * count; ++t) bins[t * 64 + lane] = 0.f;
  __syncthreads();
  const int read = min(c, a.H - 2);  // as above
  const bool second = c == a.H - 1;
  const uint32_t groups = (uint32_t)(a.V + RP_PIXELS - 1) / RP_PIXELS, items = (uint32_t)(a.B * a.U) * groups;
  const uint32_t part = blockIdx.x;
  const uint32_t w0 = min(items, (part * waves + wave) * (uint32_t)a.rows), w1 = min(items, w0 + (uint32_t)a.rows);
  float2* const mybins = (float2*)bins + lane;
  int cur = -1;
  float2 sum = {0.f, 0.f};
  for (uint32_t w = w0; w < w1; ++w) {
    const uint32_t r = w / groups;
    const int j0 = (int)(w - r * groups) * RP_PIXELS;
    const int b = (int)(r / (uint32_t)a.U), i = (int)(r - (uint32_t)b * (uint32_t)a.U);
    const P* kp = (const P*)a.kpos + b * a.k_bstride;
    const P q = ((const P*)a.qpos)[b * a.q_bstride + i];
    const T* src = (const T*)a.dout + b * a.sb + i * a.si + (int64_t)j0 * a.H + read;
    const int n = min(RP_PIXELS, a.V - j0);
#pragma unroll
    for (int k = 0; k < RP_PIXELS / 64; ++k) {  // a wave's LDS accesses stay in order
      const int p = 64 * k + lane;
      const int t = bucket_of(a.bk, border, ahead_of(kp[min(j0 + p, a.V - 1)], q, a.bk.far));
      buckets[wave][p] = p < n ? (uint16_t)t : (uint16_t)0xffff;  // in no pass's range
    }
    for (int p0 = 0; p0 < n; p0 += RP_BATCH * at_once) {
      V2 x[RP_BATCH];
#pragma unroll
      for (int k = 0; k < RP_BATCH; ++k)
        x[k] = *(const __attribute__((address_space(1))) V2U*)(src + min(p0 + k * at_once + sub, n - 1) * a.H);
#pragma unroll
      for (int k = 0; k < RP_BATCH; ++k) {
        if (p0 + k * at_once >= n) break;  // uniform
        const int t = (int)buckets[wave][p0 + k * at_once + sub] - first;
        if (t != cur) {
          if ((unsigned)cur < (unsigned)count) mybins[cur * 64] = sum;
          if ((unsigned)t < (unsigned)count) sum = mybins[t * 64];
          cur = t;
        }
        sum.x += (float)(second ? x[k][1] : x[k][0]);
        sum.y += (float)x[k][1];
      }
    }
  }
  if ((unsigned)cur < (unsigned)count) mybins[cur * 64] = sum;
  __syncthreads();
  for (int e = threadIdx.x; e < count * a.H; e += blockDim.x) {
    const int t = e / a.H, ch = e - t * a.H;
    float s = 0.f;
    for (int k = 0; k < waves; ++k)
      for (int g = 0; g < at_once; ++g) s += ((const float*)smem)[(k * count + t) * 128 + g * 2 * lanes + ch];
    a.partial[((int64_t)part * a.buckets + first + t) * a.H + ch] = s;
  }
}

RpArgs common(const gnn_relpos_args& g) {
  RpArgs a{};
  a.table = g.table, a.qpos = g.query_pos, a.kpos = g.key_pos, a.out = g.out, a.dout = g.dout, a.partial = g.partial;
  a.q_bstride = g.query_stride, a.k_bstride = g.key_stride;
  a.sb = g.stride[0], a.sh = g.stride[1], a.si = g.stride[2];
  a.B = (int)g.B, a.U = (int)g.U, a.V = (int)g.V, a.H = (int)g.H, a.buckets = (int)g.buckets;
  Buckets& k = a.bk;
  k.far = (int)g.max_distance, k.log = g.log_spacing, k.two_sided = g.two_sided;
  if (k.log) {
    k.n = a.buckets / (k.two_sided ? 2 : 1), k.near = k.n / 2;
    const int m = k.n - k.near;
    k.log_near = log2f((float)k.near);
    k.scale = (float)m / (log2f((float)k.far) - k.log_near);
    a.border[0] = k.near;
    for (int i = 1; i < m; ++i) a.border[i] = g.border[i - 1];
    a.border[m] = INT32_MAX;
  }
  return a;
}

constexpr int RP_TABLE = 48 << 10;  // LDS for the table: three workgroups of a CU
constexpr int RP_BINS = 64 << 10;   // and for a wave's bins: at least two waves a CU

template <typename T, typename P>
int forward(const gnn_relpos_args& g, hipStream_t st) {
  RpArgs a = common(g);
  constexpr int E = 16 / (int)sizeof(T);
  if (g.channels_last) {
    const size_t bytes = (size_t)a.buckets * a.H * sizeof(T), lds = bytes <= RP_TABLE ? bytes : 0;
    a.heads = lds != 0;
    const int64_t nseg = ((int64_t)a.V * a.H + RP_NT * E - 1) / (RP_NT * E);
    const int64_t grid = std::min<int64_t>((int64_t)a.B * a.U * nseg, (int64_t)compute_units() * 8);
    hipLaunchKernelGGL((relpos_last_fwd_kernel<T, P>), dim3((uint32_t)grid), dim3(RP_NT), lds, st, a);
    return (int)hipGetLastError();
  }
  a.heads = std::max<int>(1, std::min<int>(a.H, RP_TABLE / (a.buckets * (int)sizeof(T))));
  const int64_t nkey = ((int64_t)a.V + RP_NT * E - 1) / (RP_NT * E);
  // queries of a workgroup share the table and the keys, as long as the card stays full
  const int64_t full = (int64_t)compute_units() * 8;
  int64_t nh = (a.H + a.heads - 1) / a.heads;
  a.rows = (int)std::max<int64_t>(1, std::min<int64_t>(8, (int64_t)a.B * a.U * nkey * nh / full));
  if ((int64_t)a.B * a.U * nkey * nh < full) {  // few queries: fewer heads a workgroup
    const int64_t want = std::min<int64_t>(a.H, full / std::max<int64_t>(1, (int64_t)a.B * a.U * nkey));
    a.heads = (int)std::min<int64_t>(a.heads, (a.H + want - 1) / std::max<int64_t>(1, want));
    nh = (a.H + a.heads - 1) / a.heads;
  }
  const int64_t grid = nh * nkey * ((a.U + a.rows - 1) / a.rows) * a.B;
  if (grid >= ((int64_t)1 << 31)) return set_error(GNN_ERR_UNSUPPORTED, "relative_position_bias: grid too large");
  hipLaunchKernelGGL((relpos_fwd_kernel<T, P>), dim3((uint32_t)grid), dim3(RP_NT),
                     (size_t)a.heads * a.buckets * sizeof(T), st, a);
  return (int)hipGetLastError();
}

// Backward: buckets a pass, and heads last the waves of a workgroup that their bins leave room for
struct Bins {
  int count, bytes, waves;
};
Bins bins_of(const gnn_relpos_args& g) {
  Bins b;
  const int per = (g.channels_last ? 128 : 64) * 4;
  const int passes = (int)((g.buckets + RP_BINS / per - 1) / (RP_BINS / per));
  b.count = (int)((g.buckets + passes - 1) / passes);
  b.bytes = b.count * per;
  b.waves = g.channels_last ? std::max(1, std::min(4, (144 << 10) / b.bytes)) : 1;
  return b;
}
int64_t across(const gnn_relpos_args& g) { return g.channels_last ? (g.H + 127) / 128 : g.H; }
bool narrow(const gnn_relpos_args& g) { return g.channels_last && g.H <= 64; }
int64_t bwd_items(const gnn_relpos_args& g) {
  const int64_t pixels = narrow(g) ? RP_PIXELS : 64;
  return g.B * g.U * (g.channels_last ? (g.V + pixels - 1) / pixels : 1);
}

template <typename T, typename P>
int backward(const gnn_relpos_args& g, hipStream_t st) {
  RpArgs a = common(g);
  const Bins bins = bins_of(g);
  const int64_t each = g.parts * bins.waves, grid = g.parts * across(g);
  if (grid >= ((int64_t)1 << 31) || (bwd_items(g) + each - 1) / each >= ((int64_t)1 << 31))
    return set_error(GNN_ERR_UNSUPPORTED, "relative_position_bias backward: grid too large");
  a.rows = (int)((bwd_items(g) + each - 1) / each);
  for (int first = 0; first < a.buckets; first += bins.count) {
    const int n = std::min(bins.count, a.buckets - first);
    const size_t lds = (size_t)bins.waves * n * (bins.bytes / bins.count) +
                       (!g.channels_last && a.bk.far <= RP_LUT_FAR ? 2 * (2 * a.bk.far + 2) : 0);
    if (lds > 64 * 1024) {
      const void* fn = narrow(g)          ? (const void*)relpos_last_narrow_bwd_kernel<T, P>
                       : g.channels_last ? (const void*)relpos_last_bwd_kernel<T, P>
                                         : (const void*)relpos_bwd_kernel<T, P>;
      (void)hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    }
    if (narrow(g)) {
      int lanes = 1;
      while (2 * lanes < a.H) lanes *= 2;
      hipLaunchKernelGGL((relpos_last_narrow_bwd_kernel<T, P>), dim3((uint32_t)grid), dim3(64 * bins.waves), lds, st, a, first,
                         n, lanes);
    } else if (g.channels_last)
      hipLaunchKernelGGL((relpos_last_bwd_kernel<T, P>), dim3((uint32_t)grid), dim3(64 * bins.waves), lds, st, a, first, n);
    else
      hipLaunchKernelGGL((relpos_bwd_kernel<T, P>), dim3((uint32_t)grid), dim3(64), lds, st, a, first, n);
  }
  return (int)hipGetLastError();
}

template <typename P>
int by_dtype(const gnn_relpos_args& g, bool bwd, hipStream_t st) {
  switch (g.dtype) {
    case GNN_BF16: return bwd ? backward<bf16, P>(g, st) : forward<bf16, P>(g, st);
    case GNN_F16: return bwd ? backward<f16, P>(g, st) : forward<f16, P>(g, st);
    default: return bwd ? backward<float, P>(g, st) : forward<float, P>(g, st);
  }
}

}  // namespace

// One channel last is one head first
static gnn_relpos_args one_layout(gnn_relpos_args g) {
  if (g.H == 1) g.channels_last = 0;
  return g;
}

int relpos(const gnn_relpos_args& args, bool bwd, hipStream_t st) {
  const gnn_relpos_args g = one_layout(args);
  const int64_t most = (int64_t)1 << 31;
  if (g.B * g.U >= most || (g.channels_last && g.B * g.U * ((g.V * g.H + 63) / 64 + 1) >= most))
    return set_error(GNN_ERR_UNSUPPORTED, "relative_position_bias: more than 2^31 rows or pieces of rows");
  if (g.buckets > RP_MAX_BUCKETS)
    return set_error(GNN_ERR_UNSUPPORTED, "relative_position_bias: more than 4096 buckets");
  return g.pos_bytes == 8 ? by_dtype<int64_t>(g, bwd, st) : by_dtype<int32_t>(g, bwd, st);
}

// Rows of partial sums: as many workgroups as the card holds by their bins, not more than there is work
int64_t relpos_parts(const gnn_relpos_args& args) {
  const gnn_relpos_args g = one_layout(args);
  if (g.buckets > RP_MAX_BUCKETS) return 0;
  const Bins b = bins_of(g);
  const int64_t per_cu = std::max<int64_t>(1, std::min<int64_t>(16 / b.waves, (150 << 10) / (b.bytes * b.waves)));
  return std::max<int64_t>(1, std::min((bwd_items(g) + b.waves - 1) / b.waves, compute_units() * per_cu / across(g)));
}

}  // namespace gnn
