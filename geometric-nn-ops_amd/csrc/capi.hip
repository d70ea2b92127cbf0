// extern "C" entry points of libgnn_hip.so (declared in include/gnn_triangle.h): argument
// validation, the thread-local error message, and dispatch to the kernel launchers.
#include <stdio.h>
#include <string.h>

#include <string>

#include "gnn_internal.hpp"

namespace gnn {

static thread_local std::string g_last_error;

int set_error(int code, const char* msg) {
  g_last_error = msg;
  return code;
}

int compute_units() {
  int dev = 0, ncu = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&ncu, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || ncu < 1)
    ncu = 1;
  return ncu;
}

int persistent_grid(const void* fn, int threads, size_t smem) {
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, fn, threads, smem) != hipSuccess || per_cu < 1)
    per_cu = 1;
  return compute_units() * per_cu;
}

static int hip_status(hipError_t e, const char* who) {
  if (e == hipSuccess) return GNN_OK;
  char buf[256];
  snprintf(buf, sizeof buf, "%s: HIP error %d (%s)", who, (int)e, hipGetErrorString(e));
  g_last_error = buf;
  return (int)e;
}

static bool aligned(const void* p, size_t n) { return ((uintptr_t)p % n) == 0; }

// Every row of the pair bias starts on 16 bytes and has a pitch up to round_up(N, 8), which is read
static bool bias_rows_readable(const void* bias, const int64_t (&st)[4], int64_t B, int64_t H, int64_t N) {
  return st[3] == 1 && st[2] % 8 == 0 && (st[2] >= N || N % 8 == 0) && (H == 1 || st[1] % 8 == 0) &&
         (B == 1 || st[0] % 8 == 0) && aligned(bias, 16);
}

// caller_workspace: the caller provides the scratch (gnn_triattn_fwd); false for the entry
// point whose scratch is the library's static array.
static int check_triattn(const gnn_triattn_args& a, bool caller_workspace = true) {
  if (!a.q || !a.k || !a.v || !a.o)
    return set_error(GNN_ERR_ARG, "triangle_attention: q, k, v and o are required");
  if (a.B < 1 || a.S < 1 || a.N < 1 || a.H < 1 || a.D < 1)
    return set_error(GNN_ERR_ARG, "triangle_attention: B, N_seq, N_res, H and D must be positive");
  if (a.dtype != GNN_BF16 && a.dtype != GNN_F16 && a.dtype != GNN_F32)
    return set_error(GNN_ERR_ARG, "triangle_attention: unknown dtype");
  if (a.D % 8 != 0)
    return set_error(GNN_ERR_ARG, "triangle_attention: D must be a multiple of 8 (pad on the host)");
  const int64_t* st[4] = {a.q_stride, a.k_stride, a.v_stride, a.o_stride};
  const void* ptr[4] = {a.q, a.k, a.v, a.o};
  for (int t = 0; t < 4; ++t) {
    if (!aligned(ptr[t], 16))
      return set_error(GNN_ERR_ARG, "triangle_attention: q/k/v/o must be 16-byte aligned");
    for (int d = 0; d < 4; ++d)
      if (st[t][d] % 8 != 0)
        return set_error(GNN_ERR_ARG, "triangle_attention: q/k/v/o strides must be multiples of 8 elements");
  }
  if (a.bias && !triattn_row_applicable(a) && !bias_rows_readable(a.bias, a.bias_stride, a.B, a.H, a.N))
    return set_error(GNN_ERR_ARG,
                     "triangle_attention: bias needs unit key stride, other strides that are multiples of 8, rows "
                     "readable to round_up(N, 8) and 16-byte alignment");
  const size_t need = triattn_row_applicable(a) ? triattn_row_workspace_bytes(a) : 0;
  if (caller_workspace && need && (!a.workspace || a.workspace_bytes < need || !aligned(a.workspace, 16)))
    return set_error(GNN_ERR_WORKSPACE,
                     "triangle_attention: workspace missing, smaller than gnn_triattn_workspace_bytes() or "
                     "not 16-byte aligned");
  return GNN_OK;
}

}  // namespace gnn

using namespace gnn;

extern "C" {

int gnn_triattn_fwd(const gnn_triattn_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "triangle_attention: args is NULL");
  if (int rc = check_triattn(*args)) return rc;
  int rc = triattn_fwd(*args, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "triangle_attention");
}

int gnn_triattn_fwd_noalloc(const gnn_triattn_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "triangle_attention: args is NULL");
  if (int rc = check_triattn(*args, false)) return rc;
  int rc = triattn_fwd_noalloc(*args, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "triangle_attention (no-alloc)");
}

size_t gnn_triattn_workspace_bytes(const gnn_triattn_args* args) {
  if (!args) return 0;
  return triattn_row_applicable(*args) ? triattn_row_workspace_bytes(*args) : 0;
}

int gnn_triattn_bwd(const gnn_triattn_bwd_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "triangle_attention backward: args is NULL");
  const gnn_triattn_bwd_args& a = *args;
  if (!a.q || !a.k || !a.v || !a.o || !a.dout || !a.lse || !a.dq || !a.dk || !a.dv || !a.delta)
    return set_error(GNN_ERR_ARG, "triangle_attention backward: q, k, v, o, dout, lse, dq, dk, dv and delta are required");
  if (a.B < 1 || a.S < 1 || a.N < 1 || a.H < 1 || a.D < 1)
    return set_error(GNN_ERR_ARG, "triangle_attention backward: B, N_seq, N_res, H and D must be positive");
  if (a.D % 8 != 0)
    return set_error(GNN_ERR_ARG, "triangle_attention backward: D must be a multiple of 8 (pad on the host)");
  const int64_t* st[5] = {a.q_stride, a.k_stride, a.v_stride, a.o_stride, a.do_stride};
  const void* ptr[5] = {a.q, a.k, a.v, a.o, a.dout};
  for (int t = 0; t < 5; ++t) {
    if (!aligned(ptr[t], 16))
      return set_error(GNN_ERR_ARG, "triangle_attention backward: q/k/v/o/dout must be 16-byte aligned");
    for (int d = 0; d < 4; ++d)
      if (st[t][d] % 8 != 0)
        return set_error(GNN_ERR_ARG, "triangle_attention backward: q/k/v/o/dout strides must be multiples of 8 elements");
  }
  if (a.bias && !bias_rows_readable(a.bias, a.bias_stride, a.B, a.H, a.N))
    return set_error(GNN_ERR_ARG, "triangle_attention backward: bias needs unit key stride, other strides that are "
                                  "multiples of 8, rows readable to round_up(N, 8) and 16-byte alignment");
  int rc = triattn_bwd(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "triangle_attention backward");
}

size_t gnn_trimul_workspace_bytes(int64_t B, int64_t N, int64_t C, int64_t Ch, int32_t dtype,
                                  size_t off[4]) {
  const TrimulLayout L = trimul_layout(B, N, C, Ch, dtype);
  if (off) {
    off[0] = L.off_a;
    off[1] = L.off_b;
    off[2] = L.off_g;
    off[3] = L.off_o;
  }
  return L.total;
}

static int trimul_stage(const gnn_trimul_args* args, void* stream, int which) {
  if (!args) return set_error(GNN_ERR_ARG, "trimul: args is NULL");
  hipStream_t st = (hipStream_t)stream;
  int rc = GNN_OK;
  if (which & 1) rc = trimul_proj(*args, st);
  if (rc == GNN_OK && (which & 2)) rc = trimul_contract(*args, st);
  if (rc == GNN_OK && (which & 4)) rc = trimul_out(*args, st);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "trimul");
}

int gnn_trimul_fwd(const gnn_trimul_args* args, void* stream) { return trimul_stage(args, stream, 7); }
int gnn_trimul_proj(const gnn_trimul_args* args, void* stream) { return trimul_stage(args, stream, 1); }
int gnn_trimul_contract(const gnn_trimul_args* args, void* stream) {
  return trimul_stage(args, stream, 2);
}
int gnn_trimul_out(const gnn_trimul_args* args, void* stream) { return trimul_stage(args, stream, 4); }

int gnn_pair_bias_proj(const gnn_pair_bias_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "pair_bias_proj: args is NULL");
  const gnn_pair_bias_args& a = *args;
  if (!a.z || !a.proj_w || !a.out)
    return set_error(GNN_ERR_ARG, "pair_bias_proj: z, proj_w and out are required");
  if (a.B < 1 || a.U < 1 || a.V < 1 || a.Zc < 1 || a.H < 1)
    return set_error(GNN_ERR_ARG, "pair_bias_proj: B, U, V, c_z and H must be positive");
  if (!aligned(a.z, 16))
    return set_error(GNN_ERR_ARG, "pair_bias_proj: z must be 16-byte aligned");
  int rc = pair_bias_proj(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "pair_bias_proj");
}

int gnn_apb_gate_out(const gnn_apb_gate_out_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "apb_gate_out: args is NULL");
  const gnn_apb_gate_out_args& a = *args;
  if (!a.s || !a.o || !a.g_w || !a.o_w || !a.out)
    return set_error(GNN_ERR_ARG, "apb_gate_out: s, o, g_w, o_w and out are required");
  if (a.M < 1 || a.Cs < 1 || a.D < 1 || a.Co < 1)
    return set_error(GNN_ERR_ARG, "apb_gate_out: M, c_s, the attention width and c_out must be positive");
  if (a.dtype != GNN_BF16 && a.dtype != GNN_F16 && a.dtype != GNN_F32)
    return set_error(GNN_ERR_ARG, "apb_gate_out: unknown dtype");
  const int64_t e = a.dtype == GNN_F32 ? 4 : 2;
  const void* ptrs[] = {a.s, a.o, a.g_w, a.o_w, a.out};
  for (const void* p : ptrs)
    if (!aligned(p, 16)) return set_error(GNN_ERR_ARG, "apb_gate_out: tensors must be 16-byte aligned");
  if ((a.s_ld * e) % 16 || (a.o_ld * e) % 16 || (a.out_ld * e) % 16 || a.s_ld < a.Cs || a.o_ld < a.D ||
      a.out_ld < a.Co)
    return set_error(GNN_ERR_ARG, "apb_gate_out: row pitches must cover the rows and be multiples of 16 bytes");
  int rc = apb_gate_out(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "apb_gate_out");
}

int64_t gnn_layernorm_partials(int64_t rows, int64_t K) { return layernorm_partials(rows, K); }

int gnn_layernorm_rows(const gnn_layernorm_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "layernorm_rows: args is NULL");
  const gnn_layernorm_args& a = *args;
  if (!a.x || !a.out) return set_error(GNN_ERR_ARG, "layernorm_rows: x and out are required");
  if (a.rows < 1 || a.K < 1) return set_error(GNN_ERR_ARG, "layernorm_rows: rows and K must be positive");
  if (a.x_stride < a.K || a.out_stride < a.K || (a.dy && a.dy_stride < a.K))
    return set_error(GNN_ERR_ARG, "layernorm_rows: a row stride is smaller than K");
  if (a.dy && a.bias) return set_error(GNN_ERR_ARG, "layernorm_rows: bias is a forward-only argument");
  int rc = layernorm_rows(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "layernorm_rows");
}

int64_t gnn_gate_bwd_partials(int64_t rows, int64_t K) { return gate_bwd_partials(rows, K); }

int gnn_trimul_gate_bwd(const gnn_gate_bwd_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "trimul_gate_bwd: args is NULL");
  const gnn_gate_bwd_args& a = *args;
  if (!a.grad || !a.value || !a.gate_pre || !a.d_value || !a.d_gate_pre)
    return set_error(GNN_ERR_ARG, "trimul_gate_bwd: grad, value, gate_pre, d_value and d_gate_pre are required");
  if (a.rows < 1 || a.K < 1) return set_error(GNN_ERR_ARG, "trimul_gate_bwd: rows and K must be positive");
  const int64_t st[5] = {a.grad_stride, a.value_stride, a.gate_stride, a.dv_stride, a.dg_stride};
  const void* ptr[5] = {a.grad, a.value, a.gate_pre, a.d_value, a.d_gate_pre};
  const int64_t esz = a.dtype == GNN_F32 ? 4 : 2;
  for (int i = 0; i < 5; ++i) {
    if (st[i] < a.K) return set_error(GNN_ERR_ARG, "trimul_gate_bwd: a row stride is smaller than K");
    if ((st[i] * esz) % 16 != 0 || !aligned(ptr[i], 16))
      return set_error(GNN_ERR_ARG, "trimul_gate_bwd: rows must be 16-byte aligned");
  }
  int rc = gate_bwd(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "trimul_gate_bwd");
}

int64_t gnn_trimul_out_bwd_partials(int64_t B, int64_t N) { return trimul_out_bwd_partials(B, N); }

int gnn_trimul_out_bwd(const gnn_trimul_out_bwd_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "trimul_out_bwd: args is NULL");
  const gnn_trimul_out_bwd_args& a = *args;
  if (!a.o || !a.p_out_w || !a.gate || !a.dout || !a.on || !a.dy || !a.d_go || !a.d_o || !a.partial)
    return set_error(GNN_ERR_ARG, "trimul_out_bwd: o, p_out_w, gate, dout, on, dy, d_go, d_o and partial are required");
  if (a.B < 1 || a.N < 1 || a.C < 1 || a.Ch < 1)
    return set_error(GNN_ERR_ARG, "trimul_out_bwd: B, N, C and c_hidden must be positive");
  if (a.dgo_ld < a.C || (a.dgo_ld * 2) % 16 != 0)
    return set_error(GNN_ERR_ARG, "trimul_out_bwd: d_go rows must cover C and be 16-byte aligned");
  const void* ptr[9] = {a.o, a.p_out_w, a.gate, a.dout, a.on, a.dy, a.d_go, a.d_o, a.partial};
  for (const void* q : ptr)
    if (!aligned(q, 16)) return set_error(GNN_ERR_ARG, "trimul_out_bwd: tensors must be 16-byte aligned");
  int rc = trimul_out_bwd(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "trimul_out_bwd");
}

int64_t gnn_trimul_proj_bwd_partials(int64_t rows) { return trimul_proj_bwd_partials(rows); }

int gnn_trimul_proj_bwd(const gnn_trimul_proj_bwd_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "trimul_proj_bwd: args is NULL");
  const gnn_trimul_proj_bwd_args& a = *args;
  if (!a.x || !a.p_in_w || !a.g_in_w || !a.d_ab || !a.d_p || !a.d_g || !a.z || !a.partial)
    return set_error(GNN_ERR_ARG, "trimul_proj_bwd: x, p_in_w, g_in_w, d_ab, d_p, d_g, z and partial are required");
  if (a.rows < 1 || a.C < 1 || a.Ch < 1)
    return set_error(GNN_ERR_ARG, "trimul_proj_bwd: rows, C and c_hidden must be positive");
  if (a.x_ld < a.C || a.dab_ld < 2 * a.Ch || a.dl_ld < 2 * a.Ch || a.mask_stride < 0)
    return set_error(GNN_ERR_ARG, "trimul_proj_bwd: a row stride is smaller than its row");
  const int64_t st[3] = {a.x_ld, a.dab_ld, a.dl_ld};
  for (int64_t v : st)
    if ((v * 2) % 16 != 0) return set_error(GNN_ERR_ARG, "trimul_proj_bwd: rows must be 16-byte aligned");
  const void* ptr[6] = {a.x, a.d_ab, a.d_p, a.d_g, a.z, a.p_in_w};
  for (const void* q : ptr)
    if (!aligned(q, 16)) return set_error(GNN_ERR_ARG, "trimul_proj_bwd: tensors must be 16-byte aligned");
  if (!aligned(a.g_in_w, 16)) return set_error(GNN_ERR_ARG, "trimul_proj_bwd: tensors must be 16-byte aligned");
  int rc = trimul_proj_bwd(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "trimul_proj_bwd");
}

int gnn_trimul_contract_bwd(const gnn_trimul_contract_bwd_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "trimul_contract_bwd: args is NULL");
  const gnn_trimul_contract_bwd_args& a = *args;
  if (!a.a || !a.b || !a.do_i || !a.do_j || !a.da || !a.db)
    return set_error(GNN_ERR_ARG, "trimul_contract_bwd: a, b, do_i, do_j, da and db are required");
  if (a.dtype != GNN_BF16 && a.dtype != GNN_F16)
    return set_error(GNN_ERR_UNSUPPORTED, "trimul_contract_bwd: 16-bit dtypes only");
  if (a.planes < 1 || a.N < 1) return set_error(GNN_ERR_ARG, "trimul_contract_bwd: planes and N must be positive");
  const void* ptr[6] = {a.a, a.b, a.do_i, a.do_j, a.da, a.db};
  for (const void* p : ptr)
    if (!aligned(p, 16)) return set_error(GNN_ERR_ARG, "trimul_contract_bwd: pointers must be 16-byte aligned");
  if (a.planes * ((a.N + 127) / 128) * ((a.N + 255) / 256) >= ((int64_t)1 << 31) || a.N >= ((int64_t)1 << 30))
    return set_error(GNN_ERR_UNSUPPORTED, "trimul_contract_bwd: grid too large");
  int rc = trimul_contract_bwd(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "trimul_contract_bwd");
}

int gnn_relayout_f32(const gnn_trimul_relayout_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "relayout_f32: args is NULL");
  const gnn_trimul_relayout_args& a = *args;
  if (!a.src || !a.dst) return set_error(GNN_ERR_ARG, "relayout_f32: src and dst are required");
  if (a.dtype != GNN_F32) return set_error(GNN_ERR_UNSUPPORTED, "relayout_f32: fp32 only");
  const bool to_pixels = a.mode == GNN_RELAYOUT_PLANES_TO_PIXELS;
  if (!to_pixels && a.mode != GNN_RELAYOUT_PIXELS_TO_PLANES)
    return set_error(GNN_ERR_ARG, "relayout_f32: unknown mode");
  if (a.B < 1 || a.N < 1 || a.Ch < 1) return set_error(GNN_ERR_ARG, "relayout_f32: B, N and Ch must be positive");
  if (a.Ch % 4 || a.src_ld % 4 || a.dst_ld % 4 || a.src_c0 % 4 || a.dst_c0 % 4 || a.src_c0 < 0 || a.dst_c0 < 0)
    return set_error(GNN_ERR_ARG, "relayout_f32: Ch, row pitches and channel offsets must be multiples of 4");
  if (!aligned(a.src, 16) || !aligned(a.dst, 16))
    return set_error(GNN_ERR_ARG, "relayout_f32: src and dst must be 16-byte aligned");
  if (a.plane_rows != 0 && a.plane_rows < a.N)
    return set_error(GNN_ERR_ARG, "relayout_f32: plane_rows must be 0 or at least N");
  const int64_t N4 = (a.N + 3) / 4 * 4;
  if (to_pixels ? (a.src_ld < N4 || a.dst_c0 + a.Ch > a.dst_ld) : (a.dst_ld < N4 || a.src_c0 + a.Ch > a.src_ld))
    return set_error(GNN_ERR_ARG, "relayout_f32: a row pitch is too small for its rows");
  int rc = relayout_f32(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "relayout_f32");
}

static int check_rows_product(const gnn_rows_product_args* args, bool pointers) {
  if (!args) return set_error(GNN_ERR_ARG, "rows_product: args is NULL");
  const gnn_rows_product_args& a = *args;
  if (a.dtype != GNN_BF16 && a.dtype != GNN_F16 && a.dtype != GNN_F32)
    return set_error(GNN_ERR_ARG, "rows_product: unknown dtype");
  if (a.count < 1 || a.count > GNN_ROWS_PRODUCT_MAX || a.rows < 1 || a.slice_rows < 0)
    return set_error(GNN_ERR_ARG, "rows_product: rows must be positive, slice_rows not negative and count in 1 .. "
                                  "GNN_ROWS_PRODUCT_MAX");
  for (int i = 0; i < a.count; ++i) {
    const gnn_rows_product_item& p = a.p[i];
    if (p.O < 8 || p.I < 8 || p.O % 8 || p.I % 8 || p.O > (1 << 20) || p.I > (1 << 20))
      return set_error(GNN_ERR_ARG, "rows_product: O and I must be multiples of 8, at most 2^20");
    if (!pointers) continue;
    if (!p.d || !p.t || !p.partial) return set_error(GNN_ERR_ARG, "rows_product: d, t and partial are required");
    if (p.d_ld < p.O || p.t_ld < p.I || p.d_ld % 8 || p.t_ld % 8)
      return set_error(GNN_ERR_ARG, "rows_product: row pitches must cover the rows and be multiples of 8");
    if (!aligned(p.d, 16) || !aligned(p.t, 16) || !aligned(p.partial, 4))
      return set_error(GNN_ERR_ARG, "rows_product: d and t must be 16-byte aligned");
  }
  return GNN_OK;
}

int64_t gnn_rows_product_slices(const gnn_rows_product_args* args) {
  return check_rows_product(args, false) ? 0 : rows_product_slices(*args);
}

int gnn_rows_product(const gnn_rows_product_args* args, void* stream) {
  if (int rc = check_rows_product(args, true)) return rc;
  int rc = rows_product(*args, nullptr, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "rows_product");
}

int gnn_reduce_parts(const gnn_reduce_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "reduce_parts: args is NULL");
  const gnn_reduce_args& a = *args;
  if (a.count < 1 || a.count > GNN_REDUCE_MAX)
    return set_error(GNN_ERR_ARG, "reduce_parts: count must be in 1 .. GNN_REDUCE_MAX");
  for (int i = 0; i < a.count; ++i) {
    const gnn_reduce_segment& s = a.seg[i];
    if (!s.src || !s.dst || s.parts < 1 || s.n < 1 || (s.parts > 1 && s.stride < s.n))
      return set_error(GNN_ERR_ARG, "reduce_parts: src, dst, parts, n and a stride of at least n are required");
    const bool f32 = s.dtype == GNN_F32;
    if (!f32 && s.dtype != GNN_BF16 && s.dtype != GNN_F16)
      return set_error(GNN_ERR_ARG, "reduce_parts: unknown dtype");
    if (!aligned(s.src, 4) || !aligned(s.dst, f32 ? 4 : 2))
      return set_error(GNN_ERR_ARG, "reduce_parts: src and dst must be aligned to their elements");
  }
  int rc = reduce_parts(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "reduce_parts");
}

int gnn_trimul_relayout(const gnn_trimul_relayout_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "trimul_relayout: args is NULL");
  const gnn_trimul_relayout_args& a = *args;
  if (!a.src || !a.dst) return set_error(GNN_ERR_ARG, "trimul_relayout: src and dst are required");
  if (a.dtype != GNN_BF16 && a.dtype != GNN_F16)
    return set_error(GNN_ERR_UNSUPPORTED, "trimul_relayout: 16-bit dtypes only");
  if (a.mode != GNN_RELAYOUT_PLANES_TO_PIXELS && a.mode != GNN_RELAYOUT_PIXELS_TO_BLOCKED)
    return set_error(GNN_ERR_ARG, "trimul_relayout: unknown mode");
  if (a.B < 1 || a.N < 1 || a.Ch < 1) return set_error(GNN_ERR_ARG, "trimul_relayout: B, N and Ch must be positive");
  if (a.Ch % 8 || a.src_ld % 8 || a.dst_ld % 8 || a.src_c0 % 8 || a.dst_c0 % 8 || a.src_c0 < 0 || a.dst_c0 < 0)
    return set_error(GNN_ERR_ARG, "trimul_relayout: Ch, row pitches and channel offsets must be multiples of 8");
  if (!aligned(a.src, 16) || !aligned(a.dst, 16))
    return set_error(GNN_ERR_ARG, "trimul_relayout: src and dst must be 16-byte aligned");
  const int64_t N8 = (a.N + 7) / 8 * 8;
  if (a.mode == GNN_RELAYOUT_PLANES_TO_PIXELS ? (a.src_ld < N8 || a.dst_c0 + a.Ch > a.dst_ld)
                                              : (a.src_c0 + a.Ch > a.src_ld))
    return set_error(GNN_ERR_ARG, "trimul_relayout: a row pitch is too small for its rows");
  int rc = trimul_relayout(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "trimul_relayout");
}

static bool known_dtype(int32_t t) { return t == GNN_BF16 || t == GNN_F16 || t == GNN_F32; }

// Shapes, types and row addresses shared by the LayerNorm's two directions
static int check_layer_norm(int64_t rows, int64_t K, int32_t dtype, int32_t param_dtype, const void* params) {
  if (rows < 1 || K < 1) return set_error(GNN_ERR_ARG, "layer_norm: rows and K must be positive");
  if (!known_dtype(dtype)) return set_error(GNN_ERR_ARG, "layer_norm: unknown dtype");
  if (params && param_dtype != dtype && param_dtype != GNN_F32)
    return set_error(GNN_ERR_ARG, "layer_norm: parameters must be in the rows' dtype or fp32");
  return GNN_OK;
}
static int check_layer_norm_rows(const void* p, int64_t rows, int64_t inner, int64_t outer, int64_t stride, int32_t dtype) {
  if (inner < 1 || inner > rows || outer < 0 || stride < 0)
    return set_error(GNN_ERR_ARG, "layer_norm: inner rows must be in 1 .. rows and strides not negative");
  if (!aligned(p, dtype == GNN_F32 ? 4 : 2))
    return set_error(GNN_ERR_ARG, "layer_norm: tensors must be aligned to their elements");
  return GNN_OK;
}

int gnn_layer_norm_fwd(const gnn_layer_norm_fwd_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "layer_norm: args is NULL");
  const gnn_layer_norm_fwd_args& a = *args;
  if (!a.x || !a.y) return set_error(GNN_ERR_ARG, "layer_norm: x and y are required");
  if (!a.mean != !a.rstd) return set_error(GNN_ERR_ARG, "layer_norm: mean and rstd are written together");
  if (int rc = check_layer_norm(a.rows, a.K, a.dtype, a.param_dtype, a.weight ? a.weight : a.bias)) return rc;
  if (int rc = check_layer_norm_rows(a.x, a.rows, a.x_inner, a.x_outer_stride, a.x_stride, a.dtype)) return rc;
  int rc = layer_norm_fwd(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "layer_norm");
}

int64_t gnn_layer_norm_bwd_parts(int64_t rows, int64_t K, int32_t dtype) {
  return rows < 1 || K < 1 ? 0 : layer_norm_bwd_parts(rows, K, dtype);
}

int gnn_layer_norm_bwd(const gnn_layer_norm_bwd_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "layer_norm backward: args is NULL");
  const gnn_layer_norm_bwd_args& a = *args;
  if (!a.x || !a.dy || !a.mean || !a.rstd || (!a.dx && !a.partial))
    return set_error(GNN_ERR_ARG, "layer_norm backward: x, dy, mean, rstd and one of dx and partial are required");
  if (a.parts < 1 || a.parts >= ((int64_t)1 << 31))
    return set_error(GNN_ERR_ARG, "layer_norm backward: parts must be positive and fit a grid");
  if (int rc = check_layer_norm(a.rows, a.K, a.dtype, a.param_dtype, a.weight)) return rc;
  if (int rc = check_layer_norm_rows(a.x, a.rows, a.x_inner, a.x_outer_stride, a.x_stride, a.dtype)) return rc;
  if (int rc = check_layer_norm_rows(a.dy, a.rows, a.dy_inner, a.dy_outer_stride, a.dy_stride, a.dtype)) return rc;
  const int param_bytes = a.param_dtype == GNN_F32 ? 4 : 2;
  if ((a.dweight || a.dbias) && !a.partial)
    return set_error(GNN_ERR_ARG, "layer_norm backward: dweight and dbias need partial");
  if (!aligned(a.dweight, param_bytes) || !aligned(a.dbias, param_bytes))
    return set_error(GNN_ERR_ARG, "layer_norm backward: dweight and dbias must be aligned to their elements");
  int rc = layer_norm_bwd(a, (hipStream_t)stream);
  if (rc == 0 && (a.dweight || a.dbias)) {
    gnn_reduce_args r{};
    for (int i = 0; i < 2; ++i)
      if (void* dst = i ? a.dbias : a.dweight)
        r.seg[r.count++] = {a.partial + i * a.K, dst, a.parts, 2 * a.K, a.K, a.param_dtype, 0};
    rc = reduce_parts(r, (hipStream_t)stream);
  }
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "layer_norm backward");
}

static int check_relpos(const gnn_relpos_args* args) {
  if (!args) return set_error(GNN_ERR_ARG, "relative_position_bias: args is NULL");
  const gnn_relpos_args& a = *args;
  if (!known_dtype(a.dtype)) return set_error(GNN_ERR_ARG, "relative_position_bias: unknown dtype");
  if (a.pos_bytes != 4 && a.pos_bytes != 8)
    return set_error(GNN_ERR_ARG, "relative_position_bias: positions must have 4 or 8 bytes");
  const int64_t most = INT32_MAX;
  if (a.B < 1 || a.U < 1 || a.V < 1 || a.H < 1 || a.buckets < 1 || a.B > most || a.U > most || a.V > most - 4096 ||
      a.H > most || a.V * a.H > most - 4096 || a.buckets > most / a.H)
    return set_error(GNN_ERR_ARG, "relative_position_bias: B, U, V, H and buckets must be positive, V H below 2^31");
  if (a.max_distance < 1 || a.max_distance > (1 << 28))
    return set_error(GNN_ERR_ARG, "relative_position_bias: max_distance must be in 1 .. 2^28");
  if (!a.log_spacing) {
    if (a.buckets != (a.two_sided ? 2 : 1) * a.max_distance + 1)
      return set_error(GNN_ERR_ARG, "relative_position_bias: clip needs 2 max_distance + 1 buckets, one-sided max_distance + 1");
    return GNN_OK;
  }
  const int64_t n = a.buckets / (a.two_sided ? 2 : 1), near = n / 2, m = n - near;
  if (n < 2 || (a.two_sided && a.buckets % 2) || a.max_distance <= near)
    return set_error(GNN_ERR_ARG, "relative_position_bias: log needs 2 buckets a side or more and a max_distance above half of them");
  if (m > GNN_RELPOS_MAX_BORDERS)
    return set_error(GNN_ERR_UNSUPPORTED, "relative_position_bias: more than 256 logarithmic buckets a side");
  if (m > 1 && !a.border) return set_error(GNN_ERR_ARG, "relative_position_bias: log needs its borders");
  for (int64_t k = 0; k + 1 < m; ++k)
    if (a.border[k] < (k ? a.border[k - 1] : near) || a.border[k] > a.max_distance)
      return set_error(GNN_ERR_ARG, "relative_position_bias: borders must ascend and not pass max_distance");
  return GNN_OK;
}

int gnn_relpos_fwd(const gnn_relpos_args* args, void* stream) {
  if (int rc = check_relpos(args)) return rc;
  if (!args->table || !args->query_pos || !args->key_pos || !args->out)
    return set_error(GNN_ERR_ARG, "relative_position_bias: table, positions and out are required");
  if (!aligned(args->out, args->dtype == GNN_F32 ? 4 : 2))
    return set_error(GNN_ERR_ARG, "relative_position_bias: out must be aligned to its elements");
  int rc = relpos(*args, false, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "relative_position_bias");
}

int64_t gnn_relpos_parts(const gnn_relpos_args* args) { return check_relpos(args) ? 0 : relpos_parts(*args); }

int gnn_relpos_bwd(const gnn_relpos_args* args, void* stream) {
  if (int rc = check_relpos(args)) return rc;
  if (!args->query_pos || !args->key_pos || !args->dout || !args->partial || args->parts < 1)
    return set_error(GNN_ERR_ARG, "relative_position_bias backward: positions, dout, partial and parts are required");
  if (!aligned(args->dout, args->dtype == GNN_F32 ? 4 : 2))
    return set_error(GNN_ERR_ARG, "relative_position_bias backward: dout must be aligned to its elements");
  if (!aligned(args->dtable, args->dtype == GNN_F32 ? 4 : 2))
    return set_error(GNN_ERR_ARG, "relative_position_bias backward: dtable must be aligned to its elements");
  int rc = relpos(*args, true, (hipStream_t)stream);
  if (rc == 0 && args->dtable) {
    const int64_t n = args->buckets * args->H;
    gnn_reduce_args r{};
    r.seg[r.count++] = {args->partial, args->dtable, args->parts, n, n, args->dtype, 0};
    rc = reduce_parts(r, (hipStream_t)stream);
  }
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "relative_position_bias backward");
}

int gnn_linear(const gnn_linear_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "fused_linear: args is NULL");
  const gnn_linear_args& a = *args;
  if (!a.x || !a.w || !a.out || (a.dz && !a.side))
    return set_error(GNN_ERR_ARG, "fused_linear: x, w, out and, for dz, the output gradient are required");
  if (!known_dtype(a.dtype)) return set_error(GNN_ERR_ARG, "fused_linear: unknown dtype");
  if (a.precision != GNN_PREC_IEEE && a.precision != GNN_PREC_BF16X3)
    return set_error(GNN_ERR_ARG, "fused_linear: unknown precision");
  if (a.activation < GNN_ACT_NONE || a.activation > GNN_ACT_SIGMOID)
    return set_error(GNN_ERR_ARG, "fused_linear: unknown activation");
  const int64_t most = (int64_t)1 << 30;
  if (a.M < 1 || a.I < 1 || a.O < 1 || a.I > most || a.O > most || a.out_cols < a.O || a.out_cols > most)
    return set_error(GNN_ERR_ARG, "fused_linear: M, I and O must be positive, I and out_cols at most 2^30, out_cols at least O");
  const int64_t e = a.dtype == GNN_F32 ? 4 : 2;
  if (!aligned(a.x, 16) || !aligned(a.w, 16) || (a.I * e) % 16 || (a.x_ld * e) % 16 || (a.w_ld * e) % 16)
    return set_error(GNN_ERR_ARG, "fused_linear: rows of x and w must be 16-byte aligned and multiples of 16 bytes");
  if (a.x_ld < 0 || a.w_ld < (a.w_transposed ? a.O : a.I) || (a.side && a.side_ld < 0) || a.out_ld < a.out_cols ||
      (a.dx && a.dx_ld < a.I))
    return set_error(GNN_ERR_ARG, "fused_linear: row pitches must cover their rows");
  if (!aligned(a.bias, e) || !aligned(a.side, e) || !aligned(a.out, e))
    return set_error(GNN_ERR_ARG, "fused_linear: tensors must be aligned to their elements");
  if (a.dx && !linear_takes_dx(a))
    return set_error(GNN_ERR_UNSUPPORTED, "fused_linear: this call does not take dx");
  if (a.w_transposed && !linear_takes_transposed(a))
    return set_error(GNN_ERR_UNSUPPORTED, "fused_linear: this call does not take a transposed weight");
  int rc = linear(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "fused_linear");
}

int gnn_linear_takes_dx(const gnn_linear_args* args) { return args && args->dx && linear_takes_dx(*args) ? 1 : 0; }

int gnn_linear_takes_transposed(const gnn_linear_args* args) { return args && linear_takes_transposed(*args) ? 1 : 0; }

static gnn_rows_product_args wgrad_product(const gnn_linear_wgrad_args& a) {
  gnn_rows_product_args r{};
  r.rows = a.M, r.count = 1, r.dtype = a.dtype;
  r.p[0] = {a.dz, a.x, a.partial, a.dz_ld, a.x_ld, a.O, a.I};
  if (a.slices > 0 && a.M > 0) r.slice_rows = ((a.M + a.slices - 1) / a.slices + 31) / 32 * 32;
  return r;
}

int64_t gnn_linear_wgrad_slices(const gnn_linear_wgrad_args* args) {
  if (!args) return 0;
  gnn_linear_wgrad_args a = *args;
  a.slices = 0;
  const gnn_rows_product_args r = wgrad_product(a);
  return gnn_rows_product_slices(&r);
}

int gnn_linear_wgrad(const gnn_linear_wgrad_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "fused_linear gradients: args is NULL");
  const gnn_linear_wgrad_args& a = *args;
  if (a.slices < 1 || a.slices >= ((int64_t)1 << 31) || a.outputs < 1 || a.outputs > a.O)
    return set_error(GNN_ERR_ARG, "fused_linear gradients: slices must be positive, outputs from 1 to O");
  const gnn_rows_product_args r = wgrad_product(a);
  if (int rc = check_rows_product(&r, true)) return rc;
  const int bytes = a.dtype == GNN_F32 ? 4 : 2;
  if (!a.dw || !aligned(a.dw, bytes) || !aligned(a.db, bytes) || !aligned(a.partial, 4))
    return set_error(GNN_ERR_ARG, "fused_linear gradients: dw is required, dw, db and partial aligned to their elements");
  const int64_t used = (a.M + r.slice_rows - 1) / r.slice_rows, each = a.O * a.I;
  float* sums = a.db ? a.partial + used * each : nullptr;
  int rc = rows_product(r, sums, (hipStream_t)stream);
  if (rc == 0) {
    gnn_reduce_args add{};
    add.seg[add.count++] = {a.partial, a.dw, used, each, a.outputs * a.I, a.dtype, 0};
    if (a.db) add.seg[add.count++] = {sums, a.db, used, a.O, a.outputs, a.dtype, 0};
    rc = reduce_parts(add, (hipStream_t)stream);
  }
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "fused_linear gradients");
}

int gnn_pad_rows(const gnn_pad_rows_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "pad_rows: args is NULL");
  const gnn_pad_rows_args& a = *args;
  if (!a.src || !a.dst) return set_error(GNN_ERR_ARG, "pad_rows: src and dst are required");
  if (!known_dtype(a.dtype)) return set_error(GNN_ERR_ARG, "pad_rows: unknown dtype");
  const int chunk = a.dtype == GNN_F32 ? 4 : 8;
  if (a.rows < 1 || a.cols < 1 || a.ld < a.cols || a.ld > ((int64_t)1 << 24) || a.ld % chunk)
    return set_error(GNN_ERR_ARG, "pad_rows: rows and cols must be positive, ld a multiple of 16 bytes from cols to 2^24");
  if (!aligned(a.src, 16 / chunk) || !aligned(a.dst, 16))
    return set_error(GNN_ERR_ARG, "pad_rows: src must be aligned to its elements, dst to 16 bytes");
  int rc = pad_rows(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "pad_rows");
}

int64_t gnn_column_sums_parts(int64_t M, int64_t O) { return M < 1 || O < 1 ? 0 : column_sums_parts(M, O); }

int gnn_column_sums(const gnn_column_sums_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "column_sums: args is NULL");
  const gnn_column_sums_args& a = *args;
  if (!a.d || !a.partial) return set_error(GNN_ERR_ARG, "column_sums: d and partial are required");
  if (!known_dtype(a.dtype)) return set_error(GNN_ERR_ARG, "column_sums: unknown dtype");
  if (a.M < 1 || a.O < 1 || a.O > (1 << 24) || a.parts < 1 || a.parts >= ((int64_t)1 << 31) || a.ld < 0)
    return set_error(GNN_ERR_ARG, "column_sums: M, O and parts must be positive, O at most 2^24");
  if (!aligned(a.d, a.dtype == GNN_F32 ? 4 : 2))
    return set_error(GNN_ERR_ARG, "column_sums: d must be aligned to its elements");
  int rc = column_sums(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "column_sums");
}

int gnn_gated_linear(const gnn_gated_linear_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "gated_linear: args is NULL");
  const gnn_gated_linear_args& a = *args;
  if (!a.x || !a.wg || !a.wu || !a.out) return set_error(GNN_ERR_ARG, "gated_linear: x, wg, wu and out are required");
  if (!known_dtype(a.dtype)) return set_error(GNN_ERR_ARG, "gated_linear: unknown dtype");
  if (a.precision != GNN_PREC_IEEE && a.precision != GNN_PREC_BF16X3)
    return set_error(GNN_ERR_ARG, "gated_linear: unknown precision");
  if (a.activation < GNN_ACT_NONE || a.activation > GNN_ACT_SIGMOID)
    return set_error(GNN_ERR_ARG, "gated_linear: unknown activation");
  const int64_t most = (int64_t)1 << 29;
  if (a.M < 1 || a.M > (int64_t)1 << 40 || a.I < 1 || a.O < 1 || a.I > most || a.O > most || a.out_cols != (a.O + 7) / 8 * 8)
    return set_error(GNN_ERR_ARG, "gated_linear: M, I and O must be positive, M at most 2^40, I and O 2^29, out_cols O rounded up to 8");
  const int64_t e = a.dtype == GNN_F32 ? 4 : 2;
  if (!aligned(a.x, 16) || !aligned(a.wg, 16) || !aligned(a.wu, 16) || (a.I * e) % 16 || (a.x_ld * e) % 16 ||
      (a.wg_ld * e) % 16 || (a.wu_ld * e) % 16)
    return set_error(GNN_ERR_ARG, "gated_linear: rows of x, wg and wu must be 16-byte aligned and multiples of 16 bytes");
  if (a.x_ld < 0 || a.wg_ld < a.I || a.wu_ld < a.I || (a.dy && a.dy_ld < 0) || a.out_ld < (a.dy ? 2 * a.out_cols : a.O))
    return set_error(GNN_ERR_ARG, "gated_linear: row pitches must cover their rows");
  if (!aligned(a.bg, e) || !aligned(a.bu, e) || !aligned(a.dy, e) || !aligned(a.out, e))
    return set_error(GNN_ERR_ARG, "gated_linear: tensors must be aligned to their elements");
  int rc = gated_linear(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "gated_linear");
}

int gnn_gated_turn(const gnn_gated_turn_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "gated_turn: args is NULL");
  const gnn_gated_turn_args& a = *args;
  if (!a.wg || !a.wu || !a.dst) return set_error(GNN_ERR_ARG, "gated_turn: wg, wu and dst are required");
  if (!known_dtype(a.dtype)) return set_error(GNN_ERR_ARG, "gated_turn: unknown dtype");
  const int64_t most = (int64_t)1 << 29;
  if (a.I < 1 || a.O < 1 || a.I > most || a.O > most || a.out_cols < a.O || a.out_cols > most || a.out_cols % 8)
    return set_error(GNN_ERR_ARG, "gated_turn: I and O must be positive, out_cols a multiple of 8 from O on");
  const size_t e = a.dtype == GNN_F32 ? 4 : 2;
  if (a.wg_ld < a.I || a.wu_ld < a.I) return set_error(GNN_ERR_ARG, "gated_turn: row pitches must cover their rows");
  if (!aligned(a.wg, e) || !aligned(a.wu, e) || !aligned(a.dst, 16))
    return set_error(GNN_ERR_ARG, "gated_turn: weights must be aligned to their elements, dst to 16 bytes");
  int rc = gated_turn(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "gated_turn");
}

static gnn_rows_product_args gated_wgrad_product(const gnn_gated_linear_wgrad_args& a) {
  gnn_rows_product_args r{};
  r.rows = a.M, r.count = 1, r.dtype = a.dtype;
  r.p[0] = {a.dz, a.x, a.partial, a.dz_ld, a.x_ld, 2 * a.O, a.I};
  if (a.slices > 0 && a.M > 0) r.slice_rows = ((a.M + a.slices - 1) / a.slices + 31) / 32 * 32;
  return r;
}

int64_t gnn_gated_linear_wgrad_slices(const gnn_gated_linear_wgrad_args* args) {
  if (!args) return 0;
  gnn_gated_linear_wgrad_args a = *args;
  a.slices = 0;
  const gnn_rows_product_args r = gated_wgrad_product(a);
  return gnn_rows_product_slices(&r);
}

int gnn_gated_linear_wgrad(const gnn_gated_linear_wgrad_args* args, void* stream) {
  if (!args) return set_error(GNN_ERR_ARG, "gated_linear gradients: args is NULL");
  const gnn_gated_linear_wgrad_args& a = *args;
  if (a.slices < 1 || a.slices >= ((int64_t)1 << 31) || a.O < 8 || a.O % 8 || a.outputs < 1 || a.outputs > a.O)
    return set_error(GNN_ERR_ARG, "gated_linear gradients: slices must be positive, O a multiple of 8, outputs from 1 to O");
  const gnn_rows_product_args r = gated_wgrad_product(a);
  if (int rc = check_rows_product(&r, true)) return rc;
  const int bytes = a.dtype == GNN_F32 ? 4 : 2;
  void* dst[4] = {a.dwg, a.dwu, a.dbg, a.dbu};
  for (void* p : dst)
    if (!aligned(p, bytes)) return set_error(GNN_ERR_ARG, "gated_linear gradients: outputs must be aligned to their elements");
  if (!a.dwg && !a.dwu && !a.dbg && !a.dbu) return set_error(GNN_ERR_ARG, "gated_linear gradients: an output is required");
  const int64_t used = (a.M + r.slice_rows - 1) / r.slice_rows, each = 2 * a.O * a.I;
  float* sums = a.dbg || a.dbu ? a.partial + used * each : nullptr;
  int rc = rows_product(r, sums, (hipStream_t)stream);
  if (rc == 0) {
    gnn_reduce_args add{};
    for (int k = 0; k < 2; ++k) {
      if (dst[k]) add.seg[add.count++] = {a.partial + k * a.O * a.I, dst[k], used, each, a.outputs * a.I, a.dtype, 0};
      if (dst[2 + k]) add.seg[add.count++] = {sums + k * a.O, dst[2 + k], used, 2 * a.O, a.outputs, a.dtype, 0};
    }
    rc = reduce_parts(add, (hipStream_t)stream);
  }
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "gated_linear gradients");
}

// Whether a side's heads can be counted and numbered
static bool qk_rotary_rows_fit(const gnn_qk_rotary_args& a, int side) {
  const int64_t most = (int64_t)1 << 34;
  const __int128 tokens = (__int128)a.B * a.N[side];
  return tokens < most && tokens * a.H[side] < most;
}

static int check_qk_rotary(const gnn_qk_rotary_args* args, bool bwd) {
  if (!args) return set_error(GNN_ERR_ARG, "qk_norm_rotary: args is NULL");
  const gnn_qk_rotary_args& a = *args;
  if (!known_dtype(a.dtype)) return set_error(GNN_ERR_ARG, "qk_norm_rotary: unknown dtype");
  if (a.param_dtype != a.dtype && a.param_dtype != GNN_F32)
    return set_error(GNN_ERR_ARG, "qk_norm_rotary: weights must be in the rows' dtype or fp32");
  if (a.pos_bytes != 4 && a.pos_bytes != 8)
    return set_error(GNN_ERR_ARG, "qk_norm_rotary: positions must have 4 or 8 bytes");
  if (a.D < 8 || a.D > 256 || a.D % 8 || a.R < 0 || a.R > a.D || a.R % 8)
    return set_error(GNN_ERR_ARG, "qk_norm_rotary: D must be a multiple of 8 up to 256, R a multiple of 8 up to D");
  if (a.R && (a.pos[0] || a.pos[1]) && !a.frequencies)
    return set_error(GNN_ERR_ARG, "qk_norm_rotary: a rotation needs its frequencies");
  if (a.B < 0) return set_error(GNN_ERR_ARG, "qk_norm_rotary: B must not be negative");
  const size_t e = a.dtype == GNN_F32 ? 4 : 2, we = a.param_dtype == GNN_F32 ? 4 : 2;
  for (int k = 0; k < 2; ++k) {
    if (a.N[k] < 0 || a.H[k] < 0 || a.H[k] > (1 << 20))
      return set_error(GNN_ERR_ARG, "qk_norm_rotary: N must not be negative, H in 0 .. 2^20");
    if (!a.norm && (a.weight[k] || a.dweight[k])) return set_error(GNN_ERR_ARG, "qk_norm_rotary: weights go with norms");
    if (!aligned(a.x[k], e) || !aligned(a.dy[k], e) || !aligned(a.out[k], e) || !aligned(a.weight[k], we) ||
        !aligned(a.dweight[k], we) || !aligned(a.pos[k], a.pos_bytes))
      return set_error(GNN_ERR_ARG, "qk_norm_rotary: tensors must be aligned to their elements");
    if (!a.B || !a.N[k] || !a.H[k]) continue;
    if (!qk_rotary_rows_fit(a, k)) return set_error(GNN_ERR_UNSUPPORTED, "qk_norm_rotary: B N H must be below 2^34");
    if (!a.x[k] || (bwd ? !a.dy[k] : !a.out[k]))
      return set_error(GNN_ERR_ARG, "qk_norm_rotary: x and out, or in the backward x and dy, are required");
    if (bwd && (a.parts[k] < 1 || a.parts[k] >= ((int64_t)1 << 30)))
      return set_error(GNN_ERR_ARG, "qk_norm_rotary: parts must be positive and fit a grid");
    if (bwd && a.dweight[k] && !a.partial) return set_error(GNN_ERR_ARG, "qk_norm_rotary: dweight needs partial");
  }
  return GNN_OK;
}

int gnn_qk_rotary_fwd(const gnn_qk_rotary_args* args, void* stream) {
  if (int rc = check_qk_rotary(args, false)) return rc;
  int rc = qk_rotary(*args, false, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "qk_norm_rotary");
}

int64_t gnn_qk_rotary_parts(const gnn_qk_rotary_args* args, int32_t side) {
  if (!args || side < 0 || side > 1 || args->D < 8 || args->D > 256 || args->B < 0 || args->N[side] < 0 ||
      args->H[side] < 1 || args->H[side] > (1 << 20) || !qk_rotary_rows_fit(*args, side))
    return 0;
  return qk_rotary_parts(*args, side);
}

int gnn_qk_rotary_bwd(const gnn_qk_rotary_args* args, void* stream) {
  if (int rc = check_qk_rotary(args, true)) return rc;
  const gnn_qk_rotary_args& a = *args;
  int rc = qk_rotary(a, true, (hipStream_t)stream);
  if (rc == 0) {
    gnn_reduce_args r{};
    const float* partial = a.partial;
    for (int k = 0; k < 2; ++k)
      if (a.dweight[k] && a.B && a.N[k] && a.H[k]) {
        r.seg[r.count++] = {partial, a.dweight[k], a.parts[k], a.D, a.D, a.param_dtype, 0};
        partial += a.parts[k] * a.D;
      }
    if (r.count) rc = reduce_parts(r, (hipStream_t)stream);
  }
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "qk_norm_rotary backward");
}

extern "C++" {
// Whether the kernels' 32-bit offsets reach 64 rows of a product, tokens of `group` heads each
static bool within_reach(const int64_t* stride, int64_t tokens, int64_t group, size_t element) {
  const int64_t most = ((int64_t)1 << 31) / (int64_t)element, token = tokens > 1 ? stride[1] : 0;
  if (token < 0 || token >= most / 64) return false;
  return group == 1 || (stride[2] >= 0 && stride[2] <= (most - 1 - 64 * token) / (group - 1));
}
// Shapes and types that the attention's two directions share
template <typename Args>
static int check_cross_attn(const Args* args) {
  if (!args) return set_error(GNN_ERR_ARG, "cross_attention: args is NULL");
  const Args& a = *args;
  if (!known_dtype(a.dtype)) return set_error(GNN_ERR_ARG, "cross_attention: unknown dtype");
  if (a.precision != GNN_PREC_IEEE && a.precision != GNN_PREC_BF16X3)
    return set_error(GNN_ERR_ARG, "cross_attention: unknown precision");
  if (a.D < 8 || a.D > 128 || a.D % 8)
    return set_error(GNN_ERR_UNSUPPORTED, "cross_attention: the head dim must be a multiple of 8 up to 128");
  const int64_t most = (int64_t)1 << 30;
  if (a.B < 1 || a.U < 1 || a.V < 1 || a.H < 1 || a.Hk < 1 || a.B > most || a.U > most || a.V > most || a.H > most ||
      a.H % a.Hk || a.U * (a.H / a.Hk) > most)
    return set_error(GNN_ERR_ARG, "cross_attention: B, U, V, H and Hk must be positive, U H / Hk and V at most 2^30, H a multiple of Hk");
  const int64_t grid = (int64_t)1 << 31;
  if ((__int128)a.B * a.U * a.H >= grid || (__int128)a.B * a.Hk * ((a.V + 127) / 128) >= grid)
    return set_error(GNN_ERR_UNSUPPORTED, "cross_attention: grid too large");
  if (!(a.scale > 0.f) || a.scale > 3e38f) return set_error(GNN_ERR_ARG, "cross_attention: scale must be positive");
  if (!a.q || !a.k || !a.v) return set_error(GNN_ERR_ARG, "cross_attention: q, k and v are required");
  const size_t e = a.dtype == GNN_F32 ? 4 : 2;
  if (!aligned(a.q, e) || !aligned(a.k, e) || !aligned(a.v, e) || !aligned(a.bias, e) || !aligned(a.stats, 4))
    return set_error(GNN_ERR_ARG, "cross_attention: tensors must be aligned to their elements");
  if (!within_reach(a.q_stride, a.U, a.H / a.Hk, e) || !within_reach(a.k_stride, a.V, 1, e) || !within_reach(a.v_stride, a.V, 1, e))
    return set_error(GNN_ERR_UNSUPPORTED, "cross_attention: 64 tokens must span less than 2^31 bytes");
  return GNN_OK;
}
}  // extern "C++"

size_t gnn_cross_attn_workspace_bytes(const gnn_cross_attn_args* args) {
  return check_cross_attn(args) ? 0 : cross_attn_workspace_bytes(*args);
}

int gnn_cross_attn_fwd(const gnn_cross_attn_args* args, void* stream) {
  if (int rc = check_cross_attn(args)) return rc;
  if (!args->o || !aligned(args->o, 16) || !aligned(args->o_low, 16) || !aligned(args->workspace, 16))
    return set_error(GNN_ERR_ARG, "cross_attention: o is required, o, o_low and the workspace 16-byte aligned");
  int rc = cross_attn_fwd(*args, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "cross_attention");
}

size_t gnn_cross_attn_bwd_workspace_bytes(const gnn_cross_attn_bwd_args* args) {
  return check_cross_attn(args) ? 0 : cross_attn_bwd_workspace_bytes(*args);
}

int gnn_cross_attn_bwd(const gnn_cross_attn_bwd_args* args, void* stream) {
  if (int rc = check_cross_attn(args)) return rc;
  const gnn_cross_attn_bwd_args& a = *args;
  if (!a.o || !a.dout || !a.stats || !a.dq || !a.dk != !a.dv || (a.dbias && !a.bias))
    return set_error(GNN_ERR_ARG, "cross_attention backward: o, dout, stats and dq are required, dk and dv go together, dbias with bias");
  if (a.shared_bias && a.bias_stride[0] != 0)
    return set_error(GNN_ERR_ARG, "cross_attention backward: a shared bias has batch stride 0");
  const size_t e = a.dtype == GNN_F32 ? 4 : 2;
  if (!aligned(a.o, e) || !aligned(a.o_low, e) || !aligned(a.dout, e) || !aligned(a.dbias, e) || !aligned(a.dq, 16) || !aligned(a.dk, 16) ||
      !aligned(a.dv, 16) || !aligned(a.workspace, 16))
    return set_error(GNN_ERR_ARG, "cross_attention backward: o, dout and dbias must be aligned to their elements, dq, dk, dv and the workspace to 16 bytes");
  if (!within_reach(a.o_stride, a.U, a.H / a.Hk, e) || !within_reach(a.do_stride, a.U, a.H / a.Hk, e))
    return set_error(GNN_ERR_UNSUPPORTED, "cross_attention backward: 64 tokens must span less than 2^31 bytes");
  int rc = cross_attn_bwd(a, (hipStream_t)stream);
  if (rc < 0) return rc;
  return hip_status((hipError_t)rc, "cross_attention backward");
}

const char* gnn_last_error(void) { return g_last_error.c_str(); }

const char* gnn_version(void) { return "0.1.0 gfx950"; }

}  // extern "C"
