// The gated unit of a transformer MLP, y = act(gate) * up: forward (writing 8-bit checkpoints of gate
// and up in the same pass when asked to) and backward from those checkpoints.
//   silu(g) = g s,  s = 1 / (1 + e^-g)          silu'(g) = s (1 + g (1 - s))
//   gelu(g) = g P,  P = erfc(-g / sqrt 2) / 2    gelu'(g) = P + g e^(-g^2/2) / sqrt(2 pi)
//   relu(g) = max(g, 0)                          relu'(g) = 1 for g > 0, else 0
// dup = dy act(g), dgate = dy up act'(g), product = act(g) up, all in fp32, rounded once to the tensors' type.
#include "ckpt8.cuh"
#include "dwbnq_internal.h"

namespace dwbnq {

namespace {

constexpr int kThreads = 256;

// For 16-bit tensors the exponential and the division are the hardware's approximations (a few 2^-23, the exponential
// 2 + 1.2 |g| of them): the result keeps 8 or 11 bits.
template <typename T> __device__ __forceinline__ float glu_sigmoid(float g) {
  if (sizeof(T) == 4) return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-g)));
  float s;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(__fadd_rn(1.0f, __expf(-g))));
  return s;
}
template <typename T, int ACT>
__device__ __forceinline__ float act_value(float g) {
  if (ACT == DWBNQ_ACT_SILU) return __fmul_rn(g, glu_sigmoid<T>(g));
  if (ACT == DWBNQ_ACT_GELU) return __fmul_rn(g, __fmul_rn(0.5f, erfcf(__fmul_rn(g, -0.70710678118654752f))));
  return g > 0.0f ? g : (g != g ? g : 0.0f);
}
template <typename T, int ACT>
__device__ __forceinline__ void act_both(float g, float &a, float &d) {
  if (ACT == DWBNQ_ACT_SILU) {
    const float s = glu_sigmoid<T>(g);
    a = __fmul_rn(g, s);
    d = __fmul_rn(s, __fmaf_rn(g, __fsub_rn(1.0f, s), 1.0f));
  } else if (ACT == DWBNQ_ACT_GELU) {
    const float p = __fmul_rn(0.5f, erfcf(__fmul_rn(g, -0.70710678118654752f))), t = __fmul_rn(__fmul_rn(g, -0.5f), g);
    a = __fmul_rn(g, p);
    d = __fmaf_rn(__fmul_rn(g, 0.39894228040143268f), sizeof(T) == 4 ? expf(t) : __expf(t), p);
  } else {
    a = g > 0.0f ? g : (g != g ? g : 0.0f);
    d = g > 0.0f ? 1.0f : (g != g ? g : 0.0f);
  }
}

struct GluFwdArgs {
  const void *gate, *up;
  void *y;
  long long ld_gate, ld_up, ld_y, rows, cols;
  signed char *gate_codes, *up_codes;  // null: no checkpoints
  unsigned char *gate_exps, *up_exps;
  int acc_gate, acc_up, acc_y;  // OctetAccess
  OctetGrid grid;
};
struct GluBwdArgs {
  const signed char *gate_codes, *up_codes;
  const unsigned char *gate_exps, *up_exps;
  const void *dy;
  void *dgate, *dup;  // either may be null
  long long ld_dy, ld_dgate, ld_dup, rows, cols;
  signed char *prod_codes;  // null: the product is not wanted
  unsigned char *prod_exps;
  int accum;  // bit 0 dgate, bit 1 dup
  int acc_dy, acc_dgate, acc_dup;
  OctetGrid grid;
};

template <typename T, int ACT, bool CKPT>
__global__ void __launch_bounds__(kThreads) glu_fwd_kernel(const GluFwdArgs a) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  for (OctetWalk w = octet_walk(a.grid, a.rows); __any_sync(0xffffffffu, w.row < a.rows); octet_next(w)) {
    const bool in = w.row < a.rows;
    const long long c = w.col * 8LL, n = in ? a.cols - c : 0;
    float g[8], u[8], y[8];
    Octet<T>::load(static_cast<const T *>(a.gate) + w.row * a.ld_gate + c, n, a.acc_gate, g);
    Octet<T>::load(static_cast<const T *>(a.up) + w.row * a.ld_up + c, n, a.acc_up, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = __fmul_rn(act_value<T, ACT>(g[k]), u[k]);
    Octet<T>::store(static_cast<T *>(a.y) + w.row * a.ld_y + c, n, a.acc_y, y);
    if (CKPT) {
      ck_put(g, in, w.row * w.per_row + w.col, a.gate_codes, a.gate_exps);
      ck_put(u, in, w.row * w.per_row + w.col, a.up_codes, a.up_exps);
    }
  }
}

template <typename T>
__device__ __forceinline__ void put_gradient(T *p, long long n, int access, bool accum, float *v) {
  if (accum) {
    float old[8];
    Octet<T>::load(p, n, access, old);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __fadd_rn(old[k], v[k]);
  }
  Octet<T>::store(p, n, access, v);
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) glu_bwd_kernel(const GluBwdArgs a) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  for (OctetWalk w = octet_walk(a.grid, a.rows); __any_sync(0xffffffffu, w.row < a.rows); octet_next(w)) {
    const bool in = w.row < a.rows;
    const long long c = w.col * 8LL, n = in ? a.cols - c : 0, at = w.row * w.per_row + w.col;
    float g[8], u[8], dy[8], t[8], d[8];
    ck_get(a.gate_codes, a.gate_exps, in, at, g);
    ck_get(a.up_codes, a.up_exps, in, at, u);
    Octet<T>::load(static_cast<const T *>(a.dy) + w.row * a.ld_dy + c, a.dy ? n : 0, a.acc_dy, dy);
#pragma unroll
    for (int k = 0; k < 8; ++k) act_both<T, ACT>(g[k], t[k], d[k]);
    if (a.dgate) {
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] = __fmul_rn(__fmul_rn(dy[k], u[k]), d[k]);
      put_gradient(static_cast<T *>(a.dgate) + w.row * a.ld_dgate + c, n, a.acc_dgate, (a.accum & 1) != 0, d);
    }
    if (a.dup) {
#pragma unroll
      for (int k = 0; k < 8; ++k) dy[k] = __fmul_rn(dy[k], t[k]);
      put_gradient(static_cast<T *>(a.dup) + w.row * a.ld_dup + c, n, a.acc_dup, (a.accum & 2) != 0, dy);
    }
    if (a.prod_codes) {
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = k < n ? __fmul_rn(t[k], u[k]) : 0.0f;
      ck_put(t, in, at, a.prod_codes, a.prod_exps);
    }
  }
}

template <typename T, int ACT>
int fwd_t(GluFwdArgs a, cudaStream_t stream) {
  a.grid = octet_grid(a.rows, a.cols, kThreads, sm_count(-1) * 8);
  a.acc_gate = octet_access(a.gate, a.ld_gate, sizeof(T));
  a.acc_up = octet_access(a.up, a.ld_up, sizeof(T));
  a.acc_y = octet_access(a.y, a.ld_y, sizeof(T));
  const cudaError_t e = a.gate_codes ? launch_pdl(glu_fwd_kernel<T, ACT, true>, dim3(a.grid.ctas), dim3(kThreads), 0, stream, a)
                                     : launch_pdl(glu_fwd_kernel<T, ACT, false>, dim3(a.grid.ctas), dim3(kThreads), 0, stream, a);
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "glu_fwd_kernel launch");
}
template <typename T, int ACT>
int bwd_t(GluBwdArgs a, cudaStream_t stream) {
  a.grid = octet_grid(a.rows, a.cols, kThreads, sm_count(-1) * 8);
  a.acc_dy = octet_access(a.dy, a.ld_dy, sizeof(T));
  a.acc_dgate = octet_access(a.dgate, a.ld_dgate, sizeof(T));
  a.acc_dup = octet_access(a.dup, a.ld_dup, sizeof(T));
  const cudaError_t e = launch_pdl(glu_bwd_kernel<T, ACT>, dim3(a.grid.ctas), dim3(kThreads), 0, stream, a);
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "glu_bwd_kernel launch");
}
template <typename T>
int fwd_act(int act, const GluFwdArgs &a, cudaStream_t s) {
  return act == DWBNQ_ACT_SILU ? fwd_t<T, DWBNQ_ACT_SILU>(a, s)
         : act == DWBNQ_ACT_GELU ? fwd_t<T, DWBNQ_ACT_GELU>(a, s) : fwd_t<T, DWBNQ_ACT_RELU>(a, s);
}
template <typename T>
int bwd_act(int act, const GluBwdArgs &a, cudaStream_t s) {
  return act == DWBNQ_ACT_SILU ? bwd_t<T, DWBNQ_ACT_SILU>(a, s)
         : act == DWBNQ_ACT_GELU ? bwd_t<T, DWBNQ_ACT_GELU>(a, s) : bwd_t<T, DWBNQ_ACT_RELU>(a, s);
}

}  // namespace

int launch_glu_fwd(int dtype, int act, long long rows, long long cols, long long ld_gate, const void *gate, long long ld_up,
                   const void *up, long long ld_y, void *y, void *gate_codes, void *gate_exps, void *up_codes, void *up_exps,
                   cudaStream_t stream) {
  GluFwdArgs a = {};
  a.gate = gate; a.up = up; a.y = y;
  a.ld_gate = ld_gate; a.ld_up = ld_up; a.ld_y = ld_y;
  a.rows = rows; a.cols = cols;
  a.gate_codes = static_cast<signed char *>(gate_codes); a.up_codes = static_cast<signed char *>(up_codes);
  a.gate_exps = static_cast<unsigned char *>(gate_exps); a.up_exps = static_cast<unsigned char *>(up_exps);
  if (dtype == DWBNQ_F32) return fwd_act<float>(act, a, stream);
  if (dtype == DWBNQ_F16) return fwd_act<__half>(act, a, stream);
  return fwd_act<__nv_bfloat16>(act, a, stream);
}

int launch_glu_bwd(int dtype, int act, long long rows, long long cols, const void *gate_codes, const void *gate_exps,
                   const void *up_codes, const void *up_exps, long long ld_dy, const void *dy, long long ld_dgate, void *dgate,
                   long long ld_dup, void *dup, void *prod_codes, void *prod_exps, int accum, cudaStream_t stream) {
  GluBwdArgs a = {};
  a.gate_codes = static_cast<const signed char *>(gate_codes); a.up_codes = static_cast<const signed char *>(up_codes);
  a.gate_exps = static_cast<const unsigned char *>(gate_exps); a.up_exps = static_cast<const unsigned char *>(up_exps);
  a.dy = dy; a.dgate = dgate; a.dup = dup;
  a.ld_dy = ld_dy; a.ld_dgate = ld_dgate; a.ld_dup = ld_dup;
  a.rows = rows; a.cols = cols;
  a.prod_codes = static_cast<signed char *>(prod_codes); a.prod_exps = static_cast<unsigned char *>(prod_exps);
  a.accum = accum;
  if (dtype == DWBNQ_F32) return bwd_act<float>(act, a, stream);
  if (dtype == DWBNQ_F16) return bwd_act<__half>(act, a, stream);
  return bwd_act<__nv_bfloat16>(act, a, stream);
}

}  // namespace dwbnq
