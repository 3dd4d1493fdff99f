// The gated unit of a transformer MLP, y = act(gate) * up: forward (writing 8-bit checkpoints of gate
// and up in the same pass when asked to) and backward from those checkpoints.
//   silu(g) = g s,  s = 1 / (1 + e^-g)          silu'(g) = s (1 + g (1 - s))
//   gelu(g) = g P,  P = erfc(-g / sqrt 2) / 2    gelu'(g) = P + g e^(-g^2/2) / sqrt(2 pi)
//   relu(g) = max(g, 0)                          relu'(g) = 1 for g > 0, else 0
// dup = dy act(g), dgate = dy up act'(g), product = act(g) up, all in fp32, rounded once to the tensors' type.
// Bound by memory (8.06 bytes per value forward with checkpoints, 8.06 backward, bf16), with the arithmetic close behind: about 40
// instructions per value leave a third of the issue slots; and by the grid of eight CTAs per SM, of which six (16-bit forward) and
// five (16-bit backward) fit at a time. One pass, eight values per lane. [8192, 11008] bf16: silu forward with
// checkpoints 141 us (5.1 TB/s), backward 166 us (4.4 TB/s); gelu 167 and 196 us; fp32 silu 226 us each way (5.6 TB/s).
#include "ckpt8.cuh"
#include "dwbnq_internal.h"

namespace dwbnq {

namespace {

constexpr int kThreads = 256;

// For 16-bit tensors the exponential and the reciprocal are the hardware's approximations (a few 2^-23; the exponential's argument
// is rounded first, which a large one turns into more): the result keeps 8 or 11 bits. erfc, which as a library call made the
// gelu kernels compute-bound (235 and 276 us on [8192, 11008] bf16, where silu takes 147 and 165), is there
//   erfc(x) = t 2^{p(t)} e^{-x^2},  t = 1 / (1 + x / 2),  x >= 0,
// with p a polynomial of degree 8, the interpolant of log2(erfc(x) e^{x^2} / t) at the Chebyshev points of t in [0.15, 1]
// (x up to 11, beyond which e^{-x^2} is 0): off by 3.8e-7 at most, relatively, evaluated in fp32. The derivative needs e^{-x^2} too.
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Normal distribution function of g, and e^(-g^2/2).
__device__ __forceinline__ float fast_normal(float g, float &e) {
  const float t = fast_rcp(__fmaf_rn(fabsf(g), 0.35355339059327376f, 1.0f));
  float p = 0.096491605f;
  p = __fmaf_rn(p, t, -0.718809724f);
  p = __fmaf_rn(p, t, 1.9594866f);
  p = __fmaf_rn(p, t, -2.3799293f);
  p = __fmaf_rn(p, t, 1.10016215f);
  p = __fmaf_rn(p, t, -0.286739916f);
  p = __fmaf_rn(p, t, 0.620371938f);
  p = __fmaf_rn(p, t, 1.43435168f);
  p = __fmaf_rn(p, t, -1.82538545f);
  e = fast_exp2(__fmul_rn(__fmul_rn(g, -0.72134752044448170f), g));
  const float r = __fmul_rn(__fmul_rn(0.5f, t), __fmul_rn(fast_exp2(p), e));
  return g < 0.0f ? r : __fsub_rn(1.0f, r);
}
template <typename T> __device__ __forceinline__ float glu_sigmoid(float g) {
  if (sizeof(T) == 4) return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-g)));
  return fast_rcp(__fadd_rn(1.0f, fast_exp2(__fmul_rn(g, -1.4426950408889634f))));
}
template <typename T, int ACT>
__device__ __forceinline__ float act_value(float g) {
  if (ACT == DWBNQ_ACT_SILU) return __fmul_rn(g, glu_sigmoid<T>(g));
  if (ACT == DWBNQ_ACT_GELU) {
    float e;
    return __fmul_rn(g, sizeof(T) == 4 ? __fmul_rn(0.5f, erfcf(__fmul_rn(g, -0.70710678118654752f))) : fast_normal(g, e));
  }
  return g > 0.0f ? g : (g != g ? g : 0.0f);
}
template <typename T, int ACT>
__device__ __forceinline__ void act_both(float g, float &a, float &d) {
  if (ACT == DWBNQ_ACT_SILU) {
    const float s = glu_sigmoid<T>(g);
    a = __fmul_rn(g, s);
    d = __fmul_rn(s, __fmaf_rn(g, __fsub_rn(1.0f, s), 1.0f));
  } else if (ACT == DWBNQ_ACT_GELU) {
    float p, e;
    if (sizeof(T) == 4) {
      p = __fmul_rn(0.5f, erfcf(__fmul_rn(g, -0.70710678118654752f)));
      e = expf(__fmul_rn(__fmul_rn(g, -0.5f), g));
    } else {
      p = fast_normal(g, e);
    }
    a = __fmul_rn(g, p);
    d = __fmaf_rn(__fmul_rn(g, 0.39894228040143268f), e, p);
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
  OctetGrid grid;
};

template <typename T, int ACT, bool CKPT, bool VECTORS>
__global__ void __launch_bounds__(kThreads, VECTORS && sizeof(T) == 2 ? 6 : 4) glu_fwd_kernel(const GluFwdArgs a) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  float *stage = OctetStage<VECTORS>::get();
  for (OctetWalk w = octet_walk(a.grid, a.rows); __any_sync(0xffffffffu, w.row < a.rows); octet_next(w)) {
    const bool in = w.row < a.rows;
    const long long c = w.col * 8LL, n = in ? a.cols - c : 0;
    float g[8], u[8], y[8];
    Octet<T, VECTORS>::load(static_cast<const T *>(a.gate) + w.row * a.ld_gate + c, n, stage, g);
    Octet<T, VECTORS>::load(static_cast<const T *>(a.up) + w.row * a.ld_up + c, n, stage, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = __fmul_rn(act_value<T, ACT>(g[k]), u[k]);
    Octet<T, VECTORS>::store(static_cast<T *>(a.y) + w.row * a.ld_y + c, n, stage, y);
    if (CKPT) {
      ck_put(g, in, w.row * w.per_row + w.col, a.gate_codes, a.gate_exps);
      ck_put(u, in, w.row * w.per_row + w.col, a.up_codes, a.up_exps);
    }
  }
}

template <typename T, bool VECTORS>
__device__ __forceinline__ void put_gradient(T *p, long long n, bool accum, float *stage, float *v) {
  if (accum) {
    float old[8];
    Octet<T, VECTORS>::load(p, n, stage, old);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __fadd_rn(old[k], v[k]);
  }
  Octet<T, VECTORS>::store(p, n, stage, v);
}

template <typename T, int ACT, bool VECTORS>
__global__ void __launch_bounds__(kThreads, VECTORS && sizeof(T) == 2 ? 5 : 4) glu_bwd_kernel(const GluBwdArgs a) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  float *stage = OctetStage<VECTORS>::get();
  for (OctetWalk w = octet_walk(a.grid, a.rows); __any_sync(0xffffffffu, w.row < a.rows); octet_next(w)) {
    const bool in = w.row < a.rows;
    const long long c = w.col * 8LL, n = in ? a.cols - c : 0, at = w.row * w.per_row + w.col;
    float g[8], u[8], dy[8], t[8], d[8];
    ck_get(a.gate_codes, a.gate_exps, in, at, g);
    ck_get(a.up_codes, a.up_exps, in, at, u);
    Octet<T, VECTORS>::load(static_cast<const T *>(a.dy) + w.row * a.ld_dy + c, a.dy ? n : 0, stage, dy);
#pragma unroll
    for (int k = 0; k < 8; ++k) act_both<T, ACT>(g[k], t[k], d[k]);
    if (a.dgate) {
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] = __fmul_rn(__fmul_rn(dy[k], u[k]), d[k]);
      put_gradient<T, VECTORS>(static_cast<T *>(a.dgate) + w.row * a.ld_dgate + c, n, (a.accum & 1) != 0, stage, d);
    }
    if (a.dup) {
#pragma unroll
      for (int k = 0; k < 8; ++k) dy[k] = __fmul_rn(dy[k], t[k]);
      put_gradient<T, VECTORS>(static_cast<T *>(a.dup) + w.row * a.ld_dup + c, n, (a.accum & 2) != 0, stage, dy);
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
  const bool v = octet_vectors(a.gate, a.ld_gate, sizeof(T)) && octet_vectors(a.up, a.ld_up, sizeof(T)) && octet_vectors(a.y, a.ld_y, sizeof(T));
  const dim3 grid(a.grid.ctas), block(kThreads);
  const cudaError_t e = a.gate_codes ? (v ? launch_pdl(glu_fwd_kernel<T, ACT, true, true>, grid, block, 0, stream, a)
                                          : launch_pdl(glu_fwd_kernel<T, ACT, true, false>, grid, block, 0, stream, a))
                                     : (v ? launch_pdl(glu_fwd_kernel<T, ACT, false, true>, grid, block, 0, stream, a)
                                          : launch_pdl(glu_fwd_kernel<T, ACT, false, false>, grid, block, 0, stream, a));
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "glu_fwd_kernel launch");
}
template <typename T, int ACT>
int bwd_t(GluBwdArgs a, cudaStream_t stream) {
  a.grid = octet_grid(a.rows, a.cols, kThreads, sm_count(-1) * 8);
  const bool v = octet_vectors(a.dy, a.ld_dy, sizeof(T)) && (!a.dgate || octet_vectors(a.dgate, a.ld_dgate, sizeof(T))) &&
                 (!a.dup || octet_vectors(a.dup, a.ld_dup, sizeof(T)));
  const dim3 grid(a.grid.ctas), block(kThreads);
  const cudaError_t e = v ? launch_pdl(glu_bwd_kernel<T, ACT, true>, grid, block, 0, stream, a)
                          : launch_pdl(glu_bwd_kernel<T, ACT, false>, grid, block, 0, stream, a);
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
