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

template <int ACT>
__device__ __forceinline__ float act_value(float g) {
  if (ACT == DWBNQ_ACT_SILU) return __fdiv_rn(g, __fadd_rn(1.0f, expf(-g)));
  if (ACT == DWBNQ_ACT_GELU) return __fmul_rn(g, __fmul_rn(0.5f, erfcf(__fmul_rn(g, -0.70710678118654752f))));
  return g > 0.0f ? g : (g != g ? g : 0.0f);
}
template <int ACT>
__device__ __forceinline__ void act_both(float g, float &a, float &d) {
  if (ACT == DWBNQ_ACT_SILU) {
    const float s = __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-g)));
    a = __fmul_rn(g, s);
    d = __fmul_rn(s, __fmaf_rn(g, __fsub_rn(1.0f, s), 1.0f));
  } else if (ACT == DWBNQ_ACT_GELU) {
    const float p = __fmul_rn(0.5f, erfcf(__fmul_rn(g, -0.70710678118654752f)));
    a = __fmul_rn(g, p);
    d = __fmaf_rn(__fmul_rn(g, 0.39894228040143268f), expf(__fmul_rn(__fmul_rn(g, -0.5f), g)), p);
  } else {
    a = g > 0.0f ? g : (g != g ? g : 0.0f);
    d = g > 0.0f ? 1.0f : (g != g ? g : 0.0f);
  }
}

struct GluFwdArgs {
  const void *gate, *up;
  void *y;
  long long ld_gate, ld_up, ld_y, rows, cols, groups;
  signed char *gate_codes, *up_codes;  // null: no checkpoints
  unsigned char *gate_exps, *up_exps;
};
struct GluBwdArgs {
  const signed char *gate_codes, *up_codes;
  const unsigned char *gate_exps, *up_exps;
  const void *dy;
  void *dgate, *dup;  // either may be null
  long long ld_dy, ld_dgate, ld_dup, rows, cols, groups;
  signed char *prod_codes;  // null: the product is not wanted
  unsigned char *prod_exps;
  int accum;  // bit 0 dgate, bit 1 dup
};

__device__ __forceinline__ void put_group(float v, long long g, int lane, signed char *codes, unsigned char *exps) {
  const unsigned int b = ck_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
  codes[g * kCkGroup + lane] = (signed char)ck_code(v, ck_inv_step(b));
  if (lane == 0) exps[g] = (unsigned char)b;
}

// One warp per group of 32 values, one lane per value.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) glu_fwd_kernel(const GluFwdArgs a) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const int lane = threadIdx.x & 31;
  const long long total = a.rows * a.groups, step = (long long)gridDim.x * (kThreads / 32);
  for (long long g = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); g < total; g += step) {
    const long long r = g / a.groups, c = (g - r * a.groups) * kCkGroup + lane;
    float vg = 0.0f, vu = 0.0f;
    if (c < a.cols) {
      vg = Elem<T>::to_f32(static_cast<const T *>(a.gate)[r * a.ld_gate + c]);
      vu = Elem<T>::to_f32(static_cast<const T *>(a.up)[r * a.ld_up + c]);
      static_cast<T *>(a.y)[r * a.ld_y + c] = Elem<T>::from_f32(__fmul_rn(act_value<ACT>(vg), vu));
    }
    if (a.gate_codes) {
      put_group(vg, g, lane, a.gate_codes, a.gate_exps);
      put_group(vu, g, lane, a.up_codes, a.up_exps);
    }
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) glu_bwd_kernel(const GluBwdArgs a) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const int lane = threadIdx.x & 31;
  const long long total = a.rows * a.groups, step = (long long)gridDim.x * (kThreads / 32);
  for (long long g = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); g < total; g += step) {
    const long long r = g / a.groups, c = (g - r * a.groups) * kCkGroup + lane;
    const float vg = __fmul_rn((float)a.gate_codes[g * kCkGroup + lane], ck_step(a.gate_exps[g]));
    const float vu = __fmul_rn((float)a.up_codes[g * kCkGroup + lane], ck_step(a.up_exps[g]));
    float act, der;
    act_both<ACT>(vg, act, der);
    if (c < a.cols) {
      const float dy = a.dy ? Elem<T>::to_f32(static_cast<const T *>(a.dy)[r * a.ld_dy + c]) : 0.0f;
      if (a.dgate) {
        T *p = static_cast<T *>(a.dgate) + r * a.ld_dgate + c;
        float v = __fmul_rn(__fmul_rn(dy, vu), der);
        if (a.accum & 1) v = __fadd_rn(Elem<T>::to_f32(*p), v);
        *p = Elem<T>::from_f32(v);
      }
      if (a.dup) {
        T *p = static_cast<T *>(a.dup) + r * a.ld_dup + c;
        float v = __fmul_rn(dy, act);
        if (a.accum & 2) v = __fadd_rn(Elem<T>::to_f32(*p), v);
        *p = Elem<T>::from_f32(v);
      }
    }
    if (a.prod_codes) put_group(c < a.cols ? __fmul_rn(act, vu) : 0.0f, g, lane, a.prod_codes, a.prod_exps);
  }
}

unsigned int grid_for(long long warps) {
  const long long blocks = (warps + kThreads / 32 - 1) / (kThreads / 32), cap = (long long)sm_count(-1) * 16;
  return (unsigned int)(blocks > cap ? cap : blocks < 1 ? 1 : blocks);
}

template <typename T, int ACT>
int fwd_t(const GluFwdArgs &a, cudaStream_t stream) {
  const cudaError_t e = launch_pdl(glu_fwd_kernel<T, ACT>, dim3(grid_for(a.rows * a.groups)), dim3(kThreads), 0, stream, a);
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "glu_fwd_kernel launch");
}
template <typename T, int ACT>
int bwd_t(const GluBwdArgs &a, cudaStream_t stream) {
  const cudaError_t e = launch_pdl(glu_bwd_kernel<T, ACT>, dim3(grid_for(a.rows * a.groups)), dim3(kThreads), 0, stream, a);
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
  GluFwdArgs a;
  a.gate = gate; a.up = up; a.y = y;
  a.ld_gate = ld_gate; a.ld_up = ld_up; a.ld_y = ld_y;
  a.rows = rows; a.cols = cols; a.groups = (cols + kCkGroup - 1) / kCkGroup;
  a.gate_codes = static_cast<signed char *>(gate_codes); a.up_codes = static_cast<signed char *>(up_codes);
  a.gate_exps = static_cast<unsigned char *>(gate_exps); a.up_exps = static_cast<unsigned char *>(up_exps);
  if (dtype == DWBNQ_F32) return fwd_act<float>(act, a, stream);
  if (dtype == DWBNQ_F16) return fwd_act<__half>(act, a, stream);
  return fwd_act<__nv_bfloat16>(act, a, stream);
}

int launch_glu_bwd(int dtype, int act, long long rows, long long cols, const void *gate_codes, const void *gate_exps,
                   const void *up_codes, const void *up_exps, long long ld_dy, const void *dy, long long ld_dgate, void *dgate,
                   long long ld_dup, void *dup, void *prod_codes, void *prod_exps, int accum, cudaStream_t stream) {
  GluBwdArgs a;
  a.gate_codes = static_cast<const signed char *>(gate_codes); a.up_codes = static_cast<const signed char *>(up_codes);
  a.gate_exps = static_cast<const unsigned char *>(gate_exps); a.up_exps = static_cast<const unsigned char *>(up_exps);
  a.dy = dy; a.dgate = dgate; a.dup = dup;
  a.ld_dy = ld_dy; a.ld_dgate = ld_dgate; a.ld_dup = ld_dup;
  a.rows = rows; a.cols = cols; a.groups = (cols + kCkGroup - 1) / kCkGroup;
  a.prod_codes = static_cast<signed char *>(prod_codes); a.prod_exps = static_cast<unsigned char *>(prod_exps);
  a.accum = accum;
  if (dtype == DWBNQ_F32) return bwd_act<float>(act, a, stream);
  if (dtype == DWBNQ_F16) return bwd_act<__half>(act, a, stream);
  return bwd_act<__nv_bfloat16>(act, a, stream);
}

}  // namespace dwbnq
