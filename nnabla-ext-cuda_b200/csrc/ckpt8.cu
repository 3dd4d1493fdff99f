// 8-bit activation checkpoints: writing one from a tensor, and reading it back.
#include "ckpt8.cuh"
#include "dwbnq_internal.h"

namespace dwbnq {

namespace {

constexpr int kThreads = 256;

// One warp per group, one lane per value.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ckpt8_store_kernel(const T *__restrict__ x, long long ld, long long rows, long long cols, long long groups,
                       signed char *__restrict__ codes, unsigned char *__restrict__ exps) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const int lane = threadIdx.x & 31;
  const long long total = rows * groups, step = (long long)gridDim.x * (kThreads / 32);
  for (long long g = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); g < total; g += step) {
    const long long r = g / groups, c = (g - r * groups) * kCkGroup + lane;
    const float v = c < cols ? Elem<T>::to_f32(x[r * ld + c]) : 0.0f;
    const unsigned int b = ck_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
    codes[g * kCkGroup + lane] = (signed char)ck_code(v, ck_inv_step(b));
    if (lane == 0) exps[g] = (unsigned char)b;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    ckpt8_load_kernel(const signed char *__restrict__ codes, const unsigned char *__restrict__ exps, long long rows,
                      long long cols, long long groups, T *__restrict__ y, long long ld) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const int lane = threadIdx.x & 31;
  const long long total = rows * groups, step = (long long)gridDim.x * (kThreads / 32);
  for (long long g = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); g < total; g += step) {
    const long long r = g / groups, c = (g - r * groups) * kCkGroup + lane;
    if (c < cols) y[r * ld + c] = Elem<T>::from_f32(__fmul_rn((float)codes[g * kCkGroup + lane], ck_step(exps[g])));
  }
}

unsigned int grid_for(long long warps) {
  const long long blocks = (warps + kThreads / 32 - 1) / (kThreads / 32), cap = (long long)sm_count(-1) * 16;
  return (unsigned int)(blocks > cap ? cap : blocks < 1 ? 1 : blocks);
}

template <typename T>
int store_t(long long rows, long long cols, long long ld, const void *x, void *codes, void *exps, cudaStream_t stream) {
  const long long groups = (cols + kCkGroup - 1) / kCkGroup;
  const cudaError_t e = launch_pdl(ckpt8_store_kernel<T>, dim3(grid_for(rows * groups)), dim3(kThreads), 0, stream,
                                   static_cast<const T *>(x), ld, rows, cols, groups, static_cast<signed char *>(codes),
                                   static_cast<unsigned char *>(exps));
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "ckpt8_store_kernel launch");
}

template <typename T>
int load_t(long long rows, long long cols, const void *codes, const void *exps, long long ld, void *y, cudaStream_t stream) {
  const long long groups = (cols + kCkGroup - 1) / kCkGroup;
  const cudaError_t e = launch_pdl(ckpt8_load_kernel<T>, dim3(grid_for(rows * groups)), dim3(kThreads), 0, stream,
                                   static_cast<const signed char *>(codes), static_cast<const unsigned char *>(exps), rows,
                                   cols, groups, static_cast<T *>(y), ld);
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "ckpt8_load_kernel launch");
}

}  // namespace

int launch_ckpt8_store(int dtype, long long rows, long long cols, long long ld, const void *x, void *codes, void *exps,
                       cudaStream_t stream) {
  if (dtype == DWBNQ_F32) return store_t<float>(rows, cols, ld, x, codes, exps, stream);
  if (dtype == DWBNQ_F16) return store_t<__half>(rows, cols, ld, x, codes, exps, stream);
  return store_t<__nv_bfloat16>(rows, cols, ld, x, codes, exps, stream);
}

int launch_ckpt8_load(int dtype, long long rows, long long cols, const void *codes, const void *exps, long long ld, void *y,
                      cudaStream_t stream) {
  if (dtype == DWBNQ_F32) return load_t<float>(rows, cols, codes, exps, ld, y, stream);
  if (dtype == DWBNQ_F16) return load_t<__half>(rows, cols, codes, exps, ld, y, stream);
  return load_t<__nv_bfloat16>(rows, cols, codes, exps, ld, y, stream);
}

}  // namespace dwbnq
