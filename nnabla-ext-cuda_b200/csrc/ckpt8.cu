// 8-bit activation checkpoints: writing one from a tensor, and reading it back. Both are bound by memory: 3.03 bytes per 16-bit
// value each way.
#include "ckpt8.cuh"
#include "dwbnq_internal.h"

namespace dwbnq {

namespace {

constexpr int kThreads = 256, kUnroll = 2;  // octets a thread has in flight

template <typename T>
__global__ void __launch_bounds__(kThreads)
    ckpt8_store_kernel(const T *__restrict__ x, long long ld, int access, long long rows, long long cols, const OctetGrid g,
                       signed char *__restrict__ codes, unsigned char *__restrict__ exps) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  OctetWalk w = octet_walk(g, rows);
  while (__any_sync(0xffffffffu, w.row < rows)) {
    float v[kUnroll][8];
    long long at[kUnroll];
    bool in[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      in[u] = w.row < rows;
      at[u] = w.row * w.per_row + w.col;
      Octet<T>::load(x + w.row * ld + w.col * 8LL, in[u] ? cols - w.col * 8LL : 0, access, v[u]);
      octet_next(w);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) ck_put(v[u], in[u], at[u], codes, exps);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    ckpt8_load_kernel(const signed char *__restrict__ codes, const unsigned char *__restrict__ exps, long long rows,
                      long long cols, const OctetGrid g, T *__restrict__ y, long long ld, int access) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  OctetWalk w = octet_walk(g, rows);
  while (w.row < rows) {
    float v[kUnroll][8];
    T *to[kUnroll];
    long long n[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const bool in = w.row < rows;
      ck_get(codes, exps, in, w.row * w.per_row + w.col, v[u]);
      to[u] = y + w.row * ld + w.col * 8LL;
      n[u] = in ? cols - w.col * 8LL : 0;
      octet_next(w);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) Octet<T>::store(to[u], n[u], access, v[u]);
  }
}

template <typename T>
int store_t(long long rows, long long cols, long long ld, const void *x, void *codes, void *exps, cudaStream_t stream) {
  const OctetGrid g = octet_grid(rows, cols, kThreads, sm_count(-1) * 8);
  const cudaError_t e = launch_pdl(ckpt8_store_kernel<T>, dim3(g.ctas), dim3(kThreads), 0, stream, static_cast<const T *>(x), ld,
                                   octet_access(x, ld, sizeof(T)), rows, cols, g, static_cast<signed char *>(codes),
                                   static_cast<unsigned char *>(exps));
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "ckpt8_store_kernel launch");
}

template <typename T>
int load_t(long long rows, long long cols, const void *codes, const void *exps, long long ld, void *y, cudaStream_t stream) {
  const OctetGrid g = octet_grid(rows, cols, kThreads, sm_count(-1) * 8);
  const cudaError_t e = launch_pdl(ckpt8_load_kernel<T>, dim3(g.ctas), dim3(kThreads), 0, stream,
                                   static_cast<const signed char *>(codes), static_cast<const unsigned char *>(exps), rows, cols, g,
                                   static_cast<T *>(y), ld, octet_access(y, ld, sizeof(T)));
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
