// 8-bit activation checkpoints: writing one from a tensor, and reading it back. Both are bound by memory (3.03 bytes per 16-bit
// value each way, a dozen instructions), the restoring of 16-bit values also by its grid - eight CTAs per SM are launched, five fit
// with its registers, so that the last ones run by themselves: a lane has eight values, so that its access is 16 bytes and four lanes share a group; two
// such accesses in flight per thread when writing, four of the 8-byte ones when reading. [16384, 8192] bf16: written in 83 us
// (4.9 TB/s), restored in 97 us (4.2 TB/s; most of its bytes are stores); fp32 122 and 130 us (5.5 and 5.2 TB/s).
#include "ckpt8.cuh"
#include "dwbnq_internal.h"

namespace dwbnq {

namespace {

constexpr int kThreads = 256, kStoreUnroll = 2, kLoadUnroll = 4;  // octets a thread has in flight

template <typename T, bool VECTORS>
__global__ void __launch_bounds__(kThreads)
    ckpt8_store_kernel(const T *__restrict__ x, long long ld, long long rows, long long cols, const OctetGrid g,
                       signed char *__restrict__ codes, unsigned char *__restrict__ exps) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  float *stage = OctetStage<VECTORS>::get();
  OctetWalk w = octet_walk(g, rows);
  while (__any_sync(0xffffffffu, w.row < rows)) {
    float v[kStoreUnroll][8];
    long long at[kStoreUnroll];
    bool in[kStoreUnroll];
#pragma unroll
    for (int u = 0; u < kStoreUnroll; ++u) {
      in[u] = w.row < rows;
      at[u] = w.row * w.per_row + w.col;
      Octet<T, VECTORS>::load(x + w.row * ld + w.col * 8LL, in[u] ? cols - w.col * 8LL : 0, stage, v[u]);
      octet_next(w);
    }
#pragma unroll
    for (int u = 0; u < kStoreUnroll; ++u) ck_put(v[u], in[u], at[u], codes, exps);
  }
}

template <typename T, bool VECTORS>
__global__ void __launch_bounds__(kThreads)
    ckpt8_load_kernel(const signed char *__restrict__ codes, const unsigned char *__restrict__ exps, long long rows,
                      long long cols, const OctetGrid g, T *__restrict__ y, long long ld) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  float *stage = OctetStage<VECTORS>::get();
  OctetWalk w = octet_walk(g, rows);
  while (__any_sync(0xffffffffu, w.row < rows)) {
    float v[kLoadUnroll][8];
    T *to[kLoadUnroll];
    long long n[kLoadUnroll];
#pragma unroll
    for (int u = 0; u < kLoadUnroll; ++u) {
      const bool in = w.row < rows;
      ck_get(codes, exps, in, w.row * w.per_row + w.col, v[u]);
      to[u] = y + w.row * ld + w.col * 8LL;
      n[u] = in ? cols - w.col * 8LL : 0;
      octet_next(w);
    }
#pragma unroll
    for (int u = 0; u < kLoadUnroll; ++u) Octet<T, VECTORS>::store(to[u], n[u], stage, v[u]);
  }
}

template <typename T, bool VECTORS>
int store_t(long long rows, long long cols, long long ld, const void *x, void *codes, void *exps, cudaStream_t stream) {
  const OctetGrid g = octet_grid(rows, cols, kThreads, sm_count(-1) * 8);
  const cudaError_t e = launch_pdl(ckpt8_store_kernel<T, VECTORS>, dim3(g.ctas), dim3(kThreads), 0, stream, static_cast<const T *>(x), ld,
                                   rows, cols, g, static_cast<signed char *>(codes), static_cast<unsigned char *>(exps));
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "ckpt8_store_kernel launch");
}

template <typename T, bool VECTORS>
int load_t(long long rows, long long cols, const void *codes, const void *exps, long long ld, void *y, cudaStream_t stream) {
  const OctetGrid g = octet_grid(rows, cols, kThreads, sm_count(-1) * 8);
  const cudaError_t e = launch_pdl(ckpt8_load_kernel<T, VECTORS>, dim3(g.ctas), dim3(kThreads), 0, stream,
                                   static_cast<const signed char *>(codes), static_cast<const unsigned char *>(exps), rows, cols, g,
                                   static_cast<T *>(y), ld);
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "ckpt8_load_kernel launch");
}

template <typename T>
int store_a(long long rows, long long cols, long long ld, const void *x, void *codes, void *exps, cudaStream_t stream) {
  return octet_vectors(x, ld, sizeof(T)) ? store_t<T, true>(rows, cols, ld, x, codes, exps, stream)
                                         : store_t<T, false>(rows, cols, ld, x, codes, exps, stream);
}
template <typename T>
int load_a(long long rows, long long cols, const void *codes, const void *exps, long long ld, void *y, cudaStream_t stream) {
  return octet_vectors(y, ld, sizeof(T)) ? load_t<T, true>(rows, cols, codes, exps, ld, y, stream)
                                         : load_t<T, false>(rows, cols, codes, exps, ld, y, stream);
}

}  // namespace

int launch_ckpt8_store(int dtype, long long rows, long long cols, long long ld, const void *x, void *codes, void *exps,
                       cudaStream_t stream) {
  if (dtype == DWBNQ_F32) return store_a<float>(rows, cols, ld, x, codes, exps, stream);
  if (dtype == DWBNQ_F16) return store_a<__half>(rows, cols, ld, x, codes, exps, stream);
  return store_a<__nv_bfloat16>(rows, cols, ld, x, codes, exps, stream);
}

int launch_ckpt8_load(int dtype, long long rows, long long cols, const void *codes, const void *exps, long long ld, void *y,
                      cudaStream_t stream) {
  if (dtype == DWBNQ_F32) return load_a<float>(rows, cols, codes, exps, ld, y, stream);
  if (dtype == DWBNQ_F16) return load_a<__half>(rows, cols, codes, exps, ld, y, stream);
  return load_a<__nv_bfloat16>(rows, cols, codes, exps, ld, y, stream);
}

}  // namespace dwbnq
