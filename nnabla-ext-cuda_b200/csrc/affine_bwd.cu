// Weight and bias gradients of an affine layer whose input was kept as an 8-bit checkpoint:
//   dw[o][i] = sum_t dy[t][o] * x[t][i],   db[o] = sum_t dy[t][o],   x[t][i] = code * 2^(b - 133).
#include "ckpt8.cuh"
#include "dwbnq_internal.h"

namespace dwbnq {

namespace {

// 64 x 64 outputs per CTA, 4 x 4 per thread, 16 tokens per trip.
template <typename T, typename TW>
__global__ void __launch_bounds__(256)
    affine_dw_kernel(const signed char *__restrict__ codes, const unsigned char *__restrict__ exps, long long rows, int c_in,
                     int c_out, int groups, const T *__restrict__ dy, long long ld, TW *__restrict__ dw, int accum) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  __shared__ float xs[16][64 + 4], ds[16][64 + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, i0 = blockIdx.x * 64, o0 = blockIdx.y * 64;
  float acc[4][4] = {};
  for (long long t0 = 0; t0 < rows; t0 += 16) {
    for (int e = threadIdx.x; e < 16 * 64; e += 256) {
      const int t = e >> 6, j = e & 63;
      const bool in = t0 + t < rows;
      xs[t][j] = in && i0 + j < c_in ? __fmul_rn((float)codes[(t0 + t) * groups * kCkGroup + i0 + j],
                                                 ck_step(exps[(t0 + t) * groups + (i0 + j) / kCkGroup]))
                                     : 0.0f;
      ds[t][j] = in && o0 + j < c_out ? Elem<T>::to_f32(dy[(t0 + t) * ld + o0 + j]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 16; ++t)
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[p][q] = __fmaf_rn(ds[t][ty * 4 + p], xs[t][tx * 4 + q], acc[p][q]);
    __syncthreads();
  }
#pragma unroll
  for (int p = 0; p < 4; ++p)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int o = o0 + ty * 4 + p, i = i0 + tx * 4 + q;
      if (o >= c_out || i >= c_in) continue;
      TW *w = dw + (long long)o * c_in + i;
      *w = Elem<TW>::from_f32(accum ? __fadd_rn(Elem<TW>::to_f32(*w), acc[p][q]) : acc[p][q]);
    }
}

// 32 output channels per CTA, warp w sums the rows w, w + 8, ...; the eight sums are added in order.
template <typename T, typename TW>
__global__ void __launch_bounds__(256)
    affine_db_kernel(long long rows, int c_out, const T *__restrict__ dy, long long ld, TW *__restrict__ db, int accum) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, o = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (o < c_out)
    for (long long t = w; t < rows; t += 8) s = __fadd_rn(s, Elem<T>::to_f32(dy[t * ld + o]));
  part[w][lane] = s;
  __syncthreads();
  if (w || o >= c_out) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s = __fadd_rn(s, part[i][lane]);
  db[o] = Elem<TW>::from_f32(accum ? __fadd_rn(Elem<TW>::to_f32(db[o]), s) : s);
}

template <typename T, typename TW>
int run_t(const dwbnq_affine_desc &d, const void *codes, const void *exps, const void *dy, void *dw, void *db, int accum_mask,
          cudaStream_t stream) {
  const int groups = (d.c_in + kCkGroup - 1) / kCkGroup;
  cudaError_t e;
  if (dw) {
    const dim3 grid((unsigned)((d.c_in + 63) / 64), (unsigned)((d.c_out + 63) / 64));
    e = launch_pdl(affine_dw_kernel<T, TW>, grid, dim3(256), 0, stream, static_cast<const signed char *>(codes),
                   static_cast<const unsigned char *>(exps), (long long)d.rows, d.c_in, d.c_out, groups,
                   static_cast<const T *>(dy), (long long)d.ld_dy, static_cast<TW *>(dw), (accum_mask >> 1) & 1);
    if (e != cudaSuccess) return fail_cuda(e, "affine_dw_kernel launch");
  }
  if (db) {
    e = launch_pdl(affine_db_kernel<T, TW>, dim3((unsigned)((d.c_out + 31) / 32)), dim3(256), 0, stream, (long long)d.rows,
                   d.c_out, static_cast<const T *>(dy), (long long)d.ld_dy, static_cast<TW *>(db), (accum_mask >> 2) & 1);
    if (e != cudaSuccess) return fail_cuda(e, "affine_db_kernel launch");
  }
  return DWBNQ_OK;
}

}  // namespace

size_t affine_bwd_workspace_bytes(const dwbnq_affine_desc &) { return 256; }

int launch_affine_bwd(const dwbnq_affine_desc &d, const void *codes, const void *exps, const void *dy, void *dw, void *db,
                      int accum_mask, void *, int, cudaStream_t stream) {
  if (d.dtype == DWBNQ_F32) return run_t<float, float>(d, codes, exps, dy, dw, db, accum_mask, stream);
  if (d.dtype == DWBNQ_F16)
    return d.dw_dtype == DWBNQ_F32 ? run_t<__half, float>(d, codes, exps, dy, dw, db, accum_mask, stream)
                                   : run_t<__half, __half>(d, codes, exps, dy, dw, db, accum_mask, stream);
  return d.dw_dtype == DWBNQ_F32 ? run_t<__nv_bfloat16, float>(d, codes, exps, dy, dw, db, accum_mask, stream)
                                 : run_t<__nv_bfloat16, __nv_bfloat16>(d, codes, exps, dy, dw, db, accum_mask, stream);
}

}  // namespace dwbnq
