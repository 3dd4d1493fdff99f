// Affine layer with 4-bit weights in groups along the input channels, for one or a few rows:
//   y[r][o] = sum_g s[o][g] * sum_{i in g} x[r][i] * (q[o][i] - z[o][g]) + b[o].
//
// Packed weights: tiles of 16 output channels x 128 input channels, 1024 bytes each, stored one after
// the other along the input channels, so that a warp streams consecutive memory. Lane l of the warp
// that works on a tile owns the output channels l/4 and l/4 + 8: its 16 bytes at 16 l and at 512 +
// 16 l are four words each, word j holding the eight codes of input channels 32 j + 8 (l mod 4) + e.
// Code e lies in nibble e/2 + 4 (e mod 2), so that (word >> 4 p) & 0x000f000f is the pair e = 2p,
// 2p + 1, the order in which consecutive activations lie in a register. The scales follow, [tile of
// 16 output channels][group][16], then the zero points, one byte each in the same order. Channels
// past the last have scale 0.
#include "ckpt8.cuh"
#include "dwbnq_internal.h"

namespace dwbnq {

namespace {

constexpr int kTileO = 16, kTileI = 128, kTileBytes = kTileO * kTileI / 2;

struct W4Layout {
  long long o_tiles, i_tiles, groups;  // groups: of the padded row
  size_t scales, zeros, bytes;         // offsets of the two tables, and the total
};
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
W4Layout w4_layout(const dwbnq_w4_desc &d) {
  W4Layout l;
  l.o_tiles = (d.c_out + kTileO - 1) / kTileO;
  l.i_tiles = (d.c_in + kTileI - 1) / kTileI;
  l.groups = l.i_tiles * (kTileI / d.group);
  l.scales = up256((size_t)l.o_tiles * l.i_tiles * kTileBytes);
  l.zeros = l.scales + up256((size_t)l.o_tiles * l.groups * kTileO * (d.dtype == DWBNQ_F32 ? 4 : 2));
  l.bytes = l.zeros + (d.has_zeros ? up256((size_t)l.o_tiles * l.groups * kTileO) : 0);
  return l;
}

// scale = (largest magnitude of the group) / 7 in the tensor's type, code = clamp(round_half_even(w / scale), -8, 7) + 8.
// One warp per group.
template <typename T>
__global__ void __launch_bounds__(256)
    w4_quantize_kernel(const T *__restrict__ w, long long ld, int c_out, int c_in, int group, int groups,
                       unsigned char *__restrict__ codes, T *__restrict__ scales) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const int lane = threadIdx.x & 31;
  const long long total = (long long)c_out * groups, step = (long long)gridDim.x * 8;
  for (long long g = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); g < total; g += step) {
    const long long o = g / groups;
    const int i0 = (int)(g - o * groups) * group, n = min(group, c_in - i0);
    unsigned int m = 0;
    for (int i = lane; i < n; i += 32) m = max(m, __float_as_uint(Elem<T>::to_f32(w[o * ld + i0 + i])) & 0x7fffffffu);
    const T st = Elem<T>::from_f32(__fdiv_rn(__uint_as_float(__reduce_max_sync(0xffffffffu, m)), 7.0f));
    const float s = Elem<T>::to_f32(st);
    for (int i = lane; i < n; i += 32) {
      const float t = __fdiv_rn(Elem<T>::to_f32(w[o * ld + i0 + i]), s);
      // a zero scale (all zeros, or all below half the type's smallest number) and NaN give the code of zero
      codes[o * c_in + i0 + i] = (unsigned char)((s > 0.0f && t == t ? __float2int_rn(fminf(fmaxf(t, -8.0f), 7.0f)) : 0) + 8);
    }
    if (lane == 0) scales[g] = st;
  }
}

// One thread per packed word.
__global__ void __launch_bounds__(256)
    w4_pack_codes_kernel(const unsigned char *__restrict__ codes, int c_out, int c_in, long long i_tiles, long long words,
                         unsigned int *__restrict__ packed) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long w = (long long)blockIdx.x * blockDim.x + threadIdx.x; w < words; w += step) {
    const int in = (int)(w & 255), half = in >> 7, lane = (in >> 2) & 31, j = in & 3;
    const long long tile = w >> 8, ot = tile / i_tiles, it = tile - ot * i_tiles;
    const long long o = ot * kTileO + half * 8 + (lane >> 2), i = it * kTileI + 32 * j + 8 * (lane & 3);
    unsigned int v = 0;
    if (o < c_out)
      for (int e = 0; e < 8; ++e)
        if (i + e < c_in) v |= (codes[o * c_in + i + e] & 15u) << (4 * ((e >> 1) + 4 * (e & 1)));
    packed[w] = v;
  }
}
template <typename T>
__global__ void __launch_bounds__(256)
    w4_pack_tables_kernel(const T *__restrict__ scales, const unsigned char *__restrict__ zeros, int c_out, int src_groups,
                          long long groups, long long total, T *__restrict__ out_s, unsigned char *__restrict__ out_z) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int ol = (int)(i % kTileO);
    const long long tg = i / kTileO, ot = tg / groups, g = tg - ot * groups, o = ot * kTileO + ol;
    const bool in = o < c_out && g < src_groups;
    out_s[i] = in ? scales[o * src_groups + g] : Elem<T>::from_f32(0.0f);
    if (out_z) out_z[i] = in ? (unsigned char)(zeros[o * src_groups + g] & 15) : (unsigned char)8;
  }
}

// One warp per (row, output channel).
template <typename T>
__global__ void __launch_bounds__(256)
    w4_affine_kernel(const T *__restrict__ x, long long ld_x, long long rows, const unsigned int *__restrict__ words,
                     const T *__restrict__ scales, const unsigned char *__restrict__ zeros, long long i_tiles,
                     long long groups, int group, int c_in, int c_out, const T *__restrict__ b, T *__restrict__ y,
                     long long ld_y) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const int lane = threadIdx.x & 31;
  const long long total = rows * c_out, step = (long long)gridDim.x * 8;
  for (long long n = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); n < total; n += step) {
    const long long r = n / c_out;
    const int o = (int)(n - r * c_out), ol = o % kTileO;
    float acc = 0.0f;
    for (int i = lane; i < c_in; i += 32) {
      const int in = i % kTileI, e = in & 7, l = (ol & 7) * 4 + ((in >> 3) & 3);
      const unsigned int w = words[((long long)(o / kTileO) * i_tiles + i / kTileI) * 256 + (ol >> 3) * 128 + l * 4 + (in >> 5)];
      const long long t = ((long long)(o / kTileO) * groups + i / group) * kTileO + ol;
      const float q = (float)((int)((w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) - (zeros ? (int)zeros[t] : 8));
      acc = __fmaf_rn(Elem<T>::to_f32(x[r * ld_x + i]), __fmul_rn(q, Elem<T>::to_f32(scales[t])), acc);
    }
    for (int s = 16; s; s >>= 1) acc = __fadd_rn(acc, __shfl_xor_sync(0xffffffffu, acc, s));
    if (lane == 0) y[r * ld_y + o] = Elem<T>::from_f32(b ? __fadd_rn(acc, Elem<T>::to_f32(b[o])) : acc);
  }
}

unsigned int grid_for(long long items, int per_cta) {
  const long long blocks = (items + per_cta - 1) / per_cta, cap = (long long)sm_count(-1) * 16;
  return (unsigned int)(blocks > cap ? cap : blocks < 1 ? 1 : blocks);
}

template <typename T>
int quantize_t(int c_out, int c_in, int group, long long ld, const void *w, void *codes, void *scales, cudaStream_t stream) {
  const int groups = (c_in + group - 1) / group;
  const cudaError_t e = launch_pdl(w4_quantize_kernel<T>, dim3(grid_for((long long)c_out * groups, 8)), dim3(256), 0, stream,
                                   static_cast<const T *>(w), ld, c_out, c_in, group, groups,
                                   static_cast<unsigned char *>(codes), static_cast<T *>(scales));
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "w4_quantize_kernel launch");
}
template <typename T>
int pack_t(const dwbnq_w4_desc &d, const void *codes, const void *scales, const void *zeros, void *packed, cudaStream_t stream) {
  const W4Layout l = w4_layout(d);
  unsigned char *p = static_cast<unsigned char *>(packed);
  const long long words = l.o_tiles * l.i_tiles * (kTileBytes / 4), total = l.o_tiles * l.groups * kTileO;
  cudaError_t e = launch_pdl(w4_pack_codes_kernel, dim3(grid_for(words, 256)), dim3(256), 0, stream,
                             static_cast<const unsigned char *>(codes), d.c_out, d.c_in, l.i_tiles, words,
                             reinterpret_cast<unsigned int *>(p));
  if (e != cudaSuccess) return fail_cuda(e, "w4_pack_codes_kernel launch");
  e = launch_pdl(w4_pack_tables_kernel<T>, dim3(grid_for(total, 256)), dim3(256), 0, stream, static_cast<const T *>(scales),
                 static_cast<const unsigned char *>(zeros), d.c_out, (d.c_in + d.group - 1) / d.group, l.groups, total,
                 reinterpret_cast<T *>(p + l.scales), d.has_zeros ? p + l.zeros : static_cast<unsigned char *>(nullptr));
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "w4_pack_tables_kernel launch");
}
template <typename T>
int affine_t(const dwbnq_w4_desc &d, long long rows, long long ld_x, const void *x, const void *packed, const void *b,
             long long ld_y, void *y, cudaStream_t stream) {
  const W4Layout l = w4_layout(d);
  const unsigned char *p = static_cast<const unsigned char *>(packed);
  const cudaError_t e = launch_pdl(w4_affine_kernel<T>, dim3(grid_for(rows * d.c_out, 8)), dim3(256), 0, stream,
                                   static_cast<const T *>(x), ld_x, rows, reinterpret_cast<const unsigned int *>(p),
                                   reinterpret_cast<const T *>(p + l.scales),
                                   d.has_zeros ? p + l.zeros : static_cast<const unsigned char *>(nullptr), l.i_tiles, l.groups,
                                   d.group, d.c_in, d.c_out, static_cast<const T *>(b), static_cast<T *>(y), ld_y);
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "w4_affine_kernel launch");
}

}  // namespace

size_t w4_packed_bytes(const dwbnq_w4_desc &d) { return w4_layout(d).bytes; }

int launch_w4_quantize(int dtype, int c_out, int c_in, int group, long long ld, const void *w, void *codes, void *scales,
                       cudaStream_t stream) {
  if (dtype == DWBNQ_F32) return quantize_t<float>(c_out, c_in, group, ld, w, codes, scales, stream);
  if (dtype == DWBNQ_F16) return quantize_t<__half>(c_out, c_in, group, ld, w, codes, scales, stream);
  return quantize_t<__nv_bfloat16>(c_out, c_in, group, ld, w, codes, scales, stream);
}
int launch_w4_pack(const dwbnq_w4_desc &d, const void *codes, const void *scales, const void *zeros, void *packed,
                   cudaStream_t stream) {
  if (d.dtype == DWBNQ_F32) return pack_t<float>(d, codes, scales, zeros, packed, stream);
  if (d.dtype == DWBNQ_F16) return pack_t<__half>(d, codes, scales, zeros, packed, stream);
  return pack_t<__nv_bfloat16>(d, codes, scales, zeros, packed, stream);
}
int launch_w4_affine(const dwbnq_w4_desc &d, long long rows, long long ld_x, const void *x, const void *packed, const void *b,
                     long long ld_y, void *y, cudaStream_t stream) {
  if (d.dtype == DWBNQ_F32) return affine_t<float>(d, rows, ld_x, x, packed, b, ld_y, y, stream);
  if (d.dtype == DWBNQ_F16) return affine_t<__half>(d, rows, ld_x, x, packed, b, ld_y, y, stream);
  return affine_t<__nv_bfloat16>(d, rows, ld_x, x, packed, b, ld_y, y, stream);
}

}  // namespace dwbnq
