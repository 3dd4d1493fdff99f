// 8-bit activation checkpoints: the storage format and its device-side conversions, shared by the
// kernels that write and read it (ckpt8.cu, glu.cu, affine_bwd.cu).
//
// A row of `cols` values is cut into groups of 32 consecutive ones. Per group one byte
//   b = max(7, biased fp32 exponent of the largest magnitude),
// fixes the step delta = 2^(b - 133), and every value is kept as the int8 code
//   k = clamp(round_half_even(x / delta), -127, 127);  it stands for k * delta.
// The largest magnitude lies in [64, 128) steps, so |x - k*delta| <= delta / 2, except in the last
// half step of the range (above 127.5 steps), where the clamp makes it less than one delta. The
// step is a power of two on purpose: the scaling, the rounding and k * delta (seven significant
// bits, never below the normal range) are exact in fp32 and in bfloat16, so a checkpoint has one
// right value, bit for bit, and the weight gradient can feed it to the tensor cores unrounded.
// A group with a value that is not finite has b = 255 and codes 0, and stands for NaN throughout.
// Memory: codes [rows, 32 * groups], groups = ceil(cols / 32), codes past `cols` are 0, so every row
// of codes starts on a 32-byte boundary whatever `cols`; exponents [rows, groups].
#pragma once

#include <cuda_bf16.h>

#include "dwbnq_device.cuh"

namespace dwbnq {

template <> struct Elem<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
};

constexpr int kCkGroup = 32;
constexpr unsigned int kCkMinExp = 7;    // delta and 1 / delta stay normal fp32 numbers
constexpr unsigned int kCkNonFinite = 255;

// Exponent byte from the largest magnitude's bit pattern (NaN and infinity have the exponent 255).
__device__ __forceinline__ unsigned int ck_exponent(unsigned int abs_bits) {
  const unsigned int b = abs_bits >> 23;
  return b < kCkMinExp ? kCkMinExp : b;
}
// 1 / delta; 0 for a group that is not finite (then every code comes out as 0).
__device__ __forceinline__ float ck_inv_step(unsigned int b) {
  return b == kCkNonFinite ? 0.0f : __uint_as_float((260u - b) << 23);
}
// delta; NaN for a group that is not finite.
__device__ __forceinline__ float ck_step(unsigned int b) {
  return b == kCkNonFinite ? __uint_as_float(0x7fc00000u) : __uint_as_float((b - 6u) << 23);
}
// ---- eight consecutive values of a row: what a lane works on; four lanes share a group -----------------------

// Rows that all start on a 16-byte boundary are accessed in 16-byte vectors. Others value by value, but so that the lanes of a warp
// touch consecutive values: the warp's 256 values change places through 1 KB of shared memory of its own (`stage`). Lane for lane
// every instruction would touch 32 lines, and L2 saw every sector eight times (float32 [4099, 5003] restored: 72 us).
// Every lane of the warp calls load and store, those past the end with n <= 0. A kernel is compiled for either way, as both in one
// cost the first one's registers (a quarter of its speed).
inline bool octet_vectors(const void *p, long long ld, int bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * bytes)) % 16) == 0;
}
// Two values of a 16-bit type in one word, to and from fp32.
__device__ __forceinline__ void unpack_pair(const __nv_bfloat16 *, unsigned int w, float &lo, float &hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack_pair(const __half *, unsigned int w, float &lo, float &hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
  lo = f.x;
  hi = f.y;
}
__device__ __forceinline__ unsigned int pack_pair(const __nv_bfloat16 *, float lo, float hi) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned int *>(&r);
}
__device__ __forceinline__ unsigned int pack_pair(const __half *, float lo, float hi) {
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned int *>(&r);
}

template <typename T, bool VECTORS> struct Octet {
  static constexpr int WORDS = 8 * (int)sizeof(T) / 4;
  // n: values that exist (the rest are 0); p is not followed for n <= 0
  static __device__ __forceinline__ void load(const T *p, long long n, float *stage, float *v) {
    if constexpr (VECTORS) {
      unsigned int w[WORDS];
      if (n >= 8) {
#pragma unroll
        for (int k = 0; k < WORDS / 4; ++k) {
          const uint4 q = __ldcs(reinterpret_cast<const uint4 *>(p) + k);
          w[4 * k] = q.x; w[4 * k + 1] = q.y; w[4 * k + 2] = q.z; w[4 * k + 3] = q.w;
        }
      } else {
        T e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = k < n ? p[k] : Elem<T>::from_f32(0.0f);
        memcpy(w, e, sizeof(w));
      }
#pragma unroll
      for (int k = 0; k < WORDS; ++k) {
        if constexpr (sizeof(T) == 4) v[k] = __uint_as_float(w[k]);
        else unpack_pair(p, w[k], v[2 * k], v[2 * k + 1]);
      }
    } else {
      const int lane = threadIdx.x & 31, have = n < 8 ? (int)n : 8;
      float t[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // value lane % 8 of lane 4 k + lane / 8
        const int from = 4 * k + (lane >> 3);
        const T *q = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), from));
        const int m = __shfl_sync(0xffffffffu, have, from);
        t[k] = (lane & 7) < m ? Elem<T>::to_f32(q[lane & 7]) : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) stage[32 * k + lane] = t[k];
      __syncwarp();
      const float4 lo = reinterpret_cast<const float4 *>(stage)[2 * lane], hi = reinterpret_cast<const float4 *>(stage)[2 * lane + 1];
      __syncwarp();
      v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    }
  }
  static __device__ __forceinline__ void store(T *p, long long n, float *stage, const float *v) {
    if constexpr (VECTORS) {
      unsigned int w[WORDS];
#pragma unroll
      for (int k = 0; k < WORDS; ++k) {
        if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v[k]);
        else w[k] = pack_pair(p, v[2 * k], v[2 * k + 1]);
      }
      if (n >= 8) {
#pragma unroll
        for (int k = 0; k < WORDS / 4; ++k)
          __stcs(reinterpret_cast<uint4 *>(p) + k, make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]));
      } else {
        T e[8];
        memcpy(e, w, sizeof(w));
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) p[k] = e[k];
      }
    } else {
      const int lane = threadIdx.x & 31, have = n < 8 ? (int)n : 8;
      reinterpret_cast<float4 *>(stage)[2 * lane] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4 *>(stage)[2 * lane + 1] = make_float4(v[4], v[5], v[6], v[7]);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int from = 4 * k + (lane >> 3);
        T *q = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), from));
        const int m = __shfl_sync(0xffffffffu, have, from);
        if ((lane & 7) < m) q[lane & 7] = Elem<T>::from_f32(stage[32 * k + lane]);
      }
      __syncwarp();
    }
  }
};

// A walk over all octets of [rows, 4 * groups]: thread t of the grid starts at octet t and goes on by the grid's size, with one
// division at the start. A warp's lanes stay together: whole groups, and so whole warps of shuffles, as the totals are multiples of 4
// and lanes past the end take part with `in` false.
struct OctetWalk {
  long long row, rows, row_step;
  unsigned int col, per_row, col_step;  // octets
};
struct OctetGrid {  // host: the grid and its step
  unsigned int ctas;
  long long row_step;
  unsigned int col_step, per_row;
};
inline OctetGrid octet_grid(long long rows, long long cols, int threads, int max_ctas) {
  OctetGrid g;
  g.per_row = (unsigned int)((cols + kCkGroup - 1) / kCkGroup * 4);
  const long long total = rows * g.per_row, need = (total + threads - 1) / threads;
  g.ctas = (unsigned int)(need < max_ctas ? need : max_ctas);
  const long long step = (long long)g.ctas * threads;
  g.row_step = step / g.per_row;
  g.col_step = (unsigned int)(step % g.per_row);
  return g;
}
__device__ __forceinline__ OctetWalk octet_walk(const OctetGrid &g, long long rows) {
  OctetWalk w;
  const long long first = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  w.row = first / g.per_row;
  w.col = (unsigned int)(first - w.row * g.per_row);
  w.rows = rows; w.row_step = g.row_step; w.per_row = g.per_row; w.col_step = g.col_step;
  return w;
}
__device__ __forceinline__ void octet_next(OctetWalk &w) {
  w.row += w.row_step;
  w.col += w.col_step;
  if (w.col >= w.per_row) { w.col -= w.per_row; ++w.row; }
}

template <bool VECTORS> struct OctetStage {  // the shared memory of a warp's exchange; none for vectors
  static __device__ __forceinline__ float *get() {
    if constexpr (VECTORS) return nullptr;
    __shared__ float4 stages[512];  // 256 threads
    return reinterpret_cast<float *>(stages) + (threadIdx.x >> 5) * 256;
  }
};

// Writes the checkpoint of a lane's eight values; the four lanes of a group work together (all lanes of the warp call it).
__device__ __forceinline__ void ck_put(const float *v, bool in, long long octet, signed char *codes, unsigned char *exps) {
  unsigned int m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const unsigned int b = ck_exponent(m);
  const float inv = ck_inv_step(b);
  // x / delta + 1.5 * 2^23 in one rounding is the integer, half to even, in the low half of the word; the clamp works on two
  // of them at once (the conversion instructions and fp32 clamps that this replaces ran at a quarter and half of the rate)
  unsigned int w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unsigned int t[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float lo = __fmaf_rn(v[4 * h + 2 * k], inv, 12582912.0f), hi = __fmaf_rn(v[4 * h + 2 * k + 1], inv, 12582912.0f);
      t[k] = __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
      asm("min.s16x2 %0, %0, %1;" : "+r"(t[k]) : "r"(0x007f007fu));
      asm("max.s16x2 %0, %0, %1;" : "+r"(t[k]) : "r"(0xff81ff81u));
    }
    w[h] = __byte_perm(t[0], t[1], 0x6420);
  }
  if (inv == 0.0f) w[0] = w[1] = 0u;
  if (in) {
    __stcs(reinterpret_cast<uint2 *>(codes) + octet, make_uint2(w[0], w[1]));
    if ((threadIdx.x & 3) == 0) exps[octet >> 2] = (unsigned char)b;
  }
}
// Reads them back (0 for lanes past the end).
__device__ __forceinline__ void ck_get(const signed char *codes, const unsigned char *exps, bool in, long long octet, float *v) {
  const uint2 c = in ? __ldcs(reinterpret_cast<const uint2 *>(codes) + octet) : make_uint2(0u, 0u);
  const float step = ck_step(in ? __ldg(exps + (octet >> 2)) : kCkMinExp);
  // the byte, offset to 0..255, under the exponent of 2^23: 2^23 + 128 + code, exactly (no conversion instruction)
  const unsigned int w[2] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    v[k] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(w[k >> 2], 0x4b000000u, 0x7440 + (k & 3))), 8388736.0f), step);
}

}  // namespace dwbnq
