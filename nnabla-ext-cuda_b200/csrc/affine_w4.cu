// Affine layer with 4-bit weights in groups along the input channels, for one or a few rows:
//   y[r][o] = sum_g s[o][g] * sum_{i in g} x[r][i] * (q[o][i] - z[o][g]) + b[o].
//
// Packed weights: blocks of 16 output channels x 128 input channels, stored one after the other along the input channels, so that
// a warp streams consecutive memory and one bulk copy brings all it needs of a block: 1024 bytes of codes, then the scales
// [group of the block][16], then the zero points (one byte each) in the same order. Lane l of the warp that works on a block owns
// the output channels l/4 and l/4 + 8: its 16 bytes at 16 l and at 512 + 16 l are four words each, word j holding the eight codes
// of input channels 32 j + 8 (l mod 4) + e. Code e lies in nibble e/2 + 4 (e mod 2), so that (word >> 4 p) & 0x000f000f is the
// pair e = 2p, 2p + 1, the order in which consecutive activations lie in a register. Channels past the last have scale 0.
#include "ckpt8.cuh"
#include "dwbnq_internal.h"
#include "dwbnq_tc.cuh"

namespace dwbnq {

namespace {

constexpr int kPlanSms = 148;  // SMs of a B200
constexpr int kTileO = 16, kTileI = 128, kTileBytes = kTileO * kTileI / 2;

struct W4Layout {
  long long o_tiles, i_tiles;
  int block;  // bytes
};
W4Layout w4_layout(const dwbnq_w4_desc &d) {
  W4Layout l;
  l.o_tiles = (d.c_out + kTileO - 1) / kTileO;
  l.i_tiles = (d.c_in + kTileI - 1) / kTileI;
  l.block = kTileBytes + kTileI / d.group * kTileO * ((d.dtype == DWBNQ_F32 ? 4 : 2) + (d.has_zeros ? 1 : 0));
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

// One CTA per block: thread t writes word t, the first ones then a scale and a zero point.
template <typename T>
__global__ void __launch_bounds__(256)
    w4_pack_kernel(const unsigned char *__restrict__ codes, const T *__restrict__ scales, const unsigned char *__restrict__ zeros,
                   int c_out, int c_in, int group, int i_tiles, long long blocks, int block_bytes, unsigned char *__restrict__ packed) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const int half = threadIdx.x >> 7, lane = (threadIdx.x >> 2) & 31, j = threadIdx.x & 3;
  const int gb = kTileI / group, groups = (c_in + group - 1) / group;
  for (long long blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const long long ot = blk / i_tiles;
    const int it = (int)(blk - ot * i_tiles);
    unsigned char *out = packed + blk * block_bytes;
    const long long o = ot * kTileO + half * 8 + (lane >> 2);
    const int i = it * kTileI + 32 * j + 8 * (lane & 3);
    unsigned int v = 0;
    if (o < c_out)
      for (int e = 0; e < 8; ++e)
        if (i + e < c_in) v |= (codes[o * c_in + i + e] & 15u) << (4 * ((e >> 1) + 4 * (e & 1)));
    reinterpret_cast<unsigned int *>(out)[threadIdx.x] = v;
    if (threadIdx.x < gb * kTileO) {
      const int g = it * gb + threadIdx.x / kTileO;
      const long long os = ot * kTileO + threadIdx.x % kTileO;
      const bool in = os < c_out && g < groups;
      reinterpret_cast<T *>(out + kTileBytes)[threadIdx.x] = in ? scales[os * groups + g] : Elem<T>::from_f32(0.0f);
      if (zeros) (out + kTileBytes + gb * kTileO * sizeof(T))[threadIdx.x] = in ? (unsigned char)(zeros[os * groups + g] & 15) : (unsigned char)8;
    }
  }
}

// ---- the layer -----------------------------------------------------------------------------------------
//
// The weights are the A operand of mma.m16n8k16, the rows of x its B operand (eight per instruction, the missing ones zero):
// one row of x costs what eight cost, and for a handful the kernel is bound by reading the weights, 4 bits each. tcgen05 would want
// 128 output channels per tile and the weights in shared or tensor memory; here they go from global memory to the
// instruction through registers only. A lane's word of eight codes is the A operand of two instructions: (word >> 4 p) &
// 0x000f000f put under the exponent of 128 (bfloat16) or 1024 (float16) is a pair q + 128 or q + 1024, and one packed
// subtraction leaves q - z, exactly. float32 rows are the exact sum of three bfloat16 parts, one instruction each. The products
// of a group are summed by the tensor core (at most eight steps of 16, the small parts first), then scaled and added in fp32.

template <typename T> struct W4Math {  // bfloat16, and float32 in parts
  static constexpr unsigned int MAGIC = 0x43004300u;
  static __device__ __forceinline__ unsigned int zero_pair(unsigned int z) { return (0x4300u + z) * 0x10001u; }
  static __device__ __forceinline__ unsigned int sub(unsigned int a, unsigned int b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const unsigned int *>(&r);
  }
  static __device__ __forceinline__ void mma(float *c, const unsigned int *a, unsigned int b0, unsigned int b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct W4Math<__half> {
  static constexpr unsigned int MAGIC = 0x64006400u;
  static __device__ __forceinline__ unsigned int zero_pair(unsigned int z) { return (0x6400u + z) * 0x10001u; }
  static __device__ __forceinline__ unsigned int sub(unsigned int a, unsigned int b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const unsigned int *>(&r);
  }
  static __device__ __forceinline__ void mma(float *c, const unsigned int *a, unsigned int b0, unsigned int b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Eight consecutive elements of a row of x as the B operands of two instructions, part by part (float32: three bfloat16 parts).
template <typename T> struct XFrag {
  static constexpr int PARTS = 1;
  unsigned int w[1][4];
  __device__ __forceinline__ void set(const T *e) { memcpy(w[0], e, 16); }
  __device__ __forceinline__ void load_vec(const T *p) {
    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
    w[0][0] = v.x; w[0][1] = v.y; w[0][2] = v.z; w[0][3] = v.w;
  }
};
template <> struct XFrag<float> {
  static constexpr int PARTS = 3;
  unsigned int w[3][4];
  // heads by truncation, exact rests; an infinity has no rest (a NaN keeps one)
  __device__ __forceinline__ void set(const float *e) {
    float v[8];
    unsigned int top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = e[j];
      top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[q][j] = __byte_perm(__float_as_uint(v[2 * j]), __float_as_uint(v[2 * j + 1]), 0x7632);
      if (q < 2)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fsub_rn(v[j], __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u));
    }
    if (top >= 0x7f800000u) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned int half = j & 1 ? 0xffff0000u : 0xffffu;
        if ((__float_as_uint(e[j]) & 0x7fffffffu) == 0x7f800000u) { w[1][j / 2] &= ~half; w[2][j / 2] &= ~half; }
      }
    }
  }
  __device__ __forceinline__ void load_vec(const float *p) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    const float e[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    set(e);
  }
};

struct W4Args {
  const void *x, *b;
  void *y;
  const unsigned char *packed;
  long long ld_x, ld_y;
  int rows, c_in, c_out, i_tiles, o_tiles;
  int block;      // bytes of a packed block
  int has_zeros;
  int sums_at;    // where the sums lie in shared memory
  int wk;         // warps along the input channels
  int vec;        // rows of x are 16-byte aligned
  int *flag;
};

constexpr int kRing = 4;  // blocks (times R) in flight per warp

__device__ __forceinline__ void w4_copy(void *dst, const void *src, unsigned int bytes, unsigned long long *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// CTA: wo x wk warps; a warp has R tiles of 16 output channels and every wk-th tile of 128 input channels (of this CTA's share,
// where a cluster of CTAs divides them); blockIdx.y: block of 8 NB rows of x. G: group size. Rows of x that do not exist are
// read as row 0: their results are columns nobody stores.
template <typename T, int G, int NB, int R>
__global__ void __launch_bounds__(256) w4_affine_kernel(const W4Args a) {
  using M = W4Math<T>;
  constexpr int PARTS = XFrag<T>::PARTS, GB = kTileI / G;  // groups per block
  constexpr int PER_WARP = R * NB * 4 * 32;
  extern __shared__ __align__(128) unsigned char w4_smem[];
  __shared__ unsigned long long bars[8 * kRing];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, wo = warp / a.wk, wk = warp - wo * a.wk;
  const int lr = lane >> 2, lc = lane & 3;
  unsigned int crank, csize;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
  const int wos = warps / a.wk, ot0 = ((int)(blockIdx.x / csize) * wos + wo) * R;
  const int row0 = blockIdx.y * 8 * NB;
  const int stride = a.wk * (int)csize, first = wk + a.wk * (int)crank;
  // each warp fills and empties a ring of its own: no other warp is waited for before the sums
  unsigned char *ring = w4_smem + (size_t)warp * kRing * R * a.block;
  unsigned long long *bar = bars + warp * kRing;
  const int tiles = min(R, a.o_tiles - ot0);  // may be negative
  const unsigned char *src = a.packed + ((long long)ot0 * a.i_tiles + first) * a.block;
  if (lane == 0) {
    for (int k = 0; k < kRing; ++k) mbar_init(&bar[k], 1);
    mbar_fence_init();
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  auto fetch = [&](int it, int slot) {  // lane 0
    mbar_expect_tx(&bar[slot], (unsigned)(tiles * a.block));
    for (int r = 0; r < tiles; ++r)
      w4_copy(ring + (size_t)(slot * R + r) * a.block, src + ((long long)r * a.i_tiles + (it - first)) * a.block, (unsigned)a.block, &bar[slot]);
  };
  if (lane == 0 && tiles > 0)
    for (int k = 0; k < kRing && first + k * stride < a.i_tiles; ++k) fetch(first + k * stride, k);
  const T *xr[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = row0 + n * 8 + lr;
    xr[n] = static_cast<const T *>(a.x) + (long long)(row < a.rows ? row : 0) * a.ld_x + lc * 8;
  }
  float acc[R][NB][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[r][n][k] = 0.0f;
  int slot = 0;
  unsigned int ph = 0;
  bool ok = true;
  for (int it = first; tiles > 0 && it < a.i_tiles; it += stride) {
    const int i0 = it * kTileI;
    XFrag<T> x[4][NB];
    if (a.vec && i0 + kTileI <= a.c_in) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int n = 0; n < NB; ++n) x[j][n].load_vec(xr[n] + i0 + j * 32);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          T e[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) e[k] = i0 + j * 32 + lc * 8 + k < a.c_in ? __ldg(xr[n] + i0 + j * 32 + k) : Elem<T>::from_f32(0.0f);
          x[j][n].set(e);
        }
    }
    ok = pw_wait(&bar[slot], ph);
    if (!ok) break;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned char *blk = ring + (size_t)(slot * R + r) * a.block;  // a tile that does not exist is never copied: stale, and not stored
      const uint4 lo4 = reinterpret_cast<const uint4 *>(blk)[lane], hi4 = reinterpret_cast<const uint4 *>(blk)[32 + lane];
      float part[NB][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        constexpr int PER = G / 32;  // words per group
        const int g = j / PER;
        unsigned int z0 = 8, z1 = 8;
        if (a.has_zeros) {
          const unsigned char *z = blk + kTileBytes + GB * kTileO * sizeof(T) + g * kTileO + lr;
          z0 = z[0];
          z1 = z[8];
        }
        z0 = M::zero_pair(z0);
        z1 = M::zero_pair(z1);
        if (j % PER == 0)
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) part[n][k] = 0.0f;
        const unsigned int lo = j == 0 ? lo4.x : j == 1 ? lo4.y : j == 2 ? lo4.z : lo4.w;
        const unsigned int hi = j == 0 ? hi4.x : j == 1 ? hi4.y : j == 2 ? hi4.z : hi4.w;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          unsigned int f[4];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int sh = 4 * (2 * m + k);
            f[2 * k] = M::sub(((lo >> sh) & 0x000f000fu) | M::MAGIC, z0);
            f[2 * k + 1] = M::sub(((hi >> sh) & 0x000f000fu) | M::MAGIC, z1);
          }
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int q = PARTS - 1; q >= 0; --q) M::mma(part[n], f, x[j][n].w[q][2 * m], x[j][n].w[q][2 * m + 1]);
        }
        if (j % PER == PER - 1) {
          const T *sc = reinterpret_cast<const T *>(blk + kTileBytes) + g * kTileO + lr;
          const float s0 = Elem<T>::to_f32(sc[0]), s1 = Elem<T>::to_f32(sc[8]);
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[r][n][k] = __fmaf_rn(part[n][k], k < 2 ? s0 : s1, acc[r][n][k]);
        }
      }
    }
    __syncwarp();  // every lane has read the slot
    if (lane == 0 && it + kRing * stride < a.i_tiles) fetch(it + kRing * stride, slot);
    if (++slot == kRing) { slot = 0; ph ^= 1u; }
  }
  if (!ok) {  // a copy did not land in time: recorded; the others in flight are given the same time before the ring goes away
    if (lane == 0) atomicExch(a.flag, 1);
    for (int k = 1; k < kRing; ++k) pw_wait(&bar[(slot + k) % kRing], slot + k < kRing ? ph : ph ^ 1u);
  }
  __syncthreads();  // the rings have served; their memory takes the sums
  float *red = reinterpret_cast<float *>(w4_smem);  // [warp][R][NB][4][32]
  // the warps' sums (and then the CTAs') in a fixed order
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) red[warp * PER_WARP + ((r * NB + n) * 4 + k) * 32 + lane] = acc[r][n][k];
  __syncthreads();
  const int outs = wos * PER_WARP;
  float *sums = reinterpret_cast<float *>(w4_smem + a.sums_at);  // cluster: [CTA][outs], in the first CTA
  for (int e = threadIdx.x; e < outs; e += blockDim.x) {
    const int o_w = e / PER_WARP, in = e - o_w * PER_WARP;
    float v = 0.0f;
    for (int k = 0; k < a.wk; ++k) v = __fadd_rn(v, red[(o_w * a.wk + k) * PER_WARP + in]);
    if (csize > 1) {  // the first CTA's `sums` lies behind its own rings and sums, which it may still be using
      unsigned int to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"((unsigned)__cvta_generic_to_shared(sums + crank * outs + e)));
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
    } else {
      sums[e] = v;
    }
  }
  if (csize > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (crank) return;
  } else {
    __syncthreads();
  }
  for (int e = threadIdx.x; e < outs; e += blockDim.x) {
    float v = sums[e];
    for (unsigned int k = 1; k < csize; ++k) v = __fadd_rn(v, sums[k * outs + e]);
    const int l = e & 31, k = (e >> 5) & 3, n = (e >> 7) % NB, r = (e >> 7) / NB % R, o_w = e / PER_WARP;
    const int o = (((int)(blockIdx.x / csize) * wos + o_w) * R + r) * kTileO + (k >> 1) * 8 + (l >> 2), row = row0 + n * 8 + (l & 3) * 2 + (k & 1);
    if (o < a.c_out && row < a.rows) {
      if (a.b) v = __fadd_rn(v, Elem<T>::to_f32(__ldg(static_cast<const T *>(a.b) + o)));
      static_cast<T *>(a.y)[(long long)row * a.ld_y + o] = Elem<T>::from_f32(v);
    }
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
  const long long blocks = l.o_tiles * l.i_tiles;
  const cudaError_t e = launch_pdl(w4_pack_kernel<T>, dim3(grid_for(blocks, 1)), dim3(256), 0, stream,
                                   static_cast<const unsigned char *>(codes), static_cast<const T *>(scales),
                                   static_cast<const unsigned char *>(zeros), d.c_out, d.c_in, d.group, (int)l.i_tiles, blocks, l.block,
                                   static_cast<unsigned char *>(packed));
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "w4_pack_kernel launch");
}
template <typename T, int G, int NB, int R>
int affine_launch(W4Args a, int wo, int wk, int cluster, cudaStream_t stream) {
  a.wk = wk;
  const int per_warp = R * NB * 4 * 32, o_ctas = (a.o_tiles + wo * R - 1) / (wo * R);
  const size_t rings = (size_t)wo * wk * kRing * R * a.block, own = sizeof(float) * (size_t)per_warp * wo * wk;
  a.sums_at = (int)((rings > own ? rings : own) + 15) / 16 * 16;
  const size_t smem = a.sums_at + sizeof(float) * (size_t)per_warp * cluster * wo;
  auto kern = w4_affine_kernel<T, G, NB, R>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return fail_cuda(e, "w4_affine_kernel attributes");
  }
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(o_ctas * cluster), (unsigned)((a.rows + 8 * NB - 1) / (8 * NB)));
  lc.blockDim = dim3((unsigned)(32 * wo * wk));
  lc.dynamicSmemBytes = smem;
  lc.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&lc, kern, a);
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "w4_affine_kernel launch");
}
template <typename T, int G>
int affine_g(const W4Args &a, cudaStream_t stream) {
  const int nb = a.rows > 8 ? 2 : 1;
  int wo = 1, wk = 8, cluster = 1;
  if (nb == 2) { wo = 2; wk = 4; }
  while (wk > 1 && wk > a.i_tiles) wk >>= 1;
  const int R = nb == 2 ? 2 : 1;
  const int o_ctas = (a.o_tiles + wo * R - 1) / (wo * R);
  while (cluster < 8 && o_ctas * cluster * 2 <= kPlanSms && a.i_tiles >= 2 * cluster * wk) cluster *= 2;
  return nb == 2 ? affine_launch<T, G, 2, 2>(a, wo, wk, cluster, stream) : affine_launch<T, G, 1, 1>(a, wo, wk, cluster, stream);
}
template <typename T>
int affine_t(const dwbnq_w4_desc &d, long long rows, long long ld_x, const void *x, const void *packed, const void *b,
             long long ld_y, void *y, int dev, cudaStream_t stream) {
  const W4Layout l = w4_layout(d);
  W4Args a = {};
  const int st = device_flag_ptr(dev, &a.flag);
  if (st != DWBNQ_OK) return st;
  a.x = x; a.b = b; a.y = y;
  a.packed = static_cast<const unsigned char *>(packed);
  a.block = l.block; a.has_zeros = d.has_zeros;
  a.ld_x = ld_x; a.ld_y = ld_y;
  a.rows = (int)rows; a.c_in = d.c_in; a.c_out = d.c_out; a.i_tiles = (int)l.i_tiles; a.o_tiles = (int)l.o_tiles;
  a.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_x * sizeof(T) % 16 == 0;
  return d.group == 32 ? affine_g<T, 32>(a, stream) : d.group == 64 ? affine_g<T, 64>(a, stream) : affine_g<T, 128>(a, stream);
}

}  // namespace

size_t w4_packed_bytes(const dwbnq_w4_desc &d) {
  const W4Layout l = w4_layout(d);
  return ((size_t)(l.o_tiles * l.i_tiles) * l.block + 255) / 256 * 256;
}

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
                     long long ld_y, void *y, int dev, cudaStream_t stream) {
  if (d.dtype == DWBNQ_F32) return affine_t<float>(d, rows, ld_x, x, packed, b, ld_y, y, dev, stream);
  if (d.dtype == DWBNQ_F16) return affine_t<__half>(d, rows, ld_x, x, packed, b, ld_y, y, dev, stream);
  return affine_t<__nv_bfloat16>(d, rows, ld_x, x, packed, b, ld_y, y, dev, stream);
}

}  // namespace dwbnq
