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
constexpr int kSmemMax = 227 * 1024 - 1024;  // dynamic shared memory a CTA may ask for beside its static part
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
// 0x000f000f put under the exponent of 2^-4 (bfloat16) or 1024 (float16) is a pair (q + 128) / 2048 or q + 1024, and one packed
// subtraction leaves (q - z) / 2048 or q - z, exactly. float32 rows are the exact sum of three bfloat16 parts, one instruction each.
// The products of a group are summed by the tensor core (at most eight steps of 16, the small parts first), then scaled and added in
// fp32; the bfloat16 form's 2048 is multiplied in at the end. It keeps the sum of a group, at most 128 x 15 times the largest
// magnitude, in range whatever x: bfloat16 and float32 rows reach to the end of fp32's, and the scales bring the result back.
// (Giving the tensor core q + 128 and taking (128 + z) times the group's sum of x off afterwards carries 30 times the result's
// magnitude, and without bound more where an x of weight 0 is large, and turns infinities into NaN; it was 1.5% faster on one bf16
// row and 7% slower on 16.)

// What bounds it: nothing is saturated. For one bf16 row 4096 -> 14336 the 172 instructions per block of 2048 weights fill 4.4 of 11 us
// of issue slots, DRAM runs at a quarter of its rate and the tensor cores at a sixth: there are 16 warps per SM at most, each waits
// for its own copy, and the tiles of 16 x R channels do not come out even (224 CTAs here: half the SMs have one, half two). On the
// device: one bf16 row 4096 -> 14336 11.4 us (2.65 TB/s), 8192 -> 8192 11.9 us, 4096 -> 4096 5.1 us, 512 -> 512 2.1 us; one float16 row
// 4096 -> 14336 10.4 us, one float32 row 17.6 us; 16 rows: bf16 4096 -> 14336 17.4 us, fp16 8192 -> 8192 with zero points 16.6 us.

template <typename T> struct W4Math {  // bfloat16; float32 in bfloat16 parts
  static constexpr float UNIT = 2048.0f;  // what the sums are to be multiplied by
  static constexpr unsigned int MAGIC = 0x3d803d80u;  // 2^-4, twice: its last place is 1 / 2048
  static __device__ __forceinline__ unsigned int zero_pair(unsigned int z) { return (0x3d80u + z) * 0x10001u; }
  static __device__ __forceinline__ unsigned int sub(unsigned int a, unsigned int b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const unsigned int *>(&r);
  }
  // the pairs e = 0 1, 2 3, 4 5, 6 7 of a word, less the zero point
  static __device__ __forceinline__ void unpack(unsigned int w, unsigned int z, unsigned int magic, unsigned int &p0, unsigned int &p1,
                                                unsigned int &p2, unsigned int &p3) {
    p0 = sub(and_or(w, 0x000f000fu, magic), z);
    p1 = sub(and_or(w >> 4, 0x000f000fu, magic), z);
    p2 = sub(and_or(w >> 8, 0x000f000fu, magic), z);
    p3 = sub(and_or(w >> 12, 0x000f000fu, magic), z);
  }
  static __device__ __forceinline__ void mma(float *c, const unsigned int *a, unsigned int b0, unsigned int b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct W4Math<__half> {
  static constexpr float UNIT = 1.0f;
  static constexpr unsigned int MAGIC = 0x64006400u;
  static __device__ __forceinline__ unsigned int zero_pair(unsigned int z) { return (0x6400u + z) * 0x10001u; }
  static __device__ __forceinline__ unsigned int sub(unsigned int a, unsigned int b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const unsigned int *>(&r);
  }
  // as above; the ten bits of the mantissa also take a code four bits higher, 1024 + 16 q, so that one shift does:
  // (1024 + 16 q) / 16 - z' = q - z + 64 with z' = 1024 + z, less 960
  static __device__ __forceinline__ unsigned int high(unsigned int a, unsigned int z) {
    const unsigned int sixteenth = 0x2c002c00u, c960 = 0x63806380u;
    const __half2 off = __hsub2(*reinterpret_cast<const __half2 *>(&c960), *reinterpret_cast<const __half2 *>(&z));
    const __half2 q = __hfma2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&sixteenth), off);
    return *reinterpret_cast<const unsigned int *>(&q);
  }
  static __device__ __forceinline__ void unpack(unsigned int w, unsigned int z, unsigned int magic, unsigned int &p0, unsigned int &p1,
                                                unsigned int &p2, unsigned int &p3) {
    const unsigned int w8 = w >> 8;
    p0 = sub(and_or(w, 0x000f000fu, magic), z);
    p1 = high(and_or(w, 0x00f000f0u, magic), z);
    p2 = sub(and_or(w8, 0x000f000fu, magic), z);
    p3 = high(and_or(w8, 0x00f000f0u, magic), z);
  }
  static __device__ __forceinline__ void mma(float *c, const unsigned int *a, unsigned int b0, unsigned int b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Eight consecutive elements of a row of x: as they were loaded, and as the B operands of two instructions, part by part
// (float32: three bfloat16 parts, heads by truncation and exact rests; an infinity has no rest, a NaN keeps one).
template <typename T> struct XRaw {
  uint4 w[8 * (int)sizeof(T) / 16];
  __device__ __forceinline__ void load(const T *p, int n, bool vec) {  // n: elements that exist
    if (vec) {
#pragma unroll
      for (int k = 0; k < 8 * (int)sizeof(T) / 16; ++k) w[k] = __ldg(reinterpret_cast<const uint4 *>(p) + k);
    } else {
      T e[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = k < n ? __ldg(p + k) : Elem<T>::from_f32(0.0f);
      memcpy(w, e, sizeof(w));
    }
  }
};
template <typename T> struct XFrag {
  static constexpr int PARTS = 1;
  unsigned int w[1][4];
  __device__ __forceinline__ explicit XFrag(const XRaw<T> &r) { w[0][0] = r.w[0].x; w[0][1] = r.w[0].y; w[0][2] = r.w[0].z; w[0][3] = r.w[0].w; }
};
template <> struct XFrag<float> {
  static constexpr int PARTS = 3;
  unsigned int w[3][4];
  __device__ __forceinline__ explicit XFrag(const XRaw<float> &r) {
    const unsigned int e[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
    float v[8];
    unsigned int top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = __uint_as_float(e[j]);
      top = max(top, e[j] & 0x7fffffffu);
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
        if ((e[j] & 0x7fffffffu) == 0x7f800000u) { w[1][j / 2] &= ~half; w[2][j / 2] &= ~half; }
      }
    }
  }
};

struct W4Args {
  const void *x, *b;
  void *y;
  const unsigned char *packed;
  long long ld_x, ld_y;
  int rows, c_in, c_out, i_tiles, o_tiles;
  int block;      // bytes of a packed block
  int per_warp;   // blocks along the input channels per warp
  int ring;       // copies in flight per warp and tile
  int red_at, sums_at;  // where the sums lie in shared memory
  int vec;        // rows of x are 16-byte aligned
  int device;
  int *flag;
};

constexpr int kMaxRing = 2;  // copies in flight per warp: with 16 to 32 warps on an SM 64 to 130 KB, well above what latency x bandwidth asks for
__host__ __device__ constexpr int w4_step(int R) { return R <= 2 ? 2 : 1; }  // blocks per copy

__device__ __forceinline__ void w4_copy(void *dst, const void *src, unsigned int bytes, unsigned long long *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Sum e of a group's accumulators (layout [R][NB][4][32 lanes]) to its place in y.
template <typename T, int NB, int R>
__device__ __forceinline__ void store_out(const W4Args &a, int og, int row0, int e, float v) {
  const int l = e & 31, k = (e >> 5) & 3, n = (e >> 7) % NB, r = (e >> 7) / NB;
  const int o = (og * R + r) * kTileO + (k >> 1) * 8 + (l >> 2), row = row0 + n * 8 + (l & 3) * 2 + (k & 1);
  if (o < a.c_out && row < a.rows) {
    v = __fmul_rn(v, W4Math<T>::UNIT);
    if (a.b) v = __fadd_rn(v, Elem<T>::to_f32(__ldg(static_cast<const T *>(a.b) + o)));
    static_cast<T *>(a.y)[(long long)row * a.ld_y + o] = Elem<T>::from_f32(v);
  }
}

// A CTA takes R tiles of 16 output channels at a time (group blockIdx.x, then every n-th), its warps a run of per_warp tiles of
// 128 input channels each (of the CTA's share, where a cluster of CTAs divides them). The copies run on from one group to the
// next, so that memory is kept busy while the warps' sums are added. blockIdx.y: block of 8 NB rows of x. G: group size; ZEROS:
// zero points. Rows of x that do not exist are read as row 0: their results are columns nobody stores.
template <typename T, int G, int NB, int R, bool ZEROS>
__global__ void __launch_bounds__(256, 2) w4_affine_kernel(const W4Args a) {
  using M = W4Math<T>;
  constexpr int GB = kTileI / G;  // quantization groups per block
  constexpr int BLOCK = kTileBytes + GB * kTileO * ((int)sizeof(T) + (ZEROS ? 1 : 0));
  constexpr int PER_WARP = R * NB * 4 * 32, STEP = w4_step(R);
  extern __shared__ __align__(128) unsigned char w4_smem[];
  __shared__ unsigned long long bars[8 * kMaxRing];
  const int lane = threadIdx.x & 31, wk = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int lr = lane >> 2, lc = lane & 3;
  unsigned int crank, csize;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
  const int og0 = blockIdx.x / csize, og_step = gridDim.x / csize, ogs = (a.o_tiles + R - 1) / R;
  const int row0 = blockIdx.y * 8 * NB;
  const int it0 = ((int)crank * warps + wk) * a.per_warp, blocks = max(0, min(a.i_tiles - it0, a.per_warp));
  const int steps = (blocks + STEP - 1) / STEP;
  // each warp fills and empties a ring of its own: no other warp is waited for before the sums
  unsigned char *ring = w4_smem + wk * a.ring * (R * STEP * BLOCK);
  unsigned long long *bar = bars + wk * kMaxRing;
  if (lane == 0) {
    for (int k = 0; k < a.ring; ++k) mbar_init(&bar[k], 1);
    mbar_fence_init();
  }
  __syncwarp();
  // the first CTA's shared memory may only be written once it runs
  if (csize > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const long long tile_bytes = (long long)a.i_tiles * BLOCK;
  const unsigned char *src = a.packed + (long long)og0 * R * tile_bytes + (long long)it0 * BLOCK;  // of the next copy
  int og_f = og0, step_f = 0, slot_f = 0;
  auto fetch = [&]() {
    if (og_f >= ogs || steps == 0) return;
    if (elect_one()) {
      const int tiles = min(R, a.o_tiles - og_f * R);
      const unsigned int bytes = (unsigned)min(STEP, blocks - step_f * STEP) * BLOCK;
      unsigned char *dst = ring + slot_f * (R * STEP * BLOCK);
      mbar_expect_tx(&bar[slot_f], tiles * bytes);
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r < tiles) w4_copy(dst + r * (STEP * BLOCK), src + r * tile_bytes, bytes, &bar[slot_f]);
    }
    __syncwarp();
    src += STEP * BLOCK;
    if (++slot_f == a.ring) slot_f = 0;
    if (++step_f == steps) {
      step_f = 0;
      og_f += og_step;
      src += (long long)og_step * R * tile_bytes - (long long)steps * (STEP * BLOCK);
    }
  };
  for (int k = 0; k < a.ring; ++k) fetch();
  const T *x0[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = row0 + n * 8 + lr;
    x0[n] = static_cast<const T *>(a.x) + (long long)(row < a.rows ? row : 0) * a.ld_x + it0 * kTileI + lc * 8;
  }
  const unsigned int magic = opaque_constant(M::MAGIC);
  const int i_left0 = a.c_in - it0 * kTileI - lc * 8;  // input channels from this lane's first one on
  int slot = 0, buf = 0;
  unsigned int ph = 0;
  bool ok = true;
  float *red = reinterpret_cast<float *>(w4_smem + a.red_at);    // [2][warp][R][NB][4][32]
  float *sums = reinterpret_cast<float *>(w4_smem + a.sums_at);  // cluster: [2][CTA][PER_WARP], in the first CTA
  for (int og = og0; og < ogs; og += og_step) {
    float acc[R][NB][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[r][n][k] = 0.0f;
    const unsigned char *blk = ring;
    const T *xr[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) xr[n] = x0[n];
    int i_left = i_left0;
    for (int b = 0; ok && b < blocks; ++b) {
      // the rows of x are asked for before the block's copy is waited for
      XRaw<T> raw[4][NB];
      const bool vec = a.vec && i_left >= kTileI - 24;  // whole block
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int n = 0; n < NB; ++n) raw[j][n].load(xr[n] + j * 32, i_left - j * 32, vec);
#pragma unroll
      for (int n = 0; n < NB; ++n) xr[n] += kTileI;
      i_left -= kTileI;
      if (b % STEP == 0) {
        blk = ring + slot * (R * STEP * BLOCK);
        ok = pw_wait(&bar[slot], ph);
        if (!ok) break;
      }
      float part[R][NB][4];
      uint4 lo4[R], hi4[R];
      unsigned int z0[R], z1[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {  // a tile that does not exist is never copied: its slot is stale, its sums are not stored
        lo4[r] = reinterpret_cast<const uint4 *>(blk + r * (STEP * BLOCK))[lane];
        hi4[r] = reinterpret_cast<const uint4 *>(blk + r * (STEP * BLOCK))[32 + lane];
        z0[r] = z1[r] = M::zero_pair(8);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        constexpr int PER = G / 32;  // words per quantization group
        const int g = j / PER;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const XFrag<T> x(raw[j][n]);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const unsigned char *p = blk + r * (STEP * BLOCK);
            if (j % PER == 0) {
              if (ZEROS && n == 0) {
                const unsigned char *z = p + kTileBytes + GB * kTileO * sizeof(T) + g * kTileO + lr;
                z0[r] = M::zero_pair(z[0]);
                z1[r] = M::zero_pair(z[8]);
              }
#pragma unroll
              for (int k = 0; k < 4; ++k) part[r][n][k] = 0.0f;
            }
            const unsigned int lo = j == 0 ? lo4[r].x : j == 1 ? lo4[r].y : j == 2 ? lo4[r].z : lo4[r].w;
            const unsigned int hi = j == 0 ? hi4[r].x : j == 1 ? hi4[r].y : j == 2 ? hi4[r].z : hi4[r].w;
            unsigned int f[2][4];  // the same for every n: computed once
            M::unpack(lo, z0[r], magic, f[0][0], f[0][2], f[1][0], f[1][2]);
            M::unpack(hi, z1[r], magic, f[0][1], f[0][3], f[1][1], f[1][3]);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int q = XFrag<T>::PARTS - 1; q >= 0; --q) M::mma(part[r][n], f[m], x.w[q][2 * m], x.w[q][2 * m + 1]);
            if (j % PER == PER - 1) {
              const T *sc = reinterpret_cast<const T *>(p + kTileBytes) + g * kTileO + lr;
              const float s0 = Elem<T>::to_f32(sc[0]), s1 = Elem<T>::to_f32(sc[8]);
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[r][n][k] = __fmaf_rn(part[r][n][k], k < 2 ? s0 : s1, acc[r][n][k]);
            }
          }
        }
      }
      blk += BLOCK;
      if (b % STEP == STEP - 1 || b == blocks - 1) {
        __syncwarp();  // every lane has read the slot
        fetch();
        if (++slot == a.ring) { slot = 0; ph ^= 1u; }
      }
    }
    // the warps' sums (and then the CTAs') in a fixed order. One barrier per group and two buffers: whoever writes a buffer again
    // has passed the barrier that the readers of its last contents reached after reading
    float *mine = red + (buf * warps + wk) * PER_WARP;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) mine[((r * NB + n) * 4 + k) * 32 + lane] = acc[r][n][k];
    __syncthreads();
    for (int e = threadIdx.x; e < PER_WARP; e += blockDim.x) {
      const float *p = red + buf * warps * PER_WARP + e;
      float v = p[0];
      for (int k = 1; k < warps; ++k) v = __fadd_rn(v, p[k * PER_WARP]);
      if (csize > 1) {
        unsigned int to;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(sums + (buf * csize + crank) * PER_WARP + e)));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
      } else {
        store_out<T, NB, R>(a, og, row0, e, v);
      }
    }
    if (csize > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (crank == 0)
        for (int e = threadIdx.x; e < PER_WARP; e += blockDim.x) {
          const float *p = sums + buf * csize * PER_WARP + e;
          float v = p[0];
          for (unsigned int k = 1; k < csize; ++k) v = __fadd_rn(v, p[k * PER_WARP]);
          store_out<T, NB, R>(a, og, row0, e, v);
        }
    }
    buf ^= 1;
  }
  if (!ok) {  // a copy did not land in time: recorded; the others in flight are given the same time before the ring goes away
    if (lane == 0) atomicExch(a.flag, 1);
    for (int k = 1; k < a.ring; ++k) pw_wait(&bar[(slot + k) % a.ring], slot + k < a.ring ? ph : ph ^ 1u);
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
template <typename T, int G, int NB, int R, bool ZEROS>
int affine_launch(W4Args a, int warps, int cluster, int ctas, cudaStream_t stream) {
  a.per_warp = (a.i_tiles + warps * cluster - 1) / (warps * cluster);
  const int per_warp = R * NB * 4 * 32, ogs = (a.o_tiles + R - 1) / R;
  const int steps = (a.per_warp + w4_step(R) - 1) / w4_step(R), rounds = (ogs + ctas - 1) / ctas;
  a.ring = steps * rounds < kMaxRing ? steps * rounds : kMaxRing;
  a.red_at = (warps * a.ring * w4_step(R) * R * a.block + 15) / 16 * 16;
  a.sums_at = a.red_at + 2 * warps * per_warp * (int)sizeof(float);
  const size_t smem = a.sums_at + (cluster > 1 ? 2 * sizeof(float) * (size_t)per_warp * cluster : 0);
  auto kern = w4_affine_kernel<T, G, NB, R, ZEROS>;
  if (smem > (size_t)kSmemMax) return fail(DWBNQ_ERR_UNSUPPORTED, "w4: %zu bytes of shared memory", smem);
  if (smem > 40 * 1024) {  // above 48 KB with the static part
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = allow_smem(reinterpret_cast<const void *>(kern), kSmemMax, a.device, allowed);
    if (e != cudaSuccess) return fail_cuda(e, "w4_affine_kernel attributes");
  }
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)((ogs + rounds - 1) / rounds * cluster), (unsigned)((a.rows + 8 * NB - 1) / (8 * NB)));
  lc.blockDim = dim3((unsigned)(32 * warps));
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
// Output tiles per warp: a warp's rows of x, its waits and its loop cost the same for one tile and for four, but fewer warps are at
// work. With enough weights for every SM (27 blocks) a warp takes four tiles where that leaves a group for every SM, else two where
// that leaves one for every second SM (one bf16 row, us with 4 / 2 / 1 tiles: 4096 -> 14336 11.4 / 12.3 / 14.1, 8192 -> 8192 12.0 /
// 11.9 / 13.4, 4096 -> 4096 5.5 / 5.1 / 5.2, 14336 -> 4096 15.8 / 11.5 / 11.8; float32 4096 -> 14336 17.6 / 20.4 / 27.9); with fewer weights
// one (512 -> 512: 3.0 / 2.4 / 2.1). Rows 9 to 16 double the accumulators: two at most (4096 -> 14336, 16 bf16 rows: 23.2 / 17.4 / 21.6).
// Two CTAs fit an SM; while there are fewer, a cluster of CTAs divides the input channels of each group, and where there are more
// they walk over the groups in equal rounds. The plan does not look at what a type and group size need: float32 in groups of 32 with
// zero points has shared memory for one CTA where a warp takes four tiles, which then run one after the other (4096 -> 14336 25.3 us,
// 21.7 with two tiles), and the four-tile float32 and 16-row float32 forms spill some registers.
template <typename T, int G, bool ZEROS>
int affine_g(const W4Args &a, cudaStream_t stream) {
  const bool many = (long long)a.o_tiles * a.i_tiles >= 27LL * kPlanSms;
  const int nb = a.rows > 8 ? 2 : 1, R = !many || a.o_tiles < kPlanSms ? 1 : nb == 1 && a.o_tiles >= 4 * kPlanSms ? 4 : 2;
  const int ogs = (a.o_tiles + R - 1) / R, resident = 2 * kPlanSms;
  int warps = 8, cluster = 1;
  while (warps > 1 && warps > a.i_tiles) warps >>= 1;
  while (cluster < 8 && ogs * cluster * 2 <= resident && a.i_tiles >= 2 * cluster * warps) cluster *= 2;
  const int ctas = resident / cluster;
  if (nb == 2) return R == 2 ? affine_launch<T, G, 2, 2, ZEROS>(a, warps, cluster, ctas, stream) : affine_launch<T, G, 2, 1, ZEROS>(a, warps, cluster, ctas, stream);
  return R == 4 ? affine_launch<T, G, 1, 4, ZEROS>(a, warps, cluster, ctas, stream)
         : R == 2 ? affine_launch<T, G, 1, 2, ZEROS>(a, warps, cluster, ctas, stream) : affine_launch<T, G, 1, 1, ZEROS>(a, warps, cluster, ctas, stream);
}
template <typename T, int G>
int affine_z(const W4Args &a, bool zeros, cudaStream_t stream) {
  return zeros ? affine_g<T, G, true>(a, stream) : affine_g<T, G, false>(a, stream);
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
  a.block = l.block;
  a.device = dev;
  a.ld_x = ld_x; a.ld_y = ld_y;
  a.rows = (int)rows; a.c_in = d.c_in; a.c_out = d.c_out; a.i_tiles = (int)l.i_tiles; a.o_tiles = (int)l.o_tiles;
  a.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_x * sizeof(T) % 16 == 0;
  const bool z = d.has_zeros != 0;
  return d.group == 32 ? affine_z<T, 32>(a, z, stream) : d.group == 64 ? affine_z<T, 64>(a, z, stream) : affine_z<T, 128>(a, z, stream);
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
