// Weight and bias gradients of an affine layer whose input was kept as an 8-bit checkpoint:
//   dw[o][i] = sum_t dy[t][o] * x[t][i],   db[o] = sum_t dy[t][o],   x[t][i] = code * 2^(b - 133).
//
// The weight gradient is a product contracted over the tokens, D[i][o] = X^T dY, on the 5th-generation
// tensor cores (tcgen05.mma.kind::f16, both factors bfloat16, fp32 accumulators in tensor memory):
//  * the value of a checkpoint is exact in bfloat16, and so is every product; dy is taken as it is
//    (bfloat16), or as the exact sum of two (float16) or three (float32) bfloat16 parts, written once by a kernel of
//    its own and contracted one after the other, the smallest first;
//  * the 128 accumulator rows are input channels and the columns output channels: a warp that reads the
//    accumulator back holds 32 consecutive elements of one row of dw per column, so every store is a
//    coalesced line and nothing is staged. Both factors are MN-major in shared memory, as they lie in
//    global memory: no transpose anywhere;
//  * per CTA (one per SM): warps 0-15 expand the codes into the swizzled operand layout, warps 16-23 read the accumulators back,
//    warp 24 issues the TMA loads, warp 25 the MMAs, warps 26 and 27 bring the exponents. The converters work in as many groups as
//    there are stages, a chunk of 64 tokens per group: one warp needs about 1400 cycles from its wait to its next
//    one, and with all of them on every chunk that was the kernel's pace (512 cycles of MMAs per chunk);
//  * the tensor core's adder truncates, by 2^-25 of the sum per step of 16 tokens on average and up to 2^-23. Left alone over 65536
//    tokens that was half a rounding step of float16. So every sum is cut into runs of 512 tokens, which are added in fp32: the
//    accumulators are double, and while one takes the next run the epilogue adds the other's to sums that it keeps in
//    registers (128 columns per lane) until the unit is done. Adding the runs to dw in memory instead cost a quarter of the time;
//  * what bounds it: the way of a stage - copy 1600 cycles, expansion 800, issue and MMAs 1000 - against the four stages that fit;
//    8192 tokens, 4096 x 4096, inputs in L2 from the call before: bf16 254 us, 1080 TFLOP/s, with a 32-bit result 259; fp16
//    511 us, two products; fp32 786 us, three;
//  * tiles that fill whole waves of the 148 SMs are walked as they are; the tiles of the last, partial wave
//    are cut along the tokens so that it is full too, and a second kernel adds their parts in a fixed order.
#include <cstring>

#include "ckpt8.cuh"
#include "dwbnq_internal.h"
#include "dwbnq_tc.cuh"

namespace dwbnq {

namespace {

constexpr int kTileI = 128;       // input channels per tile = TMEM lanes
constexpr int kChunk = 64;        // tokens per pipeline stage
// Chunks per run. What the adder drops is relative to the sum, so the parts of dy below the leading digits (at most 2^-7 of it) may
// run longer. A run costs 128 loads and additions per epilogue lane, beside the MMAs of the next one: runs of 8, 16, 32 chunks and of
// the whole batch take the same time within 1% (8192 tokens, 4096 x 4096 bf16).
constexpr int kRun = 8, kLowRun = 64;
constexpr int kConvWarps = 16, kEpiWarps = 8, kTmaWarp = kConvWarps + kEpiWarps, kMmaWarp = kTmaWarp + 1, kExpWarp = kTmaWarp + 2;
constexpr int kThreads = 32 * (kConvWarps + kEpiWarps + 4);
// Registers per thread. The epilogue's sums want twice what a block of this size may be launched with, so the groups of four warps set
// their own number; together they are what the launch was given. (Converters with 40 and an epilogue with 136 that spills: 262 us;
// converters that load exponents themselves, with 48: 262; issuers with 40 or 24: 263 and 271.)
constexpr int kRegsLaunch = 72, kRegsConv = 32, kRegsEpi = 152, kRegsIssue = 72;
static_assert(kThreads * kRegsLaunch <= 65536 && kConvWarps % 4 == 0 && kEpiWarps % 4 == 0 &&
                  kConvWarps * kRegsConv + kEpiWarps * kRegsEpi + 4 * kRegsIssue <= kThreads / 32 * kRegsLaunch,
              "a warp that asks for more registers than the others gave back would wait for good");
constexpr int kTmemCols = 512;
constexpr int kSmemMax = 227 * 1024;
constexpr int kPlanSms = 148;     // SMs of a B200: the cut of the last wave does not depend on the device it is asked on
constexpr int kMaxParts = 2 * kPlanSms;

struct DwArgs {
  const unsigned char *exps;
  long long rows;
  int c_in, c_out, groups;
  int i_tiles;
  int token_chunks;        // ceil(rows / 64)
  int chunks;              // of a tile: token_chunks of every bfloat16 part of dy, the smallest part first
  int head;                // the first chunk of the part that holds dy's leading digits
  int exps_words;          // every row of exponents starts on a 4-byte boundary
  int full, segs, units;   // units 0 .. full-1: whole tiles; then segs parts of every further tile
  void *dw;
  float *parts;            // [unit - full][tile columns][128]
  int accum;
  int *flag;
};

// Which tile and which chunks of tokens unit u is.
__device__ __forceinline__ void dw_unit(const DwArgs &a, int u, int &tile, int &c0, int &c1) {
  if (u < a.full) {
    tile = u;
    c0 = 0;
    c1 = a.chunks;
  } else {
    const int v = u - a.full, q = v / a.segs, s = v - q * a.segs;
    tile = a.full + q;
    c0 = (int)((long long)a.chunks * s / a.segs);
    c1 = (int)((long long)a.chunks * (s + 1) / a.segs);
  }
}

// Eight codes (two words) as bfloat16 values of step `step2` (the step twice): k = (128 + low seven bits) - (128 or
// 256 for the sign bit), both exact in bfloat16, then the exact product with a power of two.
__device__ __forceinline__ unsigned int dw_pair(unsigned int two, __nv_bfloat162 step2, unsigned int magic) {  // magic: 128, twice
  const unsigned int lo = and_or(two, 0x007f007fu, magic), hi = and_or(two, 0x00800080u, magic);
  const __nv_bfloat162 k = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&lo), *reinterpret_cast<const __nv_bfloat162 *>(&hi));
  const __nv_bfloat162 v = __hmul2(k, step2);
  return *reinterpret_cast<const unsigned int *>(&v);
}
__device__ __forceinline__ uint4 dw_expand(uint2 c, unsigned int b, unsigned int magic) {
  const unsigned int s = b == kCkNonFinite ? 0x7fc07fc0u : b * 0x00800080u - 0x03000300u;  // (b - 6) << 7, twice
  const __nv_bfloat162 s2 = *reinterpret_cast<const __nv_bfloat162 *>(&s);
  uint4 r;
  r.x = dw_pair(__byte_perm(c.x, 0u, 0x4140), s2, magic);
  r.y = dw_pair(__byte_perm(c.x, 0u, 0x4342), s2, magic);
  r.z = dw_pair(__byte_perm(c.y, 0u, 0x4140), s2, magic);
  r.w = dw_pair(__byte_perm(c.y, 0u, 0x4342), s2, magic);
  return r;
}

// Eight values as PARTS vectors of eight bfloat16 that add up to them exactly: the truncated head of what is left (the upper half
// of the word, taken by the byte permutation that packs it), then the rest. A NaN stays one through every part; an infinity's rest
// would be one too, so a vector that holds a value that is not finite takes the second way.
template <int PARTS>
__device__ __forceinline__ void dw_split(float *v, uint4 *part) {
  unsigned int top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  if (PARTS > 1 && top >= 0x7f800000u) {
    const float inf = __uint_as_float(0x7f800000u);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      unsigned int w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = v[j] != v[j] ? 0x7fc0u : __float_as_uint(v[j]) >> 16;
        v[j] = fabsf(v[j]) < inf ? __fsub_rn(v[j], __uint_as_float(w[j] << 16)) : 0.0f;
      }
      part[q] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < PARTS; ++q) {
    unsigned int w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __byte_perm(__float_as_uint(v[2 * j]), __float_as_uint(v[2 * j + 1]), 0x7632);
    part[q] = make_uint4(w[0], w[1], w[2], w[3]);
    if (q + 1 < PARTS)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __fsub_rn(v[j], __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u));
  }
}

// dy as bfloat16 parts [PARTS][rows][pad] (pad: c_out up to a multiple of 8), which TMA can take whatever dy's type, address and row
// stride. A pass of its own: splitting inside the product kernel was done again for every tile of input channels, and with the
// parts beside dy itself in shared memory the pipeline was half as deep (8192 tokens, 4096 x 4096 fp16: 855 us against 509).
template <typename T, int PARTS, bool VECTORS>
__global__ void __launch_bounds__(256)
    affine_split_kernel(const T *__restrict__ dy, long long ld, long long rows, int c_out, const OctetGrid g, long long pad,
                        uint4 *__restrict__ out) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  float *stage = OctetStage<VECTORS>::get();
  for (OctetWalk w = octet_walk(g, rows); __any_sync(0xffffffffu, w.row < rows); octet_next(w)) {
    const bool in = w.row < rows;
    const long long c = w.col * 8LL;
    float v[8];
    Octet<T, VECTORS>::load(dy + w.row * ld + c, in ? c_out - c : 0, stage, v);
    uint4 part[PARTS];
    dw_split<PARTS>(v, part);
    if (in && c < pad)
#pragma unroll
      for (int q = 0; q < PARTS; ++q) out[((q * rows + w.row) * pad + c) / 8] = part[q];
  }
}

// A stage holds the expanded codes, dy, and the codes. Four stages and as many groups of converters, so that each stage's barriers are
// always awaited by the same group (a parity wait cannot tell a phase from the one after the next).
constexpr int kBn = 256, kXBytes = kChunk * kTileI * 2, kDyBytes = kChunk * kBn * 2, kStageBytes = kXBytes + kDyBytes + kChunk * kTileI;
constexpr int kStages = 4, kBox = kChunk * 128;  // a box: 64 tokens x 128 bytes
constexpr int kTileGroups = kTileI / kCkGroup, kExpBytes = kChunk * kTileGroups;  // exponents of a stage
static_assert(kStageBytes % 1024 == 0 && kStages * (kStageBytes + kExpBytes) + 1536 <= kSmemMax, "swizzle atoms; shared memory");

// pw_wait for a warp of a CTA that may be giving up: the flag is looked at only when the barrier is not ready.
__device__ __forceinline__ bool dw_wait(unsigned long long *bar, unsigned int parity, volatile int *abort_v) {
  if (__all_sync(0xffffffffu, pw_try_wait(bar, parity))) return true;
  return pw_wait(bar, parity) && !pw_giving_up(abort_v);
}

// The pointer, in a way the compiler cannot compute ahead of: all columns' addresses at once would not fit the registers.
template <typename T> __device__ __forceinline__ T *after(T *p) {
  asm volatile("" : "+l"(p));
  return p;
}
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// TW: type of dw.
template <typename TW>
__global__ void __launch_bounds__(kThreads, 1)
affine_dw_kernel(const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_codes, const DwArgs a) {
  constexpr int BN = kBn, GROUP = kConvWarps / kStages, TOKENS = kChunk / GROUP;  // converter warps per group, tokens per warp and chunk
  constexpr int NACC = kTmemCols / BN;
  constexpr int HALF = BN / 2;                        // columns per epilogue warp
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long bars[3 * kStages + 2 * NACC + 1];
  __shared__ __align__(16) unsigned char exps_s[kStages][kExpBytes];  // [token][group of channels]
  __shared__ unsigned int tmem_base_s;
  __shared__ int abort_s;
  unsigned long long *full = bars, *empty = bars + kStages, *conv = bars + 2 * kStages;
  unsigned long long *acc_full = bars + 3 * kStages, *acc_empty = acc_full + NACC, *drained = acc_empty + NACC;
  const unsigned int base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *sm = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 2);  // the copies' and the exponents'
      mbar_init(&empty[s], 1);
      mbar_init(&conv[s], GROUP);
    }
    for (int b = 0; b < NACC; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpiWarps);
    }
    mbar_init(drained, 1);
    abort_s = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const unsigned int tmem_base = tmem_base_s;
  volatile int *abort_v = &abort_s;
  int total = 0;  // chunks of this CTA
  for (int u = blockIdx.x; u < a.units; u += gridDim.x) {
    int tile, c0, c1;
    dw_unit(a, u, tile, c0, c1);
    total += c1 - c0;
  }

  if (warp == kTmaWarp) {
    // ---- TMA loads, boxes of 64 tokens x 128 bytes, zero beyond the tensors: the codes, and dy or one of its parts ----
    int s = 0, issued = 0;
    unsigned int ph = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < a.units; u += gridDim.x) {
      int tile, c0, c1;
      dw_unit(a, u, tile, c0, c1);
      const int ot = tile / a.i_tiles, o0 = ot * BN, i0 = (tile - ot * a.i_tiles) * kTileI;
      const int boxes = min(BN / 64, (a.c_out - o0 + 63) / 64);
      int part = a.chunks / a.token_chunks - 1 - c0 / a.token_chunks, ct = c0 % a.token_chunks;
      for (int c = c0; c < c1; ++c) {
        if (!dw_wait(&empty[s], ph ^ 1u, abort_v)) { ok = false; break; }
        if (elect_one()) {
          unsigned char *st = sm + s * kStageBytes;
          mbar_expect_tx(&full[s], (boxes + 1) * kBox);
          tma_load_2d(st + kXBytes + kDyBytes, &tm_codes, i0, ct * kChunk, &full[s]);
#pragma unroll
          for (int q = 0; q < BN / 64; ++q)
            if (q < boxes) tma_load_3d(st + kXBytes + q * kBox, &tm_dy, o0 + q * 64, ct * kChunk, part, &full[s]);
        }
        __syncwarp();
        if (++ct == a.token_chunks) { ct = 0; --part; }
        if (issued < kStages) ++issued;
        if (++s == kStages) { s = 0; ph ^= 1u; }
      }
    }
    if (!ok && lane == 0) {
      if (!*abort_v) { atomicExch(a.flag, 1); *abort_v = 1; }
      // the copies in flight land before the CTA gives its shared memory back
      for (; issued > 0; --issued) {
        if (--s < 0) { s = kStages - 1; ph ^= 1u; }
        pw_wait_lane(&full[s], ph);
      }
    }
  } else if (warp == kMmaWarp) {
    // ---- MMAs: the warp walks through the chunks, one elected lane issues ----
    // fp32 accumulator, bfloat16 factors, both MN-major, M = 128; N is set per tile
    const unsigned int idesc0 = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | (8u << 24);
    const unsigned long long dx0 = pw_smem_desc(base, kBox, 1024, 2), dd0 = pw_smem_desc(base + kXBytes, kBox, 1024, 2);
    const int last_steps = (int)((a.rows - (long long)(a.token_chunks - 1) * kChunk + 15) / 16);
    int s = 0, b = 0;
    unsigned int ph = 0, aph = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < a.units; u += gridDim.x) {
      int tile, c0, c1;
      dw_unit(a, u, tile, c0, c1);
      const int o0 = tile / a.i_tiles * BN;
      const int n = min(BN, (a.c_out - o0 + 15) & ~15);
      const unsigned int idesc = idesc0 | ((unsigned)(n >> 3) << 17);
      int run = 0, ct = c0 % a.token_chunks;
      for (int c = c0; c < c1; ++c) {
        // dy and the codes of the stage have landed when its converters have arrived: they waited for them
        if ((run == 0 && !dw_wait(&acc_empty[b], aph ^ 1u, abort_v)) || !dw_wait(&conv[s], ph, abort_v)) { ok = false; break; }
        tc_fence_after();
        const bool last = c == c1 - 1 || run == (c < a.head ? kLowRun : kRun) - 1 || c == a.head - 1;
        const int steps = ++ct == a.token_chunks ? last_steps : kChunk / 16;
        const unsigned long long so = (unsigned long long)(s * kStageBytes) >> 4, dx = dx0 + so, dd = dd0 + so;
        const unsigned int d = tmem_base + b * BN;
        if (ct == a.token_chunks) ct = 0;
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < kChunk / 16; ++j)  // a step is 16 rows of 128 bytes
            if (j == 0 || j < steps) tc_mma_f16(d, dx + j * 128, dd + j * 128, idesc, j ? 1u : run ? 1u : 0u);
          tc_commit(&empty[s]);
          if (last) tc_commit(&acc_full[b]);
        }
        __syncwarp();
        ++run;
        if (last) {
          run = 0;
          if (++b == NACC) { b = 0; aph ^= 1u; }
        }
        if (++s == kStages) { s = 0; ph ^= 1u; }
      }
    }
    if (!ok) {
      if (lane == 0 && !*abort_v) { atomicExch(a.flag, 1); *abort_v = 1; }
      if (elect_one()) tc_commit(drained);  // the MMAs in flight end before the tensor memory is given back
      __syncwarp();
      pw_wait(drained, 0);
    }
  } else if (warp >= kExpWarp) {
    // ---- exponents: two warps, every other chunk each, one chunk of the warp's ahead. Four groups of a token are one word where every
    // row of them starts on a word; else they come by byte loads ----
    const bool words = a.exps_words;
    int u = blockIdx.x, left = 0, ct = 0, gr = 0;  // chunks left of the unit, this one's number in its part of dy, the lane's group of channels
    // the cursor comes to the chunk `over` behind the start of unit u, which may lie in a later unit
    auto enter = [&](int over) {
      for (; u < a.units; u += gridDim.x) {
        int tile, c0, c1;
        dw_unit(a, u, tile, c0, c1);
        left = c1 - c0 - over;
        if (left > 0) {
          ct = (c0 + over) % a.token_chunks;
          gr = tile % a.i_tiles * kTileGroups + (words ? 0 : lane & 3);
          return;
        }
        over = -left;
      }
    };
    auto take = [&](unsigned int(&e)[8]) {  // those of the cursor's chunk; the cursor moves on
      unsigned int t = (unsigned)ct * kChunk + (words ? lane : lane >> 2);  // below 2^31
      const unsigned char *p = a.exps + (unsigned long long)t * (unsigned)a.groups + gr;
      const bool in = u < a.units && gr < a.groups;
      if (words) {
#pragma unroll
        for (int k = 0; k < 2; ++k, t += 32, p += 32LL * a.groups)
          e[k] = in && t < a.rows ? __ldg(reinterpret_cast<const unsigned int *>(p)) : kCkMinExp * 0x01010101u;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k, t += 8, p += 8LL * a.groups) e[k] = in && t < a.rows ? __ldg(p) : kCkMinExp;
      }
      left -= 2;
      ct += 2;
      if (left <= 0) {
        u += gridDim.x;
        enter(-left);
      } else {
        while (ct >= a.token_chunks) ct -= a.token_chunks;
      }
    };
    unsigned int e[8], next[8], ph = 0;
    bool ok = true;
    enter(warp - kExpWarp);
    take(e);
    int s = warp - kExpWarp;
    for (int n = s; n < total; n += 2) {
      take(next);
      if (!dw_wait(&empty[s], ph ^ 1u, abort_v)) { ok = false; break; }
      if (words) {
#pragma unroll
        for (int k = 0; k < 2; ++k) reinterpret_cast<unsigned int *>(exps_s[s])[k * 32 + lane] = e[k];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) exps_s[s][k * 32 + lane] = (unsigned char)e[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = next[k];
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
      s += 2;
      if (s >= kStages) { s -= kStages; ph ^= 1u; }
    }
    if (!ok && lane == 0 && !*abort_v) { atomicExch(a.flag, 1); *abort_v = 1; }
  } else if (warp < kConvWarps) {
    // ---- converters: group g has the chunks n = g, g + kStages, ... of this CTA and with them stage g; a warp has TOKENS tokens
    // of the chunk, a pass is two tokens, a lane eight channels. The code is kept short: unrolled over several chunks it threw
    // the instructions of the warps that issue the loads and the MMAs out of the instruction cache ----
    fewer_registers<kRegsConv>();
    const int g = warp / GROUP, l16 = lane & 15, hi = lane >> 4;
    const unsigned int tok0 = (warp % GROUP) * TOKENS, box = (l16 >> 3) * (unsigned)kBox;
    unsigned char *st = sm + g * kStageBytes;
    const unsigned int magic = opaque_constant(0x43004300u);
    unsigned int ph = 0;
    bool ok = true;
    for (int n = g; n < total; n += kStages) {
      if (!dw_wait(&full[g], ph, abort_v)) { ok = false; break; }
#pragma unroll
      for (int p = 0; p < TOKENS / 2; ++p) {
        const unsigned int r = tok0 + 2 * p + hi, e = exps_s[g][r * kTileGroups + (l16 >> 2)];
        const uint2 code = *reinterpret_cast<const uint2 *>(st + kXBytes + kDyBytes + r * kTileI + l16 * 8);
        *reinterpret_cast<uint4 *>(st + box + r * 128 + (((l16 & 7) ^ (r & 7)) << 4)) = dw_expand(code, e, magic);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // visible to the tensor core's reads
      __syncwarp();
      if (lane == 0) mbar_arrive(&conv[g]);
      ph ^= 1u;
    }
    if (!ok && lane == 0 && !*abort_v) { atomicExch(a.flag, 1); *abort_v = 1; }
  } else if (warp < kTmaWarp) {
    // ---- epilogue: warp (half, quarter) owns input channels [32 quarter, +32) and half of the columns. A lane keeps its columns'
    // sums in registers while the runs of a unit come in, and stores them once ----
    more_registers<kRegsEpi>();
    const int quarter = warp & 3, half = (warp - kConvWarps) >> 2;
    int b = 0;
    unsigned int aph = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < a.units; u += gridDim.x) {
      int tile, c0, c1;
      dw_unit(a, u, tile, c0, c1);
      const int ot = tile / a.i_tiles, o0 = ot * BN + half * HALF, n = min(HALF, a.c_out - o0);  // columns that exist (may be negative)
      const int low = min(max(a.head - c0, 0), c1 - c0);  // chunks of the smaller parts
      float sum[HALF];
#pragma unroll
      for (int j = 0; j < HALF; ++j) sum[j] = 0.0f;
      for (int r = (low + kLowRun - 1) / kLowRun + (c1 - c0 - low + kRun - 1) / kRun; r > 0; --r) {
        if (!dw_wait(&acc_full[b], aph, abort_v)) { ok = false; break; }
        tc_fence_after();
        const unsigned int taddr = tmem_base + ((unsigned)(quarter * 32) << 16) + b * BN + half * HALF;
#pragma unroll
        for (int q = 0; q < HALF; q += 8)
          if (q < n) {
            unsigned int acc[8];
            tc_ld8(taddr + q, acc);
            tc_ld_wait8(acc);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[q + j] = __fadd_rn(sum[q + j], __uint_as_float(acc[j]));
          }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[b]);
        if (++b == NACC) { b = 0; aph ^= 1u; }
      }
      if (!ok) break;
      const int il = quarter * 32 + lane, i = (tile - ot * a.i_tiles) * kTileI + il;
      if (u >= a.full) {
        float *part = a.parts + ((long long)(u - a.full) * BN + half * HALF) * kTileI + il;
#pragma unroll
        for (int q = 0; q < HALF; q += 8) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (q + j < n) part[j * kTileI] = sum[q + j];
          part = after(part + 8 * kTileI);
        }
      } else if (i < a.c_in) {
        TW *dw = static_cast<TW *>(a.dw) + (long long)o0 * a.c_in + i;
#pragma unroll
        for (int q = 0; q < HALF; q += 8) {
          TW *to = dw;
          if (a.accum) {  // eight loads go out together
            TW old[8];
#pragma unroll
            for (int j = 0; j < 8; ++j, to += a.c_in) old[j] = q + j < n ? *to : Elem<TW>::from_f32(0.0f);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[q + j] = __fadd_rn(Elem<TW>::to_f32(old[j]), sum[q + j]);
            to = dw;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j, to += a.c_in)
            if (q + j < n) *to = Elem<TW>::from_f32(sum[q + j]);
          dw = after(to);
        }
      }
    }
    if (!ok && lane == 0 && !*abort_v) { atomicExch(a.flag, 1); *abort_v = 1; }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// dw of the tiles whose tokens were cut into `segs` parts: the parts added in order. CTA = tile x 2 COLS of its columns; a thread has
// COLS columns and 8 or 16 loads in flight. With many tiles of few parts, four columns per thread are fewer CTAs to start (40 tiles
// of three parts, fp32: 6.5 against 9.0 us); with few tiles one per thread keeps the SMs busy.
template <typename TW, int COLS>
__global__ void __launch_bounds__(2 * kTileI)
    affine_dw_join_kernel(const float *__restrict__ parts, int first_tile, int segs, int bn, int i_tiles, int c_in, int c_out,
                          TW *__restrict__ dw, int accum) {
  constexpr int AHEAD = COLS == 1 ? 8 : 4;
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  const int tile = first_tile + blockIdx.x, ot = tile / i_tiles, il = threadIdx.x % kTileI;
  const int n = blockIdx.y * 2 * COLS + threadIdx.x / kTileI;  // and every second one after it
  const int i = (tile - ot * i_tiles) * kTileI + il, o = ot * bn + n;
  if (i >= c_in || o >= c_out) return;
  const float *p = parts + ((long long)blockIdx.x * segs * bn + n) * kTileI + il;
  const long long step = (long long)bn * kTileI;
  float s[COLS] = {};
  for (int k = 0; k < segs; k += AHEAD) {
    float v[AHEAD][COLS];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
#pragma unroll
      for (int c = 0; c < COLS; ++c) v[j][c] = k + j < segs && o + 2 * c < c_out ? p[(k + j) * step + 2 * c * kTileI] : 0.0f;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
#pragma unroll
      for (int c = 0; c < COLS; ++c) s[c] = __fadd_rn(s[c], v[j][c]);
  }
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    if (o + 2 * c >= c_out) break;
    TW *q = dw + (long long)(o + 2 * c) * c_in + i;
    *q = Elem<TW>::from_f32(accum ? __fadd_rn(Elem<TW>::to_f32(*q), s[c]) : s[c]);
  }
}

// ---- bias gradient: CTA (64 channels, slice of the rows), a lane two channels, warp w the rows w, w + 8, ..., eight of them in
// flight; then the slices in order, a sixteenth of them per thread and those in order. PAIRS: the two channels of a row are one aligned load ----
constexpr int kDbMaxSlices = 256;

template <typename T, bool PAIRS>
__global__ void __launch_bounds__(256)
    affine_db_kernel(long long rows, int c_out, const T *__restrict__ dy, long long ld, float *__restrict__ part) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  __shared__ float sums[8][64];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, o = blockIdx.x * 64 + 2 * lane;
  const long long r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  const bool a_ok = o < c_out, b_ok = o + 1 < c_out;
  float s0 = 0.0f, s1 = 0.0f;
  auto pair = [&](const T *q, float &lo, float &hi) {
    if constexpr (sizeof(T) == 4) {
      const float2 e = __ldg(reinterpret_cast<const float2 *>(q));
      lo = e.x;
      hi = e.y;
    } else {
      unpack_pair(q, __ldg(reinterpret_cast<const unsigned int *>(q)), lo, hi);
    }
  };
  const T *q = dy + (r0 + w) * ld + o;
  long long t = r0 + w;
  if (PAIRS && b_ok) {
    for (; t + 56 < r1; t += 64, q += 64 * ld) {
      float v[8][2];
#pragma unroll
      for (int j = 0; j < 8; ++j) pair(q + 8 * j * ld, v[j][0], v[j][1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s0 = __fadd_rn(s0, v[j][0]);
        s1 = __fadd_rn(s1, v[j][1]);
      }
    }
  }
  for (; t < r1; t += 8, q += 8 * ld) {
    if (a_ok) s0 = __fadd_rn(s0, Elem<T>::to_f32(q[0]));
    if (b_ok) s1 = __fadd_rn(s1, Elem<T>::to_f32(q[1]));
  }
  sums[w][2 * lane] = s0;
  sums[w][2 * lane + 1] = s1;
  __syncthreads();
  const int c = threadIdx.x;
  if (c >= 64 || blockIdx.x * 64 + c >= c_out) return;
  float s = sums[0][c];
#pragma unroll
  for (int i = 1; i < 8; ++i) s = __fadd_rn(s, sums[i][c]);
  part[(long long)blockIdx.y * c_out + blockIdx.x * 64 + c] = s;
}
template <typename TW>
__global__ void __launch_bounds__(256)
    affine_db_join_kernel(const float *__restrict__ part, int slices, int c_out, TW *__restrict__ db, int accum) {
  pdl_launch_dependents();
  pdl_wait_for_predecessor();
  __shared__ float sums[16][16];
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4, o = blockIdx.x * 16 + c;
  float s = 0.0f;
  for (int i = slices * q / 16, end = slices * (q + 1) / 16; i < end; i += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < end && o < c_out ? part[(long long)(i + j) * c_out + o] : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __fadd_rn(s, v[j]);
  }
  sums[q][c] = s;
  __syncthreads();
  if (q || o >= c_out) return;
#pragma unroll
  for (int j = 1; j < 16; ++j) s = __fadd_rn(s, sums[j][c]);
  db[o] = Elem<TW>::from_f32(accum ? __fadd_rn(Elem<TW>::to_f32(db[o]), s) : s);
}

// ---- host side ---------------------------------------------------------------------------------------------

struct DwPlan {
  int i_tiles, o_tiles, token_chunks, chunks, full, segs, units;
  size_t parts_bytes, db_at, split_at, bytes;
};
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Slices of the rows for the bias gradient: eight CTAs per SM, at least 64 rows each.
int db_slices(const dwbnq_affine_desc &d) {
  const long long ctas = (d.c_out + 63) / 64, by_rows = d.rows / 64, want = 8 * kPlanSms / (ctas > 0 ? ctas : 1);
  const long long s = by_rows < want ? by_rows : want;
  return (int)(s < 1 ? 1 : s > kDbMaxSlices ? kDbMaxSlices : s);
}

// bfloat16 parts of dy, and whether they are made in a pass of their own (float16, float32, and bfloat16 rows that TMA cannot take).
int dw_parts(const dwbnq_affine_desc &d) { return d.dtype == DWBNQ_F32 ? 3 : d.dtype == DWBNQ_F16 ? 2 : 1; }
bool dw_splits(const dwbnq_affine_desc &d) {
  return d.dtype != DWBNQ_BF16 || d.dy_unaligned || d.ld_dy % 8 != 0 || d.ld_dy >= (1LL << 36);
}
long long dw_pad(const dwbnq_affine_desc &d) { return ((long long)d.c_out + 7) / 8 * 8; }

// Whole waves of kPlanSms tiles are walked uncut; the R tiles left over are cut into the number of parts that costs least, in chunks
// on the busiest SM: ceil(R s / SMs) parts of ceil(chunks / s) chunks, each with about 4 chunks' worth of read-back, and 8 for the
// second kernel and the parts' traffic.
DwPlan dw_plan(const dwbnq_affine_desc &d) {
  DwPlan p;
  p.i_tiles = (d.c_in + kTileI - 1) / kTileI;
  p.o_tiles = (d.c_out + kBn - 1) / kBn;
  p.token_chunks = (int)((d.rows + kChunk - 1) / kChunk);
  p.chunks = p.token_chunks * dw_parts(d);
  const long long tiles = (long long)p.i_tiles * p.o_tiles;
  const int rest = (int)(tiles % kPlanSms);
  p.full = (int)(tiles - rest);
  p.segs = 1;
  long long best = 0;
  for (int s = 1; rest && s <= p.chunks && rest * s <= kMaxParts; ++s) {
    const long long cost = (long long)((rest * s + kPlanSms - 1) / kPlanSms) * ((p.chunks + s - 1) / s + 4) + (s > 1 ? 8 : 0);
    if (s == 1 || cost < best) { best = cost; p.segs = s; }
  }
  if (p.segs == 1) p.full = (int)tiles;
  p.units = p.segs == 1 ? (int)tiles : p.full + rest * p.segs;
  p.parts_bytes = p.segs == 1 ? 0 : up256((size_t)rest * p.segs * kBn * kTileI * 4);
  p.db_at = 256 + p.parts_bytes;
  p.split_at = p.db_at + up256((size_t)db_slices(d) * d.c_out * 4);
  p.bytes = p.split_at + (dw_splits(d) && d.c_in ? up256((size_t)dw_parts(d) * d.rows * dw_pad(d) * 2) : 0);
  return p;
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

template <typename TW>
int launch_dw(const CUtensorMap &tm, const CUtensorMap &tc, const DwArgs &a, int dev, cudaStream_t stream) {
  constexpr int smem = kStages * kStageBytes + 1024;
  auto kern = affine_dw_kernel<TW>;
  static std::atomic<unsigned long long> allowed{0};
  cudaError_t e;
  if (!allowed.load(std::memory_order_acquire)) {  // the split of the registers counts on what the kernel was compiled to
    cudaFuncAttributes fa;
    if ((e = cudaFuncGetAttributes(&fa, kern)) != cudaSuccess) return fail_cuda(e, "affine_dw_kernel attributes");
    if (fa.numRegs != kRegsLaunch) return fail(DWBNQ_ERR_UNSUPPORTED, "affine_dw_kernel was built with %d registers", fa.numRegs);
  }
  e = allow_smem(reinterpret_cast<const void *>(kern), smem, dev, allowed);
  if (e != cudaSuccess) return fail_cuda(e, "affine_dw_kernel attributes");
  const int sms = sm_count(-1);
  e = launch_pdl(kern, dim3((unsigned)(a.units < sms ? a.units : sms)), dim3(kThreads), (size_t)smem, stream, tm, tc, a);
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "affine_dw_kernel launch");
}

template <typename T, int PARTS>
int launch_split(const dwbnq_affine_desc &d, const void *dy, void *out, cudaStream_t stream) {
  const OctetGrid g = octet_grid(d.rows, d.c_out, 256, sm_count(-1) * 8);
  const T *p = static_cast<const T *>(dy);
  const cudaError_t e = octet_vectors(dy, d.ld_dy, sizeof(T))
                            ? launch_pdl(affine_split_kernel<T, PARTS, true>, dim3(g.ctas), dim3(256), 0, stream, p, (long long)d.ld_dy,
                                         (long long)d.rows, d.c_out, g, dw_pad(d), static_cast<uint4 *>(out))
                            : launch_pdl(affine_split_kernel<T, PARTS, false>, dim3(g.ctas), dim3(256), 0, stream, p, (long long)d.ld_dy,
                                         (long long)d.rows, d.c_out, g, dw_pad(d), static_cast<uint4 *>(out));
  return e == cudaSuccess ? DWBNQ_OK : fail_cuda(e, "affine_split_kernel launch");
}

template <typename T>
cudaError_t launch_db(const dwbnq_affine_desc &d, const T *dy, int slices, float *parts, cudaStream_t stream) {
  const dim3 grid((unsigned)((d.c_out + 63) / 64), (unsigned)slices);
  const bool pairs = reinterpret_cast<uintptr_t>(dy) % (2 * sizeof(T)) == 0 && d.ld_dy % 2 == 0;
  return pairs ? launch_pdl(affine_db_kernel<T, true>, grid, dim3(256), 0, stream, (long long)d.rows, d.c_out, dy, (long long)d.ld_dy, parts)
               : launch_pdl(affine_db_kernel<T, false>, grid, dim3(256), 0, stream, (long long)d.rows, d.c_out, dy, (long long)d.ld_dy, parts);
}

template <typename TW>
int run_t(const dwbnq_affine_desc &d, const void *codes, const void *exps, const void *dy, void *dw, void *db, int accum_mask,
          void *workspace, int dev, cudaStream_t stream) {
  cudaError_t e;
  if (d.rows == 0) {  // sums of nothing
    if (dw && !(accum_mask & 2) && (e = cudaMemsetAsync(dw, 0, sizeof(TW) * (size_t)d.c_out * d.c_in, stream)) != cudaSuccess)
      return fail_cuda(e, "cudaMemsetAsync");
    if (db && !(accum_mask & 4) && (e = cudaMemsetAsync(db, 0, sizeof(TW) * (size_t)d.c_out, stream)) != cudaSuccess)
      return fail_cuda(e, "cudaMemsetAsync");
    return DWBNQ_OK;
  }
  const DwPlan p = dw_plan(d);
  float *parts = reinterpret_cast<float *>(static_cast<char *>(workspace) + 256);
  float *dbp = reinterpret_cast<float *>(static_cast<char *>(workspace) + p.db_at);
  if (dw) {
    DwArgs a;
    std::memset(&a, 0, sizeof(a));
    a.exps = static_cast<const unsigned char *>(exps);
    a.rows = d.rows; a.c_in = d.c_in; a.c_out = d.c_out;
    a.groups = (d.c_in + kCkGroup - 1) / kCkGroup;
    a.exps_words = (reinterpret_cast<uintptr_t>(exps) | a.groups) % 4 == 0;
    a.i_tiles = p.i_tiles; a.token_chunks = p.token_chunks; a.chunks = p.chunks; a.full = p.full; a.segs = p.segs; a.units = p.units;
    a.head = p.chunks - p.token_chunks;
    a.dw = dw; a.parts = parts; a.accum = (accum_mask >> 1) & 1;
    int st = device_flag_ptr(dev, &a.flag);
    if (st != DWBNQ_OK) return st;
    const void *src = dy;
    long long pitch = d.ld_dy;
    if (dw_splits(d)) {
      void *out = static_cast<char *>(workspace) + p.split_at;
      st = d.dtype == DWBNQ_F32 ? launch_split<float, 3>(d, dy, out, stream)
           : d.dtype == DWBNQ_F16 ? launch_split<__half, 2>(d, dy, out, stream) : launch_split<__nv_bfloat16, 1>(d, dy, out, stream);
      if (st != DWBNQ_OK) return st;
      src = out;
      pitch = dw_pad(d);
    }
    if (!encode_fn()) return fail(DWBNQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    CUtensorMap tm, tc;
    const cuuint32_t es[3] = {1, 1, 1};
    const cuuint64_t cdim[2] = {(cuuint64_t)a.groups * kCkGroup, (cuuint64_t)d.rows}, cstr[1] = {cdim[0]};
    const cuuint32_t cbox[2] = {kTileI, kChunk};
    CUresult r = encode_fn()(&tc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), cdim, cstr, cbox, es,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(DWBNQ_ERR_CUDA, "cuTensorMapEncodeTiled(codes) failed with CUresult %d", (int)r);
    const cuuint64_t dim[3] = {(cuuint64_t)d.c_out, (cuuint64_t)d.rows, (cuuint64_t)dw_parts(d)};
    // a single part has no stride between parts, and rows x ld_dy may be more than one may be
    const cuuint64_t str[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)pitch * 2 * (dw_splits(d) ? (cuuint64_t)d.rows : 1)};
    const cuuint32_t box[3] = {64, kChunk, 1};
    r = encode_fn()(&tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(src), dim, str, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(DWBNQ_ERR_CUDA, "cuTensorMapEncodeTiled(dy) failed with CUresult %d", (int)r);
    st = launch_dw<TW>(tm, tc, a, dev, stream);
    if (st != DWBNQ_OK) return st;
    if (p.segs > 1) {
      const int cut = (p.units - p.full) / p.segs;
      const bool many = cut * (kBn / 2) > 16 * kPlanSms;  // more than two waves of CTAs
      e = launch_pdl(many ? affine_dw_join_kernel<TW, 4> : affine_dw_join_kernel<TW, 1>, dim3((unsigned)cut, (unsigned)(kBn / (many ? 8 : 2))),
                     dim3(2 * kTileI), 0, stream, (const float *)parts, p.full, p.segs, kBn, p.i_tiles, d.c_in, d.c_out,
                     static_cast<TW *>(dw), (accum_mask >> 1) & 1);
      if (e != cudaSuccess) return fail_cuda(e, "affine_dw_join_kernel launch");
    }
  }
  if (db) {
    const int slices = db_slices(d);
    if (d.dtype == DWBNQ_F32) e = launch_db(d, static_cast<const float *>(dy), slices, dbp, stream);
    else if (d.dtype == DWBNQ_F16) e = launch_db(d, static_cast<const __half *>(dy), slices, dbp, stream);
    else e = launch_db(d, static_cast<const __nv_bfloat16 *>(dy), slices, dbp, stream);
    if (e != cudaSuccess) return fail_cuda(e, "affine_db_kernel launch");
    e = launch_pdl(affine_db_join_kernel<TW>, dim3((unsigned)((d.c_out + 15) / 16)), dim3(256), 0, stream, (const float *)dbp, slices, d.c_out,
                   static_cast<TW *>(db), (accum_mask >> 2) & 1);
    if (e != cudaSuccess) return fail_cuda(e, "affine_db_join_kernel launch");
  }
  return DWBNQ_OK;
}

}  // namespace

size_t affine_bwd_workspace_bytes(const dwbnq_affine_desc &d) { return dw_plan(d).bytes; }

int launch_affine_bwd(const dwbnq_affine_desc &d, const void *codes, const void *exps, const void *dy, void *dw, void *db,
                      int accum_mask, void *workspace, int dev, cudaStream_t stream) {
  if (d.dw_dtype == DWBNQ_F32) return run_t<float>(d, codes, exps, dy, dw, db, accum_mask, workspace, dev, stream);
  if (d.dw_dtype == DWBNQ_F16) return run_t<__half>(d, codes, exps, dy, dw, db, accum_mask, workspace, dev, stream);
  return run_t<__nv_bfloat16>(d, codes, exps, dy, dw, db, accum_mask, workspace, dev, stream);
}

}  // namespace dwbnq
