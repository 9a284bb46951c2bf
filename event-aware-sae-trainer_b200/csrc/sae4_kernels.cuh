// Serving a sparse autoencoder from 4-bit weights.
//
//   pre[t, f] = sum_k q[f, k] s[f, k / group] xc[t, k] + b_enc[f],  xc = bf16(x - b_dec)
//   feat      = pre > theta ? pre : 0
//   x_hat[t]  = sum over the active f of feat[t, f] D[f, :] + b_dec   (D in the same format)
//
// Weights are q in [-8, 7] with a scale per `group` columns of a row. A scale
// has at most 5 significant bits, so q s is exact in bf16: the tensor cores
// multiply the weights themselves, with no rounding of their own and no
// separate accumulator per group.
//
// For few tokens everything is bound by streaming F d / 2 bytes of weights,
// and next by the instructions that unpack them.
//
// Encoder layout: a block of 16 features x 64 columns is 512 bytes, 16 per
// lane of a warp as the m16n8k32 product's A fragments need them. Lane
// (g = lane / 4, j = lane % 4) holds columns 8 j .. 8 j + 7 and 32 + 8 j .. 32 +
// 8 j + 7 of features g and g + 8; its word s (0..3) has the four columns from
// 32 (s / 2) + 8 j + 4 (s % 2) on as nibbles
//   i = 0: feature g, columns 0 | 1    i = 1: feature g + 8, columns 0 | 1
//   i = 2: feature g, columns 2 | 3    i = 3: feature g + 8, columns 2 | 3
// nibble i in the low half-word for the first column, in the high one for the
// second, each q in two's complement. The column order inside a block is free as
// long as the tokens' fragments use the same one; this one keeps the two halves
// of a block, which groups of 32 scale differently, in products of their own.
// A feature's four lanes' 16 bytes are in the order s4_unit gives, in which neither
// the 32 lanes' own words nor one j of eight features (what the many-token kernel
// reads at a time) fall on the same banks.
// The block's scales follow it: one row, or for groups of 32 two, of 8 bf16 pairs
// (feature g low, g + 8 high). Four blocks along the columns (zeros past the last)
// make a chunk of a feature tile; the chunks of eight feature tiles lie side by
// side, then those of the next columns, then the next eight tiles: a warp that
// works on one tile copies a chunk at a time, a CTA that works on 128 features
// eight of them.
#pragma once
#include <cuda_bf16.h>
#include <cstdint>
#include "wgrad8_kernels.cuh"

namespace sae {

constexpr int S4_ROWS = 16;   // features per packed block
constexpr int S4_COLS = 64;   // columns per packed block

__host__ __device__ constexpr int64_t s4_tiles(int64_t F) { return (F + S4_ROWS - 1) / S4_ROWS; }
__host__ __device__ constexpr int64_t s4_kblocks(int64_t d) { return (d + S4_COLS - 1) / S4_COLS; }

// Place of lane (g, j)'s 16 bytes in its block.
__host__ __device__ constexpr int s4_unit(int g, int j) { return 4 * g + (j ^ (g >> 1)); }
__host__ __device__ constexpr int s4_block_bytes(int spb) { return 512 + 32 * spb; }

constexpr int S4_CHUNK = 4;        // blocks per chunk
constexpr int S4_TILES = 8;        // feature tiles side by side
__host__ __device__ constexpr int s4_chunk_bytes(int spb) { return S4_CHUNK * s4_block_bytes(spb); }
__host__ __device__ constexpr int s4_kchunks(int64_t kblocks) {
  return static_cast<int>((kblocks + S4_CHUNK - 1) / S4_CHUNK);
}
// Offset of a feature tile's chunk.
__host__ __device__ constexpr int64_t s4_chunk_at(int64_t tile, int kchunks, int chunk, int spb) {
  return ((tile / S4_TILES * kchunks + chunk) * S4_TILES + tile % S4_TILES) * s4_chunk_bytes(spb);
}
__host__ __device__ constexpr int64_t s4_packed_bytes(int64_t F, int64_t d, int spb) {
  return (s4_tiles(F) + S4_TILES - 1) / S4_TILES * S4_TILES * s4_kchunks(s4_kblocks(d)) *
         s4_chunk_bytes(spb);
}

struct S4Encoder {
  const uint8_t* w;         // packed weights
  const float* b_enc;
  const float* b_dec;
  const float* theta;
  int64_t d, F;
  int kblocks, spb;         // spb: scale rows per block (2 for groups of 32)
};

// Kernels of one call are launched so that the next may be set up while the one
// before it ends; this waits until all that one wrote can be read.
__device__ __forceinline__ void wait_for_kernel_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------ weight set-up
// One thread per (row, group): scale = max|w| / 7 rounded up to 5 significant
// bits (2^-100 at least), q = rint(w / scale).
__global__ void s4_quantize_kernel(const float* __restrict__ W, int64_t F, int64_t d, int group,
                                   uint8_t* __restrict__ codes, bf16* __restrict__ scales) {
  const int64_t ng = (d + group - 1) / group;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < F * ng;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t f = i / ng, c0 = (i - f * ng) * group;
    const int64_t c1 = min(d, c0 + group);
    const float* w = W + f * d;
    float amax = 0.f;
    for (int64_t c = c0; c < c1; ++c) amax = fmaxf(amax, fabsf(w[c]));
    const uint32_t b = __float_as_uint(__fdiv_rn(amax, 7.f));
    const float s = fmaxf(__uint_as_float((b + 0x7ffffu) & 0xfff80000u), exp2f(-100.f));
    scales[i] = __float2bfloat16_rn(s);
    for (int64_t c = c0; c < c1; c += 2) {
      const int lo = max(-7, min(7, __float2int_rn(__fdiv_rn(w[c], s))));
      const int hi = max(-7, min(7, __float2int_rn(__fdiv_rn(w[c + 1], s))));
      codes[f * (d / 2) + c / 2] = static_cast<uint8_t>((lo + 8) | ((hi + 8) << 4));
    }
  }
}

// Row-major codes [F, d / 2] and scales [F, ceil(d / group)] into the encoder
// layout; padding features and columns hold q = 0.
__global__ void s4_pack_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales,
                               int64_t F, int64_t d, int group, int spb, uint32_t* __restrict__ out) {
  const int64_t ng = (d + group - 1) / group;
  const int words = s4_block_bytes(spb) / 4, kchunks = s4_kchunks(s4_kblocks(d));
  auto q = [&](int64_t f, int64_t c) -> uint32_t {
    if (f >= F || c >= d) return 0u;
    return ((codes[f * (d / 2) + c / 2] >> (4 * (c & 1))) & 15u) ^ 8u;
  };
  auto scale = [&](int64_t f, int64_t c) -> uint32_t {
    return f < F && c < d ? scales[f * ng + c / group] : 0u;
  };
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
       i < s4_packed_bytes(F, d, spb) / 4; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t block = i / words, chunk = block / S4_CHUNK;
    const int at = static_cast<int>(i - block * words);
    const int64_t tile = chunk / S4_TILES / kchunks * S4_TILES + chunk % S4_TILES;
    const int64_t f0 = tile * S4_ROWS;
    const int64_t c0 = (chunk / S4_TILES % kchunks * S4_CHUNK + block % S4_CHUNK) * S4_COLS;
    uint32_t v = 0;
    if (at < 128) {
      const int g = at / 16, j = (at / 4 % 4) ^ (g >> 1), s = at % 4;   // s4_unit is its own inverse
      const int64_t f = f0 + g, c = c0 + 32 * (s >> 1) + 8 * j + 4 * (s & 1);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v |= q(f + 8 * (k & 1), c + (k & 2)) << (4 * k) |
             q(f + 8 * (k & 1), c + (k & 2) + 1) << (16 + 4 * k);
    } else {
      const int64_t f = f0 + at % 8, c = c0 + (at - 128) / 8 * 32;
      v = scale(f, c) | scale(f + 8, c) << 16;
    }
    out[i] = v;
  }
}

// ------------------------------------------------------------- unpacking
__device__ __forceinline__ uint32_t bf2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
constexpr uint32_t S4_BF2_M24 = 0xc1c0c1c0u;   // bf16x2 {-24, -24}

// ----------------------------------------------------------------- encoder
// What the encoder writes.
struct S4Out {
  float* out;          // [T, ldo] fp32
  int64_t ldo;
  uint16_t* mask;      // [T, ldm] active bits, 16 features each; or nullptr
  int64_t ldm;
  int mode;            // 0: pre; 1: feat (0 where the gate is closed); 2: active values only
};

// A NaN passes; thresholds are not NaN.
__device__ __forceinline__ float s4_gate(float pre, float theta) {
  return pre <= theta ? 0.f : pre;
}

// Few tokens (at most 2 NT), on integer tensor cores.
//
// Unpacking 4-bit weights to bf16 costs two instructions each pair and more on
// half-rate pipes; to int8 it is three per eight weights: w & 0xf0f0f0f0 and
// (w << 4) & 0xf0f0f0f0 are eight bytes 16 q. So a token's xc is written as a
// fixed-point number: with 2^E above its largest |xc|, rint(xc 2^(30 - E)) in
// four signed bytes ("limbs"), each a column of the m16n8k32 s8 product. That
// keeps every bit of an xc of at least 2^(E - 23), which 2^-22 of the largest always
// is, and is off by at most 2^(E - 31), 2^-30 of the largest, below (bf16 itself has
// 8 bits); the products and the sums over a
// block of 64 columns are whole numbers below 2^21, exact. The integer
// accumulator starts at the bits of 1.5 * 2^23, so it ends as the bits of
// 1.5 * 2^23 + 16 S: a subtraction and one fma with the group's scale add it
// to an fp32 sum per limb. The limbs are joined at the end.
// A token that holds an infinity or a NaN gives NaN for every feature.
//
// One block per SM, whose warps take feature tiles (16 features, all columns)
// in turn, as many warps as share the SM's tiles evenly; where there are fewer
// tiles than that, ks warps split a tile's columns and their sums are added in
// warp order. Each warp streams its blocks through a ring of its own in shared
// memory by bulk copies, a chunk (256 columns) a slot; they run on from
// one tile into the next, so that the copies in flight, not the registers,
// set the bandwidth. One token, weights not in L2: 1536 x 49152 14 us
// (2.8 TB/s), 4096 x 131072 50 us (5.7 TB/s).
constexpr int S4_MAX_WARPS = 24;
constexpr int S4_MAX_SLOTS = 8;

// Bytes of a limb column: an odd multiple of 64, so that the fragment loads of
// eight columns fall on different banks.
__host__ __device__ constexpr int s4_limb_pitch(int kblocks) { return (kblocks | 1) * S4_COLS; }
__host__ __device__ constexpr int s4_slot_bytes(int spb) {   // whole 128-byte lines
  return (s4_chunk_bytes(spb) + 127) / 128 * 128;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mma_m16n8k32_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                uint32_t a3, uint32_t b0, uint32_t b1,
                                                const int (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]),
        "r"(c[3]));
}

// xc of up to four columns from c on (0 past d).
template <typename XT>
__device__ __forceinline__ void s4_xc4(const XT* __restrict__ x, const float* __restrict__ b_dec,
                                       int64_t c, int64_t d, bool vec, float (&v)[4]) {
  if (vec && c + 4 <= d) {
    load_pre<XT, 4>(x + c, v);
    const float4 b = __ldg(reinterpret_cast<const float4*>(b_dec + c));
    v[0] = bf16_round(__fsub_rn(v[0], b.x)), v[1] = bf16_round(__fsub_rn(v[1], b.y));
    v[2] = bf16_round(__fsub_rn(v[2], b.z)), v[3] = bf16_round(__fsub_rn(v[3], b.w));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = c + k < d ? bf16_round(__fsub_rn(load_f(x, c + k), b_dec[c + k])) : 0.f;
  }
}

// Biased exponent of a token's largest |xc| (as bits), at least 2^-87: limbs of a
// smaller token have fewer bits.
__device__ __forceinline__ int s4_exponent(uint32_t largest) {
  return max(static_cast<int>(largest >> 23), 40);
}

template <int NT, int SPB, typename XT>
__global__ void __launch_bounds__(32 * S4_MAX_WARPS, 1)
    s4_encode_few_kernel(const S4Encoder e, const XT* __restrict__ x, int64_t ldx, int vec,
                         int n_tok, int ks, int slots, const S4Out o) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_bar[S4_MAX_WARPS * S4_MAX_SLOTS];
  __shared__ uint32_t s_max[2 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int g = lane >> 2, j = lane & 3;
  const int pitch = s4_limb_pitch(e.kblocks);
  constexpr int slot_bytes = s4_slot_bytes(SPB), block_bytes = s4_block_bytes(SPB);
  uint8_t* s_limb = smem;                                        // [8 NT][pitch]
  uint8_t* s_ring = smem + 8 * NT * pitch + static_cast<size_t>(warp) * slots * slot_bytes;
  float* s_sum = reinterpret_cast<float*>(smem + 8 * NT * pitch + static_cast<size_t>(warps) * slots * slot_bytes);
  uint64_t* bar = s_bar + warp * S4_MAX_SLOTS;

  const int at_once = warps / ks, part = warp % ks;
  const int kchunks = s4_kchunks(e.kblocks);
  const int chunk0 = kchunks * part / ks, chunk1 = kchunks * (part + 1) / ks;
  const int kb0 = chunk0 * S4_CHUNK, kb1 = min(e.kblocks, chunk1 * S4_CHUNK);
  const int64_t tiles = s4_tiles(e.F);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * at_once;
  const int64_t tile0 = blockIdx.x + static_cast<int64_t>(gridDim.x) * (warp / ks);

  // Requests (lane 0) run ahead of the products by `slots` slots.
  int64_t rtile = tile0;
  int rleft = kb1 - kb0;
  const uint8_t* rsrc = e.w + s4_chunk_at(rtile, kchunks, chunk0, SPB);
  auto request = [&](int slot) {
    if (rtile < tiles) {
      const uint32_t bytes = min(S4_CHUNK, rleft) * block_bytes;
      mbar_arrive_expect_tx(&bar[slot], bytes);
      bulk_load(s_ring + slot * slot_bytes, rsrc, bytes, &bar[slot]);
      rsrc += S4_TILES * s4_chunk_bytes(SPB);
      rleft -= S4_CHUNK;
      if (rleft <= 0) {
        rleft = kb1 - kb0;
        rtile += stride;
        rsrc = e.w + s4_chunk_at(rtile, kchunks, chunk0, SPB);
      }
    }
  };
  if (threadIdx.x < 2 * NT) s_max[threadIdx.x] = 0;
  if (lane == 0) {
    for (int i = 0; i < slots; ++i) mbar_init(&bar[i], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < slots; ++i) request(i);
  }
  __syncthreads();

  // The tokens' limbs: largest |xc| first, then the bytes, columns 0, 2, 1, 3 of
  // each four (the order of the weights' nibbles).
  const int fours = e.kblocks * (S4_COLS / 4);
  const int per_tok = max(1, warps / n_tok), tok_step = warps / per_tok;   // warps of a token
  for (int t = warp / per_tok; t < n_tok; t += tok_step) {
    uint32_t m = 0;
    for (int i = warp % per_tok * 32 + lane; i < fours; i += per_tok * 32) {
      float v[4];
      s4_xc4(x + t * ldx, e.b_dec, 4 * i, e.d, vec, v);
#pragma unroll
      for (int k = 0; k < 4; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) atomicMax(&s_max[t], m);     // a maximum does not depend on the order
  }
  __syncthreads();
  for (int t = warp / per_tok; t < n_tok; t += tok_step) {
    // 2^(30 - E), E = exponent of the largest + 1
    const float up = __uint_as_float(static_cast<uint32_t>(283 - s4_exponent(s_max[t])) << 23);
    for (int i = warp % per_tok * 32 + lane; i < fours; i += per_tok * 32) {
      float v[4];
      s4_xc4(x + t * ldx, e.b_dec, 4 * i, e.d, vec, v);
      uint32_t limb[4] = {0, 0, 0, 0};
      // a lane's 16 columns of a block side by side
      const int at = 4 * (i & ~15) + 16 * (i >> 1 & 3) + 8 * (i >> 3 & 1) + 4 * (i & 1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        int q = __float2int_rn(v[k] * up);
        const int shift = 8 * ((k & 1) * 2 + (k >> 1));
#pragma unroll
        for (int l = 0; l < 4; ++l) {
          const int b = static_cast<int8_t>(q);
          limb[l] |= static_cast<uint32_t>(b & 0xff) << shift;
          q = (q - b) >> 8;
        }
      }
#pragma unroll
      for (int l = 0; l < 4; ++l)
        *reinterpret_cast<uint32_t*>(s_limb + (4 * t + l) * pitch + at) = limb[l];
    }
  }
  __syncthreads();

  const uint8_t* limbs = s_limb + g * pitch + 16 * j;
  const int unit = 16 * s4_unit(g, j);
  const int magic[4] = {0x4b400000, 0x4b400000, 0x4b400000, 0x4b400000};
  const int64_t rounds = (tiles + stride - 1) / stride;
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int64_t r = 0; r < rounds; ++r) {
    const int64_t tile = tile0 + r * stride;
    const bool live = tile < tiles;
    float sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[n][i] = 0.f;
    if (live) {
      auto block = [&](const uint8_t* base, int i, int kb) {
        const uint4 w = *reinterpret_cast<const uint4*>(base + i * block_bytes + unit);
        const uint32_t* pairs = reinterpret_cast<const uint32_t*>(base + i * block_bytes + 512) + g;
        const uint32_t pair = pairs[0];
        const float s0 = __uint_as_float(pair << 16), s1 = __uint_as_float(pair & 0xffff0000u);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          lo[k] = (ws[k] << 4) & 0xf0f0f0f0u;
          hi[k] = ws[k] & 0xf0f0f0f0u;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 b = *reinterpret_cast<const uint4*>(limbs + n * 8 * pitch + kb * S4_COLS);
          int c[4], d[4];
          mma_m16n8k32_s8(c, lo[0], hi[0], lo[1], hi[1], b.x, b.y, magic);
          if constexpr (SPB == 2) {     // the second half has scales of its own
            const uint32_t pair2 = pairs[8];
            const float u0 = __uint_as_float(pair2 << 16), u1 = __uint_as_float(pair2 & 0xffff0000u);
            mma_m16n8k32_s8(d, lo[2], hi[2], lo[3], hi[3], b.z, b.w, magic);
            sum[n][0] = fmaf(u0, __int_as_float(d[0]) - 12582912.f, sum[n][0]);
            sum[n][1] = fmaf(u0, __int_as_float(d[1]) - 12582912.f, sum[n][1]);
            sum[n][2] = fmaf(u1, __int_as_float(d[2]) - 12582912.f, sum[n][2]);
            sum[n][3] = fmaf(u1, __int_as_float(d[3]) - 12582912.f, sum[n][3]);
#pragma unroll
            for (int k = 0; k < 4; ++k) d[k] = c[k];
          } else {
            mma_m16n8k32_s8(d, lo[2], hi[2], lo[3], hi[3], b.z, b.w, c);
          }
          sum[n][0] = fmaf(s0, __int_as_float(d[0]) - 12582912.f, sum[n][0]);
          sum[n][1] = fmaf(s0, __int_as_float(d[1]) - 12582912.f, sum[n][1]);
          sum[n][2] = fmaf(s1, __int_as_float(d[2]) - 12582912.f, sum[n][2]);
          sum[n][3] = fmaf(s1, __int_as_float(d[3]) - 12582912.f, sum[n][3]);
        }
      };
      for (int kb = kb0; kb < kb1; kb += S4_CHUNK) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bar[slot], phase, nullptr));
        const uint8_t* base = s_ring + slot * slot_bytes;
        if (ok) {
          if (kb + S4_CHUNK <= kb1) {
#pragma unroll
            for (int i = 0; i < S4_CHUNK; ++i) block(base, i, kb + i);
          } else {
            for (int i = 0; kb + i < kb1; ++i) block(base, i, kb + i);
          }
        }
        fence_proxy_async_smem();   // the slot has been read: the next copy may write it
        __syncwarp();
        if (lane == 0 && ok) request(slot);
        if (++slot == slots) {
          slot = 0;
          phase ^= 1;
        }
      }
    }
    if (ks > 1) {
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_sum[((warp * NT + n) * 4 + i) * 32 + lane] = sum[n][i];
      __syncthreads();
      if (part == 0) {
        for (int p = 1; p < ks; ++p)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sum[n][i] += s_sum[(((warp + p) * NT + n) * 4 + i) * 32 + lane];
      }
    }
    if (!live || part != 0) continue;

    // Join the limbs: this lane has limbs 0, 1 (j even) or 2, 3 of a token, for
    // features g and g + 8; afterwards lane (g, j) has token 2 n + j / 2,
    // feature g + 8 (j & 1).
    const int64_t f = tile * S4_ROWS + g + 8 * (j & 1);
    const bool f_ok = f < e.F;
    const float bias = f_ok ? e.b_enc[f] : 0.f, th = f_ok ? e.theta[f] : 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float lo = fmaf(256.f, sum[n][1], sum[n][0]), hi = fmaf(256.f, sum[n][3], sum[n][2]);
      const float unit = (j & 1) ? 65536.f : 1.f;
      lo *= unit, hi *= unit;
      lo += __shfl_xor_sync(0xffffffffu, lo, 1);
      hi += __shfl_xor_sync(0xffffffffu, hi, 1);
      const int t = 2 * n + (j >> 1);
      const uint32_t big = t < n_tok ? s_max[t] : 0u;
      // 2^(E - 30 - 4): the limbs' unit, and the weights' factor 16
      float scale = __uint_as_float(static_cast<uint32_t>(s4_exponent(big) - 33) << 23);
      if (big >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);
      const float p = fmaf((j & 1) ? hi : lo, scale, bias);
      const float v = o.mode ? s4_gate(p, th) : p;
      const bool on = f_ok && t < n_tok && v != 0.f;
      if (f_ok && t < n_tok && (o.mode != 2 || on)) o.out[t * o.ldo + f] = v;
      if (o.mask != nullptr) {
        const uint32_t bits = __ballot_sync(0xffffffffu, on);
        if (lane < 2 && 2 * n + lane < n_tok) {
          uint32_t m = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            m |= (bits >> (4 * k + 2 * lane) & 1u) << k;
            m |= (bits >> (4 * k + 2 * lane + 1) & 1u) << (8 + k);
          }
          uint16_t* row = o.mask + (2 * n + lane) * o.ldm;
          row[tile] = static_cast<uint16_t>(m);
          if (tile == tiles - 1 && tile + 1 < o.ldm) row[tile + 1] = 0;
        }
      }
    }
  }
  if (!ok) {
    // Giving up: the copies in flight land before the block leaves.
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {
    }
  }
}

// Many tokens, on tcgen05: D[f, t] for 128 features x up to 128 tokens a CTA.
//
// The weights are the A operand and live in tensor memory: sixteen warps unpack
// them to bf16 in registers (one thread a feature row, 64 columns) and store
// them with tcgen05.st, so that they never pass through shared memory, which
// the tokens' tiles (B, by TMA) would otherwise have to share: 16 + 16 KiB a
// stage for unpacked weights against 32 KiB a stage in all for 128 tokens.
// Unpacking is exact: a half-word 0x4180 | (q + 8) << 3 is the bf16 number
// 16 + (q + 8), and one bf16 fma with s and -24 s (7 bits) makes q s of it.
// Their packed chunks (128 features x 256 columns, 17 KiB side by side) come by
// one bulk copy each into a ring of their own.
// As in the weight gradients, the tensor core's sums are closed every 512
// columns and added in fp32 registers by eight epilogue warps, from two
// accumulators in turn; the register file is divided with setmaxnreg.
// Weights not in L2, 128 tokens at 2304 x 65536 take 50 us, 300 at 1536 x 49152 56
// (tensor cores 45 and 51% busy, the integer pipe 53 and 64%). No one thing bounds it:
// with all of it in L2 the former took 40 us, 37 without the unpacking arithmetic, 35
// without the products, 35 without the stores and 24 without all three, which is the
// streaming of the weights and, to every CTA anew, of the tokens. 16 and 21 tokens at
// 1536 x 49152 take 22 us, with the integer pipe 53% busy.
constexpr int S4M_FEATURES = 128, S4M_TOKENS = 128;
// A stage is a chunk, four column blocks. (Stages of one block and finer token rings
// made no difference.)
constexpr int S4M_STAGES = 2;
constexpr int S4M_SUM_STAGES = 2;           // per tensor-core accumulation: 512 columns
constexpr int S4M_UNPACK_WARPS = 16, S4M_SETS = 4;   // four warps (128 rows) a block
constexpr int S4M_EPI_WARP0 = 4 + S4M_UNPACK_WARPS;
constexpr int S4M_THREADS = 32 * (S4M_EPI_WARP0 + 8);
constexpr int S4M_RAW_STAGES = 4;
static_assert(S4M_RAW_STAGES % (2 * S4M_STAGES) == 0, "stage parities repeat with the raw ring");
static_assert(S4M_SETS == S4_CHUNK && S4M_FEATURES == S4_TILES * S4_ROWS,
              "a set takes the same block of every chunk");
constexpr int S4M_B_BYTES = S4M_TOKENS * 128;   // per column block
constexpr int S4M_ACC_COL = 256;            // A stages in TMEM columns [0, 256), accumulators behind
constexpr int S4M_REGS_LAUNCH = 72, S4M_REGS_CONTROL = 32, S4M_REGS_UNPACK = 64,
              S4M_REGS_EPI = 104;
static_assert(S4M_REGS_CONTROL + 4 * S4M_REGS_UNPACK + 2 * S4M_REGS_EPI <= 7 * S4M_REGS_LAUNCH,
              "register shares exceed the launch's");
__host__ __device__ constexpr int s4m_raw_bytes(int spb) { return S4_TILES * s4_chunk_bytes(spb); }
__host__ __device__ constexpr size_t s4m_smem(int spb) {
  return S4M_STAGES * S4_CHUNK * S4M_B_BYTES + S4M_RAW_STAGES * s4m_raw_bytes(spb) + 512 + 1024;
}

// xc = bf16(x - b_dec) as [T, pitch], zeros past d.
template <typename XT>
__global__ void __launch_bounds__(256)
    s4_center_kernel(const XT* __restrict__ x, int64_t ldx, int vec, const float* __restrict__ b_dec,
                     int64_t n_tokens, int64_t d, int64_t pitch, bf16* __restrict__ xc) {
  for (Walk8 w(static_cast<int>(pitch / 8)); w.row < n_tokens; w.next()) {
    const int64_t c = static_cast<int64_t>(w.col) * 8;
    const int n = static_cast<int>(d - c < 8 ? (d - c > 0 ? d - c : 0) : 8);
    float v[8], b[8];
    load8(x + w.row * ldx + c, vec, n, v);
    load8(b_dec + c, true, n, b);
    uint4 o;
    __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      o2[k] = __floats2bfloat162_rn(__fsub_rn(v[2 * k], b[2 * k]), __fsub_rn(v[2 * k + 1], b[2 * k + 1]));
    *reinterpret_cast<uint4*>(xc + w.row * pitch + c) = o;
  }
}

// The four columns of one feature in a packed word, as bf16 pairs (columns 0, 1)
// and (2, 3): rotations bring the feature's nibbles to bits 3..6 of the halves.
__device__ __forceinline__ void s4_unpack_row(uint32_t w, uint32_t rot01, uint32_t rot23, uint32_t s,
                                              uint32_t s24, uint32_t& p01, uint32_t& p23) {
  // two's complement nibbles: flipping their sign bit adds 8
  p01 = bf2_fma((__funnelshift_l(w, w, rot01) & 0x00780078u) ^ 0x41c041c0u, s, s24);
  p23 = bf2_fma((__funnelshift_l(w, w, rot23) & 0x00780078u) ^ 0x41c041c0u, s, s24);
}

__device__ __forceinline__ void tmem_st_32cols(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Split as tmem_ld32_issue / tmem_ld32_wait are, for 8 columns.
__device__ __forceinline__ void tmem_ld8_issue(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld8_wait(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T
__device__ __forceinline__ void tc_mma_bf16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                               uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// base + i * stride bytes on the multiply pipe: the unpacking warps keep the ALUs busy.
template <typename T>
__device__ __forceinline__ T* s4_row(T* base, uint32_t i, uint32_t stride) {
  uint64_t r;
  asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(r) : "r"(i), "r"(stride), "l"(base));
  return reinterpret_cast<T*>(r);
}

// Bias, gate and stores of a thread's feature for n <= 64 tokens, registers having
// no index unrolled, so kept to a few instructions a token: with mode and guards
// decided per token and 64-bit pointers stepped on the ALUs a tile's stores took
// 11500 cycles, longer than its products. FULL: every lane has a feature.
template <int MODE, bool FULL>
__device__ __forceinline__ void s4m_store(const float (&sum)[S4M_TOKENS / 2], int n, float bias,
                                          float th, bool f_ok, float* p, uint32_t p_stride,
                                          uint32_t* words, uint32_t word_stride, bool word_ok) {
#pragma unroll
  for (int c = 0; c < S4M_TOKENS / 2; c += 8) {
    if (c >= n) break;
#pragma unroll
    for (int i = c; i < c + 8; ++i) {
      const float pre = sum[i] + bias;
      const float v = MODE ? s4_gate(pre, th) : pre;
      const bool in = (FULL || f_ok) && (FULL || i < n);
      if (MODE < 2) {
        if (in) *s4_row(p, i, p_stride) = v;
      } else {
        const bool on = in && v != 0.f;
        if (on) *s4_row(p, i, p_stride) = v;
        const uint32_t bits = __ballot_sync(0xffffffffu, on);
        if (word_ok && (FULL || i < n)) *s4_row(words, i, word_stride) = bits;
      }
    }
  }
}

// MODE: S4Out's (2 with a mask).
template <int SPB, int MODE>
__global__ void __launch_bounds__(S4M_THREADS, 1)
    s4_encode_many_kernel(const __grid_constant__ CUtensorMap tm_x,
                          const S4Encoder e, int n_tokens, int tile_tokens, int n_tiles,
                          const S4Out o) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);   // still known to be shared memory
  constexpr int raw_bytes = s4m_raw_bytes(SPB), block_bytes = s4_block_bytes(SPB);
  uint8_t* s_b = smem;
  uint8_t* s_raw = smem + S4M_STAGES * S4_CHUNK * S4M_B_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_raw + S4M_RAW_STAGES * raw_bytes);
  uint64_t* full = bars;                       // the tokens' copy and four unpacking warps
  uint64_t* empty = bars + S4M_STAGES;
  uint64_t* acc_full = bars + 2 * S4M_STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_full + 4;
  uint64_t* raw_full = acc_full + 5;
  uint64_t* raw_empty = raw_full + S4M_RAW_STAGES;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(raw_empty + S4M_RAW_STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((2 * S4M_STAGES + 5 + 2 * S4M_RAW_STAGES) * 8 + 8 <= 512, "barrier area too small");

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S4M_STAGES; ++s) {
      mbar_init(&full[s], 1 + S4M_UNPACK_WARPS);   // the tokens' copies, the unpacking warps
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < S4M_RAW_STAGES; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], S4M_UNPACK_WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) prefetch_tmap(&tm_x);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int m_tiles = static_cast<int>((e.F + S4M_FEATURES - 1) / S4M_FEATURES);
  const int kchunks = s4_kchunks(e.kblocks);
  const int total = m_tiles * n_tiles;     // the token tiles of a weight tile are neighbours

  if (warp < 4) {
    regs_dec<S4M_REGS_CONTROL>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------ tokens by TMA
      wait_for_kernel_before();   // the centred tokens; the weights need no waiting
      Ring<S4M_STAGES> st;
      bool ok = true;
      for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
        const int t0 = u % n_tiles * tile_tokens;
        for (int kb = 0; kb < e.kblocks; kb += S4_CHUNK, st.next()) {
          if (!wg_wait(&empty[st.s], st.ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* dst = s_b + st.s * S4_CHUNK * S4M_B_BYTES;
          const int n = min(S4_CHUNK, e.kblocks - kb);
          mbar_arrive_expect_tx(&full[st.s], tile_tokens * 128 * n);
          for (int i = 0; i < n; ++i)
            tma_load_2d(dst + i * S4M_B_BYTES, &tm_x, &full[st.s], (kb + i) * S4_COLS, t0);
        }
      }
      if (!ok) {
        // Giving up: the copies in flight (microseconds) land before the CTA leaves.
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {
        }
      }
    } else if (warp == 2 && lane == 0) {
      // -------------------------------------------------- packed weights
      Ring<S4M_RAW_STAGES> st;
      bool ok = true;
      for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
        const uint8_t* src = e.w + s4_chunk_at(static_cast<int64_t>(u / n_tiles) * S4_TILES, kchunks, 0, SPB);
        for (int i = 0; i < kchunks; ++i, st.next()) {
          if (!wg_wait(&raw_empty[st.s], st.ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&raw_full[st.s], raw_bytes);
          bulk_load(s_raw + st.s * raw_bytes, src, raw_bytes, &raw_full[st.s]);
          src += raw_bytes;
        }
      }
      if (!ok) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {
        }
      }
    } else if (warp == 1) {
      // --------------------------------------------------------- MMA issue
      const uint32_t idesc = idesc_bf16_f32(S4M_FEATURES, 8) + (static_cast<uint32_t>(tile_tokens / 8 - 1) << 17);
      const uint64_t bd0 = smem_desc_k_sw128(s_b);
      const bool issuer = elect_one();
      Ring<S4M_STAGES> st;
      Ring<2> acc;
      bool ok = true, any = false;
      for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
        int blocks = e.kblocks;
        while (blocks > 0 && ok) {
          if (!wg_wait_warp(&acc_empty[acc.s], acc.ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + S4M_ACC_COL + acc.s * S4M_TOKENS;
          for (int k = 0; k < S4M_SUM_STAGES && blocks > 0; ++k, blocks -= S4_CHUNK, st.next()) {
            if (!wg_wait_warp(&full[st.s], st.ph, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t at = tmem_base + st.s * 32 * S4_CHUNK;
            const uint64_t bd = bd0 + static_cast<uint32_t>(st.s * (S4_CHUNK * S4M_B_BYTES >> 4));
            if (issuer) {
#pragma unroll
              for (int i = 0; i < S4_CHUNK; ++i) {
                if (i < blocks) {
#pragma unroll
                  for (int kk = 0; kk < 4; ++kk)
                    tc_mma_bf16_ta(d_tmem, at + 32 * i + 8 * kk, bd + (i * S4M_B_BYTES >> 4) + 2 * kk,
                                   idesc, i + kk > 0 ? 1u : static_cast<uint32_t>(k));
                }
              }
              tc_commit(&empty[st.s]);
            }
            __syncwarp();
            any = true;
          }
          if (ok && issuer) tc_commit(&acc_full[acc.s]);
          __syncwarp();
          acc.next();
        }
      }
      if (!ok && any) {
        if (issuer) tc_commit(drain);
        __syncwarp();
        mbar_wait(drain, 0, nullptr);
      }
    }
  } else if (warp < S4M_EPI_WARP0) {
    regs_dec<S4M_REGS_UNPACK>();
    // ------------------------------------------------------ weights to TMEM
    // Set `set` unpacks every fourth block; the warp's rows are the TMEM lanes it
    // may address: feature tiles 2 q and 2 q + 1 of the eight.
    const int set = (warp - 4) >> 2, q = warp & 3;
    const int units = total > static_cast<int>(blockIdx.x)
                          ? (total - 1 - static_cast<int>(blockIdx.x)) / static_cast<int>(gridDim.x) + 1
                          : 0;
    const int r = lane & 15;                      // row of its feature tile
    const uint32_t at = (2 * q + (lane >> 4)) * s4_chunk_bytes(SPB) + set * block_bytes;
    const uint32_t rot01 = (r >> 3) ? 31 : 3, rot23 = (r >> 3) ? 23 : 27;
    const uint32_t sel = (r >> 3) ? 0x3232 : 0x1010;
    int kb = set;                                 // block of the tile
    const uint32_t a_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + set * 32;
    const uint8_t* src0 = s_raw + at;
    uint32_t unit[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) unit[j] = 16 * s4_unit(r & 7, j);
    const uint8_t* scale0 = s_raw + at + 512 + (r & 7) * 4;
    // A round of the raw ring at a time, so that slots and parities are constants
    // (rings stepped at run time: 5 us more for 300 tokens).
    uint32_t ph = 0;
#pragma unroll 1
    for (int left = units * kchunks; left > 0; left -= S4M_RAW_STAGES, ph ^= 1) {
#pragma unroll
      for (int i = 0; i < S4M_RAW_STAGES; ++i) {
        if (i >= left) break;
        if (!wg_wait_warp(&raw_full[i], ph, abort_flag)) {
          left = 0;
          break;
        }
        const uint8_t* src = src0 + i * raw_bytes;
        const uint8_t* scale = scale0 + i * raw_bytes;
        const bool some = kb < e.kblocks;
        uint32_t out[32], s[2], s24[2];
        if (some) {
#pragma unroll
          for (int h = 0; h < SPB; ++h) {
            const uint32_t pair = *reinterpret_cast<const uint32_t*>(scale + 32 * h);
            s[h] = __byte_perm(pair, pair, sel);
            s24[h] = bf2_mul(s[h], S4_BF2_M24);
          }
          if (SPB == 1) s[1] = s[0], s24[1] = s24[0];
#pragma unroll
          for (int j = 0; j < 4; ++j) {   // columns 8 j .. + 7 and 32 + 8 j .. + 7: two words each
            const uint4 w = *reinterpret_cast<const uint4*>(src + unit[j]);
            s4_unpack_row(w.x, rot01, rot23, s[0], s24[0], out[4 * j], out[4 * j + 1]);
            s4_unpack_row(w.y, rot01, rot23, s[0], s24[0], out[4 * j + 2], out[4 * j + 3]);
            s4_unpack_row(w.z, rot01, rot23, s[1], s24[1], out[16 + 4 * j], out[16 + 4 * j + 1]);
            s4_unpack_row(w.w, rot01, rot23, s[1], s24[1], out[16 + 4 * j + 2], out[16 + 4 * j + 3]);
          }
        }
        // The reads are over before the next copy: without the fence nothing makes them
        // wait, and the epilogue's stores may be queued ahead of them.
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&raw_empty[i]);
        const int stage = i % S4M_STAGES;
        if (!wg_wait_warp(&empty[stage], (i / S4M_STAGES & 1) ^ 1, abort_flag)) {
          left = 0;
          break;
        }
        tc_fence_after();
        if (some) tmem_st_32cols(a_row + stage * (S4_CHUNK * 32), out);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[stage]);
        kb += S4_CHUNK;
        if (kb >= kchunks * S4_CHUNK) kb = set;
      }
    }
  } else {
    regs_inc<S4M_REGS_EPI>();
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, h = (warp - S4M_EPI_WARP0) >> 2;
    const int n_half = tile_tokens / 2;                       // a multiple of 8
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + S4M_ACC_COL + h * n_half;
    Ring<2> acc;
    bool ok = true;
    for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
      float sum[S4M_TOKENS / 2];
#pragma unroll
      for (int i = 0; i < S4M_TOKENS / 2; ++i) sum[i] = 0.f;
      for (int left = kchunks; left > 0; left -= S4M_SUM_STAGES, acc.next()) {
        if (!wg_wait_warp(&acc_full[acc.s], acc.ph, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // a load is in flight while the one before it is added
        const uint32_t src = t_row + acc.s * S4M_TOKENS;
        uint32_t v[2][8];
        tmem_ld8_issue(src, v[0]);
#pragma unroll
        for (int c = 0; c < S4M_TOKENS / 2; c += 8) {
          if (c < n_half) {
            uint32_t(&cur)[8] = v[(c >> 3) & 1];
            tmem_ld8_wait(cur);
            if (c + 8 < n_half) tmem_ld8_issue(src + c + 8, v[((c >> 3) + 1) & 1]);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[c + i] += __uint_as_float(cur[i]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc.s]);
      }
      if (!ok) break;
      const int64_t f0 = static_cast<int64_t>(u / n_tiles) * S4M_FEATURES + q * 32;
      const int64_t f = f0 + lane;
      const bool f_ok = f < e.F;
      const float bias = f_ok ? e.b_enc[f] : 0.f, th = f_ok ? e.theta[f] : 0.f;
      const int t0 = u % n_tiles * tile_tokens + h * n_half;
      const int n = min(n_half, n_tokens - t0);
      float* p = o.out + t0 * o.ldo + f;
      uint32_t* words = MODE == 2 ? reinterpret_cast<uint32_t*>(o.mask + t0 * o.ldm) + f0 / 32 : nullptr;
      const uint32_t p_stride = static_cast<uint32_t>(o.ldo * 4), word_stride = static_cast<uint32_t>(o.ldm * 2);
      const bool word_ok = lane == 0 && f0 < e.F;
      if (f0 + 32 <= e.F && n % 8 == 0)
        s4m_store<MODE, true>(sum, n, bias, th, true, p, p_stride, words, word_stride, word_ok);
      else
        s4m_store<MODE, false>(sum, n, bias, th, f_ok, p, p_stride, words, word_stride, word_ok);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// --------------------------------------------------------------- decoder
// Active bits of dense activations [T, lda]: bit f % 16 of mask[t, f / 16] is
// acts[t, f] != 0 (a NaN counts). A warp makes S4_MASK_WORDS words (32 features
// each) at a time, its loads in flight together.
constexpr int S4_MASK_WORDS = 8;
__global__ void __launch_bounds__(256)
    s4_mask_kernel(const float* __restrict__ acts, int64_t lda, int64_t n_tokens, int64_t F,
                   uint16_t* __restrict__ mask, int64_t ldm) {
  const int lane = threadIdx.x & 31;
  const int64_t words = ldm / 2, per_row = (words + S4_MASK_WORDS - 1) / S4_MASK_WORDS;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  for (int64_t i = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
       i < n_tokens * per_row; i += warps) {
    const int64_t t = i / per_row, wd = (i - t * per_row) * S4_MASK_WORDS;
    const float* a = acts + t * lda + wd * 32 + lane;
    const int64_t left = F - wd * 32 - lane;   // features from this lane's first on
    float v[S4_MASK_WORDS];
#pragma unroll
    for (int k = 0; k < S4_MASK_WORDS; ++k) v[k] = 32 * k < left ? __ldg(a + 32 * k) : 0.f;
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < S4_MASK_WORDS; ++k) {
      const uint32_t b = __ballot_sync(0xffffffffu, v[k] != 0.f);
      if (lane == k) mine = b;
    }
    if (lane < S4_MASK_WORDS && wd + lane < words)
      reinterpret_cast<uint32_t*>(mask + t * ldm)[wd + lane] = mine;
  }
}

struct S4Decoder {
  const uint8_t* codes;    // [F, pitch] bytes, pitch a multiple of 16, column 2 i low in byte i
  const uint16_t* scale;   // [F, ng] bf16
  const float* b_dec;
  int64_t d, F, pitch;
  int ng, group_shift;     // group = 1 << group_shift
};

// x_hat[t, c0 .. c0 + 256) = sum over the active f of vals[t, f] D[f, :] + b_dec.
// Bound by a chain of dependent reads (mask, list, values, rows), not by bytes. A CTA
// lists a token's active features in ascending order from the mask (a block scan of
// the counts, S4_LIST at a time); sixteen groups of its threads take the listed rows
// in turn, a thread 16 columns (one 8-byte load), 8 rows in flight per group, and
// their sums are added in group order. 256 columns a CTA: 128 tokens at 2304 x 65536
// take 35 us more with 512 columns and 13 us more with 128.
// Tokens differ widely in their active features (thousands where most have 80:
// norms are LogNormal), and a batch waits for its longest list. So a token above
// S4_DEC_LIGHT is shared by a cluster of eight CTAs, an eighth of the features each,
// whose sums are added in rank order through distributed shared memory. How a token
// is summed depends on its own count alone, never on timing or on other tokens.
// S4_DEC_LIGHT: encoder and decoder of 128 | 400 tokens take 88 | 148 us at 96, 86 |
// 141 at 192, 86 | 133 at 384, of 40 tokens 43, 45 and 47 us.
constexpr int S4_DEC_THREADS = 256;
constexpr int S4_DEC_CTAS = 4;      // per SM, at least
constexpr int S4_DEC_COLS = 256;
constexpr int S4_DEC_LANES = S4_DEC_COLS / 16;                 // threads of a row
constexpr int S4_DEC_GROUPS = S4_DEC_THREADS / S4_DEC_LANES;   // rows at a time
constexpr int S4_LIST = 1024;
constexpr int S4_DEC_UNROLL = 8;
constexpr int S4_DEC_LIGHT = 192;
constexpr int S4_DEC_PARTS = 8;

__device__ __forceinline__ float ld_dsmem(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// acc[k] += v * (column k of eight nibbles, q + 8 each). A nibble left at bit p of
// a float's mantissa under the exponent of 2^23 is 2^23 + u 2^p; less
// 2^23 + 8 2^p it is q 2^p, exactly, which v 2^-p multiplies: five nibbles need
// no shift. (Products and sums are as for v q itself.)
struct S4Value {
  float v[5];   // v 2^-4i
  __device__ __forceinline__ explicit S4Value(float x) {
#pragma unroll
    for (int i = 0; i < 5; ++i) v[i] = x * (1.f / static_cast<float>(1 << (4 * i)));
  }
};
__device__ __forceinline__ void s4_axpy8(float* acc, uint32_t w, const S4Value& v) {
  const uint32_t top = w >> 20;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int i = k < 5 ? k : k - 5;
    const uint32_t u = ((k < 5 ? w : top) & (15u << (4 * i))) | 0x4b000000u;
    acc[k] = fmaf(v.v[i], __uint_as_float(u) - (8388608.f + static_cast<float>(8 << (4 * i))), acc[k]);
  }
}

struct S4DecodeSmem {
  int f[S4_LIST];
  float v[S4_LIST];
  float acc[S4_DEC_GROUPS][S4_DEC_COLS];
  int warp[S4_DEC_THREADS / 32];
};
struct S4DecodeIo {
  const float* vals;
  int64_t ldv;
  const uint16_t* mask;
  int64_t ldm;
  float* x_hat;
  int* counts;       // per token: given to the caller, or scratch for the shared tokens' kernel
  uint8_t* fired;
};

// This thread's words of a token's mask, among [first, first + n), with the active
// features in them, before them and in all.
struct S4Scan {
  const uint32_t* words;
  int first, w0, w1, mine, before, total;
};
__device__ __forceinline__ S4Scan s4_scan(const S4DecodeIo& o, int64_t t, int first, int n, int* s_warp) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  S4Scan s;
  s.words = reinterpret_cast<const uint32_t*>(o.mask + t * o.ldm) + first;
  s.first = first;
  const int per = (n + S4_DEC_THREADS - 1) / S4_DEC_THREADS;
  s.w0 = min(n, static_cast<int>(threadIdx.x) * per);
  s.w1 = min(n, s.w0 + per);
  s.mine = 0;
#pragma unroll 4
  for (int i = s.w0; i < s.w1; ++i) s.mine += __popc(s.words[i]);
  int before = s.mine;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, k);
    if (lane >= k) before += v;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = before;
  __syncthreads();
  s.total = 0;
  s.before = before - s.mine;
#pragma unroll
  for (int i = 0; i < S4_DEC_THREADS / 32; ++i) {
    if (i < warp) s.before += s_warp[i];
    s.total += s_warp[i];
  }
  return s;
}

// Lists a scan's active features from number `base` on, with their values; returns how many.
__device__ __forceinline__ int s4_list(const S4DecodeIo& o, int64_t t, const S4Scan& sc, int base,
                                       bool mark, S4DecodeSmem& sm) {
  int at = sc.before - base;
  if (at < S4_LIST && at + sc.mine > 0) {
    for (int i = sc.w0; i < sc.w1; ++i) {
      uint32_t b = sc.words[i];
      while (b != 0) {
        const int f = (sc.first + i) * 32 + __ffs(b) - 1;
        b &= b - 1;
        if (at >= 0 && at < S4_LIST) sm.f[at] = f;
        ++at;
      }
    }
  }
  __syncthreads();
  const int n = min(S4_LIST, sc.total - base);
  for (int i = threadIdx.x; i < n; i += S4_DEC_THREADS) {   // all values in one round trip
    const int f = sm.f[i];
    sm.v[i] = o.vals[t * o.ldv + f];
    if (mark) o.fired[f] = 1;
  }
  __syncthreads();
  return n;
}

// acc += this thread's share of the n listed rows: 16 columns from c on.
__device__ __forceinline__ void s4_rows(const S4Decoder& e, int64_t c, int n, const S4DecodeSmem& sm,
                                        float (&acc)[16]) {
  if (c >= e.d) return;
  const uint8_t* codes = e.codes + c / 2;
  const uint16_t* scale = e.scale + (c >> e.group_shift);
  for (int i0 = threadIdx.x / S4_DEC_LANES; i0 < n; i0 += S4_DEC_UNROLL * S4_DEC_GROUPS) {
    // All loads first, with no branch between them (past the list's end the last
    // row again): a scale awaited inside one made each row wait for the one before.
    uint2 w[S4_DEC_UNROLL];
    uint32_t sc[S4_DEC_UNROLL];
#pragma unroll
    for (int k = 0; k < S4_DEC_UNROLL; ++k) {
      const int64_t f = sm.f[min(i0 + k * S4_DEC_GROUPS, n - 1)];
      w[k] = __ldg(reinterpret_cast<const uint2*>(codes + f * e.pitch));
      sc[k] = __ldg(scale + f * e.ng);
    }
#pragma unroll
    for (int k = 0; k < S4_DEC_UNROLL; ++k) {
      if (i0 + k * S4_DEC_GROUPS < n) {
        const S4Value x(sm.v[i0 + k * S4_DEC_GROUPS] * __uint_as_float(sc[k] << 16));
        s4_axpy8(acc, w[k].x, x);
        s4_axpy8(acc + 8, w[k].y, x);
      }
    }
  }
}

// The threads' sums by column, added in group order, into sm.acc[0].
__device__ __forceinline__ void s4_join_rows(const float (&acc)[16], S4DecodeSmem& sm) {
  const int group = threadIdx.x / S4_DEC_LANES, lane = threadIdx.x % S4_DEC_LANES;
#pragma unroll
  for (int i = 0; i < 16; i += 4)
    *reinterpret_cast<float4*>(&sm.acc[group][lane * 16 + i]) =
        make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
  __syncthreads();
  for (int i = threadIdx.x; i < S4_DEC_COLS; i += S4_DEC_THREADS) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < S4_DEC_GROUPS; ++k) v += sm.acc[k][i];
    sm.acc[0][i] = v;
  }
}

// This CTA's eighth of a shared token; called by all CTAs of the cluster.
__device__ __forceinline__ void s4_decode_shared(const S4Decoder& e, const S4DecodeIo& o, int64_t t,
                                                 int64_t c0, int part, S4DecodeSmem& sm) {
  const int words = static_cast<int>(o.ldm / 2);
  const int first = static_cast<int>(static_cast<int64_t>(words) * part / S4_DEC_PARTS);
  const int last = static_cast<int>(static_cast<int64_t>(words) * (part + 1) / S4_DEC_PARTS);
  const S4Scan sc = s4_scan(o, t, first, last - first, sm.warp);
  float acc[16] = {};
  for (int base = 0; base < sc.total; base += S4_LIST) {
    if (base > 0) __syncthreads();
    const int n = s4_list(o, t, sc, base, o.fired != nullptr && c0 == 0, sm);
    s4_rows(e, c0 + threadIdx.x % S4_DEC_LANES * 16, n, sm, acc);
  }
  s4_join_rows(acc, sm);
  cluster_sync_all();
  // each CTA joins its share of the columns
  constexpr int share = S4_DEC_COLS / S4_DEC_PARTS;
  for (int i = part * share + threadIdx.x; i < (part + 1) * share; i += S4_DEC_THREADS) {
    const uint32_t here = smem_u32(&sm.acc[0][i]);
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < S4_DEC_PARTS; ++k) v += ld_dsmem(mapa_shared(here, k));
    if (c0 + i < e.d) o.x_hat[t * e.d + c0 + i] = v + e.b_dec[c0 + i];
  }
  cluster_sync_all();   // the sums of this CTA have been read
}

__device__ __forceinline__ void s4_decode_alone(const S4Decoder& e, const S4DecodeIo& o, int64_t t,
                                                int64_t c0, const S4Scan& sc, S4DecodeSmem& sm) {
  const int n = s4_list(o, t, sc, 0, o.fired != nullptr && c0 == 0, sm);
  float acc[16] = {};
  s4_rows(e, c0 + threadIdx.x % S4_DEC_LANES * 16, n, sm, acc);
  s4_join_rows(acc, sm);
  for (int i = threadIdx.x; i < S4_DEC_COLS; i += S4_DEC_THREADS)   // sums of this thread's own
    if (c0 + i < e.d) o.x_hat[t * e.d + c0 + i] = sm.acc[0][i] + e.b_dec[c0 + i];
}

// Few tokens: a cluster of eight CTAs per token and column range at once, seven
// of which leave a token that is not shared. (All eight count the same words.)
__global__ void __launch_bounds__(S4_DEC_THREADS, S4_DEC_CTAS)
    s4_decode_few_kernel(const S4Decoder e, const S4DecodeIo o) {
  __shared__ S4DecodeSmem sm;
  wait_for_kernel_before();
  const int64_t t = blockIdx.y, c0 = blockIdx.x * static_cast<int64_t>(S4_DEC_COLS);
  const S4Scan sc = s4_scan(o, t, 0, static_cast<int>(o.ldm / 2), sm.warp);
  const int n = sc.total;
  if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0 && o.counts != nullptr) o.counts[t] = n;
  if (n > S4_DEC_LIGHT)
    s4_decode_shared(e, o, t, c0, blockIdx.z, sm);
  else if (blockIdx.z == 0)
    s4_decode_alone(e, o, t, c0, sc, sm);
}

// Many tokens: one CTA per token and column range, which leaves the tokens to share
// to the next kernel. (Several ranges by one CTA save scans and lists, but took 26 us
// where this takes 20, for 400 tokens at 1536 x 49152.)
__global__ void __launch_bounds__(S4_DEC_THREADS, S4_DEC_CTAS)
    s4_decode_light_kernel(const S4Decoder e, const S4DecodeIo o) {
  __shared__ S4DecodeSmem sm;
  wait_for_kernel_before();
  const int64_t t = blockIdx.y, c0 = blockIdx.x * static_cast<int64_t>(S4_DEC_COLS);
  const S4Scan sc = s4_scan(o, t, 0, static_cast<int>(o.ldm / 2), sm.warp);
  if (blockIdx.x == 0 && threadIdx.x == 0) o.counts[t] = sc.total;
  if (sc.total <= S4_DEC_LIGHT) s4_decode_alone(e, o, t, c0, sc, sm);
}

// The tokens to share, clusters taking (token, column range) pairs in turn. Every
// CTA makes the same list of them from the counts, S4_DEC_THREADS tokens at a time.
__global__ void __launch_bounds__(S4_DEC_THREADS, S4_DEC_CTAS)
    s4_decode_heavy_kernel(const S4Decoder e, const S4DecodeIo o, int64_t n_tokens, int chunks) {
  __shared__ S4DecodeSmem sm;
  __shared__ int s_tok[S4_DEC_THREADS];
  __shared__ int s_heavy[S4_DEC_THREADS / 32];
  wait_for_kernel_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int skip = blockIdx.x;    // items until this cluster's next
  for (int64_t t0 = 0; t0 < n_tokens; t0 += S4_DEC_THREADS) {
    const int64_t t = t0 + threadIdx.x;
    const bool heavy = t < n_tokens && o.counts[t] > S4_DEC_LIGHT;
    const uint32_t bits = __ballot_sync(0xffffffffu, heavy);
    __syncthreads();
    if (lane == 0) s_heavy[warp] = __popc(bits);
    __syncthreads();
    int at = __popc(bits & ((1u << lane) - 1)), n = 0;
#pragma unroll
    for (int i = 0; i < S4_DEC_THREADS / 32; ++i) {
      if (i < warp) at += s_heavy[i];
      n += s_heavy[i];
    }
    if (heavy) s_tok[at] = static_cast<int>(threadIdx.x);
    __syncthreads();
    for (; skip < n * chunks; skip += gridDim.x)
      s4_decode_shared(e, o, t0 + s_tok[skip / chunks],
                       skip % chunks * static_cast<int64_t>(S4_DEC_COLS), blockIdx.z, sm);
    skip -= n * chunks;
  }
}

}  // namespace sae
