// Weight gradients from an 8-bit activation checkpoint:
//
//   D[c, n] = sum_t v[t, c] g[t, n]     v: int8 codes x power-of-two steps, g: bf16
//
// on tcgen05. The contraction runs over the tokens, and both
// operands are stored token by token, so both are used with their output
// dimension contiguous ("MN-major") and nothing is transposed:
//   * a pair of CTAs computes 256 checkpoint columns x 256 gradient columns;
//     each CTA holds 128 of the former (16 KiB) for 64 tokens per stage, and 128
//     of the latter (or all 256, see WgConfig::PAIRED);
//   * g comes by TMA, in boxes of 64 columns x 64 tokens with 128-byte swizzle;
//   * codes and steps come by TMA into a ring of their own (9 KiB a stage);
//     twelve warps expand them to bf16 (exact: 7-bit codes, power-of-two
//     steps) into the swizzled layout.
// The tensor core truncates when it adds to its accumulator, which drifts by
// about 1e-9 of the result per token summed (measured: 1.0e-6 over 1024 tokens,
// 3.8e-5 over 32768, against 4e-7 for fp32 FMAs). So it sums 512 tokens at a
// time, alternating between two TMEM accumulators, and eight epilogue warps add
// each finished one to a 128 x 256 tile of fp32 registers while the next
// accumulates; 128 tokens where g has three parts, since the small parts' products
// are cut to the large ones' last place too. That takes 128 accumulator registers a thread: the warps divide
// the register file with setmaxnreg.
//
// Where many tiles of gradient columns read the same codes, those are expanded
// once by act8_load_kernel into a bf16 workspace, and this kernel only multiplies
// (see wgrad8_plan for the rule).
//
// fp32 gradients are split into three bf16 parts (8 + 8 + 8 bits, exactly g). A
// stage then holds all three, so that codes are expanded once for three products:
// 4096 tokens x 8192 columns x 256 fp32 gradients take 51 us, 61 part after part.
// Bound by the tensor cores: 32768 tokens x 1536 columns x 49152 bf16 gradients take
// 2.8 to 3.1 ms after a pause, and 3.3 call after call under the power limit (the library's
// bf16 product of that size 3.2).
#pragma once
#include <cuda_bf16.h>
#include <cstdint>
#include "act8_kernels.cuh"
#include "tile_gemm.cuh"

namespace sae {

constexpr int WG_TOK = 64;                 // tokens per stage
constexpr int WG_BOX_BYTES = WG_TOK * 128; // 64 tokens x 64 columns bf16
constexpr int WG_OPERAND_BYTES = 2 * WG_BOX_BYTES;
constexpr int WG_RAW_CODES = WG_TOK * 128, WG_RAW_STEPS = WG_TOK * 16;
constexpr int WG_RAW_BYTES = WG_RAW_CODES + WG_RAW_STEPS;
constexpr int WG_EXPAND_WARPS = 12;        // in groups of four; a group expands every third stage
constexpr int WG_GROUP_WARPS = 4, WG_GROUPS = WG_EXPAND_WARPS / WG_GROUP_WARPS;
// EXPAND: the kernel expands the codes itself; otherwise it is given them as bf16.
// PARTS: bf16 parts of g (3 only with EXPAND).
template <bool EXPAND, int PARTS>
struct WgConfig {
  // A pair multiplies together (cta_group::2), each CTA with half of g's tile. What
  // the other CTA expands then has to be released to the leader at cluster scope,
  // and each such arrival takes about 2200 cycles. Behind the products of three parts
  // they are hidden (164 | 166 us for 4096 tokens x 16384 columns by 512 gradients, with
  // arrivals of CTA scope, which order nothing for another CTA, and these). With one
  // part they are not (4096 x 49152 by 1536: 590 | 890 us), so there each CTA
  // multiplies for itself, with a whole tile of g: 640 us, and for 8192 x 1536 by 256,
  // 768 and 1536 gradients 39, 47 and 62 as against 41, 49 and 63.
  static constexpr bool PAIRED = !EXPAND || PARTS == 3;
  static constexpr int G_BOXES = PAIRED ? 2 : 4;   // of 64 gradient columns, a part and CTA
  static constexpr int STAGES = PARTS == 3 ? 3 : EXPAND ? 4 : 7;
  static constexpr int RAW_STAGES = EXPAND ? 3 : 0;
  // Stages per tensor-core accumulation: 32 products of 16 tokens, or 24 of three parts.
  static constexpr int CHUNK = PARTS == 3 ? 2 : 8;
  static constexpr int G_BYTES = G_BOXES * WG_BOX_BYTES;
  static constexpr int STAGE_BYTES = WG_OPERAND_BYTES + PARTS * G_BYTES;
  // warpgroups: TMA + MMA, 3 x expand, 2 x epilogue
  static constexpr int EPI_WARP0 = 4 + (EXPAND ? WG_EXPAND_WARPS : 0);
  static constexpr int THREADS = 32 * (EPI_WARP0 + 8);
  static constexpr size_t SMEM = STAGES * STAGE_BYTES + RAW_STAGES * WG_RAW_BYTES + 256 + 1024;
  static_assert(SMEM <= 227 * 1024, "stages exceed the shared memory of a CTA");
  static_assert((2 * STAGES + 6 + 2 * RAW_STAGES) * 8 + 8 <= 256, "barrier area too small");
};
// Register shares per thread; the launch provides 80 x 768.
constexpr int WG_REGS_LAUNCH = 80, WG_REGS_CONTROL = 32, WG_REGS_EXPAND = 48, WG_REGS_EPI = 152;
static_assert(WG_REGS_CONTROL + 3 * WG_REGS_EXPAND + 2 * WG_REGS_EPI <= 6 * WG_REGS_LAUNCH,
              "register shares exceed the launch's");

template <int R>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

// The waits of ptx.cuh and tile_gemm.cuh, but the clock is read only after some
// failed tries: here most waits fail once, and a read of the global timer takes
// longer than what is waited for.
constexpr int WG_TRIES = 32;
__device__ __forceinline__ bool wg_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const uint32_t b = smem_u32(bar);
  for (int i = 0; i < WG_TRIES; ++i)
    if (mbar_try_wait(b, parity)) return true;
  return mbar_wait(bar, parity, abort);
}
__device__ __forceinline__ bool wg_wait_cluster(uint64_t* bar, uint32_t parity,
                                                volatile int* abort) {
  const uint32_t b = smem_u32(bar);
  for (int i = 0; i < WG_TRIES; ++i)
    if (mbar_try_wait_cluster(b, parity)) return true;
  return mbar_wait_cluster(bar, parity, abort);
}

// A wait of all 32 lanes with one answer. Lanes that time out while others do not would
// leave the loop for a barrier of the block, and the others wait at a barrier of the warp.
// (Costs 2 of 60 us for the 4-bit encoder with 300 tokens at 1536 x 49152, else nothing.)
__device__ __forceinline__ bool wg_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, wg_wait(bar, parity, abort));
}

// One lane of a converged warp. The MMA loops below keep the whole warp in step
// and elect a lane for the issue alone: inside a divergent branch the operands
// cannot stay in uniform registers, and four products took 700 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.b32 %0, 1, 0, P;\n\t}"
               : "=r"(p));
  return p != 0;
}

// Descriptor of an MN-major bf16 tile in 128-byte swizzle: boxes of 64 columns
// (128 bytes) x WG_TOK rows; the next 64 columns one box further (leading byte
// offset), the next 8 tokens 1024 bytes further (stride byte offset).
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(const void* tile) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_u32(tile) >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(WG_BOX_BYTES >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
constexpr uint32_t kIdescMnMajor = (1u << 15) | (1u << 16);   // A and B are MN-major

// 32 lanes x 16 consecutive fp32 columns. Load and wait are one statement: between
// two, nothing would keep a use of the registers behind the wait.
__device__ __forceinline__ void tmem_ld_16cols(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ uint32_t bf2_add(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Two int8 codes, each zero-extended in a half-word, times a bf16 pair of steps.
// 128 + (low 7 bits) is a bf16 number; less 128, or 256 for a negative code, it
// is the code.
__device__ __forceinline__ uint32_t act8_expand2(uint32_t halves, uint32_t step2) {
  const uint32_t a = (halves & 0x007f007fu) | 0x43004300u;
  const uint32_t b = (halves & 0x00800080u) | 0xc300c300u;
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(bf2_add(a, b)), "r"(step2));
  return r;
}
__device__ __forceinline__ uint4 act8_expand8(uint32_t lo, uint32_t hi, uint32_t step2) {
  uint4 o;
  o.x = act8_expand2(__byte_perm(lo, 0, 0x4140), step2);
  o.y = act8_expand2(__byte_perm(lo, 0, 0x4342), step2);
  o.z = act8_expand2(__byte_perm(hi, 0, 0x4140), step2);
  o.w = act8_expand2(__byte_perm(hi, 0, 0x4342), step2);
  return o;
}

struct Wgrad8Args {
  int64_t n_cols, n_grads;
  float* out;              // split s writes at out + s * split_stride
  int64_t ldo, split_stride;
  float beta;
  int transposed;          // 1: out[c, n]; 0: out[n, c]
  int vec;                 // transposed and 16-byte aligned rows
  int m_pairs, n_tiles, splits;
  int tok_blocks;          // stages: ceil(T / 64)
  int part_rows;           // rows of g's tensor map between its parts
};

// Position in a ring of barriers: slot and the parity of its current round.
template <int N>
struct Ring {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      ph ^= 1;
    }
  }
};

struct Wgrad8Unit {
  int m, n, kb0, kb1;
  int64_t out_off;
};
__device__ __forceinline__ Wgrad8Unit wgrad8_unit(const Wgrad8Args& a, int u) {
  // checkpoint columns vary fastest: the pairs at work share a few slabs of g in L2
  Wgrad8Unit w;
  const int tiles = a.m_pairs * a.n_tiles;
  const int s = u / tiles, t = u - s * tiles;
  w.m = t % a.m_pairs;
  w.n = t / a.m_pairs;
  w.kb0 = static_cast<int>(static_cast<int64_t>(a.tok_blocks) * s / a.splits);
  w.kb1 = static_cast<int>(static_cast<int64_t>(a.tok_blocks) * (s + 1) / a.splits);
  w.out_off = s * a.split_stride;
  return w;
}

// tm_codes: the codes as bytes, or (not EXPAND) the values as bf16.
template <bool EXPAND, int PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(WgConfig<EXPAND, PARTS>::THREADS, 1)
    wgrad8_kernel(const __grid_constant__ CUtensorMap tm_g,
                  const __grid_constant__ CUtensorMap tm_codes,
                  const __grid_constant__ CUtensorMap tm_steps,
                  const __grid_constant__ Wgrad8Args a) {
  using Cfg = WgConfig<EXPAND, PARTS>;
  constexpr int STAGES = Cfg::STAGES, RAW_STAGES = Cfg::RAW_STAGES, CHUNK = Cfg::CHUNK;
  constexpr bool PAIRED = Cfg::PAIRED;
  constexpr int G_BYTES = Cfg::G_BYTES, B_BYTES = PARTS * G_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);   // still known to be shared memory
  uint8_t* s_a = smem;                                   // expanded codes
  uint8_t* s_b = smem + STAGES * WG_OPERAND_BYTES;       // g
  uint8_t* s_raw = smem + STAGES * Cfg::STAGE_BYTES;     // codes and steps as stored
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_raw + RAW_STAGES * WG_RAW_BYTES);
  uint64_t* full = bars;                       // copies and expanding warps (PAIRED: both CTAs', at the leader)
  uint64_t* empty = bars + STAGES;          // each CTA: stage free
  uint64_t* acc_full = bars + 2 * STAGES;   // each CTA
  uint64_t* acc_empty = bars + 2 * STAGES + 2;   // epilogue warps (PAIRED: both CTAs', at the leader)
  uint64_t* drain = bars + 2 * STAGES + 4;
  uint64_t* done_bar = bars + 2 * STAGES + 5;
  uint64_t* raw_full = bars + 2 * STAGES + 6;    // each CTA: its own copies
  uint64_t* raw_empty = raw_full + RAW_STAGES;   // each CTA: expanding warps
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(raw_empty + RAW_STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], EXPAND ? 1 + (PAIRED ? 2 : 1) * WG_GROUP_WARPS : 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], PAIRED ? 16 : 8);
    }
    for (int s = 0; s < RAW_STAGES; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], WG_GROUP_WARPS);
    }
    mbar_init(drain, 1);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (PAIRED) {
      tmem_alloc_pair(tmem_holder, TC_TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_holder, TC_TMEM_COLS);
      tmem_relinquish();
    }
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_g);
    prefetch_tmap(&tm_codes);
    if (EXPAND) prefetch_tmap(&tm_steps);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIRED) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int pairs = gridDim.x >> 1;
  const int pair = blockIdx.x >> 1;
  const int total = a.m_pairs * a.n_tiles * a.splits;

  if (warp < 4) {
    if constexpr (EXPAND) regs_dec<WG_REGS_CONTROL>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------- g (and expanded codes) by TMA
      Ring<STAGES> st;
      bool ok = true;
      const uint32_t lbar = mapa_shared(smem_u32(full), 0);
      for (int u = pair; u < total && ok; u += pairs) {
        const Wgrad8Unit w = wgrad8_unit(a, u);
        const int n0 = w.n * 256 + (PAIRED ? static_cast<int>(rank) * 128 : 0);
        const int c0 = w.m * 256 + static_cast<int>(rank) * 128;
        for (int kb = w.kb0; kb < w.kb1; ++kb, st.next()) {
          if (!wg_wait(&empty[st.s], st.ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* dst = s_b + st.s * B_BYTES;
          if (leader || !PAIRED)
            mbar_arrive_expect_tx(&full[st.s], (PAIRED ? 2 : 1) * (EXPAND ? B_BYTES : Cfg::STAGE_BYTES));
          if constexpr (!EXPAND) {
            uint8_t* da = s_a + st.s * WG_OPERAND_BYTES;
            tma_load_2d_pair(da, &tm_codes, lbar + 8 * st.s, c0, kb * WG_TOK);
            tma_load_2d_pair(da + WG_BOX_BYTES, &tm_codes, lbar + 8 * st.s, c0 + 64, kb * WG_TOK);
          }
#pragma unroll
          for (int i = 0; i < PARTS; ++i) {
            const int row = i * a.part_rows + kb * WG_TOK;
#pragma unroll
            for (int b = 0; b < Cfg::G_BOXES; ++b) {
              uint8_t* db = dst + i * G_BYTES + b * WG_BOX_BYTES;
              if constexpr (PAIRED)
                tma_load_2d_pair(db, &tm_g, lbar + 8 * st.s, n0 + 64 * b, row);
              else
                tma_load_2d(db, &tm_g, &full[st.s], n0 + 64 * b, row);
            }
          }
        }
      }
      if (!ok) {
        // Giving up: the copies in flight (microseconds) land before the CTAs leave.
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {
        }
      }
    } else if (EXPAND && warp == 2 && lane == 0) {
      // ------------------------------------------------ codes and steps by TMA
      Ring<EXPAND ? RAW_STAGES : 1> st;
      bool ok = true;
      for (int u = pair; u < total && ok; u += pairs) {
        const Wgrad8Unit w = wgrad8_unit(a, u);
        const int c0 = w.m * 256 + static_cast<int>(rank) * 128;
        for (int kb = w.kb0; kb < w.kb1; ++kb, st.next()) {
          if (!wg_wait(&raw_empty[st.s], st.ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* raw = s_raw + st.s * WG_RAW_BYTES;
          mbar_arrive_expect_tx(&raw_full[st.s], WG_RAW_BYTES);
          tma_load_2d(raw, &tm_codes, &raw_full[st.s], c0, kb * WG_TOK);
          // 16 step bytes (512 columns), from a 16-byte boundary
          tma_load_2d(raw + WG_RAW_CODES, &tm_steps, &raw_full[st.s], c0 / A8_GROUP & ~15, kb * WG_TOK);
        }
      }
      if (!ok) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {
        }
      }
    } else if (warp == 1 && (leader || !PAIRED)) {
      // ------------------------------------------------------- MMA issue
      constexpr uint32_t idesc = idesc_bf16_f32(PAIRED ? 256 : 128, 256) | kIdescMnMajor;
      const uint64_t ad0 = smem_desc_mn_sw128(s_a), bd0 = smem_desc_mn_sw128(s_b);
      // what the other CTA's threads have written is read by the products as well
      auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return PAIRED ? wg_wait_cluster(bar, parity, abort_flag) : wg_wait(bar, parity, abort_flag);
      };
      auto commit = [](uint64_t* bar) {
        if constexpr (PAIRED) tc_commit_pair_both(bar);
        else tc_commit(bar);
      };
      Ring<STAGES> st;
      Ring<2> acc;
      bool ok = true, any = false;
      for (int u = pair; u < total && ok; u += pairs) {
        const Wgrad8Unit w = wgrad8_unit(a, u);
        for (int left = w.kb1 - w.kb0; left > 0 && ok; left -= CHUNK, acc.next()) {
          if (!__all_sync(0xffffffffu, wait_all(&acc_empty[acc.s], acc.ph ^ 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc.s * 256);
          uint32_t add = 0;
          for (int k = min(left, CHUNK); k > 0; --k, st.next()) {
            if (!__all_sync(0xffffffffu, wait_all(&full[st.s], st.ph))) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t ad = ad0 + static_cast<uint32_t>(st.s * (WG_OPERAND_BYTES >> 4));
            const uint64_t bd = bd0 + static_cast<uint32_t>(st.s * (B_BYTES >> 4));
            if (elect_one()) {
#pragma unroll
              for (int i = 0; i < PARTS; ++i) {
#pragma unroll
                for (int kk = 0; kk < WG_TOK / 16; ++kk) {
                  // 16 tokens further: two groups of 8 rows, 2048 bytes
                  const uint64_t bk = bd + i * (G_BYTES >> 4) + 128 * kk;
                  if constexpr (PAIRED)
                    tc_mma_bf16_pair(d_tmem, ad + 128 * kk, bk, idesc, i + kk > 0 ? 1u : add);
                  else
                    tc_mma_bf16(d_tmem, ad + 128 * kk, bk, idesc, i + kk > 0 ? 1u : add);
                }
              }
              commit(&empty[st.s]);
            }
            __syncwarp();
            add = 1;
            any = true;
          }
          if (ok && elect_one()) commit(&acc_full[acc.s]);
          __syncwarp();
        }
      }
      if (!ok && any) {
        if (elect_one()) {
          if constexpr (PAIRED) tc_commit_pair_local(drain);
          else tc_commit(drain);
        }
        __syncwarp();
        mbar_wait(drain, 0, nullptr);
      }
    }
  } else if (EXPAND && warp < Cfg::EPI_WARP0) {
    if constexpr (EXPAND) regs_dec<WG_REGS_EXPAND>();
    // --------------------------------------------------- codes to bf16
    // Thread: columns 16 j .. 16 j + 15 of tokens r, r + 16, .. of its group's stages.
    // The groups overlap their waits, shared-memory round trips and proxy
    // fences: all warps on every stage ran at 2220 cycles a stage.
    const int group = (warp - 4) / WG_GROUP_WARPS;
    const int tid = threadIdx.x & (32 * WG_GROUP_WARPS - 1);
    const int j = tid & 7, r = tid >> 3;
    // 16-byte chunk of the swizzled row for this thread's first and second 8
    // columns. Threads 4..7 of a row store their second half first: the eight
    // stores of a quarter-warp then fall on different banks.
    const uint32_t box = s_a - smem + (j >> 2) * WG_BOX_BYTES;
    const bool flip = (j & 4) != 0;
    const int c0 = 2 * (j & 3), c1 = c0 + 1;
    const uint32_t lbar = mapa_shared(smem_u32(full), 0);
    Ring<STAGES> st;
    Ring<EXPAND ? RAW_STAGES : 1> rst;
    int turn = 0;
    bool ok = true;
    for (int u = pair; u < total && ok; u += pairs) {
      const Wgrad8Unit w = wgrad8_unit(a, u);
      // the byte of this thread's 16 columns among the 16 that were copied
      const int sb = ((w.m * 8 + static_cast<int>(rank) * 4) & 15) + (j >> 1);
      for (int left = w.kb1 - w.kb0; left > 0; --left, st.next(), rst.next()) {
        const bool mine = turn == group;
        if (++turn == WG_GROUPS) turn = 0;
        if (!mine) continue;
        if (!wg_wait_warp(&raw_full[rst.s], rst.ph, abort_flag)) {
          ok = false;
          break;
        }
        const uint8_t* raw = s_raw + rst.s * WG_RAW_BYTES;
        uint4 code[4];
        uint32_t step2[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = r + 16 * q;
          code[q] = *reinterpret_cast<const uint4*>(raw + row * 128 + 16 * j);
          step2[q] = raw[WG_RAW_CODES + row * 16 + sb] * 0x00800080u;
        }
        // The reads above have to be over before TMA fills the buffer again. Nothing has
        // used their values yet, and behind the epilogue's stores they can wait longer
        // than the next copy takes; the fence orders them before it. (Without it the codes
        // of a later stage could be read. It cost 1 of 78 us for 4096 tokens x 8192 columns
        // by 1024 bf16 gradients, nothing for 256 of fp32.)
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&raw_empty[rst.s]);
        if (!wg_wait_warp(&empty[st.s], st.ph ^ 1, abort_flag)) {
          ok = false;
          break;
        }
        uint8_t* base = smem + box + st.s * WG_OPERAND_BYTES;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = r + 16 * q;
          const uint4 lo = act8_expand8(code[q].x, code[q].y, step2[q]);
          const uint4 hi = act8_expand8(code[q].z, code[q].w, step2[q]);
          uint8_t* line = base + row * 128;
          const int o0 = (c0 ^ (row & 7)) << 4, o1 = (c1 ^ (row & 7)) << 4;
          *reinterpret_cast<uint4*>(line + (flip ? o1 : o0)) = flip ? hi : lo;
          *reinterpret_cast<uint4*>(line + (flip ? o0 : o1)) = flip ? lo : hi;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIRED) mbar_arrive_remote(lbar + 8 * st.s);
          else mbar_arrive(&full[st.s]);
        }
      }
    }
  } else {
    if constexpr (EXPAND) regs_inc<WG_REGS_EPI>();
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, h = (warp - Cfg::EPI_WARP0) >> 2;
    const uint32_t leader_empty0 = mapa_shared(smem_u32(&acc_empty[0]), 0);
    const uint32_t leader_empty1 = mapa_shared(smem_u32(&acc_empty[1]), 0);
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + h * 128;
    Ring<2> acc;
    bool ok = true;
    for (int u = pair; u < total && ok; u += pairs) {
      const Wgrad8Unit w = wgrad8_unit(a, u);
      float sum[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) sum[i] = 0.f;
      for (int left = w.kb1 - w.kb0; left > 0; left -= CHUNK, acc.next()) {
        if (!wg_wait_warp(&acc_full[acc.s], acc.ph, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 128; c += 16) {
          float v[16];
          tmem_ld_16cols(t_row + acc.s * 256 + c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[c + i] += v[i];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIRED) mbar_arrive_remote(acc.s ? leader_empty1 : leader_empty0);
          else mbar_arrive(&acc_empty[acc.s]);
        }
      }
      if (!ok) break;
      const int64_t c = static_cast<int64_t>(w.m) * 256 + rank * 128 + q * 32 + lane;
      const int64_t n0 = static_cast<int64_t>(w.n) * 256 + h * 128;
      if (c < a.n_cols) {
        if (a.transposed) {
          float* p = a.out + w.out_off + c * a.ldo + n0;
          if (a.vec && n0 + 128 <= a.n_grads) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float4 o = make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
              if (a.beta != 0.f) {
                const float4 old = reinterpret_cast<const float4*>(p)[i];
                o.x = fmaf(a.beta, old.x, o.x), o.y = fmaf(a.beta, old.y, o.y);
                o.z = fmaf(a.beta, old.z, o.z), o.w = fmaf(a.beta, old.w, o.w);
              }
              reinterpret_cast<float4*>(p)[i] = o;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (n0 + i < a.n_grads) p[i] = a.beta != 0.f ? fmaf(a.beta, p[i], sum[i]) : sum[i];
          }
        } else {
          // a warp's lanes hold consecutive columns of a row: 128-byte stores
          float* p = a.out + w.out_off + n0 * a.ldo + c;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (n0 + i < a.n_grads)
              p[i * a.ldo] = a.beta != 0.f ? fmaf(a.beta, p[i * a.ldo], sum[i]) : sum[i];
        }
      }
    }
  }

  // The leader's MMAs write both CTAs' TMEM and read both CTAs' shared memory:
  // neither leaves before both are done.
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if constexpr (PAIRED) {
      if (lane == 0) {
        mbar_arrive_remote(mapa_shared(smem_u32(done_bar), rank ^ 1u));
        mbar_wait_cluster(done_bar, 0, nullptr);
      }
      __syncwarp();
      tc_fence_after();
      tmem_dealloc_pair(tmem_base, TC_TMEM_COLS);
    } else {
      tc_fence_after();
      tmem_dealloc(tmem_base, TC_TMEM_COLS);
    }
  }
}

// g as bf16 parts [parts][rows_padded][pitch] for the kernel's TMA: an fp32 g in
// three (its upper, middle and lower 8 bits, exactly g; a non-finite value in
// the first alone), a bf16 g whose rows TMA cannot walk in one. Padding is zero.
template <typename GT>
__global__ void __launch_bounds__(256)
    wgrad8_parts_kernel(const GT* __restrict__ g, int64_t rows, int64_t cols, int64_t ldg,
                        int64_t rows_padded, int64_t pitch, bf16* __restrict__ out) {
  constexpr int kParts = sizeof(GT) == 4 ? 3 : 1;
  for (Walk8 w(static_cast<int>(pitch / 8)); w.row < rows_padded; w.next()) {
    const int64_t c = static_cast<int64_t>(w.col) * 8;
    float v[8];
    const int n = w.row < rows ? static_cast<int>(cols - c < 8 ? (cols - c > 0 ? cols - c : 0) : 8) : 0;
    const GT* p = g + w.row * ldg + c;
    load8(p, (reinterpret_cast<uintptr_t>(p) & 15) == 0, n, v);
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t hw[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float& x = v[2 * i + j];
          const uint32_t bits = __float_as_uint(x);
          const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
          // a NaN keeps a set bit when its lower half goes
          hw[j] = (bits >> 16) | ((!finite && (bits & 0x7fffffu) != 0) ? 0x40u : 0u);
          x = finite ? x - __uint_as_float(bits & 0xffff0000u) : 0.f;
        }
        o[i] = hw[0] | (hw[1] << 16);
      }
      *reinterpret_cast<uint4*>(out + (k * rows_padded + w.row) * pitch + c) =
          make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// out = beta out + the splits' partial products [splits][rows][cols], added in
// order; V columns a thread.
template <int V>
__global__ void __launch_bounds__(256)
    wgrad8_join_kernel(const float* __restrict__ part, int splits, int64_t rows, int64_t cols,
                       float beta, float* __restrict__ out, int64_t ldo) {
  for (Walk8 w(static_cast<int>(cols / V)); w.row < rows; w.next()) {
    const int64_t c = static_cast<int64_t>(w.col) * V;
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.f;
    for (int k = 0; k < splits; ++k) {
      float v[V];
      load_pre<float, V>(part + (k * rows + w.row) * cols + c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += v[i];
    }
    float* o = out + w.row * ldo + c;
    if (beta != 0.f) {
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = fmaf(beta, o[i], s[i]);
    }
    if constexpr (V == 4)
      *reinterpret_cast<float4*>(o) = make_float4(s[0], s[1], s[2], s[3]);
    else
      o[0] = s[0];
  }
}

}  // namespace sae
