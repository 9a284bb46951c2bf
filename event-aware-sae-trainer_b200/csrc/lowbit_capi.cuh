// C-ABI entry points of the 8-bit activation checkpoints and the 4-bit serving
// weights (included by capi.cu, whose error and launch helpers they use).
#pragma once

namespace {

bool known_dtype(int t) { return t == SAE_DTYPE_F32 || t == SAE_DTYPE_BF16; }
int64_t dtype_bytes(int t) { return t == SAE_DTYPE_F32 ? 4 : 2; }

// Rows of `ld` elements that 16-byte accesses may walk.
bool vec_rows(const void* p, int64_t ld, int dtype) {
  return aligned16(p) && ld * dtype_bytes(dtype) % 16 == 0;
}

int check_act8(const void* codes, const void* steps, int64_t n_tokens, int64_t n_cols) {
  if (codes == nullptr || steps == nullptr || n_tokens <= 0 || n_cols <= 0)
    return fail(SAE_ERR_INVALID_ARGUMENT, "act8: NULL checkpoint or empty shape");
  if (n_cols > (int64_t(1) << 31) - 64)
    return fail(SAE_ERR_UNSUPPORTED_SHAPE, "act8: n_cols must be below 2^31 - 64");
  if (!aligned16(codes) || !aligned16(steps))
    return fail(SAE_ERR_MISALIGNED, "act8: codes and steps must be 16-byte aligned");
  return SAE_OK;
}

// How a weight gradient runs. g is read as it is, or as bf16 parts in the
// workspace (fp32, or rows TMA cannot walk). The codes are expanded by the
// kernel, or beforehand into the workspace. Either copy bounds the tokens per
// launch. Few output tiles are made up for by splitting the tokens, so that
// every pair of SMs has work.
constexpr int64_t kWgradPartBytes = int64_t(1) << 30;
constexpr int64_t kWgradValueBytes = int64_t(128) << 20;
// Tiles of 256 gradient columns from which expanding beforehand pays. 8192 tokens x
// 1536 columns take (beforehand | by the kernel) 48 | 40 us for 256 gradient columns,
// 67 | 65 for 1536, 77 | 80 for 2304, 122 | 133 for 4096. With three parts of g the
// kernel's own expansion is hidden behind their products. (Where the codes of all
// tokens exceed kWgradValueBytes this is not so: 4096 tokens x 49152 columns by 2304
// take 2520 | 970 us, the output being read and written for each 1024 tokens.)
constexpr int64_t kWgradExpandTiles = 7;
struct Wgrad8Plan {
  int parts;              // 0: g itself
  int64_t tokens;         // per kernel launch
  int64_t rows, pitch;    // of a part
  int m_pairs, n_tiles, splits;
  bool expanded;          // codes as bf16 in the workspace
  size_t part_bytes, value_bytes, split_bytes;
};
Wgrad8Plan wgrad8_plan(int64_t n_tokens, int64_t n_cols, const void* g, int g_dtype,
                       int64_t n_grads, int64_t ldg) {
  Wgrad8Plan p{};
  p.parts = g_dtype == SAE_DTYPE_F32 ? 3 : vec_rows(g, ldg, g_dtype) ? 0 : 1;
  p.tokens = n_tokens;
  p.pitch = (n_grads + 7) / 8 * 8;
  p.m_pairs = static_cast<int>((n_cols + 255) / 256);
  p.n_tiles = static_cast<int>((n_grads + 255) / 256);
  p.expanded = p.parts < 3 && p.n_tiles >= kWgradExpandTiles;
  auto limit = [&](int64_t bytes, int64_t per_token) {
    const int64_t fit = bytes / per_token / 512 * 512;
    p.tokens = std::min(p.tokens, std::max<int64_t>(512, fit));
  };
  if (p.parts > 0) limit(kWgradPartBytes, p.parts * p.pitch * 2);
  if (p.expanded) {
    limit(kWgradValueBytes, act8_pitch(n_cols) * 2);
    p.value_bytes = align_up(static_cast<size_t>(p.tokens) * act8_pitch(n_cols) * 2, 256);
  }
  if (p.parts > 0) {
    p.rows = (p.tokens + WG_TOK - 1) / WG_TOK * WG_TOK;
    p.part_bytes = align_up(static_cast<size_t>(p.parts) * p.rows * p.pitch * 2, 256);
  }
  const int64_t tiles = static_cast<int64_t>(p.m_pairs) * p.n_tiles;
  const int64_t blocks = (p.tokens + WG_TOK - 1) / WG_TOK;
  const int least = p.parts == 3 ? 4 : 8;   // stages of a split, a whole number of accumulations
  const int64_t room = std::max(1, device_info().sm_count / 2) / tiles;
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min(room, blocks / least)));
  if (p.splits > 1)
    p.split_bytes = align_up(static_cast<size_t>(p.splits) * n_cols * n_grads * 4, 256);
  return p;
}

// Rows of bytes in boxes of WG_TOK rows, not swizzled.
int make_byte_tmap(CUtensorMap* m, const void* base, int64_t rows, int64_t pitch, uint32_t box_cols) {
  EncodeTiledFn fn = encode_tiled();
  if (fn == nullptr) return fail(SAE_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t gdim[2] = {static_cast<cuuint64_t>(pitch), static_cast<cuuint64_t>(rows)};
  const cuuint64_t gstride[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {box_cols, WG_TOK};
  const cuuint32_t estride[2] = {1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), gdim, gstride,
                        box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SAE_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
  return SAE_OK;
}

template <bool EXPAND, int PARTS>
int wgrad8_launch(const CUtensorMap& tm_g, const CUtensorMap& tm_codes, const CUtensorMap& tm_steps,
                  const Wgrad8Args& a, cudaStream_t stream) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return fail(SAE_ERR_CUDA, "no usable current device");
  static std::once_flag once[kMaxDevices];
  static int clusters_of[kMaxDevices] = {};
  std::call_once(once[dev], [dev] {
    const auto kernel = wgrad8_kernel<EXPAND, PARTS>;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(WgConfig<EXPAND, PARTS>::SMEM));
    // The register shares wait for one another: without the launch's registers
    // to divide, the kernel must not run.
    cudaFuncAttributes fa{};
    if (EXPAND && (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess || fa.numRegs < WG_REGS_LAUNCH))
      return;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(2 * std::max(1, device_info().sm_count / 2));
    lc.blockDim = dim3(WgConfig<EXPAND, PARTS>::THREADS);
    lc.dynamicSmemBytes = WgConfig<EXPAND, PARTS>::SMEM;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2;
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    lc.attrs = &at;
    lc.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &lc) != cudaSuccess) n = 0;
    cudaGetLastError();
    clusters_of[dev] = n;
  });
  if (clusters_of[dev] <= 0)
    return fail(SAE_ERR_CUDA, "weight_grad8: this device has no room for a pair of its CTAs");
  const int64_t total = static_cast<int64_t>(a.m_pairs) * a.n_tiles * a.splits;
  const int clusters = static_cast<int>(std::min<int64_t>(total, clusters_of[dev]));
  wgrad8_kernel<EXPAND, PARTS><<<2 * clusters, WgConfig<EXPAND, PARTS>::THREADS, WgConfig<EXPAND, PARTS>::SMEM, stream>>>(
      tm_g, tm_codes, tm_steps, a);
  return check_launch("wgrad8_kernel");
}

int check_sae4(const SaeB200Sae4* m) {
  if (m == nullptr) return fail(SAE_ERR_INVALID_ARGUMENT, "sae4: model is NULL");
  if (m->d_in <= 0 || m->n_features <= 0 || m->d_in % 2 != 0)
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4: d_in must be even and positive, n_features positive");
  if (m->d_in > SAE4_MAX_D_IN || m->n_features >= (int64_t(1) << 30))
    return fail(SAE_ERR_UNSUPPORTED_SHAPE, "sae4: at most %d columns and fewer than 2^30 features",
                SAE4_MAX_D_IN);
  if (m->group != 32 && m->group != 64 && m->group != 128)
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4: group must be 32, 64 or 128");
  if (m->enc == nullptr || m->dec == nullptr || m->dec_scale == nullptr || m->b_enc == nullptr || m->b_dec == nullptr || m->theta == nullptr)
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4: NULL weight, scale, bias or threshold");
  if (!aligned16(m->enc) || !aligned16(m->dec) || !aligned16(m->b_dec))
    return fail(SAE_ERR_MISALIGNED, "sae4: packed weights and b_dec must be 16-byte aligned");
  return SAE_OK;
}

int check_tokens(const void* x, int64_t n_tokens) {
  if (x == nullptr || n_tokens <= 0)
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4: input is NULL or n_tokens <= 0");
  if (n_tokens > kMaxGridY)
    return fail(SAE_ERR_UNSUPPORTED_SHAPE, "sae4: at most %d tokens per call", kMaxGridY);
  return SAE_OK;
}

S4Encoder s4_encoder(const SaeB200Sae4* m) {
  S4Encoder e;
  e.w = static_cast<const uint8_t*>(m->enc);
  e.b_enc = m->b_enc;
  e.b_dec = m->b_dec;
  e.theta = m->theta;
  e.d = m->d_in;
  e.F = m->n_features;
  e.kblocks = static_cast<int>(s4_kblocks(m->d_in));
  e.spb = m->group == 32 ? 2 : 1;
  return e;
}

int64_t s4_dec_pitch(int64_t d) { return (d / 2 + 15) / 16 * 16; }
int64_t s4_mask_pitch(int64_t F) { return (s4_tiles(F) + 1) / 2 * 2; }

// Scratch of the 4-bit calls: the active bits and counts, then what only some of
// them use, the centred tokens (encode, reconstruct) and the active values (reconstruct).
struct S4Workspace {
  size_t counts, tokens, vals, total;
};
S4Workspace s4_workspace(int64_t n_tokens, int64_t d, int64_t F) {
  S4Workspace w{};
  w.counts = align_up(static_cast<size_t>(n_tokens) * s4_mask_pitch(F) * 2, 256);
  w.tokens = w.counts + align_up(static_cast<size_t>(n_tokens) * 4, 256);
  w.vals = w.tokens + align_up(static_cast<size_t>(n_tokens) * s4_kblocks(d) * S4_COLS * 2, 256);
  w.total = w.vals + align_up(static_cast<size_t>(n_tokens) * F * 4, 256);
  return w;
}

// Launch whose set-up may overlap the end of the kernel before it in the stream
// (the kernel waits for that one itself), with clusters of cluster_z CTAs.
template <typename... Params, typename... Args>
int launch_after(const char* what, void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                 int cluster_z, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid;
  lc.blockDim = dim3(threads);
  lc.dynamicSmemBytes = smem;
  lc.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 1;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = cluster_z;
  lc.attrs = at;
  lc.numAttrs = cluster_z > 1 ? 2 : 1;
  const cudaError_t err = cudaLaunchKernelEx(&lc, kernel, args...);
  if (err != cudaSuccess) return fail(SAE_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
  return check_launch(what);
}

constexpr size_t kS4Smem = 224 * 1024, kS4LimbBytes = 160 * 1024;   // the latter at most
static_assert(8 * s4_limb_pitch(SAE4_MAX_D_IN / S4_COLS) <= kS4LimbBytes, "one pair of tokens fits");
size_t s4_limb_bytes(const S4Encoder& e, int nt) {
  return static_cast<size_t>(8) * nt * s4_limb_pitch(e.kblocks);
}

template <int NT, int SPB, typename XT>
int s4_encode_launch(const S4Encoder& e, const void* x, int64_t ldx, int n_tok, const S4Out& o,
                     cudaStream_t stream) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return fail(SAE_ERR_CUDA, "no usable current device");
  static std::once_flag once[kMaxDevices];
  std::call_once(once[dev], [] {
    cudaFuncSetAttribute(s4_encode_few_kernel<NT, SPB, XT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(kS4Smem));
  });
  // Warps per block: the SM's tiles in even rounds. Split a tile's columns
  // while that gives warps the SM has room for, and each a slot of its ring.
  constexpr int max_warps = S4_MAX_WARPS;
  const int sms = std::max(1, device_info().sm_count);
  const int64_t per_sm = (s4_tiles(e.F) + sms - 1) / sms;
  const int64_t rounds = (per_sm + max_warps - 1) / max_warps;
  const int at_once = static_cast<int>((per_sm + rounds - 1) / rounds);
  auto fixed_bytes = [&](int split) {   // limbs, and the sums to be joined
    return s4_limb_bytes(e, NT) + (split > 1 ? static_cast<size_t>(at_once) * split * NT * 512 : 0);
  };
  auto slot_bytes = [&](int split) { return static_cast<size_t>(at_once) * split * s4_slot_bytes(SPB); };
  int ks = 1;
  while (2 * ks * at_once <= max_warps && 2 * ks <= s4_kchunks(e.kblocks) &&
         fixed_bytes(2 * ks) + slot_bytes(2 * ks) <= kS4Smem)
    ks *= 2;
  const int warps = at_once * ks;
  const size_t fixed = fixed_bytes(ks), per_slot = slot_bytes(ks);
  static_assert(kS4LimbBytes + S4_MAX_WARPS * s4_slot_bytes(SPB) <= kS4Smem,
                "a tile that is not split has room for a slot a warp");
  const int slots = static_cast<int>(std::min<size_t>(S4_MAX_SLOTS, (kS4Smem - fixed) / per_slot));
  const int grid = static_cast<int>(std::min<int64_t>(sms, s4_tiles(e.F)));
  const int vec = vec_rows(x, ldx, sizeof(XT) == 4 ? SAE_DTYPE_F32 : SAE_DTYPE_BF16);
  s4_encode_few_kernel<NT, SPB, XT><<<grid, warps * 32, fixed + slots * per_slot, stream>>>(
      e, static_cast<const XT*>(x), ldx, vec, n_tok, ks, slots, o);
  return check_launch("s4_encode_few_kernel");
}

template <int SPB, typename XT>
int s4_encode_tokens(const S4Encoder& e, const void* x, int64_t ldx, int64_t n_tokens,
                     const S4Out& o, cudaStream_t stream) {
  for (int64_t t0 = 0; t0 < n_tokens;) {
    // two tokens' limbs at a time where four tokens' leave the weights no room
    const int nt = n_tokens - t0 > 2 && s4_limb_bytes(e, 2) <= kS4LimbBytes ? 2 : 1;
    const int n_tok = static_cast<int>(std::min<int64_t>(2 * nt, n_tokens - t0));
    S4Out part = o;
    part.out += t0 * o.ldo;
    if (part.mask != nullptr) part.mask += t0 * o.ldm;
    const XT* xt = static_cast<const XT*>(x) + t0 * ldx;
    SAE_TRY(nt == 2 ? (s4_encode_launch<2, SPB, XT>(e, xt, ldx, n_tok, part, stream))
                    : (s4_encode_launch<1, SPB, XT>(e, xt, ldx, n_tok, part, stream)));
    t0 += n_tok;
  }
  return SAE_OK;
}

// Tokens from which the tcgen05 kernel is the faster one. At 1536 x 49152, weights not
// in L2, it takes 22 us for 5 to 16 tokens and 4 for the centring, the integer kernel 14
// for one, 18 for four and as much again for each further four.
constexpr int64_t kS4ManyTokens = 5;

template <int SPB, int MODE>
int s4_encode_many(const S4Encoder& e, const bf16* xc, int64_t n_tokens, const S4Out& o,
                   cudaStream_t stream) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return fail(SAE_ERR_CUDA, "no usable current device");
  static std::once_flag once[kMaxDevices];
  static bool usable[kMaxDevices] = {};
  std::call_once(once[dev], [dev] {
    // The register shares wait for one another: without the launch's registers
    // to divide, the kernel must not run.
    cudaFuncAttributes fa{};
    usable[dev] = cudaFuncSetAttribute(s4_encode_many_kernel<SPB, MODE>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(s4m_smem(SPB))) == cudaSuccess &&
                  cudaFuncGetAttributes(&fa, s4_encode_many_kernel<SPB, MODE>) == cudaSuccess &&
                  fa.numRegs >= S4M_REGS_LAUNCH;
  });
  if (!usable[dev]) return fail(SAE_ERR_CUDA, "sae4_encode: kernel attributes refused");
  const int64_t pitch = static_cast<int64_t>(e.kblocks) * S4_COLS;
  // Token tiles of even size, a multiple of 16
  const int n_tiles = static_cast<int>((n_tokens + S4M_TOKENS - 1) / S4M_TOKENS);
  const int tile = static_cast<int>(((n_tokens + n_tiles - 1) / n_tiles + 15) / 16 * 16);
  CUtensorMap tm;
  SAE_TRY(make_tmap(&tm, xc, n_tokens, pitch, tile, S4_COLS));
  const int64_t units = (e.F + S4M_FEATURES - 1) / S4M_FEATURES * n_tiles;
  if (units > (int64_t(1) << 30)) return fail(SAE_ERR_UNSUPPORTED_SHAPE, "sae4_encode: too many tiles");
  const int grid = static_cast<int>(std::min<int64_t>(std::max(1, device_info().sm_count), units));
  return launch_after("s4_encode_many_kernel", s4_encode_many_kernel<SPB, MODE>, dim3(grid),
                      S4M_THREADS, s4m_smem(SPB), 1, stream, tm, e,
                      static_cast<int>(n_tokens), tile, n_tiles, o);
}

template <int SPB>
int s4_encode_spb(const S4Encoder& e, const void* x, int x_dtype, int64_t n_tokens, int64_t ldx,
                  bf16* xc, const S4Out& o, cudaStream_t stream) {
  if (n_tokens < kS4ManyTokens)
    return x_dtype == SAE_DTYPE_BF16 ? s4_encode_tokens<SPB, bf16>(e, x, ldx, n_tokens, o, stream)
                                     : s4_encode_tokens<SPB, float>(e, x, ldx, n_tokens, o, stream);
  const int64_t pitch = static_cast<int64_t>(e.kblocks) * S4_COLS;
  const int vec = vec_rows(x, ldx, x_dtype);
  const int grid = grid_for(n_tokens * (pitch / 8), 256);
  if (x_dtype == SAE_DTYPE_BF16)
    s4_center_kernel<bf16><<<grid, 256, 0, stream>>>(static_cast<const bf16*>(x), ldx, vec, e.b_dec,
                                                     n_tokens, e.d, pitch, xc);
  else
    s4_center_kernel<float><<<grid, 256, 0, stream>>>(static_cast<const float*>(x), ldx, vec,
                                                      e.b_dec, n_tokens, e.d, pitch, xc);
  SAE_TRY(check_launch("s4_center_kernel"));
  return o.mode == 0   ? s4_encode_many<SPB, 0>(e, xc, n_tokens, o, stream)
         : o.mode == 1 ? s4_encode_many<SPB, 1>(e, xc, n_tokens, o, stream)
                       : s4_encode_many<SPB, 2>(e, xc, n_tokens, o, stream);
}

int s4_encode_any(const SaeB200Sae4* m, const void* x, int x_dtype, int64_t n_tokens, int64_t ldx,
                  bf16* xc, const S4Out& o, cudaStream_t stream) {
  const S4Encoder e = s4_encoder(m);
  return e.spb == 2 ? s4_encode_spb<2>(e, x, x_dtype, n_tokens, ldx, xc, o, stream)
                    : s4_encode_spb<1>(e, x, x_dtype, n_tokens, ldx, xc, o, stream);
}

int s4_decode_any(const SaeB200Sae4* m, const float* vals, int64_t ldv, const uint16_t* mask,
                  int64_t n_tokens, float* x_hat, int32_t* counts, uint8_t* fired,
                  cudaStream_t stream) {
  S4Decoder e;
  e.codes = static_cast<const uint8_t*>(m->dec);
  e.scale = static_cast<const uint16_t*>(m->dec_scale);
  e.b_dec = m->b_dec;
  e.d = m->d_in;
  e.F = m->n_features;
  e.pitch = s4_dec_pitch(m->d_in);
  e.ng = static_cast<int>((m->d_in + m->group - 1) / m->group);
  e.group_shift = m->group == 32 ? 5 : m->group == 64 ? 6 : 7;
  S4DecodeIo o;
  o.vals = vals;
  o.ldv = ldv;
  o.mask = mask;
  o.ldm = s4_mask_pitch(m->n_features);
  o.x_hat = x_hat;
  o.counts = counts;
  o.fired = fired;
  const unsigned chunks = static_cast<unsigned>((m->d_in + S4_DEC_COLS - 1) / S4_DEC_COLS);
  const int sms = std::max(1, device_info().sm_count);
  // The clusters of all tokens in two rounds at most: 16 tokens at 1536 x 49152 are
  // encoded and decoded in 38 us, and 46 by the two kernels below.
  if (static_cast<int64_t>(chunks) * n_tokens * S4_DEC_PARTS <= 2 * S4_DEC_CTAS * sms)
    return launch_after("s4_decode_few_kernel", s4_decode_few_kernel,
                        dim3(chunks, static_cast<unsigned>(n_tokens), S4_DEC_PARTS),
                        S4_DEC_THREADS, 0, S4_DEC_PARTS, stream, e, o);
  SAE_TRY(launch_after("s4_decode_light_kernel", s4_decode_light_kernel,
                       dim3(chunks, static_cast<unsigned>(n_tokens)), S4_DEC_THREADS, 0, 1, stream,
                       e, o));
  return launch_after("s4_decode_heavy_kernel", s4_decode_heavy_kernel,
                      dim3(static_cast<unsigned>(sms), 1, S4_DEC_PARTS),
                      S4_DEC_THREADS, 0, S4_DEC_PARTS, stream, e, o, n_tokens,
                      static_cast<int>(chunks));
}

}  // namespace

extern "C" {

int64_t sae_b200_act8_step_pitch(int64_t n_cols) { return act8_step_pitch(n_cols); }

int sae_b200_act8_save(const void* x, int x_dtype, int64_t n_tokens, int64_t n_cols, int64_t ldx,
                       int8_t* codes, uint8_t* steps, void* stream_) {
  SAE_TRY(check_act8(codes, steps, n_tokens, n_cols));
  if (x == nullptr || ldx < n_cols)
    return fail(SAE_ERR_INVALID_ARGUMENT, "act8_save: x is NULL or ldx < n_cols");
  if (!known_dtype(x_dtype)) return fail(SAE_ERR_INVALID_ARGUMENT, "x_dtype must be F32 or BF16");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int vec = vec_rows(x, ldx, x_dtype);
  const int grid = grid_for(n_tokens * (act8_pitch(n_cols) / 8), 256);
  if (x_dtype == SAE_DTYPE_BF16)
    act8_save_kernel<bf16><<<grid, 256, 0, stream>>>(static_cast<const bf16*>(x), n_tokens, n_cols,
                                                     ldx, vec, codes, steps);
  else
    act8_save_kernel<float><<<grid, 256, 0, stream>>>(static_cast<const float*>(x), n_tokens,
                                                      n_cols, ldx, vec, codes, steps);
  return check_launch("act8_save_kernel");
}

int sae_b200_act8_load(const int8_t* codes, const uint8_t* steps, int64_t n_tokens, int64_t n_cols,
                       void* out, int out_dtype, int64_t ldo, void* stream_) {
  SAE_TRY(check_act8(codes, steps, n_tokens, n_cols));
  if (out == nullptr || ldo < n_cols)
    return fail(SAE_ERR_INVALID_ARGUMENT, "act8_load: out is NULL or ldo < n_cols");
  if (!known_dtype(out_dtype))
    return fail(SAE_ERR_INVALID_ARGUMENT, "out_dtype must be F32 or BF16");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int vec = vec_rows(out, ldo, out_dtype);
  const int grid = grid_for(n_tokens * (act8_pitch(n_cols) / 8), 256);
  if (out_dtype == SAE_DTYPE_BF16)
    act8_load_kernel<bf16><<<grid, 256, 0, stream>>>(codes, steps, n_tokens, n_cols,
                                                     static_cast<bf16*>(out), ldo, vec);
  else
    act8_load_kernel<float><<<grid, 256, 0, stream>>>(codes, steps, n_tokens, n_cols,
                                                      static_cast<float*>(out), ldo, vec);
  return check_launch("act8_load_kernel");
}

static int check_weight_grad8(int64_t n_tokens, int64_t n_cols, const void* g, int g_dtype,
                              int64_t n_grads, int64_t ldg) {
  if (g == nullptr || n_tokens <= 0 || n_cols <= 0 || n_grads <= 0 || ldg < n_grads ||
      !known_dtype(g_dtype))
    return fail(SAE_ERR_INVALID_ARGUMENT,
                "weight_grad8: NULL g, empty shape, short row pitch or unknown dtype");
  if (n_tokens > (int64_t(1) << 30) || n_cols > (int64_t(1) << 30) ||
      n_grads > (int64_t(1) << 30) ||
      ((n_cols + 255) / 256) * ((n_grads + 255) / 256) > (int64_t(1) << 30))
    return fail(SAE_ERR_UNSUPPORTED_SHAPE, "weight_grad8: a dimension above 2^30");
  return SAE_OK;
}

int sae_b200_weight_grad8_workspace_bytes(int64_t n_tokens, int64_t n_cols, const void* g,
                                          int g_dtype, int64_t n_grads, int64_t ldg,
                                          size_t* bytes_out) {
  if (bytes_out == nullptr) return fail(SAE_ERR_INVALID_ARGUMENT, "bytes_out is NULL");
  SAE_TRY(check_weight_grad8(n_tokens, n_cols, g, g_dtype, n_grads, ldg));
  const Wgrad8Plan p = wgrad8_plan(n_tokens, n_cols, g, g_dtype, n_grads, ldg);
  *bytes_out = p.part_bytes + p.value_bytes + p.split_bytes;
  return SAE_OK;
}

int sae_b200_weight_grad8(const int8_t* codes, const uint8_t* steps, int64_t n_tokens,
                          int64_t n_cols, const void* g, int g_dtype, int64_t n_grads, int64_t ldg,
                          int transposed, float beta, float* out, int64_t ldo, void* workspace,
                          size_t workspace_bytes, void* stream_) {
  SAE_TRY(check_act8(codes, steps, n_tokens, n_cols));
  SAE_TRY(check_weight_grad8(n_tokens, n_cols, g, g_dtype, n_grads, ldg));
  if (out == nullptr || ldo < (transposed ? n_grads : n_cols))
    return fail(SAE_ERR_INVALID_ARGUMENT, "weight_grad8: NULL out or row pitch below its row");
  const Wgrad8Plan p = wgrad8_plan(n_tokens, n_cols, g, g_dtype, n_grads, ldg);
  const size_t need = p.part_bytes + p.value_bytes + p.split_bytes;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(SAE_ERR_WORKSPACE_TOO_SMALL, "weight_grad8 needs %zu workspace bytes", need);
  if (!aligned16(workspace))
    return fail(SAE_ERR_MISALIGNED, "weight_grad8: workspace must be 16-byte aligned");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  bf16* part = static_cast<bf16*>(workspace);
  bf16* values = reinterpret_cast<bf16*>(static_cast<uint8_t*>(workspace) + p.part_bytes);
  float* split = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.part_bytes +
                                          p.value_bytes);
  const int64_t out_rows = transposed ? n_cols : n_grads, out_cols = transposed ? n_grads : n_cols;
  for (int64_t t0 = 0; t0 < n_tokens; t0 += p.tokens) {
    const int64_t n = std::min(p.tokens, n_tokens - t0);
    const float b = t0 == 0 ? beta : 1.f;
    CUtensorMap tm, tm_codes, tm_steps;
    const int64_t pitch = act8_pitch(n_cols), spitch = act8_step_pitch(n_cols);
    if (p.expanded) {
      SAE_TRY(sae_b200_act8_load(codes + t0 * pitch, steps + t0 * spitch, n, pitch, values,
                                 SAE_DTYPE_BF16, pitch, stream_));
      SAE_TRY(make_tmap(&tm_codes, values, n, pitch, WG_TOK, 64));
      tm_steps = tm_codes;
    } else {
      SAE_TRY(make_byte_tmap(&tm_codes, codes + t0 * pitch, n, pitch, 128));
      SAE_TRY(make_byte_tmap(&tm_steps, steps + t0 * spitch, n, spitch, 16));
    }
    if (p.parts > 0) {
      const int grid = grid_for(p.rows * (p.pitch / 8), 256);
      if (g_dtype == SAE_DTYPE_F32)
        wgrad8_parts_kernel<float><<<grid, 256, 0, stream>>>(
            static_cast<const float*>(g) + t0 * ldg, n, n_grads, ldg, p.rows, p.pitch, part);
      else
        wgrad8_parts_kernel<bf16><<<grid, 256, 0, stream>>>(
            static_cast<const bf16*>(g) + t0 * ldg, n, n_grads, ldg, p.rows, p.pitch, part);
      SAE_TRY(check_launch("wgrad8_parts_kernel"));
      SAE_TRY(make_tmap(&tm, part, p.parts * p.rows, p.pitch, WG_TOK, 64));
    } else {
      SAE_TRY(make_tmap(&tm, static_cast<const bf16*>(g) + t0 * ldg, n, n_grads, WG_TOK, 64,
                        CU_TENSOR_MAP_SWIZZLE_128B, ldg));
    }
    Wgrad8Args a{};
    a.n_cols = n_cols;
    a.n_grads = n_grads;
    a.transposed = transposed != 0;
    a.m_pairs = p.m_pairs;
    a.n_tiles = p.n_tiles;
    a.tok_blocks = static_cast<int>((n + WG_TOK - 1) / WG_TOK);
    a.part_rows = static_cast<int>(p.rows);
    a.splits = std::min(p.splits, a.tok_blocks);
    if (a.splits > 1) {
      a.out = split;
      a.ldo = out_cols;
      a.split_stride = out_rows * out_cols;
      a.beta = 0.f;
    } else {
      a.out = out;
      a.ldo = ldo;
      a.beta = b;
    }
    a.vec = transposed && vec_rows(a.out, a.ldo, SAE_DTYPE_F32) && a.split_stride % 4 == 0;
    SAE_TRY(p.parts == 3 ? (wgrad8_launch<true, 3>(tm, tm_codes, tm_steps, a, stream))
            : p.expanded ? (wgrad8_launch<false, 1>(tm, tm_codes, tm_steps, a, stream))
                         : (wgrad8_launch<true, 1>(tm, tm_codes, tm_steps, a, stream)));
    if (a.splits > 1) {
      if (out_cols % 4 == 0 && vec_rows(out, ldo, SAE_DTYPE_F32))
        wgrad8_join_kernel<4><<<grid_for(out_rows * out_cols / 4, 256), 256, 0, stream>>>(
            split, a.splits, out_rows, out_cols, b, out, ldo);
      else
        wgrad8_join_kernel<1><<<grid_for(out_rows * out_cols, 256), 256, 0, stream>>>(
            split, a.splits, out_rows, out_cols, b, out, ldo);
      SAE_TRY(check_launch("wgrad8_join_kernel"));
    }
  }
  return SAE_OK;
}

int64_t sae_b200_jumprelu8_pitch(int64_t n_features) { return jump8_pitch(n_features); }

// Tokens per block: fewer where the blocks would not fill the machine.
static int jump8_rows(int64_t n_tokens, int64_t n_features) {
  const int64_t cols = (n_features + 4 * J8_THREADS - 1) / (4 * J8_THREADS);
  int rows = J8_ROWS;
  while (rows > J8_AT_ONCE &&
         cols * ((n_tokens + rows - 1) / rows) < 8 * static_cast<int64_t>(std::max(1, device_info().sm_count)))
    rows /= 2;
  while ((n_tokens + rows - 1) / rows > kMaxGridY && rows < J8_ROWS) rows *= 2;
  return rows;
}

static int check_jumprelu8(const void* codes, const float* log_threshold, int64_t n_tokens,
                           int64_t n_features, float eps) {
  if (codes == nullptr || log_threshold == nullptr || n_tokens <= 0 || n_features <= 0 ||
      !(eps > 0.f) || std::isinf(eps))
    return fail(SAE_ERR_INVALID_ARGUMENT, "invalid jumprelu8 arguments");
  if ((n_tokens + J8_ROWS - 1) / J8_ROWS > kMaxGridY || n_features > (int64_t(1) << 31) - 64)
    return fail(SAE_ERR_UNSUPPORTED_SHAPE, "jumprelu8 takes at most %lld tokens",
                static_cast<long long>(kMaxGridY) * J8_ROWS);
  if (!aligned16(codes)) return fail(SAE_ERR_MISALIGNED, "jumprelu8: codes must be 16-byte aligned");
  return SAE_OK;
}

int sae_b200_jumprelu8_forward(const void* pre, int pre_dtype, const float* log_threshold,
                               int64_t n_tokens, int64_t n_features, float eps, float* feat_out,
                               float* gate_out, int8_t* codes_out, void* stream_) {
  SAE_TRY(check_jumprelu8(codes_out, log_threshold, n_tokens, n_features, eps));
  if (pre == nullptr || feat_out == nullptr || gate_out == nullptr || !known_dtype(pre_dtype))
    return fail(SAE_ERR_INVALID_ARGUMENT, "jumprelu8_forward: NULL tensor or unknown dtype");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const bool vec = n_features % 4 == 0 && aligned16(pre) && aligned16(feat_out) && aligned16(gate_out);
  const int64_t per = static_cast<int64_t>(J8_THREADS) * (vec ? 4 : 1);
  const int rows = jump8_rows(n_tokens, n_features);
  const dim3 grid(static_cast<unsigned>((n_features + per - 1) / per),
                  static_cast<unsigned>((n_tokens + rows - 1) / rows));
  const float per_step = J8_BAND / eps;
#define SAE_J8_FWD(PT, V)                                                                       \
  jump8_forward_kernel<PT, V><<<grid, J8_THREADS, 0, stream>>>(                                 \
      static_cast<const PT*>(pre), log_threshold, n_tokens, n_features, rows, eps, per_step, feat_out, \
      gate_out, codes_out)
  if (pre_dtype == SAE_DTYPE_BF16) {
    if (vec) SAE_J8_FWD(bf16, 4); else SAE_J8_FWD(bf16, 1);
  } else {
    if (vec) SAE_J8_FWD(float, 4); else SAE_J8_FWD(float, 1);
  }
#undef SAE_J8_FWD
  return check_launch("jump8_forward_kernel");
}

int sae_b200_jumprelu8_workspace_bytes(int64_t n_tokens, int64_t n_features, size_t* bytes_out) {
  if (bytes_out == nullptr || n_tokens <= 0 || n_features <= 0)
    return fail(SAE_ERR_INVALID_ARGUMENT, "jumprelu8: invalid shape");
  const int rows = jump8_rows(n_tokens, n_features);
  *bytes_out = static_cast<size_t>((n_tokens + rows - 1) / rows) * n_features * 4;
  return SAE_OK;
}

int sae_b200_jumprelu8_backward(const int8_t* codes, const float* log_threshold, int64_t n_tokens,
                                int64_t n_features, float eps, const float* grad_feat,
                                const float* grad_gate, int64_t gate_stride_t,
                                int64_t gate_stride_f, void* grad_pre_out, int grad_pre_dtype,
                                float* grad_log_threshold_out, void* workspace,
                                size_t workspace_bytes, void* stream_) {
  SAE_TRY(check_jumprelu8(codes, log_threshold, n_tokens, n_features, eps));
  if (grad_log_threshold_out == nullptr || !known_dtype(grad_pre_dtype) || gate_stride_t < 0 ||
      gate_stride_f < 0)
    return fail(SAE_ERR_INVALID_ARGUMENT,
                "jumprelu8_backward: NULL output, unknown dtype or negative stride");
  size_t need = 0;
  SAE_TRY(sae_b200_jumprelu8_workspace_bytes(n_tokens, n_features, &need));
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SAE_ERR_WORKSPACE_TOO_SMALL, "jumprelu8_backward needs %zu workspace bytes", need);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  float* part = static_cast<float*>(workspace);
  const bool vec = n_features % 4 == 0 && aligned16(grad_feat) && aligned16(grad_pre_out);
  const int64_t per = static_cast<int64_t>(J8_THREADS) * (vec ? 4 : 1);
  const int rows = jump8_rows(n_tokens, n_features);
  const int slabs = static_cast<int>((n_tokens + rows - 1) / rows);
  const dim3 grid(static_cast<unsigned>((n_features + per - 1) / per), static_cast<unsigned>(slabs));
  const float eps_step = eps / J8_BAND;
  const int gate = grad_gate == nullptr ? 0 : gate_stride_t == 0 && gate_stride_f == 0 ? 1 : 2;
#define SAE_J8_BWD(PT, V, GATE)                                                              \
  jump8_backward_kernel<PT, V, GATE><<<grid, J8_THREADS, 0, stream>>>(                       \
      codes, log_threshold, static_cast<int>(n_tokens), n_features, rows, eps_step, grad_feat, \
      grad_gate, gate_stride_t, gate_stride_f, static_cast<PT*>(grad_pre_out), part)
#define SAE_J8_BWD_GATE(PT, V)            \
  do {                                    \
    if (gate == 0) SAE_J8_BWD(PT, V, 0);  \
    else if (gate == 1) SAE_J8_BWD(PT, V, 1); \
    else SAE_J8_BWD(PT, V, 2);            \
  } while (0)
  if (grad_pre_dtype == SAE_DTYPE_BF16) {
    if (vec) SAE_J8_BWD_GATE(bf16, 4); else SAE_J8_BWD_GATE(bf16, 1);
  } else {
    if (vec) SAE_J8_BWD_GATE(float, 4); else SAE_J8_BWD_GATE(float, 1);
  }
#undef SAE_J8_BWD_GATE
#undef SAE_J8_BWD
  SAE_TRY(check_launch("jump8_backward_kernel"));
  jump8_final_kernel<<<static_cast<unsigned>((n_features + 31) / 32), 256, 0, stream>>>(
      part, slabs, log_threshold, n_features, eps, grad_log_threshold_out);
  return check_launch("jump8_final_kernel");
}

int sae_b200_sae4_quantize(const float* W, int64_t n_features, int64_t d_in, int group,
                           uint8_t* codes, void* scales, void* stream_) {
  if (W == nullptr || codes == nullptr || scales == nullptr || n_features <= 0 || d_in <= 0 ||
      d_in % 2 != 0 || (group != 32 && group != 64 && group != 128))
    return fail(SAE_ERR_INVALID_ARGUMENT,
                "sae4_quantize: NULL tensor, odd or empty shape, or group not 32, 64 or 128");
  const int64_t n = n_features * ((d_in + group - 1) / group);
  s4_quantize_kernel<<<grid_for(n, 256), 256, 0, static_cast<cudaStream_t>(stream_)>>>(
      W, n_features, d_in, group, codes, static_cast<bf16*>(scales));
  return check_launch("s4_quantize_kernel");
}

int sae_b200_sae4_packed_bytes(int64_t n_features, int64_t d_in, int group, size_t* bytes_out) {
  if (bytes_out == nullptr || n_features <= 0 || d_in <= 0 ||
      (group != 32 && group != 64 && group != 128))
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4_packed_bytes: invalid shape or group");
  *bytes_out = static_cast<size_t>(s4_packed_bytes(n_features, d_in, group == 32 ? 2 : 1));
  return SAE_OK;
}

int sae_b200_sae4_pack(const uint8_t* codes, const void* scales, int64_t n_features, int64_t d_in,
                       int group, void* packed, void* stream_) {
  size_t bytes = 0;
  SAE_TRY(sae_b200_sae4_packed_bytes(n_features, d_in, group, &bytes));
  if (codes == nullptr || scales == nullptr || packed == nullptr || d_in % 2 != 0)
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4_pack: NULL tensor or odd d_in");
  if (!aligned16(packed))
    return fail(SAE_ERR_MISALIGNED, "sae4_pack: output must be 16-byte aligned");
  s4_pack_kernel<<<grid_for(static_cast<int64_t>(bytes / 4), 256), 256, 0,
                   static_cast<cudaStream_t>(stream_)>>>(
      codes, static_cast<const uint16_t*>(scales), n_features, d_in, group, group == 32 ? 2 : 1,
      static_cast<uint32_t*>(packed));
  return check_launch("s4_pack_kernel");
}

int sae_b200_sae4_workspace_bytes(int64_t n_tokens, int64_t d_in, int64_t n_features,
                                  size_t* encode_out, size_t* decode_out,
                                  size_t* reconstruct_out) {
  if (n_tokens <= 0 || d_in <= 0 || n_features <= 0)
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4_workspace_bytes: invalid shape");
  const S4Workspace w = s4_workspace(n_tokens, d_in, n_features);
  if (encode_out != nullptr) *encode_out = n_tokens < kS4ManyTokens ? 0 : w.vals - w.tokens;
  if (decode_out != nullptr) *decode_out = w.tokens;
  if (reconstruct_out != nullptr) *reconstruct_out = w.total;
  return SAE_OK;
}

static int check_sae4_workspace(const char* what, const void* workspace, size_t bytes, size_t need) {
  if (need > 0 && (workspace == nullptr || bytes < need))
    return fail(SAE_ERR_WORKSPACE_TOO_SMALL, "%s needs %zu workspace bytes", what, need);
  if (!aligned16(workspace))
    return fail(SAE_ERR_MISALIGNED, "%s: workspace must be 16-byte aligned", what);
  return SAE_OK;
}

int sae_b200_sae4_encode(const SaeB200Sae4* model, const void* x, int x_dtype, int64_t n_tokens,
                         int64_t ldx, int gated, float* out, int64_t ldo, void* workspace,
                         size_t workspace_bytes, void* stream_) {
  SAE_TRY(check_sae4(model));
  SAE_TRY(check_tokens(x, n_tokens));
  if (out == nullptr || ldx < model->d_in || ldo < model->n_features || !known_dtype(x_dtype))
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4_encode: NULL output, short row pitch or unknown dtype");
  if (ldo >= (int64_t(1) << 30))   // row offsets of the stores are 32-bit
    return fail(SAE_ERR_UNSUPPORTED_SHAPE, "sae4_encode: ldo must be below 2^30");
  size_t need = 0;
  SAE_TRY(sae_b200_sae4_workspace_bytes(n_tokens, model->d_in, model->n_features, &need, nullptr, nullptr));
  SAE_TRY(check_sae4_workspace("sae4_encode", workspace, workspace_bytes, need));
  S4Out o{};
  o.out = out;
  o.ldo = ldo;
  o.mode = gated ? 1 : 0;
  return s4_encode_any(model, x, x_dtype, n_tokens, ldx, static_cast<bf16*>(workspace), o,
                       static_cast<cudaStream_t>(stream_));
}

int sae_b200_sae4_decode(const SaeB200Sae4* model, const float* acts, int64_t n_tokens,
                         int64_t lda, float* x_hat_out, void* workspace, size_t workspace_bytes,
                         void* stream_) {
  SAE_TRY(check_sae4(model));
  SAE_TRY(check_tokens(acts, n_tokens));
  if (x_hat_out == nullptr || lda < model->n_features)
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4_decode: NULL output or short row pitch");
  size_t need = 0;
  SAE_TRY(sae_b200_sae4_workspace_bytes(n_tokens, model->d_in, model->n_features, nullptr, &need, nullptr));
  SAE_TRY(check_sae4_workspace("sae4_decode", workspace, workspace_bytes, need));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  uint16_t* mask = static_cast<uint16_t*>(workspace);
  const int64_t ldm = s4_mask_pitch(model->n_features);
  const int64_t mask_warps = n_tokens * ((ldm / 2 + S4_MASK_WORDS - 1) / S4_MASK_WORDS);
  s4_mask_kernel<<<grid_for(mask_warps * 32, 256), 256, 0, stream>>>(
      acts, lda, n_tokens, model->n_features, mask, ldm);
  SAE_TRY(check_launch("s4_mask_kernel"));
  const S4Workspace L = s4_workspace(n_tokens, model->d_in, model->n_features);
  int32_t* counts = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + L.counts);
  return s4_decode_any(model, acts, lda, mask, n_tokens, x_hat_out, counts, nullptr, stream);
}

int sae_b200_sae4_reconstruct(const SaeB200Sae4* model, const void* x, int x_dtype,
                              int64_t n_tokens, int64_t ldx, float* x_hat_out,
                              int32_t* active_counts_out, uint8_t* fired, void* workspace,
                              size_t workspace_bytes, void* stream_) {
  SAE_TRY(check_sae4(model));
  SAE_TRY(check_tokens(x, n_tokens));
  if (x_hat_out == nullptr || ldx < model->d_in || !known_dtype(x_dtype))
    return fail(SAE_ERR_INVALID_ARGUMENT, "sae4_reconstruct: NULL output, short row pitch or unknown dtype");
  const S4Workspace L = s4_workspace(n_tokens, model->d_in, model->n_features);
  SAE_TRY(check_sae4_workspace("sae4_reconstruct", workspace, workspace_bytes, L.total));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  S4Out o{};
  o.out = reinterpret_cast<float*>(ws + L.vals);
  o.ldo = model->n_features;
  o.mask = reinterpret_cast<uint16_t*>(ws);
  o.ldm = s4_mask_pitch(model->n_features);
  o.mode = 2;
  SAE_TRY(s4_encode_any(model, x, x_dtype, n_tokens, ldx, reinterpret_cast<bf16*>(ws + L.tokens), o,
                        stream));
  int32_t* counts = active_counts_out != nullptr ? active_counts_out
                                                 : reinterpret_cast<int32_t*>(ws + L.counts);
  return s4_decode_any(model, o.out, o.ldo, o.mask, n_tokens, x_hat_out, counts, fired, stream);
}

}  // extern "C"
