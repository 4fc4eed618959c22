// C entry points of the mixture-of-experts operators and of the saved pre-activations.
// Included at the end of swiglu_abi.cu (one translation unit; uses its validation helpers).
#pragma once

namespace {

using ExpertKernelFn = void (*)(const sgl::ExpertMaps, const sgl::ExpertParams);

struct ExpertVariant {
  ExpertKernelFn fn;
  int (*max_stages)(int groups, int a_rows, int acc_cols);
  int (*smem_bytes)(int groups, int a_rows, int acc_cols, int stages);
};

template <int F, int G, int BK>
ExpertVariant make_expert_variant() {
  using T = sgl::ExpertTraits<F, G, BK>;
  ExpertVariant v;
  v.fn = sgl::experts_kernel<F, G, BK>;
  v.max_stages = T::max_stages;
  v.smem_bytes = T::smem_bytes;
  return v;
}

constexpr int kExpertVariants = sgl::EXP_FORMS * 2;   // form * 2 + (cta_group - 1)
// Depth of a ring stage.  The weight gradient sums over a group's rows, often a few hundred: its
// operands come in steps of 64 (126 experts, about 48 rows each: 272 us instead of 280).
constexpr int kExpertBlockK = 128;
constexpr int kWgradBlockK = 64;

template <int F>
void fill_expert_form(ExpertVariant* table) {
  constexpr int kBlockK = F == sgl::EXP_WGRAD ? kWgradBlockK : kExpertBlockK;
  table[F * 2] = make_expert_variant<F, 1, kBlockK>();
  table[F * 2 + 1] = make_expert_variant<F, 2, kBlockK>();
}

const ExpertVariant& expert_variant(int form, int cta_group) {
  struct Table {
    ExpertVariant v[kExpertVariants];
    Table() {
      fill_expert_form<sgl::EXP_SWIGLU>(v);
      fill_expert_form<sgl::EXP_SAVE16>(v);
      fill_expert_form<sgl::EXP_SAVE8>(v);
      fill_expert_form<sgl::EXP_GEMM>(v);
      fill_expert_form<sgl::EXP_GEMM32>(v);
      fill_expert_form<sgl::EXP_GRAD16>(v);
      fill_expert_form<sgl::EXP_GRAD8>(v);
      fill_expert_form<sgl::EXP_WGRAD>(v);
    }
  };
  static const Table table;
  return table.v[form * 2 + cta_group - 1];
}

struct ExpertDevice {
  bool ready[kExpertVariants] = {};
  int clusters2[kExpertVariants] = {};
  bool order_ready = false;
};
std::map<int, ExpertDevice> g_expert_devices;   // by device ordinal, under g_dev_mutex

int current_device(int* dev) {
  cudaError_t e = cudaGetDevice(dev);
  return e == cudaSuccess ? SGL_OK : fail_cuda(e, "cudaGetDevice");
}

// First use of a variant on a device: its shared-memory limit, and how many CTA pairs fit.
int prepare_expert_variant(int form, int cta_group, const DeviceInfo* info, int* clusters) {
  int dev = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  std::lock_guard<std::mutex> lock(g_dev_mutex);
  ExpertDevice& d = g_expert_devices[dev];
  const int vi = form * 2 + cta_group - 1;
  const ExpertVariant& v = expert_variant(form, cta_group);
  if (!d.ready[vi]) {
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(v.fn),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return fail_cuda(e, "cudaFuncSetAttribute(max dynamic smem)");
    int n = info->sm_count / cta_group;
    if (cta_group == 2) {
      cudaLaunchConfig_t qc = {};
      qc.gridDim = dim3(static_cast<unsigned>(info->sm_count / 2 * 2), 1, 1);
      qc.blockDim = dim3(sgl::kExpThreads, 1, 1);
      qc.dynamicSmemBytes = 227 * 1024;
      cudaLaunchAttribute qa[1];
      qa[0].id = cudaLaunchAttributeClusterDimension;
      qa[0].val.clusterDim.x = 2;
      qa[0].val.clusterDim.y = 1;
      qa[0].val.clusterDim.z = 1;
      qc.attrs = qa;
      qc.numAttrs = 1;
      int q = 0;
      e = cudaOccupancyMaxActiveClusters(&q, reinterpret_cast<const void*>(v.fn), &qc);
      if (e == cudaSuccess && q > 0) {
        if (q < n) n = q;
      } else {
        cudaGetLastError();
      }
    }
    d.clusters2[vi] = n > 0 ? n : 1;
    d.ready[vi] = true;
  }
  *clusters = d.clusters2[vi];
  return SGL_OK;
}

// Tensor map over [outer][rows][cols] elements (bf16 unless said); rank 2 when outer == 0.
int make_expert_map(CUtensorMap* out, const void* base, int64_t cols, int64_t rows, int64_t outer,
                    int64_t ld_bytes, int64_t outer_bytes, int box_cols, int box_rows,
                    const char* name,
                    CUtensorMapDataType type = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                    CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B,
                    CUtensorMapL2promotion promo = CU_TENSOR_MAP_L2_PROMOTION_L2_256B) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail(SGL_ERR_NO_DRIVER, "cuTensorMapEncodeTiled is not available");
  const cuuint32_t rank = outer > 0 ? 3 : 2;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows),
                        static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld_bytes), static_cast<cuuint64_t>(outer_bytes)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(out, type, rank, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promo, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(SGL_ERR_TENSOR_MAP,
                "cuTensorMapEncodeTiled(%s) failed with CUresult %d (cols=%lld rows=%lld outer=%lld "
                "pitch=%lld)",
                name, static_cast<int>(r), static_cast<long long>(cols),
                static_cast<long long>(rows), static_cast<long long>(outer),
                static_cast<long long>(ld_bytes));
  return SGL_OK;
}

int validate_groups(int64_t R, int64_t E, const void* offsets, bool need_offsets) {
  if (R < 1 || R > 0x7fffff00ll)
    return fail(SGL_ERR_BAD_SHAPE, "R=%lld rows must be in [1, 2^31)", static_cast<long long>(R));
  if (E < 1 || E > sgl::kExpMaxGroups)
    return fail(SGL_ERR_BAD_SHAPE, "E=%lld experts outside [1, %d]", static_cast<long long>(E),
                sgl::kExpMaxGroups);
  if (!offsets && need_offsets) return fail(SGL_ERR_NULL_POINTER, "offsets is NULL");
  if (reinterpret_cast<uintptr_t>(offsets) & 3u)
    return fail(SGL_ERR_MISALIGNED, "offsets is not 4-byte aligned");
  return SGL_OK;
}

// Distance of two experts' matrices of `rows` rows.  Operands may share their last row's elements
// with the next matrix; results (`cols` columns) may not share an element.
int validate_expert_stride(int64_t stride, int64_t rows, int64_t ld, int64_t E, const char* name,
                           int64_t cols = 0) {
  if (E == 1) return SGL_OK;
  if (stride % 8 != 0 || stride < (rows - 1) * ld + cols)
    return fail(SGL_ERR_BAD_STRIDE,
                "%s=%lld: an expert's matrix must be a multiple of 8 elements and at least its "
                "rows apart from the next one's",
                name, static_cast<long long>(stride));
  return SGL_OK;
}

// One launch of experts_kernel.
struct ExpertLaunch {
  int form = sgl::EXP_GEMM;
  const char* name = "";
  const void* a = nullptr;
  const void* b = nullptr;
  void* out = nullptr;
  const int* offsets = nullptr;
  int64_t R = 0, N = 0, K = 0, M = 0, E = 0;
  int64_t lda = 0, ldb = 0, b_stride = 0, ld_out = 0, out_stride = 0;
  int b_transposed = 0;
  void* pre = nullptr;       // EXP_SAVE*: pre-activations (see preact_layout); EXP_GRAD*: their
                             // gradients, [R, 2N] bf16
  int64_t ld_pre = 0;        // EXP_GRAD*: row pitch of the gradients, elements
  const void* saved = nullptr;   // EXP_GRAD*: saved pre-activations
  void* scales = nullptr;    // 8-bit forms
  const int* slots = nullptr;    // EXP_GRAD*: the routing weight of each row, or NULL (ones)
  const void* weights = nullptr;
  int64_t ld_w = 0, k = 1;
  int w_bf16 = 0;
  int splits = 1;            // EXP_GEMM32: ranges of K, each with its own slot of the result
  int64_t k_per_split = 0;
};

// Byte layout of saved pre-activations: rows of [up | gate], each half padded to whole blocks.
struct PreactLayout {
  int64_t pitch, gate_off;             // bytes
  int64_t scale_pitch, gate_scale_off; // bytes (8-bit form)
};
PreactLayout preact_layout(int bits, int64_t N) {
  PreactLayout l;
  const int64_t half = (N + 31) / 32 * 32 * (bits / 8);
  l.pitch = 2 * half;
  l.gate_off = half;
  l.gate_scale_off = bits == 8 ? (N + 63) / 64 * 2 : 0;
  l.scale_pitch = 2 * l.gate_scale_off;
  return l;
}

int launch_experts(const ExpertLaunch& s, void* stream) {
  DeviceInfo* info = nullptr;
  int rc = check_device(&info);
  if (rc) return rc;
  const bool wgrad = s.form == sgl::EXP_WGRAD;
  const bool save = s.form == sgl::EXP_SAVE16 || s.form == sgl::EXP_SAVE8;
  const bool grad = s.form == sgl::EXP_GRAD16 || s.form == sgl::EXP_GRAD8;
  const bool swiglu = s.form == sgl::EXP_SWIGLU || save;

  // CTA pairs (256-row tiles) once the groups have that many rows on average, single CTAs (128
  // rows) below: a pair fetches each weight for twice the rows, but a group's last tile is half
  // empty on average.  64 experts, 2048 x 1024, gate/up stage: 384 rows each 206 us in pairs and
  // 225 in single CTAs, 192 rows 147 and 142, 64 rows 110 and 94.
  int cta_group = 1;
  if (wgrad) {
    cta_group = s.M > sgl::kBlockM ? 2 : 1;
  } else if (s.R / s.E >= 256) {
    cta_group = 2;
  }
  int clusters = 0;
  if ((rc = prepare_expert_variant(s.form, cta_group, info, &clusters))) return rc;
  const ExpertVariant& v = expert_variant(s.form, cta_group);

  const int tile_rows = sgl::kBlockM * cta_group;
  // tile rows there can be at most: every group may end in a partly filled one
  const int64_t groups_used = wgrad ? s.E : (s.E < s.R ? s.E : s.R);
  const int64_t max_tiles_m = wgrad ? (s.M + tile_rows - 1) / tile_rows * s.E
                                    : s.R / tile_rows + groups_used;
  // Single-CTA tiles: half as wide while there are fewer than two for each SM, four where the
  // groups are short and the weight's stream is all there is to balance (64 tokens x 8 of 64
  // experts, 1024 -> 2048: 50 us at 256 columns, 46 at 128).  (64 columns are
  // not worth it: a k-block takes 0.5 us at 64 and at 128 columns.  8 tokens x 2 of 8 experts,
  // 14336 -> 4096: 255 us at 64 columns, 142 at 128.)
  int acc_cols = sgl::kAccCols;
  const int min_cols = 128;
  if (cta_group == 1 && !wgrad) {
    const int64_t cols = swiglu ? acc_cols / 2 : acc_cols;
    if (max_tiles_m * ((s.N + cols - 1) / cols) * s.splits <
        (s.R / s.E < 64 ? 4 : 2) * info->sm_count)
      acc_cols = min_cols;
  }
  int a_rows = sgl::kBlockM;
  if (cta_group == 1 && !wgrad && s.R <= 32) a_rows = static_cast<int>((s.R + 15) / 16 * 16);
  int stages = v.max_stages(static_cast<int>(s.E), a_rows, acc_cols);
  while (stages < 2 && acc_cols > min_cols) {   // several hundred groups: their table needs room
    acc_cols /= 2;
    stages = v.max_stages(static_cast<int>(s.E), a_rows, acc_cols);
  }
  const int tile_cols = swiglu ? acc_cols / 2 : acc_cols;
  const int64_t tiles_n = (s.N + tile_cols - 1) / tile_cols;
  const int64_t units = max_tiles_m * tiles_n * s.splits;
  if (units > 0x7fffffffll) return fail(SGL_ERR_BAD_SHAPE, "too many tiles");
  const int smem = v.smem_bytes(static_cast<int>(s.E), a_rows, acc_cols, stages);

  sgl::ExpertMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  const int bits = s.form == sgl::EXP_SAVE8 || s.form == sgl::EXP_GRAD8 ? 8 : 16;
  const PreactLayout pl = preact_layout(bits, s.N);
  constexpr CUtensorMapDataType kBf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  constexpr CUtensorMapSwizzle kSw128 = CU_TENSOR_MAP_SWIZZLE_128B;
  constexpr CUtensorMapL2promotion kNoPromo = CU_TENSOR_MAP_L2_PROMOTION_NONE;
  // pitch of `pre` and distance of its halves, bytes
  const int64_t pre_pitch = grad ? s.ld_pre * 2 : pl.pitch;
  const int64_t pre_gate = grad ? s.N * 2 : pl.gate_off;
  if (wgrad) {
    if ((rc = make_expert_map(&maps.a, s.a, s.M, s.R, 0, s.lda * 2, 0, 64, kWgradBlockK, "a")) ||
        (rc = make_expert_map(&maps.b, s.b, s.N, s.R, 0, s.ldb * 2, 0, 64, kWgradBlockK, "g")) ||
        (rc = make_expert_map(&maps.out, s.out, s.N, s.M, s.E, s.ld_out * 2, s.out_stride * 2, 64,
                              32, "out", kBf16, kSw128, kNoPromo)))
      return rc;
  } else {
    const int64_t b_cols = s.b_transposed ? s.K : (swiglu ? 2 * s.N : s.N);
    const int64_t b_rows = s.b_transposed ? s.N : s.K;
    if ((rc = make_expert_map(&maps.a, s.a, s.K, s.R, 0, s.lda * 2, 0, 64, sgl::kBlockM, "a")) ||
        (rc = make_expert_map(&maps.a16, s.a, s.K, s.R, 0, s.lda * 2, 0, 64, 16, "a")) ||
        (rc = make_expert_map(&maps.b, s.b, b_cols, b_rows, s.E, s.ldb * 2, s.b_stride * 2, 64,
                              s.b_transposed ? 64 : kExpertBlockK, "b")))
      return rc;
    // boxes of the results, as the epilogue stages them: 32 rows x 128 bytes (8-bit codes: x 64);
    // the forms with three results store without maps
    const bool f32 = s.form == sgl::EXP_GEMM32;
    if (!grad && s.form != sgl::EXP_SAVE16) {
      rc = make_expert_map(&maps.out, s.out, s.N, s.R, f32 ? s.splits : 0, s.ld_out * (f32 ? 4 : 2),
                           f32 ? s.R * s.ld_out * 4 : 0, f32 ? 32 : 64, 32, "out",
                           f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : kBf16, kSw128, kNoPromo);
      if (rc) return rc;
    }
    if (s.form == sgl::EXP_SAVE8) {
      constexpr CUtensorMapDataType kU8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
      uint8_t* pre = static_cast<uint8_t*>(s.pre);
      if ((rc = make_expert_map(&maps.up, pre, s.N, s.R, 0, pre_pitch, 0, 64, 32, "up", kU8,
                                CU_TENSOR_MAP_SWIZZLE_64B, kNoPromo)) ||
          (rc = make_expert_map(&maps.gate, pre + pre_gate, s.N, s.R, 0, pre_pitch, 0, 64, 32,
                                "gate", kU8, CU_TENSOR_MAP_SWIZZLE_64B, kNoPromo)))
        return rc;
    }
  }

  sgl::ExpertParams p;
  std::memset(&p, 0, sizeof(p));
  p.offsets = s.offsets;
  p.groups = static_cast<int>(s.E);
  p.R = static_cast<int>(s.R);
  p.N = static_cast<int>(s.N);
  p.K = static_cast<int>(s.K);
  p.M = static_cast<int>(s.M);
  p.tiles_n = static_cast<int>(tiles_n);
  // (8192 tokens x 2 of 8 experts, 4096 x 14336: 4.73 ms, with 8 tile rows together 4.80, with 32
  // 4.82, with 4 5.20; no difference with small groups)
  p.group_m = 16;
  p.stages = stages;
  p.acc_cols = acc_cols;
  p.splits = s.splits;
  p.k_per_split = static_cast<int>(s.k_per_split);
  p.slot_stride = s.R * s.ld_out;
  p.a_rows = a_rows;
  p.b_kmajor = s.b_transposed;
  p.out = static_cast<__nv_bfloat16*>(s.out);
  p.ld_out = s.ld_out;
  p.pre = static_cast<uint8_t*>(s.pre);
  p.ld_pre = pre_pitch;
  p.gate_off = pre_gate;
  p.scales = static_cast<uint8_t*>(s.scales);
  p.ld_scales = pl.scale_pitch;
  p.gate_scale_off = pl.gate_scale_off;
  p.saved = static_cast<const uint8_t*>(s.saved);
  p.ld_saved = pl.pitch;
  p.saved_gate_off = pl.gate_off;
  p.slots = s.slots;
  p.weights = s.weights;
  p.ld_w = s.ld_w;
  p.num_slots = s.R;
  p.k = static_cast<int>(s.k);
  p.w_bf16 = s.w_bf16;
  // operands evict-last, results evict-first, as for the dense stage
  p.l2_hints = 2 | (2 << 2) | (1 << 4);
  p.wait_limit_ns = g_wait_limit_ns.load();

  const int64_t grid = units < clusters ? units : clusters;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(static_cast<unsigned>(grid * cta_group), 1, 1);
  lc.blockDim = dim3(sgl::kExpThreads, 1, 1);
  lc.dynamicSmemBytes = static_cast<size_t>(smem);
  lc.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = static_cast<unsigned>(cta_group);
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  lc.attrs = attrs;
  lc.numAttrs = cta_group == 2 ? 2 : 1;
  if (log_enabled())
    fprintf(stderr,
            "[libswiglu_b200] launch sgl %s R=%lld N=%lld K=%lld M=%lld E=%lld cta_group=%d "
            "acc_cols=%d splits=%d a_rows=%d stages=%d grid=%lld smem=%d\n",
            s.name, static_cast<long long>(s.R), static_cast<long long>(s.N),
            static_cast<long long>(s.K), static_cast<long long>(s.M), static_cast<long long>(s.E),
            cta_group, acc_cols, s.splits, a_rows, stages,
            static_cast<long long>(grid * cta_group), smem);
  if (nvtx_enabled()) nvtxRangePushA(s.name);
  cudaError_t e = cudaLaunchKernelEx(&lc, v.fn, maps, p);
  if (nvtx_enabled()) nvtxRangePop();
  if (e != cudaSuccess) return fail_cuda(e, "experts_kernel launch");
  g_launches.fetch_add(1);
  return SGL_OK;
}

// A launch whose grid may be set up while its predecessor in the stream still runs (the kernels
// wait with griddepcontrol.wait before they touch memory).
template <class... Args, class... Given>
int launch_after(const char* what, void (*fn)(Args...), dim3 grid, dim3 block, int smem,
                 void* stream, Given... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid;
  lc.blockDim = block;
  lc.dynamicSmemBytes = static_cast<size_t>(smem);
  lc.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attrs[1];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attrs;
  lc.numAttrs = 1;
  if (log_enabled()) fprintf(stderr, "[libswiglu_b200] launch sgl %s grid=%u\n", what, grid.x);
  cudaError_t e = cudaLaunchKernelEx(&lc, fn, args...);
  if (e != cudaSuccess) return fail_cuda(e, what);
  g_launches.fetch_add(1);
  return SGL_OK;
}

int validate_routing(int64_t T, int64_t k, int64_t E) {
  if (T < 1 || k < 1 || k > 64 || E < 1 || E > sgl::kOrderMaxExperts)
    return fail(SGL_ERR_BAD_SHAPE,
                "T=%lld >= 1 tokens, k=%lld in [1, 64], E=%lld in [1, %d] needed",
                static_cast<long long>(T), static_cast<long long>(k), static_cast<long long>(E),
                sgl::kOrderMaxExperts);
  if (T > 0x7fffff00ll / k)
    return fail(SGL_ERR_BAD_SHAPE, "T * k = %lld * %lld does not fit 31 bits",
                static_cast<long long>(T), static_cast<long long>(k));
  return SGL_OK;
}

int validate_words(const void* p, const char* name, unsigned align) {
  if (!p) return fail(SGL_ERR_NULL_POINTER, "%s is NULL", name);
  if (reinterpret_cast<uintptr_t>(p) & (align - 1))
    return fail(SGL_ERR_MISALIGNED, "%s is not %u-byte aligned", name, align);
  return SGL_OK;
}

int validate_row_call(int64_t T, int64_t k, int64_t D, int64_t R) {
  int rc = validate_routing(T, k, 1);
  if (rc) return rc;
  if (D < 8 || D % 8 != 0 || D > 0x7fffff00ll)
    return fail(SGL_ERR_BAD_SHAPE, "D=%lld must be a positive multiple of 8",
                static_cast<long long>(D));
  if (R < 1 || R > 0x7fffff00ll)
    return fail(SGL_ERR_BAD_SHAPE, "R=%lld rows must be in [1, 2^31)", static_cast<long long>(R));
  return SGL_OK;
}

// Threads of a token (a power of two of warps, at most 256) and CTAs for `T` tokens, at most
// `per_sm` per SM (16384 x 4096: dispatch 61 us without a limit and 68 us with 8; combine 73 and
// 64 us).  With few tokens, and where the kernel allows it (split), small CTAs share a token.
void row_geometry(int64_t T, int nvec, int64_t per_sm, bool split, const DeviceInfo* info,
                  dim3* grid, dim3* block) {
  unsigned tx = 32;
  while (tx < 256 && tx < static_cast<unsigned>(nvec)) tx *= 2;
  if (split && T * ((nvec + 255) / 256) < info->sm_count) {
    tx = tx < 64 ? tx : 64;
    *block = dim3(tx, 1, 1);
    const unsigned per_token = (static_cast<unsigned>(nvec) + tx - 1) / tx;
    *grid = dim3(static_cast<unsigned>(T), per_token < 64 ? per_token : 64, 1);
    return;
  }
  *block = dim3(tx, 256 / tx, 1);
  const int64_t ctas = (T + block->y - 1) / block->y;
  const int64_t cap = static_cast<int64_t>(info->sm_count) * per_sm;
  *grid = dim3(static_cast<unsigned>(ctas < cap ? ctas : cap), 1, 1);
}

int check_bits(int bits) {
  if (bits != 8 && bits != 16) return fail(SGL_ERR_BAD_ARGUMENT, "bits=%d must be 8 or 16", bits);
  return SGL_OK;
}

}  // namespace

extern "C" {

// First use on a device: the ordering kernels' shared-memory limit (1024 experts need 139 KB).
static int prepare_order_kernels() {
  int dev = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  std::lock_guard<std::mutex> lock(g_dev_mutex);
  ExpertDevice& d = g_expert_devices[dev];
  if (d.order_ready) return SGL_OK;
  const int most = sgl::order_smem_bytes(sgl::kOrderMaxExperts);
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(sgl::expert_order_kernel),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(sgl::expert_count_kernel),
                             cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(sgl::expert_order_dispatch_kernel),
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             most + sgl::kOrderRound * 4);
  if (e != cudaSuccess) return fail_cuda(e, "cudaFuncSetAttribute(expert_order)");
  d.order_ready = true;
  return SGL_OK;
}

// CTAs that order T * k slots, and the slots of each: a round of slots each if there are few, fewer
// CTAs when the table of counts, which every CTA reads, would grow past
// 64 Ki entries.
static void order_plan(int64_t total, int64_t E, int* ctas, int64_t* per_cta) {
  if (total <= sgl::kOrderRound) {
    *ctas = 1;
    *per_cta = total;
    return;
  }
  int64_t n = (total + sgl::kOrderRound - 1) / sgl::kOrderRound;
  const int64_t cap = (64 * 1024) / E;
  if (n > sgl::kOrderMaxCtas) n = sgl::kOrderMaxCtas;
  if (n > cap) n = cap;
  *per_cta = (total + n - 1) / n;
  *ctas = static_cast<int>((total + *per_cta - 1) / *per_cta);
}

int64_t sgl_expert_order_scratch_bytes(int64_t T, int64_t k, int64_t E) {
  int rc = validate_routing(T, k, E);
  if (rc) return rc;
  int ctas;
  int64_t per;
  order_plan(T * k, E, &ctas, &per);
  return ctas > 1 ? static_cast<int64_t>(ctas) * E * 4 : 0;
}

int sgl_expert_order(const void* ids, int ids_are_int64, int64_t T, int64_t k, int64_t ld_ids,
                     int64_t E, void* offsets, void* slots, void* rows, void* scratch,
                     int64_t scratch_bytes, void* stream) {
  int rc;
  if ((rc = validate_routing(T, k, E))) return rc;
  if ((rc = validate_words(ids, "ids", ids_are_int64 ? 8 : 4)) ||
      (rc = validate_words(offsets, "offsets", 4)) || (rc = validate_words(slots, "slots", 4)) ||
      (rc = validate_words(rows, "rows", 4)))
    return rc;
  if (ld_ids < k)
    return fail(SGL_ERR_BAD_STRIDE, "ld_ids=%lld is smaller than k=%lld",
                static_cast<long long>(ld_ids), static_cast<long long>(k));
  sgl::OrderParams p;
  int ctas;
  order_plan(T * k, E, &ctas, &p.per_cta);
  if (ctas > 1) {
    if ((rc = validate_words(scratch, "scratch", 4))) return rc;
    if (scratch_bytes < static_cast<int64_t>(ctas) * E * 4)
      return fail(SGL_ERR_BAD_ARGUMENT, "scratch holds %lld bytes, %lld needed",
                  static_cast<long long>(scratch_bytes), static_cast<long long>(ctas) * E * 4);
  }
  DeviceInfo* info = nullptr;
  if ((rc = check_device(&info))) return rc;
  const int smem = sgl::order_smem_bytes(static_cast<int>(E));
  if ((rc = prepare_order_kernels())) return rc;
  p.ids = ids;
  p.ld_ids = ld_ids;
  p.total = T * k;
  p.k = static_cast<int>(k);
  p.E = static_cast<int>(E);
  p.ids64 = ids_are_int64 != 0;
  p.offsets = static_cast<int*>(offsets);
  p.slots = static_cast<int*>(slots);
  p.rows = static_cast<int*>(rows);
  p.counts = static_cast<int*>(scratch);
  const dim3 threads(sgl::kOrderThreads);
  if (ctas == 1)
    return launch_after("expert_order", sgl::expert_order_kernel, dim3(1), threads, smem, stream,
                        p);
  if ((rc = launch_after("expert_count", sgl::expert_count_kernel, dim3(ctas), threads, smem,
                         stream, p)))
    return rc;
  return launch_after("expert_place", sgl::expert_place_kernel, dim3(ctas), threads,
                      (2 * static_cast<int>(E) + 40) * 4, stream, p);
}

int sgl_expert_dispatch(const void* x, const void* rows, void* out, int64_t T, int64_t k, int64_t D,
                        int64_t R, int64_t ldx, int64_t ldo, void* stream) {
  int rc;
  if ((rc = validate_row_call(T, k, D, R))) return rc;
  if ((rc = validate_ptr(x, "x")) || (rc = validate_words(rows, "rows", 4)) ||
      (rc = validate_ptr(out, "out")))
    return rc;
  if ((rc = validate_ld(ldx, D, "ldx")) || (rc = validate_ld(ldo, D, "ldo"))) return rc;
  DeviceInfo* info = nullptr;
  if ((rc = check_device(&info))) return rc;
  sgl::RowParams p;
  std::memset(&p, 0, sizeof(p));
  p.in = x;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.rows = static_cast<const int*>(rows);
  p.ld_in = ldx;
  p.ld_out = ldo;
  p.T = T;
  p.k = static_cast<int>(k);
  p.nvec = static_cast<int>(D / 8);
  p.R = R;
  dim3 grid, block;
  row_geometry(T, p.nvec, 4096, true, info, &grid, &block);
  return launch_after("expert_dispatch", sgl::expert_dispatch_kernel, grid, block, 0, stream, p);
}

// `splits`: partial sums of every fp32 row, R rows apart (sgl_experts_swiglu).
static int combine_rows(const void* in, int in_is_f32, int splits, const void* rows,
                        const void* weights, int weights_bf16, void* out, int64_t T, int64_t k,
                        int64_t D, int64_t R, int64_t ld_in, int64_t ld_w, int64_t ldo,
                        void* stream) {
  int rc;
  if ((rc = validate_row_call(T, k, D, R))) return rc;
  if ((rc = validate_ptr(in, "in")) || (rc = validate_words(rows, "rows", 4)) ||
      (rc = validate_ptr(out, "out")))
    return rc;
  if (weights) {
    if ((rc = validate_words(weights, "weights", weights_bf16 ? 2 : 4))) return rc;
    if (ld_w < k)
      return fail(SGL_ERR_BAD_STRIDE, "ld_w=%lld is smaller than k=%lld",
                  static_cast<long long>(ld_w), static_cast<long long>(k));
  }
  if ((rc = validate_ld(ld_in, D, "ld_in")) || (rc = validate_ld(ldo, D, "ldo"))) return rc;
  DeviceInfo* info = nullptr;
  if ((rc = check_device(&info))) return rc;
  sgl::RowParams p;
  std::memset(&p, 0, sizeof(p));
  p.in = in;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.rows = static_cast<const int*>(rows);
  p.splits = splits;
  p.slot_stride = R * ld_in;
  p.weights = weights;
  p.w_bf16 = weights_bf16 != 0;
  p.ld_in = ld_in;
  p.ld_out = ldo;
  p.ld_w = ld_w;
  p.T = T;
  p.k = static_cast<int>(k);
  p.nvec = static_cast<int>(D / 8);
  p.R = R;
  dim3 grid, block;
  row_geometry(T, p.nvec, 8, true, info, &grid, &block);
  if (splits > 1)
    return launch_after("expert_combine", sgl::expert_combine_parts_kernel, grid, block, 0, stream,
                        p);
  return launch_after("expert_combine",
                      k <= 2 ? (in_is_f32 ? sgl::expert_combine_kernel<true, 2, 2>
                                          : sgl::expert_combine_kernel<false, 2, 2>)
                             : (in_is_f32 ? sgl::expert_combine_kernel<true, 1, 4>
                                          : sgl::expert_combine_kernel<false, 1, 4>),
                      grid, block, 0, stream, p);
}

int sgl_expert_combine(const void* in, int in_is_f32, const void* rows, const void* weights,
                       int weights_bf16, void* out, int64_t T, int64_t k, int64_t D, int64_t R,
                       int64_t ld_in, int64_t ld_w, int64_t ldo, void* stream) {
  return combine_rows(in, in_is_f32, 1, rows, weights, weights_bf16, out, T, k, D, R, ld_in, ld_w,
                      ldo, stream);
}

int sgl_expert_combine_grad(const void* grad_out, const void* in, int in_is_f32, const void* rows,
                            const void* weights, int weights_bf16, void* grad_rows,
                            void* grad_weights, int64_t T, int64_t k, int64_t D, int64_t R,
                            int64_t ld_go, int64_t ld_in, int64_t ld_w, int64_t ld_gr,
                            void* stream) {
  int rc;
  if ((rc = validate_row_call(T, k, D, R))) return rc;
  const unsigned wa = weights_bf16 ? 2 : 4;
  if ((rc = validate_ptr(grad_out, "grad_out")) || (rc = validate_words(rows, "rows", 4)) ||
      (rc = validate_ptr(grad_rows, "grad_rows")))
    return rc;
  if (weights && (rc = validate_words(weights, "weights", wa))) return rc;
  if ((in != nullptr || grad_weights != nullptr) &&
      ((rc = validate_ptr(in, "in")) || (rc = validate_words(grad_weights, "grad_weights", wa))))
    return rc;
  if (weights && ld_w < k)
    return fail(SGL_ERR_BAD_STRIDE, "ld_w=%lld is smaller than k=%lld",
                static_cast<long long>(ld_w), static_cast<long long>(k));
  if ((rc = validate_ld(ld_go, D, "ld_go")) || (in && (rc = validate_ld(ld_in, D, "ld_in"))) ||
      (rc = validate_ld(ld_gr, D, "ld_gr")))
    return rc;
  DeviceInfo* info = nullptr;
  if ((rc = check_device(&info))) return rc;
  sgl::RowParams p;
  std::memset(&p, 0, sizeof(p));
  p.in = grad_out;
  p.in2 = in;
  p.out = static_cast<__nv_bfloat16*>(grad_rows);
  p.rows = static_cast<const int*>(rows);
  p.weights = weights;
  p.w_bf16 = weights_bf16 != 0;
  p.grad_weights = grad_weights;
  p.ld_in = ld_go;
  p.ld_in2 = ld_in;
  p.ld_out = ld_gr;
  p.ld_w = ld_w;
  p.T = T;
  p.k = static_cast<int>(k);
  p.nvec = static_cast<int>(D / 8);
  p.R = R;
  dim3 grid, block;
  row_geometry(T, p.nvec, 8, false, info, &grid, &block);
  return launch_after("expert_combine_grad",
                      k <= 2 ? (in_is_f32 ? sgl::expert_combine_grad_kernel<true, 2, 2>
                                          : sgl::expert_combine_grad_kernel<false, 2, 2>)
                             : (in_is_f32 ? sgl::expert_combine_grad_kernel<true, 1, 4>
                                          : sgl::expert_combine_grad_kernel<false, 1, 4>),
                      grid, block, 0, stream, p);
}

int64_t sgl_preact_bytes(int bits, int64_t rows, int64_t N, int64_t* pitch, int64_t* scale_bytes,
                         int64_t* scale_pitch) {
  int rc;
  if ((rc = check_bits(bits))) return rc;
  if (rows < 0)
    return fail(SGL_ERR_BAD_SHAPE, "rows=%lld must not be negative", static_cast<long long>(rows));
  if ((rc = validate_shape(rows < 1 ? 1 : rows, N, 8))) return rc;
  const PreactLayout l = preact_layout(bits, N);
  if (pitch) *pitch = l.pitch;
  if (scale_pitch) *scale_pitch = l.scale_pitch;
  if (scale_bytes) *scale_bytes = l.scale_pitch * rows;
  return l.pitch * rows;
}

static int grouped_swiglu(const char* name, const void* x, const void* w, const void* offsets,
                          void* h, void* pre, void* scales, int bits, int64_t R, int64_t N,
                          int64_t K, int64_t E, int64_t ldx, int64_t ldw, int64_t w_stride,
                          int64_t ldh, void* stream) {
  int rc;
  if ((rc = validate_groups(R, E, offsets, E > 1))) return rc;
  if ((rc = validate_ptr(x, "x")) || (rc = validate_ptr(w, "w")) || (rc = validate_ptr(h, "h")))
    return rc;
  if ((rc = validate_shape(R, N, K))) return rc;
  if ((rc = validate_ld(ldx, K, "ldx")) || (rc = validate_ld(ldw, 2 * N, "ldw")) ||
      (rc = validate_ld(ldh, N, "ldh")) ||
      (rc = validate_expert_stride(w_stride, K, ldw, E, "w_stride")))
    return rc;
  ExpertLaunch s;
  s.form = bits == 0 ? sgl::EXP_SWIGLU : (bits == 8 ? sgl::EXP_SAVE8 : sgl::EXP_SAVE16);
  if (bits != 0) {
    if ((rc = validate_ptr(pre, "pre"))) return rc;
    if (bits == 8 && (rc = validate_words(scales, "scales", 2))) return rc;
  }
  s.name = name;
  s.a = x;
  s.b = w;
  s.out = h;
  s.offsets = static_cast<const int*>(offsets);
  s.R = R;
  s.N = N;
  s.K = K;
  s.E = E;
  s.lda = ldx;
  s.ldb = ldw;
  s.b_stride = E > 1 ? w_stride : K * ldw;
  s.ld_out = ldh;
  s.pre = pre;
  s.scales = scales;
  return launch_experts(s, stream);
}

int sgl_grouped_fused_swiglu(const void* x, const void* w, const void* offsets, void* h, int64_t R,
                             int64_t N, int64_t K, int64_t E, int64_t ldx, int64_t ldw,
                             int64_t w_stride, int64_t ldh, void* stream) {
  int rc = validate_groups(R, E, offsets, true);
  if (rc) return rc;
  return grouped_swiglu("grouped_fused_swiglu", x, w, offsets, h, nullptr, nullptr, 0, R, N, K, E,
                        ldx, ldw, w_stride, ldh, stream);
}

int sgl_grouped_fused_swiglu_save(const void* x, const void* w, const void* offsets, void* h,
                                  void* pre, void* scales, int bits, int64_t R, int64_t N,
                                  int64_t K, int64_t E, int64_t ldx, int64_t ldw, int64_t w_stride,
                                  int64_t ldh, void* stream) {
  int rc = check_bits(bits);
  if (rc) return rc;
  return grouped_swiglu("grouped_fused_swiglu_save", x, w, offsets, h, pre, scales, bits, R, N, K,
                        E, ldx, ldw, w_stride, ldh, stream);
}

static int grouped_matmul(const void* a, const void* b, const void* offsets, void* c, int64_t R,
                          int64_t N, int64_t K, int64_t E, int64_t lda, int64_t ldb,
                          int64_t b_stride, int64_t ldc, int b_transposed, int c_is_f32, int splits,
                          int64_t k_per_split, void* stream) {
  int rc;
  if ((rc = validate_groups(R, E, offsets, true))) return rc;
  if ((rc = validate_ptr(a, "a")) || (rc = validate_ptr(b, "b")) || (rc = validate_ptr(c, "c")))
    return rc;
  if ((rc = validate_shape(R, N, K))) return rc;
  const int64_t b_rows = b_transposed ? N : K;
  if ((rc = validate_ld(lda, K, "lda")) || (rc = validate_ld(ldb, b_transposed ? K : N, "ldb")) ||
      (rc = validate_ld(ldc, N, "ldc")) ||
      (rc = validate_expert_stride(b_stride, b_rows, ldb, E, "b_stride")))
    return rc;
  ExpertLaunch s;
  s.form = c_is_f32 ? sgl::EXP_GEMM32 : sgl::EXP_GEMM;
  s.name = "grouped_matmul";
  s.a = a;
  s.b = b;
  s.out = c;
  s.offsets = static_cast<const int*>(offsets);
  s.R = R;
  s.N = N;
  s.K = K;
  s.E = E;
  s.lda = lda;
  s.ldb = ldb;
  s.b_stride = E > 1 ? b_stride : b_rows * ldb;
  s.ld_out = ldc;
  s.b_transposed = b_transposed != 0;
  s.splits = splits;
  s.k_per_split = k_per_split;
  return launch_experts(s, stream);
}

int sgl_grouped_matmul(const void* a, const void* b, const void* offsets, void* c, int64_t R,
                       int64_t N, int64_t K, int64_t E, int64_t lda, int64_t ldb, int64_t b_stride,
                       int64_t ldc, int b_transposed, int c_is_f32, void* stream) {
  return grouped_matmul(a, b, offsets, c, R, N, K, E, lda, ldb, b_stride, ldc, b_transposed,
                        c_is_f32, 1, 0, stream);
}

int sgl_grouped_grad_preact(const void* dy, const void* w_down, const void* offsets,
                            const void* slots, const void* weights, int weights_bf16,
                            const void* pre, const void* scales, int bits, void* grad_preact,
                            void* h, int64_t R, int64_t N, int64_t D, int64_t E, int64_t k,
                            int64_t lddy, int64_t ldw, int64_t w_stride, int64_t ld_weights,
                            int64_t ld_grad, int64_t ldh, void* stream) {
  int rc;
  if ((rc = check_bits(bits)) || (rc = validate_groups(R, E, offsets, true))) return rc;
  if ((rc = validate_ptr(dy, "dy")) || (rc = validate_ptr(w_down, "w_down")) ||
      (rc = validate_ptr(pre, "pre")) || (rc = validate_ptr(grad_preact, "grad_preact")) ||
      (rc = validate_ptr(h, "h")))
    return rc;
  if (bits == 8 && (rc = validate_words(scales, "scales", 2))) return rc;
  if (slots || weights) {
    if ((rc = validate_words(slots, "slots", 4)) ||
        (rc = validate_words(weights, "weights", weights_bf16 ? 2 : 4)))
      return rc;
    if (k < 1 || k > 64 || R % k != 0)
      return fail(SGL_ERR_BAD_SHAPE, "k=%lld outside [1, 64] or not a divisor of R=%lld",
                  static_cast<long long>(k), static_cast<long long>(R));
    if (ld_weights < k)
      return fail(SGL_ERR_BAD_STRIDE, "ld_weights=%lld is smaller than k=%lld",
                  static_cast<long long>(ld_weights), static_cast<long long>(k));
  }
  if ((rc = validate_shape(R, N, D))) return rc;
  if ((rc = validate_ld(lddy, D, "lddy")) || (rc = validate_ld(ldw, D, "ldw")) ||
      (rc = validate_ld(ld_grad, 2 * N, "ld_grad")) || (rc = validate_ld(ldh, N, "ldh")) ||
      (rc = validate_expert_stride(w_stride, N, ldw, E, "w_stride")))
    return rc;
  ExpertLaunch s;
  s.form = bits == 8 ? sgl::EXP_GRAD8 : sgl::EXP_GRAD16;
  s.name = "grouped_grad_preact";
  s.a = dy;
  s.b = w_down;
  s.out = h;
  s.offsets = static_cast<const int*>(offsets);
  s.R = R;
  s.N = N;
  s.K = D;
  s.E = E;
  s.lda = lddy;
  s.ldb = ldw;
  s.b_stride = E > 1 ? w_stride : N * ldw;
  s.b_transposed = 1;
  s.ld_out = ldh;
  s.pre = grad_preact;
  s.ld_pre = ld_grad;
  s.saved = pre;
  s.scales = const_cast<void*>(scales);
  s.slots = static_cast<const int*>(slots);
  s.weights = weights;
  s.ld_w = ld_weights;
  s.k = slots ? k : 1;
  s.w_bf16 = weights_bf16 != 0;
  return launch_experts(s, stream);
}

int sgl_grouped_weight_grad(const void* a, const void* g, const void* offsets, void* c, int64_t R,
                            int64_t M, int64_t N, int64_t E, int64_t lda, int64_t ldg, int64_t ldc,
                            int64_t c_stride, void* stream) {
  int rc;
  if ((rc = validate_groups(R, E, offsets, true))) return rc;
  if ((rc = validate_ptr(a, "a")) || (rc = validate_ptr(g, "g")) || (rc = validate_ptr(c, "c")))
    return rc;
  if ((rc = validate_shape(R, N, M))) return rc;
  if ((rc = validate_ld(lda, M, "lda")) || (rc = validate_ld(ldg, N, "ldg")) ||
      (rc = validate_ld(ldc, N, "ldc")) ||
      (rc = validate_expert_stride(c_stride, M, ldc, E, "c_stride", N)))
    return rc;
  ExpertLaunch s;
  s.form = sgl::EXP_WGRAD;
  s.name = "grouped_weight_grad";
  s.a = a;
  s.b = g;
  s.out = c;
  s.offsets = static_cast<const int*>(offsets);
  s.R = R;
  s.N = N;
  s.K = R;
  s.M = M;
  s.E = E;
  s.lda = lda;
  s.ldb = ldg;
  s.ld_out = ldc;
  s.out_stride = E > 1 ? c_stride : M * ldc;
  return launch_experts(s, stream);
}

int sgl_swiglu_grad_preact_saved(const void* dy, const void* pre, const void* scales, int bits,
                                 void* grad_preact, void* h, const void* end, int64_t rows,
                                 int64_t N, int64_t lddy, int64_t ldo, int64_t ldh, void* stream) {
  int rc;
  if ((rc = check_bits(bits))) return rc;
  if ((rc = validate_ptr(dy, "dy")) || (rc = validate_ptr(pre, "pre")) ||
      (rc = validate_ptr(grad_preact, "grad_preact")))
    return rc;
  if (bits == 8 && (rc = validate_words(scales, "scales", 2))) return rc;
  if (h && (rc = validate_ptr(h, "h"))) return rc;
  if (end && (rc = validate_words(end, "end", 4))) return rc;
  if ((rc = validate_shape(rows, N, 8))) return rc;
  if ((rc = validate_ld(lddy, N, "lddy")) || (rc = validate_ld(ldo, 2 * N, "ldo"))) return rc;
  if (h && (rc = validate_ld(ldh, N, "ldh"))) return rc;
  DeviceInfo* info = nullptr;
  if ((rc = check_device(&info))) return rc;
  const PreactLayout l = preact_layout(bits, N);
  sgl::PreactParams p;
  p.dy = static_cast<const __nv_bfloat16*>(dy);
  p.pre = static_cast<const uint8_t*>(pre);
  p.scales = static_cast<const uint8_t*>(scales);
  p.grad = static_cast<__nv_bfloat16*>(grad_preact);
  p.h = static_cast<__nv_bfloat16*>(h);
  p.end = static_cast<const int*>(end);
  p.lddy = lddy;
  p.ld_pre = l.pitch;
  p.gate_off = l.gate_off;
  p.ld_scales = l.scale_pitch;
  p.gate_scale_off = l.gate_scale_off;
  p.ld_grad = ldo;
  p.ldh = ldh;
  p.rows = rows;
  p.nvec = static_cast<int>(N / 8);
  // two vectors of 8 columns per thread where a row has more than a CTA's threads
  const int vecs = p.nvec > sgl::kPreactThreads ? 2 : 1;
  const int64_t per_cta = static_cast<int64_t>(sgl::kPreactThreads) * vecs;
  const int64_t chunks = (p.nvec + per_cta - 1) / per_cta;
  int64_t pairs = (rows + 1) / 2;
  const int64_t cap = (static_cast<int64_t>(info->sm_count) * 32 + chunks - 1) / chunks;
  if (pairs > cap) pairs = cap;
  return launch_after("grad_preact_saved",
                      bits == 8 ? (vecs == 2 ? sgl::grad_preact_saved_kernel<8, 2>
                                             : sgl::grad_preact_saved_kernel<8, 1>)
                                : (vecs == 2 ? sgl::grad_preact_saved_kernel<16, 2>
                                             : sgl::grad_preact_saved_kernel<16, 1>),
                      dim3(static_cast<unsigned>(chunks), static_cast<unsigned>(pairs)),
                      dim3(sgl::kPreactThreads), 0, stream, p);
}

int sgl_fused_swiglu_backward_saved(const void* x, const void* w, const void* dy, const void* pre,
                                    const void* scales, int bits, void* grad_preact, void* grad_x,
                                    void* grad_w, int64_t M, int64_t N, int64_t K, int64_t ldx,
                                    int64_t ldw, int64_t lddy, const sgl_config* cfg_x,
                                    const sgl_config* cfg_w, void* stream) {
  int rc;
  // everything the launches below would refuse is refused before the first of them
  if ((rc = validate_ptr(x, "x")) || (rc = validate_ptr(w, "w"))) return rc;
  if ((grad_x && (rc = validate_ptr(grad_x, "grad_x"))) ||
      (grad_w && (rc = validate_ptr(grad_w, "grad_w"))))
    return rc;
  if ((rc = validate_shape(M, N, K))) return rc;
  if ((rc = validate_ld(ldx, K, "ldx")) || (rc = validate_ld(ldw, 2 * N, "ldw"))) return rc;
  sgl_config c;
  if ((rc = resolve_config(SGL_FORM_MATMUL, cfg_x, M, &c)) ||
      (rc = resolve_config(SGL_FORM_MATMUL, cfg_w, K, &c)))
    return rc;
  if ((rc = sgl_swiglu_grad_preact_saved(dy, pre, scales, bits, grad_preact, nullptr, nullptr, M, N,
                                         lddy, 2 * N, 0, stream)))
    return rc;
  if (grad_x && (rc = sgl_matmul_bf16_ex(grad_preact, w, grad_x, M, K, 2 * N, 2 * N, ldw, K, 0, 1,
                                         cfg_x, stream)))
    return rc;
  if (grad_w)
    return sgl_matmul_bf16_ex(x, grad_preact, grad_w, K, 2 * N, M, ldx, 2 * N, 2 * N, 1, 0, cfg_w,
                              stream);
  return SGL_OK;
}

// ---- the expert layer at inference, one call ----

static int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

struct ExpertsWorkspace {
  int64_t offsets, slots, rows, scratch, scratch_bytes, xs, h, ys, total;
  int splits;              // ranges of the down projection's sum
  int64_t k_per_split;
};

// Few rows make few tiles, and the down projection (long sums, narrow results) then leaves SMs
// idle while others stream long columns of weight.  Its sum is cut into ranges of at least 512 (the
// last may be shorter, since the others are rounded up to whole blocks of 128) whose partial
// rows the combine step adds up in order: as many as give every SM about four tiles if all
// groups are used, while the partial rows written and read stay below an eighth of the weight.  A
// function of the sizes alone, a B200's 148 SMs assumed: workspaces are sized, and the order of
// the additions is fixed, without asking a device.  1 token x 2 of 8 experts, 14336 -> 4096: 59 us in
// one range, 43 us in eight.
static void down_ranges(int64_t R, int64_t E, int64_t N, int64_t D_out, int* splits,
                        int64_t* per_split) {
  *splits = 1;
  *per_split = 0;
  const int64_t groups = E < R ? E : R;
  if (R / E >= 64) return;
  const int64_t tiles = (groups + R / sgl::kBlockM) * ((D_out + 127) / 128);
  int64_t s = (4 * 148 + tiles - 1) / tiles;
  if (s > N / 512) s = N / 512;
  if (s > groups * N / (32 * R)) s = groups * N / (32 * R);
  if (s > 8) s = 8;          // (what the combine step has in flight at once)
  if (s < 2) return;
  *per_split = (((N + s - 1) / s) + 127) / 128 * 128;
  *splits = static_cast<int>((N + *per_split - 1) / *per_split);
}

static int experts_workspace(int64_t T, int64_t k, int64_t E, int64_t D, int64_t N, int64_t D_out,
                             ExpertsWorkspace* w) {
  int rc;
  if ((rc = validate_routing(T, k, E)) || (rc = validate_shape(T * k, N, D)) ||
      (rc = validate_shape(T * k, D_out, 8)))
    return rc;
  const int64_t R = T * k;
  int64_t at = 0;
  w->offsets = at;
  at += align256((E + 1) * 4);
  w->slots = at;
  at += align256(R * 4);
  w->rows = at;
  at += align256(R * 4);
  w->scratch = at;
  w->scratch_bytes = sgl_expert_order_scratch_bytes(T, k, E);
  at += align256(w->scratch_bytes);
  w->xs = at;
  at += align256(R * D * 2);
  w->h = at;
  at += align256(R * N * 2);
  w->ys = at;
  down_ranges(R, E, N, D_out, &w->splits, &w->k_per_split);
  at += align256(R * D_out * 4 * w->splits);
  w->total = at;
  return SGL_OK;
}

int64_t sgl_experts_swiglu_workspace_bytes(int64_t T, int64_t k, int64_t E, int64_t D, int64_t N,
                                           int64_t D_out) {
  ExpertsWorkspace w;
  int rc = experts_workspace(T, k, E, D, N, D_out, &w);
  return rc ? rc : w.total;
}

// What all three forms of the layer refuse, before the first launch.
struct LayerCall {
  const void *x, *ids, *weights, *w, *w_down;
  int ids_are_int64, weights_bf16;
  int64_t T, k, E, D, N, D_out;
  int64_t ldx, ld_ids, ld_weights, ldw, w_stride, ldd, d_stride;
};
static int validate_layer(const LayerCall& c, bool with_ids) {
  int rc;
  if ((rc = validate_ptr(c.x, "x")) ||
      (with_ids && (rc = validate_words(c.ids, "ids", c.ids_are_int64 ? 8 : 4))) ||
      (rc = validate_words(c.weights, "weights", c.weights_bf16 ? 2 : 4)) ||
      (rc = validate_ptr(c.w, "w")) || (rc = validate_ptr(c.w_down, "w_down")))
    return rc;
  if ((with_ids && c.ld_ids < c.k) || c.ld_weights < c.k)
    return fail(SGL_ERR_BAD_STRIDE, "ld_ids=%lld and ld_weights=%lld must be at least k=%lld",
                static_cast<long long>(c.ld_ids), static_cast<long long>(c.ld_weights),
                static_cast<long long>(c.k));
  if ((rc = validate_ld(c.ldx, c.D, "ldx")) || (rc = validate_ld(c.ldw, 2 * c.N, "ldw")) ||
      (rc = validate_ld(c.ldd, c.D_out, "ldd")) ||
      (rc = validate_expert_stride(c.w_stride, c.D, c.ldw, c.E, "w_stride")) ||
      (rc = validate_expert_stride(c.d_stride, c.N, c.ldd, c.E, "d_stride")))
    return rc;
  return SGL_OK;
}
static int validate_workspace(const void* workspace, int64_t have, int64_t need) {
  int rc = validate_ptr(workspace, "workspace");
  if (rc) return rc;
  if (have < need)
    return fail(SGL_ERR_BAD_ARGUMENT, "workspace holds %lld bytes, %lld needed",
                static_cast<long long>(have), static_cast<long long>(need));
  return SGL_OK;
}

// The slots in order and x's rows with their experts: one launch for few slots, three for more.
static int order_and_dispatch(const LayerCall& c, void* offsets, void* slots, void* rows,
                              void* scratch, int64_t scratch_bytes, void* xs, void* stream) {
  const int64_t R = c.T * c.k;
  int rc;
  if (R > sgl::kOrderRound) {
    if ((rc = sgl_expert_order(c.ids, c.ids_are_int64, c.T, c.k, c.ld_ids, c.E, offsets, slots, rows,
                               scratch, scratch_bytes, stream)))
      return rc;
    return sgl_expert_dispatch(c.x, rows, xs, c.T, c.k, c.D, R, c.ldx, c.D, stream);
  }
  DeviceInfo* info = nullptr;
  if ((rc = check_device(&info)) || (rc = prepare_order_kernels())) return rc;
  sgl::OrderParams p;
  std::memset(&p, 0, sizeof(p));
  p.ids = c.ids;
  p.ld_ids = c.ld_ids;
  p.total = p.per_cta = R;
  p.k = static_cast<int>(c.k);
  p.E = static_cast<int>(c.E);
  p.ids64 = c.ids_are_int64 != 0;
  p.offsets = static_cast<int*>(offsets);
  p.slots = static_cast<int*>(slots);
  p.rows = static_cast<int*>(rows);
  int64_t ctas = (c.T + 3) / 4;
  if (ctas > info->sm_count) ctas = info->sm_count;
  return launch_after("expert_order_dispatch", sgl::expert_order_dispatch_kernel,
                      dim3(static_cast<unsigned>(ctas)), dim3(sgl::kOrderThreads),
                      sgl::order_smem_bytes(static_cast<int>(c.E)) + sgl::kOrderRound * 4, stream, p,
                      static_cast<const __nv_bfloat16*>(c.x), static_cast<__nv_bfloat16*>(xs), c.ldx,
                      static_cast<int64_t>(c.D), static_cast<int>(c.D / 8));
}

int sgl_experts_swiglu(const void* x, const void* ids, int ids_are_int64, const void* weights,
                       int weights_bf16, const void* w, const void* w_down, void* y,
                       void* workspace, int64_t workspace_bytes, int64_t T, int64_t k, int64_t E,
                       int64_t D, int64_t N, int64_t D_out, int64_t ldx, int64_t ld_ids,
                       int64_t ld_weights, int64_t ldw, int64_t w_stride, int64_t ldd,
                       int64_t d_stride, int64_t ldy, void* stream) {
  const LayerCall c{x, ids, weights, w,   w_down, ids_are_int64, weights_bf16, T,        k,  E,
                    D, N,   D_out,   ldx, ld_ids, ld_weights,    ldw,          w_stride, ldd, d_stride};
  ExpertsWorkspace l;
  int rc;
  if ((rc = experts_workspace(T, k, E, D, N, D_out, &l)) || (rc = validate_layer(c, true)) ||
      (rc = validate_ptr(y, "y")) || (rc = validate_ld(ldy, D_out, "ldy")) ||
      (rc = validate_workspace(workspace, workspace_bytes, l.total)))
    return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t R = T * k;
  if ((rc = order_and_dispatch(c, ws + l.offsets, ws + l.slots, ws + l.rows, ws + l.scratch,
                               l.scratch_bytes, ws + l.xs, stream)) ||
      (rc = sgl_grouped_fused_swiglu(ws + l.xs, w, ws + l.offsets, ws + l.h, R, N, D, E, D, ldw,
                                     w_stride, N, stream)) ||
      (rc = grouped_matmul(ws + l.h, w_down, ws + l.offsets, ws + l.ys, R, D_out, N, E, N, ldd,
                           d_stride, D_out, 0, 1, l.splits, l.k_per_split, stream)))
    return rc;
  return combine_rows(ws + l.ys, 1, l.splits, ws + l.rows, weights, weights_bf16, y, T, k, D_out, R,
                      D_out, ld_weights, ldy, stream);
}

// ---- the expert layer in training: forward and backward, one call each ----

// An order as one int32 buffer: offsets[E + 1], slots[T * k], rows[T * k].
struct OrderBuffer {
  int *offsets, *slots, *rows;
};
static OrderBuffer split_order(const void* order, int64_t R, int64_t E) {
  int* p = static_cast<int*>(const_cast<void*>(order));
  return OrderBuffer{p, p + E + 1, p + E + 1 + R};
}

// Forward: the grouped x, h and the order's scratch.  Backward: the pre-activations' gradients, and
// one region that holds the rows' gradients and the weighted h, then the grouped x, then the rows
// of x's gradient (each is dead when the next is written).
struct TrainWorkspace {
  int64_t xs, h, scratch, scratch_bytes, forward;
  int64_t grad_pre, region, weighted_h, backward;
};
static int train_workspace(int64_t T, int64_t k, int64_t E, int64_t D, int64_t N, int64_t D_out,
                           TrainWorkspace* w) {
  int rc;
  if ((rc = validate_routing(T, k, E)) || (rc = validate_shape(T * k, N, D)) ||
      (rc = validate_shape(T * k, D_out, 8)))
    return rc;
  const int64_t R = T * k;
  w->xs = 0;
  w->h = align256(R * D * 2);
  w->scratch = w->h + align256(R * N * 2);
  w->scratch_bytes = sgl_expert_order_scratch_bytes(T, k, E);
  w->forward = w->scratch + align256(w->scratch_bytes);
  w->grad_pre = 0;
  w->region = align256(R * 2 * N * 2);
  w->weighted_h = w->region + align256(R * D_out * 2);
  const int64_t first = align256(R * D_out * 2) + align256(R * N * 2), rows = align256(R * D * 4);
  w->backward = w->region + (first > rows ? first : rows);
  return SGL_OK;
}

int64_t sgl_experts_swiglu_train_workspace_bytes(int64_t T, int64_t k, int64_t E, int64_t D,
                                                 int64_t N, int64_t D_out, int backward) {
  TrainWorkspace w;
  int rc = train_workspace(T, k, E, D, N, D_out, &w);
  return rc ? rc : (backward ? w.backward : w.forward);
}

int sgl_experts_swiglu_save(const void* x, const void* ids, int ids_are_int64, const void* weights,
                            int weights_bf16, const void* w, const void* w_down, void* y,
                            void* order, void* pre, void* scales, int bits, void* ys,
                            void* workspace, int64_t workspace_bytes, int64_t T, int64_t k,
                            int64_t E, int64_t D, int64_t N, int64_t D_out, int64_t ldx,
                            int64_t ld_ids, int64_t ld_weights, int64_t ldw, int64_t w_stride,
                            int64_t ldd, int64_t d_stride, void* stream) {
  const LayerCall c{x, ids, weights, w,   w_down, ids_are_int64, weights_bf16, T,        k,  E,
                    D, N,   D_out,   ldx, ld_ids, ld_weights,    ldw,          w_stride, ldd, d_stride};
  TrainWorkspace l;
  int rc;
  if ((rc = check_bits(bits)) || (rc = train_workspace(T, k, E, D, N, D_out, &l)) ||
      (rc = validate_layer(c, true)) || (rc = validate_ptr(y, "y")) ||
      (rc = validate_words(order, "order", 4)) || (rc = validate_ptr(pre, "pre")) ||
      (bits == 8 && (rc = validate_words(scales, "scales", 2))) || (rc = validate_ptr(ys, "ys")) ||
      (rc = validate_workspace(workspace, workspace_bytes, l.forward)))
    return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t R = T * k;
  const OrderBuffer o = split_order(order, R, E);
  if ((rc = order_and_dispatch(c, o.offsets, o.slots, o.rows, ws + l.scratch, l.scratch_bytes,
                               ws + l.xs, stream)) ||
      (rc = sgl_grouped_fused_swiglu_save(ws + l.xs, w, o.offsets, ws + l.h, pre, scales, bits, R, N,
                                          D, E, D, ldw, w_stride, N, stream)) ||
      (rc = grouped_matmul(ws + l.h, w_down, o.offsets, ys, R, D_out, N, E, N, ldd, d_stride, D_out,
                           0, 1, 1, 0, stream)))
    return rc;
  return combine_rows(ys, 1, 1, o.rows, weights, weights_bf16, y, T, k, D_out, R, D_out, ld_weights,
                      D_out, stream);
}

int sgl_experts_swiglu_backward(const void* grad_y, const void* x, const void* weights,
                                int weights_bf16, const void* w, const void* w_down,
                                const void* order, const void* pre, const void* scales, int bits,
                                const void* ys, void* grad_x, void* grad_weights, void* grad_w,
                                void* grad_down, void* workspace, int64_t workspace_bytes, int64_t T,
                                int64_t k, int64_t E, int64_t D, int64_t N, int64_t D_out,
                                int64_t ldx, int64_t ld_weights, int64_t ldw, int64_t w_stride,
                                int64_t ldd, int64_t d_stride, void* stream) {
  const LayerCall c{x, nullptr, weights, w,   w_down, 0,          weights_bf16, T,        k,  E,
                    D, N,       D_out,   ldx, 0,      ld_weights, ldw,          w_stride, ldd, d_stride};
  TrainWorkspace l;
  int rc;
  if ((rc = check_bits(bits)) || (rc = train_workspace(T, k, E, D, N, D_out, &l)) ||
      (rc = validate_layer(c, false)) || (rc = validate_ptr(grad_y, "grad_y")) ||
      (rc = validate_words(order, "order", 4)) || (rc = validate_ptr(pre, "pre")) ||
      (bits == 8 && (rc = validate_words(scales, "scales", 2))) ||
      (grad_weights && ((rc = validate_ptr(ys, "ys")) ||
                        (rc = validate_words(grad_weights, "grad_weights", weights_bf16 ? 2 : 4)))) ||
      (grad_x && (rc = validate_ptr(grad_x, "grad_x"))) ||
      (grad_w && (rc = validate_ptr(grad_w, "grad_w"))) ||
      (grad_down && (rc = validate_ptr(grad_down, "grad_down"))) ||
      (rc = validate_workspace(workspace, workspace_bytes, l.backward)))
    return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t R = T * k;
  const OrderBuffer o = split_order(order, R, E);
  void *grad_pre = ws + l.grad_pre, *region = ws + l.region, *weighted_h = ws + l.weighted_h;
  // the rows' gradients without the routing weights, and the weights' own
  if ((rc = sgl_expert_combine_grad(grad_y, grad_weights ? ys : nullptr, 1, o.rows, nullptr,
                                    weights_bf16, region, grad_weights, T, k, D_out, R, D_out, D_out,
                                    0, D_out, stream)))
    return rc;
  if (!grad_x && !grad_w && !grad_down) return SGL_OK;
  if ((rc = sgl_grouped_grad_preact(region, w_down, o.offsets, o.slots, weights, weights_bf16, pre,
                                    scales, bits, grad_pre, weighted_h, R, N, D_out, E, k, D_out,
                                    ldd, d_stride, ld_weights, 2 * N, N, stream)))
    return rc;
  if (grad_down && (rc = sgl_grouped_weight_grad(weighted_h, region, o.offsets, grad_down, R, N,
                                                 D_out, E, N, D_out, D_out, N * D_out, stream)))
    return rc;
  if (grad_w &&
      ((rc = sgl_expert_dispatch(x, o.rows, region, T, k, D, R, ldx, D, stream)) ||
       (rc = sgl_grouped_weight_grad(region, grad_pre, o.offsets, grad_w, R, D, 2 * N, E, D, 2 * N,
                                     2 * N, D * 2 * N, stream))))
    return rc;
  if (grad_x) {
    if ((rc = grouped_matmul(grad_pre, w, o.offsets, region, R, D, 2 * N, E, 2 * N, ldw, w_stride, D,
                             1, 1, 1, 0, stream)))
      return rc;
    return combine_rows(region, 1, 1, o.rows, nullptr, 0, grad_x, T, k, D, R, D, 0, D, stream);
  }
  return SGL_OK;
}

}  // extern "C"
