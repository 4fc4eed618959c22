// Products over rows that are grouped by expert, on the tensor cores (tcgen05 + TMA).
//
// Row group e is [offsets[e], offsets[e+1]) of the row tensors (device memory: the host never
// learns the sizes); groups may be empty or of any length, so their borders fall inside tiles.
//   EXP_SWIGLU   h[r]  = silu(x[r] @ Wgate[e]) * (x[r] @ Wup[e]),   W[E, K, 2N] = [W_up | W_gate]
//   EXP_SAVE16   the same, and the pre-activations [up | gate] in bf16
//   EXP_SAVE8    the same, and the pre-activations in e4m3 with a power-of-two scale per row
//                and 32 columns (1 + 1/32 bytes for each value)
//   EXP_GEMM     c[r]  = a[r] @ B[e] or a[r] @ B[e]^T, stored in bf16 (EXP_GEMM32: in fp32)
//   EXP_GRAD16, EXP_GRAD8   the backward of the gate/up stage behind the down projection: the
//                product t = dy[r] @ Wdown[e]^T stays in the accumulator; the epilogue reads the
//                saved pre-activations and writes g = [w t silu(gate) | w t up silu'(gate)] and
//                w silu(gate) up, w the routing weight of the row's slot
//   EXP_WGRAD    C[e]  = a_e^T @ g_e   (the sum runs over the rows of the group; 0 if it is empty)
// With offsets == NULL there is one group of all rows (the dense stage's 8-bit checkpoints).
//
// h and the pre-activations' gradients are rounded to bf16, the operand type of the product that reads
// them next (fp32 operands would run at half its rate or less, as tf32); everything before that
// rounding and every sum is fp32.  Results then carry two roundings: 2.3e-3 to 2.5e-3 of their
// norm against 64 bits, where the last rounding alone makes 1.7e-3.
//
// Structure as the dense kernel's (swiglu_kernel.cuh): persistent CTAs (or CTA pairs on 256-row
// tiles, tcgen05 cta_group::2), warps 0 and 6 = TMA producers (A, B), warp 1 = MMA issuer, a
// 256-column fp32 accumulator in two TMEM stages.  The epilogue has eight warps, two for each 32
// rows, which share a staging buffer and split its columns: a sum over a few hundred ends before
// four warps have worked off a tile (the backward of 8000 rows, 1024 -> 512, in 8 bits: 25.9 us
// with four warps and TMA stores of its three results, 20.5 us so).  What the groups change:
//   * every CTA turns the offsets into a table of first tile rows once, and finds the expert
//     of a tile by bisection in it;
//   * an A tile whose rows run past its group takes them along in the operand (their
//     accumulator rows are not stored).  Up to 32 rows come in one or two boxes of 16, so a
//     group of one token does not fetch 128 rows; more come in one box of 128, because many
//     small boxes hold up the one thread that issues them (16384 rows over 8 uneven experts,
//     14336 -> 4096: 1.76 ms with boxes of 16 throughout, 1.38 ms so);
//   * the epilogue stores 32 whole rows with TMA; where a group ends inside them it copies the
//     rows that exist with plain stores, so that no row of another group is touched (forms with
//     three results store every row from the registers);
//   * EXP_WGRAD sums over rows, so rows past the group must not reach the MMA: whole steps of 16
//     are not issued, and where the group ends inside a step warp 7 waits for the operands to
//     land, overwrites the rest of the step with zeros (TMA cannot clip at a border inside the
//     tensor) and only then hands the block to the MMA issuer.
// Every wait is bounded, as everywhere in this library.
#pragma once

#include <cstdint>
#include <type_traits>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "ptx_sm100.cuh"
#include "swiglu_kernel.cuh"

namespace sgl {

enum : int {
  EXP_SWIGLU = 0, EXP_SAVE16 = 1, EXP_SAVE8 = 2, EXP_GEMM = 3, EXP_GEMM32 = 4, EXP_GRAD16 = 5,
  EXP_GRAD8 = 6, EXP_WGRAD = 7, EXP_FORMS = 8
};

constexpr int kExpThreads = 384;       // two producers, MMA issuer, tail warp, 8 epilogue warps
constexpr int kExpEpiWarps = 2 * kEpiWarps;
constexpr int kExpMaxStages = 16;
constexpr int kExpBarrierBytes = 8 * (3 * kExpMaxStages + 2 * kAccStages) + 32;
constexpr int kExpMaxGroups = 1024;

enum : unsigned {
  kErrExpProducerWait = 0x111,
  kErrExpMmaFullWait = 0x112,
  kErrExpMmaTmemWait = 0x113,
  kErrExpEpilogueWait = 0x114,
  kErrExpTailWait = 0x115,
};

struct ExpertMaps {
  CUtensorMap a;        // A operand, whole-tile box
  CUtensorMap a16;      // A operand, boxes of 16 rows (forward forms, few rows)
  CUtensorMap b;        // B operand
  CUtensorMap out;      // h / c / C (forms with three results store without maps)
  CUtensorMap up;       // EXP_SAVE8: codes, up half
  CUtensorMap gate;     // the same, gate half
};

struct ExpertParams {
  const int* offsets;   // [groups + 1] or NULL (one group of R rows)
  int groups;
  int R;                // rows of the row tensors
  int N, K;             // columns of the result; extent of the sum (forward forms)
  int M;                // EXP_WGRAD: rows of each C[e]
  int tiles_n;
  int group_m;          // tile rows walked together inside a group
  int stages;
  int acc_cols;         // accumulator columns of a tile (256; single-CTA tiles also 128)
  int splits;           // EXP_GEMM32: K is cut into ranges of k_per_split (a multiple of BLOCK_K),
  int k_per_split;      // range s of a row's sum goes to slot s of the result
  int a_rows;           // rows of an A slot: 128, or a multiple of 16 below it when R is small
  int b_kmajor;         // B[e] is stored [n, k] (multiplied transposed)
  __nv_bfloat16* out;   // forward forms: raw pointers for rows that end inside a warp's 32
  int64_t ld_out, slot_stride;   // elements
  uint8_t* pre;         // pre-activations or their gradients (written), gate half at + gate_off
  int64_t ld_pre;       // row pitch, bytes
  int64_t gate_off;     // bytes from the up half to the gate half of a row
  uint8_t* scales;      // 8-bit forms: [R][2][n_blocks] exponents + 127
  int64_t ld_scales;    // row pitch, bytes
  int64_t gate_scale_off;
  const uint8_t* saved; // EXP_GRAD*: the saved pre-activations, pitch and gate half as for pre
  int64_t ld_saved, saved_gate_off;
  const int* slots;     // EXP_GRAD*: slot of each row, for its routing weight; NULL: weights of 1
  const void* weights;  // fp32 or bf16 [T, k], row pitch ld_w
  int64_t ld_w, num_slots;
  int k, w_bf16;
  int l2_hints;
  unsigned long long wait_limit_ns;
};

template <int kForm, int kCtaGroup, int kBlockK>
struct ExpertTraits {
  static constexpr bool kSwiglu = kForm == EXP_SWIGLU || kForm == EXP_SAVE16 || kForm == EXP_SAVE8;
  static constexpr bool kGrad = kForm == EXP_GRAD16 || kForm == EXP_GRAD8;
  // three bf16 results of the same shape, stored without staging (see the epilogue)
  static constexpr bool kTriple = kForm == EXP_SAVE16 || kGrad;
  // staging of 32 rows: two 64-column chunks (of fp32: 32 columns), or one chunk with its 8-bit
  // pre-activations
  static constexpr int kStagingPerRows = kTriple ? 0 : 2 * kChunkBytes;
  static constexpr int kStagingBytes = kEpiWarps * kStagingPerRows;
  static constexpr int kBSlabsMax = kAccCols / kCtaGroup / 64;
  static constexpr int kBSlabBytes = kBlockK * 128;

  __host__ __device__ static constexpr int a_stage_bytes(int a_rows) { return a_rows * kBlockK * 2; }
  __host__ __device__ static constexpr int b_stage_bytes(int acc_cols) {
    return acc_cols / kCtaGroup * kBlockK * 2;
  }
  __host__ __device__ static constexpr int table_bytes(int groups) {
    return kForm == EXP_WGRAD ? 0 : ((groups + 1) * 4 + 15) / 16 * 16;
  }
  __host__ __device__ static constexpr int fixed_bytes(int groups) {
    return 1024 + kStagingBytes + kExpBarrierBytes + table_bytes(groups);
  }
  // An MMA reads 128 A rows whatever the slot holds: past the last A slot it reads B slots.
  __host__ __device__ static int max_stages(int groups, int a_rows, int acc_cols) {
    const int s = (227 * 1024 - fixed_bytes(groups)) / (a_stage_bytes(a_rows) + b_stage_bytes(acc_cols));
    return s > kExpMaxStages ? kExpMaxStages : s;
  }
  __host__ __device__ static int smem_bytes(int groups, int a_rows, int acc_cols, int stages) {
    return fixed_bytes(groups) + stages * (a_stage_bytes(a_rows) + b_stage_bytes(acc_cols));
  }
};

// ---------------------------------------------------------------- 8-bit blocks
//
// 32 values v share the scale 2^e, e the smallest integer (>= -127) with max|v| <= 448 * 2^e,
// 448 being the largest e4m3 value: nothing saturates.  A value is off by at most 2^-4 of itself or
// 2^-10 * 2^e (half a step below e4m3's smallest normal value, 2^-6), whichever is more.  The
// block's largest lies above 224 * 2^e unless e is held at -127, so the relative bound holds down
// to 2^-13 of it.  From the bits of the maximum m * 2^x (1 <= m < 2): e = x - 8, or x - 7 when
// m > 1.75; adding 0x1fffff to the bits carries into the exponent field exactly then.  The stored
// byte is e + 127; 255 stands for a block that holds an infinity or a NaN, and every value of it
// reads as NaN.
__device__ __forceinline__ int block_exponent_code(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits >= 0x7f800000u) return 255;
  const int field = static_cast<int>((bits + 0x1fffffu) >> 23) - 8;
  return field < 0 ? 0 : field;
}
// 2^(127 - code), the factor a value is multiplied by before it is rounded to e4m3.
__device__ __forceinline__ float block_inverse_scale(int code) {
  return __uint_as_float(static_cast<uint32_t>(254 - code) << 23);   // code <= 247: normal
}
// 2^(code - 127) (NaN for 255): code 0 is the subnormal 2^-127.
__device__ __forceinline__ float block_scale(int code) {
  if (code == 255) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(code == 0 ? 0x00400000u : static_cast<uint32_t>(code) << 23);
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
// Rounds 32 values; returns the scale code.
__device__ __forceinline__ int round_block_e4m3(const float (&v)[32], uint32_t (&codes)[8]) {
  // (the bits of |v| order like the values, and a NaN's lie above every number's)
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  const int code = block_exponent_code(__uint_as_float(top));
  const float inv = block_inverse_scale(code == 255 ? 127 : code);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    codes[i] = pack_e4m3x4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv,
                           v[4 * i + 3] * inv);
  return code;
}

// ---------------------------------------------------------------- extra PTX

__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* map, int x,
                                            int y, int z, uint32_t bar, uint64_t policy,
                                            bool peer_barrier) {
  if (peer_barrier) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        ".L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(smem_dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        ".L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(smem_dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
        : "memory");
  }
}

// ptx::umma_bf16 with the two descriptors as (low word, common high word).
template <int kCtaGroup>
__device__ __forceinline__ void umma_bf16_lohi(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                               uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kCtaGroup == 2) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p;\n\t"
        "}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t"
        "}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int x, int y, int z,
                                             uint32_t smem_src, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group.L2::cache_hint"
      " [%0, {%1, %2, %3}], [%4], %5;" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(x), "r"(y), "r"(z), "r"(smem_src), "l"(policy)
      : "memory");
}

// 32 lanes x 16 consecutive fp32 columns (see ptx::tmem_ld_32x32b_x32).
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
        "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}

// Barrier of the two warps that share a staging buffer; true if the predicate holds in all their
// threads.  Both always come here together, whatever their own waits said, so that neither is
// left behind.
__device__ __forceinline__ bool pair_barrier_all(int id, bool pred) {
  uint32_t all;
  asm volatile(
      "{\n\t"
      ".reg .pred p, r;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred r, %2, 64, p;\n\t"
      "selp.u32 %0, 1, 0, r;\n\t"
      "}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(pred)), "r"(id)
      : "memory");
  return all != 0;
}
__device__ __forceinline__ void pair_barrier(int id) {
  asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory");
}

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                             uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// 16 bf16 to 16 columns of one row: 32 bytes in one store where they are aligned (`wide`), else in
// two; `cols` (a multiple of 8) of them exist.
__device__ __forceinline__ void store_row16(__nv_bfloat16* at, const float (&v)[16], int cols,
                                            bool wide) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  if (wide && cols >= 16) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(at), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    if (cols >= 8) ptx::st_global_v4(at, w[0], w[1], w[2], w[3]);
    if (cols >= 16) ptx::st_global_v4(at + 8, w[4], w[5], w[6], w[7]);
  }
}

// Copies the first `rows` of 32 staged rows (row_bytes = 128 or 64 each, in the swizzle of a TMA
// box of that width) to global memory: `bytes` of each row, a multiple of 8.  The two warps of a
// pair together (lane 0 .. 63).
template <int kRowBytes>
__device__ __forceinline__ void copy_rows(uint32_t buf, uint8_t* dst, int64_t ld, int rows,
                                          int bytes, int lane) {
  constexpr int kPieces = kRowBytes / 16;
  for (int i = lane; i < rows * kPieces; i += 64) {
    const int r = i / kPieces, piece = i % kPieces;
    if (piece * 16 >= bytes) continue;
    const int sw = kRowBytes == 128 ? (r & 7) : ((r >> 1) & 3);
    const uint4 v = ld_shared_v4(buf + static_cast<uint32_t>(r * kRowBytes + ((piece ^ sw) << 4)));
    uint8_t* at = dst + r * ld + piece * 16;
    if (bytes - piece * 16 >= 16) {
      *reinterpret_cast<uint4*>(at) = v;
    } else {
      *reinterpret_cast<uint2*>(at) = make_uint2(v.x, v.y);
    }
  }
}

// Two e4m3 values (16 bits) as fp32.
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t two) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(two)));
  return __half22float2(*reinterpret_cast<__half2*>(&h2));
}

// 16 saved up and gate values of one row, columns x .. x + 15 (half a block; the halves of a row are
// padded to whole blocks, so the last one may be read past N), kept as loaded until they are used.
template <int kBits>
struct SavedHalfBlock {
  static constexpr int kLoads = 16 * kBits / 8 / 16;
  uint4 u[kLoads] = {}, g[kLoads] = {};
  int su = 0, sg = 0;
  __device__ __forceinline__ void load(const ExpertParams& p, int64_t row, int x, bool exists) {
    if (!exists) return;
    const uint8_t* at = p.saved + row * p.ld_saved + x * (kBits / 8);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      u[i] = reinterpret_cast<const uint4*>(at)[i];
      g[i] = reinterpret_cast<const uint4*>(at + p.saved_gate_off)[i];
    }
    if constexpr (kBits == 8) {
      const uint8_t* sc = p.scales + row * p.ld_scales + (x >> 5);
      su = sc[0];
      sg = sc[p.gate_scale_off];
    }
  }
  __device__ __forceinline__ void get(float (&up)[16], float (&gate)[16]) const {
    const float fu = kBits == 8 ? block_scale(su) : 1.f, fg = kBits == 8 ? block_scale(sg) : 1.f;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t wu[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
      const uint32_t wg[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kBits == 8) {
          const int o = j * 4;
          const float2 u0 = e4m3x2_to_f32(wu[j]), u1 = e4m3x2_to_f32(wu[j] >> 16);
          const float2 g0 = e4m3x2_to_f32(wg[j]), g1 = e4m3x2_to_f32(wg[j] >> 16);
          up[o] = u0.x * fu;
          up[o + 1] = u0.y * fu;
          up[o + 2] = u1.x * fu;
          up[o + 3] = u1.y * fu;
          gate[o] = g0.x * fg;
          gate[o + 1] = g0.y * fg;
          gate[o + 2] = g1.x * fg;
          gate[o + 3] = g1.y * fg;
        } else {
          const int o = i * 8 + j * 2;
          up[o] = __uint_as_float(wu[j] << 16);
          up[o + 1] = __uint_as_float(wu[j] & 0xffff0000u);
          gate[o] = __uint_as_float(wg[j] << 16);
          gate[o + 1] = __uint_as_float(wg[j] & 0xffff0000u);
        }
      }
    }
  }
};

// ---------------------------------------------------------------- the kernel

template <int kForm, int kCtaGroup, int kBlockK>
__global__ void __launch_bounds__(kExpThreads, 1)
experts_kernel(const __grid_constant__ ExpertMaps maps, const ExpertParams p) {
  using T = ExpertTraits<kForm, kCtaGroup, kBlockK>;
  constexpr bool kWgrad = kForm == EXP_WGRAD;
  constexpr bool kSwiglu = T::kSwiglu;
  constexpr int kTileRows = kBlockM * kCtaGroup;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = (kCtaGroup == 2) ? ptx::cluster_ctarank() : 0u;
  const int cluster_id = blockIdx.x / kCtaGroup;
  const int num_clusters = gridDim.x / kCtaGroup;
  const int stages = p.stages;
  const int a_stage = T::a_stage_bytes(p.a_rows);
  const int b_stage = T::b_stage_bytes(p.acc_cols);
  const int b_slabs = p.acc_cols / kCtaGroup / 64;
  const int tile_cols = kSwiglu ? p.acc_cols / 2 : p.acc_cols;

  // ---- shared memory ----
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  const uint32_t sA = smem_base;
  const uint32_t sB = sA + stages * a_stage;
  const uint32_t sOut = sB + stages * b_stage;
  const uint32_t sBar = sOut + T::kStagingBytes;
  const uint32_t bar_full = sBar;
  const uint32_t bar_empty = bar_full + 8 * kExpMaxStages;
  const uint32_t bar_land = bar_empty + 8 * kExpMaxStages;     // EXP_WGRAD: partial blocks
  const uint32_t bar_tfull = bar_land + 8 * kExpMaxStages;
  const uint32_t bar_tempty = bar_tfull + 8 * kAccStages;
  const uint32_t tmem_slot = bar_tempty + 8 * kAccStages;
  const uint32_t abort_slot = tmem_slot + 8;
  const uint32_t table = abort_slot + 24;
  volatile uint32_t* tmem_slot_ptr =
      reinterpret_cast<volatile uint32_t*>(smem_gen + (tmem_slot - smem_base));
  int* abort_flag = reinterpret_cast<int*>(smem_gen + (abort_slot - smem_base));
  int* tile_lo = reinterpret_cast<int*>(smem_gen + (table - smem_base));   // [groups + 1]

  if (threadIdx.x == 0) {
    abort_flag[0] = 0;
    abort_flag[1] = 0;
    for (int s = 0; s < stages; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 2 * kCtaGroup);   // one arrive.expect_tx per producer
      ptx::mbar_init(bar_empty + 8 * s, 1);
      ptx::mbar_init(bar_land + 8 * s, 2);
    }
    for (int s = 0; s < kAccStages; ++s) {
      ptx::mbar_init(bar_tfull + 8 * s, 1);
      ptx::mbar_init(bar_tempty + 8 * s, kExpEpiWarps * kCtaGroup);
    }
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&maps.a);
    ptx::prefetch_tensormap(&maps.b);
    if (!T::kTriple) ptx::prefetch_tensormap(&maps.out);
  }
  if (warp == 1) ptx::tmem_alloc<kCtaGroup>(tmem_slot, kTmemCols);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- the groups: first row (clamped: rows that do not exist in the row tensors are never
  // addressed, whatever the offsets say), and a table of first tile rows ----
  const int G = p.groups;
  auto row_lo = [&](int e) {
    if (p.offsets == nullptr) return e == 0 ? 0 : p.R;
    const int lo = p.offsets[e];   // (written by a kernel this one may have started beside: no ld.nc)
    return lo < 0 ? 0 : (lo > p.R ? p.R : lo);
  };
  if constexpr (!kWgrad) {
    for (int e = threadIdx.x; e < G; e += kExpThreads) {
      const int n = row_lo(e + 1) - row_lo(e);
      tile_lo[e] = n > 0 ? (n + kTileRows - 1) / kTileRows : 0;
    }
    __syncthreads();
    if (warp == 0) {
      // exclusive sums in place: each lane a run of groups, then over the lanes
      const int per = (G + 31) / 32;
      const int e0 = lane * per, e1 = (e0 + per < G) ? e0 + per : G;
      int mine = 0;
      for (int e = e0; e < e1; ++e) mine += tile_lo[e];
      int inc = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += v;
      }
      int at = inc - mine;
      for (int e = e0; e < e1; ++e) {
        const int n = tile_lo[e];
        tile_lo[e] = at;
        at += n;
      }
      if (lane == 31) tile_lo[G] = inc;
    }
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (kCtaGroup == 2) ptx::cluster_sync();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_ptr;

  const int wgrad_tiles_m = kWgrad ? (p.M + kTileRows - 1) / kTileRows : 0;
  const int splits = kForm == EXP_GEMM32 ? p.splits : 1;
  const int total_units = (kWgrad ? wgrad_tiles_m * G : tile_lo[G]) * p.tiles_n * splits;

  struct Unit {
    int e;          // group
    int row;        // forward: first row of the tile; EXP_WGRAD: first row of the group
    int rows;       // forward: rows from there to the group's end; EXP_WGRAD: rows of the group
    int m, n;       // EXP_WGRAD: first row of C[e]; first column of the result
    int k0;         // EXP_GEMM32: first of the range of the sum
  };
  auto unit_of = [&](int u) {
    Unit r;
    const int tm = u / (p.tiles_n * splits);
    r.k0 = 0;
    if constexpr (kWgrad) {
      r.e = tm / wgrad_tiles_m;
      const TileCoord tc = tile_coord(u - r.e * wgrad_tiles_m * p.tiles_n, wgrad_tiles_m,
                                      p.tiles_n, p.group_m);
      r.row = row_lo(r.e);
      r.rows = row_lo(r.e + 1) - r.row;
      if (r.rows < 0) r.rows = 0;
      r.m = tc.m * kTileRows;
      r.n = tc.n * tile_cols;
    } else {
      int lo = 0, hi = G;    // the group whose tile rows contain tm
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tile_lo[mid] <= tm) lo = mid; else hi = mid;
      }
      r.e = lo;
      const int tiles_m = tile_lo[lo + 1] - tile_lo[lo];
      int t = u - tile_lo[lo] * p.tiles_n * splits;
      if (splits > 1) {
        // all tiles of a group for one range of the sum, then the next range: neighbouring CTAs
        // read neighbouring columns
        const int range = t / (tiles_m * p.tiles_n);
        t -= range * tiles_m * p.tiles_n;
        r.k0 = range * p.k_per_split;
      }
      const TileCoord tc = tile_coord(t, tiles_m, p.tiles_n, p.group_m);
      r.row = row_lo(lo) + tc.m * kTileRows;
      r.rows = row_lo(lo + 1) - r.row;
      r.m = 0;
      r.n = tc.n * tile_cols;
    }
    return r;
  };
  // extent of a unit's sum, and its k-blocks
  auto unit_len = [&](const Unit& un) {
    if constexpr (kWgrad) return un.rows;
    if (splits > 1) return p.K - un.k0 < p.k_per_split ? p.K - un.k0 : p.k_per_split;
    return p.K;
  };
  auto unit_kb = [&](const Unit& un) { return (unit_len(un) + kBlockK - 1) / kBlockK; };
  // EXP_WGRAD: whether block kb holds rows behind the group inside a step of 16 that is used
  auto mixed_block = [&](const Unit& un, int kb) {
    return kWgrad && un.rows - kb * kBlockK < kBlockK && (un.rows & 15) != 0;
  };

  const uint64_t limit = p.wait_limit_ns;

  // =========================== TMA producers ===========================
  // One thread each for the A and the B operand: a copy takes its thread about 230 cycles to
  // issue, and a k-block of 128 has four to six of them, more than the tensor core needs.
  auto produce = [&](auto operand) {
    constexpr bool kA = decltype(operand)::value == 0;
    const uint64_t policy = ptx::make_l2_policy((p.l2_hints >> (kA ? 0 : 2)) & 3);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    Unit next;
    if (cluster_id < total_units) next = unit_of(cluster_id);
    for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
      const Unit un = next;
      const int num_kb = unit_kb(un);
      if (num_kb == 0 && u + num_clusters < total_units) next = unit_of(u + num_clusters);
      // forward: rows of this CTA's half of the tile, and the boxes that cover them
      int left = un.rows - static_cast<int>(rank) * kBlockM;
      left = left < 0 ? 0 : (left > kBlockM ? kBlockM : left);
      [[maybe_unused]] const int my_row = un.row + static_cast<int>(rank) * kBlockM;
      const bool whole = left > 32 && p.a_rows == kBlockM;
      const int boxes16 = (left + 15) / 16;
      const uint32_t tx = static_cast<uint32_t>(
          kA ? (kWgrad || whole ? kBlockM : boxes16 * 16) * kBlockK * 2 : b_slabs * T::kBSlabBytes);
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!ptx::mbar_wait(bar_empty + 8 * s, ph ^ 1u, limit, abort_flag)) {
          report_error(kErrExpProducerWait, kb, abort_flag);
          ok = false;
          break;
        }
        const int k0 = un.k0 + kb * kBlockK;
        const uint32_t full_local = bar_full + 8 * s;
        uint32_t bar = (kCtaGroup == 2) ? ptx::mapa(full_local, 0) : full_local;
        bool peer = kCtaGroup == 2;
        if (SGL_DBG_COORD_BAD(un.row >= 0 && un.row < p.R && un.e >= 0 && un.e < G &&
                                  (un.n & 7) == 0 && un.n < p.N && un.m >= 0,
                              kb)) {
          *reinterpret_cast<volatile int*>(abort_flag) = 1;
          ok = false;
          break;
        }
        if constexpr (kWgrad) {
          // a block that the group ends in reports to this CTA's own barrier: the tail warp
          // clears the rows behind the group and passes the block on
          if (mixed_block(un, kb)) {
            bar = bar_land + 8 * s;
            peer = false;
          }
        }
        ptx::mbar_arrive_expect_tx_cluster(bar, tx);
        if constexpr (kWgrad) {
          constexpr int kSlabs = kA ? kBlockM / 64 : T::kBSlabsMax;
          const CUtensorMap* map = kA ? &maps.a : &maps.b;
          const uint32_t dst = kA ? sA + s * a_stage : sB + s * b_stage;
          const int x0 = kA ? un.m + static_cast<int>(rank) * kBlockM
                            : un.n + static_cast<int>(rank) * b_slabs * 64;
#pragma unroll
          for (int j = 0; j < kSlabs; ++j) {
            if (!kA && j >= b_slabs) break;
            if (peer) {
              ptx::tma_load_2d<true>(dst + j * (kBlockK * 128), map, x0 + j * 64, un.row + k0, bar,
                                     policy);
            } else {
              ptx::tma_load_2d<false>(dst + j * (kBlockK * 128), map, x0 + j * 64, un.row + k0, bar,
                                      policy);
            }
          }
        } else if constexpr (kA) {
          const uint32_t a_dst = sA + s * a_stage;
#pragma unroll
          for (int j = 0; j < kBlockK / 64; ++j) {
            const uint32_t dst = a_dst + j * (p.a_rows * 128);
            if (whole) {
              ptx::tma_load_2d<kCtaGroup == 2>(dst, &maps.a, k0 + j * 64, my_row, bar, policy);
            } else {
              for (int i = 0; i < boxes16; ++i)
                ptx::tma_load_2d<kCtaGroup == 2>(dst + i * (16 * 128), &maps.a16, k0 + j * 64,
                                                 my_row + i * 16, bar, policy);
            }
          }
        } else {
          const uint32_t b_dst = sB + s * b_stage;
          if (p.b_kmajor) {
            // B[e] stored [n, k]: boxes of 64 n-rows x 64 k, one 64-k slice of all this CTA's
            // rows contiguous
#pragma unroll
            for (int j = 0; j < kBlockK / 64; ++j) {
              for (int i = 0; i < b_slabs; ++i) {
                const int row = un.n + (static_cast<int>(rank) * b_slabs + i) * 64;
                tma_load_3d(b_dst + j * (b_slabs * 64 * 128) + i * (64 * 128), &maps.b, k0 + j * 64,
                            row, un.e, bar, policy, peer);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < T::kBSlabsMax; ++j) {
              if (j >= b_slabs) break;
              const int g = static_cast<int>(rank) * b_slabs + j;   // slab of the tile
              int col = un.n + g * 64;
              if constexpr (kSwiglu) {
                // the first half of the accumulator is up, the second gate
                const int half = p.acc_cols / 128;
                col = g < half ? un.n + g * 64 : p.N + un.n + (g - half) * 64;
              }
              tma_load_3d(b_dst + j * T::kBSlabBytes, &maps.b, col, k0, un.e, bar, policy, peer);
            }
          }
        }
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
        // the next tile is looked up while this one's loads are under way
        if (kb == 0 && u + num_clusters < total_units) next = unit_of(u + num_clusters);
      }
    }
    if (!ok) {
      // loads in flight land before the CTA exits
      const uint64_t t0 = ptx::globaltimer_ns();
      while (ptx::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
  };

  if (warp == 0) {
    if (lane == 0) produce(std::integral_constant<int, 0>{});
  } else if (warp == 6) {
    if (lane == 0) produce(std::integral_constant<int, 1>{});
  } else if (warp == 1) {
    // =========================== MMA issuer ===========================
    if (rank == 0 && lane == 0) {
      const uint32_t idesc =
          ptx::make_idesc_bf16(kTileRows, p.acc_cols, /*a_mn_major=*/kWgrad,
                               /*b_mn_major=*/p.b_kmajor == 0);
      const bool b_kmajor = p.b_kmajor != 0;
      // Shared-memory descriptors by halves, in units of 16 bytes: only the low word (address and
      // leading-dimension offset) changes from MMA to MMA, by constants; putting the 64-bit
      // descriptors together for each MMA kept the issuing thread busy for about 100 cycles.
      const uint64_t desc0 = ptx::smem_desc_sw128(0, 0, 1024);
      const uint32_t desc_hi = static_cast<uint32_t>(desc0 >> 32);
      const uint32_t a_lo0 = static_cast<uint32_t>(
          ptx::smem_desc_sw128(sA, kWgrad ? kBlockK * 128 : 16, 1024));
      const uint32_t b_lo0 = static_cast<uint32_t>(
          ptx::smem_desc_sw128(sB, b_kmajor ? 16 : T::kBSlabBytes, 1024));
      const uint32_t a_step = static_cast<uint32_t>(a_stage) >> 4;
      const uint32_t b_step = static_cast<uint32_t>(b_stage) >> 4;
      const uint32_t a_box = static_cast<uint32_t>(p.a_rows) * 8u;      // one 64-deep box of A
      const uint32_t b_box = static_cast<uint32_t>(b_slabs) * 512u;     // the same of B, K-major
      constexpr uint16_t mask = (kCtaGroup == 2) ? 0x3 : 0x1;
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      int i = 0;
      Unit next;
      if (cluster_id < total_units) next = unit_of(cluster_id);
      for (int u = cluster_id; u < total_units && ok; u += num_clusters, ++i) {
        const Unit un = next;
        if (unit_kb(un) == 0 && u + num_clusters < total_units) next = unit_of(u + num_clusters);
        const int as = i % kAccStages;
        const uint32_t aph = (i / kAccStages) & 1u;
        if (!ptx::mbar_wait(bar_tempty + 8 * as, aph ^ 1u, limit, abort_flag)) {
          report_error(kErrExpMmaTmemWait, i, abort_flag);
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + as * kAccCols;
        const int num_kb = unit_kb(un);
        const int last_steps = (unit_len(un) - (num_kb - 1) * kBlockK + 15) / 16;
        for (int kb = 0; kb < num_kb; ++kb) {
          // (a block that passed through the peer's tail warp carries its ordinary writes)
          const bool landed =
              (kCtaGroup == 2 && mixed_block(un, kb))
                  ? ptx::mbar_wait_acquire_cluster(bar_full + 8 * s, ph, limit, abort_flag)
                  : ptx::mbar_wait(bar_full + 8 * s, ph, limit, abort_flag);
          if (!landed) {
            report_error(kErrExpMmaFullWait, kb, abort_flag);
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t a_lo = a_lo0 + static_cast<uint32_t>(s) * a_step;
          const uint32_t b_lo = b_lo0 + static_cast<uint32_t>(s) * b_step;
          auto step = [&](int kk) {
            // 16 of the sum further: 32 bytes inside the 128-byte rows of a K-major operand (the
            // next 64 in the next box), 16 rows of an MN-major one
            const uint32_t a_off = kWgrad ? kk * 128u : (kk >> 2) * a_box + (kk & 3) * 2u;
            const uint32_t b_off = b_kmajor ? (kk >> 2) * b_box + (kk & 3) * 2u : kk * 128u;
            umma_bf16_lohi<kCtaGroup>(d_tmem, a_lo + a_off, b_lo + b_off, desc_hi, idesc,
                                      (kb > 0 || kk > 0) ? 1u : 0u);
          };
          if (kb < num_kb - 1 || last_steps == kBlockK / 16) {
#pragma unroll
            for (int kk = 0; kk < kBlockK / 16; ++kk) step(kk);
          } else {
            // the last block is padded (zero fill from TMA, or rows that the tail warp cleared
            // up to a whole step): only the steps the sum still has
#pragma unroll 1
            for (int kk = 0; kk < last_steps; ++kk) step(kk);
          }
          ptx::umma_commit<kCtaGroup>(bar_empty + 8 * s, mask);
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
          }
          if (kb == 0 && u + num_clusters < total_units) next = unit_of(u + num_clusters);
        }
        if (ok) ptx::umma_commit<kCtaGroup>(bar_tfull + 8 * as, mask);
      }
    }
  } else if (warp == 7) {
    // =========================== tail warp (EXP_WGRAD) ===========================
    if constexpr (kWgrad) {
      // Walks the same sequence of blocks as the producer; acts on the ones a group ends in.
      // The landing barrier of a slot completes a phase only for such blocks: its parity is
      // counted (one bit per slot), not derived from the ring's.
      uint32_t parities = 0;
      int64_t block = 0;    // blocks before this unit's first
      for (int u = cluster_id; u < total_units; u += num_clusters) {
        const Unit un = unit_of(u);
        const int num_kb = unit_kb(un);
        if (num_kb > 0 && mixed_block(un, num_kb - 1)) {
          const int valid = un.rows - (num_kb - 1) * kBlockK;    // rows of the last block
          const int64_t b = block + num_kb - 1;
          const int s = static_cast<int>(b % stages);
          const bool landed =
              ptx::mbar_wait(bar_land + 8 * s, (parities >> s) & 1u, limit, abort_flag);
          if (!__all_sync(0xffffffffu, landed)) {
            if (lane == 0) report_error(kErrExpTailWait, num_kb, abort_flag);
            break;
          }
          parities ^= 1u << s;
          // rows from `valid` to the end of their step of 16 in every 64-column slab: whole
          // 128-byte rows (the swizzle moves 16-byte pieces only inside a row)
          const uint32_t a0 = sA + s * a_stage, b0 = sB + s * b_stage;
          const int pieces = (16 - (valid & 15)) * 8;
          for (int slab = 0; slab < kBlockM / 64 + b_slabs; ++slab) {
            const uint32_t at = (slab < kBlockM / 64 ? a0 + slab * (kBlockK * 128)
                                                     : b0 + (slab - kBlockM / 64) * T::kBSlabBytes) +
                                static_cast<uint32_t>(valid) * 128u;
            for (int i = lane; i < pieces; i += 32) st_shared_v4(at + i * 16, 0, 0, 0, 0);
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane < 2) {   // for both producers
            const uint32_t full_local = bar_full + 8 * s;
            if constexpr (kCtaGroup == 2) {
              ptx::mbar_arrive_release_cluster(ptx::mapa(full_local, 0));
            } else {
              ptx::mbar_arrive(full_local);
            }
          }
          __syncwarp();
        }
        block += num_kb;
      }
    }
  } else {
    // =========================== epilogue ===========================
    const int q = warp & 3;                 // TMEM lane quarter: 32 rows, shared by two warps ...
    const int g = warp >= 8 ? 1 : 0;        // ... that own the first and the second half of the
    const bool issuer = g == 0 && lane == 0;   // columns of every staged chunk
    const int pair = 1 + q;                 // their named barrier
    const int pair_lane = g * 32 + lane;
    const uint32_t buf0 = sOut + q * T::kStagingPerRows;
    const uint32_t tempty = (kCtaGroup == 2) ? ptx::mapa(bar_tempty, 0) : bar_tempty;
    const uint32_t row_sw = static_cast<uint32_t>(lane & 7);
    const uint32_t row_off = static_cast<uint32_t>(lane) * 128u;
    const uint32_t off64 = static_cast<uint32_t>(lane) * 64u;          // 64-byte rows
    const uint32_t sw64 = (static_cast<uint32_t>(lane) >> 1) & 3u;
    const uint64_t pol_out = ptx::make_l2_policy((p.l2_hints >> 4) & 3);
    const int gate_col = p.acc_cols / 2;
    int stores = 0;       // staging buffers filled so far
    int i = 0;
    for (int u = cluster_id; u < total_units; u += num_clusters, ++i) {
      const Unit un = unit_of(u);
      const int as = i % kAccStages;
      const uint32_t aph = (i / kAccStages) & 1u;
      // these 32 rows of the tile, and how many of them exist
      const int in_tile = static_cast<int>(rank) * kBlockM + q * 32;
      int valid = (kWgrad ? p.M - un.m : un.rows) - in_tile;
      valid = valid < 0 ? 0 : (valid > 32 ? 32 : valid);
      const int64_t grow = un.row + in_tile;       // forward forms: first row in the row tensors
      const bool live = lane < valid;
      // EXP_GRAD*: the first saved values and the routing weight come in while the product is
      // still being made, later ones two chunks before they are used (18000 rows of 128 experts,
      // 768 -> 256: 31.1 us one chunk ahead, 28.8 two, 29.5 three)
      constexpr int kAhead = T::kGrad ? 2 : 1;
      SavedHalfBlock<kForm == EXP_GRAD8 ? 8 : 16> saved[kAhead];
      float weight = 1.0f;
      if constexpr (T::kGrad) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int x = un.n + j * 32 + g * 16;
          saved[j].load(p, grow + lane, x, live && j * 32 < tile_cols && un.n + j * 32 < p.N);
        }
        if (p.slots != nullptr && live) {
          const int64_t slot = p.slots[grow + lane];
          weight = 0.f;
          if (slot >= 0 && slot < p.num_slots) {
            const int64_t at = slot / p.k * p.ld_w + slot % p.k;
            weight = p.w_bf16
                         ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.weights)[at])
                         : reinterpret_cast<const float*>(p.weights)[at];
          }
        }
      }
      const bool w = ptx::mbar_wait(bar_tfull + 8 * as, aph, limit, abort_flag);
      __syncwarp();
      if (!pair_barrier_all(pair, w)) {
        if (lane == 0) report_error(kErrExpEpilogueWait, i, abort_flag);
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + as * kAccCols;
      auto hand_back = [&]() {
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(tempty + 8 * as);
      };
      if (valid == 0) {
        hand_back();
        continue;
      }
      // Before a staging buffer is written the store that used it has to have read it (kPending
      // younger ones may still be under way), and rows copied out by hand have to be out.
      auto buffer_free = [&](auto pending) {
        if (issuer) ptx::bulk_wait_group_read<decltype(pending)::value>();
        __syncwarp();
        pair_barrier(pair);
      };
      // Both warps' halves are in place (and, for TMA, visible to the asynchronous proxy).
      auto buffer_full = [&]() {
        ptx::fence_proxy_async_smem();
        __syncwarp();
        pair_barrier(pair);
      };
      if constexpr (T::kTriple) {
        // ---- three bf16 results, 32 columns at a time, 16 for each warp, straight from the
        // registers: a thread's 32 bytes of a row are a whole sector ----
        __nv_bfloat16* const row_h = p.out + (grow + lane) * p.ld_out;
        __nv_bfloat16* const row_up =
            reinterpret_cast<__nv_bfloat16*>(p.pre + (grow + lane) * p.ld_pre);
        __nv_bfloat16* const row_gate = reinterpret_cast<__nv_bfloat16*>(
            reinterpret_cast<uint8_t*>(row_up) + p.gate_off);
        const bool wide_h = (reinterpret_cast<uintptr_t>(row_h) & 31) == 0;
        const bool wide_pre = ((reinterpret_cast<uintptr_t>(row_up) |
                                reinterpret_cast<uintptr_t>(row_gate)) & 31) == 0;
        const int units = tile_cols / 32;
        for (int c0 = 0; c0 < units; c0 += kAhead) {
#pragma unroll
          for (int j0 = 0; j0 < kAhead; ++j0) {
            const int c = c0 + j0;
            if (c >= units) break;
            __syncwarp();             // the TMEM reads below are the whole warp's
            const int x = un.n + c * 32;
            const bool last = c == units - 1;
            if (x >= p.N) {
              if (last) hand_back();
              continue;
            }
            const int col = c * 32 + g * 16;
            float a[16], b[16], h[16];
            if constexpr (kForm == EXP_SAVE16) {
              tmem_ld_32x32b_x16(t_row + col, a);
              tmem_ld_32x32b_x16(t_row + gate_col + col, b);
              ptx::tmem_ld_wait();
              if (last) hand_back();
#pragma unroll
              for (int j = 0; j < 16; ++j) h[j] = silu_mul(b[j], a[j]);
            } else {
              // this row's saved up and gate values, then the gradients in their place
              saved[j0].get(a, b);
              saved[j0].load(p, grow + lane, x + kAhead * 32 + g * 16,
                             live && c + kAhead < units && x + kAhead * 32 < p.N);
              tmem_ld_32x32b_x16(t_row + col, h);
              ptx::tmem_ld_wait();
              if (last) hand_back();
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                float hv, sv, dv;
                silu_factors(b[j], a[j], hv, sv, dv);
                const float t = weight * h[j];
                a[j] = t * sv;
                b[j] = t * dv;
                h[j] = weight * hv;
              }
            }
            if (live) {
              const int xc = x + g * 16;
              store_row16(row_h + xc, h, p.N - xc, wide_h);
              store_row16(row_up + xc, a, p.N - xc, wide_pre);
              store_row16(row_gate + xc, b, p.N - xc, wide_pre);
            }
          }
        }
      } else if constexpr (kForm == EXP_GEMM32) {
        // ---- fp32 result, 32 columns at a time (16 for each warp), two buffers ----
        const int units = tile_cols / 32;
        const int slot = splits > 1 ? un.k0 / p.k_per_split : 0;
        for (int c = 0; c < units; ++c) {
          const int x = un.n + c * 32;
          const bool last = c == units - 1;
          if (x >= p.N) {
            if (last) hand_back();
            continue;
          }
          const uint32_t buf = buf0 + (stores & 1) * kChunkBytes;
          ++stores;
          float v[16];
          tmem_ld_32x32b_x16(t_row + c * 32 + g * 16, v);
          ptx::tmem_ld_wait();
          if (last) hand_back();
          buffer_free(std::integral_constant<int, 1>{});
#pragma unroll
          for (int j = 0; j < 4; ++j)
            st_shared_v4(buf + row_off + ((static_cast<uint32_t>(g * 4 + j) ^ row_sw) << 4),
                         __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                         __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
          buffer_full();
          if (valid == 32) {
            if (issuer) tma_store_3d(&maps.out, x, static_cast<int>(grow), slot, buf, pol_out);
          } else {
            copy_rows<128>(buf,
                           reinterpret_cast<uint8_t*>(reinterpret_cast<float*>(p.out) +
                                                      slot * p.slot_stride + grow * p.ld_out + x),
                           p.ld_out * 4, valid, (p.N - x < 32 ? p.N - x : 32) * 4, pair_lane);
          }
          if (issuer) ptx::bulk_commit_group();   // keeps the buffers' turn-taking in step
        }
      } else {
        // ---- one bf16 result, 64 columns at a time, 32 for each warp (EXP_SAVE8: with its 8-bit
        // pre-activations, of which a warp's 32 columns are one block) ----
        const int chunks = tile_cols / 64;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          const int x = un.n + c * 64;
          const bool last = c == chunks - 1;
          if (x >= p.N) {
            if (last) hand_back();
            continue;
          }
          uint32_t buf = buf0;
          if constexpr (kForm != EXP_SAVE8) buf = buf0 + (stores & 1) * kChunkBytes;
          ++stores;
          const int col = c * 64 + g * 32;
          float v0[32];
          ptx::tmem_ld_32x32b_x32(t_row + col, v0);
          uint32_t up_codes[8], gate_codes[8];
          int up_scale = 0, gate_scale = 0;
          if constexpr (kSwiglu) {
            float gate[32];
            ptx::tmem_ld_32x32b_x32(t_row + gate_col + col, gate);
            ptx::tmem_ld_wait();
            if (last) hand_back();
            if constexpr (kForm == EXP_SAVE8) {
              // columns at and past N hold sums over nothing (the operand reads as zero there,
              // or as the gate half's weights): they do not belong to the block
              const int n_left = p.N - (x + g * 32);
              if (n_left < 32) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  v0[j] = j < n_left ? v0[j] : 0.f;
                  gate[j] = j < n_left ? gate[j] : 0.f;
                }
              }
              up_scale = round_block_e4m3(v0, up_codes);
              gate_scale = round_block_e4m3(gate, gate_codes);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v0[j] = silu_mul(gate[j], v0[j]);
          } else {
            ptx::tmem_ld_wait();
            if (last) hand_back();
            if constexpr (kWgrad) {
              if (un.rows == 0) {       // a sum over nothing: the accumulator was not written
#pragma unroll
                for (int j = 0; j < 32; ++j) v0[j] = 0.f;
              }
            }
          }
          if constexpr (kForm == EXP_SAVE8) {
            buffer_free(std::integral_constant<int, 0>{});
          } else {
            buffer_free(std::integral_constant<int, 1>{});
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            st_shared_v4(buf + row_off + ((static_cast<uint32_t>(g * 4 + j) ^ row_sw) << 4),
                         pack_bf16x2(v0[8 * j], v0[8 * j + 1]),
                         pack_bf16x2(v0[8 * j + 2], v0[8 * j + 3]),
                         pack_bf16x2(v0[8 * j + 4], v0[8 * j + 5]),
                         pack_bf16x2(v0[8 * j + 6], v0[8 * j + 7]));
          if constexpr (kForm == EXP_SAVE8) {
            const uint32_t ubuf = buf + kChunkBytes, gbuf = ubuf + kChunkBytes / 2;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t off = off64 + ((static_cast<uint32_t>(g * 2 + j) ^ sw64) << 4);
              st_shared_v4(ubuf + off, up_codes[4 * j], up_codes[4 * j + 1], up_codes[4 * j + 2],
                           up_codes[4 * j + 3]);
              st_shared_v4(gbuf + off, gate_codes[4 * j], gate_codes[4 * j + 1],
                           gate_codes[4 * j + 2], gate_codes[4 * j + 3]);
            }
            if (lane < valid) {
              // this row's scale of the block (the pitch has room for a whole chunk)
              uint8_t* at = p.scales + (grow + lane) * p.ld_scales + (x >> 5) + g;
              at[0] = static_cast<uint8_t>(up_scale);
              at[p.gate_scale_off] = static_cast<uint8_t>(gate_scale);
            }
          }
          buffer_full();
          if (kWgrad || valid == 32) {
            if (issuer) {
              if constexpr (kWgrad) {
                tma_store_3d(&maps.out, x, un.m + in_tile, un.e, buf, pol_out);
              } else {
                const int y = static_cast<int>(grow);
                ptx::tma_store_2d(&maps.out, x, y, buf, pol_out);
                if constexpr (kForm == EXP_SAVE8) {
                  ptx::tma_store_2d(&maps.up, x, y, buf + kChunkBytes, pol_out);
                  ptx::tma_store_2d(&maps.gate, x, y, buf + kChunkBytes + kChunkBytes / 2, pol_out);
                }
              }
            }
          } else {
            const int cols = p.N - x < 64 ? p.N - x : 64;
            copy_rows<128>(buf, reinterpret_cast<uint8_t*>(p.out + grow * p.ld_out + x),
                           p.ld_out * 2, valid, cols * 2, pair_lane);
            if constexpr (kForm == EXP_SAVE8) {
              uint8_t* at = p.pre + grow * p.ld_pre + x;
              copy_rows<64>(buf + kChunkBytes, at, p.ld_pre, valid, cols, pair_lane);
              copy_rows<64>(buf + kChunkBytes + kChunkBytes / 2, at + p.gate_off, p.ld_pre, valid,
                            cols, pair_lane);
            }
          }
          if (issuer) ptx::bulk_commit_group();    // keeps the buffers' turn-taking in step
        }
      }
    }
    if (issuer) ptx::bulk_wait_group_read<0>();
  }

  // ---- teardown ----
  __syncwarp();
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (kCtaGroup == 2) ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<kCtaGroup>(tmem_base, kTmemCols);
  }
}

}  // namespace sgl
