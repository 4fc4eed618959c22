// Backward elementwise step of the SwiGLU stage from saved pre-activations [up | gate]:
//   grad_preact[:, 0:N]  = dy * silu(gate)        grad_preact[:, N:2N] = dy * up * silu'(gate)
//   h                    = silu(gate) * up        (optional: the down projection's weight
//                                                  gradient needs it again)
// kBits = 8: e4m3 codes with a power-of-two scale per row and 32 columns; kBits = 16: bf16.
//
// HBM bound: a row costs 2N (dy) + 2N + N/16 (codes and scales; 4N for bf16) bytes read and 4N
// (+ 2N with h) written.  One thread owns 8 columns of both halves.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "experts_order.cuh"
#include "experts_products.cuh"

namespace sgl {

struct PreactParams {
  const __nv_bfloat16* dy;
  const uint8_t* pre;          // row pitch ld_pre bytes, gate half at + gate_off bytes
  const uint8_t* scales;       // kBits = 8: row pitch ld_scales, gate half at + gate_scale_off
  __nv_bfloat16* grad;         // [rows, 2N]
  __nv_bfloat16* h;            // [rows, N] or NULL
  const int* end;              // device: rows that exist (at most `rows`), or NULL = all
  int64_t lddy, ld_pre, gate_off, ld_scales, gate_scale_off, ld_grad, ldh;
  int64_t rows;
  int nvec;                    // N / 8
};

__device__ __forceinline__ void e4m3x8_to_f32(uint2 c, float scale, float (&f)[8]) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = e4m3x2_to_f32(w[i >> 1] >> (16 * (i & 1)));
    f[2 * i] = v.x * scale;
    f[2 * i + 1] = v.y * scale;
  }
}

template <int kBits>
__global__ void __launch_bounds__(256) grad_preact_saved_kernel(const PreactParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int64_t rows = p.rows;
  if (p.end) {
    const int64_t e = *p.end;
    rows = e < 0 ? 0 : (e < rows ? e : rows);
  }
  const int64_t total = rows * p.nvec;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += stride) {
    const int64_t row = i / p.nvec;
    const int v = static_cast<int>(i - row * p.nvec);
    const uint4 g = reinterpret_cast<const uint4*>(p.dy + row * p.lddy)[v];
    float up[8], gate[8], dy[8];
    const uint8_t* pre = p.pre + row * p.ld_pre;
    if constexpr (kBits == 8) {
      const uint2 cu = reinterpret_cast<const uint2*>(pre)[v];
      const uint2 cg = reinterpret_cast<const uint2*>(pre + p.gate_off)[v];
      const uint8_t* sc = p.scales + row * p.ld_scales + (v >> 2);
      const int su = sc[0], sg = sc[p.gate_scale_off];
      e4m3x8_to_f32(cu, block_scale(su), up);
      e4m3x8_to_f32(cg, block_scale(sg), gate);
    } else {
      const uint4 cu = reinterpret_cast<const uint4*>(pre)[v];
      const uint4 cg = reinterpret_cast<const uint4*>(pre + p.gate_off)[v];
      bf16x8_to_f32(cu, up);
      bf16x8_to_f32(cg, gate);
    }
    bf16x8_to_f32(g, dy);
    float h[8], gu[8], gg[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s, d;
      silu_factors(gate[j], up[j], h[j], s, d);
      gu[j] = dy[j] * s;
      gg[j] = dy[j] * d;
    }
    __nv_bfloat16* out = p.grad + row * p.ld_grad;
    reinterpret_cast<uint4*>(out)[v] = f32_to_bf16x8(gu);
    reinterpret_cast<uint4*>(out)[p.nvec + v] = f32_to_bf16x8(gg);
    if (p.h) reinterpret_cast<uint4*>(p.h + row * p.ldh)[v] = f32_to_bf16x8(h);
  }
}

}  // namespace sgl
