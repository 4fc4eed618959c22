// Backward elementwise step of the SwiGLU stage from saved pre-activations [up | gate]:
//   grad_preact[:, 0:N]  = dy * silu(gate)        grad_preact[:, N:2N] = dy * up * silu'(gate)
//   h                    = silu(gate) * up        (optional: the down projection's weight
//                                                  gradient needs it again)
// kBits = 8: e4m3 codes with a power-of-two scale per row and 32 columns; kBits = 16: bf16.
//
// HBM bound: a row costs 2N (dy) + 2N + N/16 (codes and scales; 4N for bf16) bytes read and 4N
// (+ 2N with h) written.  A thread owns kVecs times 8 columns and walks down the rows, two at a
// time, so that the loads of both are in flight (16384 x 14336 in 8 bits without h: 292 us,
// 6.5 TB/s; one row of 8 columns at a time took 455 us).
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "experts_order.cuh"
#include "experts_products.cuh"

namespace sgl {

constexpr int kPreactThreads = 128;

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

// 8 saved values as loaded.
template <int kBits>
struct SavedVec {
  uint4 v;                     // 8 bits: x, y
  __device__ __forceinline__ void load(const uint8_t* row, int vec) {
    if constexpr (kBits == 8) {
      const uint2 c = reinterpret_cast<const uint2*>(row)[vec];
      v.x = c.x;
      v.y = c.y;
    } else {
      v = reinterpret_cast<const uint4*>(row)[vec];
    }
  }
  __device__ __forceinline__ void get(float scale, float (&f)[8]) const {
    if constexpr (kBits == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = e4m3x2_to_f32((i < 2 ? v.x : v.y) >> (16 * (i & 1)));
        f[2 * i] = t.x * scale;
        f[2 * i + 1] = t.y * scale;
      }
    } else {
      bf16x8_to_f32(v, f);
    }
  }
};

template <int kBits, int kVecs>
__global__ void __launch_bounds__(kPreactThreads) grad_preact_saved_kernel(const PreactParams p) {
  constexpr int kRows = 2;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int64_t rows = p.rows;
  if (p.end) {
    const int64_t e = *p.end;
    rows = e < 0 ? 0 : (e < rows ? e : rows);
  }
  // (neighbouring lanes own neighbouring vectors: whole sectors in every access)
  const int v0 = blockIdx.x * (kPreactThreads * kVecs) + threadIdx.x;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * kRows; r0 < rows;
       r0 += static_cast<int64_t>(gridDim.y) * kRows) {
    Vec8<false> dy[kRows][kVecs];
    SavedVec<kBits> up[kRows][kVecs], gate[kRows][kVecs];
    int su[kRows][kVecs], sg[kRows][kVecs];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t r = r0 + i;
      if (r >= rows) continue;
      const uint8_t* pre = p.pre + r * p.ld_pre;
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        const int v = v0 + j * kPreactThreads;
        if (v >= p.nvec) continue;
        dy[i][j].load(p.dy, r, p.lddy, v);
        up[i][j].load(pre, v);
        gate[i][j].load(pre + p.gate_off, v);
        if constexpr (kBits == 8) {
          const uint8_t* sc = p.scales + r * p.ld_scales + (v >> 2);
          su[i][j] = sc[0];
          sg[i][j] = sc[p.gate_scale_off];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t r = r0 + i;
      if (r >= rows) continue;
      uint4* out = reinterpret_cast<uint4*>(p.grad + r * p.ld_grad);
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        const int v = v0 + j * kPreactThreads;
        if (v >= p.nvec) continue;
        float u[8], g[8], d[8], h[8], gu[8], gg[8];
        up[i][j].get(kBits == 8 ? block_scale(su[i][j]) : 1.f, u);
        gate[i][j].get(kBits == 8 ? block_scale(sg[i][j]) : 1.f, g);
        dy[i][j].get(d);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          float sv, dv;
          silu_factors(g[c], u[c], h[c], sv, dv);
          gu[c] = d[c] * sv;
          gg[c] = d[c] * dv;
        }
        out[v] = f32_to_bf16x8(gu);
        out[p.nvec + v] = f32_to_bf16x8(gg);
        if (p.h) reinterpret_cast<uint4*>(p.h + r * p.ldh)[v] = f32_to_bf16x8(h);
      }
    }
  }
}

}  // namespace sgl
