// Token slots ordered by expert, rows sent to their experts and back, and the gradients.
//
// A slot is one (token, choice) pair, s = t * k + j, of the router's answer ids[T, k].  Slots
// whose id lies outside [0, E) are dropped (padding tokens carry -1).  The order is a stable
// counting sort by expert:
//   offsets[e]  = number of kept slots with an id below e      (offsets[E] = kept slots)
//   slots[r]    = slot that row r holds, -1 for rows at and behind offsets[E]
//   rows[t, j]  = row of slot (t, j), -1 if dropped
// Nothing here uses atomics: every result is a fixed function of the inputs, bit for bit.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "ptx_sm100.cuh"

namespace sgl {

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kOrderMaxExperts = 1024;
constexpr int kOrderCluster = 8;       // CTAs of the long form, one thread-block cluster
constexpr int kOrderUnroll = 4;

// Shared memory: a count per (warp, expert), and three words per expert.
constexpr int order_smem_bytes(int E) { return (kOrderWarps + 3) * E * 4 + 64 * 4; }

struct OrderParams {
  const void* ids;
  int64_t ld_ids;      // row pitch of ids, elements
  int64_t total;       // T * k slots
  int k, E;
  int ids64;           // ids are int64 (else int32)
  int* offsets;        // [E + 1]
  int* slots;          // [T * k]
  int* rows;           // [T * k]
};

// Expert of slot s, or -1 (dropped, or past the last slot).
__device__ __forceinline__ int order_key(const OrderParams& p, int64_t s) {
  if (s >= p.total) return -1;
  int64_t at = s;
  if (p.ld_ids != p.k) {
    const int64_t t = s / p.k;
    at = t * p.ld_ids + (s - t * p.k);
  }
  const int64_t id = p.ids64 ? reinterpret_cast<const int64_t*>(p.ids)[at]
                             : static_cast<int64_t>(reinterpret_cast<const int*>(p.ids)[at]);
  return (id >= 0 && id < p.E) ? static_cast<int>(id) : -1;
}

// One launch: the CTAs of one cluster (or a single CTA) each own a contiguous range of slots,
// and so does each warp inside its CTA.  Warps count their slots per expert (match.any groups
// the 32 slots of a step, one lane per group adds), the counts are turned into the first row of
// every (expert, CTA, warp) - CTA totals are exchanged through distributed shared memory - and
// the warps walk their slots a second time to hand out the rows in slot order.
//
// Bound by latency: 2 x (slots / (CTAs * 1024)) steps of a match and a shared-memory update.
__global__ void __launch_bounds__(kOrderThreads, 1) expert_order_kernel(const OrderParams p) {
  extern __shared__ int order_smem[];
  const int E = p.E;
  int* count = order_smem;                         // [kOrderWarps][E]
  int* cta_total = count + kOrderWarps * E;        // [E], read by the other CTAs
  int* base = cta_total + E;                       // [E]
  int* scan = base + E;                            // [E]
  int* warp_sum = scan + E;                        // [33]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t nctas = gridDim.x, rank = blockIdx.x;   // the grid is one cluster

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  for (int i = tid; i < kOrderWarps * E; i += kOrderThreads) count[i] = 0;
  __syncthreads();

  // slots of this warp: a multiple of 32, contiguous
  const int64_t per_warp =
      (p.total + static_cast<int64_t>(nctas) * kOrderThreads - 1) /
      (static_cast<int64_t>(nctas) * kOrderThreads) * 32;
  const int64_t first = (static_cast<int64_t>(rank) * kOrderWarps + warp) * per_warp;
  int64_t last = first + per_warp;
  if (last > p.total) last = p.total;
  int* my_count = count + warp * E;

  for (int64_t s0 = first; s0 < last; s0 += 32 * kOrderUnroll) {
    int key[kOrderUnroll];
#pragma unroll
    for (int u = 0; u < kOrderUnroll; ++u) {
      const int64_t s = s0 + u * 32 + lane;
      key[u] = s < last ? order_key(p, s) : -1;
    }
#pragma unroll
    for (int u = 0; u < kOrderUnroll; ++u) {
      const unsigned same = __match_any_sync(0xffffffffu, key[u]);
      if (key[u] >= 0 && lane == __ffs(same) - 1) my_count[key[u]] += __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();

  // counts -> exclusive sums over the warps of this CTA; totals for the cluster
  for (int e = tid; e < E; e += kOrderThreads) {
    int sum = 0;
#pragma unroll 8
    for (int w = 0; w < kOrderWarps; ++w) {
      const int c = count[w * E + e];
      count[w * E + e] = sum;
      sum += c;
    }
    cta_total[e] = sum;
  }
  if (nctas > 1) {
    ptx::cluster_sync();
  } else {
    __syncthreads();
  }
  // (E <= kOrderThreads: one expert per thread from here)
  int before = 0, total = 0;
  if (tid < E) {
    if (nctas > 1) {
      const uint32_t mine = ptx::smem_u32(cta_total + tid);
      for (uint32_t c = 0; c < nctas; ++c) {
        int v;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(ptx::mapa(mine, c)));
        if (c < rank) before += v;
        total += v;
      }
    } else {
      total = cta_total[tid];
    }
  }
  // exclusive scan of the totals over the experts
  int inc = total;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += v;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int mine = warp_sum[lane];
    int w = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += v;
    }
    warp_sum[lane] = w - mine;
    if (lane == 31) warp_sum[32] = w;
  }
  __syncthreads();
  const int start = warp_sum[warp] + inc - total;
  const int kept = warp_sum[32];
  if (tid < E) {
    base[tid] = start + before;
    if (rank == 0) p.offsets[tid] = start;
  }
  if (rank == 0 && tid == 0) p.offsets[E] = kept;
  __syncthreads();

  for (int64_t s0 = first; s0 < last; s0 += 32 * kOrderUnroll) {
    int key[kOrderUnroll];
#pragma unroll
    for (int u = 0; u < kOrderUnroll; ++u) {
      const int64_t s = s0 + u * 32 + lane;
      key[u] = s < last ? order_key(p, s) : -1;
    }
#pragma unroll
    for (int u = 0; u < kOrderUnroll; ++u) {
      const int64_t s = s0 + u * 32 + lane;
      const unsigned same = __match_any_sync(0xffffffffu, key[u]);
      int row = -1;
      if (key[u] >= 0) {
        row = base[key[u]] + my_count[key[u]] + __popc(same & ((1u << lane) - 1u));
        p.slots[row] = static_cast<int>(s);
      }
      __syncwarp();
      if (key[u] >= 0 && lane == __ffs(same) - 1) my_count[key[u]] += __popc(same);
      if (s < last) p.rows[s] = row;
      __syncwarp();
    }
  }
  for (int64_t r = kept + static_cast<int64_t>(rank) * kOrderThreads + tid; r < p.total;
       r += static_cast<int64_t>(nctas) * kOrderThreads)
    p.slots[r] = -1;
  // no CTA leaves while another may still read its totals
  if (nctas > 1) ptx::cluster_sync();
}

// ---------------------------------------------------------------- rows out and back
//
// All three kernels give `tx` threads (a multiple of 32) to a token, 256 / tx tokens to a CTA,
// and let each thread move 16 bytes (8 columns) of the row at a time.  HBM bound.

struct RowParams {
  const void* in;              // x [T, D] | rows [R, D] | grad_out [T, D]; bf16, rows also fp32
  const void* in2;             // combine_grad: rows [R, D] or NULL
  __nv_bfloat16* out;          // rows [R, D] | y [T, D] | grad_rows [R, D]
  const int* rows;             // [T, k]
  const void* weights;         // fp32 or bf16 [T, k], or NULL (all ones)
  void* grad_weights;          // combine_grad: dense [T, k], fp32 or bf16 (w_bf16), or NULL
  int64_t ld_in, ld_in2, ld_out, ld_w;
  int64_t T;
  int k, nvec;                 // nvec = D / 8
  int w_bf16;
  int64_t R;                   // rows the row tensors have: an index outside is not followed
};

__device__ __forceinline__ float load_weight(const RowParams& p, int64_t t, int j) {
  if (!p.weights) return 1.0f;
  const int64_t at = t * p.ld_w + j;
  return p.w_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.weights)[at])
                  : reinterpret_cast<const float*>(p.weights)[at];
}

__device__ __forceinline__ void bf16x8_to_f32(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 f32_to_bf16x8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __nv_bfloat162 r = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&r);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 8 columns of a row of bf16 or fp32, kept as loaded until they are used.
template <bool kF32>
struct Vec8 {
  uint4 v[kF32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* base, int64_t row, int64_t ld, int vec) {
    if constexpr (kF32) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + row * ld);
      v[0] = src[2 * vec];
      v[1] = src[2 * vec + 1];
    } else {
      v[0] = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + row * ld)[vec];
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (kF32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[4 * i] = __uint_as_float(v[i].x);
        f[4 * i + 1] = __uint_as_float(v[i].y);
        f[4 * i + 2] = __uint_as_float(v[i].z);
        f[4 * i + 3] = __uint_as_float(v[i].w);
      }
    } else {
      bf16x8_to_f32(v[0], f);
    }
  }
};

// The row of choice j of token t, or -1 (dropped).
__device__ __forceinline__ int row_of(const RowParams& p, int64_t t, int j) {
  const int r = p.rows[t * p.k + j];
  return (r >= 0 && r < p.R) ? r : -1;
}

// out[rows[t, j]] = x[t]: x is read once, each of its rows written once.
__global__ void __launch_bounds__(256) expert_dispatch_kernel(const RowParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < p.T;
       t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const uint4* src = reinterpret_cast<const uint4*>(
        static_cast<const __nv_bfloat16*>(p.in) + t * p.ld_in);
    for (int v = threadIdx.x; v < p.nvec; v += blockDim.x) {
      const uint4 val = src[v];
      for (int j = 0; j < p.k; ++j) {
        const int r = row_of(p, t, j);
        if (r >= 0) reinterpret_cast<uint4*>(p.out + r * p.ld_out)[v] = val;
      }
    }
  }
}

// out[t] = sum_j weights[t, j] * rows[rows[t, j]], fp32 in the order of j, rounded once.  A
// dropped choice adds nothing (its weight is not read either); a token without any is zero.
template <bool kF32>
__global__ void __launch_bounds__(256) expert_combine_kernel(const RowParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kBatch = 4;   // rows whose loads are in flight together
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < p.T;
       t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    for (int v = threadIdx.x; v < p.nvec; v += blockDim.x) {
      float acc[8] = {};
      for (int j0 = 0; j0 < p.k; j0 += kBatch) {
        Vec8<kF32> val[kBatch];
        float w[kBatch];
        bool on[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int j = j0 + u;
          const int r = j < p.k ? row_of(p, t, j) : -1;
          on[u] = r >= 0;
          if (on[u]) {
            val[u].load(p.in, r, p.ld_in, v);
            w[u] = load_weight(p, t, j);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (on[u]) {
            float f[8];
            val[u].get(f);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = fmaf(w[u], f[i], acc[i]);
          }
        }
      }
      reinterpret_cast<uint4*>(p.out + t * p.ld_out)[v] = f32_to_bf16x8(acc);
    }
  }
}

// Gradients of the weighted sum: grad_rows[r] = w * grad_out[t] (w = 1 without weights),
// grad_weights[t, j] = <grad_out[t], rows[r]> (0 for a dropped choice), in one pass over the rows.  The dot product is
// summed in fp32: by thread over its columns, then over the threads in a fixed tree.
template <bool kF32>
__global__ void __launch_bounds__(256) expert_combine_grad_kernel(const RowParams p) {
  __shared__ float part[8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warps = blockDim.x / 32;                       // warps of one token
  const int warp_in_token = threadIdx.x / 32, lane = threadIdx.x & 31;
  // every thread of the CTA makes the same number of steps (there are barriers inside)
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * blockDim.y; t0 < p.T;
       t0 += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const int64_t t = t0 + threadIdx.y;
    const bool live = t < p.T;
    const uint4* dy = reinterpret_cast<const uint4*>(
        static_cast<const __nv_bfloat16*>(p.in) + (live ? t : 0) * p.ld_in);
    for (int j = 0; j < p.k; ++j) {
      const int r = live ? row_of(p, t, j) : -1;
      float dot = 0.f;
      if (r >= 0) {
        const float w = load_weight(p, t, j);
        uint4* dst = reinterpret_cast<uint4*>(p.out + r * p.ld_out);
        for (int v = threadIdx.x; v < p.nvec; v += blockDim.x) {
          float g[8];
          bf16x8_to_f32(dy[v], g);
          if (p.in2) {
            Vec8<kF32> val;
            float y[8];
            val.load(p.in2, r, p.ld_in2, v);
            val.get(y);
#pragma unroll
            for (int i = 0; i < 8; ++i) dot = fmaf(g[i], y[i], dot);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] *= w;
          dst[v] = f32_to_bf16x8(g);
        }
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
      if (warps > 1) {
        if (lane == 0) part[threadIdx.y * warps + warp_in_token] = dot;
        __syncthreads();
        if (threadIdx.x == 0) {
          dot = 0.f;
          for (int w = 0; w < warps; ++w) dot += part[threadIdx.y * warps + w];
        }
        __syncthreads();
      }
      if (live && threadIdx.x == 0 && p.grad_weights) {
        const int64_t at = t * p.k + j;
        if (p.w_bf16) {
          reinterpret_cast<__nv_bfloat16*>(p.grad_weights)[at] = __float2bfloat16_rn(dot);
        } else {
          reinterpret_cast<float*>(p.grad_weights)[at] = dot;
        }
      }
    }
  }
}

}  // namespace sgl
