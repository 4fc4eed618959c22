// Token slots ordered by expert, rows sent to their experts and back, and the gradients.
//
// A slot is one (token, choice) pair, s = t * k + j, of the router's answer ids[T, k].  Slots
// whose id lies outside [0, E) are dropped (padding tokens carry -1).  The order is a stable
// counting sort by expert:
//   offsets[e]  = number of kept slots with an id below e      (offsets[E] = kept slots)
//   slots[r]    = slot that row r holds, -1 for rows at and behind offsets[E]
//   rows[t, j]  = row of slot (t, j), -1 if dropped
// Every result is a fixed function of the inputs, bit for bit (the only atomics are integer sums
// in shared memory).
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "ptx_sm100.cuh"

namespace sgl {

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kOrderMaxExperts = 1024;
constexpr int kOrderSteps = 2;                               // slots of a thread in one round
constexpr int kOrderRound = kOrderThreads * kOrderSteps;     // slots of a CTA in one round
constexpr int kOrderMaxCtas = 128;

// Shared memory: a count per (warp, expert), two words per expert, and the scan's scratch.
constexpr int order_smem_bytes(int E) { return (kOrderWarps + 2) * E * 4 + 40 * 4; }

struct OrderParams {
  const void* ids;
  int64_t ld_ids;      // row pitch of ids, elements
  int64_t total;       // T * k slots
  int64_t per_cta;     // slots of a CTA (a contiguous range)
  int k, E;
  int ids64;           // ids are int64 (else int32)
  int* offsets;        // [E + 1]
  int* slots;          // [T * k]
  int* rows;           // [T * k]
  int* counts;         // several CTAs: [CTAs][E], kept slots of each CTA and expert
};

// Expert of slot s, or -1 (dropped).
__device__ __forceinline__ int order_key(const OrderParams& p, int64_t s) {
  int64_t at = s;
  if (p.ld_ids != p.k) {
    const int64_t t = s / p.k;
    at = t * p.ld_ids + (s - t * p.k);
  }
  const int64_t id = p.ids64 ? reinterpret_cast<const int64_t*>(p.ids)[at]
                             : static_cast<int64_t>(reinterpret_cast<const int*>(p.ids)[at]);
  return (id >= 0 && id < p.E) ? static_cast<int>(id) : -1;
}

// Lanes whose key equals this lane's: a ballot per bit (all lanes of the warp).  768 slots of 128
// experts: 3.1 us for the whole launch, 3.5 us with one match.any instead.
__device__ __forceinline__ unsigned same_key(int key, int bits) {
  unsigned same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = (key >> b) & 1;
    const unsigned ones = __ballot_sync(0xffffffffu, one);
    same &= one ? ones : ~ones;
  }
  return same;
}

// Ranks the slots [first, last), at most kOrderRound, inside their expert: key[u] / rank[u] are
// this thread's u-th slot (index slot_of(u)), rank counting the CTA's earlier slots of the same
// expert, total[e] of earlier rounds included; total[e] is advanced.  A warp owns a contiguous run
// of slots and takes 32 at a time: lanes with equal experts find each other, one of them adds
// to the warp's counts; then the counts are summed over the warps.
struct OrderRound {
  int key[kOrderSteps], rank[kOrderSteps];
  int64_t base;        // first slot of this warp
  int steps;
  __device__ __forceinline__ int64_t slot_of(int u) const {
    return base + u * 32 + (threadIdx.x & 31);
  }
  __device__ __forceinline__ void run(const OrderParams& p, int64_t first, int64_t last, int* count,
                                      int* total) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, E = p.E;
    steps = static_cast<int>((last - first + kOrderThreads - 1) / kOrderThreads);
    base = first + static_cast<int64_t>(warp) * steps * 32;
    int* mine = count + warp * E;
    const int bits = 33 - __clz(E);   // of a key in [-1, E)
#pragma unroll
    for (int u = 0; u < kOrderSteps; ++u) {
      const int64_t s = slot_of(u);
      key[u] = (u < steps && s < last) ? order_key(p, s) : -1;
    }
    for (int i = tid; i < kOrderWarps * E; i += kOrderThreads) count[i] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kOrderSteps; ++u) {
      if (u < steps) {
        const unsigned same = same_key(key[u], bits);
        if (key[u] >= 0) rank[u] = mine[key[u]] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (key[u] >= 0 && lane == __ffs(same) - 1) mine[key[u]] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    for (int e = tid; e < E; e += kOrderThreads) {
      int sum = total[e];
#pragma unroll 8
      for (int w = 0; w < kOrderWarps; ++w) {
        const int c = count[w * E + e];
        count[w * E + e] = sum;
        sum += c;
      }
      total[e] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kOrderSteps; ++u)
      if (key[u] >= 0) rank[u] += mine[key[u]];
  }
};

// Exclusive scan over the experts (thread e holds v; E <= kOrderThreads): its result, and the sum
// of all in *sum.  scratch: 33 words.
__device__ __forceinline__ int order_scan(int v, int* scratch, int* sum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += n;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int mine = scratch[lane];
    int w = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += n;
    }
    scratch[lane] = w - mine;
    if (lane == 31) scratch[32] = w;
  }
  __syncthreads();
  *sum = scratch[32];
  return scratch[warp] + inc - v;
}

// Up to kOrderRound slots: everything in one CTA.  Bound by latency (a load, the ballots of each 32
// slots, a few barriers).
__global__ void __launch_bounds__(kOrderThreads, 1) expert_order_kernel(const OrderParams p) {
  extern __shared__ int order_smem[];
  const int E = p.E, tid = threadIdx.x;
  int* count = order_smem;
  int* total = count + kOrderWarps * E;
  int* start = total + E;
  int* scratch = start + E;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int e = tid; e < E; e += kOrderThreads) total[e] = 0;
  OrderRound r;
  r.run(p, 0, p.total, count, total);
  int kept;
  const int first = order_scan(tid < E ? total[tid] : 0, scratch, &kept);
  if (tid < E) {
    start[tid] = first;
    p.offsets[tid] = first;
  }
  if (tid == 0) p.offsets[E] = kept;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kOrderSteps; ++u) {
    const int64_t s = r.slot_of(u);
    if (u < r.steps && s < p.total) {
      const int row = r.key[u] >= 0 ? start[r.key[u]] + r.rank[u] : -1;
      p.rows[s] = row;
      if (row >= 0) p.slots[row] = static_cast<int>(s);
    }
  }
  for (int64_t i = kept + tid; i < p.total; i += kOrderThreads) p.slots[i] = -1;
}

// The same, and x's rows sent on in the same launch (sgl_experts_swiglu with few slots): every CTA
// orders all slots for itself, the first writes the order, and each copies its share of the
// tokens.  64 tokens x 8 of 64 experts, 2048 x 1024: 6 us less (4 % of the layer) than an order and a
// dispatch launch, both measured in one session.
__global__ void __launch_bounds__(kOrderThreads, 1)
expert_order_dispatch_kernel(const OrderParams p, const __nv_bfloat16* x, __nv_bfloat16* out,
                             int64_t ldx, int64_t ldo, int nvec) {
  extern __shared__ int order_smem[];
  const int E = p.E, tid = threadIdx.x;
  int* count = order_smem;
  int* total = count + kOrderWarps * E;
  int* start = total + E;
  int* scratch = start + E;
  int* row_of_slot = scratch + 40;       // [kOrderRound]
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int e = tid; e < E; e += kOrderThreads) total[e] = 0;
  OrderRound r;
  r.run(p, 0, p.total, count, total);
  int kept;
  const int first = order_scan(tid < E ? total[tid] : 0, scratch, &kept);
  const bool writer = blockIdx.x == 0;
  if (tid < E) {
    start[tid] = first;
    if (writer) p.offsets[tid] = first;
  }
  if (writer && tid == 0) p.offsets[E] = kept;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kOrderSteps; ++u) {
    const int64_t s = r.slot_of(u);
    if (u < r.steps && s < p.total) {
      const int row = r.key[u] >= 0 ? start[r.key[u]] + r.rank[u] : -1;
      row_of_slot[s] = row;
      if (writer) {
        p.rows[s] = row;
        if (row >= 0) p.slots[row] = static_cast<int>(s);
      }
    }
  }
  if (writer)
    for (int64_t i = kept + tid; i < p.total; i += kOrderThreads) p.slots[i] = -1;
  __syncthreads();
  // 256 threads to a token
  const int tokens = static_cast<int>(p.total) / p.k;
  for (int t = blockIdx.x * (kOrderThreads / 256) + tid / 256; t < tokens;
       t += gridDim.x * (kOrderThreads / 256)) {
    const uint4* src = reinterpret_cast<const uint4*>(x + t * ldx);
    for (int v = tid % 256; v < nvec; v += 256) {
      const uint4 val = src[v];
      for (int j = 0; j < p.k; ++j) {
        const int row = row_of_slot[t * p.k + j];
        if (row >= 0) reinterpret_cast<uint4*>(out + row * ldo)[v] = val;
      }
    }
  }
}

// More slots: one range per CTA.  The first kernel leaves every slot's rank inside its CTA in
// `rows` and the CTA's counts in `counts`; the second adds up the counts of the CTAs before it
// (all of them read the whole table, CTAs * E words from L2) and places its slots.  262144 slots
// of 256 experts: 10.6 us for both, where one cluster of 8 CTAs took 66 us, bound by the
// scattered stores that 8 SMs can issue.
__global__ void __launch_bounds__(kOrderThreads, 1) expert_count_kernel(const OrderParams p) {
  extern __shared__ int order_smem[];
  const int E = p.E, tid = threadIdx.x;
  int* count = order_smem;
  int* total = count + kOrderWarps * E;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int e = tid; e < E; e += kOrderThreads) total[e] = 0;
  const int64_t lo = blockIdx.x * p.per_cta;
  const int64_t hi = lo + p.per_cta < p.total ? lo + p.per_cta : p.total;
  for (int64_t s0 = lo; s0 < hi; s0 += kOrderRound) {
    OrderRound r;
    r.run(p, s0, s0 + kOrderRound < hi ? s0 + kOrderRound : hi, count, total);
#pragma unroll
    for (int u = 0; u < kOrderSteps; ++u) {
      const int64_t s = r.slot_of(u);
      if (u < r.steps && s < hi) p.rows[s] = r.key[u] >= 0 ? r.rank[u] : -1;
    }
    __syncthreads();
  }
  __syncthreads();
  for (int e = tid; e < E; e += kOrderThreads)
    p.counts[static_cast<int64_t>(blockIdx.x) * E + e] = total[e];
}

__global__ void __launch_bounds__(kOrderThreads, 1) expert_place_kernel(const OrderParams p) {
  extern __shared__ int order_smem[];
  const int E = p.E, tid = threadIdx.x;
  int* start = order_smem;       // [E] kept slots of earlier CTAs, then the first row
  int* total = start + E;        // [E]
  int* scratch = total + E;
  const int ctas = gridDim.x, cta = blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int e = tid; e < E; e += kOrderThreads) start[e] = total[e] = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  {
    // thread (group, e): every group adds up every n-th CTA's counts of expert e
    const int groups = kOrderThreads / E, e = tid % E, g = tid / E;
    if (g < groups) {
      int before = 0, all = 0;
#pragma unroll 4
      for (int c = g; c < ctas; c += groups) {
        const int n = p.counts[static_cast<int64_t>(c) * E + e];
        all += n;
        if (c < cta) before += n;
      }
      atomicAdd(&total[e], all);
      atomicAdd(&start[e], before);
    }
  }
  __syncthreads();
  int kept;
  const int first = order_scan(tid < E ? total[tid] : 0, scratch, &kept);
  if (tid < E) {
    start[tid] += first;
    if (cta == 0) p.offsets[tid] = first;
  }
  if (cta == 0 && tid == 0) p.offsets[E] = kept;
  __syncthreads();
  const int64_t lo = cta * p.per_cta;
  const int64_t hi = lo + p.per_cta < p.total ? lo + p.per_cta : p.total;
  for (int64_t s = lo + tid; s < hi; s += kOrderThreads) {
    const int rank = p.rows[s];
    if (rank >= 0) {
      const int row = start[order_key(p, s)] + rank;
      p.rows[s] = row;
      p.slots[row] = static_cast<int>(s);
    }
  }
  for (int64_t i = kept + static_cast<int64_t>(cta) * kOrderThreads + tid; i < p.total;
       i += static_cast<int64_t>(ctas) * kOrderThreads)
    p.slots[i] = -1;
}

// ---------------------------------------------------------------- rows out and back
//
// The kernels give a multiple of 32 threads to a token, 256 threads of several tokens to a CTA, and
// with few tokens several CTAs (gridDim.y) to one; a thread moves 8 columns of a row at a time.
// HBM bound.

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
  int splits;                  // combine_parts: a row is the sum of `splits` partial rows,
  int64_t slot_stride;         // slot_stride elements apart
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

// kVecs vectors of each of kBatch rows are a thread's loads in flight.  Four in all is what 64
// registers (four CTAs on an SM; three for fp32 rows) carry: 2 x 2 up to two choices a token, 1 x 4
// beyond.  16384 tokens x 2 choices x 4096 columns: combine 64 us (6.3 TB/s) so and 77 us with
// 1 x 4; 4096 tokens x 6 choices x 2048: 28 us with 2 x 2 and 23 us with 1 x 4.

// out[rows[t, j]] = x[t]: x is read once, each of its rows written once.
__global__ void __launch_bounds__(256) expert_dispatch_kernel(const RowParams p) {
  constexpr int kVecs = 2;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tx = blockDim.x * gridDim.y;     // threads of a token
  const int first = blockIdx.y * blockDim.x + threadIdx.x;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < p.T;
       t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    for (int v0 = first; v0 < p.nvec; v0 += kVecs * tx) {
      Vec8<false> val[kVecs];
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
        if (v0 + i * tx < p.nvec) val[i].load(p.in, t, p.ld_in, v0 + i * tx);
      for (int j = 0; j < p.k; ++j) {
        const int r = row_of(p, t, j);
        if (r < 0) continue;
        uint4* dst = reinterpret_cast<uint4*>(p.out + r * p.ld_out);
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
          if (v0 + i * tx < p.nvec) dst[v0 + i * tx] = val[i].v[0];
      }
    }
  }
}

// out[t] = sum_j weights[t, j] * rows[rows[t, j]], fp32 in the order of j, rounded once.  A
// dropped choice adds nothing (its weight is not read either); a token without any is zero.
template <bool kF32, int kVecs, int kBatch>
__global__ void __launch_bounds__(256, kF32 ? 3 : 4) expert_combine_kernel(const RowParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tx = blockDim.x * gridDim.y;     // threads of a token
  const int first = blockIdx.y * blockDim.x + threadIdx.x;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < p.T;
       t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    for (int v0 = first; v0 < p.nvec; v0 += kVecs * tx) {
      float acc[kVecs][8] = {};
      for (int j0 = 0; j0 < p.k; j0 += kBatch) {
        Vec8<kF32> val[kBatch][kVecs];
        float w[kBatch];
        int r[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) r[u] = j0 + u < p.k ? row_of(p, t, j0 + u) : -1;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (r[u] < 0) continue;
          w[u] = load_weight(p, t, j0 + u);
#pragma unroll
          for (int i = 0; i < kVecs; ++i)
            if (v0 + i * tx < p.nvec) val[u][i].load(p.in, r[u], p.ld_in, v0 + i * tx);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (r[u] < 0) continue;
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            float f[8];
            val[u][i].get(f);
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[i][c] = fmaf(w[u], f[c], acc[i][c]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
        if (v0 + i * tx < p.nvec)
          reinterpret_cast<uint4*>(p.out + t * p.ld_out)[v0 + i * tx] = f32_to_bf16x8(acc[i]);
    }
  }
}

// The same for rows that are sums of p.splits fp32 partial rows, added in order.  Few tokens, so
// latency bound: a thread has up to eight partial rows in flight.
__global__ void __launch_bounds__(256, 2) expert_combine_parts_kernel(const RowParams p) {
  constexpr int kParts = 8;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tx = blockDim.x * gridDim.y;     // threads of a token
  const int first = blockIdx.y * blockDim.x + threadIdx.x;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < p.T;
       t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    for (int v = first; v < p.nvec; v += tx) {
      float acc[8] = {};
      for (int j = 0; j < p.k; ++j) {
        const int r = row_of(p, t, j);
        if (r < 0) continue;
        const float w = load_weight(p, t, j);
        float sum[8] = {};
        for (int s0 = 0; s0 < p.splits; s0 += kParts) {
          Vec8<true> part[kParts];
#pragma unroll
          for (int i = 0; i < kParts; ++i)
            if (s0 + i < p.splits)
              part[i].load(static_cast<const float*>(p.in) + (s0 + i) * p.slot_stride, r, p.ld_in, v);
#pragma unroll
          for (int i = 0; i < kParts; ++i) {
            if (s0 + i >= p.splits) continue;
            float f[8];
            part[i].get(f);
#pragma unroll
            for (int c = 0; c < 8; ++c) sum[c] += f[c];
          }
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = fmaf(w, sum[c], acc[c]);
      }
      reinterpret_cast<uint4*>(p.out + t * p.ld_out)[v] = f32_to_bf16x8(acc);
    }
  }
}

// Gradients of the weighted sum: grad_rows[r] = w * grad_out[t] (w = 1 without weights),
// grad_weights[t, j] = <grad_out[t], rows[r]> (0 for a dropped choice), in one pass over the rows.
// The dot product is summed in fp32: by thread over its columns, then over the threads in a fixed
// order.
template <bool kF32, int kVecs, int kBatch>
__global__ void __launch_bounds__(256, kF32 ? 3 : 4) expert_combine_grad_kernel(const RowParams p) {
  __shared__ float part[kBatch][8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tx = blockDim.x, warps = tx / 32;              // threads and warps of one token
  const int warp_in_token = threadIdx.x / 32, lane = threadIdx.x & 31;
  // every thread of the CTA makes the same number of steps (there are barriers inside)
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * blockDim.y; t0 < p.T;
       t0 += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const int64_t t = t0 + threadIdx.y;
    const bool live = t < p.T;
    for (int j0 = 0; j0 < p.k; j0 += kBatch) {
      int r[kBatch];
      float w[kBatch], dot[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        r[u] = live && j0 + u < p.k ? row_of(p, t, j0 + u) : -1;
        w[u] = r[u] >= 0 ? load_weight(p, t, j0 + u) : 0.f;
        dot[u] = 0.f;
      }
      for (int v0 = threadIdx.x; live && v0 < p.nvec; v0 += kVecs * tx) {
        Vec8<false> g[kVecs];
        Vec8<kF32> y[kBatch][kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          if (v0 + i * tx >= p.nvec) continue;
          g[i].load(p.in, t, p.ld_in, v0 + i * tx);
          if (p.in2 != nullptr) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
              if (r[u] >= 0) y[u][i].load(p.in2, r[u], p.ld_in2, v0 + i * tx);
          }
        }
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          if (v0 + i * tx >= p.nvec) continue;
          float gf[8];
          g[i].get(gf);
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            if (r[u] < 0) continue;
            if (p.in2 != nullptr) {
              float yf[8];
              y[u][i].get(yf);
#pragma unroll
              for (int c = 0; c < 8; ++c) dot[u] = fmaf(gf[c], yf[c], dot[u]);
            }
            float o[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) o[c] = gf[c] * w[u];
            reinterpret_cast<uint4*>(p.out + r[u] * p.ld_out)[v0 + i * tx] = f32_to_bf16x8(o);
          }
        }
      }
      if (p.grad_weights == nullptr) continue;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], d);
      }
      if (warps > 1) {
        if (lane == 0) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u) part[u][threadIdx.y * warps + warp_in_token] = dot[u];
        }
        __syncthreads();
      }
      if (live && threadIdx.x < kBatch && j0 + threadIdx.x < p.k) {
        const int u = threadIdx.x;
        float sum = 0.f;
        if (warps > 1) {
          for (int i = 0; i < warps; ++i) sum += part[u][threadIdx.y * warps + i];
        } else {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) sum = u == i ? dot[i] : sum;
        }
        const int64_t at = t * p.k + j0 + u;
        if (p.w_bf16) {
          reinterpret_cast<__nv_bfloat16*>(p.grad_weights)[at] = __float2bfloat16_rn(sum);
        } else {
          reinterpret_cast<float*>(p.grad_weights)[at] = sum;
        }
      }
      if (warps > 1) __syncthreads();
    }
  }
}

}  // namespace sgl
