// Tokens to experts and back: the router's choice, the stable sort of tokens by expert, the weighted sum of the
// experts' outputs.
//
//   mq_route_experts   : logits -> the top_k experts of each token and their weights
//   mq_sort_by_expert  : expert ids -> token rows in expert order, offsets, and each choice's position in that order
//   mq_combine_experts : out[t] = sum_j weight[t, j] * Y[slot[t, j]] (_to: in another type than Y's)
#include "common.hpp"
#include "route_kernels.hpp"

namespace {

constexpr int ROUTE_MAX_E = 1024;

// ---- sort by expert -----------------------------------------------------------------------------------
// Stable counting sort of n = T * top_k choices into E + 1 bins (bin E: ids outside [0, E)).  A workgroup owns a run of
// SORT_CHUNK choices; `count` holds, bin-major, the number of choices of every (bin, workgroup).
// Measured: 146 us of kernels for 16.8 million choices over 256 experts of skewed loads (34 counting, 7 summing, 105 placing;
// 166 us a pass, with the gaps between three launches; even loads take 170 placing), 5 us for 488 in one workgroup.  Tried, at
// 102 placing: chunks of 4096 and 16384 (108 and 120); putting a workgroup's choices in order in shared memory first, so that
// rows leaves in runs (121).
constexpr int SORT_CHUNK = 8192;
constexpr int SORT_WAVES = 8;
constexpr int SORT_MAX_E = 1024;

__device__ __forceinline__ int bin_of(long id, int E) { return id < 0 || id >= E ? E : (int)id; }

__global__ __launch_bounds__(512) void sort_count_kernel(const long* __restrict__ ids, int n, int E, int blocks,
                                                         int* __restrict__ count) {
  __shared__ int hist[SORT_MAX_E + 1];
  for (int b = threadIdx.x; b <= E; b += 512) hist[b] = 0;
  __syncthreads();
  const int i0 = blockIdx.x * SORT_CHUNK, i1 = min(n, i0 + SORT_CHUNK);
  for (int i = i0 + threadIdx.x; i < i1; i += 512) atomicAdd(&hist[bin_of(ids[i], E)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b <= E; b += 512) count[(long)b * blocks + blockIdx.x] = hist[b];
}

// One workgroup per bin: its counts become their exclusive prefix sums, its total goes to total[bin].
__global__ __launch_bounds__(256) void sort_scan_kernel(int* __restrict__ count, int blocks, int* __restrict__ total) {
  __shared__ int part[4];
  int* c = count + (long)blockIdx.x * blocks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  for (int i0 = 0; i0 < blocks; i0 += 256) {
    const int i = i0 + threadIdx.x;
    const int v = i < blocks ? c[i] : 0;
    int s = v;
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(s, o);
      if (lane >= o) s += u;
    }
    if (lane == 63) part[wave] = s;
    __syncthreads();
    int before = base, all = 0;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += part[w];
      all += part[w];
    }
    if (i < blocks) c[i] = before + s - v;
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = base;
}

// n / k for 0 <= n < 2^31, k >= 1: with 2^(s-1) < k <= 2^s and mul = ceil(2^(31+s) / k) < 2^32 the quotient is
// n mul >> (31 + s), as mul exceeds 2^(31+s) / k by less than 2^s / k <= 2^(31+s) / (k n)
struct Divider {
  uint32_t mul;
  int shift;  // s - 1; k = 1: -1
  static Divider of(int k) {
    int s = 0;
    while ((1l << s) < k) ++s;
    if (s == 0) return {0, -1};
    return {(uint32_t)(((1ul << (31 + s)) + k - 1) / k), s - 1};
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return shift < 0 ? n : __umulhi(n, mul) >> shift; }
};

// A wavefront ranks its run of choices 64 at a time: the lanes that hold the same bin are found by a ballot a bit of the bin
// (stable: a lane's rank is the number of such lanes before it), then the bin's next position moves on.  The choices stay
// in registers between counting and ranking.  ALONE: one workgroup does the whole sort (n <= SORT_CHUNK) and counts for
// itself.
template <bool ALONE>
__global__ __launch_bounds__(512) void sort_scatter_kernel(const long* __restrict__ ids, int n, Divider k, int E, int bits,
                                                           int blocks, const int* __restrict__ count,
                                                           const int* __restrict__ total, long* __restrict__ rows,
                                                           long* __restrict__ offsets, int* __restrict__ slots) {
  __shared__ int pos[SORT_WAVES][SORT_MAX_E + 1];  // choices of a bin in a wavefront's run, then its next position
  __shared__ int start[SORT_MAX_E + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int STEPS = SORT_CHUNK / SORT_WAVES / 64;
  const int steps = ALONE ? ((n + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 : STEPS;
  const int i0 = (int)blockIdx.x * SORT_CHUNK + wave * steps * 64;
  int bin[STEPS];
#pragma unroll
  for (int q = 0; q < STEPS; ++q) {
    const int i = i0 + q * 64 + lane;
    bin[q] = q < steps && i < n ? bin_of(ids[i], E) : E + 1;
  }
  for (int w = 0; w < SORT_WAVES; ++w)
    for (int b = threadIdx.x; b <= E; b += 512) pos[w][b] = 0;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < STEPS; ++q)
    if (bin[q] <= E) atomicAdd(&pos[wave][bin[q]], 1);
  __syncthreads();
  if (wave == 0) {  // exclusive prefix of the bins' totals
    int base = 0;
    for (int b0 = 0; b0 <= E; b0 += 64) {
      const int b = b0 + lane;
      int v = 0;
      if (b <= E) {
        if (ALONE) {
#pragma unroll
          for (int w = 0; w < SORT_WAVES; ++w) v += pos[w][b];
        } else {
          v = total[b];
        }
      }
      int s = v;
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(s, o);
        if (lane >= o) s += u;
      }
      if (b <= E) start[b] = base + s - v;
      base += __shfl(s, 63);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b <= E; b += 512) {
    int at = start[b] + (ALONE ? 0 : count[(long)b * blocks + blockIdx.x]);
    if (blockIdx.x == 0) offsets[b] = start[b];
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int c = pos[w][b];
      pos[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < STEPS; ++q) {
    if (q >= steps) break;
    const int b = bin[q], i = i0 + q * 64 + lane;
    const bool in = b <= E;
    uint32_t lo = ~0u, hi = ~0u;  // lanes with this lane's bin
    for (int bit = 0; bit < bits; ++bit) {
      const unsigned long set = __ballot(b >> bit & 1);
      const uint32_t flip = (b >> bit & 1) - 1;
      lo &= (uint32_t)set ^ flip;
      hi &= (uint32_t)(set >> 32) ^ flip;
    }
    const int before = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
    if (in) {
      const int at = pos[wave][b] + before;
      rows[at] = k.div(i);
      if (slots) slots[i] = b == E ? -1 : at;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && before == 0) pos[wave][b] += __popc(lo) + __popc(hi);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---- combine --------------------------------------------------------------------------------------------
// One workgroup per (token, 2048 columns); the sum runs in the order of the token's choices, in 32 bits, and is rounded
// once, to the type TO of the results.  Slots outside [0, S) add nothing.  Bound by memory, for 8192 tokens of eight experts of
// 7168 columns: 397 us from fp32 to bf16 (5.0 TB/s), 223 from bf16 (4.7).
template <int DT, int TO, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(const void* __restrict__ Y, long ldy, int S, int C,
                                                      const int* __restrict__ slots, const float* __restrict__ weights, int k,
                                                      void* __restrict__ out, long ldo, int T) {
  const long t = (long)blockIdx.y * gridDim.x + blockIdx.x;
  const int c0 = (blockIdx.z * 256 + threadIdx.x) * 8;
  if (t >= T || c0 >= C) return;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < k; ++j) {
    const int s = slots[t * k + j];
    const float w = weights[t * k + j];
    if ((unsigned)s >= (unsigned)S) continue;
    const long at = (long)s * ldy + c0;
    float v[8];
    if (VEC) {
      if (DT == DT_F32) {
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>((const float*)Y + at);
        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>((const float*)Y + at + 4);
      } else {
        const uint4 u = *reinterpret_cast<const uint4*>((const uint16_t*)Y + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = load_val<DT>(&u, e);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c0 + e < C ? load_val<DT>(Y, at + e) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, v[e], acc[e]);
  }
  const long to = t * ldo + c0;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (VEC || c0 + e < C) {
      if (TO == DT_F32) ((float*)out)[to + e] = acc[e];
      else if (TO == DT_BF16) ((uint16_t*)out)[to + e] = f32_to_bf16_bits(acc[e]);
      else ((_Float16*)out)[to + e] = (_Float16)acc[e];
    }
}

template <int DT, int TO>
void combine_launch(const void* Y, long ldy, int S, int C, const int* slots, const float* weights, int T, int k, void* out,
                    long ldo, hipStream_t st) {
  constexpr int PER16 = DT == DT_F32 ? 4 : 8, PER16_TO = TO == DT_F32 ? 4 : 8;  // elements in 16 bytes
  const bool vec = C % 8 == 0 && ldy % PER16 == 0 && ldo % PER16_TO == 0 && ((uintptr_t)Y & 15) == 0 && ((uintptr_t)out & 15) == 0;
  const dim3 grid = mq_wide_grid(T, (C + 2047) / 2048);
  if (vec) hipLaunchKernelGGL((combine_kernel<DT, TO, true>), grid, dim3(256), 0, st, Y, ldy, S, C, slots, weights, k, out, ldo, T);
  else hipLaunchKernelGGL((combine_kernel<DT, TO, false>), grid, dim3(256), 0, st, Y, ldy, S, C, slots, weights, k, out, ldo, T);
}

}  // namespace

extern "C" int mq_route_experts(const void* logits, int dtype, long ldl, int T, int E, int top_k, int score, const float* bias,
                                int n_group, int topk_group, int group_top, int renormalize, float scale, float* weights,
                                long* ids, void* stream) {
  if (T < 0 || E <= 0 || E > ROUTE_MAX_E || top_k <= 0 || top_k > 64 || top_k > E || ldl < E) return MQ_ERR_ARG;
  if (score != SCORE_SOFTMAX && score != SCORE_SIGMOID) return MQ_ERR_ARG;
  if (n_group <= 0 || n_group > 64 || E % n_group || topk_group <= 0 || topk_group > n_group) return MQ_ERR_ARG;
  if (group_top < 1 || group_top > 2 || group_top > E / n_group || (long)topk_group * (E / n_group) < top_k) return MQ_ERR_ARG;
  if (dtype != DT_F32 && dtype != DT_BF16 && dtype != DT_F16) return MQ_ERR_ARG;
  if (T > 1 << 25) return MQ_ERR_TOO_LARGE;  // 64 threads a row at most, fewer than 2^32 in all
  if (T == 0) return MQ_OK;
  if (!logits || !weights || !ids) return MQ_ERR_ARG;
  RouteArgs a = {logits, ldl, T, E, top_k, score, bias, n_group, topk_group, group_top, renormalize, scale, weights, ids, 0, 0, 0, 0};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_F32) return mq_route_f32(a, st);
  if (dtype == DT_BF16) return mq_route_bf16(a, st);
  return mq_route_f16(a, st);
}

extern "C" size_t mq_sort_by_expert_workspace_bytes(int T, int top_k, int E) {
  if (T <= 0 || top_k <= 0 || E <= 0 || E > SORT_MAX_E || (long)T * top_k <= SORT_CHUNK) return 0;
  const size_t blocks = ((size_t)T * top_k + SORT_CHUNK - 1) / SORT_CHUNK;
  return (blocks + 1) * (E + 1) * sizeof(int);
}

extern "C" int mq_sort_by_expert(const long* ids, int T, int top_k, int E, long* rows, long* offsets, int* slots,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0 || top_k <= 0 || E <= 0 || E > SORT_MAX_E || (long)T * top_k > 0x7fffffffL - SORT_CHUNK) return MQ_ERR_ARG;
  if (!offsets || (T > 0 && (!ids || !rows))) return MQ_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  const int n = T * top_k;
  const Divider k = Divider::of(top_k);
  int bits = 0;
  while ((E + 1) >> bits) ++bits;
  if (n <= SORT_CHUNK) {
    hipLaunchKernelGGL((sort_scatter_kernel<true>), dim3(1), dim3(512), 0, st, ids, n, k, E, bits, 1, nullptr, nullptr, rows,
                       offsets, slots);
    return mq_check_launch();
  }
  if (!workspace || workspace_bytes < mq_sort_by_expert_workspace_bytes(T, top_k, E) || ((uintptr_t)workspace & 3)) return MQ_ERR_WORKSPACE;
  const int blocks = (n + SORT_CHUNK - 1) / SORT_CHUNK;
  int* total = reinterpret_cast<int*>(workspace);
  int* count = total + E + 1;
  hipLaunchKernelGGL(sort_count_kernel, dim3(blocks), dim3(512), 0, st, ids, n, E, blocks, count);
  hipLaunchKernelGGL(sort_scan_kernel, dim3(E + 1), dim3(256), 0, st, count, blocks, total);
  hipLaunchKernelGGL((sort_scatter_kernel<false>), dim3(blocks), dim3(512), 0, st, ids, n, k, E, bits, blocks, count, total,
                     rows, offsets, slots);
  return mq_check_launch();
}

extern "C" int mq_combine_experts_to(const void* Y, int dtype, long ldy, int S, int C, const int* slots, const float* weights,
                                     int T, int k, void* out, int out_dtype, long ldo, void* stream) {
  if (S < 0 || C <= 0 || T < 0 || k <= 0 || ldy < C || ldo < C || T > MQ_MAX_COUNT || C > 1 << 26) return MQ_ERR_ARG;
  if (dtype != DT_F32 && dtype != DT_BF16 && dtype != DT_F16) return MQ_ERR_ARG;
  if (out_dtype != dtype && (dtype != DT_F32 || (out_dtype != DT_BF16 && out_dtype != DT_F16))) return MQ_ERR_ARG;
  if (T == 0) return MQ_OK;
  if (!slots || !weights || !out || (S > 0 && !Y)) return MQ_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
#define MQ_COMBINE(DT, TO) combine_launch<DT, TO>(Y, ldy, S, C, slots, weights, T, k, out, ldo, st)
  if (dtype == DT_BF16) MQ_COMBINE(DT_BF16, DT_BF16);
  else if (dtype == DT_F16) MQ_COMBINE(DT_F16, DT_F16);
  else if (out_dtype == DT_BF16) MQ_COMBINE(DT_F32, DT_BF16);
  else if (out_dtype == DT_F16) MQ_COMBINE(DT_F32, DT_F16);
  else MQ_COMBINE(DT_F32, DT_F32);
#undef MQ_COMBINE
  return mq_check_launch();
}

extern "C" int mq_combine_experts(const void* Y, int dtype, long ldy, int S, int C, const int* slots, const float* weights,
                                  int T, int k, void* out, long ldo, void* stream) {
  return mq_combine_experts_to(Y, dtype, ldy, S, C, slots, weights, T, k, out, dtype, ldo, stream);
}
