// Tokens to experts and back: the router's choice, the stable sort of tokens by expert, the weighted sum of the
// experts' outputs.
//
//   mq_route_experts   : logits -> the top_k experts of each token and their weights
//   mq_sort_by_expert  : expert ids -> token rows in expert order, offsets, and each choice's position in that order
//   mq_combine_experts : out[t] = sum_j weight[t, j] * Y[slot[t, j]]
#include <math.h>

#include "common.hpp"

namespace {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
enum { SCORE_SOFTMAX = 0, SCORE_SIGMOID = 1 };
constexpr int ROUTE_MAX_E = 1024;

template <int DT>
__device__ __forceinline__ float load_val(const void* p, long i) {
  if (DT == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (DT == DT_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
  return (float)reinterpret_cast<const _Float16*>(p)[i];
}

struct RouteArgs {
  const void* logits;
  long ldl;
  int T, E, top_k, score;
  const float* bias;
  int n_group, topk_group, group_top, renorm;
  float scale;
  float* weights;
  long* ids;
  int vec;
  unsigned by_group;
  int group_lanes, group_shift;  // chunks of four experts in a group, where that is 1, 2, 4, 8 or 16; else 0
};

__device__ __forceinline__ double wave_max(double v) {
  for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The exact way: one wavefront routes one row, everything in 64 bits (which of two neighbouring experts is chosen hangs on
// differences far below a 32-bit step).  Lane l holds experts l, l + 64, ...; `group` (LDS, one wavefront's) holds the groups'
// scores.  NaN logits count as -inf (the expert is chosen last); an expert that is equal to the row's maximum has weight
// exp(0) even where the maximum is +inf; a row whose logits are all -inf scores 0 everywhere.
template <int DT, int V>
__device__ __forceinline__ void route_row(const RouteArgs& a, long row, double* group) {
  const int lane = threadIdx.x & 63;
  const long base = row * a.ldl;
  float l[V];
  double s[V], c[V];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane + 64 * i;
    l[i] = e < a.E ? load_val<DT>(a.logits, base + e) : -INFINITY;
    if (!(l[i] == l[i])) l[i] = -INFINITY;
    m = fmaxf(m, l[i]);
  }
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (a.score == SCORE_SIGMOID) {
      s[i] = 1.0 / (1.0 + exp(-(double)l[i]));
    } else {
      s[i] = m == -INFINITY ? 0.0 : (l[i] == m ? 1.0 : exp((double)l[i] - (double)m));
      sum += s[i];
    }
  }
  if (a.score == SCORE_SOFTMAX) {
    sum = wave_sum(sum);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
  }
  // without a bias the order of the scores is the order of the logits, which no rounding has touched
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane + 64 * i;
    if (a.bias) {
      double b = e < a.E ? (double)a.bias[e] : 0.0;
      c[i] = b == b ? s[i] + b : -INFINITY;
    } else {
      c[i] = a.n_group > 1 ? s[i] : (double)l[i];
    }
  }
  unsigned taken = 0;  // bit i: this lane's expert i is out (taken, in a dropped group, or beyond E)
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (lane + 64 * i >= a.E) taken |= 1u << i;
  if (a.n_group > 1) {
    const int per = a.E / a.n_group;
    for (int g = 0; g < a.n_group; ++g) {
      double best = -INFINITY, second = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = lane + 64 * i;
        if (e / per == g && e < a.E) {
          second = fmax(second, fmin(best, c[i]));
          best = fmax(best, c[i]);
        }
      }
      for (int o = 32; o; o >>= 1) {
        const double ob = __shfl_xor(best, o), os = __shfl_xor(second, o);
        second = fmax(fmin(best, ob), fmax(second, os));
        best = fmax(best, ob);
      }
      double total = a.group_top == 2 ? best + second : best;
      if (total != total) total = best;  // an infinite bias of each sign
      if (lane == 0) group[g] = total;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 64 * i;
      if (e < a.E) {
        const int g = e / per;
        const double mine = group[g];
        int ahead = 0;
        for (int q = 0; q < a.n_group; ++q) ahead += group[q] > mine || (group[q] == mine && q < g);
        if (ahead >= a.topk_group) taken |= 1u << i;
        if (!a.bias) c[i] = (double)l[i];
      }
    }
  }
  double sum_w = 0.0, my_w = 0.0;
  int my_e = 0;
  for (int j = 0; j < a.top_k; ++j) {
    double best = -INFINITY, bs = 0.0;
    int be = 1 << 30;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 64 * i;
      if (!(taken >> i & 1) && (c[i] > best || (c[i] == best && e < be))) best = c[i], be = e, bs = s[i];
    }
    for (int o = 32; o; o >>= 1) {
      const double ob = __shfl_xor(best, o), os = __shfl_xor(bs, o);
      const int oe = __shfl_xor(be, o);
      if (ob > best || (ob == best && oe < be)) best = ob, be = oe, bs = os;
    }
    if ((be & 63) == lane) taken |= 1u << (be >> 6);
    sum_w += bs;
    if (lane == j) my_w = bs, my_e = be;
  }
  if (lane < a.top_k) {
    if (a.renorm) my_w /= sum_w + 1e-20;
    a.ids[row * a.top_k + lane] = my_e;
    a.weights[row * a.top_k + lane] = (float)(my_w * (double)a.scale);
  }
}

template <int DT, int V>
__global__ __launch_bounds__(256) void route_exact_kernel(RouteArgs a) {
  __shared__ double group[4][64];
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row < a.T) route_row<DT, V>(a, row, group[threadIdx.x >> 6]);
}

// The fast way, for up to 16 choices: L lanes a row, V logits a lane (chunks of four: expert 4 (lane + L i) + r), scores in 32
// bits.  A lane sorts its candidates once, as 32-bit keys that end in the candidate's place in the lane; the row's best is
// then taken k + 1 times, by a maximum over the lanes' heads.  Scores in 32 bits are off by less than 2^-20 (+ their own
// rounding) and a key drops four bits, so wherever two neighbours among the first k + 1, or two groups at the border of the
// choice, are closer than that together allows, the row goes the exact way: about one row in a thousand at 256 experts.
// Without a bias the keys are the logits themselves; those of 16-bit types fit a key with the expert's number behind them,
// where nothing is left to doubt.
// Per row of 256: ~450 vector instructions for four rows (63 comparators of the sort, 9 rounds of 4 + 2 + shifts), about
// what reading 1 KB takes.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, dpp<0x128>(v));  // rotations within 16 lanes by 8, 4, 2, 1
  v = max(v, dpp<0x124>(v));
  v = max(v, dpp<0x122>(v));
  v = max(v, dpp<0x121>(v));
  if (L == 64) {
    v = max(v, (uint32_t)__shfl_xor((int)v, 16));
    v = max(v, (uint32_t)__shfl_xor((int)v, 32));
  }
  return v;
}
template <int L>
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, __uint_as_float(dpp<0x128>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(dpp<0x124>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(dpp<0x122>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(dpp<0x121>(__float_as_uint(v))));
  if (L == 64) {
    v = fmaxf(v, __shfl_xor(v, 16));
    v = fmaxf(v, __shfl_xor(v, 32));
  }
  return v;
}
template <int L>
__device__ __forceinline__ float row_sum(float v) {
  v += __uint_as_float(dpp<0x128>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x124>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x122>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x121>(__float_as_uint(v)));
  if (L == 64) {
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
  }
  return v;
}

// order-preserving bits of a float (no NaN, no -0)
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k ^ (~(uint32_t)((int)k >> 31) | 0x80000000u)); }

// descending, by odd-even merges: N = 4, 8, 16
template <int N>
__device__ __forceinline__ void sort_down(uint32_t* k) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t x = k[i + j], y = k[i + j + q];
            k[i + j] = max(x, y);
            k[i + j + q] = min(x, y);
          }
}

template <int DT, int L, int V, int KT>
__global__ __launch_bounds__(256, 5) void route_kernel(RouteArgs a) {
  constexpr int RPW = 64 / L, RPB = 4 * RPW;  // rows of a wavefront, of a workgroup
  __shared__ float cs[RPB][L * V];
  __shared__ float gs[RPB][64];
  __shared__ int res[RPB][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / L, j = lane % L, slot = wave * RPW + sub;
  const long row0 = (long)blockIdx.x * RPB + wave * RPW;
  if (row0 >= a.T) return;
  const long row = min(row0 + sub, (long)a.T - 1);
  const long base = row * a.ldl;
  const bool sigmoid = a.score == SCORE_SIGMOID, scored = a.bias || a.n_group > 1;

  float l[V];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const int e0 = 4 * (j + L * i);
    if (a.vec) {
      if (e0 < a.E) {
        if (DT == DT_F32) {
          const float4 x = *reinterpret_cast<const float4*>((const float*)a.logits + base + e0);
          l[4 * i] = x.x, l[4 * i + 1] = x.y, l[4 * i + 2] = x.z, l[4 * i + 3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>((const uint16_t*)a.logits + base + e0);
#pragma unroll
          for (int r = 0; r < 4; ++r) l[4 * i + r] = load_val<DT>(&x, r);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) l[4 * i + r] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) l[4 * i + r] = e0 + r < a.E ? load_val<DT>(a.logits, base + e0 + r) : -INFINITY;
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    l[v] = l[v] == l[v] ? l[v] + 0.f : -INFINITY;  // (+ 0: no -0)
    m = fmaxf(m, l[v]);
  }
  bool slow = false;
  float inv = 0.f;
  float c[V];
  if (!sigmoid) {
    m = row_max<L>(m);
    slow = !(fabsf(m) < INFINITY);
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      c[v] = __expf(l[v] - m);
      sum += c[v];
    }
    inv = 1.f / row_sum<L>(sum);
  }
  if (scored) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const int e0 = 4 * (j + L * i);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int v = 4 * i + r;
        const float s = sigmoid ? __builtin_amdgcn_rcpf(1.f + __expf(-l[v])) : c[v] * inv;
        c[v] = s;
        if (a.bias) {
          c[v] = s + (e0 + r < a.E ? a.bias[e0 + r] : 0.f);
          c[v] = c[v] == c[v] ? c[v] + 0.f : -INFINITY;
        }
      }
    }
  }
  unsigned out = 0;  // bit v: this lane's candidate v is none (beyond E, or in a dropped group)
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (4 * (j + L * (v >> 2)) + (v & 3) >= a.E) out |= 1u << v;
  if (a.n_group > 1) {
    const int per = a.E / a.n_group;
    if (a.group_lanes) {
      // a group is a run of 1, 2, 4, 8 or 16 lanes' chunks: exchanges with the lane 1, 2, 4, 8 away (mirrors do for the last
      // two: the quads, then the halves, agree by then)
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const float x = fmaxf(c[4 * i], c[4 * i + 1]), y = fmaxf(c[4 * i + 2], c[4 * i + 3]);
        float best = fmaxf(x, y);
        float second = fmaxf(fminf(x, y), fmaxf(fminf(c[4 * i], c[4 * i + 1]), fminf(c[4 * i + 2], c[4 * i + 3])));
        const auto meet = [&](float ob, float os) {
          second = fmaxf(fminf(best, ob), fmaxf(second, os));
          best = fmaxf(best, ob);
        };
#define MQ_MEET(CTRL) meet(__uint_as_float(dpp<CTRL>(__float_as_uint(best))), __uint_as_float(dpp<CTRL>(__float_as_uint(second))))
        if (a.group_lanes >= 2) MQ_MEET(0xB1);
        if (a.group_lanes >= 4) MQ_MEET(0x4E);
        if (a.group_lanes >= 8) MQ_MEET(0x141);
        if (a.group_lanes >= 16) MQ_MEET(0x140);
#undef MQ_MEET
        const int at = j + L * i;
        if ((at & (a.group_lanes - 1)) == 0 && 4 * at < a.E) gs[slot][at >> a.group_shift] = a.group_top == 2 ? best + second : best;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        *reinterpret_cast<float4*>(&cs[slot][4 * (j + L * i)]) = float4{c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]};
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int g = j; g < a.n_group; g += L) {
        float best = -INFINITY, second = -INFINITY;
        int at = g % per;  // (every lane starts elsewhere: equal places of equally long groups share a bank)
#pragma unroll 4
        for (int t = 0; t < per; ++t) {
          const float x = cs[slot][g * per + at];
          second = fmaxf(second, fminf(best, x));
          best = fmaxf(best, x);
          at = at + 1 == per ? 0 : at + 1;
        }
        gs[slot][g] = a.group_top == 2 ? best + second : best;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    unsigned kept = 0;
    for (int g = j, n = 0; g < a.n_group; g += L, ++n) {
      const float mine = gs[slot][g], near = 0x1p-18f + fabsf(mine) * 0x1p-20f;
      int sure = 0, maybe = 0;
#pragma unroll 4
      for (int q = 0; q < a.n_group; ++q) {
        const float other = gs[slot][q];
        sure += other > mine + near;
        maybe += q != g && !(other < mine - near);
      }
      if (maybe < a.topk_group) kept |= 1u << n;
      else if (sure < a.topk_group) slow = true;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int g = j, n = 0; g < a.n_group; g += L, ++n) gs[slot][g] = kept >> n & 1 ? 1.f : 0.f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (a.group_lanes) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        if (gs[slot][min((j + L * i) >> a.group_shift, a.n_group - 1)] == 0.f) out |= 15u << (4 * i);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = min(4 * (j + L * (v >> 2)) + (v & 3), a.E - 1);
        if (gs[slot][(unsigned)e * a.by_group >> 20] == 0.f) out |= 1u << v;
      }
    }
  }

  constexpr bool SHORT = DT != DT_F32;
  const bool sure_keys = SHORT && !a.bias;
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = 4 * (j + L * (v >> 2)) + (v & 3);
    uint32_t k;
    if (sure_keys) {
      uint32_t u;
      if (DT == DT_F16) {
        const _Float16 h = (_Float16)l[v];
        uint16_t b;
        __builtin_memcpy(&b, &h, 2);
        u = b ^ ((uint32_t)((int)(int16_t)b >> 15) & 0xffffu | 0x8000u);
      } else {
        u = ordered(l[v]) >> 16;
      }
      k = u << 16 | (0xffffu - e);
    } else {
      k = (ordered(a.bias ? c[v] : l[v]) & ~15u) | (15 - v);
    }
    key[v] = out >> v & 1 ? 0u : k;
  }
  sort_down<V>(key);

  uint32_t last = 0;
  int popped = 0;
#pragma unroll
  for (int r = 0; r <= KT; ++r) {
    if (r > a.top_k) break;  // (the same for all)
    const uint32_t best = row_max<L>(key[0]);
    const bool mine = key[0] == best && best != 0;
    if (!sure_keys && r > 0 && best != 0) {
      if (a.bias) {
        const float x = unordered(last & ~15u), y = unordered(best & ~15u);
        slow |= !(x - y > 0x1p-19f + fabsf(x) * 0x1p-18f);
      } else {
        slow |= (last ^ best) < 16u;
      }
    }
    last = best;
    if (mine) {
      ++popped;
      if (r < a.top_k) {
        const int v = 15 - (int)(best & 15);
        res[slot][r] = sure_keys ? (int)(0xffffu - (best & 0xffffu)) : 4 * (j + L * (v >> 2)) + (v & 3);
      }
#pragma unroll
      for (int v = 0; v + 1 < V && v < KT - r; ++v) key[v] = key[v + 1];
      if (V <= KT - r) key[V - 1] = 0;
    }
  }
  // equal keys in two lanes leave together: then more have been taken than rounds were run
  float taken = row_sum<L>((float)popped);
  slow |= taken > (float)(a.top_k + 1);

  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  float w = 0.f;
  int e = 0;
  if (j < a.top_k) {
    e = min(max(res[slot][j], 0), a.E - 1);  // (a slow row may have left a place empty)
    const float x = load_val<DT>(a.logits, base + e);
    if (sigmoid) {
      w = 1.f / (1.f + __expf(-x));
      slow |= !(x > -80.f);  // exp(-x) would leave 32 bits
    } else {
      w = __expf(x - m) * inv;
      slow |= !(x - m > -80.f);
    }
  }
  const float sum = row_sum<L>(w);
  const unsigned long who = __ballot(slow);
  const unsigned long mask = L == 64 ? ~0ul : ((1ul << (L & 63)) - 1) << (L * sub);
  if (!(who & mask) && row0 + sub < a.T && j < a.top_k) {
    a.ids[row * a.top_k + j] = e;
    a.weights[row * a.top_k + j] = (a.renorm ? w / (sum + 1e-20f) : w) * a.scale;
  }
  if (who) {
#pragma unroll 1
    for (int s = 0; s < RPW; ++s) {
      const unsigned long of = L == 64 ? ~0ul : ((1ul << (L & 63)) - 1) << (L * s);
      if ((who & of) && row0 + s < a.T) route_row<DT, L * V / 64>(a, row0 + s, reinterpret_cast<double*>(cs[wave * RPW]));
    }
  }
}

template <int DT, int L, int V>
void route_fast(const RouteArgs& a, hipStream_t st) {
  constexpr int RPB = 4 * (64 / L);
  const dim3 grid((a.T + RPB - 1) / RPB), block(256);
  if (a.top_k <= 8) hipLaunchKernelGGL((route_kernel<DT, L, V, 8>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((route_kernel<DT, L, V, 16>), grid, block, 0, st, a);
}

template <int DT>
void route_launch(RouteArgs a, hipStream_t st) {
  constexpr int W = DT == DT_F32 ? 4 : 2;
  a.vec = a.E % 4 == 0 && a.ldl % 4 == 0 && ((uintptr_t)a.logits % (4 * W)) == 0;
  a.by_group = ((1u << 20) + a.E / a.n_group - 1) / (a.E / a.n_group);  // e / per = e * by_group >> 20 for e < 1024
  const int per = a.E / a.n_group;
  for (int sh = 0; sh < 5; ++sh)
    if (per == 4 << sh) a.group_lanes = 1 << sh, a.group_shift = sh;
  if (a.top_k <= 16) {
    if (a.E <= 64) route_fast<DT, 16, 4>(a, st);
    else if (a.E <= 128) route_fast<DT, 16, 8>(a, st);
    else if (a.E <= 256) route_fast<DT, 16, 16>(a, st);
    else route_fast<DT, 64, 16>(a, st);
    return;
  }
  const dim3 grid((a.T + 3) / 4), block(256);
  if (a.E <= 256) hipLaunchKernelGGL((route_exact_kernel<DT, 4>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((route_exact_kernel<DT, 16>), grid, block, 0, st, a);
}

// ---- sort by expert -----------------------------------------------------------------------------------
// Stable counting sort of n = T * top_k choices into E + 1 bins (bin E: ids outside [0, E)).  A workgroup owns a run of
// SORT_CHUNK choices; `count` holds, bin-major, the number of choices of every (bin, workgroup).
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

// ALONE: one workgroup does the whole sort (n <= SORT_CHUNK) and counts for itself.
template <bool ALONE>
__global__ __launch_bounds__(512) void sort_scatter_kernel(const long* __restrict__ ids, int n, int k, int E, int blocks,
                                                           const int* __restrict__ count, const int* __restrict__ total,
                                                           long* __restrict__ rows, long* __restrict__ offsets,
                                                           int* __restrict__ slots) {
  __shared__ int pos[SORT_WAVES][SORT_MAX_E + 1];  // choices of a bin in a wavefront's run, then its next position
  __shared__ int start[SORT_MAX_E + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int w = 0; w < SORT_WAVES; ++w)
    for (int b = threadIdx.x; b <= E; b += 512) pos[w][b] = 0;
  __syncthreads();
  const int per = ALONE ? ((n + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64 : SORT_CHUNK / SORT_WAVES;
  const long i0 = (long)blockIdx.x * SORT_CHUNK + wave * per;
  for (int q = 0; q < per; q += 64) {
    const long i = i0 + q + lane;
    if (i < n) atomicAdd(&pos[wave][bin_of(ids[i], E)], 1);
  }
  __syncthreads();
  if (wave == 0) {  // exclusive prefix of the bins' totals
    int base = 0;
    for (int b0 = 0; b0 <= E; b0 += 64) {
      const int b = b0 + lane;
      int v = 0;
      if (b <= E) {
        if (ALONE)
          for (int w = 0; w < SORT_WAVES; ++w) v += pos[w][b];
        else v = total[b];
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
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int c = pos[w][b];
      pos[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int q = 0; q < per; q += 64) {
    const long i = i0 + q + lane;
    const bool in = i < n;
    const int b = in ? bin_of(ids[i], E) : E + 1;
    unsigned long same = ~0ul;  // lanes with this lane's bin
    for (int bit = 0; bit < 11; ++bit) {
      const unsigned long set = __ballot(b >> bit & 1);
      same &= (b >> bit & 1) ? set : ~set;
    }
    const int before = __popcll(same & ((1ul << lane) - 1));
    if (in) {
      const int at = pos[wave][b] + before;
      rows[at] = i / k;
      if (slots) slots[i] = b == E ? -1 : at;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && before == 0) pos[wave][b] += __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---- combine --------------------------------------------------------------------------------------------
// One workgroup per (token, 2048 columns); the sum runs in the order of the token's choices, in 32 bits, and is rounded
// once.  Slots outside [0, S) add nothing.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(const void* __restrict__ Y, long ldy, int S, int C,
                                                      const int* __restrict__ slots, const float* __restrict__ weights, int k,
                                                      void* __restrict__ out, long ldo) {
  const long t = blockIdx.x;
  const int c0 = (blockIdx.y * 256 + threadIdx.x) * 8;
  if (c0 >= C) return;
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
      if (DT == DT_F32) ((float*)out)[to + e] = acc[e];
      else if (DT == DT_BF16) ((uint16_t*)out)[to + e] = f32_to_bf16_bits(acc[e]);
      else ((_Float16*)out)[to + e] = (_Float16)acc[e];
    }
}

template <int DT>
void combine_launch(const void* Y, long ldy, int S, int C, const int* slots, const float* weights, int T, int k, void* out,
                    long ldo, hipStream_t st) {
  const int per16 = DT == DT_F32 ? 4 : 8;  // elements in 16 bytes
  const bool vec = C % 8 == 0 && ldy % per16 == 0 && ldo % per16 == 0 && ((uintptr_t)Y & 15) == 0 && ((uintptr_t)out & 15) == 0;
  const dim3 grid(T, (C + 2047) / 2048);
  if (vec) hipLaunchKernelGGL((combine_kernel<DT, true>), grid, dim3(256), 0, st, Y, ldy, S, C, slots, weights, k, out, ldo);
  else hipLaunchKernelGGL((combine_kernel<DT, false>), grid, dim3(256), 0, st, Y, ldy, S, C, slots, weights, k, out, ldo);
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
  if (T == 0) return MQ_OK;
  if (!logits || !weights || !ids) return MQ_ERR_ARG;
  RouteArgs a = {logits, ldl, T, E, top_k, score, bias, n_group, topk_group, group_top, renormalize, scale, weights, ids, 0, 0, 0, 0};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_F32) route_launch<DT_F32>(a, st);
  else if (dtype == DT_BF16) route_launch<DT_BF16>(a, st);
  else route_launch<DT_F16>(a, st);
  return mq_check_launch();
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
  if (n <= SORT_CHUNK) {
    hipLaunchKernelGGL((sort_scatter_kernel<true>), dim3(1), dim3(512), 0, st, ids, n, top_k, E, 1, nullptr, nullptr, rows,
                       offsets, slots);
    return mq_check_launch();
  }
  if (!workspace || workspace_bytes < mq_sort_by_expert_workspace_bytes(T, top_k, E)) return MQ_ERR_WORKSPACE;
  const int blocks = (n + SORT_CHUNK - 1) / SORT_CHUNK;
  int* total = reinterpret_cast<int*>(workspace);
  int* count = total + E + 1;
  hipLaunchKernelGGL(sort_count_kernel, dim3(blocks), dim3(512), 0, st, ids, n, E, blocks, count);
  hipLaunchKernelGGL(sort_scan_kernel, dim3(E + 1), dim3(256), 0, st, count, blocks, total);
  hipLaunchKernelGGL((sort_scatter_kernel<false>), dim3(blocks), dim3(512), 0, st, ids, n, top_k, E, blocks, count, total,
                     rows, offsets, slots);
  return mq_check_launch();
}

extern "C" int mq_combine_experts(const void* Y, int dtype, long ldy, int S, int C, const int* slots, const float* weights,
                                  int T, int k, void* out, long ldo, void* stream) {
  if (S < 0 || C <= 0 || T < 0 || k <= 0 || ldy < C || ldo < C) return MQ_ERR_ARG;
  if (dtype != DT_F32 && dtype != DT_BF16 && dtype != DT_F16) return MQ_ERR_ARG;
  if (T == 0) return MQ_OK;
  if (!slots || !weights || !out || (S > 0 && !Y)) return MQ_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_F32) combine_launch<DT_F32>(Y, ldy, S, C, slots, weights, T, k, out, ldo, st);
  else if (dtype == DT_BF16) combine_launch<DT_BF16>(Y, ldy, S, C, slots, weights, T, k, out, ldo, st);
  else combine_launch<DT_F16>(Y, ldy, S, C, slots, weights, T, k, out, ldo, st);
  return mq_check_launch();
}
