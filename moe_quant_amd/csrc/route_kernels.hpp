// The router's kernels, one translation unit per type of logits (they compile side by side).
#pragma once
#include <math.h>

#include <type_traits>

#include "common.hpp"

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

int mq_route_f32(const RouteArgs& a, hipStream_t st);
int mq_route_bf16(const RouteArgs& a, hipStream_t st);
int mq_route_f16(const RouteArgs& a, hipStream_t st);

namespace {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
enum { SCORE_SOFTMAX = 0, SCORE_SIGMOID = 1 };

template <int DT>
__device__ __forceinline__ float load_val(const void* p, long i) {
  if (DT == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (DT == DT_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
  return (float)reinterpret_cast<const _Float16*>(p)[i];
}

__device__ __forceinline__ double wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The exact way: one wavefront routes one row, everything in 64 bits (which of two neighbouring experts is chosen hangs on
// differences far below a 32-bit step).  `c` (LDS, E values) holds what the experts are chosen by, NaN once an expert is out;
// `group` (LDS, 64 values) the groups' scores.  NaN logits count as -inf (the expert is chosen last); an expert that is equal
// to the row's maximum has weight exp(0) even where the maximum is +inf; a row whose logits are all -inf scores 0
// everywhere.  (Loops around exp stay rolled: the fast kernels carry this code along and must not pay registers for it.)
template <int DT>
struct ExactRow {
  const RouteArgs& a;
  const long base;
  double *c, *group;
  const int lane;
  const bool sigmoid;
  float m;
  double sum;

  __device__ __forceinline__ ExactRow(const RouteArgs& args, long row, double* c_, double* group_)
      : a(args), base(row * args.ldl), c(c_), group(group_), lane(threadIdx.x & 63), sigmoid(args.score == SCORE_SIGMOID) {}

  __device__ __forceinline__ float logit(int e) const { return fmaxf(load_val<DT>(a.logits, base + e), -INFINITY); }
  __device__ __forceinline__ double score(float l, double over) const {
    if (!sigmoid && l == m) return m == -INFINITY ? 0.0 : over;
    const double x = exp(sigmoid ? -(double)l : (double)l - (double)m);
    return sigmoid ? 1.0 / (1.0 + x) : x * over;
  }

  // c = score (+ bias) of every expert
  __device__ __forceinline__ void scores() {
    m = -INFINITY;
#pragma unroll 4
    for (int e = lane; e < a.E; e += 64) {
      const float l = logit(e);
      m = fmaxf(m, l);
      c[e] = (double)l;
    }
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    sum = 0.0;
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) {
      const double s = score((float)c[e], 1.0);
      sum += s;
      c[e] = s;
    }
    if (!sigmoid) sum = wave_sum(sum);
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) {
      double v = sigmoid ? c[e] : (sum > 0.0 ? c[e] / sum : 0.0);
      if (a.bias) {
        const double b = (double)a.bias[e];
        v = b == b ? v + b : -INFINITY;
      }
      c[e] = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

  // bit g: group g stays
  __device__ __forceinline__ unsigned long groups() {
    const int per = a.E / a.n_group;
    if (lane < a.n_group) {
      double best = -INFINITY, second = -INFINITY;
      int at = lane % per;
#pragma unroll 4
      for (int t = 0; t < per; ++t) {
        const double x = c[lane * per + at];
        second = fmax(second, fmin(best, x));
        best = fmax(best, x);
        at = at + 1 == per ? 0 : at + 1;
      }
      double total = a.group_top == 2 ? best + second : best;
      if (total != total) total = best;  // an infinite bias of each sign
      group[lane] = total;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    bool stays = false;
    if (lane < a.n_group) {
      const double mine = group[lane];
      int ahead = 0;
#pragma unroll 4
      for (int q = 0; q < a.n_group; ++q) ahead += group[q] > mine || (group[q] == mine && q < lane);
      stays = ahead < a.topk_group;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return __ballot(stays);
  }

  __device__ __forceinline__ void route(long row) {
    scores();
    const unsigned long kept = a.n_group > 1 ? groups() : ~0ul;
    if (a.n_group > 1 || !a.bias) {
      const int per = a.E / a.n_group;
#pragma unroll 1
      for (int e = lane; e < a.E; e += 64) {
        if (a.n_group > 1 && !(kept >> (e / per) & 1)) c[e] = NAN;
        else if (!a.bias) c[e] = (double)logit(e);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    int my_e = 0;
#pragma unroll 1
    for (int j = 0; j < a.top_k; ++j) {
      double best = -INFINITY;
      int be = 1 << 30;
#pragma unroll 4
      for (int e = lane; e < a.E; e += 64) {
        const double x = c[e];
        if (x > best || (x == best && e < be)) best = x, be = e;
      }
#pragma unroll 1
      for (int o = 32; o; o >>= 1) {
        const double ob = __shfl_xor(best, o);
        const int oe = __shfl_xor(be, o);
        if (ob > best || (ob == best && oe < be)) best = ob, be = oe;
      }
      if ((be & 63) == lane) c[be] = NAN;
      if (lane == j) my_e = be;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    double w = lane < a.top_k ? score(logit(my_e), sum > 0.0 ? 1.0 / sum : 0.0) : 0.0;
    if (a.renorm) w /= wave_sum(w) + 1e-20;
    if (lane < a.top_k) {
      a.ids[row * a.top_k + lane] = my_e;
      a.weights[row * a.top_k + lane] = (float)(w * (double)a.scale);
    }
  }
};

template <int DT>
__global__ __launch_bounds__(256) void route_exact_kernel(RouteArgs a) {
  __shared__ double c[4][1024], group[4][64];
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row < a.T) ExactRow<DT>(a, row, c[threadIdx.x >> 6], group[threadIdx.x >> 6]).route(row);
}

// The fast way, for up to 16 choices: L lanes a row, V logits a lane (chunks of four: expert 4 (lane + L i) + r), scores in 32
// bits.  A lane sorts its candidates once, as 32-bit keys that end in the candidate's place in the lane; the row's best is
// then taken k + 1 times, by a maximum over the lanes' heads.
//   Keys: the logits themselves (sigmoid without bias), exp(l - max) (softmax without bias) or the score + bias; they drop four
//   bits, and 32-bit scores are off by less than 2^-20 (exp: 2^-18 relative).  Logits of 16-bit types without a bias fit a
//   key with the expert's number behind them, where nothing is left to doubt.
//   Doubt: wherever two neighbours among the first k + 1 are closer than these errors allow, every candidate that could
//   belong to the k best (scores down to the k-th less the error) is ranked again by its exact 64-bit score; more than 16 of
//   them, or infinite logits, send the row the exact way.  Groups too close at the border of the choice: by their exact scores.
// At 256 experts about 650 vector instructions for four rows (63 comparators of the sort, 16 exponentials, 9 rounds of 4 + 2
// + shifts); reading 4 KB takes about as long.  Measured: 251 us for 1048576 x 256 fp32 logits (4.7 TB/s; the exact way alone
// 3800), 36 to 38 for 65536 rows with groups and bias (bound by instructions), 5.3 for one row.  17 choices and more go the
// exact way: 420 us for 65536 x 256 where 16 choices take 43.
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

// MODE: bit 0 a bias, bit 1 sigmoid scores; -1: as the arguments say (more than eight choices)
template <int DT, int L, int V, int KT, int MODE>
__global__ __launch_bounds__(256, 6) void route_kernel(RouteArgs a) {
  constexpr int RPW = 64 / L, RPB = 4 * RPW;  // rows of a wavefront, of a workgroup
  __shared__ __attribute__((aligned(16))) float cs[RPB][L == 64 ? 2 * L * V : L * V];  // (also: E doubles a wavefront)
  __shared__ float gs[RPB][64];
  __shared__ int res[RPB][16], cand[RPB][16];
  __shared__ double exact[4][64];  // (16 a row, or the groups of a row that goes the exact way)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / L, j = lane % L, slot = wave * RPW + sub;
  const long row0 = (long)blockIdx.x * RPB + wave * RPW;
  if (row0 >= a.T) return;
  const long row = min(row0 + sub, (long)a.T - 1);
  const long base = row * a.ldl;
  const bool sigmoid = MODE < 0 ? a.score == SCORE_SIGMOID : (MODE & 2) != 0, biased = MODE < 0 ? a.bias != nullptr : (MODE & 1) != 0;
  const bool scored = biased || a.n_group > 1;

  float l[V];
  if (a.vec) {  // (all loads first: chunks beyond E read the first one)
    typedef typename std::conditional<DT == DT_F32, float4, uint2>::type Four;
    Four x[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const int e0 = 4 * (j + L * i);
      x[i] = *reinterpret_cast<const Four*>((const char*)a.logits + (base + (e0 < a.E ? e0 : 0)) * (DT == DT_F32 ? 4 : 2));
    }
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) l[4 * i + r] = 4 * (j + L * i) < a.E ? load_val<DT>(&x[i], r) : -INFINITY;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = 4 * (j + L * (v >> 2)) + (v & 3);
      l[v] = e < a.E ? load_val<DT>(a.logits, base + e) : -INFINITY;
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    l[v] = fmaxf(l[v], -INFINITY);  // (a NaN becomes -inf)
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
    for (int v = 0; v < V; ++v) c[v] = sigmoid ? __builtin_amdgcn_rcpf(1.f + __expf(-l[v])) : c[v] * inv;
    if (biased) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const int e0 = 4 * (j + L * i);
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (e0 + 4 <= a.E) {
          __builtin_memcpy(b, a.bias + e0, 16);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (e0 + r < a.E) b[r] = a.bias[e0 + r];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) c[4 * i + r] = fmaxf(c[4 * i + r] + b[r], -INFINITY);
      }
    }
  }
  unsigned out = 0;  // bit v: this lane's candidate v is none (beyond E, or in a dropped group)
  if (a.E < L * V) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (4 * (j + L * (v >> 2)) + (v & 3) >= a.E) out |= 1u << v;
  }
  if (a.n_group > 1) {
    const int per = a.E / a.n_group;
    // the two best of a group may cancel (large biases of both signs): then the sum's error is not small against the sum
    bool unsure = false;
    const auto sum = [&](float best, float second) {
      unsure |= fabsf(best) + fabsf(second) > 4.f * fabsf(best + second) + 4.f;
      return best + second;
    };
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
        if ((at & (a.group_lanes - 1)) == 0 && 4 * at < a.E) gs[slot][at >> a.group_shift] = a.group_top == 2 ? sum(best, second) : best;
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
        gs[slot][g] = a.group_top == 2 ? sum(best, second) : best;
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
      else if (sure < a.topk_group) unsure = true;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int g = j, n = 0; g < a.n_group; g += L, ++n) gs[slot][g] = kept >> n & 1 ? 1.f : 0.f;
    const unsigned long who = __ballot(unsure);
    if (who) {  // groups too close in 32 bits: their exact scores decide
#pragma unroll 1
      for (int s = 0; s < RPW; ++s) {
        const unsigned long of = L == 64 ? ~0ul : ((1ul << (L & 63)) - 1) << (L * s);
        if (!(who & of)) continue;
        ExactRow<DT> row_s(a, min(row0 + s, (long)a.T - 1), reinterpret_cast<double*>(cs[wave * RPW]), exact[wave]);
        row_s.scores();
        const unsigned long stay = row_s.groups();
        for (int g = lane; g < a.n_group; g += 64) gs[wave * RPW + s][g] = stay >> g & 1 ? 1.f : 0.f;
      }
    }
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
  const bool sure_keys = SHORT && !biased, exp_keys = !SHORT && !biased && !sigmoid && !scored;
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = 4 * (j + L * (v >> 2)) + (v & 3);
    uint32_t k;
    if (sure_keys) {
      const float x = l[v] + 0.f;  // (no -0)
      uint32_t u;
      if (DT == DT_F16) {
        const _Float16 h = (_Float16)x;
        uint16_t b;
        __builtin_memcpy(&b, &h, 2);
        u = b ^ ((uint32_t)((int)(int16_t)b >> 15) & 0xffffu | 0x8000u);
      } else {
        u = ordered(x) >> 16;
      }
      k = u << 16 | (0xffffu - e);
    } else if (exp_keys) {
      k = (__float_as_uint(c[v]) & ~15u) | (15 - v);
    } else {
      k = (ordered(biased ? c[v] : l[v] + 0.f) & ~15u) | (15 - v);
    }
    key[v] = k;
  }
  if (out) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (out >> v & 1) key[v] = 0;
  }
  sort_down<V>(key);

  uint32_t last = 0, kth = 0;
  int popped = 0, found = 0;  // candidates this lane gave up; rounds that found one, the same in all of the row's lanes
  bool near = false;
#pragma unroll
  for (int r = 0; r <= KT; ++r) {
    if (r > a.top_k) break;  // (the same for all)
    const uint32_t best = row_max<L>(key[0]);
    const bool mine = key[0] == best && best != 0;
    if (!sure_keys && r > 0 && best != 0) {
      if (biased) {
        const float x = unordered(last & ~15u), y = unordered(best & ~15u);
        near |= !(x - y > 0x1p-19f + fabsf(x) * 0x1p-18f);
      } else {
        near |= last - best < (exp_keys ? 96u : 16u);  // exp: 2^-18 (32 steps) each, 16 dropped
      }
    }
    if (r < a.top_k) kth = best;
    last = best;
    found += best != 0;
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
  // equal keys in two lanes leave together, with one place of `res` for both: then more candidates have left than rounds found
  // one.  (Not more than top_k + 1: where hardly more than top_k candidates exist, the last rounds find none.)  Without such
  // keys every round before the last has found one, since at least top_k candidates exist, and every place is written.
  if (!sure_keys) near |= row_sum<L>((float)popped) > (float)found;

  const unsigned long my_row = L == 64 ? ~0ul : ((1ul << (L & 63)) - 1) << (L * sub);
  if (__ballot(near)) {
    near = (__ballot(near) & my_row) != 0;
    // softmax with a bias needs the exact sum over all logits; keys that have left the range of the error bounds
    if (near && ((biased && !sigmoid) || (exp_keys && kth < 0x2b800000u))) slow = true;  // (exp(l - max) < 2^-40)
    int n = 0;
    if (near && !slow) {
      // candidates: whatever may be among the k best.  Their number is counted in the row's lanes, chunk by chunk.
      const uint32_t low = kth & ~15u;
      const float fl = unordered(low), edge = fl - (0x1p-19f + fabsf(fl) * 0x1p-18f);
#pragma unroll 1
      for (int v = 0; v < V; ++v) {
        const int ev = 4 * (j + L * (v >> 2)) + (v & 3);
        bool in = ev < a.E && !(out >> v & 1);
        if (in) {
          const float x = fmaxf(load_val<DT>(a.logits, base + ev), -INFINITY) + 0.f;
          if (biased) in = !(fmaxf(__builtin_amdgcn_rcpf(1.f + __expf(-x)) + a.bias[ev], -INFINITY) < edge);
          else if (exp_keys) in = __float_as_uint(__expf(x - m)) + 96u >= low;
          else in = ordered(x) >= low;
        }
        const unsigned long who = __ballot(in) & my_row;
        const int at = n + __popcll(who & ((1ul << lane) - 1));
        if (in && at < 16) cand[slot][at] = ev;
        n += __popcll(who);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (n > 16) slow = true, n = 0;
    int mine = 0;
    double value = 0.0;
    if (j < n) {
      mine = cand[slot][j];
      const float x = fmaxf(load_val<DT>(a.logits, base + mine), -INFINITY);
      value = x;
      if (biased) {
        const float b = a.bias[mine];
        value = b == b ? 1.0 / (1.0 + exp(-(double)x)) + (double)b : -INFINITY;
      }
      exact[wave][16 * sub + j] = value;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (j < n) {
      int rank = 0;
      for (int q = 0; q < n; ++q) {
        const double other = exact[wave][16 * sub + q];
        rank += other > value || (other == value && cand[slot][q] < mine);
      }
      if (rank < a.top_k) res[slot][rank] = mine;
    }
  }

  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  float w = 0.f;
  int e = 0;
  if (j < a.top_k) {
    e = min(max(res[slot][j], 0), a.E - 1);  // (a slow row may have left a place empty: it is routed again below)
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
  if (!(who & my_row) && row0 + sub < a.T && j < a.top_k) {
    a.ids[row * a.top_k + j] = e;
    a.weights[row * a.top_k + j] = (a.renorm ? w / (sum + 1e-20f) : w) * a.scale;
  }
  if (who) {
#pragma unroll 1
    for (int s = 0; s < RPW; ++s) {
      const unsigned long of = L == 64 ? ~0ul : ((1ul << (L & 63)) - 1) << (L * s);
      if ((who & of) && row0 + s < a.T) ExactRow<DT>(a, row0 + s, reinterpret_cast<double*>(cs[wave * RPW]), exact[wave]).route(row0 + s);
    }
  }
}

template <int DT, int L, int V>
void route_fast(const RouteArgs& a, hipStream_t st) {
  constexpr int RPB = 4 * (64 / L);
  const dim3 grid((a.T + RPB - 1) / RPB), block(256);
  const int mode = (a.score == SCORE_SIGMOID ? 2 : 0) | (a.bias ? 1 : 0);
  if (a.top_k > 8) hipLaunchKernelGGL((route_kernel<DT, L, V, 16, -1>), grid, block, 0, st, a);
  else if (mode == 0) hipLaunchKernelGGL((route_kernel<DT, L, V, 8, 0>), grid, block, 0, st, a);
  else if (mode == 1) hipLaunchKernelGGL((route_kernel<DT, L, V, 8, 1>), grid, block, 0, st, a);
  else if (mode == 2) hipLaunchKernelGGL((route_kernel<DT, L, V, 8, 2>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((route_kernel<DT, L, V, 8, 3>), grid, block, 0, st, a);
}

template <int DT>
void route_any(RouteArgs a, hipStream_t st) {
  constexpr int W = DT == DT_F32 ? 4 : 2;
  a.vec = a.E % 4 == 0 && a.ldl % 4 == 0 && ((uintptr_t)a.logits % (4 * W)) == 0;
  a.by_group = ((1u << 20) + a.E / a.n_group - 1) / (a.E / a.n_group);  // e / per = e * by_group >> 20 for e < 1024
  const int per = a.E / a.n_group;
  for (int sh = 0; sh < 5; ++sh)
    if (per == 4 << sh) a.group_lanes = 1 << sh, a.group_shift = sh;
  if (a.top_k <= 16) {
    if (a.E <= 64) route_fast<DT, 16, 4>(a, st);
    else if (a.E <= 256) route_fast<DT, 16, 16>(a, st);
    else route_fast<DT, 64, 16>(a, st);
    return;
  }
  hipLaunchKernelGGL((route_exact_kernel<DT>), dim3((a.T + 3) / 4), dim3(256), 0, st, a);
}

}  // namespace
