// Linear layers on 8-bit integers: tokens quantized with a scale each, products with a scale per token and output channel.
//
//   mq_quantize_tokens     : x -> code = rint(127 x / max|x|), scale = max|x| / 127, row by row
//   mq_matmul_int8         : y[m, n] = (sum_k A[m, k] B[n, k]) * sa[m] * sb[n] (+ bias[n]), or the SwiGLU of two such halves
//   mq_matmul_int8_grouped : the same, every run of rows with the weights of its expert
#include <math.h>

#include <mutex>

#include "common.hpp"

namespace {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

template <int DT>
__device__ __forceinline__ float load_val(const void* p, long i) {
  if (DT == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (DT == DT_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
  return (float)reinterpret_cast<const _Float16*>(p)[i];
}
template <int DT>
__device__ __forceinline__ void store_val(void* p, long i, float v) {
  if (DT == DT_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (DT == DT_BF16) reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(v);
  else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}

// ---- quantize ---------------------------------------------------------------------------------------------
// The nearest whole number to 127 x / top, ties to even, as exact arithmetic gives it: x * inv (inv = 127 / top, 32 bits)
// is within 2^-14 of the quotient, so it decides except next to a border m + 1/2; there 254 |x| and (2 m + 1) top, both
// exact in 64 bits, are compared.
__device__ __forceinline__ int code_of(float x, float top, float inv) {
  const float z = fabsf(x * inv);
  float m = floorf(z);
  const float part = z - m;
  float r;
  if (fabsf(part - 0.5f) < 1.220703125e-4f) {
    const double have = 254.0 * (double)fabsf(x), border = (2.0 * (double)m + 1.0) * (double)top;
    const bool odd = ((int)m) & 1;
    r = m + ((have > border || (have == border && odd)) ? 1.f : 0.f);
  } else {
    r = m + (part > 0.5f ? 1.f : 0.f);
  }
  const int q = (int)r;
  return x < 0.f ? -q : q;
}

// One workgroup per token: the largest magnitude, then the codes (the second read of the row comes from the cache).  A row
// that holds a NaN or an infinity gets scale NaN and codes 0: its products are NaN, no other token's are.
template <int DT>
__global__ __launch_bounds__(256) void quantize_tokens_kernel(const void* __restrict__ X, long ldx, int C,
                                                              int8_t* __restrict__ Q, long ldq, float* __restrict__ scale) {
  __shared__ float part[4];
  const long row = blockIdx.x;
  float top = 0.f;
  bool bad = false;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float v = fabsf(load_val<DT>(X, row * ldx + c));
    bad |= !(v <= 3.402823466e38f);
    top = fmaxf(top, v);
  }
  if (bad) top = INFINITY;
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const bool fine = top <= 3.402823466e38f;
  if (threadIdx.x == 0) scale[row] = fine ? top / 127.f : NAN;
  const bool zero = !fine || top == 0.f;
  const float up = top < 0x1p-90f ? 0x1p90f : 1.f;  // keeps 127 / top finite; exact
  for (int c = threadIdx.x; c < C; c += 256)
    Q[row * ldq + c] = zero ? 0 : (int8_t)code_of(load_val<DT>(X, row * ldx + c) * up, top * up, 127.f / (top * up));
}

// ---- product ------------------------------------------------------------------------------------------------
struct Int8Args {
  const int8_t* A;
  long lda;
  const float* sa;
  const long* rows;  // grouped: row m of the product takes tokens row rows[m] (nullptr: row m)
  int src_rows;      // rows of A
  const int8_t* B;
  long ldb, strideB;
  const float* sb;
  const void* bias;
  void* Y;
  long ldy;
  int M, N, K;  // N: columns of Y
  const long* offsets;  // grouped: expert e owns rows offsets[e] .. offsets[e + 1)
  int E;
  int vec_out;
};

// Which rows a workgroup's row tile covers: its tile index -> expert, first row, end.  Experts' tiles follow one another;
// every wavefront finds its own with a prefix sum over the experts, 64 at a time.  Offsets are clamped to [0, M].
__device__ __forceinline__ bool find_tile(const Int8Args& a, int tile, int bm, int& e_out, int& m0, int& mend) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int e0 = 0; e0 < a.E; e0 += 64) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < a.E) {
      lo = (int)min(max(a.offsets[e], 0l), (long)a.M);
      hi = (int)min(max(a.offsets[e + 1], (long)lo), (long)a.M);
    }
    const int tiles = (hi - lo + bm - 1) / bm;
    int s = tiles;
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(s, o);
      if (lane >= o) s += u;
    }
    const bool mine = tile >= base + s - tiles && tile < base + s;
    const unsigned long who = __ballot(mine);
    if (who) {
      const int src = __builtin_ctzll(who);
      e_out = e0 + src;
      m0 = __shfl(lo, src) + (tile - __shfl(base + s - tiles, src)) * bm;
      mend = min(m0 + bm, __shfl(hi, src));
      return true;
    }
    base += __shfl(s, 63);
  }
  return false;
}

// four results of one row, columns n .. n + 3, as far as they exist
template <int DT>
__device__ __forceinline__ void store_run(void* Y, long row, int n, int N, int vec, const float* y) {
  if (n >= N) return;
  if (vec) {
    if (DT == DT_F32) {
      *reinterpret_cast<float4*>((float*)Y + row + n) = float4{y[0], y[1], y[2], y[3]};
    } else {
      uint16_t h[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) store_val<DT>(h, v, y[v]);
      uint2 w;
      __builtin_memcpy(&w, h, 8);
      *reinterpret_cast<uint2*>((uint16_t*)Y + row + n) = w;
    }
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (n + v < N) store_val<DT>(Y, row + n + v, y[v]);
  }
}

__device__ __forceinline__ float silu_times(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// 16 bytes of a row from byte k on, zeros beyond K (any alignment)
__device__ __forceinline__ intx4 load16(const int8_t* row, int k, int K, bool in) {
  intx4 v = {0, 0, 0, 0};
  if (!in || k >= K) return v;
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
    int8_t* b = reinterpret_cast<int8_t*>(&v);
    for (int i = 0; i < 16; ++i) b[i] = k + i < K ? row[k + i] : (int8_t)0;
  }
  return v;
}

// Any sizes, strides and alignment: 128 x 128 tiles, 64 deep, staged through registers and shared memory; four wavefronts
// of 64 x 64.  The weights are the matrix instruction's first operand, so a lane holds runs of four columns of one row.
constexpr int GBM = 128, GBN = 128, GBK = 64, GLD = GBK + 16;
template <int DT, bool SWIGLU>
__global__ __launch_bounds__(256) void int8_any_kernel(Int8Args a) {
  __shared__ __attribute__((aligned(16))) int8_t As[GBM * GLD];
  __shared__ __attribute__((aligned(16))) int8_t Bs[GBN * GLD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave >> 1, wn = wave & 1;
  int e = 0, m0 = blockIdx.y * GBM, mend = min(m0 + GBM, a.M);
  if (a.offsets && !find_tile(a, blockIdx.y, GBM, e, m0, mend)) return;
  constexpr int OUTN = SWIGLU ? GBN / 2 : GBN;
  const int n0 = blockIdx.x * OUTN;
  const int8_t* B = a.B + (long)e * a.strideB;
  const float* sb = a.sb + (long)e * (SWIGLU ? 2 * a.N : a.N);

  // this thread stages rows tid / 4 and tid / 4 + 64 of both tiles, 16 bytes at 16 * (tid % 4)
  const int8_t *arow[2], *brow[2];
  bool ain[2], bin[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = (tid >> 2) + 64 * h;
    long src = m0 + r;
    ain[h] = m0 + r < mend;
    if (ain[h] && a.rows) {
      src = a.rows[src];
      ain[h] = src >= 0 && src < a.src_rows;
    }
    arow[h] = a.A + (ain[h] ? src : 0) * a.lda;
    // SwiGLU: rows 0..31 of every 64 are gate rows, 32..63 the up rows of the same columns
    const int col = SWIGLU ? n0 + (r >> 6) * 32 + (r & 31) : n0 + r;
    bin[h] = col < a.N;
    brow[h] = B + (long)(bin[h] ? (SWIGLU && (r & 32) ? a.N + col : col) : 0) * a.ldb;
  }
  intx16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
  const int kc = 16 * (tid & 3);
  for (int k0 = 0; k0 < a.K; k0 += GBK) {
    intx4 va[2], vb[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      va[h] = load16(arow[h], k0 + kc, a.K, ain[h]);
      vb[h] = load16(brow[h], k0 + kc, a.K, bin[h]);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (tid >> 2) + 64 * h;
      *reinterpret_cast<intx4*>(As + r * GLD + kc) = va[h];
      *reinterpret_cast<intx4*>(Bs + r * GLD + kc) = vb[h];
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < GBK; kk += 32) {
      intx4 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = *reinterpret_cast<const intx4*>(As + (wm * 64 + i * 32 + (lane & 31)) * GLD + kk + 16 * (lane >> 5));
        fb[i] = *reinterpret_cast<const intx4*>(Bs + (wn * 64 + i * 32 + (lane & 31)) * GLD + kk + 16 * (lane >> 5));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = m0 + wm * 64 + i * 32 + (lane & 31);
    if (m >= mend) continue;
    long src = m;
    if (a.rows) src = a.rows[m];
    const float sa = src >= 0 && src < a.src_rows ? a.sa[src] : 0.f;
    if (SWIGLU) {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int n = n0 + wn * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
        if (n >= a.N) continue;
        const float g = (float)acc[i][0][v] * sa * sb[n], u = (float)acc[i][1][v] * sa * sb[a.N + n];
        store_val<DT>(a.Y, (long)m * a.ldy + n, silu_times(g, u));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int n = n0 + wn * 64 + j * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
          if (n >= a.N) continue;
          float y = (float)acc[i][j][v] * sa * sb[n];
          if (a.bias) y += load_val<DT>(a.bias, n);
          store_val<DT>(a.Y, (long)m * a.ldy + n, y);
        }
    }
  }
}

// 256 x 256 tiles for rows of at least 16 bytes that start at multiples of 4: eight wavefronts of 128 x 64, two per SIMD,
// four stages of 64 bytes of every row in shared memory, filled by direct 16-byte loads.
//   Layout of a stage: 256 token rows, then 256 weight rows, 64 bytes each; the 16-byte chunk c of row r lies at position
//   c ^ (r / 4 % 4), so that 16 lanes reading chunk c of 16 rows touch every bank once.
//   Pipeline: while the matrix instructions of one half of a stage run, the fragments of the other half are read; the loads
//   of stage t + 4 are issued into the slot of stage t once every wavefront has read its last fragment (one barrier a stage,
//   waits for exactly the loads that must have landed).
//   The last stage: a chunk that reaches beyond K is loaded from the last 16 bytes of the row instead (never outside it),
//   and the tokens' fragments drop the bytes that belong to earlier chunks, or all of them.
constexpr int TM = 256, TN = 256, TK = 64, NST = 4, STAGE = (TM + TN) * TK;
constexpr size_t TILE_SMEM = (size_t)NST * STAGE;

// lane i copies 16 bytes from its own address to LDS byte lds_addr + 16 i.  (Inline assembly: told about an LDS-writing
// load, the compiler would drain all of them before the next LDS read.  The kernel orders loads and reads itself.)
__device__ __forceinline__ void load_lds16(const int8_t* p, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds_addr) : "memory", "m0");
}

__device__ __forceinline__ intx4 keep_from(intx4 v, int drop) {  // bytes 0 .. drop - 1 become 0
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int d = drop - 4 * w;
    v[w] = d <= 0 ? v[w] : (d >= 4 ? 0 : v[w] & (int)(0xffffffffu << (8 * d)));
  }
  return v;
}

template <int DT, bool SWIGLU>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void int8_tile_kernel(Int8Args a) {
  extern __shared__ __attribute__((aligned(1024))) int8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  constexpr int OUTN = SWIGLU ? TN / 2 : TN;
  const int nt = (a.N + OUTN - 1) / OUTN;
  int e = 0, m0, mend, tn;
  if (a.offsets) {
    const int tile = blockIdx.x / nt;
    tn = blockIdx.x % nt;
    if (!find_tile(a, tile, TM, e, m0, mend)) return;
  } else {
    // tiles in bands of eight row tiles, every XCD (workgroup index mod 8) a run of its own: the 32 tiles it works on share
    // few panels
    const int mt = (a.M + TM - 1) / TM, total = mt * nt;
    const int xcd = blockIdx.x & 7, per = total >> 3, more = total & 7;
    const int id = xcd * per + min(xcd, more) + (blockIdx.x >> 3);
    const int band = id / (8 * nt), in = id - band * 8 * nt, rows = min(8, mt - 8 * band);
    m0 = (8 * band + in % rows) * TM;
    tn = in / rows;
    mend = min(m0 + TM, a.M);
  }
  m0 = __builtin_amdgcn_readfirstlane(m0);
  mend = __builtin_amdgcn_readfirstlane(mend);
  e = __builtin_amdgcn_readfirstlane(e);
  const int n0 = __builtin_amdgcn_readfirstlane(tn) * OUTN;
  const int8_t* B = a.B + (long)e * a.strideB;
  const float* sb = a.sb + (long)e * (SWIGLU ? 2 * a.N : a.N);
  const int nk = (a.K + TK - 1) / TK;

  // loads of this wavefront: rows 32 wave + 16 q + lane / 4 of the tokens (q = 0, 1) and of the weights (q = 2, 3)
  const int chunk = (lane & 3) ^ (lane >> 4);
  const int8_t* src[4];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r = 32 * wave + 16 * q + (lane >> 2);
    // SwiGLU: rows 0..31 of every 64 are gate rows, 32..63 the up rows of the same columns
    int col = SWIGLU ? n0 + (r >> 6) * 32 + (r & 31) : n0 + r;
    if (col >= a.N) col = n0;
    src[2 + q] = B + (long)(SWIGLU && (r & 32) ? a.N + col : col) * a.ldb + 16 * chunk;
    long from = min(m0 + r, mend - 1);
    if (a.rows) from = a.rows[from];
    src[q] = from >= 0 && from < a.src_rows ? a.A + from * a.lda + 16 * chunk : src[2 + q];
  }
  const int last = TK * (nk - 1) + 16 * chunk;      // this lane's chunk of the last stage starts here
  const int back = max(0, last - (a.K - 16));       // and is loaded from this much before
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t*)smem);
  // (stages past the last one load the last one's bytes again into slots nobody reads: the waits keep their counts)
  auto issue = [&](int s, int q) {
    const int off = s < nk - 1 ? TK * s : TK * (nk - 1) - back;
    load_lds16(src[q] + off, lds0 + (unsigned)((s % NST) * STAGE + (q >> 1) * TM * TK + wave * 2048 + (q & 1) * 1024));
  };

  intx16 acc[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
#pragma unroll
  for (int s = 0; s < NST - 1; ++s)
#pragma unroll
    for (int q = 0; q < 4; ++q) issue(s, q);
#pragma unroll
  for (int q = 0; q < 2; ++q) issue(NST - 1, q);

  const int lr = lane & 31, lk = lane >> 5;
  const int pos = lk ^ ((lr >> 2) & 3);
  const int a_off = (wm * 128 + lr) * TK, b_off = TM * TK + (wn * 64 + lr) * TK;
  const int at0 = 16 * pos, at1 = 16 * (pos ^ 2);  // chunks lk and 2 + lk
  intx4 fa0[4], fb0[2], fa1[4], fb1[2];
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | 10);  // stage 0 landed: at most the 10 loads of stages 1, 2, 3 in flight
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) fa0[i] = *reinterpret_cast<const intx4*>(smem + a_off + at0 + i * 32 * TK);
#pragma unroll
  for (int j = 0; j < 2; ++j) fb0[j] = *reinterpret_cast<const intx4*>(smem + b_off + at0 + j * 32 * TK);
#pragma unroll 1
  for (int kt = 0; kt < nk; ++kt) {
    const int8_t* stg = smem + (kt % NST) * STAGE;
    const int8_t* nxt = smem + ((kt + 1) % NST) * STAGE;
    const bool ragged = kt == nk - 1 && (a.K % TK);
    if (ragged) {
      const int d = max(0, TK * (nk - 1) + 16 * lk - (a.K - 16));
#pragma unroll
      for (int i = 0; i < 4; ++i) fa0[i] = keep_from(fa0[i], d);
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      acc[m >> 1][m & 1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb0[m & 1], fa0[m >> 1], acc[m >> 1][m & 1], 0, 0, 0);
      if (m < 4) fa1[m] = *reinterpret_cast<const intx4*>(stg + a_off + at1 + m * 32 * TK);
      else if (m < 6) fb1[m - 4] = *reinterpret_cast<const intx4*>(stg + b_off + at1 + (m - 4) * 32 * TK);
      else issue(kt + NST - 1, 2 + (m - 6));
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | 8);  // stage kt+1 landed: at most the 8 loads of stages kt+2, kt+3 in flight
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (ragged) {
      const int d = max(0, TK * (nk - 1) + 32 + 16 * lk - (a.K - 16));
#pragma unroll
      for (int i = 0; i < 4; ++i) fa1[i] = keep_from(fa1[i], d);
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      acc[m >> 1][m & 1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb1[m & 1], fa1[m >> 1], acc[m >> 1][m & 1], 0, 0, 0);
      if (m < 4) fa0[m] = *reinterpret_cast<const intx4*>(nxt + a_off + at0 + m * 32 * TK);
      else if (m < 6) fb0[m - 4] = *reinterpret_cast<const intx4*>(nxt + b_off + at0 + (m - 4) * 32 * TK);
      else issue(kt + NST, m - 6);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);

#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + wm * 128 + i * 32 + lr;
    if (m >= mend) continue;
    long from = m;
    if (a.rows) from = a.rows[m];
    const float sa = from >= 0 && from < a.src_rows ? a.sa[from] : 0.f;
#pragma unroll
    for (int j = 0; j < (SWIGLU ? 1 : 2); ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = n0 + (SWIGLU ? wn * 32 : wn * 64 + j * 32) + 8 * g + 4 * lk;
        float y[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int c = min(n + v, a.N - 1);
          if (SWIGLU) {
            y[v] = silu_times((float)acc[i][0][4 * g + v] * sa * sb[c], (float)acc[i][1][4 * g + v] * sa * sb[a.N + c]);
          } else {
            y[v] = (float)acc[i][j][4 * g + v] * sa * sb[c];
            if (a.bias) y[v] += load_val<DT>(a.bias, c);
          }
        }
        store_run<DT>(a.Y, (long)m * a.ldy, n, a.N, a.vec_out, y);
      }
  }
}

bool rows_of_words(const int8_t* p, long ld) { return ((uintptr_t)p & 3) == 0 && ld % 4 == 0; }

template <int DT, bool SWIGLU>
int int8_launch(const Int8Args& a, hipStream_t st) {
  if (a.K >= 16 && a.M >= 64 && rows_of_words(a.A, a.lda) && rows_of_words(a.B, a.ldb) && a.strideB % 4 == 0) {
    static std::once_flag once;
    static bool ok = false;
    std::call_once(once, [] {
      ok = hipFuncSetAttribute((const void*)int8_tile_kernel<DT, SWIGLU>, hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)TILE_SMEM) == hipSuccess;
    });
    if (!ok) return MQ_ERR_LAUNCH;
    const long mt = a.offsets ? (long)a.M / TM + min(a.E, a.M) : ((long)a.M + TM - 1) / TM;
    const int outn = SWIGLU ? TN / 2 : TN;
    const long grid = mt * ((a.N + outn - 1) / outn);
    if (grid > 0x7fffffffL) return MQ_ERR_TOO_LARGE;
    hipLaunchKernelGGL((int8_tile_kernel<DT, SWIGLU>), dim3((unsigned)grid), dim3(512), TILE_SMEM, st, a);
    return mq_check_launch();
  }
  const long mt = a.offsets ? (long)a.M / GBM + min(a.E, a.M) : ((long)a.M + GBM - 1) / GBM;
  const int outn = SWIGLU ? GBN / 2 : GBN;
  if (mt > 65535) return MQ_ERR_TOO_LARGE;
  hipLaunchKernelGGL((int8_any_kernel<DT, SWIGLU>), dim3((a.N + outn - 1) / outn, (unsigned)mt), dim3(256), 0, st, a);
  return mq_check_launch();
}

int int8_dispatch(Int8Args a, int dtype, int swiglu, hipStream_t st) {
  // runs of four results leave in one store where rows of Y allow it
  const int run = dtype == DT_F32 ? 16 : 8;
  a.vec_out = a.N % 4 == 0 && ((uintptr_t)a.Y % run) == 0 && a.ldy % 4 == 0;
  if (dtype == DT_F32) return swiglu ? int8_launch<DT_F32, true>(a, st) : int8_launch<DT_F32, false>(a, st);
  if (dtype == DT_BF16) return swiglu ? int8_launch<DT_BF16, true>(a, st) : int8_launch<DT_BF16, false>(a, st);
  return swiglu ? int8_launch<DT_F16, true>(a, st) : int8_launch<DT_F16, false>(a, st);
}

constexpr int MAX_K = 131071;  // |sum| <= K 128 128 stays inside 32 bits

}  // namespace

extern "C" int mq_quantize_tokens(const void* X, int dtype, long ldx, int n, int C, int8_t* Q, long ldq, float* scale,
                                  void* stream) {
  if (n < 0 || C <= 0 || ldx < C || ldq < C) return MQ_ERR_ARG;
  if (dtype != DT_F32 && dtype != DT_BF16 && dtype != DT_F16) return MQ_ERR_ARG;
  if (n == 0) return MQ_OK;
  if (!X || !Q || !scale) return MQ_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_F32)
    hipLaunchKernelGGL((quantize_tokens_kernel<DT_F32>), dim3(n), dim3(256), 0, st, X, ldx, C, Q, ldq, scale);
  else if (dtype == DT_BF16)
    hipLaunchKernelGGL((quantize_tokens_kernel<DT_BF16>), dim3(n), dim3(256), 0, st, X, ldx, C, Q, ldq, scale);
  else
    hipLaunchKernelGGL((quantize_tokens_kernel<DT_F16>), dim3(n), dim3(256), 0, st, X, ldx, C, Q, ldq, scale);
  return mq_check_launch();
}

extern "C" size_t mq_matmul_int8_workspace_bytes(int M, int N, int K, int swiglu) { return 0; }

extern "C" int mq_matmul_int8(const int8_t* A, long lda, const float* a_scale, const int8_t* B, long ldb,
                              const float* b_scale, const void* bias, void* Y, long ldy, int out_dtype, int M, int N, int K,
                              int swiglu, void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || K > MAX_K || lda < K || ldb < K || ldy < N || (swiglu && bias)) return MQ_ERR_ARG;
  if (out_dtype != DT_F32 && out_dtype != DT_BF16 && out_dtype != DT_F16) return MQ_ERR_ARG;
  if (M == 0) return MQ_OK;
  if (!A || !a_scale || !B || !b_scale || !Y) return MQ_ERR_ARG;
  const Int8Args a = {A, lda, a_scale, nullptr, M, B, ldb, 0, b_scale, bias, Y, ldy, M, N, K, nullptr, 1, 0};
  return int8_dispatch(a, out_dtype, swiglu, (hipStream_t)stream);
}

extern "C" int mq_matmul_int8_grouped(const int8_t* A, long lda, const float* a_scale, int src_rows, const long* rows, int S,
                                      const int8_t* B, long ldb, long strideB, const float* b_scale, int E,
                                      const long* offsets, void* Y, long ldy, int out_dtype, int N, int K, int swiglu,
                                      void* stream) {
  if (S < 0 || E <= 0 || E > 1024 || N <= 0 || K <= 0 || K > MAX_K || lda < K || ldb < K || ldy < N) return MQ_ERR_ARG;
  if (src_rows < 0 || strideB < 0 || (!rows && src_rows < S)) return MQ_ERR_ARG;
  if (out_dtype != DT_F32 && out_dtype != DT_BF16 && out_dtype != DT_F16) return MQ_ERR_ARG;
  if (S == 0) return MQ_OK;
  if (!A || !a_scale || !B || !b_scale || !offsets || !Y) return MQ_ERR_ARG;
  const Int8Args a = {A, lda, a_scale, rows, src_rows, B, ldb, strideB, b_scale, nullptr, Y, ldy, S, N, K, offsets, E, 0};
  return int8_dispatch(a, out_dtype, swiglu, (hipStream_t)stream);
}
