// Linear layers on 8-bit integers: tokens quantized with a scale each, products with a scale per token and output channel.
//
//   mq_quantize_tokens     : x -> code = rint(127 x / max|x|), scale = max|x| / 127, row by row
//   mq_matmul_int8         : y[m, n] = (sum_k A[m, k] B[n, k]) * sa[m] * sb[n] (+ bias[n]), or the SwiGLU of two such halves
//   mq_matmul_int8_grouped : the same, every run of rows with the weights of its expert
#include "int8_kernels.hpp"

namespace {

// TPR threads per token, eight values each in turn: the largest magnitude first, then the codes, from the NV vectors a
// thread keeps in registers (NV = 0: rows too long for that, read twice, the second time from the cache).  A row that holds
// a NaN or an infinity gets scale NaN and codes 0: its products are NaN, no other token's are.
// Bound by memory: 163 to 180 us for 16384 x 16384 bf16 (4.5 to 4.9 TB/s read and written; read twice and element by element it
// took 587); 7 us for 333 x 7168.
template <int DT, int TPR, int NV>
__global__ __launch_bounds__(256) void quantize_tokens_kernel(const void* __restrict__ X, long ldx, int n, int C,
                                                              int8_t* __restrict__ Q, long ldq, float* __restrict__ scale) {
  __shared__ float part[4];
  constexpr int KEEP = NV ? NV : 1;
  const int t = threadIdx.x % TPR;
  const long row = ((long)blockIdx.y * gridDim.x + blockIdx.x) * (256 / TPR) + threadIdx.x / TPR;
  if (row >= n) return;  // (whole wavefronts, whole workgroups where they meet)
  const void* x0 = (const char*)X + row * ldx * (DT == DT_F32 ? 4 : 2);
  float x[KEEP][8];
  float top = 0.f;
  bool bad = false;
  auto look = [&](const float* v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bad |= v[i] != v[i];
      top = fmaxf(top, fabsf(v[i]));
    }
  };
  if (NV) {
#pragma unroll
    for (int v = 0; v < KEEP; ++v) load8<DT>(x0, (v * TPR + t) * 8, C, x[v]);
#pragma unroll
    for (int v = 0; v < KEEP; ++v) look(x[v]);
  } else {
    for (int c = 8 * t; c < C; c += 8 * TPR) {
      load8<DT>(x0, c, C, x[0]);
      look(x[0]);
    }
  }
  if (bad) top = INFINITY;
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (TPR == 256) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  }
  const bool fine = top <= 3.402823466e38f;
  if (t == 0) scale[row] = fine ? top / 127.f : NAN;
  const bool zero = !fine || top == 0.f;
  const float up = top < 0x1p-90f ? 0x1p90f : 1.f;  // keeps 127 / top finite; exact
  top *= up;
  const float inv = zero ? 0.f : 127.f / top;
  int8_t* q = Q + row * ldq;
  auto put = [&](float* v, int c) {
    if (c >= C) return;
    if (zero || up != 1.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = zero ? 0.f : v[i] * up;
    }
    const uint2 w = eight_codes(v, top, inv);
    if (c + 8 <= C) {
      __builtin_memcpy(q + c, &w, 8);
    } else {
      int8_t b[8];
      __builtin_memcpy(b, &w, 8);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < C) q[c + i] = b[i];
    }
  };
  if (NV) {
#pragma unroll
    for (int v = 0; v < KEEP; ++v) put(x[v], (v * TPR + t) * 8);
  } else {
    for (int c = 8 * t; c < C; c += 8 * TPR) {
      load8<DT>(x0, c, C, x[0]);
      put(x[0], c);
    }
  }
}

template <int DT>
void quantize_launch(const void* X, long ldx, int n, int C, int8_t* Q, long ldq, float* scale, hipStream_t st) {
#define MQ_QUANT(TPR, NV)                                                                                            \
  hipLaunchKernelGGL((quantize_tokens_kernel<DT, TPR, NV>), mq_wide_grid(((long)n + 256 / TPR - 1) / (256 / TPR)), dim3(256), 0, st, X, \
                     ldx, n, C, Q, ldq, scale)
  if (C <= 512) MQ_QUANT(64, 1);
  else if (C <= 1024) MQ_QUANT(64, 2);
  else if (C <= 2048) MQ_QUANT(256, 1);
  else if (C <= 4096) MQ_QUANT(256, 2);
  else if (C <= 8192) MQ_QUANT(256, 4);
  else if (C <= 16384) MQ_QUANT(256, 8);
  else if (C <= 24576) MQ_QUANT(256, 12);
  else MQ_QUANT(256, 0);
#undef MQ_QUANT
}

// Rows that start at any byte, copied to rows that start at multiples of 16 (for the tiles).
__global__ __launch_bounds__(256) void align_rows_kernel(const int8_t* __restrict__ from, long ld, int n, int K,
                                                         int8_t* __restrict__ to, long ldt) {
  const long row = (long)blockIdx.y * gridDim.x + blockIdx.x;
  if (row >= n) return;
  const int8_t* p = from + row * ld;
  int8_t* q = to + row * ldt;
  for (int c = threadIdx.x * 16; c < K; c += 256 * 16) {
    if (c + 16 <= K) {
      intx4 v;
      __builtin_memcpy(&v, p + c, 16);
      *reinterpret_cast<intx4*>(q + c) = v;
    } else {
      for (int i = c; i < K; ++i) q[i] = p[i];
    }
  }
}

size_t padded(int K) { return ((size_t)K + 15) / 16 * 16; }
// K no multiple of 4: contiguous rows start anywhere; large plain products copy them first (at 4096 x 8192 x 7781 the copies
// take 24 + 13 us and the product 250, on the rows as they are 2460).  Rows off the alignment with K a multiple of 4 are views,
// which are never copied (713 us at 4096 x 4096 x 4096 where aligned rows take 70), nor are the rows of grouped products (3600
// us for 16384 rows over 64 experts of 2048 x 4095 where 2048 x 4096 takes 180).
bool aligns_rows(int M, int N, int K, int swiglu) { return K % 4 != 0 && K >= 16 && small_tiles(M, N, swiglu); }

int int8_dispatch(Int8Args a, int dtype, int swiglu, int8_t* ws, hipStream_t st) {
  if (ws && aligns_rows(a.M, a.N, a.K, swiglu)) {
    const long ld = (long)padded(a.K);
    const int rows_b = swiglu ? 2 * a.N : a.N;
    if (!rows_of_words(a.B, a.ldb)) {
      hipLaunchKernelGGL(align_rows_kernel, mq_wide_grid(rows_b), dim3(256), 0, st, a.B, a.ldb, rows_b, a.K, ws, ld);
      a.B = ws;
      a.ldb = ld;
    }
    if (!rows_of_words(a.A, a.lda)) {
      int8_t* to = ws + (size_t)rows_b * ld;
      hipLaunchKernelGGL(align_rows_kernel, mq_wide_grid(a.M), dim3(256), 0, st, a.A, a.lda, a.M, a.K, to, ld);
      a.A = to;
      a.lda = ld;
    }
  }
  // runs of four results leave in one store where rows of Y allow it
  const int run = dtype == DT_F32 ? 16 : 8;
  a.vec_out = a.N % 4 == 0 && ((uintptr_t)a.Y % run) == 0 && a.ldy % 4 == 0;
  if (a.vec_out && a.N % 8 == 0 && ((uintptr_t)a.Y % 16) == 0 && a.ldy % 8 == 0) a.vec_out = 2;
  if (dtype == DT_F32) return mq_int8_product_f32(a, swiglu, st);
  if (dtype == DT_BF16) return mq_int8_product_bf16(a, swiglu, st);
  return mq_int8_product_f16(a, swiglu, st);
}

bool is_dtype(int d) { return d == DT_F32 || d == DT_BF16 || d == DT_F16; }

void quantize(const void* X, int dtype, long ldx, int n, int C, int8_t* Q, long ldq, float* scale, hipStream_t st) {
  if (dtype == DT_F32) quantize_launch<DT_F32>(X, ldx, n, C, Q, ldq, scale, st);
  else if (dtype == DT_BF16) quantize_launch<DT_BF16>(X, ldx, n, C, Q, ldq, scale, st);
  else quantize_launch<DT_F16>(X, ldx, n, C, Q, ldq, scale, st);
}

constexpr int MAX_K = 131071;  // |sum| <= K 128 128 stays inside 32 bits

}  // namespace

extern "C" int mq_quantize_tokens(const void* X, int dtype, long ldx, int n, int C, int8_t* Q, long ldq, float* scale,
                                  void* stream) {
  if (n < 0 || C <= 0 || ldx < C || ldq < C || n > MQ_MAX_COUNT || C > MQ_MAX_COUNT) return MQ_ERR_ARG;
  if (!is_dtype(dtype)) return MQ_ERR_ARG;
  if (n == 0) return MQ_OK;
  if (!X || !Q || !scale) return MQ_ERR_ARG;
  quantize(X, dtype, ldx, n, C, Q, ldq, scale, (hipStream_t)stream);
  return mq_check_launch();
}

extern "C" size_t mq_matmul_int8_workspace_bytes(int M, int N, int K, int swiglu) {
  if (M <= 0 || N <= 0 || K <= 0 || !aligns_rows(M, N, K, swiglu)) return 0;
  return ((size_t)M + (size_t)N * (swiglu ? 2 : 1)) * padded(K);
}

extern "C" int mq_matmul_int8(const int8_t* A, long lda, const float* a_scale, const int8_t* B, long ldb,
                              const float* b_scale, const void* bias, void* Y, long ldy, int out_dtype, int M, int N, int K,
                              int swiglu, void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || K > MAX_K || lda < K || ldb < K || ldy < N || (swiglu && bias)) return MQ_ERR_ARG;
  if (M > MQ_MAX_COUNT || N > MQ_MAX_COUNT / 2) return MQ_ERR_ARG;
  if (!is_dtype(out_dtype)) return MQ_ERR_ARG;
  if (M == 0) return MQ_OK;
  if (!A || !a_scale || !B || !b_scale || !Y) return MQ_ERR_ARG;
  const size_t need = mq_matmul_int8_workspace_bytes(M, N, K, swiglu);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return MQ_ERR_WORKSPACE;
  const Int8Args a = {A, lda, a_scale, nullptr, M, B, ldb, 0, b_scale, bias, Y, ldy, M, N, K, nullptr, 1, 0};
  return int8_dispatch(a, out_dtype, swiglu, need ? (int8_t*)workspace : nullptr, (hipStream_t)stream);
}

extern "C" int mq_matmul_int8_grouped(const int8_t* A, long lda, const float* a_scale, int src_rows, const long* rows, int S,
                                      const int8_t* B, long ldb, long strideB, const float* b_scale, int E,
                                      const long* offsets, void* Y, long ldy, int out_dtype, int N, int K, int swiglu,
                                      void* stream) {
  if (S < 0 || E <= 0 || E > 1024 || N <= 0 || K <= 0 || K > MAX_K || lda < K || ldb < K || ldy < N) return MQ_ERR_ARG;
  if (src_rows < 0 || strideB < 0 || (!rows && src_rows < S)) return MQ_ERR_ARG;
  if (S > MQ_MAX_COUNT || N > MQ_MAX_COUNT / 2) return MQ_ERR_ARG;
  if (!is_dtype(out_dtype)) return MQ_ERR_ARG;
  if (S == 0) return MQ_OK;
  if (!B || !b_scale || !offsets || !Y || (src_rows > 0 && (!A || !a_scale))) return MQ_ERR_ARG;
  const Int8Args a = {A, lda, a_scale, rows, src_rows, B, ldb, strideB, b_scale, nullptr, Y, ldy, S, N, K, offsets, E, 0};
  return int8_dispatch(a, out_dtype, swiglu, nullptr, (hipStream_t)stream);
}

extern "C" size_t mq_linear_int8_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || for_vector(M, K)) return 0;
  const size_t tokens = (size_t)M * padded(K) + ((size_t)M * sizeof(float) + 15) / 16 * 16;
  return tokens + (aligns_rows(M, N, K, 0) ? (size_t)N * padded(K) : 0);
}

extern "C" int mq_linear_int8(const void* X, int dtype, long ldx, const int8_t* B, long ldb, const float* b_scale,
                              const void* bias, void* Y, long ldy, int M, int N, int K, void* workspace,
                              size_t workspace_bytes, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || K > MAX_K || ldx < K || ldb < K || ldy < N || !is_dtype(dtype)) return MQ_ERR_ARG;
  if (M > MQ_MAX_COUNT || N > MQ_MAX_COUNT / 2) return MQ_ERR_ARG;
  if (M == 0) return MQ_OK;
  if (!X || !B || !b_scale || !Y) return MQ_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  Int8Args a = {(const int8_t*)X, ldx, nullptr, nullptr, M, B, ldb, 0, b_scale, bias, Y, ldy, M, N, K, nullptr, 1, 0};
  if (for_vector(M, K)) {  // one launch: every workgroup quantizes the row or two for itself
    if (dtype == DT_F32) return mq_int8_rows_f32(a, st);
    if (dtype == DT_BF16) return mq_int8_rows_bf16(a, st);
    return mq_int8_rows_f16(a, st);
  }
  const size_t need = mq_linear_int8_workspace_bytes(M, N, K);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) return MQ_ERR_WORKSPACE;
  float* scale = reinterpret_cast<float*>(workspace);
  int8_t* codes = reinterpret_cast<int8_t*>(workspace) + ((size_t)M * sizeof(float) + 15) / 16 * 16;
  int8_t* rest = codes + (size_t)M * padded(K);
  quantize(X, dtype, ldx, M, K, codes, (long)padded(K), scale, st);
  a.A = codes;
  a.lda = (long)padded(K);
  a.sa = scale;
  return int8_dispatch(a, dtype, 0, rest, st);
}
