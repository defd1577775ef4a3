// The kernels of the 8-bit products, one translation unit per type of results (they compile side by side).
#pragma once
#include <math.h>

#include <atomic>

#include "common.hpp"

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
  int vec_out;  // runs of four results may be stored at once; 2: of eight
};

// y = product (SwiGLU: silu(gate) * up) in the type of the name; rows: X, in that type, quantized on the way, one or two rows
int mq_int8_product_f32(const Int8Args& a, int swiglu, hipStream_t st);
int mq_int8_product_bf16(const Int8Args& a, int swiglu, hipStream_t st);
int mq_int8_product_f16(const Int8Args& a, int swiglu, hipStream_t st);
int mq_int8_rows_f32(const Int8Args& a, hipStream_t st);
int mq_int8_rows_bf16(const Int8Args& a, hipStream_t st);
int mq_int8_rows_f16(const Int8Args& a, hipStream_t st);

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
// two results in 16 bits each, rounded to nearest, ties to even (one instruction for bf16 on this chip)
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float floatx2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const floatx2 v = {a, b};
  if (DT == DT_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <int DT>
__device__ __forceinline__ void store_val(void* p, long i, float v) {
  if (DT == DT_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (DT == DT_BF16) reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(v);
  else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}

// ---- quantize ---------------------------------------------------------------------------------------------
// The nearest whole number to 127 x / top, ties to even, as exact arithmetic gives it: z = x * (127 / top) in 32 bits is
// within 2^-14 of the quotient, so rounding z decides except next to a border m + 1/2; there 254 |x| and (2 m + 1) top, both
// exact in 64 bits, are compared.
__device__ __forceinline__ int exact_code(float x, float top, float inv) {
  const float m = floorf(fabsf(x * inv) - 0.25f);  // next to a border m + 1/2: its m
  const double have = 254.0 * (double)fabsf(x), border = (2.0 * (double)m + 1.0) * (double)top;
  const int r = (int)m + (have > border || (have == border && ((int)m & 1)) ? 1 : 0);
  return x < 0.f ? -r : r;
}

// eight codes as bytes.  z + 1.5 * 2^23 rounds z to a whole number, ties to even, and ends in its two's complement.
__device__ __forceinline__ uint2 eight_codes(const float* x, float top, float inv) {
  uint32_t t[8];
  float worst = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float z = x[i] * inv, s = z + 12582912.f;
    t[i] = __float_as_uint(s);
    worst = fmaxf(worst, fabsf(z - (s - 12582912.f)));
  }
  if (worst > 0.5f - 1.220703125e-4f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float z = x[i] * inv;
      if (fabsf(z - (__uint_as_float(t[i]) - 12582912.f)) > 0.5f - 1.220703125e-4f) t[i] = (uint32_t)exact_code(x[i], top, inv);
    }
  }
  uint2 out;
  out.x = __builtin_amdgcn_perm(t[3], t[2], 0x0c0c0400u) << 16 | __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u);
  out.y = __builtin_amdgcn_perm(t[7], t[6], 0x0c0c0400u) << 16 | __builtin_amdgcn_perm(t[5], t[4], 0x0c0c0400u);
  return out;
}

// elements c .. c + 7 of a row of C, zeros beyond its end (any alignment)
template <int DT>
__device__ __forceinline__ void load8(const void* row, int c, int C, float* x) {
  if (c + 8 <= C) {
    if (DT == DT_F32) {
      __builtin_memcpy(x, (const float*)row + c, 32);
    } else {
      uint16_t h[8];
      __builtin_memcpy(h, (const uint16_t*)row + c, 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = load_val<DT>(h, i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c + i < C ? load_val<DT>(row, c + i) : 0.f;
  }
}

// ---- product ------------------------------------------------------------------------------------------------

// four results of one row, columns n .. n + 3, as far as they exist
template <int DT>
__device__ __forceinline__ void store_run(void* Y, long row, int n, int N, int vec, const float* y) {
  if (n >= N) return;
  if (vec) {
    if (DT == DT_F32) {
      *reinterpret_cast<float4*>((float*)Y + row + n) = float4{y[0], y[1], y[2], y[3]};
    } else {
      *reinterpret_cast<uint2*>((uint16_t*)Y + row + n) = make_uint2(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]));
    }
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (n + v < N) store_val<DT>(Y, row + n + v, y[v]);
  }
}

__device__ __forceinline__ float silu_times(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// bytes k .. k + 15 of a row of fewer than 16, zeros beyond its end
__device__ __forceinline__ intx4 short_row(const int8_t* row, int k, int K, bool in) {
  int8_t b[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) b[i] = in && k + i < K ? row[k + i] : (int8_t)0;
  intx4 v;
  __builtin_memcpy(&v, b, 16);
  return v;
}

// Tiles of 256 x 256 (one workgroup a CU, eight wavefronts of 128 x 64) or 128 x 128 (two a CU, four wavefronts of 64 x 64)
// for rows of at least 16 bytes that start at multiples of 4.  A workgroup takes one tile after the other; two stages of 128
// bytes of every row in shared memory, filled by direct 16-byte loads, eight lanes to a row, that is whole 128-byte lines.
//   Layout of a stage: BM token rows, then BN weight rows, 128 bytes each; the 16-byte chunk c of row r lies at position
//   c ^ (r / 2 % 8), so that 16 lanes reading chunk c of 16 rows touch every bank once.
//   Pipeline: a stage is four steps of 32 bytes; while the matrix instructions of one run, the fragments of the next are
//   read.  Once every wavefront has read the last step's (one barrier a stage), the loads of the stage after the next are
//   issued into the slot.  The stages of the next tile follow those of this one without a gap, so its first loads are in
//   flight while this tile's results are written.
//   The end of a row: a chunk that reaches beyond K is loaded from the last 16 bytes of the row instead (never outside it),
//   and the tokens' fragments drop the bytes that belong to earlier chunks, or all of them.
//   A wavefront computes only the 32-row blocks (NB of its four or two) that hold any rows.
// Measured: 476 to 571 us at 8192 x 8192 x 8192 (1.9 to 2.3 POP/s), 1.53 to 1.75 ms at 16384 x 7168 x 16384 (2.2 to 2.5; the
// clock falls to 1.6 GHz there, so power decides); large library products of 8-bit integers reach 2.1 to 2.6.  Grouped, 32
// rows for each of 128 experts of 4096 x 7168: 643 us, 5.8 TB/s of weights.  Tried: four stages of 64 bytes instead of two of 128 (5% slower
// on large products: memory serves 64-byte requests), tiles of 128 x 256 (15% slower: half again as many loads).
constexpr int TK = 128, NST = 2;
constexpr int MIN_STAGES = 3;  // what the hand-over to the next tile needs; beyond K everything counts as zero
constexpr int MAX_GROUPS = 1024;
template <int BM>
struct Tile {
  static constexpr int WAVES = BM / 32, ACROSS = WAVES / 2;  // wavefronts, of these side by side along the columns
  static constexpr int BN = 64 * ACROSS, NB = BM / 64;       // columns; 32-row blocks of a wavefront
  static constexpr int STAGE = (BM + BN) * TK, PER_CU = BM == 256 ? 1 : 2;
};
template <int BM>
struct TileShared {
  typedef Tile<BM> T;
  int8_t stage[NST][T::STAGE];
  long rows[3][BM];           // gathered products: rows of A of the last tile (a slow wavefront may still write it),
                              // of this one and of the next
  float scale[2][T::WAVES][64];  // this tile's (a slow wavefront may still use the last one's): a wavefront loads 32
                                 // columns' and 32 rows'
  float bias[2][T::BN];
  int full[MAX_GROUPS + 64], part[MAX_GROUPS + 64];  // whole tiles and partly filled ones before expert e
};
static_assert(sizeof(TileShared<256>) <= 160 * 1024 && sizeof(TileShared<128>) <= 80 * 1024, "shared memory of a CU");

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

// the same with four bytes a lane
__device__ __forceinline__ void load_lds4(const void* p, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(lds_addr) : "memory", "m0");
}

static __device__ const float no_scale = 0.f;  // of a row that is none

struct Job {
  int e, m0, mend, n0;
};

template <int DT, bool SWIGLU, int BM>
struct TileKernel {
  typedef Tile<BM> T;
  static constexpr int BN = T::BN, STAGE = T::STAGE, ROWS = BM / 2;  // ROWS of a wavefront
  static constexpr int OUTN = SWIGLU ? BN / 2 : BN;
  const Int8Args& a;
  TileShared<BM>& sh;
  const int lane, wave, wm, wn, lr, lk;
  const int nk;         // stages of a tile
  const int chunk;      // this lane's chunk of a stage's 128 bytes in direct loads of even number (of odd number: chunk ^ 4)
  const unsigned lds0;  // LDS address of the stages
  const unsigned rows0, scale0;
  intx16 acc[T::NB][2];
  intx4 fa[2][T::NB], fb[2][2];
  int src[8], next[8];  // rows of this wavefront's direct loads: four of the tokens, four of the weights
  const int8_t *from_a, *from_b, *next_b;
  int slot;

  __device__ __forceinline__ static unsigned lds_of(const void* p) {
    return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
  }
  __device__ __forceinline__ TileKernel(const Int8Args& args, TileShared<BM>& s)
      : a(args), sh(s), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), wm(wave / T::ACROSS),
        wn(wave % T::ACROSS), lr(lane & 31), lk(lane >> 5), nk(max((args.K + TK - 1) / TK, MIN_STAGES)),
        chunk((lane & 7) ^ (lane >> 4)), lds0(lds_of(&s.stage[0][0])), rows0(lds_of(&s.rows[0][0])), scale0(lds_of(&s.scale[0][0][0])),
        slot(0) {}

  // an expert's rows, clamped to [0, M]; a plain product is one expert's
  __device__ __forceinline__ void range(int e, int& lo, int& hi) const {
    lo = 0, hi = a.M;
    if (a.offsets) {
      lo = (int)min(max(a.offsets[e], 0l), (long)a.M);
      hi = (int)min(max(a.offsets[e + 1], (long)lo), (long)a.M);
    }
  }

  // the whole and partly filled row tiles before each expert; returns how many there are of both
  __device__ __forceinline__ int2 table() {
    int2 sum = {0, 0};
    if (wave == 0) {
      for (int e0 = 0; e0 < a.E; e0 += 64) {
        const int e = e0 + lane;
        int lo = 0, hi = 0;
        if (e < a.E) range(e, lo, hi);
        const int mine_f = (hi - lo) / BM, mine_p = (hi - lo) % BM ? 1 : 0;
        int f = mine_f, p = mine_p;
        for (int o = 1; o < 64; o <<= 1) {
          const int uf = __shfl_up(f, o), up = __shfl_up(p, o);
          if (lane >= o) f += uf, p += up;
        }
        sh.full[e] = sum.x + f - mine_f;  // (up to 64 entries beyond E, all = the sums)
        sh.part[e] = sum.y + p - mine_p;
        sum.x += __builtin_amdgcn_readlane(f, 63);
        sum.y += __builtin_amdgcn_readlane(p, 63);
      }
      if (lane == 0) sh.full[a.E] = sum.x, sh.part[a.E] = sum.y;
    }
    __syncthreads();
    sum.x = __builtin_amdgcn_readfirstlane(sh.full[a.E]);
    sum.y = __builtin_amdgcn_readfirstlane(sh.part[a.E]);
    return sum;
  }

  // the last expert with start[e] <= tile: 64 candidates at once, twice
  __device__ __forceinline__ int find(const int* start, int tile) const {
    const int per = (a.E + 63) >> 6;
    const int p0 = min(lane * per, a.E);
    const unsigned long w0 = __ballot(p0 < a.E && start[p0] <= tile);
    const int b0 = (63 - __builtin_clzll(w0)) * per;
    const unsigned long w1 = __ballot(lane < per && b0 + lane < a.E && start[b0 + lane] <= tile);
    return __builtin_amdgcn_readfirstlane(b0 + 63 - __builtin_clzll(w1));
  }

  // job `id` of the whole tiles (in an expert: bands of four row tiles, the rows of a band first, so that what an XCD works
  // on at a time shares few panels) or of the partly filled ones
  __device__ __forceinline__ Job job(bool whole, int id) const {
    const int nt = (a.N + OUTN - 1) / OUTN;
    const int tile = id / nt;
    Job j;
    j.e = find(whole ? sh.full : sh.part, tile);
    int lo, hi;
    range(j.e, lo, hi);
    if (whole) {
      const int in_e = id - sh.full[j.e] * nt, count = (hi - lo) / BM;
      const int band = in_e / (4 * nt), in = in_e - band * 4 * nt, rows = min(4, count - 4 * band);
      j.m0 = lo + (4 * band + in % rows) * BM;
      j.mend = j.m0 + BM;
      j.n0 = in / rows * OUTN;
    } else {
      j.mend = hi;
      j.m0 = hi - (hi - lo) % BM;
      j.n0 = (id - tile * nt) * OUTN;
    }
    j.m0 = __builtin_amdgcn_readfirstlane(j.m0);
    j.mend = __builtin_amdgcn_readfirstlane(j.mend);
    j.n0 = __builtin_amdgcn_readfirstlane(j.n0);
    return j;
  }

  // The rows of this wavefront's direct loads (eight rows each): tokens' rows 32 wave + 8 q + lane / 8, and the weights'.
  // Rows beyond a tile's are loaded as its last one, rows that are none as the first: their results are dropped or scaled by
  // 0.
  __device__ __forceinline__ void sources(const Job& j, int buf, int* rows, const int8_t** b) const {
    *b = a.B + (long)j.e * a.strideB;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = 32 * wave + 8 * q + (lane >> 3);
      // SwiGLU: rows 0..31 of every 64 are gate rows, 32..63 the up rows of the same columns
      int col = SWIGLU ? j.n0 + (r >> 6) * 32 + (r & 31) : j.n0 + r;
      if (col >= a.N) col = j.n0;
      rows[4 + q] = SWIGLU && (r & 32) ? a.N + col : col;
      const long from = a.rows ? sh.rows[buf][r] : min(j.m0 + r, j.mend - 1);
      rows[q] = from >= 0 && from < a.src_rows ? (int)from : 0;
    }
  }

  // all of stage s of this tile (of the next one, counted on, from nk on), load q
  __device__ __forceinline__ void issue(int s, int at_slot, int q) {
    const bool over = s >= nk;
    const int k = TK * (over ? s - nk : s) + 16 * (q & 1 ? chunk ^ 4 : chunk);
    const int off = min(k, a.K - 16);
    const unsigned ld = (unsigned)(q < 4 ? a.lda : a.ldb);
    const int8_t* base = q < 4 ? from_a : (over ? next_b : from_b);
    load_lds16(base + (unsigned long)(unsigned)(over ? next[q] : src[q]) * ld + off,
               lds0 + (unsigned)(at_slot * STAGE + (q >> 2) * BM * TK + wave * 4096 + (q & 3) * 1024));
  }

  // fragments of step `ks` of the stage in `at_slot`
  template <int NB>
  __device__ __forceinline__ void fragment(int at_slot, int ks, int c, intx4* ta, intx4* tb) const {
    const int8_t* stg = sh.stage[at_slot];
    const int at = 16 * ((2 * ks + lk) ^ ((lr >> 1) & 7));
    if (c < NB) ta[c] = *reinterpret_cast<const intx4*>(stg + (wm * ROWS + c * 32 + lr) * TK + at);
    else tb[c - NB] = *reinterpret_cast<const intx4*>(stg + BM * TK + (wn * 64 + (c - NB) * 32 + lr) * TK + at);
  }

  // all stages of a tile; `after` is the next tile
  template <int NB>
  __device__ __forceinline__ void loop(const Job& after, int after_buf) {
    constexpr int NR = NB ? NB + 2 : 0;   // fragments of a step; a wavefront without rows only loads
    constexpr int MF = NB ? 2 * NB : 1;   // matrix instructions of a step
#pragma unroll 1
    for (int kt = 0; kt < nk; ++kt) {
      if (kt == 1) sources(after, after_buf, next, &next_b);  // (the row numbers were loaded before kt = 0: landed by now)
      const int here = slot, there = slot ^ 1;
      const bool ragged = TK * (kt + 1) > a.K;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (ks == 3) {
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_waitcnt(0x0070);  // the next stage landed, this one's last fragments are read
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        if (ragged) {
          const int d = max(0, TK * kt + 32 * ks + 16 * lk - (a.K - 16));
#pragma unroll
          for (int i = 0; i < NB; ++i) fa[ks & 1][i] = keep_from(fa[ks & 1][i], d);
        }
        constexpr int ACTS3 = NR + 8;
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          if (NB)
            acc[m >> 1][m & 1] =
                __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[ks & 1][m & 1], fa[ks & 1][m >> 1], acc[m >> 1][m & 1], 0, 0, 0);
          const int acts = ks == 3 ? ACTS3 : NR;
#pragma unroll
          for (int c = 0; c < ACTS3; ++c)
            if (c < acts && c * MF / acts == m) {
              if (c < NR) fragment<NB>(ks == 3 ? there : here, (ks + 1) & 3, c, fa[(ks + 1) & 1], fb[(ks + 1) & 1]);
              else issue(kt + NST, here, c - NR);
            }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      slot = there;
    }
  }

  // Scales of a tile on their way to shared memory: lane 0..31 a column's, 32..63 a row's (SwiGLU: 16 gate columns', the same
  // 16 up columns', 32 rows').  Loaded while the tile is computed: 32 waits for memory in its epilogue cost 25 us a tile.
  __device__ __forceinline__ void load_scales(const Job& j, int buf, int half) {
    const float* sb = a.sb + (long)j.e * (SWIGLU ? 2 * a.N : a.N);
    const int l = lane & 31, r = 32 * wave + l;
    const float* p;
    if (lane < 32) {
      const int col = min(j.n0 + (SWIGLU ? 16 * wave + (l & 15) : r), a.N - 1);
      p = sb + (SWIGLU && l >= 16 ? a.N + col : col);
    } else {
      const long from = a.rows ? sh.rows[buf][r] : min(j.m0 + r, j.mend - 1);
      p = from >= 0 && from < a.src_rows ? a.sa + from : &no_scale;
    }
    load_lds4(p, scale0 + (unsigned)(half * T::WAVES + wave) * 256u);
    if (!SWIGLU && a.bias && threadIdx.x < BN) sh.bias[half][threadIdx.x] = load_val<DT>(a.bias, min(j.n0 + (int)threadIdx.x, a.N - 1));
  }

  __device__ __forceinline__ void results(const Job& j, int half) const {
    constexpr int RUNS = SWIGLU ? 4 : 8;  // of four columns: 8 g + 4 lk of the wavefront's 32-column blocks
    const int first = j.n0 + (SWIGLU ? wn * 32 : wn * 64) + 4 * lk;
#pragma unroll
    for (int i = 0; i < T::NB; ++i) {
      const int m = j.m0 + wm * ROWS + i * 32 + lr;
      const float sa = sh.scale[half][wm * T::NB + i][32 + lr];
      const bool in = m < j.mend;
      const long row = (long)m * a.ldy;
#pragma unroll
      for (int g = 0; g < RUNS; g += 2) {
        float y[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = (g + h) * 8 + 4 * lk;  // in the wavefront's 32 (SwiGLU) or 64 columns
          const float* s0 = SWIGLU ? &sh.scale[half][wn * 2 + (c >> 4)][c & 15] : &sh.scale[half][wn * 2 + (c >> 5)][c & 31];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if (SWIGLU) {
              y[h][v] = silu_times((float)acc[i][0][4 * (g + h) + v] * sa * s0[v], (float)acc[i][1][4 * (g + h) + v] * sa * s0[16 + v]);
            } else {
              y[h][v] = (float)acc[i][(g + h) >> 2][4 * ((g + h) & 3) + v] * sa * s0[v];
              if (a.bias) y[h][v] += sh.bias[half][wn * 64 + c + v];
            }
          }
        }
        if (DT != DT_F32 && a.vec_out == 2) {
          // lanes l and l + 32 hold columns 8 g .. + 3 and + 4 .. + 7 of one row, and the same of the next run: they swap, and
          // each stores eight columns of one run
          const auto x0 = __builtin_amdgcn_permlane32_swap(pack2<DT>(y[0][0], y[0][1]), pack2<DT>(y[1][0], y[1][1]), false, false);
          const auto x1 = __builtin_amdgcn_permlane32_swap(pack2<DT>(y[0][2], y[0][3]), pack2<DT>(y[1][2], y[1][3]), false, false);
          const int n = first - 4 * lk + 8 * (g + lk);
          if (in && n < a.N) *reinterpret_cast<uint4*>((uint16_t*)a.Y + row + n) = make_uint4(x0[0], x1[0], x0[1], x1[1]);
        } else if (in) {
          store_run<DT>(a.Y, row, first + 8 * g, a.N, a.vec_out, y[0]);
          store_run<DT>(a.Y, row, first + 8 * g + 8, a.N, a.vec_out, y[1]);
        }
      }
    }
  }

  // Jobs go to the XCDs (workgroup index mod 8) in turns, as many consecutive ones as an XCD has workgroups.  Whole tiles
  // are bound by the matrix pipes, partly filled ones by the weights' bytes: every XCD gets an equal share of both and
  // mixes them evenly, half of its workgroups half a turn later.
  struct Order {
    int per, jobs_w, jobs_p, at_w, at_p, turns, share, gone;
    __device__ __forceinline__ Order(int2 tiles, int nt) {
      const int xcd = blockIdx.x & 7, c = blockIdx.x >> 3;
      per = gridDim.x >> 3;
      jobs_w = tiles.x * nt;
      jobs_p = tiles.y * nt;
      const int tw = (jobs_w + per - 1) / per, tp = (jobs_p + per - 1) / per, xp = 7 - xcd;
      share = tw > xcd ? (tw - xcd + 7) >> 3 : 0;                    // turns of this XCD with whole tiles
      turns = share + (tp > xp ? (tp - xp + 7) >> 3 : 0);
      at_w = xcd * per + c;
      at_p = xp * per + c;
      gone = c >= per / 2 ? turns >> 1 : 0;
      left = turns;
    }
    int left;
    __device__ __forceinline__ bool next(bool& whole, int& id) {
      while (left > 0) {
        --left;
        gone += share;
        whole = gone >= turns;
        if (whole) gone -= turns;
        id = whole ? at_w : at_p;
        if (whole) at_w += 8 * per;
        else at_p += 8 * per;
        if (id < (whole ? jobs_w : jobs_p)) return true;
      }
      return false;
    }
  };

  __device__ __forceinline__ void run() {
    Order order(table(), (a.N + OUTN - 1) / OUTN);
    bool whole;
    int id;
    if (!order.next(whole, id)) return;
    Job now = job(whole, id);
    int buf = 0, half = 0;
    if (a.rows) {
      if (threadIdx.x < BM) sh.rows[0][threadIdx.x] = a.rows[min(now.m0 + (int)threadIdx.x, now.mend - 1)];
      __syncthreads();
    }
    from_a = a.src_rows > 0 ? a.A : a.B;  // (no rows at all: anything that can be read)
    sources(now, 0, src, &from_b);
#pragma unroll
    for (int s = 0; s < NST; ++s)
#pragma unroll
      for (int q = 0; q < 8; ++q) issue(s, s, q);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | 8);  // stage 0 landed
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    for (;;) {
      const bool more = order.next(whole, id);
      const Job after = more ? job(whole, id) : now;  // (after the last tile its first stages are loaded again, for nobody)
      const int buf1 = buf == 2 ? 0 : buf + 1;
      if (a.rows)  // rows 32 wave .. 32 wave + 31, two words each
        load_lds4((const int*)(a.rows + min(after.m0 + 32 * wave + (lane >> 1), after.mend - 1)) + (lane & 1),
                  rows0 + (unsigned)(buf1 * BM + 32 * wave) * 8u);
      load_scales(now, buf, half);
#pragma unroll
      for (int c = 0; c < T::NB + 2; ++c) fragment<T::NB>(slot, 0, c, fa[0], fb[0]);
#pragma unroll
      for (int i = 0; i < T::NB; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
      // (wavefronts of one workgroup may run different versions: loads, waits and barriers are the same in all)
      const int rows = now.mend - now.m0 - wm * ROWS;
      if (T::NB == 4 && rows > 96) loop<T::NB>(after, buf1);
      else if (T::NB == 4 && rows > 64) loop<T::NB == 4 ? 3 : 2>(after, buf1);
      else if (rows > 32) loop<2>(after, buf1);
      else if (rows > 0) loop<1>(after, buf1);
      else loop<0>(after, buf1);
      results(now, half);
      half ^= 1;
      if (!more) break;
      now = after;
      buf = buf1;
#pragma unroll
      for (int q = 0; q < 8; ++q) src[q] = next[q];
      from_b = next_b;
    }
    __builtin_amdgcn_s_waitcnt(0x0070);
  }
};

template <int DT, bool SWIGLU, int BM>
__global__ __launch_bounds__(64 * Tile<BM>::WAVES) __attribute__((amdgpu_waves_per_eu(2, 2))) void int8_tile_kernel(Int8Args a) {
  extern __shared__ __attribute__((aligned(1024))) int8_t smem[];
  TileKernel<DT, SWIGLU, BM>(a, *reinterpret_cast<TileShared<BM>*>(smem)).run();
}

template <int DT, bool SWIGLU, int BM>
int tile_launch(const Int8Args& a, hipStream_t st) {
  typedef Tile<BM> T;
  const int outn = SWIGLU ? T::BN / 2 : T::BN, nt = (a.N + outn - 1) / outn;
  // The kernel counts tiles in 32 bits, and offsets come from the device: were every expert's range all rows, the counts
  // would still have to fit (the table of starts ascends only then).
  if ((long)a.E * (a.M / BM + 1) * nt > 0x7fff0000L) return MQ_ERR_TOO_LARGE;  // (65535 spare, for steps of a whole grid)
  static std::atomic<int> cus[64];  // per GPU: its CUs, once the kernel may take its shared memory there
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return MQ_ERR_LAUNCH;
  int n = cus[dev].load();
  if (n == 0) {
    if (hipFuncSetAttribute((const void*)int8_tile_kernel<DT, SWIGLU, BM>, hipFuncAttributeMaxDynamicSharedMemorySize,
                            (int)sizeof(TileShared<BM>)) != hipSuccess ||
        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 8)
      return MQ_ERR_LAUNCH;
    n &= ~7;  // the same number on every XCD
    cus[dev].store(n);
  }
  const long mt = a.offsets ? (long)a.M / BM + min(a.E, a.M) : ((long)a.M + BM - 1) / BM;
  const long jobs = mt * nt;
  const int grid = (int)min((long)n * T::PER_CU, (jobs + 7) / 8 * 8);
  hipLaunchKernelGGL((int8_tile_kernel<DT, SWIGLU, BM>), dim3(grid), dim3(64 * T::WAVES), sizeof(TileShared<BM>), st, a);
  return mq_check_launch();
}

// Few rows or few tiles: a workgroup computes 16 R x 16 C results, its eight wavefronts an eighth of K each; the eight sums meet
// in shared memory.  Grouped: a workgroup belongs to an expert and walks over its rows in steps of 16 R.
//   D > 0, for rows of at least 16 bytes that start at multiples of 4: a wavefront keeps D - 1 steps of 64 bytes of its rows on
//   their way into shared memory of its own by direct loads, four lanes to a row.  (Fragments want lane l to hold row l % 16:
//   loaded like that, an instruction touches every row four times and the address unit takes 64 cycles for it.)  Chunk c of
//   row r lies at position c ^ (r / 4 % 4): 16 lanes reading chunk c of 16 rows touch every bank once.
//   D = 0: fragments straight from memory, UN steps at a time; any alignment, any K.
// Measured, on weights that no cache holds: 12 us at 333 x 576 x 7168 (D = 0: 16), 6.8 at 8 x 2048 x 7168 (D = 0: 11); bound by
// the way of the operands to the wavefronts (D = 2 has a single step in flight, which it waits for in full), or by the
// weights' bytes: 41 us at 16 x 18432 x 7168 (3.2 TB/s).
constexpr int vmcnt_is(int n) { return 0x0070 | (n & 15) | (n >> 4) << 14; }  // ... and lgkmcnt(0)

template <int DT, bool SWIGLU, int R, int C, int UN, int D>
__global__ __launch_bounds__(512) void int8_thin_kernel(Int8Args a, int gx, int by_row) {
  extern __shared__ __attribute__((aligned(1024))) int8_t smem[];
  typedef intx4 Sums[R * C][64];
  Sums* part = reinterpret_cast<Sums*>(smem);  // of every wavefront (where its steps were)
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  constexpr int OUTN = SWIGLU ? 8 * C : 16 * C;
  const int by = blockIdx.x / gx, n0 = (blockIdx.x - by * gx) * OUTN;
  int e = 0, mbeg = by * 16 * R, mend = min(mbeg + 16 * R, a.M);
  if (a.offsets) {
    e = by;
    if (by_row) {  // the expert of row `by`: as many as end before it or with it come first
      e = 0;
#pragma unroll 4
      for (int e0 = 0; e0 < a.E; e0 += 64) e += __popcll(__ballot(e0 + lane < a.E && a.offsets[min(e0 + lane, a.E - 1) + 1] <= by));
      if (e >= a.E) return;
    }
    mbeg = (int)min(max(a.offsets[e], 0l), (long)a.M);
    mend = (int)min(max(a.offsets[e + 1], (long)mbeg), (long)a.M);
    if (by_row && mbeg != by) return;  // its first row's workgroup does them all
  }
  const int8_t* B = a.B + (long)e * a.strideB;
  const float* sb = a.sb + (long)e * (SWIGLU ? 2 * a.N : a.N);
  const int steps = (a.K + 63) >> 6, per = (steps + 7) >> 3;
  const int k0 = 64 * per * wave, k1 = min(a.K, k0 + 64 * per);
  const int lrow = D ? lane >> 2 : l16;  // the row this lane loads of every 16
  const int8_t* brow[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    // SwiGLU: even blocks of 16 are gate rows, odd ones the up rows of the same columns
    int col = SWIGLU ? n0 + 16 * (c >> 1) + lrow : n0 + 16 * c + lrow;
    if (col >= a.N) col = n0;
    brow[c] = B + (long)(SWIGLU && (c & 1) ? a.N + col : col) * a.ldb;
  }
  for (int m0 = mbeg; m0 < mend; m0 += 16 * R) {
    const int8_t* arow[R];
    bool ain[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int m = m0 + 16 * r + lrow;
      long from = m;
      ain[r] = m < mend;
      if (ain[r] && a.rows) from = a.rows[m];
      ain[r] = ain[r] && from >= 0 && from < a.src_rows;
      // (a row that is none is loaded from the weights: its results are dropped, or scaled by 0)
      arow[r] = ain[r] ? a.A + from * a.lda : brow[0];
    }
    intx4 acc[R][C];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) acc[r][c] = intx4{0, 0, 0, 0};
    if (m0 != mbeg) __syncthreads();  // the sums of the rows before have been read
    if (D > 0) {
      const int mine = k1 > k0 ? (k1 - k0 + 63) >> 6 : 0;
      const int chunk = (lane & 3) ^ lq;
      int8_t* slots = smem + wave * (D ? D : 1) * (R + C) * 1024;
      const unsigned lds0 = __builtin_amdgcn_readfirstlane(
          (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t*)slots);
      // (steps past the last load it again into slots nobody reads: the waits keep their counts)
      const auto issue = [&](int s, int slot) {
        const int off = min(k0 + 64 * min(s, mine - 1) + 16 * chunk, a.K - 16);
#pragma unroll
        for (int r = 0; r < R; ++r) load_lds16(arow[r] + off, lds0 + (unsigned)(slot * (R + C) + r) * 1024u);
#pragma unroll
        for (int c = 0; c < C; ++c) load_lds16(brow[c] + off, lds0 + (unsigned)(slot * (R + C) + R + c) * 1024u);
      };
      if (mine > 0) {
#pragma unroll
        for (int s = 0; s < D - 1; ++s) issue(s, s);
        int slot = 0;
        const int at = l16 * 64 + 16 * (lq ^ (l16 >> 2));
#pragma unroll 1
        for (int t = 0; t < mine; ++t) {
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_waitcnt(vmcnt_is((D > 1 ? D - 2 : 0) * (R + C)));  // step t landed; the last step's fragments are read
          asm volatile("" ::: "memory");
          const int8_t* here = slots + slot * (R + C) * 1024 + at;
          intx4 fa[R], fb[C];
#pragma unroll
          for (int r = 0; r < R; ++r) fa[r] = *reinterpret_cast<const intx4*>(here + r * 1024);
#pragma unroll
          for (int c = 0; c < C; ++c) fb[c] = *reinterpret_cast<const intx4*>(here + (R + c) * 1024);
          issue(t + D - 1, slot == 0 ? D - 1 : slot - 1);
          slot = slot == D - 1 ? 0 : slot + 1;
          const int kc = k0 + 64 * t;
          if (kc + 64 > a.K) {
#pragma unroll
            for (int r = 0; r < R; ++r) fa[r] = keep_from(fa[r], max(0, kc + 16 * lq - (a.K - 16)));
          }
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[r][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[c], fa[r], acc[r][c], 0, 0, 0);
        }
        __builtin_amdgcn_s_waitcnt(0x0070);
      }
      __syncthreads();  // the sums go where the steps were
    } else {
      if (a.K < 16 && wave == 0) {
        intx4 ta[R], tb[C];
#pragma unroll
        for (int c = 0; c < C; ++c) tb[c] = short_row(brow[c], 16 * lq, a.K, true);
#pragma unroll
        for (int r = 0; r < R; ++r) ta[r] = short_row(arow[r], 16 * lq, a.K, ain[r]);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int c = 0; c < C; ++c) acc[r][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(tb[c], ta[r], acc[r][c], 0, 0, 0);
      }
      for (int k = a.K < 16 ? k1 : k0; k < k1; k += 64 * UN) {
        intx4 fa[UN][R], fb[UN][C];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          // chunks beyond the end of a row: the weights' last 16 bytes once more, against zeros
          const int kc = k + 64 * u + 16 * lq, at = min(kc, a.K - 16);
#pragma unroll
          for (int c = 0; c < C; ++c) __builtin_memcpy(&fb[u][c], brow[c] + at, 16);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            fa[u][r] = intx4{0, 0, 0, 0};
            if (ain[r] && kc < k1) __builtin_memcpy(&fa[u][r], arow[r] + at, 16);
          }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const int kc = k + 64 * u + 16 * lq;
          if ((a.K & 15) && a.K > 16) {
#pragma unroll
            for (int r = 0; r < R; ++r) fa[u][r] = keep_from(fa[u][r], kc - (a.K - 16));
          }
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c)
              acc[r][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[u][c], fa[u][r], acc[r][c], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) part[wave][r * C + c][lane] = acc[r][c];
    __syncthreads();
    constexpr int CB = SWIGLU ? C / 2 : C, ITEMS = R * CB * 64;
    for (int it = tid; it < ITEMS; it += 512) {
      const int ln = it & 63, r = (it >> 6) / CB, c = (it >> 6) % CB;
      const int m = m0 + 16 * r + (ln & 15), n = n0 + 16 * c + 4 * (ln >> 4);
      if (m >= mend || n >= a.N) continue;
      long from = m;
      if (a.rows) from = a.rows[m];
      const float sa = from >= 0 && from < a.src_rows ? a.sa[from] : 0.f;
      intx4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        s0 += part[w][r * C + (SWIGLU ? 2 * c : c)][ln];
        if (SWIGLU) s1 += part[w][r * C + 2 * c + 1][ln];
      }
      float y[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int col = min(n + v, a.N - 1);
        if (SWIGLU) {
          y[v] = silu_times((float)s0[v] * sa * sb[col], (float)s1[v] * sa * sb[a.N + col]);
        } else {
          y[v] = (float)s0[v] * sa * sb[col];
          if (a.bias) y[v] += load_val<DT>(a.bias, col);
        }
      }
      store_run<DT>(a.Y, (long)m * a.ldy, n, a.N, a.vec_out, y);
    }
  }
}

template <int DT, bool SWIGLU, int R, int C, int UN, int D>
int thin_launch(const Int8Args& a, hipStream_t st) {
  constexpr int SMEM = 8 * 1024 * (D * (R + C) > R * C ? D * (R + C) : R * C);
  static_assert(SMEM <= 160 * 1024, "shared memory of a CU");
  if (SMEM > 48 * 1024) {
    static std::atomic<uint64_t> set{0};  // GPUs on which the kernel may take its shared memory
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return MQ_ERR_LAUNCH;
    if (!(set.load() >> dev & 1)) {
      if (hipFuncSetAttribute((const void*)int8_thin_kernel<DT, SWIGLU, R, C, UN, D>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, SMEM) != hipSuccess)
        return MQ_ERR_LAUNCH;
      set.fetch_or(1ull << dev);
    }
  }
  const int outn = SWIGLU ? 8 * C : 16 * C, gx = (a.N + outn - 1) / outn;
  // fewer rows than experts: a workgroup a row (the others of its expert's leave at once) rather than one an expert, most
  // of which would have no rows: 16384 that leave at once take 25 us
  const int by_row = a.offsets && a.M < a.E;
  const long grid = (long)gx * (a.offsets ? min(a.M, a.E) : (a.M + 16 * R - 1) / (16 * R));
  if (grid * 512 > 0xffffffffL) return MQ_ERR_TOO_LARGE;
  hipLaunchKernelGGL((int8_thin_kernel<DT, SWIGLU, R, C, UN, D>), dim3((unsigned)grid), dim3(512), SMEM, st, a, gx, by_row);
  return mq_check_launch();
}

// One or two rows: the weights' bytes are all that counts.  A wavefront streams pairs of weight rows (SwiGLU: a gate row and
// its up row), 1 KB of a row an instruction, up to sixteen of them in flight; the tokens' codes lie in shared memory and
// meet the weights in four-byte dot products.  Tokens come as codes (XDT < 0) or are quantized here by every workgroup for
// itself (XDT = their type), under the first weights' way from memory.  Any alignment; K of at least 16.
//   A row's last chunk, where K is no multiple of 16, is its last 16 bytes, and the tokens' bytes that belong to the chunk
//   before are zero there.
// Measured: one token, quantized on the way, 8.5 us at 2048 x 7168 (6.7 on weights that a cache holds), 28.5 at 18432 x 7168
// (4.6 TB/s).
constexpr int VT = 2, VEC_THREADS = 256, VEC_CHUNKS = 8;

template <int DT, bool SWIGLU, int XDT>
struct VectorKernel {
  const Int8Args& a;
  int8_t* codes;  // VT rows of 16 ceil(K / 16) bytes
  float* scales;  // VT
  float* red;     // a value a wavefront
  const int lane, wave, chunks, pitch;

  __device__ __forceinline__ VectorKernel(const Int8Args& args, int8_t* smem)
      : a(args), codes(smem), lane(threadIdx.x & 63), wave(threadIdx.x >> 6), chunks((args.K + 15) >> 4), pitch(chunks * 16) {}

  __device__ __forceinline__ const int8_t* weight_row(int n, int second) const {
    const int r = SWIGLU ? (second ? a.N + n : n) : min(n + second, a.N - 1);
    return a.B + (long)r * a.ldb;
  }
  __device__ __forceinline__ void load(const int8_t* w0, const int8_t* w1, int c0, intx4 (*v)[2]) const {
#pragma unroll
    for (int u = 0; u < VEC_CHUNKS; ++u) {
      const int at = min(16 * min(c0 + 64 * u + lane, chunks - 1), a.K - 16);
      if (64 * (c0 / 64 + u) < chunks) {
        __builtin_memcpy(&v[u][0], w0 + at, 16);
        __builtin_memcpy(&v[u][1], w1 + at, 16);
      }
    }
  }

  // the tokens' codes and scales into shared memory
  __device__ __forceinline__ void stage() {
    for (int r = 0; r < a.M; ++r) {
      int8_t* q = codes + r * pitch;
      if (XDT < 0) {
        const int8_t* p = a.A + (long)r * a.lda;
        for (int c = threadIdx.x; c < chunks; c += VEC_THREADS) {
          intx4 v;
          __builtin_memcpy(&v, p + min(16 * c, a.K - 16), 16);
          *reinterpret_cast<intx4*>(q + 16 * c) = keep_from(v, 16 * c - (a.K - 16));
        }
        if (threadIdx.x == 0) scales[r] = a.sa[r];
      } else {
        constexpr int D = XDT < 0 ? 0 : XDT;
        const void* x0 = (const char*)a.A + (long)r * a.lda * (D == DT_F32 ? 4 : 2);
        constexpr int KEEP = 4;  // vectors of eight kept in registers; longer rows are read twice
        float x[KEEP][8];
        float top = 0.f;
        auto look = [&](const float* v) {
#pragma unroll
          for (int i = 0; i < 8; ++i) top = v[i] == v[i] ? fmaxf(top, fabsf(v[i])) : INFINITY;
        };
#pragma unroll
        for (int v = 0; v < KEEP; ++v) load8<D>(x0, (v * VEC_THREADS + threadIdx.x) * 8, a.K, x[v]);
#pragma unroll
        for (int v = 0; v < KEEP; ++v) look(x[v]);
        for (int c = (KEEP * VEC_THREADS + threadIdx.x) * 8; c < a.K; c += 8 * VEC_THREADS) {
          float y[8];
          load8<D>(x0, c, a.K, y);
          look(y);
        }
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if (r) __syncthreads();
        if (lane == 0) red[wave] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const bool fine = top <= 3.402823466e38f, zero = !fine || top == 0.f;
        if (threadIdx.x == 0) scales[r] = fine ? top / 127.f : NAN;
        const float up = top < 0x1p-90f ? 0x1p90f : 1.f;
        top *= up;
        const float inv = zero ? 0.f : 127.f / top;
        auto put = [&](float* v, int c) {
          if (c >= a.K) return;
          if (zero || up != 1.f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = zero ? 0.f : v[i] * up;
          }
          const uint2 w = eight_codes(v, top, inv);
          const int whole = a.K & ~15;
          if (c + 8 <= whole) {
            *reinterpret_cast<uint2*>(q + c) = w;
          } else {  // the last chunk starts at K - 16
            int8_t b[8];
            __builtin_memcpy(b, &w, 8);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (c + i < a.K) q[whole + c + i - (a.K - 16)] = b[i];
          }
        };
        if ((a.K & 15) && threadIdx.x < 16 - (a.K & 15)) q[(a.K & ~15) + threadIdx.x] = 0;
#pragma unroll
        for (int v = 0; v < KEEP; ++v) put(x[v], (v * VEC_THREADS + threadIdx.x) * 8);
        for (int c = (KEEP * VEC_THREADS + threadIdx.x) * 8; c < a.K; c += 8 * VEC_THREADS) {
          float y[8];
          load8<D>(x0, c, a.K, y);
          put(y, c);
        }
      }
    }
  }

  __device__ __forceinline__ void finish(int m, int n, int second, int sum0, int sum1) const {
    const float sa = scales[m];
    if (SWIGLU) {
      store_val<DT>(a.Y, (long)m * a.ldy + n, silu_times((float)sum0 * sa * a.sb[n], (float)sum1 * sa * a.sb[a.N + n]));
    } else if (n + second < a.N) {
      float y = (float)(second ? sum1 : sum0) * sa * a.sb[n + second];
      if (a.bias) y += load_val<DT>(a.bias, n + second);
      store_val<DT>(a.Y, (long)m * a.ldy + n + second, y);
    }
  }

  template <int MT>
  __device__ __forceinline__ void dots(const intx4 (*v)[2], int c0, int (*acc)[2]) const {
#pragma unroll
    for (int u = 0; u < VEC_CHUNKS; ++u) {
      const int c = c0 + 64 * u + lane;
      if (c < chunks) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const intx4 q = *reinterpret_cast<const intx4*>(codes + m * pitch + 16 * c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[m][0] = __builtin_amdgcn_sdot4(v[u][0][i], q[i], acc[m][0], false);
            acc[m][1] = __builtin_amdgcn_sdot4(v[u][1][i], q[i], acc[m][1], false);
          }
        }
      }
    }
  }

  // one pair of weight rows against MT tokens; v holds the first chunks already
  template <int MT>
  __device__ __forceinline__ void pair(int n, intx4 (*v)[2]) const {
    int acc[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = 0;
    const int8_t *w0 = weight_row(n, 0), *w1 = weight_row(n, 1);
    dots<MT>(v, 0, acc);
    for (int c0 = 64 * VEC_CHUNKS; c0 < chunks; c0 += 64 * VEC_CHUNKS) {
      load(w0, w1, c0, v);
      dots<MT>(v, c0, acc);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      int s0 = acc[m][0], s1 = acc[m][1];
      for (int o = 32; o; o >>= 1) {
        s0 += __shfl_xor(s0, o);
        s1 += __shfl_xor(s1, o);
      }
      if (lane < (SWIGLU ? 1 : 2)) finish(m, n, lane, s0, s1);
    }
  }

  __device__ __forceinline__ void run() {
    scales = reinterpret_cast<float*>(codes + VT * pitch);
    red = scales + VT;
    constexpr int WIDTH = SWIGLU ? 1 : 2;
    const int pairs = (a.N + WIDTH - 1) / WIDTH;
    const int first = blockIdx.x * (VEC_THREADS / 64) + wave, step = gridDim.x * (VEC_THREADS / 64);
    intx4 v[VEC_CHUNKS][2];
    if (first < pairs) load(weight_row(first * WIDTH, 0), weight_row(first * WIDTH, 1), 0, v);
    stage();
    __syncthreads();
    for (int p = first; p < pairs; p += step) {
      if (p != first) load(weight_row(p * WIDTH, 0), weight_row(p * WIDTH, 1), 0, v);
      if (a.M > 1) pair<2>(p * WIDTH, v);
      else pair<1>(p * WIDTH, v);
    }
  }
};

template <int DT, bool SWIGLU, int XDT>
__global__ __launch_bounds__(VEC_THREADS) void int8_vector_kernel(Int8Args a) {
  extern __shared__ __attribute__((aligned(1024))) int8_t smem[];
  VectorKernel<DT, SWIGLU, XDT>(a, smem).run();
}

size_t vector_smem(int K) { return (size_t)VT * ((K + 15) / 16 * 16) + (VT + 8) * sizeof(float); }

template <int DT, bool SWIGLU, int XDT>
int vector_launch(const Int8Args& a, hipStream_t st) {
  static std::atomic<uint64_t> set{0};  // GPUs on which the kernel may take its shared memory
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return MQ_ERR_LAUNCH;
  if (!(set.load() >> dev & 1)) {
    if (hipFuncSetAttribute((const void*)int8_vector_kernel<DT, SWIGLU, XDT>, hipFuncAttributeMaxDynamicSharedMemorySize,
                            160 * 1024) != hipSuccess)
      return MQ_ERR_LAUNCH;
    set.fetch_or(1ull << dev);
  }
  const int pairs = SWIGLU ? a.N : (a.N + 1) / 2, waves = VEC_THREADS / 64;
  // 512 workgroups, two a CU, walk over what they do not reach at once: 28.5 us at 18432 x 7168 against 35 with 256 of them and
  // 39 with 2048 (2048 x 7168 has 256)
  const int gx = min((pairs + waves - 1) / waves, 512);
  hipLaunchKernelGGL((int8_vector_kernel<DT, SWIGLU, XDT>), dim3(gx), dim3(VEC_THREADS),
                     vector_smem(a.K), st, a);
  return mq_check_launch();
}

bool rows_of_words(const int8_t* p, long ld) { return ((uintptr_t)p & 3) == 0 && ld % 4 == 0 && ld < 0x7fffffff; }

// the vector kernel takes one or two rows whose codes fit its shared memory
bool for_vector(int M, int K) { return M <= VT && K >= 16 && vector_smem(K) <= 160 * 1024; }
// a plain product's tiles of edge x edge
bool enough_tiles(int M, int N, int swiglu, int edge, int count) {
  return ((long)M + edge - 1) / edge * (((long)N * (swiglu ? 2 : 1) + edge - 1) / edge) >= count;
}
bool small_tiles(int M, int N, int swiglu) { return M > 32 && enough_tiles(M, N, swiglu, 128, 136); }
// a grouped product's tiles of 256 x 256, at most
template <bool SWIGLU>
bool enough_jobs(const Int8Args& a) {
  return ((long)a.M / 256 + min(a.E, a.M)) * ((a.N * (SWIGLU ? 2l : 1l) + 255) / 256) >= 1024;
}

template <int DT, bool SWIGLU>
int int8_launch(const Int8Args& a, hipStream_t st) {
  const bool tiles = a.K >= 16 && rows_of_words(a.A, a.lda) && rows_of_words(a.B, a.ldb) && a.strideB % 4 == 0;
  if (a.offsets) {
    // A decode step: gate/up + down of 64 experts of 7168 x 2048, skewed loads, us without shared memory against tiles: 32
    // rows 100 + 65 against 133 + 51, 64 rows 126 + 87 against 143 + 73, 128 rows 171 + 114 against 156 + 99, 256 rows 229 +
    // 145 against 221 + 122, 512 rows 322 + 191 against 237 + 148 (even loads alike).  So the border lies nearer to one row an
    // expert than to the four below, for the down product lower still.  (Staging the rows costs at 32 rows: 130 + 78 where
    // 110 + 71 was measured beside it.)
    if (!tiles || a.M <= 4l * a.E) return thin_launch<DT, SWIGLU, 2, 2, 2, 0>(a, st);
    // Few rows an expert: the weights' bytes decide, and two small workgroups a CU keep more of them in flight (5.8 against
    // 4.9 TB/s at 32 rows for each of 128 experts of 7168 x 2048).  Many rows: large tiles read both operands less often
    // (1850 against 1510 TOP/s at 256 rows), if there are enough of them to go round several times.
    if (a.M <= 128l * a.E || !enough_jobs<SWIGLU>(a)) return tile_launch<DT, SWIGLU, 128>(a, st);
    return tile_launch<DT, SWIGLU, 256>(a, st);
  }
  if (for_vector(a.M, a.K)) return vector_launch<DT, SWIGLU, -1>(a, st);
  // 70 us at 4096 x 4096 x 4096 (256 large tiles) against 97 with small ones; 66 against 51 at 2048 x 4096 x 4096 (128)
  if (tiles && enough_tiles(a.M, a.N, SWIGLU, 256, 192)) return tile_launch<DT, SWIGLU, 256>(a, st);
  // 64 us at 128 x 18432 x 7168 (144 small tiles) against 80 without tiles; 28 against 29 at 512 x 4096 x 4096 (128)
  if (tiles && small_tiles(a.M, a.N, SWIGLU)) return tile_launch<DT, SWIGLU, 128>(a, st);
  // the largest block of results that still gives 192 workgroups (and is half full, at least)
  const auto groups = [&](int R, int C) {
    const int outn = SWIGLU ? 8 * C : 16 * C;
    return a.M > 8 * R || R == 1 ? (long)((a.M + 16 * R - 1) / (16 * R)) * ((a.N + outn - 1) / outn) : 0l;
  };
  if (!tiles) {  // 16 us at 333 x 576 x 7168 against 12 for aligned rows
    if (groups(4, 4) >= 192) return thin_launch<DT, SWIGLU, 4, 4, 1, 0>(a, st);
    if (groups(2, 2) >= 192) return thin_launch<DT, SWIGLU, 2, 2, 2, 0>(a, st);
    return thin_launch<DT, SWIGLU, 1, 2, 2, 0>(a, st);
  }
  if (groups(4, 4) >= 192) return thin_launch<DT, SWIGLU, 4, 4, 1, 2>(a, st);  // 11 us at 512 x 2048 x 2048, (2, 4) 14, (2, 2) 15
  if (groups(2, 4) >= 192) return thin_launch<DT, SWIGLU, 2, 4, 1, 2>(a, st);  // 22 us at 64 x 7168 x 7168, (4, 4) 32, (2, 2) 26
  if (groups(2, 2) >= 192) return thin_launch<DT, SWIGLU, 2, 2, 1, 2>(a, st);  // 12 us at 333 x 576 x 7168, (2, 4) 16, (1, 1) 16
  if (groups(1, 2) >= 192 || SWIGLU) return thin_launch<DT, SWIGLU, 1, 2, 1, 3>(a, st);  // 5.4 us at 64 x 2048 x 2048, (1, 1) 6.0
  return thin_launch<DT, SWIGLU, 1, SWIGLU ? 2 : 1, 1, 4>(a, st);  // 6.8 us at 8 x 2048 x 7168, (1, 2) 8.7
}

}  // namespace
