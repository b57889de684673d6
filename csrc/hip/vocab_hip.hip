// Kernels over the whole vocabulary for MI355X (gfx950, CDNA4):
//
//   * softmax cross entropy of N rows h against a table w of V rows, without
//     the scores [N, V] in memory, and its gradient
//       s_nv = <h_n, w_v>          lse_n  = log sum_v exp s_nv
//       loss_n = lse_n - s_n,y(n)  c_nv   = g_n (exp(s_nv - lse_n) - [v=y(n)])
//       dh = c w                   dw     = c^T h
//   * rows in 8-bit floats (e4m3) with a power-of-two scale for each block of
//     128 columns, and the product of such rows.
//
// The scores are a matrix product whose one side is the table.  Its rows are
// the M side of the 16 x 16 matrix instructions: a lane then holds four
// neighbouring table rows of ONE sample, so that the softmax's running maximum
// and sum stay in the lane until the workgroup's last tile, coefficients are
// written as the products with them read them, and scores are stored four to an
// instruction.  Three kernels make them:
//   resident_kernel  bf16 and 8-bit rows of up to 320 columns: the samples stay
//                    in registers, and LDS is read for the table alone
//   stream_kernel    up to 16 samples: the table goes from memory to registers
//   tile_kernel      everything else: both sides by way of LDS
// The gradient takes the vocabulary a piece at a time, its coefficients c in
// memory between tile_kernel or resident_kernel and two products (grad_kernel).
//
// What bounds them, measured on one card: memory gives 4.8 TB/s in a copy; a
// loop of bf16 instructions alone runs at 2.30 PFLOP/s, one of float32
// instructions at 155 TFLOP/s; library products reach 1.35 PFLOP/s and 153
// TFLOP/s at 8192^3; a fill reaches 6.8 TB/s, and reads alone 5.6.  Figures
// beside the kernels are for the sizes they name: of whole calls, or, where it
// says so, averages of traced launches, which take up to a fifth longer.

#include <hip/hip_runtime.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <utility>

namespace py = pybind11;

#define HIP_CHECK(expr)                                                     \
  do {                                                                      \
    hipError_t _e = (expr);                                                 \
    if (_e != hipSuccess)                                                   \
      throw std::runtime_error(std::string("HIP error: ") +                 \
                               hipGetErrorString(_e) + " at " __FILE__ ":" + \
                               std::to_string(__LINE__));                   \
  } while (0)

// For lambdas with many calls: one that is not inlined keeps what it captures
// in memory.
#define INLINE __attribute__((always_inline))

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// exp(s - m) is taken as 2^(s log2e - m log2e) with one rounding of m log2e,
// which costs at most |m| 2^-25 in the exponent.  Past this |m| the exponent
// is (s - m) log2e instead: one instruction more, but it cannot overflow.
constexpr float kFar = 1e6f;

// kSplit is float32 in three parts of bf16, x = hi + mid + lo exactly (down to
// bf16's smallest subnormal, 2^-133, for numbers under 2^-109): each
// part is the nearest bf16 to what the ones before leave, so that mid and lo
// are at most 2^-9 and 2^-18 of x.  Of the nine products of two such numbers
// the six from 2^-18 up are taken; the others are 2^-26 of the product at
// most, a quarter of float32's rounding.  Six bf16 instructions take 3/8 of
// the time of the float32 ones for the same columns.
enum Type { kF32 = 0, kBF16 = 1, kFP8 = 2, kSplit = 3 };

// Bytes of one element (of kSplit, of one of its parts).  8-bit rows are
// brought to bf16 for the matrix instruction, which holds e4m3 times a power of
// two exactly.
template <int T> struct Elem;
template <> struct Elem<kF32> { static constexpr int size = 4, parts = 1; };
template <> struct Elem<kBF16> { static constexpr int size = 2, parts = 1; };
template <> struct Elem<kFP8> { static constexpr int size = 1, parts = 1; };
template <> struct Elem<kSplit> { static constexpr int size = 2, parts = 3; };

// Rows of a matrix in global memory, all of which start at multiples of
// `align` bytes: 16, 4 or less.
struct Rows {
  const char* p;
  int64_t ld;      // bytes from row to row
  int64_t rows;
  int kb;          // bytes of a row
  int align;
  const uint8_t* scales;   // 8-bit rows: exponents + 127, one per 128 columns
  int64_t lds;             // scales from row to row
};

__device__ __forceinline__ float bf16_to_f32(uint16_t h) {
  return __uint_as_float((uint32_t)h << 16);
}
__device__ __forceinline__ float exp_of(float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}
// Joins two (maximum, sum of exp(s - maximum)).
__device__ __forceinline__ void join(float& top, float& sum, float t, float s) {
  const float next = fmaxf(top, t);
  const float ref = next == -INFINITY ? 0.f : next;
  sum = sum * exp_of(top - ref) + s * exp_of(t - ref);
  top = next;
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  bf16x2 v;
  v[0] = (__bf16)a;
  v[1] = (__bf16)b;
  return __builtin_bit_cast(uint32_t, v);
}

// The three parts of x.  What is not finite is in the last, which meets the
// other side's first part alone: infinity times that has the product's sign,
// while the other parts may be 0 or of the other sign.  Its first part is 1 of
// its sign, for what is infinite on the other side.  Where bf16 would round x
// past the largest number, the parts are cut off instead of rounded: all of x's
// sign, so that no sum of them passes x.
__device__ __forceinline__ void split(float x, float& hi, float& mid, float& lo) {
  const uint32_t u = __float_as_uint(x);
  const bool finite = (u & 0x7f800000u) != 0x7f800000u;
  hi = (float)(__bf16)x;
  const bool cut = finite && __builtin_isinf(hi);
  if (cut) hi = __uint_as_float(u & 0xffff0000u);
  if (!finite) hi = __builtin_copysignf(1.f, x);
  const float rest = finite ? x - hi : 0.f;
  mid = cut ? __uint_as_float(__float_as_uint(rest) & 0xffff0000u) : (float)(__bf16)rest;
  lo = finite ? rest - mid : x;
}
__device__ __forceinline__ void split4(const f32x4& x, u32x2 (&to)[3]) {
  f32x4 t[3];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float hi, mid, lo;
    split(x[e], hi, mid, lo);
    t[0][e] = hi, t[1][e] = mid, t[2][e] = lo;
  }
#pragma unroll
  for (int p = 0; p < 3; ++p)
    to[p] = u32x2{pack_bf16(t[p][0], t[p][1]), pack_bf16(t[p][2], t[p][3])};
}

// 16 bytes of a row from byte `o` on; zeros outside of the matrix.
template <int ES>
__device__ __forceinline__ u32x4 load16(const Rows& m, int64_t row, int o) {
  u32x4 r = {0, 0, 0, 0};
  if (row >= m.rows || o >= m.kb) return r;
  const char* q = m.p + row * m.ld + o;
  if (m.align == 16) {
    // whole, as 16 bytes at a multiple of 16 are of one page; then cut
    r = *reinterpret_cast<const u32x4*>(q);
    if (o + 16 > m.kb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int have = m.kb - o - 4 * i;
        r[i] = have >= 4 ? r[i] : have <= 0 ? 0u : r[i] & ((1u << (8 * have)) - 1);
      }
    }
    return r;
  }
  if (m.align == 4 && o + 16 <= m.kb) return *reinterpret_cast<const u32x4a4*>(q);
  const int have = (m.kb - o) / ES;
  if (ES == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) r[i] = reinterpret_cast<const uint32_t*>(q)[i];
  } else if (ES == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have)
        r[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[i] << (16 * (i & 1));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < have) r[i >> 2] |= (uint32_t)(uint8_t)q[i] << (8 * (i & 3));
  }
  return r;
}

__device__ __forceinline__ float scale_of(uint8_t e) {
  // e8m0: 2^(e - 127); the quantiser writes 7..247, others are clamped into
  // the exponents of normal numbers
  const int c = e < 1 ? 1 : e > 254 ? 254 : e;
  return __uint_as_float((uint32_t)c << 23);
}

// 4 e4m3 values to bf16, times a power of two: exact.
__device__ __forceinline__ u32x2 fp8x4_to_bf16(uint32_t v, float scale) {
  u32x2 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, scale, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, scale, true));
  return r;
}
// 8 of them as the instruction takes them.
__device__ __forceinline__ u32x4 fp8x8_to_bf16(uint32_t lo, uint32_t hi, float scale) {
  const u32x2 a = fp8x4_to_bf16(lo, scale), b = fp8x4_to_bf16(hi, scale);
  return u32x4{a[0], a[1], b[0], b[1]};
}

// One step of the product: 16 bytes of k of each side per lane.  A lane's
// bytes are k = 16 * (lane >> 4) bytes of 64; as both sides take the same
// order of k, any order is right.  float32 takes four instructions for it;
// those for one result are kept apart.
template <int T, int M, int N>
__device__ __forceinline__ void mma_all(const u32x4 (&a)[M], const u32x4 (&b)[N],
                                        f32x4 (&c)[M][N]) {
  if constexpr (T == kF32) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j)
          c[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
              __uint_as_float(a[i][e]), __uint_as_float(b[j][e]), c[i][j], 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j)
        c[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, a[i]), __builtin_bit_cast(bf16x8, b[j]), c[i][j], 0, 0, 0);
  }
}

template <int T, int N>
__device__ __forceinline__ void mma_row(u32x4 a, const u32x4 (&b)[N], f32x4 (&c)[N]) {
  const u32x4 a1[1] = {a};
  mma_all<T>(a1, b, reinterpret_cast<f32x4(&)[1][N]>(c));
}

// The six products of two sides in three parts.
template <int M, int N>
__device__ __forceinline__ void mma_split(const u32x4 (&a)[3][M], const u32x4 (&b)[3][N],
                                          f32x4 (&c)[M][N]) {
  mma_all<kBF16>(a[0], b[0], c);
  mma_all<kBF16>(a[1], b[0], c);
  mma_all<kBF16>(a[2], b[0], c);
  mma_all<kBF16>(a[0], b[1], c);
  mma_all<kBF16>(a[1], b[1], c);
  mma_all<kBF16>(a[0], b[2], c);
}

// ---------------------------------------------------------------------------
// Scores: tiles of <table row, sample row>, and what is done with them.
// ---------------------------------------------------------------------------
enum Use { kLoss = 0, kCoef = 1, kStore = 2 };

struct ScoreArgs {
  Rows w, h;
  int64_t n;                // samples; h may have rows of zeros behind them
  int tiles_n, splits;      // tiles of samples; parts of the table's range
  int v_begin, v_end;       // the table rows of this launch
  // kLoss: (max, sum of exp(s - max)) per part and sample
  float2* part;
  int64_t ldp;              // samples of a part
  // kCoef
  const void* targets;
  int targets64;
  int64_t ignore, vocab;
  const float* lse;
  const float* grad;        // of every sample's loss, or null for ones
  // [coef_rows][ldc] in blocks of 16 x 16, column 0 = table row v_begin,
  // zeros in rows from N on
  char* coef;
  int64_t coef_rows, ldc;
  // kStore
  const float* col_scale;   // or null
  char* out;
  int64_t ldo;
  int out_bf16;
};

// The product of up to two numbers in memory.
__device__ __forceinline__ float scale_by(const float* a, const float* b) {
  return (a ? *a : 1.f) * (b ? *b : 1.f);
}

__device__ __forceinline__ int64_t target_of(const void* t, int is64, int64_t n) {
  return is64 ? reinterpret_cast<const int64_t*>(t)[n]
              : (int64_t) reinterpret_cast<const int32_t*>(t)[n];
}

// What a wave does with scores of NS blocks of 16 samples: a lane has sample
// n + 16 j + (lane & 15) and table rows v + 16 i + 4 (lane >> 4) + e.
template <int USE, int TC, int NS>
struct Sink {
  float top[NS], sum[NS];                      // kLoss
  bool far;                                    // of the wave: past kFar
  // kCoef; lse in powers of two, or itself where `far`
  float lse2[NS], gg[NS];
  int yy[NS];                                  // -1: no loss
  bool some;                                   // of the wave: without a loss

  __device__ __forceinline__ void start(const ScoreArgs& a, int64_t n) {
    if constexpr (USE == kLoss) {
#pragma unroll
      for (int j = 0; j < NS; ++j) top[j] = -INFINITY, sum[j] = 0.f;
      far = false;
    }
    if constexpr (USE == kCoef) {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const int64_t m = n + j * 16;
        lse2[j] = 0.f, gg[j] = 0.f, yy[j] = -1;
        if (m < a.n) {
          const int64_t y = target_of(a.targets, a.targets64, m);
          if (y != a.ignore && y >= 0 && y < a.vocab) {
            yy[j] = (int)y;
            lse2[j] = a.lse[m];
            gg[j] = a.grad ? a.grad[m] : 1.f;
          }
        }
      }
      bool f = false, none = false;
#pragma unroll
      for (int j = 0; j < NS; ++j) f |= fabsf(lse2[j]) > kFar, none |= yy[j] < 0;
      far = __any(f);
      some = __any(none);
      if (!far)
#pragma unroll
        for (int j = 0; j < NS; ++j) lse2[j] *= kLog2e;
    }
  }

  // kCoef: whether the wave has targets among `rows` table rows from v on.
  __device__ __forceinline__ bool meets(int v, int rows) const {
    bool m = false;
    if constexpr (USE == kCoef) {
#pragma unroll
      for (int j = 0; j < NS; ++j) m |= (unsigned)(yy[j] - v) < (unsigned)rows;
      m = __any(m);
    }
    return m;
  }

  // Scores of the table rows from v1 and the samples from n1 on.  `cut`: some
  // of the rows may lie past the last one; `met`: what meets() says.  These
  // four are the same for all lanes.
  template <int MR>
  __device__ __forceinline__ void take(const ScoreArgs& a, f32x4 (&acc)[MR][NS], int v1, int n1,
                                       bool cut, bool met) {
    if constexpr (USE == kLoss) take_loss(a, acc, v1, cut);
    if constexpr (USE == kCoef) take_coef(a, acc, v1 - a.v_begin, n1, cut, met);
    if constexpr (USE == kStore) take_store(a, acc, v1, n1, cut);
  }

  template <int MR>
  __device__ __forceinline__ void take_loss(const ScoreArgs& a, f32x4 (&acc)[MR][NS], int v1,
                                            bool cut) {
    if (cut) {
      const int v = v1 + (threadIdx.x >> 4 & 3) * 4;
#pragma unroll
      for (int i = 0; i < MR; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int j = 0; j < NS; ++j)
            acc[i][j][e] = v + i * 16 + e < a.v_end ? acc[i][j][e] : -INFINITY;
    }
    float most[NS];
    bool above = false;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      most[j] = acc[0][j][0];
#pragma unroll
      for (int i = 0; i < MR; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) most[j] = fmaxf(most[j], acc[i][j][e]);
      above |= most[j] > top[j];
    }
    // The reference moves only when a score is above it, which gets rare.
    if (__any(above)) {
      bool f = false;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const float next = fmaxf(top[j], most[j]);
        sum[j] *= top[j] == -INFINITY ? 0.f : exp_of(top[j] - next);
        top[j] = next;
        f |= fabsf(next) > kFar && next != -INFINITY;
      }
      far = __any(f);
    }
    // the new terms are added to each other first: one rounding of the long
    // sum for all of them
    if (far) {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const float at0 = top[j] == -INFINITY ? 0.f : top[j];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s += exp_of(acc[i][j][e] - at0);
        sum[j] += s;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        // nothing but -inf so far: any finite reference will do
        const float ref = top[j] == -INFINITY ? 0.f : top[j] * kLog2e;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -ref));
        sum[j] += s;
      }
    }
  }

  template <int MR>
  __device__ __forceinline__ void take_coef(const ScoreArgs& a, f32x4 (&acc)[MR][NS], int v1,
                                            int n1, bool cut, bool met) {
    const int lane = threadIdx.x & 63;
    // 16 samples x 16 table rows are 512 bytes (float32: 1 KB, or three times
    // 512 bytes of its parts) in one piece, as a wave writes them and with
    // every 16 bytes of one sample, as the products read them.
    // bf16 rows take bf16 coefficients: the products' instructions have one type
    // for both sides, and a second part of each coefficient would double two
    // products.  Rounding them takes the gradient's error from 1.65e-3 of it
    // (root mean square), which is its own rounding to bf16, to 1.72e-3 (256 x
    // 10k x 128).  Who wants them in 32 bits calls with float32 rows.
    constexpr int es = TC == kF32 ? 4 : 2, parts = Elem<TC>::parts;
    const int in_block = (lane & 15) * (16 * es) + (lane >> 4) * (4 * es);
    auto put = [&](int i, int j, f32x4 c) {
      char* to = a.coef + (((n1 >> 4) + j) * (a.ldc >> 4) + (v1 >> 4) + i) * (256 * es * parts);
      to += in_block;
      if constexpr (TC == kSplit) {
        u32x2 t[3];
        split4(c, t);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x2*>(to + p * 512) = t[p];
      } else if constexpr (TC == kF32) *reinterpret_cast<f32x4*>(to) = c;
      else *reinterpret_cast<u32x2*>(to) = u32x2{pack_bf16(c[0], c[1]), pack_bf16(c[2], c[3])};
    };
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      if (n1 + j * 16 >= a.coef_rows) break;
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        f32x4 c = acc[i][j];
        if (far) {
          // the difference first: it is exact for the scores that matter, while
          // lse in powers of two would be off by whole powers; lse's own
          // rounding may pass 0.  Not fminf(), which would drop a NaN
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float below = c[e] - lse2[j];
            c[e] = exp_of(below > 0.f ? 0.f : below);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            c[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(c[e], kLog2e, -lse2[j]));
        }
        const int first = a.v_begin + v1 + (lane >> 4) * 4 + i * 16;
        if (met) {
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] -= first + e == yy[j] ? 1.f : 0.f;
        }
        c *= gg[j];
        // without a loss gg is 0 and h zeros, but 0 times a table's infinity is
        // NaN (one branch that is rarely taken; with two the kernel for resident
        // samples takes 4 % longer)
        if (cut || some) {
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = yy[j] >= 0 ? c[e] : 0.f;
          if (cut) {
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = first + e < a.v_end ? c[e] : 0.f;
          }
        }
        put(i, j, c);
        // one after the other: side by side they would not fit the registers
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // 4 scores of neighbouring table rows; rows of the output start anywhere.
  __device__ __forceinline__ static void put_scores(char* o, f32x4 s, bool bf16) {
    if (bf16)
      *reinterpret_cast<u32x2a2*>(o) = u32x2{pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3])};
    else
      *reinterpret_cast<f32x4a4*>(o) = s;
  }

  // An instruction that writes 16 rows of the output, 64 bytes each, is slow:
  // half of the lanes swap one of two blocks with the other half, so that it
  // writes 8 rows, 128 bytes each (4096 x 200k float32 scores: 1.08 ms without,
  // 0.78 ms with).
  template <int MR>
  __device__ __forceinline__ void take_store(const ScoreArgs& a, f32x4 (&acc)[MR][NS], int v1,
                                             int n1, bool cut) {
    const bool bf16 = a.out_bf16;
    const int es = bf16 ? 2 : 4;
    const int r16 = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
    const int left = (int)a.n - n1;          // samples from n1 on
    char* first = a.out + ((int64_t)n1 * a.ldo + v1) * es;
    if (cut) {
#pragma unroll
      for (int i = 0; i < MR; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          if (r16 + j * 16 >= left) continue;
          char* o = first + ((r16 + j * 16) * a.ldo + 4 * g + i * 16) * es;
          const f32x4 s = acc[i][j];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (v1 + 4 * g + i * 16 + e < a.v_end) {
              if (bf16) reinterpret_cast<__bf16*>(o)[e] = (__bf16)s[e];
              else reinterpret_cast<float*>(o)[e] = s[e];
            }
          __builtin_amdgcn_sched_barrier(0);
        }
      return;
    }
    if constexpr (MR % 2 == 0) {
      const bool high = r16 & 8;
      const int64_t in = ((r16 & 7) * a.ldo + 4 * g + (high ? 16 : 0)) * es;
#pragma unroll
      for (int i = 0; i < MR; i += 2)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const f32x4 x = acc[i][j], y = acc[i + 1][j];
          f32x4 low, up;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float other = __int_as_float(__builtin_amdgcn_mov_dpp(
                __float_as_int(high ? x[e] : y[e]), 0x128, 0xf, 0xf, false));   // row_ror:8
            low[e] = high ? other : x[e];
            up[e] = high ? y[e] : other;
          }
          char* o = first + (j * 16 * a.ldo + i * 16) * es;
          if ((r16 & 7) + j * 16 < left) put_scores(o + in, low, bf16);
          if ((r16 & 7) + j * 16 + 8 < left) put_scores(o + 8 * a.ldo * es + in, up, bf16);
          __builtin_amdgcn_sched_barrier(0);      // or the registers do not do
        }
    } else {
      const int64_t in = (r16 * a.ldo + 4 * g) * es;
#pragma unroll
      for (int i = 0; i < MR; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j)
          if (r16 + j * 16 < left)
            put_scores(first + (j * 16 * a.ldo + i * 16) * es + in, acc[i][j], bf16);
    }
  }

  // kLoss, after the last tile: joins the four lanes, then the waves, that
  // hold one sample.  Wave `wave` has samples from 16 NS (wave / WV) on.
  template <int WV, int kWaves = 4>
  __device__ __forceinline__ void finish_loss(const ScoreArgs& a, char* lds, int split,
                                              int64_t n0) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int kCols = NS * 16;
    float2* red = reinterpret_cast<float2*>(lds);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NS; ++j) {
#pragma unroll
      for (int m = 16; m < 64; m <<= 1) {
        const float t = __shfl_xor(top[j], m), s = __shfl_xor(sum[j], m);
        join(top[j], sum[j], t, s);
      }
      if (lane < 16) red[wave * kCols + j * 16 + lane] = make_float2(top[j], sum[j]);
    }
    __syncthreads();
    if (threadIdx.x < kWaves / WV * kCols) {
      const int group = threadIdx.x / kCols, c = threadIdx.x % kCols;
      float2 p = red[group * WV * kCols + c];
#pragma unroll
      for (int i = 1; i < WV; ++i) {
        const float2 q = red[(group * WV + i) * kCols + c];
        join(p.x, p.y, q.x, q.y);
      }
      if (n0 + threadIdx.x < a.n) a.part[split * a.ldp + n0 + threadIdx.x] = p;
    }
  }
};

// The workgroup's tile of samples and part of the table.  Workgroups go round
// the 8 XCDs.  Where there are parts for all XCDs, those of one XCD take all
// sample tiles of one part before the next part, so that its L2 gets each
// table row from memory once.
__device__ __forceinline__ void place(const ScoreArgs& a, int& tn, int& split) {
  const int of = a.splits % 8 == 0 ? 8 : 1;
  const int at = blockIdx.x / of;
  tn = at % a.tiles_n;
  split = at / a.tiles_n * of + (of == 8 ? blockIdx.x & 7 : 0);
}

// [t0, t1): part `split` of `splits` of the tiles.
__device__ __forceinline__ void part_of(int tiles, int split, int splits, int& t0, int& t1) {
  const int each = tiles / splits, more = tiles % splits;
  t0 = split * each + min(split, more);
  t1 = t0 + each + (split < more);
}

// Where chunk c of 16 bytes of row r lies in LDS, for rows of `pitch` bytes: a
// read of 16 bytes a lane, in which lanes 0-15 have chunk c of 16 rows, 16-31
// chunk c + 1 and so on, is served 16 lanes at a time, and not in order (0-3,
// 12-15, 20-27 first): these take all 64 banks.
__device__ __forceinline__ constexpr int row_chunk(int pitch, int r, int c) {
  const int q = (r >> 2) & 3;
  return pitch % 256 == 0 ? c ^ (r & 15) : pitch % 128 == 0 ? c ^ (r & 7)
                                         : c ^ (q & 1) << 1 ^ (q >> 1) * 3;
}

// The factor of table row v in stored scores.
__device__ __forceinline__ float col_scale_of(const ScoreArgs& a, int v) {
  return a.col_scale && v < a.v_end ? a.col_scale[v] : 1.f;
}

// 16 bytes a lane from global memory straight into LDS, 1 KB from `lds` on.
// The hardware counts it as a load; wait_loads() waits for it.
// Two rules on wait states hold here that neither the hardware nor, in inline
// assembly, the compiler sees to: one between a scalar write of M0 and the load,
// and five between a vector instruction's write of a scalar register and a load
// with that address (base may come from v_readfirstlane).  The write of M0 is
// one of the five, s_nop 3 the other four (4096 samples, 1M x 300 bf16: 2 to 3 %
// of the loss; the test of the built instructions' wait states looks for both).
__device__ __forceinline__ void load_lds16(const char* p, uint32_t offset, uint32_t lds) {
  const uint64_t at = (uint64_t)p;
  const uint64_t base = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) << 32 |
                        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}
// The same, and for all reads of LDS.
__device__ __forceinline__ void wait_all() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
// load_lds16 with 4 bytes a lane.
__device__ __forceinline__ void load_lds4(const char* p, uint32_t offset, uint32_t lds) {
  const uint64_t at = (uint64_t)p;
  const uint64_t base = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) << 32 |
                        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2"
               :: "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
// Waits until only the last N loads and stores are outstanding: they end in
// the order in which they were issued.
template <int N> __device__ __forceinline__ void wait_loads_but() {
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}

// Rows of up to 32 KS columns of bf16 (or of 8 bits, on the table's side), which
// on both sides start at multiples of 16 bytes.  A wave holds its 16 NS samples
// in registers for the whole launch, so that LDS is read for the table alone:
// one fragment of 16 table rows feeds NS instructions.  Table tiles of kRows
// rows are loaded straight into LDS, up to three ahead of the tile at work; two
// workgroups fit a CU, and one's exponentials run beside the other's products.
// WN of the four waves have different samples, the others share them and take
// different rows of the tile.
// 8-bit rows are brought to bf16 with their scale: exact, while the instructions
// on 8-bit operands lose bits inside (1.5e-5 to 2.8e-5 of the result).
//   4096 samples, 1M x 300 bf16: 2.30 ms, 1.07 PFLOP/s (the matrix unit and
//     the exponentials take turns); coefficients alone 3.3 ms traced
//   1 sample: 116 us, 5.2 TB/s, bound by memory
//   4096 queries, 200k x 300 in 8 bits, float32 scores: 0.77 ms
//     (4.3 TB/s of stores, which bound it: a fill reaches 6.8)
//   1 query of 1M x 300 in 8 bits: 58 us traced, 5.2 TB/s
constexpr int resident_rows(int ks, int use, int wn, bool fp8) {
  // with stores, tiles of at most 20 KB: four of them fit, so that the stores
  // of several tiles, which are waited for in order with the loads, may be on
  // their way; without, larger tiles have fewer barriers
  const int most = use == kLoss ? 40960 : 20480, pitch = ks * (fp8 ? 32 : 64);
  const int rows = 128 * pitch <= most ? 128 : 64 * pitch <= most ? 64 : 32;
  return rows < 64 && wn == 1 ? 64 : rows;
}

template <int KS, int NS, int WN, int USE, bool FP8>
__global__ __launch_bounds__(256, 2) void resident_kernel(ScoreArgs a) {
  constexpr int WV = 4 / WN;
  constexpr int kRows = resident_rows(KS, USE, WN, FP8);
  constexpr int kPitch = KS * (FP8 ? 32 : 64);       // bytes of a row in LDS
  constexpr int kChunks = kPitch / 16;
  // two workgroups share 160 KB
  constexpr int kEach = kRows * kPitch + (FP8 ? 256 : 0) + (USE == kStore ? kRows * 4 : 0);
  constexpr int kBufs = kEach * 4 + 64 <= 81920 + (USE == kStore ? 0 : 64) ? 4 : kEach * 3 <= 81920 ? 3 : 2;
  constexpr int kAhead = kBufs - 1;
  constexpr int kLoads = kRows / 4 * kChunks / 64;   // per lane and tile
  constexpr int MR = kRows / WV >= 32 && (KS * NS <= 24 || USE == kStore) ? 2 : 1;
  constexpr int kBlocks = (KS + 3) / 4;              // scales of a row
  constexpr int kScales = kRows * kBlocks;
  static_assert(kRows / 4 * kChunks % 64 == 0 && kRows % (16 * MR * WV) == 0, "");
  __shared__ __align__(16) char lds[kBufs][kRows * kPitch];
  __shared__ __align__(16) uint8_t scales[FP8 ? kBufs : 1][256];
  __shared__ __align__(16) float col[USE == kStore ? kBufs : 1][kRows];
  static_assert(!FP8 || kScales <= 256, "");
  // stores of a wave for one whole tile
  constexpr int kStores = USE == kLoss ? 0 : kRows / (16 * WV) * NS;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wv = wave % WV, wn = wave / WV;
  const int r16 = lane & 15, g = lane >> 4;
  int tn, split;
  place(a, tn, split);
  int t0, t1;
  part_of((a.v_end - a.v_begin + kRows - 1) / kRows, split, a.splits, t0, t1);
  const int64_t n0 = (int64_t)tn * (16 * NS * WN);
  const int64_t n = n0 + wn * (16 * NS) + r16;

  // a lane reads chunks g + 4 k of row r16 and of rows 16, 32, .. on
  const uint32_t at0 = r16 * kPitch + row_chunk(kPitch, r16, g) * 16;
  constexpr int kGroup = kPitch % 256 == 0 ? 4 : kPitch % 128 == 0 ? 2 : 1;
  auto chunk = [&](const char* rows, int k) {
    return *reinterpret_cast<const u32x4*>(rows + (at0 ^ (k % kGroup * 64)) +
                                           k / kGroup * (kGroup * 64));
  };
  // the order of k within 64 columns: 8-bit fragments are 16 columns wide
  u32x4 fb[KS][NS];
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const char* row = a.h.p + min(n + j * 16, a.h.rows - 1) * a.h.ld;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int o = FP8 ? (k >> 1) * 128 + g * 32 + (k & 1) * 16 : k * 64 + g * 16;
      fb[k][j] = *reinterpret_cast<const u32x4*>(row + min(o, (a.h.kb - 1) & ~15));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int have = a.h.kb - o - 4 * q;
        fb[k][j][q] &= have >= 4 ? 0xffffffffu : have <= 0 ? 0u : 0xffffu;
      }
    }
  }
  // what lies behind the last column of a table row is cut off here
  u32x4 keep[2];
  if constexpr (!FP8) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int have = a.w.kb - ((KS - 2 + i) * 64 + g * 16 + q * 4);
        keep[i][q] = have >= 4 ? 0xffffffffu : have == 2 ? 0xffffu : 0u;
      }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int have = a.w.kb - ((KS - 2) * 32 + g * 16 + q * 4);
      keep[0][q] = have >= 4 ? 0xffffffffu : have <= 0 ? 0u : (1u << (8 * have)) - 1;
    }
  }

  // What lies outside is replaced by what is inside, and no lane sits out: the
  // waits below count the loads of each wave.
  const int last_chunk = (a.w.kb - 1) / 16;
  auto fetch = [&](int tile) {
    const int v0 = a.v_begin + tile * kRows, buf = (tile - t0) % kBufs;
    const char* base = a.w.p + v0 * a.w.ld;
    const int last = min(kRows - 1, (int)a.w.rows - 1 - v0);
    // the places are worked out anew for every tile: kept, they would take the
    // registers that the samples need
    int from = lane;
    asm volatile("" : "+v"(from));
    // all waves load the same few scales: not counted, as the rows come after
    if constexpr (FP8)
      load_lds4((const char*)a.w.scales + (int64_t)v0 * kBlocks,
                (uint32_t)min(from * 4, ((last + 1) * kBlocks - 1) & ~3),
                lds_address(scales[buf]));
    if constexpr (USE == kStore)
      if (a.col_scale)
#pragma unroll
        for (int i = 0; i < kRows; i += 64)
          load_lds4((const char*)(a.col_scale + v0), (uint32_t)min(from + i, last) * 4,
                    lds_address(&col[buf][i]));
    const uint32_t to = lds_address(&lds[buf][wave * (kRows / 4) * kPitch]);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int p = from + 64 * i;
      const int r = wave * (kRows / 4) + p / kChunks;
      const int c = row_chunk(kPitch, r, p % kChunks);
      load_lds16(base, (uint32_t)(min(r, last) * (int)a.w.ld + min(c, last_chunk) * 16),
                 to + i * 1024);
    }
  };
  static_assert(USE != kStore || kRows >= 64, "");

  Sink<USE, kBF16, NS> sink;
  sink.start(a, n);
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (t0 + i < t1) fetch(t0 + i);
  // Whether the wave makes all of kStores for every tile but the last: then
  // those made since this tile's loads need not be waited for.
  const bool whole = n0 + (wn + 1) * (16 * NS) <= a.n;
  constexpr int kLater = (kAhead - 1) * kLoads, kMost = kLater + kAhead * kStores;
  for (int tile = t0; tile < t1; ++tile) {
    const int buf = (tile - t0) % kBufs;
    // the tile has arrived for all waves, and all are done with the one before
    if (tile + kAhead - 1 >= t1) wait_loads();
    else if (kStores > 0 && whole && tile >= t0 + kAhead) wait_loads_but<(kMost < 63 ? kMost : 63)>();
    else wait_loads_but<kLater>();
    __syncthreads();
    if (tile + kAhead < t1) fetch(tile + kAhead);
    const int v0 = a.v_begin + tile * kRows;
    const bool cut = v0 + kRows > a.v_end, met = sink.meets(v0, kRows);
    // Fragments are read kLead steps before they are used, those of the next
    // rows' first steps before these rows' scores are.
    constexpr int kReads = FP8 ? KS / 2 : KS;
    constexpr int kWant = MR == 2 && KS * NS > 24 ? 2 : 4, kLead = kReads < kWant ? kReads : kWant;
    constexpr int kGroups = kRows / (16 * MR * WV);
    u32x4 fa[kLead][MR];
    auto read = [&](int m, int k) {
#pragma unroll
      for (int i = 0; i < MR; ++i)
        fa[k % kLead][i] = chunk(&lds[buf][((m * WV + wv) * MR + i) * 16 * kPitch], k);
    };
#pragma unroll
    for (int k = 0; k < kLead; ++k) read(0, k);
#pragma unroll 1
    for (int m = 0; m < kGroups; ++m) {
      const int row0 = (m * WV + wv) * 16 * MR;
      f32x4 acc[MR][NS];
#pragma unroll
      for (int i = 0; i < MR; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kReads; ++k) {
        u32x4 (&f)[MR] = fa[k % kLead];
        if constexpr (!FP8) {
          if (k >= KS - 2)
#pragma unroll
            for (int i = 0; i < MR; ++i) f[i] &= keep[k - (KS - 2)];
          mma_all<kBF16>(f, fb[k], acc);
        } else {
#pragma unroll
          for (int i = 0; i < MR; ++i) {
            if (k == kReads - 1) f[i] &= keep[0];
            const float s = scale_of(scales[buf][(row0 + i * 16 + r16) * kBlocks + k / 2]);
#pragma unroll
            for (int half = 0; half < 2; ++half)
              mma_row<kBF16>(fp8x8_to_bf16(f[i][2 * half], f[i][2 * half + 1], s),
                             fb[2 * k + half], acc[i]);
          }
        }
        if (k + kLead < kReads) read(m, k + kLead);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (m + 1 < kGroups)
#pragma unroll
        for (int k = 0; k < kLead; ++k) read(m + 1, k);
      __builtin_amdgcn_sched_barrier(0);
      if (USE == kStore && a.col_scale)
#pragma unroll
        for (int i = 0; i < MR; ++i) {
          const f32x4 cs = *reinterpret_cast<const f32x4*>(&col[buf][(row0 + i * 16 + 4 * g) % kRows]);
#pragma unroll
          for (int j = 0; j < NS; ++j) acc[i][j] *= cs;
        }
      sink.template take<MR>(a, acc, v0 + row0, (int)n0 + wn * (16 * NS), cut, met);
    }
  }
  if constexpr (USE == kLoss) sink.template finish_loss<WV>(a, lds[0], split, n0);
}

// Rows of any width, both sides by way of LDS: 64 WV table rows x 16 NS WN
// samples per workgroup, 64 x 16 NS per wave.  Steps of 64 bytes of a sample's
// row (of each part) go straight into LDS, kAhead steps ahead of the one at
// work.  Both sides' rows start at multiples of 16 bytes; 8-bit table rows are
// converted when they are read from LDS, and their scales lie by block of
// columns, then row.
//   2047 samples, 100001 x 1024 bf16, coefficients: 0.57 ms traced, 0.73
//     PFLOP/s (LDS and barriers bound it)
//   2047 samples, 30000 x 1024 float32 in parts, loss: 651 us, 193 TFLOP/s or
//     1.16 PFLOP/s of bf16 (half of the matrix unit's time; all waves of a CU
//     share one barrier a step)
//   2000 samples, 3613 x 100 float32: 24 us, 60 TFLOP/s, one round of
//     workgroups and its start
template <int TW, int TC, int USE, int WV, int WN, int NS>
__global__ __launch_bounds__(64 * WV * WN, 2) void tile_kernel(ScoreArgs a) {
  // float32 steps are long: two ahead do, and three workgroups fit a CU; the
  // small tile's are short
  constexpr int kWaves = WV * WN, MR = 4, P = Elem<TC>::parts;
  constexpr int kAhead = TC == kSplit ? 1 : TC == kF32 ? (WV == 1 ? 4 : 2) : 3;
  constexpr int kV = 64 * WV, kN = 16 * NS * WN;
  constexpr int kWideW = TW == kFP8 ? 32 : 64, kWideH = 64;   // bytes per step and part
  constexpr int kPartW = kV * kWideW, kPartH = kN * kWideH;
  constexpr int kBytesW = kPartW * P, kBytesH = kPartH * P;
  constexpr int kBytesS = TW == kFP8 ? kV : 0;
  constexpr int kInstr = (kBytesW + kBytesH) / 1024;          // loads of a whole wave
  constexpr int kEach = kInstr / kWaves, kMore = kInstr % kWaves;
  // kMid: the barrier in the middle of a step; coefficients would spill more
  // registers with it, and gain nothing.  kAmong: loads among the products.
  constexpr bool kMid = TW == kBF16 && NS == 8 && USE != kCoef;
  constexpr bool kAmong = TC == kBF16 && NS >= 4 && !kMid;
  // the scales are one more load, of the last wave
  constexpr int kScaleWave = TW == kFP8 ? kWaves - 1 : -1;
  static_assert(kBytesW % 1024 == 0 && kBytesH % 1024 == 0 && kMore < kWaves, "");
  static_assert(TW != kFP8 || kV == 256, "");
  static_assert(P == 1 || (kMore == 0 && kEach >= 2 * MR), "");
  __shared__ __align__(16) char lds[kAhead + 1][kBytesW + kBytesH + kBytesS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wv = wave % WV, wn = wave / WV;
  const int r16 = lane & 15, g = lane >> 4;
  int tn, split;
  place(a, tn, split);
  int t0, t1;
  part_of((a.v_end - a.v_begin + kV - 1) / kV, split, a.splits, t0, t1);
  const int64_t n0 = (int64_t)tn * kN;
  const int64_t n = n0 + wn * (16 * NS) + r16;
  const int steps = (a.h.kb + kWideH - 1) / kWideH;
  const int64_t all = (int64_t)(t1 - t0) * steps;
  const int last_h = (int)min((int64_t)kN - 1, a.h.rows - 1 - n0);

  // What lies outside is replaced by what is inside, and no lane sits out: the
  // waits below count the loads of each wave.
  int fetch_tile = t0, fetch_step = 0;
  constexpr int kFetches = kEach + (kMore > 0);
  // load i of kFetches of the step that is next
  auto fetch_one = [&](int buf, int i) INLINE {
    const int v0 = a.v_begin + fetch_tile * kV;
    const int ow = fetch_step * (kWideW * P), oh = fetch_step * (kWideH * P);
    const int q = wave + kWaves * i;
    if (q * 1024 < kBytesW) {
      const int part = q / (kPartW / 1024), p = (q - part * (kPartW / 1024)) * 64 + lane;
      const int r = TW == kFP8 ? p >> 1 : p >> 2;
      const int c = TW == kFP8 ? p & 1 : row_chunk(64, r, p & 3);
      const int last = min(kV - 1, (int)a.w.rows - 1 - v0);
      const int at = P > 1 ? part * 64 + c * 16 : min(c * 16, ((a.w.kb - 1) & ~15) - ow);
      load_lds16(a.w.p + v0 * a.w.ld + ow, (uint32_t)(min(r, last) * (int)a.w.ld + at),
                 lds_address(&lds[buf][q * 1024]));
    } else if (q < kInstr) {
      const int q1 = q - kBytesW / 1024;
      const int part = q1 / (kPartH / 1024), p = (q1 - part * (kPartH / 1024)) * 64 + lane;
      const int r = p >> 2, c = row_chunk(64, r, p & 3);
      const int at = P > 1 ? part * 64 + c * 16 : min(c * 16, ((a.h.kb - 1) & ~15) - oh);
      load_lds16(a.h.p + n0 * a.h.ld + oh, (uint32_t)(min(r, last_h) * (int)a.h.ld + at),
                 lds_address(&lds[buf][q * 1024]));
    }
  };
  auto fetched = [&]() INLINE {
    // kSplit loads without a branch: after the last step, that one again
    if (P > 1 && fetch_tile + 1 == t1 && fetch_step + 1 == steps) return;
    if (++fetch_step == steps) fetch_step = 0, ++fetch_tile;
  };
  auto fetch = [&](int buf) INLINE {
#pragma unroll
    for (int i = 0; i < kFetches; ++i) fetch_one(buf, i);
    if constexpr (TW == kFP8) {
      // kV bytes, four to a lane; rows past the end have room
      if (wave == kScaleWave)
        load_lds4((const char*)a.w.scales + (int64_t)(fetch_step * kWideW >> 7) * a.w.lds +
                      a.v_begin + fetch_tile * kV,
                  (uint32_t)lane * 4, lds_address(&lds[buf][kBytesW + kBytesH]));
    }
    fetched();
  };

  Sink<USE, TC, NS> sink;
  sink.start(a, n);
  f32x4 acc[MR][NS];
#pragma unroll
  for (int i = 0; i < kAhead + kMid; ++i)
    if (i < all) fetch(i);
  int tile = t0, step = 0, at_buf = 0;
  auto finish_tile = [&]() INLINE {
    const int v = a.v_begin + tile * kV + wv * 64 + 4 * g;
    if (USE == kStore && a.col_scale)
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        f32x4 cs;
#pragma unroll
        for (int e = 0; e < 4; ++e) cs[e] = col_scale_of(a, v + i * 16 + e);
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] *= cs;
      }
    const int v0 = a.v_begin + tile * kV + wv * 64;
    sink.template take<MR>(a, acc, v0, (int)n0 + wn * (16 * NS), v0 + 64 > a.v_end,
                           sink.meets(v0, 64));
    step = 0;
    ++tile;
  };
  const int at = r16 * 64 + row_chunk(64, r16, g) * 16;
  if constexpr (P > 1) {
    // The step's fragments are in registers and the next step's tiles in LDS
    // before the last two products, which run beside the next step's first
    // reads and the loads of the one after.
    u32x4 fa[P][MR], fb[P][NS], na[MR], nb[NS];
    auto read_a = [&](u32x4 (&f)[MR], int buf, int p) INLINE {
      const char* q = lds[buf] + p * kPartW + wv * 64 * 64 + at;
#pragma unroll
      for (int i = 0; i < MR; ++i) f[i] = *reinterpret_cast<const u32x4*>(q + i * 16 * 64);
    };
    auto read_b = [&](u32x4 (&f)[NS], int buf, int p) INLINE {
      const char* q = lds[buf] + kBytesW + p * kPartH + wn * (16 * NS) * 64 + at;
#pragma unroll
      for (int j = 0; j < NS; ++j) f[j] = *reinterpret_cast<const u32x4*>(q + j * 16 * 64);
    };
    wait_loads();
    __syncthreads();
    if (all > 0) fetch(1), read_a(na, 0, 0), read_b(nb, 0, 0);
    for (int64_t s = 0; s < all; ++s) {
      if (step == 0) {
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int j = 0; j < NS; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int i = 0; i < MR; ++i) fa[0][i] = na[i];
#pragma unroll
      for (int j = 0; j < NS; ++j) fb[0][j] = nb[j];
      // 4 NS results of one product, and loads or reads among them: in one
      // block they would keep the matrix unit waiting
      auto mma = [&](int p, int q, int i) INLINE {
#pragma unroll
        for (int j = 0; j < NS; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, fa[p][i]), __builtin_bit_cast(bf16x8, fb[q][j]),
              acc[i][j], 0, 0, 0);
      };
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        if (i == 0) read_a(fa[1], at_buf, 1);
        if (i == 1) read_b(fb[1], at_buf, 1);
        if (i == 2) read_a(fa[2], at_buf, 2);
        if (i == 3) read_b(fb[2], at_buf, 2);
        mma(0, 0, i);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < MR; ++i) mma(1, 0, i);
#pragma unroll
      for (int i = 0; i < MR; ++i) mma(0, 1, i);
#pragma unroll
      for (int i = 0; i < MR; ++i) mma(2, 0, i);
      __builtin_amdgcn_sched_barrier(0);
      const int to = at_buf;
      wait_all();
      __syncthreads();
      at_buf ^= 1;
      read_a(na, at_buf, 0);
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        mma(1, 1, i);
        if (i == 0) read_b(nb, at_buf, 0);
        fetch_one(to, i);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        mma(0, 2, i);
        fetch_one(to, i + MR);
        if (i + 1 == MR)
#pragma unroll
          for (int k = 2 * MR; k < kFetches; ++k) fetch_one(to, k);
        __builtin_amdgcn_sched_barrier(0);
      }
      fetched();
      if (++step == steps) finish_tile();
    }
    wait_loads();
    if constexpr (USE == kLoss) sink.template finish_loss<WV, kWaves>(a, &lds[0][0], split, n0);
    return;
  }
  if constexpr (kMid) {
    // The same with one product a step: its second half runs beside the next
    // step's first reads and the loads of four steps on (2047 samples, 100001 x
    // 1024: loss 512 us traced, with the barrier at the step's start 527).
    static_assert(kMore == 0 && kEach == MR, "");
    u32x4 fa[MR], fb[NS], na[MR];
    auto read_a = [&](int buf) INLINE {
      const char* q = lds[buf] + wv * 64 * 64 + at;
#pragma unroll
      for (int i = 0; i < MR; ++i) na[i] = *reinterpret_cast<const u32x4*>(q + i * 16 * 64);
    };
    auto mma = [&](int j) INLINE {
#pragma unroll
      for (int i = 0; i < MR; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, fa[i]), __builtin_bit_cast(bf16x8, fb[j]), acc[i][j], 0, 0, 0);
    };
    if (kAhead < all) wait_loads_but<kAhead * kEach>();
    else wait_loads();
    __syncthreads();
    if (all > 0) read_a(0);
    for (int64_t s = 0; s < all; ++s) {
      if (step == 0) {
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int j = 0; j < NS; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      const char* lh = lds[at_buf] + kBytesW + wn * (16 * NS) * kWideH + at;
#pragma unroll
      for (int j = 0; j < NS; ++j) fb[j] = *reinterpret_cast<const u32x4*>(lh + j * 16 * 64);
#pragma unroll
      for (int i = 0; i < MR; ++i) fa[i] = na[i];
      if (step + 1 == steps && (a.h.kb & 63) != 0) {
        // columns past the last one, whatever they hold
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int have = a.h.kb - (step * kWideH + g * 16 + q * 4);
          const uint32_t keep = have >= 4 ? 0xffffffffu : have <= 0 ? 0u : (1u << (8 * have)) - 1;
#pragma unroll
          for (int i = 0; i < MR; ++i) fa[i][q] &= keep;
#pragma unroll
          for (int j = 0; j < NS; ++j) fb[j][q] &= keep;
        }
      }
#pragma unroll
      for (int j = 0; j < NS / 2; ++j) mma(j);
      __builtin_amdgcn_sched_barrier(0);
      const int to = at_buf;
      const bool more = s + kAhead + 1 < all;
      at_buf = at_buf == kAhead ? 0 : at_buf + 1;
      if (s + 1 < all) {
        // step s + 1 has arrived, two more may be on their way
        if (s + kAhead < all) wait_loads_but<(kAhead - 1) * kEach>();
        else wait_loads();
        wait_lds();
        __syncthreads();
        read_a(at_buf);
      }
#pragma unroll
      for (int j = NS / 2; j < NS; ++j) {
        mma(j);
        if (more) fetch_one(to, j - NS / 2);
      }
      if (more) fetched();
      if (++step == steps) finish_tile();
    }
    if constexpr (USE == kLoss) sink.template finish_loss<WV, kWaves>(a, &lds[0][0], split, n0);
    return;
  }
  for (int64_t s = 0; s < all; ++s) {
    // step s has arrived, two more may be on their way
    if (s + kAhead - 1 < all) {
      if (wave < kMore || wave == kScaleWave) wait_loads_but<(kAhead - 1) * (kEach + 1)>();
      else wait_loads_but<(kAhead - 1) * kEach>();
    } else {
      wait_loads();
    }
    __syncthreads();
    const bool more = s + kAhead < all;
    const int to = at_buf == 0 ? kAhead : at_buf - 1;
    if (!kAmong && more) fetch(to);
    if (step == 0) {
#pragma unroll
      for (int i = 0; i < MR; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const char* buf = lds[at_buf];
    at_buf = at_buf == kAhead ? 0 : at_buf + 1;
    const char* lh = buf + kBytesW + wn * (16 * NS) * kWideH;
    u32x4 fa[MR], fb[NS];
#pragma unroll
    for (int i = 0; i < MR; ++i) {
      if constexpr (TW == kFP8) {
        const int r = wv * 64 + i * 16 + r16;
        const u32x2 q = *reinterpret_cast<const u32x2*>(buf + r * 32 + g * 8);
        const uint8_t e = *reinterpret_cast<const uint8_t*>(buf + kBytesW + kBytesH + r);
        fa[i] = fp8x8_to_bf16(q[0], q[1], scale_of(e));
      } else {
        fa[i] = *reinterpret_cast<const u32x4*>(buf + (wv * 64 + i * 16) * 64 + at);
      }
    }
#pragma unroll
    for (int j = 0; j < NS; ++j)
      fb[j] = *reinterpret_cast<const u32x4*>(lh + j * 16 * 64 + at);
    if (step + 1 == steps && (a.h.kb & 63) != 0) {
      // columns past the last one, whatever they hold
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int have = a.h.kb - (step * kWideH + g * 16 + q * 4);
        const uint32_t keep = have >= 4 ? 0xffffffffu : have <= 0 ? 0u : (1u << (8 * have)) - 1;
#pragma unroll
        for (int i = 0; i < MR; ++i) fa[i][q] &= keep;
#pragma unroll
        for (int j = 0; j < NS; ++j) fb[j][q] &= keep;
      }
    }
    if constexpr (kAmong) {
      // loads among the products: in one block they would keep the matrix unit
      // waiting
      constexpr int kPerRow = (kFetches + MR - 1) / MR;
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        mma_row<TC>(fa[i], fb, acc[i]);
        if (more)
#pragma unroll
          for (int k = i * kPerRow; k < (i + 1) * kPerRow && k < kFetches; ++k) fetch_one(to, k);
      }
      if (more) fetched();
    } else {
      mma_all<TC>(fa, fb, acc);
    }
    if (++step == steps) finish_tile();
  }
  if constexpr (USE == kLoss) sink.template finish_loss<WV, kWaves>(a, &lds[0][0], split, n0);
}

// Few samples: bound by the bytes of the table, which go from memory to the
// registers of the one wave that needs them (7 samples, 201905 x 860 float32:
// 157 us, 4.4 TB/s).  A wave takes 16 rows at a time, eight loads of 16 bytes a
// lane ahead of the eight at work; the samples lie in LDS as the instruction
// takes them.  Any type, size and alignment; VEC:
// table rows start at multiples of 16 bytes.
template <int TW, int TC, int NS, int USE, bool VEC>
__global__ __launch_bounds__(256) void stream_kernel(ScoreArgs a) {
  constexpr int kAhead = 8;
  constexpr int kSteps = TW == kFP8 ? 2 : 1;         // instructions for 16 bytes of a row
  extern __shared__ __align__(16) char samples[];    // [step][NS][64 lanes][16 bytes]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  int tn, split;
  place(a, tn, split);
  const int64_t n0 = (int64_t)tn * (16 * NS);
  const int64_t n = n0 + r16;
  const int chunks = (a.w.kb + 63) / 64;             // per lane and row
  for (int i = threadIdx.x; i < chunks * kSteps * NS * 64; i += 256) {
    const int f = i >> 6, l = i & 63, j = f % NS, k = f / NS;
    const int o = TW == kFP8 ? (k >> 1) * 128 + (l >> 4) * 32 + (k & 1) * 16
                             : k * 64 + (l >> 4) * 16;
    reinterpret_cast<u32x4*>(samples)[i] =
        load16<Elem<TC>::size>(a.h, n0 + j * 16 + (l & 15), o);
  }
  Sink<USE, TC, NS> sink;
  sink.start(a, n);
  __syncthreads();

  int t0, t1;
  part_of((a.v_end - a.v_begin + 63) / 64, split, a.splits, t0, t1);
  // this wave's rows are 16 of every 64
  const int groups = t1 - t0;
  const int v_first = a.v_begin + t0 * 64 + wave * 16;
  u32x4 next[kAhead];
  uint8_t next_scale[TW == kFP8 ? kAhead : 1];
  // rows and columns past the end are replaced by the last ones: such rows
  // are not used, such columns are cut off below
  u32x4 keep;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int have = a.w.kb - ((chunks - 1) * 64 + g * 16 + q * 4);
    keep[q] = have >= 4 ? 0xffffffffu : have <= 0 ? 0u : (1u << (8 * have)) - 1;
  }
  const int last_byte = (a.w.kb - 1) & ~15;
  auto fetch = [&](int group, int k0) {
    const int64_t row = v_first + group * 64 + r16;
    const int64_t at = min(row, a.w.rows - 1);
    const char* p = a.w.p + at * a.w.ld;
    const uint8_t* ps = a.w.scales + at * a.w.lds;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int o = (k0 + i) * 64 + g * 16;
      if constexpr (VEC) next[i] = *reinterpret_cast<const u32x4*>(p + min(o, last_byte));
      else next[i] = load16<Elem<TW>::size>(a.w, row, o);
      if constexpr (TW == kFP8)
        next_scale[i] = ps[min((k0 + i) * 64, a.w.kb - 1) >> 7];
    }
  };
  if (groups > 0) fetch(0, 0);
  for (int group = 0; group < groups; ++group) {
    f32x4 acc[1][NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int v = v_first + group * 64 + 4 * g;
    f32x4 cs = {1.f, 1.f, 1.f, 1.f};
    for (int k0 = 0; k0 < chunks; k0 += kAhead) {
      u32x4 now[kAhead];
      float scale[TW == kFP8 ? kAhead : 1];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) now[i] = next[i];
      if constexpr (TW == kFP8)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) scale[i] = scale_of(next_scale[i]);
      if (k0 + kAhead < chunks) fetch(group, k0 + kAhead);
      else if (group + 1 < groups) fetch(group + 1, 0);
      if constexpr (USE == kStore)
        if (k0 + kAhead >= chunks)
#pragma unroll
          for (int e = 0; e < 4; ++e) cs[e] = col_scale_of(a, v + e);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (k0 + i >= chunks) break;
        if (VEC && k0 + i == chunks - 1) now[i] &= keep;
        const char* fb = samples + (size_t)(k0 + i) * (kSteps * NS * 1024) + lane * 16;
        if constexpr (TW == kFP8) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const u32x4 fa = fp8x8_to_bf16(now[i][2 * half], now[i][2 * half + 1], scale[i]);
            u32x4 f[NS];
#pragma unroll
            for (int j = 0; j < NS; ++j)
              f[j] = *reinterpret_cast<const u32x4*>(fb + (half * NS + j) * 1024);
            mma_row<TC>(fa, f, acc[0]);
          }
        } else {
          u32x4 f[NS];
#pragma unroll
          for (int j = 0; j < NS; ++j) f[j] = *reinterpret_cast<const u32x4*>(fb + j * 1024);
          mma_row<TC>(now[i], f, acc[0]);
        }
      }
    }
    if constexpr (USE == kStore)
#pragma unroll
      for (int j = 0; j < NS; ++j) acc[0][j] *= cs;
    sink.template take<1>(a, acc, v - 4 * g, (int)n0, v_first + group * 64 + 16 > a.v_end, false);
  }
  if constexpr (USE == kLoss) sink.template finish_loss<4>(a, samples, split, n0);
}

// ---------------------------------------------------------------------------
// Joins the parts of one sample's softmax and takes its target's score off: one
// wave per sample, four to a workgroup.  Latency bounds it: two rows and some
// hundred pairs a sample (4096 samples of 1M x 300: 7 us).
// ---------------------------------------------------------------------------
template <int T>
__device__ __forceinline__ float elem(const char* p, int64_t i) {
  if constexpr (T == kF32) return reinterpret_cast<const float*>(p)[i];
  else return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

template <int T>
__global__ __launch_bounds__(256) void loss_join_kernel(
    int64_t block0, Rows w, Rows h, const float2* part, int splits, int64_t ldp,
    const void* targets, int targets64, int64_t ignore, float* loss, float* lse) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (block0 + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (n >= h.rows) return;
  float top = -INFINITY, sum = 0.f;
  for (int s = lane; s < splits; s += 64) {
    const float2 p = part[s * ldp + n];
    join(top, sum, p.x, p.y);
  }
  const int64_t y = target_of(targets, targets64, n);
  const bool ours = y != ignore && y >= 0 && y < w.rows;
  float right = 0.f;
  if (ours) {
    const char* wr = w.p + y * w.ld;
    const char* hr = h.p + n * h.ld;
    for (int k = lane; k < h.kb / Elem<T>::size; k += 64)
      right = __builtin_fmaf(elem<T>(wr, k), elem<T>(hr, k), right);
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const float t = __shfl_xor(top, m), s = __shfl_xor(sum, m);
    right += __shfl_xor(right, m);
    join(top, sum, t, s);
  }
  if (lane == 0) {
    const float total = top + log2f(sum) * kLn2;
    lse[n] = total;
    loss[n] = y == ignore ? 0.f : ours ? total - right : NAN;
  }
}

// Sum or mean over the samples that count, in 64 bits and a fixed order.
// factor = 1 / count for the mean, 1 for the sum; result = the sum times it.
// The mean of none is NaN, and its factor 0: no gradient, where 0 times the
// factor would be NaN too.
__global__ __launch_bounds__(1024) void loss_reduce_kernel(
    const float* loss, const void* targets, int targets64, int64_t ignore,
    int64_t n, int mean, float* result, float* factor) {
  __shared__ double sums[16];
  __shared__ long long counts[16];
  double s = 0;
  long long c = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024)
    if (target_of(targets, targets64, i) != ignore) s += loss[i], ++c;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m), c += __shfl_xor(c, m);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s, counts[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += sums[i], c += counts[i];
    const double f = mean ? 1.0 / (double)c : 1.0;
    *result = (float)(s * f);
    *factor = c || !mean ? (float)f : 0.f;
  }
}

// ---------------------------------------------------------------------------
// Products with the coefficients: out[r][d] = sum_k b(r, k) x[k][d]
//   dh: r = sample, k = table row, b = coef[r][k]
//   dw: r = table row, k = sample, b = coef[k][r]
// x has k down its rows, so its tile is read from LDS transposed, as is b's
// for dw.
// ---------------------------------------------------------------------------
struct GradArgs {
  Rows x;              // [K][D]
  const char* coef;    // in blocks of 16 samples x 16 table rows
  int64_t ldc;         // table rows of 16 samples' blocks
  int64_t r, k;
  int d;
  int tiles_d, tiles_r, splits;
  float* part;   // [splits][R][ldp], added to where `add`; or null, and
  int64_t ldp;
  int add;
  const float* scale[2];   // factors of all results, or null
  char* out;     // [R][D], of the rows' type
  int64_t ldo;
};

// Rows in parts of bf16: for each 32 columns 64 bytes of each part, and zeros
// as in pack_kernel.  A thread takes 8 columns.  Bound by memory: 4 bytes read
// and 6 written for each number.
__global__ __launch_bounds__(256) void split_kernel(
    Rows h, const void* targets, int targets64, int64_t ignore, int64_t vocab, char* out,
    int64_t rows, int ldo) {
  const int chunks = ldo / 8;
  const int64_t total = rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / chunks;
    const int c = (int)(i - r * chunks);
    u32x4 v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (r < h.rows) {
      const int64_t y = targets ? target_of(targets, targets64, r) : 0;
      if (!targets || (y != ignore && y >= 0 && y < vocab))
#pragma unroll
        for (int k = 0; k < 2; ++k) v[k] = load16<4>(h, r, c * 32 + 16 * k);
    }
    u32x2 t[2][3];
#pragma unroll
    for (int k = 0; k < 2; ++k) split4(__builtin_bit_cast(f32x4, v[k]), t[k]);
    char* to = out + r * ldo * 6 + (c >> 2) * 192 + (c & 3) * 16;
#pragma unroll
    for (int p = 0; p < 3; ++p)
      *reinterpret_cast<u32x4*>(to + p * 64) = u32x4{t[0][p][0], t[0][p][1], t[1][p][0], t[1][p][1]};
  }
}

// Rows for the gradient: [rows][ldo] of 16-byte multiples with zeros behind
// the last column and row, and (with targets) in rows that have no loss,
// whatever they hold: a coefficient of 0 would not hide a NaN.
template <int T>
__global__ __launch_bounds__(256) void pack_kernel(
    Rows h, const void* targets, int targets64, int64_t ignore, int64_t vocab, char* out,
    int64_t rows, int ldo) {
  constexpr int ES = Elem<T>::size;
  const int chunks = ldo * ES / 16;
  const int64_t total = rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / chunks;
    const int c = (int)(i - r * chunks);
    u32x4 v = {0, 0, 0, 0};
    if (r < h.rows) {
      const int64_t y = targets ? target_of(targets, targets64, r) : 0;
      if (!targets || (y != ignore && y >= 0 && y < vocab)) v = load16<ES>(h, r, c * 16);
    }
    reinterpret_cast<u32x4*>(out)[i] = v;
  }
}

// Bound by LDS and the matrix unit: 4096 samples, 1M x 300 bf16: 3.0 ms for
// dh and 2.8 ms for dw, both traced, 0.83 and 0.89 PFLOP/s.
//
// Eight waves: WR times 16 J rows r, 8 / WR times 16 ND columns d.  With 256
// rows and 32 ND columns narrow tables are read once and the coefficients, the
// larger part, as often as there are tiles of d; fewer samples than that take
// the forms with fewer rows.  Steps of 64 bytes of k (32 of bf16, 16 of
// float32) go straight into LDS, kAhead steps ahead of the one at work: three,
// two for float32, whose steps are long, or one where k is short, as several
// workgroups a CU do more there, and for kSplit, whose steps fill LDS.
template <int T, bool DW, int ND, int WR, int J, int kAhead>
__global__ __launch_bounds__(512, 2) void grad_kernel(GradArgs a) {
  constexpr int ES = Elem<T>::size, P = Elem<T>::parts, WD = 8 / WR;
  constexpr int kRowsR = 16 * J * WR, kCols = 16 * ND * WD, kStep = 64 / ES;
  constexpr int kPitchX = kCols * ES, kPitchB = kRowsR * ES;     // bytes of a row k
  constexpr int kChunksX = kPitchX / 16, kChunksB = kPitchB / 16;
  constexpr int kPartX = kStep * kPitchX, kPartB = kStep * kPitchB;
  constexpr int kBytesX = kPartX * P, kBytesB = kPartB * P;
  constexpr int kInstr = (kBytesX + kBytesB) / 1024;             // loads of a whole wave
  constexpr int kEach = kInstr / 8, kMore = kInstr % 8;          // kMore waves have one more
  constexpr int kBlock = 256 * ES * P;               // bytes of 16 x 16 coefficients
  constexpr int kLine = 16 * ES;                     // of which one sample's
  static_assert(kPartX % 1024 == 0 && kPartB % 1024 == 0, "");
  static_assert(!DW || (WR == 4 && J == 4), "");
  __shared__ __align__(16) char lds[kAhead + 1][kBytesX + kBytesB];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wd = wave % WD, wr = wave / WD;
  const int r16 = lane & 15, g = lane >> 4;
  // the parts of k go round the XCDs: the tiles of r that share rows of x are
  // in one XCD at a time
  const int tiles = a.tiles_d * a.tiles_r;
  const int of = a.splits % 8 == 0 ? 8 : 1;
  const int split = (int)(blockIdx.x / of) / tiles * of + (of == 8 ? blockIdx.x & 7 : 0);
  const int at = (int)(blockIdx.x / of) % tiles;
  const int td = at % a.tiles_d, tr = at / a.tiles_d;
  int s0, s1;
  part_of((int)((a.k + kStep - 1) / kStep), split, a.splits, s0, s1);
  const int64_t r0 = (int64_t)tr * kRowsR;
  const int d0 = td * kCols;

  // Blocks of 16 columns (of kLine bytes) of row k lie at block ^ key(k): the
  // rows that one transposing read touches spread over the banks.
  auto key = [](int k, int pitch) {
    if constexpr (T == kF32) return (k >> 2) & 3;
    else return pitch % 256 == 0 ? (k & 3) | ((k >> 3) & 1) << 2
                                 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
  };
  constexpr int kPer = kLine / 16;                   // chunks of a block's row
  // What lies outside is replaced by what is inside, and no lane sits out: the
  // waits below count the loads of each wave.  Columns d and rows r past the
  // end are not stored; past the last k, one side is zeros.
  const int have_x = (a.x.kb - d0 * ES + 15) / 16;   // chunks of x from d0 on
  const int64_t block_row = a.ldc * (kLine * P);     // 16 samples' coefficients
  const int have_b = (int)min((int64_t)(DW ? kChunksB : kRowsR),
                              DW ? ((a.r - r0) * ES + 15) / 16 : a.r - r0);
  // load i of kFetches of step s
  constexpr int kFetches = kEach + (kMore > 0);
  auto fetch_one = [&](int s, int i) INLINE {
    char* buf = lds[(s - s0) % (kAhead + 1)];
    const int64_t k0 = (int64_t)s * kStep;
    const char* xb = a.x.p + k0 * a.x.ld + d0 * (ES * P);
    const int last = (int)min((int64_t)kStep - 1, a.x.rows - 1 - k0);
    const int q = wave + 8 * i;
    if (q * 1024 < kBytesX) {
      const int part = q / (kPartX / 1024), p = (q - part * (kPartX / 1024)) * 64 + lane;
      const int k = p / kChunksX, pos = p % kChunksX;
      const int c = min(((pos / kPer) ^ key(k, kPitchX)) * kPer + pos % kPer, have_x - 1);
      const int in = P > 1 ? (c >> 2) * 192 + part * 64 + (c & 3) * 16 : c * 16;
      load_lds16(xb, (uint32_t)(min(k, last) * (int)a.x.ld + in), lds_address(buf + q * 1024));
    } else if (q < kInstr) {
      const int q1 = q - kBytesX / 1024;
      const int part = q1 / (kPartB / 1024), p = (q1 - part * (kPartB / 1024)) * 64 + lane;
      const char* from;
      uint32_t offset;
      if constexpr (DW) {
        // samples k, chunk c of the table rows
        const int k = p / kChunksB, pos = p % kChunksB;
        const int c = ((pos / kPer) ^ key(k, kPitchB)) * kPer + pos % kPer;
        const int in = min(c, have_b - 1);
        from = a.coef + (k0 >> 4) * block_row + (r0 >> 4) * kBlock;
        offset = (uint32_t)(k >> 4) * (uint32_t)block_row + part * 512 + (k & 15) * kLine +
                 in / kPer * kBlock + in % kPer * 16;
      } else {
        // 64 bytes of samples r
        const int r = p >> 2, c = row_chunk(64, r, p & 3);
        const int in = min(r, have_b - 1);
        from = a.coef + (r0 >> 4) * block_row + (k0 >> 4) * kBlock;
        offset = (uint32_t)(in >> 4) * (uint32_t)block_row + part * 512 + (in & 15) * kLine +
                 c / kPer * kBlock + c % kPer * 16;
      }
      load_lds16(from, offset, lds_address(buf + q * 1024));
    }
  };
  auto fetch = [&](int s) INLINE {
#pragma unroll
    for (int i = 0; i < kFetches; ++i) fetch_one(s, i);
  };

  f32x4 acc[ND][J];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (s0 + i < s1) fetch(s0 + i);
  // 16 columns x one step of k: for bf16 by transposing reads, in which 16
  // lanes take 4 rows k of one block; for float32 a word at a time
  auto columns = [&](const char* p, int pitch, int block) {
    if constexpr (T != kF32) {
      const int k = 8 * g + (r16 >> 2);
      const char* q = p + k * pitch + ((block ^ key(k, pitch)) << 5) + (r16 & 3) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)q);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(q + 4 * pitch));
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      return u32x4{x[0], x[1], y[0], y[1]};
    } else {
      const char* q = p + 4 * g * pitch + ((block ^ key(4 * g, pitch)) << 6) + r16 * 4;
      u32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const uint32_t*>(q + e * pitch);
      return x;
    }
  };
  for (int s = s0; s < s1; ++s) {
    // step s has arrived, kAhead - 1 more may be on their way
    if (s + kAhead - 1 < s1) {
      if (wave < kMore) wait_loads_but<(kAhead - 1) * (kEach + 1)>();
      else wait_loads_but<(kAhead - 1) * kEach>();
    } else {
      wait_loads();
    }
    __syncthreads();
    const bool more = s + kAhead < s1;
    const char* x = lds[(s - s0) % (kAhead + 1)];
    const char* b = x + kBytesX;
    u32x4 fb[P][J];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if constexpr (DW) {
          fb[p][j] = columns(b + p * kPartB, kPitchB, wr * J + j);
        } else {
          const int r = (wr * J + j) * 16 + r16;
          fb[p][j] = *reinterpret_cast<const u32x4*>(b + p * kPartB + r * 64 +
                                                     row_chunk(64, r, g) * 16);
        }
      }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      if constexpr (P > 1) {
        u32x4 fa[P][1];
#pragma unroll
        for (int p = 0; p < P; ++p)
          fa[p][0] = columns(x + p * kPartX, kPitchX, wd * ND + i);
        mma_split(fa, fb, reinterpret_cast<f32x4(&)[1][J]>(acc[i]));
      } else {
        const u32x4 fa = columns(x, kPitchX, wd * ND + i);
        mma_row<T>(fa, fb[0], acc[i]);
      }
      // loads among the products: in one block they would keep the matrix unit
      // waiting
      constexpr int kPerRow = (kFetches + ND - 1) / ND;
      if (more)
#pragma unroll
        for (int k = i * kPerRow; k < (i + 1) * kPerRow && k < kFetches; ++k)
          fetch_one(s + kAhead, k);
    }
  }
  const float scale = a.part ? 1.f : scale_by(a.scale[0], a.scale[1]);
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int64_t r = r0 + (wr * J + j) * 16 + r16;
    if (r >= a.r) continue;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const int d = d0 + (wd * ND + i) * 16 + 4 * g;
      if (d >= a.d) continue;
      acc[i][j] *= scale;
      if (a.part) {
        f32x4* o = reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.r + r) * a.ldp + d);
        *o = a.add ? *o + acc[i][j] : acc[i][j];
      } else if constexpr (T != kBF16) {
        float* o = reinterpret_cast<float*>(a.out) + r * a.ldo + d;
        if ((a.ldo & 3) == 0) {       // then d + 3 < ldo as well
          *reinterpret_cast<f32x4*>(o) = acc[i][j];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < a.d) o[e] = acc[i][j][e];
        }
      } else {
        uint16_t* o = reinterpret_cast<uint16_t*>(a.out) + r * a.ldo + d;
        const uint32_t lo = pack_bf16(acc[i][j][0], acc[i][j][1]);
        const uint32_t hi = pack_bf16(acc[i][j][2], acc[i][j][3]);
        if ((a.ldo & 3) == 0) {
          *reinterpret_cast<u32x2*>(o) = u32x2{lo, hi};
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < a.d) o[e] = (uint16_t)((e < 2 ? lo : hi) >> (16 * (e & 1)));
        }
      }
    }
  }
}

// A result from its parts: G lanes of a workgroup share a result, so that many
// parts of few results are added at the same time, in a fixed order.  Bound by
// memory, or by latency where there is little.
template <int T, int G>
__global__ __launch_bounds__(256) void sum_parts_kernel(
    int64_t block0, const float* part, int splits, int64_t rows, int64_t ldp, int d,
    const float* scale0, const float* scale1, char* out) {
  constexpr int kEach = 256 / G;
  __shared__ float sums[G][kEach];
  const int at = threadIdx.x % kEach, group = threadIdx.x / kEach;
  const int64_t total = rows * d;
  const int64_t i = (block0 + blockIdx.x) * kEach + at;
  float s = 0.f;
  if (i < total) {
    const int64_t r = i / d, c = i - r * d;
#pragma unroll 4
    for (int p = group; p < splits; p += G) s += part[((int64_t)p * rows + r) * ldp + c];
  }
  sums[group][at] = s;
  __syncthreads();
  if (group == 0 && i < total) {
#pragma unroll
    for (int k = 1; k < G; ++k) s += sums[k][at];
    s *= scale_by(scale0, scale1);
    if constexpr (T == kF32) reinterpret_cast<float*>(out)[i] = s;
    else reinterpret_cast<__bf16*>(out)[i] = (__bf16)s;
  }
}

// ---------------------------------------------------------------------------
// Rows in 8 bits.  16 lanes take one block of 128 columns, 8 to a lane.
//   e = the least integer with max|x| <= 448 * 2^e, within [-120, 120]
//   value = x / 2^e to the nearest e4m3, ties to even; NaN for what is not
//   finite (the maximum is over the finite ones).  At e = 120 the value stops
//   at 240: the next one would stand for 2^128, which float32 does not hold
// TO_BF16 writes the values that the 8-bit rows stand for instead.
// ---------------------------------------------------------------------------
//
// A workgroup takes 64 blocks of 128 columns that follow each other, four to
// a group of lanes with all loads first; the position of the first one is the
// only division by a length of 64 bits.  Bound by memory: 1M x 300 bf16 in
// 252 us traced, 3.6 TB/s (read and written).
template <int T, bool TO_BF16>
__global__ __launch_bounds__(256) void quantize_kernel(
    int64_t block0, Rows x, int blocks, char* values, int64_t ldv, uint8_t* scales, int64_t lds) {
  constexpr int kEach = 4;
  const int sub = threadIdx.x & 15;
  const int64_t first = (block0 + blockIdx.x) * (16 * kEach);
  const int64_t row0 = first / blocks;
  const int in0 = (int)(first - row0 * blocks);
  int64_t row[kEach];
  int b[kEach];
  u32x4 q[kEach][T == kBF16 ? 1 : 2];
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int t = in0 + (threadIdx.x >> 4) + 16 * u;
    const int r = t / blocks;
    row[u] = row0 + r;
    b[u] = t - r * blocks;
    const int o = (b[u] * 128 + sub * 8) * Elem<T>::size;
    q[u][0] = load16<Elem<T>::size>(x, row[u], o);
    if constexpr (T == kF32) q[u][1] = load16<4>(x, row[u], o + 16);
  }
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    if (row[u] >= x.rows) return;      // the same for the 16 lanes of a block
    const int c0 = b[u] * 128 + sub * 8;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (T == kBF16) v[k] = bf16_to_f32((uint16_t)(q[u][0][k >> 1] >> (16 * (k & 1))));
      else v[k] = __uint_as_float(q[u][k >> 2][k & 3]);
    }
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t m = __float_as_uint(v[k]) & 0x7fffffffu;
      if (m < 0x7f800000u) most = m > most ? m : most;
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
      const uint32_t o = __shfl_xor(most, m);
      most = o > most ? o : most;
    }
    // most = 1.f * 2^q; 448 = 1.75 * 2^8
    int e = (int)(most >> 23) - 127 - 8 + ((most & 0x7fffffu) > 0x600000u);
    e = e < -120 ? -120 : e > 120 ? 120 : e;
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    const float limit = e == 120 ? 240.f : 448.f;
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t m = __float_as_uint(v[k]) & 0x7fffffffu;
      v[k] = m < 0x7f800000u ? __builtin_amdgcn_fmed3f(v[k] * inv, -limit, limit) : NAN;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k], v[4 * k + 1], 0, false);
      w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2], v[4 * k + 3], r, true);
    }
    if constexpr (TO_BF16) {
      const float s = scale_of((uint8_t)(e + 127));
      const u32x2 lo = fp8x4_to_bf16(w[0], s), hi = fp8x4_to_bf16(w[1], s);
      if (c0 < ldv)      // ldv is a multiple of 8; columns past the last are 0
        *reinterpret_cast<u32x4*>(values + (row[u] * ldv + c0) * 2) =
            u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      if (c0 < ldv)      // ldv is a multiple of 16
        *reinterpret_cast<u32x2*>(values + row[u] * ldv + c0) = u32x2{w[0], w[1]};
      if (sub == 0) scales[row[u] * lds + b[u]] = (uint8_t)(e + 127);
    }
  }
}

// 8 columns to a lane, four times: rows of bf16 or f32 that follow each other
// without a gap are written in one stream.  1M x 300 to bfloat16 in 299 us
// traced, 3.0 TB/s: where the columns are no multiple of 8, as there, a lane
// makes two stores of 8 bytes instead of one of 16.
template <int TO>
__global__ __launch_bounds__(256) void dequantize_kernel(int64_t block0, Rows x, int cols, char* out,
                                                        int64_t ldo) {
  constexpr int kEach = 4;
  const int chunks = (cols + 7) / 8;
  const int64_t first = (block0 + blockIdx.x) * (256 * kEach);
  const int64_t row0 = first / chunks;
  const int in0 = (int)(first - row0 * chunks);
  int64_t row[kEach];
  int c[kEach];
  u32x2 q[kEach];
  float s[kEach];
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const uint32_t t = in0 + threadIdx.x + 256 * u;
    const uint32_t r = t / (uint32_t)chunks;
    row[u] = row0 + r;
    c[u] = (int)(t - r * chunks) * 8;
    q[u] = u32x2{0, 0};
    if (row[u] < x.rows) {
      const char* p = x.p + row[u] * x.ld + c[u];
      if (x.align == 16 && c[u] + 8 <= cols) q[u] = *reinterpret_cast<const u32x2*>(p);
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c[u] + e < cols) q[u][e >> 2] |= (uint32_t)(uint8_t)p[e] << (8 * (e & 3));
      }
      s[u] = scale_of(x.scales[row[u] * x.lds + (c[u] >> 7)]);
    }
  }
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    if (row[u] >= x.rows) return;
    const int have = cols - c[u];
    if constexpr (TO == kBF16) {
      const u32x2 lo = fp8x4_to_bf16(q[u][0], s[u]), hi = fp8x4_to_bf16(q[u][1], s[u]);
      uint16_t* o = reinterpret_cast<uint16_t*>(out) + row[u] * ldo + c[u];
      if ((ldo & 7) == 0 && have >= 8) {
        *reinterpret_cast<u32x4*>(o) = u32x4{lo[0], lo[1], hi[0], hi[1]};
      } else if ((ldo & 3) == 0 && have >= 4) {
        *reinterpret_cast<u32x2*>(o) = lo;
        if (have >= 8) *reinterpret_cast<u32x2*>(o + 4) = hi;
        else
#pragma unroll
          for (int e = 4; e < 8; ++e)
            if (e < have) o[e] = (uint16_t)(hi[(e - 4) >> 1] >> (16 * (e & 1)));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < have) o[e] = (uint16_t)((e < 4 ? lo : hi)[(e & 3) >> 1] >> (16 * (e & 1)));
      }
    } else {
      float* o = reinterpret_cast<float*>(out) + row[u] * ldo + c[u];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(q[u][k], false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(q[u][k], true);
        const f32x4 t = {lo[0] * s[u], lo[1] * s[u], hi[0] * s[u], hi[1] * s[u]};
        if ((ldo & 3) == 0 && have >= 4 * k + 4) {
          reinterpret_cast<f32x4*>(o)[k] = t;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * k + e < have) o[4 * k + e] = t[e];
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// The tensors' device for the launches of one call.
struct OnDevice {
  int before = -1, device;
  explicit OnDevice(int d) : device(d) {
    (void)hipGetLastError();      // sticky: an older error is not ours
    HIP_CHECK(hipGetDevice(&before));
    if (before != device) HIP_CHECK(hipSetDevice(device));
  }
  ~OnDevice() {
    if (before != device) (void)hipSetDevice(before);
  }
};

static Rows make_rows(uintptr_t p, int64_t ld_elems, int64_t rows, int64_t cols, int es) {
  if (rows < 0 || rows > 0x7fffffff || cols < 1 || cols > (1 << 24) || ld_elems < 0)
    throw std::runtime_error("bad shape");
  Rows r{};
  r.p = (const char*)p;
  r.ld = ld_elems * es;
  r.rows = rows;
  r.kb = (int)cols * es;
  r.align = p % 16 == 0 && r.ld % 16 == 0 ? 16 : p % 4 == 0 && r.ld % 4 == 0 ? 4 : 1;
  return r;
}

// Workgroups of a launch.  One of 2^32 threads or more would run with what is
// left of their number in 32 bits, and report nothing.
static int grid_of(int64_t blocks, int threads) {
  if (blocks < 1 || blocks * threads > 0xffffffff) throw std::runtime_error("too large a launch");
  return (int)blocks;
}

// Launches of at most 2^31 threads, with the number of the first workgroup.
template <typename K, typename... A>
static void launch_all(K kernel, int64_t blocks, hipStream_t stream, const A&... args) {
  for (int64_t b = 0; b < blocks; b += 1 << 23)
    kernel<<<(int)std::min<int64_t>(1 << 23, blocks - b), 256, 0, stream>>>(b, args...);
}

static int score_grid(const ScoreArgs& a, int threads) {
  return grid_of((int64_t)a.tiles_n * a.splits, threads);
}

// How many workgroups of a kernel the card holds at a time.
template <typename K>
static int slots_of(K kernel, int threads, int lds) {
  int per_cu = 0, cus = 0, device = 0;
  HIP_CHECK(hipGetDevice(&device));
  HIP_CHECK(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device));
  HIP_CHECK(hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, threads, lds));
  return std::max(1, per_cu * cus);
}

// Cuts the table into at most a.splits parts of whole tiles of `rows` rows.
// With `slots` workgroups at a time, R rounds of them leave room for
// R slots / tiles_n parts; of one to four rounds the one is taken in which the
// longest workgroups end first.  A workgroup's start counts as one tile.  Parts
// of several tiles are a multiple of 8, so that all XCDs have as many.
static void cut(ScoreArgs& a, int64_t rows, int slots) {
  const int64_t tiles = (a.v_end - a.v_begin + rows - 1) / rows;
  int64_t best = 1, least = INT64_MAX;
  for (int64_t rounds = 1; rounds <= 4; ++rounds) {
    int64_t parts = std::max<int64_t>(1, rounds * slots / a.tiles_n);
    parts = std::min(std::min<int64_t>(parts, a.splits), tiles);
    if (parts > 8 && parts < tiles) parts &= ~7;
    const int64_t each = (tiles + parts - 1) / parts;
    const int64_t time = (parts * a.tiles_n + slots - 1) / slots * (each + 1);
    if (time < least) least = time, best = parts;
  }
  a.splits = (int)best;
}

// The widest rows that a wave can hold in registers, in steps of 32 columns.
constexpr int kMostResident = 10;

// Whether the kernel with resident samples takes these rows.  Its offsets
// within a tile have 32 bits.
static bool is_resident(const ScoreArgs& a, int64_t cols) {
  return cols <= 32 * kMostResident && a.w.align == 16 && a.h.align == 16 && a.w.ld < (1 << 23);
}

template <int KS, int NS, int WN, int USE, bool FP8>
static void launch_resident_k(ScoreArgs& a, hipStream_t stream) {
  constexpr auto kernel = resident_kernel<KS, NS, WN, USE, FP8>;
  static const int slots = slots_of(kernel, 256, 0);
  a.tiles_n = (int)((a.n + 16 * NS * WN - 1) / (16 * NS * WN));
  cut(a, resident_rows(KS, USE, WN, FP8), slots);
  kernel<<<score_grid(a, 256), 256, 0, stream>>>(a);
}

template <int USE, bool FP8>
static void launch_resident(ScoreArgs& a, int64_t cols, hipStream_t stream) {
  const int ks = (int)((cols + 63) / 64) * 2;
  const bool few = a.n <= 64, least = a.n <= 16;
#define CASE_KS(K)                                                              \
  if (ks == K) {                                                                \
    if constexpr (USE != kCoef)                                                 \
      if (least) return launch_resident_k<K, 1, 1, USE, FP8>(a, stream);        \
    if (few) return launch_resident_k<K, 4, 1, USE, FP8>(a, stream);            \
    return launch_resident_k<K, 4, 4, USE, FP8>(a, stream);                     \
  }
  CASE_KS(2) CASE_KS(4) CASE_KS(6) CASE_KS(8) CASE_KS(10)
#undef CASE_KS
  throw std::runtime_error("rows too wide");
}

template <int TW, int TC, int USE, int WV, int WN, int NS>
static void launch_tile_k(ScoreArgs& a, hipStream_t stream) {
  constexpr auto kernel = tile_kernel<TW, TC, USE, WV, WN, NS>;
  static const int slots = slots_of(kernel, 64 * WV * WN, 0);
  a.tiles_n = (int)((a.n + 16 * NS * WN - 1) / (16 * NS * WN));
  cut(a, 64 * WV, slots);
  kernel<<<score_grid(a, 64 * WV * WN), 64 * WV * WN, 0, stream>>>(a);
}

template <int TW, int TC, int USE>
static void launch_tile(ScoreArgs& a, hipStream_t stream) {
  for (const Rows* r : {&a.w, &a.h})
    if (r->align != 16 || r->ld >= (1 << 23)) throw std::runtime_error("rows not aligned");
  if constexpr (TW == kSplit) {
    // eight waves of 64 x 64; four of 64 x 128 read less from LDS, but leave
    // one a SIMD (20000 x 8000 x 256: 425 us, with four 483)
    launch_tile_k<TW, TC, USE, 4, 2, 4>(a, stream);
  } else {
    // few results: 64 x 64, so that more of the card's matrix units work and a
    // step takes a wave a quarter of the time
    if constexpr (TC == kF32) {
      const int64_t tiles = ((a.v_end - a.v_begin + 127) / 128) * ((a.n + 127) / 128);
      if (tiles <= 128) return launch_tile_k<TW, TC, USE, 1, 4, 1>(a, stream);
    }
    if (TW == kFP8 || a.n <= 32) return launch_tile_k<TW, TC, USE, 4, 1, 2>(a, stream);
    // 128 x 128 fills the card more evenly; bf16 is bound by LDS there, and
    // takes 256 x 256 where there are enough of them
    const int64_t rows = a.v_end - a.v_begin;
    if constexpr (TW != kFP8)
      if (TC == kF32 || ((rows + 255) / 256) * ((a.n + 255) / 256) < 256)
        return launch_tile_k<TW, TC, USE, 2, 2, 4>(a, stream);
    if constexpr (TW == kBF16) launch_tile_k<TW, TC, USE, 4, 2, 8>(a, stream);
  }
}

// LDS that the samples of the streaming kernel take; 4 KB at least, for the
// joining of the softmax.
static int64_t stream_bytes(const ScoreArgs& a, int ns, bool fp8) {
  return std::max<int64_t>(4096, (int64_t)(a.w.kb + 63) / 64 * (fp8 ? 2 : 1) * ns * 1024);
}
constexpr int64_t kMostStream = 64 << 10;

template <int TW, int TC, int NS, int USE>
static void launch_stream(ScoreArgs& a, hipStream_t stream) {
  const auto kernel = a.w.align == 16 ? stream_kernel<TW, TC, NS, USE, true>
                                      : stream_kernel<TW, TC, NS, USE, false>;
  const int lds = (int)stream_bytes(a, NS, TW == kFP8);
  a.tiles_n = (int)((a.n + 16 * NS - 1) / (16 * NS));
  cut(a, 64, slots_of(kernel, 256, lds));
  kernel<<<score_grid(a, 256), 256, lds, stream>>>(a);
}

// The kernel for scores of these samples and table rows.
template <int TW, int TC, int USE>
static void launch_any(ScoreArgs& a, int64_t cols, hipStream_t stream) {
  constexpr bool fp8 = TW == kFP8;
  if constexpr (TC == kBF16)
    if (is_resident(a, cols)) return launch_resident<USE, fp8>(a, cols, stream);
  if constexpr (USE != kCoef && TC != kSplit)
    if (a.n <= 16 && stream_bytes(a, 1, fp8) <= kMostStream)
      return launch_stream<TW, TC, 1, USE>(a, stream);
  if constexpr (fp8) throw std::runtime_error("no workspace for the scales");
  else launch_tile<TW, TC, USE>(a, stream);
}

// rows [np][dp] at `to`, see pack_kernel
static Rows pack(const Rows& r, int type, const void* targets, int targets64, int64_t ignore,
                 int64_t vocab, uintptr_t to, int64_t np, int64_t dp, hipStream_t stream) {
  const int es = type == kBF16 ? 2 : type == kF32 ? 4 : 6;
  if (to % 16 != 0) throw std::runtime_error("no workspace for rows");
  const int each = type == kSplit ? 8 : 16 / es;
  const int blocks = (int)std::min<int64_t>((np * dp / each + 255) / 256, 8192);
  if (type == kBF16) pack_kernel<kBF16><<<blocks, 256, 0, stream>>>(
      r, targets, targets64, ignore, vocab, (char*)to, np, (int)dp);
  else if (type == kSplit) split_kernel<<<blocks, 256, 0, stream>>>(
      r, targets, targets64, ignore, vocab, (char*)to, np, (int)dp);
  else pack_kernel<kF32><<<blocks, 256, 0, stream>>>(
      r, targets, targets64, ignore, vocab, (char*)to, np, (int)dp);
  Rows packed = r;
  packed.p = (const char*)to;
  packed.ld = dp * es;
  packed.rows = np;
  packed.align = 16;
  if (type == kSplit) packed.kb = (int)dp * 2;
  return packed;
}

// part: part_size pairs of float, n for each part of the table.  packed_h
// [n][dp] and packed_w [piece][dp], with dp = d rounded up to 64, or null where
// rows can be read as they lie: they start at multiples of 16 bytes and less
// than 2^23 bytes apart, or the streaming kernel takes them.
static void softmax_loss(uintptr_t h, int64_t ldh, int64_t n, uintptr_t w, int64_t ldw,
                         int64_t v, int64_t d, int type, uintptr_t targets, int targets64,
                         int64_t ignore, uintptr_t part, int64_t part_size, uintptr_t packed_h,
                         uintptr_t packed_w, int64_t piece, uintptr_t loss, uintptr_t lse,
                         int reduce, uintptr_t result, uintptr_t factor, int device,
                         uintptr_t stream_ptr) {
  const OnDevice on(device);
  hipStream_t stream = (hipStream_t)stream_ptr;
  const int es = type == kBF16 ? 2 : 4;
  const int64_t dp = type == kSplit ? (d + 31) / 32 * 32 : (d + 63) / 64 * 64;
  if (n > 0) {
    const Rows rw = make_rows(w, ldw, v, d, es), rh = make_rows(h, ldh, n, d, es);
    ScoreArgs a{};
    a.n = n;
    a.h = rh;
    a.ldp = n;
    const bool pack_w = packed_w != 0;
    if (type == kSplit && !(packed_h && packed_w))
      throw std::runtime_error("no workspace for rows");
    if (packed_h)
      a.h = pack(rh, type, nullptr, 0, 0, 0, packed_h, n, dp, stream);
    if (!pack_w) piece = v;
    const int64_t pieces = (v + piece - 1) / piece;
    int parts = 0;
    for (int64_t v0 = 0; v0 < v; v0 += piece) {
      const int64_t v1 = std::min(v, v0 + piece);
      a.w = make_rows(w + v0 * ldw * es, ldw, v1 - v0, d, es);
      if (pack_w)
        a.w = pack(a.w, type, nullptr, 0, 0, 0, packed_w, v1 - v0, dp, stream);
      a.v_begin = 0;
      a.v_end = (int)(v1 - v0);
      a.part = (float2*)part + parts * n;
      a.splits = (int)std::min<int64_t>(1 << 20, part_size / n / pieces);
      if (a.splits < 1) throw std::runtime_error("workspace too small");
      if (type == kBF16) launch_any<kBF16, kBF16, kLoss>(a, d, stream);
      else if (type == kSplit) launch_any<kSplit, kSplit, kLoss>(a, d, stream);
      else launch_any<kF32, kF32, kLoss>(a, d, stream);
      parts += a.splits;
    }
    launch_all(type == kBF16 ? loss_join_kernel<kBF16> : loss_join_kernel<kF32>, (n + 3) / 4,
               stream, rw, rh, (const float2*)part, parts, n, (const void*)targets, targets64,
               ignore, (float*)loss, (float*)lse);
  }
  if (reduce)      // 1: sum, 2: mean
    loss_reduce_kernel<<<1, 1024, 0, stream>>>((const float*)loss, (const void*)targets,
                                               targets64, ignore, n, reduce == 2, (float*)result,
                                               (float*)factor);
  HIP_CHECK(hipGetLastError());
}

static void launch_sum_parts(const float* part, int splits, int64_t rows, int64_t ldp, int64_t d,
                             const float* const (&scale)[2], int is_bf16, char* out,
                             hipStream_t stream) {
  auto go = [&](auto kernel, int each) {
    launch_all(kernel, (rows * d + each - 1) / each, stream, part, splits, rows, ldp, (int)d,
               scale[0], scale[1], out);
  };
  if (splits >= 16)
    is_bf16 ? go(sum_parts_kernel<kBF16, 16>, 16) : go(sum_parts_kernel<kF32, 16>, 16);
  else
    is_bf16 ? go(sum_parts_kernel<kBF16, 4>, 64) : go(sum_parts_kernel<kF32, 4>, 64);
}

// The form of grad_kernel for a result of r x d with k terms.
struct GradForm {
  int rows;       // of a workgroup; 0: the form for a short k, of 256 rows
  int nd;         // 16 columns times this per wave
  int tiles_d;
  int slots;      // workgroups that the card holds at a time
};

static GradForm grad_form(int type, bool dw, int64_t r, int64_t k, int d) {
  GradForm f{256, 0, 0, 256};
  int wd = 2, most = 10, step = 2;    // waves along d, blocks of 16 columns a wave
  if (type == kSplit) most = 4;       // two steps of 256 x 128 fit LDS
  else if (!dw && r <= 32) f.rows = 32, wd = 8, most = 3, step = 1, f.slots = 512;
  else if (!dw && r <= 128) f.rows = 128, wd = 4, most = 5, step = 1, f.slots = 512;
  else if (dw && k <= 128) f.rows = 0, most = 4, f.slots = 768;
  if (f.rows == 0 || (f.rows == 256 && type != kF32)) {
    // bound by LDS or by what is written: the fewest tiles
    f.tiles_d = (d + 16 * wd * most - 1) / (16 * wd * most);
    f.nd = ((d + f.tiles_d - 1) / f.tiles_d + 63) / 64 * 2;
    if ((f.rows == 0 || type == kSplit) && f.nd > 2) f.nd = 4;
  } else {
    // the fewest columns past d, and of those the most tiles, which fill the
    // card more evenly; but no narrow ones where wide ones do
    int least = INT32_MAX;
    for (int n = most; n >= step; n -= step) {
      const int t = (d + 16 * n * wd - 1) / (16 * n * wd);
      if (t * n < least || (t * n == least && n > 2)) least = t * n, f.nd = n, f.tiles_d = t;
    }
  }
  if (f.rows != 256) return f;
  // Little work: narrow tiles rather than many parts of the sums.  Times of both
  // gradients, d = 300, with wide and with narrow tiles (us): bf16 1000 x 8000
  // 121 and 75, 3000 x 2000 119 and 80, 8000 x 8000 241 and 298; float32 1000 x
  // 2000 102 and 94, 8000 x 2000 262 and 278
  if ((double)r * k * d <= (type == kBF16 ? 4e9 : 1e9))
    while (f.nd > 2 && (r + 255) / 256 * f.tiles_d < 128)
      f.nd -= 2, f.tiles_d = (d + 32 * f.nd - 1) / (32 * f.nd);
  if (type == kF32 && f.nd <= 4) f.slots = 512;
  return f;
}

// Parts of k for `tiles` results on `slots` places: the fewest that fill nine
// tenths of what any number up to `most` fills.
static int grad_parts(int64_t tiles, int slots, int64_t most) {
  if (tiles >= 2 * slots) return 1;
  most = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(most, 512),
                                                (2 * slots + tiles - 1) / tiles));
  auto full = [&](int64_t s) {
    return (double)(tiles * s) / (double)((tiles * s + slots - 1) / slots * slots);
  };
  double best = 0;
  for (int64_t s = 1; s <= most; ++s) best = std::max(best, full(s));
  int64_t s = 1;
  while (full(s) < 0.9 * best) ++s;
  return (int)s;
}

// (parts of the vocabulary's pieces for dh, parts of the samples for dw)
static std::pair<int, int> softmax_plan(int64_t n, int64_t chunk, int64_t d, int type) {
  const GradForm h = grad_form(type, false, n, chunk, (int)d);
  const GradForm w = grad_form(type, true, chunk, n, (int)d);
  const int rows_w = w.rows ? w.rows : 256;
  const int64_t tiles_h = (n + h.rows - 1) / h.rows * h.tiles_d;
  const int64_t tiles_w = (chunk + rows_w - 1) / rows_w * w.tiles_d;
  // parts of dw are as large as dw: only where half of the card would idle
  return {grad_parts(tiles_h, h.slots, (chunk + 63) / 64),
          2 * tiles_w <= w.slots ? grad_parts(tiles_w, w.slots, (n + 255) / 256) : 1};
}

template <int T, bool DW, int ND, int WR, int J, int kAhead>
static void launch_grad_k(GradArgs& b, hipStream_t stream) {
  b.tiles_r = (int)((b.r + 16 * J * WR - 1) / (16 * J * WR));
  const int64_t tiles = (int64_t)b.tiles_d * b.tiles_r;
  const int blocks = grid_of(tiles * b.splits, 512);
  grad_kernel<T, DW, ND, WR, J, kAhead><<<blocks, 512, 0, stream>>>(b);
}

template <int T, bool DW>
static void launch_grad(GradArgs b, hipStream_t stream) {
  const GradForm f = grad_form(T, DW, b.r, b.k, b.d);
  b.tiles_d = f.tiles_d;
#define CASE_ND(R, N, WR, J, A) \
  if (f.rows == R && f.nd == N) return launch_grad_k<T, DW, N, WR, J, A>(b, stream);
  if constexpr (T == kSplit) {
    CASE_ND(256, 2, 4, 4, 1) CASE_ND(256, 4, 4, 4, 1)
  } else if constexpr (DW) {
    CASE_ND(0, 2, 4, 4, 1) CASE_ND(0, 4, 4, 4, 1)
  } else {
    CASE_ND(32, 1, 1, 2, 3) CASE_ND(32, 2, 1, 2, 3) CASE_ND(32, 3, 1, 2, 3)
    CASE_ND(128, 1, 2, 4, 3) CASE_ND(128, 2, 2, 4, 3) CASE_ND(128, 3, 2, 4, 3)
    CASE_ND(128, 4, 2, 4, 3) CASE_ND(128, 5, 2, 4, 3)
  }
  if constexpr (T != kSplit) {
    constexpr int kAhead = T == kF32 ? 2 : 3;
    CASE_ND(256, 2, 4, 4, kAhead) CASE_ND(256, 4, 4, 4, kAhead) CASE_ND(256, 6, 4, 4, kAhead)
    CASE_ND(256, 8, 4, 4, kAhead) CASE_ND(256, 10, 4, 4, kAhead)
  }
#undef CASE_ND
  throw std::runtime_error("no kernel for these columns");
}

// packed: [np][dp] elements with np = n rounded up to 32, dp = d rounded up to
// 64; packed_w: [chunk][dp], or null where rows of w start at multiples of 16
// bytes and less than 2^23 bytes apart; coef: [np][chunk] elements; part:
// [splits][n][ldp] floats; part_w: [splits_w][chunk][ldp] where splits_w > 1
static void softmax_grad(uintptr_t h, int64_t ldh, int64_t n, uintptr_t w, int64_t ldw,
                         int64_t v, int64_t d, int type, uintptr_t targets, int targets64,
                         int64_t ignore, uintptr_t lse, uintptr_t grad, int grad_step,
                         uintptr_t weight, uintptr_t packed, uintptr_t packed_w, int64_t chunk,
                         uintptr_t coef, int splits, uintptr_t part, int splits_w,
                         uintptr_t part_w, int64_t ldp, uintptr_t dh, uintptr_t dw, int device,
                         uintptr_t stream_ptr) {
  const OnDevice on(device);
  hipStream_t stream = (hipStream_t)stream_ptr;
  const bool is_bf16 = type == kBF16;
  const int es = is_bf16 ? 2 : 4;
  if (chunk % 256 != 0 || ldp % 4 != 0 || coef % 16 != 0)
    throw std::runtime_error("bad workspace shape");
  if (n == 0) throw std::runtime_error("no rows");
  const int64_t np = (n + 31) / 32 * 32;
  const int64_t dp = type == kSplit ? (d + 31) / 32 * 32 : (d + 63) / 64 * 64;
  const Rows rw = make_rows(w, ldw, v, d, es);
  const Rows rh = pack(make_rows(h, ldh, n, d, es), type, (const void*)targets, targets64,
                       ignore, v, packed, np, dp, stream);
  const bool pack_w = packed_w != 0;
  if (type == kSplit && !pack_w) throw std::runtime_error("no workspace for rows");
  // One gradient for all samples stays out of the coefficients: in bf16 it
  // would round all of them by the same 2^-9 or less.
  const float* const scale[2] = {grad_step ? nullptr : (const float*)grad,
                                 (const float*)weight};
  for (int64_t v0 = 0; v0 < v; v0 += chunk) {
    const int64_t v1 = std::min(v, v0 + chunk);
    // the table's rows from v0 on; v_begin and the targets count from row 0
    Rows piece = make_rows(w + v0 * ldw * es, ldw, v1 - v0, d, es);
    if (pack_w)
      piece = pack(piece, type, nullptr, 0, 0, 0, packed_w, v1 - v0, dp, stream);
    ScoreArgs a{};
    a.w = piece;
    a.w.p -= v0 * a.w.ld;
    a.w.rows = v1;
    a.h = rh;
    a.n = n;
    a.splits = 1 << 20;
    a.v_begin = (int)v0;
    a.v_end = (int)v1;
    a.vocab = v;
    a.targets = (const void*)targets;
    a.targets64 = targets64;
    a.ignore = ignore;
    a.lse = (const float*)lse;
    a.grad = grad_step ? (const float*)grad : nullptr;
    a.coef = (char*)coef;
    a.coef_rows = np;
    a.ldc = chunk;
    if (is_bf16) launch_any<kBF16, kBF16, kCoef>(a, d, stream);
    else if (type == kSplit) launch_any<kSplit, kSplit, kCoef>(a, d, stream);
    else launch_any<kF32, kF32, kCoef>(a, d, stream);
    GradArgs b{};
    b.coef = (const char*)coef;
    b.ldc = chunk;
    b.d = (int)d;
    b.ldp = ldp;
    b.scale[0] = scale[0];
    b.scale[1] = scale[1];
    if (dh) {
      b.x = piece;
      b.r = n;
      b.k = v1 - v0;
      b.splits = splits;
      b.part = (float*)part;
      b.add = v0 > 0;
      if (is_bf16) launch_grad<kBF16, false>(b, stream);
      else if (type == kSplit) launch_grad<kSplit, false>(b, stream);
      else launch_grad<kF32, false>(b, stream);
    }
    if (dw) {
      b.x = rh;
      b.r = v1 - v0;
      b.k = n;
      b.splits = splits_w;
      b.part = splits_w > 1 ? (float*)part_w : nullptr;
      b.add = 0;
      b.out = (char*)dw + v0 * d * es;
      b.ldo = d;
      if (is_bf16) launch_grad<kBF16, true>(b, stream);
      else if (type == kSplit) launch_grad<kSplit, true>(b, stream);
      else launch_grad<kF32, true>(b, stream);
      if (splits_w > 1)
        launch_sum_parts(b.part, splits_w, v1 - v0, ldp, d, scale, is_bf16, b.out, stream);
    }
  }
  if (dh)
    launch_sum_parts((const float*)part, splits, n, ldp, d, scale, is_bf16, (char*)dh, stream);
  HIP_CHECK(hipGetLastError());
}

// to_bf16: values are bf16 rows, no scales are written
static void quantize_rows(uintptr_t x, int64_t ldx, int64_t rows, int64_t cols, int is_bf16,
                          uintptr_t values, int64_t ldv, uintptr_t scales, int64_t lds,
                          int to_bf16, int device, uintptr_t stream_ptr) {
  const OnDevice on(device);
  if (rows == 0) return;
  hipStream_t stream = (hipStream_t)stream_ptr;
  if (ldv % (to_bf16 ? 8 : 16) != 0 || ldv < cols || values % 16 != 0)
    throw std::runtime_error("bad layout of the values");
  const Rows r = make_rows(x, ldx, rows, cols, is_bf16 ? 2 : 4);
  const int blocks = (int)((cols + 127) / 128);
  auto go = [&](auto kernel) {
    launch_all(kernel, (rows * blocks + 63) / 64, stream, r, blocks, (char*)values, ldv,
               (uint8_t*)scales, lds);
  };
  if (is_bf16) to_bf16 ? go(quantize_kernel<kBF16, true>) : go(quantize_kernel<kBF16, false>);
  else to_bf16 ? go(quantize_kernel<kF32, true>) : go(quantize_kernel<kF32, false>);
  HIP_CHECK(hipGetLastError());
}

static Rows make_fp8(uintptr_t values, int64_t ldv, uintptr_t scales, int64_t lds, int64_t rows,
                     int64_t cols) {
  Rows r = make_rows(values, ldv, rows, cols, 1);
  r.scales = (const uint8_t*)scales;
  r.lds = lds;
  return r;
}

static void dequantize_rows(uintptr_t values, int64_t ldv, uintptr_t scales, int64_t lds,
                            int64_t rows, int64_t cols, int is_bf16, uintptr_t out, int64_t ldo,
                            int device, uintptr_t stream_ptr) {
  const OnDevice on(device);
  if (rows == 0) return;
  hipStream_t stream = (hipStream_t)stream_ptr;
  if (out % 16 != 0) throw std::runtime_error("bad layout of the output");
  const Rows r = make_fp8(values, ldv, scales, lds, rows, cols);
  launch_all(is_bf16 ? dequantize_kernel<kBF16> : dequantize_kernel<kF32>,
             (rows * ((cols + 7) / 8) + 1023) / 1024, stream, r, (int)cols, (char*)out, ldo);
  HIP_CHECK(hipGetLastError());
}

// The scales of 8-bit rows by block of columns, as the tile kernel takes them: a
// hundredth of the table's bytes.
__global__ __launch_bounds__(256) void turn_scales_kernel(
    const uint8_t* scales, int64_t lds, int64_t rows, int blocks, uint8_t* out, int64_t ldo) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int b = 0; b < blocks; ++b)
    out[b * ldo + r] = scales[min(r, rows - 1) * lds + b];
}

// a: bf16 rows [m][k]; b: 8-bit rows [n][k]; out [m][n].  Where k > 320:
//   m <= 160, but not with m <= 16 and k <= 2048: turned, a byte for every
//   block of 128 columns and row, rows rounded up to 256
//   m > 160: wide, bf16 [piece][k rounded up to 64].  Converting 8-bit rows in
//   the product costs each workgroup registers that the product wants (1023 x
//   150001 x 1024: 0.73 ms; converted first, a piece at a time, 0.55 ms)
static void matmul_rows(uintptr_t a_ptr, int64_t lda, int64_t m, uintptr_t values, int64_t ldv,
                        uintptr_t scales, int64_t lds, int64_t n, int64_t k, uintptr_t col_scale,
                        uintptr_t out, int out_bf16, uintptr_t turned, uintptr_t wide,
                        int64_t piece, int device, uintptr_t stream_ptr) {
  const OnDevice on(device);
  if (m == 0 || n == 0) return;
  hipStream_t stream = (hipStream_t)stream_ptr;
  if (out % 16 != 0) throw std::runtime_error("bad layout of the output");
  ScoreArgs a{};
  a.w = make_fp8(values, ldv, scales, lds, n, k);
  a.h = make_rows(a_ptr, lda, m, k, 2);
  a.n = m;
  a.splits = 1 << 20;
  a.v_begin = 0;
  a.v_end = (int)n;
  a.col_scale = (const float*)col_scale;
  a.out = (char*)out;
  a.ldo = n;
  a.out_bf16 = out_bf16;
  if (wide) {
    const int64_t dp = (k + 63) / 64 * 64;
    const Rows table = a.w;
    for (int64_t v0 = 0; v0 < n; v0 += piece) {
      const int64_t rows = std::min(piece, n - v0);
      Rows part = table;
      part.p += v0 * part.ld;
      part.scales += v0 * part.lds;
      part.rows = rows;
      launch_all(dequantize_kernel<kBF16>, (rows * ((k + 7) / 8) + 1023) / 1024, stream, part,
                 (int)k, (char*)wide, dp);
      a.w = make_rows(wide, dp, rows, k, 2);
      a.v_end = (int)rows;
      a.splits = 1 << 20;
      a.col_scale = col_scale ? (const float*)col_scale + v0 : nullptr;
      a.out = (char*)out + v0 * (out_bf16 ? 2 : 4);
      launch_tile<kBF16, kBF16, kStore>(a, stream);
    }
  } else if (turned) {
    const int64_t ldo = (n + 255) / 256 * 256;
    turn_scales_kernel<<<grid_of(ldo / 256, 256), 256, 0, stream>>>(
        a.w.scales, a.w.lds, n, (int)((k + 127) / 128), (uint8_t*)turned, ldo);
    a.w.scales = (const uint8_t*)turned;
    a.w.lds = ldo;
    launch_tile<kFP8, kBF16, kStore>(a, stream);
  } else {
    launch_any<kFP8, kBF16, kStore>(a, k, stream);
  }
  HIP_CHECK(hipGetLastError());
}

PYBIND11_MODULE(_vocab_native, m) {
  m.doc() = "MI355X (gfx950) kernels over the whole vocabulary";
  m.def("softmax_loss", &softmax_loss);
  m.def("softmax_plan", &softmax_plan);
  m.def("softmax_grad", &softmax_grad);
  m.def("quantize_rows", &quantize_rows);
  m.def("dequantize_rows", &dequantize_rows);
  m.def("matmul_rows", &matmul_rows);
}
