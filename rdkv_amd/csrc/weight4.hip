// 4-bit weights with group scales: the quantizer, the layout and the products that read it.
//
// The projections of a decode step are products of one activation row (of a few, in a batch) with
// weights that are read once a step: gemv.hip streams them as fp16 / bf16, this file as 4-bit codes,
// a quarter of the bytes (4.25 bits a weight at groups of 128).
//
//   y[m, n] = sum_k x[m, k] * (q[n, k] - z[n, g(k)]) * s[n, g(k)] (+ bias[n])
//
// Layout.  A tile is 16 rows x 128 columns, 1 KiB of codes, what one wavefront reads with one
// 16-byte load per lane: lane 16 c + n holds row n, its dword d the columns 32 d + 8 c + j, j < 8,
// which is a lane's share of the 32 x 16 operand of v_mfma_f32_16x16x32.  Field j sits at bit
// 4 (j / 2) + 16 (j & 1), so a shift and a mask leave two 16-bit operands in a register.  Tiles of 16
// rows follow each other along K.  A scale word per row and group: fp32 with the zero point in its
// four lowest mantissa bits (20 significant bits are left to the scale: fp16 and bf16 scales are
// held exactly, at the whole fp32 range), [row tile][column tile][group][16 rows].  Rows and columns
// behind the matrix have zero codes and zero scale words.
//
// Nothing is dequantized in the products.  fp16: a masked code is the bit pattern of the subnormal
// q * 2^-24, which the matrix cores keep; bf16: or-ed below an exponent it is 16 + q, exactly.  Each
// group's products are summed in fp32 by the matrix cores, and the zero point (and the 16) comes
// off once per group through the sum X of the group's activations:
//   y += s * (D * 2^24 - z * X)      fp16            y += s * (D - (16 + z) * X)      bf16
// The factor that this cancels is at most (15 + 16) / 7.5 of the sum itself, in fp32.
#include "rdkv_common.h"
#include "rope_device.h"

namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = 1024;
constexpr float kSmallestScale = 0x1p-120f;      // below it a group counts as all zeros (its scale stays an ordinary number)

// Sixteen bytes at any address of a 16-bit element.
struct __attribute__((packed, aligned(2))) Loose { u32x4 v; };
__device__ __forceinline__ u32x4 load_loose(const uint16_t *p) { return reinterpret_cast<const Loose *>(p)->v; }
__device__ __forceinline__ u32x4 load_stream(const u32x4 *p) { return __builtin_nontemporal_load(p); }

template <int dtype>
__device__ __forceinline__ float load16(uint16_t bits) {
  return dtype == RDKV_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, bits) : __uint_as_float((uint32_t)bits << 16);
}
template <int dtype>
__device__ __forceinline__ uint16_t bits16(float v) {
  return dtype == RDKV_DTYPE_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : rdkv_float_to_bf16_bits(v);
}
__device__ __forceinline__ uint32_t scale_word(float s, uint32_t zero) {
  // 20 significant bits, rounded half up in magnitude; an infinity stays one, a NaN a NaN
  const uint32_t bits = __float_as_uint(s);
  const bool ordinary = (bits & 0x7f800000u) != 0x7f800000u;
  return ((ordinary ? bits + 8u : bits) & ~15u) | zero;
}
__device__ __forceinline__ float word_scale(uint32_t w) { return __uint_as_float(w & ~15u); }
__device__ __forceinline__ uint32_t word_zero(uint32_t w) { return w & 15u; }
__device__ __forceinline__ int field_shift(int j) { return 4 * (j >> 1) + 16 * (j & 1); }

// ---- quantize / pack / dequantize: a wavefront per tile ------------------------------------------

struct TileAt { int64_t tile, row; int lane, c, col0; };
__device__ __forceinline__ TileAt tile_at(uint32_t n_tiles_k) {
  TileAt t;
  t.lane = threadIdx.x & 63;
  t.c = t.lane >> 4;
  const uint32_t tile = blockIdx.x * 4u + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);     // below 2^26
  t.tile = tile;
  t.row = (int64_t)(tile / n_tiles_k) * kTileRows + (t.lane & 15);
  t.col0 = (int)(tile % n_tiles_k * kTileCols);        // (below K, which is at most 2^31 - 256)
  return t;
}

// The largest of the four lanes 16 c + n that hold a row's pieces, in each of them.
__device__ __forceinline__ float max_of_row(float v) {
  typedef unsigned uint2_t __attribute__((ext_vector_type(2)));
  uint2_t both = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
  both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// Eight elements without the first n, zeros behind the others.
__device__ __forceinline__ u32x4 drop_front(u32x4 v, int n) {
  if (n <= 0) return v;
  if (n & 4) v = u32x4{v[2], v[3], 0, 0};
  if (n & 2) v = u32x4{v[1], v[2], v[3], 0};
  if (n & 1) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
  return n >= 8 ? u32x4{0, 0, 0, 0} : v;
}
// A mask of the first n of a dword's eight fields: an even field j lies at bit 2 j, an odd one at 2 (j - 1) + 16.
__device__ __forceinline__ uint32_t fields_below(int n) {
  if (n <= 0) return 0u;
  if (n >= 8) return ~0u;
  return ((1u << (4 * ((n + 1) >> 1))) - 1) | ((1u << (4 * (n >> 1))) - 1) << 16;
}

// The value range of a group takes in zero, so that a zero weight stays zero and the zero point lies in
// 0 .. 15; quotients are the correctly rounded ones and nothing is contracted, so the codes are those of the
// expressions rint(w / s) + z.  A group that holds a NaN or an infinity has scale NaN: every product with it is NaN.
// One pass: 2 bytes read and 0.53 written for a weight (groups of 128).  28672 x 4096 fp16: 53 us, 5.6 TB/s; with a division
// for each weight that might lie between two codes it took 76.
template <int dtype, int GPC>
__global__ void __launch_bounds__(256)
w4_quantize_kernel(const uint16_t *__restrict__ W, int64_t w_stride_row, int N, int K, uint32_t n_tiles_k,
                   uint32_t n_tiles, u32x4 *__restrict__ codes, uint32_t *__restrict__ scales) {
#pragma clang fp contract(off)
  const TileAt t = tile_at(n_tiles_k);
  if (t.tile >= n_tiles) return;
  // (Read in the layout's lanes, 64 bytes of a row at a time: rows of 256 bytes turned through LDS took 59 us where this
  // takes 53.)
  u32x4 v[4];
  const uint16_t *src = W + min(t.row, (int64_t)N - 1) * w_stride_row;      // (rows behind the matrix: not stored)
  if (K >= 8) {
#pragma unroll
    for (int d = 0; d < 4; ++d) v[d] = load_loose(src + min(t.col0 + 32 * d + 8 * t.c, K - 8));
    if (t.col0 + kTileCols > K) {        // pieces over the end were read from column K - 8 on
#pragma unroll
      for (int d = 0; d < 4; ++d) v[d] = drop_front(v[d], t.col0 + 32 * d + 8 * t.c - (K - 8));
    }
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 32 * d + 8 * t.c + 2 * i;
        v[d][i] = (k < K ? src[k] : 0u) | (k + 1 < K ? (uint32_t)src[k + 1] << 16 : 0u);
      }
  }
  constexpr int DPG = 4 / GPC;           // dwords of a lane per group
  constexpr uint16_t kInfinite = dtype == RDKV_DTYPE_F16 ? 0x7c00 : 0x7f80;
  auto weight = [&](int d, int j) __attribute__((always_inline)) {
    const uint32_t pair = v[d][j >> 1];
    return load16<dtype>((uint16_t)(pair >> (16 * (j & 1))));
  };
  u32x4 out;
#pragma unroll
  for (int g = 0; g < GPC; ++g) {
    float lo = 0.0f, hi = 0.0f;
    u16x2 size = {0, 0};
#pragma unroll
    for (int d = g * DPG; d < (g + 1) * DPG; ++d) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, weight(d, j));
        hi = fmaxf(hi, weight(d, j));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t pair = v[d][i] & 0x7fff7fffu;
        size = __builtin_elementwise_max(size, __builtin_bit_cast(u16x2, pair));
      }
    }
    if (size[0] >= kInfinite || size[1] >= kInfinite) hi = INFINITY;
    hi = max_of_row(hi);
    lo = -max_of_row(-lo);
    // (hi - lo) / 15 and 1 / s by their remainders too: the first correctly rounded, the second within an ulp
    const float range = hi - lo, part = range * (1.0f / 15.0f);
    float s = word_scale(scale_word(__builtin_fmaf(__builtin_fmaf(-part, 15.0f, range), 1.0f / 15.0f, part), 0));
    if (!(s < INFINITY)) s = __builtin_nanf("");
    if (s < kSmallestScale) s = 1.0f;
    // Correctly rounded quotients without a division for each: q = v * (1 / s) is within a few ulp, its remainder v - q s is
    // exact, and q + (v - q s) (1 / s) before its rounding is within 2^-22 ulp of v / s, which, s having 20 bits, stays
    // 2^-21 ulp away from the middle of two fp32 numbers.  (Not where the remainder could be subnormal.)
    const float about = __builtin_amdgcn_rcpf(s), inv = __builtin_fmaf(__builtin_fmaf(-s, about, 1.0f), about, about);
    auto quotient = [&](float w) __attribute__((always_inline)) {
      const float q = w * inv;
      return __builtin_fmaf(__builtin_fmaf(-q, s, w), inv, q);
    };
    const bool tiny = dtype == RDKV_DTYPE_BF16 && s < 0x1p-60f;
    // Added to 1.5 * 2^23, a quotient is rounded to a whole number in the low bits, ties to even; after the clamp the bits of
    // eight of them are shifted and summed, and what they hold beside the codes is a constant.  (The clamp takes a NaN to
    // the lower end: a group whose scale is NaN has zero codes.)
    constexpr float kWhole = 0x1.8p23f;
    const float z = fminf(fmaxf(rintf(tiny ? -lo / s : quotient(-lo)), 0.0f), 15.0f);
    const float from = kWhole - z, to = from + 15.0f;
    const uint32_t beside = __float_as_uint(from) * 0x11111111u;
#pragma unroll
    for (int d = g * DPG; d < (g + 1) * DPG; ++d) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) w += __float_as_uint(__builtin_amdgcn_fmed3f(quotient(weight(d, j)) + kWhole, from, to)) << field_shift(j);
      out[d] = w - beside;
    }
    if (tiny) {
#pragma unroll
      for (int d = g * DPG; d < (g + 1) * DPG; ++d) {
        uint32_t w = 0;
        for (int j = 0; j < 8; ++j) w |= (uint32_t)fminf(fmaxf(rintf(weight(d, j) / s) + z, 0.0f), 15.0f) << field_shift(j);
        out[d] = w;
      }
    }
    if (t.c == 0) {
      const bool there = t.row < N && (int64_t)t.col0 + g * DPG * 32 < K;
      scales[(t.tile * GPC + g) * 16 + (t.lane & 15)] = there ? scale_word(s, (uint32_t)z) : 0u;
    }
  }
  if (t.col0 + kTileCols > K) {
#pragma unroll
    for (int d = 0; d < 4; ++d) out[d] &= fields_below(K - t.col0 - 32 * d - 8 * t.c);
  }
  if (t.row >= N) out = u32x4{0, 0, 0, 0};
  codes[t.tile * 64 + t.lane] = out;
}

// Codes, scales and zero points of a matrix quantized elsewhere, into the layout.
template <int GPC>
__global__ void __launch_bounds__(256)
w4_pack_kernel(const uint8_t *__restrict__ src, int64_t src_stride_row, const void *__restrict__ scale, int scale_dtype,
               int64_t scale_stride_row, const uint8_t *__restrict__ zero, int64_t zero_stride_row, int N, int K,
               uint32_t n_tiles_k, uint32_t n_tiles, u32x4 *__restrict__ codes, uint32_t *__restrict__ scales) {
  const TileAt t = tile_at(n_tiles_k);
  if (t.tile >= n_tiles) return;
  u32x4 out;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = t.col0 + 32 * d + 8 * t.c + j;
      const uint32_t q = t.row < N && k < K ? src[t.row * src_stride_row + k] & 15u : 0u;
      w |= q << field_shift(j);
    }
    out[d] = w;
  }
  codes[t.tile * 64 + t.lane] = out;
  if (t.c < GPC) {                       // lane 16 g + n: group g of row n
    const int group = t.col0 / (kTileCols / GPC) + t.c;
    uint32_t word = 0;
    if (t.row < N && group * (int64_t)(kTileCols / GPC) < K) {
      const float s = rdkv_load_as_float(scale, scale_dtype, t.row * scale_stride_row + group);
      word = scale_word(s, zero ? zero[t.row * zero_stride_row + group] & 15u : 8u);
    }
    scales[(t.tile * GPC + t.c) * 16 + (t.lane & 15)] = word;
  }
}

template <int dtype, int GPC>
__global__ void __launch_bounds__(256)
w4_dequant_kernel(const u32x4 *__restrict__ codes, const uint32_t *__restrict__ scales, int N, int K,
                  uint32_t n_tiles_k, uint32_t n_tiles, uint16_t *__restrict__ out, int64_t out_stride_row) {
  const TileAt t = tile_at(n_tiles_k);
  if (t.tile >= n_tiles) return;
  // The pieces p of the rows r change lanes through LDS, at slot 16 r + (p ^ r) of the wavefront's own, so that sixteen lanes
  // write a row's 256 bytes (28672 x 4096 bf16: 51 us, 5.8 TB/s; 82 with 64 bytes of sixteen rows at a time).
  __shared__ u32x4 s_tile[4][256];
  u32x4 *mine = s_tile[threadIdx.x >> 6];
  const int n = t.lane & 15;
  const u32x4 q = load_stream(codes + t.tile * 64 + t.lane);
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t word = scales[(t.tile * GPC + d * GPC / 4) * 16 + n];
    const float s = word_scale(word), z = (float)word_zero(word);
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (a 5-bit integer times 20 bits: exact in fp32, rounded once to the type)
      const float lo = ((float)((q[d] >> (4 * i)) & 15u) - z) * s, hi = ((float)((q[d] >> (4 * i + 16)) & 15u) - z) * s;
      w[i] = bits16<dtype>(lo) | (uint32_t)bits16<dtype>(hi) << 16;
    }
    mine[16 * n + ((4 * d + t.c) ^ n)] = w;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * i + t.c, k = t.col0 + 8 * n;
    const int64_t row = t.row - n + r;
    const u32x4 w = mine[16 * r + (n ^ r)];
    if (row >= N) continue;
    uint16_t *dst = out + row * out_stride_row + k;
    if (k + 8 <= K) {
      reinterpret_cast<Loose *>(dst)->v = w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < K) dst[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// ---- products --------------------------------------------------------------------------------------

// Two operands from one dword of codes: register r of the four that a lane gives the matrix cores.
template <int dtype>
__device__ __forceinline__ u32x4 operand(uint32_t w) {
  u32x4 b;
  if (dtype == RDKV_DTYPE_F16) {
#pragma unroll
    for (int r = 0; r < 4; ++r) b[r] = (w >> (4 * r)) & 0x000f000fu;
  } else {
    uint32_t fields = 0x00780078u;
    asm("" : "+v"(fields));              // (in a vector register: one instruction takes the mask and the exponent)
    b[0] = ((w << 3) & fields) | 0x41804180u;
#pragma unroll
    for (int r = 1; r < 4; ++r) b[r] = ((w >> (4 * r - 3)) & fields) | 0x41804180u;
  }
  return b;
}
template <int dtype>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if (dtype == RDKV_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// One group's sum D and activation sum X -> its contribution, scale word w.
template <int dtype>
__device__ __forceinline__ float add_group(uint32_t w, float D, float X, float acc) {
  const float z = (float)word_zero(w), s = word_scale(w);
  if (dtype == RDKV_DTYPE_F16) return fmaf(s * 0x1p24f, fmaf(-z * 0x1p-24f, X, D), acc);
  return fmaf(s, fmaf(-(z + 16.0f), X, D), acc);
}
template <int dtype>
__device__ __forceinline__ float round16(float v) {
  return dtype == RDKV_DTYPE_F16 ? (float)(_Float16)v : __uint_as_float((uint32_t)rdkv_float_to_bf16_bits(v) << 16);
}

// How one activation row reaches LDS, as in gemv.hip.
enum { kPlain = 0, kFromF32 = 1, kNorm = 2, kSilu = 3 };
struct RowSource {
  const void *a, *b, *c;
  float eps;
  void *residual_out;
};

// g / (1 + exp(-g)) with the hardware's exponential and reciprocal (an ulp each, 2^-17 in all at the steepest: a 64th of
// the rounding to 16 bits that follows).  Every workgroup stages the whole row: with the library's exponential and the
// correctly rounded division the staging of 14336 columns took 4 of 12 us.
__device__ __forceinline__ float silu(float g) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f));
}

// Eight elements of a 16-bit row from element k on; what lies behind the row is zero.
template <int dtype>
__device__ __forceinline__ void row8(const void *row, int k, int K, float (&f)[8]) {
  const uint16_t *p = reinterpret_cast<const uint16_t *>(row);
  if (k + 8 <= K) {
    const u32x4 w = load_loose(p + k);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = load16<dtype>((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = k + j < K ? load16<dtype>(p[k + j]) : 0.0f;
  }
}
template <int dtype>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = bits16<dtype>(f[2 * i]) | ((uint32_t)bits16<dtype>(f[2 * i + 1]) << 16);
  return w;
}

// One activation row.  A workgroup takes row tiles in turn and its wavefronts share a tile's columns (runs of
// column tiles); the wavefronts' sums are kept in LDS and added in their order, kKept tiles at a time, so that between
// them no wavefront waits for another.  Bound by HBM where there are rows enough: 128256 x 4096 bf16 46 us, 6.0 TB/s; 28672 x
// 4096 13 us; 4096 x 4096 4 us, a launch, the staging and one round of loads.
constexpr int kKept = 16;
template <int dtype, int MODE, int GPC, int WAVES, int U>
__global__ void __launch_bounds__(64 * WAVES)
w4_row_kernel(const u32x4 *__restrict__ codes, const uint32_t *__restrict__ scales, RowSource src,
              const uint16_t *__restrict__ bias, int N, int K, int n_tiles_n, int n_tiles_k, uint16_t *__restrict__ y) {
  extern __shared__ u32x4 lds[];       // the row (16 pieces of 8 per column tile), then a sum per group
  __shared__ float s_red[kKept][WAVES][16];
  __shared__ float s_part[WAVES];
  u32x4 *xs = lds;
  float *sums = reinterpret_cast<float *>(lds + n_tiles_k * 16);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, n = lane & 15;
  const int pieces = n_tiles_k * 16;
  constexpr int PPG = 16 / GPC;        // pieces per group
  // A wavefront walks its run of every row tile in steps of U column tiles; the loads of the next step are issued
  // before the current one is consumed, those of the first before the row is staged.
  struct Cur { int tn, step; };
  struct Piece { u32x4 q[U]; uint32_t w[U][GPC]; };
  // (every wavefront makes the same number of steps a tile: the barriers are met by all together)
  const int run = (n_tiles_k + WAVES - 1) / WAVES, steps = (run + U - 1) / U;
  const int k_begin = min(wave * run, n_tiles_k), k_end = min(k_begin + run, n_tiles_k);
  auto next = [&](Cur c) __attribute__((always_inline)) -> Cur {
    if (c.step + 1 < steps) return Cur{c.tn, c.step + 1};
    return Cur{c.tn + (int)gridDim.x, 0};
  };
  auto load = [&](Cur c, Piece &p) __attribute__((always_inline)) {
    const int64_t tile = (int64_t)c.tn * n_tiles_k;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = tile + min(k_begin + c.step * U + u, n_tiles_k - 1);     // (behind the run: loaded, not used)
      p.q[u] = load_stream(codes + at * 64 + lane);
#pragma unroll
      for (int g = 0; g < GPC; ++g) p.w[u][g] = scales[(at * GPC + g) * 16 + n];
    }
  };
  Piece pa, pb;
  Cur ca{(int)blockIdx.x, 0};
  if (ca.tn < n_tiles_n) load(ca, pa);
  float rs = 0.0f;
  float norm0[8];                      // the norm weight of the thread's first piece, asked for ahead of the barrier
  if (MODE == kNorm) {
    row8<dtype>(src.c, min(8 * tid, K - 1), K, norm0);
    float ss = 0.0f;
    for (int i = tid; i < pieces; i += 64 * WAVES) {
      float f[8];
      row8<dtype>(src.a, 8 * i, K, f);
      if (src.b) {
        float g[8];
        row8<dtype>(src.b, 8 * i, K, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = round16<dtype>(f[j] + g[j]);
      }
      const u32x4 r = pack8<dtype>(f);
      xs[i] = r;
      if (blockIdx.x == 0 && src.residual_out) {
        uint16_t *out = reinterpret_cast<uint16_t *>(src.residual_out);
        if (8 * i + 8 <= K) reinterpret_cast<Loose *>(out + 8 * i)->v = r;
        else
          for (int j = 0; j < 8; ++j)
            if (8 * i + j < K) out[8 * i + j] = (uint16_t)(r[j >> 1] >> (16 * (j & 1)));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
    }
    ss = rdkv_wave_sum(ss);
    if (lane == 0) s_part[wave] = ss;
    __syncthreads();
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += s_part[w];
    rs = rsqrtf(all / (float)K + src.eps);
  }
  for (int i = tid; i < pieces; i += 64 * WAVES) {
    float f[8];
    if (MODE == kFromF32) {
      const float *p = reinterpret_cast<const float *>(src.a);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 8 * i + j < K ? round16<dtype>(p[8 * i + j]) : 0.0f;
    } else if (MODE == kNorm) {
      float w[8];
      if (i == tid) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = norm0[j];
      } else {
        row8<dtype>(src.c, 8 * i, K, w);
      }
      const u32x4 r = xs[i];           // (the piece this thread wrote itself)
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = round16<dtype>(w[j] * (load16<dtype>((uint16_t)(r[j >> 1] >> (16 * (j & 1)))) * rs));
    } else if (MODE == kSilu) {
      float g[8], u[8];
      row8<dtype>(src.a, 8 * i, K, g);
      row8<dtype>(src.b, 8 * i, K, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = round16<dtype>(round16<dtype>(silu(g[j])) * u[j]);
    } else {
      row8<dtype>(src.a, 8 * i, K, f);
    }
    xs[i] = pack8<dtype>(f);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += f[j];
#pragma unroll
    for (int o = 1; o < PPG; o <<= 1) s += __shfl_xor(s, o, 64);    // (16 lanes take part together: pieces % 16 == 0)
    if (i % PPG == 0) sums[i / PPG] = s;
  }
  __syncthreads();
  float acc = 0.0f;
  int kept = 0;
  auto flush = [&](int first) __attribute__((always_inline)) {      // `kept` tiles, from row tile `first` on
    __syncthreads();
    for (int i = tid; i < kept * 16; i += 64 * WAVES) {
      const int64_t row = (int64_t)(first + (i >> 4) * (int)gridDim.x) * 16 + (i & 15);
      if (row < N) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += s_red[i >> 4][w][i & 15];
        if (bias) s += load16<dtype>(bias[row]);
        y[row] = bits16<dtype>(s);
      }
    }
  };
  auto compute = [&](Cur c, const Piece &p) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kc = k_begin + c.step * U + u;
      if (kc < k_end) {
#pragma unroll
        for (int g = 0; g < GPC; ++g) {
          f32x4 D = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int d = g * (4 / GPC); d < (g + 1) * (4 / GPC); ++d)
            D = mfma<dtype>(xs[kc * 16 + 4 * d + quarter], operand<dtype>(p.q[u][d]), D);
          acc = add_group<dtype>(p.w[u][g], D[0], sums[kc * GPC + g], acc);
        }
      }
    }
    if (c.step + 1 == steps) {
      // every lane of a column holds the same sum (all sixteen rows of the operand are the one row)
      if (lane < 16) s_red[kept][wave][lane] = acc;
      acc = 0.0f;
      if (++kept == kKept) {
        flush(c.tn - (kKept - 1) * (int)gridDim.x);
        kept = 0;
        __syncthreads();
      }
    }
  };
  while (ca.tn < n_tiles_n) {
    const Cur cb = next(ca);
    if (cb.tn < n_tiles_n) load(cb, pb);
    compute(ca, pa);
    if (cb.tn >= n_tiles_n) break;
    ca = next(cb);
    if (ca.tn < n_tiles_n) load(ca, pa);
    compute(cb, pb);
  }
  if (kept) {
    const int mine = (n_tiles_n - 1 - (int)blockIdx.x) / (int)gridDim.x;      // the workgroup's last tile
    flush((int)blockIdx.x + (mine - kept + 1) * (int)gridDim.x);
  }
}

// Eight elements of row m of the activations, from element k on; what lies behind the matrix is zero.
template <int dtype>
__device__ __forceinline__ u32x4 rows8(const void *x, int x_dtype, int64_t x_stride_row, int64_t m, int M, int k, int K) {
  if (m >= M) return u32x4{0, 0, 0, 0};
  if (x_dtype == dtype && k + 8 <= K) return load_loose(reinterpret_cast<const uint16_t *>(x) + m * x_stride_row + k);
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = k + j < K ? rdkv_load_as_float(x, x_dtype, m * x_stride_row + k + j) : 0.0f;
  return pack8<dtype>(f);
}
template <int dtype>
__device__ __forceinline__ float sum8(u32x4 v) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = v[i];
    s += load16<dtype>((uint16_t)pair);
    s += load16<dtype>((uint16_t)(pair >> 16));
  }
  return s;
}
// The sum over the lanes of a group's pieces (sixteen lanes hold the pieces of a column tile), in each of them.
template <int GPC>
__device__ __forceinline__ float sum_pieces(float s) {
  s += rdkv_dpp_mov<0xB1>(s);                    // pairs, fours, eights, sixteens
  s += rdkv_dpp_mov<0x4E>(s);
  if (GPC <= 2) s += rdkv_dpp_mov<0x141>(s);
  if (GPC == 1) s += rdkv_dpp_mov<0x140>(s);
  return s;
}

// Rows as rows of the weights' type, zeros behind their ends up to a multiple of eight elements.
template <int dtype>
__global__ void __launch_bounds__(256)
w4_stage_rows_kernel(const void *__restrict__ x, int x_dtype, int64_t x_stride_row, int K, int K_out, uint16_t *__restrict__ out) {
  const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
  if (k < K_out) out[m * K_out + k] = k < K ? bits16<dtype>(rdkv_load_as_float(x, x_dtype, m * x_stride_row + k)) : (uint16_t)0;
}

// Few products: a workgroup takes a row tile of the weights (grid.x) and 16 activation rows (grid.y), its wavefronts share
// the columns.  The rows' operands come straight from global memory (each is read by one wavefront), the sums X from a
// product with ones (all columns of it are X, where the lanes need it).  The rows start at 16-byte borders, K is a multiple
// of eight: what lies behind is taken as zero.  Bound by latency: 5 x 6144 x 4096 bf16 7.6 us for 14 MB.
template <int dtype, int GPC, int WAVES, int U>
__global__ void __launch_bounds__(64 * WAVES)
w4_few_kernel(const u32x4 *__restrict__ codes, const uint32_t *__restrict__ scales, const uint16_t *__restrict__ x,
              int64_t x_stride_row, const uint16_t *__restrict__ bias, int M, int N, int K, int n_tiles_k,
              uint16_t *__restrict__ y, int64_t y_stride_row) {
  __shared__ float s_acc[WAVES][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane >> 4, n = lane & 15;
  const int tn = blockIdx.x, m0 = blockIdx.y * 16;
  const uint16_t *row = x + (int64_t)min(m0 + n, M - 1) * x_stride_row;       // (behind the last one: not stored)
  const u32x4 *tile = codes + (int64_t)tn * n_tiles_k * 64 + lane;
  const uint32_t *words = scales + (int64_t)tn * n_tiles_k * GPC * 16 + n;
  constexpr uint32_t one2 = dtype == RDKV_DTYPE_F16 ? 0x3c003c00u : 0x3f803f80u;
  const u32x4 ones = {one2, one2, one2, one2};
  struct Piece { u32x4 q[U], a[U][4]; uint32_t w[U][GPC]; };
  const int run = (n_tiles_k + WAVES - 1) / WAVES, k_begin = min(wave * run, n_tiles_k), k_end = min(k_begin + run, n_tiles_k);
  auto load = [&](int k0, Piece &p) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kc = min(k0 + u, n_tiles_k - 1);       // (behind the run: loaded, not used)
      p.q[u] = load_stream(tile + (int64_t)kc * 64);
#pragma unroll
      for (int g = 0; g < GPC; ++g) p.w[u][g] = words[(kc * GPC + g) * 16];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int k = kc * kTileCols + 32 * d + 8 * c;
        const u32x4 v = *reinterpret_cast<const u32x4 *>(row + (k < K ? k : 0));
        p.a[u][d] = k < K ? v : u32x4{0, 0, 0, 0};
      }
    }
  };
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&](int k0, const Piece &p) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u < k_end) {
#pragma unroll
        for (int g = 0; g < GPC; ++g) {
          f32x4 D = {0.0f, 0.0f, 0.0f, 0.0f}, X = D;
#pragma unroll
          for (int d = g * (4 / GPC); d < (g + 1) * (4 / GPC); ++d) {
            D = mfma<dtype>(p.a[u][d], operand<dtype>(p.q[u][d]), D);
            X = mfma<dtype>(p.a[u][d], ones, X);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = add_group<dtype>(p.w[u][g], D[i], X[i], acc[i]);
        }
      }
    }
  };
  Piece pa, pb;
  int k0 = k_begin;
  if (k0 < k_end) load(k0, pa);
  while (k0 < k_end) {
    if (k0 + U < k_end) load(k0 + U, pb);
    compute(k0, pa);
    k0 += U;
    if (k0 >= k_end) break;
    if (k0 + U < k_end) load(k0 + U, pa);
    compute(k0, pb);
    k0 += U;
  }
  // register i of lane 16 c + n: activation row 4 c + i, weight row n
#pragma unroll
  for (int i = 0; i < 4; ++i) s_acc[wave][(4 * c + i) * 16 + n] = acc[i];
  __syncthreads();
  if (tid < 256) {
    const int m = m0 + (tid >> 4);
    const int64_t r = (int64_t)tn * 16 + (tid & 15);
    if (m < M && r < N) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += s_acc[w][tid];
      if (bias) s += load16<dtype>(bias[r]);
      y[(int64_t)m * y_stride_row + r] = bits16<dtype>(s);
    }
  }
}

// More rows.  A first launch lays the activations out in operand order, sixteen rows by a column tile at a time (piece p,
// columns 8 p .. 8 p + 7, of row m at 16-byte slot 16 p + m: what lane 16 c + m reads for p = 4 d + c), zeros behind the
// matrix, and forms the sums X; every workgroup of the second launch then copies whole blocks.  Blocks follow each other by
// column tile within MT tiles of rows: the operands of the MT tiles, then their sums [group][row].
template <int GPC, int MT>
struct Block { u32x4 x[MT * 256]; float sum[GPC][16 * MT]; };

template <int dtype, int GPC, int MT>
__global__ void __launch_bounds__(256)
w4_blocks_kernel(const void *__restrict__ x, int x_dtype, int64_t x_stride_row, int M, int K, Block<GPC, MT> *__restrict__ out) {
  const int tid = threadIdx.x, piece = tid & 15, m = tid >> 4;
  const int kc = blockIdx.x, mt = blockIdx.y % MT;
  Block<GPC, MT> &block = out[(int64_t)(blockIdx.y / MT) * gridDim.x + kc];
  const u32x4 v = rows8<dtype>(x, x_dtype, x_stride_row, (int64_t)blockIdx.y * 16 + m, M, kc * kTileCols + 8 * piece, K);
  block.x[mt * 256 + piece * 16 + m] = v;
  const float s = sum_pieces<GPC>(sum8<dtype>(v));
  if (piece % (16 / GPC) == 0) block.sum[piece / (16 / GPC)][16 * mt + m] = s;
}

// A workgroup of eight wavefronts takes 16 MT activation rows by NT row tiles of the weights for each wavefront of a set.  SETS
// sets take the column tiles in turn; a set copies the next block to LDS while it computes on the one before.  Two sets of
// four wavefronts with two row tiles each (wide: 128 rows of the weights), or, where that leaves compute units without work,
// four sets of two wavefronts with one (narrow: 32 rows).  500 rows of 14336 -> 4096 in bf16 82 us, 0.72 PFLOP/s: the matrix
// cores work 33 % of the time, vector instructions (a dword's operands, two a result and group) issue 50 %, LDS is read 29 %,
// and two wavefronts a SIMD overlap little of it; 64 rows of 4096 -> 28672 in fp16 26 us.
template <int dtype, int GPC, int MT, int NT, int SETS>
__global__ void __launch_bounds__(512)
w4_tile_kernel(const u32x4 *__restrict__ codes, const uint32_t *__restrict__ scales, const Block<GPC, MT> *__restrict__ blocks,
               const uint16_t *__restrict__ bias, int M, int N, int n_tiles_n, int n_tiles_k, uint16_t *__restrict__ y,
               int64_t y_stride_row) {
  constexpr int kWaves = 8 / SETS, kThreads = 64 * kWaves, kCopies = MT * 256 / kThreads, kSums = GPC * 16 * MT,
                kSumCopies = (kSums + kThreads - 1) / kThreads;
  __shared__ Block<GPC, MT> s_block[SETS][2];        // [set][buffer]
  const int tid = threadIdx.x, lane = tid & 63, set = __builtin_amdgcn_readfirstlane(tid / kThreads),
            wave = __builtin_amdgcn_readfirstlane(tid / 64 % kWaves), c = lane >> 4, n = lane & 15, st = tid % kThreads;
  const int tn0 = (blockIdx.x * kWaves + wave) * NT, m0 = blockIdx.y * (16 * MT);
  const Block<GPC, MT> *from = blocks + (int64_t)blockIdx.y * n_tiles_k;
  const u32x4 *tile[NT];
  const uint32_t *words[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int64_t tn = min(tn0 + nt, n_tiles_n - 1);
    tile[nt] = codes + tn * n_tiles_k * 64 + lane;
    words[nt] = scales + tn * n_tiles_k * GPC * 16 + n;
  }
  f32x4 acc[NT][MT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Weights { u32x4 q[NT]; uint32_t w[NT][GPC]; };
  struct Copy { u32x4 x[kCopies]; float sum[kSumCopies]; };
  auto load_x = [&](int kc, Copy &v) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kCopies; ++j) v.x[j] = from[kc].x[kThreads * j + st];
#pragma unroll
    for (int j = 0; j < kSumCopies; ++j) v.sum[j] = (&from[kc].sum[0][0])[min(kThreads * j + st, kSums - 1)];
  };
  auto store_x = [&](Block<GPC, MT> &to, const Copy &v) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kCopies; ++j) to.x[kThreads * j + st] = v.x[j];
#pragma unroll
    for (int j = 0; j < kSumCopies; ++j)
      if (kThreads * j + st < kSums) (&to.sum[0][0])[kThreads * j + st] = v.sum[j];
  };
  auto load_w = [&](int kc, Weights &w) __attribute__((always_inline)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      w.q[nt] = tile[nt][(int64_t)kc * 64];
#pragma unroll
      for (int g = 0; g < GPC; ++g) w.w[nt][g] = words[nt][(kc * GPC + g) * 16];
    }
  };
  // The operands of the next 32 columns are read from LDS while the matrix cores work on the current ones.
  auto compute = [&](const Block<GPC, MT> &b, const Weights &w) __attribute__((always_inline)) {
    u32x4 a[2][MT];
    f32x4 D[NT][MT], X[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) a[0][mt] = b.x[mt * 256 + lane];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      constexpr int DPG = 4 / GPC;
      if (d + 1 < 4) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) a[(d + 1) & 1][mt] = b.x[mt * 256 + (d + 1) * 64 + lane];
      }
      if ((d + 1) % DPG == 0) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) X[mt] = *reinterpret_cast<const f32x4 *>(&b.sum[d / DPG][16 * mt + 4 * c]);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const u32x4 o = operand<dtype>(w.q[nt][d]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) D[nt][mt] = mfma<dtype>(a[d & 1][mt], o, d % DPG == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : D[nt][mt]);
      }
      if ((d + 1) % DPG == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[nt][mt][i] = add_group<dtype>(w.w[nt][d / DPG], D[nt][mt][i], X[mt][i], acc[nt][mt][i]);
      }
    }
  };
  // All sets make the same number of steps.  The loads of a step are issued two steps ahead (behind the last tile: the
  // last one again, not used; without a branch, so that a wait leaves the younger loads in flight).
  const int steps = (n_tiles_k + SETS - 1) / SETS;
  auto at = [&](int step) __attribute__((always_inline)) { return min(SETS * step + set, n_tiles_k - 1); };
  Weights w[2];
  Copy xv[2];
  load_x(at(0), xv[0]);
  load_w(at(0), w[0]);
  load_x(at(1), xv[1]);
  load_w(at(1), w[1]);
  store_x(s_block[set][0], xv[0]);
  __syncthreads();
  for (int step0 = 0; step0 < steps; step0 += 2) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int step = step0 + j;
      if (step < steps) {
        load_x(at(step + 2), xv[j]);
        if (SETS * step + set < n_tiles_k) compute(s_block[set][j], w[j]);
        load_w(at(step + 2), w[j]);
        store_x(s_block[set][j ^ 1], xv[j ^ 1]);
        __syncthreads();
      }
    }
  }
  // the other sets' sums join the first one's, in their order (all reads of the blocks are behind the barrier)
  static_assert(sizeof(s_block) >= (SETS - 1) * kWaves * NT * MT * 256 * 4, "the sums of the sets fit the blocks");
  f32x4 *join = reinterpret_cast<f32x4 *>(&s_block[0][0]) + wave * (NT * MT * 64) + lane;
  constexpr int kJoin = kWaves * NT * MT * 64;       // of a set
  if (set > 0) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) join[(set - 1) * kJoin + (nt * MT + mt) * 64] = acc[nt][mt];
  }
  __syncthreads();
  if (set > 0) return;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int64_t r = (int64_t)(tn0 + nt) * 16 + n;
    const float b = bias && r < N ? load16<dtype>(bias[r]) : 0.0f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f32x4 sum = acc[nt][mt];
#pragma unroll
      for (int o = 1; o < SETS; ++o) {
        const f32x4 other = join[(o - 1) * kJoin + (nt * MT + mt) * 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += other[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + 16 * mt + 4 * c + i;
        if (m < M && r < N) y[(int64_t)m * y_stride_row + r] = bits16<dtype>(sum[i] + b);
      }
    }
  }
}

constexpr int kRowMaxK = 32768;       // what one row's LDS copy takes

int compute_units() {
  static int cu_of_device[64];
  int dev = 0, n_cu = 256;
  if (hipGetDevice(&dev) == hipSuccess && dev >= 0 && dev < 64) {
    if (cu_of_device[dev] == 0) {
      int v = 0;
      if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0)
        cu_of_device[dev] = v;
    }
    if (cu_of_device[dev] > 0) n_cu = cu_of_device[dev];
  }
  return n_cu;
}

struct Shape { int n_tiles_n, n_tiles_k, gpc; int64_t n_tiles; };

int check_shape(const char *fn, int N, int K, int group, int dtype, Shape *s) {
  RDKV_REQUIRE(N >= 0 && K > 0 && N <= 0x7ffffff0 && K <= 0x7fffff00, "%s: bad shape N=%d K=%d", fn, N, K);
  RDKV_REQUIRE(group == 32 || group == 64 || group == 128, "%s: groups of 32, 64 or 128 columns, got %d", fn, group);
  RDKV_REQUIRE(dtype == RDKV_DTYPE_F16 || dtype == RDKV_DTYPE_BF16, "%s: fp16 or bf16 only", fn);
  s->n_tiles_n = (int)rdkv_cdiv(N, kTileRows);
  s->n_tiles_k = (int)rdkv_cdiv(K, kTileCols);
  s->gpc = kTileCols / group;
  s->n_tiles = (int64_t)s->n_tiles_n * s->n_tiles_k;
  // (four tiles to 256 threads, below 2^32 of them: 1.4e11 weights)
  RDKV_REQUIRE(s->n_tiles < (int64_t)1 << 26, "%s: a matrix of %d x %d is too large", fn, N, K);
  return RDKV_OK;
}

bool aligned16(const void *p) { return ((uintptr_t)p % 16) == 0; }

template <int dtype, int MODE, int GPC>
void launch_row(const Shape &sh, const void *codes, const uint32_t *scales, const RowSource &src, const void *bias, int N,
                int K, void *y, hipStream_t s) {
  constexpr int WAVES = 16, U = 2;
  const int cus = compute_units();
  const size_t lds = (size_t)sh.n_tiles_k * (256 + 4 * GPC);
  const int grid = sh.n_tiles_n < 2 * cus ? sh.n_tiles_n : 2 * cus;
  hipLaunchKernelGGL((w4_row_kernel<dtype, MODE, GPC, WAVES, U>), dim3(grid), dim3(64 * WAVES), lds, s, (const u32x4 *)codes,
                     scales, src, (const uint16_t *)bias, N, K, sh.n_tiles_n, sh.n_tiles_k, (uint16_t *)y);
}
template <int MODE>
void launch_row_any(int dtype, const Shape &sh, const void *codes, const uint32_t *scales, const RowSource &src,
                    const void *bias, int N, int K, void *y, hipStream_t s) {
#define RDKV_W4_ROW(DT)                                                                          \
  do {                                                                                           \
    if (sh.gpc == 1) launch_row<DT, MODE, 1>(sh, codes, scales, src, bias, N, K, y, s);          \
    else if (sh.gpc == 2) launch_row<DT, MODE, 2>(sh, codes, scales, src, bias, N, K, y, s);     \
    else launch_row<DT, MODE, 4>(sh, codes, scales, src, bias, N, K, y, s);                      \
  } while (0)
  if (dtype == RDKV_DTYPE_F16) RDKV_W4_ROW(RDKV_DTYPE_F16);
  else RDKV_W4_ROW(RDKV_DTYPE_BF16);
#undef RDKV_W4_ROW
}

struct Rows {
  const void *x;
  int x_dtype;
  int64_t x_stride;
  int K;
  const uint16_t *bias;
  int M, N;
  uint16_t *y;
  int64_t y_stride;
  void *workspace;
};
// How the rows are multiplied, by the number of workgroups that each form makes; K = 4096, groups of 128, in us:
//   - up to two tiles of 16 x 16 results for each compute unit: w4_few_kernel, whose one launch keeps nothing in LDS
//     (few / narrow tiles: 2 x 4096 5.3 / 8.7, 64 x 1024 7.1 / 16.3, 32 x 4096 11.2 / 11.5, but 24 x 6144 14.2 / 11.4);
//   - beyond, wide tiles of the workgroup where they make work for three quarters of the compute units, of 64 rows if
//     possible (64 x 28672: wide 64 rows 27.5, wide 32 rows 29.5, narrow 42.8; 64 x 14336: wide 32 rows 18.6, wide 64 rows
//     25.8, narrow 25.9), narrow ones otherwise (64 x 4096: 11.8 against 17.5 wide, 16 x 16384: 12.2 against 16.6).
bool few(int M, int N) { return rdkv_cdiv(N, kTileRows) * rdkv_cdiv(M, 16) <= 2 * compute_units(); }
int64_t few_row(int K) { return rdkv_cdiv(K, 8) * 8; }        // elements of a staged row

template <int dtype, int GPC>
void launch_few(const Shape &sh, const void *codes, const uint32_t *scales, const Rows &r, hipStream_t s) {
  const uint16_t *x = (const uint16_t *)r.x;
  int64_t stride = r.x_stride;
  int K = r.K;
  if (r.x_dtype != dtype || K % 8 || !aligned16(x) || (r.M > 1 && stride % 8)) {
    stride = K = (int)few_row(K);
    x = (const uint16_t *)r.workspace;
    hipLaunchKernelGGL(w4_stage_rows_kernel<dtype>, dim3((unsigned)rdkv_cdiv(K, 256), r.M), dim3(256), 0, s, r.x, r.x_dtype,
                       r.x_stride, r.K, K, (uint16_t *)r.workspace);
  }
  // Wavefronts that share the columns, tiles a step: 8 and 2 for one to eight tiles a wavefront (5 x 6144 x 4096 7.8 us, 8.7 with
  // 8 and 1, 9.1 with 16 and 1); one tile each at most, and a second would be loaded for nothing: 12 x 1024 x 1024 3.6 against 4.4; beyond
  // K = 8192, 16 and 1: 8 x 4096 x 14336 13.8 against 15.4.
  if (sh.n_tiles_k <= 8)
    hipLaunchKernelGGL((w4_few_kernel<dtype, GPC, 8, 1>), dim3(sh.n_tiles_n, (unsigned)rdkv_cdiv(r.M, 16)), dim3(512), 0, s,
                       (const u32x4 *)codes, scales, x, stride, r.bias, r.M, r.N, K, sh.n_tiles_k, r.y, r.y_stride);
  else if (sh.n_tiles_k <= 64)
    hipLaunchKernelGGL((w4_few_kernel<dtype, GPC, 8, 2>), dim3(sh.n_tiles_n, (unsigned)rdkv_cdiv(r.M, 16)), dim3(512), 0, s,
                       (const u32x4 *)codes, scales, x, stride, r.bias, r.M, r.N, K, sh.n_tiles_k, r.y, r.y_stride);
  else
    hipLaunchKernelGGL((w4_few_kernel<dtype, GPC, 16, 1>), dim3(sh.n_tiles_n, (unsigned)rdkv_cdiv(r.M, 16)), dim3(1024), 0, s,
                       (const u32x4 *)codes, scales, x, stride, r.bias, r.M, r.N, K, sh.n_tiles_k, r.y, r.y_stride);
}
template <int dtype, int GPC, int MT, int NT, int SETS>
void launch_tile(const Shape &sh, const void *codes, const uint32_t *scales, const Rows &r, hipStream_t s) {
  const unsigned blocks = (unsigned)rdkv_cdiv(r.M, 16 * MT);
  auto *at = reinterpret_cast<Block<GPC, MT> *>(r.workspace);
  hipLaunchKernelGGL((w4_blocks_kernel<dtype, GPC, MT>), dim3(sh.n_tiles_k, blocks * MT), dim3(256), 0, s, r.x, r.x_dtype, r.x_stride,
                     r.M, r.K, at);
  hipLaunchKernelGGL((w4_tile_kernel<dtype, GPC, MT, NT, SETS>), dim3((unsigned)rdkv_cdiv(sh.n_tiles_n, 8 / SETS * NT), blocks), dim3(512), 0,
                     s, (const u32x4 *)codes, scales, at, r.bias, r.M, r.N, sh.n_tiles_n, sh.n_tiles_k, r.y, r.y_stride);
}
template <int dtype, int GPC>
void launch_rows(const Shape &sh, const void *codes, const uint32_t *scales, const Rows &r, hipStream_t s) {
  const int full = compute_units() * 3 / 4;
  const int64_t across = rdkv_cdiv(sh.n_tiles_n, 8);         // workgroups of the wide form
  if (few(r.M, r.N)) launch_few<dtype, GPC>(sh, codes, scales, r, s);
  else if (r.M <= 16 && across >= full) launch_tile<dtype, GPC, 1, 2, 2>(sh, codes, scales, r, s);
  else if (r.M <= 16) launch_tile<dtype, GPC, 1, 1, 4>(sh, codes, scales, r, s);
  else if (r.M > 32 && across * rdkv_cdiv(r.M, 64) >= full) launch_tile<dtype, GPC, 4, 2, 2>(sh, codes, scales, r, s);
  else if (across * rdkv_cdiv(r.M, 32) >= full) launch_tile<dtype, GPC, 2, 2, 2>(sh, codes, scales, r, s);
  else launch_tile<dtype, GPC, 2, 1, 4>(sh, codes, scales, r, s);
}

}  // namespace

RDKV_API int64_t rdkv_w4_codes_bytes(int N, int K) {
  if (N <= 0 || K <= 0) return 0;
  return rdkv_cdiv(N, kTileRows) * rdkv_cdiv(K, kTileCols) * kTileBytes;
}
RDKV_API int64_t rdkv_w4_scale_words(int N, int K, int group) {
  if (N <= 0 || K <= 0 || (group != 32 && group != 64 && group != 128)) return 0;
  return rdkv_cdiv(N, kTileRows) * rdkv_cdiv(K, kTileCols) * (kTileCols / group) * 16;
}

RDKV_API int rdkv_w4_quantize(const void *W, int64_t w_stride_row, int N, int K, int group, int dtype, void *codes,
                              uint32_t *scales, void *stream) {
  const char *fn = "rdkv_w4_quantize";
  Shape sh;
  const int rc = check_shape(fn, N, K, group, dtype, &sh);
  if (rc != RDKV_OK || N == 0) return rc;
  RDKV_REQUIRE(W && codes && scales && aligned16(codes), "%s: null or misaligned pointer", fn);
  RDKV_REQUIRE(w_stride_row >= K || N == 1, "%s: rows overlap (stride %lld, K=%d)", fn, (long long)w_stride_row, K);
  const dim3 grid((unsigned)rdkv_cdiv(sh.n_tiles, 4));
#define RDKV_W4_QUANTIZE(DT, GPC)                                                                                     \
  hipLaunchKernelGGL((w4_quantize_kernel<DT, GPC>), grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t *)W,      \
                     w_stride_row, N, K, (uint32_t)sh.n_tiles_k, (uint32_t)sh.n_tiles, (u32x4 *)codes, scales)
#define RDKV_W4_QUANTIZE_ANY(DT)                         \
  do {                                                   \
    if (sh.gpc == 1) RDKV_W4_QUANTIZE(DT, 1);            \
    else if (sh.gpc == 2) RDKV_W4_QUANTIZE(DT, 2);       \
    else RDKV_W4_QUANTIZE(DT, 4);                        \
  } while (0)
  if (dtype == RDKV_DTYPE_F16) RDKV_W4_QUANTIZE_ANY(RDKV_DTYPE_F16);
  else RDKV_W4_QUANTIZE_ANY(RDKV_DTYPE_BF16);
#undef RDKV_W4_QUANTIZE_ANY
#undef RDKV_W4_QUANTIZE
  RDKV_CHECK_LAUNCH(fn);
  return RDKV_OK;
}

RDKV_API int rdkv_w4_pack(const uint8_t *q, int64_t q_stride_row, const void *scale, int scale_dtype,
                          int64_t scale_stride_row, const uint8_t *zero, int64_t zero_stride_row, int N, int K, int group,
                          void *codes, uint32_t *scales, void *stream) {
  const char *fn = "rdkv_w4_pack";
  Shape sh;
  const int rc = check_shape(fn, N, K, group, RDKV_DTYPE_F16, &sh);
  if (rc != RDKV_OK || N == 0) return rc;
  RDKV_REQUIRE(q && scale && codes && scales && aligned16(codes), "%s: null or misaligned pointer", fn);
  RDKV_REQUIRE(scale_dtype >= 0 && scale_dtype <= 2, "%s: unknown scale type %d", fn, scale_dtype);
  const dim3 grid((unsigned)rdkv_cdiv(sh.n_tiles, 4));
#define RDKV_W4_PACK(GPC)                                                                                            \
  hipLaunchKernelGGL((w4_pack_kernel<GPC>), grid, dim3(256), 0, (hipStream_t)stream, q, q_stride_row, scale, scale_dtype, \
                     scale_stride_row, zero, zero_stride_row, N, K, (uint32_t)sh.n_tiles_k, (uint32_t)sh.n_tiles, (u32x4 *)codes, scales)
  if (sh.gpc == 1) RDKV_W4_PACK(1);
  else if (sh.gpc == 2) RDKV_W4_PACK(2);
  else RDKV_W4_PACK(4);
#undef RDKV_W4_PACK
  RDKV_CHECK_LAUNCH(fn);
  return RDKV_OK;
}

RDKV_API int rdkv_w4_dequant(const void *codes, const uint32_t *scales, int N, int K, int group, int dtype, void *out,
                             int64_t out_stride_row, void *stream) {
  const char *fn = "rdkv_w4_dequant";
  Shape sh;
  const int rc = check_shape(fn, N, K, group, dtype, &sh);
  if (rc != RDKV_OK || N == 0) return rc;
  RDKV_REQUIRE(codes && scales && out && aligned16(codes), "%s: null or misaligned pointer", fn);
  RDKV_REQUIRE(out_stride_row >= K || N == 1, "%s: output rows overlap", fn);
  const dim3 grid((unsigned)rdkv_cdiv(sh.n_tiles, 4));
#define RDKV_W4_DEQUANT(DT, GPC)                                                                                       \
  hipLaunchKernelGGL((w4_dequant_kernel<DT, GPC>), grid, dim3(256), 0, (hipStream_t)stream, (const u32x4 *)codes, scales, \
                     N, K, (uint32_t)sh.n_tiles_k, (uint32_t)sh.n_tiles, (uint16_t *)out, out_stride_row)
#define RDKV_W4_DEQUANT_ANY(DT)                       \
  do {                                                \
    if (sh.gpc == 1) RDKV_W4_DEQUANT(DT, 1);          \
    else if (sh.gpc == 2) RDKV_W4_DEQUANT(DT, 2);     \
    else RDKV_W4_DEQUANT(DT, 4);                      \
  } while (0)
  if (dtype == RDKV_DTYPE_F16) RDKV_W4_DEQUANT_ANY(RDKV_DTYPE_F16);
  else RDKV_W4_DEQUANT_ANY(RDKV_DTYPE_BF16);
#undef RDKV_W4_DEQUANT_ANY
#undef RDKV_W4_DEQUANT
  RDKV_CHECK_LAUNCH(fn);
  return RDKV_OK;
}

RDKV_API int64_t rdkv_w4_linear_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || (M == 1 && K <= kRowMaxK)) return 0;
  if (few(M, N)) return M * few_row(K) * 2;
  // whole blocks of 16, 32 or 64 rows, their sums at the finest groups
  const int64_t block = M <= 16 ? sizeof(Block<4, 1>) : M <= 32 ? sizeof(Block<4, 2>) : sizeof(Block<4, 4>);
  return rdkv_cdiv(M, M <= 16 ? 16 : M <= 32 ? 32 : 64) * rdkv_cdiv(K, kTileCols) * block;
}

RDKV_API int rdkv_w4_linear(const void *codes, const uint32_t *scales, const void *x, int x_dtype, int64_t x_stride_row,
                            const void *bias, int M, int N, int K, int group, int dtype, void *y, int64_t y_stride_row,
                            void *workspace, int64_t workspace_bytes, void *stream) {
  const char *fn = "rdkv_w4_linear";
  Shape sh;
  const int rc = check_shape(fn, N, K, group, dtype, &sh);
  if (rc != RDKV_OK) return rc;
  RDKV_REQUIRE(M >= 0 && M <= 1 << 19, "%s: %d rows", fn, M);
  if (N == 0 || M == 0) return RDKV_OK;
  RDKV_REQUIRE(codes && scales && x && y && aligned16(codes), "%s: null or misaligned pointer", fn);
  RDKV_REQUIRE(x_dtype == dtype || x_dtype == RDKV_DTYPE_F32, "%s: x must have the weights' type or be fp32", fn);
  RDKV_REQUIRE(M == 1 || (x_stride_row >= 0 && y_stride_row >= N), "%s: output rows overlap", fn);
  hipStream_t s = (hipStream_t)stream;
  if (M == 1 && K <= kRowMaxK) {
    const RowSource src = {x, nullptr, nullptr, 0.0f, nullptr};
    if (x_dtype == RDKV_DTYPE_F32) launch_row_any<kFromF32>(dtype, sh, codes, scales, src, bias, N, K, y, s);
    else launch_row_any<kPlain>(dtype, sh, codes, scales, src, bias, N, K, y, s);
    RDKV_CHECK_LAUNCH(fn);
    return RDKV_OK;
  }
  const int64_t need = rdkv_w4_linear_workspace_bytes(M, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
    rdkv_set_error("%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)need);
    return RDKV_EWORKSPACE;
  }
  const Rows r = {x, x_dtype, x_stride_row, K, (const uint16_t *)bias, M, N, (uint16_t *)y, y_stride_row, workspace};
#define RDKV_W4_ROWS(DT)                                              \
  do {                                                                \
    if (sh.gpc == 1) launch_rows<DT, 1>(sh, codes, scales, r, s);     \
    else if (sh.gpc == 2) launch_rows<DT, 2>(sh, codes, scales, r, s); \
    else launch_rows<DT, 4>(sh, codes, scales, r, s);                 \
  } while (0)
  if (dtype == RDKV_DTYPE_F16) RDKV_W4_ROWS(RDKV_DTYPE_F16);
  else RDKV_W4_ROWS(RDKV_DTYPE_BF16);
#undef RDKV_W4_ROWS
  RDKV_CHECK_LAUNCH(fn);
  return RDKV_OK;
}

RDKV_API int rdkv_w4_linear_norm(const void *codes, const uint32_t *scales, const void *x, const void *delta,
                                 const void *norm_weight, float eps, void *residual_out, const void *bias, int N, int K,
                                 int group, int dtype, void *y, void *stream) {
  const char *fn = "rdkv_w4_linear_norm";
  Shape sh;
  const int rc = check_shape(fn, N, K, group, dtype, &sh);
  if (rc != RDKV_OK || N == 0) return rc;
  RDKV_REQUIRE(K <= kRowMaxK, "%s: K=%d exceeds %d", fn, K, kRowMaxK);
  RDKV_REQUIRE(codes && scales && x && norm_weight && y && aligned16(codes), "%s: null or misaligned pointer", fn);
  RDKV_REQUIRE(!residual_out || (residual_out != x && residual_out != delta),
               "%s: residual_out must not alias the inputs (every workgroup reads them)", fn);
  const RowSource src = {x, delta, norm_weight, eps, residual_out};
  launch_row_any<kNorm>(dtype, sh, codes, scales, src, bias, N, K, y, (hipStream_t)stream);
  RDKV_CHECK_LAUNCH(fn);
  return RDKV_OK;
}

RDKV_API int rdkv_w4_linear_silu(const void *codes, const uint32_t *scales, const void *gate, const void *up,
                                 const void *bias, int N, int K, int group, int dtype, void *y, void *stream) {
  const char *fn = "rdkv_w4_linear_silu";
  Shape sh;
  const int rc = check_shape(fn, N, K, group, dtype, &sh);
  if (rc != RDKV_OK || N == 0) return rc;
  RDKV_REQUIRE(K <= kRowMaxK, "%s: K=%d exceeds %d", fn, K, kRowMaxK);
  RDKV_REQUIRE(codes && scales && gate && up && y && aligned16(codes), "%s: null or misaligned pointer", fn);
  const RowSource src = {gate, up, nullptr, 0.0f, nullptr};
  launch_row_any<kSilu>(dtype, sh, codes, scales, src, bias, N, K, y, (hipStream_t)stream);
  RDKV_CHECK_LAUNCH(fn);
  return RDKV_OK;
}
