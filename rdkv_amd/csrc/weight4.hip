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

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = 1024;
constexpr float kSmallestScale = 0x1p-120f;      // below it a group counts as all zeros (its scale stays an ordinary number)

__device__ __forceinline__ u32x4 load_stream(const u32x4 *p) { return __builtin_nontemporal_load(p); }

template <int dtype>
__device__ __forceinline__ float load16(uint16_t bits) {
  return dtype == RDKV_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, bits) : __uint_as_float((uint32_t)bits << 16);
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

struct TileAt { int64_t tile; int64_t row; int lane, c; int64_t col0; };
__device__ __forceinline__ TileAt tile_at(int64_t n_tiles_k) {
  TileAt t;
  t.lane = threadIdx.x & 63;
  t.c = t.lane >> 4;
  t.tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  t.row = (t.tile / n_tiles_k) * kTileRows + (t.lane & 15);
  t.col0 = (t.tile % n_tiles_k) * kTileCols;
  return t;
}

// The value range of a group takes in zero, so that a zero weight stays zero and the zero point lies in
// 0 .. 15; divisions are the correctly rounded ones and nothing is contracted, so the codes are those of the
// expressions rint(w / s) + z.  A group that holds a NaN or an infinity has scale NaN: every product with it is NaN.
template <int dtype, int GPC>
__global__ void __launch_bounds__(256)
w4_quantize_kernel(const uint16_t *__restrict__ W, int64_t w_stride_row, int N, int K, int aligned, int64_t n_tiles_k,
                   int64_t n_tiles, u32x4 *__restrict__ codes, uint32_t *__restrict__ scales) {
#pragma clang fp contract(off)
  const TileAt t = tile_at(n_tiles_k);
  if (t.tile >= n_tiles) return;
  float v[4][8];
  const uint16_t *src = W + t.row * w_stride_row;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int64_t k = t.col0 + 32 * d + 8 * t.c;
    if (t.row < N && aligned && k + 8 <= K) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(src + k);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[d][j] = load16<dtype>((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[d][j] = t.row < N && k + j < K ? load16<dtype>(src[k + j]) : 0.0f;
    }
  }
  constexpr int DPG = 4 / GPC;           // dwords of a lane per group
  u32x4 out;
#pragma unroll
  for (int g = 0; g < GPC; ++g) {
    float lo = 0.0f, hi = 0.0f;
    bool bad = false;
#pragma unroll
    for (int d = g * DPG; d < (g + 1) * DPG; ++d)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, v[d][j]);
        hi = fmaxf(hi, v[d][j]);
        bad |= !(fabsf(v[d][j]) < INFINITY);
      }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {   // the four lanes that share the row
      lo = fminf(lo, __shfl_xor(lo, o, 64));
      hi = fmaxf(hi, __shfl_xor(hi, o, 64));
      bad |= (bool)__shfl_xor((int)bad, o, 64);
    }
    float s = word_scale(scale_word((hi - lo) / 15.0f, 0));
    if (!(s < INFINITY) || bad) s = __builtin_nanf("");
    if (s < kSmallestScale) s = 1.0f;
    // (the clamps come last and take a NaN to 0: a group whose scale is NaN has zero codes)
    const float z = fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f);
#pragma unroll
    for (int d = g * DPG; d < (g + 1) * DPG; ++d) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float q = fminf(fmaxf(rintf(v[d][j] / s) + z, 0.0f), 15.0f);
        if (t.col0 + 32 * d + 8 * t.c + j < K) w |= (uint32_t)q << field_shift(j);
      }
      out[d] = t.row < N ? w : 0u;
    }
    if (t.c == 0) {
      const bool there = t.row < N && t.col0 + (int64_t)g * DPG * 32 < K;
      scales[(t.tile * GPC + g) * 16 + (t.lane & 15)] = there ? scale_word(s, (uint32_t)z) : 0u;
    }
  }
  codes[t.tile * 64 + t.lane] = out;
}

// Codes, scales and zero points of a matrix quantized elsewhere, into the layout.
template <int GPC>
__global__ void __launch_bounds__(256)
w4_pack_kernel(const uint8_t *__restrict__ src, int64_t src_stride_row, const void *__restrict__ scale, int scale_dtype,
               int64_t scale_stride_row, const uint8_t *__restrict__ zero, int64_t zero_stride_row, int N, int K,
               int64_t n_tiles_k, int64_t n_tiles, u32x4 *__restrict__ codes, uint32_t *__restrict__ scales) {
  const TileAt t = tile_at(n_tiles_k);
  if (t.tile >= n_tiles) return;
  u32x4 out;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t k = t.col0 + 32 * d + 8 * t.c + j;
      const uint32_t q = t.row < N && k < K ? src[t.row * src_stride_row + k] & 15u : 0u;
      w |= q << field_shift(j);
    }
    out[d] = w;
  }
  codes[t.tile * 64 + t.lane] = out;
  if (t.c < GPC) {                       // lane 16 g + n: group g of row n
    const int64_t group = t.col0 / (kTileCols / GPC) + t.c;
    uint32_t word = 0;
    if (t.row < N && group * (kTileCols / GPC) < K) {
      const float s = rdkv_load_as_float(scale, scale_dtype, t.row * scale_stride_row + group);
      word = scale_word(s, zero ? zero[t.row * zero_stride_row + group] & 15u : 8u);
    }
    scales[(t.tile * GPC + t.c) * 16 + (t.lane & 15)] = word;
  }
}

template <int dtype, int GPC>
__global__ void __launch_bounds__(256)
w4_dequant_kernel(const u32x4 *__restrict__ codes, const uint32_t *__restrict__ scales, int N, int K, int aligned,
                  int64_t n_tiles_k, int64_t n_tiles, uint16_t *__restrict__ out, int64_t out_stride_row) {
  const TileAt t = tile_at(n_tiles_k);
  if (t.tile >= n_tiles || t.row >= N) return;
  const u32x4 q = codes[t.tile * 64 + t.lane];
  uint16_t *dst = out + t.row * out_stride_row;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t word = scales[(t.tile * GPC + d * GPC / 4) * 16 + (t.lane & 15)];
    const float s = word_scale(word), z = (float)word_zero(word);
    const int64_t k = t.col0 + 32 * d + 8 * t.c;
    uint16_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // (a 5-bit integer times 20 bits: exact in fp32, rounded once to the type)
      const float v = ((float)((q[d] >> field_shift(j)) & 15u) - z) * s;
      h[j] = dtype == RDKV_DTYPE_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : rdkv_float_to_bf16_bits(v);
    }
    if (aligned && k + 8 <= K) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
      *reinterpret_cast<u32x4 *>(dst + k) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < K) dst[k + j] = h[j];
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
    b[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
#pragma unroll
    for (int r = 1; r < 4; ++r) b[r] = ((w >> (4 * r - 3)) & 0x00780078u) | 0x41804180u;
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
template <int dtype>
__device__ __forceinline__ uint16_t bits16(float v) {
  return dtype == RDKV_DTYPE_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : rdkv_float_to_bf16_bits(v);
}

// How one activation row reaches LDS, as in gemv.hip.
enum { kPlain = 0, kFromF32 = 1, kNorm = 2, kSilu = 3 };
struct RowSource {
  const void *a, *b, *c;
  float eps;
  void *residual_out;
  int aligned;                 // a, b, c and residual_out are 16-byte aligned
};

// Eight elements of a 16-bit row from element k on; what lies behind the row is zero.
template <int dtype>
__device__ __forceinline__ void row8(const void *row, int k, int K, int aligned, float (&f)[8]) {
  const uint16_t *p = reinterpret_cast<const uint16_t *>(row);
  if (aligned && k + 8 <= K) {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(p + k);
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
// column tiles); the wavefronts' sums meet in LDS and are added in their order.
template <int dtype, int MODE, int GPC, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
w4_row_kernel(const u32x4 *__restrict__ codes, const uint32_t *__restrict__ scales, RowSource src,
              const uint16_t *__restrict__ bias, int N, int K, int n_tiles_n, int n_tiles_k, uint16_t *__restrict__ y) {
  extern __shared__ u32x4 lds[];       // the row (16 pieces of 8 per column tile), then a sum per group
  __shared__ float s_red[2][WAVES][16];
  __shared__ float s_part[WAVES];
  u32x4 *xs = lds;
  float *sums = reinterpret_cast<float *>(lds + n_tiles_k * 16);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane >> 4, n = lane & 15;
  const int pieces = n_tiles_k * 16;
  constexpr int PPG = 16 / GPC;        // pieces per group
  float rs = 0.0f;
  if (MODE == kNorm) {
    float ss = 0.0f;
    for (int i = tid; i < pieces; i += 64 * WAVES) {
      float f[8];
      row8<dtype>(src.a, 8 * i, K, src.aligned, f);
      if (src.b) {
        float g[8];
        row8<dtype>(src.b, 8 * i, K, src.aligned, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = round16<dtype>(f[j] + g[j]);
      }
      const u32x4 r = pack8<dtype>(f);
      xs[i] = r;
      if (blockIdx.x == 0 && src.residual_out) {
        uint16_t *out = reinterpret_cast<uint16_t *>(src.residual_out);
        if (src.aligned && 8 * i + 8 <= K) *reinterpret_cast<u32x4 *>(out + 8 * i) = r;
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
      row8<dtype>(src.c, 8 * i, K, src.aligned, w);
      const u32x4 r = xs[i];           // (the piece this thread wrote itself)
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = round16<dtype>(w[j] * (load16<dtype>((uint16_t)(r[j >> 1] >> (16 * (j & 1)))) * rs));
    } else if (MODE == kSilu) {
      float g[8], u[8];
      row8<dtype>(src.a, 8 * i, K, src.aligned, g);
      row8<dtype>(src.b, 8 * i, K, src.aligned, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = round16<dtype>(round16<dtype>(g[j] / (1.0f + expf(-g[j]))) * u[j]);
    } else {
      row8<dtype>(src.a, 8 * i, K, src.aligned, f);
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
  const int run = (n_tiles_k + WAVES - 1) / WAVES;
  const int k_begin = min(wave * run, n_tiles_k), k_end = min(k_begin + run, n_tiles_k);
  int buf = 0;
  for (int tn = blockIdx.x; tn < n_tiles_n; tn += gridDim.x) {
    float acc = 0.0f;
    const u32x4 *tile = codes + (int64_t)tn * n_tiles_k * 64 + lane;
    const uint32_t *words = scales + (int64_t)tn * n_tiles_k * GPC * 16 + n;
    for (int kc = k_begin; kc < k_end; ++kc) {
      const u32x4 q = load_stream(tile + (int64_t)kc * 64);
#pragma unroll
      for (int g = 0; g < GPC; ++g) {
        const uint32_t w = words[(kc * GPC + g) * 16];
        f32x4 D = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = g * (4 / GPC); d < (g + 1) * (4 / GPC); ++d)
          D = mfma<dtype>(xs[kc * 16 + 4 * d + c], operand<dtype>(q[d]), D);
        acc = add_group<dtype>(w, D[0], sums[kc * GPC + g], acc);
      }
    }
    // every lane of a column holds the same sum (all sixteen rows of the operand are the one row)
    if (lane < 16) s_red[buf][wave][lane] = acc;
    __syncthreads();
    if (tid < 16 && tn * 16 + tid < N) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += s_red[buf][w][tid];
      const int row = tn * 16 + tid;
      if (bias) s += load16<dtype>(bias[row]);
      y[row] = bits16<dtype>(s);
    }
    buf ^= 1;      // the next tile's sums go elsewhere: one barrier a tile
  }
}

// Rows of any stride and type -> rows of the weights' type, columns padded with zeros to whole tiles.
template <int dtype>
__global__ void __launch_bounds__(256)
w4_stage_rows_kernel(const void *__restrict__ x, int x_dtype, int64_t x_stride_row, int K, int K_padded,
                     uint16_t *__restrict__ out) {
  const int k = blockIdx.x * 256 + threadIdx.x;
  const int64_t m = blockIdx.y;
  if (k >= K_padded) return;
  out[m * K_padded + k] = k < K ? bits16<dtype>(rdkv_load_as_float(x, x_dtype, m * x_stride_row + k)) : (uint16_t)0;
}

// Several activation rows: MT tiles of 16 rows by NT row tiles of the weights a workgroup, its eight wavefronts
// sharing the columns; the sums X come from a product with ones (all columns of it are X, where the lanes need it).
// x rows 16-byte aligned, K_x a multiple of 8 (what lies behind is taken as zero).
template <int dtype, int GPC, int MT, int NT>
__global__ void __launch_bounds__(512)
w4_rows_kernel(const u32x4 *__restrict__ codes, const uint32_t *__restrict__ scales, const uint16_t *__restrict__ x,
               int64_t x_stride_row, const uint16_t *__restrict__ bias, int M, int N, int K_x, int n_tiles_n,
               int n_tiles_k, uint16_t *__restrict__ y, int64_t y_stride_row) {
  extern __shared__ float s_acc[];      // [8][MT][NT][256]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane >> 4, n = lane & 15;
  const int tn0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);
  const uint16_t *rows[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) rows[mt] = x + (int64_t)min(m0 + 16 * mt + n, M - 1) * x_stride_row + 8 * c;
  const u32x4 *tile[NT];
  const uint32_t *words[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int64_t tn = min(tn0 + nt, n_tiles_n - 1);
    tile[nt] = codes + tn * n_tiles_k * 64 + lane;
    words[nt] = scales + tn * n_tiles_k * GPC * 16 + n;
  }
  f32x4 acc[MT][NT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr uint32_t one2 = dtype == RDKV_DTYPE_F16 ? 0x3c003c00u : 0x3f803f80u;
  const u32x4 ones = {one2, one2, one2, one2};
  for (int kc = wave; kc < n_tiles_k; kc += 8) {
    u32x4 q[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) q[nt] = tile[nt][(int64_t)kc * 64];
    u32x4 a[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int k = kc * kTileCols + 32 * d;
        const bool in = k + 8 * c < K_x;
        const u32x4 v = *reinterpret_cast<const u32x4 *>(rows[mt] + (in ? k : -8 * c));   // (else the row's start)
        a[mt][d] = in ? v : u32x4{0, 0, 0, 0};
      }
#pragma unroll
    for (int g = 0; g < GPC; ++g) {
      f32x4 X[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        X[mt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = g * (4 / GPC); d < (g + 1) * (4 / GPC); ++d) X[mt] = mfma<dtype>(a[mt][d], ones, X[mt]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint32_t w = words[nt][(kc * GPC + g) * 16];
        f32x4 D[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) D[mt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = g * (4 / GPC); d < (g + 1) * (4 / GPC); ++d) {
          const u32x4 b = operand<dtype>(q[nt][d]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) D[mt] = mfma<dtype>(a[mt][d], b, D[mt]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[mt][nt][i] = add_group<dtype>(w, D[mt][i], X[mt][i], acc[mt][nt][i]);
      }
    }
  }
  // register i of lane 16 c + n: activation row 4 c + i, weight row n
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s_acc[((wave * MT + mt) * NT + nt) * 256 + (4 * c + i) * 16 + n] = acc[mt][nt][i];
  __syncthreads();
  for (int e = tid; e < MT * NT * 256; e += 512) {
    const int in_tile = e & 255, nt = (e >> 8) % NT, mt = (e >> 8) / NT;
    const int m = m0 + 16 * mt + (in_tile >> 4);
    const int64_t row = (int64_t)(tn0 + nt) * 16 + (in_tile & 15);
    if (m >= M || row >= N) continue;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += s_acc[w * (MT * NT * 256) + e];
    if (bias) s += load16<dtype>(bias[row]);
    y[(int64_t)m * y_stride_row + row] = bits16<dtype>(s);
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
  RDKV_REQUIRE(s->n_tiles <= (int64_t)0x7fffffff, "%s: a matrix of %d x %d is too large", fn, N, K);
  return RDKV_OK;
}

bool aligned16(const void *p) { return ((uintptr_t)p % 16) == 0; }

template <int dtype, int MODE, int GPC>
void launch_row(const Shape &sh, const void *codes, const uint32_t *scales, const RowSource &src, const void *bias, int N,
                int K, void *y, hipStream_t s) {
  constexpr int WAVES = 8;
  const int cus = compute_units();
  const size_t lds = (size_t)sh.n_tiles_k * (256 + 4 * GPC);
  const int grid = sh.n_tiles_n < 2 * cus ? sh.n_tiles_n : 2 * cus;
  hipLaunchKernelGGL((w4_row_kernel<dtype, MODE, GPC, WAVES>), dim3(grid), dim3(64 * WAVES), lds, s, (const u32x4 *)codes,
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

struct Rows { const uint16_t *x; int64_t x_stride; int K_x; const uint16_t *bias; int M, N; uint16_t *y; int64_t y_stride; };
template <int dtype, int GPC, int MT, int NT>
void launch_rows(const Shape &sh, const void *codes, const uint32_t *scales, const Rows &r, hipStream_t s) {
  const dim3 grid((unsigned)rdkv_cdiv(sh.n_tiles_n, NT), (unsigned)rdkv_cdiv(r.M, 16 * MT));
  hipLaunchKernelGGL((w4_rows_kernel<dtype, GPC, MT, NT>), grid, dim3(512), (size_t)8 * MT * NT * 1024, s,
                     (const u32x4 *)codes, scales, r.x, r.x_stride, r.bias, r.M, r.N, r.K_x, sh.n_tiles_n, sh.n_tiles_k,
                     r.y, r.y_stride);
}
template <int dtype, int GPC>
void launch_rows_any(const Shape &sh, const void *codes, const uint32_t *scales, const Rows &r, hipStream_t s) {
  if (r.M <= 16) launch_rows<dtype, GPC, 1, 1>(sh, codes, scales, r, s);
  else if (r.M <= 32) launch_rows<dtype, GPC, 2, 1>(sh, codes, scales, r, s);
  else launch_rows<dtype, GPC, 4, 1>(sh, codes, scales, r, s);
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
  const int aligned = aligned16(W) && w_stride_row % 8 == 0;
  const dim3 grid((unsigned)rdkv_cdiv(sh.n_tiles, 4));
#define RDKV_W4_QUANTIZE(DT, GPC)                                                                                     \
  hipLaunchKernelGGL((w4_quantize_kernel<DT, GPC>), grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t *)W,      \
                     w_stride_row, N, K, aligned, (int64_t)sh.n_tiles_k, sh.n_tiles, (u32x4 *)codes, scales)
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
                     scale_stride_row, zero, zero_stride_row, N, K, (int64_t)sh.n_tiles_k, sh.n_tiles, (u32x4 *)codes, scales)
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
  const int aligned = aligned16(out) && out_stride_row % 8 == 0;
  const dim3 grid((unsigned)rdkv_cdiv(sh.n_tiles, 4));
#define RDKV_W4_DEQUANT(DT, GPC)                                                                                       \
  hipLaunchKernelGGL((w4_dequant_kernel<DT, GPC>), grid, dim3(256), 0, (hipStream_t)stream, (const u32x4 *)codes, scales, \
                     N, K, aligned, (int64_t)sh.n_tiles_k, sh.n_tiles, (uint16_t *)out, out_stride_row)
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

RDKV_API int64_t rdkv_w4_linear_workspace_bytes(int M, int K) {
  if (M <= 0 || K <= 0) return 0;
  return (int64_t)M * rdkv_cdiv(K, kTileCols) * kTileCols * 2;
}

RDKV_API int rdkv_w4_linear(const void *codes, const uint32_t *scales, const void *x, int x_dtype, int64_t x_stride_row,
                            const void *bias, int M, int N, int K, int group, int dtype, void *y, int64_t y_stride_row,
                            void *workspace, int64_t workspace_bytes, void *stream) {
  const char *fn = "rdkv_w4_linear";
  Shape sh;
  const int rc = check_shape(fn, N, K, group, dtype, &sh);
  if (rc != RDKV_OK) return rc;
  RDKV_REQUIRE(M >= 0 && M <= 65535 * 16, "%s: %d rows", fn, M);
  if (N == 0 || M == 0) return RDKV_OK;
  RDKV_REQUIRE(codes && scales && x && y && aligned16(codes), "%s: null or misaligned pointer", fn);
  RDKV_REQUIRE(x_dtype == dtype || x_dtype == RDKV_DTYPE_F32, "%s: x must have the weights' type or be fp32", fn);
  RDKV_REQUIRE(M == 1 || (x_stride_row >= 0 && y_stride_row >= N), "%s: output rows overlap", fn);
  hipStream_t s = (hipStream_t)stream;
  if (M == 1 && K <= kRowMaxK) {
    const RowSource src = {x, nullptr, nullptr, 0.0f, nullptr, aligned16(x)};
    if (x_dtype == RDKV_DTYPE_F32) launch_row_any<kFromF32>(dtype, sh, codes, scales, src, bias, N, K, y, s);
    else launch_row_any<kPlain>(dtype, sh, codes, scales, src, bias, N, K, y, s);
    RDKV_CHECK_LAUNCH(fn);
    return RDKV_OK;
  }
  Rows r = {(const uint16_t *)x, x_stride_row, K, (const uint16_t *)bias, M, N, (uint16_t *)y, y_stride_row};
  if (x_dtype != dtype || !aligned16(x) || (M > 1 && x_stride_row % 8 != 0) || K % 8 != 0) {
    // rows that cannot be read in 16-byte pieces (or are fp32): a padded copy first
    const int K_padded = sh.n_tiles_k * kTileCols;
    if (!workspace || workspace_bytes < rdkv_w4_linear_workspace_bytes(M, K) || !aligned16(workspace)) {
      rdkv_set_error("%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)rdkv_w4_linear_workspace_bytes(M, K));
      return RDKV_EWORKSPACE;
    }
    // (a grid's second dimension takes 65535 rows)
    for (int64_t m = 0; m < M; m += 65535) {
      const dim3 grid((unsigned)rdkv_cdiv(K_padded, 256), (unsigned)(M - m < 65535 ? M - m : 65535));
      const char *from = (const char *)x + m * x_stride_row * (x_dtype == RDKV_DTYPE_F32 ? 4 : 2);
      uint16_t *to = (uint16_t *)workspace + m * K_padded;
      if (dtype == RDKV_DTYPE_F16)
        hipLaunchKernelGGL(w4_stage_rows_kernel<RDKV_DTYPE_F16>, grid, dim3(256), 0, s, from, x_dtype, x_stride_row, K, K_padded, to);
      else
        hipLaunchKernelGGL(w4_stage_rows_kernel<RDKV_DTYPE_BF16>, grid, dim3(256), 0, s, from, x_dtype, x_stride_row, K, K_padded, to);
      RDKV_CHECK_LAUNCH(fn);
    }
    r.x = (const uint16_t *)workspace;
    r.x_stride = K_padded;
    r.K_x = K_padded;
  }
#define RDKV_W4_ROWS(DT)                                                  \
  do {                                                                    \
    if (sh.gpc == 1) launch_rows_any<DT, 1>(sh, codes, scales, r, s);     \
    else if (sh.gpc == 2) launch_rows_any<DT, 2>(sh, codes, scales, r, s); \
    else launch_rows_any<DT, 4>(sh, codes, scales, r, s);                 \
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
  const RowSource src = {x, delta, norm_weight, eps, residual_out,
                         aligned16(x) && aligned16(delta) && aligned16(norm_weight) && aligned16(residual_out)};
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
  const RowSource src = {gate, up, nullptr, 0.0f, nullptr, aligned16(gate) && aligned16(up)};
  launch_row_any<kSilu>(dtype, sh, codes, scales, src, bias, N, K, y, (hipStream_t)stream);
  RDKV_CHECK_LAUNCH(fn);
  return RDKV_OK;
}
