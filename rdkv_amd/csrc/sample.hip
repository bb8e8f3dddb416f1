// The next token of every sequence from its logits l and a given uniform u: temperature, top-k, top-p, min-p.
//
//   w_i = exp((l_i - max) / T), tokens in descending order of l, equal ones by index; of them stay
//   top-k: the first k; top-p: the shortest run from the front that holds p of top-k's sum; min-p: those with w_i >= min_p
//   token = the first whose running sum exceeds u times the sum of those that stay.
//
// Each filter keeps a run from the front, so what stays is the shortest of the three, and every question (the k-th token,
// the end of top-p's run, the token itself) is one search: the first token whose running count or sum exceeds a target.
// No row is sorted.  The weights are formed in fp64 and summed as 64-bit integers (2^45 for the largest, 2^62 in all),
// so that a sum does not depend on the order, the launch's shape or the atomics that form it, and a border between two
// tokens lies where 64 bits put it.
//
// Many long rows of 16-bit logits: one launch that counts the bit patterns, further below.  Otherwise three steps, of long
// rows a launch each.  Maximum: the slices of a row leave their largest logit.  Histogram: sums (and, under top-k, counts) of
// the weights in bins of 1/32 octave below the maximum; 46 octaves down the weights are 0.  Choice: one workgroup per row adds
// the bins up, which tells in which bins the searches can end, collects those bins' tokens in one pass over the row and
// resolves the searches among them, by further bins over (logit, index) while they are many.
#include "rdkv_common.h"
#include "rope_device.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kOctaves = 46, kPerOctave = 32, kBins = kOctaves * kPerOctave;
constexpr int kMaxSlices = 64;
constexpr int kMaxVocab = 1 << 24;

// Workspace of a row: the slices' maxima, then the histogram.
struct RowSpace {
  float best[kMaxSlices];                // -inf: nothing allowed
  uint64_t least_mass;                   // sum of the weights of at least min_p
  uint64_t pad;
  uint64_t mass[kBins];
  uint32_t count[kBins];
};

struct Settings {
  const float *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  float temperature_value;
  int32_t top_k_value;
  float top_p_value, min_p_value;
};
struct RowSettings { float T, top_p, min_p; int top_k; };
__device__ __forceinline__ RowSettings row_settings(const Settings &s, int row) {
  RowSettings r;
  r.T = s.temperature ? s.temperature[row] : s.temperature_value;
  r.top_k = s.top_k ? s.top_k[row] : s.top_k_value;
  r.top_p = s.top_p ? s.top_p[row] : s.top_p_value;
  r.min_p = s.min_p ? s.min_p[row] : s.min_p_value;
  return r;
}

// A logit and its index as one number in the tokens' order (larger first).
__device__ __forceinline__ uint64_t composite(float l, int index) {
  return ((uint64_t)rdkv_float_to_ordered(l + 0.0f) << 32) | (uint32_t)~index;     // (-0 counts as 0)
}
__device__ __forceinline__ float composite_logit(uint64_t c) { return rdkv_ordered_to_float((uint32_t)(c >> 32)); }
__device__ __forceinline__ int composite_index(uint64_t c) { return (int)~(uint32_t)c; }

// Bins below the maximum, in fp64 (the bin, and the place in it), and the weight there.  Two launches form them and add
// them up to the same sums, bit for bit: nothing is contracted that is not written as fma.
// A logit of +inf counts as the largest number of fp32.
struct Scale { double m, inv; int top; };           // maximum, bins per unit of logit, weight 2^top of the maximum
__device__ __forceinline__ Scale scale_of(float best, float T, int top) {
  return Scale{(double)fminf(best, 3.402823466e38f), fmax(1.44269504088896340736 * kPerOctave / (double)T, 1e-300), top};
}
// NaN for NaN, infinite for -inf, negative for +inf: the caller's comparison and `placed` put these right.
__device__ __forceinline__ double bins_below(const Scale &s, float l) {
#pragma clang fp contract(off)
  return (s.m - (double)l) * s.inv;
}
__device__ __forceinline__ double placed(double t) { return fmax(t, 0.0); }
// 2^(top - t / 32) as an integer: 2^(52 - i / 32) of the bin's place in its octave from the table, times the series of
// 2^(-f / 32) for the rest f < 1 (2e-13 of it left out), added to 2^52 for its bits as an integer, shifted.
__device__ __forceinline__ uint64_t weight(const Scale &s, const double *table, double t) {
#pragma clang fp contract(off)
  constexpr double a = 0.693147180559945309417 / kPerOctave;
  const int bin = (int)t;
  const double f = __builtin_amdgcn_fract(t);
  double p = fma(f, -a * a * a * a * a / 120, a * a * a * a / 24);
  p = fma(f, p, -a * a * a / 6);
  p = fma(f, p, a * a / 2);
  p = fma(f, p, -a);
  p = fma(f, p, 1.0);
  const double sum = fma(p, table[bin & (kPerOctave - 1)], 0x1p52);
  return (__builtin_bit_cast(uint64_t, sum) - 0x4330000000000000ull) >> (52 - s.top + (bin >> 5));
}
__device__ __forceinline__ void fill_table(double *table) {
  if (threadIdx.x < kPerOctave) table[threadIdx.x] = exp2(52.0 - (double)threadIdx.x / kPerOctave);
}

template <int dtype>
struct Row {
  static constexpr int EPP = dtype == RDKV_DTYPE_F32 ? 4 : 8;
  const void *p;
  int vocab, head, pieces;               // elements in front of the first 16-byte border, whole pieces after them
  __device__ __forceinline__ Row(const void *logits, int64_t stride, int row, int n) {
    constexpr int size = dtype == RDKV_DTYPE_F32 ? 4 : 2;
    p = reinterpret_cast<const char *>(logits) + row * stride * size;
    vocab = n;
    head = min((int)((16 - ((uintptr_t)p & 15)) & 15) / size, n);
    pieces = (n - head) / EPP;
  }
  __device__ __forceinline__ float element(int i) const { return rdkv_load_as_float(p, dtype, i); }
  __device__ __forceinline__ u32x4 piece(int i) const {
    constexpr int size = dtype == RDKV_DTYPE_F32 ? 4 : 2;
    return *reinterpret_cast<const u32x4 *>(reinterpret_cast<const char *>(p) + (int64_t)head * size + (int64_t)i * 16);
  }
  __device__ __forceinline__ static float value(u32x4 v, int e) {
    if (dtype == RDKV_DTYPE_F32) return __uint_as_float(v[e]);
    const uint16_t h = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    return dtype == RDKV_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
  }
  // take(value, index, there) for the elements of pieces [begin, end) and, `ends`, those in front of and behind the
  // pieces; every thread makes the same number of calls, in which `there` says whether it has an element.
  template <int THREADS, class F>
  __device__ __forceinline__ void each(int begin, int end, bool ends, F &&take) const {
    constexpr int U = 4;
    for (int i0 = begin; i0 < end; i0 += U * THREADS) {
      u32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * THREADS + (int)threadIdx.x;
        v[u] = piece(i < end ? i : begin);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * THREADS + (int)threadIdx.x;
        if (i0 + u * THREADS < end) {
#pragma unroll
          for (int e = 0; e < EPP; ++e) take(value(v[u], e), head + i * EPP + e, i < end);
        }
      }
    }
    if (ends) {
      const int tail = head + pieces * EPP, n = head + vocab - tail;       // at most 14 elements
      const int i = (int)threadIdx.x < head ? (int)threadIdx.x : tail + (int)threadIdx.x - head;
      const bool there = (int)threadIdx.x < n;
      take(there ? element(i) : 0.0f, i, there);
    }
  }
};

__device__ __forceinline__ uint64_t lesser(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

template <int dtype>
__global__ void __launch_bounds__(256)
sample_max_kernel(const void *__restrict__ logits, int64_t stride, int vocab, RowSpace *__restrict__ space) {
  __shared__ float s_best[4];
  const int slice = blockIdx.x, slices = gridDim.x, tid = threadIdx.x;
  RowSpace &sp = space[blockIdx.y];
  for (int i = slice * 256 + tid; i < kBins; i += slices * 256) {
    sp.mass[i] = 0;
    sp.count[i] = 0;
  }
  if (slice == 0 && tid == 0) sp.least_mass = 0;
  const Row<dtype> row(logits, stride, blockIdx.y, vocab);
  const int per = (row.pieces + slices - 1) / slices, begin = min(slice * per, row.pieces), end = min(begin + per, row.pieces);
  float best = -INFINITY;                // (a NaN is never the larger one)
  row.template each<256>(begin, end, slice == 0, [&](float l, int, bool there) __attribute__((always_inline)) {
    best = fmaxf(best, there ? l : -INFINITY);
  });
  best = rdkv_wave_max(best);
  if ((tid & 63) == 0) s_best[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) sp.best[slice] = fmaxf(fmaxf(s_best[0], s_best[1]), fmaxf(s_best[2], s_best[3]));
}

__device__ __forceinline__ float row_best(const RowSpace &sp, int slices) {
  const int lane = threadIdx.x & 63;
  return rdkv_wave_max(lane < slices ? sp.best[lane] : -INFINITY);
}

// What a row's bins take in: w >= min_p as bins below the maximum; without top-p nobody asks about what lies beyond.
struct BinRule {
  bool counts, least;
  double least_t, need;
  __device__ __forceinline__ explicit BinRule(const RowSettings &set) {
    counts = set.top_k > 0, least = set.min_p > 0.0f;
    least_t = least ? -log2((double)fminf(set.min_p, 1.0f)) * kPerOctave : 0.0;
    need = least && !(set.top_p < 1.0f) ? fmin(least_t + 1.0, (double)kBins) : (double)kBins;
  }
  __device__ __forceinline__ void add(const Scale &sc, const double *table, uint64_t *mass, uint32_t *count, uint64_t &least_mass,
                                      float l, bool there) const {
    double t = bins_below(sc, l);
    if (t < (there ? need : -INFINITY)) {
      t = placed(t);
      const uint64_t w = weight(sc, table, t);
      const int bin = (int)t;
      atomicAdd((unsigned long long *)&mass[bin], (unsigned long long)w);
      if (counts) atomicAdd(&count[bin], 1u);
      if (least && t <= least_t) least_mass += w;
    }
  }
};

template <int dtype>
__global__ void __launch_bounds__(256)
sample_bins_kernel(const void *__restrict__ logits, int64_t stride, int vocab, int top, Settings settings,
                   RowSpace *__restrict__ space) {
  __shared__ uint64_t s_mass[kBins];
  __shared__ uint32_t s_count[kBins];
  __shared__ double s_table[kPerOctave];
  __shared__ uint64_t s_least;
  const int slice = blockIdx.x, slices = gridDim.x, tid = threadIdx.x;
  RowSpace &sp = space[blockIdx.y];
  const float best = row_best(sp, slices);
  const RowSettings set = row_settings(settings, blockIdx.y);
  if (best == -INFINITY || !(set.T > 0.0f)) return;      // nothing allowed, or the largest is the choice
  const BinRule rule(set);
  fill_table(s_table);
  for (int i = tid; i < kBins; i += 256) {
    s_mass[i] = 0;
    s_count[i] = 0;
  }
  if (tid == 0) s_least = 0;
  __syncthreads();
  const Scale sc = scale_of(best, set.T, top);
  const Row<dtype> row(logits, stride, blockIdx.y, vocab);
  const int per = (row.pieces + slices - 1) / slices, begin = min(slice * per, row.pieces), end = min(begin + per, row.pieces);
  uint64_t least_mass = 0;
  row.template each<256>(begin, end, slice == 0, [&](float l, int, bool there) __attribute__((always_inline)) {
    rule.add(sc, s_table, s_mass, s_count, least_mass, l, there);
  });
  if (least_mass) atomicAdd((unsigned long long *)&s_least, (unsigned long long)least_mass);
  __syncthreads();
  for (int i = tid; i < kBins; i += 256) {
    if (s_mass[i]) atomicAdd((unsigned long long *)&sp.mass[i], (unsigned long long)s_mass[i]);
    if (rule.counts && s_count[i]) atomicAdd(&sp.count[i], s_count[i]);
  }
  if (tid == 0 && s_least) atomicAdd((unsigned long long *)&sp.least_mass, (unsigned long long)s_least);
}

struct Advance {                         // rdkv_argmax_advance's counters, of a call of one row
  int64_t *counter_a, *counter_b;
  int32_t *counts;
  int n_counts;
  uint64_t *word;
  uint32_t tag_base;
  const int64_t *uniform_index;
  int n_uniform;
};

constexpr int kList = 4096;              // tokens that the last launch sorts, and pieces that it looks into

struct Choice {                          // LDS of the last launch
  uint64_t mass[kBins + 1];              // sums (counts) in front of a bin, the whole at the end
  uint32_t count[kBins + 1];
  uint64_t list[kList];                  // the tokens of the searches' bins
  uint32_t rank[kList];                  // and how many are in front of each
  union {
    u32x4 piece[kList];                  // pieces of the row that may hold one
    struct { uint64_t before[kList], own[kList]; };      // the sum in front of each token of the list, its weight
  };
  union {
    uint32_t pieces[kList];              // the pieces' numbers
    struct {                             // of the sorted list, where a bin's run starts: its sum and its place
      uint64_t run_mass[kBins];
      uint32_t run_at[kBins];
    };
    struct {                             // further bins of the pass for crowded rows
      uint64_t sub_mass[1024];
      uint32_t sub_count[1024];
    };
  };
  uint64_t part_mass[16];
  uint32_t part_count[16];
  double table[kPerOctave];
  uint64_t lo, hi, found, upto, least;
  float best[16];
  int bin[5], n_pieces, n;
};

// Inclusive sums over the lanes of a wavefront (shifts inside rows of sixteen, then the rows' last lanes handed on).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved64(uint64_t v) {
  return ((uint64_t)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32) | moved<CTRL, ROWS>((uint32_t)v);
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v += moved64<0x111, 0xf>(v);
  v += moved64<0x112, 0xf>(v);
  v += moved64<0x114, 0xf>(v);
  v += moved64<0x118, 0xf>(v);
  v += moved64<0x142, 0xa>(v);
  return v + moved64<0x143, 0xc>(v);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  return v + moved<0x143, 0xc>(v);
}
// The sum over a wavefront, in its last lane (fewer moves than the sums in front of every lane).
template <class T, int CTRL>
__device__ __forceinline__ T partner(T v) {
  if constexpr (sizeof(T) == 8) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)v, CTRL, 0xf, 0xf, true),
                   hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(v >> 32), CTRL, 0xf, 0xf, true);
    return ((uint64_t)hi << 32) | lo;
  } else {
    return (T)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
  }
}
__device__ __forceinline__ uint64_t handed_on(uint64_t v) {
  v += moved64<0x142, 0xa>(v);
  return v + moved64<0x143, 0xc>(v);
}
__device__ __forceinline__ uint32_t handed_on(uint32_t v) {
  v += moved<0x142, 0xa>(v);
  return v + moved<0x143, 0xc>(v);
}
template <class T>
__device__ __forceinline__ T wave_total(T v) {
  v += partner<T, 0xb1>(v);              // pairs, fours, eights, sixteens
  v += partner<T, 0x4e>(v);
  v += partner<T, 0x141>(v);
  v += partner<T, 0x140>(v);
  return handed_on(v);
}
// Sums over the workgroup's threads in front of this one.
__device__ __forceinline__ void block_scan(Choice &s, uint64_t &m, uint32_t &c) {
  const int tid = threadIdx.x, wave = tid >> 6;
  const uint64_t sm = wave_scan(m);
  const uint32_t sc = wave_scan(c);
  if ((tid & 63) == 63) {
    s.part_mass[wave] = sm;
    s.part_count[wave] = sc;
  }
  __syncthreads();
  uint64_t bm = sm - m;
  uint32_t bc = sc - c;
  for (int w = 0; w < wave; ++w) {
    bm += s.part_mass[w];
    bc += s.part_count[w];
  }
  __syncthreads();
  m = bm;
  c = bc;
}

// A place in a list for every lane whose `in` holds (the whole wavefront takes part); *n counts them all.
__device__ __forceinline__ int place_in(int *n, bool in) {
  const uint64_t mask = __ballot(in);
  if (mask == 0) return kList;
  const int lane = threadIdx.x & 63, first = __ffsll((unsigned long long)mask) - 1;
  int at = 0;
  if (lane == first) at = atomicAdd(n, __popcll(mask));
  at = __shfl(at, first, 64) + __popcll(mask & ((1ull << lane) - 1));
  return in ? at : kList;
}

// Logits that can lie in bins [from, to] as a distance from a middle, wide enough for every rounding on the way; what is
// found is tested exactly.
struct Near { float middle, half; };
__device__ __forceinline__ Near near_bins(const Scale &sc, float T, int from, int to) {
  const double w = (double)T * (0.693147180559945309417 / kPerOctave);      // logits a bin
  const double lo = sc.m - ((double)to + 1.001) * w, hi = sc.m - ((double)from - 0.001) * w;
  Near n = {(float)(0.5 * (lo + hi)), (float)(0.5 * (hi - lo))};
  n.half += n.half * 0x1p-20f + fabsf(n.middle) * 0x1p-22f;
  // (+inf counts as the largest number: where that can be in reach, every piece is looked into)
  if (!(fabsf(n.middle) < 1e38f) || !(n.half < 1e38f)) n = Near{0.0f, INFINITY};
  return n;
}

// Targets of the questions.
__device__ __forceinline__ uint64_t top_p_target(float top_p, uint64_t kept) {
  const double want = ceil((double)top_p * (double)kept);
  const uint64_t target = want >= 1.0 ? (uint64_t)want - 1 : 0;
  return target < kept ? target : kept - 1;
}
__device__ __forceinline__ uint64_t token_target(float u, uint64_t run) {
  const double x = (double)u * (double)run;
  const uint64_t target = x > 0.0 ? (x < (double)run ? (uint64_t)x : run - 1) : 0;
  return target < run ? target : run - 1;
}

// Crowded rows (thousands of tokens in the bins of a search: flat rows, equal logits): the first token of `bin` whose running
// count or sum, from the bin's start on, exceeds `target`, by 1024 further bins at a time over the composites of the
// tokens in question, each from a pass over the row.  Composites are distinct and a round leaves at most a 512th of
// their range, so a handful of rounds end at one token.
template <int dtype>
__device__ __forceinline__ void crowded_search(Choice &s, const Row<dtype> &row, const Scale &sc, int bin, bool by_count,
                                               uint64_t target) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint64_t base = s.mass[bin], from = 0, to = ~0ull;
  auto each_in = [&](auto &&take) __attribute__((always_inline)) {
    row.template each<1024>(0, row.pieces, true, [&](float l, int i, bool there) __attribute__((always_inline)) {
      const double t = bins_below(sc, l);
      if (there && t < (double)kBins && (int)placed(t) == bin) {
        const uint64_t c = composite(l, i);
        if (c >= from && c <= to) take(c, placed(t));
      }
    });
  };
  for (;;) {
    if (tid == 0) {
      s.lo = ~0ull;
      s.hi = 0;
    }
    s.sub_mass[tid] = 0;
    s.sub_count[tid] = 0;
    __syncthreads();
    uint64_t lo = ~0ull, hi = 0;
    each_in([&](uint64_t c, double) __attribute__((always_inline)) {
      lo = lesser(lo, c);
      hi = larger(hi, c);
    });
    hi = wave_max64(hi);
    lo = ~wave_max64(~lo);
    if (lane == 0 && hi) {
      atomicMin((unsigned long long *)&s.lo, (unsigned long long)lo);
      atomicMax((unsigned long long *)&s.hi, (unsigned long long)hi);
    }
    __syncthreads();
    from = s.lo;
    to = s.hi;
    if (from >= to) break;
    const int bits = 64 - __clzll((long long)(to - from)), shift = bits > 10 ? bits - 10 : 0;
    each_in([&](uint64_t c, double t) __attribute__((always_inline)) {
      const int sub = (int)((to - c) >> shift);
      atomicAdd((unsigned long long *)&s.sub_mass[sub], (unsigned long long)weight(sc, s.table, t));
      atomicAdd(&s.sub_count[sub], 1u);
    });
    __syncthreads();
    uint64_t m = s.sub_mass[tid];
    uint32_t c = s.sub_count[tid];
    const uint64_t own = by_count ? c : m;
    block_scan(s, m, c);
    const uint64_t before = by_count ? c : m;
    if (before <= target && target < before + own) {
      s.bin[0] = tid;
      s.upto = m;
      s.found = before;
    }
    __syncthreads();
    const uint64_t span = (1ull << shift) - 1;
    to -= (uint64_t)s.bin[0] << shift;
    from = to - from > span ? to - span : from;
    base += s.upto;
    target -= s.found;
    __syncthreads();
  }
  const uint64_t w = weight(sc, s.table, placed(bins_below(sc, composite_logit(from))));
  __syncthreads();
  if (tid == 0) {
    s.found = from;
    s.upto = base + w;
  }
  __syncthreads();
}

template <int N> struct Count { static constexpr int value = N; };

// ALL: of a short row the maximum and the histogram as well.  The three launches of a row of 128256 fp16 logits take 2.8, 5.8 and
// 12.8 us (the pass over the row about 4), of 64 fp32 rows 6.5, 14.4 and 20.2.
template <int dtype, bool ALL>
__global__ void __launch_bounds__(1024)
sample_choose_kernel(const void *__restrict__ logits, int64_t stride, int vocab, int top, int slices, Settings settings,
                     const float *__restrict__ uniform, const RowSpace *__restrict__ space, int64_t *__restrict__ token,
                     float *__restrict__ logprob, Advance adv) {
  extern __shared__ char lds[];
  Choice &s = *reinterpret_cast<Choice *>(lds);
  const int tid = threadIdx.x, r = blockIdx.x;
  const int64_t was_a = adv.counter_a ? adv.counter_a[0] : 0, was_b = adv.counter_b ? adv.counter_b[0] : 0;
  const RowSettings set = row_settings(settings, r);
  int64_t at = r;
  if (adv.uniform_index) at = min(max(adv.uniform_index[0], (int64_t)0), (int64_t)adv.n_uniform - 1);
  const float u = uniform[at];
  const Row<dtype> row(logits, stride, r, vocab);
  // bins 2 tid and 2 tid + 1
  const bool has_bins = 2 * tid < kBins;
  static_assert(kBins % 2 == 0 && kBins <= 2048, "two bins a thread");
  u32x4 masses;
  uint64_t two_counts, least_sum;
  float best;
  if constexpr (ALL) {
    float mine = -INFINITY;
    row.template each<1024>(0, row.pieces, true, [&](float l, int, bool there) __attribute__((always_inline)) {
      mine = fmaxf(mine, there ? l : -INFINITY);
    });
    mine = rdkv_wave_max(mine);
    if ((tid & 63) == 0) s.best[tid >> 6] = mine;
    for (int i = tid; i < kBins; i += 1024) {
      s.mass[i] = 0;
      s.count[i] = 0;
    }
    if (tid == 0) s.least = 0;
    fill_table(s.table);
    __syncthreads();
    best = rdkv_wave_max(s.best[tid & 15]);
    if (best > -INFINITY && set.T > 0.0f) {
      const BinRule rule(set);
      const Scale sc = scale_of(best, set.T, top);
      uint64_t least_mass = 0;
      row.template each<1024>(0, row.pieces, true, [&](float l, int, bool there) __attribute__((always_inline)) {
        rule.add(sc, s.table, s.mass, s.count, least_mass, l, there);
      });
      if (rule.least) {
        least_mass = wave_total(least_mass);
        if ((tid & 63) == 63 && least_mass) atomicAdd((unsigned long long *)&s.least, (unsigned long long)least_mass);
      }
    }
    __syncthreads();
    const int of = has_bins ? 2 * tid : 0;
    masses = u32x4{(uint32_t)s.mass[of], (uint32_t)(s.mass[of] >> 32), (uint32_t)s.mass[of + 1], (uint32_t)(s.mass[of + 1] >> 32)};
    two_counts = s.count[of] | (uint64_t)s.count[of + 1] << 32;
    least_sum = s.least;
  } else {                               // everything that the row's launches left, asked for at once
    const RowSpace &sp = space[r];
    masses = reinterpret_cast<const u32x4 *>(sp.mass)[has_bins ? tid : 0];
    two_counts = reinterpret_cast<const uint64_t *>(sp.count)[has_bins ? tid : 0];
    least_sum = sp.least_mass;
    best = row_best(sp, slices);
    fill_table(s.table);
  }
  int64_t chosen = -1;
  float lp = -INFINITY;
  if (best > -INFINITY && !(set.T > 0.0f)) {             // the first place of the largest
    if (tid == 0) s.n = 0x7fffffff;
    __syncthreads();
    int first = 0x7fffffff;
    row.template each<1024>(0, row.pieces, true, [&](float l, int i, bool there) __attribute__((always_inline)) {
      first = there && l == best ? min(first, i) : first;
    });
    if (first != 0x7fffffff) atomicMin(&s.n, first);
    __syncthreads();
    chosen = s.n;
    lp = 0.0f;
  } else if (best > -INFINITY) {
    const Scale sc = scale_of(best, set.T, top);
    const bool counts = set.top_k > 0;
    if (tid == 0) {
      s.n_pieces = 0;
      s.n = 0;
      s.found = ~0ull;                   // (index 0)
      s.upto = 0;
    }
    // sums and counts in front of the bins: b[0], b[1] of this thread's two, b[2] behind them
    uint64_t mb[3];
    uint32_t cb[3];
    const uint64_t m0 = has_bins ? masses[0] | ((uint64_t)masses[1] << 32) : 0, m1 = has_bins ? masses[2] | ((uint64_t)masses[3] << 32) : 0;
    const uint32_t c0 = has_bins && counts ? (uint32_t)two_counts : 0, c1 = has_bins && counts ? (uint32_t)(two_counts >> 32) : 0;
    mb[0] = m0 + m1;
    cb[0] = c0 + c1;
    block_scan(s, mb[0], cb[0]);
    mb[1] = mb[0] + m0, mb[2] = mb[1] + m1;
    cb[1] = cb[0] + c0, cb[2] = cb[1] + c1;
    if (2 * tid <= kBins) {              // (the thread behind the bins holds the whole sum)
      s.mass[2 * tid] = mb[0];
      s.count[2 * tid] = cb[0];
      if (has_bins) {
        s.mass[2 * tid + 1] = mb[1];
        s.count[2 * tid + 1] = cb[1];
      }
    }
    // the bin where a running sum (count) first exceeds a target that the whole one exceeds
    auto mark = [&](int slot, uint64_t target) __attribute__((always_inline)) {
      if (mb[0] <= target && target < mb[2]) s.bin[slot] = 2 * tid + (target >= mb[1] ? 1 : 0);
    };
    if (counts && cb[0] < (uint32_t)set.top_k && (uint32_t)set.top_k <= cb[2]) s.bin[0] = 2 * tid + ((uint32_t)set.top_k > cb[1] ? 1 : 0);
    __syncthreads();
    const uint64_t total = s.mass[kBins];
    const bool by_k = counts && (uint32_t)set.top_k < s.count[kBins], by_p = set.top_p < 1.0f;     // (behind the bins the weights are 0)
    // In which bins the searches can end: top-k's sum is known to within its bin, and so on.  The first token always stays.
    const uint64_t largest = 1ull << top, least_mass = set.min_p > 0.0f ? larger(least_sum, largest) : ~0ull;
    uint64_t run_lo = total, run_hi = total;
    int from[3] = {1, 1, 1}, to[3] = {0, 0, 0};
    if (by_k) {
      from[0] = to[0] = s.bin[0];
      run_lo = larger(s.mass[from[0]], largest);
      run_hi = s.mass[to[0] + 1];
    }
    if (by_p) {
      mark(1, top_p_target(set.top_p, run_lo));
      mark(2, top_p_target(set.top_p, run_hi));
      __syncthreads();
      from[1] = s.bin[1], to[1] = s.bin[2];
      run_lo = larger(s.mass[from[1]], largest);
      run_hi = lesser(run_hi, s.mass[to[1] + 1]);
    }
    run_lo = lesser(run_lo, least_mass);
    run_hi = lesser(run_hi, least_mass);
    mark(3, token_target(u, run_lo));
    mark(4, token_target(u, run_hi));
    __syncthreads();
    from[2] = s.bin[3], to[2] = s.bin[4];
    // Pieces of the row that may hold a token of these bins: smallest distances from the middles, of the searches that there
    // are (the pass is bound by these: three always took 1.6 us more of the 25 of a row of 128256 under top-p).
    const Near near[3] = {near_bins(sc, set.T, from[2], to[2]), near_bins(sc, set.T, by_p ? from[1] : from[0], by_p ? to[1] : to[0]),
                          near_bins(sc, set.T, from[0], to[0])};
    constexpr int EPP = Row<dtype>::EPP, U = 8;
    auto scan = [&](auto ranges) __attribute__((always_inline)) {
      constexpr int R = decltype(ranges)::value;
      for (int i0 = 0; i0 < row.pieces; i0 += U * 1024) {
        u32x4 v[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int i = i0 + k * 1024 + tid;
          v[k] = row.piece(i < row.pieces ? i : 0);
        }
        uint32_t hits = 0;
#pragma unroll
        for (int k = 0; k < U; ++k) {
          float distance[R];
#pragma unroll
          for (int q = 0; q < R; ++q) distance[q] = INFINITY;
#pragma unroll
          for (int e = 0; e < EPP; ++e) {
            const float l = row.value(v[k], e);
#pragma unroll
            for (int q = 0; q < R; ++q) distance[q] = fminf(distance[q], fabsf(l - near[q].middle));
          }
          bool hit = false;
#pragma unroll
          for (int q = 0; q < R; ++q) hit |= distance[q] <= near[q].half;
          hits |= hit && i0 + k * 1024 + tid < row.pieces ? 1u << k : 0u;
        }
        if (__any(hits != 0)) {          // places in the list for all of the wavefront's pieces at once
          const uint32_t own = __popc(hits), upto = wave_scan(own);
          int at = 0;
          if ((tid & 63) == 63) at = atomicAdd(&s.n_pieces, (int)upto);
          at = __builtin_amdgcn_readlane(at, 63) + (int)(upto - own);
#pragma unroll
          for (int k = 0; k < U; ++k) {
            if ((hits >> k & 1) && at < kList) {
              s.pieces[at] = (uint32_t)(i0 + k * 1024 + tid);
              s.piece[at] = v[k];
            }
            at += hits >> k & 1;
          }
        }
      }
    };
    if (by_k && by_p) scan(Count<3>{});
    else if (by_k || by_p) scan(Count<2>{});
    else scan(Count<1>{});
    __syncthreads();
    // Their tokens in these bins (and those in front of and behind the pieces).
    const int n_pieces = s.n_pieces;
    auto put = [&](float l, int i, bool there) __attribute__((always_inline)) {
      const double t = bins_below(sc, l);
      const int bin = (int)placed(t);
      bool in = false;
#pragma unroll
      for (int k = 0; k < 3; ++k) in |= (bin >= from[k]) & (bin <= to[k]);
      const int at = place_in(&s.n, in && there && t < (double)kBins);
      if (at < kList) s.list[at] = composite(l, i);
    };
    if (n_pieces <= kList) {
      for (int i0 = 0; i0 < n_pieces; i0 += 1024) {
        const bool there = i0 + tid < n_pieces;
        const int q = there ? i0 + tid : 0, i = (int)s.pieces[q];
        const u32x4 v = s.piece[q];
#pragma unroll
        for (int e = 0; e < EPP; ++e) put(row.value(v, e), row.head + i * EPP + e, there);
      }
      const int tail = row.head + row.pieces * EPP, n_ends = row.head + vocab - tail;
      const int i = tid < row.head ? tid : tail + tid - row.head;
      put(tid < n_ends ? row.element(i) : 0.0f, i, tid < n_ends);
    }
    __syncthreads();
    const int n = s.n;
    const bool crowded = n_pieces > kList || n > kList;
    if (n <= 64 && !crowded) {
      // a lane each: a token's bin's sum and count, and those of the bin's tokens in front of it
      if (tid < 64) {
        const uint64_t c = tid < n ? s.list[tid] : 0;
        const double t = placed(bins_below(sc, composite_logit(c)));
        const int bin = tid < n ? (int)t : 0;
        const uint64_t w = weight(sc, s.table, tid < n ? t : 0.0);
        uint64_t before = s.mass[bin];
        uint32_t rank = s.count[bin];
        for (int j = 0; j < n; ++j) {
          auto of = [&](uint64_t x) __attribute__((always_inline)) {
            return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), j) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)x, j);
          };
          const bool front = of(c) > c && __builtin_amdgcn_readlane(bin, j) == bin;
          before += front ? of(w) : 0;
          rank += front ? 1 : 0;
        }
        if (tid < n) {
          s.before[tid] = before;
          s.own[tid] = w;
          s.rank[tid] = rank;
        }
      }
      __syncthreads();
    } else if (!crowded) {
      // The list in descending order: every wavefront sorts 64 tokens in registers (bitonic), then neighbouring runs are merged, a
      // token's new place being its own and the number of the neighbour's in front of it, between two buffers.  Then what lies in
      // front of every token: its bin's, and the bin's tokens in front of it.  (1199 tokens: 8.1 us, 9.5 with
      // four runs at a time, 17.5 with a bitonic sort of all; 594: 4.5, 4.6, 6.6.)
      for (int i0 = 0; i0 < n; i0 += 1024) {
        const int i = i0 + tid;
        if (i - (tid & 63) < n) {
          uint64_t v = i < n ? s.list[i] : 0;            // (no token is 0: they end up behind the others)
          auto with = [&](int k, int j, uint64_t other) __attribute__((always_inline)) {
            v = ((tid & j) == 0) == ((tid & 63 & k) == 0) ? larger(v, other) : lesser(v, other);
          };
#pragma unroll
          for (int k = 2; k <= 64; k *= 2) {
            if (k >= 64) with(k, 32, __shfl_xor(v, 32, 64));
            if (k >= 32) with(k, 16, __shfl_xor(v, 16, 64));
            if (k >= 16) with(k, 8, partner<uint64_t, 0x128>(v));
            if (k >= 8) with(k, 4, partner<uint64_t, 0x1b>(partner<uint64_t, 0x141>(v)));      // 7 ^ 3
            if (k >= 4) with(k, 2, partner<uint64_t, 0x4e>(v));
            with(k, 1, partner<uint64_t, 0xb1>(v));
          }
          if (i < n) s.list[i] = v;
        }
      }
      uint64_t *sorted = s.list, *other = s.before;
      for (int run = 64; run < n; run *= 2) {
        __syncthreads();
        for (int i = tid; i < n; i += 1024) {
          const uint64_t v = sorted[i];
          const int mine = i & -run, next = min(mine ^ run, n), end = min(next + run, n);
          int lo = next, hi = end;                       // the first of the neighbour's that is not in front
          while (lo < hi) {
            const int middle = (lo + hi) / 2;
            if (sorted[middle] > v) lo = middle + 1;
            else hi = middle;
          }
          other[(mine & ~run) + (i - mine) + (lo - next)] = v;
        }
        uint64_t *const was = sorted;
        sorted = other;
        other = was;
      }
      __syncthreads();
      if (sorted != s.list) {
        for (int i = tid; i < n; i += 1024) s.list[i] = sorted[i];
        __syncthreads();
      }
      auto bin_at = [&](int i) __attribute__((always_inline)) { return (int)placed(bins_below(sc, composite_logit(s.list[i]))); };
      const int each = (n + 1023) / 1024, first = tid * each, last = min(first + each, n);
      uint64_t sum = 0;
#pragma unroll 1
      for (int i = first; i < last; ++i) {
        const uint64_t w = weight(sc, s.table, placed(bins_below(sc, composite_logit(s.list[i]))));
        s.own[i] = w;
        sum += w;
      }
      uint32_t unused = 0;
      block_scan(s, sum, unused);
#pragma unroll 1
      for (int i = first; i < last; ++i) {
        const int bin = bin_at(i);
        if (i == 0 || bin_at(i - 1) != bin) {
          s.run_mass[bin] = sum;
          s.run_at[bin] = i;
        }
        s.before[i] = sum;
        sum += s.own[i];
      }
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < n; i += 1024) {
        const int bin = bin_at(i);
        s.before[i] += s.mass[bin] - s.run_mass[bin];
        s.rank[i] = s.count[bin] + (i - s.run_at[bin]);
      }
      __syncthreads();
    }
    uint64_t run = total;                                           // of top-k's run, then of the shortest one
#pragma unroll 1
    for (int question = by_k ? 0 : by_p ? 1 : 2; question < 3; ++question) {
      if (question == 1 && !by_p) continue;
      if (question == 2) run = lesser(run, least_mass);
      const bool by_count = question == 0;
      const uint64_t target = by_count ? (uint64_t)(set.top_k - 1) : question == 1 ? top_p_target(set.top_p, run) : token_target(u, run);
      if (!crowded) {
#pragma unroll 1
        for (int i = tid; i < n; i += 1024) {
          const uint64_t before = s.before[i], w = s.own[i];
          const bool hit = by_count ? s.rank[i] == (uint32_t)target : before <= target && target < before + w;
          if (hit) {
            s.found = s.list[i];
            s.upto = before + w;
          }
        }
      } else {
        const uint64_t t0 = by_count ? cb[0] : mb[0], t1 = by_count ? cb[1] : mb[1], t2 = by_count ? cb[2] : mb[2];
        if (t0 <= target && target < t2) s.bin[0] = 2 * tid + (target >= t1 ? 1 : 0);
        __syncthreads();
        const int bin = s.bin[0];
        __syncthreads();
        crowded_search<dtype>(s, row, sc, bin, by_count, target - (by_count ? s.count[bin] : s.mass[bin]));
      }
      __syncthreads();
      if (question < 2) {
        run = s.upto;
        __syncthreads();
      }
    }
    chosen = composite_index(s.found);
    lp = (float)(-placed(bins_below(sc, composite_logit(s.found))) * (0.693147180559945309417 / kPerOctave) - log(ldexp((double)run, -top)));
  }
  if (tid == 0) {
    token[r] = chosen;
    if (logprob) logprob[r] = lp;
    if (adv.counter_a) {
      adv.counter_a[0] = was_a + 1;
      if (adv.word) rdkv_host_word(adv.word, 0, adv.tag_base + (uint32_t)(was_a + 1), (int32_t)chosen);
    }
    if (adv.counter_b) adv.counter_b[0] = was_b + 1;
  }
  if (tid < adv.n_counts) adv.counts[tid] += 1;
}

// ---- 16-bit logits ----------------------------------------------------------------------------------
// A row of 16-bit logits holds few different values, so one pass that counts them is all that most of the work needs: the
// weight of a value is formed once, sums over values are counts times weights, and the questions are asked of values.
// One workgroup per row, one launch: LDS holds a 16-bit counter for every one of the 2^16 bit patterns (two to a word), in
// the values' order; a thread owns four blocks of 16 neighbouring patterns and forms their sums (smaller blocks share the
// crowded values out over more wavefronts, and cost more sums over the workgroup).  Only the
// token itself needs the row again: the place of its value's n-th occurrence.  A pattern that occurs 2^16 times or more
// shows in the counters' sum; the patterns are then counted again with 32 bits, half of them at a time.  240 rows of 151937
// bf16 logits take 47 us, one of 128256 33: counting 9, the sums over values 9, the rest in steps of 3.
struct Values {                          // LDS
  uint32_t words[1 << 15];               // counter of key k: word_of(k), its half k / 2^15 (or all of it, of one half)
  uint32_t aside[1024];
  uint64_t part_mass[4][16];
  uint32_t part_count[4][16];
  double table[kPerOctave];
  uint64_t least, base_mass, upto;
  uint32_t total, base_count, place, seg_count[18];
  int max_key, skipped, group, key, seg_first[18], index;
};
// Neighbouring keys lie in neighbouring banks, and so do keys 32 apart (a thread reads 16 neighbours).
__device__ __forceinline__ uint32_t word_of(uint32_t key) { return (key & 0x7fffu) ^ ((key >> 5) & 31u); }

template <int dtype>
__global__ void __launch_bounds__(1024)
sample_values_kernel(const void *__restrict__ logits, int64_t stride, int vocab, int top, Settings settings,
                     const float *__restrict__ uniform, int64_t *__restrict__ token, float *__restrict__ logprob, Advance adv) {
  extern __shared__ char lds[];
  Values &s = *reinterpret_cast<Values *>(lds);
  constexpr int kInf = dtype == RDKV_DTYPE_F16 ? 0x7c00 : 0x7f80, U = 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = blockIdx.x;
  const int64_t was_a = adv.counter_a ? adv.counter_a[0] : 0, was_b = adv.counter_b ? adv.counter_b[0] : 0;
  const RowSettings set = row_settings(settings, r);
  int64_t at = r;
  if (adv.uniform_index) at = min(max(adv.uniform_index[0], (int64_t)0), (int64_t)adv.n_uniform - 1);
  const float u = uniform[at];
  const Row<dtype> row(logits, stride, r, vocab);
  // keys: the bit patterns in the order of their values; NaN's lie beyond the infinities'
  auto allowed = [](int key) __attribute__((always_inline)) { return key > 0x7fff - kInf && key <= 0x8000 + kInf; };
  auto value = [](int key) __attribute__((always_inline)) {
    const uint16_t bits = (uint16_t)(key & 0x8000 ? key & 0x7fff : ~key);
    return dtype == RDKV_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, bits) : __uint_as_float((uint32_t)bits << 16);
  };
  // Counts the row: both halves of the keys in 16 bits each, or (half 0 or 1) those of one half in 32.
  auto count = [&](int half) __attribute__((always_inline)) {
    u32x4 *words = reinterpret_cast<u32x4 *>(s.words);
#pragma unroll
    for (int i = 0; i < (1 << 13) / 1024; ++i) words[i * 1024 + tid] = u32x4{0, 0, 0, 0};
    __syncthreads();
    // Masked tokens share one value: a value that an eighth of a wavefront's lanes start with is counted aside, in a word of
    // the lane's own, and left out if it is no number or fills half of the row (rows of 128256 with 99 % masked: 34 us; 250 with
    // their counts added up at one address, beyond the 16 bits of a counter).  Any key will do.
    uint32_t aside = 0;
    bool some = false;
    s.aside[tid] = 0;
    auto one = [&](uint32_t key, bool look_aside) __attribute__((always_inline)) {        // (the upper half is not looked at)
      const uint32_t upper = (key >> 15) & 1;
      const bool common = look_aside && (uint16_t)key == (uint16_t)aside;
      uint32_t *at = common ? &s.aside[tid] : &s.words[word_of(key)];
      if (half < 0) atomicAdd(at, !common && upper ? 0x10000u : 1u);
      else if (common || (int)upper == half) atomicAdd(at, 1u);
    };
    auto keys_of = [&](uint32_t bits) __attribute__((always_inline)) {
      if (half >= 0) {                                                  // (-0 counts as 0)
        if ((bits & 0xffffu) == 0x8000u) bits &= 0xffff0000u;
        if ((bits >> 16) == 0x8000u) bits &= 0xffffu;
      }
      typedef short short2_t __attribute__((ext_vector_type(2)));
      const uint32_t negative = __builtin_bit_cast(uint32_t, __builtin_bit_cast(short2_t, bits) >> (short)15);
      return bits ^ (negative | 0x80008000u);
    };
    for (int i0 = 0; i0 < row.pieces; i0 += U * 1024) {
      u32x4 v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * 1024 + tid;
        v[k] = row.piece(i < row.pieces ? i : 0);
      }
      if (i0 == 0) {
        const uint32_t pair = v[0][0], first = keys_of(pair) & 0xffffu;
        const uint64_t twins = __ballot((first == moved<0xb1, 0xf>(first)) | (first == moved<0x4e, 0xf>(first)) | (first == moved<0x1b, 0xf>(first)));
        if (twins) {                       // lanes of four that start with the same value
          const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)first, __ffsll((unsigned long long)twins) - 1);
          some = __popcll(__ballot(first == key)) >= 8;
          aside = some ? key : 0;
        }
      }
      auto all = [&](bool look_aside) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (i0 + k * 1024 + tid < row.pieces) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t pair = v[k][e], keys = keys_of(pair);
              one(keys, look_aside);
              one(keys >> 16, look_aside);
            }
          }
        }
      };
      if (some) all(true);
      else all(false);
    }
    const int tail = row.head + row.pieces * 8, n_ends = row.head + vocab - tail;
    if (tid < n_ends) {
      uint32_t bits = reinterpret_cast<const uint16_t *>(row.p)[tid < row.head ? tid : tail + tid - row.head];
      if (half >= 0 && bits == 0x8000u) bits = 0;
      one(bits ^ (0x8000u | ((bits >> 15) * 0x7fffu)), true);
    }
    const uint32_t n = wave_total(s.aside[tid]);                        // (the lane's own word, after its own additions)
    if (lane == 63 && n) {
      const uint32_t upper = aside >> 15;
      const bool counts = allowed((int)aside);
      if (half < 0 && (!counts || n >= 4096)) {      // (sixteen of them might not fit a counter)
        atomicAdd(&s.total, n);
        if (counts) atomicMax(&s.skipped, (int)aside);
      } else if (half < 0) {
        atomicAdd(&s.words[word_of(aside)], n << (16 * upper));
      } else if ((int)upper == half) {
        atomicAdd(&s.words[word_of(aside)], n);
      }
    }
    __syncthreads();
  };
  int half = -1;
  auto counter = [&](int key) __attribute__((always_inline)) -> uint32_t {
    const uint32_t w = s.words[word_of(key)];
    return half < 0 ? (key & 0x8000 ? w >> 16 : w & 0xffffu) : (key >> 15) == half ? w : 0;
  };
  fill_table(s.table);
  if (tid == 0) {
    s.least = 0;
    s.total = 0;
    s.max_key = s.skipped = -1;
  }
  count(-1);
  if (tid == 0) {          // -0 joins 0, its neighbour
    uint32_t &minus = s.words[word_of(0x7fff)], &zero = s.words[word_of(0x8000)];
    const uint32_t c = minus & 0xffffu;
    if (c + (zero >> 16) <= 0xffffu) {
      zero += c << 16;
      minus -= c;
    } else {
      s.total += 1;        // (the sum will not be the row's length)
    }
  }
  __syncthreads();
  // Which of the thread's keys occur, the largest of all, and, for the 16-bit counters, the sum of all.  Block b of the thread:
  // keys 16 (tid + 1024 b) and on; the blocks b and b + 2 share their words.
  uint32_t occur[2] = {0, 0};            // blocks b (lower 16 bits) and b + 2
  static_assert(kInf % 16 == 0, "a block's keys are on one side of an infinity, but for itself");
  int max_key = -1;
  auto look = [&]() __attribute__((always_inline)) {
    uint32_t total = 0;
    int largest = -1;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int first = 16 * tid + 16384 * b;
      uint32_t there = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t w = s.words[word_of(first + j)];
        typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
        if (half < 0) {
          total = __builtin_amdgcn_sad_u16(w, 0u, total);
          there |= __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(ushort2_t, w), ushort2_t{1, 1})) << j;
        } else {
          there |= min(w, 1u) << (j + 16 * half);
        }
      }
      if (first < 0x8000 - kInf) there &= 0xffff0000u;         // -inf and the NaN's behind it
      if (first >= kInf) there &= first == kInf ? 0x1ffffu : 0xffffu;
      occur[b] = there;
      if (there >> 16) largest = max(largest, 0x8000 + first + 15 - __clz((int)(there & 0xffff0000u)));
      if (there & 0xffffu) largest = max(largest, first + 31 - __clz((int)(there & 0xffffu)));
    }
    if (half < 0) {
      total = wave_total(total);
      if (lane == 63) atomicAdd(&s.total, total);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) largest = max(largest, __shfl_xor(largest, o, 64));
    if (lane == 0) atomicMax(&s.max_key, largest);
    __syncthreads();
    max_key = s.max_key;
  };
  Scale sc = {0.0, 0.0, top};
  const bool least_on = set.min_p > 0.0f;
  const double least_t = least_on ? -log2((double)fminf(set.min_p, 1.0f)) * kPerOctave : -1.0;
  // A weight times a count: below 2^63, the count below 2^24.
  auto times = [](uint64_t w, uint32_t c) __attribute__((always_inline)) {
    return (uint64_t)(uint32_t)w * c + ((uint64_t)((uint32_t)(w >> 32) * c) << 32);
  };
  // Sums of the thread's blocks; keys beyond the last bin have no weight and are not counted.
  uint64_t own[4] = {0, 0, 0, 0}, least = 0;
  uint32_t own_n[4] = {0, 0, 0, 0};
  auto sums = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      uint64_t mass = 0;
      uint32_t n = 0;
#pragma unroll 1
      for (uint32_t left = b < 2 ? occur[b] & 0xffffu : occur[b - 2] >> 16; left; left &= left - 1) {
        const int k = 16 * (tid + 1024 * b) + __ffs((int)left) - 1;
        const double t = bins_below(sc, value(k));
        if (t < (double)kBins) {
          const uint32_t c = counter(k);
          const uint64_t m = times(weight(sc, s.table, placed(t)), c);
          mass += m;
          n += c;
          least += t <= least_t ? m : 0;
        }
      }
      own[b] += mass;
      own_n[b] += n;
    }
  };
  const bool greedy = !(set.T > 0.0f);
  look();
  bool wide = s.total != (uint32_t)vocab;
  const int skipped = s.skipped;         // the largest value that was left out: it has to have no weight
  if (skipped >= 0)
    wide |= max_key <= skipped || (!greedy && bins_below(scale_of(value(max_key), set.T, top), value(skipped)) < (double)kBins);
  if (wide) {
    __syncthreads();
    if (tid == 0) s.max_key = -1;
    half = 1;
  }
#pragma unroll 1
  for (;;) {               // once, or the upper half's and the lower half's keys one after the other
    if (wide) {
      count(half);
      look();
    }
    if (max_key >= 0 && !greedy) {
      sc = scale_of(value(max_key), set.T, top);
      sums();
    }
    if (half <= 0) break;
    __syncthreads();
    half = 0;
  }
  if (least_on) {
    least = wave_total(least);
    if (lane == 63 && least) atomicAdd((unsigned long long *)&s.least, (unsigned long long)least);
  }
  __syncthreads();
  int64_t chosen = -1;
  float lp = -INFINITY;
  int key = max_key;
  uint32_t place = 0;
  if (max_key >= 0 && greedy) lp = 0.0f;
  if (max_key >= 0 && !greedy) {
    // sums in front of this thread's blocks, from the top: those behind them in the keys' order, the upper blocks first
    uint64_t before[4], total = 0;
    uint32_t before_n[4], total_n = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      before[b] = wave_scan(own[b]);
      before_n[b] = wave_scan(own_n[b]);
      if (lane == 63) {
        s.part_mass[b][wave] = before[b];
        s.part_count[b][wave] = before_n[b];
      }
    }
    __syncthreads();
    const uint64_t least_sum = s.least;
#pragma unroll
    for (int b = 3; b >= 0; --b) {
      const uint64_t m = wave_scan(lane < 16 ? s.part_mass[b][lane & 15] : 0);
      const uint32_t c = wave_scan(lane < 16 ? s.part_count[b][lane & 15] : 0u);
      auto upto = [&](int w) __attribute__((always_inline)) {
        return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(m >> 32), w) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)m, w);
      };
      const int w = wave ? wave - 1 : 0;
      total += upto(15);
      total_n += (uint32_t)__builtin_amdgcn_readlane((int)c, 15);
      before[b] = total - before[b] - (wave ? upto(w) : 0);
      before_n[b] = total_n - before_n[b] - (wave ? (uint32_t)__builtin_amdgcn_readlane((int)c, w) : 0);
    }
    const bool by_k = set.top_k > 0 && (uint32_t)set.top_k < total_n, by_p = set.top_p < 1.0f;
    const uint64_t largest = 1ull << top, least_mass = least_on ? larger(least_sum, largest) : ~0ull;
    uint64_t run = total;                // of top-k's run, then of the shortest one
#pragma unroll 1
    for (int question = by_k ? 0 : by_p ? 1 : 2; question < 3; ++question) {
      if (question == 1 && !by_p) continue;
      if (question == 2) run = lesser(run, least_mass);
      const bool by_count = question == 0;
      const uint64_t target = by_count ? (uint64_t)(set.top_k - 1) : question == 1 ? top_p_target(set.top_p, run) : token_target(u, run);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint64_t f = by_count ? before_n[b] : before[b], o = by_count ? own_n[b] : own[b];
        if (f <= target && target < f + o) {
          s.group = 1024 * b + tid;
          s.base_mass = before[b];
          s.base_count = before_n[b];
        }
      }
      __syncthreads();
      const int group = s.group;
      if (wide && (group >> 11) != half) {
        half = group >> 11;
        count(half);
      }
      if (wave == 0) {                   // the block's keys from the top
        const int k = group * 16 + 15 - (lane & 15);
        const double t = bins_below(sc, value(k));
        const bool in = lane < 16 && allowed(k) && t < (double)kBins;
        const uint32_t c = in ? counter(k) : 0;
        const uint64_t w = weight(sc, s.table, in ? placed(t) : 0.0), m = times(w, c);
        const uint64_t front = s.base_mass + wave_scan(m) - m;
        const uint32_t front_n = s.base_count + wave_scan(c) - c;
        const uint64_t f = by_count ? front_n : front, over = target - f;
        if (f <= target && over < (by_count ? (uint64_t)c : m)) {
          uint64_t n = over;
          if (!by_count) {               // the quotient of two integers below 2^62 that is below 2^24
            n = (uint64_t)((double)over / (double)w);
            if (n * w > over) --n;
            else if ((n + 1) * w <= over) ++n;
          }
          s.key = k;
          s.place = (uint32_t)n;
          s.upto = front + (n + 1) * w;
        }
      }
      __syncthreads();
      if (question < 2) run = s.upto;
    }
    key = s.key;
    place = s.place;
    lp = (float)(-placed(bins_below(sc, value(key))) * (0.693147180559945309417 / kPerOctave) - log(ldexp((double)run, -top)));
  }
  if (key >= 0) {
    // The place-th occurrence of the value: the elements in front of the pieces, sixteen runs of pieces, the rest.
    const uint32_t bits = key & 0x8000 ? key & 0x7fff : ~key & 0xffff;
    const uint32_t seen = bits == 0 ? 0x7fff7fffu : ~0u, pair = bits * 0x10001u;        // (0 in both its forms)
    const int run = (row.pieces + 15) / 16, begin = min(wave * run, row.pieces), end = min(begin + run, row.pieces);
    auto matches = [&](u32x4 v) __attribute__((always_inline)) {
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = (v[e] & seen) ^ pair;
        hits |= (x & 0xffffu) == 0 ? 1u << (2 * e) : 0u;
        hits |= (x >> 16) == 0 ? 2u << (2 * e) : 0u;
      }
      return hits;
    };
    uint32_t n = 0;
    int first = 0x7fffffff;
    for (int i0 = begin; i0 < end; i0 += U * 64) {
      u32x4 v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * 64 + lane;
        v[k] = row.piece(i < end ? i : begin);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * 64 + lane;
        const uint32_t hits = i < end ? matches(v[k]) : 0;
        if (hits) {
          n += __popc(hits);
          first = min(first, row.head + i * 8 + __ffs(hits) - 1);
        }
      }
    }
    n = wave_scan(n);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
    if (lane == 63) {
      s.seg_count[1 + wave] = n;
      s.seg_first[1 + wave] = first;
    }
    const int tail = row.head + row.pieces * 8, n_tail = vocab - tail;
    uint64_t ends = 0;                   // which of these elements match (at most seven; wavefronts 0 and 1)
    if (wave < 2) {
      const int m = wave == 0 ? row.head : n_tail, i = wave == 0 ? lane : tail + lane;
      const uint32_t x = lane < m ? reinterpret_cast<const uint16_t *>(row.p)[i] : 0;
      ends = __ballot(lane < m && ((x & seen & 0xffffu) == bits));
      if (lane == 0) s.seg_count[17 * wave] = __popcll(ends);
    }
    __syncthreads();
    const uint32_t of = lane < 18 ? s.seg_count[lane] : 0, behind = wave_scan(of);
    const uint64_t mine = __ballot(lane < 18 && behind > place);
    const int seg = mine ? __ffsll((unsigned long long)mine) - 1 : 17;
    uint32_t left = place - (uint32_t)__shfl((int)(behind - of), seg, 64);
    if (seg == 0 || seg == 17) {
      if (wave == (seg == 17)) {
        for (uint32_t q = 0; q < left; ++q) ends &= ends - 1;
        if (lane == 0) s.index = (seg == 0 ? 0 : tail) + __ffsll((unsigned long long)ends) - 1;
      }
    } else if (seg == 1 + wave) {
      if (left == 0) {
        if (lane == 0) s.index = s.seg_first[seg];
      } else {
        for (int i0 = begin; i0 < end; i0 += 64) {
          const int i = i0 + lane;
          uint32_t hits = i < end ? matches(row.piece(i)) : 0;
          const uint32_t own = __popc(hits), upto = wave_scan(own), all = (uint32_t)__shfl((int)upto, 63, 64);
          if (left < all) {
            if (upto - own <= left && left < upto) {
              for (uint32_t q = upto - own; q < left; ++q) hits &= hits - 1;
              s.index = row.head + i * 8 + __ffs(hits) - 1;
            }
            break;
          }
          left -= all;
        }
      }
    }
    __syncthreads();
    chosen = s.index;
  }
  if (tid == 0) {
    token[r] = chosen;
    if (logprob) logprob[r] = lp;
    if (adv.counter_a) {
      adv.counter_a[0] = was_a + 1;
      if (adv.word) rdkv_host_word(adv.word, 0, adv.tag_base + (uint32_t)(was_a + 1), (int32_t)chosen);
    }
    if (adv.counter_b) adv.counter_b[0] = was_b + 1;
  }
  if (tid < adv.n_counts) adv.counts[tid] += 1;
}

int weight_bits(int vocab) {             // of the largest weight: all of them together stay below 2^63
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  return 62 - bits < 45 ? 62 - bits : 45;
}

// Slices of a row: about four workgroups per compute unit over the rows, none of less than 256 pieces.
int slices_of(int rows, int vocab, int elements) {
  const int pieces = vocab / elements;
  const int want = (int)rdkv_cdiv(1024, rows), most = (int)rdkv_cdiv(pieces, 256);
  int s = want < most ? want : most;
  s = s < kMaxSlices ? s : kMaxSlices;
  return s < 1 ? 1 : s;
}

// Short rows: all three steps in one launch of a workgroup a row.  One / the others, us, 1 row and 240 rows: fp16, 1000 logits 13.7 /
// 19.1 and 16.4 / 20.5, 16000 18.6 / 20.2 and 23.3 / 25.4, 32000 23.1 / 20.5 and 29.3 / 27.8; fp32, 1000 logits 11.4 / 16.1 and
// 14.4 / 19.7, 16000 16.6 / 18.0 and 21.9 / 31.7, 32000 21.2 / 18.8 and 29.2 / 38.5.
bool in_one(int vocab) { return vocab <= 16384; }
// A few rows of 16-bit logits leave most compute units idle with one workgroup a row.  Slices / values, us, without masks and with
// 99 % masked: 128256 fp16 logits, 8 rows 30 / 37 and 24 / 34, 24 rows 35 / 37 and 27 / 34, 48 rows 41 / 38 and 31 / 35; 32000 bf16
// logits, 8 rows 22 / 26 and 20 / 24, 48 rows 28 / 27 and 22 / 25.
bool by_slices(int rows, int vocab, int dtype) { return !in_one(vocab) && (dtype == RDKV_DTYPE_F32 || rows <= 24); }

template <int dtype>
int launch_sample(const char *fn, const void *logits, int64_t stride, int rows, int vocab, const Settings &set, const float *uniform,
                  int64_t *token, float *logprob, const Advance &adv, RowSpace *space, hipStream_t s) {
  const bool one = in_one(vocab), slices_first = by_slices(rows, vocab, dtype);
  const int slices = slices_of(rows, vocab, Row<dtype>::EPP), top = weight_bits(vocab);
  for (int r = 0; r < rows; r += 65535) {                  // (a grid's second dimension)
    const int n = rows - r < 65535 ? rows - r : 65535;
    const void *from = reinterpret_cast<const char *>(logits) + (int64_t)r * stride * (dtype == RDKV_DTYPE_F32 ? 4 : 2);
    Settings part = set;
    if (part.temperature) part.temperature += r;
    if (part.top_k) part.top_k += r;
    if (part.top_p) part.top_p += r;
    if (part.min_p) part.min_p += r;
    float *lp = logprob ? logprob + r : nullptr;
    if (one) {
      hipLaunchKernelGGL((sample_choose_kernel<dtype, true>), dim3(n), dim3(1024), sizeof(Choice), s, from, stride, vocab, top, 0, part,
                         uniform + r, nullptr, token + r, lp, adv);
    } else if (slices_first) {
      hipLaunchKernelGGL(sample_max_kernel<dtype>, dim3(slices, n), dim3(256), 0, s, from, stride, vocab, space + r);
      RDKV_CHECK_LAUNCH(fn);
      hipLaunchKernelGGL(sample_bins_kernel<dtype>, dim3(slices, n), dim3(256), 0, s, from, stride, vocab, top, part, space + r);
      RDKV_CHECK_LAUNCH(fn);
      hipLaunchKernelGGL((sample_choose_kernel<dtype, false>), dim3(n), dim3(1024), sizeof(Choice), s, from, stride, vocab, top, slices, part,
                         uniform + r, space + r, token + r, lp, adv);
    } else if constexpr (dtype != RDKV_DTYPE_F32) {
      hipLaunchKernelGGL(sample_values_kernel<dtype>, dim3(n), dim3(1024), sizeof(Values), s, from, stride, vocab, top, part, uniform + r,
                         token + r, lp, adv);
    }
    RDKV_CHECK_LAUNCH(fn);
  }
  return RDKV_OK;
}

int sample(const char *fn, const void *logits, int64_t stride, int rows, int vocab, int dtype, const float *uniform,
           const RdkvSampling *sampling, int64_t *token, float *logprob, const Advance &adv, void *workspace,
           int64_t workspace_bytes, void *stream) {
  RDKV_REQUIRE(rows >= 0 && vocab >= 1 && vocab <= kMaxVocab, "%s: %d rows of %d logits", fn, rows, vocab);
  RDKV_REQUIRE(dtype >= 0 && dtype <= 2, "%s: unknown dtype %d", fn, dtype);
  RDKV_REQUIRE(sampling, "%s: no settings", fn);
  if (rows == 0) return RDKV_OK;
  RDKV_REQUIRE(logits && uniform && token, "%s: null pointer", fn);
  RDKV_REQUIRE(stride >= 0 && ((uintptr_t)logits % (dtype == RDKV_DTYPE_F32 ? 4 : 2)) == 0, "%s: bad rows", fn);
  const int64_t need = rdkv_sample_workspace_bytes(rows, vocab, dtype);
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16 != 0)) {
    rdkv_set_error("%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)need);
    return RDKV_EWORKSPACE;
  }
  const Settings set = {sampling->temperature, sampling->top_k, sampling->top_p, sampling->min_p,
                        sampling->temperature_value, sampling->top_k_value, sampling->top_p_value, sampling->min_p_value};
  auto *launch = dtype == RDKV_DTYPE_F32 ? launch_sample<RDKV_DTYPE_F32>
                 : dtype == RDKV_DTYPE_F16 ? launch_sample<RDKV_DTYPE_F16> : launch_sample<RDKV_DTYPE_BF16>;
  return launch(fn, logits, stride, rows, vocab, set, uniform, token, logprob, adv, reinterpret_cast<RowSpace *>(workspace),
                (hipStream_t)stream);
}

}  // namespace

RDKV_API int64_t rdkv_sample_workspace_bytes(int rows, int vocab, int dtype) {
  return rows <= 0 || !by_slices(rows, vocab, dtype) ? 0 : (int64_t)rows * (int64_t)sizeof(RowSpace);
}

RDKV_API int rdkv_sample_rows(const void *logits, int64_t stride_row, int rows, int vocab, int dtype,
                              const float *uniform, const RdkvSampling *sampling, int64_t *token, float *logprob,
                              void *workspace, int64_t workspace_bytes, void *stream) {
  const Advance none = {};
  return sample("rdkv_sample_rows", logits, stride_row, rows, vocab, dtype, uniform, sampling, token, logprob, none,
                workspace, workspace_bytes, stream);
}

RDKV_API int rdkv_sample_advance(const void *logits, int vocab, int dtype, const float *uniform, int n_uniform,
                                 const int64_t *uniform_index, const RdkvSampling *sampling, int64_t *token,
                                 int64_t *counter_a, int64_t *counter_b, int32_t *counts, int n_counts, uint64_t *word,
                                 uint32_t tag_base, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *fn = "rdkv_sample_advance";
  RDKV_REQUIRE(n_uniform >= 1 && uniform_index, "%s: needs uniforms and their index", fn);
  RDKV_REQUIRE(n_counts >= 0 && n_counts <= 1024 && (n_counts == 0 || counts), "%s: bad counts", fn);
  RDKV_REQUIRE(!word || counter_a, "%s: a host word is tagged with the first counter", fn);
  const Advance adv = {counter_a, counter_b, counts, n_counts, word, tag_base, uniform_index, n_uniform};
  return sample(fn, logits, vocab, 1, vocab, dtype, uniform, sampling, token, nullptr, adv, workspace, workspace_bytes, stream);
}
