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
// Three launches.  Maximum: the slices of a row leave their largest logit and its place.  Histogram: sums (and, under top-k,
// counts) of the weights in bins of 1/32 octave below the maximum; 46 octaves down the weights are 0.  Choice: one workgroup
// per row adds the bins up, finds a search's bin, collects the bin's tokens from the row and resolves them, by
// further bins over (logit, index) while they are many.
#include "rdkv_common.h"
#include "rope_device.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kOctaves = 46, kPerOctave = 32, kBins = kOctaves * kPerOctave;
constexpr int kMaxSlices = 64;
constexpr int kMaxVocab = 1 << 24;
constexpr int kList = 2048;              // tokens of a bin that LDS holds

// Workspace of a row: the slices' maxima, then the histogram.
struct RowSpace {
  uint64_t best[kMaxSlices];             // ordered logit << 32 | ~index, 0: nothing allowed
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

// A logit and its index as one number in the tokens' order (larger first); 0 where the token is masked (-inf, NaN).
__device__ __forceinline__ uint64_t composite(float l, int index) {
  if (!(l > -INFINITY)) return 0;
  return ((uint64_t)rdkv_float_to_ordered(l + 0.0f) << 32) | (uint32_t)~index;     // (-0 counts as 0)
}
__device__ __forceinline__ float composite_logit(uint64_t c) { return rdkv_ordered_to_float((uint32_t)(c >> 32)); }
__device__ __forceinline__ int composite_index(uint64_t c) { return (int)~(uint32_t)c; }

// Octaves below the maximum, in fp64; bin and weight of a token.  Two launches form them and add them up to the same
// sums, bit for bit: nothing is contracted that is not written as fma.
struct Scale { float m; double inv; int top; };     // maximum, log2(e) / T, weight 2^top of the maximum
__device__ __forceinline__ double octaves(const Scale &s, float l) {
#pragma clang fp contract(off)
  return l == s.m ? 0.0 : ((double)s.m - (double)l) * s.inv;
}
// 2^-t as an integer: 2^-(bin / 32) from the table, the rest by its series (within 2e-13)
__device__ __forceinline__ uint64_t weight(const Scale &s, const double *table, double t) {
#pragma clang fp contract(off)
  const int bin = (int)(t * kPerOctave);
  const double y = (t - bin * (1.0 / kPerOctave)) * 0.693147180559945309417;
  double p = fma(y, -1.0 / 120, 1.0 / 24);
  p = fma(y, p, -1.0 / 6);
  p = fma(y, p, 0.5);
  p = fma(y, p, -1.0);
  p = fma(y, p, 1.0) * table[bin & (kPerOctave - 1)];
  return (uint64_t)ldexp(p, s.top - (bin >> 5));
}
__device__ __forceinline__ void fill_table(double *table) {
  if (threadIdx.x < kPerOctave) table[threadIdx.x] = exp2(-(double)threadIdx.x / kPerOctave);
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
  __shared__ uint64_t s_best[4];
  const int slice = blockIdx.x, slices = gridDim.x, tid = threadIdx.x;
  RowSpace &sp = space[blockIdx.y];
  for (int i = slice * 256 + tid; i < kBins; i += slices * 256) {
    sp.mass[i] = 0;
    sp.count[i] = 0;
  }
  if (slice == 0 && tid == 0) sp.least_mass = 0;
  const Row<dtype> row(logits, stride, blockIdx.y, vocab);
  const int per = (row.pieces + slices - 1) / slices, begin = min(slice * per, row.pieces), end = min(begin + per, row.pieces);
  uint64_t best = 0;
  row.template each<256>(begin, end, slice == 0, [&](float l, int i, bool there) __attribute__((always_inline)) {
    const uint64_t c = there ? composite(l, i) : 0;
    best = best > c ? best : c;
  });
  best = wave_max64(best);
  if ((tid & 63) == 0) s_best[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 4; ++w) best = best > s_best[w] ? best : s_best[w];
    sp.best[slice] = best;
  }
}

__device__ __forceinline__ uint64_t row_best(const RowSpace &sp, int slices) {
  const int lane = threadIdx.x & 63;
  return wave_max64(lane < slices ? sp.best[lane] : 0);
}

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
  const uint64_t best = row_best(sp, slices);
  const RowSettings set = row_settings(settings, blockIdx.y);
  if (best == 0 || !(set.T > 0.0f)) return;              // nothing allowed, or the largest is the choice
  const bool counts = set.top_k > 0, least = set.min_p > 0.0f;
  fill_table(s_table);
  for (int i = tid; i < kBins; i += 256) {
    s_mass[i] = 0;
    s_count[i] = 0;
  }
  if (tid == 0) s_least = 0;
  __syncthreads();
  const Scale sc = {composite_logit(best), 1.44269504088896340736 / (double)set.T, top};
  const double least_w = (double)set.min_p * ldexp(1.0, top);
  const Row<dtype> row(logits, stride, blockIdx.y, vocab);
  const int per = (row.pieces + slices - 1) / slices, begin = min(slice * per, row.pieces), end = min(begin + per, row.pieces);
  uint64_t least_mass = 0;
  row.template each<256>(begin, end, slice == 0, [&](float l, int i, bool there) __attribute__((always_inline)) {
    const double t = octaves(sc, l);
    if (there && l > -INFINITY && t < (double)kOctaves) {
      const uint64_t w = weight(sc, s_table, t);
      const int bin = (int)(t * kPerOctave);
      atomicAdd((unsigned long long *)&s_mass[bin], (unsigned long long)w);
      if (counts) atomicAdd(&s_count[bin], 1u);
      if (least && (double)w >= least_w) least_mass += w;
    }
  });
  if (least && least_mass) atomicAdd((unsigned long long *)&s_least, (unsigned long long)least_mass);
  __syncthreads();
  for (int i = tid; i < kBins; i += 256) {
    if (s_mass[i]) atomicAdd((unsigned long long *)&sp.mass[i], (unsigned long long)s_mass[i]);
    if (counts && s_count[i]) atomicAdd(&sp.count[i], s_count[i]);
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

struct Choice {                          // LDS of the last launch
  uint64_t mass[kBins + 1];              // sums in front of a bin, the whole sum at the end
  uint32_t count[kBins + 1];
  uint64_t sub_mass[1024];
  uint32_t sub_count[1024];
  uint64_t list[2][kList];
  uint64_t part_mass[16];
  uint32_t part_count[16];
  double table[kPerOctave];
  uint64_t lo, hi, found, upto;
  int bin, n;
};

// Sums in front of each of N entries (N at most 2048: two a thread), in place; [N] takes the whole.
template <int N>
__device__ __forceinline__ void prefix(uint64_t *mass, uint32_t *count, Choice &s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int i0 = 2 * tid, i1 = i0 + 1;
  uint64_t m0 = i0 < N ? mass[i0] : 0, m1 = i1 < N ? mass[i1] : 0;
  uint32_t c0 = i0 < N ? count[i0] : 0, c1 = i1 < N ? count[i1] : 0;
  uint64_t m = m0 + m1;
  uint32_t c = c0 + c1;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t um = __shfl_up(m, o, 64);
    const uint32_t uc = __shfl_up(c, o, 64);
    if (lane >= o) {
      m += um;
      c += uc;
    }
  }
  if (lane == 63) {
    s.part_mass[wave] = m;
    s.part_count[wave] = c;
  }
  __syncthreads();
  uint64_t bm = m - m0 - m1;
  uint32_t bc = c - c0 - c1;
  for (int w = 0; w < wave; ++w) {
    bm += s.part_mass[w];
    bc += s.part_count[w];
  }
  if (i0 < N) { mass[i0] = bm; count[i0] = bc; }
  if (i1 < N) { mass[i1] = bm + m0; count[i1] = bc + c0; }
  __syncthreads();
}

// The first token, in the tokens' order, whose running count (by_count) or sum exceeds `target`, and the sum up to and
// with it; the bins' own totals exceed the target.  All threads of the workgroup take part.
template <int dtype>
__device__ void search(Choice &s, const Row<dtype> &row, const Scale &sc, bool by_count, uint64_t target) {
  const int tid = threadIdx.x;
  for (int i = tid; i < kBins; i += 1024) {
    const uint64_t a = by_count ? s.count[i] : s.mass[i], b = by_count ? s.count[i + 1] : s.mass[i + 1];
    if (a <= target && target < b) s.bin = i;            // (one bin only)
  }
  if (tid == 0) {
    s.n = 0;
    s.lo = ~0ull;
    s.hi = 0;
  }
  __syncthreads();
  const int bin = s.bin;
  uint64_t base = s.mass[bin];
  target -= by_count ? s.count[bin] : base;
  // the bin's tokens: a cheap test in fp32 (a thousandth of a bin off at most) in front of the exact one
  const float inv32 = (float)(sc.inv * kPerOctave), from = bin - 0.1f, to = bin + 1.1f;
  // (not where the factor leaves fp32, or a difference could that is fewer than 46 octaves)
  const bool coarse = sc.inv < 1e30 && sc.inv > 1e-30;
  const int lane = tid & 63;
  auto in_bin = [&](float l, bool there) __attribute__((always_inline)) {
    if (!there || !(l > -INFINITY)) return false;
    const float tf = (sc.m - l) * inv32;
    if (coarse && (tf < from || tf > to)) return false;
    const double t = octaves(sc, l);
    return t < (double)kOctaves && (int)(t * kPerOctave) == bin;
  };
  auto append = [&](uint64_t *list, bool in, uint64_t c) __attribute__((always_inline)) {
    const uint64_t mask = __ballot(in);
    if (mask == 0) return;
    int at = 0;
    if (lane == __ffsll((unsigned long long)mask) - 1) at = atomicAdd(&s.n, __popcll(mask));
    at = __shfl(at, __ffsll((unsigned long long)mask) - 1, 64) + __popcll(mask & ((1ull << lane) - 1));
    if (in && at < kList) list[at] = c;
  };
  auto bounds = [&](uint64_t lo, uint64_t hi) __attribute__((always_inline)) {
    hi = wave_max64(hi);
    lo = ~wave_max64(~lo);
    if (lane == 0 && hi) {
      atomicMin((unsigned long long *)&s.lo, (unsigned long long)lo);
      atomicMax((unsigned long long *)&s.hi, (unsigned long long)hi);
    }
  };
  {
    uint64_t lo = ~0ull, hi = 0;
    row.template each<1024>(0, row.pieces, true, [&](float l, int i, bool there) __attribute__((always_inline)) {
      const bool in = in_bin(l, there);
      const uint64_t c = in ? composite(l, i) : 0;
      if (in) {
        lo = lo < c ? lo : c;
        hi = hi > c ? hi : c;
      }
      append(s.list[0], in, c);
    });
    bounds(lo, hi);
  }
  __syncthreads();
  int n = s.n, from_list = 0;
  bool listed = n <= kList;
  while (n > 64) {
    // 1024 further bins over the range that the tokens take; every round leaves at most a 512th of it, and
    // composites are distinct, so few rounds leave few tokens
    const uint64_t lo = s.lo, hi = s.hi;
    const int bits = 64 - __clzll((long long)(hi - lo)), shift = bits > 10 ? bits - 10 : 0;
    s.sub_mass[tid] = 0;
    s.sub_count[tid] = 0;
    __syncthreads();
    if (tid == 0) {
      s.n = 0;
      s.lo = ~0ull;
      s.hi = 0;
    }
    auto add = [&](uint64_t c) __attribute__((always_inline)) {
      const int sub = (int)((hi - c) >> shift);
      atomicAdd((unsigned long long *)&s.sub_mass[sub], (unsigned long long)weight(sc, s.table, octaves(sc, composite_logit(c))));
      atomicAdd(&s.sub_count[sub], 1u);
    };
    if (listed) {
      for (int i = tid; i < n; i += 1024) add(s.list[from_list][i]);
    } else {
      row.template each<1024>(0, row.pieces, true, [&](float l, int i, bool there) __attribute__((always_inline)) {
        if (in_bin(l, there)) {
          const uint64_t c = composite(l, i);
          if (c >= lo && c <= hi) add(c);
        }
      });
    }
    __syncthreads();
    const uint64_t own_mass = s.sub_mass[tid];
    const uint32_t own_count = s.sub_count[tid];
    __syncthreads();
    prefix<1024>(s.sub_mass, s.sub_count, s);
    const uint64_t a = by_count ? s.sub_count[tid] : s.sub_mass[tid], more = by_count ? own_count : own_mass;
    if (a <= target && target < a + more) s.bin = tid;
    __syncthreads();
    const int sub = s.bin;
    const uint64_t new_hi = hi - ((uint64_t)sub << shift), span = ((1ull << shift) - 1);
    const uint64_t new_lo = new_hi - lo > span ? new_hi - span : lo;
    target -= by_count ? s.sub_count[sub] : s.sub_mass[sub];
    base += s.sub_mass[sub];
    {
      uint64_t low = ~0ull, high = 0;
      auto keep = [&](bool in, uint64_t c) __attribute__((always_inline)) {
        in = in && c >= new_lo && c <= new_hi;
        if (in) {
          low = low < c ? low : c;
          high = high > c ? high : c;
        }
        append(s.list[from_list ^ 1], in, c);
      };
      if (listed) {
        for (int i0 = 0; i0 < n; i0 += 1024) {
          const int i = i0 + tid;
          keep(i < n, i < n ? s.list[from_list][i] : 0);
        }
      } else {
        row.template each<1024>(0, row.pieces, true, [&](float l, int i, bool there) __attribute__((always_inline)) {
          const bool in = in_bin(l, there);
          keep(in, in ? composite(l, i) : 0);
        });
      }
      bounds(low, high);
    }
    __syncthreads();
    n = s.n;
    listed = n <= kList;
    from_list ^= 1;
  }
  if (tid < 64) {
    const uint64_t c = tid < n ? s.list[from_list][tid] : 0;
    const uint64_t w = tid < n ? weight(sc, s.table, octaves(sc, composite_logit(c))) : 0;
    uint64_t before = 0;
    uint32_t rank = 0;
    for (int j = 0; j < n; ++j) {
      const uint64_t cj = __shfl(c, j, 64), wj = __shfl(w, j, 64);
      if (cj > c) {
        before += wj;
        ++rank;
      }
    }
    const bool hit = by_count ? rank == target : before <= target && target < before + w;
    if (tid < n && hit) {
      s.found = c;
      s.upto = base + before + w;
    }
  }
  __syncthreads();
}

template <int dtype>
__global__ void __launch_bounds__(1024)
sample_choose_kernel(const void *__restrict__ logits, int64_t stride, int vocab, int top, int slices, Settings settings,
                     const float *__restrict__ uniform, const RowSpace *__restrict__ space, int64_t *__restrict__ token,
                     float *__restrict__ logprob, Advance adv) {
  extern __shared__ char lds[];
  Choice &s = *reinterpret_cast<Choice *>(lds);
  const int tid = threadIdx.x, r = blockIdx.x;
  const RowSpace &sp = space[r];
  const int64_t was_a = adv.counter_a ? adv.counter_a[0] : 0, was_b = adv.counter_b ? adv.counter_b[0] : 0;
  const uint64_t best = row_best(sp, slices);
  const RowSettings set = row_settings(settings, r);
  int64_t chosen = -1;
  float lp = -INFINITY;
  if (best != 0 && !(set.T > 0.0f)) {
    chosen = composite_index(best);
    lp = 0.0f;
  } else if (best != 0) {
    const Scale sc = {composite_logit(best), 1.44269504088896340736 / (double)set.T, top};
    const Row<dtype> row(logits, stride, r, vocab);
    fill_table(s.table);
    const bool counts = set.top_k > 0;
    for (int i = tid; i < kBins; i += 1024) {
      s.mass[i] = sp.mass[i];
      s.count[i] = counts ? sp.count[i] : 0;
    }
    __syncthreads();
    // the last entry takes the whole: a bin of its own without tokens
    if (tid == 0) {
      s.mass[kBins] = 0;
      s.count[kBins] = 0;
    }
    __syncthreads();
    prefix<kBins + 1>(s.mass, s.count, s);
    uint64_t kept = s.mass[kBins];                                  // of top-k's run
    if (counts && (uint32_t)set.top_k < s.count[kBins]) {           // (behind the bins the weights are 0)
      search<dtype>(s, row, sc, true, (uint64_t)(set.top_k - 1));
      kept = s.upto;
    }
    uint64_t run = kept;                                            // of the shortest run
    if (set.top_p < 1.0f) {
      const double want = ceil((double)set.top_p * (double)kept);
      uint64_t target = want >= 1.0 ? (uint64_t)want - 1 : 0;
      if (target >= kept) target = kept - 1;
      search<dtype>(s, row, sc, false, target);
      run = s.upto;
    }
    if (set.min_p > 0.0f) {
      const uint64_t largest = 1ull << top;                         // the first token always stays
      const uint64_t least = sp.least_mass > largest ? sp.least_mass : largest;
      run = run < least ? run : least;
    }
    int64_t at = r;
    if (adv.uniform_index) at = min(max(adv.uniform_index[0], (int64_t)0), (int64_t)adv.n_uniform - 1);
    const double x = (double)uniform[at] * (double)run;
    uint64_t target = x > 0.0 ? (x < (double)run ? (uint64_t)x : run - 1) : 0;
    if (target >= run) target = run - 1;
    search<dtype>(s, row, sc, false, target);
    chosen = composite_index(s.found);
    lp = (float)(-octaves(sc, composite_logit(s.found)) * 0.693147180559945309417 - log(ldexp((double)run, -top)));
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
int slices_of(int rows, int vocab, int dtype) {
  const int pieces = vocab / (dtype == RDKV_DTYPE_F32 ? 4 : 8);
  const int want = (int)rdkv_cdiv(1024, rows), most = (int)rdkv_cdiv(pieces, 256);
  int s = want < most ? want : most;
  s = s < kMaxSlices ? s : kMaxSlices;
  return s < 1 ? 1 : s;
}

template <int dtype>
int launch_sample(const char *fn, const void *logits, int64_t stride, int rows, int vocab, const Settings &set,
                  const float *uniform, int64_t *token, float *logprob, const Advance &adv, void *workspace,
                  hipStream_t s) {
  RowSpace *space = reinterpret_cast<RowSpace *>(workspace);
  const int slices = slices_of(rows, vocab, dtype), top = weight_bits(vocab);
  constexpr int size = dtype == RDKV_DTYPE_F32 ? 4 : 2;
  for (int r = 0; r < rows; r += 65535) {                  // (a grid's second dimension)
    const int n = rows - r < 65535 ? rows - r : 65535;
    const void *from = reinterpret_cast<const char *>(logits) + (int64_t)r * stride * size;
    Settings part = set;
    if (part.temperature) part.temperature += r;
    if (part.top_k) part.top_k += r;
    if (part.top_p) part.top_p += r;
    if (part.min_p) part.min_p += r;
    hipLaunchKernelGGL(sample_max_kernel<dtype>, dim3(slices, n), dim3(256), 0, s, from, stride, vocab, space + r);
    RDKV_CHECK_LAUNCH(fn);
    hipLaunchKernelGGL(sample_bins_kernel<dtype>, dim3(slices, n), dim3(256), 0, s, from, stride, vocab, top, part, space + r);
    RDKV_CHECK_LAUNCH(fn);
    hipLaunchKernelGGL(sample_choose_kernel<dtype>, dim3(n), dim3(1024), sizeof(Choice), s, from, stride, vocab, top, slices, part,
                       uniform + r, space + r, token + r, logprob ? logprob + r : nullptr, adv);
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
  if (!workspace || workspace_bytes < rdkv_sample_workspace_bytes(rows) || (uintptr_t)workspace % 16 != 0) {
    rdkv_set_error("%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)rdkv_sample_workspace_bytes(rows));
    return RDKV_EWORKSPACE;
  }
  const Settings set = {sampling->temperature, sampling->top_k, sampling->top_p, sampling->min_p,
                        sampling->temperature_value, sampling->top_k_value, sampling->top_p_value, sampling->min_p_value};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == RDKV_DTYPE_F32)
    return launch_sample<RDKV_DTYPE_F32>(fn, logits, stride, rows, vocab, set, uniform, token, logprob, adv, workspace, s);
  if (dtype == RDKV_DTYPE_F16)
    return launch_sample<RDKV_DTYPE_F16>(fn, logits, stride, rows, vocab, set, uniform, token, logprob, adv, workspace, s);
  return launch_sample<RDKV_DTYPE_BF16>(fn, logits, stride, rows, vocab, set, uniform, token, logprob, adv, workspace, s);
}

}  // namespace

RDKV_API int64_t rdkv_sample_workspace_bytes(int rows) { return rows <= 0 ? 0 : (int64_t)rows * (int64_t)sizeof(RowSpace); }

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
