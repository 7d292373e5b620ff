// One token a row from its logits and a given random number, with temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T); tokens of logit -infinity or NaN have no weight and are never drawn.
//   Order: larger logits first, the lower index among equals. top-k keeps the first k tokens; top-p keeps, of
//   those, the shortest beginning that holds p of their weight; min-p drops what weighs less than min_p.
//   Drawn: the first kept token, in index order, at which the running weight passes u times the total.
//   T not above 0: the first token of the order.
//
// Where u and p cut is decided by sums over as many as V tokens, whose shares may be far below what fp32 sums
// keep, so weights are fp64 exponentials (2^-44 relative) rounded to fixed point, 2^-46 of the largest weight, and
// every sum is an integer: exact, and so the same in any order of the additions, atomic ones among them.
//
// One workgroup of 16 waves takes a row; a wave owns a run of consecutive tokens, 16 bytes a lane at a time.
// The place where top-k or top-p cuts is found by histograms in LDS: of the distance to the maximum first, then,
// while more tokens than a list holds share the bin, of (logit, index) as one number over the bin's range; the
// tokens of the last bin are sorted.

#include "cdb_common.h"
#include "../../include/cdb_amd.h"

namespace cdb {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / kWave;
constexpr int kBins = 1024;  // one a thread
constexpr int kList = 2048;  // tokens of the bin that is sorted, two a thread
static_assert(kBins == kSampleThreads && kList == 2 * kSampleThreads, "one bin and two places a thread");

struct SampleParams {
  const void* logits;
  const double* uniform;
  const float *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int64_t* tokens;
  float* logprobs;
  int64_t row_stride;
  int32_t vocab, unit_log2;  // weights are counted in units of 2^-unit_log2
};

// 2^y for y <= 0 in fp64: 2^f for |f| <= 1/2 by a polynomial through its values at the zeros of a Chebyshev
// polynomial (off by 3.7e-14 of the value at most), exact at 0.
CDB_DEVICE double power_of_two(double y, int raise) {
  const double n = __builtin_rint(y), f = y - n;
  double p = 0x1.b63880a30e9ffp-24;
  p = __builtin_fma(p, f, 0x1.63d136366db24p-20);
  p = __builtin_fma(p, f, 0x1.ffcb9515a8016p-17);
  p = __builtin_fma(p, f, 0x1.4308ac85aa947p-13);
  p = __builtin_fma(p, f, 0x1.5d87fe86fe88ep-10);
  p = __builtin_fma(p, f, 0x1.3b2ab7181b755p-7);
  p = __builtin_fma(p, f, 0x1.c6b08d7047e52p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff823cedp-3);
  p = __builtin_fma(p, f, 0x1.62e42fefa39efp-1);
  p = __builtin_fma(p, f, 1.0);
  // Far exponents give 0 whatever they are; kept within what an int holds.
  return __builtin_ldexp(p, (int)fmax(n, -4096.0) + raise);
}

// Logits as numbers in their order, with the index below: larger logits first, the lower index among equals.
// 0 for a token that is never drawn.
CDB_DEVICE uint32_t logit_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
CDB_DEVICE float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
CDB_DEVICE uint64_t place_of(float x, int i) { return ((uint64_t)logit_key(x) << 32) | (uint32_t)~i; }

CDB_DEVICE uint64_t shfl_u64(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(lane << 2, (int)(uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_ds_bpermute(lane << 2, (int)(uint32_t)(v >> 32));
  return ((uint64_t)hi << 32) | lo;
}
CDB_DEVICE uint64_t wave_total(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += shfl_u64(v, __lane_id() ^ m);
  return v;
}
// Sum over this lane and those before it.
CDB_DEVICE uint64_t wave_running(uint64_t v) {
  const int lane = __lane_id();
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t o = shfl_u64(v, max(lane - m, 0));
    v += lane >= m ? o : 0;
  }
  return v;
}

struct SampleShared {
  uint64_t mass[kBins];
  uint64_t list[kList];
  uint32_t count[kBins];
  uint64_t wave64[kSampleWaves], lo, hi, before;
  float wave32[kSampleWaves];
  int32_t bin, found;
};

// Sum over this thread and those before it; `total` is the sum over all. Meets the workgroup twice.
CDB_DEVICE uint64_t block_running(uint64_t v, SampleShared& s, uint64_t& total) {
  const int wave = threadIdx.x >> 6;
  const uint64_t run = wave_running(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.wave64[wave] = run;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) {
    const uint64_t x = s.wave64[w];
    before += w < wave ? x : 0;
    total += x;
  }
  return before + run;
}

// A row's logits as a lane meets them: vectors of 16 bytes, aligned, of which the first and the last may stick out
// of the row. Wave w owns vectors [64 w turns, 64 (w + 1) turns), lane by lane.
template <typename T> struct SampleRow {
  static constexpr int E = 16 / (int)sizeof(T);
  const T* base;  // of vector 0, aligned
  int skip;       // elements of vector 0 before the row
  int vocab, turns, first;

  CDB_DEVICE Vec<T, E> fetch(int v) const {
    Vec<T, E> x;
    const int i0 = v * E - skip;
    if (i0 >= 0 && i0 <= vocab - E) {
      x.load(base + (int64_t)v * E);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        x.set(e, i0 + e >= 0 && i0 + e < vocab ? Elem<T>::load(base + (int64_t)v * E + e) : -INFINITY);
    }
    return x;
  }
  CDB_DEVICE void open(const T* row, int n) {
    skip = (int)(((uintptr_t)row & 15) / sizeof(T));
    base = row - skip;
    vocab = n;
    const int vectors = (skip + n + E - 1) / E;
    turns = (vectors + kSampleThreads - 1) / kSampleThreads;
    first = (threadIdx.x >> 6) * turns * kWave + (threadIdx.x & 63);
  }
  CDB_DEVICE int index(int j) const { return (first + j * kWave) * E - skip; }
  // f(vector, index of its first element) for the lane's vectors, in order.
  template <typename F> CDB_DEVICE void each_vector(F f) const {
    for (int j = 0; j < turns; ++j) f(fetch(first + j * kWave), index(j));
  }
  template <typename F> CDB_DEVICE void each(F f) const {
    each_vector([&](const Vec<T, E>& x, int i) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < E; ++e) f(x.get(e), i + e);
    });
  }
};

// What a logit weighs.
struct Weigher {
  double top, rate;  // log2(e) / T
  float top_f, bins_per;  // bins of the first histogram per unit of logit
  int unit_log2;
  bool endless;  // the maximum is infinite: nothing else weighs anything

  CDB_DEVICE double of(float x) const {
    if (endless) return x == top_f ? __builtin_ldexp(1.0, unit_log2) : 0.0;
    return power_of_two(((double)x - top) * rate, unit_log2);
  }
  CDB_DEVICE static uint64_t units(double w) {
    // Rounded to a whole number below 2^52 by the sum's own rounding.
    return __builtin_bit_cast(uint64_t, w + 0x1p52) & 0xfffffffffffffull;
  }
  // Falls, or stays, as the logit rises.
  CDB_DEVICE int bin(float x) const {
    const float d = x == top_f ? 0.f : top_f - x;
    return (int)fminf(d * bins_per, (float)(kBins - 1));
  }
};

// Tokens sorted by place, the first of the order first. n <= kList; the rest of `list` up to a power of two is
// filled with 0, which sorts last.
CDB_DEVICE void sort_places(uint64_t* list, int n) {
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kSampleThreads) list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int t = threadIdx.x; t < size / 2; t += kSampleThreads) {
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        const uint64_t x = list[a], y = list[b];
        const bool rises = (a & k) != 0;
        if ((x < y) != rises) {
          list[a] = y;
          list[b] = x;
        }
      }
      __syncthreads();
    }
  }
}

// The place of the last kept token among those at `limit` and before it in the order. Kept are those before which
// less than the goal lies: kMass, a share of what they weigh together; otherwise a number of tokens. The first is
// always kept.
template <bool kMass, typename Row>
CDB_DEVICE uint64_t cut(const Row& row, SampleShared& s, const Weigher& w, uint64_t limit, double goal) {
  const int t = threadIdx.x;
  uint64_t lo = limit, hi = ~0ull, before = 0;
  bool linear = true;
  for (;;) {
    // How much lies in each bin.
    const int shift = linear ? 0 : max(0, 64 - __clzll(hi - lo) - 10);
    auto bin_of = [&](float x, uint64_t place) __attribute__((always_inline)) -> int {
      return linear ? w.bin(x) : (int)((hi - place) >> shift);
    };
    s.mass[t] = 0;
    s.count[t] = 0;
    __syncthreads();
    row.each([&](float x, int i) __attribute__((always_inline)) {
      if (!(x > -INFINITY)) return;
      const uint64_t place = place_of(x, i);
      if (place < lo || place > hi) return;
      const int b = bin_of(x, place);
      atomicAdd(&s.count[b], 1u);
      if constexpr (kMass)
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), (unsigned long long)Weigher::units(w.of(x)));
    });
    __syncthreads();
    const uint64_t mine = kMass ? s.mass[t] : s.count[t];
    uint64_t total;
    const uint64_t upto = block_running(mine, s, total);
    if (linear) {
      if (kMass) goal *= (double)total;
      goal = fmax(goal, 0x1p-60);
    }
    // The last bin with tokens before which less than the goal lies.
    const bool starts = s.count[t] != 0 && (double)(before + upto - mine) < goal;
    if (t == 0) s.bin = -1;
    __syncthreads();
    if (starts) atomicMax(&s.bin, t);
    __syncthreads();
    const int b = s.bin;
    if (t == b) s.before = before + upto - mine;
    if (t == 0) {
      s.found = 0;
      s.lo = ~0ull;
      s.hi = 0;
    }
    __syncthreads();
    const int n = (int)min(s.count[b], 0x7fffffffu);
    before = s.before;
    auto inside = [&](float x, uint64_t place) __attribute__((always_inline)) -> bool {
      return place >= lo && place <= hi && bin_of(x, place) == b;
    };
    if (n <= kList) {
      row.each([&](float x, int i) __attribute__((always_inline)) {
        if (!(x > -INFINITY)) return;
        const uint64_t place = place_of(x, i);
        if (inside(x, place)) s.list[atomicAdd(&s.found, 1)] = place;
      });
      __syncthreads();
      sort_places(s.list, n);
      uint64_t q[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint64_t place = 2 * t + e < n ? s.list[2 * t + e] : 0;
        q[e] = place == 0 ? 0 : kMass ? Weigher::units(w.of(logit_of((uint32_t)(place >> 32)))) : 1;
      }
      const uint64_t sum = block_running(q[0] + q[1], s, total) - q[0] - q[1];
      if (t == 0) s.bin = 0;
      __syncthreads();
      if (2 * t < n && (double)(before + sum) < goal) atomicMax(&s.bin, 2 * t);
      if (2 * t + 1 < n && (double)(before + sum + q[0]) < goal) atomicMax(&s.bin, 2 * t + 1);
      __syncthreads();
      const uint64_t last = s.list[s.bin];
      __syncthreads();
      return last;
    }
    // Too many: the range that they take.
    uint64_t least = ~0ull, most = 0;
    row.each([&](float x, int i) __attribute__((always_inline)) {
      if (!(x > -INFINITY)) return;
      const uint64_t place = place_of(x, i);
      if (inside(x, place)) {
        least = min(least, place);
        most = max(most, place);
      }
    });
    atomicMin(reinterpret_cast<unsigned long long*>(&s.lo), (unsigned long long)least);
    atomicMax(reinterpret_cast<unsigned long long*>(&s.hi), (unsigned long long)most);
    __syncthreads();
    lo = s.lo;
    hi = s.hi;
    linear = false;
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleParams P) {
  __shared__ SampleShared s;
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const int64_t r = blockIdx.x;
  SampleRow<T> row;
  row.open(static_cast<const T*>(P.logits) + r * P.row_stride, P.vocab);

  float top = -INFINITY;
  row.each([&](float x, int) __attribute__((always_inline)) { top = fmaxf(top, x); });  // passes over NaN
  top = wave_max(top);
  if (lane == 0) s.wave32[wave] = top;
  if (t == 0) s.bin = 0x7fffffff;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) top = fmaxf(top, s.wave32[w]);
  if (top == -INFINITY) {
    if (t == 0) {
      P.tokens[r] = -1;
      P.logprobs[r] = -INFINITY;
    }
    return;
  }
  const float temperature = P.temperature == nullptr ? 1.f : P.temperature[r];
  if (!(temperature > 0.f)) {
    int best = 0x7fffffff;
    row.each([&](float x, int i) __attribute__((always_inline)) { if (x == top) best = min(best, i); });
    if (best != 0x7fffffff) atomicMin(&s.bin, best);
    __syncthreads();
    if (t == 0) {
      P.tokens[r] = s.bin;
      P.logprobs[r] = 0.f;
    }
    return;
  }
  Weigher w;
  w.top = top;
  w.top_f = top;
  w.rate = 1.4426950408889634 / (double)temperature;
  w.bins_per = (float)fmin(w.rate * (kBins / 46.0), 1e30);
  w.unit_log2 = P.unit_log2;
  w.endless = top == INFINITY;

  // The place of the last token that top-k and top-p keep.
  uint64_t limit = 1;
  const int k = P.top_k == nullptr ? 0 : P.top_k[r];
  if (k > 0 && k < P.vocab) limit = cut<false>(row, s, w, limit, (double)k);
  const float p = P.top_p == nullptr ? 1.f : P.top_p[r];
  if (p < 1.f) limit = cut<true>(row, s, w, limit, (double)p);
  const float last = logit_of((uint32_t)(limit >> 32));
  const bool all = limit == 1;
  const int last_index = (int)~(uint32_t)limit;
  const float m = P.min_p == nullptr ? 0.f : fminf(P.min_p[r], 1.f);
  const double least = m > 0.f ? __builtin_ldexp((double)m, P.unit_log2) : 0.0;
  auto weight = [&](float x, int i) __attribute__((always_inline)) -> uint64_t {
    const bool kept = all ? x > -INFINITY : x > last || (x == last && i <= last_index);
    if (!kept) return 0;
    const double v = w.of(x);
    return v >= least ? Weigher::units(v) : 0;
  };

  uint64_t sum = 0, total;
  row.each([&](float x, int i) __attribute__((always_inline)) { sum += weight(x, i); });
  sum = wave_total(sum);
  __syncthreads();
  if (lane == 0) s.wave64[wave] = sum;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int v = 0; v < kSampleWaves; ++v) {
    const uint64_t x = s.wave64[v];
    before += v < wave ? x : 0;
    total += x;
  }
  // The running weight that must be passed; the largest token has a weight, so one does pass.
  const double u = P.uniform[r];
  const uint64_t goal = u > 0.0 ? min((uint64_t)(fmin(u, 1.0) * (double)total), total - 1) : 0;
  if (goal < before || goal >= before + sum) return;
  row.each_vector([&](const Vec<T, SampleRow<T>::E>& x, int i) __attribute__((always_inline)) {
    uint64_t mine = 0;
#pragma unroll
    for (int e = 0; e < SampleRow<T>::E; ++e) mine += weight(x.get(e), i + e);
    const uint64_t run = wave_running(mine);
    uint64_t at = before + run - mine;
    if (goal >= at && goal < at + mine) {
      for (int e = 0; e < SampleRow<T>::E; ++e) {
        const float y = x.get(e);
        const uint64_t q = weight(y, i + e);
        if (goal >= at && goal < at + q) {
          const double share = w.endless ? 0.0 : ((double)y - w.top) * (w.rate * 0.6931471805599453);
          P.tokens[r] = i + e;
          P.logprobs[r] = (float)(share - log(__builtin_ldexp((double)total, -P.unit_log2)));
        }
        at += q;
      }
    }
    before += shfl_u64(run, 63);
  });
}

template <typename T> static int sample_type(const SampleParams& P, int rows, hipStream_t stream) {
  sample_kernel<T><<<dim3((unsigned)rows), dim3(kSampleThreads), 0, stream>>>(P);
  return hipGetLastError() == hipSuccess ? CDB_OK : CDB_ERR_HIP;
}

}  // namespace cdb

extern "C" int64_t cdb_sample_workspace_bytes(int32_t rows, int32_t vocab) {
  if (rows < 0 || vocab <= 0 || vocab > CDB_SAMPLE_MAX_VOCAB) return -1;
  return 0;
}

extern "C" int cdb_sample(const void* logits, int64_t row_stride, const double* uniform, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, int64_t* tokens,
                          float* logprobs, void* workspace, int64_t workspace_bytes, int32_t rows, int32_t vocab,
                          int32_t dtype, hipStream_t stream) {
  using namespace cdb;
  if (dtype != CDB_DTYPE_F32 && dtype != CDB_DTYPE_BF16) return CDB_ERR_UNSUPPORTED;
  if (rows < 0 || vocab <= 0 || vocab > CDB_SAMPLE_MAX_VOCAB) return CDB_ERR_SHAPE;
  if (rows == 0) return CDB_OK;
  if (logits == nullptr || uniform == nullptr || tokens == nullptr || logprobs == nullptr) return CDB_ERR_NULL;
  if (rows > 1 && row_stride < vocab) return CDB_ERR_SHAPE;
  const int size = dtype == CDB_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size != 0) return CDB_ERR_SHAPE;
  if (workspace_bytes < cdb_sample_workspace_bytes(rows, vocab)) return CDB_ERR_CAPACITY;
  (void)workspace;
  SampleParams P{};
  P.logits = logits; P.uniform = uniform; P.temperature = temperature; P.top_p = top_p; P.min_p = min_p;
  P.top_k = top_k; P.tokens = tokens; P.logprobs = logprobs; P.row_stride = row_stride; P.vocab = vocab;
  int bits = 0;  // vocab <= 2^bits: sums stay below 2^62
  while ((1ll << bits) < vocab) ++bits;
  P.unit_log2 = 62 - bits < 46 ? 62 - bits : 46;
  return dtype == CDB_DTYPE_F32 ? sample_type<float>(P, rows, stream) : sample_type<bf16_t>(P, rows, stream);
}
