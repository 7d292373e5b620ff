// One token a row from its logits and a given random number, with temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T); tokens of logit -infinity or NaN have no weight and are never drawn.
//   Order: larger logits first, the lower index among equals. top-k keeps the first k tokens; top-p keeps, of
//   those, the shortest beginning that holds p of their weight; min-p drops what weighs less than min_p.
//   Drawn: the first kept token, in index order, at which the running weight passes u times the total.
//   T not above 0: the first token of the order.
//
// Where u and p cut is decided by sums over as many as V tokens, whose shares may be far below what fp32 sums
// keep, so weights are fp64 exponentials (2^-38 relative) rounded to fixed point, 2^-46 of the largest weight, and
// every sum is an integer: exact, and so the same in any order of the additions, atomic ones among them.
//
// One workgroup takes a row; a wave owns a run of consecutive tokens, 8 of them a lane at a time.
//   A first pass leaves the largest logit of each of 2048 parts of the row.
//   top-k: the k-th largest of these is a bound that k tokens at least reach, and mostly not many more. min-p gives its
//   bound at once. A second pass collects the tokens above the bound, and the rest is done on that list, in LDS.
//   top-p: the second pass adds up what lies at each distance from the maximum (a histogram in LDS), which says where
//   the share ends; the tokens above are collected if they are few.
//   Where many tokens are kept, the pass after that collects those of the bin in which the filter ends, whose place is
//   then found on the list, and weighs the tokens above the bin, if it is not known what each wave's weigh: workgroups
//   of 16 waves have a histogram for each. Without a filter one pass weighs all tokens.
// On lists, histograms over ranges of (logit, index) as one number narrow a range down to 128 tokens, which are
// ordered by counting.
//
// Bounds: a row lies with one CU, which reads it at 25 GB/s a row where 256 run (the first pass over 256 rows of 131072
// fp32 logits takes 21 us, 6.4 TB/s, a later one 19 from the last cache), and weighs 5.5 tokens a nanosecond, some 25
// instructions of 4 cycles each. So one row of 49152 bf16 logits with all filters takes 13 us, of which the passes are
// 3 and the rest is launch, loads, meetings and instruction fetches that wait for each other; 256 rows with mixed ones
// 38, 256 of 131072 fp32 logits 88: what bounds them is a row that keeps 99 % at T = 1.5, or top-k and top-p together.
// A kernel is 160 to 170 KB of instructions, as all of this stands in it for finite and for other maxima, and holds 128
// registers a lane at four waves a SIMD: 512 threads spill 22 in bf16 and 20 in fp32 (28 and 20 bytes a lane of
// scratch), 1024 spill 64 and 73 (84 bytes).

#include <cfloat>

#include "cdb_common.h"
#include "../../include/cdb_amd.h"

namespace cdb {

constexpr int kRun = 8;  // tokens a lane takes at a time

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

// 2^(y + raise) in fp64, for y from about -1000 to 0 and a whole `raise`: 2^f for |f| <= 1/2 by a polynomial through
// its values at 0 and the zeros of a Chebyshev polynomial (off by 2.1e-12 of the value at most), exact at f = 0.
CDB_DEVICE double power_of_two(double y, double magic) {
  // magic = 1.5 * 2^52 + raise: the sum's last bits are y rounded to a whole number, and raise.
  const double t = y + magic, f = y - (t - magic);
  double p = 0x1.63b2d7971923fp-20;
  p = __builtin_fma(p, f, 0x1.00c0e4e15189cp-16);
  p = __builtin_fma(p, f, 0x1.4308c7183d6a2p-13);
  p = __builtin_fma(p, f, 0x1.5d877598350dep-10);
  p = __builtin_fma(p, f, 0x1.3b2ab70ad2565p-7);
  p = __builtin_fma(p, f, 0x1.c6b08da70cce3p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff82a734p-3);
  p = __builtin_fma(p, f, 0x1.62e42fef9cc69p-1);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)(uint32_t)__builtin_bit_cast(uint64_t, t));
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

// A word and its neighbour by DPP, 0 where there is none or the row is masked.
template <int kCtrl, int kRows = 0xf> CDB_DEVICE uint64_t dpp_u64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, kCtrl, kRows, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), kCtrl, kRows, 0xf, true);
  return ((uint64_t)hi << 32) | lo;
}
// Sum over this lane and those before it.
CDB_DEVICE uint64_t wave_running(uint64_t v) {
  v += dpp_u64<0x111>(v);  // row_shr 1, 2, 4, 8
  v += dpp_u64<0x112>(v);
  v += dpp_u64<0x114>(v);
  v += dpp_u64<0x118>(v);
  v += dpp_u64<0x142, 0xa>(v);  // lane 15 of each row to the next row, lane 31 to the upper half
  v += dpp_u64<0x143, 0xc>(v);
  return v;
}
CDB_DEVICE uint32_t wave_running32(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, true);
  return v;
}
CDB_DEVICE uint64_t read_lane(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return ((uint64_t)hi << 32) | lo;
}
CDB_DEVICE uint64_t wave_total(uint64_t v) { return read_lane(wave_running(v), 63); }
CDB_DEVICE uint64_t wave_most(uint64_t v) {
  v = max(v, dpp_u64<0x111>(v));
  v = max(v, dpp_u64<0x112>(v));
  v = max(v, dpp_u64<0x114>(v));
  v = max(v, dpp_u64<0x118>(v));
  v = max(v, dpp_u64<0x142, 0xa>(v));
  v = max(v, dpp_u64<0x143, 0xc>(v));
  return read_lane(v, 63);
}
// The largest of the wave's values.
CDB_DEVICE float wave_largest(float v) {
  v = row16_max(v);
  const float a = fmaxf(v, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 16)));
  const float b = fmaxf(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 32)),
                        __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 48)));
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(fmaxf(a, b))));
}
CDB_DEVICE void add_to(uint64_t* p, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(p), (unsigned long long)v);
}
CDB_DEVICE void raise_to(uint64_t* p, uint64_t v) {
  atomicMax(reinterpret_cast<unsigned long long*>(p), (unsigned long long)v);
}
CDB_DEVICE void lower_to(uint64_t* p, uint64_t v) {
  atomicMin(reinterpret_cast<unsigned long long*>(p), (unsigned long long)v);
}
// The range of the workgroup's places, of which a lane knows the least and the most, to words that hold ~0 and 0.
CDB_DEVICE void widen(uint64_t* lo, uint64_t* hi, uint64_t least, uint64_t most) {
  const uint64_t a = ~wave_most(~least), b = wave_most(most);
  if (__lane_id() == 0) {
    lower_to(lo, a);
    raise_to(hi, b);
  }
}

// The work of a workgroup of kSampleThreads threads on its row.
template <int kSampleThreads> struct Sampler {
  static constexpr int kSampleWaves = kSampleThreads / kWave;
  static constexpr int kBins = 1024, kBinsEach = kBins / kSampleThreads;     // a thread's lie side by side
  static constexpr int kList = 2048, kListEach = kList / kSampleThreads;     // tokens of a list
  static constexpr int kParts = 2048, kPartsEach = kParts / kSampleThreads;  // of a row: a thread's runs in turn
  // A part's maximum of this rank is reached by some 1800 tokens, where they lie as they fall.
  static constexpr int kPartRank = 1200;
  static constexpr int kShort = 128, kSharers = kSampleThreads / kShort;  // tokens ordered by counting, threads a token
  // Whether each wave has a histogram of its own, which saves weighing the kept tokens again: one workgroup to a CU has
  // the LDS for that. 64 rows of 65536 flat fp32 logits with top-p take 40 us so and 48 without, 256 rows of 131072
  // mixed ones 87 and 103.
  static constexpr bool kApart = kSampleThreads == 1024;
  static_assert(kBinsEach >= 1 && kPartsEach <= 8 && kSharers >= 1 && kSharers <= 8, "shares of a thread");

  // Sum over the kSharers lanes of a token.
  static CDB_DEVICE uint64_t sharers_total(uint64_t v) {
    if constexpr (kSharers >= 2) v += dpp_u64<0xb1>(v);   // quad_perm 1 0 3 2
    if constexpr (kSharers >= 4) v += dpp_u64<0x4e>(v);   // quad_perm 2 3 0 1
    if constexpr (kSharers >= 8) v += dpp_u64<0x141>(v);  // half mirror
    return v;
  }
  struct SampleShared {
    uint64_t mass[kBins], apart[kApart ? kSampleWaves : 1][kApart ? kBins : 1];
    uint64_t list[kList];
    uint64_t few[kShort], few_mass[kShort];
    uint64_t wave64[kSampleWaves], lo, hi, before;
    float wave32[kSampleWaves], low32[kSampleWaves], edge[2];
    int32_t bin, found, found_few;
    __align__(16) uint32_t ends[2 * kRun];  // the runs that stick out of the row, as the row's type
  };

  // Sum over this thread and those before it; `total` is the sum over all. Meets the workgroup twice.
  static CDB_DEVICE uint64_t block_running(uint64_t v, SampleShared& s, uint64_t& total) {
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

  // A row's logits as a lane meets them: runs of 8 tokens, at addresses aligned for 16-byte loads, of which the first
  // and the last may stick out of the row. Wave w owns runs [64 w turns, 64 (w + 1) turns), lane by lane.
  template <typename T> struct SampleRow {
    typedef Vec<T, kRun> Run;
    const T* base;  // of run 0, aligned
    int skip;       // elements of run 0 before the row
    const T* ends;  // run 0 and the last one, if they stick out, -infinity outside
    int vocab, turns, first, first_whole, last_whole, last;  // runs that lie in the row; the last one that touches it

    // The runs n[0..U): loaded together, those that stick out of the row (or lie behind it) mended afterwards, so that
    // no load waits for another.
    template <int U> CDB_DEVICE void fetch(const int* n, Run* x) const {
      int c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        c[u] = last_whole < first_whole ? -1 : min(max(n[u], first_whole), last_whole);
        if (last_whole >= first_whole) x[u].load(base + (int64_t)c[u] * kRun);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (n[u] != c[u]) {
          if (n[u] <= last) {
            x[u].load(ends + (n[u] == 0 ? 0 : kRun));
          } else {
#pragma unroll
            for (int e = 0; e < kRun; ++e) x[u].set(e, -INFINITY);
          }
        }
    }
    CDB_DEVICE Run fetch(int n) const {
      Run x;
      fetch<1>(&n, &x);
      return x;
    }
    CDB_DEVICE void open(SampleShared& s, const T* row, int n) {
      skip = (int)(((uintptr_t)row & 15) / sizeof(T));
      base = row - skip;
      vocab = n;
      first_whole = skip == 0 ? 0 : 1;
      last_whole = (skip + n) / kRun - 1;
      const int runs = (skip + n + kRun - 1) / kRun, t = threadIdx.x;
      last = runs - 1;
      T* to = reinterpret_cast<T*>(s.ends);
      ends = to;
      if (skip != 0 || (skip + n) % kRun != 0) {
        const int i = (t < kRun ? 0 : last * kRun) + t % kRun - skip;
        if (t < 2 * kRun) Elem<T>::store(to + t, i >= 0 && i < n ? Elem<T>::load(row + i) : -INFINITY);
        __syncthreads();
      }
      turns = (runs + kSampleThreads - 1) / kSampleThreads;
      first = (threadIdx.x >> 6) * turns * kWave + (threadIdx.x & 63);
    }
    CDB_DEVICE int wave_of(int i) const { return (skip + i) / kRun / (turns * kWave); }
    // f(turn, run, index of its first token) for the lane's runs, in order; U of them, or the next one, load together.
    template <int U, typename F> CDB_DEVICE void each(F f) const {
      if constexpr (U == 1) {
        Run x = fetch(first);
        for (int j = 0; j < turns; ++j) {
          const Run next = fetch(first + min(j + 1, turns - 1) * kWave);
          f(j, x, (first + j * kWave) * kRun - skip);
          x = next;
        }
      } else {
        for (int j0 = 0; j0 < turns; j0 += U) {
          Run x[U];
          int n[U];
#pragma unroll
          for (int u = 0; u < U; ++u) n[u] = first + min(j0 + u, turns - 1) * kWave;
          fetch<U>(n, x);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (j0 + u < turns) f(j0 + u, x[u], (first + (j0 + u) * kWave) * kRun - skip);
        }
      }
    }
  };
  // A run's logits as fp32.
  struct Logits {
    float v[kRun];
    CDB_DEVICE float get(int e) const { return v[e]; }
  };
  // The largest of a run, NaN passed over.
  template <typename Run> static CDB_DEVICE float largest(const Run& x) {
    float m = x.get(0);
#pragma unroll
    for (int e = 1; e < kRun; ++e) m = fmaxf(m, x.get(e));
    return m;
  }

  // What a logit weighs. kPlain: the maximum is finite and, over the temperature, below 2^20, so one product and sum
  // gives the exponent (all exponents are off by the same 2^-33 at most, which divides out); otherwise the difference
  // is taken first, and where the maximum is infinite nothing else weighs anything.
  template <bool kPlain> struct Weigher {
    double top, rate, offset, magic;  // rate: log2(e) / T
    float top_f, bins_per;            // bins of the first histogram per unit of logit

    // In units. -infinity and NaN give less than half a unit.
    CDB_DEVICE double of(float x) const {
      double y;
      if constexpr (kPlain) {
        y = __builtin_fma((double)x, rate, offset);
      } else {
        y = x == top_f ? 0.0 : ((double)x - top) * rate;
      }
      return power_of_two(fmax(y, -1000.0), magic);
    }
    // A weight rounded to a whole number of units, by the rounding of a sum with 2^52.
    CDB_DEVICE static uint64_t units(double w) { return __builtin_bit_cast(uint64_t, w + 0x1p52) & 0xfffffffffffffull; }
    CDB_DEVICE uint64_t units_of(float x) const { return units(of(x)); }
    // What a run's tokens weigh together, those that `keep` holds for: the sum with 2^52 stays on each until the end.
    template <typename Run, typename F> CDB_DEVICE uint64_t units_of_run(const Run& x, F keep) const {
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < kRun; ++e) {
        const double v = of(x.get(e));
        sum += __builtin_bit_cast(uint64_t, (keep(e, v) ? v : 0.0) + 0x1p52);
      }
      return sum - kRun * 0x4330000000000000ull;
    }
    template <typename Run> CDB_DEVICE uint64_t units_of_run(const Run& x) const {
      return units_of_run(x, [](int, double) { return true; });
    }
    // Falls, or stays, as the logit rises.
    CDB_DEVICE int bin(float x) const {
      const float d = !kPlain && x == top_f ? 0.f : top_f - x;
      return (int)fminf(d * bins_per, (float)(kBins - 1));
    }
    // The logits of bin b, from `lo` to `hi`, for the workgroup, which meets once: the first wave narrows the range of
    // all logits up to the maximum, half of it for each end, 32 places at a time.
    CDB_DEVICE void edges(SampleShared& s, int b, float& lo, float& hi) const {
      if (threadIdx.x < kWave) {
        const int lane = threadIdx.x;
        const bool upper = lane >= 32;
        // The bin of `in` is b - upper at most, that of `out` is not.
        uint32_t out = logit_key(-FLT_MAX) - 1, in = logit_key(top_f);
        while (__any(in - out > 1)) {
          const uint32_t mid = out + (uint32_t)(((uint64_t)(in - out) * ((lane & 31) + 1)) / 33);
          const uint64_t all = __ballot(mid != out && bin(logit_of(mid)) <= b - upper);
          const uint32_t below = upper ? (uint32_t)(all >> 32) : (uint32_t)all;
          const int first = below == 0 ? 32 : __ffs((int)below) - 1;
          const uint32_t width = in - out, start = out;
          if (first < 32) in = start + (uint32_t)(((uint64_t)width * (first + 1)) / 33);
          if (first > 0) out = start + (uint32_t)(((uint64_t)width * first) / 33);
        }
        if (lane == 0) s.edge[0] = logit_of(in);
        if (lane == 63) s.edge[1] = b == 0 ? top_f : logit_of(out);
      }
      __syncthreads();
      lo = s.edge[0];
      hi = s.edge[1];
    }
  };

  // The tokens that a cut leaves: all that can be drawn, or those up to a place of the order.
  struct Limit {
    float last;
    int index;
    bool every;
    CDB_DEVICE static Limit none() { return {0.f, 0, true}; }
    CDB_DEVICE static Limit at(uint64_t place) {
      return {logit_of((uint32_t)(place >> 32)), (int)~(uint32_t)place, false};
    }
    CDB_DEVICE bool keeps(float x, int i) const {
      return (every & (x > -INFINITY)) | (!every & ((x > last) | ((x == last) & (i <= index))));
    }
  };

  // Puts the tokens of a run whose bits are set on the list; beyond its end they are only counted. For whole waves.
  template <typename Run> static CDB_DEVICE void append(SampleShared& s, const Run& x, int i, uint32_t mask) {
    if (!__any(mask != 0)) return;
    const uint32_t upto = wave_running32(__popc(mask));
    const uint32_t all = __builtin_amdgcn_readlane(upto, 63);
    int at = 0;
    if (__lane_id() == 63) at = atomicAdd(&s.found, (int)all);
    at = __builtin_amdgcn_readlane(at, 63) + (int)upto - __popc(mask);
    while (mask != 0) {
      const int e = __ffs((int)mask) - 1;
      mask &= mask - 1;
      float y = x.get(0);
#pragma unroll
      for (int d = 1; d < kRun; ++d) y = d == e ? x.get(d) : y;
      if (at < kList) s.list[at] = place_of(y, i + e);
      ++at;
    }
  }

  // The bits of a run's tokens for which keep(logit, index) holds.
  template <typename Run, typename F> static CDB_DEVICE uint32_t bits_of(const Run& x, int i, F keep) {
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < kRun; ++e) mask |= keep(x.get(e), i + e) ? 1u << e : 0u;
    return mask;
  }

  static CDB_DEVICE void clear_bins(SampleShared& s) {
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) s.mass[threadIdx.x + e * kSampleThreads] = 0;
    if (threadIdx.x == 0) s.bin = -1;
    __syncthreads();
  }
  // Of a whole histogram in `mass`, ordered as the tokens are: the last bin that counts before which, `before`
  // included, less than the goal lies. share: the goal is that share of the histogram. `before` becomes what lies
  // before that bin.
  static CDB_DEVICE int last_bin(SampleShared& s, uint64_t& before, double& goal, bool share, uint64_t& total) {
    const int t = threadIdx.x;
    uint64_t q[kBinsEach], sum = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) {
      q[e] = s.mass[t * kBinsEach + e];
      sum += q[e];
    }
    uint64_t here = before + block_running(sum, s, total) - sum, mine_before = 0;
    if (share) goal *= (double)total;
    goal = fmax(goal, 0x1p-60);
    int mine = -1;
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) {
      if (q[e] != 0 && (double)here < goal) {
        mine = t * kBinsEach + e;
        mine_before = here;
      }
      here += q[e];
    }
    // The bins that start before the goal are the first ones that count, so a wave's last lane with one has its last.
    const uint64_t lanes = __ballot(mine >= 0);
    if (lanes != 0 && (t & 63) == 63 - __clzll(lanes)) atomicMax(&s.bin, mine);
    __syncthreads();
    const int b = max(s.bin, 0);
    if (mine == b) s.before = mine_before;
    __syncthreads();
    if (s.bin >= 0) before = s.before;
    return b;
  }

  // The place of the last kept token of the list's n whose place is `limit` at least. Kept are those before which, with
  // the `before` that is not on the list, less than the goal lies: kMass, of what they weigh; otherwise a number of
  // tokens. share: the goal is that share of what they weigh. The first is always kept.
  template <bool kMass, typename W>
  static CDB_DEVICE uint64_t pick(SampleShared& s, const W& w, int n, uint64_t limit, uint64_t before, double goal,
                                  bool share) {
    const int t = threadIdx.x;
    uint64_t place[kListEach], q[kListEach], lo = ~0ull, hi = 0, total;
#pragma unroll
    for (int e = 0; e < kListEach; ++e) {
      place[e] = t + e * kSampleThreads < n ? s.list[t + e * kSampleThreads] : 0;
      if (place[e] < limit) place[e] = 0;
      q[e] = place[e] == 0 ? 0 : kMass ? w.units_of(logit_of((uint32_t)(place[e] >> 32))) : 1;
      if (place[e] != 0) {
        lo = min(lo, place[e]);
        hi = max(hi, place[e]);
      }
    }
    if (t == 0) {
      s.lo = ~0ull;
      s.hi = 0;
    }
    __syncthreads();
    widen(&s.lo, &s.hi, lo, hi);
    __syncthreads();
    lo = s.lo;
    hi = s.hi;
    for (;;) {
      const int shift = max(0, 64 - __clzll(hi - lo) - 10);
      if (t == 0) s.found_few = 0;
      clear_bins(s);
#pragma unroll
      for (int e = 0; e < kListEach; ++e)
        if (place[e] >= lo && place[e] <= hi) add_to(&s.mass[(int)((hi - place[e]) >> shift)], q[e]);
      const int b = last_bin(s, before, goal, share, total);
      share = false;
      hi -= (uint64_t)b << shift;
      lo = max(lo, hi - (((uint64_t)1 << shift) - 1));
#pragma unroll
      for (int e = 0; e < kListEach; ++e)
        if (place[e] >= lo && place[e] <= hi) {
          const int at = atomicAdd(&s.found_few, 1);
          if (at < kShort) {
            s.few[at] = place[e];
            s.few_mass[at] = q[e];
          }
        }
      __syncthreads();
      const int m = s.found_few;
      if (m <= kShort) {
        const int i = t / kSharers, part = t % kSharers;
        const uint64_t mine = i < m ? s.few[i] : 0;
        uint64_t larger = 0;
        for (int j = part; j < m; j += kSharers) larger += s.few[j] > mine ? s.few_mass[j] : 0;
        larger = sharers_total(larger);
        if (t == 0) s.lo = hi;  // the bin holds a token: the first of its range is kept if no other is
        __syncthreads();
        if (part == 0 && i < m && (double)(before + larger) < goal) lower_to(&s.lo, mine);
        __syncthreads();
        const uint64_t last = s.lo;
        __syncthreads();
        return last;
      }
      __syncthreads();  // all have read how many there were
    }
  }

  // What the tokens that `limit` leaves weigh (or how many they are), by their distance from the maximum, to `mass`.
  template <bool kMass, typename Row, typename W>
  static CDB_DEVICE void histogram(const Row& row, SampleShared& s, const W& w, const Limit& limit) {
    clear_bins(s);
    row.template each<1>([&](int, const typename Row::Run& x, int i) __attribute__((always_inline)) {
      uint64_t q[kRun];
#pragma unroll
      for (int e = 0; e < kRun; ++e) q[e] = kMass ? w.units_of(x.get(e)) : 1;
      if (kMass && limit.every) {  // what cannot be drawn weighs nothing
#pragma unroll
        for (int e = 0; e < kRun; ++e)
          if (q[e] != 0) add_to(&s.mass[w.bin(x.get(e))], q[e]);
      } else {
#pragma unroll
        for (int e = 0; e < kRun; ++e)
          if (limit.keeps(x.get(e), i + e)) add_to(&s.mass[w.bin(x.get(e))], q[e]);
      }
    });
  }

  // The same of all tokens' weights, with what each wave's tokens weigh to `apart`.
  template <typename Row, typename W>
  static CDB_DEVICE void histogram_apart(const Row& row, SampleShared& s, const W& w) {
    const int t = threadIdx.x;
    uint64_t* mine = s.apart[t >> 6];
#pragma unroll
    for (int e = 0; e < kBins; e += kWave) mine[e + (t & 63)] = 0;
    row.template each<1>([&](int, const typename Row::Run& x, int) __attribute__((always_inline)) {
      uint64_t q[kRun];
#pragma unroll
      for (int e = 0; e < kRun; ++e) q[e] = w.units_of(x.get(e));
#pragma unroll
      for (int e = 0; e < kRun; ++e)
        if (q[e] != 0) add_to(&mine[w.bin(x.get(e))], q[e]);
    });
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kBinsEach; ++e) {
      uint64_t sum = 0;
#pragma unroll
      for (int v = 0; v < kSampleWaves; ++v) sum += s.apart[v][t * kBinsEach + e];
      s.mass[t * kBinsEach + e] = sum;
    }
    if (t == 0) s.bin = -1;
  }

  // The place of the last kept token of the row, as `pick`, among those that `limit` leaves. `bin`: of those up to the
  // first histogram's `bin`, if it was made already (0 or more), before which `before` lies.
  template <bool kMass, typename Row, typename W>
  static CDB_DEVICE uint64_t cut(const Row& row, SampleShared& s, const W& w, const Limit& limit, double goal,
                                 int bin, uint64_t before) {
    typedef typename Row::Run Run;
    const int t = threadIdx.x;
    uint64_t lo = 0, hi = ~0ull, total;
    if (bin < 0) {
      histogram<kMass>(row, s, w, limit);
      bin = last_bin(s, before, goal, kMass, total);
    }
    // The tokens of the bin; while they are too many, of a part of the range that they take.
    int shift = -1;  // of the histogram over [lo, hi], or the first one's
    for (;;) {
      auto inside = [&](float x, int i) __attribute__((always_inline)) -> bool {
        if (shift < 0) return limit.keeps(x, i) & (w.bin(x) == bin);
        const uint64_t place = place_of(x, i);
        return limit.keeps(x, i) & (place >= lo) & (place <= hi);
      };
      if (t == 0) {
        s.found = 0;
        s.lo = ~0ull;
        s.hi = 0;
      }
      __syncthreads();
      row.template each<1>([&](int, const Run& x, int i) __attribute__((always_inline)) {
        append(s, x, i, bits_of(x, i, inside));
      });
      __syncthreads();
      if (s.found <= kList) return pick<kMass>(s, w, s.found, 0, before, goal, false);
      uint64_t least = ~0ull, most = 0;
      row.template each<1>([&](int, const Run& x, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kRun; ++e)
          if (inside(x.get(e), i + e)) {
            const uint64_t place = place_of(x.get(e), i + e);
            least = min(least, place);
            most = max(most, place);
          }
      });
      widen(&s.lo, &s.hi, least, most);
      __syncthreads();
      lo = s.lo;
      hi = s.hi;
      shift = max(0, 64 - __clzll(hi - lo) - 10);
      clear_bins(s);
      row.template each<1>([&](int, const Run& x, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kRun; ++e)
          if (inside(x.get(e), i + e))
            add_to(&s.mass[(int)((hi - place_of(x.get(e), i + e)) >> shift)], kMass ? w.units_of(x.get(e)) : 1);
      });
      hi -= (uint64_t)last_bin(s, before, goal, false, total) << shift;
      lo = max(lo, hi - (((uint64_t)1 << shift) - 1));
    }
  }

  // What the filters of a row ask for.
  struct Filters {
    int k;         // 0: all
    double p;      // 1: all
    double u;      // the given number
    double size, least;  // share of the largest that a kept token weighs at least, and in units
    bool by_count, by_share, by_size;
  };

  // The share is that of the weight as it was summed, in which what all exponents are off by divides out (kPlain), and
  // one token alone has all of it: its weight may be a rounding above the total.
  template <typename W>
  static CDB_DEVICE void give(const SampleParams& P, int64_t r, const W& w, uint64_t place, uint64_t total) {
    const double weight = w.of(logit_of((uint32_t)(place >> 32)));
    P.tokens[r] = (int)~(uint32_t)place;
    P.logprobs[r] = W::units(weight) == total ? 0.f : (float)fmin(log(weight / (double)total), 0.0);
  }

  // The running weight that must be passed, of kept tokens that weigh `total` units; the largest token has a weight, so
  // one passes it.
  static CDB_DEVICE uint64_t goal_of(double u, uint64_t total) {
    return u > 0.0 ? min((uint64_t)(fmin(u, 1.0) * (double)total), total - 1) : 0;
  }

  // Draws from the list of the row's first n tokens, n <= kShort, in any order, of which top-k leaves k at most; goal:
  // the weight that top-p asks for, if it is known (0 or more).
  template <typename W>
  static CDB_DEVICE void draw_short(const SampleParams& P, int64_t r, SampleShared& s, const W& w, const Filters& f,
                                    int n, double goal) {
    // kSharers threads a token, which each compare it with their share of the others.
    const int t = threadIdx.x, i = t / kSharers, part = t % kSharers;
    const uint64_t place = i < n ? s.list[i] : 0;
    const double weight = place == 0 ? 0.0 : w.of(logit_of((uint32_t)(place >> 32)));
    const uint64_t mine = W::units(weight);
    if (part == 0) s.few_mass[i] = mine;
    if (t == 0) s.before = 0;
    __syncthreads();
    uint64_t before = 0, count = 0, total = 0;
    for (int j = part; j < n; j += kSharers) {
      const bool larger = s.list[j] > place;
      before += larger ? s.few_mass[j] : 0;
      count += larger;
    }
    before = sharers_total(before);
    count = sharers_total(count);
    bool kept = place != 0 && (!f.by_count || count < (uint64_t)f.k);
    if (f.by_share) {
      if (goal < 0.0) {
        // The last that top-k leaves has the others before it.
        if (part == 0 && place != 0 && (count + 1 == (uint64_t)f.k || (count + 1 == (uint64_t)n && n < f.k)))
          s.before = before + mine;
        __syncthreads();
        goal = f.p * (double)s.before;
      }
      kept = kept && (count == 0 || (double)before < goal);
    }
    kept = kept && weight >= f.least;
    __syncthreads();
    if (part == 0) s.few_mass[i] = kept ? mine : 0;
    __syncthreads();
    before = 0;
    for (int j = part; j < n; j += kSharers) {
      const uint64_t q = s.few_mass[j];
      before += (uint32_t)s.list[j] > (uint32_t)place ? q : 0;  // a lower index
      total += q;
    }
    before = sharers_total(before);
    total = sharers_total(total);
    const uint64_t at = goal_of(f.u, total);
    if (part == 0 && kept && at >= before && at < before + mine) give(P, r, w, place, total);
  }

  // The same for n <= kList.
  template <typename W>
  static CDB_DEVICE void draw_list(const SampleParams& P, int64_t r, SampleShared& s, const W& w, const Filters& f,
                                   int n, double goal) {
    const int t = threadIdx.x;
    uint64_t limit = 1;
    if (f.by_count) limit = pick<false>(s, w, n, limit, 0, (double)f.k, false);
    if (f.by_share) limit = pick<true>(s, w, n, limit, 0, goal < 0.0 ? f.p : goal, goal < 0.0);
    uint64_t place[kListEach], q[kListEach];
#pragma unroll
    for (int e = 0; e < kListEach; ++e) {
      place[e] = t + e * kSampleThreads < n ? s.list[t + e * kSampleThreads] : 0;
      const double weight = w.of(logit_of((uint32_t)(place[e] >> 32)));
      q[e] = place[e] >= limit && weight >= f.least ? W::units(weight) : 0;
    }
    // By index: the bin of up to 1024 neighbours, then the token.
    const int shift = max(0, 32 - __clz(P.vocab - 1) - 10);
    uint64_t total, goal_at = 0, sum = 0;
    int base = 0;
    for (int step = 0; step < 2; ++step) {
      clear_bins(s);
#pragma unroll
      for (int e = 0; e < kListEach; ++e) {
        const int i = (int)~(uint32_t)place[e] - base, at = step == 0 ? i >> shift : i;
        if (q[e] != 0 && at >= 0 && at < (step == 0 ? kBins : 1 << shift)) add_to(&s.mass[at], q[e]);
      }
      __syncthreads();
      uint64_t mine = 0, here;
#pragma unroll
      for (int e = 0; e < kBinsEach; ++e) mine += s.mass[t * kBinsEach + e];
      here = block_running(mine, s, total) - mine;
      if (step == 0) {
        sum = total;
        goal_at = goal_of(f.u, total);
      }
#pragma unroll
      for (int e = 0; e < kBinsEach; ++e) {
        const uint64_t next = here + s.mass[t * kBinsEach + e];
        if (goal_at >= here && goal_at < next) {
          s.bin = t * kBinsEach + e;
          s.before = here;
        }
        here = next;
      }
      __syncthreads();
      const int found = s.bin;
      goal_at -= s.before;
      base = step == 0 ? found << shift : base + found;
      __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < kListEach; ++e)
      if (q[e] != 0 && (int)~(uint32_t)place[e] == base) give(P, r, w, place[e], sum);
  }

  // A logit that all of the first b + 1 bins, of which `per` lie in a unit of logit, reach. (top - x) * per below b + 1
  // is off by 2^-22 of itself at most, and rounding the difference here keeps the order of the logits.
  static CDB_DEVICE float reached(float top, float per, int b) { return top - (float)(b + 1) / per * 1.000001f; }
  // Collects the tokens that reach `bound`; how many they are.
  template <typename T> static CDB_DEVICE int collect(const SampleRow<T>& row, SampleShared& s, float bound) {
    if (threadIdx.x == 0) s.found = 0;
    __syncthreads();
    auto inside = [&](float x, int) __attribute__((always_inline)) -> bool { return x >= bound; };
    row.template each<sizeof(T) == 2 ? 8 : 4>(
        [&](int, const typename SampleRow<T>::Run& x, int i) __attribute__((always_inline)) {
          if (__any(inside(largest(x), 0))) append(s, x, i, bits_of(x, i, inside));
        });
    __syncthreads();
    return s.found;
  }

  // Draws by collecting the tokens that may be kept in a list. False, for all threads, where they may be too many;
  // `bin`, `before` and `goal` then tell what is known of where top-p ends.
  template <typename T, typename W>
  static CDB_DEVICE bool draw_few(const SampleParams& P, int64_t r, const SampleRow<T>& row, SampleShared& s,
                                  const W& w, const Filters& f, const float* part_top, float least, int& bin,
                                  uint64_t& before, double& goal) {
    if (f.by_count && f.k > kPartRank) return false;
    const int t = threadIdx.x;
    uint64_t total;
    int b = kBins - 1;
    float bound = -FLT_MAX;
    // (Of top-k's tokens all are needed to tell what top-p's share of them is.)
    if (f.by_size && !(f.by_count && f.by_share))
      b = (int)fmin(-log2(f.size) * (kBins / 46.0) + 1.0, (double)(kBins - 1));
    if (f.by_count) {
      // By the bins of the weights the k-th token may lie in the last one with most of the row, too many for a list:
      // 256 mixed rows of 131072, among them k = 1000 at T = 0.3, take 275 us. With bins from the largest of the parts'
      // maxima to the least they take 87.
      const float width = (float)(kBins - 1) / (w.top_f - least), per = width <= FLT_MAX ? width : 0.f;
      clear_bins(s);
#pragma unroll
      for (int e = 0; e < kPartsEach; ++e)
        if (part_top[e] > -INFINITY) add_to(&s.mass[(int)fminf((w.top_f - part_top[e]) * per, (float)(kBins - 1))], 1);
      uint64_t parts_before = 0;
      double rank = (double)f.k;
      const int last = last_bin(s, parts_before, rank, false, total);
      if (total >= (uint64_t)f.k) bound = fmaxf(least, reached(w.top_f, per, last));
    } else if (f.by_share) {
      if (t == 0) s.found = 0;
      if constexpr (kApart) histogram_apart(row, s, w);
      else histogram<true>(row, s, w, Limit::none());
      goal = f.p;
      bin = last_bin(s, before, goal, true, total);
      b = min(b, bin);
      // The parts whose largest logit lies up to there tell about how many tokens do.
      int parts = 0;
#pragma unroll
      for (int e = 0; e < kPartsEach; ++e)
        parts += __popcll(__ballot(part_top[e] > -INFINITY && w.bin(part_top[e]) <= b));
      if ((t & 63) == 0) atomicAdd(&s.found, parts);
      __syncthreads();
      const bool many = s.found > kPartRank;
      __syncthreads();
      if (many) return false;
    }
    if (b < kBins - 1) bound = fmaxf(bound, reached(w.top_f, w.bins_per, b));
    const int n = collect(row, s, bound);
    if (n > kList) return false;
    if (n <= kShort) draw_short(P, r, s, w, f, n, goal);
    else draw_list(P, r, s, w, f, n, goal);
    return true;
  }

  // Draws by weighing every kept token in index order.
  template <typename T, typename W>
  static CDB_DEVICE void draw_many(const SampleParams& P, int64_t r, const SampleRow<T>& row, SampleShared& s,
                                   const W& w, const Filters& f, int bin, uint64_t before, double goal) {
    typedef typename SampleRow<T>::Run Run;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    Limit limit = Limit::none();
    if (f.by_count) limit = Limit::at(cut<false>(row, s, w, limit, (double)f.k, -1, 0));
    uint64_t sum = 0, total = 0;
    bool weighed = false;
    const bool apart = kApart && bin >= 0;
    if (f.by_share) {
      if (bin < 0) {
        histogram<true>(row, s, w, limit);
        goal = f.p;
        before = 0;
        bin = last_bin(s, before, goal, true, total);
      }
      // The tokens before the bin in which the share ends are kept and weighed, those of the bin collected.
      if (t == 0) s.found = 0;
      float lo, hi;
      w.edges(s, bin, lo, hi);
      if (apart && limit.every && !f.by_size) {
        // What the wave's tokens before the bin weigh is known.
        for (int e = lane; e < bin; e += kWave) sum += s.apart[kApart ? wave : 0][kApart ? e : 0];
        row.template each<sizeof(T) == 2 ? 8 : 4>([&](int, const Run& x, int i) __attribute__((always_inline)) {
          if (!__any(largest(x) >= lo)) return;
          append(s, x, i, bits_of(x, i, [&](float y, int) __attribute__((always_inline)) -> bool {
            return (y >= lo) & (y <= hi);
          }));
        });
      } else {
        row.template each<1>([&](int, const Run& x, int i) __attribute__((always_inline)) {
          const float m = largest(x);
          if (!__any(m >= lo)) return;
          Logits above;  // -infinity weighs nothing
          uint32_t here = 0;
#pragma unroll
          for (int e = 0; e < kRun; ++e) {
            const float y = x.get(e);
            above.v[e] = y > hi ? y : -INFINITY;
            here |= (y >= lo) & (y <= hi) ? 1u << e : 0u;
          }
          if (limit.every && !f.by_size) {
            sum += w.units_of_run(above);
          } else {
            uint32_t kept = 0;
#pragma unroll
            for (int e = 0; e < kRun; ++e) kept |= limit.keeps(x.get(e), i + e) ? 1u << e : 0u;
            here &= kept;
            sum += w.units_of_run(above, [&](int e, double v) __attribute__((always_inline)) -> bool {
              return (kept >> e & 1) & (v >= f.least);
            });
          }
          append(s, x, i, here);
        });
      }
      __syncthreads();
      const int n = s.found;
      weighed = n <= kList;
      __syncthreads();  // all have read it
      if (weighed) {
        const uint64_t last = pick<true>(s, w, n, 0, before, goal, false);
        limit = Limit::at(last);
        sum = wave_total(sum);
        if (lane == 0) s.wave64[wave] = sum;
        __syncthreads();
        for (int j = t; j < n; j += kSampleThreads) {
          const uint64_t place = s.list[j];
          const double v = w.of(logit_of((uint32_t)(place >> 32)));
          if (place >= last && v >= f.least) add_to(&s.wave64[row.wave_of((int)~(uint32_t)place)], W::units(v));
        }
      } else {
        limit = Limit::at(cut<true>(row, s, w, limit, goal, bin, before));
      }
    }
    auto of_run = [&](const Run& x, int i) __attribute__((always_inline)) -> uint64_t {
      if (limit.every && !f.by_size) return w.units_of_run(x);
      return w.units_of_run(x, [&](int e, double v) __attribute__((always_inline)) -> bool {
        return limit.keeps(x.get(e), i + e) & (v >= f.least);
      });
    };
    if (!weighed) {
      sum = 0;
      row.template each<1>([&](int, const Run& x, int i) __attribute__((always_inline)) {
        if (__any(limit.every || largest(x) >= limit.last)) sum += of_run(x, i);
      });
      sum = wave_total(sum);
      __syncthreads();
      if (lane == 0) s.wave64[wave] = sum;
    }
    __syncthreads();
    // Where the running weight passes the goal: the wave, the turn of that wave (a wave of this workgroup each), the
    // lane, the token.
    total = 0;
#pragma unroll
    for (int v = 0; v < kSampleWaves; ++v) total += s.wave64[v];
    const uint64_t at_goal = goal_of(f.u, total);
    int owner = 0;
    before = 0;
#pragma unroll
    for (int v = 0; v < kSampleWaves - 1; ++v) {
      const uint64_t upto = before + s.wave64[v];
      if (v == owner && upto <= at_goal) {
        before = upto;
        owner = v + 1;
      }
    }
    const int each = (row.turns + kSampleWaves - 1) / kSampleWaves;  // turns of the owner that a wave takes
    const int from = wave * each, to = min(row.turns, from + each);
    const int base = owner * row.turns * kWave + lane;
    uint64_t all = 0;
    for (int j = from; j < to; ++j)
      all += wave_total(of_run(row.fetch(base + j * kWave), (base + j * kWave) * kRun - row.skip));
    __syncthreads();
    if (lane == 0) s.wave64[wave] = all;
    __syncthreads();
    for (int v = 0; v < wave; ++v) before += s.wave64[v];
    if (at_goal < before || at_goal >= before + all) return;
    for (int j = from; j < to; ++j) {
      const int i = (base + j * kWave) * kRun - row.skip;
      const Run x = row.fetch(base + j * kWave);
      const uint64_t mine = of_run(x, i), upto = before + wave_running(mine);
      uint64_t at = upto - mine;
      if (at_goal >= at && at_goal < upto) {
#pragma unroll
        for (int e = 0; e < kRun; ++e) {
          const double v = w.of(x.get(e));
          const uint64_t q = limit.keeps(x.get(e), i + e) && v >= f.least ? W::units(v) : 0;
          if (at_goal >= at && at_goal < at + q) give(P, r, w, place_of(x.get(e), i + e), total);
          at += q;
        }
      }
      before = read_lane(upto, 63);
    }
  }

  // One row, the workgroup's.
  template <typename T> static CDB_DEVICE void draw(const SampleParams& P, SampleShared& s) {
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t r = blockIdx.x;
    SampleRow<T> row;
    row.open(s, static_cast<const T*>(P.logits) + r * P.row_stride, P.vocab);

    // Loaded with the row's first tokens: a load of its own would cost each its time.
    const float temperature = P.temperature == nullptr ? 1.f : P.temperature[r];
    const int k = P.top_k == nullptr ? 0 : P.top_k[r];
    const float p = P.top_p == nullptr ? 1.f : P.top_p[r];
    const float m = P.min_p == nullptr || !(P.min_p[r] > 0.f) ? 0.f : fminf(P.min_p[r], 1.f);
    Filters f;
    f.u = P.uniform[r];

    float part_top[kPartsEach], mine = -INFINITY, least = INFINITY;  // of the parts' largest: the largest, the least
#pragma unroll
    for (int e = 0; e < kPartsEach; ++e) part_top[e] = -INFINITY;
    for (int j0 = 0; j0 < row.turns; j0 += 8) {
      typename SampleRow<T>::Run x[8];
      int n[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) n[u] = row.first + min(j0 + u, row.turns - 1) * kWave;
      row.template fetch<8>(n, x);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (j0 + u < row.turns) part_top[u % kPartsEach] = fmaxf(part_top[u % kPartsEach], largest(x[u]));
    }
#pragma unroll
    for (int e = 0; e < kPartsEach; ++e) {
      mine = fmaxf(mine, part_top[e]);
      least = fminf(least, part_top[e] > -INFINITY ? part_top[e] : INFINITY);
    }
    float top = wave_largest(mine);
    least = -wave_largest(-least);
    if (lane == 0) {
      s.wave32[wave] = top;
      s.low32[wave] = least;
    }
    if (t == 0) s.bin = 0x7fffffff;  // the lowest index, of a greedy row
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
      top = fmaxf(top, s.wave32[w]);
      least = fminf(least, s.low32[w]);
    }
    if (__builtin_expect(top == -INFINITY, 0)) {
      if (t == 0) {
        P.tokens[r] = -1;
        P.logprobs[r] = -INFINITY;
      }
      return;
    }
    // Out of the way, as are the other rare branches here: what follows has to be fetched, and at a few instructions a
    // wave that takes longer than running it (one row 14.3 us without, 13.4 with; 33 rows of 32771 15.9 and 14.5).
    if (__builtin_expect(!(temperature > 0.f), 0)) {
      if (mine == top) {
        int best = 0x7fffffff;
        row.template each<4>([&](int, const typename SampleRow<T>::Run& x, int i) __attribute__((always_inline)) {
#pragma unroll
          for (int e = 0; e < kRun; ++e) best = x.get(e) == top ? min(best, i + e) : best;
        });
        atomicMin(&s.bin, best);
      }
      __syncthreads();
      if (t == 0) {
        P.tokens[r] = s.bin;
        P.logprobs[r] = 0.f;
      }
      return;
    }
    f.k = k;
    f.p = p;
    f.size = m;
    f.by_count = k > 0 && k < P.vocab;
    f.by_share = p < 1.f;
    f.by_size = m > 0.f;
    auto set_up = [&](auto& w) __attribute__((always_inline)) {
      w.top = top;
      w.top_f = top;
      w.rate = 1.4426950408889634 / (double)temperature;
      w.offset = -w.top * w.rate;
      w.magic = 0x1.8p52 + (double)P.unit_log2;
      w.bins_per = (float)fmin(w.rate * (kBins / 46.0), 1e30);
      f.least = f.by_size ? f.size * w.of(top) : 0.0;
    };
    if (__builtin_expect(fabs((double)top * (1.4426950408889634 / (double)temperature)) < 0x1p20, 1)) {
      Weigher<true> w;
      set_up(w);
      int bin = -1;
      uint64_t before = 0;
      double goal = -1.0;
      if ((f.by_count || f.by_share || f.by_size) && draw_few(P, r, row, s, w, f, part_top, least, bin, before, goal))
        return;
      __syncthreads();
      draw_many(P, r, row, s, w, f, bin, before, goal);
    } else {
      Weigher<false> w;
      set_up(w);
      draw_many(P, r, row, s, w, f, -1, 0, -1.0);
    }
  }
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 4) sample_kernel(SampleParams P) {
  __shared__ typename Sampler<kThreads>::SampleShared s;
  Sampler<kThreads>::template draw<T>(P, s);
}

template <typename T> static int sample_type(const SampleParams& P, int rows, hipStream_t stream) {
  // A CU holds two workgroups of 512, or one of 1024, which passes over a long row faster and has a histogram a wave:
  // 256 rows of 49152 take 38 us with 1024 threads and 46 with 512, one 13.4 and 13.8, 64 flat ones of 65536 40 and 54;
  // 356 rows of 1438 34 and 24, 298 of 82 26 and 15, 95 of 368 22 and 18, 64 of 8000 46 and 43. Of more rows than CUs
  // two run at a time: 512 rows of 49152 take 65 and 60, but 300 of them 40 and 47, 257 fp32 rows of 131072 89 and 117:
  // just above 256 rows the rule is the slower choice.
  if (rows > 256 || P.vocab <= 8192) sample_kernel<T, 512><<<dim3((unsigned)rows), dim3(512), 0, stream>>>(P);
  else sample_kernel<T, 1024><<<dim3((unsigned)rows), dim3(1024), 0, stream>>>(P);
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
