// The draw of a token from temperature, top-k, top-p and min-p with a given random number, and its log-probability.
//
// reference: Engine::Sample (app/server.cpp:237-277) sorts the weights of a row on the host and walks them; it knows a
// temperature and top-p.
//
// Tokens stand in the order (logit descending, index ascending) with weights w = exp((l - max) / T).  Kept are the first top_k;
// of those the shortest beginning whose weight reaches top_p of theirs; of those the ones with w >= min_p.  The token is the first
// whose running weight passes u times the kept weight.  Every one of these is a place where a running sum over the order crosses a
// number, so no row is sorted: a histogram over classes of gaps max - l says in which class each crossing lies, and only
// those classes' tokens (some hundreds) are brought together and sorted.
//
// Weights are whole numbers, w * 2^44 rounded (formed in 64-bit floats; 2^-45 is their error, and what is lighter is never drawn): sums
// of them are exact in any order, so atomics leave the result the same from call to call, class sums and token sums agree to the
// unit, and a crossing is found in exactly one place.
//
// Three launches: the row's maximum from its parts; weights into the parts' histograms; one workgroup a row for the rest.
#include "common.h"

namespace tlie {

constexpr int kClasses = 1024, kPickThreads = 1024, kListMost = 2048, kPartThreads = 512;

// larger for what stands earlier: the float's order, then the lower index (-0 and +0 are equal)
__device__ __forceinline__ uint64_t place_key(float v, int index) {
  const uint32_t bits = __float_as_uint(v + 0.f);
  const uint32_t order = (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
  return (static_cast<uint64_t>(order) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ float place_value(uint64_t key) {
  const uint32_t order = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((order & 0x80000000u) ? (order & 0x7fffffffu) : ~order);
}
__device__ __forceinline__ int place_index(uint64_t key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }

// What is the same for all tokens of a row.
struct RowScale {
  float max, class_scale;
  double max_wide, inv_t, one;       // one: the weight 1
};

// The classes share the gaps from 0 to 32 T (what is lighter than e^-32 rounds to no weight), or to the smallest logit if that is nearer.
__device__ __forceinline__ RowScale row_scale(float max, float min, float temperature, int shift) {
  const float span = fminf(32.f * temperature, max - min);
  RowScale row;
  row.max = max, row.class_scale = span > 0.f ? kClasses / span : 0.f;
  row.max_wide = max, row.inv_t = 1.0 / static_cast<double>(temperature), row.one = __longlong_as_double((1023ll + shift) << 52);
  return row;
}
__device__ __forceinline__ int gap_class(const RowScale& row, float v) {
  return static_cast<int>(fminf((row.max - v) * row.class_scale, static_cast<float>(kClasses - 1)));
}

// exp((v - max) / T) in units of 2^-shift, rounded; one function, each operation written out, for every kernel that forms it.
// exp(x) = 2^n exp(r), n the whole number nearest to x / ln 2, and exp(r) by its series to r^11 (|r| <= 0.347: 6e-15 of it is left).
__device__ __forceinline__ double weight_wide(const RowScale& row, float v) {
#pragma clang fp contract(off)
  const double x = fmax((static_cast<double>(v) - row.max_wide) * row.inv_t, -64.0);
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0.6931471805599453, x);
  r = fma(n, -2.3190468138462996e-17, r);
  double e = 1.0 / 39916800.0;
  e = fma(e, r, 1.0 / 3628800.0);
  e = fma(e, r, 1.0 / 362880.0);
  e = fma(e, r, 1.0 / 40320.0);
  e = fma(e, r, 1.0 / 5040.0);
  e = fma(e, r, 1.0 / 720.0);
  e = fma(e, r, 1.0 / 120.0);
  e = fma(e, r, 1.0 / 24.0);
  e = fma(e, r, 1.0 / 6.0);
  e = fma(e, r, 0.5);
  e = fma(e, r, 1.0);
  e = fma(e, r, 1.0);
  return ldexp(e * row.one, static_cast<int>(n));
}
// a weight below 2^52 to the nearest whole number: adding 2^52 leaves it in the low bits
__device__ __forceinline__ uint64_t weight_units(double wide) {
#pragma clang fp contract(off)
  return static_cast<uint64_t>(__double_as_longlong(wide + 4503599627370496.0)) & 0xfffffffffffffull;
}

// ceil(share * total) and floor(share * total), exact, for a float share in [0, 1] and total < 2^63.
__device__ __forceinline__ uint64_t share_of(float share, uint64_t total, bool up) {
  const uint32_t bits = __float_as_uint(share), exponent = (bits >> 23) & 255;
  const uint64_t mantissa = exponent ? (bits & 0x7fffffu) | 0x800000u : bits & 0x7fffffu;
  const int down = 150 - static_cast<int>(exponent ? exponent : 1);          // share = mantissa * 2^-down, down >= 23
  const unsigned __int128 product = static_cast<unsigned __int128>(mantissa) * total;
  if (down >= 128) return up && product != 0 ? 1 : 0;
  const unsigned __int128 whole = product >> down;
  return static_cast<uint64_t>(whole) + (up && (whole << down) != product ? 1 : 0);
}

// f(index, value) over the part's tokens
template <int THREADS, typename F>
__device__ __forceinline__ void scan_tokens(const float* __restrict__ row, int begin, int end, F f) {
  constexpr int kTogether = 8;
  int i = begin + threadIdx.x;
  for (; i + (kTogether - 1) * THREADS < end; i += kTogether * THREADS) {
    float v[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) v[u] = row[i + u * THREADS];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) f(i + u * THREADS, v[u]);
  }
  for (; i < end; i += THREADS) f(i, row[i]);
}

struct PartStat {
  uint64_t best;        // place_key of the part's first token in the order; 0: the part has none; all ones: a NaN or +inf
  float min;            // the smallest finite logit, +inf: none
  uint32_t unused;
};
constexpr uint64_t kBadPart = ~0ull;

__global__ void __launch_bounds__(kPartThreads)
draw_best_kernel(const float* __restrict__ logits, int vocab, int part_len, int parts, PartStat* __restrict__ stats) {
  __shared__ uint64_t best_of[kPartThreads / kWave];
  __shared__ float min_of[kPartThreads / kWave];
  const int row = blockIdx.y, part = blockIdx.x, begin = part * part_len, end = min(vocab, begin + part_len);
  uint64_t best = 0;
  float least = INFINITY;
  bool bad = false;
  scan_tokens<kPartThreads>(logits + static_cast<size_t>(row) * vocab, begin, end, [&](int i, float v) {
    bad = bad || !(v < INFINITY);
    if (v > -INFINITY) {
      const uint64_t key = place_key(v, i);
      best = key > best ? key : best;
      least = fminf(least, v);
    }
  });
  if (bad) best = kBadPart;
  for (int offset = 32; offset > 0; offset >>= 1) {
    const uint64_t other = __shfl_xor(best, offset, 64);
    best = other > best ? other : best;
    least = fminf(least, __shfl_xor(least, offset, 64));
  }
  if ((threadIdx.x & 63) == 0) best_of[threadIdx.x >> 6] = best, min_of[threadIdx.x >> 6] = least;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPartThreads / kWave; ++w) {
      best = best_of[w] > best ? best_of[w] : best;
      least = fminf(least, min_of[w]);
    }
    stats[static_cast<size_t>(row) * parts + part] = PartStat{best, least, 0};
  }
}

__device__ __forceinline__ void join_stats(const PartStat* __restrict__ stats, int parts, uint64_t& best, float& least) {
  best = 0, least = INFINITY;
  for (int p = 0; p < parts; ++p) {
    best = stats[p].best > best ? stats[p].best : best;
    least = fminf(least, stats[p].min);
  }
}

// exp(v - max) for the log-probability: the rounding of (v - max) log2(e) is made good, the exponential's own is left
__device__ __forceinline__ float plain_weight(float max, float v) {
  const float x = v - max, high = x * 1.44269502f, low = fmaf(x, 1.44269502f, -high) + x * 1.92596303e-8f;
  const float e = __builtin_amdgcn_exp2f(high);
  return x < -100.f ? 0.f : fmaf(e, low * 0.693147182f, e);
}

__global__ void __launch_bounds__(kPartThreads)
draw_weigh_kernel(const float* __restrict__ logits, int vocab, int part_len, int parts, const PartStat* __restrict__ stats,
                  const float* __restrict__ temperature, int shift, int want_sum, uint64_t* __restrict__ class_mass,
                  uint32_t* __restrict__ class_count, double* __restrict__ sums) {
  __shared__ unsigned long long mass[kClasses];
  __shared__ uint32_t count[kClasses];
  __shared__ double sum_of[kPartThreads / kWave];
  const int row = blockIdx.y, part = blockIdx.x, begin = part * part_len, end = min(vocab, begin + part_len);
  uint64_t best;
  float least;
  join_stats(stats + static_cast<size_t>(row) * parts, parts, best, least);
  if (best == kBadPart || best == 0) return;
  const float t = temperature ? temperature[row] : 0.f;
  const bool drawn = t > 0.f;
  if (!drawn && !want_sum) return;
  const RowScale scale = row_scale(place_value(best), least, t, shift);
  if (drawn) {
    for (int c = threadIdx.x; c < kClasses; c += kPartThreads) mass[c] = 0, count[c] = 0;
    __syncthreads();
  }
  double sum = 0.0;
  scan_tokens<kPartThreads>(logits + static_cast<size_t>(row) * vocab, begin, end, [&](int, float v) {
    if (drawn) {
      const uint64_t units = weight_units(weight_wide(scale, v));
      if (units != 0) {
        const int c = gap_class(scale, v);
        atomicAdd(&mass[c], static_cast<unsigned long long>(units));
        atomicAdd(&count[c], 1u);
      }
    }
    if (want_sum) sum += static_cast<double>(plain_weight(scale.max, v));
  });
  const size_t place = static_cast<size_t>(row) * parts + part;
  if (drawn) {
    __syncthreads();
    for (int c = threadIdx.x; c < kClasses; c += kPartThreads) class_mass[place * kClasses + c] = mass[c], class_count[place * kClasses + c] = count[c];
  }
  if (want_sum) {
    for (int offset = 32; offset > 0; offset >>= 1) sum += __shfl_xor(sum, offset, 64);
    if ((threadIdx.x & 63) == 0) sum_of[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kPartThreads / kWave; ++w) sum += sum_of[w];
      sums[place] = sum;
    }
  }
}

// running sums over the workgroup's threads, each thread's own included
__device__ __forceinline__ uint64_t running_sum(uint64_t v, uint64_t* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int offset = 1; offset < 64; offset <<= 1) {
    const uint64_t below = __shfl_up(v, offset, 64);
    if (lane >= offset) v += below;
  }
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += waves[w];
  __syncthreads();
  return v;
}

struct PickShared {
  uint64_t running_mass[kClasses];          // up to and with each class
  uint32_t running_count[kClasses];
  uint64_t list[kListMost];
  uint64_t waves[kPickThreads / kWave];
  uint64_t adjust[kClasses];
  uint32_t adjust_count[kClasses];
  uint64_t digit_mass[256];
  uint32_t digit_count[256];
  uint32_t wanted[kClasses / 32];           // the classes to bring together
  uint64_t result, result2;
  int found, size;
};

// The first class at which the running mass reaches `target` (> 0), or kClasses.
__device__ int class_reaching(PickShared& s, uint64_t target) {
  const int c = threadIdx.x;
  if (c == 0) s.found = kClasses;
  __syncthreads();
  const uint64_t before = c > 0 ? s.running_mass[c - 1] : 0;
  if (s.running_mass[c] >= target && before < target) s.found = c;
  __syncthreads();
  const int found = s.found;
  __syncthreads();
  return found;
}

// Without a list (more tokens than it holds share the classes in question): the place in the order where the running mass
// (or count) reaches target, found digit by digit of the place keys, eight passes over the row.  Returns the running mass there.
__device__ uint64_t descend(PickShared& s, const float* __restrict__ row, int vocab, const RowScale& scale, uint64_t target, bool by_count, uint64_t* key) {
  uint64_t prefix = 0, mass_before = 0, count_before = 0, mass = 0;
  for (int digit = 7; digit >= 0; --digit) {
    for (int b = threadIdx.x; b < 256; b += kPickThreads) s.digit_mass[b] = 0, s.digit_count[b] = 0;
    __syncthreads();
    scan_tokens<kPickThreads>(row, 0, vocab, [&](int i, float v) {
      if (!(v > -INFINITY)) return;
      const uint64_t place = place_key(v, i);
      if (digit < 7 && (place >> (8 * digit + 8)) != (prefix >> (8 * digit + 8))) return;
      const uint64_t units = weight_units(weight_wide(scale, v));
      if (units == 0) return;
      const int b = static_cast<int>((place >> (8 * digit)) & 255);
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.digit_mass[b]), static_cast<unsigned long long>(units));
      atomicAdd(&s.digit_count[b], 1u);
    });
    __syncthreads();
    if (threadIdx.x == 0) {
      int b = 255;
      uint64_t m = mass_before, n = count_before;
      for (; b > 0; --b) {
        if ((by_count ? n + s.digit_count[b] : m + s.digit_mass[b]) >= target) break;
        m += s.digit_mass[b], n += s.digit_count[b];
      }
      s.found = b, s.result = m, s.result2 = n, s.waves[0] = m + s.digit_mass[b];
    }
    __syncthreads();
    prefix |= static_cast<uint64_t>(s.found) << (8 * digit);
    mass_before = s.result, count_before = s.result2, mass = s.waves[0];
    __syncthreads();
  }
  *key = prefix;
  return mass;
}

__global__ void __launch_bounds__(kPickThreads)
draw_pick_kernel(const float* __restrict__ logits, int vocab, int parts, const PartStat* __restrict__ stats, const float* __restrict__ uniform,
                 const float* __restrict__ temperature, const int* __restrict__ top_k, const float* __restrict__ top_p,
                 const float* __restrict__ min_p, int shift, const uint64_t* __restrict__ class_mass, const uint32_t* __restrict__ class_count,
                 const double* __restrict__ sums, int* __restrict__ out, float* __restrict__ logprob) {
  __shared__ PickShared s;
  const int r = blockIdx.x, tid = threadIdx.x;
  const float* row = logits + static_cast<size_t>(r) * vocab;
  uint64_t best;
  float least;
  join_stats(stats + static_cast<size_t>(r) * parts, parts, best, least);
  if (best == kBadPart || best == 0) {
    if (tid == 0) {
      out[r] = -1;
      if (logprob) logprob[r] = __uint_as_float(0x7fc00000u);
    }
    return;
  }
  const float t = temperature ? temperature[r] : 0.f;
  uint64_t chosen = best;
  if (t > 0.f) {
    const RowScale scale = row_scale(place_value(best), least, t, shift);
    const uint64_t one = 1ull << shift;
    // ---- the row's classes, and running sums over them ----
    uint64_t mass = 0;
    uint32_t count = 0;
    for (int p = 0; p < parts; ++p) {
      const size_t place = (static_cast<size_t>(r) * parts + p) * kClasses + tid;
      mass += class_mass[place], count += class_count[place];
    }
    const uint64_t running = running_sum(mass, s.waves);
    const uint64_t running_n = running_sum(count, s.waves);
    s.running_mass[tid] = running, s.running_count[tid] = static_cast<uint32_t>(running_n);
    if (tid < kClasses / 32) s.wanted[tid] = 0;
    if (tid == 0) s.size = 0, s.result = 0;
    __syncthreads();
    auto mass_upto = [&](int c) { return c < 0 ? 0ull : static_cast<unsigned long long>(s.running_mass[min(c, kClasses - 1)]); };
    auto want = [&](int lo, int hi) {                              // (every thread: its own class)
      if (tid >= lo && tid <= hi && mass != 0) atomicOr(&s.wanted[tid >> 5], 1u << (tid & 31));
    };

    // ---- which classes the crossings can lie in.  A class that is cut leaves what follows with a range of masses. ----
    const int k = top_k ? top_k[r] : 0;
    uint64_t total_lo = s.running_mass[kClasses - 1], total_hi = total_lo;
    bool cut_k = false;
    if (k > 0 && static_cast<uint32_t>(k) < s.running_count[kClasses - 1]) {
      if (tid == 0) s.found = 0;
      __syncthreads();
      if (running_n >= static_cast<uint64_t>(k) && running_n - count < static_cast<uint64_t>(k)) s.found = tid;
      __syncthreads();
      const int c = s.found;
      __syncthreads();
      total_hi = mass_upto(c), total_lo = s.running_count[c] == static_cast<uint32_t>(k) ? total_hi : mass_upto(c - 1);
      cut_k = total_lo != total_hi;
      if (cut_k) want(c, c);
    }
    const float p_share = top_p ? top_p[r] : 1.f;
    const bool cut_p = p_share < 1.f;
    uint64_t kept_lo = total_lo, kept_hi = total_hi;
    if (cut_p) {
      const float share = fmaxf(p_share, 0.f);
      const uint64_t low = share_of(share, total_lo, true), high = share_of(share, total_hi, true);
      const int c_lo = class_reaching(s, low > 0 ? low : 1), c_hi = class_reaching(s, high > 0 ? high : 1);
      want(c_lo, c_hi);
      kept_lo = mass_upto(c_lo - 1), kept_hi = min(kept_hi, static_cast<uint64_t>(mass_upto(c_hi)));
    }
    const float floor_p = min_p ? min_p[r] : 0.f;
    const bool cut_m = floor_p > 0.f;
    uint64_t kept_floor = one;
    const double least_weight = static_cast<double>(fminf(floor_p, 1.f)) * scale.one;
    if (cut_m) {
      // the class of the gap at which the weight is min_p, and its neighbours, for the rounding of the gap
      const float gap = fmaxf(-logf(fminf(floor_p, 1.f)) * t, 0.f);
      const int c = static_cast<int>(fminf(gap * scale.class_scale, static_cast<float>(kClasses - 1)));
      want(c - 1, c + 1);
      kept_floor = max(one, static_cast<uint64_t>(mass_upto(c - 2)));
      kept_lo = min(kept_lo, kept_floor), kept_hi = min(kept_hi, static_cast<uint64_t>(mass_upto(c + 1)));
    }
    // (the first token is always kept)
    kept_lo = max(kept_lo, one);
    const float u = fmaxf(uniform[r], 0.f);                       // (a NaN counts as 0)
    auto goal_of = [&](uint64_t kept) { return u < 1.f ? share_of(u, kept, false) : kept - 1; };
    {
      const int c_lo = class_reaching(s, goal_of(kept_lo) + 1), c_hi = class_reaching(s, goal_of(kept_hi) + 1);
      want(c_lo, c_hi);
    }
    __syncthreads();

    // ---- their tokens, sorted.  The list holds every token of a wanted class, so a token's running mass over the whole row is
    // the list's own plus what the classes in between, which are not in it, hold. ----
    {
      const bool mine = (s.wanted[tid >> 5] >> (tid & 31) & 1u) != 0;
      const uint64_t listed = running_sum(mine ? mass : 0, s.waves);
      s.adjust[tid] = running - listed;                           // (of a wanted class: what is missing up to its end, and so at its start)
      if (cut_k) {
        const uint64_t listed_n = running_sum(mine ? count : 0, s.waves);
        s.adjust_count[tid] = static_cast<uint32_t>(running_n - listed_n);
      }
    }
    scan_tokens<kPickThreads>(row, 0, vocab, [&](int i, float v) {
      if (!(v > -INFINITY)) return;
      const int c = gap_class(scale, v);
      if ((s.wanted[c >> 5] >> (c & 31) & 1u) && weight_units(weight_wide(scale, v)) != 0) {
        const int at = atomicAdd(&s.size, 1);
        if (at < kListMost) s.list[at] = place_key(v, i);
      }
    });
    __syncthreads();
    const int size = s.size;
    uint64_t total = total_lo, kept;
    if (size <= kListMost) {
      int span = 64;
      while (span < size) span <<= 1;
      for (int i = size + tid; i < span; i += kPickThreads) s.list[i] = 0;
      __syncthreads();
      for (int block = 2; block <= span; block <<= 1)
        for (int step = block >> 1; step > 0; step >>= 1) {
          for (int i = tid; i < span / 2; i += kPickThreads) {
            const int a = 2 * i - (i & (step - 1)), b = a + step;
            const uint64_t x = s.list[a], y = s.list[b];
            if ((x < y) == ((a & block) == 0)) s.list[a] = y, s.list[b] = x;      // descending
          }
          __syncthreads();
        }
      // two neighbours of the list a thread
      uint64_t key[2] = {0, 0}, units[2] = {0, 0}, reached[2] = {0, 0};
      double wide[2] = {0.0, 0.0};
      int cls[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (2 * tid + j < size) {
          key[j] = s.list[2 * tid + j];
          const float v = place_value(key[j]);
          wide[j] = weight_wide(scale, v), units[j] = weight_units(wide[j]), cls[j] = gap_class(scale, v);
        }
      const uint64_t both = running_sum(units[0] + units[1], s.waves);
      reached[0] = both - units[1] + s.adjust[cls[0]], reached[1] = both + s.adjust[cls[1]];
      auto crossing = [&](uint64_t target, uint64_t otherwise, uint64_t* place) {      // the running mass where it first reaches target
        if (tid == 0) s.result = otherwise, s.result2 = best;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (units[j] != 0 && reached[j] >= target && reached[j] - units[j] < target) s.result = reached[j], s.result2 = key[j];
        __syncthreads();
        const uint64_t found = s.result;
        *place = s.result2;
        __syncthreads();
        return found;
      };
      uint64_t place;
      if (cut_k) {
        if (tid == 0) s.result = total_hi;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (units[j] != 0 && 2 * tid + j + 1 + s.adjust_count[cls[j]] == static_cast<uint32_t>(k)) s.result = reached[j];
        __syncthreads();
        total = s.result;
        __syncthreads();
      }
      kept = total;
      if (cut_p) kept = crossing(max(share_of(fmaxf(p_share, 0.f), total, true), static_cast<uint64_t>(1)), total, &place);
      if (cut_m) {
        if (tid == 0) s.result = kept_floor;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (units[j] != 0 && wide[j] >= least_weight) atomicMax(reinterpret_cast<unsigned long long*>(&s.result), static_cast<unsigned long long>(reached[j]));
        __syncthreads();
        kept = min(kept, s.result);
        __syncthreads();
      }
      crossing(goal_of(kept) + 1, 0, &place);
      chosen = place;
    } else {
      uint64_t place;
      if (cut_k) total = descend(s, row, vocab, scale, static_cast<uint64_t>(k), true, &place);
      kept = total;
      if (cut_p) kept = descend(s, row, vocab, scale, max(share_of(fmaxf(p_share, 0.f), total, true), static_cast<uint64_t>(1)), false, &place);
      if (cut_m) {
        if (tid == 0) s.result = 0;
        __syncthreads();
        scan_tokens<kPickThreads>(row, 0, vocab, [&](int, float v) {
          const double wide = weight_wide(scale, v);
          if (v > -INFINITY && wide >= least_weight)
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.result), static_cast<unsigned long long>(weight_units(wide)));
        });
        __syncthreads();
        kept = min(kept, max(s.result, one));
        __syncthreads();
      }
      descend(s, row, vocab, scale, goal_of(kept) + 1, false, &chosen);
    }
  }
  if (tid == 0) {
    out[r] = place_index(chosen);
    if (logprob) {
      double sum = 0.0;
      for (int p = 0; p < parts; ++p) sum += sums[static_cast<size_t>(r) * parts + p];
      logprob[r] = static_cast<float>(static_cast<double>(place_value(chosen)) - static_cast<double>(place_value(best)) - log(sum));
    }
  }
}

}  // namespace tlie

using namespace tlie;

// How the entry's scratch is laid out, for `parts` parts a row: the parts' statistics, their sums, their classes' masses and counts.
extern "C" long long tlie_draw_scratch_bytes(int rows, int parts) {
  if (rows <= 0 || parts <= 0) return 0;
  return static_cast<long long>(rows) * parts * (static_cast<long long>(sizeof(PartStat)) + 8 + kClasses * 12);
}

// logits: float [rows, vocab], vocab < 2^24; uniform: float [rows]; temperature, top_k, top_p, min_p: [rows] or null; out: int [rows];
// logprob: float [rows] or null.  scratch: tlie_draw_scratch_bytes(rows, parts), at a multiple of 16 bytes.
extern "C" int tlie_draw(const float* logits, int rows, int vocab, const float* uniform, const float* temperature, const int* top_k,
                         const float* top_p, const float* min_p, int parts, void* scratch, int* out, float* logprob, void* stream) {
  if (rows <= 0 || vocab <= 0 || vocab >= (1 << 24) || parts <= 0 || parts > 65535 || rows > 65535 || scratch == nullptr || uniform == nullptr)
    return kBadArgument;
  hipStream_t s = (hipStream_t)stream;
  const int part_len = (vocab + parts - 1) / parts;
  int shift = 44;                                   // the weights' sum stays below 2^62
  while (shift > 36 && (static_cast<long long>(vocab) << shift) >= (1ll << 62)) --shift;
  const size_t places = static_cast<size_t>(rows) * parts;
  PartStat* stats = static_cast<PartStat*>(scratch);
  double* sums = reinterpret_cast<double*>(stats + places);
  uint64_t* class_mass = reinterpret_cast<uint64_t*>(sums + places);
  uint32_t* class_count = reinterpret_cast<uint32_t*>(class_mass + places * kClasses);
  hipLaunchKernelGGL(draw_best_kernel, dim3(parts, rows), dim3(kPartThreads), 0, s, logits, vocab, part_len, parts, stats);
  hipLaunchKernelGGL(draw_weigh_kernel, dim3(parts, rows), dim3(kPartThreads), 0, s, logits, vocab, part_len, parts, stats, temperature, shift,
                     logprob != nullptr ? 1 : 0, class_mass, class_count, sums);
  hipLaunchKernelGGL(draw_pick_kernel, dim3(rows), dim3(kPickThreads), 0, s, logits, vocab, parts, stats, uniform, temperature, top_k, top_p, min_p,
                     shift, class_mass, class_count, sums, out, logprob);
  return launch_status();
}
