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
// Two forms.  A row in parts, four launches: its maximum; weights into the parts' histograms; the classes in question (each part's workgroup finds
// them again, which costs less than another launch) and their tokens into the row's list; and, a workgroup a row, the crossings.  Or all of
// it by one workgroup a row.
//
// What bounds them.  Few rows: reads and sums that wait for one another (1 row of 32000 tokens 20 us, its four kernels 2.5, 4.4, 7.5 and 5.1).
// Many: three readings of the row, the first from memory (64 rows of 128256, 33 MB: 5.4 us, 6.1 TB/s), and the 64-bit arithmetic of the
// weights (13.9 us, of which 9.4 without it); then 17.5 us for the tokens in question and 7.4 for the crossings, 44 in all.  256 such rows by a
// workgroup each: 21, 35, 19 (with the classes) and 3 us, 88 in all with what the slowest row takes longer.
#include "common.h"

namespace tlie {

constexpr int kClasses = 1024, kPartThreads = 512, kGatherThreads = 256, kPickThreads = 512, kRowThreads = 1024, kListMost = 2048, kPartsMost = 8;

// 2^(i / 32) and 2^(j / 1024): 2^(k / 1024) is the product of one of each
constexpr int kPowers = 1024;
__constant__ double powers_whole[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
__constant__ double powers_fine[32] = {
    1.0, 1.0006771306930664, 1.0013547198921082, 1.002032767907594,
    1.0027112750502025, 1.0033902416308227, 1.004069667960554, 1.0047495543507072,
    1.0054299011128027, 1.006110708558573, 1.0067919769999607, 1.0074737067491204,
    1.0081558981184175, 1.0088385514204294, 1.0095216669679448, 1.0102052450739643,
    1.0108892860517005, 1.011573790214578, 1.0122587578762337, 1.0129441893505169,
    1.0136300849514894, 1.0143164449934257, 1.0150032697908125, 1.0156905596583505,
    1.016378314910953, 1.0170665358637463, 1.0177552228320703, 1.0184443761314785,
    1.019133996077738, 1.0198240829868295, 1.0205146371749483, 1.0212056589585028};

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
  double max_wide, steps, least, one;       // least: the gap from which on nothing weighs; one: the weight 1
};
// With the powers 2^(j / 1024) in LDS, times the weight 1: ALL of them, for kernels that weigh every token, or 32 by 32 as they stand above, for
// those that weigh the tokens in question (their products are the same numbers: the weight 1 is a power of two).
template <bool ALL>
struct PoweredScale : RowScale {
  const double* powers;
  __device__ __forceinline__ double power(int n) const {
#pragma clang fp contract(off)
    if constexpr (ALL) return powers[n & (kPowers - 1)];
    else return powers[(n >> 5) & 31] * powers[32 + (n & 31)];
  }
};
template <bool ALL>
constexpr int kPowersHeld = ALL ? kPowers : 64;

// Every thread of the workgroup: the powers into LDS (to be read after the next barrier).
template <bool ALL, int THREADS>
__device__ __forceinline__ void bring_powers(double* powers, int shift) {
#pragma clang fp contract(off)
  const double one = __longlong_as_double((1023ll + shift) << 52);
  if constexpr (ALL) {
    for (int j = threadIdx.x; j < kPowers; j += THREADS) powers[j] = powers_whole[j >> 5] * powers_fine[j & 31] * one;
  } else {
    if (threadIdx.x < 64) powers[threadIdx.x] = threadIdx.x < 32 ? powers_whole[threadIdx.x] * one : powers_fine[threadIdx.x & 31];
  }
}

// The classes share the gaps from 0 to 32 T (what is lighter than e^-32 rounds to no weight), or to the smallest logit if that is nearer.
template <bool ALL>
__device__ __forceinline__ PoweredScale<ALL> row_scale(float max, float min, float temperature, int shift, const double* powers) {
  const float span = fminf(32.f * temperature, max - min);
  PoweredScale<ALL> row;
  row.max = max, row.class_scale = span > 0.f ? kClasses / span : 0.f;
  // (an infinite temperature as a finite one at which every finite gap is none)
  const double wide = fmin(static_cast<double>(temperature), 1e300);
  row.max_wide = max, row.steps = 1477.3197218702985 / wide, row.least = -34.0 * wide, row.one = __longlong_as_double((1023ll + shift) << 52);
  row.powers = powers;
  return row;
}
__device__ __forceinline__ int gap_class(const RowScale& row, float v) {
  return static_cast<int>(fminf((row.max - v) * row.class_scale, static_cast<float>(kClasses - 1)));
}

// exp((v - max) / T) in units of 2^-shift; one function, each operation written out, for every kernel that forms it.  The
// exponent in steps of ln 2 / 1024 is a whole number n and a rest f of half a step at most: 2^(n / 1024) from the table and its exponent, exp of
// the rest by its series to the third power (5.5e-16 of it is left).  10 operations on 64-bit floats, and a conversion: the processor's time is
// what the weights of many rows take (35 of 88 us for 256 rows of 128256 tokens; with 12 such operations 39).
template <bool ALL>
__device__ __forceinline__ double weight_wide(const PoweredScale<ALL>& row, float v) {
#pragma clang fp contract(off)
  const double gap = fmax(static_cast<double>(v) - row.max_wide, row.least);
  const double shifted = fma(gap, row.steps, 6755399441055744.0);        // 1.5 * 2^52: the nearest whole number in the low bits
  const int n = static_cast<int>(__double_as_longlong(shifted));
  const double f = fma(gap, row.steps, 6755399441055744.0 - shifted);
  constexpr double step = 0.6931471805599453 / kPowers;
  double p = fma(step * step * step / 6.0, f, step * step / 2.0);
  p = fma(p, f, step);
  p = p * f;
  const double power = row.power(n);
  const double scaled = __hiloint2double(__double2hiint(power) + ((n >> 10) << 20), __double2loint(power));
  return fma(scaled, p, scaled);
}
// a weight below 2^52 to the nearest whole number: adding 2^52 leaves it in the low bits
__device__ __forceinline__ uint64_t weight_units(double wide) {
#pragma clang fp contract(off)
  return static_cast<uint64_t>(__double_as_longlong(wide + 4503599627370496.0)) & 0xfffffffffffffull;
}

// ceil(share * total) or floor(share * total), exact, for a float share in [0, 1) and total < 2^63.
__device__ __forceinline__ uint64_t share_of(float share, uint64_t total, bool up) {
  const uint32_t bits = __float_as_uint(share), exponent = bits >> 23;
  const uint64_t mantissa = exponent ? (bits & 0x7fffffu) | 0x800000u : bits;
  const int down = 150 - static_cast<int>(exponent ? exponent : 1);          // share = mantissa * 2^-down, down >= 24
  const uint64_t low = mantissa * total, high = __umul64hi(mantissa, total);
  uint64_t whole, rest;
  if (down < 64) whole = (high << (64 - down)) | (low >> down), rest = low << (64 - down);
  else if (down < 128) whole = high >> (down - 64), rest = low | (down > 64 ? high << (128 - down) : 0);
  else whole = 0, rest = low | high;
  return whole + (up && rest != 0 ? 1 : 0);
}

// f(index, values) over the tokens begin .. end - 1 in groups of four that start at multiples of 16 bytes, the THREADS threads side
// by side; what lies outside the range is -inf, a token that nothing counts.  TOGETHER groups a thread are worked on while as many
// more are on their way: a row of 128256 tokens reaches a workgroup from beyond its L2, some 1 us for each batch that it waits for.
template <int THREADS, int TOGETHER, typename F>
__device__ __forceinline__ void scan_tokens(const float* __restrict__ row, int begin, int end, F f) {
  const int ahead = static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 2) & 3;      // tokens by which the row starts past such a place
  const int whole = (begin + ahead + 3) >> 2, past = (end + ahead) >> 2;              // the groups that lie inside
  if (begin >= end) return;
  // a group that the range's ends cut: at most one at each, by a thread each (which lie in one wave)
  if (threadIdx.x < 2) {
    const int g = threadIdx.x == 0 ? whole - 1 : past, first = 4 * g - ahead;
    const bool cut = threadIdx.x == 0 ? first + 4 > begin && first < begin : first < end && (first >= begin || whole > past);
    if (cut && !(threadIdx.x == 1 && first < begin)) {
      float4 v;
      v.x = first >= begin && first < end ? row[first] : -INFINITY;
      v.y = first + 1 >= begin && first + 1 < end ? row[first + 1] : -INFINITY;
      v.z = first + 2 >= begin && first + 2 < end ? row[first + 2] : -INFINITY;
      v.w = first + 3 >= begin && first + 3 < end ? row[first + 3] : -INFINITY;
      f(first, v);
    }
  }
  if (whole >= past) return;
  const float4* groups = reinterpret_cast<const float4*>(row - ahead);
  // (every load is made, past the end the last group's again: under a condition each would be waited for by itself)
  auto bring = [&](int g, float4 (&v)[TOGETHER]) {
#pragma unroll
    for (int u = 0; u < TOGETHER; ++u) v[u] = groups[min(g + u * THREADS, past - 1)];
  };
  float4 now[TOGETHER], next[TOGETHER];
  int g = whole + threadIdx.x;
  bring(g, now);
  for (; g < past; g += TOGETHER * THREADS) {
    bring(g + TOGETHER * THREADS, next);
#pragma unroll
    for (int u = 0; u < TOGETHER; ++u) {
      if (g + u * THREADS < past) f(4 * (g + u * THREADS) - ahead, now[u]);
      now[u] = next[u];
    }
  }
}
template <typename F>
__device__ __forceinline__ void each_of(int index, const float4& v, F f) {
  f(index, v.x), f(index + 1, v.y), f(index + 2, v.z), f(index + 3, v.w);
}

// The parts' kernels have a workgroup a part, the parts of row r on the die r % 8 (workgroups go to the dies in turn), in all of them: what one kernel
// leaves of a row, and the row itself, is in that die's L2 for the next, and the last kernel has row r there by itself.
constexpr int kDies = 8;
__device__ __forceinline__ int row_of(int parts) { return static_cast<int>(blockIdx.x / kDies) / parts * kDies + static_cast<int>(blockIdx.x % kDies); }
__device__ __forceinline__ int part_of(int parts) { return static_cast<int>(blockIdx.x / kDies) % parts; }

// What a thread has seen of the tokens begin .. end - 1: its first largest token's group, the smallest finite logit, and whether one is a NaN or
// +inf (with `finite`, or -inf).  A group of four is compared as one and kept whole, so that which of its tokens it is is asked once, at the end.
struct Seen {
  const int begin, end;
  const bool finite;
  float most = -INFINITY, least = INFINITY;
  float4 group = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  int first = 0;
  bool bad = false;
  __device__ __forceinline__ void take(int index, const float4& v) {
    bad = bad || !(v.x < INFINITY) || !(v.y < INFINITY) || !(v.z < INFINITY) || !(v.w < INFINITY);
    const float here = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
    float low = fminf(fminf(v.x, v.y), fminf(v.z, v.w));
    // a token that cannot be drawn, or none: of the others.  (A branch of the wave: taken lane by lane, 256 rows of 128256 tokens take 89.0 us for 88.4)
    if (__builtin_amdgcn_ballot_w64(low == -INFINITY) != 0) {
      const float none = INFINITY;
      low = fminf(fminf(v.x > -INFINITY ? v.x : none, v.y > -INFINITY ? v.y : none), fminf(v.z > -INFINITY ? v.z : none, v.w > -INFINITY ? v.w : none));
      auto cannot = [&](int i, float x) { return x == -INFINITY && i >= begin && i < end; };
      bad = bad || (finite && (cannot(index, v.x) || cannot(index + 1, v.y) || cannot(index + 2, v.z) || cannot(index + 3, v.w)));
    }
    least = fminf(least, low);
    const bool more = here > most || (here == most && index < first);      // (a thread may meet the range's last, cut group before others)
    most = more ? here : most, first = more ? index : first;
    group.x = more ? v.x : group.x, group.y = more ? v.y : group.y, group.z = more ? v.z : group.z;
  }
  __device__ __forceinline__ uint64_t best() const;
};

struct PartStat {
  uint64_t best;        // place_key of the part's first token in the order; 0: the part has none; all ones: the row cannot be drawn from
  float min;            // the smallest finite logit, +inf: none
  uint32_t unused;
};
constexpr uint64_t kBadPart = ~0ull;
constexpr uint32_t kNotListed = ~0u;
__device__ __forceinline__ uint64_t Seen::best() const {
  if (bad) return kBadPart;
  return most > -INFINITY ? place_key(most, first + (group.x == most ? 0 : group.y == most ? 1 : group.z == most ? 2 : 3)) : 0;
}

__global__ void __launch_bounds__(kPartThreads)
draw_best_kernel(const float* __restrict__ logits, int rows, int vocab, int part_len, int parts, int finite, PartStat* __restrict__ stats) {
  __shared__ uint64_t best_of[kPartThreads / kWave];
  __shared__ float min_of[kPartThreads / kWave];
  const int row = row_of(parts), part = part_of(parts), begin = part * part_len, end = min(vocab, begin + part_len);
  if (row >= rows) return;
  Seen seen{begin, end, finite != 0};
  scan_tokens<kPartThreads, 4>(logits + static_cast<size_t>(row) * vocab, begin, end, [&](int first, const float4& four) { seen.take(first, four); });
  uint64_t best = seen.best();
  float least = seen.least;
  for (int offset = 32; offset > 0; offset >>= 1) {
    const uint64_t other = __shfl_xor(best, offset, 64);
    best = other > best ? other : best;
    least = fminf(least, __shfl_xor(least, offset, 64));
  }
  if ((threadIdx.x & 63) == 0) best_of[threadIdx.x >> 6] = best, min_of[threadIdx.x >> 6] = least;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kPartThreads / kWave; ++w) {
      best = best_of[w] > best ? best_of[w] : best;
      least = fminf(least, min_of[w]);
    }
    stats[static_cast<size_t>(row) * parts + part] = PartStat{best, least, 0};
  }
}

// (all parts are asked for together: one after the other each waits for the one before)
__device__ __forceinline__ void join_stats(const PartStat* __restrict__ stats, int parts, uint64_t& best, float& least) {
  PartStat part[kPartsMost];
#pragma unroll
  for (int p = 0; p < kPartsMost; ++p) part[p] = stats[min(p, parts - 1)];
  best = 0, least = INFINITY;
#pragma unroll
  for (int p = 0; p < kPartsMost; ++p) {
    best = part[p].best > best ? part[p].best : best;
    least = fminf(least, part[p].min);
  }
}

// (the four weights first: with each one's sums behind it, behind a branch, every wave waits for its power alone)
template <bool ALL>
__device__ __forceinline__ void weigh_group(const PoweredScale<ALL>& scale, const float4& four, unsigned long long* mass, uint32_t* count) {
  const float v[4] = {four.x, four.y, four.z, four.w};
  uint64_t units[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) units[j] = weight_units(weight_wide(scale, v[j]));
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (units[j] != 0) {
      const int c = gap_class(scale, v[j]);
      atomicAdd(&mass[c], static_cast<unsigned long long>(units[j]));
      atomicAdd(&count[c], 1u);
    }
}
// exp(v - max), for the log-probability, in 32 bits: the difference, its product and log2(e) itself are rounded, which is 1.2 * 2^-23 of a term for
// each unit of its gap; an exponential and a sum of four add 2 * 2^-23, the rest is summed in 64 bits.  The log-probability is off by the terms' mean: (2 +
// 1.2 g) 2^-23 with g the mean gap of the softmax's tokens (under 17 in any row of 2^24), beside the rounding of its own value.
__device__ __forceinline__ double plain_weights(float max, const float4& v) {
  auto plain = [&](float x) { return __builtin_amdgcn_exp2f((x - max) * 1.44269502f); };
  return static_cast<double>((plain(v.x) + plain(v.y)) + (plain(v.z) + plain(v.w)));
}

__global__ void __launch_bounds__(kPartThreads)
draw_weigh_kernel(const float* __restrict__ logits, int rows, int vocab, int part_len, int parts, const PartStat* __restrict__ stats,
                  const float* __restrict__ temperature, int shift, int want_sum, uint64_t* __restrict__ class_mass,
                  uint32_t* __restrict__ class_count, double* __restrict__ sums) {
  __shared__ unsigned long long mass[kClasses];
  __shared__ uint32_t count[kClasses];
  __shared__ double sum_of[kPartThreads / kWave];
  __shared__ double powers[kPowersHeld<true>];
  const int row = row_of(parts), part = part_of(parts), begin = part * part_len, end = min(vocab, begin + part_len);
  if (row >= rows) return;
  uint64_t best;
  float least;
  join_stats(stats + static_cast<size_t>(row) * parts, parts, best, least);
  if (best == kBadPart || best == 0) return;
  const float t = temperature ? temperature[row] : 0.f;
  const bool drawn = t > 0.f;
  if (!drawn && !want_sum) return;
  bring_powers<true, kPartThreads>(powers, shift);
  for (int c = threadIdx.x; c < kClasses; c += kPartThreads) mass[c] = 0, count[c] = 0;
  __syncthreads();
  const auto scale = row_scale<true>(place_value(best), least, t, shift, powers);
  double sum = 0.0;
  scan_tokens<kPartThreads, 4>(logits + static_cast<size_t>(row) * vocab, begin, end, [&](int, const float4& four) {
    if (drawn) weigh_group(scale, four, mass, count);
    if (want_sum) sum += plain_weights(scale.max, four);
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
#pragma unroll
      for (int w = 1; w < kPartThreads / kWave; ++w) sum += sum_of[w];
      sums[place] = sum;
    }
  }
}

// One token of a class in question: its place in the order, its weight, and of its class the mass and the number of tokens
// before it and its tokens' range in the list.
struct Listed {
  uint64_t key, units, mass_before;
  uint32_t count_before, begin, end, unused;
};
// What the list leaves open of a row: masses that the crossings lie between, and the list's length.
struct RowState {
  uint64_t total_lo, total_hi, kept_floor;
  uint32_t size, cut_k;
};

// Running sums over a wave's lanes, each lane's own included: within the sixteens by shifts, then the sixteens' ends by broadcasts.
template <int CONTROL, int ROWS>
__device__ __forceinline__ void running_step(uint64_t& mass, uint32_t& count) {
  const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(mass), CONTROL, ROWS, 0xf, false);
  const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(mass >> 32), CONTROL, ROWS, 0xf, false);
  mass += (static_cast<uint64_t>(high) << 32) | low;
  count += __builtin_amdgcn_update_dpp(0, count, CONTROL, ROWS, 0xf, false);
}
// Running sums over the workgroup's threads; wave_mass and wave_count: an entry of LDS a wave.
template <int THREADS>
__device__ __forceinline__ void running_sums(uint64_t* wave_mass, uint32_t* wave_count, uint64_t& mass, uint32_t& count) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  running_step<0x111, 0xf>(mass, count);                        // row_shr:1, 2, 4, 8
  running_step<0x112, 0xf>(mass, count);
  running_step<0x114, 0xf>(mass, count);
  running_step<0x118, 0xf>(mass, count);
  running_step<0x142, 0xa>(mass, count);                        // row_bcast:15 into the odd sixteens, row_bcast:31 into the upper half
  running_step<0x143, 0xc>(mass, count);
  if (lane == 63) wave_mass[wave] = mass, wave_count[wave] = count;
  __syncthreads();
  uint64_t m = 0;
  uint32_t n = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) {
    const bool before = w < wave;
    m += before ? wave_mass[w] : 0, n += before ? wave_count[w] : 0;
  }
  mass += m, count += n;
}

// What a row asks for.
struct Ask {
  float t, p, floor, u;
  int k;
};
__device__ __forceinline__ Ask ask_of(int r, const float* uniform, const float* temperature, const int* top_k, const float* top_p, const float* min_p) {
  return Ask{temperature ? temperature[r] : 0.f, top_p ? top_p[r] : 1.f, min_p ? min_p[r] : 0.f, fmaxf(uniform[r], 0.f), top_k ? top_k[r] : 0};
}                                                                 // (a random number that is a NaN counts as 0)
__device__ __forceinline__ uint64_t goal_of(float u, uint64_t kept) { return (u < 1.f ? share_of(u, kept, false) : kept - 1) + 1; }
__device__ __forceinline__ uint64_t target_of(float p, uint64_t total) { return max(share_of(fmaxf(p, 0.f), total, true), static_cast<uint64_t>(1)); }

template <int THREADS>
struct ClassShared {
  uint64_t running_mass[kClasses];          // up to and with each class
  uint32_t running_count[kClasses];
  uint32_t begin[kClasses];                 // a wanted class's first place in the list, or kNotListed
  uint32_t place[kClasses];                 // where its next token goes
  uint64_t wave_mass[THREADS / kWave];
  uint32_t wave_count[THREADS / kWave], listed_count[THREADS / kWave];
  int found[7];                             // classes, a place for each question
  uint32_t held_count;                      // of list_tokens
};

// From the masses and counts of a thread's own classes (kClasses / THREADS neighbours): which classes the crossings lie in, and
// where their tokens go in the list, class after class, `ahead` of them left free at each class's start.  The whole workgroup; what it
// leaves in s may be read at once.
template <int THREADS>
__device__ RowState find_classes(ClassShared<THREADS>& s, const RowScale& scale, uint64_t one, const Ask& ask,
                                 const uint64_t (&mass)[kClasses / THREADS], const uint32_t (&count)[kClasses / THREADS],
                                 const uint32_t (&ahead)[kClasses / THREADS]) {
  constexpr int kOwn = kClasses / THREADS;
  const int tid = threadIdx.x;
  uint64_t running[kOwn];
  uint32_t running_n[kOwn];
  {
    uint64_t all = 0;
    uint32_t all_n = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) all += mass[j], all_n += count[j];
    const uint64_t own = all;
    const uint32_t own_n = all_n;
    if (tid < 7) s.found[tid] = kClasses;
    if (tid == 0) s.held_count = 0;
    running_sums<THREADS>(s.wave_mass, s.wave_count, all, all_n);
    all -= own, all_n -= own_n;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      running[j] = all += mass[j], running_n[j] = all_n += count[j];
      s.running_mass[kOwn * tid + j] = running[j], s.running_count[kOwn * tid + j] = running_n[j];
    }
  }
  __syncthreads();
  auto mass_upto = [&](int c) -> uint64_t { return c < 0 ? 0 : s.running_mass[min(c, kClasses - 1)]; };
  auto reaches = [&](int question, uint64_t target) {              // the class (if any) at which the running mass reaches a target > 0
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (running[j] >= target && running[j] - mass[j] < target) s.found[question] = kOwn * tid + j;
  };
  bool wanted[kOwn] = {};
  auto want = [&](int lo, int hi) {
#pragma unroll
    for (int j = 0; j < kOwn; ++j) wanted[j] = wanted[j] || (kOwn * tid + j >= lo && kOwn * tid + j <= hi);
  };

  // ---- which classes the crossings can lie in.  A class that is cut leaves what follows with a range of masses ----
  RowState state;
  state.total_lo = state.total_hi = s.running_mass[kClasses - 1], state.kept_floor = one, state.cut_k = 0;
  const uint32_t k = static_cast<uint32_t>(ask.k);
  if (ask.k > 0 && k < s.running_count[kClasses - 1]) {
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (running_n[j] >= k && running_n[j] - count[j] < k) s.found[0] = kOwn * tid + j;
    __syncthreads();
    const int c = s.found[0];
    state.total_hi = mass_upto(c), state.total_lo = s.running_count[c] == k ? state.total_hi : mass_upto(c - 1);
    state.cut_k = state.total_lo != state.total_hi;
    if (state.cut_k) want(c, c);
  }
  uint64_t kept_lo = state.total_lo, kept_hi = state.total_hi;
  if (ask.p < 1.f) {
    const uint64_t low = target_of(ask.p, state.total_lo);
    reaches(1, low);
    reaches(2, state.cut_k ? target_of(ask.p, state.total_hi) : low);
    __syncthreads();
    const int c_lo = s.found[1], c_hi = s.found[2];
    want(c_lo, c_hi);
    kept_lo = mass_upto(c_lo - 1), kept_hi = min(kept_hi, mass_upto(c_hi));
  }
  if (ask.floor > 1.f) {
    kept_lo = kept_hi = one;                                      // (no weight reaches it)
  } else if (ask.floor > 0.f) {
    // The class of the gap at which the weight is min_p, and its neighbours, for the rounding of the gap; of 1, up to the gap of 2^-52 T: nearer weights
    // may be rounded to the largest's, which at a very high temperature can be every token's.
    auto class_at = [&](float gap) { return static_cast<int>(fminf(gap * scale.class_scale, static_cast<float>(kClasses - 1))); };
    const float gap = fmaxf(-logf(ask.floor), 0.f);
    const int first = gap > 0.f ? class_at(gap * ask.t) : 0, last = class_at(fmaxf(gap, 2.220446e-16f) * ask.t);
    want(first - 1, last + 1);
    state.kept_floor = max(one, mass_upto(first - 2));
    kept_lo = min(kept_lo, state.kept_floor), kept_hi = min(kept_hi, mass_upto(last + 1));
  }
  kept_lo = max(kept_lo, one), kept_hi = max(kept_hi, one);       // (the first token is always kept)
  const uint64_t goal = goal_of(ask.u, kept_lo);
  reaches(3, goal);
  reaches(4, kept_lo != kept_hi ? goal_of(ask.u, kept_hi) : goal);
  __syncthreads();
  want(s.found[3], s.found[4]);

  // ---- their places in the list ----
  uint64_t nothing = 0;
  uint32_t listed = 0;
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    wanted[j] = wanted[j] && mass[j] != 0;
    if (wanted[j]) {
      listed += count[j];
      atomicMin(&s.found[5], kOwn * tid + j), atomicMin(&s.found[6], kClasses - 1 - (kOwn * tid + j));
    }
  }
  const uint32_t own_listed = listed;
  running_sums<THREADS>(s.wave_mass, s.listed_count, nothing, listed);
  listed -= own_listed;
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    s.begin[kOwn * tid + j] = wanted[j] ? listed : kNotListed;
    s.place[kOwn * tid + j] = listed + ahead[j];
    listed += wanted[j] ? count[j] : 0;
  }
  state.size = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) state.size += s.listed_count[w];
  __syncthreads();
  return state;
}

// The values between which the classes in question lie, so that the others' tokens cost a comparison (differences of logits are
// rounded to 2^-24 of the larger, and the class's bound again: room on either side).
template <int THREADS>
__device__ __forceinline__ void value_bounds(const ClassShared<THREADS>& s, const RowScale& scale, float least, float& lower, float& upper) {
  const int c_first = s.found[5], c_last = kClasses - 1 - s.found[6];
  lower = -3.4028235e38f, upper = INFINITY;
  if (scale.class_scale > 0.f) {                                  // (else every token is of the first class)
    // (tokens that weigh lie within 34 T of the first; the smallest logit may be the least there is)
    const float room = (fabsf(scale.max) + fminf(scale.max - least, static_cast<float>(-scale.least))) * 2.4e-7f;
    upper = scale.max - static_cast<float>(c_first) * 0.99999f / scale.class_scale + room;
    if (c_last < kClasses - 1) lower = scale.max - static_cast<float>(c_last + 1) * 1.00001f / scale.class_scale - room;
  }
}
__device__ __forceinline__ bool any_between(const float4& v, float lower, float upper) {
  return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= lower && fminf(fminf(v.x, v.y), fminf(v.z, v.w)) <= upper;
}
// A token that a wanted class holds, until its weight is formed.
struct Held {
  float v;
  int index;
};
// found(place in the list, key, weight, class) for each token of begin .. end - 1 that a wanted class holds, by the whole workgroup.  They are
// few: with their weights formed where they are met, nearly every wave's step waits for one lane's; held back, they are formed side by side.
// held: kListMost places (more tokens than that, of no weight then, are looked at where they are met).  Ends before a barrier that the
// caller needs for what it does with `held` or what `found` wrote.
template <int THREADS, int TOGETHER, bool ALL, typename F>
__device__ __forceinline__ void list_tokens(ClassShared<THREADS>& s, const PoweredScale<ALL>& scale, float lower, float upper, const float* __restrict__ row,
                                            int begin, int end, Held* held, F found) {
  auto list = [&](float v, int i) {
    const uint64_t units = weight_units(weight_wide(scale, v));
    const int c = gap_class(scale, v);
    if (units != 0) found(atomicAdd(&s.place[c], 1u), place_key(v, i), units, c);
  };
  scan_tokens<THREADS, TOGETHER>(row, begin, end, [&](int first, const float4& four) {
    if (!any_between(four, lower, upper)) return;
    each_of(first, four, [&](int i, float v) {
      if (!(v >= lower && v <= upper) || s.begin[gap_class(scale, v)] == kNotListed) return;
      const uint32_t place = atomicAdd(&s.held_count, 1u);
      if (place < kListMost) held[place] = Held{v, i};
      else list(v, i);
    });
  });
  __syncthreads();
  const uint32_t count = min(s.held_count, static_cast<uint32_t>(kListMost));
  for (uint32_t j = threadIdx.x; j < count; j += THREADS) list(held[j].v, held[j].index);
}
template <int THREADS>
__device__ __forceinline__ Listed listed_of(const ClassShared<THREADS>& s, uint64_t key, uint64_t units, int c) {
  const uint32_t before = c > 0 ? s.running_count[c - 1] : 0, from = s.begin[c];
  return Listed{key, units, c > 0 ? s.running_mass[c - 1] : 0, before, from, from + s.running_count[c] - before, 0};
}

struct Entry {
  uint64_t key, units;
};
template <int THREADS>
struct CrossShared {
  Entry list[kListMost];                    // bucket by bucket
  uint64_t bucket_mass[kListMost];          // of a bucket, then up to it
  uint32_t bucket_count[kListMost], place[kListMost];
  uint64_t wave_mass[THREADS / kWave];
  uint32_t wave_count[THREADS / kWave];
  uint64_t digit_mass[256];
  uint32_t digit_count[256];
  uint64_t answers[4], answer_key;          // of the crossings
  int found;
};

// The chosen token, from the list: entry(i) is its i-th.
template <int THREADS, bool ALL, typename F>
__device__ uint64_t cross(CrossShared<THREADS>& s, const PoweredScale<ALL>& scale, const Ask& ask, const RowState& state, uint64_t best, F entry) {
  constexpr int kEach = kListMost / THREADS;
  const int tid = threadIdx.x, size = static_cast<int>(state.size);
  // A token's running mass and rank: up to the class before, and of its own class what stands no later.  The list's tokens go into
  // as many buckets as they are, a class's tokens into its own by their gap, in the order; what stands in earlier buckets
  // comes from running sums, and a token is compared with those of its bucket alone.  (Compared with all of its class, 500 tokens
  // of one class took 90 us.)
  uint64_t key[kEach], units[kEach] = {}, reached[kEach];
  uint32_t rank[kEach];
  Listed own[kEach];
  int bucket[kEach];
  if (tid == 0) s.answers[0] = state.total_hi, s.answers[1] = state.total_hi, s.answers[2] = state.kept_floor, s.answer_key = best;
  for (int b = tid; b < kListMost; b += THREADS) s.bucket_mass[b] = 0, s.bucket_count[b] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = tid + j * THREADS;
    if (i >= size) continue;
    own[j] = entry(i);
    key[j] = own[j].key, units[j] = own[j].units;
    const float v = place_value(key[j]);
    // (the gap in classes without the whole ones, of the last class's tokens possibly more than one)
    const float x = v < scale.max ? (scale.max - v) * scale.class_scale : 0.f;
    const float inside = fminf(fmaxf(x - fminf(floorf(x), static_cast<float>(kClasses - 1)), 0.f) * 2048.f, 2047.f);
    bucket[j] = static_cast<int>(own[j].begin + ((static_cast<uint32_t>(inside) * (own[j].end - own[j].begin)) >> 11));
    atomicAdd(reinterpret_cast<unsigned long long*>(&s.bucket_mass[bucket[j]]), static_cast<unsigned long long>(units[j]));
    atomicAdd(&s.bucket_count[bucket[j]], 1u);
  }
  __syncthreads();
  {
    uint64_t mass[kEach], all = 0;
    uint32_t count[kEach], all_n = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) all += mass[j] = s.bucket_mass[kEach * tid + j], all_n += count[j] = s.bucket_count[kEach * tid + j];
    const uint64_t own_all = all;
    const uint32_t own_n = all_n;
    running_sums<THREADS>(s.wave_mass, s.wave_count, all, all_n);
    all -= own_all, all_n -= own_n;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      s.bucket_mass[kEach * tid + j] = all, s.place[kEach * tid + j] = all_n;              // before the bucket
      all += mass[j], all_n += count[j];
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (units[j] == 0) continue;
    // (the mass before the bucket in its class: before the class's first bucket the list holds what is not the row's)
    reached[j] = own[j].mass_before + s.bucket_mass[bucket[j]] - s.bucket_mass[own[j].begin];
    rank[j] = own[j].count_before + s.place[bucket[j]] - own[j].begin;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (units[j] != 0) s.list[atomicAdd(&s.place[bucket[j]], 1u)] = Entry{key[j], units[j]};
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (units[j] == 0) continue;
    const uint32_t end = s.place[bucket[j]];
    for (uint32_t other = end - s.bucket_count[bucket[j]]; other < end; ++other) {
      const Entry other_entry = s.list[other];
      const bool stands = other_entry.key >= key[j];
      reached[j] += stands ? other_entry.units : 0, rank[j] += stands ? 1 : 0;
    }
  }
  auto crosses = [&](int j, uint64_t target) { return units[j] != 0 && reached[j] >= target && reached[j] - units[j] < target; };
  uint64_t kept = state.total_lo;
  if (state.cut_k) {
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (units[j] != 0 && rank[j] == static_cast<uint32_t>(ask.k)) s.answers[0] = reached[j];
    __syncthreads();
    kept = s.answers[0];
  }
  if (ask.p < 1.f) {
    const uint64_t target = target_of(ask.p, kept);
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (crosses(j, target)) s.answers[1] = reached[j];
    __syncthreads();
    kept = s.answers[1];
  }
  if (ask.floor > 0.f) {
    const double least_weight = static_cast<double>(ask.floor) * scale.one;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (units[j] != 0 && weight_wide(scale, place_value(key[j])) >= least_weight)
        atomicMax(reinterpret_cast<unsigned long long*>(&s.answers[2]), static_cast<unsigned long long>(reached[j]));
    __syncthreads();
    kept = min(kept, s.answers[2]);
  }
  const uint64_t goal = goal_of(ask.u, kept);
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (crosses(j, goal)) s.answer_key = key[j];
  __syncthreads();
  return s.answer_key;
}

// Without a list (more tokens than it holds share the classes in question): the place in the order where the running mass
// (or count) reaches target, found digit by digit of the place keys, eight passes over the row.  Returns the running mass there.
template <int THREADS, bool ALL>
__device__ __forceinline__ uint64_t descend(CrossShared<THREADS>& s, const float* __restrict__ row, int vocab, const PoweredScale<ALL>& scale, uint64_t target, bool by_count,
                                         uint64_t* key) {
  uint64_t prefix = 0, mass_before = 0, count_before = 0, mass = 0;
  for (int digit = 7; digit >= 0; --digit) {
    for (int b = threadIdx.x; b < 256; b += THREADS) s.digit_mass[b] = 0, s.digit_count[b] = 0;
    __syncthreads();
    scan_tokens<THREADS, 4>(row, 0, vocab, [&](int first, const float4& four) {
      each_of(first, four, [&](int i, float v) {
        if (!(v > -INFINITY)) return;
        const uint64_t place = place_key(v, i);
        if (digit < 7 && (place >> (8 * digit + 8)) != (prefix >> (8 * digit + 8))) return;
        const uint64_t units = weight_units(weight_wide(scale, v));
        if (units == 0) return;
        const int b = static_cast<int>((place >> (8 * digit)) & 255);
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.digit_mass[b]), static_cast<unsigned long long>(units));
        atomicAdd(&s.digit_count[b], 1u);
      });
    });
    __syncthreads();
    if (threadIdx.x == 0) {
      int b = 255;
      uint64_t m = mass_before, n = count_before;
      for (; b > 0; --b) {
        if ((by_count ? n + s.digit_count[b] : m + s.digit_mass[b]) >= target) break;
        m += s.digit_mass[b], n += s.digit_count[b];
      }
      s.found = b, s.wave_mass[0] = m, s.wave_mass[1] = n, s.wave_mass[2] = m + s.digit_mass[b];
    }
    __syncthreads();
    prefix |= static_cast<uint64_t>(s.found) << (8 * digit);
    mass_before = s.wave_mass[0], count_before = s.wave_mass[1], mass = s.wave_mass[2];
    __syncthreads();
  }
  *key = prefix;
  return mass;
}
template <int THREADS, bool ALL>
__device__ uint64_t cross_without_list(CrossShared<THREADS>& s, const float* __restrict__ row, int vocab, const PoweredScale<ALL>& scale, uint64_t one, const Ask& ask,
                                       const RowState& state) {
  uint64_t place = 0, kept = state.total_lo;
  __syncthreads();
  for (int step = 0; step < 3; ++step) {                          // top_k, top_p, the draw: a loop, so that the code is there once
    if ((step == 0 && !state.cut_k) || (step == 1 && !(ask.p < 1.f))) continue;
    if (step == 2 && ask.floor > 0.f) {
      const double least_weight = static_cast<double>(ask.floor) * scale.one;
      if (threadIdx.x == 0) s.answers[3] = 0;
      __syncthreads();
      scan_tokens<THREADS, 4>(row, 0, vocab, [&](int first, const float4& four) {
        each_of(first, four, [&](int, float v) {
          const double wide = weight_wide(scale, v);
          if (v > -INFINITY && wide >= least_weight)
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.answers[3]), static_cast<unsigned long long>(weight_units(wide)));
        });
      });
      __syncthreads();
      kept = min(kept, max(s.answers[3], one));
    }
    const uint64_t target = step == 0 ? static_cast<uint64_t>(ask.k) : step == 1 ? target_of(ask.p, kept) : goal_of(ask.u, kept);
    kept = descend(s, row, vocab, scale, target, step == 0, &place);
  }
  return place;
}

__global__ void __launch_bounds__(kGatherThreads)
draw_gather_kernel(const float* __restrict__ logits, int rows, int vocab, int part_len, int parts, const PartStat* __restrict__ stats,
                   const float* __restrict__ uniform, const float* __restrict__ temperature, const int* __restrict__ top_k,
                   const float* __restrict__ top_p, const float* __restrict__ min_p, int shift, const uint64_t* __restrict__ class_mass,
                   const uint32_t* __restrict__ class_count, RowState* __restrict__ states, Listed* __restrict__ lists) {
  __shared__ ClassShared<kGatherThreads> s;
  __shared__ Held held[kListMost];
  __shared__ double powers[kPowersHeld<false>];
  const int r = row_of(parts), part = part_of(parts), tid = threadIdx.x;
  if (r >= rows) return;
  const Ask ask = ask_of(r, uniform, temperature, top_k, top_p, min_p);
  if (!(ask.t > 0.f)) return;
  uint64_t best;
  float least;
  join_stats(stats + static_cast<size_t>(r) * parts, parts, best, least);
  if (best == kBadPart || best == 0) return;
  bring_powers<false, kGatherThreads>(powers, shift);
  const auto scale = row_scale<false>(place_value(best), least, ask.t, shift, powers);
  // the row's classes, four neighbours a thread; all parts are asked for together.  (Four waves: with a class a thread, sixteen
  // waves do what is the same for all of the row, and 64 rows in 8 parts took 20 us)
  constexpr int kOwn = kClasses / kGatherThreads;
  static_assert(kOwn == 4, "classes are loaded as 16-byte pieces");
  uint64_t mass[kOwn] = {};
  uint32_t count[kOwn] = {}, ahead[kOwn] = {};                    // (ahead: of the parts before this one)
  ulonglong2 m[kPartsMost][2];
  uint4 n[kPartsMost];
#pragma unroll
  for (int p = 0; p < kPartsMost; ++p) {
    const size_t place = (static_cast<size_t>(r) * parts + min(p, parts - 1)) * kClasses + kOwn * tid;
    m[p][0] = *reinterpret_cast<const ulonglong2*>(class_mass + place), m[p][1] = *reinterpret_cast<const ulonglong2*>(class_mass + place + 2);
    n[p] = *reinterpret_cast<const uint4*>(class_count + place);
  }
#pragma unroll
  for (int p = 0; p < kPartsMost; ++p) {
    // (selected, not branched around: the loads would move behind the branch, and each be waited for by itself)
    const bool is = p < parts, before = p < part;
    mass[0] += is ? m[p][0].x : 0, mass[1] += is ? m[p][0].y : 0, mass[2] += is ? m[p][1].x : 0, mass[3] += is ? m[p][1].y : 0;
    ahead[0] += before ? n[p].x : 0, ahead[1] += before ? n[p].y : 0, ahead[2] += before ? n[p].z : 0, ahead[3] += before ? n[p].w : 0;
    count[0] += is ? n[p].x : 0, count[1] += is ? n[p].y : 0, count[2] += is ? n[p].z : 0, count[3] += is ? n[p].w : 0;
  }
  const RowState state = find_classes<kGatherThreads>(s, scale, 1ull << shift, ask, mass, count, ahead);
  if (part == 0 && tid == 0) states[r] = state;
  if (state.size > kListMost) return;
  float lower, upper;
  value_bounds(s, scale, least, lower, upper);
  const int begin = part * part_len, end = min(vocab, begin + part_len);
  Listed* list = lists + static_cast<size_t>(r) * kListMost;
  list_tokens<kGatherThreads, 8>(s, scale, lower, upper, logits + static_cast<size_t>(r) * vocab, begin, end, held,
                                 [&](uint32_t place, uint64_t key, uint64_t units, int c) { list[place] = listed_of(s, key, units, c); });
}

__global__ void __launch_bounds__(kPickThreads)
draw_pick_kernel(const float* __restrict__ logits, int vocab, int parts, const PartStat* __restrict__ stats, const float* __restrict__ uniform,
                 const float* __restrict__ temperature, const int* __restrict__ top_k, const float* __restrict__ top_p,
                 const float* __restrict__ min_p, int shift, const RowState* __restrict__ states, const Listed* __restrict__ lists,
                 const double* __restrict__ sums, int* __restrict__ out, float* __restrict__ logprob) {
  __shared__ CrossShared<kPickThreads> s;
  __shared__ double powers[kPowersHeld<false>];
  const int r = blockIdx.x, tid = threadIdx.x;
  const Ask ask = ask_of(r, uniform, temperature, top_k, top_p, min_p);
  const Listed* list = lists + static_cast<size_t>(r) * kListMost;
  const RowState state = states[r];                               // (of a row that is not drawn: anything, not looked at)
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
  double log_sum = 0.0;
  if (tid == 0 && logprob) {
    double sum = 0.0;
    for (int p = 0; p < parts; ++p) sum += sums[static_cast<size_t>(r) * parts + p];
    log_sum = log(sum);
  }
  uint64_t chosen = best;
  if (ask.t > 0.f) {
    bring_powers<false, kPickThreads>(powers, shift);
    const auto scale = row_scale<false>(place_value(best), least, ask.t, shift, powers);
    if (state.size <= kListMost)
      chosen = cross(s, scale, ask, state, best, [&](int i) { return list[i]; });
    else
      chosen = cross_without_list(s, logits + static_cast<size_t>(r) * vocab, vocab, scale, 1ull << shift, ask, state);
  }
  if (tid == 0) {
    out[r] = place_index(chosen);
    if (logprob) logprob[r] = static_cast<float>(static_cast<double>(place_value(chosen)) - static_cast<double>(place_value(best)) - log_sum);
  }
}

struct RowShared {
  ClassShared<kRowThreads> classes;
  CrossShared<kRowThreads> cross;
  double powers[kPowersHeld<true>];
  uint64_t wave_best[kRowThreads / kWave];
  float wave_least[kRowThreads / kWave];
  double wave_sum[kRowThreads / kWave];
};

// All of the above for a row by one workgroup, in one launch: three passes over the row, of which the later ones find it in the L2.
// (Kept in registers instead, 64 tokens a thread, every pass is code written out 64 times: 100 KB of it, brought from memory as it
// runs, 28 us for a row of 32000 tokens.)
__global__ void __launch_bounds__(kRowThreads)
draw_row_kernel(const float* __restrict__ logits, int vocab, const float* __restrict__ uniform, const float* __restrict__ temperature,
                const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p, int shift, int finite,
                int* __restrict__ out, float* __restrict__ logprob) {
  __shared__ RowShared s;
  constexpr int kWaves = kRowThreads / kWave, kOwn = kClasses / kRowThreads;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* row = logits + static_cast<size_t>(r) * vocab;
  const Ask ask = ask_of(r, uniform, temperature, top_k, top_p, min_p);
  // ---- the first token, the least logit, and whether the row can be drawn from ----
  Seen seen{0, vocab, finite != 0};
  scan_tokens<kRowThreads, 4>(row, 0, vocab, [&](int first, const float4& four) { seen.take(first, four); });
  uint64_t best = seen.best();
  float least = seen.least;
  for (int offset = 32; offset > 0; offset >>= 1) {
    const uint64_t other = __shfl_xor(best, offset, 64);
    best = other > best ? other : best;
    least = fminf(least, __shfl_xor(least, offset, 64));
  }
  if (lane == 0) s.wave_best[wave] = best, s.wave_least[wave] = least;
  bring_powers<true, kRowThreads>(s.powers, shift);
  unsigned long long* mass_of = reinterpret_cast<unsigned long long*>(s.classes.running_mass);       // the histogram, until it is summed up
  uint32_t* count_of = s.classes.running_count;
  for (int c = tid; c < kClasses; c += kRowThreads) mass_of[c] = 0, count_of[c] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    best = s.wave_best[w] > best ? s.wave_best[w] : best;
    least = fminf(least, s.wave_least[w]);
  }
  if (best == kBadPart || best == 0) {
    if (tid == 0) {
      out[r] = -1;
      if (logprob) logprob[r] = __uint_as_float(0x7fc00000u);
    }
    return;
  }
  const auto scale = row_scale<true>(place_value(best), least, ask.t, shift, s.powers);
  // ---- the weights, and the sum of the log-probability's ----
  double sum = 0.0;
  scan_tokens<kRowThreads, 2>(row, 0, vocab, [&](int, const float4& four) {
    if (ask.t > 0.f) weigh_group(scale, four, mass_of, count_of);
    if (logprob) sum += plain_weights(scale.max, four);
  });
  if (logprob) {
    for (int offset = 32; offset > 0; offset >>= 1) sum += __shfl_xor(sum, offset, 64);
    if (lane == 0) s.wave_sum[wave] = sum;
  }
  uint64_t chosen = best;
  if (ask.t > 0.f) {
    __syncthreads();
    uint64_t mass[kOwn];
    uint32_t count[kOwn], ahead[kOwn] = {};
#pragma unroll
    for (int j = 0; j < kOwn; ++j) mass[j] = mass_of[kOwn * tid + j], count[j] = count_of[kOwn * tid + j];
    const RowState state = find_classes<kRowThreads>(s.classes, scale, 1ull << shift, ask, mass, count, ahead);
    if (state.size <= kListMost) {
      float lower, upper;
      value_bounds(s.classes, scale, least, lower, upper);
      static_assert(sizeof(s.cross.bucket_mass) >= kListMost * sizeof(Held), "free until the crossings are looked for");
      list_tokens<kRowThreads, 4>(s.classes, scale, lower, upper, row, 0, vocab, reinterpret_cast<Held*>(s.cross.bucket_mass),
                                  [&](uint32_t place, uint64_t key, uint64_t units, int) { s.cross.list[place] = Entry{key, units}; });
      __syncthreads();
      // (the crossings read an entry before they write the list again, with barriers in between)
      chosen = cross(s.cross, scale, ask, state, best, [&](int i) {
        const Entry entry = s.cross.list[i];
        return listed_of(s.classes, entry.key, entry.units, gap_class(scale, place_value(entry.key)));
      });
    } else {
      chosen = cross_without_list(s.cross, row, vocab, scale, 1ull << shift, ask, state);
    }
  } else {
    __syncthreads();
  }
  if (tid == 0) {
    out[r] = place_index(chosen);
    if (logprob) {
      double sum = 0.0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) sum += s.wave_sum[w];
      logprob[r] = static_cast<float>(static_cast<double>(place_value(chosen)) - static_cast<double>(place_value(best)) - log(sum));
    }
  }
}

}  // namespace tlie

using namespace tlie;

// The entry's scratch, for `parts` parts a row: the rows' lists and states, the parts' statistics, masses and counts of classes, and sums.
constexpr long long kRowBytes = sizeof(RowState) + kListMost * sizeof(Listed), kPartBytes = sizeof(PartStat) + 8 + kClasses * 12;
static_assert(sizeof(RowState) == 32 && sizeof(Listed) == 40 && sizeof(PartStat) == 16, "the host's face counts them so");

// Where each begins, in bytes.  Classes are read 16 bytes at a time, so what stands before them has a multiple of 16 whatever the number of rows
// and parts (a row's list 80 KB); the sums, of 8 bytes each, stand last.
struct Scratch {
  long long lists, states, stats, class_mass, class_count, sums, end;
};
static Scratch scratch_of(long long rows, long long parts) {
  static_assert(kListMost * sizeof(Listed) % 16 == 0 && sizeof(RowState) % 16 == 0 && sizeof(PartStat) % 16 == 0 && kClasses % 4 == 0, "read in pieces of 16 bytes");
  const long long places = rows * parts;
  Scratch s{};
  s.states = s.lists + rows * kListMost * static_cast<long long>(sizeof(Listed));
  s.stats = s.states + rows * static_cast<long long>(sizeof(RowState));
  s.class_mass = s.stats + places * static_cast<long long>(sizeof(PartStat));
  s.class_count = s.class_mass + places * kClasses * 8;
  s.sums = s.class_count + places * kClasses * 4;
  s.end = s.sums + places * 8;
  return s;
}

// The starts of a scratch's seven pieces (the last: its end), for rows in `parts` parts each.
extern "C" void tlie_draw_scratch(int rows, int parts, long long* starts) {
  const Scratch s = scratch_of(rows, parts);
  const long long values[7] = {s.lists, s.states, s.stats, s.class_mass, s.class_count, s.sums, s.end};
  for (int i = 0; i < 7; ++i) starts[i] = values[i];
}

// logits: float [rows, vocab], vocab < 2^24; uniform: float [rows]; temperature, top_k, top_p, min_p: [rows] or null; parts: 1 to 8, or 0: a row by
// one workgroup (scratch is then null);
// finite: not 0, a row with a logit of -inf cannot be drawn from either; out: int [rows]; logprob: float [rows] or null.  scratch: rows * (kRowBytes + parts * kPartBytes) bytes, at a multiple of 16.
extern "C" int tlie_draw(const float* logits, int rows, int vocab, const float* uniform, const float* temperature, const int* top_k,
                         const float* top_p, const float* min_p, int finite, int parts, void* scratch, int* out, float* logprob, void* stream) {
  if (rows <= 0 || vocab <= 0 || vocab >= (1 << 24) || parts < 0 || parts > kPartsMost || rows > 65535 ||
      uniform == nullptr || (parts > 0 && (scratch == nullptr || reinterpret_cast<uintptr_t>(scratch) % 16 != 0)))
    return kBadArgument;
  hipStream_t s = (hipStream_t)stream;
  int shift = 44;                                   // the weights' sum stays below 2^62
  while ((static_cast<long long>(vocab) << shift) >= (1ll << 62)) --shift;
  if (parts == 0) {
    hipLaunchKernelGGL(draw_row_kernel, dim3(rows), dim3(kRowThreads), 0, s, logits, vocab, uniform, temperature, top_k, top_p, min_p, shift,
                       finite, out, logprob);
    return launch_status();
  }
  const int part_len = (vocab + parts - 1) / parts;
  const Scratch at = scratch_of(rows, parts);
  unsigned char* base = static_cast<unsigned char*>(scratch);
  Listed* lists = reinterpret_cast<Listed*>(base + at.lists);
  RowState* states = reinterpret_cast<RowState*>(base + at.states);
  PartStat* stats = reinterpret_cast<PartStat*>(base + at.stats);
  uint64_t* class_mass = reinterpret_cast<uint64_t*>(base + at.class_mass);
  uint32_t* class_count = reinterpret_cast<uint32_t*>(base + at.class_count);
  double* sums = reinterpret_cast<double*>(base + at.sums);
  const dim3 grid((rows + kDies - 1) / kDies * kDies * parts);
  hipLaunchKernelGGL(draw_best_kernel, grid, dim3(kPartThreads), 0, s, logits, rows, vocab, part_len, parts, finite, stats);
  hipLaunchKernelGGL(draw_weigh_kernel, grid, dim3(kPartThreads), 0, s, logits, rows, vocab, part_len, parts, stats, temperature, shift,
                     logprob != nullptr ? 1 : 0, class_mass, class_count, sums);
  if (temperature != nullptr)
    hipLaunchKernelGGL(draw_gather_kernel, grid, dim3(kGatherThreads), 0, s, logits, rows, vocab, part_len, parts, stats, uniform, temperature,
                     top_k, top_p, min_p, shift, class_mass, class_count, states, lists);
  hipLaunchKernelGGL(draw_pick_kernel, dim3(rows), dim3(kPickThreads), 0, s, logits, vocab, parts, stats, uniform, temperature, top_k, top_p, min_p,
                     shift, states, lists, sums, out, logprob);
  return launch_status();
}
