// Paged causal attention for sequences that share the keys and values of their first positions: several answers to one
// prompt, or several questions behind one document.
//
// reference: none (the reference's step reads every sequence's whole cache by itself, src/cuda/kernels.cu:147-196).
//
// The softmax over a token's keys is a sum over sets of keys that may be formed set by set: with m_i the largest score of
// set i, l_i = sum exp(s - m_i) and o_i = sum exp(s - m_i) v, the result is sum_i w_i o_i / sum_i w_i l_i with
// w_i = exp(m_i - max m).  So the keys 0 .. P - 1 that a group of sequences has in common are read once for the columns
// (token, query head) of all its tokens, as one matrix product of many columns without any mask, and the keys P .. p of
// a token at position p once for its own sequence.  The host cuts both into items, (columns, keys) ranges of about equal work,
// one workgroup each and kv head; what they leave (m, l and o in 32 bits) is joined by a second kernel in a fixed order.
//
// Inside an item scores are formed transposed, S^T = K . Q^T, so that a lane of the result holds 4 keys of one column, which
// is the layout that the second product O^T = V^T . P^T wants of P: nothing passes through LDS until the four waves, which
// take blocks of keys in turn, add up what they have.  bfloat16 on 16x16x32, 32 keys a block, p rounded to bfloat16 (its
// relative error 2^-9 is that of a value; sums, maxima and o are float); float on 16x16x4, 16 keys a block, nothing rounded.
#include "common.h"

#include <type_traits>

namespace tlie {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;

// One item: columns col0 .. of the (token, head of the kv head) pairs of `ntok` tokens from tok0 on, keys key_lo .. key_hi - 1
// that row `table` of the block table holds.  own: the tokens follow one another in one sequence, the first at
// positions[tok0], and see keys up to their own; else they see all of the item's.  part: which of its tokens' parts this is.
struct PrefixItem {
  int table, tok0, ntok, col0, key_lo, key_hi, own, part;
};

constexpr int kPrefixWaves = 4;

template <int DT, bool FLOAT, int CT>
__device__ __forceinline__ void prefix_item(const PrefixItem& item, int kvh, const void* __restrict__ q_any, const void* __restrict__ cache_any,
                                            const int* __restrict__ pages, int max_blocks, const int* __restrict__ positions,
                                            const int* __restrict__ part_first, float* __restrict__ part_o, float* __restrict__ part_ml,
                                            int nq, int nkv, int page_shift, float scale_log2, float cap_pre, float* lds) {
  using Elem = std::conditional_t<FLOAT, float, uint16_t>;
  constexpr int D = DT * 16, TILES = FLOAT ? 1 : 2, BLOCK = 16 * TILES;     // keys a block
  constexpr int KS = FLOAT ? DT : (DT + 1) / 2;                             // 16-byte pieces of a key that a lane holds
  typedef uint32_t Piece __attribute__((ext_vector_type(4)));
  typedef uint32_t Half __attribute__((ext_vector_type(2)));
  using Values = std::conditional_t<FLOAT, Piece, Half>;                    // 4 keys of a dim
  const Elem* q = static_cast<const Elem*>(q_any);
  const Elem* cache = static_cast<const Elem*>(cache_any);
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int G = nq / nkv, ncols = item.ntok * G, page_mask = (1 << page_shift) - 1;
  const int pos0 = item.own ? __builtin_amdgcn_readfirstlane(positions[item.tok0]) : 0;
  constexpr int kPiece = FLOAT ? 4 : 8;                                     // elements of a 16-byte piece
  auto has_dims = [&](int ks) { return FLOAT || DT % 2 == 0 || ks < KS - 1 || grp < 2; };

  int tok[CT], head[CT], last_key[CT];
  bool valid[CT];
  Piece query[CT][KS];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = item.col0 + ct * 16 + col;
    valid[ct] = c < ncols;
    tok[ct] = item.tok0 + (valid[ct] ? c / G : 0);
    head[ct] = kvh * G + (valid[ct] ? c % G : 0);
    last_key[ct] = !valid[ct] ? -1 : item.own ? pos0 + c / G : 0x7fffffff;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      query[ct][ks] = Piece{0, 0, 0, 0};
      if (valid[ct] && has_dims(ks))
        query[ct][ks] = *reinterpret_cast<const Piece*>(q + (static_cast<size_t>(tok[ct]) * nq + head[ct]) * D + (ks * 4 + grp) * kPiece);
    }
  }
  // keys that every column of the item sees are [open_lo, open_hi): blocks inside need no mask
  const int open_lo = item.key_lo, open_hi = item.own ? min(item.key_hi, pos0 + item.col0 / G + 1) : item.key_hi;

  const size_t page_stride = static_cast<size_t>(2 * nkv) << page_shift;    // in rows of D
  const Elem* k_base = cache + (static_cast<size_t>(kvh) << page_shift) * D;
  const Elem* v_base = cache + (static_cast<size_t>(nkv + kvh) << page_shift) * D;
  const int k_lane = col * D + grp * kPiece, v_lane = (col << page_shift) + grp * 4;

  struct Block {
    Piece k[TILES][KS];
    Values v[DT][TILES];
  };
  // Rows outside the item's keys are read with the others (their page is in the table, or page 0 stands there) and masked.
  auto load = [&](int kb, Block& block) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int first = kb + t * 16;
      const int page = __builtin_amdgcn_readfirstlane(pages[min(first >> page_shift, max_blocks - 1)]);
      const Elem* keys = k_base + (static_cast<size_t>(page) * page_stride + (first & page_mask)) * D;
      const Elem* values = v_base + static_cast<size_t>(page) * page_stride * D + (first & page_mask);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        block.k[t][ks] = has_dims(ks) ? *reinterpret_cast<const Piece*>(keys + k_lane + ks * 4 * kPiece) : Piece{0, 0, 0, 0};
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) block.v[dt][t] = *reinterpret_cast<const Values*>(values + v_lane + ((dt * 16) << page_shift));
    }
  };

  // maxima and sums in base 2: a score s enters as 2^(s * scale_log2 - maximum)
  float top[CT], sum[CT];
  floatx4 o[CT][DT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    top[ct] = -INFINITY, sum[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[ct][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  auto work = [&](int kb, Block& block, auto masked_tag) {
    constexpr bool kMasked = decltype(masked_tag)::value;
    if (kMasked) {
      // rows that are not the item's may hold anything: 0 * NaN must not arise
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kb + t * 16 + grp * 4 + j;
            const bool out = key < item.key_lo || key >= item.key_hi;
            if constexpr (FLOAT) block.v[dt][t][j] = out ? 0u : block.v[dt][t][j];
            else block.v[dt][t][j >> 1] &= out ? ((j & 1) ? 0x0000ffffu : 0xffff0000u) : 0xffffffffu;
          }
    }
    floatx4 s[CT][TILES];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        s[ct][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if constexpr (FLOAT) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(block.k[t][ks][e]), __uint_as_float(query[ct][ks][e]), s[ct][t], 0, 0, 0);
          } else {
            s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(&block.k[t][ks]),
                                                               *reinterpret_cast<const bf16x8*>(&query[ct][ks]), s[ct][t], 0, 0, 0);
          }
        }
      }
    if (cap_pre > 0.f) {
      // cap * tanh(s * scale / cap) = cap * (1 - 2 / (2^(2 log2(e) s scale / cap) + 1)); the cap is part of scale_log2
      settle(s);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float grown = __builtin_amdgcn_exp2f(s[ct][t][j] * (cap_pre * 2.8853900817779268f)) + 1.f;
            s[ct][t][j] = 1.f - (FLOAT ? 2.f / grown : 2.f * __builtin_amdgcn_rcpf(grown));
          }
    }
    float lane_top[CT];
    bool exceeds = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      lane_top[ct] = -INFINITY;
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (kMasked) {
            const int key = kb + t * 16 + grp * 4 + j;
            s[ct][t][j] = key >= item.key_lo && key < item.key_hi && key <= last_key[ct] ? s[ct][t][j] : -INFINITY;
          }
          lane_top[ct] = fmaxf(lane_top[ct], s[ct][t][j]);
        }
      lane_top[ct] *= scale_log2;                           // (the scale is positive)
      exceeds = exceeds || lane_top[ct] > top[ct];
    }
    // A column's maximum is shared by its four lane groups and moves only when a block holds a larger score, which is rare
    // after the first blocks: rescaling sits behind a branch of the wave.
    if (__builtin_amdgcn_ballot_w64(exceeds) != 0) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float most = lane_top[ct];
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        most = fmaxf(most, top[ct]);
        const float down = most == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top[ct] - most);
        top[ct] = most;
        sum[ct] *= down;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[ct][dt][j] *= down;
      }
    }
    float p[CT][TILES * 4];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float below = kMasked && top[ct] == -INFINITY ? 0.f : top[ct];         // (nothing seen yet: 2^(-inf - 0) = 0)
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[ct][t * 4 + j] = __builtin_amdgcn_exp2f(fmaf(s[ct][t][j], scale_log2, -below));
          sum[ct] += p[ct][t * 4 + j];
        }
    }
    if constexpr (FLOAT) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
            o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(block.v[dt][0][e]), p[ct][e], o[ct][dt], 0, 0, 0);
    } else {
      Piece packed[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) packed[ct][i] = pack_bf16(p[ct][2 * i], p[ct][2 * i + 1]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const Piece a = Piece{block.v[dt][0][0], block.v[dt][0][1], block.v[dt][TILES - 1][0], block.v[dt][TILES - 1][1]};
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
          o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(&a), *reinterpret_cast<const bf16x8*>(&packed[ct]),
                                                              o[ct][dt], 0, 0, 0);
      }
    }
  };

  // two blocks in registers: while one is worked on the other is on its way
  constexpr int kStride = BLOCK * kPrefixWaves;
  Block ring[2];
  const int begin = (item.key_lo & ~(BLOCK - 1)) + BLOCK * wave;
  if (begin < item.key_hi) {
    load(begin, ring[0]);
    if (begin + kStride < item.key_hi) load(begin + kStride, ring[1]);
    for (int kb = begin; kb < item.key_hi; kb += 2 * kStride) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int mine = kb + r * kStride;
        if (mine >= item.key_hi) break;
        if (mine >= open_lo && mine + BLOCK <= open_hi) work(mine, ring[r], std::false_type{});
        else work(mine, ring[r], std::true_type{});
        if (mine + 2 * kStride < item.key_hi) load(mine + 2 * kStride, ring[r]);
      }
    }
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    sum[ct] += __shfl_xor(sum[ct], 16, 64);
    sum[ct] += __shfl_xor(sum[ct], 32, 64);
  }
  settle(o);

  // The waves' results into one: every wave brings its own onto the common maximum; then, one column group after the other, the
  // values meet in LDS and each wave adds up a quarter of the dims, in the order of the waves.
  float* stats = lds;                                          // [waves][CT][16][2]
  float* slots = lds + kPrefixWaves * CT * 32;                 // [waves][DT][64][4]
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
    if (grp == 0) {
      stats[((wave * CT + ct) * 16 + col) * 2] = top[ct];
      stats[((wave * CT + ct) * 16 + col) * 2 + 1] = sum[ct];
    }
  __syncthreads();
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float most = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kPrefixWaves; ++w) most = fmaxf(most, stats[((w * CT + ct) * 16 + col) * 2]);
    const float below = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int w = 0; w < kPrefixWaves; ++w)
      total += __builtin_amdgcn_exp2f(stats[((w * CT + ct) * 16 + col) * 2] - below) * stats[((w * CT + ct) * 16 + col) * 2 + 1];
    const float down = __builtin_amdgcn_exp2f(top[ct] - below);
    if (ct > 0) __syncthreads();                               // (the slots have been read)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<float4*>(slots + ((wave * DT + dt) * 64 + lane) * 4) =
          make_float4(o[ct][dt][0] * down, o[ct][dt][1] * down, o[ct][dt][2] * down, o[ct][dt][3] * down);
    __syncthreads();
    // (a token that stands before the others of its tile may have fewer parts than they)
    const int first_part = part_first[tok[ct]];
    if (!valid[ct] || item.part >= part_first[tok[ct] + 1] - first_part) continue;
    const size_t slot = static_cast<size_t>(first_part + item.part) * nq + head[ct];
    for (int dt = wave; dt < DT; dt += kPrefixWaves) {
      float4 all = *reinterpret_cast<const float4*>(slots + (dt * 64 + lane) * 4);
#pragma unroll
      for (int w = 1; w < kPrefixWaves; ++w) {
        const float4 more = *reinterpret_cast<const float4*>(slots + ((w * DT + dt) * 64 + lane) * 4);
        all.x += more.x, all.y += more.y, all.z += more.z, all.w += more.w;
      }
      *reinterpret_cast<float4*>(part_o + slot * D + dt * 16 + grp * 4) = all;
    }
    if (wave == 0 && grp == 0) part_ml[slot * 2] = most, part_ml[slot * 2 + 1] = total;
  }
}

template <int DT, bool FLOAT, int CT>
__global__ void __launch_bounds__(64 * kPrefixWaves)
prefix_items_kernel(const void* __restrict__ q, const void* __restrict__ cache, const int* __restrict__ block_table, int max_blocks,
                    const int* __restrict__ items, const int* __restrict__ positions, const int* __restrict__ part_first, float* __restrict__ part_o,
                    float* __restrict__ part_ml, int nq, int nkv, int page_shift, float scale_log2, float cap_pre) {
  __shared__ __attribute__((aligned(16))) float lds[kPrefixWaves * (CT * 32 + DT * 256)];
  const int kvh = blockIdx.x % nkv;
  PrefixItem item;
  {
    const int* words = items + static_cast<size_t>(blockIdx.x / nkv) * 8;
    item.table = __builtin_amdgcn_readfirstlane(words[0]), item.tok0 = __builtin_amdgcn_readfirstlane(words[1]);
    item.ntok = __builtin_amdgcn_readfirstlane(words[2]), item.col0 = __builtin_amdgcn_readfirstlane(words[3]);
    item.key_lo = __builtin_amdgcn_readfirstlane(words[4]), item.key_hi = __builtin_amdgcn_readfirstlane(words[5]);
    item.own = __builtin_amdgcn_readfirstlane(words[6]), item.part = __builtin_amdgcn_readfirstlane(words[7]);
  }
  if (item.ntok <= 0) return;                                  // a list of fixed size ends in items without tokens
  const int* pages = block_table + static_cast<size_t>(item.table) * max_blocks;
  // an item of few columns is served by the form for 16 whatever the launch's width
  if (CT > 1 && item.ntok * (nq / nkv) - item.col0 > 16)
    prefix_item<DT, FLOAT, CT>(item, kvh, q, cache, pages, max_blocks, positions, part_first, part_o, part_ml, nq, nkv, page_shift, scale_log2, cap_pre, lds);
  else
    prefix_item<DT, FLOAT, 1>(item, kvh, q, cache, pages, max_blocks, positions, part_first, part_o, part_ml, nq, nkv, page_shift, scale_log2, cap_pre, lds);
}

// out[t][h] = sum_i w_i o_i / (sum_i w_i l_i + w_sink) over the token's parts, in their order.  A wave a (token, head).
template <bool FLOAT>
__global__ void __launch_bounds__(256)
prefix_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ part_first,
                   const float* __restrict__ sink, void* __restrict__ out, int rows, int nq, int d) {
  const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * 4 + (threadIdx.x >> 6)));
  if (row >= rows) return;
  const int lane = threadIdx.x & 63, token = row / nq, head = row - token * nq;
  const int first = part_first[token], count = part_first[token + 1] - first;
  const float own = sink != nullptr ? sink[head] * 1.4426950408889634f : -INFINITY;
  float most = own;
  for (int p = 0; p < count; ++p) most = fmaxf(most, part_ml[(static_cast<size_t>(first + p) * nq + head) * 2]);
  const float below = most == -INFINITY ? 0.f : most;
  float total = sink != nullptr ? __builtin_amdgcn_exp2f(own - below) : 0.f;
  for (int p = 0; p < count; ++p) {
    const size_t slot = static_cast<size_t>(first + p) * nq + head;
    total += __builtin_amdgcn_exp2f(part_ml[slot * 2] - below) * part_ml[slot * 2 + 1];
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;           // a token that no sequence brings has no parts, and gets zeros
  for (int i = lane; i < d; i += 64) {
    float value = 0.f;
    for (int p = 0; p < count; ++p) {
      const size_t slot = static_cast<size_t>(first + p) * nq + head;
      value += __builtin_amdgcn_exp2f(part_ml[slot * 2] - below) * part_o[slot * d + i];
    }
    if (FLOAT) static_cast<float*>(out)[static_cast<size_t>(row) * d + i] = value * inv;
    else static_cast<uint16_t*>(out)[static_cast<size_t>(row) * d + i] = __bfloat16_as_ushort(__float2bfloat16(value * inv));
  }
}

template <bool FLOAT, int DT>
static int launch_items(int wide, const void* q, const void* cache, const int* block_table, int max_blocks, const int* items, int num_items,
                        const int* positions, const int* part_first, float* part_o, float* part_ml, int nq, int nkv, int page_shift,
                        float scale_log2, float cap_pre, hipStream_t stream) {
  constexpr int kWide = DT <= 8 ? 2 : 1;
  if (wide != 1 && wide != kWide) return kBadArgument;
  if (wide == 1)
    hipLaunchKernelGGL((prefix_items_kernel<DT, FLOAT, 1>), dim3(num_items * nkv), dim3(64 * kPrefixWaves), 0, stream, q, cache, block_table,
                       max_blocks, items, positions, part_first, part_o, part_ml, nq, nkv, page_shift, scale_log2, cap_pre);
  else
    hipLaunchKernelGGL((prefix_items_kernel<DT, FLOAT, kWide>), dim3(num_items * nkv), dim3(64 * kPrefixWaves), 0, stream, q, cache, block_table,
                       max_blocks, items, positions, part_first, part_o, part_ml, nq, nkv, page_shift, scale_log2, cap_pre);
  return launch_status();
}

}  // namespace tlie

using namespace tlie;

// q, out: [tokens, nq, d]; cache: [pages, 2, nkv, page_size * d] (keys [row][dim], values [dim][row]); both of `dtype`.
// items: int32 [num_items, 8] (see PrefixItem), in columns of 16 * wide; part_first: int32 [tokens + 1], the first part of
// each token, so that part_first[tokens] is their number; part_o: float [parts, nq, d], part_ml: float [parts, nq, 2].
// sink: float [nq] or null.  softcap: 0, or the cap of the scaled scores.
extern "C" int tlie_attention_prefix(const void* q, const void* cache, int dtype, const int* block_table, int max_blocks, const int* items,
                                     int num_items, int wide, const int* positions, const int* part_first, float* part_o, float* part_ml,
                                     const float* sink, void* out, int tokens, int nq, int nkv, int d, int page_size, float scale,
                                     float softcap, void* stream) {
  if (tokens <= 0 || num_items <= 0 || nq <= 0 || nkv <= 0 || nq % nkv != 0 || d <= 0 || d > 256 || d % 16 != 0 || page_size < 16 ||
      (page_size & (page_size - 1)) != 0 || max_blocks <= 0 || !(scale > 0.f) || !(softcap >= 0.f) || (dtype != kF32 && dtype != kBF16) ||
      static_cast<long long>(num_items) * nkv > 0x7fffffffll || static_cast<long long>(tokens) * nq > 0x7ffffffcll)
    return kBadArgument;
  const float scale_log2 = (softcap > 0.f ? softcap : scale) * 1.4426950408889634f, cap_pre = softcap > 0.f ? scale / softcap : 0.f;
  const int page_shift = 31 - __builtin_clz(page_size);
  hipStream_t s = (hipStream_t)stream;
  int status = kBadArgument;
#define TLIE_CASE(DT)                                                                                                                              \
  case DT:                                                                                                                                         \
    status = dtype == kF32 ? launch_items<true, DT>(wide, q, cache, block_table, max_blocks, items, num_items, positions, part_first, part_o,      \
                                                    part_ml, nq, nkv, page_shift, scale_log2, cap_pre, s)                                          \
                           : launch_items<false, DT>(wide, q, cache, block_table, max_blocks, items, num_items, positions, part_first, part_o,     \
                                                     part_ml, nq, nkv, page_shift, scale_log2, cap_pre, s);                                        \
    break;
  switch (d / 16) {
    TLIE_CASE(1) TLIE_CASE(2) TLIE_CASE(3) TLIE_CASE(4) TLIE_CASE(5) TLIE_CASE(6) TLIE_CASE(7) TLIE_CASE(8)
    TLIE_CASE(9) TLIE_CASE(10) TLIE_CASE(11) TLIE_CASE(12) TLIE_CASE(13) TLIE_CASE(14) TLIE_CASE(15) TLIE_CASE(16)
  }
#undef TLIE_CASE
  if (status != kOk) return status;
  const int rows = tokens * nq;
  if (dtype == kF32)
    hipLaunchKernelGGL((prefix_join_kernel<true>), dim3((rows + 3) / 4), dim3(256), 0, s, part_o, part_ml, part_first, sink, out, rows, nq, d);
  else
    hipLaunchKernelGGL((prefix_join_kernel<false>), dim3((rows + 3) / 4), dim3(256), 0, s, part_o, part_ml, part_first, sink, out, rows, nq, d);
  return launch_status();
}
