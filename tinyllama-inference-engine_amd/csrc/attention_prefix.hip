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

#include <algorithm>
#include <cmath>
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

constexpr int kPrefixWaves = 4, kDirectWaves = 8;
// Powers may grow to 2^6 before what they are relative to moves: sums and values are float, and the rounding of a probability to
// bfloat16 is relative.  Without slack a wave of 32 columns rescales in almost every block of an item (eight
// questions behind 4000 positions 59 us against 56, three documents with capped scores 15.0 against 14.0).
constexpr float kSlack = 6.f;

// The page that position `key` lies on, of an item with keys on the pages page_lo .. page_hi; key is the same for every lane, so that the
// number comes through the scalar cache, whose lines hold sixteen.  Rows of a page outside the item's keys are read with the others and
// masked; pages that hold none of them are not: the first or last page of the keys is read again in their place, whatever the table says there.
__device__ __forceinline__ int page_of(const int* __restrict__ pages, int key, int page_shift, int page_lo, int page_hi) {
  return pages[__builtin_amdgcn_readfirstlane(min(max(key >> page_shift, page_lo), page_hi))];
}

// tanh(t) of each score, t in units of the cap.  1 - 2 / (e^2t + 1) is off by up to 2^-22, however small t: a capped score by that share of the cap (a
// cap of 10^6 left scores of 5 wrong by 0.06).  In bfloat16, up to a cap of 1024, it is an eighth of a probability's rounding of 2^-9.  Beyond, and in 32
// bits, small t by their series to the seventh power (62 / 2835 t^8 < 2^-29 of it left), from an eighth on the first form (2^-19 of t).  With both for
// all caps in bfloat16, 8 capped questions behind 4000 positions take 69.8 us in place of 60.5, three documents 15.1 in place of 14.4.
template <bool FLOAT, int CT, int TILES>
__device__ __forceinline__ void cap_scores(floatx4 (&s)[CT][TILES], float cap_pre, float scale_log2) {
  auto direct = [](float x) {
    const float grown = __builtin_amdgcn_exp2f(x * 2.8853900817779268f) + 1.f;
    return 1.f - (FLOAT ? 2.f / grown : 2.f * __builtin_amdgcn_rcpf(grown));
  };
  auto each = [&](auto f) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[ct][t][j] = f(s[ct][t][j] * cap_pre);
  };
  if (!FLOAT && scale_log2 <= 1024.f * 1.4426950408889634f) {                // (the same for the whole launch)
    each(direct);
    return;
  }
  each([&](float x) {
    const float square = x * x, series = fmaf(x * square, fmaf(square, fmaf(square, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), x);
    return fabsf(x) < 0.125f ? series : direct(x);
  });
}

// Where an item that leaves its columns' results themselves has them go, and the keys 0 .. shared - 1 that it reads through another row.
struct Direct {
  const int* pages;
  int shared;
  const float* sink;
  void* out;
};

template <int DT, bool FLOAT, int CT, int WAVES, bool DIRECT>
__device__ __forceinline__ void prefix_item(const PrefixItem& item, const Direct& direct, int kvh, const void* __restrict__ q_any, const void* __restrict__ cache_any,
                                            const int* __restrict__ pages, const int* __restrict__ positions,
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
  // keys that every column of the item sees end at open_hi: blocks inside need no mask
  const int open_hi = item.own ? min(item.key_hi, pos0 + item.col0 / G + 1) : item.key_hi;

  const size_t page_stride = static_cast<size_t>(2 * nkv) << page_shift;    // in rows of D
  const Elem* k_base = cache + (static_cast<size_t>(kvh) << page_shift) * D;
  const Elem* v_base = cache + (static_cast<size_t>(nkv + kvh) << page_shift) * D;
  const int k_lane = col * D + grp * kPiece, v_lane = (col << page_shift) + grp * 4;

  struct Block {
    Piece k[TILES][KS];
    Values v[DT][TILES];
  };
  // the item's blocks: those of the keys that it reads through another row first
  const int shared_keys = DIRECT ? direct.shared : 0, shared_blocks = (shared_keys + BLOCK - 1) / BLOCK, begin = item.key_lo & ~31;
  auto is_shared = [&](int index) { return DIRECT && index < shared_blocks; };
  auto key_of = [&](int index) { return is_shared(index) ? index * BLOCK : begin + (index - shared_blocks) * BLOCK; };
  auto load = [&](int index, Block& block) {
    const int kb = key_of(index);
    const int* from = is_shared(index) ? direct.pages : pages;
    const int page_lo = (is_shared(index) ? 0 : item.key_lo) >> page_shift, page_hi = ((is_shared(index) ? shared_keys : item.key_hi) - 1) >> page_shift;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int first = kb + t * 16;
      const int page = page_of(from, first, page_shift, page_lo, page_hi);
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

  auto work = [&](int index, Block& block) {
    const int kb = key_of(index), key_lo = is_shared(index) ? 0 : item.key_lo, key_hi = is_shared(index) ? shared_keys : item.key_hi;
    const bool ragged = kb < key_lo || kb + BLOCK > (is_shared(index) ? shared_keys : open_hi);     // (the same for the whole wave)
    if (ragged) {
      // rows that are not the item's may hold anything: 0 * NaN must not arise
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kb + t * 16 + grp * 4 + j;
            const bool out = key < key_lo || key >= key_hi;
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
    settle(s);                                            // (branches follow, behind which the scores are read)
    if (cap_pre > 0.f) cap_scores<FLOAT>(s, cap_pre, scale_log2);          // (the cap is part of scale_log2)
    if (ragged) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kb + t * 16 + grp * 4 + j;
            s[ct][t][j] = key >= key_lo && key < key_hi && key <= last_key[ct] ? s[ct][t][j] : -INFINITY;
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
        for (int j = 0; j < 4; ++j) lane_top[ct] = fmaxf(lane_top[ct], s[ct][t][j]);
      lane_top[ct] *= scale_log2;                           // (the scale is positive)
      exceeds = exceeds || lane_top[ct] > top[ct] + kSlack;
    }
    // What the scores are taken relative to (shared by a column's four lane groups) is a maximum of earlier blocks, and moves only when
    // a block exceeds it by more than the slack: rare after the first block, so rescaling sits behind a branch of the wave.
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
      const float below = top[ct] == -INFINITY ? 0.f : top[ct];         // (nothing seen yet: 2^(-inf - 0) = 0)
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
  Block ring[2];
  const int blocks = shared_blocks + (item.key_hi - begin + BLOCK - 1) / BLOCK;
  load(min(wave, blocks - 1), ring[0]);
  load(min(wave + WAVES, blocks - 1), ring[1]);
  for (int index = wave; index < blocks; index += 2 * WAVES) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int mine = index + r * WAVES;
      if (mine < blocks) work(mine, ring[r]);
      load(min(mine + 2 * WAVES, blocks - 1), ring[r]);            // (past the last block the last again: as many loads on every path)
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
  float* slots = lds + WAVES * CT * 32;                 // [waves][DT][64][4]
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
    for (int w = 0; w < WAVES; ++w) most = fmaxf(most, stats[((w * CT + ct) * 16 + col) * 2]);
    const float below = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      total += __builtin_amdgcn_exp2f(stats[((w * CT + ct) * 16 + col) * 2] - below) * stats[((w * CT + ct) * 16 + col) * 2 + 1];
    const float down = __builtin_amdgcn_exp2f(top[ct] - below);
    if (ct > 0) __syncthreads();                               // (the slots have been read)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<float4*>(slots + ((wave * DT + dt) * 64 + lane) * 4) =
          make_float4(o[ct][dt][0] * down, o[ct][dt][1] * down, o[ct][dt][2] * down, o[ct][dt][3] * down);
    __syncthreads();
    size_t slot = static_cast<size_t>(tok[ct]) * nq + head[ct];
    float scale_out = 1.f;
    if constexpr (DIRECT) {
      if (!valid[ct]) continue;
      const float own = direct.sink != nullptr ? direct.sink[head[ct]] * 1.4426950408889634f : -INFINITY;
      const float end = fmaxf(most, own), under = end == -INFINITY ? 0.f : end, weight = __builtin_amdgcn_exp2f(most - under);
      const float whole = total * weight + (direct.sink != nullptr ? __builtin_amdgcn_exp2f(own - under) : 0.f);
      scale_out = whole > 0.f ? weight / whole : 0.f;
    } else {
      // (a token that stands before the others of its tile may have fewer parts than they)
      const int first_part = part_first[tok[ct]];
      if (!valid[ct] || item.part >= part_first[tok[ct] + 1] - first_part) continue;
      slot = static_cast<size_t>(first_part + item.part) * nq + head[ct];
    }
    for (int dt = wave; dt < DT; dt += WAVES) {
      float4 all = *reinterpret_cast<const float4*>(slots + (dt * 64 + lane) * 4);
#pragma unroll
      for (int w = 1; w < WAVES; ++w) {
        const float4 more = *reinterpret_cast<const float4*>(slots + ((w * DT + dt) * 64 + lane) * 4);
        all.x += more.x, all.y += more.y, all.z += more.z, all.w += more.w;
      }
      if constexpr (DIRECT) {
        all.x *= scale_out, all.y *= scale_out, all.z *= scale_out, all.w *= scale_out;
        const size_t place = slot * D + dt * 16 + grp * 4;
        if constexpr (FLOAT) *reinterpret_cast<float4*>(static_cast<float*>(direct.out) + place) = all;
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(direct.out) + place) = make_uint2(pack_bf16(all.x, all.y), pack_bf16(all.z, all.w));
      } else {
        *reinterpret_cast<float4*>(part_o + slot * D + dt * 16 + grp * 4) = all;
      }
    }
    if (!DIRECT && wave == 0 && grp == 0) part_ml[slot * 2] = most, part_ml[slot * 2 + 1] = total;
  }
}

// An item of many columns, bfloat16: each wave has 16 * CT columns of its own, and every block of 32 keys and values is brought once
// for all four, through LDS, two at a time.  They are asked for two ahead of their turn and wait in registers; two buffers in turn, so
// that one barrier a turn is enough (a wave writes a buffer again only behind the barrier that every wave reaches after it has read it).
// Keys lie as [key][piece of 16 bytes], a key's pieces rotated by key / kPeriod so that the 16 keys that a read takes the same piece of
// are spread over the banks; values as [half of 16 keys][16 dims][4 keys][dim], of which a read takes 512 bytes in the order of the lanes.
//
// What bounds it.  128 columns of 128 dims: no one thing; of 43 us (8 questions of some 46 tokens behind 4000 positions, 24.5 GFLOP, 20 us at the
// rate of a large product) bringing the keys takes 18 by itself, and without the scores' products, the values', or the exponentials 5, 7
// and 2 us are saved.  32 sequences behind 30000 positions, keys from memory: bringing them 37 of 40 us (3.4 TB/s: two workgroups a
// compute unit have 64 KB on their way, and wait for a turn's last piece before they ask for the next).  The parts' results cost 5 us to
// write and 7 to join in both.  Eight waves a workgroup that leave one result between them halve
// that but take longer: one workgroup a unit, all its waves at the same barriers (56 against 51 us, 49 against 46, 64 sequences behind 6000 43 against 35).
template <int DT, int CT>
__device__ __forceinline__ void prefix_wide_item(const PrefixItem& item, int kvh, const uint16_t* __restrict__ q, const uint16_t* __restrict__ cache,
                                                 const int* __restrict__ pages, const int* __restrict__ positions,
                                                 const int* __restrict__ part_first, float* __restrict__ part_o, float* __restrict__ part_ml,
                                                 int nq, int nkv, int page_shift, float scale_log2, float cap_pre, unsigned char* lds) {
  constexpr int D = DT * 16, KS = (DT + 1) / 2, kPieces = 2 * DT;           // pieces of a key
  constexpr int kPeriod = 16 / (kPieces % 16 == 0 ? 16 : kPieces % 8 == 0 ? 8 : kPieces % 4 == 0 ? 4 : 2);
  constexpr int kBytes = 64 * D;                                            // of a block's keys, and of its values
  constexpr int kCalls = (2 * DT + 3) / 4;                                  // pieces a thread brings of a block: 2 * DT times 64 in all
  typedef uint32_t Piece __attribute__((ext_vector_type(4)));
  typedef uint32_t Half __attribute__((ext_vector_type(2)));
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int G = nq / nkv, ncols = item.ntok * G, page_mask = (1 << page_shift) - 1;
  const int pos0 = item.own ? __builtin_amdgcn_readfirstlane(positions[item.tok0]) : 0;
  const int col0 = item.col0 + wave * 16 * CT;
  const bool active = col0 < ncols;
  auto has_dims = [&](int ks) { return DT % 2 == 0 || ks < KS - 1 || grp < 2; };

  int last_key[CT];
  Piece query[CT][KS];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = col0 + ct * 16 + col;
    const bool valid = c < ncols;
    const int tok = item.tok0 + (valid ? c / G : 0), head = kvh * G + (valid ? c % G : 0);
    last_key[ct] = !valid ? -1 : item.own ? pos0 + c / G : 0x7fffffff;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      query[ct][ks] = Piece{0, 0, 0, 0};
      if (valid && has_dims(ks)) query[ct][ks] = *reinterpret_cast<const Piece*>(q + (static_cast<size_t>(tok) * nq + head) * D + (ks * 4 + grp) * 8);
    }
  }
  // the wave's keys end with those of its last column; keys that all its columns see need no mask
  const int last_col = min(col0 + 16 * CT, ncols) - 1;
  const int high = !active ? 0 : item.own ? min(item.key_hi, pos0 + last_col / G + 1) : item.key_hi;
  const int open_hi = item.own ? min(item.key_hi, pos0 + col0 / G + 1) : item.key_hi;

  const size_t page_stride = static_cast<size_t>(2 * nkv) << page_shift;    // in rows of D
  const uint16_t* k_base = cache + (static_cast<size_t>(kvh) << page_shift) * D;
  const uint16_t* v_base = cache + (static_cast<size_t>(nkv + kvh) << page_shift) * D;
  // A piece's place behind its half's page and row, and in the buffer, in bytes.  At 128 dims (two calls a half) a thread brings the
  // same place of both halves, so that one of each is kept for the keys and one for the values: every register counts there.
  constexpr bool kAlike = DT == 8;
  constexpr int kPlaces = kAlike ? 2 : kCalls;
  int from[kPlaces], to[kPlaces];
  bool second[kPlaces];
#pragma unroll
  for (int i = 0; i < kPlaces; ++i) {
    const int call = min(kAlike ? wave + 8 * i : wave + 4 * i, 2 * DT - 1), piece = (call % DT) * 64 + lane;      // (past the last: the last again, the same bytes)
    if (call < DT) {
      const int key = piece / kPieces, place = piece % kPieces;
      second[i] = key >= 16;
      from[i] = (key & 15) * D + place * 8;
      to[i] = (key * kPieces + (place + key / kPeriod) % kPieces) * 16;
    } else {
      const int rest = piece % (2 * D);
      second[i] = piece >= 2 * D;
      from[i] = ((rest >> 1) << page_shift) + (rest & 1) * 8;
      to[i] = kBytes + (second[i] ? D * 32 : 0) + ((rest >> 5) * 64 + (rest & 1) * 32 + ((rest >> 1) & 15)) * 8;
    }
  }
  auto is_values = [&](int i) { return kAlike ? i >= 2 : min(wave + 4 * i, 2 * DT - 1) >= DT; };       // (the same for the whole wave)
  auto to_of = [&](int i) { return kAlike ? to[i >> 1] + (i & 1) * (kBytes / 2) : to[i]; };
  Piece staged[2][kCalls];
  const int page_lo = item.key_lo >> page_shift, page_hi = (item.key_hi - 1) >> page_shift;
  auto bring = [&](int kb, Piece (&into)[kCalls]) {
    const size_t at_a = static_cast<size_t>(page_of(pages, kb, page_shift, page_lo, page_hi)) * page_stride * D;
    const size_t at_b = static_cast<size_t>(page_of(pages, kb + 16, page_shift, page_lo, page_hi)) * page_stride * D;
    const int row_a = kb & page_mask, row_b = (kb + 16) & page_mask;
    const uint16_t *keys_a = k_base + at_a + row_a * D, *keys_b = k_base + at_b + row_b * D;
    const uint16_t *values_a = v_base + at_a + row_a, *values_b = v_base + at_b + row_b;
#pragma unroll
    for (int i = 0; i < kCalls; ++i) {
      const uint16_t* base;
      if constexpr (kAlike) {
        base = i == 0 ? keys_a : i == 1 ? keys_b : i == 2 ? values_a : values_b;
      } else {
        const bool of_values = is_values(i);
        base = second[i] ? (of_values ? values_b : keys_b) : (of_values ? values_a : keys_a);
      }
      into[i] = *reinterpret_cast<const Piece*>(base + from[kAlike ? i >> 1 : i]);
    }
  };

  float top[CT], sum[CT];
  floatx4 o[CT][DT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    top[ct] = -INFINITY, sum[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[ct][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const int key_place = col * kPieces * 16;                                  // the lane's key in its half, and how far its pieces are rotated
  const int turned_a = col / kPeriod, turned_b = (col + 16) / kPeriod;

  // (one copy of the code, its masks behind branches of the wave: with a copy with and one without masks the compiler keeps 42 registers
  // in memory, and waits for the blocks on their way each time it fetches one: 67 us against 37 for the kernel)
  auto work = [&](int kb, const unsigned char* buffer) {
    const bool ragged = kb < item.key_lo || kb + 32 > open_hi;
    floatx4 s[CT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[ct][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int place = (min(ks * 4 + grp, kPieces - 1) + (t ? turned_b : turned_a)) % kPieces;
        Piece k = *reinterpret_cast<const Piece*>(buffer + key_place + t * 16 * kPieces * 16 + place * 16);
        if (!has_dims(ks)) k = Piece{0, 0, 0, 0};
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
          s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(&k), *reinterpret_cast<const bf16x8*>(&query[ct][ks]),
                                                             s[ct][t], 0, 0, 0);
      }
    }
    // (the values are asked for here, so that they are there when the probabilities are)
    Piece values[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const unsigned char* place = buffer + kBytes + (dt * 64 + lane) * 8;
      const Half a = *reinterpret_cast<const Half*>(place), b = *reinterpret_cast<const Half*>(place + D * 32);
      values[dt] = Piece{a[0], a[1], b[0], b[1]};
    }
    settle(s);                                               // (branches follow, behind which the scores are read)
    if (ragged) {
      uint32_t keep[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int key = kb + (w >> 1) * 16 + grp * 4 + (w & 1) * 2;
        keep[w] = (key >= item.key_lo && key < item.key_hi ? 0x0000ffffu : 0u) | (key + 1 >= item.key_lo && key + 1 < item.key_hi ? 0xffff0000u : 0u);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int w = 0; w < 4; ++w) values[dt][w] &= keep[w];
    }
    if (cap_pre > 0.f) cap_scores<false>(s, cap_pre, scale_log2);
    if (ragged) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kb + t * 16 + grp * 4 + j;
            s[ct][t][j] = key >= item.key_lo && key < item.key_hi && key <= last_key[ct] ? s[ct][t][j] : -INFINITY;
          }
    }
    float lane_top[CT];
    bool exceeds = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      lane_top[ct] = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) lane_top[ct] = fmaxf(lane_top[ct], s[ct][t][j]);
      lane_top[ct] *= scale_log2;
      exceeds = exceeds || lane_top[ct] > top[ct] + kSlack;
    }
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
    Piece packed[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float below = top[ct] == -INFINITY ? 0.f : top[ct];
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[ct][i >> 2][i & 3], scale_log2, -below));
      sum[ct] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
      for (int i = 0; i < 4; ++i) packed[ct][i] = pack_bf16(p[2 * i], p[2 * i + 1]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(&values[dt]), *reinterpret_cast<const bf16x8*>(&packed[ct]),
                                                            o[ct][dt], 0, 0, 0);
  };
  auto put = [&](unsigned char* place, const Piece (&waiting)[kCalls]) {
#pragma unroll
    for (int i = 0; i < kCalls; ++i) {
      unsigned char* there = place + to_of(i);
      if (is_values(i)) {
        *reinterpret_cast<Half*>(there) = Half{waiting[i][0], waiting[i][1]}, *reinterpret_cast<Half*>(there + 128) = Half{waiting[i][2], waiting[i][3]};
      } else {
        *reinterpret_cast<Piece*>(there) = waiting[i];
      }
    }
  };
  int buffer = 0;
  const int begin = item.key_lo & ~31, last = (item.key_hi - 1) & ~31;
  bring(begin, staged[0]);
  bring(min(begin + 32, last), staged[1]);
  for (int kb = begin; kb <= last; kb += 64) {
    unsigned char* place = lds + buffer * 4 * kBytes;
    put(place, staged[0]);
    put(place + 2 * kBytes, staged[1]);
    lds_barrier();
    bring(min(kb + 64, last), staged[0]);                      // (past the last block the last again: as many loads on every path)
    bring(min(kb + 96, last), staged[1]);
#pragma unroll 1
    for (int u = 0; u < 2; ++u)
      if (kb + 32 * u <= last && kb + 32 * u < high) work(kb + 32 * u, place + u * 2 * kBytes);
    buffer ^= 1;
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    sum[ct] += __shfl_xor(sum[ct], 16, 64);
    sum[ct] += __shfl_xor(sum[ct], 32, 64);
  }
  settle(o);
  int lane_again = threadIdx.x & 63;                             // (formed again: kept over the walk, the columns' places cost registers)
  asm volatile("" : "+v"(lane_again));
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = col0 + ct * 16 + (lane_again & 15), group = lane_again >> 4;
    if (c >= ncols) continue;
    const int tok = item.tok0 + c / G, head = kvh * G + c % G, first_part = part_first[tok];
    if (item.part >= part_first[tok + 1] - first_part) continue;
    const size_t slot = static_cast<size_t>(first_part + item.part) * nq + head;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<float4*>(part_o + slot * D + dt * 16 + group * 4) = make_float4(o[ct][dt][0], o[ct][dt][1], o[ct][dt][2], o[ct][dt][3]);
    if (group == 0) part_ml[slot * 2] = top[ct], part_ml[slot * 2 + 1] = sum[ct];
  }
}

// Columns that a tile has: 16 where there are no more (four waves share its keys); else 64, or 128 in bfloat16 for head sizes up to
// 128 where there are more than 64 (each wave has columns of its own).  Float items have up to 32, always by the first form.
template <int DT, bool FLOAT>
__global__ void __launch_bounds__(64 * kPrefixWaves, DT <= 8 && !FLOAT ? 2 : 1)
prefix_items_kernel(const void* __restrict__ q, const void* __restrict__ cache, const int* __restrict__ block_table, int max_blocks,
                    const int* __restrict__ items, const int* __restrict__ positions, const int* __restrict__ part_first, float* __restrict__ part_o,
                    float* __restrict__ part_ml, int nq, int nkv, int page_shift, float scale_log2, float cap_pre) {
  constexpr int kFloatWide = DT <= 8 ? 2 : 1;
  constexpr int kNarrow = kPrefixWaves * ((FLOAT ? kFloatWide : 1) * 32 + DT * 256) * 4, kWideBytes = FLOAT ? 0 : 8 * 64 * DT * 16;
  __shared__ __attribute__((aligned(16))) unsigned char lds[kNarrow > kWideBytes ? kNarrow : kWideBytes];
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
  const int columns = item.ntok * (nq / nkv) - item.col0;      // (of the tile and those behind it)
#define TLIE_ARGS positions, part_first, part_o, part_ml, nq, nkv, page_shift, scale_log2, cap_pre
  if constexpr (FLOAT) {
    if (kFloatWide > 1 && columns > 16)
      prefix_item<DT, true, kFloatWide, kPrefixWaves, false>(item, {}, kvh, q, cache, pages, TLIE_ARGS, reinterpret_cast<float*>(lds));
    else
      prefix_item<DT, true, 1, kPrefixWaves, false>(item, {}, kvh, q, cache, pages, TLIE_ARGS, reinterpret_cast<float*>(lds));
  } else {
    const uint16_t* q16 = static_cast<const uint16_t*>(q);
    const uint16_t* cache16 = static_cast<const uint16_t*>(cache);
    if (columns <= 16)
      prefix_item<DT, false, 1, kPrefixWaves, false>(item, {}, kvh, q, cache, pages, TLIE_ARGS, reinterpret_cast<float*>(lds));
    else if (DT > 8 || columns <= 64)
      prefix_wide_item<DT, 1>(item, kvh, q16, cache16, pages, TLIE_ARGS, lds);
    else
      prefix_wide_item<DT, (DT <= 8 ? 2 : 1)>(item, kvh, q16, cache16, pages, TLIE_ARGS, lds);
  }
#undef TLIE_ARGS
}

// Short steps in one launch: a workgroup of eight waves (sixteen take longer: 10.2 us in place of 7.3 for 340 keys of 64 dims) for up to 16
// columns of a sequence and all of their keys, the shared ones through another row of the table and read by every sequence for itself,
// from the second on out of a cache.  What bounds it is latency, and then the 16 addresses a clock of a compute unit's loads: 5 us per 1000 keys.
template <int DT, bool FLOAT>
__global__ void __launch_bounds__(64 * kDirectWaves, 2)
prefix_direct_kernel(const void* __restrict__ q, const void* __restrict__ cache, const int* __restrict__ block_table, int max_blocks,
                     const int* __restrict__ items, const int* __restrict__ positions, const float* __restrict__ sink, void* __restrict__ out, int nq,
                     int nkv, int page_shift, float scale_log2, float cap_pre) {
  __shared__ __attribute__((aligned(16))) float lds[kDirectWaves * (32 + DT * 256)];
  const int kvh = blockIdx.x % nkv;
  const int* words = items + static_cast<size_t>(blockIdx.x / nkv) * 8;
  auto word = [&](int i) { return __builtin_amdgcn_readfirstlane(words[i]); };
  const PrefixItem item{word(0), word(1), word(2), word(3), word(4), word(5), 1, 0};
  const Direct direct{block_table + static_cast<size_t>(word(7)) * max_blocks, item.key_lo, sink, out};
  prefix_item<DT, FLOAT, 1, kDirectWaves, true>(item, direct, kvh, q, cache, block_table + static_cast<size_t>(item.table) * max_blocks, positions, nullptr,
                                                nullptr, nullptr, nq, nkv, page_shift, scale_log2, cap_pre, lds);
}

// out[t][h] = sum_i w_i o_i / (sum_i w_i l_i + w_sink) over the token's parts.  A wave a (token, head): the lanes have a part's weight
// each first, then a sixteenth byte of it: d / 4 lanes take a part, the others the next ones.  Four loads a lane are on their way at a
// time, and the order of the additions is fixed by the number of parts.
template <bool FLOAT>
__global__ void __launch_bounds__(256)
prefix_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ part_first,
                   const float* __restrict__ sink, void* __restrict__ out, int rows, int nq, int d) {
  __shared__ float weights[4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * 4 + wave));
  if (row >= rows) return;
  const int token = row / nq, head = row - token * nq;
  const int first = __builtin_amdgcn_readfirstlane(part_first[token]), count = __builtin_amdgcn_readfirstlane(part_first[token + 1]) - first;
  const float own = sink != nullptr ? sink[head] * 1.4426950408889634f : -INFINITY;
  const int per = d >> 2, together = 64 / per, mine = lane / per, at = lane - mine * per;     // lanes a part, parts at a time
  const float* base = part_o + (static_cast<size_t>(first) * nq + head) * d + at * 4;
  const float* ml = part_ml + (static_cast<size_t>(first) * nq + head) * 2;
  float most = own, total = sink != nullptr ? 1.f : 0.f;        // (in units of 2^most)
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < count; p0 += 64) {                      // 64 parts at a time
    const int here = min(64, count - p0);
    const float2 stat = lane < here ? *reinterpret_cast<const float2*>(ml + static_cast<size_t>(p0 + lane) * nq * 2) : make_float2(-INFINITY, 0.f);
    const float next = fmaxf(most, wave_max(stat.x)), below = next == -INFINITY ? 0.f : next;
    const float down = __builtin_amdgcn_exp2f(most - below), weight = __builtin_amdgcn_exp2f(stat.x - below);
    total = total * down + wave_sum(weight * stat.y);
    sum.x *= down, sum.y *= down, sum.z *= down, sum.w *= down;
    most = next;
    weights[wave][lane] = weight;
    __builtin_amdgcn_wave_barrier();
    if (mine < together) {
      constexpr int kAhead = 4;
      for (int p = mine; p < here; p += kAhead * together) {
        float4 part[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) part[u] = *reinterpret_cast<const float4*>(base + static_cast<size_t>(p0 + min(p + u * together, here - 1)) * nq * d);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const float w = p + u * together < here ? weights[wave][min(p + u * together, here - 1)] : 0.f;
          sum.x += w * part[u].x, sum.y += w * part[u].y, sum.z += w * part[u].z, sum.w += w * part[u].w;
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  float4 all = sum;
  for (int other = 1; other < together; ++other) {              // (all lanes shuffle; the first part's lanes keep the sum)
    const int from = (at + other * per) & 63;
    all.x += __shfl(sum.x, from, 64), all.y += __shfl(sum.y, from, 64), all.z += __shfl(sum.z, from, 64), all.w += __shfl(sum.w, from, 64);
  }
  if (mine != 0) return;
  const float inv = total > 0.f ? 1.f / total : 0.f;            // a token that no sequence brings has no parts, and gets zeros
  all.x *= inv, all.y *= inv, all.z *= inv, all.w *= inv;
  if (FLOAT) *reinterpret_cast<float4*>(static_cast<float*>(out) + static_cast<size_t>(row) * d + at * 4) = all;
  else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + static_cast<size_t>(row) * d + at * 4) = make_uint2(pack_bf16(all.x, all.y), pack_bf16(all.z, all.w));
}

template <bool FLOAT, int DT>
static int launch_items(const void* q, const void* cache, const int* block_table, int max_blocks, const int* items, int num_items,
                        const int* positions, const int* part_first, float* part_o, float* part_ml, int nq, int nkv, int page_shift,
                        float scale_log2, float cap_pre, hipStream_t stream) {
  hipLaunchKernelGGL((prefix_items_kernel<DT, FLOAT>), dim3(num_items * nkv), dim3(64 * kPrefixWaves), 0, stream, q, cache, block_table, max_blocks,
                     items, positions, part_first, part_o, part_ml, nq, nkv, page_shift, scale_log2, cap_pre);
  return launch_status();
}

template <bool FLOAT, int DT>
static int launch_direct(const void* q, const void* cache, const int* block_table, int max_blocks, const int* items, int num_items, const int* positions,
                         const float* sink, void* out, int nq, int nkv, int page_shift, float scale_log2, float cap_pre, hipStream_t stream) {
  hipLaunchKernelGGL((prefix_direct_kernel<DT, FLOAT>), dim3(num_items * nkv), dim3(64 * kDirectWaves), 0, stream, q, cache, block_table, max_blocks, items,
                     positions, sink, out, nq, nkv, page_shift, scale_log2, cap_pre);
  return launch_status();
}

// ---- the host's half: which items a step has ----

// Columns of the tile that has so many of its item before it, itself included (prefix_items_kernel takes them so).
static int tile_columns(long long columns, int d, bool is_float) {
  if (columns <= 16) return 16;
  if (is_float) return d <= 128 ? 32 : 16;
  return columns > 64 && d <= 128 ? 128 : 64;
}
// A tile of 64 columns costs three times what one of 16 does a key, one of 128 five times (their products and softmax, not the keys' reading).
static double tile_cost(int columns) { return columns <= 32 ? 1.0 : columns <= 64 ? 3.0 : 5.0; }

constexpr int kLeastKeys = 128;      // that a part has, if the whole has as many

// Parts of about equal cost: a workgroup a compute unit, two where they are long.  A part more is a result more to write and to join, and
// memory's time where a prefix is long: 32 sequences behind 30000 positions, 32 heads of 128 on 8, their keys not in any cache, 46.9 us in 47 parts,
// 52.8 in 53, 50.6 in 40; eight questions behind 4000 51 in 5 parts, 57 in 4, 66 in 6.  A sixteenth of the units stays free for what the
// cuts leave over: 2 behind 8000 in one part more than there are units for 15.9 us, in two fewer 13.2.
static double part_cost(double total, int compute_units) {
  const double units = 0.9375 * compute_units;
  return std::max(total / (2.0 * units), std::min(total / units, 3200.0));
}

struct Cut {
  long long part, count;             // keys a part, and parts of the longest tile
};
// How `keys` positions, read by tiles the widest of which has `columns`, are cut.
static Cut cut_keys(long long keys, int columns, double budget, int most_parts) {
  const long long by_cost = std::llrint(static_cast<double>(keys) * tile_cost(columns) / std::max(budget, 1.0));
  const long long count = std::max(1ll, std::min({(keys + kLeastKeys - 1) / kLeastKeys, by_cost, static_cast<long long>(most_parts)}));
  // whole turns of a workgroup: wide tiles take two blocks of 32 keys each (32 sequences behind 30000 positions, keys in the caches: in parts of 544 keys 45.7 us, of 576 42.7)
  const long long turn = columns > 32 ? 64 : 32, part = ((keys + count - 1) / count + turn - 1) / turn * turn;
  return Cut{part, (keys + part - 1) / part};
}

// f(first column, columns of the tile) for the tiles of so many columns: of one width but the last, which has what is left.
template <typename F>
static void each_tile(long long columns, int d, bool is_float, F f) {
  const int step = tile_columns(columns, d, is_float);
  for (long long col0 = 0; col0 < columns; col0 += step) f(col0, columns - col0 > step ? step : tile_columns(columns - col0, d, is_float));
}

}  // namespace tlie

using namespace tlie;

// q, out: [tokens, nq, d]; cache: [pages, 2, nkv, page_size * d] (keys [row][dim], values [dim][row]); both of `dtype`.
// items: int32 [num_items, 8] (see PrefixItem; tiles of columns as prefix_items_kernel has them); part_first: int32 [tokens + 1], the first part of
// each token, so that part_first[tokens] is their number; part_o: float [parts, nq, d], part_ml: float [parts, nq, 2].
// sink: float [nq] or null.  softcap: 0, or the cap of the scaled scores.  part_o null: the items are those of tlie_prefix_direct.
extern "C" int tlie_attention_prefix(const void* q, const void* cache, int dtype, const int* block_table, int max_blocks, const int* items,
                                     int num_items, const int* positions, const int* part_first, float* part_o, float* part_ml,
                                     const float* sink, void* out, int tokens, int nq, int nkv, int d, int page_size, float scale,
                                     float softcap, void* stream) {
  // (a grid has fewer than 2^32 threads; the kernels read and write 16 bytes at a time)
  if (tokens <= 0 || num_items <= 0 || nq <= 0 || nkv <= 0 || nq % nkv != 0 || d <= 0 || d > 256 || d % 16 != 0 || page_size < 16 || page_size > 65536 ||
      (page_size & (page_size - 1)) != 0 || max_blocks <= 0 || !(scale > 0.f) || !(softcap >= 0.f) || (dtype != kF32 && dtype != kBF16) ||
      static_cast<long long>(num_items) * nkv >= 1ll << 24 || static_cast<long long>(tokens) * nq >= 1ll << 26 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(part_o)) & 15) != 0)
    return kBadArgument;
  const bool is_direct = part_o == nullptr;
  const float scale_log2 = (softcap > 0.f ? softcap : scale) * 1.4426950408889634f, cap_pre = softcap > 0.f ? scale / softcap : 0.f;
  // (below 2^-126 a number has fewer than 24 bits, and the scores would have no more)
  if (!(scale_log2 < INFINITY) || !(cap_pre < INFINITY) || (softcap > 0.f && !(cap_pre >= 1.17549435e-38f))) return kBadArgument;
  const int page_shift = 31 - __builtin_clz(page_size);
  hipStream_t s = (hipStream_t)stream;
  int status = kBadArgument;
  if (is_direct) {
#define TLIE_CASE(DT)                                                                                                                              \
  case DT:                                                                                                                                         \
    return launch_direct<false, DT>(q, cache, block_table, max_blocks, items, num_items, positions, sink, out, nq, nkv, page_shift, scale_log2,    \
                                    cap_pre, s);
#define TLIE_FLOAT(DT)                                                                                                                             \
  case DT:                                                                                                                                         \
    return launch_direct<true, DT>(q, cache, block_table, max_blocks, items, num_items, positions, sink, out, nq, nkv, page_shift, scale_log2,     \
                                   cap_pre, s);
    if (dtype == kF32) switch (d / 16) { TLIE_FLOAT(1) TLIE_FLOAT(2) TLIE_FLOAT(3) TLIE_FLOAT(4) }
    else switch (d / 16) { TLIE_CASE(1) TLIE_CASE(2) TLIE_CASE(3) TLIE_CASE(4) TLIE_CASE(5) TLIE_CASE(6) }
#undef TLIE_FLOAT
#undef TLIE_CASE
    return kBadArgument;
  }
#define TLIE_CASE(DT)                                                                                                                              \
  case DT:                                                                                                                                         \
    status = dtype == kF32 ? launch_items<true, DT>(q, cache, block_table, max_blocks, items, num_items, positions, part_first, part_o,      \
                                                    part_ml, nq, nkv, page_shift, scale_log2, cap_pre, s)                                          \
                           : launch_items<false, DT>(q, cache, block_table, max_blocks, items, num_items, positions, part_first, part_o,     \
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

// The items of a step, on the host: seq_start [sequences + 1] and seq_len [sequences] are its cumulative token counts and its sequences' lengths
// after it; groups [num_groups][3] (first sequence, sequences, prefix), in ascending order, have the keys 0 .. prefix - 1 in common.
// items: int32 [.][8], of which max_items fit; part_first: int32 [tokens + 1].  Returns the number of items, and writes nothing when they do
// not fit; or -1: sequences that do not count up, or are shorter than what they bring; -2: groups that are not runs of the step's
// sequences, apart from one another; -3: a token inside its group's prefix; -4: sizes; -5: a step beyond one launch.
extern "C" int tlie_prefix_plan(const long long* seq_start, const long long* seq_len, int sequences, const long long* groups, int num_groups, int nq,
                                int nkv, int d, int dtype, int compute_units, int most_parts, int* items, int max_items, int* part_first) {
  constexpr long long kLongest = 1ll << 30;
  const bool is_float = dtype == kF32;
  if (sequences < 0 || num_groups < 0 || nq <= 0 || nkv <= 0 || nq % nkv != 0 || d <= 0 || compute_units <= 0 || most_parts <= 0) return -4;
  const long long G = nq / nkv;
  if (seq_start[0] != 0) return -1;
  for (int s = 0; s < sequences; ++s) {
    const long long count = seq_start[s + 1] - seq_start[s];
    if (count < 0 || seq_len[s] < count) return -1;
    if (seq_len[s] > kLongest || seq_start[s + 1] >= (1ll << 26) / nq) return -5;
  }
  const long long tokens = seq_start[sequences];
  // ---- the groups, checked, and what the step costs ----
  double cost = 0.0;
  long long after = 0;
  for (int g = 0; g < num_groups; ++g) {
    const long long first = groups[3 * g], count = groups[3 * g + 1], prefix = groups[3 * g + 2];
    if (count < 1 || prefix < 0 || first < after || count > sequences || first > sequences - count) return -2;
    after = first + count;
    for (long long s = first; s < after; ++s)
      if (seq_start[s + 1] > seq_start[s] && seq_len[s] - (seq_start[s + 1] - seq_start[s]) < prefix) return -3;
    each_tile((seq_start[after] - seq_start[first]) * G, d, is_float, [&](long long, int width) { cost += static_cast<double>(prefix) * tile_cost(width); });
  }
  // f(sequence, its tokens, its own first key), for those that bring tokens, and of its group's place (or -1)
  auto each_sequence = [&](auto f) {
    int g = 0;
    for (int s = 0; s < sequences; ++s) {
      while (g < num_groups && groups[3 * g] + groups[3 * g + 1] <= s) ++g;
      const bool grouped = g < num_groups && groups[3 * g] <= s;
      if (seq_start[s + 1] > seq_start[s]) f(s, seq_start[s + 1] - seq_start[s], grouped ? groups[3 * g + 2] : 0ll, grouped ? g : -1);
    }
  };
  // a tile's keys end with the last token that it has columns of
  auto own_end = [&](int s, long long count, long long col0, int width) { return seq_len[s] - count + std::min(count - 1, (col0 + width - 1) / G) + 1; };
  each_sequence([&](int s, long long count, long long from, int) {
    each_tile(count * G, d, is_float, [&](long long col0, int width) { cost += static_cast<double>(own_end(s, count, col0, width) - from) * tile_cost(width); });
  });
  const double budget = part_cost(cost * nkv, compute_units);
  // All tiles of a group's prefix, and all of a sequence's own keys, are cut alike: as their widest and longest are.
  auto cut_of_group = [&](int g) {
    const long long columns = (seq_start[groups[3 * g] + groups[3 * g + 1]] - seq_start[groups[3 * g]]) * G;
    return groups[3 * g + 2] > 0 && columns > 0 ? cut_keys(groups[3 * g + 2], tile_columns(columns, d, is_float), budget, most_parts) : Cut{1, 0};
  };
  auto cut_of_own = [&](int s, long long count, long long from) { return cut_keys(seq_len[s] - from, tile_columns(count * G, d, is_float), budget, most_parts); };

  // ---- twice over the tiles: how many items, then the items ----
  long long total = 0;
  auto walk = [&](auto put) {                        // put(table row, tile's tokens from, tokens, first column, first key, end, own, keys a part, first part)
    for (int g = 0; g < num_groups; ++g) {
      const long long first = groups[3 * g], last = first + groups[3 * g + 1];
      const Cut cut = cut_of_group(g);
      if (cut.count == 0) continue;
      long long reader = first;                      // a sequence that brings no tokens may be shorter than the prefix: the first that does holds it
      while (seq_start[reader + 1] == seq_start[reader]) ++reader;
      each_tile((seq_start[last] - seq_start[first]) * G, d, is_float, [&](long long col0, int) {
        put(reader, seq_start[first], seq_start[last] - seq_start[first], col0, 0ll, groups[3 * g + 2], 0, cut.part, 0ll);
      });
    }
    int group = -1;
    long long ahead = 0;
    each_sequence([&](int s, long long count, long long from, int g) {
      if (g != group) group = g, ahead = g >= 0 ? cut_of_group(g).count : 0;
      const Cut cut = cut_of_own(s, count, from);
      each_tile(count * G, d, is_float, [&](long long col0, int width) {
        put(s, seq_start[s], count, col0, from, own_end(s, count, col0, width), 1, cut.part, ahead);
      });
    });
  };
  walk([&](long long, long long, long long, long long, long long lo, long long hi, int, long long part, long long) { total += (hi - lo + part - 1) / part; });
  if (total * nkv >= 1ll << 24) return -5;
  if (total > max_items) return static_cast<int>(total);
  int* word = items;
  walk([&](long long table, long long tok0, long long ntok, long long col0, long long lo, long long hi, int own, long long part, long long place) {
    for (long long key = lo; key < hi; key += part, ++place, word += 8) {
      const long long values[8] = {table, tok0, ntok, col0, key, std::min(hi, key + part), own, place};
      for (int i = 0; i < 8; ++i) word[i] = static_cast<int>(values[i]);
    }
  });
  // a token's parts: its group's, then those of its own keys that begin at or before it
  long long parts = 0, token = 0;
  int group = -1;
  long long ahead = 0;
  each_sequence([&](int s, long long count, long long from, int g) {
    if (g != group) group = g, ahead = g >= 0 ? cut_of_group(g).count : 0;
    const Cut cut = cut_of_own(s, count, from);
    for (long long i = 0; i < count; ++i, ++token) {
      part_first[token] = static_cast<int>(std::min(parts, 0x7fffffffll));
      parts += ahead + (seq_len[s] - count + i - from) / cut.part + 1;
    }
  });
  part_first[tokens] = static_cast<int>(std::min(parts, 0x7fffffffll));
  return parts * nq > 0x7fffffffll ? -5 : static_cast<int>(total);
}

// The items of a short step that one launch takes (part_o null in tlie_attention_prefix), for a step that tlie_prefix_plan has a plan for: [.][8]
// (sequence, first token, tokens, first column, shared keys, end of the keys, 1, the row that the shared keys are read through).  Returns
// their number; 0: such a step takes longer this way.
extern "C" int tlie_prefix_direct(const long long* seq_start, const long long* seq_len, int sequences, const long long* groups, int num_groups, int nq,
                                  int nkv, int d, int dtype, int compute_units, int* items, int max_items) {
  const long long G = nq / nkv;
  // bytes of a plane of keys, and head sizes, up to which one launch is no slower in a recording either (16 sequences, 32 heads of 64 on 4, 440
  // keys 7.4 us, in parts 10.4; 12 heads of 32 on 4, 940 keys 6.6 and 8.2; 16 heads of 96, 540 keys 9.3 and 10.4; of 128 on 8, 160 keys
  // 10.1 and 9.9, 300 11.9 and 9.7); from eager calls 9.8 us and 14.1.  More workgroups than units run one after the other (48
  // sequences, 24 heads of 80 on 8: 13.9 and 11.9).
  constexpr long long kMostBytes = 98304;
  if (d > (dtype == kF32 ? 64 : 96)) return 0;
  long long count = 0;
  int g = 0;
  for (int s = 0; s < sequences; ++s) {
    const long long tokens = seq_start[s + 1] - seq_start[s];
    while (g < num_groups && groups[3 * g] + groups[3 * g + 1] <= s) ++g;
    if (tokens == 0) continue;
    const bool grouped = g < num_groups && groups[3 * g] <= s;
    long long reader = s;
    if (grouped) {
      reader = groups[3 * g];
      while (seq_start[reader + 1] == seq_start[reader]) ++reader;
    }
    for (long long col0 = 0; col0 < tokens * G; col0 += 16, ++count) {
      const long long end = seq_len[s] - tokens + std::min(tokens - 1, (col0 + 15) / G) + 1;
      if (end * d * (dtype == kF32 ? 4 : 2) > kMostBytes || count >= max_items) return 0;
      const long long values[8] = {s, seq_start[s], tokens, col0, grouped ? groups[3 * g + 2] : 0, end, 1, reader};
      for (int i = 0; i < 8; ++i) items[count * 8 + i] = static_cast<int>(values[i]);
    }
  }
  return count * nkv <= compute_units ? static_cast<int>(count) : 0;
}
