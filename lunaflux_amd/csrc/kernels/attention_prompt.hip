// attention_prompt.hip - attention of the rows of prompts, or of parts of them, over the
// paged key / value cache (the attention section of include/lunaflux_fp8.h).
#include "device_common.h"

#include "attention_index.h"

namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// One pass over the keys with the running maximum and sum of each row's softmax. A block holds a
// query tile (attention_index.h, QueryTile) of which each wave has 32 rows in registers, as the
// B operand of S^T = K Q^T; that leaves a lane the scores of one row, so its statistics are
// lane values, and 16 weights per 32 keys in the order of the B operand of O^T = V^T P^T. Key and
// value tiles go through LDS, shared by the waves; values are read from it transposed.
// The waves are two groups, one wave of each on every SIMD, half a tile apart: between two
// barriers one group's waves have the products of a tile and the other's its softmax.
// Blocks are dealt equal ranges of the step's weight (attention_index.h); a query tile cut
// between ranges leaves fp32 partial results, which a second launch adds up in their order.
//
// Weights are rounded to bf16 once, for the second product, and their sum is of the rounded ones, so
// that equal values come out equal. A weight is off by up to 2^-8 of itself, as a value of out is: for values
// without a common part the errors are as large as out's own rounding (1.7e-3 to 2.4e-3 of out in all against
// 64 bits, more the more keys; 1.6e-3 to 1.7e-3 where only out is rounded). A second bf16 term would take that away for half as many
// products again.
//
// Matrix products bound it, with the softmax close behind: of a tile of heads of 128 a wave has 32 products,
// 1024 cycles of the matrix unit, and some 190 vector instructions, 900 of the vector unit. 8192 rows, 32/8 heads
// of 128: 555-570 us, 0.97-0.99 PFLOP/s of 1.39 that an 8192^3 product reaches, at the 1.9 GHz that the card holds
// under it; under the counters matrix units 47 % of the cycles, LDS reads 23 % without conflicts. By steps: waves
// of 16 rows with tiles through registers 1652 us; two groups of waves with 32 rows and loads that go
// straight to LDS 696; operands read ahead and code of their own for the groups 584; a third stage of
// tiles 551. Loads issued by the second group instead of the first: 591 at the time of 554. Tiles of 32 keys
// for heads of 256, whose sums and queries take 192 registers of a lane: 170 us for 2045 rows behind 2500 tokens each.
template <int D>
struct Prompts {
  static constexpr int kWaves = 8, kThreads = 64 * kWaves, kBlocks = 256;
  static constexpr int kRows = 32 * kWaves;
  static constexpr int kKeys = D == 256 ? 32 : 64;
  static constexpr int kKeyTiles = kKeys / 32;
  static constexpr int kTileBytes = kKeys * D * 2;
  static constexpr int kFloats = kRows * (D + 2);  // of a partial result: sums, maxima, weight sums
};
constexpr int kJoinSlices = 8, kMostSequences = 2048;  // LF_FP8_ATTN_MAX_SEQUENCES

// The step's prompts, their weights added up in LDS.
struct PromptPlan {
  int n, rows;
  QueryTile tile;
  int heads;             // pairs of key head and part of its group
  int token_of;          // rows of a tile to tokens: row token_of >> 16 (exact: both are at most 256)
  int64_t total, share;
};

template <int D, int THREADS>
LF_DEVICE PromptPlan plan_of(const Desc &d, const int32_t *counts, const int32_t *row_offsets, const int32_t *lengths,
                             const int32_t *page_offsets, int64_t *prefix, bool &bad) {
  __shared__ int64_t wave_total[THREADS / 64], wave_rows[THREADS / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  PromptPlan plan;
  plan.rows = live_rows(counts, d.max_tokens);
  plan.n = decoded_of(d, 0, counts[0], counts[2]).n;
  plan.tile = query_tile_of(d, Prompts<D>::kRows);
  plan.heads = d.kv_heads * plan.tile.subs;
  plan.token_of = plan.tile.subs > 1 ? 0 : (65536 + plan.tile.heads - 1) / plan.tile.heads;
  int64_t carry = 0, rows = 0;
  for (int base = 0; base < plan.n; base += THREADS) {
    const int i = base + static_cast<int>(threadIdx.x);
    int64_t weight = 0;
    int mine = 0;
    if (i < plan.n) {
      const Prompt p = prompt_of(d, row_offsets, lengths, page_offsets, i, plan.rows, bad);
      const Weights w = weights_of(d, plan.tile, p);
      weight = weight_before(w, w.tiles);
      mine = p.rows;
    }
    int64_t sum = weight, some = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int64_t up = __shfl_up(sum, m), more = __shfl_up(some, m);
      if (lane >= m) sum += up, some += more;
    }
    if (lane == 63) wave_total[wave] = sum, wave_rows[wave] = some;
    __syncthreads();
    int64_t before = carry;
    for (int k = 0; k < THREADS / 64; ++k) {
      if (k < wave) before += wave_total[k];
      carry += wave_total[k];
      rows += wave_rows[k];
    }
    if (i < plan.n) prefix[i] = before + sum - weight;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[plan.n] = carry;
  __syncthreads();
  if (rows > plan.rows) {  // sequences that share rows
    bad = true;
    carry = 0;
  }
  plan.total = carry * plan.heads;
  plan.share = (plan.total + Prompts<D>::kBlocks - 1) / Prompts<D>::kBlocks;
  return plan;
}

// A pair of the step: its sequence, head (key head and part of its group), query tile, and place in the weight.
struct PromptPair {
  int i, x, head;
  int64_t begin, weight;
  Prompt p;
  Weights w;
};
// Query heads of a pair: key head, first query head and number.
struct PairHeads {
  int h, first, count;
};
LF_DEVICE PairHeads heads_of(const Desc &d, const PromptPlan &plan, const PromptPair &pair) {
  const int group = d.query_heads / d.kv_heads;
  if (plan.tile.subs == 1) return {pair.head, pair.head * group, group};
  const int h = pair.head / plan.tile.subs, from = (pair.head - h * plan.tile.subs) * plan.tile.heads;
  return {h, h * group + from, group - from < plan.tile.heads ? group - from : plan.tile.heads};
}
LF_DEVICE void read_prompt(const Desc &d, const PromptPlan &plan, const int32_t *row_offsets, const int32_t *lengths,
                           const int32_t *page_offsets, PromptPair &pair) {
  bool unused = false;
  pair.p = prompt_of(d, row_offsets, lengths, page_offsets, pair.i, plan.rows, unused);
  pair.w = weights_of(d, plan.tile, pair.p);
}
LF_DEVICE PromptPair pair_at(const Desc &d, const PromptPlan &plan, const int32_t *row_offsets, const int32_t *lengths,
                             const int32_t *page_offsets, const int64_t *prefix, int64_t u) {
  PromptPair pair;
  pair.i = __builtin_amdgcn_readfirstlane(prompt_at(prefix, plan.n, plan.heads, u));
  read_prompt(d, plan, row_offsets, lengths, page_offsets, pair);
  const int64_t first = prefix[pair.i] * plan.heads, each = prefix[pair.i + 1] - prefix[pair.i];
  int64_t head = quotient(u - first, each);  // up to one off where the weights pass 2^52
  if (head * each > u - first) --head;
  if ((head + 1) * each <= u - first) ++head;
  pair.head = __builtin_amdgcn_readfirstlane(static_cast<int>(head));
  const int64_t within = u - first - pair.head * each;
  pair.x = __builtin_amdgcn_readfirstlane(tile_at(pair.w, within));
  pair.begin = first + pair.head * each + weight_before(pair.w, pair.x);
  pair.weight = weight_of(pair.w, pair.x);
  return pair;
}

// One v_cvt_pk_bf16_f32, rounded to nearest even.
LF_DEVICE uint32_t pack_bf16(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// Byte of 16-byte chunk `chunk` of a key's row in an LDS tile of rows of D bf16 values.
template <int D>
LF_DEVICE uint32_t tile_byte(int key, int chunk) {
  return static_cast<uint32_t>(key * D * 2 + ((chunk ^ (chunk_swizzle(key & 15) & (D / 8 - 1))) << 4));
}

// Partial results, their maxima and their weight sums in the workspace, behind a line with the error word.
template <int D>
LF_DEVICE float *partial_of(uint8_t *ws, int slot) {
  return reinterpret_cast<float *>(ws + 256) + static_cast<uint64_t>(slot) * Prompts<D>::kFloats;
}

// What the join has to know of a range: the first query tile in it, of weights [begin, begin + weight) of the step's.
// The first launch writes it (weight 0 where the range is empty) in the place of partial result 0, so that the
// second, of whose blocks a CU holds eight, does not look for it once more: 20 and 9 us for four prompts, 27 and 16
// for 8192 rows.
struct RangeStart {
  int64_t share, begin, weight;
  int tiles, row0, head0, heads, rows, token_of, h;
};
LF_DEVICE RangeStart *start_of(uint8_t *ws, int range) { return reinterpret_cast<RangeStart *>(ws + 256) + range; }
static_assert(Prompts<64>::kBlocks * sizeof(RangeStart) <= Prompts<64>::kFloats * 4, "");

// One global_load_lds_dwordx4: every lane's 16 bytes from its address go to LDS at lds + 16 lane
// (wave-uniform; M0, whose write has to be a wait state before the load, which the compiler does not
// see to inside an asm). As assembly, so that the compiler does not make every LDS read wait for it:
// the kernel orders it by itself, with vmcnt and barriers. No read of the interval that it is issued in
// touches what it writes, so the two may change places (interval_end holds both).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // M0 is listed as clobbered on purpose
LF_DEVICE void load_to_lds(const uint8_t *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "m0");
}
// The same for 4 bytes a lane.
LF_DEVICE void load_word_to_lds(const float *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               :
               : "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "m0");
}
// All but the last LEFT of this wave's loads to LDS have arrived.
template <int LEFT>
LF_DEVICE void loads_arrived() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
#pragma clang diagnostic pop
LF_DEVICE uint32_t lds_at(const uint8_t *p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) uint8_t *)p));
}
template <class T>
LF_DEVICE T lds_read(uint32_t at) {
  return *(const __attribute__((address_space(3))) T *)at;
}
template <class T>
LF_DEVICE void lds_write(uint32_t at, T v) {
  *(__attribute__((address_space(3))) T *)at = v;
}

// The block's barrier between intervals: this wave's LDS accesses are over, and no instruction
// moves past it. LOADS: its loads have arrived too, but for the last LEFT.
template <bool LOADS, int LEFT = 0>
LF_DEVICE void interval_end() {
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (LOADS) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
  } else {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
  __builtin_amdgcn_sched_barrier(0);
}

// v times a weight above zero that may have vanished in fp32: an infinite value stays what it is. So a row that counts
// one has the same result wherever its largest score is and wherever its keys are cut.
LF_DEVICE float weighted(float v, float weight) { return fabsf(v) == INFINITY ? v : v * weight; }

// The rows of a query tile that one wave has, without the matrix units: for rows that some infinity or NaN
// reached, since in products of tiles zero times such a value of a key that a row does not count is NaN
// too, for ones with scores so large that their differences need the scores rounded as the maximum is, and
// for tables with pages outside the cache. Here only the keys that it counts enter. Lanes c and
// c + 32 hold the halves of row c. Apart from the kernel's registers, and slow, which such rows bear: a
// prompt of 8192 rows that all hold a NaN takes 233 ms, 400 times as long as without.
struct CarefulRow {
  const uint16_t *q;
  const uint8_t *kc, *vc;
  const int32_t *table;
  PromptKeys keys;
  int k0, k1, h, position;
  float factor;
};
template <int D, int CACHE>
__device__ __attribute__((noinline)) void careful_row(const Desc &d, const CarefulRow &r, bool flip, float (&acc)[D / 2], float &top, float &sum) {
  constexpr int kKeys = Prompts<D>::kKeys;
  constexpr bool E4M3 = CACHE != kCacheBf16;
  const int half = (threadIdx.x >> 5) & 1;
  const int shift = __builtin_ctz(d.page_size), slot_mask = d.page_size - 1;
  auto value = [&](const uint8_t *cache, int page, int slot, int e) {
    const uint64_t at = cache_byte<E4M3>(d, page, r.h, slot);
    if constexpr (E4M3) {
      const float v = __builtin_amdgcn_cvt_f32_fp8(cache[at + e], 0);
      return CACHE == kCacheBlocks ? v * reinterpret_cast<const float *>(cache + d.block_scales)[scale_index(d, page, slot, r.h)] : v;
    } else {
      return bf16_to_f32(*reinterpret_cast<const uint16_t *>(cache + at + 2 * e));
    }
  };
  top = -INFINITY;
  sum = 0.0f;
  for (int e = 0; e < D / 2; ++e) acc[e] = 0.0f;
  for (int t = r.k0; t < r.k1; ++t) {
    const int base = kKeys * (t < r.keys.sink_tiles ? t : t + r.keys.first - r.keys.sink_tiles);
    for (int j = base; j < base + kKeys && j <= r.keys.last; ++j) {
      if (j >= r.keys.sink && j < r.keys.lo) continue;
      const int page = r.table[j >> shift], slot = j & slot_mask;
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(d.pages)) continue;
      float score = 0.0f;
      for (int e = 0; e < D / 2; ++e) score += bf16_to_f32(r.q[half * (D / 2) + e]) * value(r.kc, page, slot, half * (D / 2) + e);
      score += __shfl_xor(score, 32);
      if (j > r.position || !(d.window == 0 || j > r.position - d.window || j < d.sinks)) continue;
      float z = (flip ? -score : score) * r.factor;
      asm("" : "+v"(z));  // rounded, for the difference below too: a fused one is not zero at the maximum
      const float next = fmaxf(top, z), from = next == -INFINITY ? 0.0f : next;
      const float keep = __builtin_amdgcn_exp2f(top - from), p = __builtin_amdgcn_exp2f(z - from);
      top = next;
      sum = sum * keep + p;
      for (int e = 0; e < D / 2; ++e) {
        const float v = value(r.vc, page, slot, half * (D / 2) + e);
        acc[e] = weighted(acc[e], keep) + (z == -INFINITY ? v * p : weighted(v, p));
      }
    }
  }
}

template <int D, int CACHE>
LF_DEVICE void prefill(const int32_t *counts, const int32_t *row_offsets, const int32_t *lengths,
                       const int32_t *page_offsets, const int32_t *page_indices, const uint8_t *attn,
                       const uint16_t *q, uint16_t *out, const uint8_t *kc, const uint8_t *vc, uint8_t *ws) {
  using P = Prompts<D>;
  constexpr int KT = P::kKeyTiles, kKeys = P::kKeys, kSteps = D / 16, kBands = D / 32;
  constexpr bool E4M3 = CACHE != kCacheBf16;
  extern __shared__ __attribute__((aligned(1024))) uint8_t stages[];
  const Desc &d = desc_of(attn);
  if (d.magic != kMagic) return;
  int *error = reinterpret_cast<int *>(ws);
  // Stage i: the keys of tile i and the values of tile i - 1. Three of them where tiles go straight to LDS, so that
  // two are on their way; of codes two, and two more of the codes themselves, which their waves convert.
  constexpr int kStages = E4M3 ? 2 : 3;
  __shared__ int64_t prefix[kMostSequences + 1];
  __shared__ float code_scales[CACHE == kCacheBlocks ? 2 * 2 * P::kThreads : 1];
  const uint32_t stages_at = lds_at(stages), codes_at = stages_at + 4 * P::kTileBytes, scales_at = lds_at(reinterpret_cast<const uint8_t *>(code_scales));
  auto keys_at = [&](int i) { return stages_at + i % kStages * 2 * P::kTileBytes; };
  auto values_at = [&](int i) { return stages_at + (i + 1) % kStages * 2 * P::kTileBytes + P::kTileBytes; };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __shared__ int once_more;
  const bool late = wave >= P::kWaves / 2;  // the group that is half a tile behind
  const int c = lane & 31, half = lane >> 5;
  bool bad = false;
  const PromptPlan plan = plan_of<D, P::kThreads>(d, counts, row_offsets, lengths, page_offsets, prefix, bad);
  const int range = range_of_block(blockIdx.x, P::kBlocks);
  const int64_t u0 = range * plan.share, u1 = u0 + plan.share < plan.total ? u0 + plan.share : plan.total;
  if (bad) flag_error(error);
  const bool cuts = cuts_prompts(d, P::kRows, kKeys);
  if (u0 >= u1) {
    if (cuts && threadIdx.x == 0) start_of(ws, range)->weight = 0;
    return;
  }

  const int Hq = d.query_heads, Hkv = d.kv_heads;
  const int shift = __builtin_ctz(d.page_size), slot_mask = d.page_size - 1, pages = d.pages;
  const float *scales = reinterpret_cast<const float *>(attn + d.scale_offset);
  const bool flip = d.softmax_scale < 0.0f;
  const int window = d.window > 0 ? d.window : INT32_MAX, sinks = d.sinks;
  constexpr uint32_t kSize = E4M3 ? 1 : 2;
  const uint32_t page_bytes = static_cast<uint32_t>(d.page_stride) * kSize, token_bytes = static_cast<uint32_t>(d.token_stride) * kSize;
  const uint32_t head_bytes = static_cast<uint32_t>(d.head_stride) * kSize;
  const int64_t d_block_scales = d.block_scales;

  PromptPair pair = pair_at(d, plan, row_offsets, lengths, page_offsets, prefix, u0);
  for (;;) {
    const PromptKeys pk = keys_of(d, plan.tile, pair.p, pair.x, kKeys);
    const int cut = cut_tiles(plan.share, kKeys);
    const int k0 = cut_of(u0, pair.begin, pair.weight, pk.tiles, cut), k1 = cut_of(u1, pair.begin, pair.weight, pk.tiles, cut);
    const PairHeads of = heads_of(d, plan, pair);
    const int h = of.h, head0 = of.first, heads = of.count, tokens = pk.last - pk.first_position + 1;
    const int row0 = pair.p.row + pair.x * plan.tile.tokens;
    if (cuts && pair.begin <= u0 && threadIdx.x == 0) {
      *start_of(ws, range) = {plan.share, pair.begin, pair.weight, pk.tiles, row0, head0, heads, tokens * heads, plan.token_of, h};
    }
    if (k0 < k1) {
      const int32_t *table = page_indices + pair.p.entry;
      const int page_first = pk.lo >> shift, page_end = (pk.last >> shift) + 1, sink_end = (pk.sink + slot_mask) >> shift;
      // (a scale of zero as one that leaves -infinity, a masked score, what it is)
      const float factor = fmaxf(fabsf(d.softmax_scale) * 1.44269504088896341f * (CACHE == kCacheE4m3 ? scales[h] : 1.0f), 0x1p-126f);
      const int n = k1 - k0;
      auto base_of = [&](int i) { return kKeys * (k0 + i < pk.sink_tiles ? k0 + i : k0 + i + pk.first - pk.sink_tiles); };

      // Tiles are loaded by the first group's waves, or by all of them where codes are converted (of heads of 64 keys
      // by the first group's and values by the second's); kLoaders waves share a tile's rows.
      constexpr int kLoaders = E4M3 && D != 64 ? P::kWaves : P::kWaves / 2, kWaveKeys = kKeys / kLoaders, kGroups = (kWaveKeys + 7) / 8;
      // Pages of the groups of eight keys of a tile that are this wave's to load, by scalar loads, so that no wait
      // for them is one for the tiles on their way (they share a counter with LDS reads, so they are on their way
      // only during a softmax). One that the cache does not have is read as page 0: the
      // tiles' results are not used then.
      int tile_pages[2][kGroups];  // of the tile whose keys are loaded next, and of the one before
      int loading[kGroups];
      bool outside = false;
      auto pages_of_tile = [&](int i) {
        typedef const __attribute__((address_space(4))) int32_t *Constant;
        const int base = base_of(i < n ? i : n - 1);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int j = base + ((wave & (kLoaders - 1)) * kWaveKeys & ~7) + 8 * g;
          loading[g] = ((Constant)table)[__builtin_amdgcn_readfirstlane(sink_entry_of(sink_end, page_first, page_end, shift, j))];
        }
      };
      auto arrived = [&]() {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const bool in = static_cast<uint32_t>(loading[g]) < static_cast<uint32_t>(pages);
          outside |= !in;
          tile_pages[1][g] = tile_pages[0][g];
          tile_pages[0][g] = in ? loading[g] : 0;
        }
      };
      auto slot_of = [&](int base, int key) {
        const int j = base + key;
        return (j < pk.last ? j : pk.last) & slot_mask;
      };
      const uint8_t *head_keys = kc + static_cast<uint64_t>(static_cast<uint32_t>(h)) * head_bytes;
      const uint8_t *head_values = vc + static_cast<uint64_t>(static_cast<uint32_t>(h)) * head_bytes;
      auto load_tile = [&](const uint8_t *cache, uint32_t to, int base, const int (&p)[kGroups]) {  // bf16
        constexpr int kChunks = D / 8, kRowsAtOnce = 64 / kChunks;
        const int first = wave * kWaveKeys;
#pragma unroll
        for (int r = 0; r < kWaveKeys; r += kRowsAtOnce) {
          const int key = first + r + lane / kChunks, chunk = lane & (kChunks - 1);
          const int from = chunk ^ (chunk_swizzle(key & 15) & (kChunks - 1));
          const uint8_t *page = cache + static_cast<uint64_t>(static_cast<uint32_t>(p[r / 8])) * page_bytes;
          load_to_lds(page + (static_cast<uint64_t>(static_cast<uint32_t>(slot_of(base, key))) * token_bytes + 16 * from), to + (first + r) * D * 2);
        }
      };
      // e4m3: a thread's 16 codes of a row of keys and of one of values (heads of 64: of either, by the wave's group).
      constexpr int kSides = D == 64 ? 1 : 2, kKeyLanes = D / 16, kSideBytes = kKeys * D;
      const int code_thread = D == 64 ? static_cast<int>(threadIdx.x) & 255 : static_cast<int>(threadIdx.x);
      const int code_key = code_thread / kKeyLanes, code_at = code_thread % kKeyLanes;
      auto load_codes = [&](const uint8_t *head, const uint8_t *cache, bool value, int stage, int base, const int (&of_groups)[kGroups]) {
        const int p = kGroups == 2 && (code_key & 8) != 0 ? of_groups[kGroups - 1] : of_groups[0];
        const int slot = slot_of(base, code_key), place = (stage & 1) * 2 + value;
        load_to_lds(head + (row_byte(p, slot, page_bytes, token_bytes) + 16 * code_at), codes_at + place * kSideBytes + (code_thread & ~63) * 16);
        if constexpr (CACHE == kCacheBlocks) {
          load_word_to_lds(reinterpret_cast<const float *>(cache + d_block_scales) + scale_index(d, p, slot, h),
                           scales_at + place * P::kThreads * 4 + (code_thread & ~63) * 4);
        }
      };
      struct Codes {
        u32x4 w;
        float scale;
      };
      auto read_codes = [&](bool value, int stage, Codes &x) {
        const int place = (stage & 1) * 2 + value;
        x.w = lds_read<u32x4>(codes_at + place * kSideBytes + code_thread * 16);
        x.scale = 1.0f;
        if constexpr (CACHE == kCacheBlocks) x.scale = lds_read<float>(scales_at + (place * P::kThreads + code_thread) * 4);
      };
      auto convert = [&](const Codes &x, uint32_t to) {
        uint32_t b[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          b[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(x.w[e]), x.scale, false));
          b[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(x.w[e]), x.scale, true));
        }
        lds_write(to + tile_byte<D>(code_key, 2 * code_at), u32x4{b[0], b[1], b[2], b[3]});
        lds_write(to + tile_byte<D>(code_key, 2 * code_at + 1), u32x4{b[4], b[5], b[6], b[7]});
      };
      // Begins to load stage i (behind the last tile the last one's keys, of no use).
      auto load_stage = [&](int i) {
        const int key_base = base_of(i < n ? i : n - 1), value_base = base_of(i > 0 ? i - 1 : 0);
        if constexpr (!E4M3) {
          load_tile(head_keys, keys_at(i), key_base, tile_pages[0]);
          if (i > 0) load_tile(head_values, values_at(i - 1), value_base, tile_pages[1]);
        } else {
          if (kSides == 2 || !late) load_codes(head_keys, kc, false, i, key_base, tile_pages[0]);
          if (kSides == 2 || late) load_codes(head_values, vc, true, i, value_base, tile_pages[1]);
        }
      };
      // Codes that have arrived to their places as bf16 values.
      auto convert_stage = [&](int i) {
        Codes keys, values;
        if (kSides == 2 || !late) read_codes(false, i, keys);
        if (i > 0 && (kSides == 2 || late)) read_codes(true, i, values);
        if (kSides == 2 || !late) convert(keys, keys_at(i));
        if (i > 0 && (kSides == 2 || late)) convert(values, values_at(i - 1));
      };

      // this lane's row: query operand, position, statistics
      u32x4 qv[kSteps];
      const int m = wave * 32 + c, token = (m * plan.token_of) >> 16, head = m - token * heads;
      const bool live = m < tokens * heads;
      const int position = live ? pk.first_position + token : pk.first_position;
      const uint32_t row_at = static_cast<uint32_t>(live ? row0 + token : row0) * Hq + head0 + (live ? head : 0);
      {
        const uint16_t *src = q + static_cast<uint64_t>(row_at) * D + 8 * half;
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
          u32x4 w = *reinterpret_cast<const u32x4 *>(src + 16 * t);
          if (flip) w ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
          qv[t] = w;
        }
      }
      // Weights are relative to `top`, the row's maximum in the first tile that it counts a key of. It need not be
      // the row's largest score, only near it: a weight of 2^kNear and sums of 2^31 of them are as exact in fp32
      // and bf16 as ones. Past that the tiles are gone through once more, with the largest that was seen. So the
      // sums are never scaled, which would take a multiplication of each for every tile (heads of 128: 64 of a
      // lane's; with them the kernel did not fit its registers).
      constexpr float kNear = 40.0f;
      float top = -INFINITY, seen = -INFINITY, sum;
      int redo;
      f32x16 o[kBands];
      do {
        const bool loads = E4M3 || !late;
        constexpr int kStageLoads = E4M3 ? kSides * (CACHE == kCacheBlocks ? 2 : 1) : 2 * kWaveKeys * (D / 8) / 64;
        if (loads) {
          pages_of_tile(0);
          arrived();
#pragma unroll
          for (int g = 0; g < kGroups; ++g) tile_pages[1][g] = tile_pages[0][g];  // stage 0 of codes has values too, of no use
          pages_of_tile(1);
          load_stage(0);
          arrived();
          load_stage(1);
          if constexpr (E4M3) {
            pages_of_tile(2);
            loads_arrived<kStageLoads>();
            convert_stage(0);
            arrived();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the codes of stage 0 have been read
            if (2 <= n) load_stage(2);
          }
        }
        top = seen;
        sum = 0.0f;
#pragma unroll
        for (int b = 0; b < kBands; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
        interval_end<!E4M3>();
        if (threadIdx.x == 0) once_more = 0;  // every wave has read it by now

        u32x4 weights[2 * KT];
        f32x16 s[KT];
        // This lane's place in a tile of keys (key c of 32, chunk `half`) and in one of values (key 4 half + .. of
        // 16, its columns of 32). Other chunks and columns are the place with bits of it flipped, other keys are
        // further on by a constant, so that a tile's reads share a few addresses.
        const int l16 = lane & 15, value_key = 4 * half + (l16 >> 2), value_column = 16 * ((lane >> 4) & 1) + 4 * (l16 & 3);
        const uint32_t key_place = tile_byte<D>(c, half), value_place = tile_byte<D>(value_key, value_column / 8) + (value_column % 8) * 2;
        auto key_words = [&](uint32_t at, int st, int kt) { return lds_read<u32x4>((at ^ (st << 5)) + kt * 32 * D * 2); };
        // values of keys 16 kk + 4 half + 0 .. 3 and of those 8 further, column 32 b + lane % 32
        auto value_words = [&](uint32_t at, int kk, int b) {
          const uint32_t band = at ^ (b << 6);
          typedef __attribute__((address_space(3))) s16x4 *LdsWords;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsWords)(band + kk * 16 * D * 2));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsWords)((band ^ 32) + (kk * 16 + 8) * D * 2));
          const uint2 w0 = __builtin_bit_cast(uint2, lo), w1 = __builtin_bit_cast(uint2, hi);
          return u32x4{w0.x, w0.y, w1.x, w1.y};
        };
        auto product = [&](u32x4 a, u32x4 b, f32x16 acc) {
          return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
        };
        // Products of an interval: V^T P^T of tile i - 1 onto O^T (VALUES), then K Q^T of tile i (SCORES). Operands are
        // read from LDS kRing products ahead.
        auto products = [&](int i, auto with_values, auto with_scores) {
          constexpr bool VALUES = decltype(with_values)::value, SCORES = decltype(with_scores)::value;
          constexpr int kValues = VALUES ? 2 * KT * kBands : 0, kScores = SCORES ? kSteps * KT : 0;
          constexpr int kRing = VALUES && D < 256 ? 8 : 4, kKeyRing = 4;
          uint32_t value_at = VALUES ? values_at(i - 1) + value_place : 0, key_at = SCORES ? keys_at(i) + key_place : 0;
          asm volatile("" : "+v"(value_at), "+v"(key_at));  // or every address of both stages stays in a register
          u32x4 v[kRing], k[kKeyRing];
          if constexpr (VALUES) {
#pragma unroll
            for (int f = 0; f < kRing; ++f) v[f] = value_words(value_at, f / kBands, f % kBands);
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * kRing, 0);
#pragma unroll
            for (int f = 0; f < kValues; ++f) {
              o[f % kBands] = product(v[f % kRing], weights[f / kBands], o[f % kBands]);
              if (f + kRing < kValues) v[f % kRing] = value_words(value_at, (f + kRing) / kBands, (f + kRing) % kBands);
            }
          }
          if constexpr (SCORES) {
#pragma unroll
            for (int f = 0; f < kKeyRing; ++f) k[f] = key_words(key_at, f / KT, f % KT);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
              for (int e = 0; e < 16; ++e) s[kt][e] = 0.0f;
#pragma unroll
            for (int f = 0; f < kScores; ++f) {
              s[f % KT] = product(k[f % kKeyRing], qv[f / KT], s[f % KT]);
              if (f + kKeyRing < kScores) k[f % kKeyRing] = key_words(key_at, (f + kKeyRing) / KT, (f + kKeyRing) % KT);
            }
          }
          // the order: after the first reads, a product, then the reads that its operands' registers are free for
#pragma unroll
          for (int f = 0; f < kValues; ++f) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (f + kRing < kValues) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            else if (SCORES && f + kKeyRing >= kValues) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
          if constexpr (SCORES) {
            if constexpr (!VALUES) __builtin_amdgcn_sched_group_barrier(0x100, kKeyRing, 0);
#pragma unroll
            for (int f = 0; f < kScores; ++f) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              if (f + kKeyRing < kScores) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
          }
        };
        constexpr std::true_type kYes{};
        constexpr std::false_type kNo{};
        // positions of the wave's rows
        const int wave_first = pk.first_position + (wave * 32 < tokens * heads ? (wave * 32 * plan.token_of) >> 16 : 0);
        const int wave_last = pk.first_position + (wave * 32 + 31 < tokens * heads ? ((wave * 32 + 31) * plan.token_of) >> 16 : tokens - 1);
        auto softmax = [&](int i) {
          const int base = base_of(i);
          float z[16 * KT];
#pragma unroll
          for (int e = 0; e < 16 * KT; ++e) z[e] = s[e / 16][e % 16];
          if (base + kKeys - 1 > wave_first || (base <= wave_last - window && base + kKeys > sinks)) {
            // some row does not count some key: it counts those low < j <= to and j < sink (no short circuits: each
            // would be a branch)
            const int to = position - base - 4 * half, sink = sinks - base - 4 * half;
            const int low = static_cast<int>(static_cast<uint32_t>(to) - static_cast<uint32_t>(window));  // (of no use for to < 0)
#pragma unroll
            for (int e = 0; e < 16 * KT; ++e) {
              const int j = 32 * (e >> 4) + 8 * ((e >> 2) & 3) + (e & 3);
              const bool counts = (j <= to) & ((j > low) | (j < sink));
              z[e] = counts ? z[e] : -INFINITY;
            }
          }
          float most = z[0], other = z[1];
#pragma unroll
          for (int e = 2; e < 16 * KT; e += 2) most = fmaxf(most, z[e]), other = fmaxf(other, z[e + 1]);
          {
            const uint32_t a = __float_as_uint(fmaxf(most, other));
            const auto x = __builtin_amdgcn_permlane32_swap(a, a, false, false);
            most = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * factor;
          }
          seen = fmaxf(seen, most);
          top = top == -INFINITY ? most : top;
          const float from = top == -INFINITY ? 0.0f : top;
          float sums[4] = {sum, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int e = 0; e < 8 * KT; ++e) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(z[2 * e], factor, -from));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(z[2 * e + 1], factor, -from));
            const uint32_t w = pack_bf16(p0, p1);
            weights[e / 4][e % 4] = w;
            sums[e & 3] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), sums[e & 3], false);
          }
          sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
          for (int e = 0; e < 2 * KT; ++e) asm volatile("" : "+v"(weights[e]));  // here, not with the products
        };
        // Intervals of a wave, by its group: products of tile i (and of tile i - 1's values), softmax of tile i. Stage i
        // is read in the products i of both groups. Its place is free once the first group begins products i + 1,
        // for which the stage after has to be there: the first group then loads stage i + 3 into it, or both turn
        // the codes of stage i + 2 into it in their products i + 1 and load those of stage i + 4.
        // (Code of their own: where paths meet, the compiler waits for what either may have on its way.)
        auto tiles = [&](auto behind) {
          constexpr bool LATE = decltype(behind)::value, LOADS = !LATE || E4M3;
          // Converts stage i + 1, and loads stage i + 3: the first group behind softmax i, the second behind its
          // products i, or, where products are the longer part, behind the softmax before them.
          constexpr bool kEarly = E4M3 && LATE && D == 256;
          auto convert_next = [&](int i) {
            if (i + 1 <= n) {
              if (i + 2 <= n) {
                loads_arrived<kStageLoads>();
              } else {
                loads_arrived<0>();
              }
              convert_stage(i + 1);
            }
            if (i + 3 <= n) {
              asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the codes of stage i + 1 have been read
              load_stage(i + 3);
            }
          };
          if constexpr (LOADS) {
            pages_of_tile(E4M3 ? 3 : 2);
            arrived();
          }
          if constexpr (kEarly) convert_next(0);
          if constexpr (LATE) interval_end<false>();
          if constexpr (!LATE && !E4M3) {
            if (2 <= n) load_stage(2);
          }
          products(0, kNo, kYes);
          if constexpr (LATE && E4M3 && !kEarly) convert_next(0);
          interval_end<false>();
          for (int i = 0; i < n;) {
            if constexpr (LOADS && !(E4M3 && !LATE)) pages_of_tile(i + (E4M3 ? 4 : 3));
            softmax(i);
            if constexpr (!LATE && E4M3) {
              convert_next(i);
              pages_of_tile(i + 4);
            }
            if constexpr (LOADS) arrived();
            if constexpr (kEarly) convert_next(i + 1);
            if constexpr (E4M3 || LATE) {
              interval_end<false>();
            } else if (i + 2 <= n) {
              interval_end<true, kStageLoads>();
            } else {
              interval_end<true>();
            }
            ++i;
            if constexpr (!LATE && !E4M3) {
              if (i + 2 <= n) load_stage(i + 2);
            }
            products(i, kYes, kYes);  // behind the last tile's values, scores of no use
            if constexpr (LATE && E4M3 && !kEarly) convert_next(i);
            interval_end<false>();
          }
          if constexpr (!LATE) interval_end<false>();
        };
        if (late) {
          tiles(kYes);
        } else {
          tiles(kNo);
        }
        // 1: once more; 2: a page outside the cache
        const int after = outside ? 2 : __ballot(live && seen > top + kNear) != 0 ? 1 : 0;
        if (after != 0 && lane == 0) atomicOr(&once_more, after);
        interval_end<false>();
        redo = __builtin_amdgcn_readfirstlane(once_more);
      } while (redo == 1);
      if (redo >= 2) bad = true;

      const uint32_t sum_bits = __float_as_uint(sum);
      const auto both = __builtin_amdgcn_permlane32_swap(sum_bits, sum_bits, false, false);
      const float total = __uint_as_float(both[0]) + __uint_as_float(both[1]);
      const bool whole = k0 == 0 && k1 == pk.tiles;
      const float scale = whole ? (CACHE == kCacheE4m3 ? scales[Hkv + h] : 1.0f) / total : 1.0f;
      uint16_t *dst = out + static_cast<uint64_t>(row_at) * D;
      float *part = partial_of<D>(ws, prompt_slot(range, k0 > 0));
      float finite = total;  // a NaN once a value is not: x - x is then
#pragma unroll
      for (int b = 0; b < kBands; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) finite += o[b][e] - o[b][e];
      if (live && whole) {
#pragma unroll
        for (int b = 0; b < kBands; ++b)
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            // columns 2 e + 4 half .. and 2 e + 8 + 4 half ..: the lanes of a row trade for eight in a row each
            u32x4 w;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t lo = pack_bf16(o[b][e + 2 * k] * scale, o[b][e + 2 * k + 1] * scale);
              uint32_t hi = pack_bf16(o[b][e + 4 + 2 * k] * scale, o[b][e + 5 + 2 * k] * scale);
              if (total == 0.0f) lo = hi = 0;
              const auto x = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
              w[k] = x[0];
              w[2 + k] = x[1];
            }
            *reinterpret_cast<u32x4 *>(dst + 32 * b + 2 * e + 8 * half) = w;
          }
      } else if (live) {
#pragma unroll
        for (int b = 0; b < kBands; ++b)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<f32x4 *>(part + m * D + 32 * b + 2 * e + 4 * half) = f32x4{o[b][e], o[b][e + 1], o[b][e + 2], o[b][e + 3]};
        if (half == 0) {
          part[P::kRows * D + m] = top;
          part[P::kRows * D + P::kRows + m] = total;
        }
      }
      // A maximum of 2^29 or more is rounded by 16 or more, and a score, whose product is not, may be as far from it:
      // from 2^31 on, weights relative to it could all be zero.
      const bool coarse = !(fabsf(top) < 0x1p29f) && top != -INFINITY;
      if (__ballot(live && (!(finite < INFINITY) || coarse)) != 0 || redo >= 2) {
        const CarefulRow r = {q + static_cast<uint64_t>(row_at) * D, kc, vc, table, pk, k0, k1, h, position, factor};
        float acc[D / 2], careful_top, careful_sum;
        careful_row<D, CACHE>(d, r, flip, acc, careful_top, careful_sum);
        if (live) {
          for (int e = 0; e < D / 2; ++e) {
            const int column = half * (D / 2) + e;
            if (whole) {
              const float v = acc[e] * ((CACHE == kCacheE4m3 ? scales[Hkv + h] : 1.0f) / careful_sum);
              dst[column] = static_cast<uint16_t>(careful_sum == 0.0f ? 0u : f32_to_bf16(v));
            } else {
              part[m * D + column] = acc[e];
            }
          }
          if (!whole && half == 0) {
            part[P::kRows * D + m] = careful_top;
            part[P::kRows * D + P::kRows + m] = careful_sum;
          }
        }
      }
    }
    // the next pair
    if (pair.begin + pair.weight >= u1) break;
    pair.begin += pair.weight;
    if (++pair.x == pair.w.tiles) {
      pair.x = 0;
      if (++pair.head == plan.heads) {
        pair.head = 0;
        do ++pair.i;
        while (prefix[pair.i] == prefix[pair.i + 1]);
        pair.i = __builtin_amdgcn_readfirstlane(pair.i);
        read_prompt(d, plan, row_offsets, lengths, page_offsets, pair);
      }
    }
    pair.weight = weight_of(pair.w, pair.x);
  }
  if (bad) flag_error(error);
}

// Adds up the parts of the query tiles that were cut: the block of range b and slice k takes its
// part of the rows of a tile of which range b holds a part that is not its first. HBM bounds
// it where there are many parts: heads of 256, 512 of 2045 rows behind 2500 tokens 20 us for 105 MB, four
// prompts of up to 2039 rows of heads of 128 9 us, of which a launch that does nothing is 4.
template <int D, int CACHE>
LF_DEVICE void prefill_join(const uint8_t *attn, uint16_t *out, uint8_t *ws) {
  using P = Prompts<D>;
  __shared__ int slots[P::kBlocks], counted[4], own;
  const Desc &d = desc_of(attn);
  const int range = blockIdx.x / kJoinSlices, slice = blockIdx.x % kJoinSlices;
  const RangeStart tile = *start_of(ws, range);
  if (d.magic != kMagic || tile.weight == 0) return;
  auto cut = [&](int b) { return cut_of(b * tile.share, tile.begin, tile.weight, tile.tiles, cut_tiles(tile.share, P::kKeys)); };
  if (cut(range) == 0 || cut(range) >= cut(range + 1)) return;

  // the ranges with a part of the tile, in order
  const int first = static_cast<int>(tile.begin / tile.share);
  const int mine = first + static_cast<int>(threadIdx.x);
  const int from = cut(mine), to = cut(mine + 1);
  const bool some = mine < P::kBlocks && from < to;
  const uint64_t ballot = __ballot(some);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) counted[wave] = __popcll(ballot);
  __syncthreads();
  int at = __popcll(ballot & ((1ull << lane) - 1)), parts = 0;
  for (int k = 0; k < 4; ++k) {
    if (k < wave) at += counted[k];
    parts += counted[k];
  }
  if (some) slots[at] = prompt_slot(mine, from > 0);
  if (some && mine == range) own = at;
  __syncthreads();
  const int worker = (own - 1) * kJoinSlices + slice, workers = (parts - 1) * kJoinSlices;

  const int Hq = d.query_heads, head0 = tile.head0, heads = tile.heads, rows = tile.rows, row0 = tile.row0;
  const float vscale = CACHE == kCacheE4m3 ? reinterpret_cast<const float *>(attn + d.scale_offset)[d.kv_heads + tile.h] : 1.0f;
  constexpr int kQuads = D / 4;
  const int m0 = rows * worker / workers, m1 = rows * (worker + 1) / workers;
  struct Joined {
    f32x4 acc;
    float top, sum;
  };
  auto add = [](Joined &x, const f32x4 &v, float t, float l) {
    const float next = fmaxf(x.top, t), base = next == -INFINITY ? 0.0f : next;
    const float keep = __builtin_amdgcn_exp2f(x.top - base), f = __builtin_amdgcn_exp2f(t - base);
    x.acc = x.acc * keep + v * f;
    x.sum = x.sum * keep + l * f;
    x.top = next;
  };
  // The parts of a row that has an infinity, once more. (All parts so take 1 to 2 us more: 170 and 172 for 61 rows behind
  // 131010 tokens; this way they take what they did without it.)
  auto odd_values = [&](int quad) {
    Joined x = {{0.0f, 0.0f, 0.0f, 0.0f}, -INFINITY, 0.0f};
    for (int p = 0; p < parts; ++p) {
      const float *part = partial_of<D>(ws, slots[p]);
      const float t = part[P::kRows * D + quad / kQuads], next = fmaxf(x.top, t), base = next == -INFINITY ? 0.0f : next;
      const float keep = __builtin_amdgcn_exp2f(x.top - base), f = __builtin_amdgcn_exp2f(t - base);
      for (int e = 0; e < 4; ++e) x.acc[e] = weighted(x.acc[e], keep) + weighted(part[4 * quad + e], f);
      x.sum = x.sum * keep + part[P::kRows * D + P::kRows + quad / kQuads] * f;
      x.top = next;
    }
    return x;
  };
  auto finish = [&](int quad, Joined x) {
    const float some = (x.acc[0] + x.acc[1]) + (x.acc[2] + x.acc[3]);
    if (some != some) x = odd_values(quad);
    const int m = quad / kQuads, column = quad % kQuads * 4, token = (m * tile.token_of) >> 16;
    const float scale = vscale / x.sum;
    uint2 w = {pack_bf16(x.acc[0] * scale, x.acc[1] * scale), pack_bf16(x.acc[2] * scale, x.acc[3] * scale)};
    if (x.sum == 0.0f) w = {0u, 0u};
    *reinterpret_cast<uint2 *>(out + (static_cast<uint64_t>(row0 + token) * Hq + head0 + m - token * heads) * D + column) = w;
  };
  // Few parts: two of them at a time for four values of a thread. Many: eight groups of threads share them, and
  // their sums are added up in their order.
  constexpr Joined kNone = {{0.0f, 0.0f, 0.0f, 0.0f}, -INFINITY, 0.0f};
  if (parts <= 4) {
    constexpr int kAtOnce = 4;
    for (int q0 = m0 * kQuads + static_cast<int>(threadIdx.x); q0 < m1 * kQuads; q0 += kAtOnce * 256) {
      Joined x[kAtOnce] = {kNone, kNone, kNone, kNone};
      for (int p0 = 0; p0 < parts; p0 += 2) {
        f32x4 v[2][kAtOnce];
        float t[2][kAtOnce], l[2][kAtOnce];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const float *part = partial_of<D>(ws, slots[p0 + p < parts ? p0 + p : p0]);
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) {
            const int quad = q0 + k * 256 < m1 * kQuads ? q0 + k * 256 : q0;
            v[p][k] = *reinterpret_cast<const f32x4 *>(part + 4 * quad);
            t[p][k] = part[P::kRows * D + quad / kQuads];
            l[p][k] = part[P::kRows * D + P::kRows + quad / kQuads];
          }
        }
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k)
            if (p0 + p < parts) add(x[k], v[p][k], t[p][k], l[p][k]);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k)
        if (q0 + k * 256 < m1 * kQuads) finish(q0 + k * 256, x[k]);
    }
  } else {
    constexpr int kGroups = 8, kItems = 256 / kGroups, kAtOnce = 4;
    __shared__ Joined joined[kGroups][kItems];
    const int g = static_cast<int>(threadIdx.x) / kItems, item = static_cast<int>(threadIdx.x) % kItems;
    for (int q0 = m0 * kQuads; q0 < m1 * kQuads; q0 += kItems) {
      const int quad = q0 + item < m1 * kQuads ? q0 + item : q0;
      Joined x = kNone;
      for (int p0 = g; p0 < parts; p0 += kAtOnce * kGroups) {
        f32x4 v[kAtOnce];
        float t[kAtOnce], l[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const float *part = partial_of<D>(ws, slots[p0 + k * kGroups < parts ? p0 + k * kGroups : p0]);
          v[k] = *reinterpret_cast<const f32x4 *>(part + 4 * quad);
          t[k] = part[P::kRows * D + quad / kQuads];
          l[k] = part[P::kRows * D + P::kRows + quad / kQuads];
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (p0 + k * kGroups < parts) add(x, v[k], t[k], l[k]);
      }
      joined[g][item] = x;
      __syncthreads();
      if (g == 0) {
        for (int k = 1; k < kGroups; ++k) add(x, joined[k][item].acc, joined[k][item].top, joined[k][item].sum);
        if (q0 + item < m1 * kQuads) finish(quad, x);
      }
      __syncthreads();
    }
  }
}

}  // namespace attn

#define LF_ATTN_PREFILL(D, TYPE, CACHE)                                                                        \
  extern "C" __global__ __launch_bounds__(512, 2) void lf_attn_prefill_d##D##_##TYPE(                          \
      const int32_t *__restrict__ counts, const int32_t *__restrict__ row_offsets,                             \
      const int32_t *__restrict__ lengths, const int32_t *__restrict__ page_offsets,                           \
      const int32_t *__restrict__ page_indices, const uint8_t *__restrict__ desc,                              \
      const uint16_t *__restrict__ q, uint16_t *__restrict__ out, const uint8_t *__restrict__ kc,              \
      const uint8_t *__restrict__ vc, uint8_t *__restrict__ ws) {                                              \
    attn::prefill<D, attn::CACHE>(counts, row_offsets, lengths, page_offsets, page_indices, desc, q, out, kc,  \
                                  vc, ws);                                                                     \
  }                                                                                                            \
  extern "C" __global__ __launch_bounds__(256) void lf_attn_prefill_join_d##D##_##TYPE(                        \
      const uint8_t *__restrict__ desc, uint16_t *__restrict__ out, uint8_t *__restrict__ ws) {                \
    attn::prefill_join<D, attn::CACHE>(desc, out, ws);                                                         \
  }
LF_ATTN_PREFILL(64, bf16, kCacheBf16)
LF_ATTN_PREFILL(128, bf16, kCacheBf16)
LF_ATTN_PREFILL(256, bf16, kCacheBf16)
LF_ATTN_PREFILL(64, e4m3, kCacheE4m3)
LF_ATTN_PREFILL(128, e4m3, kCacheE4m3)
LF_ATTN_PREFILL(256, e4m3, kCacheE4m3)
LF_ATTN_PREFILL(64, e4m3_blocks, kCacheBlocks)
LF_ATTN_PREFILL(128, e4m3_blocks, kCacheBlocks)
LF_ATTN_PREFILL(256, e4m3_blocks, kCacheBlocks)
