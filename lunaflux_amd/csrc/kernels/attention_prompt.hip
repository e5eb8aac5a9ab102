// attention_prompt.hip - attention of the rows of prompts, or of parts of them, over the
// paged key / value cache (the attention section of include/lunaflux_fp8.h).
#include "device_common.h"

#include "attention_index.h"

namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// One pass over the keys with the running maximum and sum of each row's softmax. A block holds a
// query tile (attention_index.h, QueryTile) of which each wave has kRowTiles tiles of 32 rows in
// registers, as the B operand of S^T = K Q^T; that leaves a lane the scores of one row, so
// its statistics are lane values, and 16 weights per 32 keys in the order of the B operand of
// O^T = V^T P^T. Key and value tiles go through LDS, shared by the waves; values are read from it
// transposed.
// Blocks are dealt equal ranges of the step's weight (attention_index.h); a query tile cut
// between ranges leaves fp32 partial results, which a second launch adds up in their order.
template <int D>
struct Prompts {
  static constexpr int kWaves = 4, kBlocks = 256;
  static constexpr int kRowTiles = D == 256 ? 1 : 2;
  static constexpr int kRows = 32 * kRowTiles * kWaves;
  static constexpr int kKeys = D == 256 ? 32 : 64;
  static constexpr int kKeyTiles = kKeys / 32;
  static constexpr int kTileBytes = kKeys * D * 2;
  static constexpr int kFloats = kRows * (D + 2);  // of a partial result: sums, maxima, weight sums
};
constexpr int kJoinSlices = 4;

// The step's prompts, their weights added up in LDS.
struct PromptPlan {
  int n, rows;
  QueryTile tile;
  int64_t heads, total, share;  // heads: pairs of key head and part of its group
};

template <int D>
LF_DEVICE PromptPlan plan_of(const Desc &d, const int32_t *counts, const int32_t *row_offsets, const int32_t *lengths,
                             const int32_t *page_offsets, int64_t *prefix, bool &bad) {
  __shared__ int64_t wave_total[4], wave_rows[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  PromptPlan plan;
  plan.rows = live_rows(counts, d.max_tokens);
  plan.n = decoded_of(d, 0, counts[0], counts[2]).n;
  plan.tile = query_tile_of(d, Prompts<D>::kRows);
  plan.heads = static_cast<int64_t>(d.kv_heads) * plan.tile.subs;
  int64_t carry = 0, rows = 0;
  for (int base = 0; base < plan.n; base += 256) {
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
    for (int k = 0; k < 4; ++k) {
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
  int i, x;
  int64_t head, begin, weight;
  Prompt p;
  Weights w;
};
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
  pair.head = (u - first) / each;
  const int64_t within = u - first - pair.head * each;
  pair.x = __builtin_amdgcn_readfirstlane(tile_at(pair.w, within));
  pair.begin = first + pair.head * each + weight_before(pair.w, pair.x);
  pair.weight = weight_of(pair.w, pair.x);
  return pair;
}

LF_DEVICE uint32_t pack_bf16(float a, float b) { return f32_to_bf16(a) | (f32_to_bf16(b) << 16); }

// Byte of 16-byte chunk `chunk` of a key's row in an LDS tile of rows of D bf16 values.
template <int D>
LF_DEVICE uint32_t tile_byte(int key, int chunk) {
  return static_cast<uint32_t>(key * D * 2 + ((chunk ^ (chunk_swizzle(key & 15) & (D / 8 - 1))) << 4));
}

// A bf16 pair with an infinity or NaN among the two, and its values: finite ones kept and
// others zero, or +infinity, -infinity, NaN as 1, 256, 65536 and finite ones zero.
LF_DEVICE bool odd_half(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }
LF_DEVICE uint32_t finite_pair(uint32_t w) {
  return (odd_half(w) ? 0u : w & 0xffffu) | (odd_half(w >> 16) ? 0u : w & 0xffff0000u);
}
LF_DEVICE uint32_t odd_code(uint32_t h) {
  return !odd_half(h) ? 0u : (h & 0x7fu) != 0 ? 0x4780u : (h & 0x8000u) != 0 ? 0x4380u : 0x3f80u;
}
LF_DEVICE uint32_t odd_pair(uint32_t w) { return odd_code(w & 0xffffu) | (odd_code(w >> 16) << 16); }
LF_DEVICE bool odd_word(uint32_t w) { return odd_half(w) || odd_half(w >> 16); }

LF_DEVICE u32x4 finite4(u32x4 w) {
  return u32x4{finite_pair(w[0]), finite_pair(w[1]), finite_pair(w[2]), finite_pair(w[3])};
}
LF_DEVICE u32x4 odd4(u32x4 w) { return u32x4{odd_pair(w[0]), odd_pair(w[1]), odd_pair(w[2]), odd_pair(w[3])}; }

// Partial results, their maxima and their weight sums in the workspace.
template <int D>
LF_DEVICE float *partial_of(uint8_t *ws, int slot) {
  return reinterpret_cast<float *>(ws + 256) + static_cast<uint64_t>(slot) * Prompts<D>::kFloats;
}

template <int D, int CACHE>
LF_DEVICE void prefill(const int32_t *counts, const int32_t *row_offsets, const int32_t *lengths,
                       const int32_t *page_offsets, const int32_t *page_indices, const uint8_t *attn,
                       const uint16_t *q, uint16_t *out, const uint8_t *kc, const uint8_t *vc, uint8_t *ws) {
  using P = Prompts<D>;
  constexpr int RT = P::kRowTiles, KT = P::kKeyTiles, kKeys = P::kKeys, kSteps = D / 16, kBands = D / 32;
  constexpr bool E4M3 = CACHE != kCacheBf16;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const Desc &d = desc_of(attn);
  if (d.magic != kMagic) return;
  int *error = reinterpret_cast<int *>(ws);
  int64_t *prefix = reinterpret_cast<int64_t *>(lds);
  uint8_t *keys = lds + ((static_cast<uint32_t>(d.max_sequences) + 1) / 2 * 16 + 16), *values = keys + P::kTileBytes;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, half = lane >> 5;
  bool bad = false;
  const PromptPlan plan = plan_of<D>(d, counts, row_offsets, lengths, page_offsets, prefix, bad);
  const int range = range_of_block(blockIdx.x, P::kBlocks);
  const int64_t u0 = range * plan.share, u1 = u0 + plan.share < plan.total ? u0 + plan.share : plan.total;
  if (bad) flag_error(error);
  if (u0 >= u1) return;

  const int Hq = d.query_heads, Hkv = d.kv_heads, group = Hq / Hkv;
  const int shift = __builtin_ctz(d.page_size), slot_mask = d.page_size - 1;
  const float *scales = reinterpret_cast<const float *>(attn + d.scale_offset);
  const bool flip = d.softmax_scale < 0.0f;
  const int window = d.window > 0 ? d.window : INT32_MAX, sinks = d.sinks;

  PromptPair pair = pair_at(d, plan, row_offsets, lengths, page_offsets, prefix, u0);
  for (;;) {
    const PromptKeys pk = keys_of(d, plan.tile, pair.p, pair.x, kKeys);
    const int k0 = cut_of(u0, pair.begin, pair.weight, pk.tiles), k1 = cut_of(u1, pair.begin, pair.weight, pk.tiles);
    if (k0 < k1) {
      const int h = static_cast<int>(pair.head / plan.tile.subs), sub = static_cast<int>(pair.head - static_cast<int64_t>(h) * plan.tile.subs);
      const int tokens = pk.last - pk.first_position + 1;
      const int head0 = h * group + sub * plan.tile.heads;
      const int heads = group - sub * plan.tile.heads < plan.tile.heads ? group - sub * plan.tile.heads : plan.tile.heads;
      const int live_rows_here = tokens * heads;
      const int row0 = pair.p.row + pair.x * plan.tile.tokens;
      const int32_t *table = page_indices + pair.p.entry;
      // (a scale of zero as one that leaves -infinity, a masked score, what it is)
      const float factor = fmaxf(fabsf(d.softmax_scale) * 1.44269504088896341f * (CACHE == kCacheE4m3 ? scales[h] : 1.0f), 0x1p-126f);

      // this lane's rows: query operands, positions, statistics
      u32x4 qv[RT][kSteps];
      int position[RT];
      uint32_t row_at[RT];  // row and head of q and out, or none
      float top[RT], sum[RT];
      f32x16 o[RT][kBands];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int m = (wave * RT + rt) * 32 + c;
        const int token = m / heads, head = m - token * heads;
        const bool live = m < live_rows_here;
        position[rt] = live ? pk.first_position + token : pk.first_position;
        row_at[rt] = live ? static_cast<uint32_t>(row0 + token) * Hq + head0 + head : ~0u;
        const uint16_t *src = q + static_cast<uint64_t>(live ? row_at[rt] : static_cast<uint32_t>(row0) * Hq + head0) * D + 8 * half;
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
          u32x4 w = *reinterpret_cast<const u32x4 *>(src + 16 * t);
          if (flip) w ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
          qv[rt][t] = w;
        }
        top[rt] = -INFINITY;
        sum[rt] = 0.0f;
#pragma unroll
        for (int b = 0; b < kBands; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[rt][b][i] = 0.0f;
      }

      const int page_first = pk.lo >> shift, page_end = (pk.last >> shift) + 1, sink_end = (pk.sink + slot_mask) >> shift;
      for (int t = k0; t < k1; ++t) {
        const int base = kKeys * (t < pk.sink_tiles ? t : t + pk.first - pk.sink_tiles);
        // pages of the tile's groups of eight keys
        int page = 0;
        bool in = true;
        if (lane < kKeys / 8) {
          page = table[sink_entry_of(sink_end, page_first, page_end, shift, base + 8 * lane)];
          in = static_cast<uint32_t>(page) < static_cast<uint32_t>(d.pages);
          page = in ? page : 0;
        }
        const uint32_t outside = static_cast<uint32_t>(__ballot(!in));
        if (outside != 0) bad = true;
        constexpr int kChunks = D * (E4M3 ? 1 : 2) / 16;  // 16-byte chunks of a key in the cache
        bool odd = false;
        __syncthreads();  // the tile before has been read
        for (int side = 0; side < 2; ++side) {
#pragma unroll
          for (int i = 0; i < kKeys * kChunks / 256; ++i) {
            const int id = i * 256 + static_cast<int>(threadIdx.x), key = id / kChunks, chunk = id % kChunks;
            const int p = __shfl(page, key >> 3);
            const int j = base + key < pk.last ? base + key : pk.last, slot = j & slot_mask;
            const uint8_t *src = (side == 0 ? kc : vc) + cache_byte<E4M3>(d, p, h, slot) + 16 * chunk;
            const u32x4 w = *reinterpret_cast<const u32x4 *>(src);
            uint8_t *dst = side == 0 ? keys : values;
            if constexpr (E4M3) {
              float scale = 1.0f;
              if constexpr (CACHE == kCacheBlocks) {
                scale = reinterpret_cast<const float *>((side == 0 ? kc : vc) + d.block_scales)[scale_index(d, p, slot, h)];
              }
              uint32_t b[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                b[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w[e]), scale, false));
                b[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w[e]), scale, true));
                odd |= odd_word(b[2 * e]) | odd_word(b[2 * e + 1]);
              }
              *reinterpret_cast<u32x4 *>(dst + tile_byte<D>(key, 2 * chunk)) = u32x4{b[0], b[1], b[2], b[3]};
              *reinterpret_cast<u32x4 *>(dst + tile_byte<D>(key, 2 * chunk + 1)) = u32x4{b[4], b[5], b[6], b[7]};
            } else {
              odd |= odd_word(w[0]) | odd_word(w[1]) | odd_word(w[2]) | odd_word(w[3]);
              *reinterpret_cast<u32x4 *>(dst + tile_byte<D>(key, chunk)) = w;
            }
          }
        }
        odd = __syncthreads_or(odd) != 0;

        // whether the row at `at` counts the tile's key `within` (no short circuits: each would be a branch)
        auto counts_key = [&](int at, int within) {
          const int j = base + within, low = at - window;
          return static_cast<int>(j <= at) & (static_cast<int>(j > low) | static_cast<int>(j < sinks)) &
                 static_cast<int>(((outside >> (within >> 3)) & 1) == 0);
        };
        const bool masked = base + kKeys - 1 > pk.first_position || outside != 0 ||
                            (base <= pk.last - window && base + kKeys > sinks);
        f32x16 s[RT][KT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[rt][kt][i] = 0.0f;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const bf16x8 a = *reinterpret_cast<const bf16x8 *>(keys + tile_byte<D>(32 * kt + c, 2 * st + half));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              s[rt][kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, qv[rt][st]), s[rt][kt], 0, 0, 0);
          }
        }
        u32x4 weights[RT][2 * KT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          if (masked) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                s[rt][kt][i] = counts_key(position[rt], 32 * kt + 8 * (i >> 2) + 4 * half + (i & 3)) != 0 ? s[rt][kt][i] : -INFINITY;
              }
          }
          float most = s[rt][0][0];
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, s[rt][kt][i]);
          {
            const uint32_t a = __float_as_uint(most);
            const auto x = __builtin_amdgcn_permlane32_swap(a, a, false, false);
            most = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
          }
          const float next = fmaxf(top[rt], most * factor), from = next == -INFINITY ? 0.0f : next;
          const float shrink = __builtin_amdgcn_exp2f(top[rt] - from);
          top[rt] = next;
          sum[rt] *= shrink;
#pragma unroll
          for (int b = 0; b < kBands; ++b) o[rt][b] *= shrink;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][kt][2 * i], factor, -from));
              const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][kt][2 * i + 1], factor, -from));
              const uint32_t w = pack_bf16(p0, p1);
              weights[rt][2 * kt + i / 4][i % 4] = w;
              sum[rt] += __uint_as_float(w << 16) + __uint_as_float(w & 0xffff0000u);
            }
          }
        }
        // values of keys 16 kk + 4 half + 0 .. 3 and of those 8 further, column 32 b + lane % 32
        auto values_at = [&](int kk, int b) {
          const int l16 = lane & 15, key = 16 * kk + 4 * half + (l16 >> 2);
          const int column = 32 * b + 16 * ((lane >> 4) & 1) + 4 * (l16 & 3);
          typedef __attribute__((address_space(3))) s16x4 *LdsWords;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsWords)(values + tile_byte<D>(key, column / 8) + (column % 8) * 2));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsWords)(values + tile_byte<D>(key + 8, column / 8) + (column % 8) * 2));
          const uint2 w0 = __builtin_bit_cast(uint2, lo), w1 = __builtin_bit_cast(uint2, hi);
          return u32x4{w0.x, w0.y, w1.x, w1.y};
        };
        if (odd) {
          // Infinities and NaN among the values: a row that does not count their key, or gives it a weight that
          // is zero in fp32, would take zero times those, which is NaN. Products of zeros and ones count the infinities and NaN that a row does count; they go to
          // its sum by themselves, and the tile keeps its finite values.
#pragma unroll
          for (int b = 0; b < kBands; ++b)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              f32x16 found;
#pragma unroll
              for (int i = 0; i < 16; ++i) found[i] = 0.0f;
#pragma unroll 1
              for (int kk = 0; kk < 2 * KT; ++kk) {
                uint32_t seen[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int within = 16 * kk + 8 * (i >> 1) + 4 * half + 2 * (i & 1);
                  seen[i] = 0x3f80u * counts_key(position[rt], within) + 0x3f800000u * counts_key(position[rt], within + 1);
                }
                found = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, odd4(values_at(kk, b))),
                                                                __builtin_bit_cast(bf16x8, u32x4{seen[0], seen[1], seen[2], seen[3]}), found, 0, 0, 0);
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int n = static_cast<int>(found[i]), plus = n & 255, minus = (n >> 8) & 255;
                if (n != 0) o[rt][b][i] += n >= 65536 || (plus != 0 && minus != 0) ? __builtin_nanf("") : plus != 0 ? INFINITY : -INFINITY;
              }
            }
          __syncthreads();
          for (int i = threadIdx.x; i < P::kTileBytes / 16; i += 256) {
            u32x4 *w = reinterpret_cast<u32x4 *>(values) + i;
            *w = finite4(*w);
          }
          __syncthreads();
        }
#pragma unroll
        for (int b = 0; b < kBands; ++b) {
#pragma unroll
          for (int kk = 0; kk < 2 * KT; ++kk) {
            const bf16x8 a = __builtin_bit_cast(bf16x8, values_at(kk, b));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              o[rt][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, weights[rt][kk]), o[rt][b], 0, 0, 0);
          }
        }
      }

#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const uint32_t a = __float_as_uint(sum[rt]);
        const auto x = __builtin_amdgcn_permlane32_swap(a, a, false, false);
        const float total = __uint_as_float(x[0]) + __uint_as_float(x[1]);
        if (row_at[rt] == ~0u) continue;
        if (k0 == 0 && k1 == pk.tiles) {
          const float scale = (CACHE == kCacheE4m3 ? scales[Hkv + h] : 1.0f) / total;
          uint16_t *dst = out + static_cast<uint64_t>(row_at[rt]) * D + 4 * half;
#pragma unroll
          for (int b = 0; b < kBands; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              uint2 w = {pack_bf16(o[rt][b][i] * scale, o[rt][b][i + 1] * scale), pack_bf16(o[rt][b][i + 2] * scale, o[rt][b][i + 3] * scale)};
              if (total == 0.0f) w = {0u, 0u};
              *reinterpret_cast<uint2 *>(dst + 32 * b + 2 * i) = w;
            }
        } else {
          float *part = partial_of<D>(ws, prompt_slot(range, k0 > 0));
          const int m = (wave * RT + rt) * 32 + c;
#pragma unroll
          for (int b = 0; b < kBands; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<f32x4 *>(part + m * D + 32 * b + 2 * i + 4 * half) = f32x4{o[rt][b][i], o[rt][b][i + 1], o[rt][b][i + 2], o[rt][b][i + 3]};
          if (half == 0) {
            part[P::kRows * D + m] = top[rt];
            part[P::kRows * D + P::kRows + m] = total;
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
// part of the rows of a tile of which range b holds a part that is not its first.
template <int D, int CACHE>
LF_DEVICE void prefill_join(const int32_t *counts, const int32_t *row_offsets, const int32_t *lengths,
                            const int32_t *page_offsets, const uint8_t *attn, uint16_t *out, uint8_t *ws) {
  using P = Prompts<D>;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int slots[P::kBlocks], counted[4], own;
  const Desc &d = desc_of(attn);
  if (d.magic != kMagic) return;
  int64_t *prefix = reinterpret_cast<int64_t *>(lds);
  bool bad = false;  // reported by the launch before
  const PromptPlan plan = plan_of<D>(d, counts, row_offsets, lengths, page_offsets, prefix, bad);
  const int range = blockIdx.x / kJoinSlices, slice = blockIdx.x % kJoinSlices;
  const int64_t u = range * plan.share;
  if (range == 0 || u >= plan.total) return;
  const PromptPair pair = pair_at(d, plan, row_offsets, lengths, page_offsets, prefix, u);
  const PromptKeys pk = keys_of(d, plan.tile, pair.p, pair.x, P::kKeys);
  auto cut = [&](int b) { return cut_of(b * plan.share, pair.begin, pair.weight, pk.tiles); };
  if (cut(range) == 0 || cut(range) >= cut(range + 1)) return;

  // the ranges with a part of the tile, in order
  const int first = static_cast<int>(pair.begin / plan.share);
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

  const int Hq = d.query_heads, group = Hq / d.kv_heads;
  const int h = static_cast<int>(pair.head / plan.tile.subs), sub = static_cast<int>(pair.head - static_cast<int64_t>(h) * plan.tile.subs);
  const int head0 = h * group + sub * plan.tile.heads;
  const int heads = group - sub * plan.tile.heads < plan.tile.heads ? group - sub * plan.tile.heads : plan.tile.heads;
  const int rows = (pk.last - pk.first_position + 1) * heads;
  const int row0 = pair.p.row + pair.x * plan.tile.tokens;
  const float vscale = CACHE == kCacheE4m3 ? reinterpret_cast<const float *>(attn + d.scale_offset)[d.kv_heads + h] : 1.0f;
  constexpr int kQuads = D / 4;
  const int m0 = rows * worker / workers, m1 = rows * (worker + 1) / workers;
  for (int i = m0 * kQuads + static_cast<int>(threadIdx.x); i < m1 * kQuads; i += 256) {
    const int m = i / kQuads, column = i % kQuads * 4;
    float top = -INFINITY, sum = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < parts; ++p) {
      const float *part = partial_of<D>(ws, slots[p]);
      const f32x4 v = *reinterpret_cast<const f32x4 *>(part + m * D + column);
      const float t = part[P::kRows * D + m], l = part[P::kRows * D + P::kRows + m];
      const float next = fmaxf(top, t), base = next == -INFINITY ? 0.0f : next;
      const float keep = __builtin_amdgcn_exp2f(top - base), f = __builtin_amdgcn_exp2f(t - base);
      acc = acc * keep + v * f;
      sum = sum * keep + l * f;
      top = next;
    }
    const float scale = vscale / sum;
    uint2 w = {pack_bf16(acc[0] * scale, acc[1] * scale), pack_bf16(acc[2] * scale, acc[3] * scale)};
    if (sum == 0.0f) w = {0u, 0u};
    const int token = m / heads;
    *reinterpret_cast<uint2 *>(out + (static_cast<uint64_t>(row0 + token) * Hq + head0 + m - token * heads) * D + column) = w;
  }
}

}  // namespace attn

#define LF_ATTN_PREFILL(D, TYPE, CACHE)                                                                        \
  extern "C" __global__ __launch_bounds__(256, 1) void lf_attn_prefill_d##D##_##TYPE(                          \
      const int32_t *__restrict__ counts, const int32_t *__restrict__ row_offsets,                             \
      const int32_t *__restrict__ lengths, const int32_t *__restrict__ page_offsets,                           \
      const int32_t *__restrict__ page_indices, const uint8_t *__restrict__ desc,                              \
      const uint16_t *__restrict__ q, uint16_t *__restrict__ out, const uint8_t *__restrict__ kc,              \
      const uint8_t *__restrict__ vc, uint8_t *__restrict__ ws) {                                              \
    attn::prefill<D, attn::CACHE>(counts, row_offsets, lengths, page_offsets, page_indices, desc, q, out, kc,  \
                                  vc, ws);                                                                     \
  }                                                                                                            \
  extern "C" __global__ __launch_bounds__(256) void lf_attn_prefill_join_d##D##_##TYPE(                        \
      const int32_t *__restrict__ counts, const int32_t *__restrict__ row_offsets,                             \
      const int32_t *__restrict__ lengths, const int32_t *__restrict__ page_offsets,                           \
      const uint8_t *__restrict__ desc, uint16_t *__restrict__ out, uint8_t *__restrict__ ws) {                \
    attn::prefill_join<D, attn::CACHE>(counts, row_offsets, lengths, page_offsets, desc, out, ws);             \
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
