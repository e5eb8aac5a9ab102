// attention.hip - the steps between the QKV and the output projection over a
// paged key / value cache (the attention section of include/lunaflux_fp8.h):
// per-head norm, rotary positions and cache append in one pass over the packed
// rows, and attention of one new token per sequence.
#include "device_common.h"

#include "attention_index.h"

namespace attn {

LF_DEVICE const Desc &desc_of(const uint8_t *region) { return *reinterpret_cast<const Desc *>(region); }

LF_DEVICE void flag_error(int *word) { __hip_atomic_store(word, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// ---- norm, rotation, append ---------------------------------------------------

LF_DEVICE u32x4 bf16x8_of(const float *v) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = f32_to_bf16(v[2 * i]) | (f32_to_bf16(v[2 * i + 1]) << 16);
  return w;
}

// x / scale cut to the e4m3 range, a NaN kept.
LF_DEVICE float e4m3_range(float x, float inv_scale) {
  const float v = x * inv_scale;
  return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f);
}
LF_DEVICE uint2 e4m3x8_of(const float *v, float inv_scale) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(v[4 * i], inv_scale), e4m3_range(v[4 * i + 1], inv_scale), 0,
                                            false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(v[4 * i + 2], inv_scale), e4m3_range(v[4 * i + 3], inv_scale), p,
                                        true);
    w[i] = static_cast<uint32_t>(p);
  }
  return make_uint2(w[0], w[1]);
}

// The sequence of a row: the number of sequences that end at or before it.
LF_DEVICE int sequence_of(const int32_t *row_offsets, int sequences, int row) {
  int s = 0;
  for (int base = 0; base < sequences; base += 64) {
    const int i = base + (threadIdx.x & 63);
    const bool before = i < sequences && row_offsets[i + 1] <= row;
    s += __popcll(__ballot(before));
  }
  return s;
}

// One block per row, D / 16 lanes per head: a lane holds the 16 values
// [o0, o0 + 8) and [o1, o1 + 8) of its head, which are eight whole rotary
// pairs, so the rotation needs no exchange and every load and store is 16
// bytes.
template <bool E4M3>
LF_DEVICE void qk_norm_rope(const int32_t *counts, const int32_t *positions, const int32_t *row_offsets,
                            const int32_t *lengths, const int32_t *page_offsets, const int32_t *page_indices,
                            const uint8_t *attn, const uint16_t *qkv, const uint16_t *gq, const uint16_t *gk,
                            uint16_t *q, uint8_t *kc, uint8_t *vc, int *status) {
  __shared__ float2 turn[128];
  const Desc &d = desc_of(attn);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int row = blockIdx.x;
  if (row >= rows) return;
  int sequences = counts[2];
  sequences = sequences < 0 ? 0 : sequences > d.max_sequences ? d.max_sequences : sequences;
  const int s = sequence_of(row_offsets, sequences, row);
  if (s >= sequences || row < row_offsets[0]) return;

  const int R = d.rotary_dim;
  if (static_cast<int>(threadIdx.x) < R / 2) {
    const int i = threadIdx.x;
    const double *turns = reinterpret_cast<const double *>(attn + d.turns_offset);
    const int32_t *axis = reinterpret_cast<const int32_t *>(attn + d.axis_offset);
    const double t = static_cast<double>(positions[row * d.axes + axis[i]]) * turns[i];
    float sin_t, cos_t;
    sincospif(static_cast<float>(2.0 * (t - rint(t))), &sin_t, &cos_t);
    turn[i] = make_float2(cos_t, sin_t);
  }
  __syncthreads();

  const Place place = place_of(d, row_offsets, lengths, page_offsets, page_indices, s, row);
  if (place.page < 0 && threadIdx.x == 0) flag_error(status);

  const int D = d.head_dim, lanes = D >> 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int j = lane & (lanes - 1);
  const bool turned = 16 * j < R;
  const bool half = d.pairing == 0 && turned;
  const int o0 = half ? 8 * j : 16 * j;
  const int o1 = half ? R / 2 + 8 * j : 16 * j + 8;
  float c[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 t = turned ? turn[8 * j + e] : make_float2(1.0f, 0.0f);
    c[e] = t.x;
    sn[e] = t.y;
  }
  const int Hq = d.query_heads, Hkv = d.kv_heads, heads = Hq + 2 * Hkv;
  const int per_wave = 64 / lanes;
  const float *scales = reinterpret_cast<const float *>(attn + d.scale_offset);
  for (int base = wave * per_wave; base < heads; base += 4 * per_wave) {
    const int h = base + lane / lanes;
    if (h >= heads) continue;
    const uint16_t *src = qkv + (static_cast<uint64_t>(row) * heads + h) * D;
    const u32x4 w0 = *reinterpret_cast<const u32x4 *>(src + o0);
    const u32x4 w1 = *reinterpret_cast<const u32x4 *>(src + o1);
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[2 * i] = bf16_to_f32(w0[i] & 0xffffu);
      a[2 * i + 1] = bf16_to_f32(w0[i] >> 16);
      b[2 * i] = bf16_to_f32(w1[i] & 0xffffu);
      b[2 * i + 1] = bf16_to_f32(w1[i] >> 16);
    }
    if (h < Hq + Hkv) {
      if (d.norm) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + b[e] * b[e];
        for (int m = 1; m < lanes; m <<= 1) ss += __shfl_xor(ss, m);
        const float inv = 1.0f / __builtin_sqrtf(ss / static_cast<float>(D) + d.norm_epsilon);
        const uint16_t *g = h < Hq ? gq : gk;
        const u32x4 g0 = *reinterpret_cast<const u32x4 *>(g + o0);
        const u32x4 g1 = *reinterpret_cast<const u32x4 *>(g + o1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[2 * i] *= inv * bf16_to_f32(g0[i] & 0xffffu);
          a[2 * i + 1] *= inv * bf16_to_f32(g0[i] >> 16);
          b[2 * i] *= inv * bf16_to_f32(g1[i] & 0xffffu);
          b[2 * i + 1] *= inv * bf16_to_f32(g1[i] >> 16);
        }
      }
      if (turned) {
        if (half) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = a[e], y = b[e];
            a[e] = x * c[e] - y * sn[e];
            b[e] = y * c[e] + x * sn[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = a[2 * e], y = a[2 * e + 1];
            a[2 * e] = x * c[e] - y * sn[e];
            a[2 * e + 1] = y * c[e] + x * sn[e];
            x = b[2 * e];
            y = b[2 * e + 1];
            b[2 * e] = x * c[4 + e] - y * sn[4 + e];
            b[2 * e + 1] = y * c[4 + e] + x * sn[4 + e];
          }
        }
      }
    }
    if (h < Hq) {
      uint16_t *dst = q + (static_cast<uint64_t>(row) * Hq + h) * D;
      *reinterpret_cast<u32x4 *>(dst + o0) = bf16x8_of(a);
      *reinterpret_cast<u32x4 *>(dst + o1) = bf16x8_of(b);
    } else if (place.page >= 0) {
      const bool value = h >= Hq + Hkv;
      const int kh = h - Hq - (value ? Hkv : 0);
      uint8_t *dst = (value ? vc : kc) + cache_byte<E4M3>(d, place.page, kh, place.slot);
      if constexpr (E4M3) {
        const float inv_scale = 1.0f / scales[(value ? Hkv : 0) + kh];
        *reinterpret_cast<uint2 *>(dst + o0) = e4m3x8_of(a, inv_scale);
        *reinterpret_cast<uint2 *>(dst + o1) = e4m3x8_of(b, inv_scale);
      } else {
        *reinterpret_cast<u32x4 *>(dst + 2 * o0) = bf16x8_of(a);
        *reinterpret_cast<u32x4 *>(dst + 2 * o1) = bf16x8_of(b);
      }
    }
  }
}

// ---- attention of one new token per sequence -------------------------------

// The step's work in tiles of 128 keys: (sequence, head tile, key tile), key
// tiles innermost, cut into equal ranges of `share` tiles, one per block. A
// pair (sequence, head tile) that one block holds whole is finished there;
// others leave a partial result per block (fp32 sums, maximum and weight sum
// of each of its 16 rows), which the join adds up in block order.
constexpr int kWaves = 4;
constexpr int kBlocks = 1024;

// Workspace: error word, live sequences, share, then the tile prefix and two
// partial results per block (first range of the block, last one).
struct Ws {
  int *head;
  int *prefix;
  float *slots;
};
LF_DEVICE Ws ws_of(const Desc &d, uint8_t *ws) {
  Ws w;
  w.head = reinterpret_cast<int *>(ws);
  w.prefix = reinterpret_cast<int *>(ws + 256);
  w.slots = reinterpret_cast<float *>(ws + 256 + align256((static_cast<uint64_t>(d.max_sequences) + 1) * 4));
  return w;
}
template <int D>
LF_DEVICE float *slot_of(const Ws &w, int slot) {
  return w.slots + static_cast<uint64_t>(slot) * (kHeadTile * D + 2 * kHeadTile);
}

// Keys and values of 32 consecutive keys in a wave's registers.
//  keys:   A operand of 16x16x32 products: lane l holds, of key l % 16 of each
//          half, the 16-byte chunks l / 16, l / 16 + 4, ...
//  values: lane l holds, of the eight keys 4 g + e and 16 + 4 g + e (g = l / 16,
//          e = 0 .. 3), the D / 16 values from (l % 16) D / 16 on. Those are the
//          keys whose scores the first product leaves in this lane, so its
//          weights are the B operand of the second one as they are.
template <int D, bool E4M3>
struct Tile {
  static constexpr int kSize = E4M3 ? 1 : 2;
  static constexpr int kChunks = D * kSize / 64;        // 16-byte chunks of a key per lane
  static constexpr int kWords = D / 16 * kSize / 4;     // words of a value row per lane
  u32x4 k[2][kChunks];
  uint32_t v[8][kWords];
};

template <int WORDS>
LF_DEVICE void load_words(uint32_t (&dst)[WORDS], const uint8_t *src) {
  if constexpr (WORDS == 1) {
    dst[0] = *reinterpret_cast<const uint32_t *>(src);
  } else if constexpr (WORDS == 2) {
    const uint2 w = *reinterpret_cast<const uint2 *>(src);
    dst[0] = w.x;
    dst[1] = w.y;
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(src + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[i + e] = w[e];
    }
  }
}

LF_DEVICE bf16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(bf16x8, u32x4{a, b, c, d});
}

template <int D, bool E4M3>
LF_DEVICE void decode(const int32_t *counts, const int32_t *row_offsets, const int32_t *lengths,
                      const int32_t *page_offsets, const int32_t *page_indices, const uint8_t *attn,
                      const uint16_t *q, uint16_t *out, const uint8_t *kc, const uint8_t *vc, uint8_t *ws) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int wave_total[kWaves];
  const Desc &d = desc_of(attn);
  if (d.magic != kMagic) return;
  const Ws w = ws_of(d, ws);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rows = live_rows(counts, d.max_tokens);
  const int s0 = decoded_of(d, counts).s0, n = decoded_of(d, counts).n;

  int *prefix = reinterpret_cast<int *>(lds);
  bool bad = false;
  int64_t carry = 0;
  for (int base = 0; base < n; base += 256) {
    const int i = base + static_cast<int>(threadIdx.x);
    const int tiles = i < n ? span_of(d, lengths, page_offsets, s0 + i, bad).tiles : 0;
    int sum = tiles;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int up = __shfl_up(sum, m);
      if (lane >= m) sum += up;
    }
    if (lane == 63) wave_total[wave] = sum;
    __syncthreads();
    int64_t before = carry;
    for (int k = 0; k < kWaves; ++k) {
      if (k < wave) before += wave_total[k];
      carry += wave_total[k];
    }
    if (i < n) prefix[i] = static_cast<int>(before) + sum - tiles;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[n] = static_cast<int>(carry);
  __syncthreads();

  const int Hq = d.query_heads, Hkv = d.kv_heads, group = Hq / Hkv;
  const int group_tiles = (group + kHeadTile - 1) / kHeadTile;
  const int head_tiles = head_tiles_of(d);
  // (page ranges that overlap may add up to more than the descriptor's bound)
  const bool counted = carry * head_tiles <= INT32_MAX;
  if (!counted) bad = true;
  const int items = counted ? static_cast<int>(carry) * head_tiles : 0;
  const int share = share_of(items, kBlocks);
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) {
      w.head[1] = n;
      w.head[2] = share;
      w.head[3] = s0;
    }
    for (int i = threadIdx.x; i <= n; i += 256) w.prefix[i] = prefix[i];
  }
  if (bad) flag_error(w.head);
  if (share == 0) return;
  const int begin = static_cast<int>(blockIdx.x) * share;
  const int end = begin + share < items ? begin + share : items;

  const int shift = __builtin_ctz(d.page_size);
  const float *scales = reinterpret_cast<const float *>(attn + d.scale_offset);
  const int g = lane >> 4, c = lane & 15;
  const int tile_rows = group < kHeadTile ? group : kHeadTile;
  float *join = reinterpret_cast<float *>(lds + ((static_cast<uint64_t>(d.max_sequences) * 4 + 4 + 15) & ~uint64_t(15)));

  for (int u = begin; u < end;) {
    const int i = sequence_at(prefix, n, head_tiles, u);
    const int s = s0 + i;
    bool unused = false;
    const Span span = span_of(d, lengths, page_offsets, s, unused);
    const Pages pages = pages_of(d, page_offsets, s, unused);
    const int32_t *table = page_indices + pages.first;
    const int first_page = span.lo >> shift, end_page = (span.len + d.page_size - 1) >> shift;
    const int within = u - prefix[i] * head_tiles;
    const int ht = within / span.tiles, t0 = within - ht * span.tiles;
    const int t1 = span.tiles - t0 < end - u ? span.tiles : t0 + (end - u);
    const int h = ht / group_tiles;
    const int row0 = (ht - h * group_tiles) * kHeadTile;  // first query head of the tile in its group
    const int tile_live = group - row0 < kHeadTile ? group - row0 : kHeadTile;
    const int row = row_offsets[s];
    const bool row_ok = row >= 0 && row < rows;
    if (!row_ok) bad = true;

    // B operand of the first product: query head c, the values of its key chunk
    bf16x8 qv[D / 32];
    {
      const uint16_t *src = q + (static_cast<uint64_t>(row_ok ? row : 0) * Hq + h * group + row0 + c) * D;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        // bf16 keys: chunk k holds values 32 k + 8 g ..; e4m3: 64 (k / 2) + 16 g + 8 (k % 2) ..
        const int at = E4M3 ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 32 * k + 8 * g;
        qv[k] = c < tile_live && row_ok ? *reinterpret_cast<const bf16x8 *>(src + at) : operand(0, 0, 0, 0);
      }
    }
    const float factor = d.softmax_scale * 1.44269504088896341f * (E4M3 ? scales[h] : 1.0f);
    const uint8_t *kh = kc + cache_byte<E4M3>(d, 0, h, 0);
    const uint8_t *vh = vc + cache_byte<E4M3>(d, 0, h, 0);

    f32x4 o[D / 16];
#pragma unroll
    for (int k = 0; k < D / 16; ++k) o[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 sum4 = {0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY;

    for (int t = t0; t < t1; ++t) {
      const int base = (span.first_tile + t) * kTileKeys + 32 * wave;
      if (base >= span.len || base + 32 <= span.lo) continue;
      Tile<D, E4M3> x;
      int vpage[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int j = base + 16 * half + c;
        const int page = page_of(d, table, first_page, end_page, shift, j, bad);
        const uint8_t *src = kh + cache_byte<E4M3>(d, page < 0 ? 0 : page, 0, j & (d.page_size - 1)) + 16 * g;
#pragma unroll
        for (int k = 0; k < Tile<D, E4M3>::kChunks; ++k) x.k[half][k] = *reinterpret_cast<const u32x4 *>(src + 64 * k);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int j = base + 16 * half + 4 * g;  // four keys of one page
        vpage[half] = page_of(d, table, first_page, end_page, shift, j, bad);
        const uint8_t *src = vh + cache_byte<E4M3>(d, vpage[half] < 0 ? 0 : vpage[half], 0, j & (d.page_size - 1)) +
                             c * (D / 16 * Tile<D, E4M3>::kSize);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          load_words(x.v[4 * half + e], src + static_cast<uint64_t>(e) * static_cast<uint32_t>(d.token_stride) *
                                                  Tile<D, E4M3>::kSize);
        }
      }
      // scores: rows = keys 16 half + 4 g + r, column = query head c
      f32x4 sc[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        sc[half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < Tile<D, E4M3>::kChunks; ++k) {
          const u32x4 kw = x.k[half][k];
          if constexpr (E4M3) {
            uint32_t b[8];
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) e4m3x4_to_bf16x4(kw[i4], b[2 * i4], b[2 * i4 + 1]);
            sc[half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(b[0], b[1], b[2], b[3]), qv[2 * k], sc[half], 0,
                                                               0, 0);
            sc[half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(b[4], b[5], b[6], b[7]), qv[2 * k + 1],
                                                               sc[half], 0, 0, 0);
          } else {
            sc[half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kw), qv[k], sc[half], 0, 0, 0);
          }
        }
      }
      float z[8];
      const bool edge = base < span.lo || base + 32 > span.len;
      const bool masked = __any(edge || vpage[0] < 0 || vpage[1] < 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = sc[e >> 2][e & 3] * factor;
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = base + 16 * (e >> 2) + 4 * g + (e & 3);
          const bool live = j >= span.lo && j < span.len && vpage[e >> 2] >= 0;
          z[e] = live ? z[e] : -INFINITY;
          // a weight of zero times what the place holds would let an infinity or NaN through
#pragma unroll
          for (int i4 = 0; i4 < Tile<D, E4M3>::kWords; ++i4) x.v[e][i4] = live ? x.v[e][i4] : 0u;
        }
      }
      float most = z[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) most = fmaxf(most, z[e]);
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      if (__any(most > top)) {
        const float next = fmaxf(top, most);
        const float shrink = __builtin_amdgcn_exp2f(top - (next == -INFINITY ? 0.0f : next));
        top = next;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) o[k] *= shrink;
        sum4 *= shrink;
      }
      const float from = top == -INFINITY ? 0.0f : top;
      uint32_t pw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pw[e] = f32_to_bf16(__builtin_amdgcn_exp2f(z[2 * e] - from)) |
                (f32_to_bf16(__builtin_amdgcn_exp2f(z[2 * e + 1] - from)) << 16);
      }
      const bf16x8 p = operand(pw[0], pw[1], pw[2], pw[3]);
      constexpr uint32_t kOne2 = 0x3f803f80u;
      sum4 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(kOne2, kOne2, kOne2, kOne2), p, sum4, 0, 0, 0);
      // values as pairs of neighbouring columns, bf16
      constexpr int kPairs = D / 32;
      uint32_t vp[8][kPairs];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int i4 = 0; i4 < Tile<D, E4M3>::kWords; ++i4) {
          if constexpr (E4M3) {
            e4m3x4_to_bf16x4(x.v[e][i4], vp[e][2 * i4], vp[e][2 * i4 + 1]);
          } else {
            vp[e][i4] = x.v[e][i4];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t sel = (k & 1) ? 0x07060302u : 0x05040100u;
        uint32_t a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = __builtin_amdgcn_perm(vp[2 * e + 1][k >> 1], vp[2 * e][k >> 1], sel);
        o[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(a[0], a[1], a[2], a[3]), p, o[k], 0, 0, 0);
      }
    }

    // The four waves' results joined in wave order. o[k][r] is the sum of
    // query head c at column (4 g + r) D / 16 + k.
    float *mine = join + static_cast<uint64_t>(wave) * tile_rows * (D + 2);
    if (c < tile_live) {
      float *dst = mine + c * (D + 2);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) dst[(4 * g + r) * (D / 16) + k] = o[k][r];
      }
      if (g == 0) {
        dst[D] = top;
        dst[D + 1] = sum4[0];
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == span.tiles;
    float *slot = slot_of<D>(w, part_slot(blockIdx.x, u - t0, share));
    const float vscale = E4M3 ? scales[Hkv + h] : 1.0f;
    for (int x = threadIdx.x; x < tile_live * D; x += 256) {
      const int r = x / D, col = x % D;
      const float *src = join + r * (D + 2);
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) m = fmaxf(m, src[k * tile_rows * (D + 2) + D]);
      const float from = m == -INFINITY ? 0.0f : m;
      float acc = 0.0f, sum = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const float *p = src + k * tile_rows * (D + 2);
        const float f = __builtin_amdgcn_exp2f(p[D] - from);
        acc += f * p[col];
        sum += f * p[D + 1];
      }
      if (whole) {
        const float y = sum == 0.0f ? 0.0f : acc / sum * vscale;
        if (row_ok) {
          out[(static_cast<uint64_t>(row) * Hq + h * group + row0 + r) * D + col] =
              static_cast<uint16_t>(f32_to_bf16(y));
        }
      } else {
        slot[r * D + col] = acc;
        if (col == 0) {
          slot[kHeadTile * D + r] = m;
          slot[kHeadTile * D + kHeadTile + r] = sum;
        }
      }
    }
    __syncthreads();
    u += t1 - t0;
  }
  if (bad) flag_error(w.head);
}

// One wave per (sequence, query head): the partial results of its pair, in
// block order; pairs that one block finished are left alone.
template <int D>
LF_DEVICE void join(const int32_t *counts, const int32_t *row_offsets, const uint8_t *attn, uint16_t *out,
                    uint8_t *ws) {
  const Desc &d = desc_of(attn);
  if (d.magic != kMagic) return;
  const Ws w = ws_of(d, ws);
  const int lane = threadIdx.x & 63;
  const int item = static_cast<int>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  const int Hq = d.query_heads, Hkv = d.kv_heads, group = Hq / Hkv;
  const int i = item / Hq, qh = item - i * Hq;
  const int n = w.head[1], share = w.head[2];
  if (i >= n || share <= 0) return;
  const int row = row_offsets[w.head[3] + i];
  if (row < 0 || row >= live_rows(counts, d.max_tokens)) return;
  const int group_tiles = (group + kHeadTile - 1) / kHeadTile;
  const int h = qh / group, in_group = qh - h * group;
  const int ht = h * group_tiles + in_group / kHeadTile, r = in_group & (kHeadTile - 1);
  const int tiles = w.prefix[i + 1] - w.prefix[i];
  const int begin = w.prefix[i] * head_tiles_of(d) + ht * tiles;
  const Parts parts = parts_of(begin, tiles, share);
  if (parts.first == parts.last) return;
  constexpr int kPer = D / 64;
  float m = -INFINITY;
  for (int b = parts.first; b <= parts.last; ++b) {
    const float *slot = slot_of<D>(w, part_slot(b, begin, share));
    m = fmaxf(m, slot[kHeadTile * D + r]);
  }
  const float from = m == -INFINITY ? 0.0f : m;
  float acc[kPer], sum = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  for (int b = parts.first; b <= parts.last; ++b) {
    const float *slot = slot_of<D>(w, part_slot(b, begin, share));
    const float f = __builtin_amdgcn_exp2f(slot[kHeadTile * D + r] - from);
    sum += f * slot[kHeadTile * D + kHeadTile + r];
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] += f * slot[r * D + lane * kPer + e];
  }
  const float *scales = reinterpret_cast<const float *>(attn + d.scale_offset);
  const float vscale = scales[Hkv + h];
  uint16_t *dst = out + (static_cast<uint64_t>(row) * Hq + qh) * D + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    dst[e] = static_cast<uint16_t>(f32_to_bf16(sum == 0.0f ? 0.0f : acc[e] / sum * vscale));
  }
}

}  // namespace attn

#define LF_ATTN_ROPE(TYPE, E4M3)                                                                             \
  extern "C" __global__ __launch_bounds__(256) void lf_attn_qk_norm_rope_##TYPE(                             \
      const int32_t *counts, const int32_t *positions, const int32_t *row_offsets, const int32_t *lengths,   \
      const int32_t *page_offsets, const int32_t *page_indices, const uint8_t *desc, const uint16_t *qkv,    \
      const uint16_t *gq, const uint16_t *gk, uint16_t *q, uint8_t *kc, uint8_t *vc, int *status) {          \
    attn::qk_norm_rope<E4M3>(counts, positions, row_offsets, lengths, page_offsets, page_indices, desc, qkv, \
                             gq, gk, q, kc, vc, status);                                                     \
  }
LF_ATTN_ROPE(bf16, false)
LF_ATTN_ROPE(e4m3, true)

#define LF_ATTN_DECODE(D, TYPE, E4M3)                                                                          \
  extern "C" __global__ __launch_bounds__(256) void lf_attn_decode_d##D##_##TYPE(                              \
      const int32_t *counts, const int32_t *row_offsets, const int32_t *lengths, const int32_t *page_offsets,  \
      const int32_t *page_indices, const uint8_t *desc, const uint16_t *q, uint16_t *out, const uint8_t *kc,   \
      const uint8_t *vc, uint8_t *ws) {                                                                        \
    attn::decode<D, E4M3>(counts, row_offsets, lengths, page_offsets, page_indices, desc, q, out, kc, vc, ws); \
  }
LF_ATTN_DECODE(64, bf16, false)
LF_ATTN_DECODE(128, bf16, false)
LF_ATTN_DECODE(256, bf16, false)
LF_ATTN_DECODE(64, e4m3, true)
LF_ATTN_DECODE(128, e4m3, true)
LF_ATTN_DECODE(256, e4m3, true)

#define LF_ATTN_JOIN(D)                                                                                     \
  extern "C" __global__ __launch_bounds__(256) void lf_attn_join_d##D(                                      \
      const int32_t *counts, const int32_t *row_offsets, const uint8_t *desc, uint16_t *out, uint8_t *ws) { \
    attn::join<D>(counts, row_offsets, desc, out, ws);                                                      \
  }
LF_ATTN_JOIN(64)
LF_ATTN_JOIN(128)
LF_ATTN_JOIN(256)
