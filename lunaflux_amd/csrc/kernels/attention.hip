// attention.hip - the steps between the QKV and the output projection over a
// paged key / value cache (the attention section of include/lunaflux_fp8.h):
// per-head norm, rotary positions and cache append in one pass over the packed
// rows, and attention of one new token per sequence.
#include "device_common.h"

#include "attention_index.h"
#include "phases.h"

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
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
LF_DEVICE u32x2 e4m3x8_of(const float *v, float inv_scale) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(v[4 * i], inv_scale), e4m3_range(v[4 * i + 1], inv_scale), 0,
                                            false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(v[4 * i + 2], inv_scale), e4m3_range(v[4 * i + 3], inv_scale), p,
                                        true);
    w[i] = static_cast<uint32_t>(p);
  }
  return u32x2{w[0], w[1]};
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
// bytes. Loads and stores are nontemporal: 8192 rows of 32 + 16 heads of 128 take
// 37.7 us so (201 MB at 5.3 TB/s, the rate of a copy), 46.5 otherwise; the rows'
// loads a step ahead of their use cost occupancy (50).
template <class T, class P>
LF_DEVICE void put(P *to, T value) {
  __builtin_nontemporal_store(value, reinterpret_cast<T *>(to));
}

// The 16 values that a lane holds of a head of D, in pairs (a[e], b[e]) of the "half" pairing
// or as two runs of eight, and where they are in the head.
struct HeadLane {
  int o0, o1;
  bool turned, half;
};
LF_DEVICE HeadLane head_lane(const Desc &d, int j) {
  const int R = d.rotary_dim;
  HeadLane x;
  x.turned = 16 * j < R;
  x.half = d.pairing == 0 && x.turned;
  x.o0 = x.half ? 8 * j : 16 * j;
  x.o1 = x.half ? R / 2 + 8 * j : 16 * j + 8;
  return x;
}
LF_DEVICE void load_head(const uint16_t *src, const HeadLane &x, float (&a)[8], float (&b)[8]) {
  const u32x4 w0 = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + x.o0));
  const u32x4 w1 = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + x.o1));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[2 * i] = bf16_to_f32(w0[i] & 0xffffu);
    a[2 * i + 1] = bf16_to_f32(w0[i] >> 16);
    b[2 * i] = bf16_to_f32(w1[i] & 0xffffu);
    b[2 * i + 1] = bf16_to_f32(w1[i] >> 16);
  }
}
LF_DEVICE void norm_head(const Desc &d, const uint16_t *g, int lanes, const HeadLane &x, float (&a)[8], float (&b)[8]) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + b[e] * b[e];
  for (int m = 1; m < lanes; m <<= 1) ss += __shfl_xor(ss, m);
  const float inv = 1.0f / __builtin_sqrtf(ss / static_cast<float>(d.head_dim) + d.norm_epsilon);
  const u32x4 g0 = *reinterpret_cast<const u32x4 *>(g + x.o0);
  const u32x4 g1 = *reinterpret_cast<const u32x4 *>(g + x.o1);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[2 * i] *= inv * bf16_to_f32(g0[i] & 0xffffu);
    a[2 * i + 1] *= inv * bf16_to_f32(g0[i] >> 16);
    b[2 * i] *= inv * bf16_to_f32(g1[i] & 0xffffu);
    b[2 * i + 1] *= inv * bf16_to_f32(g1[i] >> 16);
  }
}
LF_DEVICE void turn_head(const HeadLane &w, const float (&c)[8], const float (&sn)[8], float (&a)[8], float (&b)[8]) {
  if (w.half) {
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
// Cosine and sine of pair i of the row's rotation.
LF_DEVICE float2 turn_of(const Desc &d, const uint8_t *attn, const int32_t *positions, int row, int i) {
  const double *turns = reinterpret_cast<const double *>(attn + d.turns_offset);
  const int32_t *axis = reinterpret_cast<const int32_t *>(attn + d.axis_offset);
  const double t = static_cast<double>(positions[row * d.axes + axis[i]]) * turns[i];
  float sin_t, cos_t;
  sincospif(static_cast<float>(2.0 * (t - rint(t))), &sin_t, &cos_t);
  return make_float2(cos_t, sin_t);
}

// Keys and values of the rows go to the cache too (CACHE kCacheBf16, kCacheE4m3), or are
// append_blocks' part (kCacheBlocks).
template <int CACHE>
LF_DEVICE void qk_norm_rope(int row, const int32_t *counts, const int32_t *positions, const int32_t *row_offsets,
                            const int32_t *lengths, const int32_t *page_offsets, const int32_t *page_indices,
                            const uint8_t *attn, const uint16_t *qkv, const uint16_t *gq, const uint16_t *gk,
                            uint16_t *q, uint8_t *kc, uint8_t *vc, int *status) {
  __shared__ float2 turn[128];
  const Desc &d = desc_of(attn);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  if (row >= rows) return;
  int sequences = counts[2];
  sequences = sequences < 0 ? 0 : sequences > d.max_sequences ? d.max_sequences : sequences;
  const int s = sequence_of(row_offsets, sequences, row);
  if (s >= sequences || row < row_offsets[0]) return;

  const int R = d.rotary_dim;
  if (static_cast<int>(threadIdx.x) < R / 2) turn[threadIdx.x] = turn_of(d, attn, positions, row, threadIdx.x);
  __syncthreads();

  Place place = {-1, 0};
  if constexpr (CACHE != kCacheBlocks) {
    place = place_of(d, row_offsets, lengths, page_offsets, page_indices, s, row);
    if (place.page < 0 && threadIdx.x == 0) flag_error(status);
  }

  const int D = d.head_dim, lanes = D >> 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int j = lane & (lanes - 1);
  const HeadLane at = head_lane(d, j);
  float c[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 t = at.turned ? turn[8 * j + e] : make_float2(1.0f, 0.0f);
    c[e] = t.x;
    sn[e] = t.y;
  }
  const int Hq = d.query_heads, Hkv = d.kv_heads, heads = Hq + 2 * Hkv;
  const int done = CACHE == kCacheBlocks ? Hq : heads;
  const int per_wave = 64 / lanes;
  const float *scales = reinterpret_cast<const float *>(attn + d.scale_offset);
  for (int base = wave * per_wave; base < done; base += 4 * per_wave) {
    const int h = base + lane / lanes;
    if (h >= done) continue;
    float a[8], b[8];
    load_head(qkv + (static_cast<uint64_t>(row) * heads + h) * D, at, a, b);
    if (h < Hq + Hkv) {
      if (d.norm) norm_head(d, h < Hq ? gq : gk, lanes, at, a, b);
      if (at.turned) turn_head(at, c, sn, a, b);
    }
    if (h < Hq) {
      uint16_t *dst = q + (static_cast<uint64_t>(row) * Hq + h) * D;
      put(dst + at.o0, bf16x8_of(a));
      put(dst + at.o1, bf16x8_of(b));
    } else if (place.page >= 0) {
      const bool value = h >= Hq + Hkv;
      const int kh = h - Hq - (value ? Hkv : 0);
      uint8_t *dst = (value ? vc : kc) + cache_byte<CACHE == kCacheE4m3>(d, place.page, kh, place.slot);
      if constexpr (CACHE == kCacheE4m3) {
        const float inv_scale = 1.0f / scales[(value ? Hkv : 0) + kh];
        put(dst + at.o0, e4m3x8_of(a, inv_scale));
        put(dst + at.o1, e4m3x8_of(b, inv_scale));
      } else {
        put(dst + 2 * at.o0, bf16x8_of(a));
        put(dst + 2 * at.o1, bf16x8_of(b));
      }
    }
  }
}

// ---- append with a scale per block of tokens and head --------------------------------

// The scale is the least power of two, of 2^-100 to 2^119, by which the block's largest finite
// magnitude is at most 448, e4m3's largest. As a power of two it costs no rounding: neither at
// the append nor where codes become bf16 values, and codes that are raised to a larger
// scale are rounded again only below 2^-6 of it.
LF_DEVICE float scale_of(float amax) {
  const int e = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;  // 448 = 1.75 2^8
  return __uint_as_float(static_cast<uint32_t>((e < -100 ? -100 : e > 119 ? 119 : e) + 127) << 23);
}

LF_DEVICE u32x2 raised(u32x2 codes, float ratio) {
  u32x2 out;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes[i]), false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes[i]), true);
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * ratio, lo[1] * ratio, 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * ratio, hi[1] * ratio, p, true);
    out[i] = static_cast<uint32_t>(p);
  }
  return out;
}

// A wave holds the rows of one block of tokens (at most 16) of one head's keys or values in
// registers: their largest magnitude, the scale, the codes. Blocks of the grid take four heads
// of one block of tokens, found by the number of blocks that the sequences before have. A block
// of tokens that holds older ones keeps its scale or raises it, and then their codes.
// HBM bounds it: 8191 rows of 32/8 heads of 128 with norm and rotation 44.6 us with the queries, 4.2 TB/s
// (a copy of as many bytes 36). The grid's blocks of the cache come before the rows of queries, whose
// work is shorter, so that the launch does not end with them: 52 us the other way round, with one kernel for
// all head sizes.
template <int D>
LF_DEVICE void append_rows(const Desc &d, const uint16_t *qkv, const uint16_t *gk, const float2 (*turn)[128],
                           const Block &x, int page, int unit_head, bool value, uint8_t *cache) {
  constexpr int kLanes = D / 16, kRows = 64 / kLanes, kPasses = (16 + kRows - 1) / kRows;
  const int lane = threadIdx.x & 63, j = lane & (kLanes - 1), r = lane / kLanes;
  const HeadLane at = head_lane(d, j);
  const int Hq = d.query_heads, Hkv = d.kv_heads, heads = Hq + 2 * Hkv;
  const int h = Hq + (value ? Hkv : 0) + unit_head;
  float *scales = reinterpret_cast<float *>(cache + d.block_scales) + scale_index(d, page, x.slot, unit_head);
  const float old = x.lo > 0 ? *scales : 0.0f;
  float a[kPasses][8], b[kPasses][8];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int slot = p * kRows + r;
    const bool mine = slot >= x.lo && slot < x.hi;
    load_head(qkv + (static_cast<uint64_t>(x.row + (mine ? slot - x.lo : 0)) * heads + h) * D, at, a[p], b[p]);
  }
  float amax = 0.0f;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int slot = p * kRows + r;
    const bool mine = slot >= x.lo && slot < x.hi;
    if (!value) {
      if (d.norm) norm_head(d, gk, kLanes, at, a[p], b[p]);
      if (at.turned) {
        float c[8], sn[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 t = turn[mine ? slot - x.lo : 0][8 * j + e];
          c[e] = t.x;
          sn[e] = t.y;
        }
        turn_head(at, c, sn, a[p], b[p]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = fabsf(a[p][e]), v = fabsf(b[p][e]);
      amax = fmaxf(amax, mine && u < INFINITY ? u : 0.0f);
      amax = fmaxf(amax, mine && v < INFINITY ? v : 0.0f);
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m));
  float scale = scale_of(amax);
  if (old > scale) scale = old;
  const bool grows = x.lo > 0 && old != scale;
  const float inv_scale = 1.0f / scale, ratio = old * inv_scale;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int slot = p * kRows + r;
    uint8_t *dst = cache + cache_byte<true>(d, page, unit_head, x.slot + slot);
    if (slot >= x.lo && slot < x.hi) {
      put(dst + at.o0, e4m3x8_of(a[p], inv_scale));
      put(dst + at.o1, e4m3x8_of(b[p], inv_scale));
    } else if (grows && slot < x.lo) {
      u32x2 *o0 = reinterpret_cast<u32x2 *>(dst + at.o0), *o1 = reinterpret_cast<u32x2 *>(dst + at.o1);
      const u32x2 w0 = *o0, w1 = *o1;
      *o0 = raised(w0, ratio);
      *o1 = raised(w1, ratio);
    }
  }
  if (lane == 0) *scales = scale;
}

template <int D>
LF_DEVICE void append_blocks(const int32_t *counts, const int32_t *positions, const int32_t *row_offsets,
                             const int32_t *lengths, const int32_t *page_offsets, const int32_t *page_indices,
                             const uint8_t *attn, const uint16_t *qkv, const uint16_t *gk, uint8_t *kc, uint8_t *vc,
                             int *status) {
  __shared__ int prefix[2048];  // LF_FP8_ATTN_MAX_SEQUENCES
  __shared__ int wave_total[4];
  __shared__ float2 turn[16][128];
  const Desc &d = desc_of(attn);
  if (d.magic != kMagic) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = live_rows(counts, d.max_tokens);
  int n = counts[2];
  n = n < 0 ? 0 : n > d.max_sequences ? d.max_sequences : n;
  bool bad = false;
  int64_t carry = 0;
  for (int base = 0; base < n; base += 256) {
    const int i = base + static_cast<int>(threadIdx.x);
    int blocks = 0;
    if (i < n) blocks = blocks_of(d, prompt_of(d, row_offsets, lengths, page_offsets, i, rows, bad));
    int sum = blocks;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int up = __shfl_up(sum, m);
      if (lane >= m) sum += up;
    }
    if (lane == 63) wave_total[wave] = sum;
    __syncthreads();
    int64_t before = carry;
    for (int k = 0; k < 4; ++k) {
      if (k < wave) before += wave_total[k];
      carry += wave_total[k];
    }
    if (i < n) prefix[i] = static_cast<int>(before) + sum - blocks;
    __syncthreads();
  }
  __syncthreads();
  if (carry > rows) {  // sequences that share rows: a block of tokens has a row at least
    flag_error(status);
    return;
  }
  const int Hkv = d.kv_heads, groups = (Hkv + 3) / 4;
  const int64_t items = carry * 2 * groups;
  for (int64_t u = blockIdx.x; u < items; u += gridDim.x - d.max_tokens) {
    const int b = static_cast<int>(u / (2 * groups)), unit = static_cast<int>(u - static_cast<int64_t>(b) * 2 * groups);
    const bool value = unit >= groups;
    int s = 0;  // the last with prefix[s] <= b, so one with blocks
    for (int hi = n; hi - s > 1;) {
      const int mid = (s + hi) >> 1;
      if (prefix[mid] <= b) {
        s = mid;
      } else {
        hi = mid;
      }
    }
    bool unused = false;
    const Prompt p = prompt_of(d, row_offsets, lengths, page_offsets, s, rows, unused);
    const Block x = block_of(d, p, b - prefix[s]);
    const int page = page_indices[x.entry];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(d.pages)) {
      bad = true;
      continue;
    }
    if (!value && d.rotary_dim > 0) {
      const int pairs = d.rotary_dim / 2;
      __syncthreads();  // the turns of the item before have been read
      for (int i = threadIdx.x; i < (x.hi - x.lo) * pairs; i += 256) {
        const int r = i / pairs;
        turn[r][i - r * pairs] = turn_of(d, attn, positions, x.row + r, i - r * pairs);
      }
      __syncthreads();
    }
    const int h = (value ? unit - groups : unit) * 4 + wave;
    if (h >= Hkv) continue;
    uint8_t *cache = value ? vc : kc;
    append_rows<D>(d, qkv, gk, turn, x, page, h, value, cache);
  }
  if (bad) flag_error(status);
}

// ---- attention of one new token per sequence -------------------------------

// The step's work is cut into tiles of 32 keys, (sequence, head tile, key tile)
// with key tiles innermost, and the tiles into equal ranges, one per block (by whole
// pairs (sequence, head tile) if all are short); a block's four waves take a pair's
// tiles in turn and join through LDS. A pair that one block holds whole is finished
// there. Other blocks leave a partial result (fp32 sums, maximum and weight sum of
// each of the tile's rows) in the workspace; of every kGroup neighbours the last to
// arrive adds the group's up in order, and the last group to arrive the groups'.
// HBM bounds it (5.8 TB/s of 131071 keys); a launch with nothing to read takes 5 us,
// the join 3 to 6, and the XCDs' rates differ by a tenth while their shares are
// equal. Partial results are stored and loaded at agent scope (past the XCD's L2),
// and a block counts itself only once its stores have completed.
constexpr int kWaves = 4;

// Blocks of the grid: one per CU, two where a key is 128 bytes or less and one
// would have too few bytes in flight: 96 sequences of up to 5003 keys, heads of 128
// in e4m3, 126 us with one and 111 with two; in bf16 92 and 102 for 131071 keys, 44
// and 49 for 32 sequences.
template <int D, bool E4M3>
LF_DEVICE constexpr int blocks() { return D * (E4M3 ? 1 : 2) <= 128 ? 512 : 256; }

// Workspace: a line with the error word, arrival counters of groups (at their
// first part's place) and of pairs (at theirs), the partial results, two per
// block, and the groups' sums.
struct Ws {
  int *error, *group_arrivals, *pair_arrivals;
  float *parts, *groups;
  int floats;  // of a partial result: [rows][D] sums, rows maxima, rows weight sums
};
template <int D, bool E4M3>
LF_DEVICE Ws ws_of(uint8_t *ws, int tile_rows) {
  constexpr int places = 2 * blocks<D, E4M3>();
  Ws w;
  w.error = reinterpret_cast<int *>(ws);
  w.group_arrivals = reinterpret_cast<int *>(ws + 256);
  w.pair_arrivals = w.group_arrivals + places;
  w.parts = reinterpret_cast<float *>(w.pair_arrivals + places);
  w.floats = tile_rows * (D + 2);
  w.groups = w.parts + static_cast<uint64_t>(places) * w.floats;
  return w;
}

LF_DEVICE float load_agent(const float *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
LF_DEVICE void store_agent(float *p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Counts this block, whose stores at agent scope came before; true for the last
// of `total`, which puts the counter back to zero.
LF_DEVICE bool arrive(int *counter, int total, int *flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before == total - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = before == total - 1 ? 1 : 0;
  }
  __syncthreads();
  const bool last = __builtin_amdgcn_readfirstlane(*flag) != 0;
  asm volatile("" ::: "memory");
  return last;
}

// The block adds up `count` partial results of `rows` rows in their order, the
// first at float `first` of `from` and the p-th of the others at rest + p step,
// and hands every value on: write(row, column, sum, weight sum, maximum).
// kGroup results of a few values per thread are in flight at a time. stats:
// LDS, the maxima and weight sums of kGroup results. (The empty asm keeps the
// compiler from holding an address per result and thread.)
template <int D, class W>
LF_DEVICE void add_parts(const float *from, int first, int rest, int step, int count, int rows, int tile_rows,
                         float (*stats)[kGroup][kHeadTile], W &&write) {
  constexpr int kThreads = 64 * kWaves, kAtOnce = 2;
  static_assert(2 * kThreads == kGroup * kHeadTile, "two statistics per thread");
  for (int x0 = 0; x0 < rows * D; x0 += kAtOnce * kThreads) {
    float acc[kAtOnce], sum[kAtOnce], top[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) acc[i] = sum[i] = 0.0f, top[i] = -INFINITY;
    for (int p0 = 0; p0 < count; p0 += kGroup) {
      float v[kGroup][kAtOnce];
#pragma unroll
      for (int p = 0; p < kGroup; ++p) {
        const int part = p0 + p < count ? p0 + p : p0;
        uint32_t at = static_cast<uint32_t>(part == 0 ? first : rest + part * step);
        asm("" : "+s"(at));
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const int x = x0 + i * kThreads + static_cast<int>(threadIdx.x);
          v[p][i] = load_agent(from + at + static_cast<uint32_t>(x < rows * D ? x : 0));
        }
      }
      const int sr = threadIdx.x % kHeadTile;
      float m[2], l[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int sp = p0 + static_cast<int>(threadIdx.x) / kHeadTile + i * (kGroup / 2);
        const bool some = sp < count && sr < rows;
        const float *src = from + (sp == 0 || !some ? first : rest + sp * step) + tile_rows * D + (some ? sr : 0);
        m[i] = load_agent(src);
        l[i] = load_agent(src + tile_rows);
        m[i] = some ? m[i] : -INFINITY;
        l[i] = some ? l[i] : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        stats[0][threadIdx.x / kHeadTile + i * (kGroup / 2)][sr] = m[i];
        stats[1][threadIdx.x / kHeadTile + i * (kGroup / 2)][sr] = l[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int x = x0 + i * kThreads + static_cast<int>(threadIdx.x), r = x < rows * D ? x / D : 0;
        float next = top[i];
#pragma unroll
        for (int p = 0; p < kGroup; ++p) next = fmaxf(next, stats[0][p][r]);
        const float base = next == -INFINITY ? 0.0f : next;
        const float keep = __builtin_amdgcn_exp2f(top[i] - base);
        top[i] = next;
        acc[i] *= keep;
        sum[i] *= keep;
#pragma unroll
        for (int p = 0; p < kGroup; ++p) {
          const float f = __builtin_amdgcn_exp2f(stats[0][p][r] - base);
          sum[i] += f * stats[1][p][r];
          acc[i] += p0 + p < count ? f * v[p][i] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int x = x0 + i * kThreads + static_cast<int>(threadIdx.x);
      if (x < rows * D) write(x / D, x % D, acc[i], sum[i], top[i]);
    }
  }
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

// Values of one row, 16 lanes taking the whole of it: nontemporal, since nothing
// reads them again (131071 keys 102 us with plain loads and 92 so, 32 sequences 49
// and 44). Keys, whose lines two loads share, are faster so in bf16 (94, 47) and
// slower in e4m3 (129, 132), with values so both ways: they are loaded plainly.
template <int WORDS>
LF_DEVICE void load_words(uint32_t (&dst)[WORDS], const uint8_t *src) {
  typedef uint32_t Words __attribute__((ext_vector_type(WORDS < 4 ? WORDS : 4)));
#pragma unroll
  for (int i = 0; i < WORDS; i += 4) {
    const Words w = __builtin_nontemporal_load(reinterpret_cast<const Words *>(src + 4 * i));
#pragma unroll
    for (int e = 0; e < (WORDS < 4 ? WORDS : 4); ++e) dst[i + e] = w[e];
  }
}

template <int WORDS>
LF_DEVICE void store_words(uint16_t *dst, const uint32_t (&src)[WORDS]) {
  if constexpr (WORDS == 2) {
    *reinterpret_cast<uint2 *>(dst) = make_uint2(src[0], src[1]);
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4)
      *reinterpret_cast<u32x4 *>(dst + 2 * i) = u32x4{src[i], src[i + 1], src[i + 2], src[i + 3]};
  }
}

LF_DEVICE bf16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(bf16x8, u32x4{a, b, c, d});
}

// The bf16 values of two fp32 values' upper halves, and what such a half leaves.
LF_DEVICE uint32_t upper_halves(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
LF_DEVICE float rest_of(float v) {
  return fmaxf(v - __uint_as_float(__float_as_uint(v) & 0xffff0000u), v * 0x1p-64f);
}

// Where a tile's four groups of keys are: byte offsets of their first rows from
// the head's first, and which of them lie in the cache.
struct Groups {
  uint64_t at0, at1, at2, at3;
  int in;
};
// page: the groups' page indices in lanes 0 .. 3.
LF_DEVICE Groups groups_of(int page, int pages, uint32_t page_bytes, uint32_t token_bytes, int slot_mask, int base) {
  int in = 0;
  auto at = [&](int p, int k) {
    const bool ok = static_cast<uint32_t>(p) < static_cast<uint32_t>(pages);
    in |= ok ? 1 << k : 0;
    return row_byte(ok ? p : 0, (base + 8 * k) & slot_mask, page_bytes, token_bytes);
  };
  const uint64_t a = at(__builtin_amdgcn_readlane(page, 0), 0), b = at(__builtin_amdgcn_readlane(page, 1), 1);
  const uint64_t c = at(__builtin_amdgcn_readlane(page, 2), 2), d = at(__builtin_amdgcn_readlane(page, 3), 3);
  return {a, b, c, d, in};
}
LF_DEVICE uint64_t pick(bool first, uint64_t a, uint64_t b) { return first ? a : b; }

// keys: this lane's part of the first row of its group of eight (c % 8 rows
// further, chunk g); values: that of row 4 g of its half.
template <int D, bool E4M3>
LF_DEVICE void load_keys(Tile<D, E4M3> &x, const uint8_t *keys, const Groups &at, int c) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint8_t *src = keys + pick(c < 8, half == 0 ? +at.at0 : +at.at2, half == 0 ? +at.at1 : +at.at3);
#pragma unroll
    for (int k = 0; k < Tile<D, E4M3>::kChunks; ++k) x.k[half][k] = *reinterpret_cast<const u32x4 *>(src + 64 * k);
  }
}
template <int D, bool E4M3>
LF_DEVICE void load_values(Tile<D, E4M3> &x, const uint8_t *values, const Groups &at, uint32_t token_bytes, int g) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint8_t *src = values + pick(g < 2, half == 0 ? +at.at0 : +at.at2, half == 0 ? +at.at1 : +at.at3);
#pragma unroll
    for (int e = 0; e < 4; ++e) load_words(x.v[4 * half + e], src + static_cast<uint64_t>(e) * token_bytes);
  }
}

// The larger of a value over the four lane groups, in all of them.
LF_DEVICE float max_over_groups(float v) {
  const uint32_t a = __float_as_uint(v);
  const auto x = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t b = __float_as_uint(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
  const auto y = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// A part of a pair: the tiles of keys [base, stop) of a sequence whose keys [lo,
// len) count, stop at most len, for `live` query heads from head `row0` of key
// head h's group on.
struct PlainPiece {
  const int32_t *table;
  int lo, len, base, stop;
  int h, row0, live, row;  // row of q and out, or -1
  int pair, tiles;         // its pair's first item and tiles
};
struct SinkPiece : PlainPiece {
  int sink, edge, jump;  // the first keys that count too; from `edge` on, keys are `jump` further
};

// What a block keeps of each of the first sequences in LDS.
struct Sequence {
  Span span;
  int entry, row;  // first page table entry, row of q and out
};
struct Sinks {
  int sink, tiles;
};

// BLOCKS: an e4m3 cache with scales by blocks of tokens. A lane's keys of a half of the tile
// lie in one block, so its key scale multiplies the half's scores and its value scale the
// weights, which are powers of two and leave the weights' mantissas; the sum of the weights
// takes its ones divided by them. 96 sequences of up to 5003 keys, 32/8 heads of 128: 115 us, 1 to 3 more
// than with scales per head for 1.6 % more bytes and the loads of the scales.
// SINKS: Piece's base, stop and the tiles are counted along the keys that are read, the sinks' tiles and
// then the window's (64 sequences, windows of 4093 and 5 sinks in bf16 98 us, HBM at the copy's rate).
template <int D, bool E4M3, bool BLOCKS, bool SINKS>
LF_DEVICE void decode(const int32_t *counts, const int32_t *row_offsets, const int32_t *lengths,
                      const int32_t *page_offsets, const int32_t *page_indices, const uint8_t *attn,
                      const uint16_t *q, uint16_t *out, const uint8_t *kc, const uint8_t *vc, uint8_t *ws) {
  using Piece = std::conditional_t<SINKS, SinkPiece, PlainPiece>;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int wave_total[kWaves], wave_long[kWaves];
  __shared__ int arrived;
  __shared__ float stats[2][kGroup][kHeadTile];
  __shared__ Sequence near[64 * kWaves];
  __shared__ Sinks near_sinks[SINKS ? 64 * kWaves : 1];
  const Desc &d = desc_of(attn);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (the loads before the first wait: each further round trip to memory delays
  // every block's first keys)
  const int magic = d.magic, count0 = counts[0], count1 = counts[1], count2 = counts[2];
  int rows = counts[kQueryTokensIndex];
  rows = rows < 0 ? 0 : rows > d.max_tokens ? d.max_tokens : rows;
  if (magic != static_cast<int>(kMagic)) return;
  const Decoded decoded = decoded_of(d, count0, count1, count2);
  const int s0 = decoded.s0, n = decoded.n;
  auto load_sequence = [&](int s, bool &is_bad, Sinks &sinks) {
    const int len = lengths[s], first = page_offsets[s], end = page_offsets[s + 1], row = row_offsets[s];
    const Pages pages = pages_of(d, first, end, is_bad);
    if constexpr (SINKS) {
      const SinkSpan span = sink_span_of(d, len, pages, is_bad);
      sinks = {span.sink, span.sink_tiles};
      return Sequence{span.span, pages.first, row};
    } else {
      return Sequence{span_of(d, len, pages, is_bad), pages.first, row};
    }
  };

  int *prefix = reinterpret_cast<int *>(lds);
  const int most_tiles = whole_tiles(n * head_tiles_of(d));
  bool bad = false, longer = false;
  int64_t carry = 0;
  for (int base = 0; base < n; base += 256) {
    const int i = base + static_cast<int>(threadIdx.x);
    int tiles = 0;
    if (i < n) {
      Sinks sinks;
      const Sequence q1 = load_sequence(s0 + i, bad, sinks);
      tiles = q1.span.tiles;
      if (base == 0) {
        near[i] = q1;
        if constexpr (SINKS) near_sinks[i] = sinks;
      }
    }
    longer |= tiles > most_tiles;
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
  const bool some_longer = __ballot(longer) != 0;
  if (lane == 0) wave_long[wave] = some_longer ? 1 : 0;
  __syncthreads();

  const int Hq = d.query_heads, Hkv = d.kv_heads, group = Hq / Hkv;
  const int group_tiles = (group + kHeadTile - 1) / kHeadTile;
  const int head_tiles = head_tiles_of(d);
  // (page ranges that overlap may add up to more than the descriptor's bound; a wave's
  // own sums fit 31 bits, since at most every other range of a list of offsets can
  // rise past another: 32 of 2^26 - 32 tiles and 32 of one)
  const bool counted = carry * head_tiles <= kMostItems;
  if (!counted) bad = true;
  const int items = __builtin_amdgcn_readfirstlane(counted ? static_cast<int>(carry) * head_tiles : 0);
  const int share = share_of(items, n * head_tiles, blocks<D, E4M3>());
  const int tile_rows = group < kHeadTile ? group : kHeadTile;
  const Ws w = ws_of<D, E4M3>(ws, tile_rows);
  if (bad) flag_error(w.error);

  const int shift = __builtin_ctz(d.page_size);
  constexpr uint32_t kSize = E4M3 ? 1 : 2;
  const uint32_t page_bytes = static_cast<uint32_t>(d.page_stride) * kSize;
  const uint32_t token_bytes = static_cast<uint32_t>(d.token_stride) * kSize;
  const int slot_mask = d.page_size - 1, pages = d.pages;
  const float *scales = reinterpret_cast<const float *>(attn + d.scale_offset);
  const int g = lane >> 4, c = lane & 15;

  const int block = blockIdx.x;
  const bool by_pair = __builtin_amdgcn_readfirstlane(wave_long[0] | wave_long[1] | wave_long[2] | wave_long[3]) == 0;
  int u, end;
  if (by_pair) {
    int tiles = 0;  // of the pair whose first item it gives
    auto start = [&](int pair) {
      const int i = pair / head_tiles, before = prefix[i];
      tiles = __builtin_amdgcn_readfirstlane(prefix[i + 1] - before);
      return __builtin_amdgcn_readfirstlane(before) * head_tiles + (pair - i * head_tiles) * tiles;
    };
    const PairRange mine = pairs_of(block, n * head_tiles, blocks<D, E4M3>());
    if (items == 0 || mine.first >= mine.end) return;
    u = start(mine.first);
    end = u + tiles;
    if (mine.end - mine.first > 1) end = start(mine.end - 1) + tiles;
  } else {
    const int64_t begin64 = static_cast<int64_t>(block) * share;
    if (begin64 >= items) return;
    u = static_cast<int>(begin64);
    end = items - u < share ? items : u + share;
  }

  // the next part of a pair in the block's range
  auto take = [&](Piece &x) {
    while (u < end) {
      const int i = __builtin_amdgcn_readfirstlane(sequence_at(prefix, n, head_tiles, u));
      bool unused = false;
      Sinks sinks = SINKS && i < 64 * kWaves ? near_sinks[i] : Sinks{0, 0};
      const Sequence seq = i < 64 * kWaves ? near[i] : load_sequence(s0 + i, unused, sinks);
      auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
      const Span span = {same(seq.span.first_tile), same(seq.span.tiles), same(seq.span.lo), same(seq.span.len)};
      const int within = u - __builtin_amdgcn_readfirstlane(prefix[i]) * head_tiles;
      const int ht = within / span.tiles, t0 = within - ht * span.tiles;
      const int t1 = span.tiles - t0 < end - u ? span.tiles : t0 + (end - u);
      x.pair = u - t0;
      x.tiles = span.tiles;
      x.h = ht / group_tiles;
      x.row0 = (ht - x.h * group_tiles) * kHeadTile;
      x.live = group - x.row0 < kHeadTile ? group - x.row0 : kHeadTile;
      x.row = __builtin_amdgcn_readfirstlane(seq.row);
      if (x.row < 0 || x.row >= rows) {
        x.row = -1;
        bad = true;
      }
      x.table = page_indices + __builtin_amdgcn_readfirstlane(seq.entry);
      x.lo = span.lo;
      x.len = span.len;
      if constexpr (SINKS) {
        const int sink_tiles = same(sinks.tiles);
        x.sink = same(sinks.sink);
        x.edge = sink_tiles * kTileKeys;
        x.jump = (span.first_tile - sink_tiles) * kTileKeys;
        x.base = t0 * kTileKeys;
        x.stop = t1 * kTileKeys < span.len - x.jump ? t1 * kTileKeys : span.len - x.jump;
      } else {
        x.base = (span.first_tile + t0) * kTileKeys;
        x.stop = (span.first_tile + t1) * kTileKeys < span.len ? (span.first_tile + t1) * kTileKeys : span.len;
      }
      u += t1 - t0;
      if (span.len > 0) return true;
      if (x.row >= 0) {  // no keys
        uint16_t *dst = out + (static_cast<uint64_t>(x.row) * Hq + x.h * group + x.row0) * D;
        for (int k = threadIdx.x; k < x.live * D; k += 64 * kWaves) dst[k] = 0;
      }
    }
    return false;
  };
  // the key that a tile counted along the piece begins with
  auto key_of = [&](const Piece &x, int base) {
    if constexpr (SINKS) base += base >= x.edge ? x.jump : 0;
    return base;
  };
  auto indices = [&](const int32_t *table, int lo, int len, int base) {
    return table[entry_of(lo >> shift, (len + slot_mask) >> shift, shift, base + 8 * (lane & 3))];
  };
  auto pages_at = [&](const Piece &x, int base) {
    if constexpr (SINKS) {
      return x.table[sink_entry_of((x.sink + slot_mask) >> shift, x.lo >> shift, (x.len + slot_mask) >> shift, shift,
                                   key_of(x, base) + 8 * (lane & 3))];
    } else {
      return indices(x.table, x.lo, x.len, base);
    }
  };
  auto tile_groups = [&](int page, int base) {
    return groups_of(page, pages, page_bytes, token_bytes, slot_mask, base);
  };
  // this lane's part of a head's rows
  const uint64_t key_at = key_lane(c, g, token_bytes), value_at = value_lane(c, g, token_bytes, D / 16 * kSize);
  const uint32_t head_bytes = static_cast<uint32_t>(d.head_stride) * kSize;
  auto keys_of = [&](uint32_t h) { return kc + static_cast<uint64_t>(h) * head_bytes + key_at; };
  auto values_of = [&](uint32_t h) { return vc + static_cast<uint64_t>(h) * head_bytes + value_at; };
  // B operand of the first product: query head c, the values of its key chunk
  bf16x8 qv[D / 32];
  auto load_queries = [&](const Piece &x) {
    const uint16_t *src =
        q + (static_cast<uint64_t>(x.row < 0 ? 0 : x.row) * Hq + x.h * group + x.row0 + (c < x.live ? c : 0)) * D;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      // bf16 keys: chunk k holds values 32 k + 8 g ..; e4m3: 64 (k / 2) + 16 g + 8 (k % 2) ..
      const int at = E4M3 ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 32 * k + 8 * g;
      qv[k] = *reinterpret_cast<const bf16x8 *>(src + at);
    }
  };

  // Loads run one tile ahead, over the ends of pieces too: keys, values and
  // queries each into the registers just consumed, page indices one further.
  // The wave's tiles of a piece are its own-th of every four; a piece without one
  // for it gives it one tile of keys that are all masked.
  constexpr int kStep = kWaves * kTileKeys;
  auto take_mine = [&](Piece &x) {
    const bool some = take(x);
    x.base += wave * kTileKeys;
    return some;
  };
  Piece now, next;
  if (!take_mine(now)) {
    if (bad) flag_error(w.error);
    return;
  }
  Tile<D, E4M3> x;
  // BLOCKS: lanes 0 .. 3 (of every eight) hold the key scales of a tile's groups, 4 .. 7 the value
  // scales (a finite one also where no key counts).
  float steps = 1.0f;
  auto load_steps = [&](int page, int h, int base) {
    if constexpr (BLOCKS) {
      const uint8_t *side = (lane & 4) != 0 ? vc : kc;
      const int p = static_cast<uint32_t>(page) < static_cast<uint32_t>(pages) ? page : 0;
      const float v = reinterpret_cast<const float *>(side + d.block_scales)[scale_index(d, p, (base + 8 * (lane & 3)) & slot_mask, h)];
      return fminf(fmaxf(v, 0x1p-100f), 0x1p119f);
    } else {
      return 1.0f;
    }
  };
  const int first_page = pages_at(now, now.base);
  Groups at = tile_groups(first_page, key_of(now, now.base));
  load_keys(x, keys_of(now.h), at, c);
  steps = load_steps(first_page, now.h, key_of(now, now.base));
  load_queries(now);
  int ahead = pages_at(now, now.base + kStep);
  asm volatile("" ::: "memory");  // values last, as in the loop
  load_values(x, values_of(now.h), at, token_bytes, g);
  bool has_next = take_mine(next);
  if (!has_next) next = now;  // what is loaded behind the last tile
  auto after_one_tile = [&]() {  // a piece of one tile: the tile ahead is the next piece's
    if (now.base + kStep >= now.stop) {
      ahead = pages_at(next, next.base);
      asm volatile("" : "+v"(ahead));  // waited for here, not where every tile's is
    }
  };
  after_one_tile();

  for (;;) {
    const float factor = d.softmax_scale * 1.44269504088896341f * (E4M3 && !BLOCKS ? scales[now.h] : 1.0f);
    f32x4 o[D / 16];
#pragma unroll
    for (int k = 0; k < D / 16; ++k) o[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 sum4 = {0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY;
    int base = now.base;
    do {
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
      // The tile after this one, in this piece or the next; behind the last, any.
      // (All loads are issued on every path: a load that a branch may skip makes
      // the wait for an older one a wait for all.)
      const bool more = base + kStep < now.stop;
      const int then_base = more ? key_of(now, base + kStep) : key_of(next, next.base);
      const Groups then = tile_groups(ahead, then_base);
      const uint32_t then_h = more ? now.h : next.h;
      load_keys(x, keys_of(then_h), then, c);
      float step[2][2] = {{1.0f, 1.0f}, {1.0f, 1.0f}};  // [key, value][half]
      if constexpr (BLOCKS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) step[i >> 1][i & 1] = __shfl(steps, 4 * (i >> 1) + 2 * (i & 1) + (g >> 1));
        steps = load_steps(ahead, then_h, then_base);
      }
      if (!more) load_queries(next);
      {
        const bool same = base + 2 * kStep < now.stop;
        if constexpr (SINKS) {
          ahead = pages_at(same ? now : next, same ? base + 2 * kStep : more ? next.base : next.base + kStep);
        } else {
          ahead = indices(same ? now.table : next.table, same ? now.lo : next.lo, same ? now.len : next.len,
                          same ? base + 2 * kStep : more ? next.base : next.base + kStep);
        }
      }
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = sc[e >> 2][e & 3] * (BLOCKS ? factor * step[0][e >> 2] : factor);
      if (at.in != 15 && base < now.stop) bad = true;
      const int key = key_of(now, base);
      int sink = 0;
      if constexpr (SINKS) sink = now.sink;
      if ((key < now.lo && (!SINKS || key + kTileKeys > sink)) || base + kTileKeys > now.stop || at.in != 15) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int within = 16 * (e >> 2) + 4 * g + (e & 3), j = key + within;
          const bool live = (j >= now.lo || (SINKS && j < sink)) && base + within < now.stop &&
                            ((at.in >> (2 * (e >> 2) + (g >> 1))) & 1) != 0;
          z[e] = live ? z[e] : -INFINITY;
          // a weight of zero times what the place holds would let an infinity or NaN through
#pragma unroll
          for (int i4 = 0; i4 < Tile<D, E4M3>::kWords; ++i4) x.v[e][i4] = live ? x.v[e][i4] : 0u;
        }
      }
      float most = z[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) most = fmaxf(most, z[e]);
      most = max_over_groups(most);
      const float before = top;
      top = fmaxf(top, most);
      const float from = top == -INFINITY ? 0.0f : top;
      const float shrink = __builtin_amdgcn_exp2f(before - from);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) o[k] *= shrink;
      sum4 *= shrink;
      // Weights as two bf16 terms, the upper half of the fp32 bits and the rest, which
      // leave 2^-15 of a weight; one term alone leaves 2^-8, which shows in bf16
      // outputs (relative to fp32 weights 1.9e-3, and 1e-4 so; 131071 keys 90 us
      // either way, 96 sequences over e4m3 108.7 and 110.2). A weight above zero has
      // a rest above zero: any other would make NaN of an infinite value.
      uint32_t pw[4], rw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float p0 = __builtin_amdgcn_exp2f(z[2 * e] - from), p1 = __builtin_amdgcn_exp2f(z[2 * e + 1] - from);
        if constexpr (BLOCKS) {
          p0 *= step[1][e >> 1];
          p1 *= step[1][e >> 1];
        }
        pw[e] = upper_halves(p0, p1);
        rw[e] = f32_to_bf16(rest_of(p0)) | (f32_to_bf16(rest_of(p1)) << 16);
      }
      const bf16x8 p = operand(pw[0], pw[1], pw[2], pw[3]), rest = operand(rw[0], rw[1], rw[2], rw[3]);
      constexpr uint32_t kOne2 = 0x3f803f80u;
      uint32_t one[2] = {kOne2, kOne2};
      if constexpr (BLOCKS) {  // 2^-e of the halves' value scales 2^e, in bf16
#pragma unroll
        for (int half = 0; half < 2; ++half) one[half] = (0x7f00u - (__float_as_uint(step[1][half]) >> 16)) * 0x10001u;
      }
      const bf16x8 ones = operand(one[0], one[0], one[1], one[1]);
      sum4 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p, sum4, 0, 0, 0);
      sum4 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, rest, sum4, 0, 0, 0);
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
        const bf16x8 columns = operand(a[0], a[1], a[2], a[3]);
        o[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(columns, p, o[k], 0, 0, 0);
        o[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(columns, rest, o[k], 0, 0, 0);
      }
      load_values(x, values_of(then_h), then, token_bytes, g);
      at = then;
      base += kStep;
    } while (base < now.stop);

    // The waves' results joined in wave order. o[k][r] is the sum of query head
    // c at column (4 g + r) D / 16 + k.
    float *join = reinterpret_cast<float *>(lds + ((static_cast<uint32_t>(d.max_sequences) * 4 + 4 + 15) & ~15u));
    constexpr int kRow = D + 4;  // of a row in LDS: D sums, maximum, weight sum
    if (c < now.live) {
      float *dst = join + (wave * tile_rows + c) * kRow;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int k = 0; k < D / 16; k += 4)
          *reinterpret_cast<f32x4 *>(dst + (4 * g + r) * (D / 16) + k) =
              f32x4{o[k][r], o[k + 1][r], o[k + 2][r], o[k + 3][r]};
      }
      if (g == 0) {
        dst[D] = top;
        dst[D + 1] = sum4[0];
      }
    }
    __syncthreads();
    const Parts parts = parts_of(now.pair, now.tiles, share);
    const bool whole = by_pair || parts.first == parts.last;
    const float vscale = E4M3 && !BLOCKS ? scales[Hkv + now.h] : 1.0f;
    const int live = now.live;
    uint16_t *dst = out + (static_cast<uint64_t>(now.row < 0 ? 0 : now.row) * Hq + now.h * group + now.row0) * D;
    float *part = w.parts + static_cast<uint64_t>(part_slot(block, now.pair, share)) * w.floats;
    auto finish = [&](int r, int col, float acc, float sum) {
      if (now.row >= 0) dst[r * D + col] = static_cast<uint16_t>(f32_to_bf16(sum == 0.0f ? 0.0f : acc / sum * vscale));
    };
    for (int x1 = threadIdx.x; x1 < live * D; x1 += 64 * kWaves) {
      const int r = x1 / D, col = x1 % D;
      const float *src = join + r * kRow;
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) m = fmaxf(m, src[k * tile_rows * kRow + D]);
      const float from = m == -INFINITY ? 0.0f : m;
      float acc = 0.0f, sum = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const float *p = src + k * tile_rows * kRow;
        const float f = __builtin_amdgcn_exp2f(p[D] - from);
        acc += f * p[col];
        sum += f * p[D + 1];
      }
      if (whole) {
        finish(r, col, acc, sum);
      } else {
        store_agent(part + x1, acc);
        if (col == 0) {
          store_agent(part + tile_rows * D + r, m);
          store_agent(part + tile_rows * (D + 1) + r, sum);
        }
      }
    }
    if (!whole) {
      const int count = parts.last - parts.first + 1, group_count = (count + kGroup - 1) / kGroup;
      const int start = parts.first + (block - parts.first) / kGroup * kGroup;
      const int in_group = parts.last + 1 - start < kGroup ? parts.last + 1 - start : kGroup;
      // the group's parts, then, if there are several groups, their sums
      float *sums = w.groups + static_cast<uint64_t>(group_slot(start, parts.first)) * w.floats;
      const float *from = w.parts;
      int first = part_slot(start, now.pair, share) * w.floats, rest = 2 * start * w.floats, adds = in_group;
      bool done = group_count == 1;
      bool go_on = arrive(w.group_arrivals + part_slot(start, now.pair, share), in_group, &arrived);
      while (go_on) {
        add_parts<D>(from, first, rest, 2 * w.floats, adds, live, tile_rows, stats,
                     [&](int r, int col, float acc, float sum, float m) {
                       if (done) {
                         finish(r, col, acc, sum);
                       } else {
                         store_agent(sums + r * D + col, acc);
                         if (col == 0) {
                           store_agent(sums + tile_rows * D + r, m);
                           store_agent(sums + tile_rows * (D + 1) + r, sum);
                         }
                       }
                     });
        go_on = !done && arrive(w.pair_arrivals + part_slot(parts.first, now.pair, share), group_count, &arrived);
        done = true;
        adds = group_count;
        from = w.groups;
        first = group_slot(parts.first, parts.first) * w.floats;
        rest = first - w.floats;
      }
    }
    __syncthreads();  // the join area has been read
    if (!has_next) break;
    now = next;
    has_next = take_mine(next);
    if (!has_next) next = now;
    after_one_tile();
  }
  if (bad) flag_error(w.error);
}

}  // namespace attn

#define LF_ATTN_ROPE_ARGUMENTS                                                                                 \
  const int32_t *__restrict__ counts, const int32_t *__restrict__ positions,                                   \
      const int32_t *__restrict__ row_offsets, const int32_t *__restrict__ lengths,                            \
      const int32_t *__restrict__ page_offsets, const int32_t *__restrict__ page_indices,                      \
      const uint8_t *__restrict__ desc, const uint16_t *__restrict__ qkv,                                      \
      const uint16_t *__restrict__ gq, const uint16_t *__restrict__ gk, uint16_t *__restrict__ q,              \
      uint8_t *__restrict__ kc, uint8_t *__restrict__ vc, int *__restrict__ status
#define LF_ATTN_ROPE(TYPE, CACHE)                                                                              \
  extern "C" __global__ __launch_bounds__(256, CACHE == attn::kCacheBf16 ? 8 : 7)                              \
  void lf_attn_qk_norm_rope_##TYPE(LF_ATTN_ROPE_ARGUMENTS) {                                                   \
    attn::qk_norm_rope<CACHE>(blockIdx.x, counts, positions, row_offsets, lengths, page_offsets, page_indices, \
                              desc, qkv, gq, gk, q, kc, vc, status);                                           \
  }
LF_ATTN_ROPE(bf16, attn::kCacheBf16)
LF_ATTN_ROPE(e4m3, attn::kCacheE4m3)

// The first blocks of the grid write the cache, the last max_tokens the queries.
#define LF_ATTN_ROPE_BLOCKS(D)                                                                                 \
  extern "C" __global__ __launch_bounds__(256)                                                                 \
  void lf_attn_qk_norm_rope_e4m3_blocks_d##D(LF_ATTN_ROPE_ARGUMENTS) {                                         \
    const int row = static_cast<int>(blockIdx.x) - static_cast<int>(gridDim.x) + attn::desc_of(desc).max_tokens; \
    if (row < 0) {                                                                                             \
      attn::append_blocks<D>(counts, positions, row_offsets, lengths, page_offsets, page_indices, desc, qkv,   \
                             gk, kc, vc, status);                                                              \
    } else {                                                                                                   \
      attn::qk_norm_rope<attn::kCacheBlocks>(row, counts, positions, row_offsets, lengths, page_offsets,       \
                                             page_indices, desc, qkv, gq, gk, q, kc, vc, status);              \
    }                                                                                                          \
  }
LF_ATTN_ROPE_BLOCKS(64)
LF_ATTN_ROPE_BLOCKS(128)
LF_ATTN_ROPE_BLOCKS(256)

#define LF_ATTN_DECODE(D, TYPE, ...)                                                                           \
  extern "C" __global__ __launch_bounds__(256, D == 256 ? 1 : 2) void lf_attn_decode_d##D##_##TYPE(            \
      const int32_t *__restrict__ counts, const int32_t *__restrict__ row_offsets,                             \
      const int32_t *__restrict__ lengths, const int32_t *__restrict__ page_offsets,                           \
      const int32_t *__restrict__ page_indices, const uint8_t *__restrict__ desc,                              \
      const uint16_t *__restrict__ q, uint16_t *__restrict__ out, const uint8_t *__restrict__ kc,              \
      const uint8_t *__restrict__ vc, uint8_t *__restrict__ ws) {                                              \
    attn::decode<D, __VA_ARGS__>(counts, row_offsets, lengths, page_offsets, page_indices, desc, q, out, kc,   \
                                 vc, ws);                                                                      \
  }
LF_ATTN_DECODE(64, bf16, false, false, false)
LF_ATTN_DECODE(128, bf16, false, false, false)
LF_ATTN_DECODE(256, bf16, false, false, false)
LF_ATTN_DECODE(64, e4m3, true, false, false)
LF_ATTN_DECODE(128, e4m3, true, false, false)
LF_ATTN_DECODE(256, e4m3, true, false, false)
LF_ATTN_DECODE(64, bf16_sinks, false, false, true)
LF_ATTN_DECODE(128, bf16_sinks, false, false, true)
LF_ATTN_DECODE(256, bf16_sinks, false, false, true)
LF_ATTN_DECODE(64, e4m3_sinks, true, false, true)
LF_ATTN_DECODE(128, e4m3_sinks, true, false, true)
LF_ATTN_DECODE(256, e4m3_sinks, true, false, true)
LF_ATTN_DECODE(64, e4m3_blocks, true, true, true)
LF_ATTN_DECODE(128, e4m3_blocks, true, true, true)
LF_ATTN_DECODE(256, e4m3_blocks, true, true, true)
