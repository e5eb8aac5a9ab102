// attention_index.h - which memory the attention kernels touch and how their
// work is cut: the descriptor as the device sees it, a sequence's pages and
// live keys, and the split of a step's key tiles over blocks. Integer code
// only, no device builtins, so it also compiles for the host.
#pragma once

#include <stdint.h>

namespace attn {

// Mirror of lf_fp8_attn_desc.
struct Desc {
  uint32_t magic;
  int32_t query_heads, kv_heads, head_dim, cache, page_size, pages;
  int32_t max_tokens, max_sequences, table_entries, window;
  int32_t rotary_dim, axes, pairing, norm;
  float norm_epsilon, softmax_scale;
  int32_t reserved;
  int64_t page_stride, head_stride, token_stride;
  int64_t scale_offset, turns_offset, axis_offset, region_bytes;
};
constexpr uint32_t kMagic = 0x4E54414Cu;

// A sequence's entries [first, end) of the page table; none where they leave it.
struct Pages {
  int first, count;
};
LF_DEVICE Pages pages_of(const Desc &d, int first, int end, bool &bad) {
  if (first < 0 || end < first || end > d.table_entries) {
    bad = true;
    return {0, 0};
  }
  return {first, end - first};
}

// Byte of (page, head, slot) in a cache region. Strides fit 31 bits, so each
// product is one 32 x 32 -> 64 multiplication.
template <bool E4M3>
LF_DEVICE uint64_t cache_byte(const Desc &d, int page, int head, int slot) {
  constexpr uint64_t size = E4M3 ? 1 : 2;
  return size * (static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(d.page_stride) +
                 static_cast<uint64_t>(static_cast<uint32_t>(head)) * static_cast<uint32_t>(d.head_stride) +
                 static_cast<uint64_t>(static_cast<uint32_t>(slot)) * static_cast<uint32_t>(d.token_stride));
}

// ---- append ---------------------------------------------------------------------

// Page and slot of a row of sequence s; page -1 where there is none.
struct Place {
  int page, slot;
};
LF_DEVICE Place place_of(const Desc &d, const int32_t *row_offsets, const int32_t *lengths,
                         const int32_t *page_offsets, const int32_t *page_indices, int s, int row) {
  bool bad = false;
  const Pages pages = pages_of(d, page_offsets[s], page_offsets[s + 1], bad);
  const int64_t token = static_cast<int64_t>(lengths[s]) - row_offsets[s + 1] + row;
  const int shift = __builtin_ctz(static_cast<uint32_t>(d.page_size));
  if (token < 0 || (token >> shift) >= pages.count) return {-1, 0};
  const int page = page_indices[pages.first + static_cast<int>(token >> shift)];
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(d.pages)) return {-1, 0};
  return {page, static_cast<int>(token & (d.page_size - 1))};
}

// ---- single-token attention -------------------------------------------------------

constexpr int kTileKeys = 32;
constexpr int kHeadTile = 16;

// Keys [lo, len) of a sequence, in `tiles` tiles from the one that holds lo;
// a sequence without keys has one tile, whose block writes its zeros.
struct Span {
  int first_tile, tiles, lo, len;
};
LF_DEVICE Span span_of(const Desc &d, int len, Pages p, bool &bad) {
  const int most = p.count * d.page_size;
  if (len < 0 || len > most) {
    bad = true;
    len = len < 0 ? 0 : most;
  }
  const int lo = d.window > 0 && len > d.window ? len - d.window : 0;
  const int first = lo / kTileKeys;
  const int end = (len + kTileKeys - 1) / kTileKeys;
  return {first, end > first ? end - first : 1, lo, len};
}

// A key tile is four groups of eight keys, each in one page. The table entry of
// the group that starts at key j, of a sequence whose keys that count are in the
// entries [first, end), end > first: groups before and behind those (a released
// page before the window, an unused one behind the length) take the nearest of
// them, and their keys are masked.
LF_DEVICE int entry_of(int first, int end, int shift, int j) {
  const int e = j >> shift;
  return e < first ? first : e < end ? e : end - 1;
}

// Bytes, all in 64 bits (a page's or a token's step may be up to 2^31 - 1 of them):
// of slot `slot` of a page from the head's first row, and from the first of a group
// of eight rows of lane 16 g + c's part of them, which is row c % 8, 16-byte chunk g,
// of keys, and row 4 g % 8, the c-th of 16 pieces of `piece` bytes, of values.
LF_DEVICE uint64_t row_byte(int page, int slot, uint32_t page_bytes, uint32_t token_bytes) {
  return static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_bytes +
         static_cast<uint64_t>(static_cast<uint32_t>(slot)) * token_bytes;
}
LF_DEVICE uint64_t key_lane(int c, int g, uint32_t token_bytes) {
  return static_cast<uint64_t>(static_cast<uint32_t>(c & 7)) * token_bytes + static_cast<uint32_t>(16 * g);
}
LF_DEVICE uint64_t value_lane(int c, int g, uint32_t token_bytes, int piece) {
  return static_cast<uint64_t>(static_cast<uint32_t>(4 * g & 7)) * token_bytes + static_cast<uint32_t>(c * piece);
}

LF_DEVICE int head_tiles_of(const Desc &d) {
  const int group = d.query_heads / d.kv_heads;
  return d.kv_heads * ((group + kHeadTile - 1) / kHeadTile);
}

// The step's sequences s0 .. s0 + n - 1 that are decoded.
struct Decoded {
  int s0, n;
};
LF_DEVICE Decoded decoded_of(const Desc &d, int s0, int n, int total) {
  total = total < 0 ? 0 : total > d.max_sequences ? d.max_sequences : total;
  s0 = s0 < 0 ? 0 : s0 > total ? total : s0;
  n = n < 0 ? 0 : n > total - s0 ? total - s0 : n;
  return {s0, n};
}

// The step's items are the key tiles of every (sequence, head tile) pair in
// turn: pair (i, ht) starts at prefix[i] head_tiles + ht tiles(i), where prefix
// adds up the tiles of the sequences before i. Block b holds the items [b share,
// (b + 1) share): a part of a pair is worth adding up from about kLeastShare
// tiles on, and pairs shorter than that get a block each while there are enough.
constexpr int kLeastShare = 8;
constexpr int kMostItems = INT32_MAX - (1 << 22);  // leaves the sums below room for blocks and pairs
LF_DEVICE int share_of(int items, int pairs, int blocks) {
  if (pairs < 1) return 1;
  const int share = (items + blocks - 1) / blocks, whole = (items + pairs - 1) / pairs;
  const int least = whole < kLeastShare ? whole : kLeastShare;
  return share > least ? share : least;
}

// A step whose pairs all are short is dealt out by pairs instead: block b holds the
// pairs [first, end), and none is cut. Heads of 128, 8 key heads, us by items and by
// pairs: 15 sequences of up to 179 keys 19.3 and 9.0, 64 of up to 300 27.7 and 19.8,
// 16 of up to 1000 23.8 and 19.0, 128 of up to 1000 88 and 84; one of 1000 13.2 and
// 15.2, so few pairs have to be shorter; steps of one tile per pair 0.3 slower. One
// longer sequence among short ones does not mind: 15 of 30 and one of 1000 18.7 and
// 16.5, 3 of 30 and one of 500 22.5 and 11.6. The rule does not see where pairs of full
// length leave blocks without one, or give some two: 4 of 1000 (32 pairs) 14.5 and
// 17.5, 33 of 1000 (264 pairs on 256 blocks) 31.5 and 37.0.
LF_DEVICE int whole_tiles(int pairs) { return pairs < 32 ? 16 : 32; }
struct PairRange {
  int first, end;
};
LF_DEVICE PairRange pairs_of(int block, int pairs, int blocks) {
  if (pairs <= blocks) return {block, block < pairs ? block + 1 : block};
  return {static_cast<int>(static_cast<int64_t>(block) * pairs / blocks),
          static_cast<int>(static_cast<int64_t>(block + 1) * pairs / blocks)};
}

// The sequence that item u belongs to (prefix rises by at least 1 a sequence).
LF_DEVICE int sequence_at(const int *prefix, int n, int head_tiles, int u) {
  int i = 0;
  for (int lo = 0, hi = n; lo < hi;) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] * head_tiles <= u) {
      i = mid;
      lo = mid + 1;
    } else {
      hi = mid;
    }
  }
  return i;
}

// The blocks first .. last that hold parts of the pair whose items are [begin,
// begin + tiles), and where block b's part goes: partial result 2 b if the pair
// is the first thing in the block's range, 2 b + 1 if it comes after another
// (only the pair's first block can, so no two parts share a place).
struct Parts {
  int first, last;
};
LF_DEVICE Parts parts_of(int begin, int tiles, int share) {
  return {begin / share, (begin + tiles - 1) / share};
}
LF_DEVICE int part_slot(int block, int begin, int share) { return 2 * block + (begin > block * share ? 1 : 0); }

// Parts are added up in groups of kGroup neighbours, from the pair's first on,
// then the groups. The sum of the group that starts at block `start` has a
// place of its own among the pairs of more than one group: of those, at most
// one first group and one later group start in a window of kGroup blocks.
constexpr int kGroup = 32;
LF_DEVICE int group_slot(int start, int first) { return 2 * (start / kGroup) + (start == first ? 1 : 0); }

}  // namespace attn
