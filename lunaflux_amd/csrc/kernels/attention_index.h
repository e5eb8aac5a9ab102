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
  int32_t sinks, block_tokens;
  int64_t block_scales;
};
constexpr uint32_t kMagic = 0x4E54414Cu;
constexpr int kCacheBf16 = 1, kCacheE4m3 = 2, kCacheBlocks = 3;

// A block of a cache with a scale per block and head: 8 or 16 tokens of one page.
// Index of its scale in the table behind a cache's codes.
LF_DEVICE int block_shift(const Desc &d) { return d.block_tokens == 8 ? 3 : 4; }
LF_DEVICE uint64_t scale_index(const Desc &d, int page, int slot, int head) {
  const int shift = block_shift(d);
  return (static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(d.page_size >> shift) +
          static_cast<uint32_t>(slot >> shift)) *
             static_cast<uint32_t>(d.kv_heads) +
         static_cast<uint32_t>(head);
}

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

// Rows of a step that one sequence has, with what is cached before them; none where the
// step contradicts itself or leaves its bounds (rows: the step's live rows).
struct Prompt {
  int row, rows, before, entry;  // first row, their number, tokens before, first page table entry
};
LF_DEVICE Prompt prompt_of(const Desc &d, const int32_t *row_offsets, const int32_t *lengths,
                           const int32_t *page_offsets, int s, int rows, bool &bad) {
  const int r0 = row_offsets[s], r1 = row_offsets[s + 1], len = lengths[s];
  const Pages pages = pages_of(d, page_offsets[s], page_offsets[s + 1], bad);
  if (r0 < 0 || r1 < r0 || r1 > rows || len < r1 - r0 || len > pages.count * d.page_size) {
    bad = true;
    return {0, 0, 0, 0};
  }
  return {r0, r1 - r0, len - (r1 - r0), pages.first};
}

// Blocks of tokens with a scale of their own that the rows fall into.
LF_DEVICE int blocks_of(const Desc &d, const Prompt &p) {
  const int shift = block_shift(d);
  return p.rows < 1 ? 0 : ((p.before + p.rows - 1) >> shift) - (p.before >> shift) + 1;
}

// The b-th of them: its first slot in its page, the slots [lo, hi) that rows are written
// to, the row of the first, and the page table entry.
struct Block {
  int entry, slot, lo, hi, row;
};
LF_DEVICE Block block_of(const Desc &d, const Prompt &p, int b) {
  const int shift = block_shift(d), first = ((p.before >> shift) + b) << shift;  // token
  const int lo = first < p.before ? p.before - first : 0;
  const int end = p.before + p.rows - first, hi = end < d.block_tokens ? end : d.block_tokens;
  return {p.entry + (first >> __builtin_ctz(static_cast<uint32_t>(d.page_size))), first & (d.page_size - 1), lo, hi,
          p.row + first + lo - p.before};
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

// With sinks: the first `sink` keys count too. The tiles are those of the sinks, then
// those of the window, without the ones between: tile t holds the keys from
// kTileKeys (t, or t + first_tile - sink_tiles from sink_tiles on).
struct SinkSpan {
  Span span;
  int sink, sink_tiles;
};
LF_DEVICE int sink_tiles_of(int sink, int first_tile, int tile_keys) {
  const int t = (sink + tile_keys - 1) / tile_keys;
  return t < first_tile ? t : first_tile;
}
LF_DEVICE SinkSpan sink_span_of(const Desc &d, int len, Pages p, bool &bad) {
  SinkSpan s = {span_of(d, len, p, bad), 0, 0};
  s.sink = d.sinks < s.span.lo ? d.sinks : s.span.lo;
  s.sink_tiles = sink_tiles_of(s.sink, s.span.first_tile, kTileKeys);
  s.span.tiles += s.sink_tiles;
  return s;
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

// With sinks, where the keys that count are in the entries [0, sink_end) and [first, end):
// a group between takes the last of the sinks' (of the window's first, without sinks).
LF_DEVICE int sink_entry_of(int sink_end, int first, int end, int shift, int j) {
  const int e = j >> shift;
  if (e >= first) return e < end ? e : end - 1;
  return e < sink_end ? e : sink_end > 0 ? sink_end - 1 : first;
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

// ---- attention of prompts -------------------------------------------------------------

// A block's query tile: `tokens` consecutive rows of a sequence with all `heads` query heads
// of a key head, row-major (token, head) in the tile; where a group has more heads than the
// tile has rows, one token with `heads` of them at a time, `subs` times.
struct QueryTile {
  int tokens, heads, subs;
};
LF_DEVICE QueryTile query_tile_of(const Desc &d, int tile_rows) {
  const int group = d.query_heads / d.kv_heads;
  if (group > tile_rows) return {1, tile_rows, (group + tile_rows - 1) / tile_rows};
  return {tile_rows / group, group, 1};
}

// The step's pairs are (sequence, key head and part of its group, query tile), tiles
// innermost. A pair weighs the keys that its tile sees, without their rounding to key tiles,
// and kPairKeys for what it takes whatever its keys are: min(a + step x, cap) for tile x of a
// sequence, so that sums over x have a closed form. The blocks take equal ranges of weight.
// (kPairKeys by what pairs take apart from their keys, us with 64, 256 and 512 of them: 8192 rows of heads of 128
// 619, 564 and 566, four prompts of up to 2039 rows 174, 158 and 163, of heads of 64 114, 105 and 110, windows of
// 1021 146, 150 and 152; few rows behind a cache, 1209 to 2545 of heads of 256 and one prompt of 1506 within 2 %.)
constexpr int kPairKeys = 256;
struct Weights {
  int64_t a, step, cap, rising;  // rising: the tiles that weigh less than cap
  int tiles;
};
// floor(a / b) for 0 <= a < 2^52 and 0 < b < 2^52 with a quotient below 2^31 (or what the rounded division gives):
// a twentieth of the instructions of a 64-bit integer division.
LF_DEVICE int64_t quotient(int64_t a, int64_t b) {
  return static_cast<int64_t>(static_cast<double>(a) / static_cast<double>(b));
}
LF_DEVICE Weights weights_of(const Desc &d, const QueryTile &q, const Prompt &p) {
  Weights w;
  w.tiles = (p.rows + q.tokens - 1) / q.tokens;
  w.step = q.tokens;
  w.a = static_cast<int64_t>(p.before) + q.tokens + kPairKeys;
  w.cap = d.window > 0 ? static_cast<int64_t>(d.window) + d.sinks + q.tokens + kPairKeys : int64_t(1) << 40;
  w.rising = d.window == 0 ? w.cap : w.a < w.cap ? quotient(w.cap - w.a + w.step - 1, w.step) : 0;
  return w;
}
LF_DEVICE int64_t weight_of(const Weights &w, int x) {
  const int64_t v = w.a + w.step * x;
  return v < w.cap ? v : w.cap;
}
// Weight of the tiles before x.
LF_DEVICE int64_t weight_before(const Weights &w, int x) {
  const int64_t rising = w.rising < x ? w.rising : x;
  return w.a * rising + w.step * (rising * (rising - 1) / 2) + w.cap * (x - rising);
}
// The tile in which weight r < weight_before(tiles) lies.
LF_DEVICE int tile_at(const Weights &w, int64_t r) {
  int lo = 0;
  for (int hi = w.tiles; hi - lo > 1;) {
    const int mid = lo + ((hi - lo) >> 1);
    if (weight_before(w, mid) <= r) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// The sequence that weight u of the step belongs to: prefix[i] (of n + 1) adds up the
// weights of one head's tiles in the sequences before i, and each has `heads` of them.
LF_DEVICE int prompt_at(const int64_t *prefix, int n, int64_t heads, int64_t u) {
  int lo = 0;  // the last i with prefix[i] heads <= u, so one with tiles
  for (int hi = n; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] * heads <= u) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// Keys of query tile x: those of [lo, last] and the first `sink`; key tiles as those of a
// SinkSpan, tile t from key tile_keys (t, or t + first - sink_tiles from sink_tiles on).
struct PromptKeys {
  int first_position, last;  // of the tile's rows
  int lo, sink, sink_tiles, first, tiles;
};
LF_DEVICE PromptKeys keys_of(const Desc &d, const QueryTile &q, const Prompt &p, int x, int tile_keys) {
  PromptKeys k;
  const int from = x * q.tokens, rest = p.rows - from;
  k.first_position = p.before + from;
  k.last = k.first_position + (rest < q.tokens ? rest : q.tokens) - 1;
  k.lo = d.window > 0 && k.first_position >= d.window ? k.first_position + 1 - d.window : 0;
  k.sink = d.sinks < k.lo ? d.sinks : k.lo;
  k.first = k.lo / tile_keys;
  k.sink_tiles = sink_tiles_of(k.sink, k.first, tile_keys);
  k.tiles = k.sink_tiles + k.last / tile_keys + 1 - k.first;
  return k;
}

// Where weight u cuts a pair of [begin, begin + weight) with `tiles` key tiles: at a multiple
// of `cut` of them, so that no part is shorter (but a pair itself may be). Does not fall as u rises.
// (Shorter parts cost their beginning, end and place in the join, longer ones equal ranges. us with 8 and 16:
// windows of 1021 150 and 135, four prompts of heads of 128 158 and 167, of 64 105 and 116, heads of 256 170 and
// 178, 8192 rows alike.)
constexpr int kCut = 8;
// In steps of little work (share, a block's weight, below 8 tiles of 64 keys) long pairs are cut at every fourth
// tile instead. us with 8 and 4: 69 rows behind 3244 tokens, 28/4 heads of 128, 47 and 34; 3 prompts of 8 rows
// behind 6566, 16/2, 41 and 30; 2 of 14 behind 40776, 5/1 of 64, 36 and 32. Cut at 4 beyond that (when the rule was
// made, before later steps): windows of 1021 156 and 166, pairs of up to 24 tiles (1506 rows of 8 heads of 64) 35 and
// 42, tiles of 32 keys (1209 rows, 16/8 heads of 256) 69 and 102.
LF_DEVICE int cut_tiles(int64_t share, int tile_keys) { return tile_keys == 64 && share < kCut * 64 ? kCut / 2 : kCut; }
LF_DEVICE int cut_of(int64_t u, int64_t begin, int64_t weight, int tiles, int cut = kCut) {
  if (u <= begin) return 0;
  if (u >= begin + weight) return tiles;
  const int k = static_cast<int>(static_cast<double>(u - begin) * tiles / static_cast<double>(weight) + 0.5);
  if (tiles < 4 * kCut) cut = kCut;
  const int c = (k + cut / 2) / cut * cut;
  return tiles - c < cut ? tiles : c;
}

// Whether the rows of a query tile can count keys enough for it to be cut: 2 kCut key tiles. (The host sizes the
// workspace and leaves out the join by it. T: Desc, or the structure that it mirrors.)
template <class T>
LF_DEVICE bool cuts_prompts(const T &d, int tile_rows, int tile_keys) {
  const int group = d.query_heads / d.kv_heads;
  int64_t longest = static_cast<int64_t>(d.table_entries) * d.page_size;
  const int64_t seen = static_cast<int64_t>(d.window) + (group > tile_rows ? 1 : tile_rows / group) + d.sinks + 2 * tile_keys;
  if (d.window > 0 && seen < longest) longest = seen;
  return (longest + tile_keys - 1) / tile_keys >= 2 * kCut;
}

// Block b of the grid (as many blocks as CUs) takes the b-th range of weight of those with
// the XCD in the upper bits: neighbours in weight, which share keys, share an XCD's L2.
LF_DEVICE int range_of_block(int b, int blocks) { return (b & 7) * (blocks >> 3) + (b >> 3); }

// Partial result of range b: of a pair cut before it, or of one that it begins and does not end. (The first, of a
// pair cut before range 0, never is.)
LF_DEVICE int prompt_slot(int b, bool begun_before) { return 2 * b + (begun_before ? 0 : 1); }

}  // namespace attn
