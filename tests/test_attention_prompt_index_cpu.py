"""The index arithmetic of prompts, windows with sinks and caches with scales by
blocks (csrc/kernels/attention_index.h), run on the CPU: for garbage steps no
place lies outside the regions that the descriptor bounds; for sound ones every
row and visible key is covered once, whatever the ranges are cut at, and the
join reads the partial results that the ranges leave."""
import os
import subprocess

from lunaflux_amd import build as native_build

KERNELS = os.path.join(native_build.CSRC, "kernels")

PROGRAM = r"""
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <algorithm>
#include <map>
#include <random>
#include <set>
#include <vector>
#define LF_DEVICE static inline
#include "attention_index.h"
using namespace attn;
#define CHECK(x) do { if (!(x)) { std::printf("FAIL line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)
static std::mt19937 rng(11);
static int pick(int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); }

static Desc desc() {
  Desc d{};
  d.kv_heads = pick(1, 8);
  d.query_heads = d.kv_heads * (pick(0, 5) ? pick(1, 40) : pick(100, 128));
  d.head_dim = 64 << pick(0, 2);
  d.page_size = 8 << pick(0, 7);
  d.pages = pick(1, 50);
  d.max_tokens = pick(1, 300);
  d.max_sequences = pick(1, 20);
  d.table_entries = pick(1, 200);
  d.window = pick(0, 2) ? 0 : pick(1, 700);
  d.sinks = pick(0, 1) ? 0 : pick(1, 200);
  d.block_tokens = std::min(16, d.page_size);
  d.token_stride = d.head_dim;
  d.head_stride = d.token_stride * d.page_size;
  d.page_stride = d.head_stride * d.kv_heads;
  return d;
}

struct Step {
  std::vector<int32_t> row_offsets, lengths, page_offsets, table;
  int n, rows;
};
static Step garbage(const Desc &d) {
  auto some = [&](size_t n) {
    std::vector<int32_t> v(n);
    for (auto &x : v) {
      const int kind = pick(0, 3);
      x = kind == 0 ? pick(-5, 5) : kind == 1 ? pick(0, 3000) : kind == 2 ? static_cast<int32_t>(rng()) : pick(0, 40);
    }
    return v;
  };
  return {some(d.max_sequences + 1), some(d.max_sequences), some(d.max_sequences + 1), some(d.table_entries), d.max_sequences,
          pick(0, d.max_tokens)};
}
// Sequences that fit: rows, and tokens before them.
static Step sound(const Desc &d) {
  Step s;
  s.n = pick(0, d.max_sequences);
  s.row_offsets = {0};
  s.page_offsets = {0};
  int rows = d.max_tokens, entries = d.table_entries;
  for (int i = 0; i < s.n; ++i) {
    const int most = entries * d.page_size;
    const int r = std::min(pick(0, 3) ? pick(0, 4) : pick(0, rows), std::min(rows, most));
    const int before = pick(0, 2) ? pick(0, std::min(most - r, 50)) : pick(0, most - r);
    const int pages = (r + before + d.page_size - 1) / d.page_size;
    s.row_offsets.push_back(s.row_offsets.back() + r);
    s.lengths.push_back(r + before);
    s.page_offsets.push_back(s.page_offsets.back() + pages);
    rows -= r;
    entries -= pages;
  }
  s.rows = s.row_offsets.back();
  s.table.assign(d.table_entries, 0);
  return s;
}

static void entries_of(const Desc &d, const Prompt &p, const PromptKeys &k, int tile_keys, int pages) {
  const int shift = __builtin_ctz(d.page_size);
  const int first = k.lo >> shift, end = (k.last >> shift) + 1, sink_end = (k.sink + d.page_size - 1) >> shift;
  CHECK(k.tiles >= 1 && k.sink_tiles <= k.first && k.last < pages * d.page_size);
  int before = -1;
  for (int t = 0; t < k.tiles; ++t) {
    const int base = tile_keys * (t < k.sink_tiles ? t : t + k.first - k.sink_tiles);
    CHECK(base > before && base <= k.last);
    before = base;
    for (int j = base; j < base + tile_keys; j += 8) {
      const int e = sink_entry_of(sink_end, first, end, shift, j);
      CHECK(e >= 0 && e < pages && p.entry + e < d.table_entries);
      for (int i = j; i < j + 8; ++i) {
        if (i <= k.last && (i >= k.lo || i < k.sink)) CHECK(e == i >> shift);  // keys that some row counts
      }
    }
  }
}

static void hostile() {
  const Desc d = desc();
  const Step s = garbage(d);
  const int tile_rows = 256, tile_keys = d.head_dim == 256 ? 32 : 64;
  const QueryTile q = query_tile_of(d, tile_rows);
  for (int i = 0; i < s.n; ++i) {
    bool bad = false;
    const Prompt p = prompt_of(d, s.row_offsets.data(), s.lengths.data(), s.page_offsets.data(), i, s.rows, bad);
    CHECK(p.rows >= 0 && p.row >= 0 && p.row + p.rows <= s.rows && p.before >= 0);
    if (p.rows == 0) continue;
    const int pages = s.page_offsets[i + 1] - s.page_offsets[i];
    CHECK(!bad && p.before + p.rows <= pages * d.page_size);
    int row = p.row;
    for (int b = 0; b < blocks_of(d, p); ++b) {
      const Block x = block_of(d, p, b);
      CHECK(x.entry >= 0 && x.entry < p.entry + pages && x.entry < d.table_entries);
      CHECK(x.slot >= 0 && x.slot % d.block_tokens == 0 && x.slot + d.block_tokens <= d.page_size);
      CHECK(x.lo >= 0 && x.lo < x.hi && x.hi <= d.block_tokens && x.row == row);
      CHECK(x.lo == 0 || b == 0);
      row += x.hi - x.lo;
      for (int page = 0; page < d.pages; ++page) {
        CHECK(scale_index(d, page, x.slot, d.kv_heads - 1) < uint64_t(d.pages) * (d.page_size / d.block_tokens) * d.kv_heads);
      }
    }
    CHECK(row == p.row + p.rows);
    for (int x = 0; x < weights_of(d, q, p).tiles; ++x) entries_of(d, p, keys_of(d, q, p, x, tile_keys), tile_keys, pages);
  }
  // decode
  for (int i = 0; i < s.n; ++i) {
    bool bad = false;
    const Pages pages = pages_of(d, s.page_offsets[i], s.page_offsets[i + 1], bad);
    const SinkSpan span = sink_span_of(d, s.lengths[i], pages, bad);
    const int len = span.span.len, lo = span.span.lo, shift = __builtin_ctz(d.page_size);
    if (len == 0) continue;
    const int first = lo >> shift, end = (len + d.page_size - 1) >> shift, sink_end = (span.sink + d.page_size - 1) >> shift;
    std::set<int> seen;
    for (int t = 0; t < span.span.tiles; ++t) {
      const int base = kTileKeys * (t < span.sink_tiles ? t : t + span.span.first_tile - span.sink_tiles);
      CHECK(base < len);
      for (int j = base; j < base + kTileKeys; j += 8) {
        const int e = sink_entry_of(sink_end, first, end, shift, j);
        CHECK(e >= 0 && e < pages.count);
        for (int k = j; k < j + 8 && k < len; ++k) {
          if (k < span.sink || k >= lo) CHECK(e == k >> shift && seen.insert(k).second);
        }
      }
    }
    CHECK(static_cast<int>(seen.size()) == len - lo + span.sink);
  }
}

static void weights() {
  Weights w{pick(1, 5000), pick(1, 300), 0, pick(1, 200)};
  w.cap = pick(0, 1) ? int64_t(1) << 40 : pick(1, 20000);
  int64_t sum = 0;
  for (int x = 0; x <= w.tiles; ++x) {
    CHECK(weight_before(w, x) == sum);
    if (x < w.tiles) {
      CHECK(tile_at(w, sum) == x && tile_at(w, sum + weight_of(w, x) - 1) == x);
      sum += weight_of(w, x);
    }
  }
}

// As the kernels go through a step, with `blocks` ranges.
static void cut(int blocks) {
  Desc d = desc();
  d.table_entries = pick(1, 1000);
  const Step s = sound(d);
  const int tile_rows = 256, tile_keys = d.head_dim == 256 ? 32 : 64;
  const QueryTile q = query_tile_of(d, tile_rows);
  const int64_t heads = int64_t(d.kv_heads) * q.subs;
  CHECK(q.heads * q.tokens <= tile_rows && q.heads * q.subs >= d.query_heads / d.kv_heads);
  std::vector<int64_t> prefix(s.n + 1, 0);
  std::vector<Prompt> prompts(s.n);
  for (int i = 0; i < s.n; ++i) {
    bool bad = false;
    prompts[i] = prompt_of(d, s.row_offsets.data(), s.lengths.data(), s.page_offsets.data(), i, s.rows, bad);
    CHECK(!bad && prompts[i].rows == s.row_offsets[i + 1] - s.row_offsets[i]);
    const Weights w = weights_of(d, q, prompts[i]);
    prefix[i + 1] = prefix[i] + weight_before(w, w.tiles);
  }
  const int64_t total = prefix[s.n] * heads, share = (total + blocks - 1) / blocks;
  typedef std::tuple<int, int64_t, int> Pair;
  std::map<Pair, std::vector<int>> seen;  // of each pair: how often each key tile
  std::map<Pair, std::vector<int>> left;  // partial results in order
  std::set<int> slots;
  for (int b = 0; b < blocks; ++b) {
    const int64_t u0 = b * share, u1 = std::min(u0 + share, total);
    if (u0 >= u1) continue;
    int i = prompt_at(prefix.data(), s.n, heads, u0);
    CHECK(prefix[i] * heads <= u0 && u0 < prefix[i + 1] * heads);
    Weights w = weights_of(d, q, prompts[i]);
    const int64_t first = prefix[i] * heads, each = prefix[i + 1] - prefix[i];
    int64_t head = (u0 - first) / each;
    int x = tile_at(w, u0 - first - head * each);
    int64_t begin = first + head * each + weight_before(w, x), weight = weight_of(w, x);
    CHECK(begin <= u0 && u0 < begin + weight);
    for (;;) {
      const PromptKeys k = keys_of(d, q, prompts[i], x, tile_keys);
      const int k0 = cut_of(u0, begin, weight, k.tiles), k1 = cut_of(u1, begin, weight, k.tiles);
      CHECK(k0 >= 0 && k1 <= k.tiles && k0 <= k1);
      if (k0 < k1) {
        auto &v = seen[{i, head, x}];
        v.resize(k.tiles);
        for (int t = k0; t < k1; ++t) v[t]++;
        if (k0 > 0 || k1 < k.tiles) {
          CHECK(k1 - k0 >= kCut && k.tiles >= 2 * kCut);
          const int slot = prompt_slot(b, k0 > 0);
          CHECK(slot >= 0 && slot < 2 * blocks && slots.insert(slot).second);
          left[{i, head, x}].push_back(slot);
        }
      }
      if (begin + weight >= u1) break;
      begin += weight;
      if (++x == w.tiles) {
        x = 0;
        if (++head == heads) {
          head = 0;
          do ++i;
          while (prefix[i] == prefix[i + 1]);
          w = weights_of(d, q, prompts[i]);
        }
      }
      weight = weight_of(w, x);
    }
  }
  for (int i = 0; i < s.n; ++i) {
    const Weights w = weights_of(d, q, prompts[i]);
    for (int64_t head = 0; head < heads; ++head) {
      for (int x = 0; x < w.tiles; ++x) {
        const PromptKeys k = keys_of(d, q, prompts[i], x, tile_keys);
        const auto &v = seen[{i, head, x}];
        CHECK(static_cast<int>(v.size()) == k.tiles);
        for (int n : v) CHECK(n == 1);
        // what a row counts lies in the tile's keys
        for (int p = k.first_position; p <= k.last; ++p) {
          const int lo = d.window > 0 ? std::max(0, p + 1 - d.window) : 0;
          CHECK(lo >= k.lo && (std::min(d.sinks, lo) <= k.sink || k.sink == k.lo));
        }
      }
    }
  }
  // the join: every range that holds a later part of a cut pair finds all its parts
  std::set<Pair> joined;
  for (int range = 1; range < blocks; ++range) {
    const int64_t u = range * share;
    if (u >= total) continue;
    const int i = prompt_at(prefix.data(), s.n, heads, u);
    const Weights w = weights_of(d, q, prompts[i]);
    const int64_t first = prefix[i] * heads, each = prefix[i + 1] - prefix[i], head = (u - first) / each;
    const int x = tile_at(w, u - first - head * each);
    const int64_t begin = first + head * each + weight_before(w, x), weight = weight_of(w, x);
    const PromptKeys k = keys_of(d, q, prompts[i], x, tile_keys);
    auto at = [&](int b) { return cut_of(b * share, begin, weight, k.tiles); };
    if (at(range) == 0 || at(range) >= at(range + 1)) continue;
    std::vector<int> parts;
    int own = -1;
    for (int t = 0; t < 256; ++t) {
      const int b = static_cast<int>(begin / share) + t;
      if (b < blocks && at(b) < at(b + 1)) {
        if (b == range) own = static_cast<int>(parts.size());
        parts.push_back(prompt_slot(b, at(b) > 0));
      }
    }
    CHECK((parts == left[{i, head, x}]) && own >= 1);
    joined.insert({i, head, x});
  }
  for (auto &l : left) CHECK(joined.count(l.first) == 1);
}

int main() {
  for (int i = 0; i < 4000; ++i) hostile();
  for (int i = 0; i < 2000; ++i) weights();
  const int blocks[] = {1, 2, 7, 40, 256};
  for (int i = 0; i < 1500; ++i) cut(blocks[i % 5]);
  std::set<int> ranges;
  for (int b = 0; b < 256; ++b) CHECK(range_of_block(b, 256) < 256 && ranges.insert(range_of_block(b, 256)).second);
  std::printf("ok\n");
}
"""


def test_prompts_stay_in_bounds_and_are_covered_once(tmp_path):
    src = tmp_path / "index.cpp"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "index")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", KERNELS,
                    str(src), "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
