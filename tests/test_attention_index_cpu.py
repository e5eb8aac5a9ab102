"""The attention kernels' index arithmetic (csrc/kernels/attention_index.h), run
on the CPU: for descriptors and steps of any kind, also ones whose offsets,
lengths and page indices are garbage, no place read or written lies outside
the regions the descriptor bounds; and for sound steps the cut of the key tiles
over blocks covers every tile once, and the join reads exactly the partial
results that the blocks leave."""
import os
import subprocess


from lunaflux_amd import build as native_build

KERNELS = os.path.join(native_build.CSRC, "kernels")

PROGRAM = r"""
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>
#define LF_DEVICE static inline
#include "attention_index.h"
using namespace attn;
#define CHECK(x) do { if (!(x)) { std::printf("FAIL line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)
static std::mt19937 rng(7);
static int pick(int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); }

static Desc desc() {
  Desc d{};
  d.kv_heads = pick(1, 8);
  d.query_heads = d.kv_heads * pick(1, 40);
  d.head_dim = 64 << pick(0, 2);
  d.page_size = 8 << pick(0, 7);
  d.pages = pick(1, 50);
  d.max_tokens = pick(1, 60);
  d.max_sequences = pick(1, 20);
  d.table_entries = pick(1, 100);
  d.window = pick(0, 2) ? 0 : pick(1, 700);
  d.token_stride = d.head_dim;
  d.head_stride = d.token_stride * d.page_size;
  d.page_stride = d.head_stride * d.kv_heads;
  return d;
}
static int64_t elements(const Desc &d) {
  return (d.pages - 1) * d.page_stride + (d.kv_heads - 1) * d.head_stride + (d.page_size - 1) * d.token_stride +
         d.head_dim;
}

// by pairs: every pair once, in order, in no more blocks than there are
static void by_pairs() {
  const int blocks = pick(0, 1) ? 256 : 512, pairs = pick(0, 3) ? pick(0, 3000) : 2048 * 1024 - pick(0, 3);
  int next = 0;
  for (int b = 0; b < blocks; ++b) {
    const PairRange r = pairs_of(b, pairs, blocks);
    if (r.first >= r.end) continue;
    CHECK(r.first == next && r.end <= pairs);
    CHECK(r.end - r.first <= (pairs + blocks - 1) / blocks);
    next = r.end;
  }
  CHECK(next == pairs);
}

static void hostile() {
  const Desc d = desc();
  auto garbage = [&](size_t n) {
    std::vector<int32_t> v(n);
    for (auto &x : v) {
      const int kind = pick(0, 3);
      x = kind == 0 ? pick(-5, 5) : kind == 1 ? pick(0, 3000) : kind == 2 ? static_cast<int32_t>(rng()) : pick(0, 40);
    }
    return v;
  };
  // regions of exactly the descriptor's sizes; .at() faults outside them
  auto counts = garbage(5), row_offsets = garbage(d.max_sequences + 1), lengths = garbage(d.max_sequences);
  auto page_offsets = garbage(d.max_sequences + 1), table = garbage(d.table_entries);
  const Decoded dec = decoded_of(d, counts[0], counts[1], counts[2]);
  CHECK(dec.s0 >= 0 && dec.n >= 0 && dec.s0 + dec.n <= d.max_sequences);
  for (int s = 0; s < d.max_sequences; ++s) {
    bool bad = false;
    const Pages p = pages_of(d, page_offsets[s], page_offsets[s + 1], bad);
    CHECK(p.first >= 0 && p.count >= 0 && p.first + p.count <= d.table_entries);
    const Span span = span_of(d, lengths[s], p, bad);
    CHECK(span.len >= 0 && span.len <= int64_t(p.count) * d.page_size && span.lo >= 0 && span.lo <= span.len);
    CHECK(span.tiles >= 1);
    const int shift = __builtin_ctz(d.page_size), first = span.lo >> shift, end = (span.len + d.page_size - 1) >> shift;
    CHECK(end <= p.count);
    if (span.len > 0) CHECK(end > first);
    for (int t = 0; t < span.tiles && span.len > 0; ++t) {
      const int base = (span.first_tile + t) * kTileKeys;
      CHECK(base < span.len);
      for (int j = base; j < base + kTileKeys; j += 8) {
        const int e = entry_of(first, end, shift, j);
        CHECK(e >= first && e < end && p.first + e < d.table_entries);
        for (int i = j; i < j + 8; ++i) {
          if (i >= span.lo && i < span.len) CHECK(e == i >> shift);   // keys that count are in their page
          // pages outside the cache are read as page 0
          for (int page = 0; page < d.pages; page += d.pages > 1 ? d.pages - 1 : 1) {
            for (int h = 0; h < d.kv_heads; ++h) {
              const uint64_t at = cache_byte<true>(d, page, h, i & (d.page_size - 1));
              CHECK(at + d.head_dim <= static_cast<uint64_t>(elements(d)));
              CHECK(cache_byte<false>(d, page, h, i & (d.page_size - 1)) == 2 * at);
            }
          }
        }
      }
    }
    for (int row = 0; row < d.max_tokens; ++row) {
      const Place place = place_of(d, row_offsets.data(), lengths.data(), page_offsets.data(), table.data(), s, row);
      CHECK(place.page >= -1 && place.page < d.pages && place.slot >= 0 && place.slot < d.page_size);
    }
  }
}

static void cut(int workers) {  // ranges
  Desc d = desc();
  const int n = pick(0, d.max_sequences), head_tiles = head_tiles_of(d);
  std::vector<int> prefix(n + 1, 0), tiles(n);
  for (int i = 0; i < n; ++i) {
    tiles[i] = pick(0, 4) ? pick(1, 5) : pick(1, 400);
    prefix[i + 1] = prefix[i] + tiles[i];
  }
  const int items = prefix[n] * head_tiles, share = share_of(items, n * head_tiles, workers);
  CHECK(share > 0 && int64_t(share) * workers >= items);
  std::vector<int> seen(items, 0);
  std::set<int> left, read, sums;
  for (int b = 0; b < workers; ++b) {
    const int begin = b * share, end = begin + share < items ? begin + share : items;
    for (int u = begin; u < end;) {
      const int i = sequence_at(prefix.data(), n, head_tiles, u);
      CHECK(prefix[i] * head_tiles <= u && u < prefix[i + 1] * head_tiles);
      const int within = u - prefix[i] * head_tiles, ht = within / tiles[i], t0 = within - ht * tiles[i];
      const int t1 = tiles[i] - t0 < end - u ? tiles[i] : t0 + (end - u);
      CHECK(t1 > t0 && ht < head_tiles);
      for (int t = t0; t < t1; ++t) seen[prefix[i] * head_tiles + ht * tiles[i] + t]++;
      if (t0 != 0 || t1 != tiles[i]) {
        const int slot = part_slot(b, u - t0, share);
        CHECK(slot >= 0 && slot < 2 * workers && left.insert(slot).second);
      }
      u += t1 - t0;
    }
  }
  for (int x : seen) CHECK(x == 1);
  for (int i = 0; i < n; ++i) {
    for (int ht = 0; ht < head_tiles; ++ht) {
      const int begin = prefix[i] * head_tiles + ht * tiles[i];
      const Parts parts = parts_of(begin, tiles[i], share);
      if (parts.first == parts.last) continue;
      for (int b = parts.first; b <= parts.last; ++b) {
        CHECK(read.insert(part_slot(b, begin, share)).second);
        if (b > parts.first) CHECK(part_slot(b, begin, share) == 2 * b);   // the kernel steps from part to part
      }
      if (parts.last - parts.first < kGroup) continue;
      for (int start = parts.first; start <= parts.last; start += kGroup) {
        const int place = group_slot(start, parts.first);
        CHECK(place >= 0 && place <= 2 * workers / kGroup + 1 && sums.insert(place).second);
        if (start > parts.first)
          CHECK(place == group_slot(parts.first, parts.first) - 1 + 2 * ((start - parts.first) / kGroup));
      }
    }
  }
  CHECK(left == read);
}

int main() {
  for (int i = 0; i < 300; ++i) by_pairs();
    hostile();
  const int workers[] = {1, 2, 7, 256, 1024, 2048};
  for (int i = 0; i < 600; ++i) cut(workers[i % 6]);
  std::printf("ok\n");
}
"""


def test_places_stay_in_bounds_and_tiles_are_covered_once(tmp_path):
    src = tmp_path / "index.cpp"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "index")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", KERNELS,
                    str(src), "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
