// low_rank.cpp - host side of the low-rank adapter section of
// include/lunaflux_fp8.h: the descriptor, workspace size and launch geometry.
// No device code here.
#include "lunaflux_fp8.h"
#include "lunaflux_hip.h"

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>

namespace {

constexpr int64_t kMaxWidth = int64_t(1) << 20;
constexpr int64_t kHeaderBytes = 256;  // kernels/low_rank.hip, kPartsAt

int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
int64_t cut(int64_t v, int64_t by) { return (v + by - 1) / by; }

// The one launch reads a slice's A once per 1024 columns and 16 rows, so A has to
// be small enough to come from L2 quickly, and gives each adapter of 16 rows a
// block. Against two launches (columns 4096 + 2 x 1024, hidden 4096, an adapter per
// row or so): 16 rows of rank 16, 64 and 128 9 us and 20, 17 and 24, 26 and 37; 61
// rows 13 and 25, 33 and 35, 53 and 45; 128 rows 19 and 31, 50 and 47, 84 and 64; 256
// rows 31 and 39, 83 and 83, 139 and 88.
int32_t one_launch_of(const lf_fp8_low_rank_desc *d) {
  const int64_t values = int64_t(d->rank) * d->hidden;
  return d->max_tokens <= 256 && values <= (1 << 19) && d->max_tokens * values <= (1 << 24) ? 1 : 0;
}

// A shrink block's rows and columns of x A^T; with 32 columns where there are no
// more, it does not load A's rows twice (509 rows, rank 32: 18.3 us, with 64 19.5).
constexpr int64_t kTileRows = 64;
int64_t chunk_of(const lf_fp8_low_rank_desc *d) { return int64_t(d->slices) * d->rank <= 32 ? 32 : 64; }
int64_t shrink_blocks(const lf_fp8_low_rank_desc *d) {
  return cut(d->max_tokens, kTileRows) * cut(int64_t(d->slices) * d->rank, chunk_of(d));
}

// Slices of hidden: four or more steps of 64 for each of a block's eight waves, and
// no more blocks than the chip has compute units. Every block of the second launch
// adds the slices up again: 509 rows of 14336 take 16.9 us in slices of 2048, 17.7 of
// 1024 and 18.5 of 2560, 800 rows 23, 31 and 24, 1000 rows of 4096 27, 30 and 32.
int32_t splits_of(const lf_fp8_low_rank_desc *d) {
  if (one_launch_of(d)) return 1;
  return static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>({16, d->hidden / 2048, 256 / shrink_blocks(d)})));
}

// Blocks that share a tile's adapters. In the two launches most tiles of long
// prompts have one, so that the other blocks are idle, but a tile of two must not
// take twice as long: 4093 rows of 8 adapters 84 us with one slot, 69 with two, 66
// with four.
int32_t slots_of(const lf_fp8_low_rank_desc *d) {
  const int64_t most = one_launch_of(d) ? 16 : std::max<int64_t>(2, std::min<int64_t>(8, 768 / shrink_blocks(d)));
  return static_cast<int32_t>(std::min<int64_t>(d->adapters, most));
}

// Rows of an expand block: 16, so that few rows still fill the chip, while that
// reads B from L2 rarely enough. Both launches with 16 and with 64: 200 rows of rank
// 16 15 us and 18, of rank 64 18 and 21; 509 rows 19 and 20, 29 and 23; 1600 rows 35
// and 23, 68 and 38.
int64_t expand_rows(const lf_fp8_low_rank_desc *d) {
  return d->max_tokens <= 512 && d->rank <= 64 && int64_t(d->max_tokens) * d->rank <= 16384 ? 16 : 64;
}

int64_t blocks_of(const lf_fp8_low_rank_desc *d, int64_t columns) {
  int64_t blocks = 0, begin = 0;
  for (int32_t i = 0; i < d->slices; ++i) {
    blocks += cut(d->ends[i] - begin, columns);
    begin = d->ends[i];
  }
  return blocks;
}

// Columns of a block: 1024 in one launch; 512 for 16 rows, 128 for each of four
// waves; 512 or 1024 for 64 rows, where each block starts with a chain of loads: 1024
// if that leaves most of the compute units a block. Columns 4096 + 2 x 1024, rank 64:
// 192 blocks of 1024 (2000 rows) take 40.0 us and as many rows with 512 38.5, 228 46.6
// and 48.4, 264 44.2 and 47.2, 300 46.3 and 49.5, 384 (4093 rows) 52.3 and 56.4, 768 94
// and 100 (112 with 2048); rank 16, 264 blocks 34.7 and 37.9.
int32_t block_columns_of(const lf_fp8_low_rank_desc *d) {
  if (one_launch_of(d)) return 1024;
  return expand_rows(d) == 64 && cut(d->max_tokens, 64) * blocks_of(d, 1024) >= 224 ? 1024 : 512;
}

int32_t column_blocks_of(const lf_fp8_low_rank_desc *d) { return static_cast<int32_t>(blocks_of(d, block_columns_of(d))); }

// Multiples of 8: XCDs have neighbouring blocks each.
int64_t shrink_grid(const lf_fp8_low_rank_desc *d) { return align_up(shrink_blocks(d) * splits_of(d), 8); }
int64_t expand_grid(const lf_fp8_low_rank_desc *d) {
  return align_up(cut(d->max_tokens, expand_rows(d)) * column_blocks_of(d), 8);
}

bool fields_ok(const lf_fp8_low_rank_desc *d) {
  if (d->adapters < 1 || d->adapters > 65536 || d->rank < 16 || d->rank > 128 || d->rank % 16 != 0 ||
      d->hidden < 128 || d->hidden > kMaxWidth || d->hidden % 128 != 0 || d->slices < 1 ||
      d->slices > LF_FP8_LOW_RANK_SLICES || d->max_tokens < 1 || d->max_tokens > (1 << 24) ||
      d->columns < 64 || d->columns > kMaxWidth) {
    return false;
  }
  int32_t before = 0;
  for (int32_t i = 0; i < d->slices; ++i) {
    if (d->ends[i] <= before || d->ends[i] % 64 != 0) return false;
    before = d->ends[i];
  }
  // HIP counts a grid's threads in 32 bits.
  return before == d->columns && shrink_grid(d) * 512 <= UINT32_MAX && expand_grid(d) * 256 <= UINT32_MAX;
}

bool desc_ok(const lf_fp8_low_rank_desc *d) {
  return d != nullptr && d->magic == LF_FP8_LOW_RANK_MAGIC && fields_ok(d) && d->splits == splits_of(d) &&
         d->slots == slots_of(d) && d->one_launch == one_launch_of(d) && d->column_blocks == column_blocks_of(d) &&
         d->block_columns == block_columns_of(d);
}

}  // namespace

extern "C" {

int32_t lunaflux_fp8_low_rank_descriptor(int32_t adapters, int32_t rank, int64_t hidden, const int64_t *widths,
                                         int32_t slices, int32_t max_tokens, lf_fp8_low_rank_desc *out) {
  if (out == nullptr || widths == nullptr || slices < 1 || slices > LF_FP8_LOW_RANK_SLICES || hidden < 1 ||
      hidden > kMaxWidth) {
    return LF_INVALID_ARGUMENT;
  }
  lf_fp8_low_rank_desc d;
  std::memset(&d, 0, sizeof(d));
  d.magic = LF_FP8_LOW_RANK_MAGIC;
  d.adapters = adapters;
  d.rank = rank;
  d.hidden = static_cast<int32_t>(hidden);
  d.slices = slices;
  d.max_tokens = max_tokens;
  int64_t columns = 0;
  for (int32_t i = 0; i < slices; ++i) {
    if (widths[i] < 1 || widths[i] > kMaxWidth) return LF_INVALID_ARGUMENT;
    columns += widths[i];
    d.ends[i] = static_cast<int32_t>(columns);
  }
  d.columns = static_cast<int32_t>(columns);
  if (!fields_ok(&d)) return LF_INVALID_ARGUMENT;
  d.splits = splits_of(&d);
  d.slots = slots_of(&d);
  d.one_launch = one_launch_of(&d);
  d.column_blocks = column_blocks_of(&d);
  d.block_columns = block_columns_of(&d);
  *out = d;
  return LF_OK;
}

int64_t lunaflux_fp8_low_rank_workspace_bytes(const lf_fp8_low_rank_desc *d) {
  if (!desc_ok(d)) return -1;
  if (d->one_launch) return kHeaderBytes;
  return kHeaderBytes + int64_t(d->splits) * d->max_tokens * d->slices * d->rank * 4;
}

int32_t lunaflux_fp8_low_rank_launch_geometry(int32_t entry, const lf_fp8_low_rank_desc *d, int32_t dims[7],
                                              char symbol[LF_FP8_SYMBOL_BYTES]) {
  if (!desc_ok(d) || dims == nullptr || symbol == nullptr) return LF_INVALID_ARGUMENT;
  if (entry < LF_FP8_LOW_RANK_ONE_LAUNCH || entry > LF_FP8_LOW_RANK_EXPAND) return LF_INVALID_ARGUMENT;
  if ((d->one_launch != 0) != (entry == LF_FP8_LOW_RANK_ONE_LAUNCH)) return LF_UNSUPPORTED;
  int64_t gx = 0, gy = 1, threads = 256;
  if (entry == LF_FP8_LOW_RANK_ONE_LAUNCH) {
    std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_low_rank_n%d", d->rank == 16 ? 1 : d->rank == 32 ? 2 : 4);
    gx = cut(d->max_tokens, 16) * d->slots;
    threads = 512;
    gy = d->column_blocks;
  } else if (entry == LF_FP8_LOW_RANK_SHRINK) {
    std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_low_rank_shrink_%dx%d", static_cast<int>(kTileRows),
                  static_cast<int>(chunk_of(d)));
    threads = 512;
    gx = shrink_grid(d);
  } else {
    std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_low_rank_expand_%dx%d", static_cast<int>(expand_rows(d)),
                  d->rank <= 32 ? 32 : d->rank <= 64 ? 64 : 128);
    gx = expand_grid(d);
  }
  // (the second launch's blocks come to a tile's adapters sooner: 400 rows of 16
  // adapters 55 us with eight slots there, 50 with four or two; 1600 rows of 5 in
  // runs of 100 44 with five or four, 45 with two, 48 with one)
  if (entry == LF_FP8_LOW_RANK_SHRINK) gy = d->slots;
  if (entry == LF_FP8_LOW_RANK_EXPAND) gy = std::min(d->slots, 4);
  dims[0] = static_cast<int32_t>(gx);
  dims[1] = static_cast<int32_t>(gy);
  dims[2] = 1;
  dims[3] = static_cast<int32_t>(threads);
  dims[4] = dims[5] = 1;
  dims[6] = 0;
  return LF_OK;
}

}  // extern "C"
