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
// kernels/low_rank.hip
constexpr int64_t kChunk = 64;         // columns of x A^T per block
constexpr int64_t kColumnBlock = 512;  // output columns per block
constexpr int64_t kHeaderBytes = 256, kCounterBytes = 256;

// Rows of a block's tile: batches of few rows hold many adapters, so a tile is
// one 16-row product and its adapters go to blocks of their own; long runs of
// one adapter share its weights over 64 rows.
int64_t tile_rows(const lf_fp8_low_rank_desc *d) { return d->max_tokens <= 512 ? 16 : 64; }

int64_t tiles(const lf_fp8_low_rank_desc *d) {
  const int64_t rows = tile_rows(d);
  return (d->max_tokens + rows - 1) / rows;
}

int64_t chunks(const lf_fp8_low_rank_desc *d) { return (int64_t(d->slices) * d->rank + kChunk - 1) / kChunk; }

// Blocks per tile, each taking every slots-th adapter of the tile's rows.
int32_t slots_of(const lf_fp8_low_rank_desc *d) {
  return std::min<int32_t>(d->adapters, d->max_tokens <= 128 ? 16 : d->max_tokens <= 512 ? 4 : 2);
}

// Slices of hidden: two or more steps of 64 for each of a block's four waves,
// and no more blocks than the chip holds at once.
int32_t splits_of(const lf_fp8_low_rank_desc *d) {
  const int64_t blocks = tiles(d) * chunks(d);
  const int64_t most = std::min<int64_t>(16, std::max<int64_t>(1, d->hidden / 512));
  return static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(most, 768 / std::min<int64_t>(blocks, 768))));
}

int32_t column_blocks_of(const lf_fp8_low_rank_desc *d) {
  int64_t blocks = 0, begin = 0;
  for (int32_t i = 0; i < d->slices; ++i) {
    blocks += (d->ends[i] - begin + kColumnBlock - 1) / kColumnBlock;
    begin = d->ends[i];
  }
  return static_cast<int32_t>(blocks);
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
  return before == d->columns;
}

bool desc_ok(const lf_fp8_low_rank_desc *d) {
  return d != nullptr && d->magic == LF_FP8_LOW_RANK_MAGIC && fields_ok(d) && d->splits == splits_of(d) &&
         d->slots == slots_of(d) && d->column_blocks == column_blocks_of(d);
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
  d.column_blocks = column_blocks_of(&d);
  *out = d;
  return LF_OK;
}

int64_t lunaflux_fp8_low_rank_workspace_bytes(const lf_fp8_low_rank_desc *d) {
  if (!desc_ok(d)) return -1;
  const int64_t counted = tile_rows(d) == 16 ? tiles(d) * d->slots : 0;
  return kHeaderBytes + counted * kCounterBytes + int64_t(d->splits) * d->max_tokens * d->slices * d->rank * 4;
}

int32_t lunaflux_fp8_low_rank_launch_geometry(int32_t entry, const lf_fp8_low_rank_desc *d, int32_t dims[7],
                                              char symbol[LF_FP8_SYMBOL_BYTES]) {
  if (!desc_ok(d) || dims == nullptr || symbol == nullptr) return LF_INVALID_ARGUMENT;
  const bool one = tile_rows(d) == 16;
  if (entry < LF_FP8_LOW_RANK_ONE_LAUNCH || entry > LF_FP8_LOW_RANK_EXPAND) return LF_INVALID_ARGUMENT;
  if (one != (entry == LF_FP8_LOW_RANK_ONE_LAUNCH)) return LF_UNSUPPORTED;
  const int64_t pairs = tiles(d) * d->slots;
  int64_t gx = pairs, gy = 1, gz = 1;
  const char *name = "lf_low_rank_r16";
  if (one) {
    gx = pairs * (chunks(d) * d->splits + d->column_blocks);
  } else if (entry == LF_FP8_LOW_RANK_SHRINK) {
    name = "lf_low_rank_shrink_r64";
    gy = chunks(d);
    gz = d->splits;
  } else {
    name = "lf_low_rank_expand_r64";
    gy = d->column_blocks;
  }
  std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "%s", name);
  dims[0] = static_cast<int32_t>(gx);
  dims[1] = static_cast<int32_t>(gy);
  dims[2] = static_cast<int32_t>(gz);
  dims[3] = 256;
  dims[4] = dims[5] = 1;
  dims[6] = 0;
  return LF_OK;
}

}  // extern "C"
