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

constexpr int64_t kMaxWidth = int64_t(1) << 24;
// kernels/low_rank.hip
constexpr int64_t kChunk = 64;        // columns of x A^T per block
constexpr int64_t kColumnBlock = 256; // output columns per block
constexpr int64_t kHeaderBytes = 256;

// Rows of a block's tile: batches of single-token rows hold many adapters, so
// a tile is one 16-row product and its adapters go to blocks of their own; long
// runs of one adapter share its weights over 64 rows.
int64_t tile_rows(int64_t max_tokens) { return max_tokens <= 128 ? 16 : 64; }

// Blocks per tile, each taking every slots-th adapter of the tile's rows.
int64_t tile_slots(const lf_fp8_low_rank_desc *d) {
  return tile_rows(d->max_tokens) == 16 ? std::min<int64_t>(d->adapters, 16) : 1;
}

int64_t tiles(const lf_fp8_low_rank_desc *d) {
  const int64_t rows = tile_rows(d->max_tokens);
  return (d->max_tokens + rows - 1) / rows;
}

int64_t chunks(const lf_fp8_low_rank_desc *d) { return (int64_t(d->slices) * d->rank + kChunk - 1) / kChunk; }

int32_t splits_of(const lf_fp8_low_rank_desc *d) {
  const int64_t blocks = tiles(d) * tile_slots(d) * chunks(d);
  const int64_t most = std::max<int64_t>(1, d->hidden / 512);
  return static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(most, 512 / std::min<int64_t>(blocks, 512))));
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
  return d != nullptr && d->magic == LF_FP8_LOW_RANK_MAGIC && fields_ok(d) && d->splits == splits_of(d);
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
  *out = d;
  return LF_OK;
}

int64_t lunaflux_fp8_low_rank_workspace_bytes(const lf_fp8_low_rank_desc *d) {
  if (!desc_ok(d)) return -1;
  return kHeaderBytes + int64_t(d->splits) * d->max_tokens * d->slices * d->rank * 4;
}

int32_t lunaflux_fp8_low_rank_launch_geometry(int32_t entry, const lf_fp8_low_rank_desc *d, int32_t dims[7],
                                              char symbol[LF_FP8_SYMBOL_BYTES]) {
  if (!desc_ok(d) || dims == nullptr || symbol == nullptr) return LF_INVALID_ARGUMENT;
  const int rows = static_cast<int>(tile_rows(d->max_tokens));
  dims[0] = static_cast<int32_t>(tiles(d) * tile_slots(d));
  dims[2] = 1;
  switch (entry) {
    case LF_FP8_LOW_RANK_SHRINK:
      dims[1] = static_cast<int32_t>(chunks(d));
      dims[2] = d->splits;
      std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_low_rank_shrink_r%d", rows);
      break;
    case LF_FP8_LOW_RANK_EXPAND:
      dims[1] = static_cast<int32_t>((d->columns + kColumnBlock - 1) / kColumnBlock);
      std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_low_rank_expand_r%d", rows);
      break;
    default: return LF_INVALID_ARGUMENT;
  }
  if (dims[1] > LF_MAX_GRID_YZ) return LF_UNSUPPORTED;
  dims[3] = 256;
  dims[4] = dims[5] = 1;
  dims[6] = 0;
  return LF_OK;
}

}  // extern "C"
