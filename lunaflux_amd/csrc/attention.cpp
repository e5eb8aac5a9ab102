// attention.cpp - host side of the attention section of
// include/lunaflux_fp8.h: the descriptor region, workspace sizes and launch
// geometry. No device code here.
#include "lunaflux_fp8.h"
#include "lunaflux_hip.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>

#define LF_DEVICE static inline
#include "kernels/attention_index.h"

namespace {

constexpr int64_t kLimit32 = (int64_t(1) << 31) - 1;
// kernels/attention.hip
constexpr int64_t kTileKeys = 32;
constexpr int64_t kGroup = 32;
constexpr int64_t kHeadTile = 16;
constexpr int64_t kMostItems = kLimit32 - (1 << 22);  // attention_index.h
constexpr int64_t kWaves = 4;
// kernels/attention_prompt.hip
constexpr int64_t kPromptBlocks = 256;
constexpr int64_t kJoinSlices = 8;
// Blocks of the append to an E4M3_BLOCKS cache that write keys and values; each goes on
// in steps of the grid.
constexpr int64_t kMostAppendBlocks = 1 << 14;

int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

bool power_of_two(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }

int64_t element_bytes(const lf_fp8_attn_desc *d) { return d->cache == LF_FP8_CACHE_BF16 ? 2 : 1; }

// Tiles of up to 16 query heads that read one key head.
int64_t head_tiles(const lf_fp8_attn_desc *d) {
  return d->kv_heads * ((d->query_heads / d->kv_heads + kHeadTile - 1) / kHeadTile);
}

int64_t last_element(const lf_fp8_attn_desc *d) {
  return (d->pages - 1) * d->page_stride + (d->kv_heads - 1) * d->head_stride +
         (d->page_size - 1) * d->token_stride + d->head_dim;
}

// No two rows of D elements overlap: with the dimensions sorted by stride,
// each stride steps over everything the smaller ones span.
bool strides_ok(const lf_fp8_attn_desc *d) {
  struct Dim {
    int64_t stride, count;
  } dims[3] = {{d->page_stride, d->pages}, {d->head_stride, d->kv_heads}, {d->token_stride, d->page_size}};
  for (const Dim &x : dims) {
    const int64_t bytes = x.stride > 0 && x.stride <= kLimit32 ? x.stride * element_bytes(d) : 0;
    if (bytes <= 0 || bytes > kLimit32 || bytes % 16 != 0) return false;
  }
  std::sort(dims, dims + 3, [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
  int64_t span = d->head_dim;
  for (const Dim &x : dims) {
    if (x.count == 1) continue;  // its stride is not stepped
    if (x.stride < span) return false;
    span += (x.count - 1) * x.stride;
  }
  return true;
}

bool fields_ok(const lf_fp8_attn_desc *d) {
  if (d->query_heads < 1 || d->kv_heads < 1 || d->query_heads > 1024 || d->query_heads % d->kv_heads != 0 ||
      (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) ||
      (d->cache != LF_FP8_CACHE_BF16 && d->cache != LF_FP8_CACHE_E4M3 && d->cache != LF_FP8_CACHE_E4M3_BLOCKS) || !power_of_two(d->page_size) ||
      d->page_size < 8 || d->page_size > 1024 || d->pages < 1 || d->max_tokens < 1 || d->max_sequences < 1 ||
      d->max_sequences > LF_FP8_ATTN_MAX_SEQUENCES || d->table_entries < 1 || d->window < 0 || d->sinks < 0) {
    return false;
  }
  if (d->rotary_dim < 0 || d->rotary_dim % 16 != 0 || d->rotary_dim > d->head_dim || d->axes < 1 ||
      d->axes > 4 || (d->pairing != LF_FP8_PAIR_HALF && d->pairing != LF_FP8_PAIR_NEIGHBOUR) ||
      (d->norm != 0 && d->norm != 1) || !std::isfinite(d->softmax_scale)) {
    return false;
  }
  if (d->norm == 1 && !(d->norm_epsilon >= 0.0f && std::isfinite(d->norm_epsilon))) return false;
  // The kernels count cached tokens, positions and (key tile, head tile) items in 31
  // bits, HIP a grid's threads in 32.
  if (int64_t(d->table_entries) * d->page_size > kLimit32 - 1024 ||
      int64_t(d->max_tokens) * d->axes > kLimit32 || d->max_tokens >= (1 << 24) ||
      (int64_t(d->table_entries) * d->page_size / kTileKeys + 2 * d->max_sequences) * head_tiles(d) > kMostItems) {
    return false;
  }
  if (d->cache == LF_FP8_CACHE_E4M3_BLOCKS && d->max_tokens >= (1 << 24) - kMostAppendBlocks) return false;
  return true;
}

// The region's parts behind the descriptor.
void lay_out(lf_fp8_attn_desc *d) {
  d->scale_offset = LF_FP8_ATTN_DESC_BYTES;
  d->turns_offset = d->scale_offset + align_up(int64_t(2) * d->kv_heads * 4, 256);
  d->axis_offset = d->turns_offset + align_up(int64_t(d->rotary_dim) / 2 * 8, 256);
  d->region_bytes = d->axis_offset + align_up(int64_t(d->rotary_dim) / 2 * 4, 256);
  const bool blocks = d->cache == LF_FP8_CACHE_E4M3_BLOCKS;
  d->block_tokens = blocks ? std::min<int32_t>(d->page_size, 16) : 0;
  d->block_scales = blocks ? align_up(last_element(d), 256) : 0;
}

bool laid_out(const lf_fp8_attn_desc *d) {
  lf_fp8_attn_desc r = *d;
  lay_out(&r);
  return d->scale_offset == r.scale_offset && d->turns_offset == r.turns_offset && d->axis_offset == r.axis_offset &&
         d->region_bytes == r.region_bytes && d->block_tokens == r.block_tokens && d->block_scales == r.block_scales;
}

bool desc_ok(const lf_fp8_attn_desc *d) {
  return d != nullptr && d->magic == LF_FP8_ATTN_MAGIC && fields_ok(d) && strides_ok(d) && laid_out(d);
}

int64_t tile_rows(const lf_fp8_attn_desc *d) {
  return std::min<int64_t>(d->query_heads / d->kv_heads, kHeadTile);
}

// kernels/attention.hip, blocks: blocks of the decode grid.
int64_t decode_blocks(const lf_fp8_attn_desc *d) {
  return d->head_dim * element_bytes(d) <= 128 ? 512 : 256;
}

// The decode workspace: a line with the error word, two arrival counters per
// partial result, two partial results per block (fp32 [rows][D] sums, maxima
// and weight sums of a head tile's rows) and the groups' sums.
int64_t decode_bytes(const lf_fp8_attn_desc *d) {
  const int64_t places = 2 * decode_blocks(d);
  return LF_FP8_ATTN_STATUS_BYTES + 2 * places * 4 +
         (places + places / kGroup + 2) * tile_rows(d) * (d->head_dim + 2) * 4;
}

// kernels/attention_prompt.hip: query rows and keys of a block's tiles.
constexpr int kPromptRows = 256;
int64_t prompt_keys(const lf_fp8_attn_desc *d) { return d->head_dim == 256 ? 32 : 64; }

bool prompt_cuts(const lf_fp8_attn_desc *d) { return attn::cuts_prompts(*d, kPromptRows, static_cast<int>(prompt_keys(d))); }

// Its workspace: a line with the error word, and, if tiles can be cut, two partial results per block (fp32 [rows][D]
// sums, maxima and weight sums; the first, of no use, has the starts of the blocks' ranges).
int64_t prompt_bytes(const lf_fp8_attn_desc *d) {
  return LF_FP8_ATTN_STATUS_BYTES +
         (prompt_cuts(d) ? 2 * kPromptBlocks * kPromptRows * (d->head_dim + 2) * 4 : 0);
}

// Blocks that write an E4M3_BLOCKS cache: four heads' keys or values of one block of tokens each.
int64_t append_blocks(const lf_fp8_attn_desc *d) {
  const int64_t touched = std::min<int64_t>(d->max_tokens, d->max_tokens / d->block_tokens + 2 * int64_t(d->max_sequences));
  return std::min(kMostAppendBlocks, touched * 2 * ((d->kv_heads + kWaves - 1) / kWaves));
}

const char *cache_name(const lf_fp8_attn_desc *d) {
  return d->cache == LF_FP8_CACHE_BF16 ? "bf16" : d->cache == LF_FP8_CACHE_E4M3 ? "e4m3" : "e4m3_blocks";
}

}  // namespace

extern "C" {

int32_t lunaflux_fp8_attn_descriptor(lf_fp8_attn_desc *d) { return lunaflux_fp8_attn_descriptor_sinks(d, 0); }

int32_t lunaflux_fp8_attn_descriptor_sinks(lf_fp8_attn_desc *d, int32_t sinks) {
  if (d == nullptr) return LF_INVALID_ARGUMENT;
  lf_fp8_attn_desc r = *d;
  r.magic = LF_FP8_ATTN_MAGIC;
  r.reserved = 0;
  r.sinks = sinks;
  std::memset(r.padding, 0, sizeof(r.padding));
  if (!fields_ok(&r)) return LF_INVALID_ARGUMENT;
  if (r.page_stride == 0 && r.head_stride == 0 && r.token_stride == 0) {
    r.token_stride = r.head_dim;
    r.head_stride = int64_t(r.page_size) * r.head_dim;
    r.page_stride = r.kv_heads * r.head_stride;
  }
  if (!strides_ok(&r)) return LF_INVALID_ARGUMENT;
  lay_out(&r);
  *d = r;
  return LF_OK;
}

int32_t lunaflux_fp8_attn_region(const lf_fp8_attn_desc *d, const float *scales, int64_t scale_count,
                                 const double *turns, const int32_t *axis, int64_t pair_count,
                                 uint8_t *region, int64_t region_bytes) {
  if (!desc_ok(d) || region == nullptr || region_bytes != d->region_bytes) return LF_INVALID_ARGUMENT;
  const int64_t pairs = d->rotary_dim / 2;
  if (pair_count != pairs || (pairs > 0 && (turns == nullptr || axis == nullptr))) return LF_INVALID_ARGUMENT;
  if (scales == nullptr ? (scale_count != 0 || d->cache == LF_FP8_CACHE_E4M3)
                        : scale_count != 2 * d->kv_heads || d->cache == LF_FP8_CACHE_E4M3_BLOCKS) {
    return LF_INVALID_ARGUMENT;
  }
  for (int64_t i = 0; i < scale_count; ++i) {
    // 1 / scale is what the append multiplies by: it has to be finite too
    if (!(scales[i] > 0.0f) || !std::isfinite(scales[i]) || !std::isfinite(1.0f / scales[i])) {
      return LF_INVALID_ARGUMENT;
    }
    if (d->cache == LF_FP8_CACHE_BF16 && scales[i] != 1.0f) return LF_INVALID_ARGUMENT;
  }
  for (int64_t i = 0; i < pairs; ++i) {
    if (!std::isfinite(turns[i]) || axis[i] < 0 || axis[i] >= d->axes) return LF_INVALID_ARGUMENT;
  }
  std::memset(region, 0, static_cast<size_t>(region_bytes));
  std::memcpy(region, d, sizeof(*d));
  float *s = reinterpret_cast<float *>(region + d->scale_offset);
  for (int64_t i = 0; i < 2 * d->kv_heads; ++i) s[i] = scales == nullptr ? 1.0f : scales[i];
  if (pairs > 0) {
    std::memcpy(region + d->turns_offset, turns, static_cast<size_t>(pairs) * 8);
    std::memcpy(region + d->axis_offset, axis, static_cast<size_t>(pairs) * 4);
  }
  return LF_OK;
}

int64_t lunaflux_fp8_attn_cache_bytes(const lf_fp8_attn_desc *d) {
  if (!desc_ok(d)) return -1;
  if (d->cache != LF_FP8_CACHE_E4M3_BLOCKS) return last_element(d) * element_bytes(d);
  return d->block_scales + int64_t(d->pages) * (d->page_size / d->block_tokens) * d->kv_heads * 4;
}

int64_t lunaflux_fp8_attn_workspace_bytes(int32_t entry, const lf_fp8_attn_desc *d) {
  if (!desc_ok(d)) return -1;
  switch (entry) {
    case LF_FP8_ATTN_QK_NORM_ROPE: return LF_FP8_ATTN_STATUS_BYTES;
    case LF_FP8_ATTN_DECODE: return decode_bytes(d);
    case LF_FP8_ATTN_PREFILL:
    case LF_FP8_ATTN_PREFILL_JOIN: return prompt_bytes(d);
    default: return -1;
  }
}

int32_t lunaflux_fp8_attn_launch_geometry(int32_t entry, const lf_fp8_attn_desc *d, int32_t dims[7],
                                          char symbol[LF_FP8_SYMBOL_BYTES]) {
  if (!desc_ok(d) || dims == nullptr || symbol == nullptr) return LF_INVALID_ARGUMENT;
  const char *type = cache_name(d);
  int64_t gx = 0, lds = 0;
  switch (entry) {
    case LF_FP8_ATTN_QK_NORM_ROPE:
      gx = d->max_tokens + (d->cache == LF_FP8_CACHE_E4M3_BLOCKS ? append_blocks(d) : 0);
      if (d->cache == LF_FP8_CACHE_E4M3_BLOCKS) {
        std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_attn_qk_norm_rope_%s_d%d", type, d->head_dim);
      } else {
        std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_attn_qk_norm_rope_%s", type);
      }
      break;
    case LF_FP8_ATTN_DECODE:
      gx = decode_blocks(d);
      lds = align_up((int64_t(d->max_sequences) + 1) * 4, 16) + kWaves * tile_rows(d) * (d->head_dim + 4) * 4;
      std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_attn_decode_d%d_%s%s", d->head_dim, type,
                    d->cache != LF_FP8_CACHE_E4M3_BLOCKS && d->window > 0 && d->sinks > 0 ? "_sinks" : "");
      break;
    case LF_FP8_ATTN_PREFILL:
      gx = kPromptBlocks;
      lds = 6 * prompt_keys(d) * d->head_dim * 2;
      std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_attn_prefill_d%d_%s", d->head_dim, type);
      break;
    case LF_FP8_ATTN_PREFILL_JOIN:
      gx = prompt_cuts(d) ? kPromptBlocks * kJoinSlices : 0;
      std::snprintf(symbol, LF_FP8_SYMBOL_BYTES, "lf_attn_prefill_join_d%d_%s", d->head_dim, type);
      break;
    default: return LF_INVALID_ARGUMENT;
  }
  dims[0] = static_cast<int32_t>(gx);
  dims[1] = dims[2] = dims[4] = dims[5] = 1;
  dims[3] = static_cast<int32_t>(64 * (entry == LF_FP8_ATTN_PREFILL ? 2 * kWaves : kWaves));
  dims[6] = static_cast<int32_t>(lds);
  return LF_OK;
}

}  // extern "C"
