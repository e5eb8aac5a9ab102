// low_rank.hip - low-rank adapters of many requests beside a shared projection
// (the low-rank section of include/lunaflux_fp8.h): out = y + s_a (x A_a^T)
// B_a^T per row, a the row's adapter.
//
// Both products run on tiles of consecutive rows. A tile's rows may belong to
// any adapters: the block goes through the distinct ones, computes the product
// of the whole tile with each and keeps the columns (= rows of x) that are the
// adapter's own, so nothing is sorted and a row never meets another adapter's
// weights.
#include "device_common.h"

namespace low_rank {

// Mirror of lf_fp8_low_rank_desc.
struct Desc {
  uint32_t magic;
  int32_t adapters, rank, hidden, slices, columns, max_tokens, splits;
  int32_t ends[4];
};
constexpr uint32_t kMagic = 0x4B4E524Cu;
constexpr uint64_t kHeaderBytes = 256;
constexpr int kWaves = 4;

LF_DEVICE const Desc &desc_of(const uint8_t *region) { return *reinterpret_cast<const Desc *>(region); }

// Adapter of each row of a tile, lane l holding row l; -1: none.
template <int MT>
LF_DEVICE int tile_ids(const Desc &d, const int32_t *ids, int row0, int rows, int *error) {
  const int lane = threadIdx.x & 63;
  int id = lane < 16 * MT && row0 + lane < rows ? ids[row0 + lane] : -1;
  if (id >= d.adapters) {
    __hip_atomic_store(error, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    id = -1;
  }
  return id < 0 ? -1 : id;
}

// f(adapter, rows of it as a bit mask) for every slots-th distinct adapter of
// a tile from the slot-th on, in the order of their first rows.
template <class F>
LF_DEVICE void for_adapters(int id, int slot, int slots, F &&f) {
  uint64_t left = __ballot(id >= 0);
  for (int j = 0; left != 0; ++j) {
    const int adapter = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t mine = __ballot(id == adapter);
    left &= ~mine;
    if (j % slots == slot) f(adapter, mine);
  }
}

// x A^T of one tile, 64 of its columns and one slice of hidden. Operands of the
// 16x16x32 products: rows = rows of A, columns = rows of x; a lane's 32 values
// of k (a step of 64 over the four lane groups) are consecutive in both, so each
// row is read in 128-byte pieces. The block's waves take the steps in turn and
// add up in wave order through LDS.
template <int MT>
LF_DEVICE void shrink(const int32_t *counts, const int32_t *ids, const uint8_t *desc, const uint16_t *x,
                      const uint16_t *a, uint8_t *ws) {
  constexpr int NT = 4;
  __shared__ f32x4 part[kWaves][NT * MT][64];
  const Desc &d = desc_of(desc);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int slots = MT == 1 ? (d.adapters < 16 ? d.adapters : 16) : 1;
  const int tile = blockIdx.x / slots, slot = blockIdx.x - tile * slots;
  const int row0 = tile * 16 * MT;
  if (row0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int id = tile_ids<MT>(d, ids, row0, rows, reinterpret_cast<int *>(ws));
  const int SR = d.slices * d.rank, K = d.hidden;
  const int col0 = blockIdx.y * 64;
  const int live = (SR - col0) / 16 < NT ? (SR - col0) / 16 : NT;  // 16-column tiles
  const int steps = K / 64, per = (steps + d.splits - 1) / d.splits;
  const int first = blockIdx.z * per, end = first + per < steps ? first + per : steps;
  float *v = reinterpret_cast<float *>(ws + kHeaderBytes) + static_cast<uint64_t>(blockIdx.z) * d.max_tokens * SR;

  const uint16_t *xr[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 16 * mt + c;
    xr[mt] = x + static_cast<uint64_t>(row < rows ? row : rows - 1) * K + 16 * g;
  }
  for_adapters(id, slot, slots, [&](int adapter, uint64_t mine) {
    const uint16_t *ar = a + (static_cast<uint64_t>(adapter) * SR + col0 + c) * K + 16 * g;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = first + wave; s < end; s += kWaves) {
      const int k = 64 * s;
      bf16x8 xf[MT][2], af[NT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) xf[mt][h] = *reinterpret_cast<const bf16x8 *>(xr[mt] + k + 8 * h);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t < live) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            af[t][h] = *reinterpret_cast<const bf16x8 *>(ar + static_cast<uint64_t>(16 * t) * K + k + 8 * h);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t < live) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              acc[t][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[t][h], xf[mt][h], acc[t][mt], 0, 0, 0);
        }
      }
    }
    __syncthreads();  // the adapter before has been read
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) part[wave][t * MT + mt][lane] = acc[t][mt];
    __syncthreads();
    for (int i = wave; i < live * MT; i += kWaves) {
      const int t = i / MT, m = 16 * (i % MT) + c;
      f32x4 sum = part[0][i][lane];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += part[w][i][lane];
      if ((mine >> m) & 1) {
        *reinterpret_cast<f32x4 *>(v + static_cast<uint64_t>(row0 + m) * SR + col0 + 16 * t + 4 * g) = sum;
      }
    }
  });
}

// y + s (x A^T) B^T of one tile and 64 columns per wave. Rows of the products
// are output columns, arranged so that lane group g ends up with 16 consecutive
// ones (column 16 g + 4 t + i in element i of tile t); columns are rows of y.
// A value of x A^T goes in as its bf16 rounding and the rounding of the rest:
// lane groups 0 and 1 hold the first, 2 and 3 the second, of the same 16 ranks.
template <int MT>
LF_DEVICE void expand(const int32_t *counts, const int32_t *ids, const uint8_t *desc, const float *scaling,
                      const uint16_t *b, const uint16_t *y, uint16_t *out, uint8_t *ws) {
  const Desc &d = desc_of(desc);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int slots = MT == 1 ? (d.adapters < 16 ? d.adapters : 16) : 1;
  const int tile = blockIdx.x / slots, slot = blockIdx.x - tile * slots;
  const int row0 = tile * 16 * MT;
  if (row0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int n0 = (static_cast<int>(blockIdx.y) * kWaves + wave) * 64;
  if (n0 >= d.columns) return;
  const int id = tile_ids<MT>(d, ids, row0, rows, reinterpret_cast<int *>(ws));
  int slice = 0;
  while (n0 >= d.ends[slice]) ++slice;
  const int R = d.rank, SR = d.slices * R;
  const float *v = reinterpret_cast<const float *>(ws + kHeaderBytes) + slice * R + 8 * (g & 1);
  const uint64_t split_stride = static_cast<uint64_t>(d.max_tokens) * SR;

  for_adapters(id, slot, slots, [&](int adapter, uint64_t mine) {
    f32x4 acc[4][MT];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint16_t *br = b + (static_cast<uint64_t>(adapter) * d.columns + n0 + 16 * (c >> 2) + (c & 3)) * R + 8 * (g & 1);
    for (int r = 0; r < R; r += 16) {
      bf16x8 bf[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) bf[t] = *reinterpret_cast<const bf16x8 *>(br + static_cast<uint64_t>(4 * t) * R + r);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int row = row0 + 16 * mt + c;
        const float *src = v + static_cast<uint64_t>(row < rows ? row : rows - 1) * SR + r;
        f32x4 lo = *reinterpret_cast<const f32x4 *>(src), hi = *reinterpret_cast<const f32x4 *>(src + 4);
        for (int s = 1; s < d.splits; ++s) {
          lo += *reinterpret_cast<const f32x4 *>(src + s * split_stride);
          hi += *reinterpret_cast<const f32x4 *>(src + s * split_stride + 4);
        }
        bf16x8 vf;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float full = e < 4 ? lo[e] : hi[e - 4];
          const __bf16 top = static_cast<__bf16>(full);
          // (an infinity leaves no rest, not NaN)
          const float kept = static_cast<float>(top);
          const float rest = __builtin_isinf(kept) ? 0.0f : full - kept;
          vf[e] = g < 2 ? top : static_cast<__bf16>(rest);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[t], vf, acc[t][mt], 0, 0, 0);
      }
    }
    const float scale = scaling[adapter];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int m = 16 * mt + c;
      if ((mine >> m) & 1) {
        const uint64_t at = static_cast<uint64_t>(row0 + m) * d.columns + n0 + 16 * g;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 w = *reinterpret_cast<const u32x4 *>(y + at + 8 * h);
          u32x4 o;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 &p = acc[2 * h + (i >> 1)][mt];
            o[i] = f32_to_bf16(bf16_to_f32(w[i] & 0xffffu) + scale * p[2 * (i & 1)]) |
                   (f32_to_bf16(bf16_to_f32(w[i] >> 16) + scale * p[2 * (i & 1) + 1]) << 16);
          }
          *reinterpret_cast<u32x4 *>(out + at + 8 * h) = o;
        }
      }
    }
  });
  if (slot == 0 && out != y) {  // rows without an adapter
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int m = 16 * mt + c;
      const int owner = __shfl(id, m);
      if (row0 + m < rows && owner < 0) {
        const uint64_t at = static_cast<uint64_t>(row0 + m) * d.columns + n0 + 16 * g;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          *reinterpret_cast<u32x4 *>(out + at + 8 * h) = *reinterpret_cast<const u32x4 *>(y + at + 8 * h);
        }
      }
    }
  }
}

}  // namespace low_rank

#define LF_LOW_RANK(ROWS, MT)                                                                               \
  extern "C" __global__ __launch_bounds__(256) void lf_low_rank_shrink_r##ROWS(                             \
      const int32_t *counts, const int32_t *ids, const uint8_t *desc, const uint16_t *x, const uint16_t *a, \
      uint8_t *ws) {                                                                                        \
    low_rank::shrink<MT>(counts, ids, desc, x, a, ws);                                                      \
  }                                                                                                         \
  extern "C" __global__ __launch_bounds__(256) void lf_low_rank_expand_r##ROWS(                             \
      const int32_t *counts, const int32_t *ids, const uint8_t *desc, const float *scaling,                 \
      const uint16_t *b, const uint16_t *y, uint16_t *out, uint8_t *ws) {                                   \
    low_rank::expand<MT>(counts, ids, desc, scaling, b, y, out, ws);                                        \
  }
LF_LOW_RANK(16, 1)
LF_LOW_RANK(64, 4)
