// low_rank.hip - low-rank adapters of many requests beside a shared projection
// (the low-rank section of include/lunaflux_fp8.h): out = y + s_a (x A_a^T)
// B_a^T per row, a the row's adapter.
//
// Both products run on tiles of consecutive rows. A tile's rows may belong to
// any adapters: a block goes through the distinct ones, computes the product of
// the whole tile with each and keeps the columns (= rows of x) that are the
// adapter's own, so nothing is sorted and a row never meets another adapter's
// weights.
#include "device_common.h"
#include "phases.h"

namespace low_rank {

// Mirror of lf_fp8_low_rank_desc.
struct Desc {
  uint32_t magic;
  int32_t adapters, rank, hidden, slices, columns, max_tokens, splits;
  int32_t ends[4];
  int32_t slots, column_blocks, reserved[2];
};
constexpr uint32_t kMagic = 0x4B4E524Cu;
constexpr int kWaves = 4;
constexpr int kColumnBlock = 512;  // output columns per block, 128 per wave

LF_DEVICE const Desc &desc_of(const uint8_t *region) { return *reinterpret_cast<const Desc *>(region); }

// Workspace: a line with the error word (a wait ran out; 0 after every correct
// launch) and, at 64, the word of ids past the adapters; two counters per (tile,
// slot), each in a line of its own, for the one-launch form; x A^T fp32 [splits]
// [max_tokens][slices * rank].
struct Ws {
  int *error, *bad_id;
  uint8_t *counters;
  float *v;
};
LF_DEVICE Ws ws_of(const Desc &d, uint8_t *ws, int counted) {
  return {reinterpret_cast<int *>(ws), reinterpret_cast<int *>(ws + 64), ws + 256,
          reinterpret_cast<float *>(ws + 256 + static_cast<uint64_t>(counted) * 256)};
}

// Adapter of each row of a tile, lane l holding row l; -1: none.
template <int MT>
LF_DEVICE int tile_ids(const Desc &d, const int32_t *ids, int row0, int rows, int *bad_id) {
  const int lane = threadIdx.x & 63;
  int id = lane < 16 * MT && row0 + lane < rows ? ids[row0 + lane] : -1;
  if (id >= d.adapters) {
    __hip_atomic_store(bad_id, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    id = -1;
  }
  return id < 0 ? -1 : id;
}

// f(adapter, rows of it as a bit mask) for every slots-th distinct adapter of
// a tile from the slot-th on, in the order of their first rows; how many.
template <class F>
LF_DEVICE int for_adapters(int id, int slot, int slots, F &&f) {
  uint64_t left = __ballot(id >= 0);
  int found = 0;
  for (int j = 0; left != 0; ++j) {
    const int adapter = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t mine = __ballot(id == adapter);
    left &= ~mine;
    if (j % slots == slot) {
      f(adapter, mine);
      ++found;
    }
  }
  return found;
}

// x A^T of one tile, 64 of its columns and one slice of hidden. Operands of the
// 16x16x32 products: rows = rows of A, columns = rows of x; a lane's 32 values
// of k (a step of 64 over the four lane groups) are consecutive in both, so each
// row is read in 128-byte pieces. The block's waves take the steps in turn, one
// step's loads ahead, and add up in wave order through LDS.
template <int MT>
struct Shrink {
  static constexpr int NT = 4;
  f32x4 part[kWaves][NT * MT][64];
};
template <int MT>
LF_DEVICE int shrink(const Desc &d, int id, int slot, int row0, int rows, int chunk, int split, const uint16_t *x,
                     const uint16_t *a, float *v, Shrink<MT> &lds) {
  constexpr int NT = Shrink<MT>::NT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int SR = d.slices * d.rank, K = d.hidden;
  const int col0 = chunk * 64;
  const int live = (SR - col0) / 16 < NT ? (SR - col0) / 16 : NT;  // 16-column tiles
  const int steps = K / 64, per = (steps + d.splits - 1) / d.splits;
  const int first = split * per, end = first + per < steps ? first + per : steps;
  v += static_cast<uint64_t>(split) * d.max_tokens * SR;

  const uint16_t *xr[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 16 * mt + c;
    xr[mt] = x + static_cast<uint64_t>(row < rows ? row : rows - 1) * K + 16 * g;
  }
  struct Step {
    bf16x8 x[MT][2], a[NT][2];
  };
  return for_adapters(id, slot, d.slots, [&](int adapter, uint64_t mine) {
    // (tiles past the last read the last again)
    const uint16_t *ar[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
      ar[t] = a + (static_cast<uint64_t>(adapter) * SR + col0 + 16 * (t < live ? t : live - 1) + c) * K + 16 * g;
    auto load = [&](Step &s, int step) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) s.x[mt][h] = *reinterpret_cast<const bf16x8 *>(xr[mt] + 64 * step + 8 * h);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) s.a[t][h] = *reinterpret_cast<const bf16x8 *>(ar[t] + 64 * step + 8 * h);
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Step &s) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            acc[t][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(s.a[t][h], s.x[mt][h], acc[t][mt], 0, 0, 0);
    };
    if (first + wave < end) {
      Step s0, s1;
      const int last = end - 1 - (end - 1 - first - wave) % kWaves;  // this wave's last step
      load(s0, first + wave);
      for (int s = first + wave; s < end; s += 2 * kWaves) {
        load(s1, s + kWaves < end ? s + kWaves : last);
        multiply(s0);
        if (s + kWaves >= end) break;
        load(s0, s + 2 * kWaves < end ? s + 2 * kWaves : last);
        multiply(s1);
      }
    }
    __syncthreads();  // the adapter before has been read
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) lds.part[wave][t * MT + mt][lane] = acc[t][mt];
    __syncthreads();
    for (int i = wave; i < live * MT; i += kWaves) {
      const int t = i / MT, m = 16 * (i % MT) + c;
      f32x4 sum = lds.part[0][i][lane];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += lds.part[w][i][lane];
      if ((mine >> m) & 1) {
        phase::store16_through(v + static_cast<uint64_t>(row0 + m) * SR + col0 + 16 * t + 4 * g,
                               __builtin_bit_cast(u32x4, sum));
      }
    }
  });
}

// The columns of a block: a slice, its first column there and behind it.
struct Columns {
  int slice, first, end;
};
LF_DEVICE Columns columns_of(const Desc &d, int block) {
  int begin = 0;
  for (int s = 0; s < d.slices; ++s) {
    const int blocks = (d.ends[s] - begin + kColumnBlock - 1) / kColumnBlock;
    if (block < blocks) {
      const int first = begin + block * kColumnBlock;
      return {s, first, first + kColumnBlock < d.ends[s] ? first + kColumnBlock : d.ends[s]};
    }
    block -= blocks;
    begin = d.ends[s];
  }
  return {0, 0, 0};
}

// x A^T of a tile's rows, the splits added up in order, as its bf16 rounding and
// the rounding of the rest, in LDS.
template <int MT>
struct Expand {
  static constexpr int kStride = 128 + 8;  // ranks of a row, and a shift of banks
  __bf16 v[2][16 * MT][kStride];
};
template <int MT>
LF_DEVICE void load_low(const Desc &d, int row0, int rows, int slice, const float *v, Expand<MT> &lds) {
  const int R = d.rank, SR = d.slices * R, quads = R / 4;
  const uint64_t split_stride = static_cast<uint64_t>(d.max_tokens) * SR;
  for (int i = threadIdx.x; i < 16 * MT * quads; i += 64 * kWaves) {
    const int m = i / quads, r = 4 * (i - m * quads);
    const float *src = v + static_cast<uint64_t>(row0 + m < rows ? row0 + m : rows - 1) * SR + slice * R + r;
    f32x4 sum = *reinterpret_cast<const f32x4 *>(src);
    int s = 1;
    for (; s + 4 <= d.splits; s += 4) {
      f32x4 p[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k] = *reinterpret_cast<const f32x4 *>(src + (s + k) * split_stride);
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += p[k];
    }
    for (; s < d.splits; ++s) sum += *reinterpret_cast<const f32x4 *>(src + s * split_stride);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __bf16 top = static_cast<__bf16>(sum[e]);
      const float kept = static_cast<float>(top);
      lds.v[0][m][r + e] = top;
      // (an infinity leaves no rest, not NaN)
      lds.v[1][m][r + e] = static_cast<__bf16>(__builtin_isinf(kept) ? 0.0f : sum[e] - kept);
    }
  }
}

// y + s v B^T of one tile and the block's columns, v = x A^T in LDS. Rows of the
// products are output columns, arranged so that lane group g ends up with 16
// consecutive ones of every 64 (column 16 g + 4 t + i in element i of tile t);
// columns are rows of y. Of each 16 ranks, lane groups 0 and 1 hold the bf16
// values of v and 2 and 3 the rests, so one 16x16x32 product adds both.
// ready(): v is in LDS afterwards (false: it never came, and nothing is stored);
// what does not depend on it is requested before.
template <int MT, class F>
LF_DEVICE void expand(const Desc &d, int id, int slot, int row0, int rows, Columns cols, const float *scaling,
                      const uint16_t *b, const uint16_t *y, uint16_t *out, Expand<MT> &lds, F &&ready) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int R = d.rank;
  bool waited = false, came = true;
  for_adapters(id, slot, d.slots, [&](int adapter, uint64_t mine) {
    const float scale = scaling[adapter];
    for (int n0 = cols.first + 64 * wave; n0 < cols.end || !waited; n0 += 64 * kWaves) {
      const bool some = n0 < cols.end;
      const int n = some ? n0 : cols.first;
      const uint16_t *br = b + (static_cast<uint64_t>(adapter) * d.columns + n + 16 * (c >> 2) + (c & 3)) * R + 8 * (g & 1);
      bf16x8 bf[4], bn[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) bf[t] = *reinterpret_cast<const bf16x8 *>(br + static_cast<uint64_t>(4 * t) * R);
      u32x4 yw[MT][2];
      uint64_t at[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int m = 16 * mt + c;
        at[mt] = static_cast<uint64_t>((mine >> m) & 1 ? row0 + m : row0) * d.columns + n + 16 * g;
#pragma unroll
        for (int h = 0; h < 2; ++h) yw[mt][h] = *reinterpret_cast<const u32x4 *>(y + at[mt] + 8 * h);
      }
      if (!waited) {
        came = ready();
        waited = true;
      }
      if (!some || !came) break;
      f32x4 acc[4][MT];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int r = 0; r < R; r += 16) {
        const int next = r + 16 < R ? r + 16 : r;
#pragma unroll
        for (int t = 0; t < 4; ++t) bn[t] = *reinterpret_cast<const bf16x8 *>(br + static_cast<uint64_t>(4 * t) * R + next);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const bf16x8 vf = *reinterpret_cast<const bf16x8 *>(&lds.v[g >> 1][16 * mt + c][r + 8 * (g & 1)]);
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[t][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[t], vf, acc[t][mt], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) bf[t] = bn[t];
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if ((mine >> (16 * mt + c)) & 1) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4 o;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const f32x4 &p = acc[2 * h + (i >> 1)][mt];
              o[i] = f32_to_bf16(bf16_to_f32(yw[mt][h][i] & 0xffffu) + scale * p[2 * (i & 1)]) |
                     (f32_to_bf16(bf16_to_f32(yw[mt][h][i] >> 16) + scale * p[2 * (i & 1) + 1]) << 16);
            }
            *reinterpret_cast<u32x4 *>(out + at[mt] + 8 * h) = o;
          }
        }
      }
    }
  });
  if (slot == 0 && out != y) {  // rows without an adapter
    for (int n0 = cols.first + 64 * wave; n0 < cols.end; n0 += 64 * kWaves) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int m = 16 * mt + c;
        const int owner = __shfl(id, m);
        if (row0 + m < rows && owner < 0) {
          const uint64_t at = static_cast<uint64_t>(row0 + m) * d.columns + n0 + 16 * g;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<u32x4 *>(out + at + 8 * h) = *reinterpret_cast<const u32x4 *>(y + at + 8 * h);
        }
      }
    }
  }
}

// Long runs of an adapter (64-row tiles): two launches.
LF_DEVICE void shrink_launch(const int32_t *counts, const int32_t *ids, const uint8_t *desc, const uint16_t *x,
                             const uint16_t *a, uint8_t *ws) {
  __shared__ Shrink<4> lds;
  const Desc &d = desc_of(desc);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int tile = blockIdx.x / d.slots, slot = blockIdx.x - tile * d.slots;
  if (64 * tile >= rows) return;
  const Ws w = ws_of(d, ws, 0);
  const int id = tile_ids<4>(d, ids, 64 * tile, rows, w.bad_id);
  shrink<4>(d, id, slot, 64 * tile, rows, blockIdx.y, blockIdx.z, x, a, w.v, lds);
}
LF_DEVICE void expand_launch(const int32_t *counts, const int32_t *ids, const uint8_t *desc, const float *scaling,
                             const uint16_t *b, const uint16_t *y, uint16_t *out, uint8_t *ws) {
  __shared__ Expand<4> lds;
  const Desc &d = desc_of(desc);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int tile = blockIdx.x / d.slots, slot = blockIdx.x - tile * d.slots;
  if (64 * tile >= rows) return;
  const Ws w = ws_of(d, ws, 0);
  const int id = tile_ids<4>(d, ids, 64 * tile, rows, w.bad_id);
  const Columns cols = columns_of(d, blockIdx.y);
  expand<4>(d, id, slot, 64 * tile, rows, cols, scaling, b, y, out, lds, [&]() {
    load_low<4>(d, 64 * tile, rows, cols.slice, w.v, lds);
    __syncthreads();
    return true;
  });
}

// Few rows (16-row tiles): one launch. The grid's first blocks compute x A^T,
// the others wait for their tile's and slot's, counted (phases.h), with their
// part of B and y on the way. The last block behind a wait puts both counters of
// its tile and slot back to zero.
LF_DEVICE void one_launch(const int32_t *counts, const int32_t *ids, const uint8_t *desc, const float *scaling,
                          const uint16_t *x, const uint16_t *a, const uint16_t *b, const uint16_t *y, uint16_t *out,
                          uint8_t *ws) {
  __shared__ union {
    Shrink<1> shrink;
    Expand<1> expand;
  } lds;
  __shared__ phase::Flag flag;
  const Desc &d = desc_of(desc);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int tiles = (d.max_tokens + 15) / 16, pairs = tiles * d.slots;
  const int chunks = (d.slices * d.rank + 63) / 64, each = chunks * d.splits;
  const Ws w = ws_of(d, ws, pairs);
  int block = blockIdx.x;
  const bool first_step = block < pairs * each;
  if (!first_step) block -= pairs * each;
  const int share = first_step ? each : d.column_blocks;
  const int pair = block / share, part = block - pair * share;
  const int tile = pair / d.slots, slot = pair - tile * d.slots;
  if (16 * tile >= rows) return;
  const int id = tile_ids<1>(d, ids, 16 * tile, rows, w.bad_id);
  int *done = reinterpret_cast<int *>(w.counters + static_cast<uint64_t>(pair) * 256), *left = done + phase::kLineInts;
  if (first_step) {
    const int split = part / chunks;
    if (shrink<1>(d, id, slot, 16 * tile, rows, part - split * chunks, split, x, a, w.v, lds.shrink) > 0)
      phase::signal(done);
    return;
  }
  const Columns cols = columns_of(d, part);
  bool waited = false, ok = true;
  expand<1>(d, id, slot, 16 * tile, rows, cols, scaling, b, y, out, lds.expand, [&]() {
    waited = true;
    ok = phase::wait_for(done, each, w.error, flag);
    if (ok) {
      load_low<1>(d, 16 * tile, rows, cols.slice, w.v, lds.expand);
      __syncthreads();
    }
    return ok;
  });
  if (!waited) return;
  __syncthreads();
  if (threadIdx.x == 0 && ok) {
    const int before = __hip_atomic_fetch_add(left, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before == d.column_blocks - 1) {
      phase::store_agent(done, 0);
      phase::store_agent(left, 0);
    }
  }
}

}  // namespace low_rank

extern "C" __global__ __launch_bounds__(256) void lf_low_rank_shrink_r64(const int32_t *counts, const int32_t *ids,
                                                                         const uint8_t *desc, const uint16_t *x,
                                                                         const uint16_t *a, uint8_t *ws) {
  low_rank::shrink_launch(counts, ids, desc, x, a, ws);
}
extern "C" __global__ __launch_bounds__(256) void lf_low_rank_expand_r64(const int32_t *counts, const int32_t *ids,
                                                                         const uint8_t *desc, const float *scaling,
                                                                         const uint16_t *b, const uint16_t *y,
                                                                         uint16_t *out, uint8_t *ws) {
  low_rank::expand_launch(counts, ids, desc, scaling, b, y, out, ws);
}
extern "C" __global__ __launch_bounds__(256) void lf_low_rank_r16(const int32_t *counts, const int32_t *ids,
                                                                  const uint8_t *desc, const float *scaling,
                                                                  const uint16_t *x, const uint16_t *a,
                                                                  const uint16_t *b, const uint16_t *y, uint16_t *out,
                                                                  uint8_t *ws) {
  low_rank::one_launch(counts, ids, desc, scaling, x, a, b, y, out, ws);
}
