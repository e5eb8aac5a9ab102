// low_rank.hip - low-rank adapters of many requests beside a shared projection
// (the low-rank section of include/lunaflux_fp8.h): out = y + s_a (x A_a^T)
// B_a^T per row, a the row's adapter.
//
// Both products run on tiles of consecutive rows. A tile's rows may belong to
// any adapters: the blocks of its slots share out the distinct ones, compute the
// product of the whole tile with each and keep the rows that are the adapter's
// own, so nothing is sorted and a row never meets another adapter's weights.
//
// 61 rows of 16 adapters, hidden 4096, rank 16, columns 4096 + 2 x 1024: 13 us in
// one launch, of which launch and the chain of loads (ids, x and A, B, y) are nearly
// all; the bytes, at the rate of a copy, would take 2. 4093 rows, rank 64: 25 us for x
// A^T (8 TB/s from L2) and 27 for the rest (4 TB/s from and to HBM; 7 less without
// the products), 52 together, the bytes 28. Operands loaded from memory straight into
// the layout of the matrix instructions took 82 + 51.
#include "device_common.h"
#include "phases.h"

namespace low_rank {

// Mirror of lf_fp8_low_rank_desc.
struct Desc {
  uint32_t magic;
  int32_t adapters, rank, hidden, slices, columns, max_tokens, splits;
  int32_t ends[4];
  int32_t slots, one_launch, column_blocks, block_columns;
};
constexpr uint32_t kMagic = 0x4B4E524Cu;
LF_DEVICE const Desc &desc_of(const uint8_t *region) { return *reinterpret_cast<const Desc *>(region); }

// Workspace: a line with the word of ids past the adapters; in the two-launch
// form x A^T, per split of hidden, fp32 [splits][max_tokens][slices * rank].
constexpr uint64_t kPartsAt = 256;

// Adapter of each row of a tile, lane l holding row l; -1: none.
template <int ROWS>
LF_DEVICE int tile_ids(const Desc &d, const int32_t *ids, int row0, int rows, int *bad_id) {
  const int lane = threadIdx.x & 63;
  int id = lane < ROWS && row0 + lane < rows ? ids[row0 + lane] : -1;
  if (id >= d.adapters) {
    __hip_atomic_store(bad_id, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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

// A wave's part of x A^T: `steps` steps of 64 of k, `stride` apart, for 16 MT rows
// of x and 16 NT rows of A. Operands of the 16x16x32 products (rows = rows of A,
// columns = rows of x) want neighbouring lanes on different rows, which the
// vector memory would serve lane by lane; so rows are loaded in pieces of 128
// bytes, eight lanes each, and pass through the wave's own LDS (16-byte chunk j
// of row r at chunk j ^ (r % 8)). Two steps are in flight (four cost registers: 61
// rows of rank 32 21 us and 22.5); LDS serves a wave's accesses in their order, so
// no wait is needed between them.
constexpr int kAhead = 2;
LF_DEVICE void wave_order() {  // of what the wave's lanes pass each other through LDS
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
template <int MT, int NT>
constexpr int kStageBytes = (MT + NT) * 2048;
template <int MT, int NT>
LF_DEVICE void shrink_steps(f32x4 (&acc)[NT][MT], const uint8_t *x, const uint32_t (&xo)[2 * MT], const uint8_t *a,
                            int live, uint32_t row_bytes, int first, int steps, int stride, uint8_t *lds) {
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, r8 = lane >> 3, ch = lane & 7;
  struct Step {
    u32x4 x[2 * MT], a[2 * NT];
  } s[kAhead];
  const uint32_t ao = r8 * row_bytes + 16 * ch;
  if (steps <= 0) return;
  // (the last step again behind it: a load that a branch may skip would make the
  // wait for an older one a wait for all)
  auto load = [&](Step &to, int i) {
    const uint64_t k = 128ull * static_cast<uint32_t>(first + stride * (i < steps ? i : steps - 1));
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) to.x[j] = *reinterpret_cast<const u32x4 *>(x + k + xo[j]);
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      to.a[j] = *reinterpret_cast<const u32x4 *>(a + k + (j < 2 * live ? 8u * j : 0u) * row_bytes + ao);
    }
  };
  uint8_t *put = lds + r8 * 128 + ((ch ^ r8) * 16);
  const uint8_t *get[2] = {lds + c * 128 + ((g ^ (c & 7)) * 16), lds + c * 128 + (((4 + g) ^ (c & 7)) * 16)};
  auto multiply = [&](const Step &of) {
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) *reinterpret_cast<u32x4 *>(put + 1024 * j) = of.x[j];
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) *reinterpret_cast<u32x4 *>(put + 2048 * MT + 1024 * j) = of.a[j];
    wave_order();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 xf[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) xf[mt] = *reinterpret_cast<const bf16x8 *>(get[h] + 2048 * mt);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const bf16x8 af = *reinterpret_cast<const bf16x8 *>(get[h] + 2048 * (MT + t));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          acc[t][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, xf[mt], acc[t][mt], 0, 0, 0);
      }
    }
    wave_order();
  };
  static_for<kAhead>([&](auto j) { load(s[j], j); });
  int i = 0;
  for (; i + kAhead <= steps; i += kAhead) {
    static_for<kAhead>([&](auto j) {
      multiply(s[j]);
      __builtin_amdgcn_sched_barrier(0);  // the loads stay behind the products
      load(s[j], i + kAhead + j);
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  static_for<kAhead>([&](auto j) {
    if (i + j < steps) multiply(s[j]);
  });
}

// A value of x A^T as a bf16 value and the bf16 value of the rest (an infinity
// leaves none, not NaN).
LF_DEVICE void split_bf16(float v, __bf16 &top, __bf16 &rest) {
  top = static_cast<__bf16>(v);
  const float kept = static_cast<float>(top);
  rest = static_cast<__bf16>(__builtin_isinf(kept) ? 0.0f : v - kept);
}

// The columns [first, end) of a block, and the slice they lie in.
struct Columns {
  int slice, first, end;
};
LF_DEVICE Columns columns_of(const Desc &d, int block) {
  const int width = d.block_columns;
  int begin = 0;
  for (int s = 0; s < d.slices; ++s) {
    const int blocks = (d.ends[s] - begin + width - 1) / width;
    if (block < blocks) {
      const int first = begin + block * width;
      return {s, first, first + width < d.ends[s] ? first + width : d.ends[s]};
    }
    block -= blocks;
    begin = d.ends[s];
  }
  return {0, 0, 0};
}

// 128 columns of y + s v B^T for the wave's 16 rows, v = x A^T in two bf16 terms.
// Rows of the products are rows of y, columns output columns, arranged so that
// lane c has the eight columns 8 c + t of product t and each load and store of y
// takes 256 consecutive bytes of four rows. B comes in chunks of RANKS ranks
// through LDS, row 8 c + t as row 16 t + c, its 16-byte pieces turned so that
// eight rows' pieces lie in different banks; both terms are multiplied by it.
constexpr int kGroupColumns = 128;
template <int RANKS>
constexpr int kChunkBytes = kGroupColumns * 2 * RANKS;
template <int RANKS>
LF_DEVICE int chunk_at(int row, int piece) {
  constexpr int kPieces = RANKS / 8, kRows = kPieces < 8 ? 8 / kPieces : 1;  // rows per 128 bytes
  return row * 2 * RANKS + (piece ^ ((row / kRows) & (kPieces < 8 ? kPieces - 1 : 7))) * 16;
}
template <int LOADS, int RANKS>
struct ColumnChunk {
  static constexpr int kPieces = RANKS / 8, kRows = kGroupColumns / LOADS;
  u32x4 b[LOADS];
  // thread `id` of kRows * kPieces takes 16 bytes of every kRows-th row; zeros past
  // the rank
  LF_DEVICE void load(const Desc &d, int adapter, int n, int end, int r, int id, const uint16_t *w) {
    const int piece = id & (kPieces - 1), rank = r + 8 * piece < d.rank ? r + 8 * piece : r;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = n + id / kPieces + kRows * i;
      b[i] = *reinterpret_cast<const u32x4 *>(
          w + (static_cast<uint64_t>(adapter) * d.columns + (row < end ? row : end - 1)) * d.rank + rank);
      if constexpr (RANKS > 16) b[i] = r + 8 * piece < d.rank ? b[i] : u32x4{0, 0, 0, 0};
    }
  }
  LF_DEVICE void put(uint8_t *lds, int id) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = id / kPieces + kRows * i;
      *reinterpret_cast<u32x4 *>(lds + chunk_at<RANKS>((row & 7) * 16 + (row >> 3), id & (kPieces - 1))) = b[i];
    }
  }
};
// y of rows `row` + 4 g + i; rows and columns that are not to be written read
// others. Stores are nontemporal, and where many rows make a stream of it the
// loads too: 4093 rows 58.3 us with both, 60.0 with the stores alone, 62.0 with
// neither; 509 rows 18.7, 17.8 and 17.9.
template <bool STREAM>
struct ColumnRows {
  u32x4 y[4];
  LF_DEVICE void load(const Desc &d, uint32_t mine, int row, int any, int n, int end, const uint16_t *yp) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int col = n + 8 * c < end ? n + 8 * c : n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = (mine >> (4 * g + i)) & 1 ? row + 4 * g + i : any;
      const u32x4 *src = reinterpret_cast<const u32x4 *>(yp + static_cast<uint64_t>(m) * d.columns + col);
      y[i] = STREAM ? __builtin_nontemporal_load(src) : *src;
    }
  }
  LF_DEVICE void store(const Desc &d, const f32x4 (&acc)[8], float scale, uint32_t mine, int row, int n, int end,
                       uint16_t *out) const {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (((mine >> (4 * g + i)) & 1) && n + 8 * c < end) {
        u32x4 o;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          typedef float f32x2 __attribute__((ext_vector_type(2)));
          const f32x2 sum = {__builtin_bit_cast(float, y[i][k] << 16) + scale * acc[2 * k][i],
                             __builtin_bit_cast(float, y[i][k] & 0xffff0000u) + scale * acc[2 * k + 1][i]};
          o[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(sum, bf16x2));
        }
        uint16_t *to = out + static_cast<uint64_t>(row + 4 * g + i) * d.columns + n + 8 * c;
        __builtin_nontemporal_store(o, reinterpret_cast<u32x4 *>(to));
      }
    }
  }
};
// acc += v times the chunk, step h 32 ranks of it: lane group g has first(h) = the
// first terms of ranks 32 h + 8 g .. of row c, and rest(h) the second. A chunk of 16
// ranks takes both terms in one product: groups 0 and 1 the first, 2 and 3 the second.
template <int RANKS, class First, class Rest>
LF_DEVICE void multiply_chunk(f32x4 (&acc)[8], const uint8_t *lds, First &&first, Rest &&rest) {
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  static_for<(RANKS + 31) / 32>([&](auto h) {
    const int piece = 4 * h + (RANKS > 16 ? g : g & 1);
    bf16x8 w[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) w[t] = *reinterpret_cast<const bf16x8 *>(lds + chunk_at<RANKS>(16 * t + c, piece));
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(first(h), w[t], acc[t], 0, 0, 0);
    if constexpr (RANKS > 16) {
#pragma unroll
      for (int t = 0; t < 8; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(rest(h), w[t], acc[t], 0, 0, 0);
    }
  });
}

// Rows row .. row + 15 without an adapter, columns n .. n + 127.
LF_DEVICE void copy_others(const Desc &d, uint32_t none, int row, int n, int end, const uint16_t *y, uint16_t *out) {
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (((none >> (4 * g + i)) & 1) && n + 8 * c < end) {
      const uint64_t at = static_cast<uint64_t>(row + 4 * g + i) * d.columns + n + 8 * c;
      *reinterpret_cast<u32x4 *>(out + at) = *reinterpret_cast<const u32x4 *>(y + at);
    }
  }
}

// Few rows and small A: one launch. A block of eight waves has one 16-row tile,
// one slot of its adapters and up to 1024 columns of a slice, and computes x A^T
// of the slice by itself (the waves take the steps in turn and add up in wave
// order through LDS): reading A again per 1024 columns, from L2, costs less than
// passing x A^T from block to block.
constexpr int kOneWaves = 8;  // of 128 columns each
template <int NT>
LF_DEVICE void one_launch(const int32_t *counts, const int32_t *ids, const uint8_t *desc, const float *scaling,
                          const uint16_t *x, const uint16_t *a, const uint16_t *b, const uint16_t *y, uint16_t *out,
                          uint8_t *ws) {
  constexpr int kRanks = NT == 1 ? 16 : 32;  // of a chunk of B
  constexpr int kLowStride = 128 + 8;        // a row of x A^T, and a shift of banks
  constexpr int kWaveBytes = kStageBytes<1, NT> > kChunkBytes<kRanks> ? kStageBytes<1, NT> : kChunkBytes<kRanks>;
  __shared__ __attribute__((aligned(16))) uint8_t stage[kOneWaves][kWaveBytes];
  __shared__ __attribute__((aligned(16))) __bf16 low[2][16][kLowStride];
  const Desc &d = desc_of(desc);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int tile = blockIdx.x / d.slots, row0 = 16 * tile;
  // (turned by two per tile: the XCDs take blocks in turn, and the last slots are
  // often empty)
  const int slot = (blockIdx.x - tile * d.slots + 2 * tile) % d.slots;
  if (row0 >= rows) return;
  const int id = tile_ids<16>(d, ids, row0, rows, reinterpret_cast<int *>(ws));
  const Columns cols = columns_of(d, blockIdx.y);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int r8 = lane >> 3, ch = lane & 7;
  const int R = d.rank, SR = d.slices * R, K = d.hidden;
  const int n = cols.first + kGroupColumns * wave;
  const int steps = (K / 64 - wave + kOneWaves - 1) / kOneWaves;
  for_adapters(id, slot, d.slots, [&](int adapter, uint64_t mine) {
    const float scale = scaling[adapter];
    const int any = __builtin_ctzll(mine);
    ColumnChunk<kRanks / 4, kRanks> chunk;
    ColumnRows<false> column;
    if (n < cols.end) {
      chunk.load(d, adapter, n, cols.end, 0, lane, b);
      column.load(d, static_cast<uint32_t>(mine), row0, row0 + any, n, cols.end, y);
    }
    uint32_t xo[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = 8 * j + r8;
      xo[j] = static_cast<uint32_t>((mine >> m) & 1 ? m : any) * K * 2 + 16 * ch;
    }
    for (int r0 = 0; r0 < R; r0 += 16 * NT) {
      const int live = (R - r0) / 16 < NT ? (R - r0) / 16 : NT;
      f32x4 acc[NT][1];
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][0] = f32x4{0.f, 0.f, 0.f, 0.f};
      __syncthreads();  // what the stages and `low` held has been read
      shrink_steps<1, NT>(
          acc, reinterpret_cast<const uint8_t *>(x + static_cast<uint64_t>(row0) * K), xo,
          reinterpret_cast<const uint8_t *>(a + (static_cast<uint64_t>(adapter) * SR + cols.slice * R + r0) * K), live,
          2 * K, wave, steps, kOneWaves, stage[wave]);
#pragma unroll
      for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4 *>(stage[wave] + 1024 * t + 16 * lane) = acc[t][0];
      __syncthreads();
      if (wave < live) {
        f32x4 sum = *reinterpret_cast<const f32x4 *>(stage[0] + 1024 * wave + 16 * lane);
#pragma unroll
        for (int w = 1; w < kOneWaves; ++w) sum += *reinterpret_cast<const f32x4 *>(stage[w] + 1024 * wave + 16 * lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + 16 * wave + 4 * g + e;
          split_bf16(sum[e], low[0][c][r], low[1][c][r]);
        }
      } else if (NT > 1 && wave == live && live % 2 == 1) {  // the other half of a last step of 32
#pragma unroll
        for (int e = 0; e < 4; ++e) low[0][c][r0 + 16 * wave + 4 * g + e] = low[1][c][r0 + 16 * wave + 4 * g + e] = 0.f;
      }
    }
    __syncthreads();
    if (n < cols.end) {
      f32x4 acc[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int r = 0; r < R; r += kRanks) {
        chunk.put(stage[wave], lane);
        wave_order();
        if constexpr (NT == 4) chunk.load(d, adapter, n, cols.end, r + 32 < R ? r + 32 : r, lane, b);
        multiply_chunk<kRanks>(
            acc, stage[wave],
            [&](auto) {
              return *reinterpret_cast<const bf16x8 *>(NT > 1 ? &low[0][c][r + 8 * g] : &low[g >> 1][c][8 * (g & 1)]);
            },
            [&](auto) { return *reinterpret_cast<const bf16x8 *>(&low[1][c][r + 8 * g]); });
        wave_order();
      }
      column.store(d, acc, scale, static_cast<uint32_t>(mine), row0, n, cols.end, out);
    }
  });
  if (slot == 0 && out != y && n < cols.end) {
    const uint64_t none = __ballot(lane < 16 && row0 + lane < rows && id < 0);
    copy_others(d, static_cast<uint32_t>(none), row0, n, cols.end, y, out);
  }
}

// Blocks are dealt to the eight XCDs in turn: the `position`-th of `total` work
// items of block `block`, so that each XCD has neighbouring items, which share
// an adapter's weights in its L2. (A grid of a multiple of eight blocks; items
// past the last are none.)
LF_DEVICE int item_of(int block, int blocks) { return (block & 7) * (blocks >> 3) + (block >> 3); }

// x A^T of one tile of 16 MT rows, 16 NT of its columns and one split of hidden;
// the waves take the steps in turn and add up in wave order through LDS.
constexpr int kShrinkWaves = 8;
template <int MT, int NT>
LF_DEVICE void shrink(const int32_t *counts, const int32_t *ids, const uint8_t *desc, const uint16_t *x,
                      const uint16_t *a, uint8_t *ws) {
  constexpr int kRows = 16 * MT, kChunk = 16 * NT;
  __shared__ __attribute__((aligned(16))) uint8_t stage[kShrinkWaves][kStageBytes<MT, NT>];
  const Desc &d = desc_of(desc);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int SR = d.slices * d.rank, K = d.hidden, chunks = (SR + kChunk - 1) / kChunk;
  const int item = item_of(blockIdx.x, gridDim.x), slot = blockIdx.y;
  const int tile = item / (chunks * d.splits), chunk = item / d.splits - tile * chunks, split = item % d.splits;
  const int row0 = tile * kRows;
  if (row0 >= rows) return;
  const int id = tile_ids<kRows>(d, ids, row0, rows, reinterpret_cast<int *>(ws));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int r8 = lane >> 3, ch = lane & 7;
  const int col0 = chunk * kChunk;
  const int live = (SR - col0) / 16 < NT ? (SR - col0) / 16 : NT;
  const int all = K / 64, per = (all + d.splits - 1) / d.splits;
  const int first = split * per + wave, end = split * per + per < all ? split * per + per : all;
  const int steps = __builtin_amdgcn_readfirstlane(first < end ? (end - first + kShrinkWaves - 1) / kShrinkWaves : 0);
  float *part = reinterpret_cast<float *>(ws + kPartsAt) +
                (static_cast<uint64_t>(split) * d.max_tokens + row0) * SR + col0;

  uint32_t xo[2 * MT];
#pragma unroll
  for (int j = 0; j < 2 * MT; ++j) {
    const int m = 8 * j + r8;
    xo[j] = static_cast<uint32_t>(row0 + m < rows ? m : rows - 1 - row0) * K * 2 + 16 * ch;
  }
  for_adapters(id, slot, gridDim.y, [&](int adapter, uint64_t mine) {
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();  // what the stages held has been read
    shrink_steps<MT, NT>(acc, reinterpret_cast<const uint8_t *>(x + static_cast<uint64_t>(row0) * K), xo,
                            reinterpret_cast<const uint8_t *>(a + (static_cast<uint64_t>(adapter) * SR + col0) * K),
                            live, 2 * K, first, steps, kShrinkWaves, stage[wave]);
    static_assert(NT * MT * 1024 <= kStageBytes<MT, NT>, "a wave's sums fit its stage");
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        *reinterpret_cast<f32x4 *>(stage[wave] + 1024 * (t * MT + mt) + 16 * lane) = acc[t][mt];
    __syncthreads();
    for (int i = wave; i < live * MT; i += kShrinkWaves) {
      const int m = 16 * (i % MT) + c, r = 16 * (i / MT) + 4 * g;
      f32x4 sum = *reinterpret_cast<const f32x4 *>(stage[0] + 1024 * i + 16 * lane);
#pragma unroll
      for (int k = 1; k < kShrinkWaves; ++k) sum += *reinterpret_cast<const f32x4 *>(stage[k] + 1024 * i + 16 * lane);
      if ((mine >> m) & 1) *reinterpret_cast<f32x4 *>(part + static_cast<uint32_t>(m * SR + r)) = sum;
    }
  });
}

// y + s v B^T, v from the workspace, for 16 RW rows and a block's columns of a
// slice; RANKS = the rank, up to a power of two. RW 4: four waves of 16 rows each go
// through the columns together, with one copy of B in LDS; RW 1: each wave has 128
// columns of the same 16 rows. The next columns' B and y are loaded while these are
// multiplied; B first, so that the wait for it leaves y in flight, and it goes to
// LDS before the results are stored, so that no wait for a load is one for a store
// behind it.
template <int RW, int RANKS>
LF_DEVICE void expand(const int32_t *counts, const int32_t *ids, const uint8_t *desc, const float *scaling,
                      const uint16_t *b, const uint16_t *y, uint16_t *out, uint8_t *ws) {
  constexpr int kSide = 4 / RW;  // column groups side by side
  __shared__ __attribute__((aligned(16))) uint8_t stage[2][kSide][kChunkBytes<RANKS>];
  const Desc &d = desc_of(desc);
  if (d.magic != kMagic) return;
  const int rows = live_rows(counts, d.max_tokens);
  const int item = item_of(blockIdx.x, gridDim.x), tile = item / d.column_blocks, row0 = tile * 16 * RW;
  const int slot = blockIdx.y;
  if (row0 >= rows) return;
  const int id = tile_ids<16 * RW>(d, ids, row0, rows, reinterpret_cast<int *>(ws));
  bool some = false;
  for_adapters(id, slot, gridDim.y, [&](int, uint64_t) { some = true; });
  if (!some && slot > 0) return;
  const Columns cols = columns_of(d, item - tile * d.column_blocks);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int side = RW == 4 ? 0 : wave, part = RW == 4 ? wave : 0, row = row0 + 16 * part;
  const int loader = RW == 4 ? static_cast<int>(threadIdx.x) : lane;
  const int R = d.rank, SR = d.slices * R;
  auto sync = [&]() {
    if constexpr (RW == 4) {
      __syncthreads();
    } else {
      wave_order();
    }
  };
  // x A^T of the block's rows: the splits added up in order, then as two bf16 terms,
  // through the second stage, which is free until the first columns' products
  typedef __bf16 Low[2][16][RANKS];
  static_assert(RW * sizeof(Low) <= sizeof(stage[1]), "x A^T fits a stage");
  Low *low = reinterpret_cast<Low *>(stage[1]);
  const float *parts = reinterpret_cast<const float *>(ws + kPartsAt);
#pragma unroll 1
  for (int i = threadIdx.x; i < RW * 4 * RANKS; i += 256) {
    const int m = i / (RANKS / 4), k = 4 * (i % (RANKS / 4));
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (k < R) {
      const int at = row0 + m < rows ? row0 + m : rows - 1;
      const float *from = parts + static_cast<uint64_t>(at) * SR + cols.slice * R + k;
      constexpr int kBatch = RW == 4 ? 4 : 8;  // (4093 rows, one split: 56 us, with 8 58)
      for (int s0 = 0; s0 < d.splits; s0 += kBatch) {
        f32x4 v[kBatch];
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
          const uint64_t split = s0 + s < d.splits ? s0 + s : s0;
          v[s] = *reinterpret_cast<const f32x4 *>(from + split * d.max_tokens * SR);
        }
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
          if (s0 + s < d.splits) sum += v[s];
        }
      }
    }
    __bf16 t[4], u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split_bf16(sum[e], t[e], u[e]);
    *reinterpret_cast<uint2 *>(&low[m >> 4][0][m & 15][k]) = *reinterpret_cast<uint2 *>(t);
    *reinterpret_cast<uint2 *>(&low[m >> 4][1][m & 15][k]) = *reinterpret_cast<uint2 *>(u);
  }
  __syncthreads();
  bf16x8 first[RANKS / 32], rest[RANKS / 32];
#pragma unroll
  for (int h = 0; h < RANKS / 32; ++h) {
    first[h] = *reinterpret_cast<const bf16x8 *>(&low[part][0][c][32 * h + 8 * g]);
    rest[h] = *reinterpret_cast<const bf16x8 *>(&low[part][1][c][32 * h + 8 * g]);
  }
  __syncthreads();
  for_adapters(id, slot, gridDim.y, [&](int adapter, uint64_t block_rows) {
    const float scale = scaling[adapter];
    const uint32_t mine = static_cast<uint32_t>(block_rows >> (16 * part)) & 0xffffu;
    const int any = row0 + __builtin_ctzll(block_rows);
    const int begin = cols.first + kGroupColumns * side;
    if (begin >= cols.end) return;  // (alike for all waves that share a stage)
    ColumnChunk<RANKS / (RW == 4 ? 16 : 4), RANKS> chunk;
    ColumnRows<RW == 4> column[2];
    chunk.load(d, adapter, begin, cols.end, 0, loader, b);
    column[0].load(d, mine, row, any, begin, cols.end, y);
    sync();  // what the stage held has been read
    chunk.put(stage[0][side], loader);
    sync();
    auto group = [&](int n, auto k) {
      // (behind the last group the same again, see shrink_steps)
      const int n1 = n + kGroupColumns * kSide < cols.end ? n + kGroupColumns * kSide : n;
      chunk.load(d, adapter, n1, cols.end, 0, loader, b);
      column[1 - k].load(d, mine, row, any, n1, cols.end, y);
      f32x4 acc[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      __builtin_amdgcn_sched_barrier(0);
      multiply_chunk<RANKS>(acc, stage[k][side], [&](auto h) { return first[h]; }, [&](auto h) { return rest[h]; });
      __builtin_amdgcn_sched_barrier(0);
      chunk.put(stage[1 - k][side], loader);
      column[k].store(d, acc, scale, mine, row, n, cols.end, out);
      sync();
    };
    for (int n = begin; n < cols.end; n += 2 * kGroupColumns * kSide) {
      group(n, std::integral_constant<int, 0>());
      if (n + kGroupColumns * kSide < cols.end) group(n + kGroupColumns * kSide, std::integral_constant<int, 1>());
    }
  });
  if (slot == 0 && out != y) {
    const uint64_t none = __ballot(lane < 16 * RW && row0 + lane < rows && id < 0);
    const uint32_t mine = static_cast<uint32_t>(none >> (16 * part)) & 0xffffu;
    for (int n = cols.first + kGroupColumns * side; n < cols.end; n += kGroupColumns * kSide)
      copy_others(d, mine, row, n, cols.end, y, out);
  }
}

}  // namespace low_rank

#define LF_LOW_RANK_ONE(NT)                                                                                    \
  extern "C" __global__ __launch_bounds__(512, NT == 1 ? 4 : 2) void lf_low_rank_n##NT(                        \
      const int32_t *__restrict__ counts, const int32_t *__restrict__ ids, const uint8_t *__restrict__ desc,   \
      const float *__restrict__ scaling, const uint16_t *__restrict__ x, const uint16_t *__restrict__ a,       \
      const uint16_t *__restrict__ b, const uint16_t *y, uint16_t *out, uint8_t *__restrict__ ws) {            \
    low_rank::one_launch<NT>(counts, ids, desc, scaling, x, a, b, y, out, ws);                                 \
  }
LF_LOW_RANK_ONE(1)
LF_LOW_RANK_ONE(2)
LF_LOW_RANK_ONE(4)

#define LF_LOW_RANK_SHRINK(ROWS, COLUMNS)                                                                      \
  extern "C" __global__ __launch_bounds__(512) void lf_low_rank_shrink_##ROWS##x##COLUMNS(                     \
      const int32_t *__restrict__ counts, const int32_t *__restrict__ ids, const uint8_t *__restrict__ desc,   \
      const uint16_t *__restrict__ x, const uint16_t *__restrict__ a, uint8_t *__restrict__ ws) {              \
    low_rank::shrink<ROWS / 16, COLUMNS / 16>(counts, ids, desc, x, a, ws);                                    \
  }
LF_LOW_RANK_SHRINK(64, 32)
LF_LOW_RANK_SHRINK(64, 64)

#define LF_LOW_RANK_EXPAND(ROWS, RANKS)                                                                        \
  extern "C" __global__ __launch_bounds__(256, 2) void lf_low_rank_expand_##ROWS##x##RANKS(                    \
      const int32_t *__restrict__ counts, const int32_t *__restrict__ ids, const uint8_t *__restrict__ desc,   \
      const float *__restrict__ scaling, const uint16_t *__restrict__ b, const uint16_t *y, uint16_t *out,     \
      uint8_t *__restrict__ ws) {                                                                              \
    low_rank::expand<ROWS / 16, RANKS>(counts, ids, desc, scaling, b, y, out, ws);                             \
  }
LF_LOW_RANK_EXPAND(16, 32)
LF_LOW_RANK_EXPAND(16, 64)
LF_LOW_RANK_EXPAND(64, 32)
LF_LOW_RANK_EXPAND(64, 64)
LF_LOW_RANK_EXPAND(64, 128)
