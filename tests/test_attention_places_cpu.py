"""The attention kernels' index arithmetic on the CPU beyond
test_attention_index_cpu.py, whose program this one builds on: steps of garbage
on many descriptors, and caches whose strides are as long as the descriptor allows."""
import subprocess

from test_attention_index_cpu import KERNELS, PROGRAM

MAIN = "int main() {"


def run(tmp_path, body):
    """The program's functions with `body` (a definition of main, and what it calls) behind them."""
    src, exe = tmp_path / "places.cpp", str(tmp_path / "places")
    src.write_text(PROGRAM[:PROGRAM.index(MAIN)] + body)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", KERNELS,
                    "-Wno-unused-function", str(src), "-o", exe], check=True)
    done = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stdout + done.stderr


LANES = r"""
// Every lane's part of a group of eight rows is where cache_byte has the row.
template <bool E4M3>
static void lanes(int64_t page_stride, int64_t head_stride, int64_t token_stride, int dim) {
  Desc d{};
  d.page_size = 16;
  d.pages = 1 << 20;
  d.kv_heads = 8;
  d.page_stride = page_stride;
  d.head_stride = head_stride;
  d.token_stride = token_stride;
  constexpr int size = E4M3 ? 1 : 2;
  const uint32_t page_bytes = static_cast<uint32_t>(page_stride) * size;
  const uint32_t token_bytes = static_cast<uint32_t>(token_stride) * size;
  for (int page : {0, 1, (1 << 20) - 1}) {
    for (int slot : {0, 8}) {
      const uint64_t group = row_byte(page, slot, page_bytes, token_bytes);
      const uint64_t head = static_cast<uint64_t>(7) * static_cast<uint64_t>(head_stride) * size;
      for (int g = 0; g < 4; ++g) {
        for (int c = 0; c < 16; ++c) {
          CHECK(head + group + key_lane(c, g, token_bytes) ==
                cache_byte<E4M3>(d, page, 7, slot + c % 8) + static_cast<uint64_t>(16 * g));
          CHECK(head + group + value_lane(c, g, token_bytes, dim / 16 * size) ==
                cache_byte<E4M3>(d, page, 7, slot + 4 * g % 8) + static_cast<uint64_t>(c * (dim / 16) * size));
        }
      }
    }
  }
}
int main() {
  const int64_t most = (int64_t(1) << 31) - 16;   // bytes of a stride
  for (int dim : {64, 128, 256}) {
    lanes<true>(16 * 8 * dim, 16 * dim, dim, dim);
    lanes<false>(16 * 8 * dim, 16 * dim, dim, dim);
    for (int64_t token : {int64_t(613566752), int64_t(613566768), int64_t(1) << 30, most}) {
      lanes<true>(8 * dim, dim, token, dim);
      lanes<false>(8 * dim, dim, token / 2, dim);
    }
    lanes<true>(most, 16 * dim, dim, dim);
    lanes<true>(dim, most, 1024 * dim, dim);
  }
  std::printf("ok\n");
}
"""


def test_lanes_of_long_strides(tmp_path):
    run(tmp_path, LANES)


OVERLAPS = r"""
// The tiles of 64 consecutive sequences, whatever the page offsets, stay in the 31 bits
// that a wave adds them up in: a range that overlaps one before it comes after a range
// that falls, which has no pages and one tile.
static void offsets(const Desc &d, const std::vector<int> &ends) {
  int64_t sum = 0;
  for (size_t s = 0; s + 1 < ends.size(); ++s) {
    bool bad = false;
    const Pages p = pages_of(d, ends[s], ends[s + 1], bad);
    if (bad) CHECK(p.count == 0);
    const Span span = span_of(d, INT32_MAX, p, bad);
    CHECK(span.tiles >= 1 && span.tiles <= (1 << 26) - 32);
    sum += span.tiles;
    if ((s + 1) % 64 == 0) {
      CHECK(sum <= INT32_MAX);
      sum = 0;
    }
  }
}
int main() {
  for (int page : {8, 32, 1024}) {
    Desc d{};
    d.page_size = page;
    d.table_entries = (INT32_MAX - 1024) / page;
    std::vector<int> ends(2049);
    for (int phase = 0; phase < 2; ++phase) {
      for (size_t i = 0; i < ends.size(); ++i) ends[i] = i % 2 == static_cast<size_t>(phase) ? 0 : d.table_entries;
      offsets(d, ends);
    }
    for (int i = 0; i < 500; ++i) {
      for (auto &e : ends) e = pick(0, 3) ? pick(0, 1) * d.table_entries : pick(-2, d.table_entries);
      offsets(d, ends);
    }
  }
  std::printf("ok\n");
}
"""


def test_a_wave_of_overlapping_page_ranges_fits_31_bits(tmp_path):
    run(tmp_path, OVERLAPS)


def test_steps_of_garbage_on_many_descriptors(tmp_path):
    """hostile() on a descriptor of its own each time, and the cut for both grids of
    the decode kernels (256 and 512 blocks)."""
    run(tmp_path, r"""
int main() {
  for (int i = 0; i < 400; ++i) hostile();
  for (int i = 0; i < 400; ++i) cut(i % 2 ? 256 : 512);
  std::printf("ok\n");
}
""")
