"""The ranges, partial results and join of test_attention_prompt_index_cpu.py with the cuts that the kernels make:
both launches cut by cut_tiles, every fourth tile of long pairs in steps of little work."""
import subprocess

import test_attention_prompt_index_cpu as index

CHANGES = [  # (of its program, as the kernels have it, how often)
    ("share = (total + blocks - 1) / blocks;", "share = (total + blocks - 1) / blocks;\n  const int by = cut_tiles(share, tile_keys);", 1),
    ("cut_of(u0, begin, weight, k.tiles), k1 = cut_of(u1, begin, weight, k.tiles);",
     "cut_of(u0, begin, weight, k.tiles, by), k1 = cut_of(u1, begin, weight, k.tiles, by);", 1),
    ("CHECK(k1 - k0 >= kCut && k.tiles >= 2 * kCut);",
     "CHECK(k1 - k0 >= (k.tiles < 4 * kCut ? kCut : by) && k.tiles >= 2 * kCut);\n"
     "          (by < kCut && k.tiles >= 4 * kCut ? (k0 % kCut != 0 || k1 % kCut != 0) ? fourth : fourth_whole : eighth)++;", 1),
    ("return cut_of(b * share, begin, weight, k.tiles);", "return cut_of(b * share, begin, weight, k.tiles, by);", 1),
    ("// As the kernels go through a step", "static int fourth, fourth_whole, eighth;  // parts\n// As the kernels go through a step", 1),
    ("static Desc desc() {", "static bool little;\nstatic Desc desc() {", 1),
    ("  d.table_entries = pick(1, 1000);\n", "  d.table_entries = little ? pick(1, 100) : pick(1, 1000);\n"
     "  if (little) d.max_tokens = pick(1, 30), d.page_size = 64, d.kv_heads = pick(1, 2), d.query_heads = d.kv_heads * pick(1, 8), d.window = 0;\n", 1),
    ("cut(blocks[i % 5]);", "little = i % 2 != 0, cut(i % 2 != 0 ? 256 : blocks[i % 5]);", 1),
    ('std::printf("ok\\n");', 'std::printf("ok %d\\n", fourth > 1000 && eighth > 1000);', 1),
]


def test_steps_are_covered_and_joined_as_the_kernels_cut_them(tmp_path):
    program = index.PROGRAM
    for old, new, times in CHANGES:
        assert program.count(old) == times, old
        program = program.replace(old, new)
    src, exe = tmp_path / "steps.cpp", str(tmp_path / "steps")
    src.write_text(program)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", index.KERNELS,
                    str(src), "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "ok 1", run.stdout + run.stderr
