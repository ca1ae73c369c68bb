"""The packed attention's search for a workgroup's sequence, block and chunk, run on the CPU with every index checked
(native/packed_ranges.cpp): starts and lengths of any content keep each address inside its tensor, consistent ones meet every
block of work exactly once."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("packed_ranges")
    text = open(os.path.join(ROOT, "efficientvlm_amd", "csrc", "packed_attention.hip")).read()
    cut = lambda first, last: text[text.index(first):text.index(last)]
    source = cut("struct PkArgs {", "// ---- 16-byte fragments") + cut("// ---- sequences ---", "// ---- staging")
    source += cut("#define PK_BLOCKS", "// dK / dV, the shape of a block")
    source, n = re.subn(r"const int32_t \*cu_q, \*cu_k, \*k_lens;", "Starts cu_q, cu_k, k_lens;", source)
    assert n == 1
    source = source.replace("outside_rows(const int32_t* cu,", "outside_rows(const Starts& cu,")
    (folder / "source.h").write_text(source)
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wno-unused-function", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    "-I", os.path.join(ROOT, "include"), f'-DPACKED_SOURCE="{folder / "source.h"}"',
                    os.path.join(ROOT, "tests", "native", "packed_ranges.cpp"), "-o", str(folder / "packed_ranges")], check=True)
    return str(folder / "packed_ranges")


@pytest.mark.parametrize("seed", range(3))
def test_every_range_stays_inside_and_every_block_is_met_once(program, seed):
    run = subprocess.run([program, str(seed), "12"], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
