"""Host rules of the 8-bit linear path that pick a kernel by size, compiled on the
CPU from the header that the launches use (csrc/blocks.h)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "onnx-rs_b200", "csrc")


def cuda_include():
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")


def run_cpp(tmp_path, body):
    """The integers that a program around csrc/blocks.h prints, a tuple per line."""
    cxx = shutil.which("g++") or shutil.which("c++")
    if not cxx or not os.path.exists(os.path.join(cuda_include(), "cuda_runtime.h")):
        pytest.skip("no C++ compiler or CUDA headers")
    src, out = tmp_path / "rules.cpp", tmp_path / "rules"
    src.write_text('#include <cstdio>\n#include "blocks.h"\nusing namespace ob2;\nint main() {\n%s\n}\n' % body)
    r = subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-I", CSRC, "-isystem", cuda_include(), str(src), "-o", str(out)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([str(out)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0
    return [tuple(map(int, line.split())) for line in r.stdout.splitlines()]


def test_shared_memory_of_the_product_for_one_or_two_rows(tmp_path):
    """Rows of a that do not fit shared memory never take the kernel that keeps them there, up to the
    longest k the entry accepts (2^31 - 257): around 2^31 a 32-bit count of the bytes comes out small."""
    ks = [1, 16, 128, 4096, 48000, 51200, 60000, 100000, 1 << 26, (1 << 30) - 1, 1 << 30, 2114445439, 2114445440, 2114470000,
          2114495840, 2114495841, (1 << 31) - 257]
    got = run_cpp(tmp_path, "for (int k : {%s}) for (int m : {1, 2, 3})\n"
                  '  printf("%%d %%d %%lld %%d\\n", m, k, (long long)matmul_vec_smem(m, k), (int)matmul_takes_vec(m, k));'
                  % ", ".join(map(str, ks)))
    assert len(got) == 3 * len(ks)
    for m, k, smem, takes in got:
        assert smem == m * (-(-k // 16) * 32 + -(-k // 128) * 4)
        assert takes == (m <= 2 and smem <= 100 * 1024)


# Products with several tiles for a pair of thread blocks, on the 148 SMs of a B200: (m, n, whether tiles are 256 wide)
TILED = [(1777, 5000, True), (2300, 4700, True), (1800, 5003, True), (4096, 4096, True), (8192, 8192, True), (1500, 6700, True),
         (700, 6400, False), (600, 6404, False), (200, 8192, False), (256, 512, False), (1500, 777, False), (70000, 300, False)]


def test_tile_width_of_products_with_many_rows(tmp_path):
    """Wide tiles where their waves take no longer: a wave of narrow ones takes 0.6 of theirs."""
    got = run_cpp(tmp_path, "const int mn[][2] = {%s};\nfor (auto& v : mn) printf(\"%%d %%d %%d\\n\", v[0], v[1], "
                  "(int)matmul_takes_wide(v[0], v[1], 148));" % ", ".join("{%d, %d}" % t[:2] for t in TILED))
    assert [(m, n, bool(w)) for m, n, w in got] == TILED
    for m, n, wide in got:
        waves = [-(-(-(-m // 256) * -(-n // bn)) // 74) for bn in (128, 256)]
        assert wide == (3 * waves[0] >= 5 * waves[1])
