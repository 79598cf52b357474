"""What the operators on the text side take and refuse at the edges of their documented limits, on the CPU (their C entry points with no
rows, which check everything else and launch nothing), and which tiles their products take."""

import ctypes
import pathlib
import subprocess

from attention_forms import SHARED
from fp8_tiles import TILES


def test_strides_of_attention_over_packed_rows(pkg):
    """Rows lie less than 2^22 elements apart (24-bit and 32-bit offsets inside a tile); heads up to 2^40."""
    lib, arg = pkg._lib.load(), pkg._lib.WANMI_ERR_ARG

    def cross(ss=256, hs=64, k_hs=64):
        return lib.wanmi_packed_cross_attention(16, ss, hs, 16, ss, k_hs, 16, ss, k_hs, 16, 16, 2, 0, 4, 4, 4, 64, 0.5, 16, 256, None, 1, None)

    def bias(ss=256, hs=64):
        starts = (ctypes.c_int * 4)(0, 1, 2, 5)
        return lib.wanmi_relative_bias_attention(16, ss, hs, 16, ss, hs, 16, ss, hs, 16, 2, 0, 4, 64, 1.0, 16, 0, starts, 4, 1, 16, 256, 1, None)

    for fn in (cross, bias):
        for kw in (dict(), dict(hs=1 << 22), dict(hs=75600 * 128), dict(hs=(1 << 40) - 8), dict(ss=(1 << 22) - 8)):
            assert fn(**kw) == 0, (fn.__name__, kw)
        for kw in (dict(ss=1 << 22), dict(hs=1 << 40), dict(hs=(1 << 22) + 4), dict(hs=-64), dict(ss=-256)):
            assert fn(**kw) == arg, (fn.__name__, kw)
    assert cross(k_hs=1 << 23) == 0 and cross(k_hs=1 << 40) == arg


def _plans(tmp_path, body, header="fp8_plan.h"):
    """What a program around a header of rules prints, line by line."""
    root = pathlib.Path(__file__).resolve().parents[1]
    (tmp_path / "main.cc").write_text(f'#include "{header}"\n#include <cstdio>\nusing namespace wanmi;\n' + body)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{root / 'vllm-omni-neuron_amd' / 'csrc'}", str(tmp_path / "main.cc"), "-o",
                    str(tmp_path / "main")], check=True)
    return subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True, timeout=120).stdout.splitlines()


def test_the_measured_and_tested_tiles_are_taken(tmp_path):
    """The sizes of the GPU tests take the tiles and parts that they are there for, and every kind has some."""
    names = {"64": "kFp8Tiles64", "128 deep": "kFp8Tiles128Deep", "128": "kFp8Tiles128", "256": "kFp8Tiles256"}
    lines = "".join(f"  {{ const Fp8Plan p = fp8_plan({M}, {N}, {-(-K // 128)}); printf(\"%d %d\\n\", p.tiles == {names[tile]}, p.splits); }}\n"
                    for (M, K, N), (tile, _) in TILES.items())
    got = _plans(tmp_path, "int main() {\n" + lines + "}\n")
    assert [(size, line) for (size, (_, parts)), line in zip(TILES.items(), got) if line != f"1 {parts}"] == []
    kinds = {(tile, parts > 1) for tile, parts in TILES.values()}
    assert kinds == {("64", False), ("64", True), ("128 deep", False), ("128 deep", True), ("128", False), ("256", False)}


def test_the_parts_of_a_sum_are_no_larger_than_its_operands_twice(tmp_path):
    """Their workspace against codes, weight and output of the product: 1.9 times as much at most over the range (722 x 5120 x 640: 14.8 MB
    beside 7.9), and below 400 MB."""
    out = _plans(tmp_path, r"""
int main() {
  double share = 0, most = 0;
  for (int64_t N : {8, 64, 640, 2568, 5120, 13824, 15360, 1 << 20})
    for (int64_t KB : {1, 2, 3, 5, 33, 40, 108, 864})
      for (int64_t M = 17; M <= 33000; M += M < 600 ? 1 : 61) {
        const Fp8Plan p = fp8_plan(M, N, KB);
        if (p.splits == 1) continue;
        const double parts = 4.0 * p.splits * M * N, own = (M + N) * KB * 128.0 + 2.0 * M * N;
        share = std::max(share, parts / own);
        most = std::max(most, parts);
      }
  printf("%f\n%f\n", share, most);
}
""")
    assert 1.0 < float(out[0]) < 1.9 and float(out[1]) < 400e6


def test_the_tiles_of_attention_over_packed_rows(tmp_path):
    """Shared keys where every tile is on the chip at once and has more than 64 keys; one long request beside many short ones, short texts
    and many requests take 128 rows a tile, whatever their average."""
    shared = [(sum(q) + pad, sum(k), len(q), heads, D) for q, k, pad, heads, _, D in SHARED]
    shared += [(1, 512, 1, 40, 128), (128, 2000, 1, 40, 128), (128, 2048, 4, 40, 128), (32, 16384, 32, 8, 64), (1024, 1024, 1, 12, 64), (100, 100, 1, 12, 64),
               (270, 270, 3, 4, 128), (201, 201, 2, 8, 64)]
    rows = [(3127, 65536, 128, 40, 128), (1063, 32768, 64, 40, 128), (531, 16384, 32, 64, 64), (1280, 32768, 64, 40, 128), (12, 12, 1, 64, 64), (16, 64, 1, 40, 128),
            (1, 1, 1, 1, 64), (200, 512, 1, 40, 128), (32760, 1024, 2, 40, 128), (256, 8192, 16, 40, 128)]
    lines = "".join(f'  printf("%d\\n", packed_keys_shared({T}, {Tk}, {R}, {H}, {D}));\n' for T, Tk, R, H, D in shared + rows)
    got = _plans(tmp_path, "int main() {\n" + lines + "}\n", "packed_attention_plan.h")
    assert got == ["1"] * len(shared) + ["0"] * len(rows)
