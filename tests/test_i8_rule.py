"""Which kernel takes an 8-bit product (helixml_amd/csrc/hx_i8_rule.h), on the host: one that is made for many rows does not take one token's
logits, however many outputs there are."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    exe = tmp_path_factory.mktemp("i8") / "i8_rule"
    if shutil.which("g++") is None:
        pytest.skip("g++ needed")
    r = subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'helixml_amd' / 'csrc'}", str(ROOT / "tests" / "cpp" / "i8_rule.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def of(sizes):
        r = subprocess.run([str(exe)], input="\n".join(" ".join(str(int(v)) for v in s) for s in sizes), capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        return r.stdout.split("\n")[:-1]
    return of


def test_few_rows_of_a_large_vocabulary(rule):
    """Up to 16 rows go through the few rows' kernel, up to 128 never through tiles of 256 rows."""
    outs = [1, 1000, 65280, 65281, 128256, 131072, 1 << 20, (1 << 26) - 1]
    inner = [64, 2048, 4096, 8192, (1 << 17) - 1]
    for m in (1, 2, 15, 16):
        assert set(rule([(m, n, k, 1) for n in outs for k in inner])) == {"rows 16x16"}, m
    for m in (17, 33, 64, 127, 128):
        assert "tiles 256" not in rule([(m, n, k, 1) for n in outs for k in inner]), m


def test_measured_sizes(rule):
    """The faster one of those that were timed."""
    cases = {(48, 2048, 8192): "rows 32x32", (32, 2048, 8192): "rows 16x16", (256, 1024, 8192): "rows 32x32", (512, 2048, 2048): "rows 32x32",
             (1024, 2048, 2048): "tiles 128", (4096, 4096, 8192): "tiles 256", (8192, 8192, 4096): "tiles 256", (13479, 13976, 272): "tiles 128",
             (1, 131072, 4096): "rows 16x16", (32, 131072, 4096): "tiles 128", (64, 131072, 4096): "tiles 128", (128, 131072, 4096): "tiles 128",
             (129, 131072, 4096): "tiles 256", (256, 131072, 4096): "tiles 256", (64, 65536, 8192): "tiles 128", (512, 65536, 8192): "tiles 256"}
    assert dict(zip(cases, rule([(*s, 1) for s in cases]))) == cases


def test_rows_that_start_anywhere(rule):
    """Tiles take rows of X in pieces of 16 bytes."""
    sizes = [(m, n, k, 0) for m in (1, 128, 129, 8192) for n in (2048, 131072) for k in (2048, 8192)]
    assert all(k.startswith("rows") for k in rule(sizes))
