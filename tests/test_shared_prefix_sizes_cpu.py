"""How attention over a shared prefix cuts its work where that passes 32 bits: the plan's arithmetic, compiled for the host."""
import subprocess

import pytest

from tests.conftest import ROOT

CTAS = 148

PROGRAM = r"""
#include <cstdint>
#include <cstdio>

#include "shared_prefix.cuh"

int main() {
    long long tiles, each;
    int ctas;
    while (std::scanf("%lld %lld %d", &tiles, &each, &ctas) == 3) {
        const int64_t work = b200::shared_unit_work(static_cast<int>(tiles), static_cast<int>(each));
        std::printf("%lld %d\n", static_cast<long long>(work), b200::shared_stages_per_item(work, ctas));
    }
}
"""

# (row tiles, stages that each of them goes over): one request's rows behind its own keys
WORK = [(1, 1), (1, 2), (1, 6), (1, 149), (8, 100), (148, 5), (148, 6), (149, 7), (64, 65536), (4096, 4096), (16384, 65535), (16384, 65536),
        (16385, 65536), (32767, 65536), (32768, 65536), (65536, 65536), (131072, 32768), (2 ** 20, 2 ** 25), (2 ** 28, 2 ** 25), (3, 2 ** 25)]


@pytest.fixture(scope="module")
def answers(pkg, tmp_path_factory):
    from sglang_cpp_b200 import build
    where = tmp_path_factory.mktemp("sizes")
    source, program = where / "sizes.cu", where / "sizes"
    source.write_text(PROGRAM)
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-I", str(build.CSRC), "-I", str(ROOT / "include"), "-o", str(program), str(source)],
                   check=True, capture_output=True, text=True)
    said = subprocess.run([str(program)], input="".join(f"{t} {s} {CTAS}\n" for t, s in WORK), check=True, capture_output=True, text=True).stdout
    return dict(zip(WORK, (tuple(map(int, line.split())) for line in said.splitlines())))


@pytest.mark.parametrize("tiles,stages", WORK)
def test_stages_per_item(answers, tiles, stages):
    """Counted in full, and no more items than there is room for: four per CTA and one per row tile."""
    work, piece = answers[tiles, stages]
    assert work == tiles * stages
    assert piece >= 2
    assert tiles * -(-stages // piece) <= 4 * CTAS + tiles
    if work >= 4 * CTAS * 6:     # ... of which a good part is made use of
        assert piece <= max(-(-work // (2 * CTAS)), 6)
