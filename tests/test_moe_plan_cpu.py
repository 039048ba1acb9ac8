"""How the mixture-of-experts kernel deals its work out, walked through on the host.

tests/c_runtime/moe_plan.cpp includes the kernel's own partition and checks, for every
CTA of a grid, that each K block is done once, that shared tiles' partial sums are
looked for where they were left, and that no CTA overwrites sums which others may
still be reading."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
SRC = Path(__file__).resolve().parent / "c_runtime" / "moe_plan.cpp"


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is missing")
    exe = tmp_path_factory.mktemp("moe_plan") / "moe_plan"
    proc = subprocess.run([gxx, "-O2", "-std=c++17", "-Wno-unknown-pragmas", str(SRC),
                           f"-I{ROOT / 'deepx_op_gpukernelcompiler_b200' / 'csrc'}", "-o", str(exe)],
                          capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-3000:]

    def run(*args):
        proc = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, timeout=60)
        return proc.stdout.strip()

    return run


@pytest.mark.parametrize("grid,D,H,chosen", [
    # More output tiles than CTAs, and CTAs whose split units lie in two tiles.
    (148, 65536, 192, 1), (148, 40072, 1448, 3), (148, 49152, 1024, 8), (148, 65536, 65536, 2),
    # The same on a part of the SMs, at ordinary widths.
    (24, 7168, 2048, 8), (8, 2880, 2880, 1), (16, 5120, 1536, 6), (1, 512, 256, 2),
    # Fewer tiles than CTAs; both phases whole; one K block.
    (148, 4096, 14336, 2), (148, 2048, 1024, 64), (148, 1032, 2824, 16), (148, 40072, 72, 3),
    (148, 136, 20000, 3), (148, 8, 8, 1), (148, 64, 64, 256),
])
def test_plan(plan, grid, D, H, chosen):
    assert plan(grid, D, H, chosen) == "ok"


def test_drawn_plans(plan):
    rng = random.Random(1)
    for _ in range(120):
        grid = rng.choice([1, 2, 8, 16, 24, 40, 74, 132, 148])
        D, H = (8 * round(2 ** rng.uniform(0, 13)) for _ in range(2))
        chosen = rng.randint(1, min(256, max(1, 2 ** 27 // (D * H))))
        assert plan(grid, D, H, chosen) == "ok", (grid, D, H, chosen)
