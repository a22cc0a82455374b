"""The rules by which a 4-bit product is cut (csrc/xv_fp4_plan.h, compiled here
without HIP): the GPU tests' shapes reach every kernel that any product
reaches, and the workspace that a caller asks for is what the cut needs."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

from mxfp4_shapes import SHAPES

CSRC = Path(__file__).resolve().parents[1] / "xixi-vllm_amd" / "csrc"
WRAPPER = """
#include "xv_fp4_plan.h"
extern "C" int is_short(int m) { return m <= kShort; }
extern "C" void plan(int m, int n, int k, int silu, int* out) {
  if (m <= kShort) { const ShortPlan p = short_plan(m, n, k, silu != 0); out[0] = p.tiles; out[1] = 0; out[2] = p.parts; }
  else { const TilePlan p = tile_plan(m, n, k, silu != 0); out[0] = p.mtw; out[1] = p.nt; out[2] = p.parts; }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(WRAPPER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "plan.cpp"), "-o", str(d / "plan.so")],
                   check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    out = (ctypes.c_int * 3)()

    def call(m, n, k, silu):
        lib.plan(m, n, k, int(silu), out)
        return bool(lib.is_short(m)), tuple(out)

    return call


def _kernels(plan, m, n, k, silu):
    """What a product runs: its kernel's template arguments and the branches that sizes choose."""
    short, (a, b, parts) = plan(m, n, k, silu)
    whole = (n // 2 if silu else n) % 4 == 0  # outputs in fours
    if short:
        rows = next(r for r in (8, 16, 32, 48, 64) if m <= r)
        return {("short", rows, a, silu, k // 32 % 4 != 0), ("short parts", rows, parts, silu), ("sum", parts > 1, silu, whole)}
    blocks = -(-m // (32 * a))
    full = m - 32 * a * (blocks - 1) > (2 * a - 1) * 16
    return {("tile", a, b, silu), ("tile end", a, full), ("tile scales", b, silu, k // 32 % 4 != 0), ("tile parts", parts, silu),
            ("sum", parts > 1, silu, whole), ("tile blocks", min(blocks, 3))}


def test_test_shapes_reach_every_kernel(plan):
    reached = set().union(*(_kernels(plan, *s, silu) for s in SHAPES for silu in (False, True)))
    assert len([r for r in reached if r[0] == "short"]) == 2 * 5 * (4 + 3)  # 1, 2, 4, 6 tiles; an even number with SiLU
    assert len([r for r in reached if r[0] == "tile"]) == 5 * (3 + 2)       # 1, 2, 4 row tiles; 2, 4 with SiLU
    rng = random.Random(3)
    for _ in range(100000):
        m = min(int(2 ** rng.uniform(0, 10)), 700)
        n, k = 2 * int(2 ** rng.uniform(0, 18)), 32 * int(2 ** rng.uniform(0, 11))
        silu = rng.random() < 0.5
        more = _kernels(plan, m, n, k, silu) - reached
        assert not more, (m, n, k, silu, more)


def test_workspace_is_that_of_the_parts(plan):
    from xvllm import _C
    from xvllm.layers.linear import MXFP4_WHOLE_ROWS

    rng = random.Random(4)
    for _ in range(3000):
        m, n, k = rng.randint(1, 300), 2 * int(2 ** rng.uniform(0, 15)), 32 * int(2 ** rng.uniform(0, 10))
        silu = rng.random() < 0.5
        parts = plan(m, n, k, silu)[1][2]
        assert _C.lib().xv_mxfp4_gemm_workspace_size(m, n, k, silu) == (parts * m * n * 4 if parts > 1 else 0)
        assert parts == 1 or m > MXFP4_WHOLE_ROWS
