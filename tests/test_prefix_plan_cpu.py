"""The plan of tt_shared_prefix_attention (tritiercache_b200/csrc/tt_prefix_plan.cuh), checked on the host by
tests/prefix_plan_check.cu, and that the GPU tests' shapes take the plans they are there for.  nvcc builds the check as
a host program; no GPU is used."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


def plans(tmp_path, shapes):
    """(walk_prefix, tile rows, row tiles, lanes, spans a unit, key tiles a span, most spans and most units of a CTA,
    workspace) of each shape."""
    if not os.path.exists(NVCC):
        pytest.skip("nvcc not available")
    exe = str(tmp_path / "prefix_plan_check")
    subprocess.run([NVCC, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a", "-o", exe,
                    os.path.join(HERE, "prefix_plan_check.cu")], check=True, capture_output=True, timeout=300)
    out = subprocess.run([exe], input="\n".join(" ".join(map(str, s)) for s in shapes), capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.splitlines()[-1].startswith("ok"), out.stdout + out.stderr
    return [tuple(map(int, line.split()[1:])) for line in out.stdout.splitlines()[:-1]]


def test_plans_cover_every_tile_once_and_the_gpu_tests_reach_them(tmp_path):
    from test_gpu_prefix_plans import CROSSING
    got = plans(tmp_path, [(R, nq, nkv, hd, prefix, P, most // P + 2) for R, nq, nkv, hd, prefix, most, P, *_ in CROSSING])
    assert len(got) == len(CROSSING)
    kinds = set()
    for case, (walk, tile_rows, row_tiles, lanes, spans, per, most_spans, most_units, _) in zip(CROSSING, got):
        # each case crosses: a CTA takes spans of several units
        assert not walk and spans == 0 and most_spans > 1 and most_units > 1, case
        kinds.add((tile_rows, row_tiles > 1, lanes > 1, case[3]))
        # a last key tile that is not whole, in the middle of a CTA's life: V is cleared and the pass goes on
        kinds.add(("cut", tile_rows, case[4] % 128 != 0))
    for hd in (64, 128):
        assert {(128, False, False, hd), (256, False, False, hd), (256, True, False, hd)} <= kinds
    assert (256, True, True, 128) in kinds  # row tiles side by side
    assert {("cut", 128, True), ("cut", 256, True)} <= kinds
    assert any(p[6] > 2 for p in got)  # three spans of a CTA
