"""How the work of scores from features and weights is cut (csrc/linear_plan.hpp), compiled with g++."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "lvd-pg_amd", "csrc")


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "linear_plan")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, "-o", exe, os.path.join(HERE, "linear_plan_test.cpp")], check=True)

    def run(*args):
        out = subprocess.run([exe, *map(str, args)], check=True, capture_output=True, text=True).stdout
        return dict((l.split()[0], int(l.split()[1])) for l in out.splitlines())
    return run


@pytest.fixture(scope="module")
def got(run):
    return run()


def test_no_launch_has_two_to_the_32_threads(got):
    assert got["tiles_none"] == 0 and got["tiles_past"] == 0 and got["few_past"] == 0
    assert got["tiles_several"] > 0                    # (there are sizes that take several)
    assert got["few_512"] == 2 ** 23 - 1 and got["few_256"] == 2 ** 24 - 1


def test_pieces_and_parts_have_bounds(got):
    assert got["pieces_uneven"] == 0 and got["pieces_large"] == 0 and got["pieces_parts"] > 0


def test_the_sizes_for_wide_tiles_select_them(run):
    """What the GPU tests take for products of 256 x 256 tiles is cut into such, so that a change of the rule cannot empty them"""
    import linear_reference as R
    steps = lambda n, each: -(-n // each)
    for (rows, length, cats), which, pieces in R.WIDE:
        planes = 2 if rows < 1024 else 1
        most = min(cats, run(rows, length)["piece"])
        assert steps(cats, most) == pieces
        for piece in {most} if pieces == 1 else range(most // 2 + 256, most + 1, 256):      # (pieces may be cut smaller, down to half)
            is_wide = {"scores": run(piece, rows, steps(length, 64)), "features": run(length, rows, planes * steps(piece, 64)),
                       "weight": run(length, piece, planes * steps(rows, 64))}
            assert all(is_wide[name]["wide"] == 1 for name in which), (rows, length, piece, is_wide)
    for rows, length, cats in R.WIDE8:
        assert run(cats, rows, steps(length, 128))["wide"] == 1
