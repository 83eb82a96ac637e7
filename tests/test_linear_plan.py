"""How the work of scores from features and weights is cut (csrc/linear_plan.hpp), compiled with g++."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "lvd-pg_amd", "csrc")


@pytest.fixture(scope="module")
def got(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "linear_plan")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, "-o", exe, os.path.join(HERE, "linear_plan_test.cpp")], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    return dict((l.split()[0], int(l.split()[1])) for l in out.splitlines())


def test_no_launch_has_two_to_the_32_threads(got):
    assert got["tiles_none"] == 0 and got["tiles_past"] == 0 and got["few_past"] == 0
    assert got["tiles_several"] > 0                    # (there are sizes that take several)
    assert got["few_512"] == 2 ** 23 - 1 and got["few_256"] == 2 ** 24 - 1


def test_pieces_and_parts_have_bounds(got):
    assert got["pieces_uneven"] == 0 and got["pieces_large"] == 0 and got["pieces_parts"] > 0
