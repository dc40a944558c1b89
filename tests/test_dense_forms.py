"""CPU suite: what the host classes of clipped gradients refuse (tests/cpp/test_dense_objects.cpp); which form (straight or packed, wavefronts, tiles, shared k axes, pieces) a size of a dense layer or of the loss on top of one takes (tests/cpp/test_dense_forms.cpp)."""
import os
import subprocess

import pytest

import dense_sizes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def tool(*args, name="test_dense_forms"):
    exe = os.path.join(ROOT, "tests", "cpp", name)
    if not os.path.exists(exe):
        from binarybrain_amd.build import build_cpp_tests
        build_cpp_tests()
    res = subprocess.run([exe, *map(str, args)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert res.returncode == 0, res.stdout
    return res.stdout.strip()


def test_rules():
    """no rule asks for a number of wavefronts that no kernel has"""
    tool("--rules")


def test_objects():
    tool(name="test_dense_objects")


@pytest.mark.parametrize("what,size", [(what, size) for what, sizes in (("forward", dense_sizes.FORWARD), ("backward", dense_sizes.BACKWARD), ("loss", dense_sizes.LOSS)) for size in sizes])
def test_sizes_take_the_forms_that_they_are_there_for(what, size):
    assert tool(what, *size) == getattr(dense_sizes, what.upper())[size]
