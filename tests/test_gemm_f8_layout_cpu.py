"""The LDS layout of the block-scaled 8-bit product, walked through on the host: tests/gemm_f8_slab_host.cpp compiles
csrc/och_gemm_f8_slab.h and checks that every byte of a fragment is the element it has to be, that the chunks cover the
slab once, and that the lanes which read together meet different banks."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def slab(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("slab") / "gemm_f8_slab_host.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "ocean-tensor-package_amd", "csrc"),
                    os.path.join(ROOT, "tests", "gemm_f8_slab_host.cpp"), "-o", so], check=True)
    lib = C.CDLL(so)
    lib.gemm_f8_slab_check.restype = C.c_long
    return lib


@pytest.mark.parametrize("rows", [32, 64, 128, 256])
@pytest.mark.parametrize("kc", [0, 1], ids=["contiguous_along_rows", "contiguous_along_k"])
def test_every_fragment_byte_is_the_element_it_has_to_be(slab, kc, rows):
    assert slab.gemm_f8_slab_check(kc, rows) == 0
