"""The check of test_float8_asm_cpu on every other source whose kernels load to LDS with inline assembly: M0 is used by those
loads alone. The sources are found by what they include, so that a new one is not missed."""
import os
import re

import pytest

import test_float8_asm_cpu as A

CSRC = os.path.join(A.ROOT, "ocean-tensor-package_amd", "csrc")
LOADING = re.compile(r'#include "och_gemm_f8_(few|pipe)\.h"')
SOURCES = sorted(n for n in os.listdir(CSRC) if n.endswith(".hip") and LOADING.search(open(os.path.join(CSRC, n)).read()))


def test_every_pair_of_code_types_is_there():
    assert SOURCES == ["och_gemm_f8_%s_%d%d.hip" % (k, a, b) for k in ("few", "pipe") for a in (4, 5) for b in (4, 5)]
    assert set(A.SOURCES) <= set(SOURCES)


@pytest.mark.parametrize("source", [s for s in SOURCES if s not in A.SOURCES])
def test_m0_is_used_by_the_loads_to_lds_only(source, tmp_path):
    A.test_m0_is_used_by_the_loads_to_lds_only(source, tmp_path)
