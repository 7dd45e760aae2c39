"""Loads of single 16-bit elements in the kernels' sources (no GPU needed).  The toolkit's own is assembly without effects: the compiler may
move it before the condition that it stands under, to an address behind the last row or to none at all."""
import glob
import os
import re

import pytest

from conftest import ROOT

SOURCES = sorted(glob.glob(os.path.join(ROOT, "actnn_b200", "csrc", "*.cu*")))


def elements(text):
    """The toolkit's loads of elements whose type is a kernel's: turned to float, put beside a zero of the type, or into a vector of one."""
    return re.findall(r"[^\n]*(?:2float\(__ldg\(|__ldg\([^\n]*from_float<T>|\br\.v = __ldg\()[^\n]*", text)


def test_what_is_looked_for():
    for line in ("  return __half2float(__ldg(p + i));", "v = e + i < K ? __ldg(p + e + i) : from_float<T>(0.f);", "    r.v = __ldg(p);"):
        assert elements(line) == [line]
    for line in ("const float s = __ldg(scale + row);", "v = c < n ? load_one(p + c) : from_float<T>(0.f);"):
        assert not elements(line)


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_no_element_is_loaded_by_assembly_that_may_move(path):
    assert not elements(open(path).read())


def test_the_loads_of_an_element_stay():
    text = open(os.path.join(ROOT, "actnn_b200", "csrc", "load_one.cuh")).read()
    assert len(re.findall(r"ACTNN_DEV \S+ load_one\(const \S+ p\) \{", text)) == len(re.findall(r"asm volatile\(\"ld\.global\.nc", text)) == 4
