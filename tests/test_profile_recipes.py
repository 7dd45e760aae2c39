"""The capture commands of profiles/*.md: a capture of more than the launches' times takes a kernel's launch many times over, so each command asks
for a few launches of what it names, leaves the clocks alone, and follows a run of the same program without the profiler (no GPU needed)."""
import glob
import os
import re

import pytest

from conftest import ROOT

FILES = sorted(glob.glob(os.path.join(ROOT, "profiles", "*.md")))


def commands(text):
    """The capturing commands of the fenced blocks, continued lines joined, without the comments' own."""
    for block in re.findall(r"```\n(.*?)```", text, re.S):
        for line in block.replace("\\\n", " ").splitlines():
            if re.search(r"(^|\s)ncu\s", line) and not line.startswith("#") and not re.search(r"ncu -i ", line):
                yield line


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_a_capture_is_of_a_few_launches(path):
    for line in commands(open(path).read()):
        if "same options" in line:
            continue
        assert "--clock-control none" in line and "&&" in line[:line.index("ncu ")], line
        if "--section" in line or "--set" in line:
            count = re.search(r"\s-c (\d+|\$COUNT)\s", line)
            assert count and (count.group(1) == "$COUNT" or int(count.group(1)) <= 3), line
            assert re.search(r'-k regex:(\w+|\$KERNEL|"\$KERNELS")\s', line), line
