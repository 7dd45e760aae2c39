"""The cut that the 8-bit floating-point product makes of its sizes: `plan` of its source, compiled for the host (no GPU needed)."""
import ctypes
import functools
import os
import shutil
import subprocess
import tempfile

import pytest

from conftest import ROOT

FIELDS = "tokens splits pair wide boxes stages atoms sets set_columns columns first channel_tiles tiles stage_scales k_blocks".split()


@functools.lru_cache(None)
def _library():
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    text = open(os.path.join(ROOT, "actnn_b200", "csrc", "fp8_matmul.cu")).read()

    def part(first, last):
        return text[text.index(first):text.index(last, text.index(first))]

    source = "\n".join([
        "#include <algorithm>", "#include <cstdint>", "struct Device { int sm_count; };", "static Device device;", "static Device& device_info() { return device; }",
        part("constexpr int kFpThreads", "struct FpShared"), part("void plan(FpArgs& a) {", "struct FpMaps"),
        'extern "C" int limit() { return kFpSmem; }', 'extern "C" int staging() { return kFpStaging; }',
        'extern "C" void cut(int64_t T, int64_t N, int K, int boxes, int sms, int64_t* out) {',
        "  device.sm_count = sms;", "  FpArgs a{};", "  a.T = T, a.N = N, a.K = K, a.boxes = boxes != 0;", "  plan(a);",
        "  const int64_t v[] = {%s};" % ", ".join("(int64_t)a." + f for f in FIELDS), "  for (int64_t i : v) *out++ = i;", "}"])
    with tempfile.TemporaryDirectory() as folder:
        path = os.path.join(folder, "cut.cpp")
        with open(path, "w") as f:
            f.write(source)
        subprocess.run([compiler, "-std=c++17", "-O1", "-shared", "-fPIC", path, "-o", path + ".so"], check=True, capture_output=True)
        lib = ctypes.CDLL(path + ".so")
    lib.cut.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    return lib


class Cut:
    """What `plan` says of a product of t tokens by n channels over k on a device of `sms` multiprocessors; `boxes`: rows of the result are whole
    16 bytes."""

    def __init__(self, t, n, k, boxes=True, sms=148):
        out = (ctypes.c_int64 * len(FIELDS))()
        _library().cut(t, n, k, int(boxes), sms, out)
        for name, value in zip(FIELDS, out):
            setattr(self, name, int(value))
        self.bytes, self.staging = _library().limit(), _library().staging()

    def kernel(self):
        """Which of the four kernels, tokens of a tile, whether outputs leave as boxes."""
        return ("wide" if self.wide else "pair" if self.pair else "split%d" % self.splits if self.splits > 1 else "single"), self.tokens, bool(self.boxes)
