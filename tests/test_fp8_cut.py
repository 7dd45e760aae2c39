"""The cuts of the 8-bit floating-point product, as its own source makes them (no GPU needed): that their layout holds over all sizes, and which
kernels the sizes of the tests on the GPU take."""
import os
import random
import re

import pytest

from conftest import ROOT
from fp8_cut import Cut

TEXT = open(os.path.join(ROOT, "actnn_b200", "csrc", "fp8_matmul.cu")).read()


def sizes(count, seed):
    rng = random.Random(seed)
    for _ in range(count):
        t, n, k = (int(2 ** rng.uniform(0, top)) for top in (15, 15, 14))
        yield t, n if rng.random() < 0.5 else (n + 7) // 8 * 8, k, rng.choice([148, 148, 132, 160, 74])


def holds(t, n, k, sms):
    c = Cut(t, n, k, n % 8 == 0, sms)
    channels = 256 if c.pair else 128
    assert c.channel_tiles == -(-n // channels) and c.tiles == c.channel_tiles * -(-t // c.tokens) and c.k_blocks == -(-k // 128)
    assert not (c.pair and c.splits > 1) and not (c.wide and not c.pair) and 1 <= c.splits <= 8 and (c.splits == 1 or c.k_blocks >= 2 * c.splits)
    assert c.tokens >= t or c.tokens % 64 == 0
    # what an instruction takes: 16 columns at a time of 128 channels, 32 of 256, 256 at most
    if c.wide:
        assert 256 <= c.tokens <= 448 and c.first % 64 == 0 and (c.tokens - c.first) % 64 == 0 and 0 < c.tokens - c.first <= c.first <= 256
    else:
        assert c.first == c.tokens <= 224 and c.tokens % (32 if c.pair or c.boxes else 16) == 0
    # scales: every tile's lie in its sets of 128 tokens; the copies that the kernel makes
    several = c.tokens < t
    assert all((i * c.tokens & 127) + c.tokens <= c.atoms * 128 for i in range(8 if several else 1))
    assert c.atoms <= (4 if c.wide else 2) and c.set_columns == 4 + 4 * c.atoms and c.stage_scales == 512 * (1 + c.atoms)
    # tensor memory
    sums = c.tokens * (1 if c.wide or c.splits > 1 else 2)
    assert sums + c.sets * c.set_columns <= c.columns <= 512 and c.columns & (c.columns - 1) == 0
    assert 3 <= c.sets <= 4 and 4 * c.sets - 3 >= c.stages
    # shared memory
    stage = (128 + (c.tokens // 2 if c.pair else c.tokens)) * 128
    assert stage % 1024 == 0 and 2 <= c.stages <= 8
    assert c.stages * (stage + c.stage_scales) + (c.staging if c.boxes else 0) + 1024 <= c.bytes
    if c.splits > 1:
        assert not c.boxes and c.tokens * 512 <= c.bytes - 1024 and c.tiles * c.splits <= sms
    return c


@pytest.mark.parametrize("seed", range(4))
def test_the_layout_holds(seed):
    for t, n, k, sms in sizes(20000, seed):
        holds(t, n, k, sms)


def test_the_layout_holds_at_the_ends():
    for t in list(range(1, 520)) + [16383, 16384, 16385, 1 << 20, 1 << 24]:
        for n, k in ((1, 1), (128, 128), (256, 4096), (4096, 129), (16384, 8192), (9810, 3466), (4096, 65536)):
            holds(t, n, k, 148)


def test_scales_beyond_two_sets_are_copied_for_wide_tiles_alone():
    assert max(holds(*s).atoms for s in sizes(3000, 9) if not Cut(*s[:3], s[1] % 8 == 0, s[3]).wide) == 2
    copies = re.findall(r"if \((.*?)\) scales_to_tmem", TEXT)
    assert copies == ["a.atoms > 1", "WIDE && a.atoms > 2", "WIDE && a.atoms > 3"]


def test_the_limits_of_a_tile_are_met():
    """No limit in the offer lies above what is offered."""
    seen = {True: 0, False: 0}
    for t, n, k, sms in sizes(20000, 5):
        c = Cut(t, n, k, n % 8 == 0, sms)
        seen[c.wide] = max(seen[c.wide], c.tokens)
    assert seen == {False: 224, True: 448}
    assert re.search(r"if \(tokens > \(wide \? kFpWide : kFpTokens\) \|\| \(wide && tokens < 256\)\) return;", TEXT)


def test_which_kernels_the_products_on_the_gpu_take():
    from test_fp8_linear_gpu import PRODUCTS
    from test_fp8_wide_tiles_gpu import PRODUCTS as more
    kernels = {}
    for t, n, k in PRODUCTS + [p for p, _ in more]:
        for whole in (n % 8 == 0, n % 4 == 0):                 # results of 16 and of 32 bits
            c = holds(t, n, k, 148)
            kernels.setdefault(Cut(t, n, k, whole).kernel(), set()).add((c.tiles > 74, min(c.k_blocks, 9)))
    for pair in (96, 128, 160, 192, 224):
        assert {("pair", pair, True), ("pair", pair, False)} <= set(kernels)
    for wide in (256, 320, 384, 448):
        for boxes in (True, False):
            assert {many for many, _ in kernels[("wide", wide, boxes)]} == {True, False}      # one round of tiles, and several
    assert {("split%d" % s) for s in (2, 4, 8)} | {"single", "pair", "wide"} == {k for k, _, _ in kernels}
    assert {k for b in (True, False) for _, k in kernels[("wide", 448, b)]} >= {4, 5, 6, 7, 8}       # as many stages as there are, and more
    for (t, n, k), name in more:
        c = Cut(t, n, k, n % 8 == 0)
        assert name == "%s %d" % (c.kernel()[0], c.tokens)
