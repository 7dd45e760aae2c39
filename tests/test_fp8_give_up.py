"""What the 8-bit floating-point product does when one of its waits runs out, read from its source: the rules of the integer product,
whose orders of steps tests/test_int8_give_up.py follows one by one, and one for warps that issue by an elected lane."""
import os
import re

from conftest import ROOT

TEXT = open(os.path.join(ROOT, "actnn_b200", "csrc", "fp8_matmul.cu")).read()


def part(first, last):
    return TEXT[TEXT.index(first):TEXT.index(last)]


def test_the_epilogue_leaves_together():
    code = part("---------------- epilogue", "nobody leaves while its sums are read")
    assert re.search(r"const bool ok = warp != 0 \|\| fp_wait\(smem_addr\(&s\.sum_full\[buf\]\)[^;]*;\s*(\w+\(\);\s*)*"
                     r"if \(!epilogue_agrees\(ok\)\) break;", code)
    assert len(re.findall(r"\bbreak;", code)) == 1
    assert re.search(r"barrier\.cta\.red\.and\.pred q, 1, 256, p", TEXT)


def test_lanes_that_elect_one_have_all_come_through_their_wait():
    """Copies and matrix instructions: no wait of a single lane, and every way out of a loop follows a vote."""
    assert re.search(r"return __all_sync\(kFull, ready \|\| fp_wait\(bar, parity, s, gave_up\)\);", TEXT)
    for code in (part("---------------- copies", "---------------- matrix instructions"), part("---------------- matrix instructions", "---------------- epilogue")):
        assert "elect_one()" in code and not re.search(r"\bfp_wait\(|mm_wait\(", code)
        for line in code.splitlines():
            if "break;" in line:
                assert "fp_warp_waits(" in line or line.strip() == "if (!ok) break;"


def test_a_pairs_second_block_waits_for_what_the_first_one_sends():
    copies = part("---------------- copies", "---------------- matrix instructions")
    stages = re.search(r"for \(int i = 0, at = copy_stage; PAIR && copied && i < a\.stages; \+\+i\) \{\s*"
                       r"copied = fp_warp_waits\(false, smem_addr\(&s\.empty\[at\]\), copy_phase \^ \(at < copy_stage \? 0 : 1\)", copies)
    last = re.search(r"if \(PAIR && copied\) copied = fp_warp_waits\(false, smem_addr\(&s\.drained\), 0", copies)
    assert stages and last and stages.start() < last.start()


def test_copies_under_way_are_waited_for_whichever_wait_ran_out():
    end = part("nobody leaves while its sums are read", "// ------------------------------------------------------------------ host")
    drain = re.search(r"__syncthreads\(\);\s*if \(warp == 8 && lane == 0 && s\.dead\) \{", end)
    assert drain and drain.end() < end.index("mbar_wait(smem_addr(&s.full[copy_stage]), copy_phase);") < end.index("if constexpr (PAIR) cluster_sync();")


def test_a_cluster_writes_all_of_a_tile_or_nothing():
    assert TEXT.index("s.gone = 0;") < TEXT.index("if constexpr (SPLIT) cluster_arrive();")
    shared = part("if constexpr (SPLIT) {\n    __syncwarp();", "nobody leaves while its sums are read")
    told = re.search(r"cluster_wait\(\);[^;]*\n(\s*//[^\n]*\n)*\s*if \(s\.dead\)\s*for \(int k = 0; k < a\.splits; \+\+k\) "
                     r"peer_store1\(smem_addr\(&s\.gone\), k, 1\);\s*cluster_sync\(\);\s*if \(warp < 8 && !s\.gone\) \{", shared)
    assert told and told.end() < shared.index("peer_load4") and "fp_wait" not in shared


def plan_tiles():
    """Every tile that the cut can choose: (tokens, whether there are several, wide)."""
    for several in (False, True):
        for tokens in range(16, 225, 16):
            if not several or tokens % 64 == 0:
                yield tokens, several, False
        for tokens in range(256, 449, 64):
            yield tokens, several, True


def test_scales_begin_where_the_instructions_take_them():
    """At an even column of tensor memory: the second operand's scales of a tile, and of a wide tile's second half; and the sets of
    columns fit beside the accumulators, at least as many as keep one from being overwritten while it is read."""
    for tokens, several, wide in plan_tiles():
        first = (tokens // 2 + 63) // 64 * 64 if wide else tokens
        for tile in range(8 if several else 1):
            shift = (tile * tokens & 127) // 32
            assert shift % 2 == 0
            if wide:
                assert (shift + first // 32) % 2 == 0 and first % 64 == 0 and (tokens - first) % 64 == 0 and 0 < tokens - first <= first <= 256
        common = 128
        while tokens % common:
            common //= 2
        atoms = (128 - common + tokens + 127) // 128 if several else (tokens + 127) // 128
        assert atoms <= (4 if wide else 3) and all((t * tokens & 127) + tokens <= atoms * 128 for t in range(8 if several else 1))
        sums = tokens if wide else 2 * tokens
        sets = min(4, (512 - sums) // (4 + 4 * atoms))
        stages = min(8, (216 * 1024 - 1024 - 32 * 1024) // ((128 + tokens // 2) * 128 + 512 * (1 + atoms)))
        assert sets >= 3 and (not wide or 4 * sets - 3 >= stages)
    assert re.search(r"if \(tokens < a\.T\) tokens = \(tokens \+ 63\) / 64 \* 64;", TEXT)
