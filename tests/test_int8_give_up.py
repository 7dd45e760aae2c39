"""What the integer product does when one of its waits runs out, shown on the CPU: every order in which its warps can take their
steps is followed, and none may end with some of them waiting for others that have left."""
import os
import re

import pytest

from conftest import ROOT

SOURCE = os.path.join(ROOT, "actnn_b200", "csrc", "int8_matmul.cu")


def ends(warps, tiles, together):
    """All ends of an epilogue of `warps` warps over `tiles` tiles, each warp's last place.  A warp waits for its tile (the phase may
    complete at any time, another wait of the block may run out at any time; a try looks at the phase first, then at the flag)
    and passes a barrier that counts all warps.  `together`: the barrier also tells whether every wait was good, and all leave
    where one was not; otherwise a warp whose wait was not good leaves by itself."""
    start = (tuple(("try", 0) for _ in range(warps)), 0, False)         # places, tiles complete, flag
    seen, todo, found = {start}, [start], set()
    while todo:
        places, complete, dead = todo.pop()
        after = []
        if complete < tiles:
            after.append((places, complete + 1, dead))
        if not dead:
            after.append((places, complete, True))
        for i, (what, tile) in enumerate(places):
            def to(place):
                return places[:i] + (place,) + places[i + 1:]
            if what == "try":                               # the phase
                after.append((to(("through", tile) if tile < complete else ("flag", tile)), complete, dead))
            elif what == "flag":                            # then the flag
                bad = ("bad", tile) if together else ("left", tile)
                after.append((to(bad if dead else ("try", tile)), complete, dead))
        at = [w for w, _ in places]
        if all(w in ("through", "bad") for w in at):        # the barrier is complete
            on = ("try", places[0][1] + 1) if places[0][1] + 1 < tiles else ("done", tiles)
            after.append((tuple(("left", t) if "bad" in at else on for _, t in places), complete, dead))
        moved = [s for s in after if s != (places, complete, dead)]
        if not moved:
            found.add(places)
        for s in moved:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return found


@pytest.mark.parametrize("warps,tiles", [(2, 1), (2, 3), (3, 2), (4, 2)])
def test_the_epilogue_leaves_together(warps, tiles):
    alone = ends(warps, tiles, False)
    assert any({"left", "through"} <= {w for w, _ in e} for e in alone)         # what leaving one by one can end with
    for e in ends(warps, tiles, True):
        assert {w for w, _ in e} in ({"left"}, {"done"})


def epilogue():
    text = open(SOURCE).read()
    return text[text.index("---------------- epilogue"):text.index("host")]


def test_the_kernel_asks_all_warps_before_it_goes_on():
    """Between the wait for a tile's sums and anything else of the tile stands the vote of all eight warps, and no warp leaves by
    its own result."""
    code = epilogue()
    assert re.search(r"const bool ok = (warp != 0 \|\| )?mm_wait\(smem_addr\(&s\.sum_full\[buf\]\)[^;]*;\s*(\w+\(\);\s*)*"
                     r"if \(!epilogue_agrees\(ok\)\) break;", code)
    assert len(re.findall(r"\bbreak;", code)) == 1 and "bar.sync 1" not in code
    assert re.search(r"barrier\.cta\.red\.and\.pred q, 1, 256, p", open(SOURCE).read())


@pytest.mark.parametrize("stages", [1, 2, 3, 5, 8])
def test_every_stage_is_waited_for_at_the_end(stages):
    """The thread that requests copies waits, before its block may leave, for the last arrival at every stage's barrier: the parity it asks
    for is that of the last phase that the stage's matrix instructions complete, and one that is over where there were none."""
    for issued in range(4 * stages + 1):
        stage, phase, rounds = 0, 0, [0] * stages          # rounds: how often a stage was filled, so how many phases will complete
        for _ in range(issued):
            rounds[stage] += 1
            stage += 1
            if stage == stages:
                stage, phase = 0, phase ^ 1
        at, asked = stage, []
        for _ in range(stages):
            asked.append((at, phase ^ (0 if at < stage else 1)))
            at = (at + 1) % stages
        assert sorted(a for a, _ in asked) == list(range(stages))
        for a, parity in asked:
            # a wait for a parity ends when the phase that runs has the other one, and no sooner than after the last arrival
            assert [done for done in range(rounds[a] + 1) if done % 2 != parity][-1] == rounds[a]
            assert rounds[a] == 0 or (rounds[a] - 1) % 2 == parity


def test_the_kernel_waits_for_what_the_pairs_first_block_sends():
    text = open(SOURCE).read()
    copies = text[text.index("---------------- copies"):text.index("---------------- matrix instructions")]
    stages = re.search(r"for \(int i = 0, at = copy_stage; PAIR && copied && i < a\.stages; \+\+i\) \{\s*"
                       r"copied = mm_wait\(smem_addr\(&s\.empty\[at\]\), copy_phase \^ \(at < copy_stage \? 0 : 1\), s, gave_up\);", copies)
    last = re.search(r"if \(PAIR && copied\) copied = mm_wait\(smem_addr\(&s\.drained\), 0", copies)
    assert stages and last and stages.start() < last.start()


def test_copies_under_way_are_waited_for_whichever_wait_ran_out():
    """Behind the block's last barrier, when every thread's waits are over."""
    text = open(SOURCE).read()
    end = text[text.index("nobody leaves while its sums are read"):text.index("host")]
    drain = re.search(r"__syncthreads\(\);\s*if \(warp == 8 && lane == 0 && s\.dead\) \{", end)
    assert drain and drain.end() < end.index("mbar_wait(smem_addr(&s.full[copy_stage]), copy_phase);") < end.index("if constexpr (PAIR) cluster_sync();")


def test_a_cluster_writes_all_of_a_tile_or_nothing():
    """A reduction that blocks share: a thread whose wait ran out tells every block of the cluster, between the barrier that says that all have
    set their flags and the one behind which the sums are read, and nothing is written where one has told.  No wait for a phase
    stands behind the latter."""
    text = open(SOURCE).read()
    assert re.search(r"s\.dead = s\.gone = 0;", text) and text.index("s.gone = 0;") < text.index("if constexpr (SPLIT) cluster_arrive();")
    shared = text[text.index("if constexpr (SPLIT) {\n    __syncwarp();"):text.index("nobody leaves while its sums are read")]
    told = re.search(r"cluster_wait\(\);[^;]*\n(\s*//[^\n]*\n)*\s*if \(s\.dead\)\s*for \(int k = 0; k < a\.splits; \+\+k\) "
                     r"peer_store1\(smem_addr\(&s\.gone\), k, 1\);\s*cluster_sync\(\);\s*if \(warp < 8 && !s\.gone\) \{", shared)
    assert told and told.end() < shared.index("peer_load4i") and "mm_wait" not in shared
