"""What the blocks that share a row of the norm's backward pass do when a wait for one another's sums runs out: their steps are played on the
CPU in many orders, sums delayed, waits run out, and the rules that make every order safe are read from the kernel's source (no GPU needed)."""
import os
import random
import re

import pytest

from conftest import ROOT

TEXT = open(os.path.join(ROOT, "actnn_b200", "csrc", "residual_norm.cuh")).read()
KERNEL = TEXT[TEXT.index("rn_backward_kernel(const __grid_constant__"):TEXT.index("// The partial sums of the runs, added in order")]


class Barrier:
    """Counts one arrival, which says how many messages to expect, and the messages; a phase is over when both are there."""

    def __init__(self):
        self.phase, self.pending, self.missing, self.broken = 0, 1, 0, False

    def over(self):
        if self.pending == 0 and self.missing == 0:
            self.phase, self.pending = self.phase + 1, 1

    def expect(self, messages):
        self.broken |= self.pending == 0                     # a second arrival in one phase
        self.pending, self.missing = self.pending - 1, self.missing + messages
        self.over()

    def message(self):
        self.missing -= 1
        self.over()

    def done(self, parity):
        return self.phase % 2 != parity


def play(rng, blocks, warps, rows, quiet, outlast):
    """One order of the steps: what went wrong in it.  `quiet`: a warp whose wait ran out sends nothing more; `outlast`: before its block may
    go, it waits for what is on its way there."""
    bars = [[Barrier(), Barrier()] for _ in range(blocks)]
    sums = [[{}, {}] for _ in range(blocks)]                 # [block][place]: sender -> row
    flying, wrong, state, time = [], set(), {}, 0
    team = [(b, w) for b in range(blocks) for w in range(warps)]
    for who in team:
        state[who] = dict(row=0, at="send", ok=True, seen=[], since=0)
    arrived = set()
    while True:
        moves = [("land", m) for m in flying]
        for who in team:
            s = state[who]
            if s["at"] == "wait":
                bar = bars[who[0]][s["row"] & 1]
                if bar.done(s["row"] >> 1 & 1):
                    moves.append(("go", who))
                elif not any(m[0] == who[0] and m[4] < s["since"] for m in flying):      # a limit outlasts what was sent before it began
                    moves.append(("out", who))
            elif s["at"] == "leave":
                if len(arrived) == len(team) and (s["ok"] or not outlast or not any(m[0] == who[0] for m in flying)):
                    moves.append(("go", who))
            elif s["at"] != "gone":
                moves.append(("go", who))
        moves = [m for m in moves if m[0] != "out" or rng.random() < 0.3] or moves
        if not moves:
            break
        kind, what = rng.choice(moves)
        time += 1
        if kind == "land":
            flying.remove(what)
            to, place, sender, row, _ = what
            if all(state[(to, w)]["at"] == "gone" for w in range(warps)):
                wrong.add("sums reach a block that has left")
            sums[to][place][sender] = row
            bars[to][place].message()
            continue
        s = state[what]
        place, me = s["row"] & 1, what[0]
        if kind == "out":
            s["ok"], s["at"], s["seen"] = False, "read", []
        elif s["at"] == "send":
            if s["ok"] or not quiet:
                if what[1] == 0:
                    bars[me][place].expect(len(team))
                flying += [(to, place, what, s["row"], time) for to in range(blocks)]
            s["at"], s["since"], s["seen"] = "wait" if s["ok"] else "read", time, []
        elif s["at"] == "wait":
            s["at"] = "read"
        elif s["at"] == "read":                              # one sender's sums at a time
            sender = team[len(s["seen"])]
            s["seen"].append(sums[me][place].get(sender))
            if len(s["seen"]) == len(team):
                if s["ok"] and any(row != s["row"] for row in s["seen"]):
                    wrong.add("a gradient of other sums that is not NaN")
                s["row"] += 1
                s["at"] = "send" if s["row"] < rows else "leave"
                if s["at"] == "leave":
                    arrived.add(what)
        elif s["at"] == "leave":
            s["at"] = "gone"
    if any(bar.broken for pair in bars for bar in pair):
        wrong.add("a barrier is arrived at twice in a phase")
    assert all(s["at"] == "gone" for s in state.values())
    return wrong


def played(quiet, outlast, times=1500):
    wrong = set()
    for seed in range(times):
        rng = random.Random(seed)
        wrong |= play(rng, rng.choice([2, 2, 3]), rng.choice([1, 2]), rng.choice([1, 2, 3, 5]), quiet, outlast)
    return wrong


def test_what_a_warp_that_goes_on_sending_does():
    assert {"a gradient of other sums that is not NaN", "a barrier is arrived at twice in a phase"} <= played(False, True)


def test_what_a_block_that_leaves_at_once_does():
    assert played(True, False) == {"sums reach a block that has left"}


def test_no_order_is_wrong():
    assert played(True, True) == set()


@pytest.mark.parametrize("what", [r"if \(ok && threadIdx\.x == 0\) mbar_expect_tx\(", r"if \(ok && lane < a\.cluster\) \{[^}]*peer_send4\("])
def test_a_warp_whose_wait_ran_out_sends_nothing_more(what):
    assert len(re.findall(what, KERNEL)) == 1 and len(re.findall(r"mbar_expect_tx\(|peer_send4\(", KERNEL)) == 2


def test_what_is_on_its_way_is_waited_for():
    """Behind the cluster's last barrier, when all has been sent: of each of the two places both parities, of which one is that of the phase
    that runs.  It ends when all of the phase's sums are there, or the limit outlasts them."""
    last = KERNEL.index("if (a.cluster > 1) cluster_sync();                    // nobody leaves")
    assert re.search(r"cluster_sync\(\);[^;]*nobody leaves[^\n]*\n\s*if \(!ok\) rn_outlast\(there_s\);", KERNEL[last:])
    helper = TEXT[TEXT.index("void rn_outlast("):]
    helper = helper[:helper.index("\n}\n")]
    assert re.search(r"for \(int i = 0; i < 4; \+\+i\) mbar_wait\(smem_addr\(&bars\[i >> 1\]\), i & 1\);", helper)
    bar = Barrier()
    for _ in range(5):
        assert sum(bar.done(parity) for parity in (0, 1)) == 1
        bar.expect(1), bar.message()
