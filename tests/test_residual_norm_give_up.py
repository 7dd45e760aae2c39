"""What the norm's backward pass does when a wait between the blocks of a row runs out, read from its source; and codes of a weight that is
no longer the layer's."""
import os
import re

import torch

from conftest import ROOT

TEXT = open(os.path.join(ROOT, "actnn_b200", "csrc", "residual_norm.cuh")).read()
KERNEL = TEXT[TEXT.index("rn_backward_kernel(const __grid_constant__"):TEXT.index("// The partial sums of the runs, added in order")]


def test_the_only_wait_is_bounded_and_its_warp_goes_on_together():
    assert len(re.findall(r"mbar_(try_)?wait\(|while \(", KERNEL)) == 1
    assert re.search(r"if \(ok\) \{\s*ok = __all_sync\(kFull, mbar_wait\(bar, phase >> place & 1\)\);\s*"
                     r"if \(!ok && lane == 0\) atomicAdd\(gave_up, 1u\);\s*\}\s*phase \^= 1u << place;", KERNEL)


def test_rows_without_their_sums_are_nan():
    assert KERNEL.index("mbar_wait(") < KERNEL.index("if (!ok) joined = __int_as_float(0x7fffffff);") < KERNEL.index("total[i] = __shfl_sync(kFull, joined")


def test_nobody_leaves_while_sums_are_on_their_way():
    """The last thing that all blocks of a cluster do together comes after the loop, and nothing is sent after it."""
    end = KERNEL.index("if (a.cluster > 1) cluster_sync();                    // nobody leaves")
    assert "peer_send4" not in KERNEL[end:] and KERNEL.index("peer_send4") < end and not re.search(r"\breturn;", KERNEL)


def test_codes_of_another_weight_are_not_served():
    import actnn_b200 as actnn
    for drop in (lambda m: m.load_state_dict(actnn.QFp8Linear(8, 4).state_dict()), lambda m: m.half(), lambda m: m.train(), lambda m: m.unfreeze()):
        layer = actnn.QFp8Linear(8, 4).eval()
        layer.frozen = (torch.zeros(1), torch.zeros(1))
        drop(layer)
        assert layer.frozen is None
