"""The kernels' way out of a wait that ran out, by their source (no GPU may be made to get there). The warps of a CTA share a word that
says that one of them gives up. A warp that works together - votes, shuffles, .aligned instructions - has to leave its loop as one:
lanes that read the word at different times would wait for one another for good."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnabla-ext-cuda_b200", "csrc")
RECORD = re.compile(r"!\*abort_v\) \{ atomicExch\(a\.flag, 1\); \*abort_v = 1; \}")


def kernel_lines(name):
    with open(os.path.join(CSRC, name)) as f:
        return [line.split("//")[0].strip() for line in f]


@pytest.mark.parametrize("name", ["affine_bwd.cu", "pointwise.cu"])
def test_a_warp_gives_up_as_one(name):
    lines = kernel_lines(name)
    reads = [l for l in lines if "*abort_v" in l and not l.startswith("volatile int") and "volatile int *abort_v)" not in l]
    assert reads
    for l in reads:
        rest = RECORD.sub("", l)
        # one thread's own loop may look at the word by itself
        assert "*abort_v" not in rest or "pw_wait_lane(" in rest or rest == "if (*abort_v) ok = false;", l
    assert any("pw_giving_up(abort_v)" in l for l in lines)


def test_the_question_is_put_to_the_warp():
    with open(os.path.join(CSRC, "dwbnq_tc.cuh")) as f:
        body = re.search(r"bool pw_giving_up\(volatile int \*abort_v\) \{(.*?)\n?\}", f.read(), re.S).group(1)
    assert "__any_sync(0xffffffffu, *abort_v" in body
