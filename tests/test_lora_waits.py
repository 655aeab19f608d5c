"""Waits of the adapters' tensor core kernels, by their source: what happens when one runs out cannot be run without making a GPU
fault, so the rules that keep it harmless are looked for in the text."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = open(os.path.join(ROOT, "lib_b200", "csrc", "qm_lora.cu")).read()


def body(name):
    """The text of a function from its name to the brace that closes it."""
    start = SOURCE.index(" %s(" % name)
    at, depth = SOURCE.index("{", start), 0
    for i in range(at, len(SOURCE)):
        depth += {"{": 1, "}": -1}.get(SOURCE[i], 0)
        if depth == 0:
            return SOURCE[start:i + 1]


def test_a_warp_takes_one_answer():
    """Only one thread on its own (pipe_multiply) waits without the vote of its warp."""
    waits = SOURCE.count("mbar_wait_bounded(")
    assert "__all_sync(0xffffffffu, qm::mbar_wait_bounded(" in body("warp_wait")
    assert waits == 1 + body("pipe_multiply").count("mbar_wait_bounded(")
    for call in re.finditer(r"pipe_multiply<", SOURCE):
        assert SOURCE[:call.start()].rstrip().endswith("if (lane == 0)")


def test_what_is_given_up_is_waited_for():
    """Every wait that runs out marks its CTA, and a marked CTA lets its copies land before their memory is used again."""
    assert SOURCE.count("QM_STATUS_TIMEOUT") == 1 and "*p.failed = 1" in body("give_up")
    assert "*p.failed" in body("pipe_done")
    for kernel in ("shrink", "outer"):
        text = body(kernel)
        last = max(text.index("pipe_multiply<"), text.index("pipe_read<"))
        assert text.index("pipe_done(pipe)") > last and not re.search(r"part \+ .*=", text[last:text.index("pipe_done(pipe)")])


def test_warps_are_together_for_tensor_memory():
    for step in ("tcgen05.alloc", "tcgen05.dealloc"):
        before = SOURCE[:SOURCE.index(step)].rsplit("if (threadIdx.x < 32)", 1)[0]
        assert "__syncwarp();" in "".join(before.rstrip().splitlines()[-1:])
