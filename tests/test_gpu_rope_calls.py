"""Calls of the heads' norm and rotation at the edges of what their documentation allows."""
import pytest
import torch

import lib_b200
from lib_b200 import _capi
from tests import capture
from tests.test_gpu_rope import U32, turned, turns

pytestmark = pytest.mark.gpu


def test_handle_is_not_made_under_capture(ctx):
    codes, made = [], []

    def call():
        try:
            made.append(ctx.rope(64, 64, 10000.0))
        except lib_b200.QmError as e:
            codes.append(e.code)

    capture.launches(ctx, call)     # (ends the capture: fails if it was invalidated)
    for r in made:
        r.close()
    assert codes == [900]           # CUDA_ERROR_STREAM_CAPTURE_UNSUPPORTED


def test_handles_are_ready_at_once(ctx):
    """A handle's frequencies are there for the first call on any stream, whatever the stream that made it is busy with."""
    pos = torch.tensor([5], dtype=torch.int32, device="cuda")
    x, q = torch.randn(1, 512, device="cuda"), torch.empty(1, 512, device="cuda")
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        for i in range(20):
            ctx.set_stream(first.cuda_stream)
            with torch.cuda.stream(first):
                torch.cuda._sleep(2_000_000)
            rope = ctx.rope(512, 512, 100.0 + i)
            ctx.set_stream(second.cuda_stream)
            rope.qk_norm(x.data_ptr(), 512, 1, 1, 0, 0, 0, 0.0, pos.data_ptr(), q.data_ptr(), 512, 0, 0, _capi.QK_NO_NORM)
            ctx.sync()
            want = turned(x.double()[:, None], turns(pos, 512, 100.0 + i, None), 512, False)[:, 0]
            assert ((q.double() - want).abs() <= 24 * U32 * float(x.abs().max())).all()
            rope.close()
    finally:
        ctx.set_stream(0)
