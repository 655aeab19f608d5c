"""Calls of the heads' norm and rotation at the edges of what their documentation allows."""
import pytest
import torch

import lib_b200
from lib_b200 import _capi
from tests import capture
from tests.test_gpu_rope import BF16, U32, turned, turns

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e-17, 1e-14, 1e-6, 1.0, 1e14, 1e17])
@pytest.mark.parametrize("dim", [128, 130, 256, 512])
@pytest.mark.parametrize("bf16", [False, True])
def test_gradient_of_heads_of_any_magnitude(ctx, scale, dim, bf16):
    """As far as the squares fit float32 (eps 0): dx = r (dz g - n mean(dz g n)) holds its bits."""
    tokens, hq, hk, rot = 21, 3, 2, dim // 2 // 2 * 2
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    x = torch.randn(tokens, (hq + hk) * dim, generator=g, device="cuda") * scale
    gq, gk = (torch.rand(dim, generator=g, device="cuda") + 0.5 for _ in range(2))
    pos = torch.randint(0, 10 ** 6, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    dq, dk = (torch.randn(tokens, h * dim, generator=g, device="cuda").to(BF16 if bf16 else torch.float32) for h in (hq, hk))
    dx, dgq, dgk = torch.empty_like(x), torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")
    rope = ctx.rope(dim, rot, 10000.0)
    torch.cuda.synchronize()
    rope.qk_norm_backward(x.data_ptr(), x.shape[1], tokens, hq, hk, gq.data_ptr(), gk.data_ptr(), 0.0, pos.data_ptr(), dq.data_ptr(), hq * dim,
                          dk.data_ptr(), hk * dim, dx.data_ptr(), x.shape[1], dgq.data_ptr(), dgk.data_ptr(), _capi.QK_BF16 if bf16 else 0)
    ctx.sync()
    ang = turns(pos, rot, 10000.0, None)
    at = 0
    for h, gain, dy, dgain in ((hq, gq, dq, dgq), (hk, gk, dk, dgk)):
        z, got = (t[:, at * dim:(at + h) * dim].reshape(tokens, h, dim).double() for t in (x, dx))
        at += h
        dz = turned(dy.double().reshape(tokens, h, dim), -ang, rot, False)
        r = 1 / z.square().mean(-1, keepdim=True).sqrt()
        n, dn = z * r, dz * gain.double()
        want = r * (dn - n * (dn * n).mean(-1, keepdim=True))
        # the turn, the factors and the sums of a head: as for ordinary heads
        top = dn.abs().amax(-1, keepdim=True) * (1 + n.abs() * n.abs().mean(-1, keepdim=True))
        assert ((got - want).abs() <= (32 + dim // 32) * U32 * r * top).all(), ((got - want).abs() / (U32 * r * top)).max()
        mag = (dz.abs().amax(-1, keepdim=True) * n.abs()).sum((0, 1))
        assert ((dgain.double() - (dz * n).sum((0, 1))).abs() <= (48 + tokens * (hq + hk) / 64) * U32 * mag).all()
    rope.close()


@pytest.mark.parametrize("dim,interleaved", [(128, False), (128, True), (130, False)])
def test_slow_pairs_at_small_positions(ctx, dim, interleaved):
    """The sine of a slow pair's small angle keeps all its bits: (1, 0) turned, and turned back."""
    theta, half = 500000.0, dim // 2
    pos = torch.tensor([1, 2, 3, -1, 7, 100, -5], dtype=torch.int32, device="cuda")
    t = pos.numel()
    one = torch.zeros(t, dim, device="cuda")
    one[:, 0:dim:2 if interleaved else 1][:, :half] = 1.0
    q, dx = torch.empty(t, dim, device="cuda"), torch.empty(t, dim, device="cuda")
    rope = ctx.rope(dim, dim, theta, interleaved=interleaved)
    torch.cuda.synchronize()
    common = (one.data_ptr(), dim, t, 1, 0, 0, 0, 0.0, pos.data_ptr())
    rope.qk_norm(*common, q.data_ptr(), dim, 0, 0, _capi.QK_NO_NORM)
    rope.qk_norm_backward(*common, one.data_ptr(), dim, 0, 0, dx.data_ptr(), dim, 0, 0, _capi.QK_NO_NORM)
    ctx.sync()
    ang = turns(pos, dim, theta, None)[:, 0]
    small = ang.abs() < 1.5     # (beyond, a rounding of the angle weighs more than the sine's own)
    assert small[:, half - 1].all()
    for got, sign in ((q, 1.0), (dx, -1.0)):
        sine = (got[:, 1::2] if interleaved else got[:, half:]).double()
        want = sign * ang.sin()
        # the angle's rounding to float32 (its weight in the sine is at most one here), a unit of sincospif, and 2^-64 turns
        # per position of the frequency, 2^-41 of the slowest pair's
        assert ((sine - want).abs() <= 4 * U32 * want.abs())[small].all(), ((sine - want).abs() / want.abs())[small].max()
    rope.close()


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


@pytest.mark.parametrize("backward", [False, True])
def test_rotation_alone_ignores_gains_and_eps(ctx, backward):
    tokens, dim = 9, 64
    rope = ctx.rope(dim, dim, 10000.0)
    x, d = torch.randn(tokens, 2 * dim, device="cuda"), torch.randn(tokens, 2 * dim, device="cuda")
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    gain = torch.full((dim + 1,), float("nan"), device="cuda")
    results, names = [], []
    for gq, gk, eps in ((0, 0, 0.0), (gain.data_ptr(), gain.data_ptr() + 4, 1e-5), (gain.data_ptr() + 1, 3, float("nan")), (0, 0, -1.0), (0, 0, float("inf"))):
        out = torch.zeros(tokens, 2 * dim, device="cuda")
        torch.cuda.synchronize()
        common = (x.data_ptr(), 2 * dim, tokens, 1, 1, gq, gk, eps, pos.data_ptr())
        if backward:
            call = lambda: rope.qk_norm_backward(*common, d.data_ptr(), 2 * dim, d.data_ptr() + 4 * dim, 2 * dim, out.data_ptr(), 2 * dim,  # noqa: E731
                                                 0, 0, _capi.QK_NO_NORM)
        else:
            call = lambda: rope.qk_norm(*common, out.data_ptr(), 2 * dim, out.data_ptr() + 4 * dim, 2 * dim, _capi.QK_NO_NORM)  # noqa: E731
        call()
        ctx.sync()
        results.append(out)
        names.append([l.name for l in capture.launches(ctx, call)])
    assert all(torch.equal(results[0], r) for r in results) and names.count(names[0]) == len(names)
    # a result on what is ignored is an ordinary result
    out = torch.zeros(tokens, 2 * dim, device="cuda")
    torch.cuda.synchronize()
    if not backward:
        rope.qk_norm(x.data_ptr(), 2 * dim, tokens, 1, 1, out.data_ptr(), 0, 0.0, pos.data_ptr(), out.data_ptr(), 2 * dim, out.data_ptr() + 4 * dim,
                     2 * dim, _capi.QK_NO_NORM)
        ctx.sync()
        assert torch.equal(out, results[0])
    rope.close()
