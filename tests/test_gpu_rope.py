"""Norm and rotation of query and key heads against the formulas in float64, forward and backward, and their refusals."""
import pytest
import torch

import lib_b200
from lib_b200 import _capi

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
BF16 = torch.bfloat16


def turns(pos, rot, theta, factors):
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    f = torch.ones_like(i) if factors is None else torch.tensor(factors, device="cuda", dtype=torch.float32).double()
    return pos.double()[:, None, None] * theta ** (-2.0 * i / max(rot, 1)) / f


def turned(z, ang, rot, interleaved):
    c, s = ang.cos(), ang.sin()
    p, q = (z[..., 0:rot:2], z[..., 1:rot:2]) if interleaved else (z[..., :rot // 2], z[..., rot // 2:rot])
    a, b = p * c - q * s, q * c + p * s
    first = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((first, z[..., rot:]), -1)


def forward(x, gain, ang, rot, interleaved, eps, norm):
    if norm:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        if gain is not None:
            x = x * gain
    return turned(x, ang, rot, interleaved)


CASES = [
    # tokens, q heads, k heads, dim, rot, interleaved, bf16, norm, gains, shift of the pointers in elements, extra pitch
    (1, 32, 8, 128, 128, False, False, True, True, 0, 0),
    (1, 1, 0, 2, 2, False, False, True, True, 0, 0),
    (3, 0, 1, 128, 64, True, False, True, False, 0, 4),
    (777, 12, 3, 96, 64, True, False, True, True, 0, 8),
    (777, 12, 3, 96, 64, False, True, True, True, 0, 8),
    (500, 5, 2, 80, 40, False, True, True, True, 0, 2),
    (130, 7, 7, 64, 64, True, True, False, False, 0, 0),
    (257, 3, 1, 256, 128, False, False, True, True, 0, 6),
    (64, 2, 1, 512, 512, False, True, True, True, 0, 0),
    (33, 3, 2, 130, 66, False, False, True, True, 0, 0),      # halves of no whole vectors
    (33, 3, 2, 6, 2, True, True, True, True, 0, 1),           # an odd row pitch
    (65, 4, 4, 128, 128, False, False, True, True, 1, 3),     # nothing aligned to more than an element
    (65, 4, 4, 128, 0, False, True, True, True, 1, 0),        # norm alone
    (2500, 9, 2, 128, 128, False, True, True, True, 0, 0),    # several heads per warp, an odd number of them
    (300, 3, 1, 510, 254, True, False, True, True, 0, 0),
    (3, 1500, 2, 64, 64, False, False, True, True, 0, 0),     # more heads than CTAs
    (5000, 2, 1, 192, 96, True, True, True, True, 0, 4),
]


def heads_of(tokens, hq, hk, dim, dtype, shift, extra, g, spare=0):
    """[tokens][(hq + hk + spare) * dim] values in a buffer with a shifted start and a wider pitch: (pointer, pitch, view)."""
    ld = (hq + hk + spare) * dim + extra
    whole = torch.full((tokens * ld + shift + 8,), -7.0, dtype=dtype, device="cuda")
    view = whole[shift:shift + tokens * ld].view(tokens, ld)[:, :(hq + hk + spare) * dim]
    view.copy_(torch.randn(view.shape, generator=g, device="cuda") * 0.7)
    return whole, ld, view


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("backward", [False, True])
def test_against_float64(ctx, case, backward):
    tokens, hq, hk, dim, rot, interleaved, bf16, norm, gains, shift, extra = case
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens * dim + rot)
    dtype = BF16 if bf16 else torch.float32
    eps, theta = 1e-5, 500000.0
    factors = [1.0 + (i % 5) for i in range(rot // 2)] if tokens % 2 else None
    rope = ctx.rope(dim, rot, theta, factors, interleaved)
    xw, ldx, x = heads_of(tokens, hq, hk, dim, torch.float32, shift, extra, g, spare=hk)
    gq, gk = (torch.rand(dim + 1, generator=g, device="cuda")[shift:shift + dim] + 0.5 for _ in range(2))
    pos = torch.randint(-1000, 2 ** 31 - 1, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = 0
    qw, ldq, q = heads_of(tokens, hq, 0, dim, dtype, shift, extra, g)
    kw, ldk, k = heads_of(tokens, 0, hk, dim, dtype, shift, extra + 4, g)
    flags = (0 if norm else _capi.QK_NO_NORM) | (_capi.QK_BF16 if bf16 else 0)
    p = lambda w, there=True: w.data_ptr() + shift * w.element_size() if there else 0  # noqa: E731
    gp = (gq.data_ptr(), gk.data_ptr()) if gains else (0, 0)
    ang = turns(pos, rot, theta, factors)
    parts = [(x[:, :hq * dim].reshape(tokens, hq, dim).double(), q, gq), (x[:, hq * dim:(hq + hk) * dim].reshape(tokens, hk, dim).double(), k, gk)]
    torch.cuda.synchronize()
    if not backward:
        rope.qk_norm(p(xw), ldx, tokens, hq, hk, *gp, eps, pos.data_ptr(), p(qw, hq), ldq, p(kw, hk), ldk, flags)
        ctx.sync()
        for z, got, gain in parts:
            want = forward(z, gain.double() if gains else None, ang, rot, interleaved, eps, norm).reshape(tokens, -1)
            mag = (z.abs() if not norm else z.abs() / (z.square().mean(-1, keepdim=True) + eps).sqrt() * (gain.double() if gains else 1.0))
            # both elements of a pair enter with a magnitude of at most the head's largest; float32: the turn (half a step of
            # half a turn, 2 pi 2^-25, and sincospif's two units) and a handful of roundings; the norm's sum is dim / 64 + 5 deep
            top = mag.amax(-1, keepdim=True).expand(mag.shape).reshape(tokens, -1)
            tol = (24 + dim // 64) * U32 * top
            if bf16:
                tol = tol + want.abs() * 2.0 ** -8
            assert ((got.double() - want).abs() <= tol + 1e-30).all()
        assert (kw.view(-1)[shift + tokens * ldk:] == -7.0).all() and (qw.view(-1)[shift + tokens * ldq:] == -7.0).all()
        assert extra == 0 or (qw[shift:shift + tokens * ldq].view(tokens, ldq)[:, hq * dim:] == -7.0).all()
    else:
        dxw, lddx, dx = heads_of(tokens, hq, hk, dim, torch.float32, shift, extra, g)
        dgq, dgk = (torch.full((dim,), -7.0, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        args = (p(xw), ldx, tokens, hq, hk, *gp, eps, pos.data_ptr(), p(qw, hq), ldq, p(kw, hk), ldk, p(dxw), lddx)
        grads = (dgq.data_ptr(), dgk.data_ptr()) if norm else (0, 0)
        rope.qk_norm_backward(*args, *grads, flags)
        ctx.sync()
        first = 0
        for (z, dy, gain), dgain, h in zip(parts, (dgq, dgk), (hq, hk)):
            got = dx[:, first * dim:(first + h) * dim].reshape(tokens, h, dim).double()
            first += h
            dz = turned(dy.double().reshape(tokens, h, dim), -ang, rot, interleaved)
            if not norm:
                want, top = dz, dz.abs().amax(-1, keepdim=True) if h else dz
                tol = 24 * U32 * top
            else:
                r = 1 / (z.square().mean(-1, keepdim=True) + eps).sqrt()
                dn = dz * gain.double() if gains else dz
                n = z * r
                want = r * (dn - n * (dn * n).mean(-1, keepdim=True))
                top = dn.abs().amax(-1, keepdim=True) * (1 + n.abs() * n.abs().mean(-1, keepdim=True)) if h else dz
                tol = (32 + dim // 32) * U32 * r * top
                wantg = (dz * n).sum((0, 1))
                mag = (dz.abs().amax(-1, keepdim=True) * n.abs()).sum((0, 1)) if h else wantg.abs()
                # a warp's chain of tokens and heads, eight warps, then float64
                chain = 40 + tokens * (hq + hk) / 64 + 8
                assert ((dgain.double() - wantg).abs() <= chain * U32 * mag + 1e-30).all()
            assert ((got - want).abs() <= tol + 1e-30).all()
        before = [t.clone() for t in (dxw, dgq, dgk)]
        torch.cuda.synchronize()
        rope.qk_norm_backward(*args, *grads, flags)      # the same bits again
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(before, (dxw, dgq, dgk)))
    rope.close()


def test_gradient_against_differences(ctx):
    tokens, hq, hk, dim, rot = 4, 2, 1, 16, 8
    rope = ctx.rope(dim, rot, 100.0)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randn(tokens, 3 * dim, generator=g, device="cuda")
    gq, gk = torch.rand(dim, generator=g, device="cuda") + 0.5, torch.rand(dim, generator=g, device="cuda") + 0.5
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda") * 5
    dq, dk = torch.randn(tokens, 2 * dim, generator=g, device="cuda"), torch.randn(tokens, dim, generator=g, device="cuda")
    q, k, dx = torch.empty_like(dq), torch.empty_like(dk), torch.empty_like(x)
    dgq, dgk = torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")
    torch.cuda.synchronize()
    rope.qk_norm_backward(x.data_ptr(), 48, tokens, hq, hk, gq.data_ptr(), gk.data_ptr(), 1e-5, pos.data_ptr(), dq.data_ptr(), 32, dk.data_ptr(), 16,
                          dx.data_ptr(), 48, dgq.data_ptr(), dgk.data_ptr())
    ctx.sync()

    def value():
        torch.cuda.synchronize()
        rope.qk_norm(x.data_ptr(), 48, tokens, hq, hk, gq.data_ptr(), gk.data_ptr(), 1e-5, pos.data_ptr(), q.data_ptr(), 32, k.data_ptr(), 16)
        ctx.sync()
        return float((q.double() * dq.double()).sum() + (k.double() * dk.double()).sum())

    # central differences: an error of the third derivative times h^2 / 6, and of 2^-24 * |values| / h
    h = 2.0 ** -7
    for t, grad in ((x, dx), (gq, dgq), (gk, dgk)):
        for at in (0, 5, t.numel() - 1):
            flat = t.view(-1)
            old = float(flat[at])
            flat[at] = old + h
            up = value()
            flat[at] = old - h
            down = value()
            flat[at] = old
            got, want = (up - down) / (2 * h), float(grad.view(-1)[at])
            assert abs(got - want) <= 2e-3 * (1 + abs(want))
    rope.close()


def test_in_place(ctx):
    tokens, hq, hk, dim = 300, 6, 2, 128
    rope = ctx.rope(dim, dim, 10000.0)
    x = torch.randn(tokens, (hq + 2 * hk) * dim, device="cuda")
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    ld = x.shape[1]
    q, k = torch.empty(tokens, hq * dim, device="cuda"), torch.empty(tokens, hk * dim, device="cuda")
    y = x.clone()
    torch.cuda.synchronize()
    rope.qk_norm(x.data_ptr(), ld, tokens, hq, hk, 0, 0, 1e-5, pos.data_ptr(), q.data_ptr(), hq * dim, k.data_ptr(), hk * dim)
    rope.qk_norm(y.data_ptr(), ld, tokens, hq, hk, 0, 0, 1e-5, pos.data_ptr(), y.data_ptr(), ld, y.data_ptr() + hq * dim * 4, ld)
    ctx.sync()
    assert torch.equal(y[:, :hq * dim], q) and torch.equal(y[:, hq * dim:(hq + hk) * dim], k) and torch.equal(y[:, (hq + hk) * dim:], x[:, (hq + hk) * dim:])
    # backward: dx on the gradients of the results, which lie side by side
    n = (hq + hk) * dim
    d = torch.randn(tokens, n, device="cuda")
    dx, both = torch.empty(tokens, n, device="cuda"), d.clone()
    torch.cuda.synchronize()
    common = (x.data_ptr(), ld, tokens, hq, hk, 0, 0, 1e-5, pos.data_ptr())
    rope.qk_norm_backward(*common, d.data_ptr(), n, d.data_ptr() + hq * dim * 4, n, dx.data_ptr(), n)
    rope.qk_norm_backward(*common, both.data_ptr(), n, both.data_ptr() + hq * dim * 4, n, both.data_ptr(), n)
    ctx.sync()
    assert torch.equal(both, dx)
    rope.close()


def test_unturned_elements_keep_to_themselves(ctx):
    """Rotation alone: an infinity behind the turning part does not reach its neighbour."""
    rope = ctx.rope(8, 4, 100.0)
    x = torch.arange(8, dtype=torch.float32, device="cuda")[None].clone()
    x[0, 5] = float("inf")
    pos = torch.tensor([3], dtype=torch.int32, device="cuda")
    q = torch.empty(1, 8, device="cuda")
    torch.cuda.synchronize()
    rope.qk_norm(x.data_ptr(), 8, 1, 1, 0, 0, 0, 0.0, pos.data_ptr(), q.data_ptr(), 8, 0, 0, _capi.QK_NO_NORM)
    ctx.sync()
    assert torch.equal(q[0, 4:], x[0, 4:]) and q[0, :4].isfinite().all()
    rope.close()


def test_no_tokens_and_zero_heads(ctx):
    rope = ctx.rope(16, 16, 10000.0)
    dgq, dgk = torch.full((16,), 5.0, device="cuda"), torch.full((16,), 5.0, device="cuda")
    torch.cuda.synchronize()
    rope.qk_norm(0, 16, 0, 1, 0, 0, 0, 1e-5, 0, 0, 16, 0, 0)
    rope.qk_norm_backward(0, 16, 0, 1, 0, 0, 0, 1e-5, 0, 0, 16, 0, 0, 0, 16, dgq.data_ptr(), dgk.data_ptr())
    ctx.sync()
    assert (dgq == 0).all() and (dgk == 0).all()
    # a head of zeros: zeros, and a finite gradient
    x, pos = torch.zeros(1, 16, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    q, dx = torch.ones(1, 16, device="cuda"), torch.empty(1, 16, device="cuda")
    torch.cuda.synchronize()
    rope.qk_norm_backward(x.data_ptr(), 16, 1, 1, 0, 0, 0, 1e-5, pos.data_ptr(), q.data_ptr(), 16, 0, 0, dx.data_ptr(), 16)
    rope.qk_norm(x.data_ptr(), 16, 1, 1, 0, 0, 0, 1e-5, pos.data_ptr(), q.data_ptr(), 16, 0, 0)
    ctx.sync()
    assert (q == 0).all() and dx.isfinite().all()
    rope.close()


def test_captured_and_replayed(ctx):
    tokens, hq, hk, dim = 50, 4, 2, 64
    rope = ctx.rope(dim, dim, 10000.0)
    n = (hq + hk) * dim
    x, dq, dk = torch.randn(tokens, n, device="cuda"), torch.randn(tokens, hq * dim, device="cuda"), torch.randn(tokens, hk * dim, device="cuda")
    pos = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    q, k, dx = torch.empty_like(dq), torch.empty_like(dk), torch.empty_like(x)
    dgq, dgk = torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")

    def step():
        rope.qk_norm(x.data_ptr(), n, tokens, hq, hk, 0, 0, 1e-5, pos.data_ptr(), q.data_ptr(), hq * dim, k.data_ptr(), hk * dim)
        rope.qk_norm_backward(x.data_ptr(), n, tokens, hq, hk, 0, 0, 1e-5, pos.data_ptr(), dq.data_ptr(), hq * dim, dk.data_ptr(), hk * dim,
                              dx.data_ptr(), n, dgq.data_ptr(), dgk.data_ptr())

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph, stream=stream):
            ctx.set_stream(stream.cuda_stream)
            step()
    finally:
        ctx.set_stream(0)
    for first in (3, 900000):
        pos.copy_(torch.arange(tokens, device="cuda") + first)
        x.copy_(torch.randn(tokens, n, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, k, dx, dgq, dgk)]
        torch.cuda.synchronize()
        step()
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, (q, k, dx, dgq, dgk)))
    del graph
    rope.close()


def test_refusals(ctx):
    def code(call, *args, **kw):
        with pytest.raises(lib_b200.QmError) as e:
            call(*args, **kw)
        return e.value.code

    SHAPE, ARG, LIMIT = -4, -5, -11
    for args, want in [((0, 0, 1e4), SHAPE), ((7, 2, 1e4), SHAPE), ((8, 3, 1e4), SHAPE), ((8, 10, 1e4), SHAPE), ((8, -2, 1e4), SHAPE), ((514, 2, 1e4), LIMIT),
                       ((8, 8, 0.0), ARG), ((8, 8, -1.0), ARG), ((8, 8, float("nan")), ARG), ((8, 8, float("inf")), ARG), ((8, 8, 1e4, [1, 1, 0, 1]), ARG),
                       ((8, 8, 1e4, [1, 1, float("nan"), 1]), ARG)]:
        assert code(ctx.rope, *args) == want, args
    with pytest.raises(ValueError):
        ctx.rope(8, 8, 1e4, [1.0, 1.0])
    rope = ctx.rope(8, 8, 1e4)
    p = torch.zeros(1 << 14, device="cuda").data_ptr()
    X, Q, K, P, D = p, p + 16384, p + 32768, p + 49152, p + 57344
    ok = dict(x_dev=X, ldx=32, tokens=4, q_heads=2, k_heads=1, q_gain_dev=0, k_gain_dev=0, eps=1e-5, pos_dev=P, q_dev=Q, ldq=16, k_dev=K, ldk=8, flags=0)
    bad = [(dict(tokens=-1), SHAPE), (dict(q_heads=-1), SHAPE), (dict(q_heads=0, k_heads=0), SHAPE), (dict(ldx=23), SHAPE), (dict(ldq=15), SHAPE), (dict(ldk=7), SHAPE),
           (dict(ldx=1 << 40), SHAPE), (dict(eps=-1.0), SHAPE), (dict(eps=float("nan")), SHAPE), (dict(x_dev=0), ARG), (dict(pos_dev=0), ARG), (dict(q_dev=0), ARG),
           (dict(k_dev=0), ARG), (dict(x_dev=X + 2), ARG), (dict(q_dev=Q + 2), ARG), (dict(flags=4), ARG), (dict(q_gain_dev=P + 1), ARG), (dict(pos_dev=P + 2), ARG)]
    for change, want in bad + [(dict(q_dev=X + 4), ARG), (dict(q_dev=X, ldq=36), ARG), (dict(k_dev=Q), ARG), (dict(k_dev=Q + 32), ARG), (dict(q_dev=P), ARG), (dict(k_gain_dev=K), ARG), (dict(q_dev=X, ldq=32, flags=2), ARG)]:
        assert code(rope.qk_norm, **{**ok, **change}) == want, change
    both = {**ok, "ldq": 24, "ldk": 24, "k_dev": Q + 64}
    rope.qk_norm(**both)          # q and k side by side in rows of their own
    ok = {**{k: v for k, v in ok.items() if k[:2] not in ("q_", "k_", "ld")}, "ldx": 32, "q_heads": 2, "k_heads": 1, "q_gain_dev": 0, "k_gain_dev": 0, "dq_dev": Q, "lddq": 16,
          "dk_dev": K, "lddk": 8, "dx_dev": D, "lddx": 24}
    for change, want in [(dict(dx_dev=0), ARG), (dict(lddx=23), SHAPE), (dict(dx_dev=D + 1), ARG), (dict(dq_dev=0), ARG), (dict(lddq=15), SHAPE), (dict(dx_dev=X + 32), ARG),
                         (dict(dx_dev=Q), ARG), (dict(dx_dev=K), ARG), (dict(flags=1, dq_gain_dev=D), ARG), (dict(dk_gain_dev=D + 2), ARG), (dict(tokens=-1), SHAPE), (dict(dk_gain_dev=D), ARG),
                         (dict(dq_gain_dev=P + 64, dk_gain_dev=P + 68), ARG)]:
        assert code(rope.qk_norm_backward, **{**ok, **change}) == want, change
    assert lib_b200.lib.qm_rope_destroy(ctx._h, None) == ARG
    ctx.sync()
    rope.close()
