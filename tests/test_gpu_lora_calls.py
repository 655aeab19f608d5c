"""Calls of the adapters at the edges of what their documentation allows."""
import pytest
import torch

import lib_b200
from lib_b200 import _capi, synth
from tests import capture
from tests.test_gpu_lora import BF16, U32, adapters  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def same_specials(got, want):
    """The same infinities and NaN, place for place."""
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()] > 0, want[want.isinf()] > 0)


@pytest.mark.parametrize("tokens", [1, 2, 9, 16, 17, 100, 128, 129])
@pytest.mark.parametrize("rows", [40, 512, 4096, 28673])
@pytest.mark.parametrize("how", ["apart", "in place", "none"])
def test_empty_slot_without_ids(ctx, tokens, rows, how):
    """No ids, slot 0 never filled: every row is its base row, or zeros."""
    cols = 64
    h = ctx.lora(rows, cols, 2, 16, tokens)
    x = torch.full((tokens, cols), float("nan"), dtype=BF16, device="cuda")
    base = torch.randn(tokens, rows, device="cuda")
    y = torch.full((tokens + 1, rows + 3), -7.0, device="cuda")
    if how == "in place":
        y[:tokens, :rows] = base
    bp, lb = {"apart": (base.data_ptr(), rows), "in place": (y.data_ptr(), rows + 3), "none": (0, 0)}[how]
    torch.cuda.synchronize()
    h.matmul_bf16(x.data_ptr(), tokens, cols, 0, bp, lb, y.data_ptr(), rows + 3)
    ctx.sync()
    assert torch.equal(y[:tokens, :rows], base if how != "none" else torch.zeros_like(base))
    assert (y[:tokens, rows:] == -7.0).all() and (y[tokens] == -7.0).all()
    h.close()


# tokens of slot 1 (rank 5) among bare ones: none, one, a whole item, one item and a bit
@pytest.mark.parametrize("tokens,held", [(1, 0), (33, 1), (128, 0), (128, 16), (128, 17), (128, 111), (100, 99)])
@pytest.mark.parametrize("how", ["apart", "in place", "none"])
def test_mostly_bare_tokens(ctx, adapters, tokens, held, how):  # noqa: F811
    rows, cols = 6150, 96
    ad = adapters(rows, cols, 3, 16, tokens, {1: 5}, seed=tokens + held)
    g = torch.Generator(device="cuda")
    g.manual_seed(held)
    ids = torch.tensor([-1, 0, 2, 3, 10 ** 9], dtype=torch.int32, device="cuda")[torch.randint(0, 5, (tokens,), generator=g, device="cuda")]
    ids[torch.randperm(tokens, generator=g, device="cuda")[:held]] = 1
    x = torch.randn(tokens, cols, generator=g, device="cuda").to(BF16)
    x[ids != 1] = float("nan")
    base = torch.randn(tokens, rows, generator=g, device="cuda")
    start = base if how != "none" else torch.zeros_like(base)
    y = base.clone() if how == "in place" else torch.full((tokens, rows), -7.0, device="cuda")
    bp = {"apart": base.data_ptr(), "in place": y.data_ptr(), "none": 0}[how]
    torch.cuda.synchronize()
    ad.h.matmul_bf16(x.data_ptr(), tokens, cols, ids.data_ptr(), bp, rows, y.data_ptr(), rows)
    ctx.sync()
    want, mag = ad.forward(x.double(), ids, start)
    # 4 per stage of 64 columns, two stages, 8 CTAs; 3 parts of 16 ranks, the base, the scale: truncated, a unit each
    assert ((y.double() - want).abs() <= 2 * (4 + 2 + 8 + 3 + 4) * U32 * mag + 1e-30).all()
    assert torch.equal(y[ids != 1], start[ids != 1])


def test_handle_made_on_a_busy_stream(ctx):
    """A handle made while its context's stream has work queued is ready for any other stream."""
    rows, cols, r = 96, 64, 8
    a, b = torch.randn(r, cols, device="cuda").to(BF16), torch.randn(rows, r, device="cuda").to(BF16)
    x, y = torch.randn(2, cols, device="cuda"), torch.zeros(2, rows, device="cuda")
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        ctx.set_stream(first.cuda_stream)
        with torch.cuda.stream(first):
            torch.cuda._sleep(200_000_000)      # about a tenth of a second
        h = ctx.lora(rows, cols, 1, r, 2)
        ctx.set_stream(second.cuda_stream)
        h.set(0, r, 1.0, a.data_ptr(), b.data_ptr())
        ctx.sync()
        first.synchronize()
        h.matvec(x.data_ptr(), 2, cols, 0, 0, 0, y.data_ptr(), rows)
        ctx.sync()
    finally:
        ctx.set_stream(0)
    want, mag = x.double() @ a.double().t() @ b.double().t(), x.double().abs() @ a.double().abs().t() @ b.double().abs().t()
    assert ((y.double() - want).abs() <= 60 * U32 * mag).all()
    h.close()


def test_handle_is_not_made_under_capture(ctx):
    """The slots' first clear would run again with the graph: refused, and the capture goes on."""
    codes, made = [], []

    def call():
        try:
            made.append(ctx.lora(96, 64, 1, 8, 2))
        except lib_b200.QmError as e:
            codes.append(e.code)

    capture.launches(ctx, call)     # (ends the capture: fails if it was invalidated)
    for h in made:
        h.close()
    assert codes == [900]           # CUDA_ERROR_STREAM_CAPTURE_UNSUPPORTED


@pytest.mark.parametrize("tokens", [3, 100, 300])
def test_pitch_of_an_absent_base(ctx, adapters, tokens):  # noqa: F811
    """Without a base its pitch means nothing: no other kernel, no refusal."""
    rows, cols = 256, 128
    ad = adapters(rows, cols, 1, 16, 300, {0: 16})
    x, y = torch.randn(tokens, cols, device="cuda").to(BF16), torch.zeros(tokens, rows, device="cuda")
    torch.cuda.synchronize()
    call = lambda ldb: ad.h.matmul_bf16(x.data_ptr(), tokens, cols, 0, 0, ldb, y.data_ptr(), rows)  # noqa: E731
    names = [[l.name for l in capture.launches(ctx, lambda: call(ldb))] for ldb in (0, 1, rows + 1, 1 << 40, -1)]
    assert names.count(names[0]) == len(names)
    if tokens <= 8:
        xf = x.float()
        torch.cuda.synchronize()
        for ldb in (0, 1, 1 << 40):
            ad.h.matvec(xf.data_ptr(), tokens, cols, 0, 0, ldb, y.data_ptr(), rows)
    # the backward pass without dx: base and its pitch are not used
    dy = torch.randn(tokens, rows, device="cuda").to(BF16)
    da, db = torch.zeros(16, cols, device="cuda"), torch.zeros(rows, 16, device="cuda")
    torch.cuda.synchronize()
    ad.h.backward(x.data_ptr(), cols, dy.data_ptr(), rows, tokens, 0, da.data_ptr(), 1 << 40, 0, 1 << 62, da.data_ptr(), db.data_ptr())
    ad.h.backward(x.data_ptr(), cols, dy.data_ptr(), rows, tokens, 0, 0, 1 << 40, y.data_ptr(), cols, da.data_ptr(), db.data_ptr())
    ctx.sync()


@pytest.mark.parametrize("m", [128, 129, 391])
def test_batched_product_with_adapters(ctx, adapters, m):  # noqa: F811
    """qm_matmul_bf16_lora in the forms for few tokens and for prompts: the product's own result, the adapters on it."""
    rows, cols = 520, 1024
    w = ctx.store_upload(_capi.Q4_K, rows, cols, synth.weights(_capi.Q4_K, rows, cols, seed=3))
    ad = adapters(rows, cols, 3, 24, m, {0: 24, 2: 7})
    x = torch.tensor(synth.activations(m, cols, seed=4), device="cuda").to(BF16)
    ids = torch.tensor([0, -1, 2, 1], dtype=torch.int32, device="cuda")[torch.arange(m, device="cuda") * 4 // m]
    c, c2 = torch.full((m + 1, rows + 4), -7.0, device="cuda"), torch.empty(m, rows, device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_bf16(w, x.data_ptr(), m, cols, c2.data_ptr(), rows)
    ctx.matmul_bf16_lora(w, ad.h, x.data_ptr(), m, cols, ids.data_ptr(), c.data_ptr(), rows + 4)
    ctx.sync()
    want, mag = ad.forward(x.double(), ids, c2)
    # as in the batches beside a base
    assert ((c[:m, :rows].double() - want).abs() <= 2 * (4 + cols // 64 + 8 + 3 * 2 + 4) * U32 * mag).all()
    bare = (ids != 0) & (ids != 2)
    assert torch.equal(c[:m, :rows][bare], c2[bare]) and (c[:m, rows:] == -7.0).all() and (c[m] == -7.0).all()
    w.free()


@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("rank", [1, 5, 24, 40, 70])
@pytest.mark.parametrize("where", ["x", "dy", "A", "B", "x and dy"])
def test_infinities_are_those_of_the_formulas(ctx, adapters, tokens, rank, where):  # noqa: F811
    """An infinite element gives the infinities (and the NaN of unlike ones) that the formulas give, in every form."""
    rows, cols = 136, 96
    ad = adapters(rows, cols, 2, rank, tokens, {0: rank, 1: max(1, rank // 2)}, seed=rank)
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens + rank)
    x, dy = torch.randn(tokens, cols, generator=g, device="cuda").to(BF16), torch.randn(tokens, rows, generator=g, device="cuda").to(BF16)
    a, b = ad.a[0].to(BF16), ad.b[0].to(BF16)
    if "x" in where:
        x[2, 5] = float("inf")
    if "dy" in where:
        dy[4, 7] = -float("inf")
    if where == "A":
        a[rank // 2, 9] = float("inf")
    if where == "B":
        b[11, rank // 2] = -float("inf")
    for t in (x, dy, a, b):     # (nothing is zero: an infinity times zero is NaN by the formulas too)
        t[t == 0] = 1.0
    ad.put(0, rank, ad.s[0], a, b, _capi.TYPE_BF16)
    ids = torch.arange(tokens, device="cuda", dtype=torch.int32) // 8 % 3 - 1
    ids[:8] = 0
    base, dbase = torch.randn(tokens, rows, generator=g, device="cuda"), torch.randn(tokens, cols, generator=g, device="cuda")
    y, dx = torch.empty(tokens, rows, device="cuda"), torch.empty(tokens, cols, device="cuda")
    da, db = torch.empty(2, rank, cols, device="cuda"), torch.empty(2, rows, rank, device="cuda")
    torch.cuda.synchronize()
    ad.h.matmul_bf16(x.data_ptr(), tokens, cols, ids.data_ptr(), base.data_ptr(), rows, y.data_ptr(), rows)
    ad.h.backward(x.data_ptr(), cols, dy.data_ptr(), rows, tokens, ids.data_ptr(), dbase.data_ptr(), cols, dx.data_ptr(), cols, da.data_ptr(), db.data_ptr())
    ctx.sync()
    # (sums written out: a matrix product of the library may skip or rearrange what is special)
    want, wantx = base.double().clone(), dbase.double().clone()
    for e, at in ad.of(ids):
        A, B, s, xe, de = ad.a[e], ad.b[e], ad.s[e], x[at].double(), dy[at].double()
        u, v = s * (xe[:, None] * A[None]).sum(2), s * (de[:, :, None] * B[None]).sum(1)
        want[at] += (u[:, None] * B[None]).sum(2)
        wantx[at] += (v[:, :, None] * A[None]).sum(1)
        r = A.shape[0]
        assert same_specials(da[e, :r], (v[:, :, None] * xe[:, None]).sum(0))
        assert same_specials(db[e, :, :r], (de[:, :, None] * u[:, None]).sum(0))
    assert same_specials(y, want) and same_specials(dx, wantx)
    xf, yr = x[:8].float(), torch.empty(8, rows, device="cuda")
    torch.cuda.synchronize()
    ad.h.matvec(xf.data_ptr(), 8, cols, ids.data_ptr(), base.data_ptr(), rows, yr.data_ptr(), rows)
    ctx.sync()
    assert same_specials(yr, want[:8])


@pytest.mark.parametrize("tokens", [40, 300])
def test_values_at_the_ends_of_float32(ctx, adapters, tokens):  # noqa: F811
    """Narrow products next to the largest float32, and far below the smallest bf16 part, keep their bits."""
    rows, cols = 40, 32
    ad = adapters(rows, cols, 1, 1, tokens, {0: 1})
    a, b = torch.zeros(1, cols, device="cuda").to(BF16), torch.full((rows, 1), 2.0 ** -100, device="cuda").to(BF16)
    a[0, :2] = torch.tensor([1.0, 2.0 ** -8], device="cuda").to(BF16)
    ad.put(0, 1, 1.0, a, b, _capi.TYPE_BF16)
    x = torch.zeros(tokens, cols, device="cuda").to(BF16)
    x[:, 0] = x[:, 1] = 3.3895313892515355e38       # the largest bf16; the sum rounds to nothing finite there
    x[1::2, :2] = 2.0 ** -100 * 1.0078125
    y = torch.empty(tokens, rows, device="cuda")
    torch.cuda.synchronize()
    b2 = torch.full((rows, 1), 2.0 ** 90, device="cuda").to(BF16)
    for bb in (b, b2):
        ad.put(0, 1, 1.0, a, bb, _capi.TYPE_BF16)
        torch.cuda.synchronize()
        ad.h.matmul_bf16(x.data_ptr(), tokens, cols, 0, 0, 0, y.data_ptr(), rows)
        ctx.sync()
        want, _ = ad.forward(x.double(), torch.zeros(tokens, dtype=torch.int32, device="cuda"), torch.zeros(tokens, rows, device="cuda"))
        at = slice(0, None, 2) if bb is b else slice(1, None, 2)     # (the others leave float32's range)
        # two products, their sum, three parts: a unit each
        assert ((y[at].double() - want[at]).abs() <= 2 * 6 * U32 * want[at].abs()).all()


def test_small_calls_of_one_handle_overlap(ctx, adapters):  # noqa: F811
    """Rows and few tokens use no workspace: calls on one handle may run at once, captured ones among them."""
    rows, cols, tokens = 4100, 2048, 100
    ad = adapters(rows, cols, 3, 32, tokens, {0: 32, 2: 9})
    ids = torch.tensor([0, -1, 2], dtype=torch.int32, device="cuda")[torch.arange(tokens, device="cuda") % 3]
    x = [torch.randn(tokens, cols, device="cuda").to(BF16) for _ in range(3)]
    xf = [t[:8].float() for t in x]
    y = [torch.empty(tokens, rows, device="cuda") for _ in x]
    yr = [torch.empty(8, rows, device="cuda") for _ in x]
    streams, graph = [torch.cuda.Stream() for _ in x], torch.cuda.CUDAGraph()

    def both(i):
        ad.h.matmul_bf16(x[i].data_ptr(), tokens, cols, ids.data_ptr(), 0, 0, y[i].data_ptr(), rows)
        ad.h.matvec(xf[i].data_ptr(), 8, cols, ids.data_ptr(), 0, 0, yr[i].data_ptr(), rows)

    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph, stream=streams[2]):
            ctx.set_stream(streams[2].cuda_stream)
            both(2)
        for _ in range(10):
            with torch.cuda.stream(streams[2]):
                graph.replay()
            for i in range(2):
                ctx.set_stream(streams[i].cuda_stream)
                both(i)
        torch.cuda.synchronize()
    finally:
        ctx.set_stream(0)
    for i in range(3):
        for got, inp in ((y[i], x[i]), (yr[i], xf[i])):
            n = inp.shape[0]
            want, mag = ad.forward(inp.double(), ids[:n], torch.zeros(n, rows, device="cuda"))
            assert ((got.double() - want).abs() <= 2 * (4 + cols // 64 + 8 + 3 * 2 + 4) * U32 * mag + 1e-30).all()
    del graph
