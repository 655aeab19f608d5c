"""Low-rank adapters beside a stored projection against the same in float64: single rows, bf16 batches, gradients, refusals."""
import numpy as np
import pytest
import torch

import lib_b200
from lib_b200 import _capi, synth
from oracle import oracle
from tests import capture

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24   # half a step of float32
BF16 = torch.bfloat16


class Adapters:
    """A handle and what its slots hold, in float64."""

    def __init__(self, ctx, rows, cols, slots, max_rank, max_tokens, ranks, seed=0, type=_capi.TYPE_BF16):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.ctx, self.rows, self.cols, self.ranks = ctx, rows, cols, ranks
        self.h = ctx.lora(rows, cols, slots, max_rank, max_tokens)
        self.a, self.b, self.s = {}, {}, {}
        kept = {_capi.TYPE_F32: torch.float32, _capi.TYPE_F16: torch.float16, _capi.TYPE_BF16: BF16}[type]
        for slot, r in ranks.items():
            a = (torch.randn(r, cols, generator=g, device="cuda") * cols ** -0.5).to(kept)
            b = (torch.randn(rows, r, generator=g, device="cuda") * 0.3).to(kept)
            self.put(slot, r, 0.5 + 0.25 * slot, a, b, type)

    def put(self, slot, r, scale, a, b, type):
        torch.cuda.synchronize()
        self.h.set(slot, r, scale, a.data_ptr(), b.data_ptr(), type)
        self.ctx.sync()
        self.a[slot], self.b[slot], self.s[slot] = a.to(BF16).double(), b.to(BF16).double(), float(np.float32(scale))

    def of(self, ids):
        """(slot, its tokens) of every slot that holds an adapter."""
        for slot in self.a:
            at = torch.nonzero(ids == slot).flatten()
            if at.numel():
                yield slot, at

    def forward(self, x, ids, base):
        """y in float64, and the same sum with every term's magnitude."""
        y, mag = base.double().clone(), base.double().abs()
        for e, at in self.of(ids):
            y[at] += self.s[e] * (x[at] @ self.a[e].t()) @ self.b[e].t()
            mag[at] += abs(self.s[e]) * (x[at].abs() @ self.a[e].abs().t()) @ self.b[e].abs().t()
        return y, mag

    def close(self):
        self.h.close()


@pytest.fixture
def adapters(ctx):
    made = []

    def make(*args, **kw):
        made.append(Adapters(ctx, *args, **kw))
        return made[-1]

    yield make
    for m in made:
        m.close()


def padded(rows, width, ld, fill=float("nan"), dtype=torch.float32):
    """A [rows][ld] buffer full of `fill`, and its [rows][width] part."""
    whole = torch.full((rows, ld), fill, dtype=dtype, device="cuda")
    return whole, whole[:, :width]


def transformed(x, x2, xop):
    x = x.double()
    if xop == _capi.XOP_ADD_RMSNORM:
        x = x + x2.double()
    if xop in (_capi.XOP_RMSNORM, _capi.XOP_ADD_RMSNORM):
        x = x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt()
    if xop == _capi.XOP_SWIGLU:
        x = x / (1 + torch.exp(-x)) * x2.double()
    return x


ROWS = [
    # rows, cols, m, ranks of the slots, ids, xop, base
    (256, 256, 1, {0: 16}, [0], 0, "apart"),
    (4096, 4096, 1, {0: 16}, None, 1, "in place"),
    (129, 32, 3, {0: 1, 2: 7}, [2, 0, 2], 0, "apart"),          # K of one block, most CTAs of the cluster without columns
    (1, 64, 2, {1: 3}, [1, -1], 0, "none"),
    (10007, 2304, 5, {0: 24, 1: 15, 2: 24}, [1, 0, -1, 1, 2], 0, "apart"),
    (6144, 4096, 8, {i: 64 - 9 * (i % 2) for i in range(8)}, [7, 6, 5, 4, 3, 2, 1, 0], 1, "in place"),
    (4096, 14336, 8, {0: 128}, [0] * 8, 3, "none"),
    (4100, 14336, 6, {0: 128, 3: 100}, [3, 0, 3, 0, 99, 1], 2, "apart"),   # 99 names no slot, 1 an empty one
    (28672, 32768, 8, {0: 33, 1: 2}, [0, 1, 0, 1, 0, 1, 0, -2147483648], 0, "in place"),
    (40000, 96, 2, {0: 8}, [0, 0], 1, "apart"),                 # several chunks of columns per CTA
]


@pytest.mark.parametrize("rows,cols,m,ranks,ids,xop,how", ROWS)
def test_rows(ctx, adapters, rows, cols, m, ranks, ids, xop, how):
    ad = adapters(rows, cols, max(ranks) + 1 + (ids is not None), max(ranks.values()), 1, ranks, seed=rows + m)
    g = torch.Generator(device="cuda")
    g.manual_seed(m * 7 + cols)
    ldx, ldy, ldb = cols + 12, rows + 5, rows + 3
    xw, x = padded(m, cols, ldx)
    x.copy_(torch.randn(m, cols, generator=g, device="cuda"))
    x2w, x2 = padded(m, cols, ldx)
    x2.copy_(torch.randn(m, cols, generator=g, device="cuda"))
    base = torch.randn(m, rows, generator=g, device="cuda")
    yw, y = padded(m + 1, rows, ldy, -7.0)
    bw, b = padded(m, rows, ldb)
    b.copy_(base)
    idt = torch.tensor(ids if ids is not None else [0] * m, dtype=torch.int32, device="cuda")
    if how == "in place":
        y[:m].copy_(base)
        bp, lb = yw.data_ptr(), ldy
    else:
        bp, lb = (bw.data_ptr(), ldb) if how == "apart" else (0, 0)
    torch.cuda.synchronize()
    ad.h.matvec(xw.data_ptr(), m, ldx, idt.data_ptr() if ids is not None else 0, bp, lb, yw.data_ptr(), ldy, xop, x2w.data_ptr() if xop >= 2 else 0)
    ctx.sync()
    want, mag = ad.forward(transformed(x, x2, xop), idt, base if how != "none" else torch.zeros_like(base))
    # longest chain of additions behind one value: a lane's share of K (eight per step), shuffles, cluster; ranks of a
    # thread; the four groups, the base; the factors, and the transform's own roundings (square root, expf: a few units)
    chain = cols // 256 + 8 + 5 + 8 + max(ranks.values()) // 4 + 3 + 1 + 16
    assert ((y[:m].double() - want).abs() <= chain * U32 * mag + 1e-30).all(), ((y[:m].double() - want).abs() / (U32 * mag + 1e-30)).max()
    # rows without an adapter are the base's bits; nothing beside or behind the rows is touched
    for j, e in enumerate(idt.tolist()):
        if e not in ranks:
            assert torch.equal(y[j], base[j] if how != "none" else torch.zeros_like(base[j]))
    assert (yw[:m, rows:] == -7.0).all() and (yw[m:] == -7.0).all()


BATCHES = [
    # rows, cols, tokens, ranks, base, how the ids lie
    (64, 64, 1, {0: 16}, "apart", "one"),
    (128, 32, 63, {0: 1}, "none", "all"),
    (129, 96, 64, {0: 16, 1: 5}, "apart", "mixed"),
    (1, 64, 65, {0: 3, 2: 16}, "in place", "mixed"),
    (4096, 4096, 130, {0: 32, 1: 17, 5: 20}, "apart", "runs"),
    (1031, 416, 777, {i: 1 + 4 * i for i in range(16)}, "in place", "mixed"),
    (512, 14336, 300, {0: 64, 1: 40}, "apart", "runs"),
    (770, 2080, 200, {0: 128, 3: 65}, "apart", "mixed"),
    (256, 1024, 4099, {0: 8, 1: 16}, "none", "runs"),
    (300, 128, 256, {i: 4 for i in range(256)}, "apart", "each"),
    (130, 32, 129, {0: 2}, "apart", "all"),                     # fewer columns than a cluster has CTAs
    (1, 64, 200, {1: 33, 0: 1}, "in place", "mixed"),
    (64, 64, 200001, {0: 4, 3: 2}, "apart", "runs"),            # many tiles of one adapter
    # up to 128 tokens: one launch
    (4096, 4096, 100, {0: 128, 1: 65, 2: 33}, "apart", "mixed"),
    (1031, 2080, 128, {0: 64, 1: 40, 7: 9}, "in place", "runs"),
    (6144, 14336, 100, {0: 32}, "none", "all"),
    (28672, 96, 17, {0: 16, 1: 3}, "apart", "mixed"),
    (512, 1024, 128, {i: 1 + i % 16 for i in range(128)}, "apart", "each"),
]


def make_ids(how, tokens, ranks, slots):
    r = np.random.default_rng(tokens)
    names = list(ranks)
    if how in ("one", "all"):
        ids = np.full(tokens, names[0])
    elif how == "each":
        ids = r.permutation(tokens)
    elif how == "mixed":
        ids = r.choice(names + [-1, slots, 10 ** 9, slots - 1], tokens)
    else:
        cuts = np.sort(r.choice(tokens, 4, replace=False))
        ids = np.array(names + [-1])[np.searchsorted(cuts, np.arange(tokens), "right") % (len(names) + 1)]
    return torch.tensor(ids.astype(np.int32), device="cuda")


@pytest.mark.parametrize("rows,cols,tokens,ranks,base_how,ids_how", BATCHES)
def test_batch(ctx, adapters, rows, cols, tokens, ranks, base_how, ids_how):
    slots = min(256, max(ranks) + 2)
    ad = adapters(rows, cols, slots, max(ranks.values()), tokens + 3, ranks, seed=tokens)
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens + cols)
    ldx, ldy, ldb = cols + 8, rows + 3, rows + 6
    xw, x = padded(tokens, cols, ldx, dtype=BF16)
    x.copy_(torch.randn(tokens, cols, generator=g, device="cuda"))
    ids = make_ids(ids_how, tokens, ranks, slots)
    base = torch.randn(tokens, rows, generator=g, device="cuda")
    yw, y = padded(tokens + 1, rows, ldy, -7.0)
    bw, b = padded(tokens, rows, ldb)
    b.copy_(base)
    bare = ~torch.isin(ids, torch.tensor(list(ranks), device="cuda", dtype=torch.int32))
    x[bare] = float("nan")      # what no adapter reads may hold anything
    if base_how == "in place":
        y[:tokens].copy_(base)
        bp, lb = yw.data_ptr(), ldy
    else:
        bp, lb = (bw.data_ptr(), ldb) if base_how == "apart" else (0, 0)
    torch.cuda.synchronize()
    ad.h.matmul_bf16(xw.data_ptr(), tokens, ldx, 0 if ids_how == "all" else ids.data_ptr(), bp, lb, yw.data_ptr(), ldy)
    ctx.sync()
    start = base if base_how != "none" else torch.zeros_like(base)
    want, mag = ad.forward(x.double(), ids, start)
    # tensor core sums truncate (a unit, not half of one): 4 per stage, the stages and 8 CTAs of a cluster; then 3 per 16
    # ranks, the parts, the base and the scale
    chain = 2 * (4 + cols // 64 + 8 + 3 * ((max(ranks.values()) + 15) // 16) + 4)
    assert ((y[:tokens].double() - want).abs() <= chain * U32 * mag + 1e-30).all(), ((y[:tokens].double() - want).abs() / (U32 * mag + 1e-30)).max()
    assert torch.equal(y[:tokens][bare], start[bare])
    assert (yw[:tokens, rows:] == -7.0).all() and (yw[tokens:] == -7.0).all()


def test_infinities_stay_with_their_token(ctx, adapters):
    ad = adapters(96, 64, 2, 20, 8, {0: 20, 1: 3})
    x = torch.randn(8, 64, device="cuda").to(BF16)
    x[2, 5] = float("inf")
    x[5, 7] = float("nan")
    ids = torch.tensor([0, 1] * 4, dtype=torch.int32, device="cuda")
    base, y = torch.randn(8, 96, device="cuda"), torch.empty(8, 96, device="cuda")
    torch.cuda.synchronize()
    ad.h.matmul_bf16(x.data_ptr(), 8, 64, ids.data_ptr(), base.data_ptr(), 96, y.data_ptr(), 96)
    ctx.sync()
    want, _ = ad.forward(x.double(), ids, base)
    clean = torch.tensor([0, 1, 3, 4, 6, 7], device="cuda")
    assert torch.allclose(y[clean].double(), want[clean], rtol=1e-5, atol=1e-5)
    assert y[5].isnan().all() and not y[2].isfinite().any()


GRADS = [
    # rows, cols, tokens, ranks, ids
    (64, 32, 1, {0: 2}, "one"),
    (72, 96, 33, {0: 16}, "all"),
    (129, 160, 200, {0: 7, 1: 32, 2: 1}, "mixed"),
    (1000, 416, 777, {0: 64, 3: 33}, "mixed"),
    (4096, 2048, 1025, {0: 16}, "all"),
    (520, 1024, 515, {0: 128, 1: 90, 2: 3}, "runs"),
    (264, 64, 64, {i: 4 for i in range(64)}, "each"),
    (72, 96, 70001, {0: 9, 1: 16}, "runs"),
]


@pytest.mark.parametrize("rows,cols,tokens,ranks,ids_how", GRADS)
@pytest.mark.parametrize("base_how", ["apart", "in place", "none"])
def test_backward(ctx, adapters, rows, cols, tokens, ranks, ids_how, base_how):
    slots, R = max(ranks) + 2, max(ranks.values())
    ad = adapters(rows, cols, slots, R, tokens, ranks, seed=tokens + 1)
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    ldx, lddy, lddx = cols + 16, (rows + 15) // 8 * 8, cols + 1
    xw, x = padded(tokens, cols, ldx, dtype=BF16)
    x.copy_(torch.randn(tokens, cols, generator=g, device="cuda"))
    dyw, dy = padded(tokens, rows, lddy, dtype=BF16)
    dy.copy_(torch.randn(tokens, rows, generator=g, device="cuda"))
    ids = make_ids(ids_how, tokens, ranks, slots)
    bare = ~torch.isin(ids, torch.tensor(list(ranks), device="cuda", dtype=torch.int32))
    x[bare] = float("nan")
    dy[bare] = float("nan")
    base = torch.randn(tokens, cols, generator=g, device="cuda")
    dxw, dx = padded(tokens + 1, cols, lddx, -7.0)
    da, db = torch.full((slots, R, cols), -7.0, device="cuda"), torch.full((slots, rows, R), -7.0, device="cuda")
    if base_how == "in place":
        dx[:tokens].copy_(base)
    args = {"apart": (base.data_ptr(), cols), "in place": (dxw.data_ptr(), lddx), "none": (0, 0)}[base_how]
    torch.cuda.synchronize()
    ad.h.backward(xw.data_ptr(), ldx, dyw.data_ptr(), lddy, tokens, 0 if ids_how == "all" else ids.data_ptr(), *args, dxw.data_ptr(), lddx,
                  da.data_ptr(), db.data_ptr())
    ctx.sync()
    start = base if base_how != "none" else torch.zeros_like(base)
    want, mag = start.double().clone(), start.double().abs()
    wa, wb = torch.zeros(da.shape, dtype=torch.float64, device="cuda"), torch.zeros(db.shape, dtype=torch.float64, device="cuda")
    ma, mb = wa.clone(), wb.clone()
    for e, at in ad.of(ids):
        a, b, s, xe, de, r = ad.a[e], ad.b[e], ad.s[e], x[at].double(), dy[at].double(), ranks[e]
        for sign, o, ga, gb in ((lambda t: t, want, wa, wb), (torch.abs, mag, ma, mb)):
            v, u = s * sign(de) @ sign(b), s * sign(xe) @ sign(a).t()
            o[at] += v @ sign(a)
            ga[e, :r] = v.t() @ sign(xe)
            gb[e, :, :r] = sign(de).t() @ u
    wide = max(rows, cols)
    low = 2 * (4 + wide // 64 + 8 + 2)                      # of u and v, as in test_batch
    chain = low + 2 * (3 * ((R + 15) // 16) + 3)
    assert ((dx[:tokens].double() - want).abs() <= chain * U32 * mag + 1e-30).all()
    chain = low + 2 * (6 + tokens // 32 + 8 + 1)            # six per stage, the stages, the cluster
    assert ((da.double() - wa).abs() <= chain * U32 * ma).all(), ((da.double() - wa).abs() / (U32 * ma + 1e-30)).max()
    assert ((db.double() - wb).abs() <= chain * U32 * mb).all(), ((db.double() - wb).abs() / (U32 * mb + 1e-30)).max()
    assert torch.equal(dx[:tokens][bare], start[bare])
    assert (dxw[:tokens, cols:] == -7.0).all() and (dxw[tokens:] == -7.0).all()


def test_gradients_against_differences(ctx, adapters):
    """d<dy, y>/d(one element) by central differences of the forward call, in steps that bf16 holds."""
    rows, cols, tokens, r = 40, 64, 48, 5
    ad = adapters(rows, cols, 1, r, tokens, {0: r})
    a, b = ad.a[0].to(BF16), ad.b[0].to(BF16)
    x, dy = torch.randn(tokens, cols, device="cuda").to(BF16), torch.randn(tokens, rows, device="cuda").to(BF16)
    dx, da, db = torch.empty(tokens, cols, device="cuda"), torch.empty(1, r, cols, device="cuda"), torch.empty(1, rows, r, device="cuda")
    y = torch.empty(tokens, rows, device="cuda")
    torch.cuda.synchronize()
    ad.h.backward(x.data_ptr(), cols, dy.data_ptr(), rows, tokens, 0, 0, 0, dx.data_ptr(), cols, da.data_ptr(), db.data_ptr())
    ctx.sync()

    def value(x, a, b):
        torch.cuda.synchronize()
        ad.h.set(0, r, ad.s[0], a.data_ptr(), b.data_ptr(), _capi.TYPE_BF16)
        ad.h.matmul_bf16(x.data_ptr(), tokens, cols, 0, 0, 0, y.data_ptr(), rows)
        ctx.sync()
        return float((y.double() * dy.double()).sum())

    for name, grad, which in (("x", dx, 0), ("a", da[0], 1), ("b", db[0], 2)):
        for i, j in ((0, 0), (3, 4), (grad.shape[0] - 1, grad.shape[1] - 1)):
            up, down = [t.clone() for t in (x, a, b)], [t.clone() for t in (x, a, b)]
            up[which][i, j] += 0.5
            down[which][i, j] -= 0.5
            step = float(up[which][i, j].double() - down[which][i, j].double())
            # y is linear in each of the three: the quotient is the gradient up to the float32 sums behind both values
            got = (value(*up) - value(*down)) / step
            assert abs(got - float(grad[i, j])) <= 1e-4 * (1 + abs(got)), (name, i, j)


def test_backward_parts_and_repeats(ctx, adapters):
    """Every output may be left out; the same call gives the same bits; no tokens give zero gradients."""
    rows, cols, tokens = 264, 128, 300
    ad = adapters(rows, cols, 3, 24, tokens, {0: 24, 2: 8})
    x, dy = torch.randn(tokens, cols, device="cuda").to(BF16), torch.randn(tokens, rows, device="cuda").to(BF16)
    ids = make_ids("mixed", tokens, {0: 24, 2: 8}, 3)

    def once(want, n=tokens):
        out = [torch.full((tokens, cols), 5.0, device="cuda"), torch.full((3, 24, cols), 5.0, device="cuda"), torch.full((3, rows, 24), 5.0, device="cuda")]
        torch.cuda.synchronize()
        p = [t.data_ptr() if w else 0 for t, w in zip(out, want)]
        ad.h.backward(x.data_ptr(), cols, dy.data_ptr(), rows, n, ids.data_ptr(), 0, 0, p[0], cols, p[1], p[2])
        ctx.sync()
        return out

    full = once((1, 1, 1))
    for want in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
        for got, ref, w in zip(once(want), full, want):
            assert torch.equal(got, ref if w else torch.full_like(ref, 5.0))
    dx, da, db = once((1, 1, 1), 0)
    assert (dx == 5.0).all() and (da == 0).all() and (db == 0).all()


@pytest.mark.parametrize("shift,lddy", [(0, 129), (1, 136), (3, 131), (8, 133)])
def test_backward_of_unaligned_gradients(ctx, adapters, shift, lddy):
    """dy rows at any address and pitch give the bits of aligned ones; the first such call is refused under capture."""
    rows, cols, tokens = 129, 96, 150
    ad = adapters(rows, cols, 2, 16, tokens, {0: 16, 1: 3})
    x, ids = torch.randn(tokens, cols, device="cuda").to(BF16), make_ids("mixed", tokens, {0: 16, 1: 3}, 2)
    flat = torch.full((tokens * lddy + 16,), float("nan"), dtype=BF16, device="cuda")
    dy = flat[shift:shift + tokens * lddy].view(tokens, lddy)[:, :rows]
    dy.copy_(torch.randn(tokens, rows, device="cuda"))
    even = torch.full((tokens, 136), float("nan"), dtype=BF16, device="cuda")
    even[:, :rows].copy_(dy)

    def call(dev, ld):
        out = [torch.empty(tokens, cols, device="cuda"), torch.empty(2, 16, cols, device="cuda"), torch.empty(2, rows, 16, device="cuda")]
        torch.cuda.synchronize()
        ad.h.backward(x.data_ptr(), cols, dev, ld, tokens, ids.data_ptr(), 0, 0, out[0].data_ptr(), cols, out[1].data_ptr(), out[2].data_ptr())
        ctx.sync()
        return out

    with pytest.raises(lib_b200.QmError) as e:
        capture.launches(ctx, lambda: ad.h.backward(x.data_ptr(), cols, flat.data_ptr() + 2 * shift, lddy, tokens, ids.data_ptr(), 0, 0,
                                                    even.data_ptr(), cols, 0, 0))
    assert e.value.code == 900      # CUDA_ERROR_STREAM_CAPTURE_UNSUPPORTED
    for a, b in zip(call(flat.data_ptr() + 2 * shift, lddy), call(even.data_ptr(), 136)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("type,kept", [(_capi.TYPE_F32, torch.float32), (_capi.TYPE_F16, torch.float16), (_capi.TYPE_BF16, BF16)])
def test_slots_are_replaced_and_emptied(ctx, adapters, type, kept):
    rows, cols = 130, 64
    ad = adapters(rows, cols, 2, 40, 4, {0: 40, 1: 9}, type=type)
    x = torch.randn(4, cols, device="cuda")
    ids = torch.tensor([0, 1, 0, 1], dtype=torch.int32, device="cuda")
    y, yb = torch.empty(4, rows, device="cuda"), torch.empty(4, rows, device="cuda")

    def check():
        xb = x.to(BF16)
        torch.cuda.synchronize()
        ad.h.matvec(x.data_ptr(), 4, cols, ids.data_ptr(), 0, 0, y.data_ptr(), rows)
        ad.h.matmul_bf16(xb.data_ptr(), 4, cols, ids.data_ptr(), 0, 0, yb.data_ptr(), rows)
        ctx.sync()
        for got, inp in ((y, x), (yb, xb)):
            want, mag = ad.forward(inp.double(), ids, torch.zeros_like(got))
            assert ((got.double() - want).abs() <= 80 * U32 * mag + 1e-30).all()

    check()
    ad.put(0, 3, -1.5, torch.randn(3, cols, device="cuda").to(kept), torch.randn(rows, 3, device="cuda").to(kept), type)   # a smaller one
    check()
    ad.h.set(1, 0, 1.0, 0, 0)      # empty
    del ad.a[1]
    check()


@pytest.mark.parametrize("R,used", [(16, 3), (16, 256), (32, 64), (64, 40), (128, 32)])
def test_many_slots(ctx, adapters, R, used):
    """Hundreds of slots, few or all of them with tokens: the grids are smaller than the tiles there may be."""
    rows, cols, tokens, slots = 4096, 4224, 1100, 256
    held = list(range(0, slots, slots // used))[:used]
    ad = adapters(rows, cols, slots, R, tokens, {e: 1 + (R - 1 + 7 * i) % R for i, e in enumerate(held)}, seed=R + used)
    g = torch.Generator(device="cuda")
    g.manual_seed(R * used)
    x = torch.randn(tokens, cols, generator=g, device="cuda").to(BF16)
    dy = torch.randn(tokens, rows, generator=g, device="cuda").to(BF16)
    base, dbase = torch.randn(tokens, rows, generator=g, device="cuda"), torch.randn(tokens, cols, generator=g, device="cuda")
    y, dx = torch.full((tokens + 1, rows), -7.0, device="cuda"), torch.full((tokens + 1, cols), -7.0, device="cuda")
    names = torch.tensor(held + [-1], dtype=torch.int32, device="cuda")
    for mixed in (True, False):
        pick = torch.randint(0, len(names), (tokens,), generator=g, device="cuda")
        ids = names[pick if mixed else pick.sort().values]
        torch.cuda.synchronize()
        ad.h.matmul_bf16(x.data_ptr(), tokens, cols, ids.data_ptr(), base.data_ptr(), rows, y.data_ptr(), rows)
        ad.h.backward(x.data_ptr(), cols, dy.data_ptr(), rows, tokens, ids.data_ptr(), dbase.data_ptr(), cols, dx.data_ptr(), cols, 0, 0)
        ctx.sync()
        want, mag = ad.forward(x.double(), ids, base)
        low = 2 * (4 + cols // 64 + 8 + 2)                  # as in test_batch and test_backward
        chain = low + 2 * (3 * ((R + 15) // 16) + 3)
        assert ((y[:tokens].double() - want).abs() <= chain * U32 * mag).all()
        want, mag = dbase.double().clone(), dbase.double().abs()
        for e, at in ad.of(ids):
            de = dy[at].double()
            want[at] += ad.s[e] * de @ ad.b[e] @ ad.a[e]
            mag[at] += ad.s[e] * de.abs() @ ad.b[e].abs() @ ad.a[e].abs()
        assert ((dx[:tokens].double() - want).abs() <= chain * U32 * mag).all()
        bare = ids < 0
        assert torch.equal(y[:tokens][bare], base[bare]) and torch.equal(dx[:tokens][bare], dbase[bare])
        assert (y[tokens] == -7.0).all() and (dx[tokens] == -7.0).all()
    where = {l.name for l in capture.launches(ctx, lambda: ad.h.matmul_bf16(x.data_ptr(), tokens, cols, ids.data_ptr(), base.data_ptr(), rows, y.data_ptr(), rows))}
    assert where == {"qm_lora_lists", "qm_lora_shrink_r%d_m" % R, "qm_lora_expand_r%d_m" % R}


def test_rows_far_apart(ctx, adapters):
    """Row pitches whose byte offsets pass 32 bits."""
    rows, cols, ld = 200, 64, 1 << 30
    ad = adapters(rows, cols, 1, 8, 3, {0: 8})
    x = torch.randn(3, cols, device="cuda").to(BF16)
    far = torch.empty(2 * ld + 256, device="cuda")
    ad_y = far.as_strided((3, rows), (ld, 1))
    torch.cuda.synchronize()
    ad.h.matmul_bf16(x.data_ptr(), 3, cols, 0, 0, 0, far.data_ptr(), ld)
    ctx.sync()
    want, mag = ad.forward(x.double(), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, rows, device="cuda"))
    assert ((ad_y.double() - want).abs() <= 60 * U32 * mag + 1e-30).all()
    xf = x.float()
    torch.cuda.synchronize()
    ad.h.matvec(xf.data_ptr(), 3, cols, 0, 0, 0, far.data_ptr(), ld)
    ctx.sync()
    assert ((ad_y.double() - want).abs() <= 60 * U32 * mag + 1e-30).all()


def test_captured_calls_follow_their_inputs(ctx, adapters):
    """Forward and backward in one graph, adapters set in it too; replayed on other inputs, on another stream."""
    rows, cols, tokens = 256, 128, 100
    ad = adapters(rows, cols, 2, 16, tokens, {0: 16, 1: 5})
    x, dy = torch.zeros(tokens, cols, dtype=BF16, device="cuda"), torch.zeros(tokens, rows, dtype=BF16, device="cuda")
    ids = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    a, b = torch.zeros(16, cols, device="cuda"), torch.zeros(rows, 16, device="cuda")
    y, dx = torch.zeros(tokens, rows, device="cuda"), torch.zeros(tokens, cols, device="cuda")
    da, db = torch.zeros(2, 16, cols, device="cuda"), torch.zeros(2, rows, 16, device="cuda")

    def step():
        ad.h.set(0, 16, 0.5, a.data_ptr(), b.data_ptr(), _capi.TYPE_F32)
        ad.h.matmul_bf16(x.data_ptr(), tokens, cols, ids.data_ptr(), 0, 0, y.data_ptr(), rows)
        ad.h.backward(x.data_ptr(), cols, dy.data_ptr(), rows, tokens, ids.data_ptr(), 0, 0, dx.data_ptr(), cols, da.data_ptr(), db.data_ptr())

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph, stream=stream):
            ctx.set_stream(stream.cuda_stream)
            step()
    finally:
        ctx.set_stream(0)
    for seed in (1, 2):
        r = torch.Generator(device="cuda")
        r.manual_seed(seed)
        x.copy_(torch.randn(tokens, cols, generator=r, device="cuda"))
        dy.copy_(torch.randn(tokens, rows, generator=r, device="cuda"))
        ids.copy_(torch.randint(-1, 2, (tokens,), generator=r, device="cuda"))
        a.copy_(torch.randn(16, cols, generator=r, device="cuda"))
        b.copy_(torch.randn(rows, 16, generator=r, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (y, dx, da, db)]
        torch.cuda.synchronize()
        step()
        ctx.sync()
        for got, want in zip(replayed, (y, dx, da, db)):
            assert torch.equal(got, want)
    del graph


def test_two_handles_on_two_streams(ctx, adapters):
    """Handles share nothing: their calls may overlap."""
    rows, cols, tokens = 512, 1024, 500
    two = [adapters(rows, cols, 2, 32, tokens, {0: 32, 1: 7}, seed=i) for i in range(2)]
    x = [torch.randn(tokens, cols, device="cuda").to(BF16) for _ in two]
    ids = make_ids("mixed", tokens, {0: 32, 1: 7}, 2)
    y = [torch.empty(tokens, rows, device="cuda") for _ in two]
    streams = [torch.cuda.Stream() for _ in two]
    torch.cuda.synchronize()
    try:
        for _ in range(10):
            for ad, xs, ys, st in zip(two, x, y, streams):
                ctx.set_stream(st.cuda_stream)
                ad.h.matmul_bf16(xs.data_ptr(), tokens, cols, ids.data_ptr(), 0, 0, ys.data_ptr(), rows)
        torch.cuda.synchronize()
    finally:
        ctx.set_stream(0)
    for ad, xs, ys in zip(two, x, y):
        want, mag = ad.forward(xs.double(), ids, torch.zeros_like(ys))
        assert ((ys.double() - want).abs() <= 100 * U32 * mag + 1e-30).all()


@pytest.mark.parametrize("fmt", [_capi.Q8_0, _capi.Q4_K])
def test_product_adapters_norm_and_rotation_together(ctx, adapters, fmt):
    """A decode step's q|k|v: stored weights with the RMSNorm in the product, two requests' adapters, then norm and rotation
    of the heads; against the oracle's product and the formulas in float64."""
    heads, kv, dim, cols, m = 4, 2, 64, 512, 3
    rows = (heads + 2 * kv) * dim
    raw = synth.weights(fmt, rows, cols, seed=5)
    w = ctx.store_upload(fmt, rows, cols, raw)
    ad = adapters(rows, cols, 2, 8, 8, {0: 8, 1: 4})
    x = torch.tensor(synth.activations(m, cols, seed=6), device="cuda")
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    qkv = torch.empty(m, rows, device="cuda")
    pos = torch.tensor([7, 100000, 3], dtype=torch.int32, device="cuda")
    gq, gk = torch.rand(dim, device="cuda") + 0.5, torch.rand(dim, device="cuda") + 0.5
    q, k = torch.empty(m, heads * dim, device="cuda"), torch.empty(m, kv * dim, device="cuda")
    rope = ctx.rope(dim, dim, 10000.0)
    torch.cuda.synchronize()

    def step():
        ctx.matvec_lora(w, ad.h, x.data_ptr(), m, cols, ids.data_ptr(), qkv.data_ptr(), rows, _capi.XOP_RMSNORM)
        rope.qk_norm(qkv.data_ptr(), rows, m, heads, kv, gq.data_ptr(), gk.data_ptr(), 1e-5, pos.data_ptr(), q.data_ptr(), heads * dim,
                     k.data_ptr(), kv * dim)

    step()
    ctx.sync()
    normed = transformed(x, None, _capi.XOP_RMSNORM)
    product = torch.tensor(oracle.MatVec(fmt, raw, rows, cols, normed.float().cpu().numpy()), device="cuda").double()
    want, _ = ad.forward(normed, ids, product)
    # the product of three rows takes its activations with 14 bits of their group's maximum
    assert float((qkv.double() - want).norm() / want.norm()) <= 4e-4
    z = qkv.double().view(m, -1, dim)
    for got, part, gain in ((q, z[:, :heads], gq), (k, z[:, heads:heads + kv], gk)):
        n = part / (part.square().mean(-1, keepdim=True) + 1e-5).sqrt() * gain.double()
        ang = pos.double()[:, None, None] * 10000.0 ** (-2.0 * torch.arange(dim // 2, device="cuda", dtype=torch.float64) / dim)
        f, s = n[..., :dim // 2], n[..., dim // 2:]
        turned = torch.cat((f * ang.cos() - s * ang.sin(), s * ang.cos() + f * ang.sin()), -1).reshape(m, -1)
        assert torch.allclose(got.double(), turned, rtol=0, atol=2e-6 * float(n.abs().max()))
    # the launches follow one another by programmatic edges, as those of the matvecs do
    made = capture.launches(ctx, step)
    assert [l.name for l in made][-2:] == ["qm_lora_rows", "qm_qk_norm_w1"] and made[-1].overlaps == "qm_lora_rows"
    # the batched product with its adapters
    if fmt == _capi.Q4_K:
        xb = x.to(BF16)
        c, c2 = torch.empty(m, rows, device="cuda"), torch.empty(m, rows, device="cuda")
        torch.cuda.synchronize()
        ctx.matmul_bf16_lora(w, ad.h, xb.data_ptr(), m, cols, ids.data_ptr(), c.data_ptr(), rows)
        ctx.matmul_bf16(w, xb.data_ptr(), m, cols, c2.data_ptr(), rows)
        ctx.sync()
        want, mag = ad.forward(xb.double(), ids, c2)
        assert ((c.double() - want).abs() <= 80 * U32 * mag).all()
    rope.close()
    w.free()


def test_refusals(ctx, adapters):
    def code(call, *args):
        with pytest.raises(lib_b200.QmError) as e:
            call(*args)
        return e.value.code

    SHAPE, ARG, FORMAT, LIMIT = -4, -5, -3, -11
    for args, want in [((0, 64, 1, 1, 1), SHAPE), ((8, 48, 1, 1, 1), SHAPE), ((8, 0, 1, 1, 1), SHAPE), ((8, 64, 0, 1, 1), SHAPE), ((8, 64, 1, 0, 1), SHAPE),
                       ((8, 64, 1, 1, 0), SHAPE), ((8, 64, 257, 1, 1), LIMIT), ((8, 64, 1, 129, 1), LIMIT), ((8, 65536, 1, 1, 1), LIMIT),
                       ((1 << 23, 64, 1, 1, 1), LIMIT), ((8, 64, 1, 1, (1 << 20) + 1), LIMIT)]:
        assert code(ctx.lora, *args) == want, args
    ad = adapters(64, 64, 2, 8, 16, {0: 8})
    h = ad.h
    buf = torch.zeros(1 << 16, device="cuda")
    p = buf.data_ptr()
    X, Y, B, I, D = p, p + 65536, p + 131072, p + 196608, p + 212992
    for args, want in [((2, 4, 1.0, X, Y), SHAPE), ((-1, 4, 1.0, X, Y), SHAPE), ((0, 9, 1.0, X, Y), SHAPE), ((0, -1, 1.0, X, Y), SHAPE), ((0, 4, 1.0, 0, Y), ARG),
                       ((0, 4, 1.0, X, 0), ARG), ((0, 4, float("nan"), X, Y), ARG), ((0, 4, 1.0, X + 1, Y), ARG), ((0, 4, 1.0, X, Y, 2), FORMAT)]:
        assert code(h.set, *args) == want, args
    ok = dict(x_dev=X, m=4, ldx=64, ids_dev=I, base_dev=B, ldb=64, y_dev=Y, ldy=64)
    for change, want in [(dict(m=0), SHAPE), (dict(m=9), SHAPE), (dict(ldx=60), SHAPE), (dict(ldy=63), SHAPE), (dict(ldb=63), SHAPE), (dict(ldx=1 << 40), SHAPE),
                         (dict(x_dev=0), ARG), (dict(y_dev=0), ARG), (dict(x_dev=X + 4), ARG), (dict(ldx=66), ARG), (dict(y_dev=Y + 2), ARG), (dict(ids_dev=I + 1), ARG),
                         (dict(base_dev=Y + 256), ARG), (dict(base_dev=Y, ldb=68), ARG), (dict(y_dev=X + 512), ARG), (dict(flags=4), ARG), (dict(flags=0x200), ARG),
                         (dict(flags=2), ARG), (dict(flags=3, x2_dev=B + 4), ARG), (dict(ids_dev=Y), ARG)]:
        assert code(lambda: h.matvec(**{**ok, **change})) == want, change
    ok = dict(x_dev=X, tokens=4, ldx=64, ids_dev=I, base_dev=B, ldb=64, y_dev=Y, ldy=64)
    for change, want in [(dict(tokens=-1), SHAPE), (dict(tokens=17), LIMIT), (dict(ldx=56), SHAPE), (dict(ldy=63), SHAPE), (dict(ldb=1), SHAPE), (dict(x_dev=0), ARG),
                         (dict(y_dev=0), ARG), (dict(x_dev=X + 8), ARG), (dict(ldx=68), ARG), (dict(base_dev=Y + 4), ARG), (dict(y_dev=X), ARG)]:
        assert code(lambda: h.matmul_bf16(**{**ok, **change})) == want, change
    h.matmul_bf16(X, 0, 64, I, 0, 0, Y, 64)      # no tokens: nothing to do
    ok = dict(x_dev=X, ldx=64, dy_dev=D, lddy=64, tokens=4, ids_dev=I, base_dev=B, ldb=64, dx_dev=Y, lddx=64, da_dev=B + 8192, db_dev=B + 16384)
    for change, want in [(dict(dx_dev=0, da_dev=0, db_dev=0), ARG), (dict(tokens=17), LIMIT), (dict(tokens=-1), SHAPE), (dict(lddy=56), SHAPE),
                         (dict(dy_dev=D + 1), ARG), (dict(dy_dev=0), ARG), (dict(x_dev=0), ARG), (dict(lddx=63), SHAPE), (dict(dx_dev=D), ARG), (dict(dx_dev=X), ARG),
                         (dict(da_dev=B + 2), ARG), (dict(base_dev=Y + 4), ARG), (dict(da_dev=X), ARG), (dict(db_dev=B + 8192), ARG), (dict(db_dev=Y + 8), ARG)]:
        assert code(lambda: h.backward(**{**ok, **change})) == want, change
    w = ctx.store_create(_capi.Q8_0, 96, 64)
    assert code(ctx.matvec_lora, w, h, X, 1, 64, 0, Y, 96) == SHAPE     # a matrix of another shape
    w.free()
    assert lib_b200.lib.qm_lora_destroy(ctx._h, None) == ARG
    other = lib_b200.Context(0)
    assert lib_b200.lib.qm_lora_destroy(other._h, h._h) == ARG          # a handle of another context
    other.close()
    ctx.sync()
    assert ctx.last_status() == (0, 0)
