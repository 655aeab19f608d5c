"""Low-rank adapters beside stored weights and the normalised, rotated queries and keys behind the q|k|v product, as cases
that can be timed and compared: in a plain form of elementary torch operations, and as the calls of this library.

Kinds of cases (each stands for one real use):
  lora_rows   a decode step of 1..8 requests: base + scale * B (A f(x)) for each row with its own request's adapter, float32
              activations, f the plain row or its RMS normalised form (as qm_matvec stages it)
  lora_batch  the same over a batch of tokens with bf16 activations: prompts of several requests one after the other, or a
              large decode batch (every request one token); requests without an adapter keep their base rows
  lora_grad   the backward pass of lora_batch in a training step: the adapters as the optimizer left them, then the gradients
              of the activations, of every A and of every B
  qk          per head RMSNorm with gain and rotary positions for the q and k parts of q|k|v rows in one pass
  qk_grad     its backward pass: gradients of the raw q|k rows and of both gains
"""
import functools

import torch

own = False

BF16 = torch.bfloat16


def listed():
    return [
        # the smallest call: one token of one request, a square projection of a 4096-wide model
        {"name": "lora rows 1", "kind": "lora_rows", "rows": 4096, "cols": 4096, "m": 1, "adapters": 1, "rank": 16, "xop": 0, "bare": 0},
        # eight requests with eight adapters on the stacked q|k|v matrix, RMSNorm fused
        {"name": "lora rows 8", "kind": "lora_rows", "rows": 6144, "cols": 4096, "m": 8, "adapters": 8, "rank": 64, "xop": 1, "bare": 0},
        # an odd one: rows that are no whole tiles, five rows that share three adapters, one without any
        {"name": "lora rows ragged", "kind": "lora_rows", "rows": 10007, "cols": 2304, "m": 5, "adapters": 3, "rank": 24, "xop": 0, "bare": 1},
        # a decode batch of 64 requests over 32 small adapters
        {"name": "lora batch 64", "kind": "lora_batch", "rows": 6144, "cols": 4096, "tokens": 64, "requests": 64, "adapters": 32, "rank": 16, "bare": 0},
        # short prompts of five requests on the stacked gate|up matrix, the last one without an adapter
        {"name": "lora batch 391", "kind": "lora_batch", "rows": 28672, "cols": 4096, "tokens": 391, "requests": 5, "adapters": 4, "rank": 32, "bare": 1},
        # long prompts of eight requests with large adapters on the down projection
        {"name": "lora batch 2048", "kind": "lora_batch", "rows": 4096, "cols": 14336, "tokens": 2048, "requests": 8, "adapters": 8, "rank": 64, "bare": 0},
        # a small training step: three sequences of odd lengths, two adapters
        {"name": "lora grad 777", "kind": "lora_grad", "rows": 6144, "cols": 4096, "tokens": 777, "requests": 3, "adapters": 2, "rank": 8, "bare": 0},
        # a large one: one adapter on gate|up, 4096 tokens
        {"name": "lora grad 4096", "kind": "lora_grad", "rows": 28672, "cols": 4096, "tokens": 4096, "requests": 1, "adapters": 1, "rank": 32, "bare": 0},
        # one token behind the q|k|v product of an 8B-parameter model
        {"name": "qk 1", "kind": "qk", "tokens": 1, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "interleaved": 0, "norm": 1, "bf16": 0, "far": 4096},
        # an odd one: heads of 96 of which 64 rotate, adjacent pairs, far positions
        {"name": "qk 777", "kind": "qk", "tokens": 777, "q_heads": 12, "k_heads": 3, "dim": 96, "rot": 64, "interleaved": 1, "norm": 1, "bf16": 0, "far": 1000000},
        # a long prompt, bf16 results for the attention and the cache
        {"name": "qk 8192", "kind": "qk", "tokens": 8192, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "interleaved": 0, "norm": 1, "bf16": 1, "far": 131072},
        # the training step's backward pass, bf16 gradients from the attention
        {"name": "qk grad 4096", "kind": "qk_grad", "tokens": 4096, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "interleaved": 0, "norm": 1, "bf16": 1, "far": 8192},
    ]


def draw(rng):
    def log(lo, hi, step=1):
        """A multiple of `step` between lo and hi, even over the logarithm."""
        v = lo * (hi / lo) ** rng.random()
        return max(lo, min(hi, int(round(v / step)) * step))

    kind = rng.choice(["lora_rows", "lora_rows", "lora_batch", "lora_batch", "lora_grad", "lora_grad", "qk", "qk", "qk_grad"])
    if kind == "lora_rows":
        m = rng.randint(1, 8)
        return {"kind": kind, "rows": log(512, 28672), "cols": log(512, 14336, 32), "m": m, "adapters": rng.randint(1, m),
                "rank": log(4, 128), "xop": rng.randint(0, 1), "bare": rng.randint(0, 1) if m > 1 else 0}
    if kind == "lora_batch":
        tokens, most = log(9, 2048), 32
        requests = log(1, min(tokens, 128))
        return {"kind": kind, "rows": log(512, 14336), "cols": log(512, 14336, 32), "tokens": tokens, "requests": requests,
                "adapters": rng.randint(1, min(requests, most)), "rank": log(4, 128), "bare": rng.randint(0, 1) if requests > 1 else 0}
    if kind == "lora_grad":
        tokens = log(32, 4096)
        requests = log(1, 8)
        return {"kind": kind, "rows": log(512, 14336), "cols": log(512, 14336, 32), "tokens": tokens, "requests": requests,
                "adapters": rng.randint(1, min(requests, 4)), "rank": log(4, 128), "bare": rng.randint(0, 1) if requests > 1 else 0}
    dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
    k_heads = rng.choice([1, 2, 4, 8])
    return {"kind": kind, "tokens": log(1, 4096) if kind == "qk" else log(16, 2048), "q_heads": k_heads * rng.choice([1, 3, 4, 8]),
            "k_heads": k_heads, "dim": dim, "rot": rng.choice([dim, dim, dim // 2]), "interleaved": rng.randint(0, 1),
            "norm": rng.choice([0, 1, 1]) if kind == "qk" else 1, "bf16": rng.randint(0, 1), "far": log(64, 4000000)}


THETA = 500000.0
EPS_ROW = 1e-6     # of the RMS normalised activation row (qm_matvec's)
EPS_HEAD = 1e-5    # of the per head norm


def ranks_of(case):
    """Adapters as servers hold them: every second one has a smaller rank (odd sizes among them)."""
    return [case["rank"] if i % 2 == 0 else max(1, case["rank"] * 5 // 8) for i in range(case["adapters"])]


def used(case):
    """Adapters that at least one token of the case uses."""
    return min(case["adapters"], case.get("requests", case.get("m")) - case["bare"])


@functools.lru_cache(maxsize=None)
def context():
    """The program's one library context."""
    import lib_b200
    torch.cuda.init()
    return lib_b200.Context(0)


class Owned:
    """A library object of one state, given back with it."""

    def __init__(self, obj):
        self.obj = obj

    def __del__(self):
        self.obj.close()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = (prepare_qk if case["kind"].startswith("qk") else prepare_lora)(case, g, normal)
    torch.cuda.synchronize()   # the library works on a stream of its own
    return s


def prepare_lora(case, g, normal):
    kind, rows, cols, count, rank = case["kind"], case["rows"], case["cols"], case["adapters"], case["rank"]
    tokens = case["m"] if kind == "lora_rows" else case["tokens"]
    requests = tokens if kind == "lora_rows" else case["requests"]
    # every request has at least one token; the adapters go round the requests, in a shuffled order
    cuts = torch.randperm(tokens - 1, generator=g, device="cuda")[:requests - 1].sort().values + 1
    owner = torch.zeros(tokens, dtype=torch.int64, device="cuda")
    owner[cuts] = 1
    owner = owner.cumsum(0)
    with_one = requests - case["bare"]
    of_request = torch.full((requests,), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(with_one, generator=g, device="cuda")
    of_request[:with_one] = (order % count).to(torch.int32)
    ranks = torch.tensor(ranks_of(case), device="cuda")
    there = torch.arange(rank, device="cuda")[None, :] < ranks[:, None]
    # trained adapters: A keeps its initial spread, B and the scale give changes of a fraction of the base result
    a = (normal(count, rank, cols) * cols ** -0.5 * there[:, :, None]).to(BF16)
    b = (normal(count, rows, rank) * 0.05 * there[:, None, :]).to(BF16)
    scale = 0.5 + torch.rand(count, generator=g, device="cuda")
    s = {"kind": kind, "tokens": tokens, "rows": rows, "cols": cols, "xop": case.get("xop", 0), "ids": of_request[owner], "a": a, "b": b, "scale": scale}
    if kind == "lora_rows":
        s["x"] = normal(tokens, cols)
    else:
        s["x"] = normal(tokens, cols).to(BF16)
    if kind == "lora_grad":
        s["dy"] = (normal(tokens, rows) * 0.01).to(BF16)
        s["base"] = normal(tokens, cols) * 0.05      # the frozen weights' share of the activations' gradient
        s["out"] = torch.empty(tokens, cols, device="cuda")
        s["da"] = torch.empty(count, rank, cols, device="cuda")
        s["db"] = torch.empty(count, rows, rank, device="cuda")
    else:
        s["base"] = normal(tokens, rows)             # the stored weights' product
        s["out"] = torch.empty(tokens, rows, device="cuda")
    if own:
        # the adapters as a program holds them: each cut to its rank, and the handle of the projection
        s["parts"] = [(i, r, float(f), a[i, :r].contiguous(), b[i, :, :r].contiguous())
                      for i, (r, f) in enumerate(zip(ranks_of(case), scale.tolist()))]
        torch.cuda.synchronize()
        s["lora"] = Owned(context().lora(rows, cols, count, rank, tokens))
        set_adapters(s)
        context().sync()
        s["ptr"] = {k: s[k].data_ptr() for k in ("x", "ids", "base", "out", "dy", "da", "db") if k in s}
    return s


def set_adapters(s):
    for slot, r, factor, a, b in s["parts"]:
        s["lora"].obj.set(slot, r, factor, a.data_ptr(), b.data_ptr(), 30)


def prepare_qk(case, g, normal):
    tokens, hq, hk, dim, rot = (case[k] for k in ("tokens", "q_heads", "k_heads", "dim", "rot"))
    grads = BF16 if case["bf16"] else torch.float32
    first = int(torch.randint(0, case["far"], (1,), generator=g, device="cuda"))
    s = {"kind": case["kind"], "tokens": tokens, "hq": hq, "hk": hk, "dim": dim, "rot": rot, "interleaved": case["interleaved"],
         "norm": case["norm"], "out_type": grads, "x": normal(tokens, (hq + 2 * hk) * dim) * 0.7,
         "gq": torch.rand(dim, generator=g, device="cuda") + 0.5, "gk": torch.rand(dim, generator=g, device="cuda") + 0.5,
         "pos": (torch.arange(tokens, device="cuda") + first).to(torch.int32)}
    if case["kind"] == "qk":
        s["q"] = torch.empty(tokens, hq * dim, dtype=grads, device="cuda")
        s["k"] = torch.empty(tokens, hk * dim, dtype=grads, device="cuda")
    else:
        s["q"] = (normal(tokens, hq * dim) * 0.01).to(grads)
        s["k"] = (normal(tokens, hk * dim) * 0.01).to(grads)
        s["dx"] = torch.empty(tokens, (hq + hk) * dim, device="cuda")
        s["dgq"], s["dgk"] = torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")
    if own:
        s["rope"] = Owned(context().rope(dim, rot, THETA, interleaved=bool(case["interleaved"])))
        s["ptr"] = {k: s[k].data_ptr() for k in ("x", "gq", "gk", "pos", "q", "k", "dx", "dgq", "dgk") if k in s}
        s["flags"] = (0 if case["norm"] else 1) | (2 if case["bf16"] else 0)
    return s


def run(s):
    return (OWN if own else PLAIN)[s["kind"]](s)


# ---- the library's calls ------------------------------------------------------------------------------------------------
def own_lora_rows(s):
    p = s["ptr"]
    s["lora"].obj.matvec(p["x"], s["tokens"], s["cols"], p["ids"], p["base"], s["rows"], p["out"], s["rows"], s["xop"])
    return s["out"]


def own_lora_batch(s):
    p = s["ptr"]
    s["lora"].obj.matmul_bf16(p["x"], s["tokens"], s["cols"], p["ids"], p["base"], s["rows"], p["out"], s["rows"])
    return s["out"]


def own_lora_grad(s):
    p = s["ptr"]
    set_adapters(s)     # the optimizer changed them
    s["lora"].obj.backward(p["x"], s["cols"], p["dy"], s["rows"], s["tokens"], p["ids"], p["base"], s["cols"], p["out"], s["cols"],
                           p["da"], p["db"])
    return {"dx": s["out"], "da": s["da"], "db": s["db"]}


def own_qk(s):
    p, dim, hq, hk = s["ptr"], s["dim"], s["hq"], s["hk"]
    s["rope"].obj.qk_norm(p["x"], (hq + 2 * hk) * dim, s["tokens"], hq, hk, p["gq"], p["gk"], EPS_HEAD, p["pos"], p["q"], hq * dim, p["k"],
                          hk * dim, s["flags"])
    return {"q": s["q"], "k": s["k"]}


def own_qk_grad(s):
    p, dim, hq, hk = s["ptr"], s["dim"], s["hq"], s["hk"]
    s["rope"].obj.qk_norm_backward(p["x"], (hq + 2 * hk) * dim, s["tokens"], hq, hk, p["gq"], p["gk"], EPS_HEAD, p["pos"], p["q"], hq * dim,
                                   p["k"], hk * dim, p["dx"], (hq + hk) * dim, p["dgq"], p["dgk"], s["flags"])
    return {"dx": s["dx"], "dgq": s["dgq"], "dgk": s["dgk"]}


# ---- the plain forms ----------------------------------------------------------------------------------------------------
def chosen(s):
    """[tokens][adapters]: the scale of the token's adapter at its place, zeros elsewhere."""
    mine = s["ids"][:, None] == torch.arange(s["a"].shape[0], device="cuda", dtype=torch.int32)[None, :]
    return mine.float() * s["scale"][None, :]


def masked(products, mask):
    """[tokens][adapters * rank] with every adapter's columns times the token's mask for it."""
    return (products.view(*mask.shape, -1) * mask[:, :, None]).reshape(products.shape)


def plain_lora(s):
    x = s["x"].float()
    if s["xop"]:
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS_ROW)
    count, rank, cols = s["a"].shape
    low = masked(x @ s["a"].float().view(count * rank, cols).t(), chosen(s))
    return s["base"] + low @ s["b"].float().transpose(1, 2).reshape(count * rank, -1)


def plain_lora_grad(s):
    x, dy, mask = s["x"].float(), s["dy"].float(), chosen(s)
    count, rank, cols = s["a"].shape
    a, b = s["a"].float().view(count * rank, cols), s["b"].float().transpose(1, 2).reshape(count * rank, -1)
    u, v = masked(x @ a.t(), mask), masked(dy @ b.t(), mask)
    return {"dx": s["base"] + v @ a, "da": (v.t() @ x).view(count, rank, cols), "db": (u.t() @ dy).view(count, rank, -1).transpose(1, 2).contiguous()}


def turns(s):
    """cos and sin of position * theta^(-2i/rot): [tokens][1][rot/2], angles in 64 bits (far positions)."""
    i = torch.arange(s["rot"] // 2, device="cuda", dtype=torch.float64)
    angle = s["pos"].double()[:, None] * torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"), -2.0 * i / s["rot"])[None, :]
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def turned(s, z, cos, sin):
    """The first `rot` elements of every head turned pairwise, the others as they are."""
    rot, half = s["rot"], s["rot"] // 2
    if s["interleaved"]:
        p, q = z[..., 0:rot:2], z[..., 1:rot:2]
        first = torch.stack((p * cos - q * sin, q * cos + p * sin), -1).flatten(-2)
    else:
        p, q = z[..., :half], z[..., half:rot]
        first = torch.cat((p * cos - q * sin, q * cos + p * sin), -1)
    return torch.cat((first, z[..., rot:]), -1)


def heads(s):
    """The raw q and k heads as [tokens][heads][dim]."""
    q, k, _ = s["x"].split((s["hq"] * s["dim"], s["hk"] * s["dim"], s["hk"] * s["dim"]), 1)
    return q.reshape(s["tokens"], s["hq"], s["dim"]), k.reshape(s["tokens"], s["hk"], s["dim"])


def plain_qk(s):
    cos, sin = turns(s)

    def one(x, gain):
        if s["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS_HEAD) * gain
        return turned(s, x, cos, sin).reshape(s["tokens"], -1).to(s["out_type"])

    q, k = heads(s)
    return {"q": one(q, s["gq"]), "k": one(k, s["gk"])}


def plain_qk_grad(s):
    cos, sin = turns(s)

    def one(x, gain, dy):
        dz = turned(s, dy.float().view(x.shape), cos, -sin)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS_HEAD)
        n = x * r
        dn = dz * gain
        dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
        return dx.reshape(s["tokens"], -1), (dz * n).sum((0, 1), dtype=torch.float64).float()

    q, k = heads(s)
    (dq, dgq), (dk, dgk) = one(q, s["gq"], s["q"]), one(k, s["gk"], s["k"])
    return {"dx": torch.cat((dq, dk), 1), "dgq": dgq, "dgk": dgk}


PLAIN = {"lora_rows": plain_lora, "lora_batch": plain_lora, "lora_grad": plain_lora_grad, "qk": plain_qk, "qk_grad": plain_qk_grad}
OWN = {"lora_rows": own_lora_rows, "lora_batch": own_lora_batch, "lora_grad": own_lora_grad, "qk": own_qk, "qk_grad": own_qk_grad}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    """Inputs once (of the adapters those that a token uses, at their ranks), outputs once; two operations per product."""
    kind = case["kind"]
    if kind.startswith("qk"):
        tokens, dim = case["tokens"], case["dim"]
        n = tokens * (case["q_heads"] + case["k_heads"]) * dim
        side = 2 if case["bf16"] else 4
        if kind == "qk":
            return {"bytes": n * (4 + side) + tokens * 4 + 8 * dim * case["norm"], "flops": 10 * n}
        return {"bytes": n * (4 + side + 4) + tokens * 4 + 16 * dim, "flops": 20 * n}
    n, k = case["rows"], case["cols"]
    t = case["m"] if kind == "lora_rows" else case["tokens"]
    rank = sum(ranks_of(case)[:used(case)])
    weights = rank * (n + k) * 2
    mean = sum(ranks_of(case)) / case["adapters"]
    if kind == "lora_grad":
        grads = case["adapters"] * case["rank"] * (n + k) * 4
        return {"bytes": weights + grads + t * (k * 2 + n * 2 + k * 8 + 4), "flops": 2 * t * mean * (3 * k + 2 * n)}
    return {"bytes": weights + t * (k * (4 if kind == "lora_rows" else 2) + n * 8 + 4), "flops": 2 * t * mean * (n + k)}


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("qk"):
        return exact_qk(s, case["kind"] == "qk_grad")
    grad = case["kind"] == "lora_grad"
    x = s["x"].double()
    if s["xop"]:
        x = x / torch.linalg.vector_norm(x, dim=1, keepdim=True).square().div(x.shape[1]).add(EPS_ROW).sqrt()
    out = s["base"].double()
    da, db = torch.zeros(s["a"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["b"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["adapters"]):
        at = torch.nonzero(s["ids"] == i).flatten()
        a, b, f = s["a"][i].double(), s["b"][i].double(), s["scale"][i].double()
        if not grad:
            out[at] += f * torch.einsum("tk,rk,nr->tn", x[at], a, b)
        else:
            dy = s["dy"][at].double()
            da[i] = f * torch.einsum("nr,tn,tk->rk", b, dy, x[at])
            db[i] = f * torch.einsum("tn,tk,rk->nr", dy, x[at], a)
            out[at] += f * torch.einsum("tn,nr,rk->tk", dy, b, a)
    return {"dx": out, "da": da, "db": db} if grad else out


def exact_qk(s, grad):
    rot, t = s["rot"], s["tokens"]
    power = torch.arange(rot // 2, device="cuda", dtype=torch.float64) * (2.0 / rot)
    wheel = torch.polar(torch.ones(t, 1, rot // 2, dtype=torch.float64, device="cuda"),
                        (s["pos"].double().view(-1, 1) / THETA ** power).view(t, 1, -1))
    x = s["x"].double().requires_grad_(grad)
    gains = [s["gq"].double().requires_grad_(grad), s["gk"].double().requires_grad_(grad)]
    done, at = [], 0
    for h, gain in zip((s["hq"], s["hk"]), gains):
        z = x[:, at * s["dim"]:(at + h) * s["dim"]].reshape(t, h, s["dim"])
        at += h
        if s["norm"]:
            z = z / (z.square().sum(-1, keepdim=True) / s["dim"] + EPS_HEAD).sqrt() * gain
        pairs = z[..., :rot].unflatten(-1, (rot // 2, 2)) if s["interleaved"] else z[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        spun = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * wheel)
        spun = (spun if s["interleaved"] else spun.transpose(-1, -2)).flatten(-2)
        done.append(torch.cat((spun, z[..., rot:]), -1).reshape(t, -1))
    if not grad:
        return {"q": done[0], "k": done[1]}
    loss = (done[0] * s["q"].double()).sum() + (done[1] * s["k"].double()).sum()
    dx, dgq, dgk = torch.autograd.grad(loss, [x] + gains)
    return {"dx": dx[:, :s["dx"].shape[1]].contiguous(), "dgq": dgq, "dgk": dgk}
