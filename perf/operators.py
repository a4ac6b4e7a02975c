"""What is measured of three groups of operators, and their plain forms:

  lookup      rows of an embedding table by id, scaled, and the table's gradient: the rows of the incoming gradient
              summed by token
  checkpoint  a dense layer's saved activations in 8 bits (int8 or e4m3, one power-of-two scale per 32 columns of a
              row), and the layer's backward pass out of them
  scores      penalties for items a row has had before, biases and masks on a table of scores

`own` decides what run() calls: the plain form in elementary torch operations, or the package's operators."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
GROUP = 32        # columns of a row that share a scale
LOWEST = -110     # smallest exponent of a scale


def listed():
    return [
        # one user's row, as a service that answers one request at a time reads it
        dict(name="lookup_one", kind="lookup", n=1, rows=31882, dim=64, pitch=64, type="float32", ids="int64", scale=1.0, padding=-1, train=False),
        # a training batch's three id lists against the Tmall-shaped table at latdim 128, forward and gradient
        dict(name="lookup_batch", kind="lookup", n=6144, rows=63114, dim=128, pitch=128, type="float32", ids="int64", scale=1.0, padding=-1, train=True),
        # sequences of item ids with a padding id, the row width no multiple of anything, a table that is a view of a wider one
        dict(name="lookup_ragged", kind="lookup", n=5003, rows=30113, dim=100, pitch=103, type="float16", ids="int32", scale=10.0, padding=0, train=True),
        # a long batch of tokens against a large vocabulary, scaled by the root of the width
        dict(name="lookup_tokens", kind="lookup", n=65536, rows=131072, dim=1024, pitch=1024, type="bfloat16", ids="int64", scale=32.0, padding=-1, train=True),
        # activations put away and read back, odd sizes
        dict(name="keep_ragged", kind="keep", n=4097, k=333, type="float16", format="e4m3"),
        # a denoiser's first layer, latdim 128 + 8 -> 32, over the Tmall-shaped graph's users
        dict(name="dense_tmall", kind="dense", n=31882, k=136, m=32, type="float32", format="int8", tanh=True),
        # the hidden layer of a denoiser over a million users
        dict(name="dense_million", kind="dense", n=1000000, k=128, m=64, type="float32", format="e4m3", tanh=True),
        # a wide layer in 16 bits, where the product counts
        dict(name="dense_wide", kind="dense", n=16384, k=1000, m=1000, type="bfloat16", format="int8", tanh=False),
        # one user's scores over all items: the next recommendation of a session
        dict(name="scores_one", kind="scores", rows=1, items=31232, type="float32", history=37, penalties=True, bias=False, states=0, exclude=False),
        # an evaluation batch of 1024 test users, the training items taken out
        dict(name="scores_eval", kind="scores", rows=1024, items=31232, type="float32", history=40, penalties=False, bias=False, states=0, exclude=True),
        # decoding under a grammar: long histories, a state's mask of allowed tokens per row, an odd vocabulary
        dict(name="scores_grammar", kind="scores", rows=64, items=131071, type="float16", history=4096, penalties=True, bias=True, states=17, exclude=False),
        # a large batch with penalties and a bias
        dict(name="scores_large", kind="scores", rows=4096, items=65537, type="bfloat16", history=300, penalties=True, bias=True, states=0, exclude=False),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm, odd as often as not."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    return min(hi, v | 1) if rng.random() < 0.5 else v


def draw(rng):
    kind = rng.choice(["lookup", "lookup", "keep", "dense", "dense", "scores", "scores"])
    t = rng.choice(sorted(TYPES))
    if kind == "lookup":
        dim = _between(rng, 1, 1024)
        n = min(_between(rng, 1, 70000), (64 << 20) // dim)
        rows = min(_between(rng, 1, 200000), (128 << 20) // dim)
        return dict(kind=kind, n=n, rows=rows, dim=dim, pitch=dim + rng.choice([0, 0, 1, 8]), type=t, ids=rng.choice(["int64", "int32"]),
                    scale=rng.choice([1.0, 0.5, round(math.sqrt(dim), 3)]), padding=rng.choice([-1, -1, 0, rows - 1]), train=rng.random() < 0.75)
    if kind == "keep":
        k = _between(rng, 1, 1100)
        return dict(kind=kind, n=min(_between(rng, 1, 300000), (32 << 20) // k), k=k, type=t, format=rng.choice(["int8", "e4m3"]))
    if kind == "dense":
        k, m = _between(rng, 1, 1024), _between(rng, 1, 1024)
        n = min(_between(rng, 1, 500000), (96 << 20) // max(k, m), (16 << 30) // (k * m))
        return dict(kind=kind, n=n, k=k, m=m, type=t, format=rng.choice(["int8", "e4m3"]), tanh=rng.random() < 0.6)
    items = _between(rng, 2, 131072)
    rows = min(_between(rng, 1, 4096), (256 << 20) // items)
    return dict(kind=kind, rows=rows, items=items, type=t, history=min(_between(rng, 1, 4096), (4 << 20) // rows), penalties=rng.random() < 0.8,
                bias=rng.random() < 0.5, states=rng.choice([0, 0, 1, 9]), exclude=rng.random() < 0.3)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _zipf(count, n, g):
    """Ids of which a few come very often (about one over their rank), spread over [0, n) by a fixed stride."""
    rank = (torch.exp(torch.rand(count, generator=g, device=DEV, dtype=torch.float64) * math.log(n + 1.0)) - 1.0).long().clamp_(0, n - 1)
    stride = 7919 if n % 7919 else 1
    return (rank * stride) % n


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 17)
    c, dtype = dict(case), TYPES[case["type"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    s = {"case": c}
    if c["kind"] == "lookup":
        s["table"] = (normal(c["rows"], c["pitch"]) / math.sqrt(c["dim"])).to(dtype)[:, : c["dim"]]
        ids = _zipf(c["n"], c["rows"], g)
        if c["padding"] >= 0:
            ids = torch.where(torch.rand(c["n"], generator=g, device=DEV) < 0.2, torch.full_like(ids, c["padding"]), ids)
        s["ids"] = ids.to(torch.int32 if c["ids"] == "int32" else torch.int64)
        s["d_out"] = (normal(c["n"], c["dim"]) * 0.05).to(dtype) if c["train"] else None
    elif c["kind"] in ("keep", "dense"):
        s["x"] = torch.tanh(normal(c["n"], c["k"]) * torch.exp(normal(c["n"], 1))).to(dtype)
        if c["kind"] == "dense":
            s["y"] = torch.tanh(normal(c["n"], c["m"])).to(dtype) if c["tanh"] else None
            s["d_y"] = (normal(c["n"], c["m"]) * 0.01).to(dtype)
    else:
        B, V = c["rows"], c["items"]
        s["scores"] = (normal(B, V) * 3).to(dtype)
        lengths = (torch.rand(B, generator=g, device=DEV) * (2 * c["history"] + 1)).long()
        lengths[0] = c["history"]
        rowptr = torch.zeros(B + 1, dtype=torch.int64, device=DEV)
        rowptr[1:] = torch.cumsum(lengths, 0)
        s["rowptr"], s["col"] = rowptr.to(torch.int32), _zipf(max(1, int(rowptr[-1])), V, g).to(torch.int32)
        one = lambda lo, hi: torch.rand(B, generator=g, device=DEV) * (hi - lo) + lo  # noqa: E731
        s["repetition"], s["frequency"], s["presence"] = (one(1.0, 1.6), one(0.0, 0.7), one(-0.2, 0.9)) if c["penalties"] else (None, None, None)
        s["bias"] = normal(V) if c["bias"] else None
        s["allowed"] = s["state"] = None
        if c["states"]:
            words = (V + 31) // 32
            bits = torch.rand(c["states"], words, 32, generator=g, device=DEV) < torch.rand(c["states"], 1, 1, generator=g, device=DEV)
            s["allowed"] = (bits.long() << torch.arange(32, device=DEV)).sum(-1).to(torch.int32)       # (the top bit is the sign)
            s["state"] = (torch.rand(B, generator=g, device=DEV) * (c["states"] + 1)).long().clamp_(max=c["states"]).to(torch.int32) - 1
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return _own(state, c)
    if c["kind"] == "lookup":
        return _plain_lookup(state, c)
    if c["kind"] == "keep":
        return _plain_kept(state["x"], c["format"]).to(state["x"].dtype)
    if c["kind"] == "dense":
        return _plain_dense(state, c)
    return _plain_scores(state, c)


def _own(s, c):
    from diffgraph_amd import ops
    if c["kind"] == "lookup":
        pad = c["padding"] if c["padding"] >= 0 else None
        out = {"rows": ops.embedding_lookup(s["table"], s["ids"], c["scale"])}
        if c["train"]:
            out["gradient"] = ops.embedding_grad(s["d_out"], s["ids"], c["rows"], c["scale"], pad)
        return out
    if c["kind"] == "keep":
        return ops.checkpoint8(s["x"], c["format"]).values(s["x"].dtype)
    if c["kind"] == "dense":
        x = ops.checkpoint8(s["x"], c["format"])
        y = ops.checkpoint8(s["y"], c["format"]) if c["tanh"] else None
        d_z, d_w, d_b = ops.checkpoint8_backward(s["d_y"], x, y)
        return {"weight": d_w, "bias": d_b, "inner": d_z} if c["tanh"] else {"weight": d_w, "bias": d_b}
    return ops.adjust_scores(s["scores"], history=(s["rowptr"], s["col"]), repetition=s["repetition"], frequency=s["frequency"],
                             presence=s["presence"], bias=s["bias"], allowed=s["allowed"], allowed_rows=s["state"], exclude=c["exclude"])


def _plain_lookup(s, c):
    ids = s["ids"].long()
    out = {"rows": (s["table"][ids].float() * c["scale"]).to(s["table"].dtype)}
    if c["train"]:
        d = s["d_out"].float() * c["scale"]
        if c["padding"] >= 0:
            d = torch.where((ids == c["padding"])[:, None], torch.zeros_like(d), d)
        out["gradient"] = torch.zeros(c["rows"], c["dim"], device=DEV).index_add_(0, ids, d).to(s["d_out"].dtype)
    return out


def _plain_kept(x, form):
    """The values that x [n, k]'s 8-bit codes stand for, in 32 bits."""
    n, k = x.shape
    groups = -(-k // GROUP)
    v = torch.nn.functional.pad(x.float(), (0, groups * GROUP - k)).view(n, groups, GROUP)
    part, e = torch.frexp(v.abs().amax(-1, keepdim=True))            # largest = part * 2^e, part in [1/2, 1)
    top, bits = (0.875, 9) if form == "e4m3" else (127 / 128, 7)     # largest code = top * 2^bits
    e = torch.where(part > 0, torch.where(part <= top, e - bits, e - bits + 1), torch.full_like(e, LOWEST)).clamp(min=LOWEST)
    q = torch.ldexp(v, -e)
    if form == "e4m3":
        step = torch.ldexp(torch.ones_like(q), torch.frexp(q)[1].clamp(min=-5) - 4)    # three bits behind the leading one; 2^-9 below 2^-6
        q = torch.round(q / step) * step
    else:
        q = torch.round(q)
    return torch.ldexp(q, e).view(n, groups * GROUP)[:, :k]


def _plain_dense(s, c):
    d = s["d_y"].float()
    if c["tanh"]:
        y = _plain_kept(s["y"], c["format"])
        d = d * (1 - y * y)
    w = d.t() @ _plain_kept(s["x"], c["format"])
    out = {"weight": w.to(s["d_y"].dtype), "bias": d.sum(0).to(s["d_y"].dtype)}
    if c["tanh"]:
        out["inner"] = d.to(s["d_y"].dtype)
    return out


def _plain_scores(s, c):
    B, V = s["scores"].shape
    v = s["scores"].float()
    row = torch.repeat_interleave(torch.arange(B, device=DEV), (s["rowptr"][1:] - s["rowptr"][:-1]).long(), output_size=s["col"].numel()) \
        if int(c["history"]) else None
    count = torch.zeros(B * V, device=DEV)
    if row is not None:
        count.index_add_(0, row * V + s["col"].long(), torch.ones(row.numel(), device=DEV))
    count = count.view(B, V)
    had = count > 0
    if c["penalties"]:
        r = s["repetition"][:, None]
        v = torch.where(had, torch.where(v > 0, v / r, v * r) - (s["frequency"][:, None] * count + s["presence"][:, None]), v)
    if s["bias"] is not None:
        v = v + s["bias"]
    if s["allowed"] is not None:
        bits = ((s["allowed"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).view(c["states"], -1)[:, :V].bool()
        ok = bits[s["state"].long().clamp(min=0)] | (s["state"] < 0)[:, None]
        v = torch.where(ok, v, torch.full_like(v, -math.inf))
    if c["exclude"]:
        v = torch.where(had, torch.full_like(v, -math.inf), v)
    return v.to(s["scores"].dtype)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c, z = case, SIZE[case["type"]]
    if c["kind"] == "lookup":
        i = 8 if c["ids"] == "int64" else 4
        seen = min(c["n"], c["rows"])
        b, f = c["n"] * i + seen * c["dim"] * z + c["n"] * c["dim"] * z, c["n"] * c["dim"]
        if c["train"]:
            b, f = b + c["n"] * i + c["n"] * c["dim"] * z + c["rows"] * c["dim"] * z, 3 * f
        return {"bytes": b, "flops": f}
    if c["kind"] == "keep":
        return {"bytes": 2 * c["n"] * c["k"] * z + 2 * c["n"] * (c["k"] + -(-c["k"] // GROUP)), "flops": 3 * c["n"] * c["k"]}
    if c["kind"] == "dense":
        n, k, m = c["n"], c["k"], c["m"]
        codes = lambda w: 2 * n * (w + -(-w // GROUP))  # noqa: E731  (written, and read by the backward pass)
        b = n * k * z + codes(k) + n * m * z + m * k * z + m * z + (n * m * z * 2 + codes(m) if c["tanh"] else 0)
        return {"bytes": b, "flops": 2 * n * k * m + 4 * n * m}
    B, V = c["rows"], c["items"]
    b = 2 * B * V * z + B * c["history"] * 4 + (4 * V if c["bias"] else 0) + c["states"] * V // 8
    return {"bytes": b, "flops": 4 * B * V}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), dict(case)
    if c["kind"] == "lookup":
        ids = s["ids"].long()
        out = {"rows": torch.index_select(s["table"].double(), 0, ids).mul_(c["scale"])}
        if c["train"]:
            keep = torch.nonzero(ids != c["padding"]).flatten() if c["padding"] >= 0 else torch.arange(ids.numel(), device=DEV)
            g = torch.zeros(c["rows"], c["dim"], dtype=torch.float64, device=DEV)
            g.index_put_((ids[keep],), s["d_out"].double()[keep], accumulate=True)
            out["gradient"] = g.mul_(c["scale"])
        return out
    if c["kind"] == "keep":
        return _exact_kept(s["x"], c["format"])
    if c["kind"] == "dense":
        d = s["d_y"].double()
        if c["tanh"]:
            d = d - d * _exact_kept(s["y"], c["format"]).square()
        out = {"weight": torch.mm(d.t().contiguous(), _exact_kept(s["x"], c["format"])), "bias": torch.mv(d.t().contiguous(), torch.ones(c["n"], dtype=torch.float64, device=DEV))}
        if c["tanh"]:
            out["inner"] = d
        return out
    B, V = c["rows"], c["items"]
    v = s["scores"].double().flatten()
    owner = torch.searchsorted(s["rowptr"][1:].long(), torch.arange(int(s["rowptr"][-1]), device=DEV), right=True)
    place, times = torch.unique(owner * V + s["col"][: owner.numel()].long(), return_counts=True)
    at, row = v[place], place // V
    if c["penalties"]:
        r = s["repetition"].double()[row]
        at = at * torch.where(at > 0, 1 / r, r) - s["presence"].double()[row] - times * s["frequency"].double()[row]
    v[place] = at
    v = v.view(B, V)
    if s["bias"] is not None:
        v += s["bias"].double()
    if s["allowed"] is not None:
        item = torch.arange(V, device=DEV)
        for b in range(B):
            if int(s["state"][b]) >= 0:
                word = s["allowed"][int(s["state"][b])].long()[item // 32]
                v[b, ((word >> (item % 32)) & 1) == 0] = -math.inf
    if c["exclude"]:
        v.view(-1)[place] = -math.inf
    return v


def _exact_kept(x, form):
    """The same values from the definition: the smallest power of two that brings the group's largest within the codes'
    range, and the nearest code, found in a list of all of them (a tie goes to the even one)."""
    n, k = x.shape
    v = x.double()
    out = torch.empty_like(v)
    if form == "e4m3":
        whole = torch.arange(127, dtype=torch.float64, device=DEV)       # codes 0 .. 126 stand for these, code 127 for no number
        code = torch.where(whole < 8, whole * 2.0 ** -9, (8 + whole % 8) * torch.exp2(torch.floor(whole / 8) - 10))
    else:
        code = torch.arange(128, dtype=torch.float64, device=DEV)
    middle = (code[1:] + code[:-1]) / 2
    exponents = torch.arange(LOWEST, 128, device=DEV, dtype=torch.float64)
    for at in range(0, k, GROUP):
        part = v[:, at: at + GROUP]
        big = part.abs().amax(1)
        e = torch.searchsorted(code[-1] * torch.exp2(exponents), big)    # the first power that is large enough
        unit = torch.exp2(exponents[e])[:, None]
        q = part.abs() / unit
        below = torch.searchsorted(middle, q, right=False)
        above = torch.searchsorted(middle, q, right=True)                # differs from `below` on a tie alone
        out[:, at: at + GROUP] = torch.sign(part) * code[torch.where(below % 2 == 0, below, above)] * unit
    return out
