"""The operators in the framework's own paths, one after the other as they are used: denoisers that keep their
activations in 8 bits (Denoise(act_ckpt=...), args.act_ckpt), the wide model's batch rows by embedding lookup, its
evaluation and evaluate.recommend over adjusted scores."""
import copy
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import diffgraph_amd as dg
from diffgraph_amd import DiffGraphHipError, data as dgdata, evaluate as ev, ops
from diffgraph_amd.model_rec import DEFAULT_ARGS
from tests.helpers import GRAD_TOL, assert_close_to_max, assert_rows_close

gpu = pytest.mark.gpu
DEV = "cuda"


def denoiser(fmt, latdim=96, dims=(128, 40), emb=10, seed=0):
    torch.manual_seed(seed)
    out = list(dims) + [latdim]
    return dg.Denoise(out[::-1], out, emb, norm=True, act_ckpt=fmt).to(DEV)


def dense_layers(dn):
    return [(l, True) for l in dn.in_layers] + [(l, i != len(dn.out_layers) - 1) for i, l in enumerate(dn.out_layers)]


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n", [1, 77, 1500])
def test_denoiser_forward_is_unchanged_and_gradients_follow_the_kept_values(n, fmt):
    dn, plain = denoiser(fmt), denoiser(None)
    plain.load_state_dict(dn.state_dict())
    x = torch.randn(n, 96, device=DEV, requires_grad=True)
    t = torch.randint(0, 200, (n,), device=DEV)
    keep = torch.rand(n, 96, device=DEV) < 0.5
    out = dn(x, t, True, keep)
    assert torch.equal(out, plain(x.detach(), t, True, keep))                   # the same forward values
    with torch.no_grad():
        assert torch.equal(out, dn(x, t, True, keep))
    d_out = torch.randn_like(out)
    out.backward(d_out)
    # the backward pass in 64 bits, from the values that the codes of the very same activations stand for
    acts = []
    with torch.no_grad():
        e = torch.arange(5, device=DEV, dtype=torch.float32)
        f = t[:, None].float() * torch.exp(-math.log(10000) * e / 5)[None]
        emb = ops.linear_fwd(torch.cat([torch.cos(f), torch.sin(f)], 1).contiguous(), dn.emb_layer.weight, dn.emb_layer.bias)
        h = torch.cat([torch.nn.functional.normalize(x) * (keep.float() * 2.0), emb], 1)
        for layer, tanh in dense_layers(dn):
            kept = ops.checkpoint8(h, fmt).values().double()
            h = ops.linear_fwd(h.contiguous(), layer.weight, layer.bias)
            h = torch.tanh(h) if tanh else h
            acts.append((kept, ops.checkpoint8(h, fmt).values().double() if tanh else None))
        assert torch.equal(h, out)
    d = d_out.double()
    for (layer, tanh), (xv, yv) in reversed(list(zip(dense_layers(dn), acts))):
        d = d * (1 - yv * yv) if tanh else d
        assert_close_to_max(layer.weight.grad, d.t() @ xv, GRAD_TOL, "d weight")
        assert_close_to_max(layer.bias.grad, d.sum(0), GRAD_TOL, "d bias")
        d = d @ layer.weight.detach().double()
    xd = x.detach().double().requires_grad_()
    (torch.nn.functional.normalize(xd) * (keep.double() * 2.0)).backward(d[:, :96])
    # (through normalize, whose backward takes g's part along the row away: what is left may be a tenth of g)
    assert_rows_close(x.grad, xd.grad, rtol=1e-4, what="d x")
    # and they stay within what the rounding of the codes explains: the last layer's weight, whose d_z is the same
    x2 = x.detach().requires_grad_()
    plain(x2, t, True, keep).backward(d_out)
    last, ref = dn.out_layers[-1].weight.grad.double(), plain.out_layers[-1].weight.grad.double()
    half = 2.0 ** -7 if fmt == "int8" else 2.0 ** -4                  # of |h| <= 1: half a scale of at most 2^-6; half a step
    bound = half * d_out.double().abs().sum(0)[:, None] + GRAD_TOL * ref.abs().max()
    assert bool(((last - ref).abs() <= bound).all())


def code_error(v, fmt):
    """How far a code's value may be from v [n, k], by the definition: half a scale in int8, half a step of three bits in
    e4m3 (below its normal numbers: 2^-10 of the scale).  The scale is at most the power of two above largest / Q."""
    n, k = v.shape
    q = 127.0 if fmt == "int8" else 448.0
    top = torch.nn.functional.pad(v.abs(), (0, -k % 32)).view(n, -1, 32).amax(2)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-30) / q)) + 1).repeat_interleave(32, 1)[:, :k]
    return scale / 2 if fmt == "int8" else torch.maximum(v.abs() * 2.0 ** -4, scale * 2.0 ** -10)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n,gain", [(1, 1.0), (77, 1.0), (1500, 1.0), (1, 4.0), (77, 4.0)])
def test_every_gradient_stays_within_what_the_codes_explain(n, gain, fmt):
    """The denoiser that keeps 8 bits against the one that keeps everything: inputs, weights and biases of every layer.  With
    X and Y the errors of the codes of a layer's input x and output y, and E that of the gradient d that reaches it:
    tanh' = 1 - y^2 is off by T <= 2 |y| Y + Y^2, d_z by Z <= E tanh' + |d| T + E T (Z = E without tanh), d_w by
    Z^T (|x| + X) + |d_z|^T X, d_b by the column sums of Z, and the layer before gets E = Z |W|.  Beside these, sums of n (or
    m) products in fp32 in either pass.  gain 4: most units beyond |z| = 2."""
    U = 2.0 ** -24
    dn, plain = denoiser(fmt, seed=2), denoiser(None)
    with torch.no_grad():
        for layer, tanh in dense_layers(dn):
            if tanh:
                layer.weight.mul_(gain)
    plain.load_state_dict(dn.state_dict())
    g = torch.Generator().manual_seed(n)
    x1 = torch.randn(n, 96, generator=g).to(DEV).requires_grad_()
    x2 = x1.detach().clone().requires_grad_()
    t, keep = torch.randint(0, 200, (n,), generator=g).to(DEV), (torch.rand(n, 96, generator=g) < 0.5).to(DEV)
    d_out = torch.randn(n, 96, generator=g).to(DEV)
    dn(x1, t, True, keep).backward(d_out)
    plain(x2, t, True, keep).backward(d_out)
    layers, acts = list(zip(dense_layers(dn), dense_layers(plain))), []
    with torch.no_grad():
        e = torch.arange(5, device=DEV, dtype=torch.float32)
        f = t[:, None].float() * torch.exp(-math.log(10000) * e / 5)[None]
        emb = ops.linear_fwd(torch.cat([torch.cos(f), torch.sin(f)], 1).contiguous(), dn.emb_layer.weight, dn.emb_layer.bias)
        h = torch.cat([torch.nn.functional.normalize(x1) * (keep.float() * 2.0), emb], 1)
        for (layer, tanh), _ in layers:
            x = h.double()
            h = ops.linear_fwd(h.contiguous(), layer.weight, layer.bias)
            h = torch.tanh(h) if tanh else h
            acts.append((x, h.double()))
    d, E, saturated, close = d_out.double(), torch.zeros(n, 96, dtype=torch.float64, device=DEV), 0, []
    for ((layer, tanh), (ref, _)), (x, y) in reversed(list(zip(layers, acts))):
        X = code_error(x, fmt)
        if tanh:
            Y, slope = code_error(y, fmt), 1 - y * y
            T = 2 * y.abs() * Y + Y * Y
            Z, d = E * slope + d.abs() * T + E * T + 8 * U * (d.abs() + E), d * slope
            saturated += int((y.abs() > 1 - 2.0 ** -7).sum())
        else:
            Z = E
        sums = (n + 1000) * 8 * U
        w_off = Z.t() @ (x.abs() + X) + d.abs().t() @ X + sums * (d.abs() + Z).t() @ (x.abs() + X)
        b_off = Z.sum(0) + sums * (d.abs() + Z).sum(0)
        assert bool(((layer.weight.grad.double() - ref.weight.grad.double()).abs() <= w_off).all()), (layer, "d weight")
        assert bool(((layer.bias.grad.double() - ref.bias.grad.double()).abs() <= b_off).all()), (layer, "d bias")
        close.append(float((w_off < 0.5 * ref.weight.grad.double().abs()).double().mean()))
        W = layer.weight.detach().double()
        E, d = (Z + (layer.weight.shape[0] + 10) * 8 * U * (d.abs() + Z)) @ W.abs(), d @ W
    # through the kept part of the rows and normalize: (g - u (u . g)) / |x|, u = x / |x|
    g, g_off = d[:, :96] * keep.double() * 2, E[:, :96] * keep.double() * 2 + 1e-5 * d[:, :96].abs()
    norm = x1.detach().double().norm(dim=1, keepdim=True)
    u = x1.detach().double() / norm
    off = (g_off + u.abs() * (u.abs() * g_off).sum(1, keepdim=True) + 1e-5 * (g.abs() + u.abs() * (u * g).abs().sum(1, keepdim=True))) / norm
    assert bool(((x1.grad.double() - x2.grad.double()).abs() <= off).all()), "d x"
    assert bool(x1.grad.any()) and bool(x1.grad.isfinite().all())
    assert (saturated > 0) == (gain > 1) or n > 1
    if n == 1 and gain == 1 and fmt == "int8":      # one row, where nothing cancels: the bounds of the last two layers say something
        assert min(close[:2]) > 0.5, close


@gpu
@pytest.mark.parametrize("fmt,flat", [("int8", 1 - 2.0 ** -7), ("e4m3", 1 - 2.0 ** -5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_the_slope_of_saturated_units(dtype, fmt, flat):
    """tanh' out of the codes, beside a unit at 1: within 2 |y| Y + Y^2 of the true one, and exactly 0 where y is kept as 1, from
    half a step below 1 on; not 0 before."""
    z = torch.cat([torch.linspace(-6, 6, 31 * 40, dtype=torch.float64).view(40, 31), torch.full((40, 1), 9.0, dtype=torch.float64)], 1)
    y = torch.tanh(z).to(dtype).to(DEV)
    x = ops.checkpoint8(torch.ones(40, 3, dtype=dtype, device=DEV), fmt)
    d_z, _, d_b = ops.checkpoint8_backward(torch.ones(40, 32, dtype=dtype, device=DEV), x, ops.checkpoint8(y, fmt))
    v = y.double()
    off = 2.0 ** -7 if fmt == "int8" else torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -18)).clamp(max=2.0 ** -5)
    bound = 2 * v.abs() * off + off * off
    assert bool(((d_z.double() - (1 - v * v)).abs() <= bound + torch.finfo(dtype).eps / 2 + 2.0 ** -23).all())
    assert not bool(d_z[v.abs() > flat].any()) and bool((d_z[v.abs() < flat] > 0).all())
    assert bool((d_b > 0).any())


@gpu
def test_kept_bytes():
    """What autograd holds between the passes, apart from the weights: a quarter of the fp32 activations and a little."""
    n, held = 4096, {}
    for fmt in (None, "int8"):
        dn = denoiser(fmt, dims=(256, 128))
        weights = {p.data_ptr() for p in dn.parameters()}
        seen = {}

        def pack(v):
            if v.data_ptr() not in weights:
                seen[v.data_ptr()] = v.numel() * v.element_size()
            return v
        x, t = torch.randn(n, 96, device=DEV), torch.randint(0, 200, (n,), device=DEV)
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v):
            out = dn(x, t, False)
        held[fmt] = sum(seen.values())
        del out
    # per row: 106 + 128 + 256 + 128 inner columns... each a byte and its scale's share, the time embedding's 10 floats beside them
    cols = 96 + 10 + 128 + 256 + 128
    assert held["int8"] <= n * (cols * 1.2 + 2 * 10 * 4 + 64) < 0.45 * held[None]


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_backward_against_differences(fmt):
    """One row, its bias chosen so that tanh(z) is a code's value: d_w is then the gradient of sum c tanh(x^ w^T + b)."""
    torch.manual_seed(4)
    m, k = 9, 40
    x = ops.checkpoint8(torch.randn(1, k, device=DEV), fmt)
    y = ops.checkpoint8(torch.tanh(torch.randn(1, m, device=DEV)) * 0.9, fmt)
    xv, yv = x.values().double(), y.values().double()
    c = torch.randn(1, m, device=DEV)
    _, d_w, d_b = ops.checkpoint8_backward(c, x, y)
    w = torch.randn(m, k, dtype=torch.float64, device=DEV)
    b = torch.atanh(yv) - xv @ w.t()
    loss = lambda w, b: (c.double() * torch.tanh(xv @ w.t() + b)).sum()  # noqa: E731
    h = 1e-5
    for o, i in ((0, 0), (8, 39), (4, 31), (5, 32)):
        e = torch.zeros_like(w)
        e[o, i] = h
        diff = float(loss(w + e, b) - loss(w - e, b)) / (2 * h)
        # central difference: (h x)^2 / 6 of the third derivative (at most 2) and 64-bit rounding / h; the kernel: three roundings
        tol = abs(float(c[0, o])) * (abs(float(xv[0, i])) ** 3 * h * h + 1e-10) + 4 * 2.0 ** -24 * abs(diff) + 1e-10
        assert abs(float(d_w[o, i]) - diff) <= tol
        e = torch.zeros_like(b)
        e[0, o] = h
        diff = float(loss(w, b + e) - loss(w, b - e)) / (2 * h)
        assert abs(float(d_b[o]) - diff) <= abs(float(c[0, o])) * (h * h + 1e-10) + 4 * 2.0 ** -24 * abs(diff) + 1e-10


def test_a_denoiser_pickled_before_it_kept_anything():
    """A whole pickled module of a version without act_ckpt (as the reference saves its models) keeps nothing in 8 bits."""
    import pickle
    d = dg.Denoise([96, 40], [40, 96], 8)
    del d.__dict__["act_ckpt"]
    assert pickle.loads(pickle.dumps(d)).act_ckpt is None


def _on_the_cpu(monkeypatch):
    """The operators that a dense layer with kept activations calls, by plain stand-ins that keep every bit."""
    from diffgraph_amd import diffusion
    kept = {}

    def keep(x, fmt):
        ck = ops.Checkpoint8(torch.full((x.numel(),), len(kept), dtype=torch.uint8), tuple(x.shape), fmt)
        kept[len(kept)] = x.detach().clone()
        return ck

    def backward(d_y, x, y=None):
        d_z = d_y if y is None else d_y * (1 - kept[int(y.data[0])] ** 2)
        return d_z, d_z.t() @ kept[int(x.data[0])], d_z.sum(0)
    monkeypatch.setattr(diffusion.ops, "checkpoint8", keep)
    monkeypatch.setattr(diffusion.ops, "checkpoint8_backward", backward)
    monkeypatch.setattr(diffusion.ops, "linear_fwd", lambda x, w, b: torch.nn.functional.linear(x, w, b))
    return diffusion._Dense8Fn


def test_no_gradient_is_made_for_the_codes(monkeypatch):
    """The codes are a second output of a layer with tanh: its backward pass gets none for them, where autograd would fill a
    tensor of their size with zeros."""
    fn = _on_the_cpu(monkeypatch)
    got, inner = [], fn.backward

    def spy(ctx, dy, codes):
        got.append((dy is None, codes is None))
        return inner(ctx, dy, codes)
    monkeypatch.setattr(fn, "backward", staticmethod(spy))
    x, w, b = torch.randn(5, 6, requires_grad=True), torch.randn(4, 6, requires_grad=True), torch.randn(4, requires_grad=True)
    w2, b2 = torch.randn(3, 4, requires_grad=True), torch.randn(3, requires_grad=True)
    h, kept = fn.apply(x, None, w, b, "int8", True)
    y, none = fn.apply(h, kept, w2, b2, "int8", False)
    assert kept.dtype == torch.uint8 and not kept.requires_grad and none is None
    d = torch.randn_like(y)
    grads = torch.autograd.grad(y, (x, w, b, w2, b2), d)
    want = torch.autograd.grad(torch.tanh(x @ w.t() + b) @ w2.t() + b2, (x, w, b, w2, b2), d)
    for a, c in zip(grads, want):
        torch.testing.assert_close(a, c)
    assert got == [(False, True), (False, True)]


def test_a_layer_that_no_gradient_reaches(monkeypatch):
    """Its output goes into a function that passes none on."""
    class Stop(torch.autograd.Function):
        @staticmethod
        def forward(ctx, h, x):
            return h + x

        @staticmethod
        def backward(ctx, d):
            return None, d
    fn = _on_the_cpu(monkeypatch)
    x, w, b = torch.randn(5, 4, requires_grad=True), torch.randn(4, 4, requires_grad=True), torch.randn(4, requires_grad=True)
    h, _ = fn.apply(x, None, w, b, "e4m3", True)
    Stop.apply(h, x).sum().backward()
    assert torch.equal(x.grad, torch.ones(5, 4)) and (w.grad is None or not bool(w.grad.any()))


def test_denoiser_refuses_another_format():
    with pytest.raises(ValueError, match="act_ckpt"):
        dg.Denoise([96, 40], [40, 96], 8, act_ckpt="int4")


@gpu
@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("fmt,latdim", [("int8", 64), ("e4m3", 128)])
def test_coach_epochs_with_kept_activations_then_recommendations(fmt, latdim, use_graph):
    """A run of all three together: training steps whose denoisers keep 8 bits (at latdim 128 the batch rows by lookup and
    gradient by token), eagerly and recorded; evaluation; recommendations out of the trained tables."""
    from diffgraph_amd.train import Coach
    from tests.test_gpu_train import _handler
    args = copy.copy(DEFAULT_ARGS)
    args.batch, args.dims, args.d_emb_size, args.epoch, args.latdim, args.act_ckpt = 64, "[128, 32]", 10, 2, latdim, fmt
    torch.manual_seed(5)
    handler = _handler()
    c = Coach(handler, args, device=DEV, use_graph=use_graph, seed=3)
    lines = []
    res = c.run(log=lines.append)
    assert c.model.usr_denoiser.act_ckpt == fmt and not c.model.usr_denoiser.fused
    assert len(lines) == 4 and all("nan" not in ln.lower() for ln in lines), lines
    assert 0.0 <= res["Recall"] <= 1.0
    with torch.no_grad():
        pu, pi = c.model.predict()
    data = handler.tst_data
    val, idx = ev.recommend(pu, pi, data.test_users_dev, data, 5)
    v2, i2 = ev.all_rank_topk(pu, pi, data.test_users_dev, data, 5)
    kept = torch.isfinite(val)
    np.testing.assert_allclose(val[kept].cpu().numpy(), v2[kept].cpu().numpy(), rtol=2e-5, atol=2e-5 * float(v2[kept].abs().max()))
    assert i2.shape == idx.shape


@gpu
def test_recorded_and_eager_steps_agree_with_kept_activations():
    """The same draws, the same steps: a recorded training step with 8-bit activations gives the eager step's bits."""
    from diffgraph_amd.train import Coach
    from tests.test_gpu_train import _handler
    got = []
    for use_graph in (False, True):
        args = copy.copy(DEFAULT_ARGS)
        args.batch, args.dims, args.epoch, args.latdim, args.act_ckpt = 64, "[48]", 1, 128, "int8"
        torch.manual_seed(6)
        handler = _handler()
        c = Coach(handler, args, device=DEV, use_graph=use_graph, seed=3)
        c.prepareModel()
        # (the warm-up steps before a recording take draws beyond the step's own and give them back: a few more than steps)
        n, steps = c.model.n_user + c.model.n_item, c._n_batches + 4
        g = torch.Generator().manual_seed(9)
        c.set_draws(torch.randint(0, 200, (steps, n), generator=g), torch.randn(steps, n, 128, generator=g),
                    (torch.rand(steps, n, 128, generator=g) < 0.5).to(torch.uint8))
        c.trainEpoch()
        got.append([p.detach().clone() for p in c.model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ---- wide model, evaluation, recommendations ------------------------------------------------------------------------
def interactions(nu, ni, seed=3):
    import scipy.sparse as sp
    trn_u, trn_i = dgdata.synth_interactions(nu, ni, nu * 20, seed)
    rng = np.random.default_rng(5)
    coo = lambda u, i: sp.coo_matrix((np.ones(len(u), np.float32), (u, i)), shape=(nu, ni))  # noqa: E731
    data = ev.AllRankTestData(coo(np.arange(nu, dtype=np.int32), rng.integers(0, ni, nu).astype(np.int32)), coo(trn_u, trn_i))
    had = torch.zeros(nu, ni, dtype=torch.bool)
    had[torch.from_numpy(trn_u).long(), torch.from_numpy(trn_i).long()] = True
    return data, had


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("width", [64, 100])
def test_recommend(width, dtype):
    nu, ni, k = 70, 900, 20
    data, had = interactions(nu, ni)
    g = torch.Generator().manual_seed(1)
    usr, itm = torch.randn(nu, width, generator=g).to(dtype).to(DEV), torch.randn(ni, width, generator=g).to(dtype).to(DEV)
    users = torch.tensor([3, 69, 3, 0, 41], device=DEV)
    scores = torch.mm(usr[users], itm.t())                        # the operators' part starts here
    rep = torch.tensor([1.0, 1.5, 2.0, 1.2, 0.9], device=DEV)
    bias = torch.randn(ni, generator=g).to(DEV)
    words = torch.randint(-2 ** 31, 2 ** 31, (3, (ni + 31) // 32), generator=g).to(torch.int32).to(DEV)
    which = torch.tensor([0, -1, 2, 1, 1], dtype=torch.int32, device=DEV)
    stays = ((words.cpu().long()[:, torch.arange(ni) // 32] >> (torch.arange(ni) % 32)) & 1).bool()
    for exclude, batch in ((True, 1024), (False, 2)):
        val, idx = ev.recommend(usr, itm, users, data, k, exclude=exclude, repetition=rep, presence=0.1, bias=bias, allowed=words,
                                allowed_rows=which, batch=batch)
        assert val.dtype == dtype and idx.dtype == torch.int32 and val.shape == idx.shape == (5, k)
        s, h = scores.cpu().double(), had[users.cpu()]
        r = rep.cpu().double()[:, None]
        s = torch.where(h, torch.where(s > 0, s / r, s * r) - 0.1, s) + bias.cpu().double()
        out = ~(stays[which.cpu().long().clamp(min=0)] | (which.cpu() < 0)[:, None])
        s[out | h if exclude else out] = -math.inf
        want = s.topk(k).values
        # each score: four fp32 roundings of values below size, one to the type; a product of another shape may differ in
        # its last bit itself (2 eps of its value)
        size = s.masked_fill(torch.isinf(s), 0).abs().max() + 4
        tol = 8 * 2.0 ** -24 * size + 3 * torch.finfo(dtype).eps * size
        assert torch.equal(torch.isinf(val).cpu(), torch.isinf(want))
        fin = torch.isfinite(want)
        assert bool(((val.cpu().double() - want).abs()[fin] <= tol).all())
        at = s.gather(1, idx.cpu().long())
        assert bool(((at - val.cpu().double()).abs()[fin] <= tol).all())
    one = ev.recommend(usr, itm, users[:1], data, 1)
    assert one[0].shape == (1, 1) and not bool(had[3, int(one[1])])
    assert ev.recommend(usr, itm, users[:0], data, 3)[0].shape == (0, 3)
    odd = ev.recommend(usr, itm, torch.tensor([nu, 2], device=DEV), data, 3)
    assert bool(odd[0][0].isnan().all()) and bool(odd[0][1].isfinite().all())
    leaves = ev.recommend(usr.clone().requires_grad_(), itm, users[:1], data, 1, bias=torch.zeros(ni, device=DEV, requires_grad=True))
    assert torch.equal(leaves[1], one[1]) and not leaves[0].requires_grad


@gpu
def test_recommend_refusals():
    data, _ = interactions(30, 50)
    usr, itm, users = torch.zeros(30, 8, device=DEV), torch.zeros(50, 8, device=DEV), torch.tensor([1, 2], device=DEV)
    for args, kw, what in (((usr[:29], itm, users), {}, "match"), ((usr, itm.half(), users), {}, "one type"), ((usr, itm, users.int()), {}, "users"),
                           ((usr, itm, users), dict(topk=0), "topk"), ((usr, itm, users), dict(topk=51), "topk"), ((usr, itm, users), dict(batch=0), "batch"),
                           ((usr, itm, users), dict(repetition=torch.ones(3, device=DEV)), "repetition"),
                           ((usr, itm, users), dict(bias=torch.ones(2, 50, device=DEV)), "bias"),
                           ((usr, itm, users), dict(allowed=torch.zeros(5, 2, dtype=torch.int32, device=DEV)), "allowed")):
        with pytest.raises(DiffGraphHipError, match=what):
            ev.recommend(args[0], args[1], args[2], data, **kw)


@gpu
def test_wide_loss_with_rows_named_many_times():
    """wide.cal_loss: the gradient of a batch that names rows many times is the sum over the batch."""
    from diffgraph_amd import wide
    wl = dgdata.rec_workload("tiny")
    nu, ni = wl.n_user, wl.n_item
    graphs = [dg.CSRGraph.from_bipartite(u, i, nu, ni) for (u, i) in [wl.target] + wl.behaviours]
    handler = SimpleNamespace(userNum=nu, itemNum=ni, target_adj=graphs[0], behavior_mats=graphs[1:])
    args = SimpleNamespace(**{**vars(DEFAULT_ARGS), "latdim": 80, "batch": 300, "act_ckpt": "int8"})
    torch.manual_seed(1)
    m = dg.rec.HGDM(handler, args).eval()
    n = 300
    ids = [torch.randint(0, hi, (n,), device=DEV) for hi in (3, 2, ni)]
    draws = (torch.randint(0, 200, (nu,), device=DEV), torch.randn(nu, 80, device=DEV), torch.randint(0, 200, (ni,), device=DEV),
             torch.randn(ni, 80, device=DEV))
    grads = []
    for lookup in (wide.embedding, lambda table, i: table[i]):         # the kernels, and torch's own indexing
        old, wide.embedding = wide.embedding, lookup
        try:
            m.zero_grad()
            wide.cal_loss(m, *ids, *draws)[0].backward()
        finally:
            wide.embedding = old
        grads.append(m.embedding_table.grad.clone())
    assert_rows_close(grads[0], grads[1], rtol=1e-5, what="table gradient")


def test_wide_evaluation_refuses_users_that_are_not_there():
    """As the narrow tables' evaluation does (and torch's index check did): before anything touches the GPU."""
    from diffgraph_amd import wide
    usr, itm = torch.zeros(6, 80), torch.zeros(9, 80)
    rowptr, col = torch.zeros(7, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for users in ([6], [0, -1], [5, 6, 1], [-7]):
        with pytest.raises(DiffGraphHipError, match="users must lie in"):
            wide.all_rank_topk(usr, itm, torch.tensor(users), rowptr, col, 3)
    with pytest.raises(DiffGraphHipError, match="users must lie in"):      # a user without a line in the interactions
        wide.all_rank_topk(usr, itm, torch.tensor([5]), rowptr[:6], col, 3)


@gpu
def test_wide_evaluation_refuses_users_that_are_not_there_through_its_entry_point():
    data, _ = interactions(30, 50)
    usr, itm = torch.randn(30, 80, device=DEV), torch.randn(50, 80, device=DEV)
    for users in ([30], [3, -1]):
        for width in (64, 80):
            with pytest.raises(DiffGraphHipError, match="users must lie in"):
                ev.all_rank_topk(usr[:, :width].contiguous(), itm[:, :width].contiguous(), torch.tensor(users, device=DEV), data, 5)
    val, idx = ev.all_rank_topk(usr, itm, torch.tensor([29, 0], device=DEV), data, 5)
    assert bool(val.isfinite().all()) and idx.shape == (2, 5)


def wide_model(latdim, batch, **kw):
    wl = dgdata.rec_workload("tiny")
    nu, ni = wl.n_user, wl.n_item
    graphs = [dg.CSRGraph.from_bipartite(u, i, nu, ni) for (u, i) in [wl.target] + wl.behaviours]
    handler = SimpleNamespace(userNum=nu, itemNum=ni, target_adj=graphs[0], behavior_mats=graphs[1:])
    torch.manual_seed(1)
    m = dg.rec.HGDM(handler, SimpleNamespace(**{**vars(DEFAULT_ARGS), "latdim": latdim, "batch": batch, **kw})).eval()
    draws = (torch.randint(0, 200, (nu,), device=DEV), torch.randn(nu, latdim, device=DEV), torch.randint(0, 200, (ni,), device=DEV),
             torch.randn(ni, latdim, device=DEV))
    return m, nu, ni, draws


@gpu
def test_wide_loss_counts_negative_ids_from_the_end():
    """As torch's indexing does: the loss and its gradient, bit for bit."""
    from diffgraph_amd import wide
    m, nu, ni, draws = wide_model(80, 50)
    ids = [torch.randint(0, hi, (50,), device=DEV) for hi in (nu, ni, ni)]
    got = []
    for turned in ([], [0], [1], [2], [0, 1, 2]):
        m.zero_grad()
        part = [v - hi if k in turned else v for k, (v, hi) in enumerate(zip(ids, (nu, ni, ni)))]
        loss = wide.cal_loss(m, *part, *draws)
        loss[0].backward()
        got.append((loss.detach().clone(), m.embedding_table.grad.clone()))
    assert bool(got[0][0].isfinite().all())
    for loss, grad in got[1:]:
        assert torch.equal(loss, got[0][0]) and torch.equal(grad, got[0][1])


def test_ids_outside_a_table_raise():
    """(On the GPU by torch's own assertion there, at the next synchronisation.)"""
    from diffgraph_amd import wide
    rows = torch.arange(9)
    assert wide.row_ids(torch.tensor([0, 6, -1, -7]), rows[:7]).tolist() == [0, 6, 6, 0]
    assert wide.row_ids(torch.tensor([3], dtype=torch.int32), rows[:7]).dtype == torch.int64
    for bad in (7, -8, 1 << 40):
        with pytest.raises(IndexError):
            wide.row_ids(torch.tensor([0, bad]), rows[:7])


def _wide_tables(nu=40, ni=300, width=80, dtype=torch.float32):
    data, had = interactions(nu, ni)
    g = torch.Generator().manual_seed(2)
    return data, had.to(DEV), torch.randn(nu, width, generator=g).to(dtype).to(DEV), torch.randn(ni, width, generator=g).to(dtype).to(DEV)


@gpu
@pytest.mark.parametrize("rowptr_type,col_type", [(torch.int64, torch.int64), (torch.int64, torch.int32), (torch.int32, torch.int64)])
def test_wide_evaluation_takes_interactions_of_either_width(rowptr_type, col_type):
    from diffgraph_amd import wide
    data, had, usr, itm = _wide_tables()
    users = torch.tensor([0, 39, 7, 7], device=DEV)
    want = wide.all_rank_topk(usr, itm, users, data.trn_rowptr, data.trn_col, 9)
    got = wide.all_rank_topk(usr, itm, users, data.trn_rowptr.to(rowptr_type), data.trn_col.to(col_type), 9)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert not bool(had[users[:, None], want[1].long()].any())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.float16], ids=str)
def test_wide_evaluation_passes_gradients_to_its_tables(dtype):
    """The values are scores of the tables, and differentiable in them as torch's mm, mask and topk are: d usr[u] = sum of
    d value * itm[item], nothing through a masked place; with gradients off the same values and items."""
    from diffgraph_amd import wide
    data, had, usr, itm = _wide_tables(dtype=dtype)
    users, k = torch.tensor([0, 39, 7, 7], device=DEV), 295                  # more than some rows have left
    with torch.no_grad():
        plain = wide.all_rank_topk(usr, itm, users, data.trn_rowptr, data.trn_col, k, batch=3)
    usr.requires_grad_(), itm.requires_grad_()
    val, idx = wide.all_rank_topk(usr, itm, users, data.trn_rowptr, data.trn_col, k, batch=3)
    assert val.dtype == dtype and torch.equal(val, plain[0]) and torch.equal(idx, plain[1])
    masked = had[users[:, None], idx.long()]
    assert bool(masked.any()) and torch.equal(masked, val.double() < -1e7)
    d = torch.randn(val.shape, device=DEV).to(dtype)
    val.backward(d)
    c = torch.zeros(4, 300, dtype=torch.float64, device=DEV).scatter_(1, idx.long(), d.double().masked_fill(masked, 0))
    du = torch.zeros(40, 80, dtype=torch.float64, device=DEV).index_add_(0, users, c @ itm.detach().double())
    di = c.t().contiguous() @ usr.detach().double()[users]
    # sums of at most 300 products (and two lookups of one row): each rounding a half step of a partial sum, the rows' sums and
    # the results rounded to the type
    eps = torch.finfo(dtype).eps
    size_u = torch.zeros_like(du).index_add_(0, users, c.abs() @ itm.detach().double().abs())
    size_i = c.abs().t().contiguous() @ usr.detach().double()[users].abs()
    half = max(2.0 ** -24, eps / 2) if dtype != torch.float64 else eps / 2
    for got, want, size in ((usr.grad, du, size_u), (itm.grad, di, size_i)):
        assert got.dtype == dtype
        assert bool(((got.double() - want).abs() <= (304 * min(half, 2.0 ** -24) * 2 + 4 * half) * size + 1e-30).all())


@gpu
def test_wide_evaluation_out_of_wide_numbers():
    from diffgraph_amd import wide
    data, had, usr, itm = _wide_tables(dtype=torch.float64)
    users = torch.arange(40, device=DEV)
    val, idx = wide.all_rank_topk(usr, itm, users, data.trn_rowptr, data.trn_col, 6)
    want = (usr @ itm.t()).masked_fill(had, -1e8).topk(6)
    assert val.dtype == torch.float64 and torch.equal(val, want.values) and torch.equal(idx.long(), want.indices)


@gpu
def test_recommendations_out_of_trained_tables_are_the_best_that_are_left():
    """After a training epoch with kept activations and looked-up rows: every returned item's own score is its value, in
    descending order, no training item is among the finite ones, and nothing better was left out."""
    from diffgraph_amd.train import Coach
    from tests.test_gpu_train import _handler
    args = copy.copy(DEFAULT_ARGS)
    args.batch, args.dims, args.d_emb_size, args.epoch, args.latdim, args.act_ckpt = 64, "[128, 32]", 10, 1, 128, "int8"
    torch.manual_seed(8)
    handler = _handler()
    c = Coach(handler, args, device=DEV, seed=3)
    c.prepareModel()
    c.trainEpoch()
    with torch.no_grad():
        usr, itm = c.model.predict()
    data = handler.tst_data
    users = data.test_users_dev
    val, idx = ev.recommend(usr, itm, users, data, 5)
    v2, i2 = ev.all_rank_topk(usr, itm, users, data, 5)
    scores = torch.mm(usr[users], itm.t()).double()
    size = usr.abs().double()[users] @ itm.abs().double().t()
    off = 2 * (usr.shape[1] + 1) * 2.0 ** -24 * size.max()          # products of other shapes may add in another order
    ptr, col = data.trn_rowptr.cpu().tolist(), data.trn_col.cpu().tolist()
    for r, u in enumerate(users.tolist()):
        had = set(col[ptr[u]: ptr[u + 1]])
        left = torch.tensor([i for i in range(data.n_item) if i not in had], device=DEV)
        for v, i, out in ((val[r], idx[r], -math.inf), (v2[r], i2[r], -1e8)):
            items, n = i.tolist(), min(5, left.numel())
            assert len(set(items)) == 5 and not any(k in had for k in items[:n]) and bool((v[n:] == out).all())
            best = scores[r, left].topk(n).values
            assert bool(((scores[r, i[:n].long()] - v[:n].double()).abs() <= off).all()) and bool(((best - v[:n].double()).abs() <= off).all())
            assert bool((v[1:n] <= v[:n - 1]).all()) if n > 1 else True


@gpu
@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("fmt,dims,latdim", [("int8", "[128, 32]", 64), ("e4m3", "[64]", 128)])
def test_nc_epochs_with_kept_activations(fmt, dims, latdim, use_graph):
    """The classification model's denoiser with args.act_ckpt, eagerly and with the step recorded."""
    from diffgraph_amd.train_nc import NCCoach
    from tests.test_gpu_train import _nc_handler
    args = copy.copy(dg.nc.DEFAULT_ARGS)
    args.dims, args.d_emb_size, args.latdim, args.batch, args.act_ckpt = dims, 8, latdim, 8, fmt
    torch.manual_seed(3)
    c = NCCoach(_nc_handler(), args, device=DEV, use_graph=use_graph, seed=3)
    lines = []
    res = c.run(epochs=2, log=lines.append)
    dn = c.model.user_denoise_model
    assert dn.act_ckpt == fmt and not dn.fused
    assert len(lines) == 2 and all("nan" not in ln.lower() for ln in lines) and 0.0 <= res["macro"] <= 1.0
    assert all(bool(p.isfinite().all()) for p in c.model.parameters())


@gpu
@pytest.mark.parametrize("col_type", [torch.uint8, torch.int16])
def test_wide_evaluation_takes_interactions_in_short_types(col_type):
    from diffgraph_amd import wide
    ni = 200 if col_type == torch.uint8 else 40000               # (more items than the type's numbers: none of them interacted with)
    g = torch.Generator().manual_seed(6)
    usr, itm = torch.randn(3, 80, generator=g).to(DEV), torch.randn(ni, 80, generator=g).to(DEV)
    rowptr, col = torch.tensor([0, 2, 2, 5], device=DEV), torch.tensor([0, 7, 100, 3, 120], device=DEV)
    users = torch.tensor([2, 0, 1], device=DEV)
    want = wide.all_rank_topk(usr, itm, users, rowptr, col, 9)
    got = wide.all_rank_topk(usr, itm, users, rowptr.to(torch.int16), col.to(col_type), 9)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
