"""Activation checkpoints in 8 bits (ops.checkpoint8) and the dense layer's backward pass out of them
(ops.checkpoint8_backward) against the definition in 64 bits.

Codes and their values are compared exactly.  So is the backward pass on whole-number inputs whose products and sums stay
below 2^24: every order of adding them gives the same number.  On real-valued inputs an element of d_w is a sum of n
products per piece of d_z, exact in fp32 themselves, whose additions are each off by at most 2^-23 (the matrix instruction
may cut instead of round) of a partial sum no larger than S = sum |d_z x|; d_z itself carries two roundings under tanh and
the pieces' cut (2^-15 for two pieces); one rounding to the type (eps / 2) ends it."""
import math

import pytest
import torch

from diffgraph_amd import DiffGraphHipError, _lib, ops

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
FORMATS = ["int8", "e4m3"]
gpu = pytest.mark.gpu
DEV = "cuda"


def codes_of(fmt):
    """The magnitudes a code can stand for at scale 1, in 64 bits."""
    if fmt == "int8":
        return torch.arange(128, dtype=torch.float64)
    c = torch.arange(127, dtype=torch.float64)
    return torch.where(c < 8, c * 2.0 ** -9, (8 + c % 8) * 2.0 ** (torch.floor(c / 8) - 10))


def want_values(x, fmt):
    """(values, scales) of x [n, k] by the definition, on the CPU in 64 bits."""
    x = x.cpu().double()
    n, k = x.shape
    code = codes_of(fmt)
    mid = (code[1:] + code[:-1]) / 2
    groups = -(-k // 32)
    out, scale = torch.empty_like(x), torch.empty(n, groups, dtype=torch.float64)
    powers = 2.0 ** torch.arange(-110, 129, dtype=torch.float64)
    for g in range(groups):
        v = x[:, 32 * g: 32 * g + 32]
        whole = torch.isfinite(v).all(1)
        u = torch.where(whole[:, None], v, torch.zeros_like(v))
        s = powers[torch.searchsorted(powers * code[-1], u.abs().amax(1))]
        q = u.abs() / s[:, None]
        lo, hi = torch.searchsorted(mid, q), torch.searchsorted(mid, q, right=True)
        val = torch.sign(u) * code[torch.where(lo % 2 == 0, lo, hi)] * s[:, None]
        out[:, 32 * g: 32 * g + 32] = torch.where(whole[:, None], val, torch.full_like(val, math.nan))
        scale[:, g] = torch.where(whole, s, torch.full_like(s, math.nan))
    return out, scale


def check_kept(x, fmt):
    ck = ops.checkpoint8(x, fmt)
    n, k = x.shape
    want, scale = want_values(x, fmt)
    pitch, groups, quads = (k + 15) // 16 * 16, (k + 31) // 32, (n + 3) // 4
    assert ck.shape == (n, k) and ck.data.numel() == _lib.load().dg_checkpoint8_bytes(n, k) == 4 * quads * (pitch + groups)
    codes = ck.data[: 4 * quads * pitch].view(quads, pitch, 4).permute(0, 2, 1).reshape(4 * quads, pitch).cpu()
    byte = ck.data[4 * quads * pitch:].view(quads, groups, 4).permute(0, 2, 1).reshape(4 * quads, groups)[:n].cpu().double()
    assert torch.equal(torch.where(byte == 255, torch.full_like(byte, math.nan), 2.0 ** (byte - 127)).nan_to_num(-1), scale.nan_to_num(-1))
    assert not bool(codes[:, k:].any()) and not bool(codes[n:].any())
    for t in TYPES:
        got = ck.values(t).cpu()
        assert got.dtype == t and torch.equal(got.double().nan_to_num(7e37), want.to(torch.float32).to(t).double().nan_to_num(7e37))
    return ck, want


SIZES = [(1, 1), (1, 7), (2, 3), (3, 8), (1, 16), (5, 31), (64, 32), (7, 33), (129, 72), (33, 100), (4, 333), (17, 1000), (3, 2050), (300, 64)]


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,k", SIZES)
def test_codes_and_values(n, k, dtype, fmt):
    g = torch.Generator().manual_seed(n * 1000 + k)
    x = torch.randn(n, k + 3, generator=g) * torch.exp(3 * torch.randn(n, 1, generator=g))
    x[torch.rand(n, k + 3, generator=g) < 0.2] = 0
    check_kept(x.to(dtype).to(DEV)[:, :k], fmt)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_every_16_bit_value_beside_a_larger_one(dtype, fmt):
    """Every finite value of the type, 31 to a group whose largest is 1, 0.99 or 448: each to the nearest code."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    v = bits.view(dtype)
    v = v[torch.isfinite(v)]
    v = torch.nn.functional.pad(v, (0, -v.numel() % 31)).view(-1, 31)
    for big in (1.0, 0.99, 448.0):
        x = torch.cat([torch.full((v.shape[0], 1), big, dtype=dtype), torch.where(v.abs().float() <= big, v, torch.zeros_like(v))], 1)
        check_kept(x.to(DEV), fmt)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_largest_of_a_group_at_the_borders_of_the_scale(fmt):
    one = torch.tensor(1.0)
    tops = [0.0, 2.0 ** -149, 2.0 ** -126, 448 * 2.0 ** -110, torch.finfo(torch.float32).max]
    for edge in (448.0, 127.0, 1.75, 127 / 64, 1.0):
        tops += [edge, float(torch.nextafter(edge * one, one * 1e9)), float(torch.nextafter(edge * one, one * 0))]
    x = torch.zeros(len(tops), 40)
    x[:, 3], x[:, 35] = torch.tensor(tops), -torch.tensor(tops)
    x[:, 5] = torch.tensor(tops) / 3
    check_kept(x.to(DEV), fmt)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_group_with_an_infinity_or_nan_stands_for_nan_alone(fmt):
    x = torch.randn(4, 70, device=DEV)
    x[1, 2], x[2, 40], x[3, 69] = math.inf, math.nan, -math.inf
    ck, want = check_kept(x, fmt)
    assert want.isnan().sum(1).tolist() == [0, 32, 32, 6]
    # ... and reaches the columns of d_w that belong to it, no others
    _, d_w, d_b = ops.checkpoint8_backward(torch.ones(4, 5, device=DEV), ck)
    assert torch.equal(d_w.isnan().any(0), want.isnan().any(0).to(DEV)) and not bool(d_b.isnan().any())


BACK = [(1, 1, 1), (1, 64, 64), (2, 8, 72), (31, 5, 3), (33, 33, 129), (64, 64, 64), (65, 100, 64), (300, 32, 136), (1000, 128, 128),
        (257, 65, 65), (4097, 1, 200), (700, 200, 1), (515, 260, 300), (70000, 16, 24), (12, 1000, 130)]


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tanh", [False, True], ids=["linear", "tanh"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,m,k", BACK)
def test_backward_of_whole_numbers_is_exact(n, m, k, dtype, tanh, fmt):
    g = torch.Generator().manual_seed(n + 17 * m + 291 * k)
    x = torch.randint(-8, 9, (n, k), generator=g).float()
    d = torch.randint(-4, 5, (n, m), generator=g).float() * 4
    y = torch.randint(-1, 2, (n, m), generator=g).float() / 2
    assert n * 8 * 16 < 2 ** 24 or n > 60000
    if n > 60000:
        d[torch.rand(n, m, generator=g) < 0.9] = 0              # (n * 0.1 * 8 * 16 < 2^24)
    dy = torch.cat([d, d[:, :1]], 1).to(dtype).to(DEV)[:, :m]   # rows further apart than their width
    xk, yk = ops.checkpoint8(x.to(dtype).to(DEV), fmt), ops.checkpoint8(y.to(dtype).to(DEV), fmt) if tanh else None
    d_z, d_w, d_b = ops.checkpoint8_backward(dy, xk, yk)
    z = d.double() * (1 - y.double() ** 2) if tanh else d.double()
    w, b = z.t() @ x.double(), z.sum(0)
    for got, want in ((d_z, z), (d_w, w), (d_b, b)):
        assert got.dtype == dtype and torch.equal(got.cpu(), want.to(torch.float32).to(dtype))
    if not tanh:
        assert d_z is dy


@gpu
def test_every_bit_of_an_fp32_gradient_reaches_the_product():
    """One row per column of d_w: each element is one product, 24 bits times a power of two."""
    n, m = 96, 70
    g = torch.Generator().manual_seed(3)
    d = (torch.randint(1 << 23, 1 << 24, (n, m), generator=g) | 1).float() * 2.0 ** torch.randint(-60, 60, (n, m), generator=g).float()
    x = torch.diag(2.0 ** torch.randint(-3, 4, (n,), generator=g).float())
    for fmt in FORMATS:
        _, d_w, _ = ops.checkpoint8_backward(d.to(DEV), ops.checkpoint8(x.to(DEV), fmt))
        assert torch.equal(d_w.cpu().double(), d.double().t() @ x.double())


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_bit_of_d_z_under_tanh_reaches_the_product(dtype, fmt):
    """Pairs of rows with x = 1 and -1, the same d_y and different y = c 2^-9, |c| <= 15 (codes of either format): an element
    of d_w is the difference of two d_z that agree in their leading bits, exact in fp32 whatever the order of its pieces'
    sums (each is a multiple of the smaller one's last place and no larger than d_z), and rounded once to the type."""
    pairs, m = 32, 70
    g = torch.Generator().manual_seed(11)
    d = torch.randn(pairs, 1, m, generator=g).to(dtype).expand(pairs, 2, m).reshape(2 * pairs, m)
    y = torch.randint(-15, 16, (2 * pairs, m), generator=g).float() * 2.0 ** -9
    x = torch.zeros(2 * pairs, pairs)
    x[torch.arange(2 * pairs), torch.arange(2 * pairs) // 2] = torch.tensor([1.0, -1.0]).repeat(pairs)
    xk, yk = ops.checkpoint8(x.to(dtype).to(DEV), fmt), ops.checkpoint8(y.to(dtype).to(DEV), fmt)
    assert torch.equal(yk.values().cpu(), y)
    _, d_w, _ = ops.checkpoint8_backward(d.to(DEV), xk, yk)
    z = (d.float() * (1 - y * y)).double()                      # (fp32, as the definition of d_z is held)
    want = (z[0::2] - z[1::2]).t()
    assert torch.equal(want.float().double(), want) and bool((want != 0).any())
    assert torch.equal(d_w.cpu(), want.float().to(dtype))


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tanh", [False, True], ids=["linear", "tanh"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,m,k", [(40, 64, 72), (515, 130, 260), (2049, 32, 128), (9000, 100, 50)])
def test_backward_of_real_numbers(n, m, k, dtype, tanh, fmt):
    g = torch.Generator(device=DEV).manual_seed(n)
    x = torch.randn(n, k, generator=g, device=DEV).to(dtype)
    y = torch.tanh(torch.randn(n, m, generator=g, device=DEV)).to(dtype)
    dy = torch.randn(n, m, generator=g, device=DEV).to(dtype)
    xk, yk = ops.checkpoint8(x, fmt), ops.checkpoint8(y, fmt) if tanh else None
    d_z, d_w, d_b = ops.checkpoint8_backward(dy, xk, yk)
    again = ops.checkpoint8_backward(dy, xk, yk)
    assert all(torch.equal(a, b) for a, b in zip((d_z, d_w, d_b), again))
    xv = xk.values().double()
    z = dy.double() * (1 - yk.values().double() ** 2) if tanh else dy.double()
    f = torch.finfo(dtype)
    step = lambda v: f.eps / 2 * v.abs() + f.smallest_normal * f.eps / 2  # noqa: E731
    assert bool(((d_z.double() - z).abs() <= 2 * U * z.abs() + step(z)).all())
    pieces = 3 if dtype == torch.float32 else 2 if tanh or dtype == torch.float16 else 1
    cut = 2.0 ** -15 if pieces == 2 else 0.0
    z_off = (2 * U if tanh else 0) + cut
    size = z.abs().t() @ xv.abs()
    want = z.t() @ xv
    assert bool(((d_w.double() - want).abs() <= ((n + 600) * pieces * 2 * U + z_off) * size + step(want)).all())
    size, want = z.abs().sum(0), z.sum(0)
    assert bool(((d_b.double() - want).abs() <= ((n + 600) * U + 2 * U) * size + step(want)).all())
    # as a whole: roundings add up like a random walk, far below their worst case (measured against nothing: 64 bits)
    rel = (d_w.double() - z.t() @ xv).norm() / (z.t() @ xv).norm()
    assert rel <= 8 * math.sqrt(n) * U + cut + f.eps / 2


@gpu
def test_rows_of_the_gradient_far_apart_or_the_same():
    xk = ops.checkpoint8(torch.randn(5, 40, device=DEV))
    far = torch.zeros(5, (1 << 24) + 3, device=DEV)[:, :6]
    far.normal_()
    same = torch.randn(1, 6, device=DEV).expand(5, 6)
    for d in (far, same):
        _, d_w, d_b = ops.checkpoint8_backward(d, xk)
        _, w, b = ops.checkpoint8_backward(d.clone(memory_format=torch.contiguous_format), xk)
        assert torch.equal(d_w, w) and torch.equal(d_b, b)


@gpu
def test_no_rows_give_zeros():
    for tanh in (False, True):
        xk, yk = ops.checkpoint8(torch.zeros(0, 40, device=DEV)), ops.checkpoint8(torch.zeros(0, 9, device=DEV))
        d_z, d_w, d_b = ops.checkpoint8_backward(torch.zeros(0, 9, device=DEV), xk, yk if tanh else None)
        assert d_z.shape == (0, 9) and d_w.shape == (9, 40) and not bool(d_w.any()) and not bool(d_b.any())
    assert xk.values().shape == (0, 40)


@gpu
def test_codes_past_32_bits():
    n, k = (1 << 31) // 1024 + 3, 1024
    x = torch.zeros(n, k, dtype=torch.bfloat16, device=DEV)
    x[-1], x[0, 0] = 3.0, 1.0
    ck = ops.checkpoint8(x, "e4m3")
    del x
    d = torch.zeros(n, 8, dtype=torch.bfloat16, device=DEV)
    d[-1], d[0] = 2.0, 5.0
    _, d_w, d_b = ops.checkpoint8_backward(d, ck)
    want = torch.full((8, k), 6.0)
    want[:, 0] = 11.0
    assert torch.equal(d_w.cpu().float(), want) and bool((d_b == 7).all())
    assert torch.equal(ck.values(torch.bfloat16)[-1].cpu().float(), torch.full((k,), 3.0))


@gpu
def test_on_another_stream_and_in_a_graph():
    n, k, m = 700, 90, 70
    x, y, d = torch.randn(n, k, device=DEV), torch.tanh(torch.randn(n, m, device=DEV)), torch.randn(n, m, device=DEV)

    def call():
        xk, yk = ops.checkpoint8(x, "e4m3"), ops.checkpoint8(y, "e4m3")
        return ops.checkpoint8_backward(d, xk, yk)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        x.normal_(), d.normal_()
        y.copy_(torch.tanh(torch.randn(n, m, device=DEV)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, call()))


@gpu
def test_two_calls_at_once_on_two_streams():
    g = torch.Generator().manual_seed(14)
    work = []
    for n, m, k, dtype in ((20000, 64, 100, torch.float32), (3001, 130, 257, torch.bfloat16)):
        x, y, d = (torch.randn(n, c, generator=g).to(DEV).to(dtype) for c in (k, m, m))
        work.append((d, x, torch.tanh(y)))
    run = lambda d, x, y: ops.checkpoint8_backward(d, ops.checkpoint8(x), ops.checkpoint8(y))  # noqa: E731
    alone = [run(*w) for w in work]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for s, w, out in zip(streams, work, got):
            with torch.cuda.stream(s):
                out.append(run(*w))
    torch.cuda.synchronize()
    for want, outs in zip(alone, got):
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


# ---- refusals (no GPU needed) ---------------------------------------------------------------------------------------
def test_c_entry_refuses_bad_arguments():
    lib, p = _lib.load(), 1 << 20
    assert lib.dg_checkpoint8_bytes(5, 33) == 8 * (48 + 2) and lib.dg_checkpoint8_bytes(5, 0) == 0 and lib.dg_checkpoint8_bytes(-1, 4) == 0
    assert lib.dg_checkpoint8(p, 8, 2, 8, 0, 5, p, None) == -1 and b"format" in lib.dg_last_error()
    assert lib.dg_checkpoint8(p, 8, 2, 8, 9, 0, p, None) == -1 and b"type" in lib.dg_last_error()
    assert lib.dg_checkpoint8(p, 8, 2, 0, 0, 0, p, None) == -1
    assert lib.dg_checkpoint8(p, -8, 2, 8, 0, 0, p, None) == -1
    assert lib.dg_checkpoint8(p, 8, 2, 8, 0, 0, p + 8, None) == -1 and b"aligned" in lib.dg_last_error()
    assert lib.dg_checkpoint8(None, 8, 2, 8, 0, 0, p, None) == -1
    assert lib.dg_checkpoint8(None, 8, 0, 8, 0, 0, None, None) == 0
    assert lib.dg_checkpoint8(p, 8, 1 << 31, 8, 0, 0, p, None) == -3
    assert lib.dg_checkpoint8_values(p, 2, 8, 0, 9, p, None) == -1 and lib.dg_checkpoint8_values(None, 2, 8, 0, 0, p, None) == -1
    need = lib.dg_checkpoint8_backward_workspace(100, 8, 8)
    back = lambda **k: lib.dg_checkpoint8_backward(*{**dict(d_y=p, stride=8, n=100, m=8, k=8, dtype=0, fmt=0, xk=p, yk=p, dz=p,  # noqa: E731
                                                            dw=p, db=p, ws=p, bytes=need, stream=None), **k}.values())
    for bad, text in ((dict(fmt=2), b"format"), (dict(dtype=3), b"type"), (dict(m=0), b"sizes"), (dict(n=-1), b"sizes"), (dict(stride=7), b"overlap"),
                      (dict(xk=None), b"NULL"), (dict(dz=None), b"NULL"), (dict(dw=None), b"NULL"),
                      (dict(xk=p + 4), b"aligned"), (dict(yk=p + 8), b"aligned"), (dict(ws=p + 4), b"aligned")):
        assert back(**bad) == -1 and text in lib.dg_last_error(), bad
    assert back(stride=(1 << 24) + 1) == -3 and b"apart" in lib.dg_last_error()
    assert back(bytes=need - 1) == -3 and b"workspace" in lib.dg_last_error()


def test_cpu_tensors_are_refused():
    with pytest.raises(DiffGraphHipError, match="GPU"):
        ops.checkpoint8(torch.zeros(2, 8))
    with pytest.raises(DiffGraphHipError, match="GPU"):
        ops.checkpoint8_backward(torch.zeros(2, 8), None)


@gpu
def test_wrong_arguments_are_refused():
    x, d = torch.zeros(6, 40, device=DEV), torch.zeros(6, 9, device=DEV)
    xk = ops.checkpoint8(x)
    for call, what in ((lambda: ops.checkpoint8(x, "int4"), "format"), (lambda: ops.checkpoint8(x.t()), "next to each other"),
                       (lambda: ops.checkpoint8(x.double()), "float32"), (lambda: xk.values(torch.float64), "values"),
                       (lambda: ops.checkpoint8_backward(d, x), "checkpoint8 returns"), (lambda: ops.checkpoint8_backward(d[:5], xk), "rows"),
                       (lambda: ops.checkpoint8_backward(d, xk, xk), "columns"),
                       (lambda: ops.checkpoint8_backward(d, xk, ops.checkpoint8(d, "e4m3")), "format"),
                       (lambda: ops.checkpoint8_backward(d, ops.Checkpoint8(xk.data[:-1], (6, 40), "int8")), "keeps"),
                       (lambda: ops.Checkpoint8(xk.data, (6, 49), "int8").values(), "keeps")):
        with pytest.raises(DiffGraphHipError, match=what):
            call()
