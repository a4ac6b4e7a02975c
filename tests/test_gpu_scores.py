"""Penalties, biases and masks on scores (ops.adjust_scores) against the definition in 64 bits.

Tolerance: three fp32 roundings at most on the way of a penalised score (quotient or product; frequency * had, its sum with
presence, and their difference count together below as four), one of the bias's sum, each 2^-24 of a value no larger than
the sum of the terms' sizes; then one rounding to the type (eps / 2)."""
import math

import pytest
import torch

from diffgraph_amd import DiffGraphHipError, _lib, ops

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu
DEV = "cuda"


def counts_of(rowptr, col, lines, items):
    """[len(lines), items] counts of the CSR's lines on the CPU; a line outside the CSR is empty, ids outside fall away."""
    rowptr, col = rowptr.cpu().tolist(), col.cpu().long()
    had = torch.zeros(len(lines), items, dtype=torch.float64)
    for r, line in enumerate(lines):
        if 0 <= line < len(rowptr) - 1:
            c = col[rowptr[line]: rowptr[line + 1]]
            had[r] = torch.bincount(c[(c >= 0) & (c < items)], minlength=items).double()
    return had


def bits_of(words, items):
    """[masks, items] truth values of int32 words."""
    w = words.cpu().reshape(-1, words.shape[-1])
    item = torch.arange(items)
    return ((w[:, item // 32].long() >> (item % 32)) & 1).bool()


def want_scores(scores, had, rep, fre, pre, bias, stays, exclude, fill):
    """(value, size of the terms, which places are masked), in 64 bits on the CPU."""
    v = scores.cpu().double()
    col = lambda x: x.cpu().double()[:, None] if isinstance(x, torch.Tensor) else torch.tensor(float(x), dtype=torch.float64)  # noqa: E731
    rep, fre, pre = col(rep), col(fre), col(pre)
    off = fre * had + pre
    pen = torch.where(v > 0, v / rep, v * rep)
    size = torch.where(had > 0, pen.abs() + (fre * had).abs() + pre.abs(), v.abs())
    v = torch.where(had > 0, pen - off, v)
    if bias is not None:
        v, size = v + bias.cpu().double(), size + bias.cpu().double().abs()
    masked = torch.zeros_like(v, dtype=torch.bool)
    if stays is not None:
        masked |= ~stays
    if exclude:
        masked |= had > 0
    return torch.where(masked, torch.full_like(v, fill), v), torch.where(masked, torch.zeros_like(v), size)


def check(got, want, size, dtype):
    got = got.cpu()
    assert got.dtype == dtype
    target = want.to(torch.float32).to(dtype).double()         # (fills beyond the range become infinities)
    special = ~torch.isfinite(target)
    assert torch.equal(got.isnan(), target.isnan())
    assert torch.equal(got.double()[special & ~target.isnan()], target[special & ~target.isnan()])
    f = torch.finfo(dtype)
    bound = 6 * U * size + f.eps / 2 * (want.abs() + 6 * U * size) + f.smallest_normal * f.eps / 2
    err = (got.double() - want).abs()[~special]
    assert bool((err <= bound[~special]).all()), f"worst {(err / bound[~special]).max().item():.3g} bounds"


def history(n, items, longest, g):
    lengths = torch.randint(0, longest + 1, (n,), generator=g)
    lengths[0] = longest
    if n > 2:
        lengths[n // 2] = 0
    rowptr = torch.zeros(n + 1, dtype=torch.int64)
    rowptr[1:] = lengths.cumsum(0)
    col = (torch.rand(int(rowptr[-1]), generator=g) ** 2 * items).long().clamp(0, items - 1)
    if col.numel() > 4:
        col[1], col[3] = items, -1                              # outside: passed over
    return rowptr.to(torch.int32), col.to(torch.int32)


SIZES = [(1, 1, 3), (1, 2, 9), (1, 31232, 37), (3, 33, 40), (5, 4095, 300), (2, 4096, 5000), (7, 4097, 64), (4, 8193, 20000), (33, 1000, 12),
         (64, 5, 4), (2, 131071, 4096)]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,items,longest", SIZES)
@pytest.mark.parametrize("form", ["penalties", "everything", "exclude", "mask", "bias per row"])
def test_scores_against_the_definition(form, n, items, longest, dtype):
    g = torch.Generator().manual_seed(items * 13 + n)
    pitch = items + (n % 3)
    scores = (torch.randn(n, pitch, generator=g) * 4).to(dtype).to(DEV)[:, :items]
    rowptr, col = (v.to(DEV) for v in history(n, items, longest, g))
    had = counts_of(rowptr, col, range(n), items)
    one = lambda lo, hi: (torch.rand(n, generator=g) * (hi - lo) + lo).to(DEV)  # noqa: E731
    kw, want = {}, dict(rep=1.0, fre=0.0, pre=0.0, bias=None, stays=None, exclude=False, fill=-math.inf)
    if form in ("penalties", "everything"):
        want.update(rep=one(0.5, 2.0), fre=one(-0.3, 1.0), pre=0.25)
        kw = dict(repetition=want["rep"], frequency=want["fre"], presence=0.25)
    if form in ("everything", "mask"):
        words = torch.randint(-2 ** 31, 2 ** 31, (4, (items + 31) // 32 + 1), generator=g).to(torch.int32).to(DEV)
        words[2] = 0                                            # leaves nothing
        which = (torch.arange(n, dtype=torch.int32) % 6 - 1).to(DEV)       # -1 and 4: no mask
        inside = (which >= 0) & (which < 4)
        want["stays"] = bits_of(words, items)[which.cpu().long().clamp(0, 3)] | ~inside.cpu()[:, None]
        kw.update(allowed=words, allowed_rows=which)
    if form == "everything":
        want["bias"] = torch.randn(items, generator=g).to(DEV)
        kw["bias"] = want["bias"]
    if form == "bias per row":
        want["bias"] = torch.randn(n, items + 3, generator=g).to(DEV)[:, :items]
        kw["bias"] = want["bias"]
    if form in ("exclude", "everything"):
        want.update(exclude=True, fill=-1e8 if form == "exclude" else torch.finfo(dtype).min)
        kw.update(exclude=True, fill=want["fill"])
    got = ops.adjust_scores(scores, history=(rowptr, col), **kw)
    v, size = want_scores(scores, had, want["rep"], want["fre"], want["pre"], want["bias"], want["stays"], want["exclude"], want["fill"])
    check(got, v, size, dtype)
    inplace = scores.clone() if pitch == items else torch.cat([scores, scores[:, :1]], 1)[:, :items]
    assert ops.adjust_scores(inplace, history=(rowptr, col), out=inplace, **kw) is inplace
    assert torch.equal(inplace, got)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_masked_places_may_hold_anything_and_rows_behind_stay(dtype):
    big = torch.randn(9, 700, device=DEV).to(dtype)
    big[0, 5], big[0, 6], big[1, 7] = float("nan"), float("inf"), -float("inf")
    before = big.clone()
    words = torch.full((3, 22), -1, dtype=torch.int32, device=DEV)
    words[0, 0] = ~((1 << 5) | (1 << 6))
    words[2] = 0
    got = ops.adjust_scores(big[:3], allowed=words, out=big[:3], fill=-3.0)
    assert bool((got[0, 5:7] == -3).all()) and bool((got[2] == -3).all()) and got[1, 7] == -float("inf")
    assert torch.equal(big[3:], before[3:])
    # an infinity that stays goes through the penalties as the formula says; nothing else is touched
    rowptr, col = torch.tensor([0, 2], dtype=torch.int32, device=DEV), torch.tensor([6, 9], dtype=torch.int32, device=DEV)
    row = ops.adjust_scores(before[:1], history=(rowptr, col), repetition=2.0)
    assert row[0, 6] == float("inf") and bool(row[0, 5].isnan()) and torch.equal(row[0, 10:], before[0, 10:])


@gpu
def test_history_lines_by_number_and_no_history_at_all():
    g = torch.Generator().manual_seed(5)
    rowptr, col = (v.to(DEV) for v in history(20, 900, 50, g))
    scores = torch.randn(6, 900, device=DEV)
    lines = [3, 3, 0, 19, 20, -1]
    got = ops.adjust_scores(scores, history=(rowptr, col), rows=torch.tensor(lines, device=DEV), exclude=True, fill=-1e8)
    v, size = want_scores(scores, counts_of(rowptr, col, lines, 900), 1.0, 0.0, 0.0, None, None, True, -1e8)
    check(got, v, size, torch.float32)
    empty = (torch.zeros(7, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV))
    assert torch.equal(ops.adjust_scores(scores, history=empty, exclude=True), scores)
    assert torch.equal(ops.adjust_scores(scores), scores)
    for shape in ((0, 900), (6, 0)):
        if shape[1]:
            assert ops.adjust_scores(scores[: shape[0]]).shape == shape


@gpu
def test_many_rows_and_offsets_past_32_bits():
    scores = torch.zeros(70001, 9, device=DEV)
    rowptr = torch.arange(70002, dtype=torch.int32, device=DEV)
    col = (torch.arange(70001, device=DEV) % 9).to(torch.int32)
    got = ops.adjust_scores(scores, history=(rowptr, col), presence=1.0)
    assert torch.equal(got, -torch.nn.functional.one_hot(col.long(), 9).float())
    far = torch.zeros(1 << 15, (1 << 17) + 8, dtype=torch.bfloat16, device=DEV)           # 2^32 elements and more
    rowptr = torch.zeros((1 << 15) + 1, dtype=torch.int32, device=DEV)
    rowptr[-1] = 2
    col = torch.tensor([(1 << 17) + 7, 0], dtype=torch.int32, device=DEV)
    ops.adjust_scores(far, history=(rowptr, col), presence=2.0, out=far)
    assert far[-1, -1] == -2 and far[-1, 0] == -2 and int(far[-1].count_nonzero()) == 2 and not bool(far[:2].any())


@gpu
def test_the_longest_row():
    """2^31 - 1 items: the last tile ends where a 32-bit count of items does."""
    items = (1 << 31) - 1
    scores = torch.zeros(1, items, dtype=torch.bfloat16, device=DEV)
    at = [0, 4095, 4096, items - 4096, items - 4095, items - 1]
    col = torch.tensor(at + at[-1:], dtype=torch.int32, device=DEV)
    rowptr = torch.tensor([0, len(at) + 1], dtype=torch.int32, device=DEV)
    ops.adjust_scores(scores, history=(rowptr, col), frequency=2.0, out=scores)
    assert scores[0, at].tolist() == [-2.0] * (len(at) - 1) + [-4.0]
    scores[0, at] = 0
    assert not bool(scores.any())


@gpu
def test_the_most_rows():
    """2^31 - 1 rows of one item: the launches' first rows end where a 32-bit one would."""
    n = (1 << 31) - 1
    scores = torch.zeros(n, 1, dtype=torch.bfloat16, device=DEV)
    ops.adjust_scores(scores, bias=torch.ones(1, device=DEV), out=scores)
    assert bool((scores == 1).all())


@gpu
def test_in_place_calls_are_seen_by_autograd():
    """A tensor that a backward pass still needs: changed by the call, it is refused there, as after torch's own."""
    bias = torch.ones(64, device=DEV)
    p = torch.randn(2, 64, device=DEV, requires_grad=True)
    for write in (lambda q: ops.adjust_scores(q, bias=bias, out=q), lambda q: ops.adjust_scores(torch.zeros_like(q), bias=bias, out=q)):
        q = p * 1
        loss = (q * q).sum()
        before, seen = q._version, q.detach()
        assert write(seen) is seen and q._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    q = p * 1
    loss, before = (q * q).sum(), q._version
    ops.adjust_scores(q.detach(), bias=bias)                    # reads alone
    with pytest.raises(DiffGraphHipError, match="own"):
        ops.adjust_scores(q.detach()[:1], bias=bias, out=q.detach()[1:])
    assert q._version == before
    loss.backward()
    assert torch.equal(p.grad, 2 * p)
    with torch.inference_mode():
        s = torch.randn(2, 64, device=DEV)
        want = s + 1
        assert torch.equal(ops.adjust_scores(s, bias=bias, out=s), want)


@gpu
def test_on_another_stream_and_in_a_graph():
    g = torch.Generator().manual_seed(8)
    rowptr, col = (v.to(DEV) for v in history(16, 5000, 200, g))
    scores, bias = torch.randn(16, 5000, device=DEV), torch.randn(5000, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call = lambda: ops.adjust_scores(scores, history=(rowptr, col), repetition=1.3, frequency=0.2, bias=bias)  # noqa: E731
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        scores.normal_()
        col.copy_(torch.randint(0, 5000, (col.numel(),), device=DEV).to(torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


# ---- refusals (no GPU needed) ---------------------------------------------------------------------------------------
def test_c_entry_refuses_bad_tasks():
    import ctypes as C
    lib, p = _lib.load(), 1 << 20

    def rc(**kw):
        t = _lib.ScoreTask(scores=p, out=p, row_stride=8, out_stride=8, n_rows=2, n_items=8, repetition_all=1.0)
        for k, v in kw.items():
            setattr(t, k, v)
        return lib.dg_adjust_scores(C.byref(t), None)

    assert lib.dg_adjust_scores(None, None) == -1
    assert rc(n_rows=0) == 0 and rc(n_items=0) == 0
    for bad, text in ((dict(dtype=7), b"type"), (dict(n_rows=-1), b"sizes"), (dict(scores=None), b"NULL"), (dict(out_stride=7), b"overlap"),
                      (dict(row_stride=-8), b"stride"), (dict(hist_rowptr=p), b"history"), (dict(hist_rows=p), b"history"),
                      (dict(hist_rowptr=p, hist_col=p, n_hist=1), b"histories"), (dict(repetition_all=0.0), b"positive"),
                      (dict(repetition_all=float("nan")), b"positive"), (dict(allowed=p, n_masks=0, mask_words=1), b"mask"),
                      (dict(allowed=p, n_masks=1, mask_words=0), b"words"), (dict(allowed=p, n_masks=3, n_rows=4, mask_words=1), b"masks"),
                      (dict(bias=p, bias_stride=-1), b"bias")):
        assert rc(**bad) == -1 and text in lib.dg_last_error(), (bad, lib.dg_last_error())


def test_cpu_tensors_are_refused():
    with pytest.raises(DiffGraphHipError, match="GPU"):
        ops.adjust_scores(torch.zeros(2, 8))


@gpu
def test_wrong_arguments_are_refused():
    s = torch.zeros(2, 64, device=DEV)
    h = (torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    i32 = lambda *a: torch.zeros(*a, dtype=torch.int32, device=DEV)  # noqa: E731
    for kw, what in ((dict(exclude=True), "history"), (dict(repetition=1.2), "history"), (dict(history=(h[0][:2], h[1])), "lines"),
                     (dict(history=(h[0].long(), h[1])), "history"), (dict(history=h, rows=torch.zeros(3, dtype=torch.int64, device=DEV)), "rows"),
                     (dict(history=h, repetition=0.0), "positive"), (dict(history=h, repetition=torch.ones(3, device=DEV)), "one value"),
                     (dict(bias=torch.zeros(63, device=DEV)), "bias"), (dict(bias=torch.zeros(64)), "bias"), (dict(allowed=i32(1)), "words"),
                     (dict(allowed=i32(3, 2)), "masks"), (dict(allowed=i32(0, 2), allowed_rows=i32(2)), "no mask"),
                     (dict(allowed_rows=i32(2)), "masks"), (dict(allowed=i32(3, 2), allowed_rows=i32(3)), "allowed_rows"),
                     (dict(out=s.half()), "out"), (dict(out=s[:, :32]), "out")):
        with pytest.raises(DiffGraphHipError, match=what):
            ops.adjust_scores(s, **kw)
    both = torch.zeros(4, 64, device=DEV)
    with pytest.raises(DiffGraphHipError, match="memory of its own"):
        ops.adjust_scores(both[:2], out=both[1:3])
    with pytest.raises(DiffGraphHipError, match="overlap"):
        ops.adjust_scores(s, out=torch.zeros(64, device=DEV).expand(2, 64))
    with pytest.raises(DiffGraphHipError, match="next to each other"):
        ops.adjust_scores(s.t())
    with pytest.raises(DiffGraphHipError, match="2\\^31"):
        ops.adjust_scores(torch.zeros(1, 1, dtype=torch.bfloat16, device=DEV).expand(1 << 31, 1))


@gpu
def test_tensors_that_ask_for_a_gradient():
    """The call is not recorded: where a gradient would be lost, it is refused."""
    s, b = torch.randn(2, 64, device=DEV, requires_grad=True), torch.zeros(64, device=DEV, requires_grad=True)
    for scores, bias in ((s, None), (s * 2, None), (s.detach(), b)):
        with pytest.raises(DiffGraphHipError, match="autograd"):
            ops.adjust_scores(scores, bias=bias)
        with torch.no_grad():
            assert torch.equal(ops.adjust_scores(scores, bias=bias), scores)
    assert torch.equal(ops.adjust_scores(s.detach(), bias=b.detach()), s.detach())


@gpu
@pytest.mark.parametrize("name", ["repetition", "frequency", "presence", "out"])
def test_penalties_and_outputs_that_ask_for_a_gradient(name):
    """A penalty's gradient would be lost as a score's would; an output that asks for one takes no unrecorded values."""
    s = torch.randn(2, 64, device=DEV)
    h = (torch.tensor([0, 1, 3], dtype=torch.int32, device=DEV), torch.tensor([5, 7, 7], dtype=torch.int32, device=DEV))
    asks = torch.ones(2, 64, device=DEV, requires_grad=True) if name == "out" else torch.full((2,), 1.5, device=DEV, requires_grad=True)
    with pytest.raises(DiffGraphHipError, match="autograd"):
        ops.adjust_scores(s, history=h, **{name: asks})
    want = ops.adjust_scores(s, history=h, **({} if name == "out" else {name: asks.detach()}))
    with torch.no_grad():
        assert torch.equal(ops.adjust_scores(s, history=h, **{name: asks}), want)
    with pytest.raises(DiffGraphHipError, match="bias"):
        ops.adjust_scores(s, bias=[0.0] * 64)


def test_c_entry_refuses_one_table_with_two_strides():
    import ctypes as C
    p = 1 << 20
    t = _lib.ScoreTask(scores=p, out=p, row_stride=16, out_stride=8, n_rows=2, n_items=8, repetition_all=1.0)
    assert _lib.load().dg_adjust_scores(C.byref(t), None) == -1 and b"overlap" in _lib.load().dg_last_error()


def test_c_entry_names_the_words_of_the_longest_mask():
    import ctypes as C
    items, p = (1 << 31) - 1, 1 << 20
    t = _lib.ScoreTask(scores=p, out=p, row_stride=items, out_stride=items, n_rows=1, n_items=items, repetition_all=1.0, allowed=p, n_masks=1,
                       mask_words=(1 << 26) - 1)
    assert _lib.load().dg_adjust_scores(C.byref(t), None) == -1 and b"at least 67108864 words" in _lib.load().dg_last_error()
