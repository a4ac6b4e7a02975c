"""Embedding lookup with scaling and its gradient by sorted tokens (ops.embedding_lookup / embedding_grad,
layers.embedding / Embedding) against the definition in 64 bits.

Tolerances.  A looked-up element is one fp32 product (2^-24) and one rounding to the table's type (eps / 2; below the
type's normal range half of its smallest step).  A gradient element is a sum of c terms in fp32, one product and one
rounding: c - 1 additions, each off by at most 2^-24 of a partial sum that is at most S = sum |d_out|, so
c 2^-24 S |scale| covers additions and product."""
import pytest
import torch

from diffgraph_amd import DiffGraphHipError, _lib, layers, ops

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu
DEV = "cuda"


def half_step(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def want_lookup(table, ids, scale):
    n = table.shape[0]
    ok = (ids >= 0) & (ids < n)
    rows = table.double()[ids.clamp(0, n - 1).long()] * scale
    return torch.where(ok[..., None], rows, torch.full_like(rows, float("nan")))


def check_lookup(got, table, ids, scale):
    want = want_lookup(table, ids, scale)
    assert got.dtype == table.dtype and got.shape == want.shape
    rel, low = half_step(table.dtype)
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    err = (got.double() - want).abs()[~nan]
    assert bool((err <= (rel + 2 * U) * want[~nan].abs() + low).all())


def check_grad(got, d_out, ids, n_rows, scale, padding):
    flat, d = ids.reshape(-1).long(), d_out.reshape(-1, d_out.shape[-1]).double()
    ok = (flat >= 0) & (flat < n_rows)
    if padding is not None:
        ok &= flat != padding
    at, d = flat[ok], d[ok]
    zero = torch.zeros(n_rows, d.shape[1], dtype=torch.float64, device=d.device)
    want, size = zero.clone().index_add_(0, at, d) * scale, zero.index_add_(0, at, d.abs())
    c = torch.bincount(at, minlength=n_rows).double()[:, None]
    rel, low = half_step(d_out.dtype)
    sums = c * U * size * abs(scale)
    assert got.dtype == d_out.dtype and got.shape == want.shape
    err = (got.double() - want).abs()
    bound = sums + rel * (want.abs() + sums) + low
    bound[size.expand_as(bound) == 0] = 0                       # rows that nothing reaches are zeros
    assert bool((err <= bound).all()), f"worst {(err / bound.clamp(min=1e-300)).max().item():.3g} bounds"


# rows, width, ids, pitch
SHAPES = [(1, 1, 1, 1), (40, 64, 1, 64), (40, 64, 7, 64), (61, 100, 333, 103), (31882, 64, 2048, 64), (1000, 33, 1025, 33),
          (257, 130, 4097, 136), (30113, 129, 5003, 129), (5, 8, 20000, 8), (1 << 20, 16, 3000, 16), (2100000, 3, 1500, 3),
          (70000, 24, 300001, 24), (3, 1, 270000, 1), (63114, 128, 6144, 128), (512, 1100, 700, 1100)]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width,n,pitch", SHAPES)
def test_lookup_and_gradient(rows, width, n, pitch, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + 7 * width + 31 * n)
    table = torch.randn(rows, pitch, generator=g, device=DEV).to(dtype)[:, :width]
    ids = (torch.rand(n, generator=g, device=DEV) ** 3 * rows).long().clamp(0, rows - 1)
    if n >= 7:
        ids[3], ids[5] = rows, -1                                 # outside the table
    ids = ids.to(torch.int32) if n % 2 else ids
    d = torch.randn(n, pitch, generator=g, device=DEV).to(dtype)[:, :width]
    scale, padding = (1.0, None) if n % 3 else (width ** 0.5, 0)
    check_lookup(ops.embedding_lookup(table, ids, scale), table, ids, scale)
    got = ops.embedding_grad(d, ids, rows, scale, padding)
    check_grad(got, d, ids, rows, scale, padding)
    assert torch.equal(got, ops.embedding_grad(d, ids, rows, scale, padding))        # the same bits again


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n", [9001, 70001])
@pytest.mark.parametrize("case", ["one token", "two tokens over chunk borders", "all padding", "all outside", "none", "sorted", "reversed"])
def test_gradient_of_long_runs(case, n, dtype):
    rows, width = 37, 72
    g = torch.Generator(device=DEV).manual_seed(11)
    d = torch.randn(n, width, generator=g, device=DEV).to(dtype)
    ids = torch.randint(0, rows, (n,), generator=g, device=DEV)
    padding = None
    if case == "one token":
        ids.fill_(36)
    elif case == "two tokens over chunk borders":
        ids.copy_((torch.arange(n, device=DEV) >= 4100).long() * 5)
    elif case == "all padding":
        ids.fill_(4)
        padding = 4
    elif case == "all outside":
        ids.fill_(rows)
        ids[::2] = -(1 << 40)
    elif case == "none":
        ids, d = ids[:0], d[:0]
    else:
        ids = ids.sort(descending=case == "reversed").values
    check_grad(ops.embedding_grad(d, ids, rows, 0.5, padding), d, ids, rows, 0.5, padding)


@gpu
def test_infinities_and_nan_stay_in_their_rows():
    table = torch.randn(50, 64, device=DEV)
    table[7, 3], table[8, 0] = float("inf"), float("nan")
    ids = torch.tensor([6, 7, 8, 9], device=DEV)
    got = ops.embedding_lookup(table, ids, 2.0)
    assert torch.equal(got.isfinite().all(1), torch.tensor([True, False, False, True], device=DEV))
    d = torch.randn(4, 64, device=DEV)
    d[1, 5] = float("nan")
    grad = ops.embedding_grad(d, ids, 50)
    assert bool(grad[7, 5].isnan()) and int(grad.isnan().sum()) == 1
    padded = ops.embedding_grad(d, ids, 50, padding_idx=7)
    assert not bool(padded[7].any()) and not bool(padded.isnan().any())              # what padding holds does not count


@gpu
def test_ids_of_other_shapes_and_orders():
    table = torch.randn(90, 40, device=DEV)
    ids = torch.randint(0, 90, (6, 5, 4), device=DEV)
    for v in (ids, ids.transpose(0, 2), ids[:, ::2], ids[0, 0, 0], ids[:0]):
        check_lookup(ops.embedding_lookup(table, v, 1.5), table, v, 1.5)
        d = torch.randn(*v.shape, 40, device=DEV)
        check_grad(ops.embedding_grad(d, v, 90, 1.5), d, v, 90, 1.5, None)
    d = torch.randn(6, 4, 5, 40, device=DEV).transpose(1, 2)                         # rows in another order than the ids
    check_grad(ops.embedding_grad(d, ids, 90), d, ids, 90, 1.0, None)
    d = torch.randn(40, 30, device=DEV).t()                                          # columns next to each other
    check_grad(ops.embedding_grad(d, ids[:, :, 0].reshape(-1), 90), d, ids[:, :, 0].reshape(-1), 90, 1.0, None)
    check_grad(ops.embedding_grad(torch.ones((), device=DEV).expand(6, 5, 4, 40), ids, 90), torch.ones(6, 5, 4, 40, device=DEV), ids, 90, 1.0, None)


@gpu
def test_differentiable_lookup_against_differences_and_torch():
    torch.manual_seed(2)
    m = layers.Embedding(30, 12, scale=3.0, padding_idx=4)
    assert not bool(m.weight[4].any())
    ids = torch.tensor([[1, 4, 4], [29, 1, 0]], device=DEV)
    coef = torch.randn(2, 3, 12, device=DEV)
    m(ids).mul(coef).sum().backward()
    grad = m.weight.grad.double()
    # central differences of the (linear) loss in 64 bits: each is the coefficient sum itself
    w = m.weight.detach().double().requires_grad_()
    loss = lambda v: (3.0 * v[ids] * coef.double()).sum()  # noqa: E731
    for r, c in ((1, 0), (29, 11), (0, 5), (17, 3)):
        e = torch.zeros_like(w)
        e[r, c] = 1e-3
        diff = ((loss(w + e) - loss(w - e)) / 2e-3).item()
        # two terms at most, scale and sum: 4 roundings of values below 3 * sum |coef|; the difference itself 1e-9 off
        assert abs(float(grad[r, c] - diff)) <= 4 * U * 3 * float(coef.abs().sum()) + 1e-9
    assert not bool(grad[4].any())
    # two lookups of one table add up
    t = torch.randn(30, 12, device=DEV, requires_grad=True)
    a, b = torch.tensor([3, 3, 5], device=DEV), torch.tensor([5, 7, 3], device=DEV)
    (layers.embedding(t, a) * layers.embedding(t, b)).sum().backward()
    w = t.detach().double().requires_grad_()
    (w[a] * w[b]).sum().backward()
    # at most four terms, each an element of the table: three additions of partial sums below 4 max |table|
    assert bool(((t.grad.double() - w.grad).abs() <= 3 * U * 4 * w.detach().abs().max()).all())


@gpu
def test_on_another_stream_and_in_a_graph():
    rows, width, n = 3000, 96, 1500
    table = torch.randn(rows, width, device=DEV)
    ids = torch.randint(0, rows, (n,), device=DEV)
    d = torch.randn(n, width, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.embedding_lookup(table, ids), ops.embedding_grad(d, ids, rows)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = ops.embedding_lookup(table, ids, 2.0)
            grad = ops.embedding_grad(d, ids, rows, 2.0)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        ids.copy_(torch.randint(0, rows, (n,), device=DEV) if k else torch.full((n,), 7, device=DEV))
        d.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = ops.embedding_lookup(table, ids, 2.0), ops.embedding_grad(d, ids, rows, 2.0)
        assert torch.equal(out, want[0]) and torch.equal(grad, want[1])
        check_grad(grad, d, ids, rows, 2.0, None)


@gpu
def test_an_output_row_past_32_bits():
    """A table whose last rows lie beyond 2^32 bytes (and 2^31 elements), looked up and given a gradient."""
    rows, width = (1 << 31) // 1024 + 5, 1024
    table = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    table[-1] = 3.0
    ids = torch.tensor([rows - 1, 0, rows - 1], device=DEV)
    assert torch.equal(ops.embedding_lookup(table, ids)[:, 0].float(), torch.tensor([3.0, 0.0, 3.0], device=DEV))
    del table
    grad = ops.embedding_grad(torch.ones(3, width, dtype=torch.bfloat16, device=DEV), ids, rows)
    assert bool((grad[-1] == 2).all()) and bool((grad[0] == 1).all()) and not bool(grad[1:-1].any())


@gpu
def test_more_ids_than_one_launch_takes():
    """16 lanes an id at one column: more than 2^26 ids take a second launch."""
    table = torch.tensor([[1.0], [2.0], [3.0]], dtype=torch.bfloat16, device=DEV)
    ids = torch.zeros((1 << 26) + 37, dtype=torch.int32, device=DEV)
    ids[::1 << 18] = 2
    ids[-17:] = 1
    rows = ops.embedding_lookup(table, ids)
    assert bool((rows[-17:] == 2).all()) and bool((rows[::1 << 18] == 3).all())
    assert rows.view(torch.int16).ne(table.view(torch.int16)[0, 0]).sum().item() == 257 + 17      # (the others: 1)


@gpu
def test_two_calls_at_once_on_two_streams():
    g = torch.Generator().manual_seed(12)
    work = []
    for n, rows in ((50000, 3000), (7000, 90000)):
        ids = torch.randint(0, rows, (n,), generator=g).to(DEV)
        work.append((torch.randn(n, 96, generator=g).to(DEV), ids, rows))
    alone = [ops.embedding_grad(*w) for w in work]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for s, w, out in zip(streams, work, got):
            with torch.cuda.stream(s):
                out.append(ops.embedding_grad(*w))
    torch.cuda.synchronize()
    for want, outs in zip(alone, got):
        assert all(torch.equal(o, want) for o in outs)


# ---- refusals (no GPU needed) ---------------------------------------------------------------------------------------
def test_cpu_tensors_and_bad_types_are_refused():
    t, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(DiffGraphHipError, match="table"):
        ops.embedding_lookup(t, ids)
    with pytest.raises(DiffGraphHipError, match="d_out"):
        ops.embedding_grad(torch.zeros(3, 8), ids, 4)
    with pytest.raises(DiffGraphHipError, match="shape"):
        ops.embedding_grad(torch.zeros(2, 8), ids, 4)
    with pytest.raises(DiffGraphHipError, match="ids a tensor"):
        ops.embedding_grad(torch.zeros(3, 8), [0, 1, 2], 4)
    with pytest.raises(DiffGraphHipError, match="n_rows"):
        ops.embedding_grad(torch.zeros(3, 8), ids, 0)
    with pytest.raises(DiffGraphHipError, match="padding_idx"):
        layers.embedding(t, ids, padding_idx=4)
    with pytest.raises(DiffGraphHipError, match="padding_idx"):
        layers.Embedding(4, 8, padding_idx=-1, device="cpu")


def test_c_entry_refuses_bad_arguments():
    lib, some = _lib.load(), 1 << 20
    assert lib.dg_embedding_lookup(some, 4, 8, 8, 3, some, 1, 2, 1.0, some, None) == -1 and b"element type" in lib.dg_last_error()
    assert lib.dg_embedding_lookup(some, 4, 8, 8, 0, None, 1, 2, 1.0, some, None) == -1 and b"NULL" in lib.dg_last_error()
    assert lib.dg_embedding_lookup(some, 4, -8, 8, 0, some, 1, 2, 1.0, some, None) == -1
    assert lib.dg_embedding_lookup(some, 0, 8, 8, 0, some, 1, 2, 1.0, some, None) == -1
    assert lib.dg_embedding_lookup(some, 1 << 31, 8, 8, 0, some, 1, 2, 1.0, some, None) == -3
    assert lib.dg_embedding_lookup(some, 4, 8, 8, 0, some, 1, 0, 1.0, some, None) == 0           # nothing to look up
    assert lib.dg_embedding_grad(some, 1, some, 1, 0, (1 << 29) + 1, 1, 0, 1.0, -1, some, some, 0, None) == -3
    assert b"2^29" in lib.dg_last_error()
    need = lib.dg_embedding_grad_workspace(100, 4, 8)
    assert need > 0 and lib.dg_embedding_grad_workspace(-1, 4, 8) == 0
    assert lib.dg_embedding_grad(some, 8, some, 1, 100, 4, 8, 0, 1.0, -1, some, some, need - 1, None) == -3
    assert b"workspace" in lib.dg_last_error()
    assert lib.dg_embedding_grad(some, 8, some, 1, 100, 4, 8, 0, 1.0, -1, some, some + 4, need, None) == -3
    assert lib.dg_embedding_grad(some, 8, some, 1, 100, 4, 8, 0, 1.0, -1, None, some, need, None) == -1


@gpu
def test_wrong_layouts_are_refused():
    t, ids = torch.zeros(8, 4, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(DiffGraphHipError, match="no rows"):
        ops.embedding_lookup(t[:0], ids[:0])
    for bad, what in ((t.t(), "next to each other"), (t.double(), "float32"), (t[0], "2-D")):
        with pytest.raises(DiffGraphHipError, match=what):
            ops.embedding_lookup(bad, ids)
    with pytest.raises(DiffGraphHipError, match="ids"):
        ops.embedding_lookup(t, ids.cpu())
    with pytest.raises(DiffGraphHipError, match="ids"):
        ops.embedding_lookup(t, ids.float())
    with pytest.raises(DiffGraphHipError, match="padding_idx"):
        ops.embedding_grad(torch.zeros(3, 4, device=DEV), ids, 8, padding_idx=8)
