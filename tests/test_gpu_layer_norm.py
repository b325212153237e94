"""Layer norm, forward and backward, against the 64-bit oracle and its derived bounds."""
import pytest
import torch

import cppmega_amd
from cppmega_amd import LayerNorm, layer_norm, layer_norm_backward
from oracle import layer_norm as orc

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _inputs(gen, rows, n, dtype, wdtype, weight=True, bias=True):
    x = (torch.randn(rows, n, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen)) + torch.randn(rows, 1, generator=gen)).to(dtype)
    w = (1 + 0.3 * torch.randn(n, generator=gen)).to(wdtype) if weight else None
    b = torch.randn(n, generator=gen).to(wdtype) if bias else None
    return x, torch.randn(rows, n, generator=gen).to(dtype), w, b


def _check(got, ref, names):
    for name in names:
        a, e, tol = got[name].double().cpu(), ref[name], ref["e_" + name]
        a = a.reshape(e.shape)
        bad = ~((a - e).abs() <= tol)
        assert not bad.any(), (name, int(bad.sum()), a[bad][:4], e[bad][:4], tol[bad][:4])


def _step(dev, x, dy, w, b, eps):
    """One training step's results from tensors on the device."""
    leaves = [t if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = LayerNorm.apply(*leaves, eps)
    wanted = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, wanted, dy))
    got = dict(y=y.detach())
    for name, t in zip(("dx", "dweight", "dbias"), leaves):
        if t is not None:
            got[name] = next(grads)
            assert got[name].dtype == t.dtype and got[name].shape == t.shape
    return got


def _run(dev, x, dy, w, b, eps=1e-5):
    on = [t if t is None else t.to(dev) for t in (x, dy, w, b)]
    got = _step(dev, *on, eps)
    pd = next((t.dtype for t in (w, b) if t is not None), F32)
    ref = orc.layer_norm(x.reshape(-1, x.shape[-1]), w, b, eps, dy.reshape(-1, x.shape[-1]), x.dtype, pd)
    _check(got, ref, list(got))
    return got


WIDTHS = [1, 2, 7, 8, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1001, 1024, 1025, 2048, 2049, 4095, 4096, 4097, 8192, 8193,
          16383, 16384]


@pytest.mark.parametrize("n", WIDTHS)
def test_widths(dev, n):
    gen = torch.Generator().manual_seed(n)
    for rows, dtype, wdtype in ((37, BF, BF), (5, BF, F32), (3, F32, F32), (1, F32, BF)):
        _run(dev, *_inputs(gen, rows, n, dtype, wdtype))


@pytest.mark.parametrize("rows,n", [(1, 64), (31, 64), (33, 64), (8192, 64), (20001, 64), (9000, 128), (1500, 300), (3001, 1000), (700, 2048),
                                    (600, 4096), (520, 8200)])
def test_many_rows(dev, rows, n):
    gen = torch.Generator().manual_seed(rows)
    _run(dev, *_inputs(gen, rows, n, BF, BF), eps=1e-6)


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("n", [64, 700, 5000])
def test_without_parameters(dev, weight, bias, n):
    gen = torch.Generator().manual_seed(n)
    _run(dev, *_inputs(gen, 50, n, BF, F32, weight, bias))


def test_a_column_of_very_many_equal_values(dev):
    """2^26 rows, whose value rounds down by almost half a step of the sum where a lane's 4096 are added one after the other."""
    rows, n = 1 << 26, 8
    c = 1 + 2.0 ** -13 - 2.0 ** -23
    x, dy = torch.ones(1, n, device=dev).expand(rows, n), torch.full((1, n), c, device=dev).expand(rows, n)
    mean, rstd = torch.zeros(rows, device=dev), torch.ones(rows, device=dev)
    _, dw, db = layer_norm_backward(dy, x, None, mean, rstd, (False, True, True))
    for got in (dw, db):
        assert ((got.double().cpu() - rows * c).abs() <= orc.WIDEN * (orc.ROWS + orc.V) * rows * c).all()


def test_an_infinite_gradient_among_very_many(dev):
    """It stays in its column, and a sum of one sign of infinity is that infinity."""
    rows, n = 2_200_003, 4
    x, dy = torch.ones(rows, n, device=dev), torch.ones(rows, n, device=dev)
    dy[77, 1], dy[1_900_000, 2], dy[2_000_000, 2] = float("inf"), float("inf"), -float("inf")
    _, dw, db = layer_norm_backward(dy, x, None, torch.zeros(rows, device=dev), torch.ones(rows, device=dev), (False, True, True))
    for got in (dw, db):
        assert got[0] == got[3] == rows and got[1] == float("inf") and got[2].isnan()


@pytest.mark.parametrize("rows,n", [(2_200_003, 3), (270_001, 300), (70_001, 1100), (33_001, 9000)])
def test_columns_over_very_many_rows(dev, rows, n):
    """More rows than a lane adds in a run, in every form of the workgroup; the sums in 64 bits beside them."""
    gen = torch.Generator(device=dev).manual_seed(n)
    x, dy = (torch.randn(rows, n, generator=gen, device=dev, dtype=F32).to(BF) for _ in range(2))
    mean, rstd = 0.1 * torch.randn(rows, generator=gen, device=dev), 0.5 + torch.rand(rows, generator=gen, device=dev)
    got = layer_norm_backward(dy, x, None, mean, rstd)
    again = layer_norm_backward(dy, x, None, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    part = slice(rows - 40, None)
    assert torch.equal(got[0][part], layer_norm_backward(dy[part], x[part], None, mean[part], rstd[part], (True, False, False))[0])
    sums = torch.zeros(4, n, dtype=torch.float64, device=dev)
    for at in range(0, rows, 1 << 14):
        a, g = x[at:at + (1 << 14)].double(), dy[at:at + (1 << 14)].double()
        t = g * ((a - mean[at:at + (1 << 14), None].double()) * rstd[at:at + (1 << 14), None].double())
        sums += torch.stack([t.sum(0), g.sum(0), t.abs().sum(0), g.abs().sum(0)])
    sums = sums.cpu()                                                  # (xhat: two roundings)
    _check(dict(dweight=got[1], dbias=got[2]),
           dict(dweight=sums[0], dbias=sums[1], e_dweight=orc.WIDEN * ((orc.ROWS + 2 * orc.V) * sums[2] + orc.V * sums[0].abs()),
                e_dbias=orc.WIDEN * (orc.ROWS * sums[3] + orc.V * sums[1].abs())), ("dweight", "dbias"))


def test_shapes_strides_and_alignment(dev):
    """Leading axes, rows inside a wider tensor at any element, broadcast and transposed gradients."""
    gen = torch.Generator().manual_seed(4)
    for n in (64, 97, 1100):
        x, dy, w, b = _inputs(gen, 24, n, BF, BF)
        on = [t.to(dev) for t in (x, dy, w, b)]
        ref = orc.layer_norm(x, w, b, 1e-5, dy)
        _check(_step(dev, on[0].view(2, 3, 4, n), on[1].view(2, 3, 4, n), *on[2:], 1e-5), ref, ("y", "dx", "dweight", "dbias"))
        for off, width in ((1, n + 5), (3, 2 * n + 3)):
            wide, wide_dy = torch.full((24, width), float("nan"), dtype=BF, device=dev), torch.full((24, width), float("nan"), dtype=BF, device=dev)
            wide[:, off:off + n], wide_dy[:, off:off + n] = on[0], on[1]
            _check(_step(dev, wide[:, off:off + n], wide_dy[:, off:off + n], *on[2:], 1e-5), ref, ("y", "dx", "dweight", "dbias"))
        _check(_step(dev, on[0], on[1].t().contiguous().t(), *on[2:], 1e-5), ref, ("y", "dx", "dweight", "dbias"))
        one = dy[:1].expand(24, n)
        ref1 = orc.layer_norm(x, w, b, 1e-5, one)
        _check(_step(dev, on[0], on[1][:1].expand(24, n), *on[2:], 1e-5), ref1, ("y", "dx", "dweight", "dbias"))
        same = dy[:, :1].expand(24, n)                 # what sum(-1) gives
        _check(_step(dev, on[0], on[1][:, :1].expand(24, n), *on[2:], 1e-5), orc.layer_norm(x, w, b, 1e-5, same), ("y", "dx", "dweight", "dbias"))
        _check(_step(dev, on[0][:1].expand(24, n), on[1], *on[2:], 1e-5), orc.layer_norm(x[:1].expand(24, n), w, b, 1e-5, dy),
               ("y", "dx", "dweight", "dbias"))


def test_rows_past_a_grid_and_past_four_gigabytes(dev):
    """The last rows of a call with more than 2^32 threads, and of one whose rows lie past 2^32 bytes: those of a call on them alone."""
    w, b = torch.tensor([1.0, 2.0, -0.5], device=dev), torch.tensor([0.0, 1.0, 0.25], device=dev)
    x = torch.randn((1 << 29) + 77, 3, dtype=BF, device=dev)
    y, mean, rstd = layer_norm(x, w, b, return_stats=True)
    for part in (slice(0, 50), slice((1 << 29) - 40, None)):
        assert torch.equal(y[part], layer_norm(x[part], w, b))
    dx, _, _ = layer_norm_backward(y, x, w, mean, rstd, (True, False, False))
    part = slice((1 << 29) - 40, None)
    assert torch.equal(dx[part], layer_norm_backward(y[part], x[part], w, mean[part], rstd[part], (True, False, False))[0])
    del x, y, mean, rstd, dx
    x = torch.zeros((1 << 22) + 9, 1024, dtype=BF, device=dev)[:, 5:69]
    x[-40:] = torch.randn(40, 64, device=dev).to(BF)
    y, mean, rstd = layer_norm(x, return_stats=True)
    assert (y[:-40] == 0).all() and torch.equal(y[-40:], layer_norm(x[-40:].contiguous()))
    dw = layer_norm_backward(x, x, None, mean, rstd)[1]                # (rows of zeros add nothing)
    ref = orc.layer_norm(x[-40:].cpu(), None, None, 1e-5, x[-40:].cpu(), BF, F32)
    assert ((dw.double().cpu() - ref["dweight"]).abs() <= ref["e_dweight"]).all()


def test_no_rows(dev):
    x = torch.zeros(0, 96, dtype=BF, device=dev)
    w, b = torch.ones(96, device=dev), torch.ones(96, device=dev)
    got = _step(dev, x, x, w, b, 1e-5)
    assert got["y"].shape == (0, 96) and got["dx"].shape == (0, 96)
    assert (got["dweight"] == 0).all() and (got["dbias"] == 0).all()


def test_statistics_and_a_far_mean(dev):
    """The variance is that of the differences: a mean of 1000 standard deviations costs the rounding of the mean alone."""
    gen = torch.Generator().manual_seed(8)
    for n in (64, 1000, 4096):
        x = torch.randn(40, n, generator=gen) + 1000.0
        y, mean, rstd = layer_norm(x.to(dev), eps=1e-5, return_stats=True)
        ref = orc.layer_norm(x, None, None, 1e-5, dtype=F32)
        _check(dict(y=y, mean=mean, rstd=rstd), ref, ("y", "mean", "rstd"))


def test_constant_rows(dev):
    x = torch.full((9, 128), 3.0, dtype=BF, device=dev)
    got = _step(dev, x, torch.ones_like(x), torch.ones(128, device=dev), torch.full((128,), 0.5, device=dev), 1e-5)
    assert (got["y"] == 0.5).all() and (got["dx"] == 0).all() and (got["dweight"] == 0).all() and (got["dbias"] == 9).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [14, 28, 56, 97, 1001, 3584, 7168, 16383])
def test_constant_rows_at_any_width(dev, n, dtype):
    """1 / n is no binary number: the mean is the rows' value all the same, and the differences from it vanish.  The first mean is
    off by MEAN of the value c, what is left of that by MEAN again, and eps = 1e-6 makes 1000 times that of it."""
    value = torch.tensor([3.0, 50.0, 100.0, 1000.0, -0.0078125, 0.0]).to(dtype)
    x = value[:, None].expand(6, n).contiguous().to(dev)
    y, mean, rstd = layer_norm(x, eps=1e-6, return_stats=True)
    assert torch.equal(mean.cpu(), value.float())
    assert (y.double().cpu().abs() <= orc.WIDEN * 1000 * orc.MEAN ** 2 * value.double().abs()[:, None]).all()
    gen = torch.Generator().manual_seed(n)
    dy = torch.randn(6, n, generator=gen).to(dtype)
    dx, dw, _ = layer_norm_backward(dy.to(dev), x, None, mean, rstd)
    assert (dw == 0).all()
    _check(dict(dx=dx), orc.layer_norm(x.cpu(), None, None, 1e-6, dy, dtype), ("dx",))


@pytest.mark.parametrize("n", [97, 1001, 3584, 7168, 16383])
def test_a_far_mean_and_a_small_spread(dev, n):
    """Rows of 1000 +- 0.05: the forward holds their mean to more than 32 bits, the backward to those."""
    gen = torch.Generator().manual_seed(n)
    x, dy = 1000.0 + 0.05 * torch.randn(12, n, generator=gen), torch.randn(12, n, generator=gen)
    w, b = (1 + 0.3 * torch.randn(n, generator=gen)), torch.randn(n, generator=gen)
    _run(dev, x, dy, w, b, eps=1e-6)


@pytest.mark.parametrize("n", [4096, 16384])
def test_small_elements_behind_a_large_one(dev, n):
    """Rows with 64 elements a lane: one of them 1, whose square swallows each of 63 squares of just below half its last step where
    they are added to it one by one."""
    col = torch.arange(n)
    x = torch.where((col < n // 8) & (col % 8 == 0), 1.0, (0.99 * 2.0 ** -24) ** 0.5) * torch.where((col // 8) % 2 == 0, 1.0, -1.0)
    x = x.repeat(5, 1)
    y, mean, rstd = layer_norm(x.to(dev), eps=1e-9, return_stats=True)
    _check(dict(y=y, mean=mean, rstd=rstd), orc.layer_norm(x, None, None, 1e-9, dtype=F32), ("y", "mean", "rstd"))


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("n", [64, 640, 3000])
def test_a_row_that_is_not_finite(dev, n, what):
    """It stays with its row in y and dx."""
    gen = torch.Generator().manual_seed(n)
    x, dy, w, b = _inputs(gen, 40, n, BF, F32)
    ref = orc.layer_norm(x, w, b, 1e-5, dy)
    x[17, n // 2] = what
    got = _step(dev, *(t.to(dev) for t in (x, dy, w, b)), 1e-5)
    keep = torch.arange(40) != 17
    _check({k: got[k][keep.to(dev)] for k in ("y", "dx")}, {k: v[keep] for k, v in ref.items() if k in ("y", "dx", "e_y", "e_dx")}, ("y", "dx"))
    assert got["y"][17].isnan().all() and got["dx"][17].isnan().all()


def test_wanted_gradients_alone(dev):
    gen = torch.Generator().manual_seed(2)
    x, dy, w, b = (t.to(dev) for t in _inputs(gen, 300, 640, BF, F32))
    y, mean, rstd = layer_norm(x, w, b, return_stats=True)
    full = layer_norm_backward(dy, x, w, mean, rstd)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        part = layer_norm_backward(dy, x, w, mean, rstd, need)
        for k, a, e in zip(need, part, full):
            assert (a is None) if not k else torch.equal(a, e)
    again = layer_norm_backward(dy, x, w, mean, rstd)
    assert all(torch.equal(a, e) for a, e in zip(again, full))     # the same bits


def test_on_another_stream_and_in_a_graph(dev):
    """A step captured and replayed on new data beside eager steps of the same leaves."""
    gen = torch.Generator().manual_seed(6)
    x, dy, w, b = (t.to(dev) for t in _inputs(gen, 600, 128, BF, BF))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(dev, x, dy, w, b, 1e-5)
    torch.cuda.current_stream().wait_stream(side)
    eager = _step(dev, x, dy, w, b, 1e-5)
    assert all(torch.equal(got[k], eager[k]) for k in eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(dev, x, dy, w, b, 1e-5)
    for i in range(4):
        x.copy_(torch.randn(600, 128, generator=gen).to(BF))
        graph.replay()
        eager = _step(dev, x, dy, w, b, 1e-5)
        torch.cuda.synchronize()
        assert all(torch.equal(held[k], eager[k]) for k in eager), i


def test_capture_beside_a_living_graph(dev):
    """Captured on leaves of its own while an eager graph of the same tensors waits for its backward."""
    gen = torch.Generator().manual_seed(16)
    x, dy, w, b = (t.to(dev) for t in _inputs(gen, 200, 64, BF, F32))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    living = LayerNorm.apply(*leaves, 1e-5)
    _step(dev, leaves[0], dy, leaves[1], leaves[2], 1e-5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(dev, leaves[0], dy, leaves[1], leaves[2], 1e-5)
    graph.replay()
    living.backward(dy)
    torch.cuda.synchronize()
    for name, t in zip(("dx", "dweight", "dbias"), leaves):
        assert torch.equal(held[name], t.grad)


def test_second_gradients_are_refused(dev):
    x = torch.randn(4, 64, device=dev, requires_grad=True)
    (g,) = torch.autograd.grad(LayerNorm.apply(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("of", ["x", "weight", "bias"])
def test_a_penalty_on_a_gradient_is_refused_not_dropped(dev, of):
    """The gradient hangs on x and weight though the upstream one hangs on nothing; its values are those without create_graph."""
    x, w, b = torch.randn(4, 64, device=dev, requires_grad=True), torch.ones(64, device=dev, requires_grad=True), torch.zeros(64, device=dev, requires_grad=True)
    leaf = dict(x=x, weight=w, bias=b)[of]
    up = torch.randn(4, 64, device=dev)
    (plain,) = torch.autograd.grad(LayerNorm.apply(x, w, b), leaf, up)
    assert not plain.requires_grad
    (g,) = torch.autograd.grad(LayerNorm.apply(x, w, b), leaf, up, create_graph=True)
    assert torch.equal(g, plain) and g.requires_grad
    with pytest.raises(RuntimeError, match="second gradients"):
        (g.square().sum() + x.square().sum()).backward()
    fixed = x.detach()
    (g,) = torch.autograd.grad(LayerNorm.apply(fixed, None, b), b, up, create_graph=True)
    assert not g.requires_grad                                        # of nothing that asks for a gradient
    (g.square().sum() + b.square().sum()).backward()
    assert (b.grad == 0).all()


def test_in_front_of_the_indexer(dev):
    """Normed keys through the indexer's scores and loss: the gradient reaches the norm's weight and its input."""
    gen = torch.Generator().manual_seed(11)
    s, h, d = 96, 16, 64
    x = torch.randn(s, 1, d, generator=gen).to(BF).to(dev).requires_grad_()
    w, b = torch.ones(d, device=dev, requires_grad=True), torch.zeros(d, device=dev, requires_grad=True)
    q, wt = torch.randn(s, 1, h, d, generator=gen).to(BF).to(dev), torch.randn(s, 1, h, generator=gen).to(dev)
    k = LayerNorm.apply(x, w, b, 1e-6)
    scores = cppmega_amd.IndexScores.apply(q, wt, k, True, 2)
    up = torch.randn(1, s, s, generator=gen).to(dev).tril()
    scores.backward(torch.where(up.isfinite(), up, 0))
    _, _, dk = cppmega_amd.index_scores_backward(up, q, wt, k.detach(), causal=True)
    ref = orc.layer_norm(x.detach().cpu()[:, 0], w.detach().cpu(), b.detach().cpu(), 1e-6, dk.cpu()[:, 0])
    _check(dict(dx=x.grad[:, 0], dweight=w.grad, dbias=b.grad), ref, ("dx", "dweight", "dbias"))
