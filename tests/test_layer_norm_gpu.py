"""layer_norm (bpt_layer_norm_forward / _backward) against the formula in 64 bits on the same inputs.

Tolerances, with u = 2^-24.  a = x + r is rounded once; a row's mean and variance are fp32 sums of at most 16 terms a
thread and 9 levels above, so with S = max|a| rstd the normalised n is off by at most 32 u S and rstd by 32 u S of
itself.  With Q = max|gy w| and N = max|n| of the row that gives, to first order,
    y:  32 u S (N + 1) max|w|          da: 32 u S rstd Q (2 + 2 N)
    dw: sum over rows of 32 u S (1 + |n|) |gy|, and the rounding of the sum
each plus half a step of the output's type.  The sums over rows are chains of at most 128 additions (rows of a thread,
rows of a block, partial rows of a column): 128 u times the sum of the absolute terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
FP32 = 2.0 ** -19  # 32 u
CHAIN = 128 * 2.0 ** -24


def inputs(rows, dim, dtype, residual, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = (rnd(rows, dim) * 1.5 + 0.3).to(dtype)
    r = rnd(rows, dim).to(dtype) if residual else None
    w = (1 + 0.2 * rnd(dim)).to(dtype)
    b = (0.2 * rnd(dim)).to(dtype)
    gy = rnd(rows, dim).to(dtype)
    return x, r, w, b, gy


def formula(x, r, w, b, gy, eps):
    """(y, da, dw, db) in 64 bits and what each may be off by before it is rounded to its type."""
    a = x.double() if r is None else x.double() + r.double()
    one = torch.ones(x.size(-1), dtype=torch.float64, device=x.device)
    wd, bd = one if w is None else w.double(), 0 * one if b is None else b.double()
    c = a - a.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    n = c * rstd
    g = gy.double()
    q = g * wd
    da = rstd * (q - q.mean(-1, keepdim=True) - n * (q * n).mean(-1, keepdim=True))
    top = lambda t: t.abs().amax(-1, keepdim=True)
    S, N = top(a) * rstd + 1, top(n)
    off = (FP32 * S * (N + 1) * wd.abs().max() + FP32 * top(bd), FP32 * S * rstd * top(q) * (2 + 2 * N),
           (FP32 * S * (1 + n.abs()) * g.abs()).sum(0) + CHAIN * (g * n).abs().sum(0), CHAIN * g.abs().sum(0))
    return (n * wd + bd, da, (g * n).sum(0), g.sum(0)), off


def near(got, want, slack):
    """|got - want| <= half a step of got's type + slack."""
    info = torch.finfo(got.dtype)
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((off <= info.eps / 2 * (want.abs() + slack) + slack + info.smallest_normal * info.eps).all()), \
        float((off - info.eps / 2 * want.abs() - slack).max())


def check(x, r, w, b, gy, eps=1e-5):
    from bpt_b200.norm import layer_norm
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, r, w, b)]  # the same memory
    y = layer_norm(leaves[0], leaves[2], leaves[3], eps, residual=leaves[1])
    assert y.dtype == x.dtype and y.shape == x.shape
    with torch.no_grad():  # without gradients: the same values
        assert torch.equal(layer_norm(x, w, b, eps, residual=r), y)
    y.backward(gy)
    want, off = formula(x, r, w, b, gy, eps)
    near(y.detach(), want[0], off[0])
    near(leaves[0].grad, want[1], off[1])
    if r is not None:
        assert torch.equal(leaves[0].grad, leaves[1].grad)
    if w is not None:
        near(leaves[2].grad, want[2], off[2])
    if b is not None:
        near(leaves[3].grad, want[3], off[3])
    return [None if t is None else t.grad for t in leaves]


# widths on both sides of every layout switch: pieces of 8, 4 and 1, 32 to 512 threads a row
@pytest.mark.parametrize("dim", [2, 3, 8, 31, 36, 64, 300, 500, 512, 513, 520, 1000, 1024, 1028, 2047, 2048, 4096, 4100, 8191, 8192])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_and_gradients(dim, dtype):
    for rows, residual in ((1, True), (7, False), (70, True)):
        check(*inputs(rows, dim, dtype, residual, seed=dim + rows))


# widths that are even, but no multiple of 4: pieces of 2
@pytest.mark.parametrize("dim", [6, 62, 130, 254, 370, 474, 514, 1026, 1330, 4098, 8190])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pairs(dim, dtype):
    for rows, residual in ((1, True), (9, False), (2500 if dim < 1000 else 300, True)):
        check(*inputs(rows, dim, dtype, residual, seed=dim + rows))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(dtype):
    """More rows than the grid holds at once: every block loops, and the last round is ragged."""
    check(*inputs(20011, 512, dtype, True))
    check(*inputs(5003, 1100, dtype, False))


@pytest.mark.parametrize("dtype", DTYPES)
def test_bitwise_reproducible(dtype):
    args = inputs(9001, 300, dtype, True)
    first, second = check(*args), check(*args)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_width_one_and_constant_rows():
    """One element a row, or equal ones: the variance is 0, y is the bias, and the gradient of x is 0 by the formula
    (q - mean q = 0 for one element; finite for constant rows)."""
    from bpt_b200.norm import layer_norm
    x, r, w, b, gy = inputs(33, 1, torch.float32, False)
    xl = x.clone().requires_grad_(True)
    y = layer_norm(xl, w, b)
    assert torch.equal(y, b.expand_as(y).clone())
    y.backward(gy)
    assert torch.equal(xl.grad, torch.zeros_like(x))
    c = torch.full((5, 64), 2.0, device="cuda")
    y = layer_norm(c, None, None)
    assert torch.equal(y, torch.zeros_like(y))


@pytest.mark.parametrize("dtype", DTYPES)
def test_optional_arguments(dtype):
    x, r, w, b, gy = inputs(50, 300, dtype, True)
    check(x, r, None, None, gy)
    check(x, None, w, None, gy)
    check(x, r, None, b, gy)


def test_only_some_gradients():
    from bpt_b200.norm import layer_norm
    x, r, w, b, gy = inputs(200, 512, torch.bfloat16, True)
    full = check(x, r, w, b, gy)
    for which in range(4):
        leaves = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, r, w, b))]
        layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1]).backward(gy)
        for i, t in enumerate(leaves):
            assert (t.grad is None) == (i != which)
        assert torch.equal(leaves[which].grad, full[which])


def test_no_rows():
    from bpt_b200.norm import layer_norm
    x, r, w, b, gy = [t.requires_grad_(True) for t in inputs(0, 512, torch.bfloat16, True)]
    y = layer_norm(x, w, b, residual=r)
    assert y.shape == (0, 512)
    y.backward(torch.empty_like(y))
    assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b)) and x.grad.shape == x.shape


def test_strides_and_alignment():
    """Transposed, sliced and expanded inputs, and contiguous ones that start off a 16-byte boundary."""
    from bpt_b200.norm import layer_norm
    for dtype in DTYPES:
        x, r, w, b, gy = inputs(96, 64, dtype, True)
        want = layer_norm(x, w, b, residual=r)
        assert torch.equal(layer_norm(x.t().contiguous().t(), w, b, residual=r), want)
        wide = torch.cat([x, x], 1)
        assert torch.equal(layer_norm(wide[:, :64], w, b, residual=r), want)
        for shift in (1, 2, 4):
            buf = torch.empty(96 * 64 + 8, dtype=dtype, device="cuda")
            moved = buf[shift:shift + 96 * 64].view(96, 64)
            moved.copy_(x)
            got = check(moved, r, w, b, gy)
            for a, e in zip(got, check(x, r, w, b, gy)):
                assert torch.allclose(a.float(), e.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-4)
        grad = torch.zeros((), dtype=dtype, device="cuda").expand(96, 64)  # an expanded gradient, stride 0
        xl = x.clone().requires_grad_(True)
        layer_norm(xl, w, b).backward(grad)
        assert torch.equal(xl.grad, torch.zeros_like(x))
        batch = layer_norm(x.view(2, 6, 8, 64), w, b, residual=r.view(2, 6, 8, 64))
        assert torch.equal(batch.view(96, 64), want)


def test_large_mean_and_nonfinite_rows_stay_to_themselves():
    from bpt_b200.norm import layer_norm
    x, _, w, b, _ = inputs(64, 512, torch.float32, False)
    want = layer_norm(x, w, b)
    bad = x.clone()
    bad[3, 5] = float("nan")
    bad[10, 0] = float("inf")
    got = layer_norm(bad, w, b)
    rows = [i for i in range(64) if i not in (3, 10)]
    assert torch.equal(got[rows], want[rows])
    assert bool(torch.isnan(got[3]).all()) and bool(torch.isnan(got[10]).any())
    # a mean 1000 times the spread: the variance is taken about the mean, so what is left is the inputs' own rounding
    far = x + 1000.0
    got = layer_norm(far, None, None).double()
    exact = formula(far, None, None, None, far, 1e-5)[0][0]
    assert float((got - exact).abs().max()) < 2e3 * 16 * 2.0 ** -24  # |mean| rstd * 16 u


def test_gradient_against_differences():
    """<dL/dx, d> against (L(x + h d) - L(x - h d)) / 2h of the formula in 64 bits, L = <y, gy>."""
    x, r, w, b, gy = inputs(6, 40, torch.float32, True)
    got = check(x, r, w, b, gy)
    gen = torch.Generator(device="cuda").manual_seed(9)
    h = 1e-4
    for i, t in enumerate((x, r, w, b)):
        d = torch.randn(t.shape, generator=gen, device="cuda", dtype=torch.float64)
        loss = []
        for s in (h, -h):
            moved = [u.double() for u in (x, r, w, b)]
            moved[i] = moved[i] + s * d
            loss.append(float((formula(*moved, gy, 1e-5)[0][0] * gy.double()).sum()))
        diff = (loss[0] - loss[1]) / (2 * h)
        scale = float((got[i].double() * d).abs().sum())
        # the difference is off by h^2 times a third derivative (order 10): 1e-7 of the scale; the gradient by a few 32 u
        assert abs(float((got[i].double() * d).sum()) - diff) < 4e-5 * scale


def test_other_stream_device_guard_and_graph():
    from bpt_b200.norm import layer_norm
    x, r, w, b, gy = inputs(3000, 512, torch.bfloat16, True)
    want = layer_norm(x, w, b, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer_norm(x, w, b, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # a whole forward + backward captured and replayed with new inputs
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w, b)]

    def step():
        y = layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
        return (y.detach(),) + torch.autograd.grad(y, leaves, gy)

    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        leaves[0].mul_(0.5)
        gy.mul_(2.0)
    graph.replay()
    again = [t.clone() for t in out]
    eager = step()
    assert all(torch.equal(a, e) for a, e in zip(again, eager))


def test_refusals():
    from bpt_b200.norm import layer_norm
    x, r, w, b, _ = inputs(4, 16, torch.bfloat16, True)
    for bad in (dict(weight=w.float()), dict(bias=b[:8]), dict(residual=r[:2]), dict(residual=r.float()), dict(weight=w.cpu()),
                dict(x=x.double()), dict(x=torch.empty(2, 8193, device="cuda", dtype=torch.bfloat16)),
                dict(x=torch.empty(2, 0, device="cuda", dtype=torch.bfloat16)), dict(x=x.cpu())):
        a = dict(x=x, weight=w, bias=b, residual=r)
        a.update(bad)
        if "x" in bad:
            a.update(weight=None, bias=None, residual=None)
        with pytest.raises(RuntimeError, match="bpt_b200"):
            layer_norm(a["x"], a["weight"], a["bias"], residual=a["residual"])
    y = layer_norm(x.clone().requires_grad_(True), w, b)
    first = torch.autograd.grad(y.sum(), [y], create_graph=True)  # the first derivative is fine to ask for
    assert first[0] is not None


def test_blocks_train_through_it():
    """Blocks at two widths: gradients of every parameter against torch's layer norm."""
    from bpt_b200 import csr as csrmod, graphbuilder
    from bpt_b200 import model as models
    from bpt_b200.attention import AttentionPlan
    for dim, heads in ((128, 4), (512, 8)):
        torch.manual_seed(0)
        batch = csrmod.batch_graphs([graphbuilder.BinaryPartition(100, True, 4, 6)])
        plan = AttentionPlan.from_batch(batch, n_etypes=1000)
        blk = models.BPTBlock(dim, heads, 2 * dim, rel_pos=True, drop_h=0.0).cuda()
        h = torch.randn(batch.n_nodes, dim, device="cuda")
        gy = torch.randn(batch.n_nodes, dim, device="cuda")
        blk(h, plan).backward(gy)
        got = {k: p.grad.clone() for k, p in blk.named_parameters()}
        blk.zero_grad()
        kept = models.add_layer_norm
        models.add_layer_norm = lambda a, r, norm: norm(a + r)
        try:
            blk(h, plan).backward(gy)
        finally:
            models.add_layer_norm = kept
        for k, p in blk.named_parameters():
            assert float((p.grad - got[k]).abs().max()) <= 1e-4 * float(p.grad.abs().max()), k


def test_second_derivative_is_refused():
    """create_graph may be asked for (other parts of a model may need it); the derivative of this backward is an error."""
    from bpt_b200.loss import linear_cross_entropy
    from bpt_b200.norm import layer_norm
    x, r, w, b, _ = inputs(4, 16, torch.float32, True)
    x.requires_grad_(True)
    t = torch.zeros(4, dtype=torch.long, device="cuda")
    for f in (lambda: layer_norm(x, w, b, residual=r).square().sum(), lambda: linear_cross_entropy(x, r.detach(), t)):
        plain, = torch.autograd.grad(f(), x)
        g, = torch.autograd.grad(f(), x, create_graph=True)
        assert torch.equal(g.detach(), plain)
        with pytest.raises(RuntimeError, match="once"):
            g.sum().backward()
