"""linear_cross_entropy (bpt_linear_ce_forward / _backward) against the formula in 64 bits on the same inputs.

Tolerances (u = 2^-24; h = half a step of the operands' type relative to the value: 2^-8 bf16, 2^-11 fp16).
Logits: exact products summed in fp32, 16 at a time; each of the D / 16 (+ a few) additions is off by at most a step
2 u of the partial sum, which is at most A = max over cells of sum |x w| + |b|:  Ez = (D / 16 + 16) 2 u A.  For fp32 the
plane products that are left out and the roundings of the other planes stay below 16 of these steps as well.
Probabilities: exp is good to 2^-20 with its argument's rounding (|z log2 e| below 64), and the row's lse is off by no
more than Ez + 2^-20 max(1, |lse|):  Ep = 2 Ez + 2^-19 relative.  The loss is off by 2 Ez + 2^-20 max(1, |lse|, |loss|).
The gradient of a logit: Ep p, and for 16-bit operands its rounding h |dz| (half a step of the sum of both for the
target).  Products over V or N cells: those errors with absolute values of the other operand, and the fp32 sum's own
(K / 16 + 16) 2 u sum |terms|.  Each result is then rounded to its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24
IGNORE = -100


def inputs(n, vocab, dim, dtype, bias=True, padded=0.0, seed=0, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = rnd(n, dim).to(dtype)
    w = (rnd(vocab, dim) * spread / dim ** 0.5).to(dtype)
    b = (0.2 * rnd(vocab)).to(dtype) if bias else None
    t = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
    if padded:
        t = torch.where(torch.rand(n, generator=gen, device="cuda") < padded, torch.full_like(t, IGNORE), t)
    return x, w, b, t


def formula(x, w, b, t, smoothing, reduction, grad):
    """Values (loss, dx, dw, db) in 64 bits and what each may be off by before its own rounding."""
    n, vocab, dim = x.size(0), w.size(0), x.size(1)
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    A = float((xd.abs() @ wd.abs().t()).max())
    if b is not None:
        z = z + b.double()
        A += float(b.double().abs()[torch.isfinite(b)].max())
    counted = t != IGNORE
    at = torch.where(counted, t, torch.zeros_like(t)).unsqueeze(1)
    lse = torch.logsumexp(z, 1)
    row = lse - (1 - smoothing) * z.gather(1, at).squeeze(1)
    if smoothing:
        row = row - smoothing * z.mean(1)
    row = torch.where(counted, row, torch.zeros_like(row))
    count = counted.sum().double()
    loss = row if reduction == "none" else row.sum() if reduction == "sum" else row.sum() / count
    Ez = (dim / 16 + 16) * 2 * U * A
    Erow = (2 * Ez + 2.0 ** -20 * torch.maximum(lse.abs(), row.abs()).clamp(min=1)) * counted
    Eloss = Erow if reduction == "none" else Erow.sum() if reduction == "sum" else Erow.sum() / count
    g = grad.double() if reduction == "none" else grad.double().expand(n) / (count if reduction == "mean" else 1)
    g = torch.where(counted, g, torch.zeros((), device=x.device, dtype=torch.float64))
    p = torch.exp(z - lse.unsqueeze(1))
    dz = p - smoothing / vocab
    dz.scatter_add_(1, at, torch.full((n, 1), -(1 - smoothing), device=x.device, dtype=torch.float64))
    h = 0.0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
    G = g.abs().unsqueeze(1)
    Edz = ((2 * Ez + 2.0 ** -19) * p + h * dz.abs()) * G
    if x.dtype == torch.float16:
        Edz = Edz + 2.0 ** -39 * g.abs().max()  # half the smallest number of the type, which is kept times 2^14
    dz = dz * g.unsqueeze(1)
    cells = dz.abs()
    Edx = Edz @ wd.abs() + (vocab / 16 + 16) * 2 * U * (cells @ wd.abs())
    Edw = Edz.t() @ xd.abs() + (n / 16 + 16) * 2 * U * (cells.t() @ xd.abs())
    Edb = Edz.sum(0) + (n / 16 + 16) * 2 * U * cells.sum(0)
    return (loss, dz @ wd, dz.t() @ xd, dz.sum(0)), (Eloss, Edx, Edw, Edb)


def near(got, want, slack, what):
    info = torch.finfo(got.dtype)
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), what
    off = (got.double() - want).abs()
    most = info.eps / 2 * (want.abs() + slack) + slack + info.smallest_normal * info.eps
    assert bool((off <= most).all()), (what, float((off / most).max()))


def check(x, w, b, t, smoothing=0.0, reduction="mean", grad=None, formula_inputs=None):
    """Values and gradients, and the forward alone; returns them."""
    from bpt_b200.loss import linear_cross_entropy
    if grad is None:
        grad = torch.ones((), device="cuda")
    leaves = [None if v is None else v.detach().requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], ignore_index=IGNORE, label_smoothing=smoothing,
                                reduction=reduction)
    assert loss.dtype == torch.float32
    with torch.no_grad():
        alone = linear_cross_entropy(x, w, t, bias=b, ignore_index=IGNORE, label_smoothing=smoothing, reduction=reduction)
    assert torch.equal(alone, loss.detach())
    loss.backward(grad if reduction != "none" or grad.dim() else grad.expand(t.shape))
    grads = [None if v is None else v.grad for v in leaves]
    fx, ft = formula_inputs or (x, t)
    want, off = formula(fx, w, b, ft, smoothing, reduction, grad if reduction != "none" or grad.dim() else grad.expand(t.shape))
    near(loss.detach(), want[0], off[0], "loss")
    for name, got, v, e in zip(("dx", "dw", "db"), grads, want[1:], off[1:]):
        if got is not None:
            assert got.dtype == x.dtype
            near(got, v, e, name)
    return loss.detach(), grads


SHAPES = [(1, 1, 1), (1, 50, 8), (3, 2, 16), (5, 17, 24), (64, 256, 64), (128, 256, 64), (129, 257, 65), (127, 255, 63),
          (200, 1000, 300), (130, 513, 512), (300, 5000, 72), (1, 50257, 64), (777, 1001, 40), (256, 128, 1030), (2, 33, 7)]


@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_and_gradients(shape, dtype):
    n, vocab, dim = shape
    check(*inputs(n, vocab, dim, dtype, seed=n + vocab + dim))
    check(*inputs(n, vocab, dim, dtype, bias=False, padded=0.3 if n > 8 else 0.0, seed=vocab), smoothing=0.1, reduction="sum")
    gen = torch.Generator(device="cuda").manual_seed(7)
    check(*inputs(n, vocab, dim, dtype, seed=dim), smoothing=0.25, reduction="none",
          grad=torch.randn(n, generator=gen, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2100, 20000, 64), (20000, 2100, 64), (34000, 4000, 32), (12000, 12000, 40), (6000, 40000, 32),
                                   (40000, 6000, 32), (20, 300000, 16), (300000, 20, 16)])
def test_pieces(shape, dtype):
    """More cells than are kept at a time: the vocabulary is cut, the tokens are, and both; few, many and all but a few of
    the tokens ignored, so that a piece has fewer tokens than it was planned for, or none."""
    check(*inputs(*shape, dtype, padded=0.1), smoothing=0.1)
    if shape[0] * shape[1] > 1.4e8:
        x, w, b, t = inputs(*shape, dtype, padded=0.7)
        check(x, w, b, t)
        t[3:-2] = IGNORE
        t[0] = t[-1] = 1
        check(x, w, b, t, reduction="sum")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_millions_of_tokens(dtype, reduction):
    """More than the blocks that list the tokens have at 256 each: they go through theirs in turns."""
    n = 2 * 1048576 + 77
    x, w, b, t = inputs(n, 5, 8, dtype, padded=0.3, seed=11)
    grad = torch.linspace(0.5, 1.5, n, device="cuda") if reduction == "none" else None
    check(x, w, b, t, reduction=reduction, grad=grad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_bitwise_reproducible(dtype):
    args = inputs(3001, 12345, 128, dtype, padded=0.2)
    first, second = check(*args), check(*args)
    assert torch.equal(first[0], second[0])
    assert all(torch.equal(a, b) for a, b in zip(first[1], second[1]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 65])
def test_ignored_rows_may_hold_anything(dtype, dim):
    """NaN, infinities and huge numbers in the rows of ignored tokens: the same loss and gradients as with zeros there,
    and exact zeros in their rows of dx.  Both where x is read in place (64) and where it is copied (65, fp32)."""
    x, w, b, t = inputs(700, 300, dim, dtype, padded=0.4)
    t[64:200] = IGNORE  # whole blocks of 64 and more
    ignored = t == IGNORE
    clean = torch.where(ignored.unsqueeze(1), torch.zeros_like(x), x)
    dirty = clean.clone()
    junk = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max], device="cuda", dtype=dtype)
    dirty[ignored] = junk[torch.arange(dim, device="cuda") % 4]
    for reduction in ("mean", "sum", "none"):
        want, wg = check(clean, w, b, t, reduction=reduction)
        got, gg = check(dirty, w, b, t, reduction=reduction, formula_inputs=(clean, t))
        assert torch.equal(want, got) and all(torch.equal(a, e) for a, e in zip(gg, wg))
        assert bool((gg[0][ignored] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_counts(dtype):
    """Every target ignored: the sum is 0, the mean 0 / 0, the gradients are zero; and no tokens at all."""
    from bpt_b200.loss import linear_cross_entropy
    for n in (0, 70):
        x, w, b, t = [v.requires_grad_(True) if v.is_floating_point() else v for v in inputs(n, 90, 48, dtype)]
        t = torch.full_like(t, IGNORE)
        for reduction in ("mean", "sum", "none"):
            loss = linear_cross_entropy(x, w, t, bias=b, reduction=reduction)
            if reduction == "mean":
                assert bool(torch.isnan(loss))
            else:
                assert bool((loss == 0).all()) and loss.numel() == (1 if reduction == "sum" else n)
            for got, v in zip(torch.autograd.grad(loss.sum(), (x, w, b)), (x, w, b)):
                assert torch.equal(got, torch.zeros_like(v))


def test_target_out_of_range_says_so():
    from bpt_b200.loss import linear_cross_entropy
    x, w, b, t = inputs(200, 300, 64, torch.bfloat16)
    for wrong in (300, -1, -99, 2 ** 40, -2 ** 40):
        bad = t.clone()
        bad[17] = wrong
        rows = linear_cross_entropy(x, w, bad, bias=b, reduction="none")
        assert bool(torch.isnan(rows[17])) and int(torch.isnan(rows).sum()) == 1
        xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(xl, wl, bad, bias=b)
        loss.backward()
        assert bool(torch.isnan(loss)) and bool(torch.isnan(xl.grad[17]).all()) and bool(torch.isnan(wl.grad).all())
        assert bool(torch.isfinite(xl.grad[16]).all())
    # another ignore_index, also one that is a class
    for index in (5, -1, 299):
        moved = torch.where(t % 3 == 0, torch.full_like(t, index), t)
        got = linear_cross_entropy(x, w, moved, bias=b, ignore_index=index)
        want = torch.nn.functional.cross_entropy(x.double() @ w.double().t() + b.double(), moved, ignore_index=index)
        assert abs(float(got) - float(want)) < 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_classes_and_large_logits(dtype):
    """A bias of -inf takes classes out (probability and gradient 0); logits in the thousands do not overflow."""
    x, w, b, t = inputs(150, 400, 64, dtype)
    b[200:] = -float("inf")
    b[:3] = -float("inf")
    t = t % 190 + 5
    from bpt_b200.loss import linear_cross_entropy
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    loss.backward()
    keep = torch.arange(400, device="cuda")
    keep = (keep >= 3) & (keep < 200)
    want, grads = check(x, w[keep].contiguous(), b[keep].contiguous(), t - 3)
    assert abs(float(loss) - float(want)) <= 2e-6 * float(want)
    assert bool((leaves[1].grad[~keep] == 0).all()) and bool((leaves[2].grad[~keep] == 0).all())
    assert bool(torch.isfinite(leaves[0].grad).all())
    big = inputs(150, 400, 64, dtype, spread=800.0)
    loss = linear_cross_entropy(big[0], big[1], big[3], bias=big[2])
    exact = torch.nn.functional.cross_entropy(big[0].double() @ big[1].double().t() + big[2].double(), big[3])
    # Ez of the module's note for logits up to 4000: (4 + 16) 2 u 2e4 = 0.05
    assert abs(float(loss) - float(exact)) < 0.1


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_alignment_and_shapes(dtype):
    x, w, b, t = inputs(96, 200, 64, dtype, padded=0.2)
    want, grads = check(x, w, b, t)

    def same(got):  # the same numbers went in; a copied operand takes the same tiles
        assert torch.equal(got[0], want) and all(torch.equal(a, e) for a, e in zip(got[1], grads))

    wide = lambda v, extra: torch.cat([v, torch.full((v.size(0), extra), float("nan"), dtype=dtype, device="cuda")], 1)[:, :v.size(1)]
    same(check(wide(x, 8), wide(w, 16), b, t))   # rows apart, still on 16 bytes
    same(check(wide(x, 3), wide(w, 5), b, t))    # rows off 16 bytes
    same(check(x.t().contiguous().t(), w.t().contiguous().t(), b, t))
    buf = torch.empty(200 * 64 + 1, dtype=dtype, device="cuda")
    moved = buf[1:].view(200, 64)
    moved.copy_(w)
    same(check(x, moved, b, t))
    same(check(x, w, torch.stack([b, b], 1)[:, 0], t))
    from bpt_b200.loss import linear_cross_entropy
    t2 = torch.stack([t, t], 1)[:, 0]
    assert torch.equal(linear_cross_entropy(x, w, t2, bias=b), want)
    folded = linear_cross_entropy(x.view(4, 24, 64), w, t.view(4, 24), bias=b, reduction="none")
    assert folded.shape == (4, 24)
    assert torch.equal(folded.view(-1), linear_cross_entropy(x, w, t, bias=b, reduction="none"))
    one = linear_cross_entropy(x[3], w, t[3], bias=b, reduction="sum")
    assert torch.equal(one, linear_cross_entropy(x[3:4], w, t[3:4], bias=b, reduction="sum"))
    row = x[:1].expand(96, 64)  # stride 0: broadcast features, gradients summed by autograd
    leaf = x[:1].detach().requires_grad_(True)
    linear_cross_entropy(leaf.expand(96, 64), w, t, bias=b).backward()
    _, got = check(row.contiguous(), w, b, t)
    ref = got[0].double().sum(0)
    assert float((leaf.grad.double() - ref).abs().max()) <= 96 * torch.finfo(dtype).eps * float(got[0].abs().sum(0).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2100, 22000, 32), (150, 700, 134), (40, 300, 72)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_that_start_anywhere(dtype, shape):
    """The library's own entry points: outputs off 16 bytes, in one piece and in several, with nothing written around them."""
    from bpt_b200 import _lib
    n, vocab, dim = shape
    x, w, b, t = inputs(n, vocab, dim, dtype, padded=0.2, seed=5)
    _, want = check(x, w, b, t, reduction="sum")
    L, code, p = _lib.lib(), _lib.dtype_code(dtype), lambda v: v.data_ptr()
    loss, lse, count, grad = (torch.empty(k, device="cuda") for k in (1, n, 1, 1))
    grad.fill_(1.0)
    size = L.bpt_linear_ce_forward_workspace_bytes(p(x), dim, p(w), dim, n, vocab, dim, code)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    _lib.check(L.bpt_linear_ce_forward(p(x), dim, p(w), dim, p(b), p(t), IGNORE, 0.0, 2, p(loss), p(lse), p(count), n, vocab, dim, code,
                                       p(ws), size, _lib.stream()))
    size = L.bpt_linear_ce_backward_workspace_bytes(p(x), dim, p(w), dim, n, vocab, dim, code, 1, 1, 1)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    for off in (1, 2, 3, 4):
        held = [torch.full((v.numel() + 16,), 7.0, dtype=dtype, device="cuda") for v in want]
        outs = [h[off:off + v.numel()] for h, v in zip(held, want)]
        _lib.check(L.bpt_linear_ce_backward(p(x), dim, p(w), dim, p(b), p(t), IGNORE, 0.0, 2, p(lse), p(count), p(grad), p(outs[0]),
                                            p(outs[1]), p(outs[2]), n, vocab, dim, code, p(ws), size, _lib.stream()))
        for h, o, v in zip(held, outs, want):
            assert torch.equal(o.view(v.shape), v)
            assert bool((h[:off] == 7.0).all()) and bool((h[off + v.numel():] == 7.0).all())


def test_only_some_gradients():
    from bpt_b200.loss import linear_cross_entropy
    x, w, b, t = inputs(500, 700, 128, torch.bfloat16, padded=0.1)
    _, full = check(x, w, b, t)
    for which in range(3):
        leaves = [v.detach().clone().requires_grad_(i == which) for i, v in enumerate((x, w, b))]
        linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2]).backward()
        assert [v.grad is None for v in leaves] == [i != which for i in range(3)]
        assert torch.equal(leaves[which].grad, full[which])


def test_gradients_of_zero_and_large_grad():
    """reduction none: a zero gradient, one of 2^40 and one of 2^-60 for all tokens; the scale is a power of two."""
    x, w, b, t = inputs(300, 500, 64, torch.bfloat16)
    _, one = check(x, w, b, t, reduction="none", grad=torch.ones(300, device="cuda"))
    for scale in (2.0 ** 40, 2.0 ** -60, 0.0):
        _, got = check(x, w, b, t, reduction="none", grad=torch.full((300,), scale, device="cuda"))
        assert all(torch.equal(a, e * scale) for a, e in zip(got, one))


def test_gradient_against_differences():
    """<dL/dv, d> against (L(v + h d) - L(v - h d)) / 2h of the loss in 64 bits."""
    x, w, b, t = inputs(40, 60, 24, torch.float32, padded=0.2)
    _, grads = check(x, w, b, t, smoothing=0.1)
    gen = torch.Generator(device="cuda").manual_seed(3)
    h = 1e-4
    for i in range(3):
        moved = [v.double() for v in (x, w, b)]
        d = torch.randn(moved[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        value = []
        for s in (h, -h):
            m = list(moved)
            m[i] = m[i] + s * d
            value.append(float(torch.nn.functional.cross_entropy(m[0] @ m[1].t() + m[2], t, label_smoothing=0.1)))
        diff = (value[0] - value[1]) / (2 * h)
        # h^2 times a third derivative of order 10: 1e-7; the gradients are good to a few 1e-6 of their terms
        assert abs(float((grads[i].double() * d).sum()) - diff) < 1e-5 * float((grads[i].double() * d).abs().sum()) + 1e-6


def test_streams_and_graphs():
    from bpt_b200.loss import linear_cross_entropy
    x, w, b, t = inputs(3000, 9000, 128, torch.bfloat16, padded=0.1)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]

    def step():
        loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], label_smoothing=0.1)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves)

    want = step()
    streams = [torch.cuda.Stream() for _ in range(3)]
    out = []
    for s in streams:  # calls that overlap on three streams
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out.append([step() for _ in range(3)])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for runs in out:
        for run in runs:
            assert all(torch.equal(a, e) for a, e in zip(run, want))
    del out
    # two graphs that share a memory pool, replayed in turn with new inputs
    with torch.cuda.stream(streams[0]):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(streams[0])
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        a = step()
    with torch.cuda.graph(second, pool=first.pool()):
        c = step()
    with torch.no_grad():
        leaves[0].mul_(0.5)
        t.copy_(t.flip(0))
    first.replay()
    got_a = [v.clone() for v in a]
    second.replay()
    got_c = [v.clone() for v in c]
    fresh = step()
    assert all(torch.equal(p, e) for p, e in zip(got_a, fresh)) and all(torch.equal(p, e) for p, e in zip(got_c, fresh))


@pytest.mark.parametrize("shape", [(6, 5194, 134, torch.float16, 0.0), (17599, 2078, 652, torch.float16, 0.12),
                                   (4099, 803, 300, torch.float32, 0.12), (700, 1000, 65, torch.bfloat16, 0.3),
                                   (3000, 900, 128, torch.bfloat16, 0.3), (100, 300, 40, torch.float32, 0.0)],
                         ids=lambda s: "x".join(map(str, s[:3])))
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_workspaces_that_held_something_else(shape, reduction):
    """Kernels of a call start before those ahead of them have ended: none may read what they are about to write.  The
    memory that the call's workspaces come from is filled just before it, calls follow each other without a wait."""
    from bpt_b200.loss import linear_cross_entropy
    n, vocab, dim, dtype, padded = shape
    states = [inputs(n, vocab, dim, dtype, padded=padded, seed=k) for k in (3, 4)]

    def step(x, w, b, t):
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], ignore_index=IGNORE, reduction=reduction)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves, torch.ones_like(loss))

    want = []
    for state in states:
        torch.cuda.synchronize()
        want.append(step(*state))
        torch.cuda.synchronize()
    checked, _ = check(*states[0], reduction=reduction, grad=torch.ones(n, device="cuda") if reduction == "none" else None)
    assert torch.equal(checked, want[0][0])
    size = 64 << 20
    for turn in range(24):
        for fill in (0, 255):  # a handful of blocks of every size class, back in the allocator when the call asks
            held = [torch.full((size >> k,), fill, dtype=torch.uint8, device="cuda") for k in range(0, 18, 2)]
            del held
            got = step(*states[turn % 2])
            assert all(torch.equal(a, e) for a, e in zip(got, want[turn % 2])), (turn, fill)


def test_refusals():
    from bpt_b200.loss import linear_cross_entropy
    x, w, b, t = inputs(10, 20, 16, torch.bfloat16)
    for bad in (dict(x=x.cpu()), dict(x=x.double(), w=w.double()), dict(w=w.float()), dict(w=w[:, :8]), dict(w=w.cpu()), dict(w=w[:0]),
                dict(b=b.float()), dict(b=b[:4]), dict(b=b.cpu()), dict(t=t.int()), dict(t=t[:4]), dict(t=t.cpu()),
                dict(reduction="max"), dict(smoothing=-0.5), dict(smoothing=1.5)):
        a = dict(x=x, w=w, b=b, t=t, reduction="mean", smoothing=0.0)
        a.update(bad)
        with pytest.raises(RuntimeError, match="bpt_b200"):
            linear_cross_entropy(a["x"], a["w"], a["t"], bias=a["b"], reduction=a["reduction"], label_smoothing=a["smoothing"])


def test_models_train_on_it():
    """The models' loss against nll_loss of their forward: value and every parameter's gradient (fp32)."""
    from bpt_b200 import csr as csrmod, graphbuilder
    from bpt_b200.attention import AttentionPlan
    from bpt_b200.model import BPTClassifier, BPTEncoderDecoder, BPTLanguageModel
    torch.manual_seed(0)
    lengths = [100, 37, 64]
    batch = csrmod.batch_graphs([graphbuilder.BinaryPartition(n, True, 4, 6) for n in lengths])
    plan = AttentionPlan.from_batch(batch, n_etypes=1000)
    tokens = torch.randint(0, 256, (sum(lengths),), device="cuda")
    target = torch.randint(0, 256, (sum(lengths),), device="cuda")
    target[5:20] = IGNORE

    def compare(model, loss, logp, target):
        got = loss()
        got.backward()
        mine = {k: p.grad.clone() for k, p in model.named_parameters()}
        model.zero_grad()
        want = torch.nn.functional.nll_loss(logp(), target, ignore_index=IGNORE)
        want.backward()
        assert abs(float(got) - float(want)) < 1e-5 * float(want)
        for k, p in model.named_parameters():
            assert float((p.grad - mine[k]).abs().max()) <= 1e-4 * float(p.grad.abs().max()) + 1e-9, k

    lm = BPTLanguageModel(256, 128, 256, 2, 2).cuda()
    compare(lm, lambda: lm.loss(tokens, batch.leaf_ids(), plan, target), lambda: lm(tokens, batch.leaf_ids(), plan), target)
    cls = BPTClassifier(256, 300, 600, 6, 2, 3, readout="mean").cuda()
    labels, lens = torch.tensor([0, 2, 1], device="cuda"), torch.tensor(lengths, device="cuda")
    compare(cls, lambda: cls.loss(tokens, batch.leaf_ids(), plan, batch.root_ids(), labels, lens),
            lambda: cls(tokens, batch.leaf_ids(), plan, batch.root_ids(), lens), labels)
    enc = csrmod.batch_graphs([graphbuilder.BinaryPartition(n, False, 2, 3) for n in (20, 33)])
    dec = csrmod.batch_graphs([graphbuilder.BinaryPartition(n, True, 2, 3) for n in (12, 25)])
    isrc, idst = csrmod.inter_graph([(enc.node_offsets[i], n) for i, n in enumerate((20, 33))],
                                    [(dec.node_offsets[i], n) for i, n in enumerate((12, 25))])
    mt = BPTEncoderDecoder([100, 1003], 128, 256, 2, 1, 1).cuda()
    args = (torch.randint(0, 100, (53,), device="cuda"), enc.leaf_ids(), AttentionPlan.from_batch(enc, n_etypes=1000),
            torch.randint(0, 1003, (37,), device="cuda"), dec.leaf_ids(), AttentionPlan.from_batch(dec, n_etypes=1000),
            AttentionPlan(isrc, idst, None, dec.n_nodes, n_src=enc.n_nodes), dec.leaf_ids())
    words = torch.randint(0, 1003, (37,), device="cuda")
    compare(mt, lambda: mt.loss(*args, words), lambda: mt(*args), words)
    smooth = mt.loss(*args, words, label_smoothing=0.1)
    with torch.no_grad():
        logp = mt(*args)
        want = -(0.9 * logp.gather(1, words.unsqueeze(1)).squeeze(1) + 0.1 * logp.mean(1)).mean()
    assert abs(float(smooth) - float(want)) < 1e-5 * float(want)


@pytest.mark.parametrize("spread", [0, 12, 24, 25, 40, 100])
@pytest.mark.parametrize("of", ["x", "w", "all"])
def test_fp32_rows_of_very_different_size(spread, of):
    """fp32 operands are split by what their rows' sizes allow: two scaled planes, or three with the whole range.  Each token's
    loss has to be as good as its own numbers allow (Ez with the row's own A), whatever the other rows are; and the
    gradients of a token of ordinary size have to be as good as in a batch of such tokens alone."""
    from bpt_b200.loss import linear_cross_entropy
    n, vocab, dim = 300, 500, 72
    x, w, b, t = inputs(n, vocab, dim, torch.float32)
    down = torch.ones(n, device="cuda", dtype=torch.float64)
    if of in ("x", "all"):
        down = 2.0 ** -(torch.arange(n, device="cuda", dtype=torch.float64) % (spread + 1))
        x = (x.double() * down.unsqueeze(1)).float()
    if of in ("w", "all"):
        w = (w.double() * 2.0 ** -(torch.arange(vocab, device="cuda", dtype=torch.float64) % (spread + 1)).unsqueeze(1)).float()
    if of == "all":  # and far from 1 altogether
        x, w = x * 2.0 ** -20, w * 2.0 ** 20
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    rows = linear_cross_entropy(xl, wl, t, bias=b, reduction="none")
    rows.sum().backward()
    xd, wd = x.double().requires_grad_(True), w.double().requires_grad_(True)
    exact = torch.nn.functional.cross_entropy(xd @ wd.t() + b.double(), t, reduction="none")
    exact.sum().backward()
    A = (x.double().abs() @ w.double().abs().t()).amax(1) + b.double().abs().max()
    Ez = (dim / 16 + 16) * 2 * U * A
    assert bool(((rows.detach().double() - exact.detach()).abs() <= 2 * Ez + 2.0 ** -20 * exact.detach().clamp(min=1)).all())
    # gradients: errors of probabilities (relative, by the row's Ez), of the planes, and of the sums
    p = torch.softmax(x.double() @ w.double().t() + b.double(), 1)
    dz = p.clone()
    dz[torch.arange(n, device="cuda"), t] -= 1
    Edz = (2 * Ez.unsqueeze(1) + 2.0 ** -19) * p + (vocab / 16 + 16) * 2 * U * dz.abs()
    near(xl.grad, xd.grad, Edz @ w.double().abs(), "dx")
    near(wl.grad, wd.grad, (Edz + (n / 16 + 16) * 2 * U * dz.abs()).t() @ x.double().abs(), "dw")


def test_fp32_nonfinite_rows_stay_to_themselves():
    from bpt_b200.loss import linear_cross_entropy
    x, w, b, t = inputs(300, 500, 72, torch.float32)
    want = linear_cross_entropy(x, w, t, bias=b, reduction="none")
    for bad in (float("nan"), float("inf"), 3e38):
        y = x.clone()
        y[7, 3] = bad
        got = linear_cross_entropy(y, w, t, bias=b, reduction="none")
        keep = torch.arange(300, device="cuda") != 7
        assert torch.allclose(got[keep], want[keep], rtol=4e-6, atol=4e-6)  # 2 Ez of the module's note
        if bad != 3e38:
            assert bool(torch.isnan(got[7]))
