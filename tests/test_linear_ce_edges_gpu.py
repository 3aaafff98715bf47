"""linear_cross_entropy at the edges of its number formats, against the formula in 64 bits.

Tolerances are those of test_linear_ce_gpu's note (u = 2^-24, Ez, Ep), which hold for every entry with the absolute values of
its own row and column; what is added to them stands at each test."""
import pytest
import torch

from bpt_b200.loss import linear_cross_entropy
from test_linear_ce_gpu import DTYPES, IGNORE, check, formula, inputs, near

pytestmark = pytest.mark.gpu

# fp32 in two fp16 planes: an entry of dZ times 2^14 has a second plane times 2^11, whose smallest half step is 2^-25: 2^-50 of
# dZ.  The product of second planes is left out: that of dZ is up to 2^-25 (where the first is at its smallest step), 2^-39
# of dZ, and the other operand's up to 2^-11 of its numbers: 2^-50 again.
FLOOR = 2.0 ** -49


@pytest.mark.parametrize("down", [12, 40, 52, 90])
@pytest.mark.parametrize("of", ["x", "w", "x up, w down"])
def test_fp32_columns_of_very_different_size(of, down):
    """One feature far below the others: its column of d w has what that column of x keeps, its column of d x what that of w
    does.  One far above the others in x and as far below in w: the logits have what the other columns of x keep."""
    for n, dim in ((300, 72), (70, 73), (90, 1100), (65, 150), (40, 270), (33, 642), (50, 401)):
        x, w, b, t = inputs(n, 500, dim, torch.float32, padded=0.1)
        for c in (5, dim - 100) if dim > 512 else (5,):
            if of == "x":
                x[:, c] *= 2.0 ** -down
            elif of == "w":
                w[:, c] *= 2.0 ** -down
            else:
                x[:, c] *= 2.0 ** down
                w[:, c] *= 2.0 ** -down
        check(x, w, b, t, smoothing=0.1)


@pytest.mark.parametrize("up", [100, 108, 110, -100, -108, -110])
def test_fp32_sizes_far_from_one(up):
    """x times 2^up and w times 2^-up: the same logits."""
    x, w, b, t = inputs(300, 500, 72, torch.float32, padded=0.1)
    check(x * 2.0 ** up, w * 2.0 ** -up, b, t, smoothing=0.1)


def off_by(x, w, t, most):
    """What d x, d w, d b may be off by when every entry of dZ that counts is off by `most`."""
    counted = (t != IGNORE).double().unsqueeze(1)
    dz = most * counted.expand(-1, w.size(0))
    return dz @ w.double().abs(), dz.t() @ x.double().abs(), dz.sum(0)


@pytest.mark.parametrize("spread", [12, 24, 26, 40, 60, 110])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_of_very_different_weight(dtype, spread):
    """reduction none: weights from 1 to 2^-spread.  Each token's row of d x is as good as its own weight allows.  In fp32 an
    entry of dZ may also be off by FLOOR of the largest weight while no weight is below 2^-24 of it."""
    x, w, b, t = inputs(300, 500, 72, dtype, padded=0.1)
    g = 2.0 ** -(torch.arange(300, device="cuda") % (spread + 1)).float()
    g[7] = 0.0
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
    linear_cross_entropy(*leaves[:2], t, bias=leaves[2], reduction="none").backward(g)
    want, off = formula(x, w, b, t, 0.0, "none", g)
    more = off_by(x, w, t, FLOOR if dtype == torch.float32 and spread <= 24 else 0.0)
    for name, leaf, v, e, m in zip(("dx", "dw", "db"), leaves, want[1:], off[1:], more):
        near(leaf.grad, v, e + m, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_a_gradient_that_is_not_finite_spoils_its_own_row(dtype, bad):
    """reduction none: that token's row of d x and the sums over tokens are not finite, the other rows are as without it."""
    for n in (300, 20):  # dZ in one plane and in two
        x, w, b, t = inputs(n, 500, 72, dtype, padded=0.1)
        t[17] = 3
        g = torch.linspace(0.5, 1.5, n, device="cuda")

        def grads(of_17):
            leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
            weight = g.clone()
            weight[17] = of_17
            linear_cross_entropy(*leaves[:2], t, bias=leaves[2], reduction="none").backward(weight)
            return [v.grad for v in leaves]

        want, got = grads(1.0), grads(bad)
        keep = torch.arange(n, device="cuda") != 17
        assert torch.equal(got[0][keep], want[0][keep])
        assert not bool(torch.isfinite(got[0][17]).any())
        assert not bool(torch.isfinite(got[1]).any()) and not bool(torch.isfinite(got[2]).any())


@pytest.mark.parametrize("shape", [(9000, 40000, 128, torch.bfloat16), (3000, 90000, 128, torch.float16), (60000, 3000, 256, torch.float32)],
                         ids=lambda s: "x".join(map(str, s[:3])))
def test_a_wait_that_ran_out_marks_every_gradient(shape):
    """A kernel whose wait ran out sets the status word, the first of the workspace; no wait runs out here, the word is set from
    the host while the kernels of several pieces run.  Every gradient's first element is NaN then, whichever piece it was."""
    from bpt_b200 import _lib
    n, vocab, dim, dtype = shape
    x, w, b, t = inputs(n, vocab, dim, dtype, padded=0.1)
    t[0] = IGNORE  # the first row of d x is written by no product
    L, code, p = _lib.lib(), _lib.dtype_code(dtype), lambda v: v.data_ptr()
    loss, lse, count = (torch.empty(k, device="cuda") for k in (1, n, 1))
    grad = torch.ones(1, device="cuda")
    size = L.bpt_linear_ce_forward_workspace_bytes(p(x), dim, p(w), dim, n, vocab, dim, code)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    _lib.check(L.bpt_linear_ce_forward(p(x), dim, p(w), dim, p(b), p(t), IGNORE, 0.0, 1, p(loss), p(lse), p(count), n, vocab, dim, code,
                                       p(ws), size, _lib.stream()))
    size = L.bpt_linear_ce_backward_workspace_bytes(p(x), dim, p(w), dim, n, vocab, dim, code, 1, 1, 1)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert ws.data_ptr() % 256 == 0
    outs = [torch.empty(s, dtype=dtype, device="cuda") for s in ((n, dim), (vocab, dim), (vocab,))]
    word, one = ws[:4].view(torch.int32), torch.ones(1, dtype=torch.int32).pin_memory()
    side, end = torch.cuda.Stream(), torch.cuda.Event()

    def backward():
        _lib.check(L.bpt_linear_ce_backward(p(x), dim, p(w), dim, p(b), p(t), IGNORE, 0.0, 1, p(lse), p(count), p(grad), p(outs[0]),
                                            p(outs[1]), p(outs[2]), n, vocab, dim, code, p(ws), size, _lib.stream()))

    backward()  # warm
    torch.cuda.synchronize()
    assert all(bool(torch.isfinite(v).all()) for v in outs)
    for _ in range(50):  # again if the host was held up while the kernels ran
        backward()
        end.record()
        sent = 0
        with torch.cuda.stream(side):  # copies need no SM, which the kernels hold
            while not end.query():
                word.copy_(one, non_blocking=True)
                sent += 1
        torch.cuda.synchronize()
        if sent > 10:
            break
    assert sent > 10
    for name, v in zip(("dx", "dw", "db"), outs):
        assert bool(torch.isnan(v.view(-1)[0])), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 5, 300])
def test_smoothing_over_classes_that_are_masked(n, dtype):
    """A bias of -inf and label smoothing: the loss is infinite (not NaN), also of a token whose target is masked, and the
    gradients, which need no logarithm, are the formula's."""
    x, w, b, t = inputs(n, 400, 64, dtype)
    b[3] = b[200] = -float("inf")
    t[0] = 3
    t[1:] = t[1:].clamp(min=4)
    t[t == 200] = 201
    for smoothing, row0, rows in ((0.0, float("inf"), None), (0.1, float("inf"), float("inf"))):
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        loss = linear_cross_entropy(*leaves[:2], t, bias=leaves[2], label_smoothing=smoothing, reduction="none")
        with torch.no_grad():
            assert torch.equal(loss, linear_cross_entropy(x, w, t, bias=b, label_smoothing=smoothing, reduction="none"))
        assert float(loss[0].detach()) == row0
        assert bool(torch.isfinite(loss[1:]).all()) if rows is None else bool((loss[1:] == rows).all())
        loss.backward(torch.ones_like(loss))
        want, off = formula(x, w, b, t, smoothing, "none", torch.ones(n, device="cuda"))
        for name, leaf, v, e in zip(("dx", "dw", "db"), leaves, want[1:], off[1:]):
            near(leaf.grad, v, e, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 5, 300])
def test_classes_masked_with_the_lowest_number(n, dtype):
    """The bias of masked classes is the type's lowest number, whole blocks of classes among them.  Losses stay finite, and
    gradients are those of a bias of -inf.  Losses of ordinary tokens without smoothing, too; the others are sums of at most 432 additions,
    so off by 2^-15 of themselves."""
    x, w, b, t = inputs(n, 400, 64, dtype)
    masked = torch.zeros(400, dtype=torch.bool, device="cuda")
    masked[:64] = masked[200:300] = masked[399] = True
    t = t % 90 + 70
    t[0] = 3
    low, none = b.clone(), b.clone()
    low[masked], none[masked] = torch.finfo(dtype).min, -float("inf")
    z = x.double() @ w.double().t() + low.double()
    for smoothing in (0.0, 0.1):
        leaves = [v.clone().requires_grad_(True) for v in (x, w, low)]
        loss = linear_cross_entropy(*leaves[:2], t, bias=leaves[2], label_smoothing=smoothing, reduction="none")
        loss.backward(torch.ones_like(loss))
        exact = torch.nn.functional.cross_entropy(z, t, label_smoothing=smoothing, reduction="none")
        assert bool(((loss.detach().double() - exact).abs() <= 2.0 ** -15 * exact.abs()).all())
        want, off = formula(x, w, none, t, smoothing, "none", torch.ones(n, device="cuda"))
        if not smoothing and n > 1:
            near(loss.detach()[1:], want[0][1:], off[0][1:], "loss")
        for name, leaf, v, e in zip(("dx", "dw", "db"), leaves, want[1:], off[1:]):
            near(leaf.grad, v, e, name)
    for smoothing in (0.0, 0.1):  # nothing is left
        leaves = [v.clone().requires_grad_(True) for v in (x, w, torch.full_like(b, torch.finfo(dtype).min))]
        loss = linear_cross_entropy(*leaves[:2], t, bias=leaves[2], label_smoothing=smoothing, reduction="none")
        loss.backward(torch.ones_like(loss))
        assert bool(torch.isfinite(loss).all()) and all(bool(torch.isfinite(v.grad).all()) for v in leaves)


@pytest.mark.parametrize("dtype", DTYPES)
def test_probabilities_of_very_different_size(dtype):
    """Classes whose probability is from 2^-4 down to 2^-60 for every token: rows of d w that are as small.  An entry of dZ is off by
    the note's bound and, in fp32, by no more than FLOOR beside it (in fp16 by 2^-39, which the formula has)."""
    for n in (300, 90):
        x, w, b, t = inputs(n, 600, 72, dtype, spread=0.3)
        b = (b.float() - 0.6931 * (torch.arange(600, device="cuda") % 60)).to(dtype)
        t = t // 60 * 60  # classes that are probable
        t[::7] = IGNORE
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        linear_cross_entropy(*leaves[:2], t, bias=leaves[2], reduction="sum").backward()
        want, off = formula(x, w, b, t, 0.0, "sum", torch.ones((), device="cuda"))
        p = torch.softmax(x.double() @ w.double().t() + b.double(), 1)
        assert float(p.max()) > 2.0 ** -5 and float(p.min()) < 2.0 ** -60
        more = off_by(x, w, t, FLOOR if dtype == torch.float32 else 0.0)
        for name, leaf, v, e, m in zip(("dx", "dw", "db"), leaves, want[1:], off[1:], more):
            near(leaf.grad, v, e + m, name)


def test_label_smoothing_and_a_summed_divergence():
    """KLDivLoss(reduction="sum") of the log-probabilities against targets with smoothing / vocab on every class is the summed
    loss minus the targets' entropy, a constant for each token that counts: the same gradients.  Tolerances: the module's note."""
    x, w, b, t = inputs(200, 300, 64, torch.float32, padded=0.2)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(*leaves[:2], t, bias=leaves[2], label_smoothing=0.1, reduction="sum")
    loss.backward()
    exact = [v.double().requires_grad_(True) for v in (x, w, b)]
    counted = t != IGNORE
    logp = torch.log_softmax(exact[0] @ exact[1].t() + exact[2], 1)[counted]
    q = torch.full_like(logp, 0.1 / 300).scatter_(1, t[counted].unsqueeze(1), 0.9 + 0.1 / 300)
    divergence = torch.nn.functional.kl_div(logp, q, reduction="sum")
    divergence.backward()
    entropy = -(q * q.log()).sum()
    want, off = formula(x, w, b, t, 0.1, "sum", torch.ones((), device="cuda"))
    near(loss.detach(), (divergence + entropy).detach(), off[0], "loss")
    for name, leaf, e, slack in zip(("dx", "dw", "db"), leaves, exact, off[1:]):
        near(leaf.grad, e.grad, slack, name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_far_apart_in_memory(dtype):
    """Rows whose offsets pass 2^31 elements, read in place and copied: the same as close together."""
    n, step, dim = 140000, 16384, 64
    big = torch.empty(n * step, dtype=dtype, device="cuda").view(n, step)
    x, w, b, t = inputs(n, 100, dim, dtype, padded=0.1)
    want = linear_cross_entropy(x, w, t, bias=b, reduction="none")
    for at in (8, 3):
        far = big[:, at:at + dim]
        far.copy_(x)
        assert torch.equal(linear_cross_entropy(far, w, t, bias=b, reduction="none"), want)
    leaves = [v.clone().requires_grad_(True) for v in (x, w)]
    linear_cross_entropy(*leaves, t, bias=b).backward()
    held = far.detach().requires_grad_(True)
    again = w.clone().requires_grad_(True)
    linear_cross_entropy(held, again, t, bias=b).backward()
    assert torch.equal(held.grad, leaves[0].grad) and torch.equal(again.grad, leaves[1].grad)


@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_replayed_graphs_choose_the_planes_again(reduction):
    """fp32: which planes the operands take is found on the device.  A step captured with ordinary numbers is replayed with a
    column far below the others and tokens of far smaller weight, then with ordinary ones again."""
    x, w, b, t = inputs(300, 500, 72, torch.float32, padded=0.1)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
    weight = torch.ones(300, device="cuda") if reduction == "none" else torch.ones((), device="cuda")

    def step():
        loss = linear_cross_entropy(*leaves[:2], t, bias=leaves[2], reduction=reduction)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves, weight)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for column, small in ((1.0, 0), (2.0 ** -40, 0), (1.0, 50), (2.0 ** -40, 50), (1.0, 0)):
        with torch.no_grad():
            leaves[0].copy_(x)
            leaves[0][:, 5] *= column
            if reduction == "none":
                weight.copy_(2.0 ** -(torch.arange(300, device="cuda") % (small + 1)).float())
        graph.replay()
        got = [v.clone() for v in out]
        assert all(torch.equal(a, e) for a, e in zip(got, step()))
