"""A build without the torch extensions (build.py --no-torch-ext) still runs the blocks, the models and decoding: their layer
norm reaches the library through ctypes."""
import sys

import pytest
import torch

import bpt_b200
from bpt_b200 import model as models

pytestmark = pytest.mark.gpu


@pytest.fixture
def without_extension(monkeypatch):
    def remove():
        monkeypatch.setitem(sys.modules, "bpt_b200._train_ext", None)  # importing it raises ImportError
        monkeypatch.delattr(bpt_b200, "_train_ext", raising=False)
        models._has_train_extension.cache_clear()
    yield remove
    monkeypatch.undo()
    models._has_train_extension.cache_clear()


def language_model():
    from bpt_b200 import csr, graphbuilder
    from bpt_b200.attention import AttentionPlan
    torch.manual_seed(0)
    batch = csr.batch_graphs([graphbuilder.BinaryPartition(n, True, 4, 6) for n in (100, 37)])
    plan = AttentionPlan.from_batch(batch, n_etypes=1000)
    tokens = torch.randint(0, 50, (137,), device="cuda")
    return models.BPTLanguageModel(50, 128, 256, 2, 2).cuda(), (tokens, batch.leaf_ids(), plan)


def test_models_run_and_train(without_extension):
    lm, args = language_model()
    want = lm(*args)
    want.sum().backward()
    grads = [p.grad.clone() for p in lm.parameters()]
    lm.zero_grad()
    without_extension()
    with pytest.raises(ImportError, match="bpt_b200.build"):
        bpt_b200.train_extension()
    got = lm(*args)
    got.sum().backward()
    assert torch.equal(got, want)
    assert all(torch.equal(p.grad, g) for p, g in zip(lm.parameters(), grads))
    with torch.no_grad():
        assert torch.equal(lm(*args), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_add_layer_norm(without_extension, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    cases = []
    for rows, dim in ((0, 64), (5, 8), (1000, 512), (33, 520), (9, 4096)):
        x, r, gy = (torch.randn(rows, 2 * dim, generator=gen, device="cuda").to(dtype)[:, ::2] for _ in range(3))
        cases.append((x, r, torch.nn.LayerNorm(dim).cuda().to(dtype), gy))

    def run(x, r, norm, gy):
        leaves = [x.detach().requires_grad_(True), r.detach().requires_grad_(True)]
        y = models.add_layer_norm(*leaves, norm)
        return [y] + list(torch.autograd.grad(y, leaves + [norm.weight, norm.bias], gy))

    want = [run(*c) for c in cases]
    without_extension()
    assert not models._has_train_extension()
    for c, w in zip(cases, want):
        assert all(torch.equal(a, e) for a, e in zip(run(*c), w))
    x, r, norm, gy = cases[1]
    leaf = x.detach().requires_grad_(True)
    first = torch.autograd.grad(models.add_layer_norm(leaf, r, norm), leaf, gy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once"):
        first.sum().backward()
