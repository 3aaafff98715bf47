"""Measured cases of two training operators: softmax cross entropy fused with the generator's projection
(`bpt_b200.loss.linear_cross_entropy`) and layer norm with a residual (`bpt_b200.norm.layer_norm`), each in its
forward form and with its gradients.

A case is one call as a training or scoring program makes it.  `run` computes it either through the library
(`own`) or in elementary torch operations in 32 bits.

Sizes: the character language model reads 8 sequences of 8192 bytes (65536 tokens, 256 symbols, model width 512;
its causal binary-partition graphs have 8 x 16383 nodes), the translation model has a vocabulary of 8000 and about
28.7 thousand target tokens a batch, the classifier has 50 thousand words and a model width of 300.
"""
import math

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

# The most work a drawn case may have: multiply-adds x products, cells of the logit matrix, elements of a norm.
MOST_PRODUCT = 6e11
MOST_CELLS = 4.1e8
MOST_NORM = 6.7e7


def loss_case(name, n, vocab, dim, dtype, train, bias=True, smoothing=0.0, padded=0.0, reduction="mean"):
    return {"name": name, "op": "loss", "n": n, "vocab": vocab, "dim": dim, "dtype": dtype, "train": train, "bias": bias,
            "smoothing": smoothing, "padded": padded, "reduction": reduction}


def norm_case(name, rows, dim, dtype, train, residual=True):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "train": train, "residual": residual}


def listed():
    return [
        # one training step's loss of the character language model: a small vocabulary, as many tokens as a batch has
        loss_case("loss train char lm", 65536, 256, 512, "bf16", True),
        # translation training: padded sentences, label smoothing, a middling vocabulary
        loss_case("loss train translation", 28701, 8000, 512, "bf16", True, smoothing=0.1, padded=0.12),
        # word-level language model: the vocabulary is the long axis
        loss_case("loss train words", 8192, 50000, 512, "bf16", True),
        # single precision training at the classifier's width, odd token count and vocabulary
        loss_case("loss train fp32", 4099, 8003, 300, "fp32", True, smoothing=0.1, padded=0.12),
        # half precision with a summed (scaled) loss, an output layer without bias, a short ragged batch
        loss_case("loss train fp16 ragged", 777, 10001, 512, "fp16", True, bias=False, reduction="sum"),
        # scoring one token against every word: latency, the weight is all there is to read
        loss_case("loss score one token", 1, 50000, 512, "bf16", False, reduction="none"),
        # perplexity of a validation set: forward only
        loss_case("loss evaluate", 65536, 8000, 512, "bf16", False),
        # every node of the language model's batch, twice a layer and step
        norm_case("norm train lm nodes", 131064, 512, "bf16", True),
        # one decoding step: the nodes of one position of 16 sequences
        norm_case("norm decode step", 20, 512, "bf16", False),
        # the classifier's width in single precision, a ragged batch
        norm_case("norm train fp32 300", 14207, 300, "fp32", True),
        # a wide model in half precision without a residual
        norm_case("norm train fp16 wide", 4096, 4096, "fp16", True, residual=False),
        # a small training batch: few rows, so the weight gradient's reduction and the launches count
        norm_case("norm train short", 555, 512, "bf16", True),
    ]


def log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
    train = rng.random() < 0.7
    if rng.random() < 0.5:
        dim = log_uniform(rng, 64, 1024)
        step = rng.choice([1, 4, 8, 64])
        dim = max(step, dim // step * step)
        n = log_uniform(rng, 1, 65536)
        vocab = log_uniform(rng, 17, 50257)
        while n * vocab * dim * (3 if train else 1) > MOST_PRODUCT or n * vocab > MOST_CELLS:
            n = n * 2 // 3
        n = max(n, 1)
        reduction = "sum" if dtype == "fp16" else rng.choice(["mean", "mean", "sum", "none"])
        case = loss_case("", n, vocab, dim, dtype, train, rng.random() < 0.7, rng.choice([0.0, 0.0, 0.1]),
                         rng.choice([0.0, 0.12, 0.4]) if n > 64 else 0.0, reduction)
    else:
        dim = log_uniform(rng, 64, 4096)
        step = rng.choice([1, 4, 8, 64])
        dim = max(step, dim // step * step)
        rows = log_uniform(rng, 1, 131072)
        rows = max(1, min(rows, int(MOST_NORM // dim)))
        case = norm_case("", rows, dim, dtype, train, rng.random() < 0.7)
    del case["name"]
    return case


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    gen = generator(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).add_(shift).to(dtype)

    state = dict(case)
    if case["op"] == "loss":
        n, vocab, dim = case["n"], case["vocab"], case["dim"]
        # the last layer's normalised features; a weight that spreads the logits by about two
        state["x"] = normal(n, dim)
        state["weight"] = normal(vocab, dim, scale=2.0 / math.sqrt(dim))
        state["bias"] = normal(vocab, scale=0.2) if case["bias"] else None
        # word frequencies fall as one over the rank
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        target = (torch.exp(u * math.log(vocab)).long() - 1).clamp_(0, vocab - 1)
        if case["padded"]:
            # sentences in slots of 64, their tails padding
            slots = (n + 63) // 64
            least = max(1, int(64 * (1 - 2 * case["padded"])))
            length = torch.randint(least, 65, (slots,), generator=gen, device="cuda")
            at = torch.arange(n, device="cuda")
            target = torch.where(at % 64 < length[at // 64], target, torch.full_like(target, IGNORE))
        state["target"] = target
        # the gradient that reaches the loss: ones, or one weight a token
        state["grad"] = (torch.rand(n, generator=gen, device="cuda") + 0.5 if case["reduction"] == "none"
                         else torch.ones((), device="cuda"))
        leaves = ["x", "weight", "bias"]
    else:
        rows, dim = case["rows"], case["dim"]
        state["x"] = normal(rows, dim, scale=1.5, shift=0.3)
        state["residual"] = normal(rows, dim) if case["residual"] else None
        state["weight"] = normal(dim, scale=0.2, shift=1.0)
        state["bias"] = normal(dim, scale=0.2)
        state["grad"] = normal(rows, dim)
        leaves = ["x", "residual", "weight", "bias"]
    if case["train"]:
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


def run(state):
    if own:
        return own_loss(state) if state["op"] == "loss" else own_norm(state)
    with torch.no_grad():
        return plain_loss(state) if state["op"] == "loss" else plain_norm(state)


def with_grads(names, state, out, more):
    """The outputs as a dict: the result and the gradients of the inputs that the case has."""
    kept = [k for k in names if state[k] is not None]
    grads = more([state[k] for k in kept])
    return {"out": out, **{"d_" + k: g for k, g in zip(kept, grads)}}


def own_loss(s):
    from bpt_b200.loss import linear_cross_entropy
    if not s["train"]:
        with torch.no_grad():
            return {"out": linear_cross_entropy(s["x"], s["weight"], s["target"], bias=s["bias"], ignore_index=IGNORE,
                                                label_smoothing=s["smoothing"], reduction=s["reduction"])}
    loss = linear_cross_entropy(s["x"], s["weight"], s["target"], bias=s["bias"], ignore_index=IGNORE,
                                label_smoothing=s["smoothing"], reduction=s["reduction"])
    return with_grads(["x", "weight", "bias"], s, loss.detach(), lambda at: torch.autograd.grad(loss, at, s["grad"]))


def own_norm(s):
    from bpt_b200.norm import layer_norm
    if not s["train"]:
        with torch.no_grad():
            return {"out": layer_norm(s["x"], s["weight"], s["bias"], residual=s["residual"])}
    y = layer_norm(s["x"], s["weight"], s["bias"], residual=s["residual"])
    return with_grads(["x", "residual", "weight", "bias"], s, y.detach(), lambda at: torch.autograd.grad(y, at, s["grad"]))


def plain_loss(s):
    """lse_i = log sum_v exp(z_iv), z = x W^T + b; loss_i = lse_i - (1 - e) z_i,t - e mean_v z_iv;
    d z_iv = g_i (softmax_iv - (1 - e) [v = t_i] - e / V)."""
    x, w, target, eps = s["x"].float(), s["weight"].float(), s["target"], s["smoothing"]
    vocab = w.size(0)
    z = x @ w.t()
    if s["bias"] is not None:
        z += s["bias"].float()
    counted = target != IGNORE
    at = torch.where(counted, target, torch.zeros_like(target)).unsqueeze(1)
    top = z.amax(1, keepdim=True)
    loss = -(1.0 - eps) * z.gather(1, at)
    if eps:
        loss -= eps * z.mean(1, keepdim=True)
    z = torch.exp(z.sub_(top))
    total = z.sum(1, keepdim=True)
    loss = torch.where(counted, (loss + top + torch.log(total)).squeeze(1), torch.zeros((), device=x.device))
    n_counted = counted.sum()
    out = loss if s["reduction"] == "none" else loss.sum() if s["reduction"] == "sum" else loss.sum() / n_counted
    if not s["train"]:
        return {"out": out}
    g = s["grad"] / n_counted if s["reduction"] == "mean" else s["grad"]
    g = torch.where(counted, g, torch.zeros((), device=x.device)).unsqueeze(1)
    z /= total
    if eps:
        z -= eps / vocab
    z.scatter_add_(1, at, torch.full_like(total, -(1.0 - eps)))
    z *= g
    dtype = s["x"].dtype
    made = {"x": lambda: (z @ w).to(dtype), "weight": lambda: (z.t() @ x).to(dtype), "bias": lambda: z.sum(0).to(dtype)}
    names = ["x", "weight", "bias"]
    return with_grads(names, s, out, lambda at: [made[k]() for k in names if s[k] is not None])


def plain_norm(s):
    """y = (a - mean) / sqrt(var + eps) * w + b with a = x + residual; with n the normalised a and q = gy w:
    d a = (q - mean(q) - n mean(q n)) / sqrt(var + eps), d w = sum gy n, d b = sum gy."""
    dtype = s["x"].dtype
    a = s["x"].float()
    if s["residual"] is not None:
        a = a + s["residual"].float()
    w = s["weight"].float()
    a = a - a.mean(1, keepdim=True)
    r = torch.rsqrt((a * a).mean(1, keepdim=True) + 1e-5)
    n = a * r
    out = (n * w + s["bias"].float()).to(dtype)
    if not s["train"]:
        return {"out": out}
    gy = s["grad"].float()
    q = gy * w
    da = ((q - q.mean(1, keepdim=True) - n * (q * n).mean(1, keepdim=True)) * r).to(dtype)
    made = {"x": da, "residual": da, "weight": (gy * n).sum(0).to(dtype), "bias": gy.sum(0).to(dtype)}
    names = ["x", "residual", "weight", "bias"]
    return with_grads(names, s, out, lambda at: [made[k] for k in names if s[k] is not None])


def work(case):
    """Each input read once, each output written once; the products that the definition has: the logits, and for a
    training step the products of their gradient with the weight and with the features, of the tokens that count."""
    b = SIZE[case["dtype"]]
    if case["op"] == "loss":
        n, vocab, dim = case["n"], case["vocab"], case["dim"]
        counted = n * (1.0 - case["padded"])
        read = (counted * dim + vocab * dim + (vocab if case["bias"] else 0)) * b + 8 * n
        wrote = 4 * n if case["reduction"] == "none" else 4
        if case["train"]:
            wrote += (n * dim + vocab * dim + (vocab if case["bias"] else 0)) * b
        return {"bytes": read + wrote, "flops": (6.0 if case["train"] else 2.0) * counted * vocab * dim}
    rows, dim = case["rows"], case["dim"]
    inputs = 2 if case["residual"] else 1
    matrices = inputs + 1 + (2 if case["train"] else 0)  # inputs, y; gy and the one gradient that both inputs share
    return {"bytes": (matrices * rows * dim + (4 if case["train"] else 2) * dim) * b,
            "flops": (20.0 if case["train"] else 8.0) * rows * dim}


def exact(case, seed):
    """The same from torch's own definitions in 64 bits, the gradients by automatic differentiation."""
    s = prepare(case, seed)

    def double(k):
        return None if s[k] is None else s[k].detach().double().requires_grad_(case["train"])

    if case["op"] == "loss":
        at = {k: double(k) for k in ("x", "weight", "bias")}
        z = torch.nn.functional.linear(at["x"], at["weight"], at["bias"])
        out = torch.nn.functional.cross_entropy(z, s["target"], ignore_index=IGNORE, reduction=s["reduction"],
                                                label_smoothing=s["smoothing"])
    else:
        at = {k: double(k) for k in ("x", "residual", "weight", "bias")}
        a = at["x"] if at["residual"] is None else at["x"] + at["residual"]
        out = torch.nn.functional.layer_norm(a, (case["dim"],), at["weight"], at["bias"], 1e-5)
    if not case["train"]:
        return {"out": out}
    at = {k: v for k, v in at.items() if v is not None}
    grads = torch.autograd.grad(out, list(at.values()), s["grad"].double())
    return {"out": out.detach(), **{"d_" + k: g for k, g in zip(at, grads)}}
