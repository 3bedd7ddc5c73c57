"""What is timed of the last stretch of a language model's training step, and its plain forms.

Three operators, in the order a step runs them:

``loss`` / ``step``   softmax cross entropy over a vocabulary straight from the hidden states and the
                      token table, without the logits: the losses alone (evaluation), or the loss and its
                      gradients for the hidden states and the table (training);
``embedding``         the gradient of the token + position embedding, added into the tables' gradients;
``adamw``             one AdamW step over every tensor of a model, its states in 32 bits or in 8.

Where ``own`` is false `run` computes them from elementary torch operations; where it is true it makes
the calls a user of the package makes.  Integers below 0 in ``labels`` leave their row out.

AdamW, t the number of the step, b1 / b2 the decay rates:
    m <- m + (g - m) (1 - b1)        v <- v + (g g - v) (1 - b2)
    p <- p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
States in 8 bits hold m and r = sqrt(v) in blocks of 256 consecutive elements of a tensor: a number
scale = max(|largest of the block| / 448, 2^-126) and one e4m3 number (4 exponent, 3 mantissa bits) per
element, the element over scale rounded to nearest; p takes the step of the unrounded m and v.
"""
import importlib
import math

import numpy as np
import torch

own = False

BLOCK = 256          # elements of a tensor that share one scale of the 8-bit states
TINY = 2.0 ** -126   # the least scale
HYPER = dict(lr=6e-4, eps=1e-8, beta1=0.9, beta2=0.95)
DECAY = 0.1          # on matrices; vectors (gains, biases) are not decayed


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # evaluation of a few words with the smallest model of the tests: nothing but latency
        dict(name="loss tiny", op="loss", rows=24, dim=64, vocab=300, left_out=0.0),
        # scoring one short, ragged batch of candidate answers: odd counts, bound by the read of the table
        dict(name="loss 61 rows", op="loss", rows=61, dim=768, vocab=50257, left_out=0.1),
        # perplexity over eight sequences of 1024 tokens
        dict(name="loss 8192 rows", op="loss", rows=8192, dim=768, vocab=50257, left_out=0.0),
        # a training step of the tests' smallest model
        dict(name="step tiny", op="step", rows=48, dim=64, vocab=300, left_out=0.0, reduction="mean"),
        # a micro-batch whose losses are weighted one by one, sequences padded, nothing a multiple of a tile
        dict(name="step 1000 rows weighted", op="step", rows=1000, dim=770, vocab=50257, left_out=0.2, reduction="none"),
        # the training step of the block benchmark's batch, 8 x 1024 tokens
        dict(name="step 8192 rows", op="step", rows=8192, dim=768, vocab=50257, left_out=0.02, reduction="mean"),
        # the embedding's gradient for the tests' smallest model, and for 8 x 1024 tokens of a skewed text
        dict(name="embedding tiny", op="embedding", sentences=2, seq=24, vocab=300, positions=32, dim=64),
        dict(name="embedding 8x1024", op="embedding", sentences=8, seq=1024, vocab=50257, positions=1024, dim=768),
        # AdamW over a small model (28 tensors, latency) and over one with GPT-2's 148 tensors
        dict(name="adamw32 small", op="adamw", bits=32, layers=2, width=64, vocab=300, positions=32, t=1),
        dict(name="adamw32 148 tensors", op="adamw", bits=32, layers=12, width=768, vocab=50257, positions=1024, t=1000),
        dict(name="adamw8 small", op="adamw", bits=8, layers=2, width=100, vocab=301, positions=33, t=1),
        dict(name="adamw8 148 tensors", op="adamw", bits=8, layers=12, width=768, vocab=50257, positions=1024, t=1000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("loss", "step", "step", "embedding", "adamw", "adamw"))
    if op in ("loss", "step"):
        while True:
            c = dict(op=op, rows=_log(rng, 1, 8192), dim=_log(rng, 16, 1600), vocab=_log(rng, 50, 60000),
                     left_out=rng.choice((0.0, 0.05, 0.5)))
            if c["rows"] * c["dim"] * c["vocab"] <= 8192 * 768 * 50257:
                break
        if op == "step":
            c["reduction"] = rng.choice(("mean", "mean", "sum", "none"))
        return c
    if op == "embedding":
        seq = _log(rng, 1, 1024)
        return dict(op=op, sentences=_log(rng, 1, 8), seq=seq, vocab=_log(rng, 50, 50257), positions=seq + rng.randrange(64),
                    dim=_log(rng, 16, 768))
    while True:
        c = dict(op=op, bits=rng.choice((32, 8)), layers=rng.randrange(1, 13), width=_log(rng, 16, 1024),
                 vocab=_log(rng, 50, 50257), positions=_log(rng, 16, 1024), t=_log(rng, 1, 100000))
        if sum(math.prod(s) for s in _shapes(c)) <= 124439808:
            return c


def _shapes(c):
    """The tensors of a model with learned positions: tables, per layer two LayerNorms and four linear
    layers with biases, the last LayerNorm."""
    w = c["width"]
    layer = [(w,), (w,), (w, 3 * w), (3 * w,), (w, w), (w,), (w,), (w,), (w, 4 * w), (4 * w,), (4 * w, w), (w,)]
    return [(c["vocab"], w), (c["positions"], w)] + c["layers"] * layer + [(w,), (w,)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class _Held:
    """A torch tensor's memory as the storage of a HIPTensor."""

    def __init__(self, t):
        self.tensor, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


_HIP_TYPES = {torch.float32: "float", torch.int32: "int32", torch.uint8: "uint8"}


def _hip(t):
    package = importlib.import_module("cl-waffe2_amd")
    package.lib.get()
    return package.HIPTensor(list(t.shape), vec=_Held(t), dtype=_HIP_TYPES[t.dtype])


def _text(n, vocab, gen, device):
    """Token ids with a text's skew: id k about as often as 1 / (k + 3)."""
    u = torch.rand(n, generator=gen, device=device, dtype=torch.float64)
    return ((3.0 * ((vocab + 3.0) / 3.0) ** u) - 3.0).long().clamp_(0, vocab - 1)


def _inputs(case, seed, device):
    """The case's inputs as torch tensors, from the seed alone."""
    gen = torch.Generator(device=device).manual_seed(int(seed))
    normal = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    if case["op"] in ("loss", "step"):
        n, d, v = case["rows"], case["dim"], case["vocab"]
        w = normal(v, d) * 0.14                                 # a trained token table's spread
        labels = _text(n, v, gen, device)
        # hidden states as a trained model leaves them: noise, and the way towards the right token
        x = normal(n, d) + torch.rand(n, 1, generator=gen, device=device) * (10.0 / (0.14 * d ** 0.5)) * w[labels] / (0.14 * d ** 0.5)
        labels = labels.int()
        labels[torch.rand(n, generator=gen, device=device) < case["left_out"]] = -1   # padding
        s = dict(x=x, w=w, labels=labels)
        if case.get("reduction") == "none":
            s["dy"] = torch.rand(n, generator=gen, device=device) + 0.5
        return s
    if case["op"] == "embedding":
        b, t, v, d = case["sentences"], case["seq"], case["vocab"], case["dim"]
        return dict(ids=_text(b * t, v, gen, device).float().view(b, t), dout=normal(b, t, d) * 1e-3,
                    dwte=normal(v, d) * 1e-3, dwpe=normal(case["positions"], d) * 1e-3)
    shapes = _shapes(case)
    rows = [-(-math.prod(s) // BLOCK) for s in shapes]            # blocks of each tensor in one flat storage
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    live = torch.ones(total, BLOCK, device=device)
    decay = torch.zeros(total, 1, device=device)
    for s, a, b in zip(shapes, start[:-1], start[1:]):
        n = math.prod(s)
        live[a:b].view(-1)[n:] = 0                                # what a tensor's last block does not fill
        if len(s) == 2:
            decay[a:b] = DECAY
    p = normal(total, BLOCK) * 0.05 * live
    # gradients whose sizes differ from element to element by orders of magnitude, as a network's do
    size = torch.exp(2.0 * normal(total, BLOCK)) * 1e-4
    g = normal(total, BLOCK) * size * live
    s = dict(p=p, g=g, decay=decay, shapes=shapes, start=[int(a) for a in start])
    if case["t"] == 1:                                            # the first step starts from nothing
        m, v = torch.zeros_like(p), torch.zeros_like(p)
    else:
        m = normal(total, BLOCK) * size * 0.3 * live
        v = (size * (0.5 + torch.rand(total, BLOCK, generator=gen, device=device))) ** 2 * live
    if case["bits"] == 32:
        s.update(m=m, v=v)
    else:
        s["m"], s["m_scale"] = _encode(m)
        s["r"], s["r_scale"] = _encode(torch.sqrt(v))
    return s


def prepare(case, seed):
    s = _inputs(case, seed, "cuda")
    s["case"] = case
    if case["op"] in ("loss", "step"):
        n = case["rows"]
        scalar = case.get("reduction") in ("mean", "sum")
        s.update(loss=torch.empty(1 if scalar else n, device="cuda"), lse=torch.empty(n, device="cuda"))
        if case["op"] == "step":
            s.update(dx=torch.empty_like(s["x"]), dw=torch.empty_like(s["w"]))
    if case["op"] == "adamw":
        s["steps"] = case["t"] - 1
    if own:
        s["hip"] = {k: _hip(t) for k, t in s.items() if isinstance(t, torch.Tensor) and t.dtype in _HIP_TYPES}
        if case["op"] == "adamw":
            s["optimizer"], s["grads"] = _optimizer(s, case)
    return s


def _optimizer(s, case):
    """The package's AdamW over the tensors of the flat storages, resumed after t - 1 steps."""
    optimizers = importlib.import_module("cl-waffe2_amd.optimizers")
    windows = {k: [] for k in ("p", "g", "m", "v", "r", "m_scale", "r_scale") if k in s}
    for shape, a, b in zip(s["shapes"], s["start"][:-1], s["start"][1:]):
        for k, found in windows.items():
            t = s[k][a:b].reshape(-1)
            found.append(_hip(t if k.endswith("scale") else t[:math.prod(shape)].view(shape)))
    decay = [DECAY if len(shape) == 2 else 0.0 for shape in s["shapes"]]
    states = {k: windows[k] for k in windows if k not in ("p", "g")}
    return optimizers.AdamW(windows["p"], weight_decay=decay, state_bits=case["bits"],
                            resume=dict(n=case["t"] - 1, **states), **HYPER), windows["g"]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if op in ("loss", "step"):
        return _run_loss(state)
    return _run_embedding(state) if op == "embedding" else _run_adamw(state)


def _run_loss(s):
    case = s["case"]
    reduction = case.get("reduction", "none")
    if own:
        nn = importlib.import_module("cl-waffe2_amd.nn")
        h = s["hip"]
        how = None if reduction == "none" else reduction
        nn.linear_cross_entropy(h["x"], h["w"], h["labels"], reduction=how, loss=h["loss"], lse=h["lse"])
        if case["op"] == "loss":
            return s["loss"], s["lse"]
        nn.linear_cross_entropy_backward(h["dy"] if how is None else 1.0, h["x"], h["w"], h["labels"], h["lse"],
                                         reduction=how, dx=h["dx"], dw=h["dw"])
        return s["loss"], s["dx"], s["dw"]
    x, w, labels = s["x"], s["w"], s["labels"].long()
    held = labels >= 0
    at = labels.clamp(min=0).unsqueeze(1)
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    loss = torch.where(held, lse - logits.gather(1, at).squeeze(1), 0.0)
    if case["op"] == "loss":
        return loss, lse
    if reduction == "none":
        g = torch.where(held, s["dy"], 0.0)
    else:
        weight = 1.0 / held.sum() if reduction == "mean" else torch.ones((), device=x.device)
        g = torch.where(held, weight, 0.0)
        loss = (loss.sum() * weight).view(1)
    e *= (g.unsqueeze(1) / total)                                # softmax times the row's gradient
    e.scatter_add_(1, at, -g.unsqueeze(1))
    return loss, e @ w, e.t() @ x


def _run_embedding(s):
    if own:
        gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
        h = s["hip"]
        gpt2.positional_embedding_backward(h["ids"], h["dout"], h["dwte"], h["dwpe"])
    else:
        seq, dim = s["case"]["seq"], s["case"]["dim"]
        s["dwte"].index_add_(0, s["ids"].view(-1).long(), s["dout"].view(-1, dim))
        s["dwpe"][:seq] += s["dout"].sum(0)
    return s["dwte"], s["dwpe"]


def _run_adamw(s):
    case = s["case"]
    if own:
        s["optimizer"].step(s["grads"])
    else:
        lr, eps, b1, b2 = (HYPER[k] for k in ("lr", "eps", "beta1", "beta2"))
        s["steps"] += 1
        c1, c2 = 1.0 - b1 ** s["steps"], 1.0 - b2 ** s["steps"]
        p, g = s["p"], s["g"]
        if case["bits"] == 32:
            m, v = s["m"], s["v"]
        else:
            m = _decode(s["m"], s["m_scale"])
            v = _decode(s["r"], s["r_scale"]) ** 2
        m += (g - m) * (1.0 - b1)
        v += (g * g - v) * (1.0 - b2)
        p -= lr * s["decay"] * p + (lr / c1) * m / (torch.sqrt(v / c2) + eps)
        if case["bits"] == 8:
            for name, values in (("m", m), ("r", torch.sqrt(v))):
                codes, scale = _encode(values)
                s[name].copy_(codes)
                s[name + "_scale"].copy_(scale)
    if case["bits"] == 32:
        return s["p"], s["m"], s["v"]
    e4m3 = torch.float8_e4m3fn
    return s["p"], s["m"].view(e4m3), s["m_scale"], s["r"].view(e4m3), s["r_scale"]


def _encode(a):
    """(e4m3 codes as bytes, one scale per block)."""
    scale = (a.abs().amax(1, keepdim=True) / 448.0).clamp(min=TINY)
    return (a / scale).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _decode(codes, scale):
    return codes.view(torch.float8_e4m3fn).float() * scale


# ---------------------------------------------------------------------------
# what a pass cannot do without, and what it should return
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] in ("loss", "step"):
        n, d, v = case["rows"], case["dim"], case["vocab"]
        if case["op"] == "loss":       # x, the table and the labels in, losses and row statistics out; the logits
            return dict(bytes=4 * (n * d + v * d + 3 * n), flops=2 * n * d * v)
        return dict(bytes=4 * (2 * n * d + 2 * v * d + 3 * n), flops=6 * n * d * v)   # and both gradients
    if case["op"] == "embedding":
        n, d = case["sentences"] * case["seq"], case["dim"]
        # rows of the table that are touched: about v (1 - (1 - share)^n) of them, here by the ids' distribution
        k = np.arange(case["vocab"], dtype=np.float64)
        share = np.log((k + 4.0) / (k + 3.0)) / math.log((case["vocab"] + 3.0) / 3.0)
        touched = float(np.sum(1.0 - (1.0 - np.minimum(share, 1.0)) ** n))
        return dict(bytes=int(4 * (n + n * d + 2 * touched * d + 2 * case["seq"] * d)), flops=2 * n * d)
    sizes = [math.prod(s) for s in _shapes(case)]
    n = sum(sizes)
    if case["bits"] == 32:             # p, m, v in and out, g in
        return dict(bytes=28 * n, flops=14 * n)
    return dict(bytes=16 * n + 16 * sum(-(-k // BLOCK) for k in sizes), flops=22 * n)


def exact(case, seed):
    s = _inputs(case, seed, "cuda")
    f8 = torch.float64
    if case["op"] in ("loss", "step"):
        n, reduction = case["rows"], case.get("reduction", "none")
        labels, w = s["labels"].long(), s["w"].to(f8)
        count = int((labels >= 0).sum())
        losses, lses, dxs, dw = [], [], [], torch.zeros_like(w) if case["op"] == "step" else None
        for a in range(0, n, 2048):                              # a slice of the rows at a time
            x, l = s["x"][a:a + 2048].to(f8), labels[a:a + 2048]
            z = torch.log_softmax(x @ w.t(), 1)
            row = torch.arange(len(l), device=l.device)
            hit = l >= 0
            losses.append(torch.where(hit, -z[row, l.clamp(min=0)], 0.0))
            lses.append(torch.logsumexp(x @ w.t(), 1))
            if case["op"] == "step":
                z = z.exp()
                z[row, l.clamp(min=0)] -= 1.0
                weight = s["dy"][a:a + 2048].to(f8) if reduction == "none" else 1.0 / max(count, 1) if reduction == "mean" else 1.0
                z *= (hit * weight).unsqueeze(1)
                dxs.append(z @ w)
                dw += z.t() @ x
        loss = torch.cat(losses)
        if case["op"] == "loss":
            return loss, torch.cat(lses)
        if reduction != "none":
            loss = (loss.sum() / (count if reduction == "mean" else 1)).view(1)
        return loss, torch.cat(dxs), dw
    if case["op"] == "embedding":
        ids, dout = s["ids"].view(-1).long(), s["dout"].to(f8)
        dwte, dwpe = s["dwte"].to(f8), s["dwpe"].to(f8)
        dwte.index_put_((ids,), dout.view(-1, case["dim"]), accumulate=True)
        for t in range(case["seq"]):
            dwpe[t] += dout[:, t].sum(0)
        return dwte, dwpe
    h, t = HYPER, case["t"]
    p, g, wd = s["p"].to(f8), s["g"].to(f8), s["decay"].to(f8)
    if case["bits"] == 32:
        m, v = s["m"].to(f8), s["v"].to(f8)
    else:
        value = torch.from_numpy(_e4m3_values()).to(p.device)
        m = value[s["m"].long()] * s["m_scale"].to(f8)
        v = (value[s["r"].long()] * s["r_scale"].to(f8)).square()
    m = h["beta1"] * m + (1 - h["beta1"]) * g
    v = h["beta2"] * v + (1 - h["beta2"]) * g.square()
    step = (m / (1 - h["beta1"] ** t)) / ((v / (1 - h["beta2"] ** t)).sqrt() + h["eps"])
    p = p * (1 - h["lr"] * wd) - h["lr"] * step
    if case["bits"] == 32:
        return p, m, v
    out = [p]
    for a in (m, v.sqrt()):
        scale = torch.clamp(a.abs().amax(1, keepdim=True) / 448.0, min=TINY)
        out += [_nearest_e4m3(a / scale), scale]
    return tuple(out)


def _e4m3_values():
    """The numbers that the 256 codes stand for."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    a = np.where(e == 0, f * 2.0 ** -9, (1.0 + f / 8.0) * 2.0 ** (e - 7.0))
    a[(c & 127) == 127] = np.nan
    return np.where(c & 128, -a, a)


def _nearest_e4m3(y):
    """The e4m3 number nearest to each y (|y| at most about 448), ties to the even code."""
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3.0)
    return torch.round(y / step) * step
