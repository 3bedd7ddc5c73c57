"""A language model's training step on the device: embedding, blocks, loss over the vocabulary, every gradient, AdamW.

The gradients are held against a float64 backward that central differences pin (below, on the CPU), the steps against
AdamW in float64 on the device's own gradients (the loss, its gradients, the embedding's gradient and AdamW run
together as a user runs them)."""
import importlib

import numpy as np
import pytest

from oracle import gpt2_block_ref as ref
from test_gpu_adamw import HYPER, U, decode, reference

f32 = np.float32
CFG = dict(batch=2, seq=24, d_model=64, n_head=4, head_dim=16, d_ff=128, eps=1e-5)
VOCAB, N_CTX, LAYERS = 300, 32, 2


def make_model(seed=12):
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    rng = np.random.default_rng(seed)
    model = {"wte": (rng.standard_normal((VOCAB, 64)) * 0.1).astype(f32),
             "wpe": (rng.standard_normal((N_CTX, 64)) * 0.1).astype(f32),
             "ln_f_g": (1 + 0.1 * rng.standard_normal(64)).astype(f32), "ln_f_b": (0.1 * rng.standard_normal(64)).astype(f32),
             "layers": []}
    for i in range(LAYERS):
        p = gpt2.make_block_params(20 + i, CFG)
        for k in p:
            if k.startswith("w_"):
                p[k] = (rng.standard_normal(p[k].shape) * 0.1).astype(f32)
            else:
                p[k] = (p[k] + 0.1 * rng.standard_normal(p[k].shape)).astype(f32)
        model["layers"].append(p)
    tokens = rng.integers(0, VOCAB, (2, 25))
    labels = tokens[:, 1:].astype(np.int32)
    labels[1, 18:] = -1        # a padded sentence
    return model, tokens[:, :-1].astype(f32), labels


def names(model):
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    return ["wte", "wpe"] + [(i, k) for i in range(len(model["layers"])) for k in gpt2.BLOCK_PARAMETERS] + ["ln_f_g", "ln_f_b"]


def test_float64_gradients_by_differences():
    model, tokens, labels = make_model()
    grads, _ = ref.model_gradients(tokens, labels, model, CFG["n_head"], CFG["eps"])
    wide = {k: (v.astype(np.float64) if k != "layers" else [{n: a.astype(np.float64) for n, a in p.items()} for p in v])
            for k, v in model.items()}
    rng = np.random.default_rng(3)
    for name in ("wte", "wpe", "ln_f_g", (0, "w_qkv"), (1, "w_fc"), (1, "ln2_g"), (0, "b_o")):
        at = wide[name] if isinstance(name, str) else wide["layers"][name[0]][name[1]]
        direction = rng.standard_normal(at.shape)
        h, value = 1e-5, []
        for sign in (1, -1):
            at += sign * h * direction
            value.append(ref.model_loss(tokens, labels, wide, CFG["n_head"], CFG["eps"]))
            at -= sign * h * direction
        numeric, exact = (value[0] - value[1]) / (2 * h), (grads[name] * direction).sum()
        assert abs(numeric - exact) <= 1e-6 * max(abs(exact), 1e-3), name


def device_model(W, model):
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    return {k: (W.HIPTensor.from_numpy(v) if k != "layers" else [gpt2.to_device(p) for p in v]) for k, v in model.items()}


@pytest.mark.gpu
def test_loss_and_gradients(gpu):
    W = gpu
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    model, tokens, labels = make_model()
    dev = device_model(W, model)
    saved = {}
    t, l = W.HIPTensor.from_numpy(tokens), W.HIPTensor.from_numpy(labels, dtype="int32")
    loss = gpt2.model_loss(t, l, dev, CFG, saved=saved)
    want = ref.model_loss(tokens, labels, model, CFG["n_head"], CFG["eps"])
    assert abs(float(loss.numpy()[0]) - want) <= 1e-5 * abs(want)
    assert float(gpt2.model_loss(t, l, dev, CFG).numpy()[0]) == float(loss.numpy()[0])
    got = gpt2.model_gradients(saved, dev, CFG)
    grads, scales = ref.model_gradients(tokens, labels, model, CFG["n_head"], CFG["eps"])
    assert len(got) == len(gpt2.model_parameters(dev)) == len(names(model))
    for name, g, p in zip(names(model), got, gpt2.model_parameters(dev)):
        assert g.shape == p.shape, name
        # the yardstick of the block's backward: 2e-4 of the magnitude that the gradient's last product or sum adds up
        assert np.all(np.abs(g.numpy() - grads[name]) <= 2e-4 * scales[name] + 1e-7), name


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(gpu, bits):
    """Six steps; each is AdamW's on the gradients and the states of the moment, to the bounds of the optimiser's own
    tests."""
    W = gpu
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    model, tokens, labels = make_model(seed=5)
    dev = device_model(W, model)
    t, l = W.HIPTensor.from_numpy(tokens), W.HIPTensor.from_numpy(labels, dtype="int32")
    params = gpt2.model_parameters(dev)
    decay = [0.1 if len(p.shape) == 2 else 0.0 for p in params]
    opt = W.optimizers.AdamW(params, weight_decay=decay, state_bits=bits, **HYPER)
    for step in range(1, 7):
        before = [p.numpy().ravel() for p in params]
        states = {k: ([W.HIPTensor.from_numpy(t_.numpy(), dtype=t_.dtype) for t_ in v] if k != "n" else v)
                  for k, v in opt.state().items()}     # copies: the step moves the tensors themselves
        saved = {}
        loss = gpt2.model_loss(t, l, dev, CFG, saved=saved)
        grads = [g.numpy().ravel() for g in gpt2.model_gradients(saved, dev, CFG)]
        again = gpt2.train_step(t, l, dev, opt, CFG) if step % 2 else None
        if again is None:
            opt.step([W.HIPTensor.from_numpy(g.reshape(p.shape)) for g, p in zip(grads, params)])
        else:
            assert float(again.numpy()[0]) == float(loss.numpy()[0])
        assert opt.n == step
        for i, p in enumerate(params):
            if bits == 32:
                m, v = states["m"][i].numpy().ravel(), states["v"][i].numpy().ravel()
                want, _, _, bound, _, _ = reference(before[i], grads[i], m, v, step, decay[i])
            else:
                m = decode(states["m"][i].numpy(), states["m_scale"][i].numpy())
                v = decode(states["r"][i].numpy(), states["r_scale"][i].numpy()) ** 2
                want, m1, v1, bound, _, _ = reference(before[i], grads[i], m, v, step, decay[i])
                root = np.sqrt(v1 / (1 - HYPER["beta2"] ** step)) + HYPER["eps"]
                bound = bound + HYPER["lr"] / (1 - HYPER["beta1"] ** step) * (
                    2 * U * np.abs(m) + np.abs(m1) * 2 * U * v / np.maximum(v1, 1e-300)) / root
            assert np.all(np.abs(p.numpy().ravel() - want) <= bound), (names(model)[i], step)
    assert all(np.isfinite(p.numpy()).all() for p in params)


@pytest.mark.gpu
def test_recorded_training_step(gpu):
    """The whole step recorded once and replayed: parameters and loss follow the eager steps bit for bit."""
    W = gpu
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    model, tokens, labels = make_model(seed=8)
    runs = []
    for recorded in (False, True):
        dev = device_model(W, model)
        t, l = W.HIPTensor.from_numpy(tokens), W.HIPTensor.from_numpy(labels, dtype="int32")
        opt = W.optimizers.AdamW(gpt2.model_parameters(dev), lr=1e-3, state_bits=8)
        losses = [gpt2.train_step(t, l, dev, opt, CFG).numpy()[0]]
        if recorded:
            with W.lib.Graph() as g:
                out = gpt2.train_step(t, l, dev, opt, CFG)
            for _ in range(4):
                g.launch()
                losses.append(out.numpy()[0])
                junk = W.functional.exp(W.HIPTensor([300, 64], initial_element=0.5))   # eager work between replays
                assert junk.numpy()[0, 0] == f32(np.exp(np.float64(0.5)))
            g.destroy()
        else:
            for _ in range(4):
                losses.append(gpt2.train_step(t, l, dev, opt, CFG).numpy()[0])
        assert opt.n == 5
        runs.append((losses, [p.numpy() for p in gpt2.model_parameters(dev)]))
    assert runs[0][0] == runs[1][0]
    assert all(np.array_equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))
