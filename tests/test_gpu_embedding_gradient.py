"""The gradient of the GPT-2 example's embedding node against float64.

Tolerance: a token's k rows are added up in binary32 and then to the table: k additions, each within half a step, 2^-24 of
a partial sum, which the sum of the magnitudes bounds."""
import ctypes as C
import importlib

import numpy as np
import pytest

f32 = np.float32
U = 2.0 ** -24


def reference(ids, dout, dwte, dwpe):
    vocab = dwte.shape[0]
    nearest = np.rint(np.nan_to_num(ids, nan=-1.0, posinf=3e38, neginf=-1.0).astype(np.float64))
    tokens = np.clip(nearest, 0, vocab - 1).astype(np.int64).ravel()
    d = dout.astype(np.float64).reshape(len(tokens), -1)
    a, b = dwte.astype(np.float64), dwpe.astype(np.float64)
    ma, mb, count = np.abs(a), np.abs(b), np.zeros(vocab)
    np.add.at(a, tokens, d)
    np.add.at(ma, tokens, np.abs(d))
    np.add.at(count, tokens, 1)
    t = ids.shape[1]
    b[:t] += dout.astype(np.float64).sum(axis=0)
    mb[:t] += np.abs(dout).astype(np.float64).sum(axis=0)
    return a, b, (count[:, None] + 1) * U * ma, (ids.shape[0] + 1) * U * mb


def numbers(n, t, vocab, n_ctx, dim, seed=0):
    rng = np.random.default_rng(seed + n * 1000 + t)
    ids = np.floor(vocab * rng.random((n, t)) ** 3).astype(f32)     # a few words often, most seldom
    return ids, rng.standard_normal((n, t, dim)).astype(f32), rng.standard_normal((vocab, dim)).astype(f32), \
        rng.standard_normal((n_ctx, dim)).astype(f32)


def run(W, ids, dout, dwte, dwpe):
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    h = [W.HIPTensor.from_numpy(a) for a in (ids, dout, dwte, dwpe)]
    a, b = gpt2.positional_embedding_backward(*h)
    assert a is h[2] and b is h[3]
    return a.numpy(), b.numpy()


def check(W, *data):
    got = run(W, *data)
    a, b, ea, eb = reference(*data)
    assert np.all(np.abs(got[0] - a) <= ea), np.max(np.abs(got[0] - a) / np.maximum(ea, 1e-30))
    assert np.all(np.abs(got[1] - b) <= eb)
    assert all(np.array_equal(x, y) for x, y in zip(got, run(W, *data))), "the same call gives the same bits"
    # rows that no id names and positions behind the sentence are left as they were
    named = np.unique(np.clip(np.rint(np.nan_to_num(data[0], nan=0, posinf=3e38, neginf=0)), 0, len(a) - 1).astype(np.int64))
    rest = np.setdiff1d(np.arange(len(a)), named)
    assert np.array_equal(got[0][rest], data[2][rest]) and np.array_equal(got[1][data[0].shape[1]:], data[3][data[0].shape[1]:])


SHAPES = [(1, 1, 1, 1, 1), (1, 1, 5, 3, 4), (2, 7, 50, 16, 12), (2, 24, 300, 32, 64), (3, 33, 1000, 64, 70), (5, 51, 3, 51, 33),
          (1, 257, 70000, 300, 20), (2, 100, 5000, 128, 768), (8, 1024, 50257, 1024, 96), (9, 200, 13, 200, 1025), (64, 17, 97, 17, 8),
          (700, 3, 40, 4, 36), (300, 1, 5000, 2, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,t,vocab,n_ctx,dim", SHAPES)
def test_against_float64(gpu, n, t, vocab, n_ctx, dim):
    check(gpu, *numbers(n, t, vocab, n_ctx, dim))


@pytest.mark.gpu
def test_one_token_everywhere(gpu):
    """All rows name one token: a list sorted bit by bit, a token in every run."""
    ids, dout, dwte, dwpe = numbers(5, 1000, 40, 1000, 36)
    ids[:] = 17
    check(gpu, ids, dout, dwte, dwpe)
    ids[0, ::2] = 16
    check(gpu, ids, dout, dwte, dwpe)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [3, 2000])
def test_more_rows_of_a_class_than_its_lists_hold(gpu, vocab):
    """26000 rows of a few tokens of one class (lists hold 8192): turns one after the other into the same rows."""
    ids, dout, dwte, dwpe = numbers(13, 2000, vocab, 2000, 12)
    ids[:] = 1 if vocab == 3 else 1 + 256 * (np.arange(2000) % 5)
    ids[5, :700] = 2
    check(gpu, ids, dout, dwte, dwpe)


@pytest.mark.gpu
@pytest.mark.parametrize("n,t,vocab,n_ctx,dim", [(4, 300, 50, 300, 1600), (2, 500, 3000, 512, 1284), (3, 40, 9, 40, 401),
                                                 (20, 500, 4000, 500, 260), (3, 70, 500, 70, 2052)])
def test_columns_shared_out(gpu, n, t, vocab, n_ctx, dim):
    """Rows of several slices of 64 vectors (64 elements where a row is no multiple of 16 bytes), which up to four
    workgroups share: two, three and four of them, equal and unequal shares."""
    check(gpu, *numbers(n, t, vocab, n_ctx, dim))


@pytest.mark.gpu
@pytest.mark.parametrize("distinct", [2, 17, 4096])
def test_long_lists_of_many_tokens(gpu, distinct):
    """9600 rows of one class whose tokens differ in up to twelve bits above those of the class."""
    ids, dout, dwte, dwpe = numbers(16, 600, (1 << 20) + 3, 600, 4)
    ids[:] = 1 + 256 * np.random.default_rng(distinct).integers(0, distinct, ids.shape)
    check(gpu, ids, dout, dwte, dwpe)
    ids[:] = np.random.default_rng(distinct).integers(0, (1 << 20) + 3, ids.shape)
    check(gpu, ids, dout, dwte, dwpe)


@pytest.mark.gpu
def test_ids_are_read_as_the_forward_reads_them(gpu):
    ids, dout, dwte, dwpe = numbers(1, 11, 10, 16, 8)
    ids[0] = [0.5, 1.5, 2.5, 3.49, 8.6, 9.0, 42.0, -3.0, np.nan, np.inf, -np.inf]
    check(gpu, ids, dout, dwte, dwpe)


@pytest.mark.gpu
def test_gradient_is_the_forwards(gpu):
    """<dout, forward(wte + h a, wpe + h b) - forward(wte, wpe)> = h (<dwte, a> + <dwpe, b>): the node is linear in its tables."""
    W = gpu
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    ids, dout, _, _ = numbers(3, 20, 60, 24, 16)
    rng = np.random.default_rng(4)
    a, b = rng.standard_normal((60, 16)).astype(f32), rng.standard_normal((24, 16)).astype(f32)
    out = gpt2.positional_embedding(*(W.HIPTensor.from_numpy(x) for x in (ids, a, b))).numpy()
    dwte, dwpe = run(W, ids, dout, np.zeros_like(a), np.zeros_like(b))
    left = (dout.astype(np.float64) * out).sum()
    right = (dwte.astype(np.float64) * a).sum() + (dwpe.astype(np.float64) * b).sum()
    assert abs(left - right) <= 1e-5 * np.abs(dout.astype(np.float64) * out).sum()


@pytest.mark.gpu
def test_replay_adds_once_more(gpu):
    W = gpu
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    data = numbers(4, 64, 500, 64, 48)
    h = [W.HIPTensor.from_numpy(a) for a in data]
    e = [W.HIPTensor.from_numpy(a) for a in data]
    with W.lib.Graph() as g:
        gpt2.positional_embedding_backward(*h)
    for _ in range(3):
        g.launch()
        gpt2.positional_embedding_backward(*e)
        assert all(np.array_equal(x.numpy(), y.numpy()) for x, y in zip(h[2:], e[2:]))
    g.destroy()


@pytest.mark.gpu
def test_argument_checks(gpu):
    W = gpu
    gpt2 = importlib.import_module("cl-waffe2_amd.gpt2")
    lib = W.lib.get()
    ctx, dout, dwte, dwpe = W.HIPTensor([2, 6]), W.HIPTensor([2, 6, 8]), W.HIPTensor([10, 8]), W.HIPTensor([7, 8])
    p = lambda t: C.c_void_p(t.ptr)  # noqa: E731
    f = lib.wf2hip_embedding_gradient_f32
    assert f(12, 6, 8, p(ctx), p(dout), p(dwte), 10, p(dwpe), 7) == 0
    assert f(0, 6, 8, None, None, None, 10, None, 7) == 0
    assert f(-1, 6, 8, p(ctx), p(dout), p(dwte), 10, p(dwpe), 7) == W.lib.EINVAL
    assert f(12, 5, 8, p(ctx), p(dout), p(dwte), 10, p(dwpe), 7) == W.lib.EINVAL
    assert f(12, 12, 8, p(ctx), p(dout), p(dwte), 10, p(dwpe), 7) == W.lib.EINVAL
    assert f(12, 6, 8, p(ctx), p(dout), p(dwte), 0, p(dwpe), 7) == W.lib.EINVAL
    assert f(12, 6, 8, None, p(dout), p(dwte), 10, p(dwpe), 7) == W.lib.EINVAL
    assert f(2 ** 31, 2, 8, p(ctx), p(dout), p(dwte), 10, p(dwpe), 7) == W.lib.EUNSUPPORTED
    assert f(12, 6, 8, p(ctx), p(dout), p(dout), 10, p(dwpe), 7) == W.lib.EOVERLAP
    assert f(12, 6, 8, p(ctx), p(dout), p(dwte), 10, p(dwte), 7) == W.lib.EOVERLAP
    for bad in (lambda: gpt2.positional_embedding_backward(ctx, W.HIPTensor([2, 6, 7]), dwte, dwpe),
                lambda: gpt2.positional_embedding_backward(ctx, dout, W.HIPTensor([10, 8], dtype="double"), dwpe),
                lambda: gpt2.positional_embedding_backward(ctx, dout, dwte.view((0, 5), True), dwpe),
                lambda: gpt2.positional_embedding_backward(ctx, dout, dwte, W.HIPTensor([7, 9]))):
        with pytest.raises(ValueError):
            bad()
