"""Token log probabilities, entropy, alternatives and their gradient against plain 64-bit arithmetic."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from rustingbrain_b200 import InvalidInput, _lib

INF = float("inf")


# ---- refusals: no device needed -------------------------------------------------------------------------------------
def _forward(x=None, stride=8, targets=None, rows=1, vocab=8, top=0, precision=_lib.PRECISION_F32, tl=None, ti=None):
    msg = C.create_string_buffer(128)
    rc = _lib.lib().logprobs_forward(x, stride, targets, rows, vocab, top, precision, None, None, None, tl, ti, None, msg, 128)
    return rc, msg.value.decode()


def test_arguments_are_checked_before_any_device_work():
    buf = (C.c_float * 64)()
    p = C.cast(buf, C.c_void_p)
    assert _forward(p, rows=0)[0] == _lib.OK
    assert _forward(None, rows=0)[0] == _lib.OK
    assert _forward(p, precision=_lib.PRECISION_Q8)[0] == _lib.INVALID_CONFIG
    for bad in (dict(rows=-1), dict(vocab=0), dict(stride=7), dict(top=-1), dict(top=9), dict(top=33, vocab=64, stride=64), dict(top=2, tl=p),
                dict(top=2, ti=p)):
        rc, text = _forward(p, **bad)
        assert rc == _lib.INVALID_INPUT and text, bad
    assert _forward(None)[0] == _lib.INVALID_INPUT
    assert _forward(C.c_void_p(p.value + 2))[0] == _lib.INVALID_INPUT           # not aligned to its type

    def back(x=p, xs=8, lse=p, h=p, gl=p, gh=p, rows=1, vocab=8, g=p, gs=8, precision=_lib.PRECISION_F32):
        msg = C.create_string_buffer(128)
        return _lib.lib().logprobs_backward(x, xs, None, lse, h, gl, gh, rows, vocab, precision, g, gs, None, msg, 128)
    assert back(rows=0) == _lib.OK
    assert back(precision=7) == _lib.INVALID_CONFIG
    for bad in (dict(x=None), dict(g=None), dict(lse=None), dict(h=None), dict(gs=7), dict(xs=7), dict(vocab=0), dict(rows=-1), dict(gs=16),
                dict(g=C.c_void_p(p.value + 1)), dict(rows=0x7fffffff, vocab=1 << 20, xs=1 << 20, gs=1 << 20)):
        assert back(**bad) == _lib.INVALID_INPUT, bad


def test_the_wrapper_refuses_what_the_kernels_do_not_read():
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    x = torch.zeros(2, 8)
    with pytest.raises(InvalidInput):
        token_logprobs(x)                                                        # not on a device
    with pytest.raises(InvalidInput):
        token_logprobs_backward(x, None, torch.zeros(2))


# ---- against 64 bits ------------------------------------------------------------------------------------------------
def _plain(x, t, top):
    """x as the device sees it, float64."""
    lse = torch.logsumexp(x, 1)
    logp = x - lse[:, None]
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    t = t.long()
    lp = torch.where(t >= 0, logp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0], torch.zeros_like(lse))
    ids = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -x.cpu().numpy()), axis=1)[:, :top]
    return lp, entropy, lse, ids


def _tolerances(x, lse, entropy):
    """A thread adds at most vocab / 256 + 2 vectors' logits one after the other, each sum off by half a unit (2^-24); the exponentials
    are good to 2^-22 and their arguments to 2^-24 of themselves; the result is scaled by two rounded constants."""
    V = x.shape[1]
    s = (V / 256 + 80) * 2.0 ** -24 + 2.0 ** -22
    big = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(1)
    at = s + 2.0 ** -22 * (big + torch.nan_to_num(lse, 0, 0, 0).abs())
    return at, at * (1 + entropy) + 2.0 ** -23 * entropy


def _check(x, t, top, got):
    xd = x.double()
    lp, entropy, lse, ids = _plain(xd, t, top)
    a, ah = _tolerances(xd, lse, entropy)
    for name, mine, want, tol in (("lse", got.lse, lse, a), ("logprob", got.logprob, lp, a), ("entropy", got.entropy, entropy, ah)):
        same = (mine.double() == want) | ((mine.double() - want).abs() <= tol)
        assert bool(same.all()), (name, float((mine.double() - want).abs().max()))
    if top:
        assert np.array_equal(got.top_ids.cpu().numpy(), ids)
        want = xd.gather(1, torch.from_numpy(ids).cuda()) - lse[:, None]
        d = (got.top_logprobs.double() - want).abs()
        assert bool(((d <= a[:, None]) | (got.top_logprobs.double() == want)).all())


def _logits(rows, vocab, dtype, seed, stride=None, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, device="cuda", generator=g) * 3
    if stride is None:
        return x.to(dtype)
    flat = torch.full((rows * stride + offset,), 1e4, device="cuda", dtype=dtype)      # what lies between rows must not be read as logits
    view = flat[offset:].view(rows, stride)[:, :vocab]
    view.copy_(x)
    return view


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 2), (5, 7, 7), (3, 8, 1), (2, 31, 31), (70, 1000, 5), (1, 4097, 32), (3, 32003, 20),
                                            (1, 131072, 32), (1, 131071, 3), (300, 2049, 4), (700, 513, 0), (1200, 100, 8)])
def test_rows_of_every_length(dtype, rows, vocab, top):
    from rustingbrain_b200.logprobs import token_logprobs
    x = _logits(rows, vocab, dtype, rows + vocab)
    t = torch.randint(0, vocab, (rows,), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(1))
    t[1::3] = -1
    _check(x, t, top, token_logprobs(x, t, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("stride,offset", [(1008, 0), (1003, 0), (1003, 1), (1001, 5), (2000, 3)])
def test_rows_apart_and_off_the_16_byte_boundary(dtype, stride, offset):
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    x = _logits(9, 1001, dtype, 3, stride, offset)
    t = torch.arange(9, device="cuda", dtype=torch.int32) * 111
    got = token_logprobs(x, t, top=6)
    _check(x, t, 6, got)
    g = torch.linspace(-1, 1, 9, device="cuda")
    want = token_logprobs_backward(x.contiguous(), t, got.lse, got.entropy, g, g)
    for out in (None, _logits(9, 1001, dtype, 4, stride, offset), _logits(9, 1001, dtype, 4, 1007, 2)):
        assert torch.equal(token_logprobs_backward(x, t, got.lse, got.entropy, g, g, out=out), want)
    base = x.clone()
    assert token_logprobs_backward(x, t, got.lse, got.entropy, g, g, out=x) is x and torch.equal(x, want)      # in place
    assert not torch.equal(base, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [2, 700])
def test_ties_go_to_the_lower_index(dtype, rows):
    from rustingbrain_b200.logprobs import token_logprobs
    V = 9001
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-3, 3, (rows, V), device="cuda", generator=g).to(dtype)
    x[0] = 2.5                                                  # a constant row
    x[1] = torch.arange(V, device="cuda").to(dtype)             # ascending: the best sit in neighbouring vectors
    if rows > 2:
        x[2] = -torch.arange(V, device="cuda").to(dtype)
        x[3], x[3, 17], x[3, 5000] = 0.0, -0.0, -0.0            # zeros of both signs are equal
    t = torch.zeros(rows, device="cuda", dtype=torch.int32)
    _check(x, t, 32, token_logprobs(x, t, top=32))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 300])
def test_thousands_of_logits_above_the_bound(rows):
    """Nineteen threads' vectors hold everything that is large, and the twentieth best thread has nothing of it: all of the large
    ones pass the bound."""
    from rustingbrain_b200.logprobs import token_logprobs
    V, step = 16384, 256 if rows > 1 else 2048
    x = _logits(rows, V, torch.float32, 5)
    x += 50.0 * (((torch.arange(V, device="cuda") // 4) % step) < 19)
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    _check(x, t, 20, token_logprobs(x, t, top=20))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [40, 5000])
def test_masked_rows_and_extreme_values(dtype, vocab):
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = _logits(12, vocab, dtype, 6)
    x[0] = -INF                                  # nothing left
    x[1] = -INF; x[1, 7] = 3.0                   # one token left
    x[2, 3:] = -INF
    x[3] = low                                   # everything masked with the lowest value: uniform
    x[4, 5:] = low
    x[5, ::2] = -INF; x[5, 1::2] = low
    x[6, 9] = high
    x[7] *= 1e30
    x[8, 4] = float("nan")
    x[9, 4] = INF
    x[10, : vocab // 2] = -INF
    t = torch.full((12,), 7, device="cuda", dtype=torch.int32)
    t[11] = vocab
    top = 10
    got = token_logprobs(x, t, top=top)
    fine = torch.tensor([1, 2, 3, 4, 5, 6, 7, 10], device="cuda")
    _check(x[fine], t[fine], top, type(got)(*(f[fine] for f in got)))
    assert float(got.lse[0]) == -INF and float(got.logprob[0]) == -INF and float(got.entropy[0]) == 0
    assert got.top_ids[0].tolist() == list(range(top)) and bool((got.top_logprobs[0] == -INF).all())
    assert bool(got.lse[8:10].isnan().all()) and bool(got.entropy[8:10].isnan().all()) and bool(got.logprob[8:10].isnan().all())
    assert bool(((got.top_ids >= -1) & (got.top_ids < vocab)).all())
    assert bool(got.logprob[11].isnan()) and bool(got.lse[11].isfinite())        # a token that does not exist
    g = torch.ones(12, device="cuda")
    grad = token_logprobs_backward(x, t, got.lse, got.entropy, g, g)
    assert float(grad[0].abs().max()) == 0
    assert bool(grad[[8, 9, 11]].isnan().all()) and bool(grad[fine].isfinite().all())
    assert float(grad[10, 8: vocab // 2].abs().max()) == 0                       # masked tokens other than the given one


def _plain_grad(x, t, gl, gh):
    """By automatic differentiation of the definition, in 64 bits."""
    x = x.double().requires_grad_(True)
    logp = torch.log_softmax(x, 1)
    keep = t >= 0
    lp = logp.gather(1, t.long().clamp(min=0)[:, None])[:, 0]
    entropy = -(logp.exp() * torch.where(torch.isfinite(logp), logp, torch.zeros_like(logp))).sum(1)
    ((lp * gl.double())[keep].sum() + (entropy * gh.double()).sum()).backward()
    return x.grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 3), (4, 9), (33, 1000), (5, 32003), (2, 8192)])
def test_gradient(dtype, rows, vocab):
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    x = _logits(rows, vocab, dtype, 7)
    if vocab > 4:
        x[:, 2:4] = -INF
    gen = torch.Generator(device="cuda").manual_seed(8)
    t = torch.zeros(rows, device="cuda", dtype=torch.int32)
    t[1::2] = -1
    gl, gh = torch.randn(rows, device="cuda", generator=gen), torch.randn(rows, device="cuda", generator=gen)
    fwd = token_logprobs(x, t)
    for a, b in ((gl, gh), (gl, None), (None, gh), (None, None)):
        got = token_logprobs_backward(x, t, fwd.lse, fwd.entropy, a, b)
        zero = torch.zeros_like(gl)
        want = _plain_grad(x, t, zero if a is None else a, zero if b is None else b)
        # lse and entropy are off by some 2^-21, p by as much of itself; then the gradient's own rounding
        scale = (0 if a is None else a.abs().double()) + (0 if b is None else b.abs().double() * (40 + fwd.entropy.double()))
        p = torch.softmax(x.double(), 1)
        hot = torch.zeros_like(p).scatter_(1, t.long().clamp(min=0)[:, None], 1.0)
        s = (vocab / 256 + 80) * 2.0 ** -24 + 2.0 ** -20
        tol = (p + hot * 2.0 ** -3) * s * (scale[:, None] if torch.is_tensor(scale) else scale) + want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + 1e-38
        assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() - tol).max())


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the 64-bit forward formula around the very logits the kernel saw."""
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    V = 37
    x = _logits(2, V, torch.float32, 9)
    t = torch.tensor([5, -1], device="cuda", dtype=torch.int32)
    gl, gh = torch.tensor([0.7, 0.3], device="cuda"), torch.tensor([-0.4, 1.1], device="cuda")
    fwd = token_logprobs(x, t)
    got = token_logprobs_backward(x, t, fwd.lse, fwd.entropy, gl, gh).double()

    def value(y):
        lp, h, _, _ = _plain(y, t, 0)
        return lp * gl.double() + h * gh.double()
    h = 1e-5
    for v in range(V):
        e = torch.zeros(2, V, device="cuda", dtype=torch.float64)
        e[:, v] = h
        want = (value(x.double() + e) - value(x.double() - e)) / (2 * h)
        assert float((got[:, v] - want).abs().max()) < 2e-6       # h^2 of the third derivative, 1e-16 / h of the rounding, f32


@pytest.mark.gpu
def test_streams_graphs_and_no_rows():
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    x = _logits(4, 5003, torch.bfloat16, 10)
    t = torch.tensor([1, 2, 3, -1], device="cuda", dtype=torch.int32)
    want = token_logprobs(x, t, top=3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = token_logprobs(x, t, top=3)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    g = torch.ones(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = token_logprobs(x, t, top=3)
        grad = token_logprobs_backward(x, t, got.lse, got.entropy, g, g)
    x.copy_(_logits(4, 5003, torch.bfloat16, 11))
    graph.replay()
    torch.cuda.synchronize()
    want = token_logprobs(x, t, top=3)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert torch.equal(grad, token_logprobs_backward(x, t, want.lse, want.entropy, g, g))
    none = token_logprobs(x[:0], t[:0], top=2)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 2)
    assert token_logprobs_backward(x[:0], t[:0], none.lse).shape == (0, 5003)
    for bad in (dict(targets=t.long()), dict(targets=t[:2]), dict(top=33), dict(top=-1)):
        with pytest.raises(InvalidInput):
            token_logprobs(x, **{**dict(targets=t), **bad})
    with pytest.raises(InvalidInput):
        token_logprobs(x.t())
    with pytest.raises(InvalidInput):
        token_logprobs(x.half())
    with pytest.raises(InvalidInput):
        token_logprobs_backward(x, t, None, None, g)
    with pytest.raises(InvalidInput):
        token_logprobs_backward(x, t, want.lse, None, None, g)


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run():
    from rustingbrain_b200.logprobs import token_logprobs
    x = _logits(64, 32003, torch.bfloat16, 12)
    t = torch.zeros(64, device="cuda", dtype=torch.int32)
    first = token_logprobs(x, t, top=8)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, token_logprobs(x, t, top=8)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_probability_above_one(dtype):
    """One token left, logits of every size: its log probability is 0, and what rounding leaves of it is not above 0."""
    from rustingbrain_b200.logprobs import token_logprobs
    rows, V = 4096, 40
    x = torch.full((rows, V), -INF, device="cuda")
    t = torch.arange(rows, device="cuda") % V
    x[torch.arange(rows, device="cuda"), t] = torch.linspace(-40, 40, rows, device="cuda")
    x, t = x.to(dtype), t.to(torch.int32)
    got = token_logprobs(x, t, top=2)
    _check(x, t, 2, got)
    assert float(got.logprob.max()) <= 0 and float(got.top_logprobs.max()) <= 0
    assert float(got.entropy.min()) >= 0
    x[1::2, :] = 0.0                             # a peak far above the others
    x[torch.arange(rows, device="cuda"), t.long()] += 30.0
    got = token_logprobs(x, t, top=2)
    _check(x, t, 2, got)
    assert float(got.logprob.max()) <= 0 and float(got.top_logprobs.max()) <= 0


def test_a_gradient_that_overlaps_the_logits_is_refused():
    """In place, or beside the logits: anything else would overwrite logits that another row's gradient has yet to read."""
    buf = (C.c_float * 256)()
    p = C.addressof(buf)

    def back(x, xs, g, gs, rows, vocab=8, precision=_lib.PRECISION_F32):
        msg = C.create_string_buffer(128)
        o = C.c_void_p(p)
        rc = _lib.lib().logprobs_backward(C.c_void_p(p + x), xs, None, o, o, o, o, rows, vocab, precision, C.c_void_p(p + g), gs, None, msg, 128)
        return rc, msg.value
    for bad in ((0, 8, 4, 8, 1), (4, 8, 0, 8, 1), (0, 8, 28, 8, 1), (0, 8, 32, 8, 2), (0, 16, 16, 16, 3), (0, 16, 60, 16, 3), (0, 16, 36, 16, 3),
                (0, 16, 32, 24, 3), (64, 16, 4, 8, 3), (0, 8, 8, 8, 1, 8, _lib.PRECISION_BF16)):
        rc, text = back(*bad)
        assert rc == _lib.INVALID_INPUT and b"overlap" in text, bad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_beside_their_logits(dtype):
    """Rows of the gradient between those of the logits, on either side and at distances of their own."""
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    V, rows = 100, 5
    g = torch.linspace(-1, 1, rows, device="cuda")
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    for x_at, x_step, d_at, d_step in ((0, 200, 100, 200), (100, 200, 0, 200), (0, 213, 107, 213), (0, 200, 100, 400), (100, 600, 0, 300), (0, 100, 500, 300)):
        buf = torch.full((4000,), 7.0, device="cuda", dtype=dtype)
        x = buf.as_strided((rows, V), (x_step, 1), x_at)
        d = buf.as_strided((rows, V), (d_step, 1), d_at)
        x.copy_(_logits(rows, V, dtype, 50))
        base = x.clone()
        f = token_logprobs(x, t)
        want = token_logprobs_backward(base, t, f.lse, f.entropy, g, g)
        token_logprobs_backward(x, t, f.lse, f.entropy, g, g, out=d)
        assert torch.equal(d, want) and torch.equal(x, base)
    with pytest.raises(InvalidInput, match="overlap"):
        token_logprobs_backward(x, t, f.lse, f.entropy, g, g, out=buf.as_strided((rows, V), (x_step, 1), 50))


@pytest.mark.gpu
def test_the_largest_vocabulary():
    """A row of 2^31 - 1 logits, whose gradient lies off their 16-byte boundary: indices end at the last number of 31 bits."""
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    V = 2 ** 31 - 1
    x = torch.zeros(1, V, device="cuda", dtype=torch.bfloat16)
    x[0, V - 1], x[0, 5] = 4.0, 3.0
    t = torch.tensor([V - 1], device="cuda", dtype=torch.int32)
    got = token_logprobs(x, t, top=3)
    assert got.top_ids[0].tolist() == [V - 1, 5, 0]
    lse, g = torch.ones(1, device="cuda"), torch.ones(1, device="cuda")
    for shift in (0, 1):
        flat = torch.full((V + 9,), 7.0, device="cuda", dtype=torch.bfloat16)
        out = flat[shift:shift + V].view(1, V)
        token_logprobs_backward(x, t, lse, grad_logprob=g, out=out)
        for at, want in ((0, -np.exp(-1.0)), (5, -np.exp(2.0)), (V // 2, -np.exp(-1.0)), (V - 2, -np.exp(-1.0)), (V - 1, 1 - np.exp(3.0))):
            assert abs(float(out[0, at]) - want) <= abs(want) * (2.0 ** -8 + 2.0 ** -20), (shift, at)
        assert int((out == out[0, 0]).sum()) == V - 2
        assert bool((flat[:shift] == 7).all()) and bool((flat[shift + V:] == 7).all())
        del flat, out
