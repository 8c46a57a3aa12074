"""4-bit projections, 4-bit cache, log probabilities: together as a decode step uses them, and inside the language model."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from helpers import rel_l2
from oracle import norm as rms
from oracle import transformer as T
from oracle.kv_q4 import Q4CacheOracle, to_bf16
from rustingbrain_b200 import InvalidConfig, InvalidInput, _lib
from rustingbrain_b200 import transformer as D
from rustingbrain_b200.kv_attention import KvCache
from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
from rustingbrain_b200.q4_linear import Q4Linear


# ---- no device needed -----------------------------------------------------------------------------------------------
def test_the_models_entry_points_refuse_without_a_model():
    L = _lib.lib()
    h = C.c_void_p()
    assert L.lm_decoder_create_q4(None, 1, 1, C.byref(h)) == _lib.INVALID_INPUT
    assert L.lm_score(None, None, None, None, 1, 1, 0, None, None, None, None) == _lib.INVALID_INPUT


# ---- the operators one behind the other -----------------------------------------------------------------------------
class _Step:
    """One attention block with 4-bit projections and a 4-bit head, around a 4-bit cache."""

    def __init__(self, d, H, Hkv, hd, vocab, sequences, cap, group=32):
        self.d, self.H, self.Hkv, self.hd, self.vocab = d, H, Hkv, hd, vocab
        g = torch.Generator(device="cuda").manual_seed(5)
        self.weights = []
        def linear(d_in, d_out):
            w = Q4Linear(d_in, d_out, group_size=group)
            w.set_weight(torch.randn(d_out, d_in, generator=g, device="cuda") * d_in ** -0.5)
            return w
        self.wqkv, self.wo, self.head = linear(d, (H + 2 * Hkv) * hd), linear(H * hd, d), linear(d, vocab)
        self.cache = KvCache(sequences, H, Hkv, hd, capacity=cap, precision="q4")

    def run(self, x, tokens, g_lp, g_h, rows):
        qkv = self.wqkv(x)
        q, k, v = (t.contiguous() for t in qkv.split([self.H * self.hd, self.Hkv * self.hd, self.Hkv * self.hd], dim=1))
        merged = self.cache.forward_cached(q, k, v, rows_per_sequence=rows)
        y = self.wo(merged) + x
        logits = self.head(y)
        s = token_logprobs(logits, tokens, top=4)
        return q, k, v, merged, y, logits, s, token_logprobs_backward(logits, tokens, s.lse, s.entropy, g_lp, g_h)


def _near(got, want, tol):
    d = (got.double().cpu() - want).abs()
    assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("d,H,Hkv,hd,vocab,sequences,rows", [(128, 4, 1, 64, 301, 3, 1), (256, 4, 2, 128, 1000, 2, 3), (64, 2, 2, 32, 77, 1, 9)])
def test_a_run_of_the_operators(d, H, Hkv, hd, vocab, sequences, rows):
    """Each stage against 64-bit arithmetic on what it was given; then the same steps captured, replayed over an empty cache: the same bits."""
    steps, cap = 4, 4 * rows + 2
    st = _Step(d, H, Hkv, hd, vocab, sequences, cap)
    n = sequences * rows
    g = torch.Generator(device="cuda").manual_seed(6)
    xs = [torch.randn(n, d, generator=g, device="cuda").bfloat16() for _ in range(steps)]
    ts = [torch.randint(-1, vocab, (n,), generator=g, device="cuda", dtype=torch.int32) for _ in range(steps)]
    g_lp, g_h = torch.randn(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    oracles = [Q4CacheOracle(H, Hkv, hd, cap) for _ in range(sequences)]
    half = 2.0 ** -8                                                   # of a step of bf16, relative
    eager = []
    for x, t in zip(xs, ts):
        q, k, v, merged, y, logits, s, dx = st.run(x, t, g_lp, g_h, rows)
        eager.append([a.clone() for a in (merged, logits, s.logprob, s.entropy, s.top_logprobs, s.top_ids, dx)])
        for layer, given, got in ((st.wqkv, x, torch.cat([q, k, v], 1)), (st.head, y, logits)):
            w = layer.weight().double().cpu()
            a = given.double().cpu()
            # one rounding of the result, and f32 sums: at most 2^-23 of the terms' magnitudes for each term
            _near(got, a @ w.T, (a @ w.T).abs() * half * 1.0001 + a.abs() @ w.abs().T * (w.shape[1] * 1.2 * 2.0 ** -23))
        for i in range(sequences):
            sl = slice(i * rows, (i + 1) * rows)
            want, tol = oracles[i].forward_cached(*(a[sl].float().cpu().numpy() for a in (q, k, v)))
            _near(merged[sl], torch.from_numpy(want), torch.from_numpy(tol))
        w, a = st.wo.weight().double().cpu(), merged.double().cpu()
        z = a @ w.T
        # two roundings: the projection's and the sum's
        _near(y, z + x.double().cpu(), (z.abs() + (z + x.double().cpu()).abs() + 2.0 ** -6 * z.abs()) * half + a.abs() @ w.abs().T * (w.shape[1] * 1.2 * 2.0 ** -23))
        lg, tt = logits.double().cpu(), t.cpu().long()
        lse = torch.logsumexp(lg, 1)
        logp = lg - lse[:, None]
        entropy = -(logp.exp() * logp).sum(1)
        lp = torch.where(tt >= 0, logp.gather(1, tt.clamp(min=0)[:, None])[:, 0], torch.zeros(()).double())
        # f32 exponentials (relative 2^-20 with the rounding of their arguments, which are below 2^7 in magnitude) and sums of `vocab` of them
        e = 2.0 ** -17 + vocab * 2.0 ** -24
        _near(s.logprob, lp, e * (1 + lse.abs() + logp.abs().amax(1)))
        _near(s.entropy, entropy, e * (1 + lse.abs() + logp.abs().amax(1)))
        top, ids = torch.topk(lg, 4, dim=1)
        assert torch.equal(logits.gather(1, s.top_ids.long()).double().cpu(), top)
        p, hot = logp.exp(), torch.nn.functional.one_hot(tt.clamp(min=0), vocab).double() * (tt >= 0)[:, None]
        gl, gh = g_lp.double().cpu()[:, None] * (tt >= 0)[:, None], g_h.double().cpu()[:, None]
        want = gl * (hot - p) - gh * p * (logp + entropy[:, None])
        size = (gl.abs() + gh.abs() * (1 + logp.abs() + entropy[:, None])) * (p + hot)
        _near(dx, want, want.abs() * half * 1.01 + size * 16 * e + 1e-30)
    assert st.cache.lengths() == [steps * rows] * sequences
    # captured: one graph a step, in one pool
    st.cache.clear()
    side = torch.cuda.Stream()
    outs, graphs = [], []
    side.wait_stream(torch.cuda.current_stream())
    for x, t in zip(xs, ts):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            r = st.run(x, t, g_lp, g_h, rows)
        graphs.append(graph)
        outs.append((r[3], r[5], r[6].logprob, r[6].entropy, r[6].top_logprobs, r[6].top_ids, r[7]))
    st.cache.clear()
    for i, graph in enumerate(graphs):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs[i], eager[i]):
            assert torch.equal(a, b) or bool(((a == b) | (a != a)).all())
    assert st.cache.lengths() == [steps * rows] * sequences


# ---- inside the language model --------------------------------------------------------------------------------------
def _config(**over):
    c = T.default_config(vocab_size=101, d_model=128, n_layers=3, n_heads=4, n_kv_heads=2, head_dim=64, d_ff=96, moe_d_ff=64,
                         num_experts=4, experts_per_token=2, moe_layers=(1, 2), max_seq_len=64)
    c.update(over)
    return c


def _model(c, seed=3, std=0.08, rows=256):
    w = T.seeded_model_weights(c, seed, std=std)
    dev = D.TransformerLm.builder().config(D.TransformerConfig(**c)).max_batch_rows(rows).optimizer(D.Adam(1e-2)).build()
    dev.load_weights(w)
    return dev, w


def _sequences(vocab, lengths, seed=1):
    g = np.random.Generator(np.random.Philox(seed))
    return [list(g.integers(0, vocab, n)) for n in lengths]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,lengths,top,masked", [(101, [16, 16], 0, False), (101, [30, 7, 2], 5, False), (1000, [20, 33], 32, True), (3, [5, 9], 3, False)])
def test_scores_of_a_batch(vocab, lengths, top, masked):
    c = _config(vocab_size=vocab)
    dev, _ = _model(c)
    seqs = _sequences(vocab, lengths)
    S, B = max(lengths), len(lengths)
    mask = (np.arange(B * S) % 3 != 0) if masked else None
    batch = D.TokenBatch(seqs, mask)
    logits = dev.forward_batch(batch).astype(np.float64)              # bf16 numbers, as on the device
    lse = np.log(np.exp(logits - logits.max(1, keepdims=True)).sum(1)) + logits.max(1)
    logp = logits - lse[:, None]
    got = dev.score_batch(batch, top=top)
    e = (2.0 ** -17 + vocab * 2.0 ** -24) * (1 + np.abs(lse) + np.abs(logp).max(1))   # as above
    picked, n = 0.0, 0
    for i, s in enumerate(seqs):
        for t in range(S):
            r = i * S + t
            if t >= len(s):
                assert got.logprob[r] == 0 and got.entropy[r] == 0
                if top:
                    assert (got.top_ids[r] == -1).all() and (got.top_logprobs[r] == 0).all()
                continue
            if t + 1 < len(s) and (mask is None or mask[r + 1]):
                assert abs(got.logprob[r] - logp[r, s[t + 1]]) <= e[r]
                picked, n = picked + got.logprob[r], n + 1
            else:
                assert got.logprob[r] == 0
            assert abs(got.entropy[r] + (np.exp(logp[r]) * logp[r]).sum()) <= e[r]
            if top:
                order = np.lexsort((np.arange(vocab), -logits[r]))[:top]
                assert np.array_equal(got.top_ids[r], order)
                assert (np.abs(got.top_logprobs[r] - logp[r, order]) <= e[r]).all()
    dev.zero_grad()
    loss = dev.accumulate_step(batch).lm_loss
    assert abs(loss + picked / n) <= 2 * e.max()                       # both are f32 sums over the same logits
    dev.close()


@pytest.mark.gpu
def test_the_model_refuses_what_it_cannot_do():
    dev, _ = _model(_config())
    seqs = _sequences(101, [8, 8])
    for top in (-1, 33):
        with pytest.raises(InvalidInput):
            dev.score_batch(seqs, top=top)
    with pytest.raises(InvalidInput, match="TokenOutOfRange"):
        dev.score_batch([[1, 101]])
    with pytest.raises(InvalidInput, match="SequenceTooLong"):
        dev.score_batch(_sequences(101, [65]))
    with pytest.raises(InvalidConfig):
        dev.new_kv_caches(1, 8, precision="f32")
    with pytest.raises(InvalidConfig):
        dev.new_kv_caches(1, 65, precision="q4")
    lp = np.zeros(16, np.float32)
    ids = np.zeros(16, np.uint32)
    p = lambda a: a.ctypes.data_as(C.c_void_p)
    assert _lib.lib().lm_score(dev._h, p(ids), None, None, 2, 8, 2, p(lp), None, None, None) == _lib.INVALID_INPUT
    assert _lib.lib().lm_score(dev._h, p(ids), None, None, 2, 8, 0, None, None, None, None) == _lib.INVALID_INPUT
    assert _lib.lib().lm_score(dev._h, p(ids), None, None, 2, 8, 0, p(lp), None, None, None) == _lib.OK      # the entropy is optional
    dev.close()


def _decode_oracle(c, w, ids):
    """One sequence through dense blocks: norms and products in 32 bits on bf16 weights, the attention over what a 4-bit cache stands for."""
    bf = to_bf16
    x = bf(w["embedding"])[np.asarray(ids)]
    for b in w["blocks"]:
        n1 = bf(rms.forward(x, b["attention_norm"], c["rmsnorm_eps"]))
        q, k, v = (bf(T.linear_forward(n1, bf(b[m]))) for m in ("wq", "wk", "wv"))
        cache = Q4CacheOracle(c["n_heads"], c["n_kv_heads"], c["head_dim"], c["max_seq_len"], c["rope_base"])
        merged = cache.forward_cached(q, k, v)[0].astype(np.float32)
        x = bf(bf(T.linear_forward(bf(merged), bf(b["wo"]))) + x)
        n2 = bf(rms.forward(x, b["ffn_norm"], c["rmsnorm_eps"]))
        x = bf(bf(T.swiglu_forward(n2, bf(b["gate"]), bf(b["up"]), bf(b["down"]))[0]) + x)
    return T.linear_forward(bf(rms.forward(x, w["final_norm"], c["rmsnorm_eps"])), bf(w["embedding"] if c["tie_embeddings"] else w["lm_head"]))


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,hd", [(4, 2, 64), (4, 1, 32), (2, 2, 128)])
def test_the_models_decode_over_a_cache_in_4_bits(H, Hkv, hd):
    """A prompt, then single tokens, for three sequences.  Both sides round at the same places, but a sum's last bit decides some roundings,
    and a changed key or value may take the next code: with groups of about four standard deviations a step is 0.27 of one, a bf16
    half step moves about one code in a hundred by that, 0.03 of the cached rows' size, and the rows are averaged over positions and
    stand beside the residual.  So 4e-2 of the logits; the bf16 cache's own bar is 2e-2."""
    c = _config(n_heads=H, n_kv_heads=Hkv, head_dim=hd, moe_layers=(), n_layers=2)
    dev, w = _model(c)
    seqs = _sequences(101, [40, 40, 40], seed=4)
    want = np.stack([_decode_oracle(c, w, s) for s in seqs])
    caches = dev.new_kv_caches(sequences=3, capacity=44, precision="q4")
    got = np.empty_like(want)
    got[:, :30] = dev.forward_cached([s[:30] for s in seqs], caches).reshape(3, 30, -1)
    for t in range(30, 40):
        got[:, t] = dev.forward_cached([[s[t]] for s in seqs], caches)
    assert rel_l2(got, want) <= 4e-2
    caches.clear(1)
    again = dev.forward_cached([seqs[1][:8]], caches, first_sequence=1).reshape(8, -1)
    assert rel_l2(again, want[1, :8]) <= 4e-2
    with pytest.raises(InvalidInput, match="SequenceTooLong"):
        dev.forward_cached([list(seqs[0][:10])], caches, first_sequence=0)
    dev.close()


@pytest.mark.gpu
def test_inputs_that_come_from_another_stream():
    """Kernels that are let in while their predecessor runs: what they read comes from a second stream, eager and captured, and each call's
    input is overwritten as soon as it has been read."""
    L = Q4Linear(256, 512)
    g = torch.Generator(device="cuda").manual_seed(8)
    L.set_weight(torch.randn(512, 256, generator=g, device="cuda"))
    xs = torch.randn(20, 4, 256, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, 512, (4,), generator=g, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    want = []
    for x in xs:
        y = L(x)
        torch.cuda.synchronize()
        s = token_logprobs(y, t)
        torch.cuda.synchronize()
        want.append((y, s.logprob, token_logprobs_backward(y, t, s.lse, s.entropy, s.lse, s.entropy)))
    torch.cuda.synchronize()
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    x, y, d = torch.zeros_like(xs[0]), torch.zeros_like(want[0][0]), torch.zeros_like(want[0][2])
    pile = [(torch.zeros_like(y), torch.zeros_like(want[0][1]), torch.zeros_like(d)) for _ in xs]

    def run():
        for i in range(len(xs)):
            side.wait_stream(main)
            with torch.cuda.stream(side):
                x.copy_(xs[i])
            main.wait_stream(side)
            L(x, out=y)
            s = token_logprobs(y, t)
            token_logprobs_backward(y, t, s.lse, s.entropy, s.lse, s.entropy, out=d)
            for a, b in zip(pile[i], (y, s.logprob, d)):
                a.copy_(b)

    def check():
        torch.cuda.synchronize()
        for got, w in zip(pile, want):
            for a, b in zip(got, w):
                assert torch.equal(a, b)
                a.zero_()
        torch.cuda.synchronize()

    with torch.cuda.stream(main):
        run()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        run()
    for _ in range(3):
        graph.replay()
        check()


def _busy():
    torch.cuda._sleep(100_000_000)               # about 50 ms of the current stream


@pytest.mark.gpu
def test_weights_set_on_a_stream_of_their_own():
    """The zeros that a new layer starts with do not land on top of weights that another stream has packed."""
    g = torch.Generator(device="cuda").manual_seed(40)
    codes = torch.randint(-8, 8, (64, 128), device="cuda", generator=g).to(torch.int8)
    scales = torch.rand(64, 4, device="cuda", generator=g).bfloat16()
    weight = torch.randn(64, 128, device="cuda", generator=g)
    want = codes.float() * scales.float().repeat_interleave(32, dim=1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for set_it in (lambda l: l.set_codes(codes, scales, stream=side.cuda_stream), lambda l: l.set_weight(weight, stream=side.cuda_stream)):
        _busy()
        layer = Q4Linear(128, 64)
        set_it(layer)
        torch.cuda.synchronize()
        assert float(layer.weight().abs().max()) > 0
    _busy()
    layer = Q4Linear(128, 64)
    layer.set_codes(codes, scales, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(layer.weight(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["linear", "weight", "logprobs", "gradient", "step", "newest"])
def test_results_of_a_given_stream_are_its_own_memory(what):
    """A result that is dropped before its stream has written it is not handed out on another stream meanwhile."""
    side = torch.cuda.Stream()
    layer = Q4Linear(128, 4096)
    layer.set_weight(torch.ones(4096, 128, device="cuda"))
    x = torch.ones(64, 128, device="cuda")
    logits, lse = torch.ones(64, 4096, device="cuda"), torch.ones(64, device="cuda")
    cache = KvCache(64, 16, 16, 128, capacity=4, precision="bf16")
    qkv = [torch.ones(64, 2048, device="cuda").bfloat16() for _ in range(3)]
    cache.append(qkv[1], qkv[2])
    st = side.cuda_stream
    call = {"linear": lambda: [layer.forward(x, stream=st)], "weight": lambda: [layer.weight(stream=st)],
            "logprobs": lambda: [t for t in token_logprobs(logits, None, top=32, stream=st)],
            "gradient": lambda: [token_logprobs_backward(logits, None, lse, grad_logprob=lse, stream=st)],
            "step": lambda: [cache.forward_cached(*qkv, stream=st)], "newest": lambda: list(cache.newest(stream=st))}[what]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        _busy()
    got = call()
    shapes = [(t.shape, t.dtype) for t in got]
    del got
    mine = [torch.full(s, 7, device="cuda", dtype=d) for s, d in shapes]
    torch.cuda.synchronize()
    assert all(bool((t == 7).all()) for t in mine)
    with torch.cuda.stream(side):                              # ... and the default stream, given by its number
        again = call()
    torch.cuda.synchronize()
    st = 0
    if what != "step":
        for a, b in zip(again, call()):
            assert torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["q4", "bf16", "f32"])
def test_a_cache_is_cut_read_and_cleared_in_the_order_of_its_stream(precision):
    dt = torch.float32 if precision == "f32" else torch.bfloat16
    cache = KvCache(2, 2, 1, 64, capacity=40, precision=precision)
    k = torch.ones(20, 64, device="cuda", dtype=dt)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        _busy()
        cache.append(k, k, rows_per_sequence=10)
        cache.truncate(7, sequence=0)
        assert cache.lengths() == [7, 10]
        _busy()
        cache.append(k, k, rows_per_sequence=10)
        values = cache.keys_values(1)[1]
        assert values.shape == (20, 64) and (values == 1).all()
        _busy()
        cache.append(k[:2], k[:2])
        cache.clear(1)
    side.synchronize()
    assert cache.lengths() == [18, 0]
