"""KV cache held in 4 bits: the format bit for bit, the attention against 64-bit arithmetic on what the cache stands for."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from oracle.kv_q4 import Q4CacheOracle, quantise, to_bf16
from rustingbrain_b200 import InvalidConfig, InvalidInput, _lib
from rustingbrain_b200.kv_attention import KvCache


# ---- no device needed -----------------------------------------------------------------------------------------------
def test_the_format_rounds_to_the_nearest_of_sixteen_values():
    x = np.random.Generator(np.random.Philox(1)).standard_normal((50, 3, 64)).astype(np.float32)
    x[3, 1] = 2.5
    y, code = quantise(x)
    assert code.min() == 0 and code.max() == 15
    assert np.array_equal(y[3, 1], x[3, 1])                                # a constant group is its base
    g = x.reshape(50, 3, 2, 32)
    spread = (g.max(-1) - g.min(-1)).repeat(32, axis=-1).reshape(x.shape)
    # half a step, the base's rounding (2^-8 of it) and the step's over fifteen steps
    assert (np.abs(y - x) <= spread / 30 * 1.01 + np.abs(x).max() * 2.0 ** -8).all()
    assert np.array_equal(to_bf16(np.float32([1.00390625, -1.01171875])), np.float32([1.0, -1.015625]))      # ties to even


def _create(**kw):
    cfg = dict(sequences=2, num_heads=4, kv_heads=2, head_dim=64, capacity=16, max_seq_len=16, rope_base=10000.0, rope=1,
               precision=_lib.PRECISION_Q4, device=0)
    cfg.update(kw)
    h = C.c_void_p()
    rc = _lib.lib().kv_cache_create(C.byref(_lib.KvCacheConfigC(**cfg)), C.byref(h))
    text = _lib.lib().kv_cache_last_error(h).decode()
    _lib.lib().kv_cache_destroy(h)
    return rc, text


def test_configurations_are_checked_before_any_device_work():
    for hd in (8, 16):
        rc, text = _create(head_dim=hd)
        assert rc == _lib.UNSUPPORTED and "4-bit" in text
    for bad in (dict(num_heads=3), dict(head_dim=7), dict(sequences=0), dict(capacity=17), dict(precision=4), dict(precision=_lib.PRECISION_Q8)):
        assert _create(**bad)[0] == _lib.INVALID_CONFIG, bad
    rc, text = _create(capacity=(1 << 30) + 1, max_seq_len=(1 << 30) + 1)
    assert rc == _lib.UNSUPPORTED and "2^30" in text
    L = _lib.lib()
    assert L.kv_cache_append(None, 0, 1, None, None, 1, None) == _lib.INVALID_INPUT
    assert L.kv_cache_rollback(None, 0, 1, 1, None) == _lib.INVALID_INPUT
    assert L.kv_cache_newest(None, 0, 1, 1, None, None, None) == _lib.INVALID_INPUT
    with pytest.raises(InvalidConfig):
        KvCache(1, 2, 2, 64, 8, precision="q2")
    msg = C.create_string_buffer(128)
    cfg = _lib.MoeConfigC(d_model=64, num_experts=4, experts_per_token=2, d_ff=32, precision=_lib.PRECISION_Q4, max_tokens=16, ep_size=1)
    assert L.moe_config_validate(C.byref(cfg), msg, 128) == _lib.INVALID_CONFIG      # a cache's precision, not a layer's


# ---- on the device --------------------------------------------------------------------------------------------------
def _rows(n, H, Hkv, hd, seed, scale=1.0):
    g = np.random.Generator(np.random.Philox(seed))
    bf = lambda *s: to_bf16(g.standard_normal(s).astype(np.float32) * np.float32(scale))
    return bf(n, H * hd), bf(n, Hkv * hd), bf(n, Hkv * hd)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda().bfloat16()


def _same_cache(cache, s, o):
    k, v = cache.keys_values(s)
    np.testing.assert_array_equal(k, o.keys.reshape(len(o), -1))
    np.testing.assert_array_equal(v, o.values.reshape(len(o), -1))


def _close(got, want):
    out, tol = want
    d = np.abs(got.double().cpu().numpy() - out)
    assert (d <= tol).all(), float((d / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,hd,rows", [(8, 2, 64, 1), (4, 4, 64, 3), (2, 2, 32, 1), (3, 1, 32, 2), (8, 1, 128, 1), (16, 1, 128, 1), (20, 1, 64, 1),
                                           (32, 4, 128, 2), (4, 2, 256, 1), (12, 1, 256, 2), (16, 2, 64, 5), (6, 2, 32, 9)])
def test_steps_of_sequences_of_different_lengths(H, Hkv, hd, rows):
    """Histories that end in, at and behind the edges of a page; groups of 1 to 20 query heads; one pass and several."""
    lens = [0, 1, 62, 63, 64, 65, 130, 700]
    S, cap = len(lens), 760
    cache = KvCache(S, H, Hkv, hd, capacity=cap, precision="q4")
    oracles = [Q4CacheOracle(H, Hkv, hd, cap) for _ in lens]
    for s, n in enumerate(lens):
        if n:
            _, k, v = _rows(n, H, Hkv, hd, 100 + s)
            cache.append(_dev(k), _dev(v), rows_per_sequence=n, first_sequence=s, n_sequences=1)
            oracles[s].append(k, v)
    assert cache.lengths() == lens
    for step in range(3):
        q, k, v = _rows(S * rows, H, Hkv, hd, 200 + step)
        qd = _dev(q)
        got = cache.forward_cached(qd, _dev(k), _dev(v), rows_per_sequence=rows)
        assert np.array_equal(qd.float().cpu().numpy(), q)                       # the queries are left alone
        for s in range(S):
            sl = slice(s * rows, (s + 1) * rows)
            _close(got[sl], oracles[s].forward_cached(q[sl], k[sl], v[sl]))
        keys, values = cache.newest(rows)
        want = np.concatenate([o.keys[-rows:].reshape(rows, -1) for o in oracles])
        np.testing.assert_array_equal(keys.cpu().numpy(), want)
        np.testing.assert_array_equal(values.cpu().numpy(), np.concatenate([o.values[-rows:].reshape(rows, -1) for o in oracles]))
    assert cache.lengths() == [n + 3 * rows for n in lens]
    for s in (0, 3, 7):
        _same_cache(cache, s, oracles[s])


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,hd,n,rows", [(8, 2, 64, 2500, 1), (2, 1, 128, 5000, 1), (4, 1, 64, 9000, 3), (2, 2, 256, 2700, 1), (8, 1, 32, 3000, 40)])
def test_one_long_sequence(H, Hkv, hd, n, rows):
    """Enough pages for more slices than one cluster joins."""
    cache, o = KvCache(1, H, Hkv, hd, capacity=n + 100, precision="q4"), Q4CacheOracle(H, Hkv, hd, n + 100)
    _, k, v = _rows(n, H, Hkv, hd, 1)
    cache.append(_dev(k), _dev(v), rows_per_sequence=n)
    o.append(k, v)
    for step in range(2):
        q, k, v = _rows(rows, H, Hkv, hd, 2 + step)
        _close(cache.forward_cached(_dev(q), _dev(k), _dev(v), rows_per_sequence=rows), o.forward_cached(q, k, v))
    assert cache.lengths() == [n + 2 * rows]
    _same_cache(cache, 0, o)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,hd,rows", [(8, 2, 64, 1), (4, 1, 128, 3), (2, 2, 256, 1), (24, 2, 32, 2)])
def test_slices_of_sequences_that_differ_much(H, Hkv, hd, rows):
    """From an empty sequence to a long one: slices of one size for all, most of them not there, joined by a second launch."""
    lens = [3000, 0, 9000, 5, 63, 700, 4000]
    S, cap = len(lens), 9100
    cache, o = KvCache(S, H, Hkv, hd, cap, precision="q4"), [Q4CacheOracle(H, Hkv, hd, cap) for _ in lens]
    for s, n in enumerate(lens):
        if n:
            _, k, v = _rows(n, H, Hkv, hd, 300 + s)
            cache.append(_dev(k), _dev(v), rows_per_sequence=n, first_sequence=s, n_sequences=1)
            o[s].append(k, v)
    for step in range(2):
        q, k, v = _rows(S * rows, H, Hkv, hd, 400 + step)
        got = cache.forward_cached(_dev(q), _dev(k), _dev(v), rows_per_sequence=rows)
        for s in range(S):
            sl = slice(s * rows, (s + 1) * rows)
            _close(got[sl], o[s].forward_cached(q[sl], k[sl], v[sl]))
    assert cache.lengths() == [n + 2 * rows for n in lens]
    q, k, v = _rows(2 * rows, H, Hkv, hd, 500)                 # a part of the cache: the others stay
    got = cache.forward_cached(_dev(q), _dev(k), _dev(v), rows_per_sequence=rows, first_sequence=2, n_sequences=2)
    for j, s in enumerate((2, 3)):
        sl = slice(j * rows, (j + 1) * rows)
        _close(got[sl], o[s].forward_cached(q[sl], k[sl], v[sl]))
    assert cache.lengths() == [n + (3 if s in (2, 3) else 2) * rows for s, n in enumerate(lens)]


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,hd,n", [(8, 2, 64, 200), (4, 1, 128, 97), (2, 2, 32, 64), (4, 4, 256, 70)])
def test_a_prompt_at_once_equals_row_by_row(H, Hkv, hd, n):
    one, many, o = KvCache(1, H, Hkv, hd, 256, precision="q4"), KvCache(1, H, Hkv, hd, 256, precision="q4"), Q4CacheOracle(H, Hkv, hd, 256)
    q, k, v = _rows(n, H, Hkv, hd, 5)
    got = one.forward_cached(_dev(q), _dev(k), _dev(v), rows_per_sequence=n)
    want = o.forward_cached(q, k, v)
    _close(got, want)
    for i in range(n):
        _close(many.forward_cached(_dev(q[i:i + 1]), _dev(k[i:i + 1]), _dev(v[i:i + 1])), (want[0][i:i + 1], want[1][i:i + 1]))
    _same_cache(one, 0, o)
    _same_cache(many, 0, o)


@pytest.mark.gpu
def test_rollback_clear_truncate_and_other_sequences_stay():
    H, Hkv, hd, cap = 8, 2, 64, 200
    cache, o = KvCache(4, H, Hkv, hd, cap, precision="q4"), [Q4CacheOracle(H, Hkv, hd, cap) for _ in range(4)]
    for s, n in enumerate((70, 100, 127, 60)):
        _, k, v = _rows(n, H, Hkv, hd, s)
        cache.append(_dev(k), _dev(v), rows_per_sequence=n, first_sequence=s, n_sequences=1)
        o[s].append(k, v)
    q, k, v = _rows(2 * 3, H, Hkv, hd, 9)
    cache.forward_cached(_dev(q), _dev(k), _dev(v), rows_per_sequence=3, first_sequence=1, n_sequences=2)
    assert cache.lengths() == [70, 103, 130, 60]
    cache.rollback(2, first_sequence=1, n_sequences=2)                      # one of three drafts was accepted
    assert cache.lengths() == [70, 101, 128, 60]
    for j, s in enumerate((1, 2)):
        o[s].append(k[3 * j:3 * j + 1], v[3 * j:3 * j + 1])
    for s in range(4):
        _same_cache(cache, s, o[s])
    q, k, v = _rows(2, H, Hkv, hd, 10)
    got = cache.forward_cached(_dev(q), _dev(k), _dev(v), first_sequence=1, n_sequences=2)
    for j, s in enumerate((1, 2)):
        _close(got[j:j + 1], o[s].forward_cached(q[j:j + 1], k[j:j + 1], v[j:j + 1]))
    cache.clear(2)
    cache.truncate(65, sequence=1)
    o[1].truncate(65)
    assert cache.lengths() == [70, 65, 0, 60]
    q, k, v = _rows(2, H, Hkv, hd, 11)
    got = cache.forward_cached(_dev(q), _dev(k), _dev(v), first_sequence=1, n_sequences=2)
    o[2] = Q4CacheOracle(H, Hkv, hd, cap)
    for j, s in enumerate((1, 2)):
        _close(got[j:j + 1], o[s].forward_cached(q[j:j + 1], k[j:j + 1], v[j:j + 1]))
    for bad in (lambda: cache.rollback(2, 2, 1), lambda: cache.rollback(0), lambda: cache.newest(2, 2, 1), lambda: cache.newest(1, 3, 2),
                lambda: cache.rollback(1, -1, 1), lambda: cache.append(_dev(k), _dev(v)), lambda: cache.append(_dev(k).float(), _dev(v), 1, 1, 2),
                lambda: cache.append(_dev(k), _dev(v), rows_per_sequence=2, first_sequence=4, n_sequences=1)):
        with pytest.raises(InvalidInput):
            bad()
    long = _rows(141, H, Hkv, hd, 12)
    with pytest.raises(InvalidInput, match="SequenceTooLong"):
        cache.append(_dev(long[1]), _dev(long[2]), rows_per_sequence=141, first_sequence=3, n_sequences=1)
    assert cache.lengths() == [70, 66, 1, 60]


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 2.0 ** 127])
@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("rows", [4, 30])
def test_a_position_that_is_not_finite_reaches_only_those_who_see_it(bad, where, rows):
    H, Hkv, hd, j = 4, 2, 64, 2
    cache, o = KvCache(1, H, Hkv, hd, 256, precision="q4"), Q4CacheOracle(H, Hkv, hd, 256)
    _, k, v = _rows(61, H, Hkv, hd, 1)
    cache.append(_dev(k), _dev(v), rows_per_sequence=61)
    o.append(k, v)
    q, k, v = _rows(rows, H, Hkv, hd, 2)
    (k if where == "key" else v)[j, 7] = bad                   # the first kv head of the third new row
    got = cache.forward_cached(_dev(q), _dev(k), _dev(v), rows_per_sequence=rows)
    out, tol = o.forward_cached(q, k, v)
    first = H // Hkv * hd
    assert bool(got[j:, :first].isnan().all())
    _close(got[:j], (out[:j], tol[:j]))
    _close(got[:, first:], (out[:, first:], tol[:, first:]))
    _same_cache(cache, 0, o)
    # rolled back, the slots hold finite numbers again
    cache.rollback(rows)
    o.truncate(61)
    q, k, v = _rows(2, H, Hkv, hd, 3)
    _close(cache.forward_cached(_dev(q), _dev(k), _dev(v), rows_per_sequence=2), o.forward_cached(q, k, v))


@pytest.mark.gpu
def test_rolled_back_positions_that_are_not_finite_do_not_come_back():
    H, Hkv, hd = 4, 1, 128
    cache, o = KvCache(1, H, Hkv, hd, 256, precision="q4"), Q4CacheOracle(H, Hkv, hd, 256)
    _, k, v = _rows(60, H, Hkv, hd, 4)
    k[20:], v[25:] = np.nan, np.inf
    cache.append(_dev(k), _dev(v), rows_per_sequence=60)
    cache.truncate(10)
    o.append(k[:10], v[:10])
    q, k, v = _rows(1, H, Hkv, hd, 5)
    _close(cache.forward_cached(_dev(q), _dev(k), _dev(v)), o.forward_cached(q, k, v))
    q[0, :hd] = np.nan                                         # one head's query
    got = cache.forward_cached(_dev(q), _dev(k), _dev(v))
    assert bool(got[0, :hd].isnan().all()) and bool(got[0, hd:].isfinite().all())


@pytest.mark.gpu
def test_large_and_small_numbers_and_no_rotation():
    H, Hkv, hd = 4, 2, 64
    for scale in (1e-30, 1e-3, 300.0, 1e6):
        cache, o = KvCache(1, H, Hkv, hd, 128, precision="q4", rope=False), Q4CacheOracle(H, Hkv, hd, 128, rope=False)
        _, _, v = _rows(80, H, Hkv, hd, 6, scale)
        _, k, _ = _rows(80, H, Hkv, hd, 7)
        cache.append(_dev(k), _dev(v), rows_per_sequence=80)
        o.append(k, v)
        q, k, _ = _rows(3, H, Hkv, hd, 8)
        _, _, v = _rows(3, H, Hkv, hd, 9, scale)
        _close(cache.forward_cached(_dev(q), _dev(k), _dev(v), rows_per_sequence=3), o.forward_cached(q, k, v))
        _same_cache(cache, 0, o)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    H, Hkv, hd, cap, S = 8, 8, 128, 131072, 30                 # 168 MB a sequence
    cache, o = KvCache(S, H, Hkv, hd, cap, precision="q4"), Q4CacheOracle(H, Hkv, hd, 300)
    _, k, v = _rows(200, H, Hkv, hd, 13)
    cache.append(_dev(k), _dev(v), rows_per_sequence=200, first_sequence=S - 1, n_sequences=1)
    o.append(k, v)
    q, k, v = _rows(1, H, Hkv, hd, 14)
    _close(cache.forward_cached(_dev(q), _dev(k), _dev(v), first_sequence=S - 1, n_sequences=1), o.forward_cached(q, k, v))
    _same_cache(cache, S - 1, o)
    assert cache.lengths() == [0] * (S - 1) + [201]


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,hd,rows,n", [(4, 2, 64, 1, 2), (4, 1, 64, 6, 2), (2, 1, 128, 1, 2600)])
def test_captured_steps_and_the_end_of_the_cache(H, Hkv, hd, rows, n):
    """A replayed step advances the device lengths only; one that finds no room stores nothing, returns zeros and marks the sequence."""
    S, cap = 2, n + 3 * rows + 3
    cache = KvCache(S, H, Hkv, hd, cap, precision="q4")
    o = [Q4CacheOracle(H, Hkv, hd, cap) for _ in range(S)]
    for s, m in enumerate((n + 3, n)):
        _, k, v = _rows(m, H, Hkv, hd, 20 + s)
        cache.append(_dev(k), _dev(v), rows_per_sequence=m, first_sequence=s, n_sequences=1)
        o[s].append(k, v)
    a, b = _rows(S * rows, H, Hkv, hd, 22), _rows(S * rows, H, Hkv, hd, 23)
    q, k, v = (_dev(x) for x in a)
    out = torch.empty_like(q)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        cache.forward_cached(q, k, v, out=out, rows_per_sequence=rows)
        cache.rollback(rows)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        cache.forward_cached(q, k, v, out=out, rows_per_sequence=rows)
    for x in (a, b, a):
        for t, y in zip((q, k, v), x):
            t.copy_(_dev(y))
        graph.replay()
        torch.cuda.synchronize()
        for s in range(S):
            sl = slice(s * rows, (s + 1) * rows)
            _close(out[sl], o[s].forward_cached(x[0][sl], x[1][sl], x[2][sl]))
    assert cache.lengths() == [cap, cap - 3]
    graph.replay()                                             # the first is full, the second too unless three rows fit
    torch.cuda.synchronize()
    assert float(out[:rows].abs().max()) == 0
    with pytest.raises(InvalidInput, match="SequenceTooLong"):
        cache.lengths()
    assert cache.lengths() == [cap, cap - 3 + (rows if rows <= 3 else 0)]
    _same_cache(cache, 0, o[0])
    cache.truncate(n, sequence=0)
    cache.truncate(n, sequence=1)
    for s in range(S):
        o[s].truncate(n)
    graph.replay()
    torch.cuda.synchronize()
    for s in range(S):
        sl = slice(s * rows, (s + 1) * rows)
        _close(out[sl], o[s].forward_cached(a[0][sl], a[1][sl], a[2][sl]))
    assert cache.lengths() == [n + rows] * S


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run():
    H, Hkv, hd, S = 16, 4, 64, 8
    cache = KvCache(S, H, Hkv, hd, 2048, precision="q4")
    _, k, v = _rows(S * 1500, H, Hkv, hd, 30)
    cache.append(_dev(k), _dev(v), rows_per_sequence=1500)
    q, k, v = (_dev(x) for x in _rows(S, H, Hkv, hd, 31))
    first = cache.forward_cached(q, k, v)
    for _ in range(5):
        cache.rollback(1)
        assert torch.equal(cache.forward_cached(q, k, v), first)


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["f32", "bf16"])
def test_append_newest_and_rollback_on_the_other_caches(precision):
    from oracle.attention import KvCacheOracle
    H, Hkv, hd = 4, 2, 64
    dt = torch.float32 if precision == "f32" else torch.bfloat16
    cache, o = KvCache(2, H, Hkv, hd, 64, precision=precision), KvCacheOracle(H, Hkv, hd, 64)
    q, k, v = _rows(30, H, Hkv, hd, 40)
    cache.append(torch.from_numpy(k[:29]).cuda().to(dt), torch.from_numpy(v[:29]).cuda().to(dt), rows_per_sequence=29, first_sequence=1, n_sequences=1)
    o.forward_cached(q[:29], k[:29], v[:29])
    assert cache.lengths() == [0, 29]
    keys, values = cache.newest(5, 1, 1)
    assert np.abs(keys.cpu().numpy() - np.asarray(o.keys)[24:29]).max() <= (1e-5 if precision == "f32" else 2.0 ** -8 * 5)
    assert np.array_equal(values.cpu().numpy(), np.asarray(o.values)[24:29])
    d = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda().to(dt)
    got = cache.forward_cached(d(q[29:]), d(k[29:]), d(v[29:]), first_sequence=1, n_sequences=1)
    want = o.forward_cached(q[29:], k[29:], v[29:])
    assert np.linalg.norm(got.float().cpu().numpy() - want) / np.linalg.norm(want) <= (1e-5 if precision == "f32" else 2e-2)
    cache.rollback(1, 1, 1)
    again = cache.forward_cached(d(q[29:]), d(k[29:]), d(v[29:]), first_sequence=1, n_sequences=1)
    assert torch.equal(got, again) and cache.lengths() == [0, 30]


@pytest.mark.gpu
def test_ranges_that_wrap_around():
    """A first sequence or a number of rows whose sum with what is there passes 31 bits is refused like any other."""
    for precision, dt in (("q4", torch.bfloat16), ("f32", torch.float32)):
        cache = KvCache(2, 1, 1, 32, capacity=8, precision=precision)
        k = torch.ones(2, 32, device="cuda", dtype=dt)
        cache.append(k, k)
        p, L, st = C.c_void_p(k.data_ptr()), _lib.lib(), 0
        big = 2 ** 31 - 1
        for first, n, rows in ((big, 1, 1), (1, big, 1), (2, 1, 1), (0, 1, big), (0, 1, 8), (1, 2, 1)):
            assert L.kv_cache_append(cache._h, first, n, p, p, rows, st) == _lib.INVALID_INPUT, (first, n, rows)
            assert L.kv_attention_forward_cached(cache._h, first, n, p, p, p, rows, p, st) == _lib.INVALID_INPUT
            assert L.kv_cache_rollback(cache._h, first, n, rows, st) == _lib.INVALID_INPUT
            assert L.kv_cache_newest(cache._h, first, n, rows, p, p, st) == _lib.INVALID_INPUT
        assert cache.lengths() == [1, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,hd", [(4, 1, 64), (10, 1, 32), (16, 1, 128), (4, 1, 256)])
def test_queries_of_any_size(H, Hkv, hd):
    """Queries of 2^110 against keys of 2^-112, and the other way round; small and large queries in one pass keep their own scale."""
    for up, down in ((110, -112), (-110, 30), (0, 0)):
        cache, o = KvCache(1, H, Hkv, hd, capacity=100, precision="q4"), Q4CacheOracle(H, Hkv, hd, 100)
        _, k, v = _rows(90, H, Hkv, hd, 31)
        k = k * np.float32(2.0 ** down)
        cache.append(_dev(k), _dev(v), rows_per_sequence=90)
        o.append(k, v)
        q, k, v = _rows(1, H, Hkv, hd, 32)
        q = q.reshape(H, hd) * np.float32(2.0) ** (up - 3 * np.arange(H, dtype=np.float32))[:, None] if up <= 0 else q * np.float32(2.0 ** up)
        q, k = q.reshape(1, -1), k * np.float32(2.0 ** down)
        _close(cache.forward_cached(_dev(q), _dev(k), _dev(v)), o.forward_cached(q, k, v))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,rows", [([70, 70], 1), ([3, 900], 1), ([600, 20], 5), ([0, 64], 40)])
def test_the_result_may_take_the_queries_place(lens, rows):
    """Clusters, slices and several passes; rows behind the last sequence stay as they were."""
    H, Hkv, hd, S = 8, 2, 64, len(lens)
    caches = [KvCache(S, H, Hkv, hd, capacity=1000, precision="q4") for _ in range(2)]
    for c in caches:
        for s, n in enumerate(lens):
            if n:
                _, k, v = _rows(n, H, Hkv, hd, 50 + s)
                c.append(_dev(k), _dev(v), rows_per_sequence=n, first_sequence=s, n_sequences=1)
    q, k, v = (_dev(a) for a in _rows(S * rows, H, Hkv, hd, 60))
    want = caches[0].forward_cached(q, k, v, rows_per_sequence=rows)
    buf = torch.cat([q, torch.full((3, H * hd), 7.0, device="cuda").bfloat16()])
    got = caches[1].forward_cached(buf[:S * rows], k, v, rows_per_sequence=rows, out=buf[:S * rows])
    assert torch.equal(got, want) and bool((buf[S * rows:] == 7).all())
    with pytest.raises(InvalidInput):
        caches[1].forward_cached(q, k, v, rows_per_sequence=rows, out=torch.empty(S * rows, Hkv * hd, device="cuda", dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("precision,what", [("q4", "step"), ("q4", "append"), ("bf16", "append"), ("f32", "append")])
@pytest.mark.parametrize("drafts", [1, 3])
def test_rollback_behind_a_step_that_was_skipped(precision, what, drafts):
    """Captured: a step of four rows that does not fit, `drafts` steps of one row that do, and their rollback.  What was skipped left
    nothing behind, what was taken goes again; a rollback over both takes back only what is there."""
    H, Hkv, hd, cap, n = 4, 2, 64, 12, 9
    cache = KvCache(2, H, Hkv, hd, cap, precision=precision)
    dt = torch.float32 if precision == "f32" else torch.bfloat16
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda().to(dt)
    _, k0, v0 = _rows(n, H, Hkv, hd, 70)
    cache.append(dev(k0[:6]), dev(v0[:6]), rows_per_sequence=6, first_sequence=0, n_sequences=1)
    cache.append(dev(k0[:2]), dev(v0[:2]), rows_per_sequence=2, first_sequence=1, n_sequences=1)
    side, graphs, data = torch.cuda.Stream(), {}, {}
    torch.cuda.synchronize()
    for rows in (4, 1):                                        # captured while the host's copy of the lengths says that they fit
        data[rows] = tuple(dev(a) for a in _rows(rows, H, Hkv, hd, 71 + rows))
        graphs[rows] = torch.cuda.CUDAGraph()
        q, k, v = data[rows]
        with torch.cuda.graph(graphs[rows], stream=side):
            if what == "step":
                data[rows] += (cache.forward_cached(q, k, v, rows_per_sequence=rows, first_sequence=0, n_sequences=1),)
            else:
                cache.append(k, v, rows_per_sequence=rows, first_sequence=0, n_sequences=1)
    assert cache.lengths() == [6, 2]
    cache.append(dev(k0[6:]), dev(v0[6:]), rows_per_sequence=n - 6, first_sequence=0, n_sequences=1)
    before = None if precision != "q4" else Q4CacheOracle(H, Hkv, hd, cap)
    if before is not None:
        before.append(k0, v0)
    torch.cuda.synchronize()
    graphs[4].replay()                                         # 9 + 4 > 12: skipped
    for _ in range(drafts):
        graphs[1].replay()                                     # up to 12
    torch.cuda.synchronize()
    if what == "step":
        assert float(data[4][3].abs().max()) == 0 and float(data[1][3].abs().max()) > 0
    cache.rollback(drafts, first_sequence=0, n_sequences=1)
    with pytest.raises(InvalidInput, match="SequenceTooLong"):
        cache.lengths()
    assert cache.lengths() == [n, 2]
    if before is not None:
        _same_cache(cache, 0, before)
    for _ in range(5):                                         # three fit, two do not
        graphs[1].replay()
    torch.cuda.synchronize()
    cache.rollback(1, first_sequence=0, n_sequences=1)         # of the two
    cache.rollback(2, first_sequence=0, n_sequences=1)         # the other, and the newest that is there
    with pytest.raises(InvalidInput, match="SequenceTooLong"):
        cache.lengths()
    assert cache.lengths() == [cap - 1, 2]
    cache.rollback(1)                                          # nothing is owed any more, and the other sequence is an ordinary one
    assert cache.lengths() == [cap - 2, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["bf16", "f32"])
def test_rollback_of_steps_that_a_marked_cache_skips(precision):
    """The caches of 16 and 32 bits take no step while a mark is unread: those rows are taken back without a trace too."""
    H, Hkv, hd, cap = 4, 2, 64, 8
    cache = KvCache(1, H, Hkv, hd, cap, precision=precision)
    dt = torch.float32 if precision == "f32" else torch.bfloat16
    q, k, v = (torch.from_numpy(a).cuda().to(dt) for a in _rows(3, H, Hkv, hd, 80))
    cache.forward_cached(q, k, v, rows_per_sequence=3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.forward_cached(q.clone(), k, v, rows_per_sequence=3)
    assert cache.lengths() == [3]
    for _ in range(3):                                         # 6, then twice no room
        graph.replay()
    torch.cuda.synchronize()
    cache.rollback(1)
    cache.rollback(2)                                          # the second of the skipped steps
    with pytest.raises(InvalidInput, match="SequenceTooLong"):
        cache.lengths()
    assert cache.lengths() == [6]
    graph.replay()
    torch.cuda.synchronize()
    cache.rollback(4)                                          # a skipped step and one row
    with pytest.raises(InvalidInput, match="SequenceTooLong"):
        cache.lengths()
    assert cache.lengths() == [5]


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["q4", "bf16", "f32"])
def test_out_has_any_shape(precision):
    H, Hkv, hd, S, rows = 4, 2, 64, 3, 2
    dt = torch.float32 if precision == "f32" else torch.bfloat16
    caches = [KvCache(S, H, Hkv, hd, 16, precision=precision) for _ in range(2)]
    q, k, v = (torch.from_numpy(a).cuda().to(dt) for a in _rows(S * rows, H, Hkv, hd, 90))
    want = caches[0].forward_cached(q.clone(), k, v, rows_per_sequence=rows)
    out = torch.empty(S, rows, H, hd, device="cuda", dtype=dt)
    got = caches[1].forward_cached(q.clone(), k, v, rows_per_sequence=rows, out=out)
    assert got is out and torch.equal(out.view(S * rows, H * hd), want)
    for bad in (torch.empty(S * rows, H * hd + 1, device="cuda", dtype=dt), torch.empty(S * rows, H * hd, dtype=dt), torch.empty(S, H, rows, hd, device="cuda", dtype=dt).transpose(1, 2),
                torch.empty(S * rows, H * hd, device="cuda", dtype=torch.float64)):
        with pytest.raises(InvalidInput):
            caches[0].forward_cached(q, k, v, rows_per_sequence=rows, out=bad)
    assert caches[0].lengths() == [rows] * S


@pytest.mark.gpu
@pytest.mark.parametrize("precision,hd,off,ok", [("bf16", 64, 1, False), ("bf16", 64, 2, True), ("bf16", 32, 2, False), ("bf16", 32, 8, True), ("f32", 64, 1, False),
                                                 ("f32", 64, 4, True), ("q4", 64, 1, True), ("q4", 64, 3, True)])
def test_queries_off_their_boundary(precision, hd, off, ok):
    """The kernels of the older caches load several channels of a query at once; where those would straddle a boundary the call is refused."""
    H, Hkv = 4, 2
    dt = torch.float32 if precision == "f32" else torch.bfloat16
    cache, other = (KvCache(2, H, Hkv, hd, 8, precision=precision) for _ in range(2))
    q, k, v = (torch.from_numpy(a).cuda().to(dt) for a in _rows(2, H, Hkv, hd, 91))
    flat = torch.zeros(q.numel() + 16, device="cuda", dtype=dt)
    moved = flat[off:off + q.numel()].view(q.shape)
    moved.copy_(q)
    if ok:
        odd = torch.zeros(k.numel() + 1, device="cuda", dtype=dt)[1:].view(k.shape)     # keys and values are taken one by one
        odd.copy_(k)
        assert torch.equal(cache.forward_cached(moved, odd, v), other.forward_cached(q, k, v))
    else:
        with pytest.raises(InvalidInput, match="boundary"):
            cache.forward_cached(moved, k, v)
        assert cache.lengths() == [0, 0]


@pytest.mark.gpu
def test_a_result_on_top_of_what_a_4_bit_step_reads_is_refused():
    H, Hkv, hd, S = 4, 2, 64, 2
    cache, other = (KvCache(S, H, Hkv, hd, 8, precision="q4") for _ in range(2))
    q, k, v = (_dev(a) for a in _rows(S, H, Hkv, hd, 95))
    n, w = q.numel(), k.numel()
    flat = torch.zeros(2 * n + 2 * w, device="cuda").bfloat16()
    at = {"q": 0, "k": n, "v": n + w, "free": n + 2 * w}
    for name, t in (("q", q), ("k", k), ("v", v)):
        flat[at[name]:at[name] + t.numel()] = t.view(-1)
    view = lambda start, t: flat[start:start + t.numel()].view(t.shape)
    args = view(0, q), view(n, k), view(n + w, v)
    for start in (8, n // 2, n, n + w - 8, n + w, n + 2 * w - 1):
        with pytest.raises(InvalidInput, match="overlaps"):
            cache.forward_cached(*args, out=view(start, q))
    assert cache.lengths() == [0] * S
    want = other.forward_cached(q, k, v)
    assert torch.equal(cache.forward_cached(*args, out=view(n + 2 * w, q)), want)      # right behind them
    cache.rollback(1)
    assert torch.equal(cache.forward_cached(*args, out=args[0]), want)


@pytest.mark.gpu
def test_rollback_of_more_rows_than_queries_would_be_allowed():
    """256 sequences of 140000 positions take back 135000 each: with 64 query heads that is past 31 bits, but no query is asked."""
    S, n = 256, 140000
    cache = KvCache(S, 64, 1, 32, capacity=n, precision="q4")
    k = torch.ones(128 * 70000, 32, device="cuda").bfloat16()
    for half in (0, 0, 1, 1):
        cache.append(k, k, rows_per_sequence=70000, first_sequence=128 * half, n_sequences=128)
    cache.rollback(135000)
    assert cache.lengths() == [5000] * S
