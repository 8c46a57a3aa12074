"""The operators of a decode step in four bits, and of the log probabilities it answers with: what is measured.

`linear`     y = x W^T for a matrix of 4-bit codes with one bf16 scale per group of input channels
             (`rustingbrain_b200.q4_linear.Q4Linear`).
`attention`  one step of a KV cache held in 4 bits: rotate, quantise and append the new keys and values, then
             softmax(q K^T / sqrt(head_dim)) V over the cache (`rustingbrain_b200.kv_attention.KvCache`, precision "q4").
`logprobs`   log probabilities of given tokens, the entropy of each row and its most likely tokens, and the gradient
             of the first two (`rustingbrain_b200.logprobs`).

With `own` false, `run` computes them in elementary torch operations in 32 bits; with `own` true it calls the library.
"""
import math

import torch

own = False

DEV = "cuda"
KV_GROUP = 32          # channels of a key or value head that share a scale and a minimum
ROPE_BASE = 10000.0
LARGEST = 16 * 16384 * 8 * 128      # cached channels of the largest attention case
LARGEST_W = 24576 * 4096            # weights of the largest linear case
LARGEST_L = 8192 * 32000            # logits of the largest log-probability case


def listed():
    return [
        # one token through the up projection of one expert of the int8 decode workload: latency
        {"name": "linear 1x1024-2816 bf16", "op": "linear", "rows": 1, "k": 1024, "n": 2816, "group": 32, "dtype": "bf16"},
        # the 64 concurrent sequences of the decode workload through gate and up together
        {"name": "linear 64x1024-5632 bf16", "op": "linear", "rows": 64, "k": 1024, "n": 5632, "group": 128, "dtype": "bf16"},
        # a small batch through a wide gate and up product of the 4096-channel layer
        {"name": "linear 8x4096-24576 bf16", "op": "linear", "rows": 8, "k": 4096, "n": 24576, "group": 64, "dtype": "bf16"},
        # an output head over an odd vocabulary, f32 activations, an odd batch
        {"name": "linear 3x2048-32003 f32", "op": "linear", "rows": 3, "k": 2048, "n": 32003, "group": 32, "dtype": "f32"},
        # a single conversation of the 55M model: latency
        {"name": "attention 1x700 8/2x64", "op": "attention", "seqs": 1, "heads": 8, "kv_heads": 2, "hd": 64, "lo": 700, "hi": 700, "rows": 1},
        # the decode workload's attention: 64 sequences of 4096 positions
        {"name": "attention 64x4096 16/4x64", "op": "attention", "seqs": 64, "heads": 16, "kv_heads": 4, "hd": 64, "lo": 4096, "hi": 4096, "rows": 1},
        # a ragged batch, from an empty cache to a long one, three draft tokens a sequence
        {"name": "attention 16x0..32767 32/8x128", "op": "attention", "seqs": 16, "heads": 32, "kv_heads": 8, "hd": 128, "lo": 0, "hi": 32767, "rows": 3},
        # a chunk of two prompts behind what is cached already
        {"name": "attention chunk 2x256 on 1500", "op": "attention", "seqs": 2, "heads": 8, "kv_heads": 2, "hd": 64, "lo": 1500, "hi": 1601, "rows": 256},
        # the answer of one decode step, with 20 alternatives: latency
        {"name": "logprobs 1x32000 bf16 top 20", "op": "logprobs", "back": False, "rows": 1, "vocab": 32000, "top": 20, "dtype": "bf16", "mask": False},
        # 64 decoding sequences, a large odd vocabulary, part of it forbidden
        {"name": "logprobs 64x131071 f32 top 5", "op": "logprobs", "back": False, "rows": 64, "vocab": 131071, "top": 5, "dtype": "f32", "mask": True},
        # scoring the 8 x 1024 tokens of a training batch
        {"name": "logprobs 8192x32000 bf16", "op": "logprobs", "back": False, "rows": 8192, "vocab": 32000, "top": 0, "dtype": "bf16", "mask": False},
        # the gradient of a policy loss with an entropy bonus over such a batch
        {"name": "logprobs back 4096x32000 bf16", "op": "logprobs", "back": True, "rows": 4096, "vocab": 32000, "top": 0, "dtype": "bf16", "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "attention", "logprobs"])
    if op == "linear":
        group = rng.choice([32, 64, 128])
        k = max(1, _log(rng, 256, 8192) // group) * group
        n = min(_log(rng, 64, 32768), LARGEST_W // k)
        return {"op": op, "rows": _log(rng, 1, 64), "k": k, "n": n, "group": group, "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if op == "attention":
        hd, kv = rng.choice([32, 64, 64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 8])
        if rng.random() < 0.25:      # a chunk of a prompt
            seqs, rows = rng.randint(1, 3), _log(rng, 16, 300)
            hi = _log(rng, 64, 4000)
        else:                        # a decode step, some with drafts
            seqs, rows = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 5])
            hi = min(_log(rng, 100, 32000), LARGEST // (seqs * kv * hd))
        return {"op": op, "seqs": seqs, "heads": heads, "kv_heads": kv, "hd": hd, "lo": rng.randint(0, hi), "hi": hi, "rows": rows}
    vocab = _log(rng, 1000, 131072)
    back = rng.random() < 0.4
    return {"op": op, "back": back, "rows": min(_log(rng, 1, 8192), LARGEST_L // vocab), "vocab": vocab, "top": 0 if back else rng.randint(0, 20),
            "dtype": rng.choice(["bf16", "f32"]), "mask": rng.random() < 0.5}


def _lengths(case):
    """Cached positions of each sequence: spread evenly from lo to hi, the long ones not all at one end."""
    s, lo, hi = case["seqs"], case["lo"], case["hi"]
    even = [lo + (hi - lo) * i // max(1, s - 1) for i in range(s)] if s > 1 else [hi]
    return even[::2] + even[1::2][::-1]


def work(case):
    if case["op"] == "linear":
        r, k, n = case["rows"], case["k"], case["n"]
        act = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * k / 2 + n * (k // case["group"]) * 2 + r * (k + n) * act, "flops": 2 * r * n * k}
    if case["op"] == "attention":
        H, Hkv, hd, r = case["heads"], case["kv_heads"], case["hd"], case["rows"]
        row = Hkv * hd * 2 * (0.5 + 4 / KV_GROUP)     # one position's key and value: half a byte a channel, 4 bytes a group
        cached = sum(_lengths(case)) * row
        new = case["seqs"] * r * (row + Hkv * hd * (2 * 2 + 2 * 4) + 2 * H * hd * 2)
        seen = sum(n * r + r * (r + 1) // 2 for n in _lengths(case))
        return {"bytes": cached + new, "flops": 4 * H * hd * seen}
    r, v = case["rows"], case["vocab"]
    size = r * v * (2 if case["dtype"] == "bf16" else 4)
    return {"bytes": size * (2 if case["back"] else 1) + r * (20 + 8 * case["top"]), "flops": 6 * r * v}


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _linear_inputs(case, seed):
    g, r, k, n = _gen(seed), case["rows"], case["k"], case["n"]
    x = torch.randn(r, k, device=DEV, generator=g).to(_dtype(case))
    codes = (torch.randn(n, k, device=DEV, generator=g) * 2.7).round().clamp(-8, 7).to(torch.int8)
    scales = ((0.5 + torch.rand(n, k // case["group"], device=DEV, generator=g)) * 0.008).bfloat16()
    return x, codes, scales


def _attention_inputs(case, seed):
    """New q, k, v rows, and the keys (before rotation) and values that are cached already."""
    g, r = _gen(seed), case["rows"] * case["seqs"]
    H, W = case["heads"] * case["hd"], case["kv_heads"] * case["hd"]
    draw_rows = lambda *shape: torch.randn(*shape, device=DEV, generator=g).bfloat16()
    longest = max(_lengths(case))
    tone = 0.5 + torch.rand(W, device=DEV, generator=g)       # key channels differ in size
    q, k, v = draw_rows(r, H), draw_rows(r, W) * tone.bfloat16(), draw_rows(r, W)
    old_k = draw_rows(case["seqs"], longest, W) * tone.bfloat16()
    old_v = draw_rows(case["seqs"], longest, W)
    return q, k, v, old_k, old_v


def _logprob_inputs(case, seed):
    g, r, v = _gen(seed), case["rows"], case["vocab"]
    x = torch.randn(r, v, device=DEV, generator=g).mul_(2.5)
    peak = torch.randint(0, v, (r,), device=DEV, generator=g)
    rows = torch.arange(r, device=DEV)
    x[rows, peak] += 12 * torch.rand(r, device=DEV, generator=g)
    t = torch.where(torch.rand(r, device=DEV, generator=g) < 0.5, peak, torch.randint(0, v, (r,), device=DEV, generator=g))
    if case["mask"]:      # a stretch of the vocabulary is forbidden, and every 16th row has no token
        x[:, v // 3: v // 2] = float("-inf")
        t = torch.where((t >= v // 3) & (t < v // 2), torch.zeros_like(t), t)
        t[15::16] = -1
    x, t = x.to(_dtype(case)), t.to(torch.int32)
    out = {"x": x, "t": t}
    if case["back"]:
        out["g_lp"] = torch.randn(r, device=DEV, generator=g) / r
        out["g_h"] = 0.05 * torch.randn(r, device=DEV, generator=g) / r
        lse, h = torch.empty(r, device=DEV), torch.empty(r, device=DEV)
        for a in range(0, r, 512):      # what the forward pass of the same step has left behind
            y = x[a:a + 512].double()
            z = torch.logsumexp(y, 1, keepdim=True)
            p = (y - z).exp()
            lse[a:a + 512] = z[:, 0].float()
            h[a:a + 512] = -torch.where(p > 0, p * (y - z), torch.zeros_like(p)).sum(1).float()
        out["lse"], out["h"] = lse, h
    return out


def prepare(case, seed):
    st = {"case": case}
    if case["op"] == "linear":
        st["x"], codes, scales = _linear_inputs(case, seed)
        if own:
            from rustingbrain_b200.q4_linear import Q4Linear
            st["layer"] = Q4Linear(case["k"], case["n"], group_size=case["group"])
            st["layer"].set_codes(codes, scales)
        else:
            st["codes"], st["scales"] = codes, scales
    elif case["op"] == "attention":
        st["q"], st["k"], st["v"], old_k, old_v = _attention_inputs(case, seed)
        lens, r = _lengths(case), case["rows"]
        if own:
            from rustingbrain_b200.kv_attention import KvCache
            st["cache"] = KvCache(case["seqs"], case["heads"], case["kv_heads"], case["hd"], capacity=max(lens) + r, rope_base=ROPE_BASE, precision="q4")
            for i, n in enumerate(lens):
                if n:
                    st["cache"].append(old_k[i, :n], old_v[i, :n], rows_per_sequence=n, first_sequence=i, n_sequences=1)
        else:
            S, L, Hkv, hd = case["seqs"], max(lens) + r, case["kv_heads"], case["hd"]
            st["len"] = torch.tensor(lens, device=DEV)
            st["cos"], st["sin"] = _tables(L, hd)
            st["kq"], st["vq"] = _empty_cache(S, L, Hkv, hd), _empty_cache(S, L, Hkv, hd)
            n = max(lens)
            if n:
                keys = _rotate(old_k.view(S, n, Hkv, hd).float(), st["cos"][:n, None], st["sin"][:n, None])
                for where, new in ((st["kq"], _quantise(keys)), (st["vq"], _quantise(old_v.view(S, n, Hkv, hd).float()))):
                    for a, b in zip(where, new):
                        a[:, :n] = b
    else:
        st.update(_logprob_inputs(case, seed))
    torch.cuda.synchronize()
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------------
def _plain_linear(st):
    w = st["codes"].float().view(st["codes"].shape[0], -1, st["case"]["group"]) * st["scales"].float()[:, :, None]
    return (st["x"].float() @ w.view(st["codes"].shape).t()).to(st["x"].dtype)


def _tables(length, hd):
    """cos and sin of position x base^(-2 c / head_dim), the angles in 64 bits."""
    freq = ROPE_BASE ** (-2.0 * torch.arange(hd // 2, device=DEV, dtype=torch.float64) / hd)
    angle = torch.arange(length, device=DEV, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _rotate(x, cos, sin):
    lo, hi = x.chunk(2, dim=-1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], dim=-1)


def _empty_cache(s, length, heads, hd):
    flat = lambda: torch.zeros(s, length, heads, hd // KV_GROUP, 1, device=DEV)
    return torch.zeros(s, length, heads, hd // KV_GROUP, KV_GROUP, device=DEV, dtype=torch.uint8), flat(), flat()


def _quantise(x):
    """Codes 0 .. 15, scale and minimum of each group of 32 channels; scale and minimum are bf16 numbers."""
    x = x.unflatten(-1, (-1, KV_GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / torch.full_like(low, 15)).bfloat16().float()
    low = low.bfloat16().float()
    code = torch.where(scale > 0, (x - low) / scale, torch.zeros_like(x)).round().clamp(0, 15)
    return code.to(torch.uint8), scale, low


def _values(cache):
    code, scale, low = cache
    return (code.float() * scale + low).flatten(-2)


def _plain_attention(st):
    c = st["case"]
    S, R, H, Hkv, hd = c["seqs"], c["rows"], c["heads"], c["kv_heads"], c["hd"]
    pos = st["len"][:, None] + torch.arange(R, device=DEV)                   # [S, R]
    cos, sin = st["cos"][pos][:, :, None], st["sin"][pos][:, :, None]
    q = _rotate(st["q"].float().view(S, R, H, hd), cos, sin).view(S, R, Hkv, H // Hkv, hd)
    k = _quantise(_rotate(st["k"].float().view(S, R, Hkv, hd), cos, sin))
    v = _quantise(st["v"].float().view(S, R, Hkv, hd))
    seq = torch.arange(S, device=DEV)[:, None].expand(S, R)
    for where, new in ((st["kq"], k), (st["vq"], v)):
        for a, b in zip(where, new):
            a[seq, pos] = b
    keys, values = _values(st["kq"]), _values(st["vq"])                      # [S, L, Hkv, hd]
    score = torch.einsum("srkgd,slkd->skgrl", q, keys) / math.sqrt(hd)
    seen = torch.arange(keys.shape[1], device=DEV) <= pos[:, :, None]        # [S, R, L]
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = torch.einsum("skgrl,slkd->srkgd", p, values).reshape(S * R, H * hd).bfloat16()
    return out, _values(k).reshape(S * R, Hkv * hd), _values(v).reshape(S * R, Hkv * hd)


def _plain_logprobs(st):
    x, t, n = st["x"].float(), st["t"].long(), st["case"]["top"]
    top = x.amax(1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    lse = (top + total.log())[:, 0]
    entropy = total.log()[:, 0] - torch.where(e > 0, e * (x - top), torch.zeros_like(e)).sum(1) / total[:, 0]
    lp = torch.where(t >= 0, x.gather(1, t.clamp(min=0)[:, None])[:, 0] - lse, torch.zeros_like(lse))
    out = {"logprob": lp, "entropy": entropy, "lse": lse}
    if n:
        # one whole number a logit, larger for a larger logit, and for the lower index of two equal ones
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits)
        key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=DEV))
        ids = (1 << 20) - 1 - (key.topk(n, dim=1, sorted=True).values & ((1 << 20) - 1))
        out["top_ids"], out["top_logprobs"] = ids.to(torch.int32), x.gather(1, ids) - lse[:, None]
    return out


def _plain_logprobs_back(st):
    x, t = st["x"].float(), st["t"].long()
    logp = x - st["lse"][:, None]
    p = logp.exp()
    g = torch.where(t >= 0, st["g_lp"], torch.zeros_like(st["g_lp"]))
    grad = -p * g[:, None] - torch.where(p > 0, p * (logp + st["h"][:, None]), torch.zeros_like(p)) * st["g_h"][:, None]
    grad.scatter_add_(1, t.clamp(min=0)[:, None], g[:, None])
    return grad.to(st["x"].dtype)


def run(state):
    op = state["case"]["op"]
    if not own:
        if op == "linear":
            return _plain_linear(state)
        if op == "attention":
            return _plain_attention(state)
        return _plain_logprobs_back(state) if state["case"]["back"] else _plain_logprobs(state)
    if op == "linear":
        return state["layer"].forward(state["x"])
    if op == "attention":
        cache, r = state["cache"], state["case"]["rows"]
        merged = cache.forward_cached(state["q"], state["k"], state["v"], rows_per_sequence=r)
        keys, values = cache.newest(r)       # what the new rows stand for in the cache
        cache.rollback(r)                    # as after draft tokens that were not accepted
        return merged, keys, values
    from rustingbrain_b200.logprobs import token_logprobs, token_logprobs_backward
    if state["case"]["back"]:
        return token_logprobs_backward(state["x"], state["t"], state["lse"], state["h"], state["g_lp"], state["g_h"])
    got = token_logprobs(state["x"], state["t"], top=state["case"]["top"])
    out = {"logprob": got.logprob, "entropy": got.entropy, "lse": got.lse}
    if state["case"]["top"]:
        out["top_ids"], out["top_logprobs"] = got.top_ids, got.top_logprobs
    return out


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def _exact_quantised(x):
    """What a cached head stands for. The format is defined in 32-bit steps, so this follows them on 32-bit numbers; 64 bits hold every
    product of a code and a scale."""
    shape = x.shape
    x = x.reshape(-1, KV_GROUP)
    low, _ = x.min(dim=1)
    high, _ = x.max(dim=1)
    step = ((high - low).double() / 15.0).float().bfloat16()
    base = low.bfloat16()
    frac = ((x - base.float()[:, None]).double() / step.double()[:, None]).float().double()
    code = torch.where(step[:, None] > 0, torch.round(frac), torch.zeros_like(frac)).clamp_(0.0, 15.0)
    return (code * step.double()[:, None] + base.double()[:, None]).reshape(shape)


def _exact_attention(case, seed):
    q, k, v, old_k, old_v = _attention_inputs(case, seed)
    R, H, Hkv, hd = case["rows"], case["heads"], case["kv_heads"], case["hd"]
    half, g = hd // 2, H // Hkv
    freq = torch.tensor([ROPE_BASE ** (-2.0 * c / hd) for c in range(half)], dtype=torch.float64, device=DEV)
    outs, ks, vs = [], [], []
    for s, n in enumerate(_lengths(case)):
        rows = slice(s * R, (s + 1) * R)
        angle = torch.outer(torch.arange(n + R, dtype=torch.float64, device=DEV), freq)
        co, si = torch.cos(angle), torch.sin(angle)
        raw = torch.cat([old_k[s, :n], k[rows]]).reshape(n + R, Hkv, hd).float()
        c32, s32 = co.float()[:, None, :], si.float()[:, None, :]
        keys = torch.empty_like(raw)
        keys[..., :half] = raw[..., :half] * c32 - raw[..., half:] * s32
        keys[..., half:] = raw[..., half:] * c32 + raw[..., :half] * s32
        keys = _exact_quantised(keys)
        values = _exact_quantised(torch.cat([old_v[s, :n], v[rows]]).reshape(n + R, Hkv, hd).float())
        qs = q[rows].reshape(R, H, hd).double()
        cq, sq = co[n:, None, :], si[n:, None, :]
        turned = torch.cat([qs[..., :half] * cq - qs[..., half:] * sq, qs[..., half:] * cq + qs[..., :half] * sq], -1)
        merged = torch.empty(R, H, hd, dtype=torch.float64, device=DEV)
        hidden = torch.arange(n + R, device=DEV)[None, :] > n + torch.arange(R, device=DEV)[:, None]
        for h in range(H):
            score = turned[:, h] @ keys[:, h // g].t() * hd ** -0.5
            score[hidden] = -math.inf
            merged[:, h] = torch.softmax(score, dim=1) @ values[:, h // g]
        outs.append(merged.reshape(R, H * hd))
        ks.append(keys[n:].reshape(R, Hkv * hd))
        vs.append(values[n:].reshape(R, Hkv * hd))
    return torch.cat(outs), torch.cat(ks), torch.cat(vs)


def _exact_logprobs(case, seed):
    st = _logprob_inputs(case, seed)
    r, v, n = case["rows"], case["vocab"], case["top"]
    kept = {k: [] for k in ("logprob", "entropy", "lse", "top_logprobs", "grad")}
    step = max(1, (1 << 26) // v)
    for a in range(0, r, step):
        x, t = st["x"][a:a + step].double(), st["t"][a:a + step].long()
        if case["back"]:
            # d/dx of g_lp log p_t + g_h H at the given lse and H
            lse, h = st["lse"][a:a + step].double()[:, None], st["h"][a:a + step].double()[:, None]
            p = torch.exp(x - lse)
            mark = (torch.arange(v, device=DEV)[None] == t[:, None]).double()
            real = (t >= 0).double()[:, None]
            kept["grad"].append((st["g_lp"][a:a + step].double()[:, None] * real * (mark - p) - st["g_h"][a:a + step].double()[:, None]
                                 * (torch.special.xlogy(p, p) + p * h)))
            if step < r:
                kept["grad"][-1] = kept["grad"][-1].float()      # room: 32 bits say enough of a bf16 gradient
            continue
        logp = torch.log_softmax(x, dim=1)
        lse = torch.logsumexp(x, dim=1)
        kept["lse"].append(lse)
        kept["entropy"].append(torch.special.entr(logp.exp()).sum(dim=1))
        kept["logprob"].append(torch.where(t >= 0, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lse)))
        if n:
            kept["top_logprobs"].append(torch.sort(logp, dim=1, descending=True).values[:, :n])
    if case["back"]:
        return torch.cat(kept["grad"])
    out = {k: torch.cat(kept[k]) for k in ("logprob", "entropy", "lse")}
    if n:
        out["top_ids"], out["top_logprobs"] = None, torch.cat(kept["top_logprobs"])
    return out


def exact(case, seed):
    if case["op"] == "linear":
        x, codes, scales = _linear_inputs(case, seed)
        out, step = [], max(1, (1 << 27) // case["k"])
        for a in range(0, case["n"], step):
            w = codes[a:a + step].double() * scales[a:a + step].double().repeat_interleave(case["group"], dim=1)
            out.append(x.double() @ w.t())
        return torch.cat(out, dim=1)
    return _exact_attention(case, seed) if case["op"] == "attention" else _exact_logprobs(case, seed)
