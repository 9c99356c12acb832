"""New tokens of sequences whose keys and values are kept in pages, and attention that looks back over a window: the calls that are measured, their plain forms and their values in 64 bits.

Three kinds of pass:
  append   ``cache_append``: the new tokens' queries and keys are normalised (``norm``) and turned by their positions, keys and values are written into their pages
  attend   ``cache_attention`` of the last ``new[i]`` tokens of each sequence over its pages (``single``: one token of each, without offsets); with ``append`` they are appended first
  prompt   ``attention_ragged`` over packed sequences with a window and first tokens that stay visible (``sinks``); with ``train`` its gradients as well

Lengths are texts of numbers, one a sequence.  Heads: ``Hq`` of queries, ``Hkv`` of keys and values.  ``kind`` of a cache: bf16, fp16, e4m3 or int8 (8 bits with one fp32 scale for each
row of a head).  ``window``: how many keys a query looks back on, its own among them; 0: all.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
HEADS = [(8, 8), (16, 16), (16, 4), (32, 8), (40, 8), (12, 4), (14, 2), (16, 1)]
EPS = 1e-6
MAX_PAIRS = 1.2e9            # (query, key, head) triples of a drawn call, visible or not: its plain form keeps them all

_pkg = None


def package():
    global _pkg
    if _pkg is None:
        import __graft_entry__
        _pkg = __graft_entry__.load_package()
    return _pkg


def numbers(text):
    return [int(x) for x in text.split(",")]


def texts(values):
    return ",".join(str(v) for v in values)


def listed():
    heads = lambda Hq, Hkv, D, dtype, kind: {"Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "kind": kind}
    plain = {"axes": 0, "norm": False, "interleaved": False, "rot": 0}
    return [
        # one conversation's next token: latency
        {"name": "append_one", "op": "append", "lens": "333", "new": "1", "page": 16, **heads(16, 4, 64, "fp16", "fp16"), **plain, "rot": 64},
        # whole prompts into an 8-bit cache, queries and keys with their norms, and back for what reads them in 16 bits
        {"name": "append_prompt", "op": "append", "lens": "8192,4099,1,777", "new": "8192,4099,1,777", "page": 64, **heads(32, 8, 128, "bf16", "e4m3"), **plain, "norm": True, "rot": 128},
        # tokens of videos with positions in time, height and width
        {"name": "append_frames", "op": "append", "lens": "9360,1560,5000", "new": "7040,1560,880", "page": 128, **heads(16, 16, 128, "bf16", "bf16"), "axes": 3, "norm": True, "interleaved": False, "rot": 128},
        # few short pieces: latency
        {"name": "chunk_small", "op": "attend", "lens": "300,45,33", "new": "16,5,1", "single": False, "append": False, "window": 0, "sinks": 0, "page": 16, **heads(8, 2, 64, "fp16", "int8"), **plain},
        # the next pieces of long prompts
        {"name": "chunk_prompt", "op": "attend", "lens": "16384,9001,1301", "new": "2048,512,77", "single": False, "append": False, "window": 0, "sinks": 0, "page": 64, **heads(32, 8, 128, "bf16", "bf16"), **plain},
        # a serving step: two prompts' pieces between the next tokens of others, 8 bits
        {"name": "chunk_mixed", "op": "attend", "lens": texts([6000] + _ragged(46, 8000) + [1999]), "new": texts([512] + [1] * 46 + [300]), "single": False, "append": False, "window": 0, "sinks": 0, "page": 32,
         **heads(16, 8, 128, "bf16", "e4m3"), **plain},
        # long documents, every token looks back on a window and on the first four
        {"name": "window_prompt", "op": "prompt", "lens": "16384,5000,1777,1", "window": 1024, "sinks": 4, **heads(16, 4, 128, "bf16", ""), "train": False},
        # training on packed documents with a window
        {"name": "window_train", "op": "prompt", "lens": "8192,3001,511,1024", "window": 1024, "sinks": 4, **heads(32, 8, 128, "bf16", ""), "train": True},
        # smaller ones, a short window without first tokens
        {"name": "window_train_small", "op": "prompt", "lens": "1560,880,390", "window": 250, "sinks": 0, **heads(16, 16, 64, "fp16", ""), "train": True},
        # a batch's next tokens over the last 4096 keys of long conversations in 8 bits
        {"name": "window_decode", "op": "attend", "lens": texts(_ragged(64, 30000)), "new": texts([1] * 64), "single": True, "append": False, "window": 4096, "sinks": 4, "page": 64,
         **heads(32, 8, 128, "bf16", "int8"), **plain},
        # one conversation's next token: latency
        {"name": "window_decode_one", "op": "attend", "lens": "5001", "new": "1", "single": True, "append": False, "window": 500, "sinks": 16, "page": 16, **heads(16, 4, 64, "fp16", "fp16"), **plain},
        # a layer's step: new tokens of a batch appended, then attended to over a window
        {"name": "window_step", "op": "attend", "lens": texts(_ragged(30, 6000) + [5000, 700]), "new": texts([1] * 30 + [256, 33]), "single": False, "append": True, "window": 2048, "sinks": 4, "page": 32,
         **heads(32, 8, 128, "bf16", "bf16"), **plain, "norm": True, "rot": 64, "interleaved": True},
    ]


def _ragged(n, most):
    """n lengths from 1 to about `most`, spread over their logarithm."""
    return [max(1, int(most ** ((i * 0.6180339887) % 1.0))) if i % 3 else max(1, most - 61 * i) for i in range(1, n + 1)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "prompt", "prompt"])
    (Hq, Hkv), D, dtype = rng.choice(HEADS), rng.choice([64, 128]), rng.choice(["bf16", "fp16"])
    kind, page = rng.choice([dtype, "e4m3", "int8"]), rng.choice([16, 32, 64, 128])
    case = {"op": op, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "kind": kind}
    window, sinks = rng.choice([0, _log(rng, 1, 4096)]), rng.choice([0, 1, 4, 4, 64, 100])
    if op == "prompt":
        train, n, most = rng.random() < 0.5, _log(rng, 1, 24), _log(rng, 16, 8192)
        while n * Hq * most * most > MAX_PAIRS / (4 if train else 1):
            most = most * 2 // 3
        return {**case, "lens": texts([_log(rng, 1, most) for _ in range(n)]), "window": max(1, window), "sinks": sinks, "kind": "", "train": train}
    turned = {"axes": rng.choice([0, 0, 1, 3]), "norm": rng.random() < 0.5, "interleaved": rng.random() < 0.3, "rot": rng.choice([D, D, D // 2, 16])}
    if op == "append":
        n = _log(rng, 1, 64)
        most = _log(rng, 2, 32768 // n)
        new = [_log(rng, 1, most) for _ in range(n)]
        known = [0 if kind in QMAX else rng.choice([0, 1, _log(rng, 1, 4096)]) for _ in new]
        return {**case, "lens": texts([a + b for a, b in zip(known, new)]), "new": texts(new), "page": page, **turned}
    single, append, n = rng.random() < 0.35, rng.random() < 0.3, _log(rng, 1, 96)
    most = min(65536, _log(rng, 16, 1600000 // (n * Hkv)))
    lens = [_log(rng, 1, most) for _ in range(n)]
    new = [1 if single else min(m, rng.choice([1, 1, _log(rng, 1, 1024)])) for m in lens]
    while sum(a * b for a, b in zip(lens, new)) * Hq > MAX_PAIRS:
        new = [-(-a // 2) for a in new]
    if append:
        case["kind"] = dtype
    return {**case, "lens": texts(lens), "new": texts(new), "single": single, "append": append, "window": window, "sinks": sinks if window else 0, "page": page, **turned}


def _offsets(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows(gen, shape, dtype):
    """Rows whose channels differ in size, as those of a projection do."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return (x * (0.4 * torch.randn(shape[-1], generator=gen, device="cuda")).exp()).to(dtype)


def _filled(gen, pages, heads, page, D, kind):
    """One half of a cache that holds something everywhere, and its scales."""
    x = _rows(gen, (pages, heads, page, D), torch.float32)
    if kind not in QMAX:
        return x.to(DTYPES[kind]), None
    scale = x.abs().amax(-1) / QMAX[kind]
    x = x / scale[..., None]
    return (x.round() if kind == "int8" else x).to(DTYPES[kind]), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    D, dtype, Hq, Hkv = case["D"], DTYPES[case["dtype"]], case["Hq"], case["Hkv"]
    lens = numbers(case["lens"])
    if case["op"] == "prompt":
        s["cu"] = _int32(_offsets(lens))
        for name, heads in (("q", Hq), ("k", Hkv), ("v", Hkv)):
            s[name] = _rows(gen, (sum(lens), heads, D), dtype).requires_grad_(case["train"])
        if case["train"]:
            s["do"] = _rows(gen, (sum(lens), Hq, D), dtype)
        return s
    new, page = numbers(case["new"]), case["page"]
    rows = sum(new)
    s["cu"], s["lens_on"], s["cu_all"] = _int32(_offsets(new)), _int32(lens), _int32(_offsets(lens))
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 3
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    # entries behind a sequence's last page say nothing: page 0 here
    s["table"] = _int32([[free.pop() for _ in range(h)] + [0] * (max(held) - h) for h in held])
    parts = [_filled(gen, pages, Hkv, page, D, case["kind"]) for _ in range(2)]
    s["parts"] = [parts[0][0], parts[1][0], parts[0][1], parts[1][1]]
    s["q"] = _rows(gen, (rows, Hq, D), dtype)
    if case["op"] == "append" or case["append"]:
        s["k"], s["v"] = _rows(gen, (rows, Hkv, D), dtype), _rows(gen, (rows, Hkv, D), dtype)
        pairs, axes = case["rot"] // 2, max(1, case["axes"])
        freqs = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
        # (each axis turns channels of its own)
        of = torch.arange(pairs, device="cuda") * axes // pairs
        s["freqs"] = torch.stack([torch.where(of == a, freqs, 0.0) for a in range(axes)]).float()
        s["positions"] = None
        if case["axes"]:
            s["positions"] = torch.stack([torch.randint(0, most, (rows,), generator=gen, device="cuda") for most in (4096, 45, 80)[:axes]], 1).int()
        s["weights"] = [(1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(dtype) for _ in range(2)] if case["norm"] else [None, None]
    return s


# ---- plain forms
def _places(s):
    """The sequence of each new row, and its place there."""
    at = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu"], at, right=True) - 1
    return seq, (at - s["cu"][seq + 1] + s["lens_on"][seq]).long()


def _turned(x, weight, s, place, real=torch.float32):
    """Rows normalised and turned, in `real` (angles in 64 bits)."""
    x = x.to(real)
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(real)
    positions = place[:, None].double() if s["positions"] is None else s["positions"].double()
    angles = (positions[:, :, None] * s["freqs"].double()).sum(1)[:, None]
    cos, sin, pairs = angles.cos().to(real), angles.sin().to(real), s["rot"] // 2
    turned = x.clone()
    if s["interleaved"]:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned[..., 0:2 * pairs:2], turned[..., 1:2 * pairs:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned[..., :pairs], turned[..., pairs:2 * pairs] = a * cos - b * sin, b * cos + a * sin
    return turned


def _bytes(x):
    """(8 bits of floats are indexed as bytes)"""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _plain_append(s):
    seq, place = _places(s)
    q, k = (_turned(x, w, s, place) for x, w in zip((s["q"], s["k"]), s["weights"]))
    page, row = s["table"][seq, place // s["page"]].long(), place % s["page"]
    for x, to, scale in zip((k, s["v"].float()), s["parts"][:2], s["parts"][2:]):
        if scale is not None:
            by = x.abs().amax(-1) * (1 / QMAX[s["kind"]])
            scale[page, :, row] = by
            x = x / torch.where(by > 0, by, torch.ones_like(by))[..., None]
            x = x.round() if s["kind"] == "int8" else x
        _bytes(to)[page, :, row] = _bytes(x.to(to.dtype))
    return q.to(s["q"].dtype)


def _plain_pages(s, i, n):
    """The first n rows of sequence i, keys and values, [Hkv, n, D] in fp32."""
    table, got = s["table"][i, :-(-n // s["page"])].long(), []
    for x, scale in zip(s["parts"][:2], s["parts"][2:]):
        y = _bytes(x)[table].view(x.dtype).float()
        y = y if scale is None else y * scale[table][..., None]
        got.append(y.transpose(0, 1).reshape(s["Hkv"], -1, s["D"])[:, :n])
    return got


def _attend(q, k, v, window, sinks):
    """One sequence: q [n, Hq, D], k and v [Hkv, m, D] in fp32; the queries are the last n positions.  o and the log-sum-exp, [n, Hq]."""
    (n, Hq, D), (Hkv, m) = q.shape, k.shape[:2]
    Q = q.transpose(0, 1).reshape(Hkv, -1, D)
    scores = (Q @ k.transpose(-1, -2)).reshape(Hkv, -1, n, m) * D ** -0.5
    at, key = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")
    visible = key <= at
    if window:
        visible = visible & ((key > at - window) | (key < sinks))
    scores = torch.where(visible, scores, torch.full((), -math.inf, device="cuda"))
    top = scores.amax(-1, keepdim=True)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    out = ((p / total).reshape(Hkv, -1, m) @ v).reshape(Hq, n, D).transpose(0, 1)
    return out, (top + total.log()).reshape(Hq, n).t()


def _plain_attend(s):
    q = _plain_append(s) if s["append"] else s["q"]
    lens, at, got = numbers(s["lens"]), _offsets(numbers(s["new"])), []
    for i, m in enumerate(lens):
        got.append(_attend(q[at[i]:at[i + 1]].float(), *_plain_pages(s, i, m), s["window"], s["sinks"]))
    out = torch.cat([o for o, _ in got]).to(q.dtype), torch.cat([lse for _, lse in got])
    return (*out, *s["parts"][:2]) if s["append"] else out


def _plain_prompt(s, q, k, v):
    at = _offsets(numbers(s["lens"]))
    got = [_attend(q[a:b], k[a:b].transpose(0, 1), v[a:b].transpose(0, 1), s["window"], s["sinks"]) for a, b in zip(at[:-1], at[1:])]
    return torch.cat([o for o, _ in got]), torch.cat([lse for _, lse in got]).t()


def _plain(s):
    dtype = s["q"].dtype
    if s["op"] == "append":
        q = _plain_append(s)
        if s["kind"] not in QMAX:
            return (q, *s["parts"][:2])
        rows = [_plain_pages(s, i, m) for i, m in enumerate(numbers(s["lens"]))]
        return (q, *(torch.cat([r[j].transpose(0, 1) for r in rows]).to(dtype) for j in range(2)))
    if s["op"] == "attend":
        return _plain_attend(s)
    if not s["train"]:
        out, lse = _plain_prompt(s, *(s[n].float() for n in "qkv"))
        return out.to(dtype), lse
    leaves = [s[n].detach().float().requires_grad_() for n in "qkv"]
    out, _ = _plain_prompt(s, *leaves)
    grads = torch.autograd.grad(out, leaves, s["do"].float())
    return (out.detach().to(dtype), *(g.to(dtype) for g in grads))


# ---- the framework's calls
def _calls(s):
    P = package()
    if s["op"] == "prompt":
        if not s["train"]:
            return P.ragged_fwd(s["q"], s["k"], s["v"], s["cu"], causal=True, window=s["window"], sinks=s["sinks"])
        out = P.attention_ragged(s["q"], s["k"], s["v"], s["cu"], causal=True, window=s["window"], sinks=s["sinks"])
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"]))
    cache = s.get("cache")
    if cache is None:           # (a program makes it once)
        cache = s["cache"] = P.KVCache(*s["parts"])
    q, table, lens = s["q"], s["table"], s["lens_on"]
    if s["op"] == "append" or s["append"]:
        q = P.cache_append(cache, q, s["k"], s["v"], table, lens, s["cu"], freqs=s["freqs"], positions=s["positions"], interleaved=s["interleaved"], q_weight=s["weights"][0],
                           k_weight=s["weights"][1], eps=EPS)
    if s["op"] == "append":
        if s["kind"] not in QMAX:
            return (q, *s["parts"][:2])
        return (q, *P.cache_read(cache, table, s["cu_all"], sum(numbers(s["lens"])), dtype=q.dtype))
    out = P.cache_attention(q, cache, table, lens, need_lse=True, cu=None if s["single"] else s["cu"], window=s["window"] or None, sinks=s["sinks"])
    return (*out, *s["parts"][:2]) if s["append"] else out


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


# ---- what a pass cannot do without
def _pairs(case):
    """Visible (query, key) pairs of all sequences."""
    lens, total = numbers(case["lens"]), 0
    for m, n in zip(lens, numbers(case["new"]) if case["op"] == "attend" else lens):
        W, S = (case["window"], case["sinks"]) if case["window"] else (m, 0)
        # position p sees min(p + 1, W) keys of its window, and of the S first ones those before it
        upto = lambda p: _sum(min(p, W)) + max(0, p - W) * W + _sum(min(max(0, p - W), S)) + max(0, p - W - S) * S
        total += upto(m) - upto(m - n)
    return total


def _sum(n):
    return n * (n + 1) // 2


def _seen(case):
    """Keys that some query of their sequence sees."""
    total = 0
    for m, n in zip(numbers(case["lens"]), numbers(case["new"])):
        first = max(0, m - n - case["window"] + 1) if case["window"] else 0
        total += m - first + min(first, case["sinks"])
    return total


def work(case):
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    if case["op"] == "prompt":
        rows, products = sum(numbers(case["lens"])), Hq * D * _pairs(case)
        q, k = rows * Hq * D * 2, rows * Hkv * D * 2
        if case["train"]:       # forward 2 products, backward 5; q, k, v, do in, o and the gradients out
            return {"bytes": 4 * q + 4 * k, "flops": 14 * products}
        return {"bytes": 2 * q + 2 * k + rows * Hq * 4, "flops": 4 * products}
    rows, cached = sum(numbers(case["new"])), D * 2 if case["kind"] not in QMAX else D + 4        # (bytes of a row of a head)
    turned = {"bytes": rows * (2 * Hq * D * 2 + 2 * Hkv * (D * 2 + cached) + 4 * case["axes"]), "flops": rows * (Hq + Hkv) * (3 * case["rot"] + (4 * D if case["norm"] else 0))}
    if case["op"] == "append":
        if case["kind"] in QMAX:                # (and back)
            turned["bytes"] += rows * 2 * Hkv * (cached + D * 2)
        return turned
    attended = {"bytes": _seen(case) * 2 * Hkv * cached + rows * Hq * (2 * D * 2 + 4), "flops": 4 * Hq * D * _pairs(case)}
    return {n: attended[n] + turned[n] for n in attended} if case["append"] else attended


# ---- 64 bits
def _attend64(q, k, v, window, sinks, first):
    """One head: rows `first` .. of a sequence's positions.  softmax(q k^T / sqrt D) and its log-sum-exp."""
    s = q @ k.t() * q.shape[1] ** -0.5
    t, j = torch.arange(first, first + q.shape[0], device="cuda")[:, None], torch.arange(k.shape[0], device="cuda")
    hidden = j > t
    if window:
        hidden |= (j <= t - window) & (j >= sinks)
    s.masked_fill_(hidden, -math.inf)
    lse = torch.logsumexp(s, -1)
    return torch.exp(s - lse[:, None]), lse


def _exact_prompt(case, s):
    q, k, v = (s[n].detach().double() for n in "qkv")
    out, lse = torch.zeros_like(q), torch.zeros((case["Hq"], q.shape[0]), dtype=torch.float64, device="cuda")
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    scale, group, at = case["D"] ** -0.5, case["Hq"] // case["Hkv"], _offsets(numbers(case["lens"]))
    for a, b in zip(at[:-1], at[1:]):
        for h in range(case["Hq"]):
            for t in range(0, b - a, 4096):
                rows, end = slice(a + t, min(b, a + t + 4096)), min(b, a + t + 4096)       # (later keys are hidden from all of them)
                K, V = k[a:end, h // group], v[a:end, h // group]
                P, lse[h, rows] = _attend64(q[rows, h], K, V, case["window"], case["sinks"], t)
                out[rows, h] = P @ V
                if case["train"]:
                    g = s["do"][rows, h].double()
                    dS = P * (g @ V.t() - (g * out[rows, h]).sum(-1, keepdim=True)) * scale
                    grads[0][rows, h] = dS @ K
                    grads[1][a:end, h // group] += dS.t() @ q[rows, h]
                    grads[2][a:end, h // group] += P.t() @ g
    return (out, *grads) if case["train"] else (out, lse)


def _turned64(x, weight, s, place):
    """By products of complex numbers."""
    x = x.double()
    if weight is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    positions = place[:, None].double() if s["positions"] is None else s["positions"].double()
    by = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions @ s["freqs"].double())[:, None]
    R, y = s["rot"] // 2, x.clone()
    first, second = (slice(0, 2 * R, 2), slice(1, 2 * R, 2)) if s["interleaved"] else (slice(0, R), slice(R, 2 * R))
    z = torch.complex(x[..., first], x[..., second]) * by
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _places64(case):
    return torch.cat([torch.arange(m - n, m, device="cuda") for m, n in zip(numbers(case["lens"]), numbers(case["new"]))])


def _held64(x, case):
    """What rows stand for once they lie in the cache."""
    if case["kind"] not in QMAX:
        return x
    # (a scale is the largest times 1 / QMAX, all in fp32, and a code the quotient rounded once: 16-bit values often lie on a border between two codes)
    by = (x.abs().amax(-1, keepdim=True).float() * torch.tensor(1 / QMAX[case["kind"]], device="cuda")).double()
    codes = (x / by.clamp(min=1e-300)).float()
    return (codes.round() if case["kind"] == "int8" else codes.to(torch.float8_e4m3fn)).double() * by


def _pages64(case, s, i, m):
    table, at, got = s["table"][i].long(), torch.arange(m, device="cuda"), []
    for x, by in zip(s["parts"][:2], s["parts"][2:]):
        y = _bytes(x)[table[at // case["page"]], :, at % case["page"]].view(x.dtype).double()
        got.append(y if by is None else y * by[table[at // case["page"]], :, at % case["page"]].double()[..., None])
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":
        return _exact_prompt(case, s)
    lens, at, q = numbers(case["lens"]), _offsets(numbers(case["new"])), s["q"].double()
    fresh, pools = None, []
    if case["op"] == "append" or case["append"]:
        place = _places64(case)
        q, k = (_turned64(x, w, s, place) for x, w in zip((s["q"], s["k"]), s["weights"]))
        fresh = [_held64(x, case) for x in (k, s["v"].double())]
        if case["kind"] not in QMAX:
            seq = torch.cat([torch.full((b - a,), i, device="cuda") for i, (a, b) in enumerate(zip(at[:-1], at[1:]))])
            for x, y in zip(s["parts"][:2], fresh):
                pool = x.double()
                pool[s["table"][seq, place // case["page"]].long(), :, place % case["page"]] = y
                pools.append(pool)
    if case["op"] == "append":
        return (q, *(fresh if case["kind"] in QMAX else pools))       # (in 8 bits every position is a new one)
    if fresh:       # (between the two calls queries, keys and values are held in 16 bits)
        q, fresh = q.to(s["q"].dtype).double(), [x.to(s["q"].dtype).double() for x in fresh]
    out, lse, group = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda"), case["Hq"] // case["Hkv"]
    for i, m in enumerate(lens):
        rows = slice(at[i], at[i + 1])
        K, V = _pages64(case, s, i, m)
        if fresh:
            K[m - at[i + 1] + at[i]:], V[m - at[i + 1] + at[i]:] = fresh[0][rows], fresh[1][rows]
        for h in range(case["Hq"]):
            P, lse[rows, h] = _attend64(q[rows, h], K[:, h // group], V[:, h // group], case["window"], case["sinks"], m - at[i + 1] + at[i])
            out[rows, h] = P @ V[:, h // group]
    return (out, lse, *pools) if case["append"] else (out, lse)
