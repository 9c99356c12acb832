"""Attention over sequences of different lengths and over a paged key-value cache: the calls that are measured, their plain forms and their values in 64 bits.

Three kinds of pass:
  prompt   ``attention_ragged``: packed sequences, grouped heads, causal (aligned at the sequences' ends) or not; with ``train`` its gradients as well
  decode   ``cache_attention``: one new token of each sequence over its pages; with ``write`` that token's key and value are written first (``cache_write``)
  cache    ``cache_write`` of packed rows into pages and ``cache_read`` of all of them

Lengths are texts of numbers, one a sequence.  Heads: ``Hq`` of queries, ``Hkv`` of keys and values.  ``kind`` of a cache: bf16, fp16, e4m3 or int8 (8 bits with one fp32
scale for each row of a head).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
HEADS = [(8, 8), (16, 16), (16, 4), (32, 8), (40, 8), (12, 4), (14, 2), (16, 1)]
MAX_PAIRS = 1.2e9            # visible or hidden (query, key, head) triples of a drawn prompt: its plain form keeps them all

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
    return [
        # a short request alone, as it arrives: latency
        {"name": "prompt_one", "op": "prompt", "q_lens": "37", "k_lens": "37", "Hq": 8, "Hkv": 2, "D": 64, "dtype": "fp16", "causal": True, "train": False},
        # a serving batch's prompts of every length, one of them a single token
        {"name": "prompt_ragged", "op": "prompt", "q_lens": "1777,64,511,1,2048,129,1000,333,1531,700,48,255", "k_lens": "1777,64,511,1,2048,129,1000,333,1531,700,48,255",
         "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16", "causal": True, "train": False},
        # one long document
        {"name": "prompt_long", "op": "prompt", "q_lens": "16384", "k_lens": "16384", "Hq": 16, "Hkv": 4, "D": 128, "dtype": "bf16", "causal": True, "train": False},
        # the next piece of prompts whose first parts are known already: few queries, many keys
        {"name": "prompt_chunk", "op": "prompt", "q_lens": "512,77,1", "k_lens": "8192,1301,4097", "Hq": 16, "Hkv": 2, "D": 128, "dtype": "fp16", "causal": True, "train": False},
        # training on packed documents, grouped heads
        {"name": "train_ragged", "op": "prompt", "q_lens": "2048,1023,4096,511", "k_lens": "2048,1023,4096,511", "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16", "causal": True, "train": True},
        # training on packed images of three sizes: every token sees its whole image
        {"name": "train_frames", "op": "prompt", "q_lens": "1560,880,390", "k_lens": "1560,880,390", "Hq": 16, "Hkv": 16, "D": 64, "dtype": "fp16", "causal": False, "train": True},
        # one conversation, its next token: latency
        {"name": "decode_one", "op": "decode", "lens": "333", "capacity": 512, "page": 16, "Hq": 16, "Hkv": 4, "D": 64, "dtype": "fp16", "kind": "fp16", "write": False},
        # a serving batch's next tokens, conversations of every length
        {"name": "decode_ragged", "op": "decode", "lens": texts(_ragged(48, 8000)), "capacity": 8192, "page": 64, "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16", "kind": "bf16", "write": False},
        # few very long contexts in 8 bits
        {"name": "decode_long", "op": "decode", "lens": "131072,70001,99", "capacity": 131072, "page": 128, "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16", "kind": "e4m3", "write": False},
        # a layer's step: the new tokens into an 8-bit cache, then attention over it
        {"name": "step_int8", "op": "decode", "lens": texts(_ragged(32, 3000)), "capacity": 4096, "page": 32, "Hq": 16, "Hkv": 8, "D": 128, "dtype": "bf16", "kind": "int8", "write": True},
        # a prompt's keys and values into the cache and back, for its next piece
        {"name": "cache_prompt", "op": "cache", "lens": "16384,9999,1,4096", "page": 64, "Hkv": 8, "D": 128, "dtype": "bf16", "kind": "e4m3"},
        # a few short prompts
        {"name": "cache_small", "op": "cache", "lens": "17,5,40", "page": 16, "Hkv": 2, "D": 64, "dtype": "fp16", "kind": "int8"},
    ]


def _ragged(n, most):
    """n lengths from 1 to about `most`, spread over their logarithm."""
    return [max(1, int(most ** ((i * 0.6180339887) % 1.0))) if i % 3 else max(1, most - 61 * i) for i in range(1, n + 1)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "decode", "decode", "cache"])
    (Hq, Hkv), D, dtype = rng.choice(HEADS), rng.choice([64, 128]), rng.choice(["bf16", "fp16"])
    if op == "prompt":
        train, n, most = rng.random() < 0.4, _log(rng, 1, 24), _log(rng, 16, 8192)
        while n * Hq * most * most > MAX_PAIRS / (4 if train else 1):
            most = most * 2 // 3
        q = [_log(rng, 1, most) for _ in range(n)]
        causal = rng.random() < 0.75
        k = [min(most, v + rng.choice([0, 0, 1, 63, most])) for v in q] if causal and rng.random() < 0.3 else q
        return {"op": "prompt", "q_lens": texts(q), "k_lens": texts(k), "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "causal": causal, "train": train}
    page = rng.choice([16, 32, 64, 128])
    kind = rng.choice([dtype, "e4m3", "int8"])
    if op == "decode":
        n = _log(rng, 1, 128)
        most = min(131072, _log(rng, 16, 3200000 // (n * Hkv)))
        lens = [_log(rng, 1, most) for _ in range(n)]
        return {"op": "decode", "lens": texts(lens), "capacity": -(-most // page) * page, "page": page, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "kind": kind, "write": rng.random() < 0.4}
    n = _log(rng, 1, 32)
    most = _log(rng, 4, 32768 // n)
    return {"op": "cache", "lens": texts([_log(rng, 1, most) for _ in range(n)]), "page": page, "Hkv": Hkv, "D": D, "dtype": dtype, "kind": kind}


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
    D, dtype, Hkv = case["D"], DTYPES[case["dtype"]], case["Hkv"]
    if case["op"] == "prompt":
        ql, kl = numbers(case["q_lens"]), numbers(case["k_lens"])
        s["cu_q"], s["cu_k"] = _int32(_offsets(ql)), _int32(_offsets(kl))
        s["q_most"], s["k_most"] = max(ql), max(kl)
        for name, rows, heads in (("q", sum(ql), case["Hq"]), ("k", sum(kl), Hkv), ("v", sum(kl), Hkv)):
            s[name] = _rows(gen, (rows, heads, D), dtype).requires_grad_(case["train"])
        if case["train"]:
            s["do"] = _rows(gen, (sum(ql), case["Hq"], D), dtype)
        return s
    lens, page = numbers(case["lens"]), case["page"]
    s["lens"] = _int32(lens)
    width = -(-(case["capacity"] if case["op"] == "decode" else max(lens)) // page)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 3
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    # entries behind a sequence's last page say nothing: page 0 here
    s["table"] = _int32([[free.pop() for _ in range(h)] + [0] * (width - h) for h in held])
    parts = [_filled(gen, pages, Hkv, page, D, case["kind"]) for _ in range(2)]
    s["parts"] = [parts[0][0], parts[1][0], parts[0][1], parts[1][1]]
    if case["op"] == "decode":
        s["q"] = _rows(gen, (len(lens), case["Hq"], D), dtype)
        fresh = len(lens) if case["write"] else 0
    else:
        fresh = sum(lens)
        s["cu"] = _int32(_offsets(lens))
    s["fresh"] = [_rows(gen, (fresh, Hkv, D), dtype) for _ in range(2)] if fresh else None
    return s


# ---- plain forms
def _padded(x, cu, most):
    """Packed rows [T, H, D] as [B, H, most, D] in fp32, zeros behind a sequence's end."""
    start, at = cu[:-1, None].long(), torch.arange(most, device=x.device)
    live = at < (cu[1:, None] - cu[:-1, None])
    y = x.float()[(start + at).clamp(max=x.shape[0] - 1)]
    return torch.where(live[:, :, None, None], y, torch.zeros((), device=x.device)).transpose(1, 2)


def _places(cu, rows):
    """The sequence of each of the packed rows, and its place there."""
    at = torch.arange(rows, device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(cu, at, right=True) - 1
    return seq, at.long() - cu[seq].long()


def _softmax(scores, visible):
    """exp(scores - max) where visible, its sum, and its logarithm with the max put back."""
    scores = torch.where(visible, scores, torch.full((), -math.inf, device=scores.device))
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top.isinf(), torch.zeros_like(top), top)).exp()
    total = p.sum(-1, keepdim=True)
    return p, total, (top + total.log()).squeeze(-1)


def _plain_prompt(s, q, k, v):
    cu_q, cu_k, group = s["cu_q"], s["cu_k"], s["Hq"] // s["Hkv"]
    Q, K, V = _padded(q, cu_q, s["q_most"]), _padded(k, cu_k, s["k_most"]), _padded(v, cu_k, s["k_most"])
    B, n, m, D = Q.shape[0], s["q_most"], s["k_most"], s["D"]
    Q = Q.reshape(B, s["Hkv"], group * n, D)
    scores = (Q @ K.transpose(-1, -2)).reshape(B, s["Hkv"], group, n, m) * D ** -0.5
    lq, lk = (cu_q[1:] - cu_q[:-1])[:, None, None], (cu_k[1:] - cu_k[:-1])[:, None, None]
    at, key = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)
    visible = (key < lk).expand(B, n, m) if not s["causal"] else (key < lk) & (key <= at + lk - lq)
    p, total, lse = _softmax(scores, visible[:, None, None])
    out = (p / total.clamp(min=1e-30)).reshape(B, s["Hkv"], group * n, m) @ V
    seq, place = _places(cu_q, q.shape[0])
    out = out.reshape(B, s["Hq"], n, D)[seq, :, place]
    return out, lse.reshape(B, s["Hq"], n)[seq, :, place].t()


def _plain_write(s, rows, new):
    """Writes fresh rows, the last `new[i]` positions of sequence i each."""
    k, v, k_scale, v_scale = s["parts"]
    cu = torch.cat([new.new_zeros(1), new.cumsum(0, dtype=torch.int32)])
    seq, place = _places(cu, rows[0].shape[0])
    place = place + (s["lens"] - new)[seq].long()
    page, row = s["table"][seq, place // s["page"]].long(), place % s["page"]
    for x, to, scale in ((rows[0], k, k_scale), (rows[1], v, v_scale)):
        x = x.float()
        if scale is not None:
            by = x.abs().amax(-1) / QMAX[s["kind"]]
            scale[page, :, row] = by
            x = x / torch.where(by > 0, by, torch.ones_like(by))[..., None]
            x = x.round() if s["kind"] == "int8" else x
        # (8 bits of floats are written as bytes: indexing is not there for them)
        to.view(torch.uint8 if s["kind"] == "e4m3" else to.dtype)[page, :, row] = x.to(to.dtype).view(torch.uint8) if s["kind"] == "e4m3" else x.to(to.dtype)


def _plain_pages(s):
    """Every sequence's pages side by side, [B, Hkv, capacity, D] in fp32, for keys and for values."""
    table, got = s["table"].long(), []
    for x, scale in zip(s["parts"][:2], s["parts"][2:]):
        y = x.view(torch.uint8)[table].view(x.dtype).float() if s["kind"] == "e4m3" else x[table].float()
        y = y if scale is None else y * scale[table][..., None]
        got.append(y.transpose(1, 2).reshape(table.shape[0], s["Hkv"], -1, s["D"]))
    return got


def _plain_decode(s):
    if s["write"]:
        _plain_write(s, s["fresh"], torch.ones_like(s["lens"]))
    K, V = _plain_pages(s)
    B = K.shape[0]
    Q = s["q"].float().reshape(B, s["Hkv"], -1, s["D"])
    visible = torch.arange(K.shape[2], device=K.device) < s["lens"][:, None]
    p, total, lse = _softmax(Q @ K.transpose(-1, -2) * s["D"] ** -0.5, visible[:, None, None])
    out = (p / total) @ V
    return out.reshape(s["q"].shape).to(s["q"].dtype), lse.reshape(B, -1)


def _plain_cache(s):
    _plain_write(s, s["fresh"], s["lens"])
    seq, place = _places(s["cu"], s["fresh"][0].shape[0])
    return tuple(x[seq, :, place].to(s["fresh"][0].dtype) for x in _plain_pages(s))


def _plain(s):
    if s["op"] == "decode":
        return _plain_decode(s)
    if s["op"] == "cache":
        return _plain_cache(s)
    if not s["train"]:
        out, lse = _plain_prompt(s, s["q"], s["k"], s["v"])
        return out.to(s["q"].dtype), lse
    leaves = [s[n].detach().float().requires_grad_() for n in "qkv"]
    out, _ = _plain_prompt(s, *leaves)
    grads = torch.autograd.grad(out, leaves, s["do"].float())
    return (out.detach().to(s["q"].dtype), *(g.to(s["q"].dtype) for g in grads))


# ---- the framework's calls
def _calls(s):
    P = package()
    if s["op"] == "prompt":
        if not s["train"]:
            return P.ragged_fwd(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["causal"])
        out = P.attention_ragged(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["causal"])
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"]))
    cache = s.get("cache")
    if cache is None:           # (a program makes it once)
        cache = s["cache"] = P.KVCache(*s["parts"])
    if s["op"] == "decode":
        if s["write"]:
            P.cache_write(cache, *s["fresh"], s["table"], s["lens"])
        return P.cache_attention(s["q"], cache, s["table"], s["lens"], need_lse=True)
    P.cache_write(cache, *s["fresh"], s["table"], s["lens"], s["cu"])
    return P.cache_read(cache, s["table"], s["cu"], s["fresh"][0].shape[0], dtype=s["fresh"][0].dtype)


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


# ---- what a pass cannot do without
def _pairs(case):
    """Visible (query, key) pairs of all sequences."""
    total = 0
    for n, m in zip(numbers(case["q_lens"]), numbers(case["k_lens"])):
        if case["causal"]:      # row t sees max(0, t + 1 + m - n) keys
            first = max(0, n - m)
            total += sum_to(m) - sum_to(first + m - n)
        else:
            total += n * m
    return total


def sum_to(n):
    return n * (n + 1) // 2


def work(case):
    D, Hkv = case["D"], case["Hkv"]
    if case["op"] == "prompt":
        q, k = sum(numbers(case["q_lens"])) * case["Hq"] * D * 2, sum(numbers(case["k_lens"])) * Hkv * D * 2
        products = case["Hq"] * D * _pairs(case)
        if case["train"]:       # forward 2 products, backward 5; q, k, v, do in, o and the gradients out
            return {"bytes": 2 * q + 2 * k + 2 * q + 2 * k, "flops": 14 * products}
        return {"bytes": 2 * q + 2 * k + sum(numbers(case["q_lens"])) * case["Hq"] * 4, "flops": 4 * products}
    lens = numbers(case["lens"])
    rows = sum(lens) * Hkv * 2
    cached = rows * (D * 2 if case["kind"] not in QMAX else D + 4)
    if case["op"] == "decode":
        q = len(lens) * case["Hq"] * D * 2
        return {"bytes": cached + 2 * q + (len(lens) * Hkv * 4 * D if case["write"] else 0), "flops": 4 * sum(lens) * case["Hq"] * D}
    return {"bytes": 2 * rows * D * 2 + 2 * cached, "flops": 2 * rows * D}


# ---- 64 bits
def _attend64(q, k, v, scale, hidden_from=None):
    """One head of one sequence: softmax(scale q k^T) v and its log-sum-exp; row t sees the keys below hidden_from[t]."""
    s = q @ k.t() * scale
    if hidden_from is not None:
        s.masked_fill_(torch.arange(k.shape[0], device=q.device) >= hidden_from[:, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    return torch.exp(s - lse.clamp(min=-1e300)[:, None]), lse


def _exact_prompt(case, s):
    q, k, v = (s[n].detach().double() for n in "qkv")
    out, lse = torch.zeros_like(q), torch.full((case["Hq"], q.shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    scale, group = case["D"] ** -0.5, case["Hq"] // case["Hkv"]
    qa, ka = _offsets(numbers(case["q_lens"])), _offsets(numbers(case["k_lens"]))
    for i in range(len(qa) - 1):
        n, m = qa[i + 1] - qa[i], ka[i + 1] - ka[i]
        for h in range(case["Hq"]):
            K, V = k[ka[i]:ka[i + 1], h // group], v[ka[i]:ka[i + 1], h // group]
            for a in range(0, n, 4096):
                rows = slice(qa[i] + a, qa[i] + min(n, a + 4096))
                t = torch.arange(a, min(n, a + 4096), device="cuda")
                P, lse[h, rows] = _attend64(q[rows, h], K, V, scale, t + 1 + m - n if case["causal"] else None)
                out[rows, h] = P @ V
                if case["train"]:
                    g = s["do"][rows, h].double()
                    dS = P * (g @ V.t() - (g * out[rows, h]).sum(-1, keepdim=True)) * scale
                    grads[0][rows, h] = dS @ K
                    grads[1][ka[i]:ka[i + 1], h // group] += dS.t() @ q[rows, h]
                    grads[2][ka[i]:ka[i + 1], h // group] += P.t() @ g
    return (out, *grads) if case["train"] else (out, lse)


def _written64(case, s, new):
    """The rows of the cache that sequence i's positions stand for, [lens[i], Hkv, D], keys and values."""
    lens, page, rows = numbers(case["lens"]), case["page"], []
    start = _offsets(new)
    for i, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        pages = s["table"][i].long()[at // page]
        pair = []
        for j in range(2):
            x, by = s["parts"][j], s["parts"][2 + j]
            y = x.view(torch.uint8)[pages, :, at % page].view(x.dtype).double() if case["kind"] == "e4m3" else x[pages, :, at % page].double()
            y = y if by is None else y * by[pages, :, at % page].double()[..., None]
            if new[i]:
                fresh = s["fresh"][j][start[i]:start[i + 1]].double()
                if case["kind"] in QMAX:
                    # (a scale is held in fp32, and a code is the quotient in fp32 rounded once more: what lies next to a border is the operator's to say)
                    by = (fresh.abs().amax(-1, keepdim=True) / QMAX[case["kind"]]).float().double()
                    codes = (fresh / by.clamp(min=1e-300)).float()
                    fresh = (codes.round() if case["kind"] == "int8" else codes.to(torch.float8_e4m3fn)).double() * by
                y[n - new[i]:] = fresh
            pair.append(y)
        rows.append(pair)
    return rows


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":
        return _exact_prompt(case, s)
    lens = numbers(case["lens"])
    if case["op"] == "cache":
        rows = _written64(case, s, lens)
        return tuple(torch.cat([pair[j] for pair in rows]) for j in range(2))
    rows = _written64(case, s, [1 if case["write"] else 0] * len(lens))
    q, group = s["q"].double(), case["Hq"] // case["Hkv"]
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    for i, (K, V) in enumerate(rows):
        for h in range(case["Hkv"]):
            heads = slice(h * group, (h + 1) * group)
            P, lse[i, heads] = _attend64(q[i, heads], K[:, h], V[:, h], case["D"] ** -0.5)
            out[i, heads] = P @ V[:, h]
    return out, lse
