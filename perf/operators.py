"""The paged-cache and draft operators as performance cases: inputs, one pass through each in plain torch
or through the framework, the work a pass cannot do without, and the same results in 64 bits.

A case is a dict of plain values; `op` says which operator a pass runs:
  append     new K / V rows of several sequences into the pages of a quantised cache, then read back
             as the values that the cache now holds
  read       every cached row of several sequences, dense and dequantised
  attention  new tokens of several sequences over their pages (one token each when decoding, a few
             when a draft is checked, many when a prompt is read)
  verify     drafted tokens against the target's probabilities with given random numbers
Sequences have `new_lo` to `new_hi` new tokens behind `old_lo` to `old_hi` cached ones, spread over the
logarithm and fixed by the case. q, k and v are columns of one projection output, as a layer has them.

The pages: a byte tensor [layer][K, V][page][kv head][cell]. A cell is the codes, then the scales: K
codes [head_dim / 32][position][32], V codes [head_dim][position] (Q4_0: 16 bytes in place of 32 codes,
byte j holding element j in its low half and element j + 16 in its high half), scales
[head_dim / 32][position] in half precision.
"""
import math
import random

import torch

own = False  # False: plain torch; True: the framework's operators

ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
NO_WINDOW = 0x7FFFFFFF


def _cache(name, op, cache, act, heads, kv_heads, head_dim, page, seqs, new, old, window=NO_WINDOW, softcap=0.0):
    c = dict(op=op, cache=cache, act=act, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, seqs=seqs,
             new_lo=new[0], new_hi=new[1], old_lo=old[0], old_hi=old[1], window=window, softcap=softcap)
    return dict(c, name=name) if name else c


def _verify(name, seqs, drafts, vocab, greedy):
    c = dict(op="verify", seqs=seqs, drafts=drafts, vocab=vocab, greedy=greedy)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decode step of 64 requests: a row each, the launch-bound end
        _cache("append-decode", "append", "q8_0", "f32", 32, 8, 128, 64, 64, (1, 1), (100, 4000)),
        # the prompts of four requests go in, thousands of rows
        _cache("append-prompts", "append", "q4_0", "f32", 28, 4, 128, 32, 4, (900, 4000), (0, 300)),
        # a small model's session read back by its host
        _cache("read-session", "read", "f16", "f32", 8, 2, 64, 16, 1, (1, 1), (700, 800)),
        # long sessions taken out of the pages into dense half-precision rows
        _cache("read-long", "read", "q8_0", "f16", 16, 8, 256, 64, 8, (1, 1), (3000, 16000)),
        # one chat request decodes at an ordinary context: latency
        _cache("decode-chat", "attention", "q8_0", "f32", 32, 8, 128, 64, 1, (1, 1), (518, 518)),
        # 64 requests decode, short and long ones in one batch
        _cache("decode-batch", "attention", "q8_0", "f32", 28, 4, 128, 64, 64, (1, 1), (200, 8000)),
        # one request with a very long context decodes from a 4-bit cache
        _cache("decode-long", "attention", "q4_0", "f32", 32, 8, 128, 128, 1, (1, 1), (131070, 131070)),
        # four drafted tokens and the last accepted one of 16 requests are scored
        _cache("draft-chunk", "attention", "f16", "bf16", 32, 8, 128, 32, 16, (5, 5), (1000, 6000)),
        # prompts of three requests in one pass, half precision throughout
        _cache("prompt-chunk", "attention", "f16", "bf16", 32, 8, 128, 64, 3, (1500, 3500), (500, 5000)),
        # a chunk of a long prompt: sliding window, soft cap, wide heads, 8-bit cache, full precision
        _cache("prompt-window", "attention", "q8_0", "f32", 16, 8, 256, 64, 1, (2047, 2047), (4097, 4097), 4096, 50.0),
        # a draft of four tokens for one request
        _verify("verify-one", 1, 4, 128256, False),
        # drafts of up to eight tokens for 64 requests
        _verify("verify-batch", 64, 8, 152064, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attention", "attention", "attention", "verify"])
    if op == "verify":
        seqs = _log(rng, 1, 64)
        return _verify(None, seqs, rng.randint(1, 8), _log(rng, 500, 152064), rng.random() < 0.3)
    heads, kv, hd = rng.choice([(32, 8, 128), (28, 4, 128), (16, 8, 256), (8, 2, 64), (12, 2, 128), (8, 4, 256),
                                (4, 4, 96), (16, 1, 128), (10, 5, 160), (8, 8, 32)])
    cache, act = rng.choice(["f16", "q8_0", "q4_0"]), rng.choice(["f32", "f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op != "attention":
        seqs = _log(rng, 1, 64)
        rows = _log(rng, 64, 16384)
        new = max(1, rows // seqs)
        if op == "append":
            return _cache(None, op, cache, act, heads, kv, hd, page, seqs, (max(1, new // 3), new), (0, 500))
        return _cache(None, op, cache, act, heads, kv, hd, page, seqs, (1, 1), (new // 3, new))
    window, softcap = rng.choice([NO_WINDOW, NO_WINDOW, _log(rng, 5, 4096)]), rng.choice([0.0, 0.0, 50.0])
    kind = rng.choice(["decode", "draft", "prompt"])
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        most = min(100000, 300000 // seqs)
        old = _log(rng, 20, most)
        new = (1, 1)
    elif kind == "draft":
        seqs = _log(rng, 1, 32)
        old = _log(rng, 20, min(30000, 100000 // seqs))
        new = (1, rng.randint(2, 16))
    else:
        seqs = rng.randint(1, 4)
        old = _log(rng, 1, 3000)
        n = _log(rng, 33, 4000 // seqs)
        new = (max(1, n // 3), n)
    return _cache(None, op, cache, act, heads, kv, hd, page, seqs, new, (old // 4, old), window, softcap)


def _lengths(c):
    """(new tokens, cached tokens before them) of each sequence."""
    rng = random.Random("%(seqs)d %(new_lo)d %(new_hi)d %(old_lo)d %(old_hi)d %(page)d" % c)
    spread = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1) + 1e-9)) - 0.5)  # noqa: E731
    both = [(spread(c["new_lo"], c["new_hi"]), spread(c["old_lo"], c["old_hi"])) for _ in range(c["seqs"])]
    return [max(n, c["new_lo"]) for n, _ in both], [o for _, o in both]


def _seen(new, old, window):
    """Query-key pairs of one sequence."""
    return sum(min(p + 1, window) for p in range(old, old + new))


def work(c):
    if c["op"] == "verify":
        b = c["seqs"] * (2 * c["vocab"] * 4 + c["drafts"] * 20 + 12)
        return {"bytes": b, "flops": 2 * c["seqs"] * c["vocab"]}
    new, old = _lengths(c)
    width = c["kv_heads"] * c["head_dim"]
    elem = {"f16": 2, "q8_0": 34 / 32, "q4_0": 18 / 32}[c["cache"]]
    act = 4 if c["act"] == "f32" else 2
    t = sum(new)
    if c["op"] == "append":  # rows in, codes out and in again, values out
        return {"bytes": 2 * t * width * (act + elem + elem + 4), "flops": 8 * t * width}
    if c["op"] == "read":
        return {"bytes": 2 * (t + sum(old)) * width * (elem + act), "flops": 2 * (t + sum(old)) * width}
    live = sum(min(n + o, c["window"] + n - 1) for n, o in zip(new, old))
    pairs = sum(_seen(n, o, c["window"]) for n, o in zip(new, old))
    return {"bytes": 2 * live * width * elem + 2 * t * c["heads"] * c["head_dim"] * act,
            "flops": 4 * pairs * c["heads"] * c["head_dim"]}


# ---------------------------------------------------------------------------------------
# the pages in plain torch
# ---------------------------------------------------------------------------------------
def _cell_bytes(c):
    n = c["page"] * c["head_dim"]
    return {"f16": 2 * n, "q8_0": n + n // 16, "q4_0": n // 2 + n // 16}[c["cache"]]


def _parts(pool, c, kind):
    """Views of one kind's codes and scales over all cells of a [pages][kv heads][cell] byte tensor:
    codes [.., block, position, 32 or 16] for K, [.., block, 32 or 16, position] for V."""
    nb, page, n = c["head_dim"] // 32, c["page"], c["page"] * c["head_dim"]
    inner = (nb, page, -1) if kind == 0 else (nb, -1, page)
    if c["cache"] == "f16":
        return pool.view(torch.float16).unflatten(-1, inner), None
    size = n if c["cache"] == "q8_0" else n // 2
    codes = pool.narrow(-1, 0, size)
    codes = codes.view(torch.int8) if c["cache"] == "q8_0" else codes
    return codes.unflatten(-1, inner), pool.narrow(-1, size, n // 16).view(torch.float16).unflatten(-1, (nb, page))


def _quantise(x, c):
    """x [.., 32] -> (codes [.., 32 or 16], scales [..]): the codes are the quotients by the half-precision
    scale rounded to even, taken in 64 bits."""
    if c["cache"] == "f16":
        return x.to(torch.float16), None
    x = x.float()
    if c["cache"] == "q8_0":
        d, lo, hi = x.abs().amax(-1) / torch.tensor(127.0, device=x.device), -127, 127
    else:
        first = x.abs().argmax(-1, keepdim=True)
        d, lo, hi = x.gather(-1, first).squeeze(-1) * -0.125, -8, 7
    d = d.to(torch.float16).clamp(-65504, 65504)
    q = torch.where(d[..., None] != 0, torch.round(x.double() / d.double()[..., None]).clamp(lo, hi), 0.0)
    if c["cache"] == "q8_0":
        return q.to(torch.int8), d
    q = (q + 8).to(torch.uint8)
    return q[..., :16] | (q[..., 16:] << 4), d


def _values(codes, d, c, dim):
    """Codes (their block of 32 or 16 along `dim`) and scales as float32 values, 32 along `dim`."""
    if c["cache"] == "f16":
        return codes.float()
    if c["cache"] == "q4_0":
        codes = torch.cat([codes & 15, codes >> 4], dim).to(torch.int8) - 8
    return codes.float() * d.float().unsqueeze(dim)


def _write(pool, c, layer, kind, page, off, x):
    """Rows x [token][kv head][head_dim] into positions (page, off)."""
    codes, scales = _parts(pool[layer, kind], c, kind)
    q, d = _quantise(x.unflatten(-1, (-1, 32)), c)  # [token][kv head][block][32 or 16]
    if kind == 0:
        codes[page, :, :, off, :] = q
    else:
        codes[page, :, :, :, off] = q
    if d is not None:
        scales[page, :, :, off] = d


def _rows(pool, c, layer, kind, page, off):
    """The rows at (page, off) as float32 [token][kv head * head_dim]."""
    codes, scales = _parts(pool[layer, kind], c, kind)
    q = codes[page, :, :, off, :] if kind == 0 else codes[page, :, :, :, off]
    return _values(q, None if scales is None else scales[page, :, :, off], c, -1).flatten(1)


def _pages(pool, c, layer, kind, table):
    """Whole pages of every sequence: [seq][kv head][position][head_dim] for K, [..][head_dim][position] for V."""
    codes, scales = _parts(pool[layer, kind], c, kind)
    dim = -1 if kind == 0 else -2
    x = _values(codes[table], None if scales is None else scales[table], c, dim)  # [seq][page][kv head][block]..
    if kind == 0:
        return x.permute(0, 2, 1, 4, 3, 5).flatten(2, 3).flatten(-2)
    return x.permute(0, 2, 3, 4, 1, 5).flatten(2, 3).flatten(-2)


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def prepare(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = _prepare_verify(c, gen) if c["op"] == "verify" else _prepare_cache(c, gen)
    if own:
        s["call"] = _Own(c, s)
    return s


def _prepare_verify(c, gen):
    b, n, v = c["seqs"], c["drafts"], c["vocab"]
    s = {"case": c}
    logits = 2.5 * _normal(gen, b, n + 1, v)
    s["target"] = torch.softmax(logits, -1)
    near = logits[:, :n] + 0.7 * _normal(gen, b, n, v)  # a smaller model's guess
    if c["greedy"]:  # the draft is the smaller model's best token: a distribution of one point
        s["draft"], s["tokens"] = None, near.argmax(-1).int()
    else:
        s["draft"] = torch.softmax(near, -1)
        cut = torch.rand(b, n, 1, device=DEV, generator=gen)
        s["tokens"] = (s["draft"].double().cumsum(-1) < cut).sum(-1).clamp(max=v - 1).int()
    s["counts"] = torch.randint(n if b == 1 else 0, n + 1, (b,), device=DEV, generator=gen, dtype=torch.int32)
    s["u_accept"] = torch.rand(b, n, device=DEV, generator=gen)
    s["u_sample"] = torch.rand(b, device=DEV, generator=gen)
    s["out_tokens"] = torch.empty(b, n + 1, device=DEV, dtype=torch.int32)
    s["out_counts"] = torch.empty(b, device=DEV, dtype=torch.int32)
    return s


def _prepare_cache(c, gen):
    new, old = _lengths(c)
    length = [n + o for n, o in zip(new, old)]
    page, nkv, hd = c["page"], c["kv_heads"], c["head_dim"]
    need = [-(-n // page) for n in length]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, device=DEV, generator=gen).int()
    wide = max(1, max(need))
    first = [sum(need[:i]) for i in range(len(need))]
    at = torch.arange(wide, device=DEV)[None, :]
    t = lambda v: torch.tensor(v, device=DEV)  # noqa: E731
    table = torch.where(at < t(need)[:, None], order[(t(first)[:, None] + at).clamp(max=n_pages - 1)], 0)
    pool = torch.zeros(2, 2, n_pages, nkv, _cell_bytes(c), device=DEV, dtype=torch.uint8)
    # a layer's keys have a few strong channels, its values do not; the first layer is another one's
    strong = torch.exp(0.5 * _normal(gen, nkv, 1, hd))
    for kind in (0, 1):
        codes, scales = _parts(pool[1, kind], c, kind)
        for lo in range(0, n_pages, 2048):
            n = min(2048, n_pages - lo)
            x = _normal(gen, n, nkv, page, hd) * (strong if kind == 0 else 0.5)
            q, d = _quantise(x.unflatten(-1, (-1, 32)), c)  # [page][kv head][position][block][32 or 16]
            codes[lo:lo + n] = q.permute(0, 1, 3, 2, 4) if kind == 0 else q.permute(0, 1, 3, 4, 2)
            if d is not None:
                scales[lo:lo + n] = d.transpose(-1, -2)
    tokens = sum(new)
    qkv = _normal(gen, tokens, (c["heads"] + 2 * nkv) * hd).to(ACT[c["act"]])
    s = {"case": c, "pool": pool, "n_pages": n_pages, "table": table.long(), "qkv": qkv, "new": new, "length": length}
    s["host_table"] = table.int().cpu().numpy()
    # where each new token and each cached position lies
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), t(new))
    start = t([sum(new[:i]) for i in range(len(new))])
    pos = torch.arange(tokens, device=DEV) - start[seq] + t(old)[seq]
    s["pos"], s["seq"], s["slot"] = pos, seq, torch.arange(tokens, device=DEV) - start[seq]
    if c["op"] == "append":
        s["page"], s["off"] = table[seq, pos // page].long(), pos % page
        s["out_k"] = torch.empty(tokens, nkv * hd, device=DEV)
        s["out_v"] = torch.empty(tokens, nkv * hd, device=DEV)
    elif c["op"] == "read":
        every = torch.repeat_interleave(torch.arange(len(new), device=DEV), t(length))
        p = torch.arange(sum(length), device=DEV) - t([sum(length[:i]) for i in range(len(new))])[every]
        s["page"], s["off"] = table[every, p // page].long(), p % page
        s["out_k"] = torch.empty(sum(length), nkv * hd, device=DEV, dtype=ACT[c["act"]])
        s["out_v"] = torch.empty_like(s["out_k"])
    else:
        s["out"] = torch.empty(tokens, c["heads"] * hd, device=DEV, dtype=ACT[c["act"]])
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(s):
    if own:
        return s["call"].run()
    c = s["case"]
    if c["op"] == "verify":
        return _plain_verify(s)
    if c["op"] == "attention":
        return _plain_attention(s)
    if c["op"] == "read":
        return {"k": _rows(s["pool"], c, 1, 0, s["page"], s["off"]).to(ACT[c["act"]]),
                "v": _rows(s["pool"], c, 1, 1, s["page"], s["off"]).to(ACT[c["act"]])}
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    k, v = s["qkv"][:, h * hd:(h + kv) * hd], s["qkv"][:, (h + kv) * hd:]
    _write(s["pool"], c, 1, 0, s["page"], s["off"], k.unflatten(-1, (kv, hd)))
    _write(s["pool"], c, 1, 1, s["page"], s["off"], v.unflatten(-1, (kv, hd)))
    return {"k": _rows(s["pool"], c, 1, 0, s["page"], s["off"]), "v": _rows(s["pool"], c, 1, 1, s["page"], s["off"])}


def _plain_attention(s):
    c = s["case"]
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    b, most = len(s["new"]), max(s["new"])
    q = torch.zeros(b, most, h * hd, device=DEV)
    q[s["seq"], s["slot"]] = s["qkv"][:, :h * hd].float()
    q = q.view(b, most, kv, h // kv, hd).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, hd)
    at = torch.full((b, most), -1, device=DEV)
    at[s["seq"], s["slot"]] = s["pos"]
    key = _pages(s["pool"], c, 1, 0, s["table"])
    x = (q @ key.transpose(-1, -2).contiguous()) * _scale(c)
    del key
    if c["softcap"] > 0:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    j = torch.arange(x.shape[-1], device=DEV)
    seen = (j <= at[..., None]) & (j > at[..., None] - c["window"])  # [seq][new][position]
    x = x.view(b, kv, most, h // kv, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    x = (x / x.sum(-1, keepdim=True).clamp(min=1e-30)).flatten(2, 3)
    val = _pages(s["pool"], c, 1, 1, s["table"]).transpose(-1, -2).contiguous()
    # behind a sequence's last position the pages hold whatever was there
    val = torch.where((j <= at.amax(-1, keepdim=True))[:, None, :, None], val, 0.0)
    o = (x @ val).view(b, kv, most, h // kv, hd).permute(0, 2, 1, 3, 4).reshape(b, most, h * hd)
    return o[s["seq"], s["slot"]].to(ACT[c["act"]])


def _plain_verify(s):
    b, n = s["tokens"].shape
    at, i, tok = torch.arange(b, device=DEV), torch.arange(n, device=DEV), s["tokens"].long()
    p = s["target"][at[:, None], i, tok].double()
    q = s["draft"][at[:, None], i, tok].double() if s["draft"] is not None else torch.ones_like(p)
    good = (s["u_accept"].double() * q < p) & (i < s["counts"][:, None])
    count = good.int().cumprod(-1).sum(-1)
    refused, last = count < s["counts"], count.clamp(max=n - 1)
    w = s["target"][at, count].double()
    if s["draft"] is not None:
        less = s["draft"][at, last].double()
    else:
        less = torch.zeros_like(w).scatter_(1, tok[at, last][:, None], 1.0)
    rest = (w - less * refused[:, None]).clamp(min=0)
    w = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    total = w.cumsum(-1)
    past = (total > s["u_sample"].double()[:, None] * total[:, -1:]) & (w > 0)
    token = past.int().argmax(-1).int()
    out = torch.where(i < count[:, None], s["tokens"], -1)
    out = torch.cat([out, torch.full_like(out[:, :1], -1)], 1)
    out[at, count] = token
    return {"tokens": out, "counts": count.int()}


def _scale(c):
    return 1.0 / math.sqrt(c["head_dim"])


class _Own:
    """What a program that uses the framework keeps: the context, the pages over its memory, the batch of
    its sequences, and the buffers that the calls read and write."""

    context = None

    def __init__(self, c, s):
        import dotnetfoundryllm_amd as F
        if _Own.context is None:
            _Own.context = F.Context(0)
        ctx, self.F, self.c, self.s = _Own.context, F, c, s
        torch.cuda.synchronize()
        buf = self.buf = lambda x: F.DeviceBuffer.wrap(ctx, x.data_ptr(), x.numel() * x.element_size())
        if c["op"] == "verify":
            self.given = dict(target=F.Rows(buf(s["target"]), c["vocab"]), tokens=buf(s["tokens"]),
                              counts=buf(s["counts"]), u_accept=buf(s["u_accept"]), u_sample=buf(s["u_sample"]),
                              out_tokens=buf(s["out_tokens"]), out_counts=buf(s["out_counts"]),
                              draft=None if s["draft"] is None else F.Rows(buf(s["draft"]), c["vocab"]))
            return
        kind = {"f16": F.F16, "q8_0": F.Q8_0, "q4_0": F.Q4_0}[c["cache"]]
        act = {"f32": F.F32, "f16": F.F16, "bf16": F.BF16}[c["act"]]
        h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
        self.pages = F.PagedKvCache(ctx, kind, 2, kv, hd, c["page"], s["n_pages"], memory=buf(s["pool"]))
        self.batch = self.pages.batch(h, c["window"])
        self.batch.set(s["new"], s["length"], s["host_table"])
        qkv, ld, size = buf(s["qkv"]), (h + 2 * kv) * hd, s["qkv"].element_size()
        self.q = F.Rows(qkv, ld, act)
        self.k = F.Rows(qkv, ld, act, h * hd * size)
        self.v = F.Rows(qkv, ld, act, (h + kv) * hd * size)
        if c["op"] == "attention":
            self.out = F.Rows(buf(s["out"]), h * hd, act)
        else:
            to = act if c["op"] == "read" else F.F32
            self.out_k, self.out_v = F.Rows(buf(s["out_k"]), kv * hd, to), F.Rows(buf(s["out_v"]), kv * hd, to)

    def run(self):
        c, s = self.c, self.s
        if c["op"] == "verify":
            self.F.draft_verify(_Own.context, c["seqs"], c["drafts"], c["vocab"], **self.given)
            return {"tokens": s["out_tokens"], "counts": s["out_counts"]}
        if c["op"] == "attention":
            self.batch.attention(1, self.q, self.out, _scale(c), c["softcap"])
            return s["out"]
        if c["op"] == "append":
            self.batch.append(1, self.k, self.v)
        self.batch.read(1, self.out_k, self.out_v, new_only=c["op"] == "append")
        return {"k": s["out_k"], "v": s["out_v"]}

    def __del__(self):
        if hasattr(self, "batch"):
            self.batch.close()
            self.pages.close()


# ---------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------
def _exact_block(raw, scale, cache):
    """One block's 32 values in 64 bits from its raw bytes [.., 32 or 16] and scale [..]."""
    if cache == "q8_0":
        return raw.view(torch.int8).double() * scale.double()[..., None]
    low, high = torch.bitwise_and(raw, 15).double(), torch.div(raw, 16, rounding_mode="floor").double()
    return (torch.cat((low, high), -1) - 8.0) * scale.double()[..., None]


def _exact_kv(s, kind, i):
    """Every cached row of sequence i: [kv head][position][head_dim] in 64 bits, read cell by cell."""
    c, size = s["case"], s["length"][i]
    nb, page, cache = c["head_dim"] // 32, c["page"], c["cache"]
    cells = s["pool"][1, kind][s["table"][i][: -(-size // page)]]  # [page][kv head][bytes]
    n, nkv, _ = cells.shape
    if cache == "f16":
        x = cells.contiguous().view(torch.float16).double()
        x = x.reshape(n, nkv, nb, page, 32) if kind == 0 else x.reshape(n, nkv, nb, 32, page).transpose(-1, -2)
    else:
        per = 32 if cache == "q8_0" else 16
        raw = cells[..., : nb * page * per].contiguous()
        raw = raw.reshape(n, nkv, nb, page, per) if kind == 0 else raw.reshape(n, nkv, nb, per, page).transpose(-1, -2)
        scale = cells[..., nb * page * per:].contiguous().view(torch.float16).reshape(n, nkv, nb, page)
        x = _exact_block(raw.contiguous(), scale, cache)
    return x.permute(1, 0, 3, 2, 4).reshape(nkv, n * page, nb * 32)[:, :size]


def _exact_stored(x, cache):
    """The values that a cache of this type holds of x [.., 32]."""
    x = x.double()
    if cache == "f16":
        return x.float().to(torch.float16).double()
    if cache == "q8_0":
        step = (x.abs().max(-1).values / 127).float().half().double()[..., None]
        code = (x / step).round().clamp(-127, 127)
    else:
        most, least = x.max(-1).values, x.min(-1).values
        even = most == -least
        lead = torch.where(most > -least, most, least)
        up, down = (x == most[..., None]).int().argmax(-1), (x == least[..., None]).int().argmax(-1)
        lead = torch.where(even & (up < down), most, lead)
        step = (lead.float() / -8).half().double()[..., None]
        code = (x / step).round().clamp(-8, 7)
    return torch.where(step == 0, 0.0, code * step)


def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["op"] == "verify":
        return _exact_verify(s)
    if c["op"] == "append":
        h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
        at = {"k": h * hd, "v": (h + kv) * hd}
        return {k: _exact_stored(s["qkv"][:, lo:lo + kv * hd].unflatten(-1, (-1, 32)), c["cache"]).flatten(1)
                for k, lo in at.items()}
    if c["op"] == "read":
        return {k: torch.cat([_exact_kv(s, kind, i).transpose(0, 1).flatten(1) for i in range(c["seqs"])])
                for k, kind in (("k", 0), ("v", 1))}
    out, row, hd, group = [], 0, c["head_dim"], c["heads"] // c["kv_heads"]
    for i, (n, size) in enumerate(zip(s["new"], s["length"])):
        if n == 0:
            continue
        key, val = _exact_kv(s, 0, i), _exact_kv(s, 1, i)
        q = s["qkv"][row:row + n, : c["heads"] * hd].double().view(n, c["heads"], hd)
        p, j = torch.arange(size - n, size, device=DEV)[:, None], torch.arange(size, device=DEV)[None]
        hide = (j > p) | (p - j >= c["window"])
        o = torch.empty(n, c["heads"], hd, device=DEV, dtype=torch.float64)
        for a in range(c["heads"]):
            x = torch.mm(q[:, a], key[a // group].t().contiguous()) / math.sqrt(hd)
            if c["softcap"] > 0:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            x = torch.softmax(x.masked_fill(hide, -math.inf), -1)
            o[:, a] = torch.mm(x, val[a // group])
        out.append(o.flatten(1))
        row += n
    return torch.cat(out)


def _exact_verify(s):
    b, n = s["tokens"].shape
    out, counts = torch.full((b, n + 1), -1, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        k, most = 0, int(s["counts"][i])
        target, tokens, ua = s["target"][i].double(), s["tokens"][i].tolist(), s["u_accept"][i].tolist()
        given = None if s["draft"] is None else s["draft"][i].double()
        while k < most:
            qx = 1.0 if given is None else float(given[k, tokens[k]])
            if not ua[k] * qx < float(target[k, tokens[k]]):
                break
            out[i, k] = tokens[k]
            k += 1
        w = target[k].clone()
        if k < most:
            if given is None:
                w[tokens[k]] = 0 if w[tokens[k]] <= 1 else w[tokens[k]] - 1
            else:
                w = torch.relu(w - given[k])
            if float(w.sum()) == 0:
                w = target[k]
        run_sum = torch.cumsum(w, 0)
        out[i, k] = int(torch.nonzero((run_sum > float(s["u_sample"][i]) * run_sum[-1]) & (w > 0))[0, 0])
        counts[i] = k
    return {"tokens": out, "counts": counts}
