"""Cases for timing the operators of the 4-bit paged KV cache, with their plain forms.

A cache is a uint8 tensor ``[pages, kv_heads, page_size, head_dim / 2 + 8]``. Sixteen tokens of one page and head are a
unit: 16 rows of codes (two channels a byte, the even one in the low bits), then 16 rows of parameters (bf16
``s0, c0, s1, c1``). Channels come in words of eight; even words form group 0, odd words group 1, and a value is
``c + s * (code - 8)`` with its group's pair.

``append``  QK norm, rotary embedding and the quantising write of one step's tokens, then the values read back
``read``    the values of cached tokens, as bf16
``attend``  causal attention of packed query rows (single tokens first, then chunks) over the paged cache
"""
import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
D = 128              # head_dim of every architecture that the GPU kernels run
ROW = D // 2 + 8     # bytes of one token and head
EPS = 1e-6
THETA = 1e6
SCALE = D ** -0.5


# ---- cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 32 running sequences, 32 query / 8 KV heads: latency
        {"name": "append 32 decode rows", "kind": "append", "tokens": 32, "hq": 32, "hkv": 8, "page": 16, "skip": 0},
        # a prompt step of ragged length whose last rows are padding (slot -1), group of 5, pages of 48
        {"name": "append 997 ragged", "kind": "append", "tokens": 997, "hq": 40, "hkv": 8, "page": 48, "skip": 21},
        # a full prompt step: max_num_batched_tokens of the default configuration
        {"name": "append 8192 prompt rows", "kind": "append", "tokens": 8192, "hq": 32, "hkv": 8, "page": 16, "skip": 0},
        # one prompt's cached values on a rank that holds a single KV head
        {"name": "read 777 one head", "kind": "read", "tokens": 777, "hkv": 1, "page": 16},
        # a long shared prefix read back whole
        {"name": "read 32768", "kind": "read", "tokens": 32768, "hkv": 8, "page": 16},
        # the first tokens of one short request: nothing but latency
        {"name": "decode 1 x 17", "kind": "attend", "hq": 16, "hkv": 8, "page": 16, "decodes": 1, "lo": 17, "hi": 17,
         "chunks": 0, "chunk": 0, "prefix": 0},
        # an ordinary decode step: 32 sequences of 128 to 1280 tokens
        {"name": "decode 32 x 128-1280", "kind": "attend", "hq": 16, "hkv": 8, "page": 16, "decodes": 32, "lo": 128,
         "hi": 1280, "chunks": 0, "chunk": 0, "prefix": 0},
        # group of 5, pages of 48, empty rows among the sequences (a padded step)
        {"name": "decode 9 odd", "kind": "attend", "hq": 40, "hkv": 8, "page": 48, "decodes": 9, "lo": 0, "hi": 3001,
         "chunks": 0, "chunk": 0, "prefix": 0},
        # one request at the end of the longest context, 64 query heads
        {"name": "decode 1 x 40960", "kind": "attend", "hq": 64, "hkv": 8, "page": 16, "decodes": 1, "lo": 40960,
         "hi": 40960, "chunks": 0, "chunk": 0, "prefix": 0},
        # a full decode step: 256 sequences anywhere in the default context
        {"name": "decode 256 x 256-4096", "kind": "attend", "hq": 32, "hkv": 8, "page": 16, "decodes": 256, "lo": 256,
         "hi": 4096, "chunks": 0, "chunk": 0, "prefix": 0},
        # running sequences next to short last chunks of long prompts
        {"name": "mixed 8 + 3 x 61", "kind": "attend", "hq": 32, "hkv": 8, "page": 16, "decodes": 8, "lo": 100,
         "hi": 2000, "chunks": 3, "chunk": 61, "prefix": 1536},
        # a full prompt step: four chunks of 2048 rows behind a cached prefix
        {"name": "prompt 4 x 2048", "kind": "attend", "hq": 32, "hkv": 8, "page": 16, "decodes": 0, "lo": 0, "hi": 0,
         "chunks": 4, "chunk": 2048, "prefix": 512},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    kind = rng.choice(["append", "read", "decode", "decode", "chunks", "mixed"])
    if kind == "append":
        t = _log(rng, 1, 6000)
        return {"kind": "append", "tokens": t, "hq": hq, "hkv": hkv, "page": page, "skip": rng.choice([0, t // 3])}
    if kind == "read":
        return {"kind": "read", "tokens": _log(rng, 1, 32000), "hkv": hkv, "page": page}
    c = {"kind": "attend", "hq": hq, "hkv": hkv, "page": page, "decodes": 0, "lo": 0, "hi": 0, "chunks": 0, "chunk": 0,
         "prefix": 0}
    if kind != "chunks":
        n = _log(rng, 1, 200)
        hi = _log(rng, 1, min(40960, max(4, 400000 // n)))
        c.update(decodes=n, lo=rng.randint(0 if n > 3 else 1, hi), hi=hi)
    if kind != "decode":
        n = rng.randint(1, 4)
        chunk, prefix = _log(rng, 2, 2000 if kind == "chunks" else 300), rng.choice([0, _log(rng, 1, 2000)])
        while n * chunk * (chunk + prefix) * hq > 4 * 2048 * 2560 * 32:      # no more than the largest listed
            chunk, prefix = chunk // 2, prefix // 2
        c.update(chunks=n, chunk=chunk, prefix=prefix)
        if kind == "mixed":     # the plain form pads every sequence to the longest chunk
            c.update(decodes=min(c["decodes"], 16), hi=min(c["hi"], 4000), lo=min(c["lo"], c["hi"], 4000))
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------
def _groups(x):
    """``[..., D]`` as ``[..., 2, D / 2]``: the channels of even words, then those of odd words."""
    return x.unflatten(-1, (D // 16, 2, 8)).transpose(-2, -3).flatten(-2)


def _ungroup(x):
    return x.unflatten(-1, (D // 16, 8)).transpose(-2, -3).flatten(-3)


def _quantise(x):
    """Codes ``[..., D]`` (int32) and parameters ``s, c`` (``[..., 2]`` bf16) of bf16 values ``[..., D]``."""
    g = _groups(x.float())
    hi, lo = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    s = ((0.5 * hi - 0.5 * lo) / 7.5).bfloat16().float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    c = (0.5 * hi + 0.5 * lo + 0.5 * s).bfloat16().float()
    n = torch.where(s > 0, torch.round((g - c) / s) + 8, 8.0).clamp(0, 15).to(torch.int32)
    return _ungroup(n), s.squeeze(-1).bfloat16(), c.squeeze(-1).bfloat16()


def _value(n, s, c):
    """fp32 values of codes ``[..., D]`` under ``s, c`` ``[..., 2]``."""
    return _ungroup(c.float().unsqueeze(-1) + s.float().unsqueeze(-1) * (_groups(n).float() - 8))


def _pack(n, s, c):
    """Rows of codes and parameters ``[pages, heads, page, ...]`` as cache bytes."""
    p, h, bs, _ = n.shape
    n = n.to(torch.uint8).view(p, h, bs // 16, 16, D // 2, 2)
    codes = (n[..., 0] | (n[..., 1] << 4)).flatten(-2)
    pars = torch.stack([s, c], -1).contiguous().view(torch.uint8).view(p, h, bs // 16, 16 * 8)
    return torch.cat([codes, pars], -1).view(p, h, bs, ROW)


def _unpack(cache):
    """Codes ``[pages, heads, page, D]`` and parameters of cache bytes."""
    p, h, bs, _ = cache.shape
    u = cache.reshape(p, h, bs // 16, 16 * ROW)
    b = u[..., :8 * D].reshape(p, h, bs, D // 2)
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    sc = u[..., 8 * D:].contiguous().view(torch.bfloat16).view(p, h, bs, 2, 2)
    return n, sc[..., 0], sc[..., 1]


def _cache(pages, hkv, page, gen):
    """A cache as a model leaves it: values near a normal distribution, a few channels larger than the rest."""
    out = torch.empty(pages, hkv, page, ROW, dtype=torch.uint8, device=DEV)
    gain = torch.exp(0.3 * torch.randn(hkv, 1, D, device=DEV, generator=gen))
    step = max(1, (1 << 26) // (hkv * page * D))
    for p in range(0, pages, step):
        m = min(step, pages - p)
        x = torch.randn(m, hkv, page, D, device=DEV, generator=gen) * gain
        out[p:p + m] = _pack(*_quantise(x.bfloat16()))
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    hkv, page = case["hkv"], case["page"]
    st = {"case": case}
    if case["kind"] in ("append", "read"):
        t = case["tokens"]
        pages = -(-t // page) + 3
        order = torch.randperm(pages, device=DEV, generator=gen)[: -(-t // page)]
        st["slots"] = (order[:, None] * page + torch.arange(page, device=DEV)).flatten()[:t].to(torch.int32)
    if case["kind"] == "read":
        st["k"], st["v"] = _cache(pages, hkv, page, gen), _cache(pages, hkv, page, gen)
        return st
    hq = case["hq"]
    if case["kind"] == "append":
        if case["skip"]:
            st["slots"][t - case["skip"]:] = -1
        st["k"] = torch.zeros(pages, hkv, page, ROW, dtype=torch.uint8, device=DEV)
        st["v"] = torch.zeros_like(st["k"])
        st["qkv"] = torch.randn(t, (hq + 2 * hkv) * D, device=DEV, generator=gen).bfloat16()
        st["qw"] = torch.exp(0.1 * torch.randn(D, device=DEV, generator=gen)).bfloat16()
        st["kw"] = torch.exp(0.1 * torch.randn(D, device=DEV, generator=gen)).bfloat16()
        st["pos"] = torch.arange(t, device=DEV, dtype=torch.int32) + int(torch.randint(0, 1000, (1,), device=DEV, generator=gen))
        ang = torch.arange(t + 1000, device=DEV, dtype=torch.float64)[:, None] * THETA ** (
            -torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        st["cs"] = torch.cat([ang.cos(), ang.sin()], -1).float()
        return st
    lens = torch.randint(case["lo"], case["hi"] + 1, (case["decodes"],), device=DEV, generator=gen).tolist()
    q_lens = [1] * len(lens)
    for i in range(case["chunks"]):          # ragged: every chunk a little shorter than the one before
        n = max(1, case["chunk"] - 3 * i)
        q_lens.append(n)
        lens.append(case["prefix"] + n)
    per = max(1, max(-(-n // page) for n in lens))
    pages = sum(-(-n // page) for n in lens) + 3
    order = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.zeros(len(lens), per, dtype=torch.int32)
    at, order_h = 0, order.cpu()
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = order_h[at:at + m]
        at += m
    cu = torch.tensor([0] + q_lens).cumsum(0)
    st.update(table=table.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV), cu=cu.to(torch.int32).to(DEV),
              max_q=max(q_lens), max_kv=max(lens), rows=int(cu[-1]))
    st["k"], st["v"] = _cache(pages, hkv, page, gen), _cache(pages, hkv, page, gen)
    st["q"] = (1.5 * torch.randn(st["rows"], hq * D, device=DEV, generator=gen)).bfloat16()
    # what the engine's stager hands to attention for a packed step
    st["attn"] = SimpleNamespace(cu_q=st["cu"], kv_lens=st["lens"], block_tables=st["table"], num_seqs=len(lens),
                                 num_decode=case["decodes"], max_q_len=st["max_q"], max_kv_len=st["max_kv"],
                                 num_tokens=st["rows"], cu_q_host=None, kv_lens_host=None)
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------
def _append_plain(st):
    case = st["case"]
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    t = case["tokens"]
    x = st["qkv"].view(t, hq + 2 * hkv, D)
    cs = st["cs"][st["pos"].long()]

    def normed(h, w, dt):
        h = h.to(dt)
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.to(dt)
        a, b = h.chunk(2, -1)
        cos, sin = cs[:, None].to(dt).chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float().bfloat16()

    q = normed(x[:, :hq], st["qw"], torch.float32).view(t, hq * D)
    # a code is a choice between two levels: K is taken to 64 bits so that values next to a border fall alike
    k, v = normed(x[:, hq:hq + hkv], st["kw"], torch.float64), x[:, hq + hkv:]
    keep = st["slots"] >= 0
    p, r = st["slots"][keep].long() // page, st["slots"][keep].long() % page
    vals = []
    for cache, new in ((st["k"], k), (st["v"], v)):
        n, s, c = _quantise(new[keep])
        rows = cache.view(cache.shape[0], hkv, page // 16, 16 * ROW)
        codes = (n[..., 0::2] | (n[..., 1::2] << 4)).to(torch.uint8)
        pars = torch.stack([s, c], -1).view(torch.uint8).view(-1, hkv, 8)
        base = (r % 16)[:, None, None]
        h = torch.arange(hkv, device=DEV)[None, :, None]
        rows[p[:, None, None], h, (r // 16)[:, None, None], base * (D // 2) + torch.arange(D // 2, device=DEV)] = codes
        rows[p[:, None, None], h, (r // 16)[:, None, None], 8 * D + base * 8 + torch.arange(8, device=DEV)] = pars
        vals.append(_rows_plain(cache, st["slots"]))
    return q, vals[0], vals[1]


def _rows_plain(cache, slots):
    pages, hkv, page, _ = cache.shape
    s = slots.clamp_min(0).long()
    p, r = s // page, s % page
    u = cache.view(pages, hkv, page // 16, 16 * ROW)[p, :, r // 16]                     # [T, hkv, unit]
    i = (r % 16)[:, None, None]
    b = u.gather(-1, (i * (D // 2) + torch.arange(D // 2, device=DEV)).expand(-1, hkv, -1))
    sc = u.gather(-1, (8 * D + i * 8 + torch.arange(8, device=DEV)).expand(-1, hkv, -1)).view(torch.bfloat16)
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    x = _value(n, sc[..., 0::2], sc[..., 1::2])
    return torch.where((slots >= 0)[:, None, None], x, torch.zeros_like(x)).bfloat16()


def _attend_plain(st):
    case = st["case"]
    hq, hkv = case["hq"], case["hkv"]
    g = hq // hkv
    B, L = st["table"].shape[0], st["table"].shape[1] * case["page"]
    lens, cu, mq = st["lens"].long(), st["cu"].long(), st["max_q"]

    def seqs(cache):
        n, s, c = _unpack(cache[st["table"].long().flatten()])
        return _value(n, s, c).view(B, -1, hkv, case["page"], D).transpose(1, 2).reshape(B, hkv, L, D)

    k, v = seqs(st["k"]), seqs(st["v"])
    q_len = cu[1:] - cu[:-1]
    i = torch.arange(mq, device=DEV)
    real = i < q_len[:, None]
    row = torch.where(real, cu[:-1, None] + i, 0)                                          # [B, mq]
    q = st["q"][row].float().view(B, mq, hkv, g, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, g * mq, D)
    s = (q @ k.transpose(-1, -2)).mul_(SCALE).view(B, hkv, g, mq, L)
    t = torch.arange(L, device=DEV)
    seen = t <= (lens[:, None] - q_len[:, None] + i)[..., None]                            # causal, last q_len positions
    seen &= (t < lens[:, None])[:, None]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    z = s.sum(-1, keepdim=True)
    o = (s.view(B, hkv, g * mq, L) @ v).view(B, hkv, g, mq, D) / torch.where(z > 0, z, torch.ones_like(z))
    o = o.permute(0, 3, 1, 2, 4).reshape(B, mq, hq * D).bfloat16()
    return o[real]


def run(st):
    case = st["case"]
    if own:
        from xixi_vllm_b200.ops import dispatch as ops
        if case["kind"] == "append":
            q = ops.qk_norm_rope_cache(st["qkv"], st["qw"], st["kw"], EPS, st["cs"], st["pos"], st["slots"], st["k"],
                                       st["v"], case["hq"], case["hkv"], D)
            return (q, *ops.read_cache(st["k"], st["v"], st["slots"], D))
        if case["kind"] == "read":
            return ops.read_cache(st["k"], st["v"], st["slots"], D)
        return ops.paged_attention(st["q"], st["k"], st["v"], st["attn"], SCALE, case["hq"], case["hkv"], D)
    if case["kind"] == "append":
        return _append_plain(st)
    if case["kind"] == "read":
        return _rows_plain(st["k"], st["slots"]), _rows_plain(st["v"], st["slots"])
    return _attend_plain(st)


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def _mean_len(case):
    return (case["lo"] + case["hi"]) / 2


def work(case):
    hkv = case["hkv"]
    if case["kind"] == "read":
        return {"bytes": case["tokens"] * hkv * 2 * (ROW + 2 * D), "flops": case["tokens"] * hkv * 2 * D * 2}
    hq = case["hq"]
    if case["kind"] == "append":
        t = case["tokens"]
        return {"bytes": t * ((hq + 2 * hkv) * 2 * D + hq * 2 * D + hkv * 2 * (ROW + 2 * D)),
                "flops": t * (hq + 2 * hkv) * D * 10}
    tokens, pairs, rows = case["decodes"] * _mean_len(case), case["decodes"] * _mean_len(case), case["decodes"]
    for i in range(case["chunks"]):
        n = max(1, case["chunk"] - 3 * i)
        tokens += case["prefix"] + n
        pairs += n * case["prefix"] + n * (n + 1) / 2
        rows += n
    return {"bytes": tokens * hkv * 2 * ROW + rows * hq * D * 4, "flops": 4 * pairs * hq * D}


# ---- from the definition, in 64 bits ----------------------------------------------------------------------------
def _decode64(cache):
    """Every value of a cache ``[pages, heads, page, D]`` in 64 bits, byte by byte from the layout."""
    pages, hkv, page, _ = cache.shape
    out = torch.empty(pages, hkv, page, D, dtype=torch.float64, device=cache.device)
    flat = cache.reshape(pages, hkv, page * ROW)
    for i in range(page):
        base = (i // 16) * 16 * ROW
        byte = flat[..., base + (i % 16) * (D // 2):][..., :D // 2].long()
        par = flat[..., base + 8 * D + (i % 16) * 8:][..., :8].contiguous().view(torch.bfloat16).double()
        for ch in range(16):                        # channel ch of every run of 16 channels: word parity ch // 8
            code = (byte[..., ch // 2::8] >> (4 * (ch % 2))) % 16
            s, c = par[..., 2 * (ch // 8)], par[..., 2 * (ch // 8) + 1]
            out[:, :, i, ch::16] = c[..., None] + s[..., None] * (code - 8)
    return out


def _levels64(x):
    """What the 4-bit form of bf16 values stands for, in 64 bits."""
    x = x.double()
    out = torch.empty_like(x)
    for par in (0, 1):
        ch = [c for c in range(D) if (c // 8) % 2 == par]
        g = x[..., ch]
        top, low = g.max(-1, keepdim=True).values, g.min(-1, keepdim=True).values
        s = ((top - low) / 15).bfloat16().double()
        c = ((top + low + s) / 2).bfloat16().double()
        n = torch.where(s > 0, torch.round((g - c) / torch.where(s > 0, s, 1.0)).clamp(-8, 7), 0.0)
        out[..., ch] = c + s * n
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "read":
        page = case["page"]
        s = st["slots"].long()
        return tuple(_decode64(st[n])[s // page, :, s % page] for n in ("k", "v"))
    hq, hkv = case["hq"], case["hkv"]
    if case["kind"] == "append":
        t = case["tokens"]
        x = st["qkv"].double().view(t, hq + 2 * hkv, D)
        ang = st["cs"].double()[st["pos"].long()]
        half = D // 2

        def rotated(h, w):
            h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / D + EPS) * w.double()
            z = torch.complex(h[..., :half], h[..., half:]) * torch.complex(ang[:, None, :half], ang[:, None, half:])
            return torch.cat([z.real, z.imag], -1)

        live = (st["slots"] >= 0).double()[:, None, None]
        k = _levels64(rotated(x[:, hq:hq + hkv], st["kw"]).bfloat16()) * live
        v = _levels64(x[:, hq + hkv:].bfloat16()) * live
        return rotated(x[:, :hq], st["qw"]).reshape(t, hq * D), k, v
    out = torch.zeros(st["rows"], hq, D, dtype=torch.float64, device=DEV)
    cu, lens = st["cu"].tolist(), st["lens"].tolist()
    g = hq // hkv
    for b, n in enumerate(lens):
        if n == 0:
            continue
        used = st["table"][b, :-(-n // case["page"])].long()
        k, v = (_decode64(st[c][used]).transpose(0, 1).reshape(hkv, -1, D)[:, :n] for c in ("k", "v"))
        q = st["q"][cu[b]:cu[b + 1]].double().view(-1, hq, D)
        hide = torch.ones(q.shape[0], n, dtype=torch.bool, device=DEV).triu(n - q.shape[0] + 1)
        for h in range(hq):
            s = (q[:, h] @ k[h // g].T / math.sqrt(D)).masked_fill(hide, -math.inf)
            out[cu[b]:cu[b + 1], h] = torch.softmax(s, -1) @ v[h // g]
    return out.view(st["rows"], hq * D)
