"""A 4-bit KV cache from its definition, in 64 bits and apart from the package's own code (numpy, byte by byte)."""
import numpy as np
import torch


def to_bf16(x):
    """fp64 array -> nearest bf16 values, as fp64 (through fp32, as every producer does)."""
    return torch.from_numpy(np.asarray(x, dtype=np.float64)).float().bfloat16().double().numpy()


def levels(x):
    """What the 4-bit form of bf16 values ``x [..., D]`` stands for; a group is the channels with equal word parity."""
    x = np.asarray(x, dtype=np.float64)
    out = np.empty_like(x)
    parity = (np.arange(x.shape[-1]) // 8) % 2
    for g in (0, 1):
        v = x[..., parity == g]
        hi, lo = v.max(-1, keepdims=True), v.min(-1, keepdims=True)
        s = to_bf16((hi / 2 - lo / 2) / 7.5)
        s = np.where(s < 2.0 ** -126, 0.0, s)
        c = to_bf16(hi / 2 + lo / 2 + s / 2)
        with np.errstate(invalid="ignore", divide="ignore"):
            n = np.where(s > 0, np.clip(np.rint((v - c) / np.where(s > 0, s, 1.0)), -8, 7), 0.0)
        out[..., parity == g] = c + s * n
    return out


def parts(cache, page, head, r):
    """(codes [D] int, s [D], c [D]) of row ``r`` of a page of a uint8 cache tensor."""
    row = cache.shape[3]
    d = (row - 8) * 2
    unit = cache[page, head].reshape(-1)[(r // 16) * 16 * row:][:16 * row].cpu().numpy()
    i = r % 16
    code_bytes = unit[i * (d // 2):(i + 1) * (d // 2)]
    par = torch.from_numpy(unit[16 * (d // 2) + 8 * i:][:8].copy()).view(torch.bfloat16).double().numpy()
    codes = np.empty(d, dtype=np.int64)
    codes[0::2], codes[1::2] = code_bytes & 15, code_bytes >> 4
    g = (np.arange(d) // 8) % 2
    return codes, par[2 * g], par[2 * g + 1]


def rows(cache, slots):
    """Values ``[T, heads, D]`` at ``slots`` (negative: zeros), and the same without the centres (``s (n - 8)``)."""
    nb, heads, bs, row = cache.shape
    cache = cache.cpu()
    vals = np.zeros((len(slots), heads, (row - 8) * 2))
    swing = np.zeros_like(vals)
    for i, s in enumerate(slots):
        if s >= 0:
            for h in range(heads):
                n, sc, c = parts(cache, s // bs, h, s % bs)
                swing[i, h] = sc * (n - 8)
                vals[i, h] = c + swing[i, h]
    return vals, swing


def attention(q, k_cache, v_cache, q_lens, kv_lens, tables, scale, hq):
    """Causal attention in fp64. Returns per packed query row: the output ``[T, hq, D]``, ``sum p |v|``,
    ``sum p |s (n - 8)|`` of V and ``max_j scale * sum |q| |k_j|`` ``[T, hq]``, from which tests bound rounding."""
    _, hkv, bs, row = k_cache.shape
    d = (row - 8) * 2
    q = q.double().cpu().numpy().reshape(-1, hq, d)
    out, mag, swing = (np.zeros(q.shape) for _ in range(3))
    qk = np.zeros(q.shape[:2])
    at = 0
    for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
        if L > 0:
            slots = [int(tables[b, t // bs]) * bs + t % bs for t in range(L)]
            k, _ = rows(k_cache, slots)
            v, vs = rows(v_cache, slots)
            for i in range(n):
                seen = min(L, L - n + i + 1)
                if seen <= 0:
                    continue
                for h in range(hq):
                    hk = h // (hq // hkv)
                    s = scale * (k[:seen, hk] @ q[at + i, h])
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[at + i, h] = p @ v[:seen, hk]
                    mag[at + i, h] = p @ np.abs(v[:seen, hk])
                    swing[at + i, h] = p @ np.abs(vs[:seen, hk])
                    qk[at + i, h] = scale * (np.abs(k[:seen, hk]) @ np.abs(q[at + i, h])).max()
        at += n
    return out, mag, swing, qk
