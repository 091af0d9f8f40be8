"""Kernels of the 4-bit KV cache against plain implementations in 64 bits."""
import numpy as np
import pytest
import torch

import kv4_ref
from xixi_vllm_b200.ops import cpu_ref, kv4
from xixi_vllm_b200.runtime.staging import AttnBatch

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128
HALF_BF16 = 2.0 ** -8          # largest relative error of one rounding to bf16


def _ops():
    from xixi_vllm_b200.ops import dispatch
    return dispatch


def _cuda():
    from xixi_vllm_b200.ops import cuda
    return cuda


def _empty(nb, hkv, bs):
    return [torch.zeros(nb, hkv, bs, kv4.row_bytes(D), dtype=torch.uint8, device=DEV) for _ in range(2)]


def _random(nb, hkv, bs, seed, scale=1.0):
    """A cache whose every row holds quantised normal values (made on the CPU by the oracle)."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        c = torch.zeros(nb, hkv, bs, kv4.row_bytes(D), dtype=torch.uint8)
        kv4.write_rows(c, torch.arange(nb * bs), torch.randn(nb * bs, hkv, D, generator=g) * scale)
        out.append(c.to(DEV))
    return out


# ---- writing and reading ----

def _write_case(T, hq, hkv, bs, seed, skip=(), parts=0):
    g = torch.Generator().manual_seed(seed)
    nb = -(-T // bs) + 2
    qkv = (torch.randn(T, (hq + 2 * hkv) * D, generator=g) * torch.exp(torch.randn(1, (hq + 2 * hkv) * D, generator=g))).bfloat16()
    qw, kw = (torch.exp(0.3 * torch.randn(D, generator=g)).bfloat16() for _ in range(2))
    cs = cpu_ref.build_cos_sin_cache(D, 5000, 1e6)
    pos = torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32)
    slots = torch.randperm(nb * bs, generator=g)[:T].to(torch.int32)
    for i in skip:
        slots[i] = -1
    return nb, qkv, qw, kw, cs, pos, slots


def _rotated(x, w, cs, pos, eps):
    x = x.double().numpy()
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.double().numpy()
    a, b = x[..., :D // 2], x[..., D // 2:]
    c, s = np.split(cs[pos.long()].double().numpy()[:, None], 2, -1)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("T,hq,hkv,bs,skip", [(1, 16, 8, 16, ()), (2, 3, 1, 16, (0,)), (33, 32, 8, 48, (0, 5, 32)),
                                              (130, 40, 8, 128, ()), (7, 0, 2, 16, ())])
def test_write_then_read(T, hq, hkv, bs, skip):
    nb, qkv, qw, kw, cs, pos, slots = _write_case(T, hq, hkv, bs, T, skip)
    k, v = _empty(nb, hkv, bs)
    q = _ops().qk_norm_rope_cache(qkv.to(DEV), qw.to(DEV), kw.to(DEV), 1e-6, cs.to(DEV), pos.to(DEV), slots.to(DEV), k, v,
                                  hq, hkv, D)
    _cuda().check_status()
    x = qkv.view(T, hq + 2 * hkv, D)
    live = np.array([s >= 0 for s in slots.tolist()])
    # V: the kernel and the definition do the same exact or correctly rounded steps, so the levels are equal
    want_v = kv4_ref.levels(x[:, hq + hkv:].double().numpy()) * live[:, None, None]
    got_v, _ = kv4_ref.rows(v, slots.tolist())
    np.testing.assert_allclose(got_v, want_v, rtol=1e-12)
    # K: 64-bit norm and rotation, rounded to fp32 and bf16 alike
    want_k = kv4_ref.levels(kv4_ref.to_bf16(_rotated(x[:, hq:hq + hkv], kw, cs, pos, 1e-6))) * live[:, None, None]
    got_k, _ = kv4_ref.rows(k, slots.tolist())
    np.testing.assert_allclose(got_k, want_k, rtol=1e-12)
    # q: fp32 (a dozen roundings of 2^-24 on terms no larger than the pair's norm), then one rounding to bf16
    if hq:
        want_q = _rotated(x[:, :hq], qw, cs, pos, 1e-6)
        norm = np.sqrt(want_q ** 2 + np.roll(want_q, D // 2, -1) ** 2)
        assert (np.abs(q.double().cpu().numpy().reshape(T, hq, D) - want_q) <= HALF_BF16 * np.abs(want_q) + 2.0 ** -19 * norm + 1e-30).all()
    kk, vv = _ops().read_cache(k, v, slots.to(DEV), D)
    _cuda().check_status()
    for got, want in ((kk, got_k), (vv, got_v)):
        assert got.shape == (T, hkv, D)
        assert (np.abs(got.double().cpu().numpy() - want) <= HALF_BF16 * np.abs(want) * (1 + 2.0 ** -14)).all()
    # nothing else was written
    used = torch.zeros(nb * bs, dtype=torch.bool)
    used[slots[slots >= 0].long()] = True
    rest = [s for s in range(nb * bs) if not used[s]]
    for c in (k, v):
        vals, swing = kv4_ref.rows(c, rest)
        assert not vals.any() and not swing.any()


def test_write_sums_split_k_planes():
    T, hq, hkv, bs = 5, 4, 2, 16
    nb, qkv, qw, kw, cs, pos, slots = _write_case(T, hq, hkv, bs, 3)
    cuda = _cuda()
    planes = torch.randn(3, *qkv.shape, generator=torch.Generator().manual_seed(4)).to(DEV)
    part = cuda.SplitKPartial(planes.view(torch.uint8).flatten(), 3, *qkv.shape)
    # ((p0 + p1) + p2) in fp32, then bf16: the kernel's order
    whole = ((planes[0] + planes[1]) + planes[2]).bfloat16()
    a, b = _empty(nb, hkv, bs), _empty(nb, hkv, bs)
    args = (qw.to(DEV), kw.to(DEV), 1e-6, cs.to(DEV), pos.to(DEV), slots.to(DEV))
    qa = cuda.qk_norm_rope_cache(part, *args, *a, hq, hkv, D)
    qb = cuda.qk_norm_rope_cache(whole, *args, *b, hq, hkv, D)
    cuda.check_status()
    assert torch.equal(qa, qb) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_write_matches_the_cpu_backend_byte_for_byte():
    T, hq, hkv, bs = 70, 8, 4, 32
    nb, qkv, qw, kw, cs, pos, slots = _write_case(T, hq, hkv, bs, 9, (3,))
    qkv[11, 5] = float("nan")
    qkv[12, (hq + hkv) * D + 20] = float("inf")                # one group of a V row
    qkv[13] = 0.0                                              # constant groups
    qkv[14, (hq + hkv) * D:] = 1.5
    gpu = _empty(nb, hkv, bs)
    cpu = [c.cpu() for c in gpu]
    _ops().qk_norm_rope_cache(qkv.to(DEV), qw.to(DEV), kw.to(DEV), 1e-6, cs.to(DEV), pos.to(DEV), slots.to(DEV), *gpu, hq, hkv, D)
    cpu_ref.qk_norm_rope_cache(qkv, qw, kw, 1e-6, cs, pos, slots, *cpu, hq, hkv, D)
    _cuda().check_status()
    live = slots[slots >= 0].long()
    for a, b in zip(gpu, cpu):
        torch.testing.assert_close(kv4.read_rows(a.cpu(), live), kv4.read_rows(b, live), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e-3, 1e15, 1e25, 3e38])
def test_rows_of_any_size_and_infinite_ones(size):
    """The sum of squares of a K row leaves fp32, or is lost beside eps (which counts in 64 bits); an infinity makes its own
    group NaN and, through the norm, zeros of the rest."""
    T, hq, hkv, bs = 600, 2, 2, 16
    nb, qkv, qw, kw, cs, pos, slots = _write_case(T, hq, hkv, bs, 12)
    qkv[:, hq * D:] = (qkv[:, hq * D:].float().clamp(-1, 1) * size).bfloat16()
    qkv[1, hq * D + 3] = float("inf")
    qkv[2, hq * D + D] = float("-inf")
    qkv[4, hq * D] = float("nan")
    gpu, cpu = _empty(nb, hkv, bs), [c.cpu() for c in _empty(nb, hkv, bs)]
    _ops().qk_norm_rope_cache(qkv.to(DEV), qw.to(DEV), kw.to(DEV), 1e-6, cs.to(DEV), pos.to(DEV), slots.to(DEV), *gpu, hq, hkv, D)
    _ops().qk_norm_rope_cache(qkv, qw, kw, 1e-6, cs, pos, slots, *cpu, hq, hkv, D)
    live = slots[slots >= 0].long()
    for a, b in zip(gpu, cpu):
        torch.testing.assert_close(kv4.read_rows(a.cpu(), live), kv4.read_rows(b, live), rtol=0, atol=0, equal_nan=True)
    assert bool(kv4.read_rows(cpu[0], live).any())


def test_bad_slots_and_positions_are_reported_and_not_followed():
    T, hq, hkv, bs = 4, 2, 1, 16
    nb, qkv, qw, kw, cs, pos, slots = _write_case(T, hq, hkv, bs, 5)
    k, v = _empty(nb, hkv, bs)
    args = (qkv.to(DEV), qw.to(DEV), kw.to(DEV), 1e-6, cs.to(DEV))
    slots[1] = nb * bs
    _ops().qk_norm_rope_cache(*args, pos.to(DEV), slots.to(DEV), k, v, hq, hkv, D)
    with pytest.raises(RuntimeError, match="status 5"):
        _cuda().check_status()
    kk, _ = _ops().read_cache(k, v, slots.to(DEV), D)
    assert not kk[1].any() and bool(kk[0].any())
    with pytest.raises(RuntimeError, match="status 5"):
        _cuda().check_status()
    pos[2] = 5000
    slots[1] = -1
    _ops().qk_norm_rope_cache(*args, pos.to(DEV), slots.to(DEV), k, v, hq, hkv, D)
    with pytest.raises(RuntimeError, match="status 5"):
        _cuda().check_status()


# ---- attention ----

def _attend(q_lens, kv_lens, hq, hkv, bs=16, n_decode=0, seed=0, poison=False, q_scale=1.0, extra_pages=1, v_scale=1.0):
    B = len(kv_lens)
    maxb = max(1, max(-(-n // bs) for n in kv_lens)) + extra_pages
    nb = sum(-(-n // bs) for n in kv_lens) + 2
    g = torch.Generator().manual_seed(seed + 100)
    perm = torch.randperm(nb, generator=g).tolist()
    table = torch.zeros(B, maxb, dtype=torch.int32)
    for b, n in enumerate(kv_lens):
        for i in range(-(-n // bs)):
            table[b, i] = perm.pop()
    k, v = _random(nb, hkv, bs, seed, v_scale)
    if poison:                     # parameters of every row that no sequence holds are NaN
        live = torch.zeros(nb * bs, dtype=torch.bool)
        for b, n in enumerate(kv_lens):
            for t in range(n):
                live[int(table[b, t // bs]) * bs + t % bs] = True
        dead = (~live).nonzero().flatten()
        if len(dead):
            for c in (k, v):
                host = c.cpu()
                kv4.write_rows(host, dead, torch.full((len(dead), hkv, D), float("nan")))
                c.copy_(host)
    T = sum(q_lens)
    q = (torch.randn(T, hq * D, generator=g) * q_scale).bfloat16()
    cu = torch.tensor([0] + list(np.cumsum(q_lens)), dtype=torch.int32)
    scale = D ** -0.5
    attn = AttnBatch(cu_q=cu.to(DEV), kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device=DEV), block_tables=table.to(DEV),
                     num_seqs=B, num_decode=n_decode, max_q_len=max(q_lens), max_kv_len=max(kv_lens), num_tokens=T)
    out = _ops().paged_attention(q.to(DEV), k, v, attn, scale, hq, hkv, D)
    torch.cuda.synchronize()
    _cuda().check_status()
    ref, mag, swing, qk = kv4_ref.attention(q, k, v, q_lens, kv_lens, table, scale, hq)
    got = out.double().cpu().numpy().reshape(T, hq, D)
    qk = qk[..., None]
    # Decode rows: the output is rounded to bf16 and P s_g to fp16 once (held to bf16's bound here); scores are fp32 sums
    # of at most 2 * 64 products no larger than 17 times those of q and k, so 2^-24 * 17 * 8 bounds their relative error.
    tol = HALF_BF16 * (np.abs(ref) + swing) + 2 * (2.0 ** -24 * 17 * 8 * qk + 2.0 ** -20) * mag
    # Chunks: K, V and P are each rounded to fp16 once, c + s (n - 8) from an exact n - 8, with s and c exact (8 bits): a
    # score moves by at most 2^-11 of sum |q| |k|, a probability by twice that, V and P by 2^-11 of p |v| each. The output is
    # rounded to bf16.
    chunk = HALF_BF16 * np.abs(ref) + 2.0 ** -9 * (mag + swing) + (np.exp(2.0 ** -9 * qk) - 1) * mag + 2.0 ** -18 * mag
    tol[n_decode:] = chunk[n_decode:]
    worst = (np.abs(got - ref) - tol).max()
    assert worst <= 0, worst
    if ref.any():
        rel = np.linalg.norm(got - ref) / np.linalg.norm(ref)
        assert rel <= HALF_BF16, rel
    return out


@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 8), (3, 1), (32, 8), (5, 1), (8, 1), (9, 1), (32, 2)])
def test_decode_groups(hq, hkv):
    _attend([1] * 5, [1, 15, 16, 17, 150], hq, hkv, n_decode=5, seed=hq)


@pytest.mark.parametrize("bs", [16, 48, 128])
def test_decode_page_sizes_and_empty_rows(bs):
    _attend([1] * 6, [0, 1, bs, bs + 1, 2 * bs - 1, 0], 8, 2, bs=bs, n_decode=6, seed=bs)


def test_decode_all_rows_empty():
    assert not _attend([1] * 2, [0, 0], 4, 2, n_decode=2).any()


def test_decode_many_splits_and_long_tables():
    _attend([1, 1], [1100, 513], 8, 2, n_decode=2, extra_pages=2000)       # most splits see nothing


WIDE = 20000       # pages of block table: the launch bound that makes decode deal its tokens in even shares


@pytest.mark.parametrize("hq,hkv", [(8, 8), (3, 1), (16, 2), (9, 1)])
def test_even_shares_groups_and_ragged_lengths(hq, hkv):
    _attend([1] * 7, [0, 1, 150, 0, 17, 400, 33], hq, hkv, n_decode=7, seed=hq, extra_pages=WIDE)


@pytest.mark.parametrize("bs", [48, 128])
def test_even_shares_page_sizes_and_nan_around_the_sequences(bs):
    _attend([1] * 5, [bs - 1, 3 * bs, 1, 0, 2 * bs + 5], 8, 2, bs=bs, n_decode=5, poison=True, extra_pages=WIDE)


def test_even_shares_one_sequence_many_runs_and_mixed_batch():
    _attend([1], [1500], 8, 2, n_decode=1, q_scale=3.0, extra_pages=WIDE)
    _attend([1, 1, 40], [90, 333, 56], 8, 2, n_decode=2, extra_pages=WIDE)


def test_even_shares_all_rows_empty():
    assert not _attend([1] * 3, [0, 0, 0], 4, 2, n_decode=3, extra_pages=WIDE).any()


def test_even_shares_more_sequences_than_threads_of_the_scan():
    lens = [(i * 7) % 23 for i in range(300)]
    _attend([1] * 300, lens, 2, 2, n_decode=300, extra_pages=600)


def test_decode_growing_maxima():
    _attend([1, 1], [400, 700], 8, 1, n_decode=2, q_scale=8.0, seed=4)


def test_decode_values_near_zero_of_a_large_step():
    """Rows that one token dominates, where codes of 8 and small centres make outputs a thousandth of a step: nothing of the
    8 that comes off may be left."""
    _attend([1] * 20, [9, 0, 11, 9, 2, 7, 15, 6, 3, 18, 11, 12, 14, 4, 11, 12, 3, 8, 3, 3], 24, 3, bs=64, n_decode=20, seed=84421,
            q_scale=4.0, extra_pages=300)
    _attend([1] * 20, [16, 156, 81, 98, 52, 181, 75, 24, 111, 1, 89, 23, 104, 39, 28, 136, 187, 45, 192, 87], 48, 3, bs=128,
            n_decode=20, seed=990221, q_scale=4.0)
    _attend([1] * 64, [1] * 64, 8, 8, n_decode=64, seed=5)


@pytest.mark.parametrize("extra_pages", [1, WIDE])
@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (1, 2, 0)])
def test_decode_values_of_mixed_magnitude(order, extra_pages):
    """V rows of 2^-20, 1 and 2^20 times normal values behind rows that are constant, in runs that a warp meets one after
    the other: the power of two that P * s is held in moves up. A term's rounding is at most half a step of fp16, 2^-11 of
    it, or of the smallest subnormal, 2^-25 in units that the largest scale met so far is at least 2^2 of: relative to the
    largest |v| (at least 2^-7 of it is in `mag`, a tenth of the weights being on such rows) 400 * 8 * 2^-27 / 12 is below 2^-18."""
    hq, hkv, bs, n = 4, 1, 16, 400
    nb = n // bs
    g = torch.Generator().manual_seed(31)
    k, v = (torch.zeros(nb, hkv, bs, kv4.row_bytes(D), dtype=torch.uint8) for _ in range(2))
    size = torch.tensor([2.0 ** (20 * (order[t // 5 % 3] - 1)) for t in range(n)])[:, None, None]
    values = torch.randn(n, hkv, D, generator=g) * size
    values[:7] = 3.0
    kv4.write_rows(k, torch.arange(n), torch.randn(n, hkv, D, generator=g))
    kv4.write_rows(v, torch.arange(n), values)
    q = (torch.randn(1, hq * D, generator=g) * 0.25).bfloat16()
    table = torch.zeros(1, nb + extra_pages, dtype=torch.int32)
    table[0, :nb] = torch.arange(nb)
    i32 = dict(dtype=torch.int32, device=DEV)
    attn = AttnBatch(torch.tensor([0, 1], **i32), torch.tensor([n], **i32), table.to(DEV), 1, 1, 1, n, 1)
    out = _ops().paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), attn, D ** -0.5, hq, hkv, D)
    _cuda().check_status()
    ref, mag, swing, qk = kv4_ref.attention(q, k, v, [1], [n], table, D ** -0.5, hq)
    got = out.double().cpu().numpy().reshape(1, hq, D)
    tol = HALF_BF16 * (np.abs(ref) + swing) + 2 * (2.0 ** -24 * 17 * 8 * qk[..., None] + 2.0 ** -18) * mag
    assert ((np.abs(got - ref) - tol) <= 0).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("extra_pages", [1, WIDE])
def test_decode_query_head_that_is_not_finite_stays_alone(bad, extra_pages):
    k, v = _random(8, 2, 16, 3)
    q = torch.randn(2, 8 * D, generator=torch.Generator().manual_seed(8)).bfloat16()
    q[0, 2 * D + 5] = 0.0
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.zeros(2, 4 + extra_pages, **i32)
    table[0, :4], table[1, :4] = torch.arange(4, **i32), torch.arange(4, 8, **i32)
    attn = AttnBatch(torch.tensor([0, 1, 2], **i32), torch.tensor([50, 61], **i32), table, 2, 2, 1, 61, 2)
    clean = _ops().paged_attention(q.to(DEV), k, v, attn, 0.09, 8, 2, D)
    q[0, 2 * D + 5] = bad
    out = _ops().paged_attention(q.to(DEV), k, v, attn, 0.09, 8, 2, D)
    _cuda().check_status()
    assert not bool(out[0, 2 * D:3 * D].isfinite().any())
    out[0, 2 * D:3 * D] = clean[0, 2 * D:3 * D]
    assert torch.equal(out, clean)


def test_rows_beyond_the_sequence_may_hold_nan():
    _attend([1, 1, 1, 20, 70], [1, 15, 33, 20, 100], 8, 2, n_decode=3, poison=True)
    _attend([1, 65], [47, 130], 4, 2, bs=48, n_decode=1, poison=True)


def test_nan_inside_a_sequence_reaches_its_rows_only():
    k, v = _random(4, 1, 16, 1)
    host = k.cpu()
    kv4.write_rows(host, torch.arange(16), torch.full((16, 1, D), float("nan")))
    k.copy_(host)
    q = torch.ones(2, 2 * D, device=DEV).bfloat16()
    i32 = dict(dtype=torch.int32, device=DEV)
    attn = AttnBatch(cu_q=torch.tensor([0, 1, 2], **i32), kv_lens=torch.tensor([16, 20], **i32),
                     block_tables=torch.tensor([[0, 0], [1, 2]], **i32), num_seqs=2, num_decode=2, max_q_len=1,
                     max_kv_len=20, num_tokens=2)
    out = _ops().paged_attention(q, k, v, attn, 0.1, 2, 1, D)
    assert bool(out[0].isnan().all()) and bool(out[1].isfinite().all())


@pytest.mark.parametrize("hq,hkv,bs", [(8, 2, 16), (3, 1, 48), (4, 4, 64)])
def test_chunks(hq, hkv, bs):
    _attend([1, 15, 64, 65, 33], [1, 15, 64, 65, 33 + 40], hq, hkv, bs=bs, seed=hq)


def test_chunk_with_no_context_is_zero_and_mixed_batch():
    _attend([1, 1, 40, 70], [33, 1, 40, 16 + 70], 8, 2, n_decode=2, seed=7)


@pytest.mark.parametrize("q_len,kv_len", [(130, 130), (200, 333), (128, 512)])
def test_long_chunks(q_len, kv_len):
    _attend([q_len, 67], [kv_len, 67], 4, 2, seed=q_len)


@pytest.mark.parametrize("hq,hkv,bs", [(8, 8, 16), (2, 1, 48), (5, 1, 16), (8, 1, 128), (16, 1, 32), (12, 1, 16)])
def test_chunks_of_every_group_size(hq, hkv, bs):
    _attend([70, 1, 33], [70 + 131, 1, 33], hq, hkv, bs=bs, seed=hq)


@pytest.mark.parametrize("hq,hkv", [(4, 1), (5, 1), (16, 2)])
def test_short_chunks_behind_long_prefixes_split_the_range(hq, hkv):
    _attend([1, 9, 40], [1400, 1209, 40], hq, hkv, seed=hq, extra_pages=300)


def test_split_chunks_with_nan_around_and_bad_pages():
    _attend([30, 2], [700, 130], 4, 2, poison=True, extra_pages=300)


def test_chunk_growing_maxima():
    _attend([150], [500], 4, 1, q_scale=8.0, seed=9)


def test_chunk_values_of_mixed_magnitude():
    """Tiles of K and V whose magnitudes differ by 2^20 either way: the tile exponents move up and down."""
    hq, hkv, bs, n = 4, 1, 16, 400
    nb = n // bs + 2
    g = torch.Generator().manual_seed(3)
    ramp = torch.tensor([2.0 ** (20 * ((t // 130) % 3 - 1)) for t in range(nb * bs)])[:, None, None]
    k, v = (torch.zeros(nb, hkv, bs, kv4.row_bytes(D), dtype=torch.uint8) for _ in range(2))
    kv4.write_rows(k, torch.arange(nb * bs), torch.randn(nb * bs, hkv, D, generator=g) * ramp.clamp(max=1.0))
    kv4.write_rows(v, torch.arange(nb * bs), torch.randn(nb * bs, hkv, D, generator=g) * ramp)
    q = (torch.randn(n, hq * D, generator=g) * 0.5).bfloat16()
    table = torch.arange(nb, dtype=torch.int32)[None]
    i32 = dict(dtype=torch.int32, device=DEV)
    attn = AttnBatch(torch.tensor([0, n], **i32), torch.tensor([n], **i32), table.to(DEV), 1, 0, n, n, n)
    out = _ops().paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), attn, D ** -0.5, hq, hkv, D)
    _cuda().check_status()
    ref, mag, swing, qk = kv4_ref.attention(q, k, v, [n], [n], table, D ** -0.5, hq)
    got = out.double().cpu().numpy().reshape(n, hq, D)
    tol = HALF_BF16 * np.abs(ref) + 2.0 ** -9 * (mag + swing) + (np.exp(2.0 ** -9 * qk[..., None]) - 1) * mag + 2.0 ** -18 * mag
    assert ((np.abs(got - ref) - tol) <= 0).all()


@pytest.mark.parametrize("q_len", [40, 200])
def test_chunk_nan_in_the_sequence_reaches_the_rows_that_see_it(q_len):
    """NaN parameters of K and of V at single positions: rows before them are as if they were not there."""
    hq, hkv, bs = 4, 1, 16
    n = q_len + 30
    nb = n // bs + 2
    k, v = _random(nb, hkv, bs, 5)
    hk, hv = k.cpu(), v.cpu()
    bad_k, bad_v = 30 + q_len // 2, 30 + 3 * q_len // 4
    kv4.write_rows(hk, torch.tensor([bad_k]), torch.full((1, hkv, D), float("nan")))
    kv4.write_rows(hv, torch.tensor([bad_v]), torch.full((1, hkv, D), float("nan")))
    q = torch.randn(q_len, hq * D, generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.arange(nb, **i32)[None]
    attn = AttnBatch(torch.tensor([0, q_len], **i32), torch.tensor([n], **i32), table, 1, 0, q_len, n, q_len)
    clean = _ops().paged_attention(q, k, v, attn, 0.09, hq, hkv, D)
    for c, b in ((hk, bad_k), (hv, bad_v)):
        args = (c.to(DEV), v) if c is hk else (k, c.to(DEV))
        out = _ops().paged_attention(q, *args, attn, 0.09, hq, hkv, D)
        first = b - 30                                       # the query row at that position
        assert torch.equal(out[:first], clean[:first])
        assert bool(out[first:].isnan().any(-1).all())
    _cuda().check_status()


def test_small_and_large_values():
    _attend([1, 30], [40, 60], 4, 2, n_decode=1, v_scale=2.0 ** -60, q_scale=2.0 ** 60)
    _attend([1, 30], [40, 60], 4, 2, n_decode=1, v_scale=2.0 ** 40, q_scale=2.0 ** -40)


@pytest.mark.parametrize("extra_pages", [1, 300])
def test_rows_before_position_0_and_behind_the_last_sequence_are_zero(extra_pages):
    out = _attend([1, 40, 150], [9, 25, 130], 4, 2, n_decode=1, extra_pages=extra_pages)
    assert not out[1:16].any() and not out[41:61].any() and bool(out[16:41].any(-1).all())
    ops = _ops()
    q, k, v, attn = _small()
    padded = torch.cat([q, torch.ones(300, q.shape[1], dtype=q.dtype, device=DEV)])
    for n_decode in (2, 1, 0):
        attn.num_decode = n_decode
        torch.full_like(padded, 7.0)                         # what the allocator may hand out again
        got = ops.paged_attention(padded, k, v, attn, 0.1, 4, 2, D)
        assert not got[2:].any()
        torch.testing.assert_close(got[:2], ops.paged_attention(q, k, v, attn, 0.1, 4, 2, D), rtol=0, atol=0)
    _cuda().check_status()


@pytest.mark.parametrize("power", [100, -100])
@pytest.mark.parametrize("extra_pages", [1, 300, WIDE])
def test_values_near_the_ends_of_the_range(power, extra_pages):
    """K and V of 2^100 or 2^-100 times normal values against queries that bring the scores back to size."""
    _attend([1, 1, 30, 140], [40, 700, 60, 333], 6, 2, n_decode=2, v_scale=2.0 ** power, q_scale=2.0 ** -power, extra_pages=extra_pages)


def test_scores_below_the_smallest_float_leave_equal_weights():
    """The scale of a score underflows; what the mask takes out still has weight 0, not NaN."""
    _attend([1, 30, 200], [40, 60, 200], 4, 2, n_decode=1, v_scale=2.0 ** -60, q_scale=2.0 ** -70)
    _attend([1, 30, 200], [40, 60, 200], 4, 2, n_decode=1, v_scale=2.0 ** -40, q_scale=0.0)


def _small(n_decode=2):
    k, v = _random(4, 2, 16, 0)
    i32 = dict(dtype=torch.int32, device=DEV)
    attn = AttnBatch(cu_q=torch.tensor([0, 1, 2], **i32), kv_lens=torch.tensor([20, 7], **i32),
                     block_tables=torch.tensor([[0, 1], [2, 0]], **i32), num_seqs=2, num_decode=n_decode, max_q_len=1,
                     max_kv_len=20, num_tokens=2)
    return torch.randn(2, 4 * D, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV), k, v, attn


@pytest.mark.parametrize("n_decode", [2, 0])
def test_bad_pages_lengths_and_ranges_are_reported_and_not_followed(n_decode):
    ops, cuda = _ops(), _cuda()
    for field, value in (("block_tables", [[0, 9], [2, 0]]), ("block_tables", [[0, -1], [2, 0]]), ("kv_lens", [33, 7])):
        q, k, v, attn = _small(n_decode)
        setattr(attn, field, torch.tensor(value, dtype=torch.int32, device=DEV))
        out = ops.paged_attention(q, k, v, attn, 0.1, 4, 2, D)
        with pytest.raises(RuntimeError, match="status 5"):
            cuda.check_status()
        assert bool(out[1].isfinite().all())
    if n_decode == 0:
        q, k, v, attn = _small(0)
        attn.cu_q = torch.tensor([0, 1, 3], dtype=torch.int32, device=DEV)
        ops.paged_attention(q, k, v, attn, 0.1, 4, 2, D)
        with pytest.raises(RuntimeError, match="status 5"):
            cuda.check_status()


def test_refusals():
    ops = _ops()
    q, k, v, attn = _small()
    for bad, args in ((TypeError, (q.float(), k, v)), (ValueError, (q.t().contiguous().t(), k, v)),
                      (TypeError, (q, k, v.float())), (ValueError, (q, k[:, :1], v[:, :1])), (ValueError, (q[:1], k, v)),
                      (ValueError, (q, k.cpu(), v.cpu()))):
        with pytest.raises(bad):
            ops.paged_attention(*args, attn, 0.1, 4, 2, D)
    for bad in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="finite"):
            ops.paged_attention(q, k, v, attn, bad, 4, 2, D)
    with pytest.raises(ValueError, match="16 to one"):
        ops.paged_attention(torch.zeros(2, 34 * D, device=DEV).bfloat16(), k, v, attn, 0.1, 34, 2, D)
    with pytest.raises(ValueError, match="head_dim 128"):
        ops.read_cache(torch.zeros(1, 1, 16, 40, dtype=torch.uint8, device=DEV),
                       torch.zeros(1, 1, 16, 40, dtype=torch.uint8, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), 64)
    with pytest.raises(ValueError, match="slots"):
        ops.read_cache(k, v, torch.zeros(1, dtype=torch.int64, device=DEV), D)
    attn.block_tables = torch.zeros(2, 4, dtype=torch.int32, device=DEV)[:, ::2]
    with pytest.raises(ValueError, match="block_tables"):
        ops.paged_attention(q, k, v, attn, 0.1, 4, 2, D)
    attn.block_tables = attn.block_tables.contiguous()
    with pytest.raises(RuntimeError, match="misaligned"):
        ops.paged_attention(torch.zeros(2 * 4 * D + 1, device=DEV).bfloat16()[1:].view(2, 4 * D), k, v, attn, 0.1, 4, 2, D)
    attn.kv_lens = attn.kv_lens.long()
    with pytest.raises(ValueError, match="kv_lens"):
        ops.paged_attention(q, k, v, attn, 0.1, 4, 2, D)
    e = ops.paged_attention(q[:0], k, v, AttnBatch(attn.cu_q[:1], attn.kv_lens[:0].int(), attn.block_tables[:0], 0, 0, 0, 0, 0),
                            0.1, 4, 2, D)
    assert e.shape == (0, 4 * D)


def test_two_streams_and_graph_replay_do_not_share_scratch():
    """Two captured decode calls with a workspace, replayed at the same time on two streams, and an eager one between."""
    ops = _ops()
    runs = []
    for seed in (1, 2):
        k, v = _random(70, 2, 16, seed)
        g = torch.Generator().manual_seed(seed)
        q = torch.randn(1, 8 * D, generator=g).bfloat16().to(DEV)
        i32 = dict(dtype=torch.int32, device=DEV)
        table = torch.zeros(1, WIDE, **i32)
        table[0, :70] = torch.randperm(70, generator=g).to(**i32)
        attn = AttnBatch(torch.tensor([0, 1], **i32), torch.tensor([1100], **i32), table, 1, 1, 1, 1100, 1)
        want = ops.paged_attention(q, k, v, attn, 0.09, 8, 2, D).clone()
        torch.cuda.synchronize()
        gr, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(gr, stream=s):
            out = ops.paged_attention(q, k, v, attn, 0.09, 8, 2, D)
        runs.append((gr, s, out, want, (q, k, v, attn)))
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, s, out, want, _ in runs:
            with torch.cuda.stream(s):
                gr.replay()
        q, k, v, attn = runs[0][4]
        eager = ops.paged_attention(q, k, v, attn, 0.09, 8, 2, D)
        torch.cuda.synchronize()
        assert torch.equal(eager, runs[0][3])
        for _, _, out, want, _ in runs:
            assert torch.equal(out, want)
    _cuda().check_status()


def test_split_chunks_on_two_streams_do_not_share_scratch():
    """Two captured chunk calls whose KV range is split, replayed at the same time on two streams."""
    ops = _ops()
    runs = []
    for seed in (1, 2):
        k, v = _random(80, 2, 16, seed)
        g = torch.Generator().manual_seed(seed)
        q = torch.randn(40, 8 * D, generator=g).bfloat16().to(DEV)
        i32 = dict(dtype=torch.int32, device=DEV)
        attn = AttnBatch(torch.tensor([0, 40], **i32), torch.tensor([1200], **i32), torch.randperm(80, generator=g)[None].to(**i32),
                         1, 0, 40, 1200, 40)
        want = ops.paged_attention(q, k, v, attn, 0.09, 8, 2, D).clone()
        torch.cuda.synchronize()
        gr, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(gr, stream=s):
            out = ops.paged_attention(q, k, v, attn, 0.09, 8, 2, D)
        runs.append((gr, s, out, want, (q, k, v, attn)))
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, s, out, want, _ in runs:
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for _, _, out, want, _ in runs:
            assert torch.equal(out, want)
    _cuda().check_status()


def test_captured_step_follows_its_inputs():
    """One graph of append, decode attention and read-back on a side stream: every replay takes what the inputs hold then,
    padded rows (slot -1, no cached tokens) among them."""
    ops, B, hq, hkv, bs = _ops(), 5, 8, 2, 16
    k, v = _random(64, hkv, bs, 4)
    ek, ev = k.clone(), v.clone()
    g = torch.Generator().manual_seed(4)
    i32 = dict(dtype=torch.int32, device=DEV)
    qw, kw = (torch.exp(0.3 * torch.randn(D, generator=g)).bfloat16().to(DEV) for _ in range(2))
    cs = cpu_ref.build_cos_sin_cache(D, 5000, 1e6).to(DEV)
    qkv = torch.zeros(B, (hq + 2 * hkv) * D, device=DEV).bfloat16()
    pos, slots, lens = (torch.zeros(B, **i32) for _ in range(3))
    slots.fill_(-1)
    table = torch.arange(60, **i32).view(B, 12).contiguous()
    attn = AttnBatch(torch.arange(B + 1, **i32), lens, table, B, B, 1, 192, B)

    def step(k, v):
        q = ops.qk_norm_rope_cache(qkv, qw, kw, 1e-6, cs, pos, slots, k, v, hq, hkv, D)
        return (ops.paged_attention(q, k, v, attn, 0.09, hq, hkv, D), *ops.read_cache(k, v, slots, D))

    step(k, v)
    torch.cuda.synchronize()
    gr, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(gr, stream=s):
        got = step(k, v)
    for i in range(6):
        n = torch.randint(1, 190, (B,), generator=g)
        live = torch.arange(B) != i % B
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        pos.copy_(n)
        lens.copy_(torch.where(live, n + 1, 0))
        slots.copy_(torch.where(live, torch.arange(B) * 192 + n, -1))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(ek, ev)):
            assert torch.equal(a, b)
        assert torch.equal(k, ek) and torch.equal(v, ev) and not got[0][i % B].any() and not got[1][i % B].any()
    _cuda().check_status()


# ---- the operators together, as the engine runs them ----

def _engine(model_dir, prompts, max_tokens, **kw):
    from xixi_vllm_b200 import Engine, EngineConfig, SamplingParams
    base = dict(device="cuda", dtype="bfloat16", num_kvcache_blocks=256, max_num_seqs=16, max_num_batched_tokens=256,
                context_len=512, kv_cache_dtype="int4")
    base.update(kw)
    eng = Engine(EngineConfig(model=model_dir, **base))
    try:
        seqs = [eng.add_request(p, SamplingParams(max_tokens=max_tokens, ignore_eos=True)) for p in prompts]
        while eng.has_unfinished():
            eng.step()
        return [s.token_ids[s.num_prompt_tokens:] for s in seqs]
    finally:
        eng.destroy()


@pytest.fixture(scope="module")
def model_dir(tmp_path_factory):
    from xixi_vllm_b200.models.synth import make_model_dir
    return make_model_dir(str(tmp_path_factory.mktemp("kv4_model")), "tiny", std=0.08, num_hidden_layers=2, hidden_size=512,
                          num_attention_heads=4, num_key_value_heads=2, head_dim=128, intermediate_size=1024,
                          vocab_size=2048, torch_dtype="bfloat16", tie_word_embeddings=False)


def _prompts(lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 2048, (n,), generator=g).tolist() for n in lens]


def test_engine_native_and_module_forwards_agree_on_a_4_bit_cache(model_dir, monkeypatch):
    """Graph-replayed native executor against the Python forward: the same kernels, so identical tokens. Four sequences
    are a graph bucket of their own and 240 tokens of context one KV split, so both run the same launch shapes (another
    split count adds in another order)."""
    prompts = _prompts((7, 33, 120, 200), 2)
    kw = dict(context_len=240)
    native = _engine(model_dir, prompts, 10, enforce_eager=False, **kw)
    late = _engine(model_dir, prompts, 10, enforce_eager=False, async_scheduling="off", **kw)
    monkeypatch.setenv("XV_NATIVE_FORWARD", "0")
    assert native == _engine(model_dir, prompts, 10, enforce_eager=True, **kw) == late


def test_engine_on_a_4_bit_cache_follows_the_cpu_backend(model_dir):
    """First sampled token of every prompt: one forward from equal inputs. Later ones depend on it."""
    prompts = _prompts((5, 16, 17, 40, 100, 3, 230), 0)
    gpu = _engine(model_dir, prompts, 12)
    cpu = _engine(model_dir, prompts, 12, device="cpu")
    assert sum(a[0] == b[0] for a, b in zip(gpu, cpu)) >= len(prompts) - 1, (gpu, cpu)


def test_append_attend_and_read_back_as_one_run():
    """Prompt chunk, two more chunks on top of it, then decode steps: every output against 64-bit attention over the
    bytes that the steps before it wrote."""
    ops, cuda = _ops(), _cuda()
    hq, hkv, bs = 8, 2, 16
    g = torch.Generator().manual_seed(11)
    k, v = _empty(12, hkv, bs)
    table = torch.randperm(12, generator=g)[None].to(torch.int32)
    cs = cpu_ref.build_cos_sin_cache(D, 400, 1e6).to(DEV)
    w = torch.ones(D).bfloat16().to(DEV)
    have = 0
    for n in (70, 37, 1, 1, 2, 1):
        qkv = torch.randn(n, (hq + 2 * hkv) * D, generator=g).bfloat16().to(DEV)
        pos = torch.arange(have, have + n, dtype=torch.int32)
        slots = torch.tensor([int(table[0, t // bs]) * bs + t % bs for t in range(have, have + n)], dtype=torch.int32)
        q = ops.qk_norm_rope_cache(qkv, w, w, 1e-6, cs, pos.to(DEV), slots.to(DEV), k, v, hq, hkv, D)
        have += n
        i32 = dict(dtype=torch.int32, device=DEV)
        attn = AttnBatch(torch.tensor([0, n], **i32), torch.tensor([have], **i32), table.to(DEV), 1, 1 if n == 1 else 0, n, have, n)
        out = ops.paged_attention(q, k, v, attn, D ** -0.5, hq, hkv, D)
        cuda.check_status()
        ref, *_ = kv4_ref.attention(q, k, v, [n], [have], table, D ** -0.5, hq)
        got = out.double().cpu().numpy().reshape(n, hq, D)
        assert np.linalg.norm(got - ref) <= HALF_BF16 * 2 * np.linalg.norm(ref)
    every = torch.tensor([int(table[0, t // bs]) * bs + t % bs for t in range(have)], dtype=torch.int32, device=DEV)
    kk, vv = ops.read_cache(k, v, every, D)
    for got, cache in ((kk, k), (vv, v)):
        want, _ = kv4_ref.rows(cache, every.tolist())
        assert (np.abs(got.double().cpu().numpy() - want) <= HALF_BF16 * np.abs(want) * (1 + 2.0 ** -14)).all()
