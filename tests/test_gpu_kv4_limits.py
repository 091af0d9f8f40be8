"""Calls on 4-bit caches at the ends of what they take: magnitudes, scales, values that are not finite, launch bounds."""
import numpy as np
import pytest
import torch

import kv4_ref
from test_gpu_kv4 import D, DEV, HALF_BF16, WIDE, _cuda, _ops
from xixi_vllm_b200.ops import kv4
from xixi_vllm_b200.runtime.staging import AttnBatch

pytestmark = pytest.mark.gpu
SCALE = D ** -0.5
I32 = dict(dtype=torch.int32, device=DEV)


class Case:
    """One packed batch on pages of 16 tokens, made on the CPU: k, v ``[sequence][tokens, hkv, D]``, q ``[rows, hq, D]``."""

    def __init__(self, q_lens, kv_lens, hq, hkv, n_decode=0, extra_pages=1, seed=0, crowd=0):
        """``crowd``: so many one-token sequences more, which make a launch of chunks too large for its range to be split."""
        q_lens, kv_lens = q_lens + [1] * crowd, kv_lens + [1] * crowd
        self.q_lens, self.kv_lens, self.hq, self.hkv, self.n_decode = q_lens, kv_lens, hq, hkv, n_decode
        g = torch.Generator().manual_seed(seed)
        per = max(1, max(-(-n // 16) for n in kv_lens))
        self.table = torch.zeros(len(kv_lens), per + extra_pages, dtype=torch.int32)
        self.table[:, :per] = torch.arange(len(kv_lens) * per).view(-1, per)
        self.pages = len(kv_lens) * per
        self.k, self.v = ([torch.randn(n, hkv, D, generator=g) for n in kv_lens] for _ in range(2))
        self.q = torch.randn(sum(q_lens), hq, D, generator=g)

    def attn(self):
        cu = torch.tensor([0] + list(np.cumsum(self.q_lens)))
        return AttnBatch(cu.to(**I32), torch.tensor(self.kv_lens, **I32), self.table.to(DEV), len(self.kv_lens), self.n_decode,
                         max(self.q_lens), max(self.kv_lens), sum(self.q_lens))

    def caches(self):
        out = []
        for values in (self.k, self.v):
            c = torch.zeros(self.pages, self.hkv, 16, kv4.row_bytes(D), dtype=torch.uint8)
            for b, x in enumerate(values):
                slots = self.table[b, torch.arange(len(x)) // 16] * 16 + torch.arange(len(x)) % 16
                kv4.write_rows(c, slots, x)
            out.append(c)
        return out

    def run(self, scale=SCALE):
        k, v = self.caches()
        q = self.q.bfloat16().flatten(1)
        out = _ops().paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), self.attn(), scale, self.hq, self.hkv, D)
        _cuda().check_status()
        return out.view(-1, self.hq, D).cpu()

    def reference(self, scale):
        """64-bit outputs ``[rows, hq, D]`` and how far a call may be from them. A decode score is an fp32 sum of at most 2 * 64
        products no larger than 17 times those of q and k, so it is off by 2^-24 * 17 * 8 of sum |q| |k|; P s is rounded to
        fp16 and the output to bf16 (both held to bf16's bound). A chunk's K, V and P are rounded to fp16 once each, 2^-11.
        An error d of token j's score moves p_j by p_j (e^d - 1), in the numerator and in the sum. What falls below fp16's
        smallest number, and fp32 sums, are 2^-18 of sum p |v| at these lengths."""
        k_cache, v_cache = self.caches()
        q = self.q.bfloat16().double().numpy() * scale
        ref, tol = np.zeros(q.shape), np.zeros(q.shape)
        at = 0
        for b, (n, L) in enumerate(zip(self.q_lens, self.kv_lens)):
            slots = [int(self.table[b, t // 16]) * 16 + t % 16 for t in range(L)]
            k, (v, codes) = kv4_ref.rows(k_cache, slots)[0], kv4_ref.rows(v_cache, slots)
            for h in range(self.hq):
                hk = h // (self.hq // self.hkv)
                x = q[at:at + n, h]
                s = x @ k[:, hk].T
                s[np.arange(L) > (L - n + np.arange(n))[:, None]] = -np.inf
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                decode = np.arange(b, b + n)[:, None] < self.n_decode
                with np.errstate(over="ignore", invalid="ignore"):
                    moved = np.where(p > 0, p * np.expm1(np.minimum(np.where(decode, 2.0 ** -24 * 17 * 8, 2.0 ** -11) * (np.abs(x) @ np.abs(k[:, hk]).T), 700)), 0)
                out, mag, swing = p @ v[:, hk], p @ np.abs(v[:, hk]), p @ np.abs(codes[:, hk])
                ref[at:at + n, h] = out
                rounded = np.where(decode, HALF_BF16 * swing, 2.0 ** -10 * (mag + swing))
                tol[at:at + n, h] = (HALF_BF16 * np.abs(out) + rounded + 2.0 ** -18 * mag + moved @ np.abs(v[:, hk]) +
                                     moved.sum(-1, keepdims=True) * np.abs(out))
            at += n
        return ref, tol

    def check(self, scale=SCALE):
        got = self.run(scale).double().numpy()
        ref, tol = self.reference(scale)
        bad = ~(np.abs(got - ref) <= tol)                    # NaN is bad
        assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4].tolist(), got[bad][:4], ref[bad][:4], tol[bad][:4])
        return got


@pytest.mark.parametrize("extra_pages", [1, WIDE])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (7, 1), (16, 1)])
def test_decode_head_of_any_finite_size_stays_alone(hq, hkv, extra_pages):
    """Query heads of 2^120 beside ordinary ones and beside heads of 2^-100: each head has its own power of two."""
    c = Case([1, 1], [40, 700], hq, hkv, n_decode=2, extra_pages=extra_pages, seed=3)
    c.q[:, 1] *= 2.0 ** 120
    c.q[:, 2] *= 2.0 ** -100
    got = c.check()
    # one token has all of the large head's weight: its scores are 2^100 and more apart
    vals, swing = kv4_ref.rows(c.caches()[1], [(int(c.table[1, t // 16])) * 16 + t % 16 for t in range(700)])
    k, _ = kv4_ref.rows(c.caches()[0], [(int(c.table[1, t // 16])) * 16 + t % 16 for t in range(700)])
    s = k[:, 0] @ c.q[1, 1].bfloat16().double().numpy()
    first, second = np.argsort(s)[::-1][:2]
    assert s[first] - s[second] > 2.0 ** -12 * np.abs(k[first, 0]) @ np.abs(c.q[1, 1].double().numpy())
    want, sw = vals[first, 0], np.abs(swing[first, 0])
    assert (np.abs(got[1, 1] - want) <= HALF_BF16 * (np.abs(want) + sw) + 2.0 ** -18 * np.abs(want)).all()


@pytest.mark.parametrize("power", [124, 110, -110, -118])
@pytest.mark.parametrize("extra_pages", [1, WIDE])
def test_decode_queries_at_the_ends_of_the_range(power, extra_pages):
    """Queries of 2^124 down to 2^-118 times normal values on keys that bring the scores back to size."""
    c = Case([1, 1], [40, 700], 6, 2, n_decode=2, extra_pages=extra_pages, seed=4)
    c.q.clamp_(-4, 4).mul_(2.0 ** power)
    c.q[:, ::2].abs_()                                       # their sum leaves fp32
    c.k = [k * 2.0 ** -min(power, 120) for k in c.k]
    c.check(SCALE * 2.0 ** (-power + min(power, 120)))


@pytest.mark.parametrize("extra_pages", [1, WIDE])
def test_decode_scores_beyond_2_to_the_30(extra_pages):
    """Weights are 1 and 0 there: the maximum's own exponent has to be 0, not what rounding leaves of it."""
    c = Case([1, 1], [40, 700], 6, 2, n_decode=2, extra_pages=extra_pages, seed=15)
    c.q *= 2.0 ** 31
    assert not np.isnan(c.run().double().numpy()).any()
    c.q.mul_(2.0 ** 8)
    k, v = c.caches()
    at = [int(c.table[1, t // 16]) * 16 + t % 16 for t in range(700)]
    (keys, _), (vals, swing) = kv4_ref.rows(k, at), kv4_ref.rows(v, at)
    got = c.run().double().numpy()[1]
    for h in range(6):
        q = c.q[1, h].bfloat16().double().numpy()
        s = keys[:, h // 3] @ q
        first, second = np.argsort(s)[::-1][:2]
        if s[first] - s[second] > 2.0 ** -12 * (np.abs(keys[first, h // 3]) @ np.abs(q)):       # well apart: fp32 sums see it
            want, sw = vals[first, h // 3], np.abs(swing[first, h // 3])
            assert (np.abs(got[h] - want) <= HALF_BF16 * (np.abs(want) + sw) + 2.0 ** -18 * np.abs(want)).all()


@pytest.mark.parametrize("scale", [0.0, 1e-33, -1e-33, 2.0 ** -120, 1e30])
@pytest.mark.parametrize("extra_pages,crowd", [(1, 0), (300, 0), (1, 160), (WIDE, 0)])
def test_scales_of_any_size(scale, extra_pages, crowd):
    """Zero leaves equal weights whatever the scores; a scale of 1e-33 is not a larger one."""
    c = Case([1, 1, 30, 200], [40, 700, 60, 333], 6, 2, n_decode=2, extra_pages=extra_pages, seed=5, crowd=crowd)
    size = 2.0 ** 110 if scale == 0 else 0.1 / abs(scale)
    c.q *= size ** 0.5
    c.k = [k * size ** 0.5 for k in c.k]
    c.check(scale)


@pytest.mark.parametrize("qp,kp,scale", [(-110, 120, 2.0 ** -13), (-100, 60, 2.0 ** 37), (100, -110, 2.0 ** 7), (100, -60, 2.0 ** -43)])
def test_products_of_scale_query_and_key_powers(qp, kp, scale):
    c = Case([1, 30, 200], [40, 60, 333], 6, 2, n_decode=1, seed=6)
    c.q *= 2.0 ** qp
    c.k = [k * 2.0 ** kp for k in c.k]
    c.check(scale)


@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_scores_beyond_2_to_the_30(crowd):
    """As for decode rows. A row whose best score is well apart from the next is that token's value."""
    c = Case([70, 30], [70, 560], 6, 2, extra_pages=300, crowd=crowd, seed=16)
    c.q *= 2.0 ** 31
    assert not np.isnan(c.run().double().numpy()).any()
    c.q *= 2.0 ** 8
    got, at, seen = c.run().double().numpy(), 0, 0
    k_cache, v_cache = c.caches()
    for b, (n, L) in enumerate(zip(c.q_lens[:2], c.kv_lens)):
        slots = [int(c.table[b, t // 16]) * 16 + t % 16 for t in range(L)]
        keys, vals = kv4_ref.rows(k_cache, slots)[0], kv4_ref.rows(v_cache, slots)[0]
        for i in range(n):
            for h in range(6):
                q = c.q[at + i, h].bfloat16().double().numpy()
                s = keys[:L - n + i + 1, h // 3] @ q
                best = int(np.argmax(s))
                rest = np.delete(s, best)
                if len(rest) == 0 or s[best] - rest.max() > 2.0 ** -10 * 2 * (np.abs(keys[:L - n + i + 1, h // 3]) @ np.abs(q)).max():
                    want = vals[best, h // 3]                # V rounded to fp16 once, P exact, the output to bf16
                    assert (np.abs(got[at + i, h] - want) <= (HALF_BF16 + 2.0 ** -11) * np.abs(want) + 2.0 ** -11 * np.abs(want).max()).all()
                    seen += 1
        at += n
    assert seen > 100


@pytest.mark.parametrize("crowd", [0, 160])
@pytest.mark.parametrize("first,second", [(10, 500), (500, 10), (300, 20)])
def test_chunk_scores_around_2_to_the_24(first, second, crowd):
    """Two tokens of 1.01 and 0.9 times 2^24 in log2 units, in different tiles (and CTAs): rows beyond 2^24 leave the scale's
    mantissa out, which must not turn their order."""
    c = Case([30], [560], 4, 1, extra_pages=300, crowd=crowd, seed=17)
    c.q = torch.ones_like(c.q)
    for b, k in enumerate(c.k):
        k.mul_(0.0)
    c.k[0][first], c.k[0][second] = 1.0, 0.9
    one = float(kv4_ref.rows(c.caches()[0], [int(c.table[0, first // 16]) * 16 + first % 16])[0].sum())
    target = 1.01 * 2.0 ** 24 / np.log2(np.e)
    size = max((1.0, 1.0625, 1.25, 1.5, 1.75), key=lambda a: np.frexp(target * np.log2(np.e) / (one * a))[0])
    assert np.frexp(target * np.log2(np.e) / (one * size))[0] > 0.85
    c.q *= size
    got = c.run(target / (one * size)).double().numpy()[:30]
    want = kv4_ref.rows(c.caches()[1], [int(c.table[0, first // 16]) * 16 + first % 16])[0][0, 0]
    assert (np.abs(got - want) <= (HALF_BF16 + 2.0 ** -11) * np.abs(want) + 2.0 ** -11 * np.abs(want).max()).all()


@pytest.mark.parametrize("hq,hkv", [(4, 1), (3, 1), (16, 1)])
@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_row_of_any_finite_size_stays_alone(hq, hkv, crowd):
    c = Case([40, 33], [40, 633], hq, hkv, extra_pages=300, crowd=crowd, seed=7)
    c.q[5, 1] *= 2.0 ** 120
    c.q[50, 0] *= 2.0 ** 60
    c.q[9] *= 2.0 ** -90
    c.check()


@pytest.mark.parametrize("crowd", [0, 160])
def test_small_values_over_a_long_context(crowd):
    c = Case([1, 100], [1100, 1500], 4, 1, n_decode=1, extra_pages=300, crowd=crowd, seed=10)
    c.v = [v * 2.0 ** -112 for v in c.v]
    c.q *= 0.3
    c.check()


@pytest.mark.parametrize("powers", [(20, -110), (0, -120, 0), (100, -20, -110, 60), (-110, 20), (10, -40, -10, -100)])
@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_values_whose_tiles_differ_by_any_power(powers, crowd):
    """128 tokens each of V at 2^p: the accumulator's unit must never take it out of fp32."""
    n = 128 * len(powers)
    c = Case([100], [n], 4, 1, extra_pages=300, crowd=crowd, seed=8)
    c.v[0] *= torch.tensor([2.0 ** powers[t // 128] for t in range(n)])[:, None, None]
    c.check()


@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_small_values_behind_large_ones_that_no_longer_count(crowd):
    """Later keys score about 200 higher, so the weights of the first 256 tokens, whose values are 2^80, are 2^-250 and less."""
    c = Case([100], [512], 4, 1, seed=9, crowd=crowd)
    c.q = 2.5 * (c.q.abs() + 0.5)
    c.k[0][256:] = c.k[0][256:].abs() + 2
    c.k[0][:256] = -c.k[0][:256].abs() - 2
    c.v[0][:256] *= 2.0 ** 80
    c.v[0][256:] *= 2.0 ** -30
    c.check()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_query_row_that_is_not_finite_is_nan_and_stays_alone(bad, sign, crowd):
    """Also where all its scores are -inf: a softmax of those is NaN, not zeros."""
    c = Case([40, 3], [40, 600], 4, 2, extra_pages=300, crowd=crowd, seed=11)
    for k in c.k:
        k[..., 5] = sign * (k[..., 5].abs() + 1)
    c.q[7, 2, 5] = c.q[41, 0, 5] = 0.0
    clean = c.run()
    c.q[7, 2, 5] = c.q[41, 0, 5] = bad
    out = c.run()
    assert not bool(out[7, 2].isfinite().any()) and not bool(out[41, 0].isfinite().any())
    out[7, 2], out[41, 0] = clean[7, 2], clean[41, 0]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("q_len,n_decode,extra_pages", [(1, 1, 1), (1, 1, WIDE), (40, 0, 1), (200, 0, 1), (40, 0, 300)])
def test_values_that_are_not_finite_reach_the_channels_of_their_group(q_len, n_decode, extra_pages):
    """One channel of a V row is infinite: its group's half of the row is held as NaN, and the rows that see it are NaN
    there; the other half is as if the group held zeros."""
    c = Case([q_len], [q_len + 600], 4, 1, n_decode=n_decode, extra_pages=extra_pages, seed=12)
    at = 600 + q_len // 2
    of = torch.arange(D) // 8 % 2 == 1
    c.v[0][at, 0, of] = 0.0
    clean = c.run()
    c.v[0][at, 0, 9] = float("inf")
    out = c.run()
    first = q_len // 2
    assert bool(out[first:, :, of].isnan().all())
    out[first:, :, of] = clean[first:, :, of]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("power", [124, 110, -110, -118])
@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_queries_at_the_ends_of_the_range(power, crowd):
    c = Case([30, 140], [60, 333], 6, 2, extra_pages=300, seed=4, crowd=crowd)
    c.q.clamp_(-4, 4).mul_(2.0 ** power)
    c.q[:, ::2].abs_()
    c.k = [k * 2.0 ** -min(power, 120) for k in c.k]
    c.check(SCALE * 2.0 ** (-power + min(power, 120)))


def test_chunks_without_rows_and_chunks_beyond_max_q_len():
    """Rows that no chunk covers are zeros whatever max_q_len says; a chunk that is longer than it is reported and comes
    out as zeros, its neighbours untouched."""
    ops, cuda = _ops(), _cuda()
    for extra_pages in (1, 300):
        c = Case([1, 5, 70, 9], [30, 45, 600, 9], 4, 2, n_decode=1, extra_pages=extra_pages, seed=13)
        k, v = (x.to(DEV) for x in c.caches())
        q = torch.cat([c.q, torch.ones(300, 4, D)]).bfloat16().flatten(1).to(DEV)
        want = ops.paged_attention(q, k, v, c.attn(), SCALE, 4, 2, D)
        assert bool(want[:85].any(-1).all()) and not want[85:].any()
        for most in (0, 1, 8, 9, 64, 69):
            torch.full_like(q, 7.0)                          # what the allocator may hand out again
            attn = c.attn()
            attn.max_q_len = most
            got = ops.paged_attention(q, k, v, attn, SCALE, 4, 2, D)
            with pytest.raises(RuntimeError, match="status 5"):
                cuda.check_status()
            at = 0
            for n in c.q_lens:
                if n == 1 or n <= most:
                    torch.testing.assert_close(got[at:at + n], want[at:at + n], rtol=2 * HALF_BF16, atol=2.0 ** -8)
                else:
                    assert not got[at:at + n].any()
                at += n
            assert not got[85:].any()
        for most in (0, 2 ** 31 - 1):                        # empty chunks only; a bound far above any row count
            attn = c.attn()
            if most == 0:
                attn.cu_q = torch.tensor([0, 1, 1, 1, 1], **I32)
            attn.max_q_len = most
            torch.full_like(q, 7.0)
            got = ops.paged_attention(q, k, v, attn, SCALE, 4, 2, D)
            cuda.check_status()
            torch.testing.assert_close(got, want if most else torch.cat([want[:1], torch.zeros_like(want[1:])]),
                                       rtol=2 * HALF_BF16, atol=2.0 ** -8)
        attn.max_q_len = -1
        with pytest.raises(ValueError, match="max_q_len"):
            ops.paged_attention(q, k, v, attn, SCALE, 4, 2, D)
        attn = c.attn()
        attn.cu_q = torch.tensor([0, 1, 6, 76, 2000], **I32)          # beyond the rows of q
        torch.full_like(q, 7.0)
        got = ops.paged_attention(q, k, v, attn, SCALE, 4, 2, D)
        with pytest.raises(RuntimeError, match="status 5"):
            cuda.check_status()
        torch.testing.assert_close(got[:76], want[:76], rtol=2 * HALF_BF16, atol=2.0 ** -8)
        assert not got[76:].any()
        attn.cu_q = torch.tensor([0, 4, 9, 79, 88], **I32)            # three rows between the decode row and the chunks
        torch.full_like(q, 7.0)
        moved = torch.cat([q[:1], torch.ones_like(q[:3]), q[1:-3]])
        got = ops.paged_attention(moved, k, v, attn, SCALE, 4, 2, D)
        cuda.check_status()
        assert torch.equal(got[:1], want[:1]) and torch.equal(got[4:88], want[1:85]) and not got[1:4].any() and not got[88:].any()
        attn.cu_q = torch.tensor([0, 0, 6, 76, 85], **I32)            # the first chunk begins on the decode row
        torch.full_like(q, 7.0)
        got = ops.paged_attention(q, k, v, attn, SCALE, 4, 2, D)
        with pytest.raises(RuntimeError, match="status 5"):
            cuda.check_status()
        assert torch.equal(got[:1], want[:1]) and torch.equal(got[6:], want[6:]) and not got[1:6].any()


@pytest.mark.parametrize("power", [60, 110])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_tokens_far_larger_than_their_neighbours(which, power, crowd):
    """Two tokens of 2^60 times the others' size inside one tile of a chunk: rows before them do not see them, rows behind
    them give them no weight (their scores are the lowest) or all of what they are worth."""
    c = Case([100, 30], [100, 560], 4, 1, extra_pages=300, crowd=crowd, seed=14)
    c.q = c.q.abs() + 0.5
    for b, at in ((0, 50), (0, 90), (1, 545)):
        if which == "k":
            c.k[b][at] = -(c.k[b][at].abs() + 1) * 2.0 ** power
        else:
            c.v[b][at] *= 2.0 ** power
    c.check()


def test_write_does_not_depend_on_how_heads_are_dealt_to_warps(monkeypatch):
    """One pair of heads a warp up to eight, for a device of many and of few SMs."""
    from test_gpu_kv4 import _empty, _write_case
    T, hq, hkv, bs = 33, 40, 9, 32
    nb, qkv, qw, kw, cs, pos, slots = _write_case(T, hq, hkv, bs, 21, (4,))
    args = [x.to(DEV) for x in (qkv, qw, kw)] + [1e-6] + [x.to(DEV) for x in (cs, pos, slots)]
    st, runs = _cuda()._kv4_state(args[0]), []
    for sms in (1000, 148, 10, 5, 4, 3, 2, 1):
        monkeypatch.setattr(st, "num_sms", sms)
        caches = _empty(nb, hkv, bs)
        runs.append((_ops().qk_norm_rope_cache(*args, *caches, hq, hkv, D), *caches))
    _cuda().check_status()
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


# ---- the engine on long contexts ----

@pytest.fixture(scope="module")
def long_model_dir(tmp_path_factory):
    from xixi_vllm_b200.models.synth import make_model_dir
    return make_model_dir(str(tmp_path_factory.mktemp("kv4_long")), "tiny", std=0.08, num_hidden_layers=2, hidden_size=512,
                          num_attention_heads=4, num_key_value_heads=2, head_dim=128, intermediate_size=1024, vocab_size=2048,
                          torch_dtype="bfloat16", tie_word_embeddings=False, max_position_embeddings=32768)


@pytest.mark.parametrize("lens,context,batched", [((9, 40, 1500), 4096, 256), ((9, 40, 17500, 3000), 20480, 2048)])
def test_engine_forwards_agree_on_long_contexts(long_model_dir, monkeypatch, lens, context, batched):
    """Captured decode over wide tables and mixed steps whose chunk lies behind a long prefix: even shares and split chunks, one
    after the other in the native executor's one scratch buffer, layer by layer. The Python forward gives every call scratch of
    its own; both capture the same shapes, so the tokens are identical."""
    from test_gpu_kv4 import _engine, _prompts
    L = _cuda().lib()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert L.xv_kv4_prefill_splits(1, batched, 4, 2, max(lens), sms) > 1
    assert (L.xv_kv4_decode_splits(2, 2, sms, context) == 0) == (context > 16384) == (L.xv_kv4_decode_splits(2, 2, sms, max(lens)) == 0)
    kw = dict(context_len=context, max_num_batched_tokens=batched, num_kvcache_blocks=1600, enforce_eager=False)
    prompts = _prompts(lens, 5)
    native = _engine(long_model_dir, prompts, 40, **kw)
    monkeypatch.setenv("XV_NATIVE_FORWARD", "0")
    assert native == _engine(long_model_dir, prompts, 40, **kw)


@pytest.mark.parametrize("hq", [4, 6, 16])
@pytest.mark.parametrize("group", [0, 1])
@pytest.mark.parametrize("extra_pages", [1, WIDE])
def test_decode_nan_in_a_group_of_v_stays_in_its_channels(hq, group, extra_pages):
    """At every number of heads to a KV head: up to four have columns for each group, more of them share."""
    c = Case([1, 1], [50, 61], hq, 1, n_decode=2, extra_pages=extra_pages, seed=22)
    of = torch.arange(D) // 8 % 2 == group
    c.v[0][33, 0, of] = 0.0
    clean = c.run()
    c.v[0][33, 0, 8 * group + 3] = float("inf")
    out = c.run()
    assert bool(out[0][:, of].isnan().all())
    out[0][:, of] = clean[0][:, of]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_tokens_of_every_size(crowd):
    """V of 2^-100 to 2^100 token by token, with weights and without; and tokens of 2^-6 between ordinary ones, in a tile with one
    of 2^22 that the rows before it do not see."""
    c = Case([100, 30], [100, 560], 4, 1, extra_pages=300, seed=23, crowd=crowd)
    ordinary = [v.clone() for v in c.v]
    g = torch.Generator().manual_seed(23)
    c.v = [v * torch.exp2(torch.rand(len(v), 1, 1, generator=g) * 200 - 100) for v in c.v]
    c.check()
    c.q *= 0.0
    c.check()
    c.v = ordinary
    c.v[0][1::2] *= 2.0 ** -6
    c.v[0][90] *= 2.0 ** 22
    c.check()


@pytest.mark.parametrize("crowd", [0, 160])
def test_chunk_large_values_without_weight_in_front_of_small_ones(crowd):
    """Tiles of V of 2^80 (and single tokens of it) whose scores are hundreds below the others': nothing of them may be left,
    nor anything of the others lost."""
    c = Case([100], [640], 4, 1, extra_pages=300, seed=24, crowd=crowd)
    c.q = 2.5 * (c.q.abs() + 0.5)
    c.k[0] = c.k[0].abs() + 2
    low = torch.zeros(640, dtype=torch.bool)
    low[128:256] = low[[300, 520, 560, 600]] = True
    c.k[0][low] *= -1
    c.v[0][low] *= 2.0 ** 80
    c.check()


@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("power,weight", [(-60, 0), (-80, 0), (-110, 0), (-130, 0), (0, -120), (-40, -90)])
def test_write_of_small_keys_matches_the_cpu_backend(eps, power, weight):
    """K rows whose squares, and products with the weights, leave fp32; without an eps the norm brings them back to size."""
    from test_gpu_kv4 import _empty, _write_case
    T, hq, hkv, bs = 65, 2, 3, 16
    nb, qkv, qw, kw, cs, pos, slots = _write_case(T, hq, hkv, bs, 31)
    k = qkv[:, hq * D:(hq + hkv) * D]
    k.copy_((k.double() * 2.0 ** power).bfloat16())
    kw = (kw.double() * 2.0 ** weight).bfloat16()
    gpu = _empty(nb, hkv, bs)
    cpu = [c.cpu() for c in gpu]
    _ops().qk_norm_rope_cache(*[x.to(DEV) for x in (qkv, qw, kw)], eps, *[x.to(DEV) for x in (cs, pos, slots)], *gpu, hq, hkv, D)
    _ops().qk_norm_rope_cache(qkv, qw, kw, eps, cs, pos, slots, *cpu, hq, hkv, D)
    _cuda().check_status()
    a, b = (kv4.read_rows(c.cpu(), slots.long()) for c in (gpu[0], cpu[0]))
    assert bool(b.isfinite().all()) and bool(b.any())
    # at this step the quantiser's own last bit below 2^-102 is left out of it
    quantum = 2.0 ** -100 if float(b.abs().max()) < 2.0 ** -90 else 0.0
    assert float((a - b).abs().max()) <= quantum


@pytest.mark.parametrize("power", [-63, -64, -66, -95, -104, -118, -124, -127, -131])
def test_write_of_small_values_matches_the_cpu_backend(power):
    """Groups whose quotients' remainders, steps or centres are below fp32's smallest normal number."""
    from test_gpu_kv4 import _empty, _write_case
    T, hq, hkv, bs = 600, 0, 2, 16
    nb, qkv, qw, kw, cs, pos, slots = _write_case(T, hq, hkv, bs, 32)
    g = torch.Generator().manual_seed(32)
    v = qkv[:, hkv * D:]
    v.copy_((torch.randn(v.shape, generator=g).double() * 2.0 ** power).bfloat16())
    v[100:200].abs_()
    v[200:300, ::2] = 0.0
    v[300:310] = v[300:310, :1]                                # constant groups
    gpu = _empty(nb, hkv, bs)
    cpu = [c.cpu() for c in gpu]
    _ops().qk_norm_rope_cache(*[x.to(DEV) for x in (qkv, qw, kw)], 1e-6, *[x.to(DEV) for x in (cs, pos, slots)], *gpu, hq, hkv, D)
    _ops().qk_norm_rope_cache(qkv, qw, kw, 1e-6, cs, pos, slots, *cpu, hq, hkv, D)
    _cuda().check_status()
    for a, b in zip(gpu, cpu):
        assert torch.equal(a.cpu(), b)


def test_long_padding_is_cleared():
    """Thousands of rows behind one short chunk, and behind chunks of which one is long."""
    for q_lens, most in (([61], 61), ([300] + [1] * 40, 300), ([5, 3], 4000)):
        c = Case(q_lens, [n + 20 for n in q_lens], 4, 2, n_decode=0, seed=33)
        k, v = (x.to(DEV) for x in c.caches())
        rows = sum(q_lens)
        q = torch.cat([c.q, torch.ones(9000 - rows, 4, D)]).bfloat16().flatten(1).to(DEV)
        want = c.run().flatten(1).to(DEV)
        torch.full_like(q, 7.0)                              # what the allocator may hand out again
        attn = c.attn()
        attn.max_q_len = most
        got = _ops().paged_attention(q, k, v, attn, SCALE, 4, 2, D)
        _cuda().check_status()
        torch.testing.assert_close(got[:rows], want, rtol=2 * HALF_BF16, atol=2.0 ** -8)
        assert not got[rows:].any()


@pytest.mark.parametrize("hq", [4, 6, 16])
@pytest.mark.parametrize("power", [30, 75])
@pytest.mark.parametrize("extra_pages", [1, WIDE])
def test_decode_large_values_without_weight(hq, power, extra_pages):
    """V of 2^30 and 2^75 at tokens that all heads but one give no weight: those heads see nothing of it, in nor beside their sums."""
    c = Case([1, 1], [70, 700], hq, 1, n_decode=2, extra_pages=extra_pages, seed=25)
    for b, k in enumerate(c.k):
        at = [3, 40] if b == 0 else [5, 330, 331, 650]
        k[at] = 0.0
        k[at, :, 0] = -40.0                                  # channel 0 decides: far below for heads with a positive q
        c.v[b][at] *= 2.0 ** power
        c.q[b, :, 0] = 100.0
        c.q[b, 1, 0] = -1.0                                  # and far above for head 1
        k[[i for i in range(len(k)) if i not in at], :, 0] = 0.0
    c.check()


@pytest.mark.parametrize("hq", [4, 6])
@pytest.mark.parametrize("extra_pages", [1, WIDE])
def test_decode_large_values_of_many_tokens(hq, extra_pages):
    """Sums over 1500 tokens of V of 2^112: scaled sums and centres must stay in fp32."""
    c = Case([1, 1], [70, 1500], hq, 1, n_decode=2, extra_pages=extra_pages, seed=26)
    c.q *= 0.1
    c.v = [(v.abs() + 1) * 2.0 ** 112 for v in c.v]
    c.check()
