"""Entry points used by model code. A CUDA tensor goes to the sm_100a kernels, a CPU tensor
to the PyTorch oracle. There is exactly one GPU implementation per op; if the CUDA library
is missing on a machine with a GPU the call raises instead of falling back.
"""

from __future__ import annotations

import math

import torch

from . import cpu_ref, kv4

__all__ = [
    "rmsnorm", "add_rmsnorm", "linear", "linear_silu_mul", "silu_mul", "embedding", "qk_norm_rope_cache",
    "read_cache", "paged_attention", "sample", "argmax", "build_cos_sin_cache", "gather_rows",
    "resolve_token_refs",
]

build_cos_sin_cache = cpu_ref.build_cos_sin_cache


_cuda_ops = None


def _cuda():
    global _cuda_ops
    if _cuda_ops is None:
        from . import cuda

        _cuda_ops = cuda
    return _cuda_ops


def rmsnorm(x, w, eps):
    return _cuda().rmsnorm(x, w, eps) if x.is_cuda else cpu_ref.rmsnorm(x, w, eps)


def add_rmsnorm(x, residual, w, eps):
    return _cuda().add_rmsnorm(x, residual, w, eps) if x.is_cuda else cpu_ref.add_rmsnorm(x, residual, w, eps)


def linear(x, w, bias=None, out=None, defer=False):
    """``defer=True`` lets the GPU GEMM hand back unreduced split-K partials; only pass the result
    to ``add_rmsnorm`` or ``qk_norm_rope_cache`` (they sum the partials themselves)."""
    if x.is_cuda:
        return _cuda().linear(x, w, bias, out, defer)
    y = cpu_ref.linear(x, w, bias)
    if out is not None:
        out.copy_(y)
        return out
    return y


def linear_silu_mul(x, w):
    """GPU only: fused gate/up projection + SiLU-mul over an interleaved weight (see ops.cuda)."""
    return _cuda().linear_silu_mul(x, w)


def silu_mul(x):
    return _cuda().silu_mul(x) if x.is_cuda else cpu_ref.silu_mul(x)


def embedding(ids, w, vocab_start=0, out=None):
    if w.is_cuda:
        return _cuda().embedding(ids, w, vocab_start, out)
    y = cpu_ref.embedding(ids, w, vocab_start)
    if out is not None:
        out.copy_(y)
        return out
    return y


def qk_norm_rope_cache(qkv, q_w, k_w, eps, cos_sin, positions, slots, k_cache, v_cache,
                       num_q_heads, num_kv_heads, head_dim, prefill_begin: int = 0):
    """``prefill_begin``: index of the first prefill row of the packed batch (decode rows come first).
    The GPU kernel clears the V rows that follow a prefill chunk's last row inside its page.
    uint8 caches (``ops.kv4``) receive the rows quantised to 4 bits; every other argument is the same. Slots that are
    not negative must be distinct: of two rows for one slot, either may be stored, or a mixture."""
    if qkv.is_cuda:
        return _cuda().qk_norm_rope_cache(qkv, q_w, k_w, eps, cos_sin, positions, slots, k_cache, v_cache,
                                          num_q_heads, num_kv_heads, head_dim, prefill_begin)
    if kv4.is_kv4(k_cache) or kv4.is_kv4(v_cache):
        kv4.check_caches(k_cache, v_cache, head_dim, num_kv_heads)
        if qkv.shape[-1] != (num_q_heads + 2 * num_kv_heads) * head_dim:
            raise ValueError(f"qk_norm_rope_cache: qkv of shape {tuple(qkv.shape)} for {num_q_heads} query and {num_kv_heads} KV heads")
    return cpu_ref.qk_norm_rope_cache(qkv, q_w, k_w, eps, cos_sin, positions, slots, k_cache, v_cache,
                                      num_q_heads, num_kv_heads, head_dim)


def read_cache(k_cache, v_cache, slots, head_dim):
    """What a 4-bit cache holds at ``slots [T]`` (int32, as ``qk_norm_rope_cache`` takes them): bf16 ``k, v`` of shape
    ``[T, kv_heads, head_dim]``. Rows whose slot is negative are zero. A slot may be named any number of times."""
    if k_cache.is_cuda:
        return _cuda().read_cache(k_cache, v_cache, slots, head_dim)
    kv4.check_caches(k_cache, v_cache, head_dim)
    return cpu_ref.read_cache(k_cache, v_cache, slots)


def paged_attention(q, k_cache, v_cache, attn, scale, num_q_heads, num_kv_heads, head_dim):
    """``attn`` is a ``runtime.staging.AttnBatch`` (cu_q, kv_lens, block_tables, decode split). The caches are bf16
    pages or, as uint8, pages held in 4 bits (``ops.kv4``). On a 4-bit cache rows of ``q`` that no sequence names, rows of
    a sequence without cached tokens and rows before position 0 come out as zeros; ``scale`` is finite. On the GPU a chunk
    that is longer than ``attn.max_q_len`` or reaches beyond ``q`` is reported through the status word and is zeros. Finite
    values of any size are taken; a row with a score beyond fp32 is NaN."""
    if q.is_cuda:
        return _cuda().paged_attention(q, k_cache, v_cache, attn, scale, num_q_heads, num_kv_heads, head_dim)
    if kv4.is_kv4(k_cache) or kv4.is_kv4(v_cache):
        kv4.check_caches(k_cache, v_cache, head_dim, num_kv_heads)
        if q.shape[-1] != num_q_heads * head_dim or num_q_heads % num_kv_heads:
            raise ValueError(f"paged_attention: q of shape {tuple(q.shape)} for {num_q_heads} query and {num_kv_heads} KV heads")
        if not math.isfinite(scale):
            raise ValueError("paged_attention: scale must be finite")
    return cpu_ref.paged_attention(q, k_cache, v_cache, attn.cu_q, attn.kv_lens, attn.block_tables,
                                   scale, num_q_heads, num_kv_heads, head_dim)


def argmax(logits):
    return _cuda().argmax(logits) if logits.is_cuda else cpu_ref.argmax(logits)


def sample(logits, temperature, top_k, top_p, min_p, *, rng=None, generator=None):
    """``rng``: device int32 ``[seed, step]`` (GPU path); ``generator``: torch generator (CPU path)."""
    if logits.is_cuda:
        return _cuda().sample(logits, temperature, top_k, top_p, min_p, rng)
    return cpu_ref.sample(logits, temperature, top_k, top_p, min_p, generator)


def resolve_token_refs(ids, prev) -> None:
    """In place: input ids < 0 name rows of the previous step's sample buffer (``-(row) - 1``)."""
    if ids.is_cuda:
        _cuda().resolve_token_refs(ids, prev)
        return
    neg = ids < 0
    if bool(neg.any()):
        ids[neg] = prev[(-ids[neg] - 1).long()].to(ids.dtype)


def gather_rows(x, rows):
    """``x[rows]`` for int32 row indices."""
    if x.is_cuda:
        return _cuda().gather_rows(x, rows)
    return x.index_select(0, rows.long())
