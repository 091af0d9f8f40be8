"""4-bit KV cache on the CPU backend: byte format, quantiser, refusals and the engine that uses it."""
import os

import numpy as np
import pytest
import torch

import kv4_ref
from xixi_vllm_b200.ops import cpu_ref, dispatch as ops, kv4
from xixi_vllm_b200.runtime.staging import AttnBatch


def caches(nb, heads, bs, d):
    return tuple(torch.zeros(nb, heads, bs, kv4.row_bytes(d), dtype=torch.uint8) for _ in range(2))


@pytest.mark.parametrize("d", [16, 64, 128])
def test_quantise_matches_the_definition_in_64_bits(d):
    g = torch.Generator().manual_seed(d)
    x = torch.randn(200, d, generator=g) * torch.exp(2 * torch.randn(200, 1, generator=g))
    x[3], x[4, ::2], x[5] = 0.7, 5.0, 0.0
    x = x.bfloat16()
    got = kv4.dequantize(*kv4.quantize(x)).double().numpy()
    want = kv4_ref.levels(x.double().numpy())
    # c + s (n - 8) in fp32 rounds once
    np.testing.assert_allclose(got, want, rtol=2.0 ** -23, atol=0)


def test_quantise_error_is_half_a_step_and_constant_groups_are_exact():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(500, 128, generator=g).bfloat16()
    x[0] = -3.25
    codes, par = kv4.quantize(x)
    err = kv4._to_groups((kv4.dequantize(codes, par) - x.float()).abs())
    step = par[..., 0:1].float()
    centre = par[..., 1:2].float().abs()
    # half a step; the ends of the range move by the rounding of s (7.5 steps of 2^-8) and of c
    assert bool((err <= step * (0.5 + 7.5 * 2.0 ** -8) + centre * 2.0 ** -8 + 1e-6).all())
    assert torch.equal(kv4.dequantize(codes, par)[0], x[0].float())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_group_with_a_non_finite_value_reads_back_as_nan_and_the_other_group_does_not(value):
    x = torch.randn(2, 128, generator=torch.Generator().manual_seed(2))
    x[0, 9] = value                              # word 1: group 1
    y = kv4.dequantize(*kv4.quantize(x))
    odd = (torch.arange(128) // 8) % 2 == 1
    assert bool(y[0, odd].isnan().all()) and bool(y[0, ~odd].isfinite().all()) and bool(y[1].isfinite().all())


def test_largest_and_smallest_values():
    big = 2.0 ** 126                             # eight steps of the largest bf16 would leave fp32
    x = torch.zeros(3, 128)
    x[0, 0], x[0, 1] = big, -big
    x[1, 0] = 1e-38                              # a step below the smallest normal number counts as 0
    x[2] = 2.0 ** -126
    y = kv4.dequantize(*kv4.quantize(x))
    assert bool(y.isfinite().all())
    assert float((y[0, :2] - x[0, :2]).abs().max()) <= big / 15
    assert float((y[1] - x[1]).abs().max()) <= 1e-38
    assert torch.equal(y[2], x[2])


@pytest.mark.parametrize("d,bs", [(64, 16), (128, 48)])
def test_rows_land_where_the_format_says(d, bs):
    k, _ = caches(3, 2, bs, d)
    x = torch.randn(5, 2, d, generator=torch.Generator().manual_seed(3))
    slots = torch.tensor([0, bs + 15, 2 * bs + 1, bs - 1, 2 * bs + 10])
    kv4.write_rows(k, slots, x)
    want = kv4_ref.levels(x.bfloat16().double().numpy())
    got, _ = kv4_ref.rows(k, slots.tolist())
    np.testing.assert_allclose(got, want, rtol=1e-12)
    np.testing.assert_allclose(kv4.read_rows(k, slots).numpy(), want, rtol=2.0 ** -23)
    untouched, _ = kv4_ref.rows(k, [1, bs, 2 * bs])
    assert not untouched.any()


def test_read_cache_negative_slots_and_repeats():
    k, v = caches(2, 1, 16, 64)
    kv4.write_rows(k, torch.tensor([5]), torch.ones(1, 1, 64))
    kv4.write_rows(v, torch.tensor([5]), torch.full((1, 1, 64), 2.0))
    kk, vv = ops.read_cache(k, v, torch.tensor([5, -1, 5], dtype=torch.int32), 64)
    assert kk.dtype == torch.bfloat16 and kk.shape == (3, 1, 64)
    assert kk[:, 0, 0].tolist() == [1, 0, 1] and vv[:, 0, 0].tolist() == [2, 0, 2]
    e, _ = ops.read_cache(k, v, torch.zeros(0, dtype=torch.int32), 64)
    assert e.shape == (0, 1, 64)


def test_refusals():
    k, v = caches(2, 1, 16, 64)
    s = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError, match="uint8"):
        ops.read_cache(k, v.float(), s, 64)
    with pytest.raises(TypeError, match="uint8"):
        ops.read_cache(torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16), s, 64)
    with pytest.raises(ValueError, match="expected"):
        ops.read_cache(k, v, s, 128)                              # row size of another head_dim
    with pytest.raises(ValueError, match="one 4-d shape"):
        ops.read_cache(k, v[:1], s, 64)
    with pytest.raises(ValueError, match="contiguous"):
        ops.read_cache(k.repeat(1, 2, 1, 1).transpose(0, 1), v.repeat(1, 2, 1, 1).transpose(0, 1), s, 64)
    with pytest.raises(ValueError, match="expected"):
        kv4.check_caches(k[:, :, :8], v[:, :, :8], 64)            # a page of half a unit
    with pytest.raises(ValueError, match="head_dim % 16"):
        kv4.row_bytes(72)


def test_the_cpu_form_refuses_what_the_kernels_refuse():
    """Writing and attending, with caches that do not fit each other or the call, scales and pages that mean nothing."""
    hq, hkv, d, bs = 4, 2, 64, 16
    k, v = caches(3, hkv, bs, d)
    i32 = dict(dtype=torch.int32)
    cs, w = cpu_ref.build_cos_sin_cache(d, 10, 1e4), torch.ones(d)
    wide = torch.zeros(3, hkv, bs, d)

    def write(k, v, qkv=torch.ones(1, (hq + 2 * hkv) * d), hkv=hkv):
        return ops.qk_norm_rope_cache(qkv, w, w, 1e-6, cs, torch.zeros(1, **i32), torch.zeros(1, **i32), k, v, hq, hkv, d)

    def attend(k, v, scale=0.1, hq=hq, hkv=hkv, pages=(0, 1), length=20):
        attn = AttnBatch(torch.tensor([0, 1], **i32), torch.tensor([length], **i32), torch.tensor([pages], **i32), 1, 1, 1, length, 1)
        return ops.paged_attention(torch.ones(1, 4 * d), k, v, attn, scale, hq, hkv, d)

    write(k, v)
    assert bool(attend(k, v).isfinite().all())
    for call in (write, attend):
        for bad in ((k, wide), (wide, v)):
            with pytest.raises(TypeError, match="uint8"):
                call(*bad)
        with pytest.raises(ValueError, match="one 4-d shape"):
            call(k, v[:2])
        with pytest.raises(ValueError, match="expected"):
            call(k[:, :, :8].contiguous(), v[:, :, :8].contiguous())
        with pytest.raises(ValueError, match="expected"):
            call(k, v, hkv=1)
        with pytest.raises(ValueError, match="contiguous"):
            call(k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(0, 1).contiguous().transpose(0, 1))
    assert not bool(wide.any())
    with pytest.raises(ValueError, match="qkv of shape"):
        write(k, v, torch.ones(1, (hq + 2 * hkv) * d + 8))
    with pytest.raises(ValueError, match="q of shape"):
        attend(k, v, hq=3)
    for scale in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="finite"):
            attend(k, v, scale)
    for pages, length in (((0, 3), 20), ((0, -1), 20), ((0, 1), 33)):
        with pytest.raises(IndexError, match="pages"):
            attend(k, v, pages=pages, length=length)


def test_append_then_attend_matches_64_bits():
    torch.manual_seed(0)
    hq, hkv, d, bs = 4, 2, 64, 32
    k, v = caches(6, hkv, bs, d)
    T = 41
    qkv = torch.randn(T, (hq + 2 * hkv) * d)
    cs = cpu_ref.build_cos_sin_cache(d, 100, 1e4)
    w = torch.ones(d)
    table = torch.tensor([[4, 2]], dtype=torch.int32)
    slots = torch.tensor([int(table[0, t // bs]) * bs + t % bs for t in range(T)], dtype=torch.int32)
    slots_w = slots.clone()
    q = ops.qk_norm_rope_cache(qkv, w, w, 1e-6, cs, torch.arange(T, dtype=torch.int32), slots_w, k, v, hq, hkv, d)
    want_v = kv4_ref.levels(qkv[:, (hq + hkv) * d:].view(T, hkv, d).bfloat16().double().numpy())
    np.testing.assert_allclose(kv4_ref.rows(v, slots.tolist())[0], want_v, rtol=1e-12)
    attn = AttnBatch(cu_q=torch.tensor([0, T], dtype=torch.int32), kv_lens=torch.tensor([T], dtype=torch.int32),
                     block_tables=table, num_seqs=1, num_decode=0, max_q_len=T, max_kv_len=T, num_tokens=T)
    out = ops.paged_attention(q, k, v, attn, d ** -0.5, hq, hkv, d)
    ref, *_ = kv4_ref.attention(q, k, v, [T], [T], table, d ** -0.5, hq)
    np.testing.assert_allclose(out.view(T, hq, d).numpy(), ref, atol=1e-5)


def test_what_a_row_does_not_see_cannot_reach_it():
    """NaN under a negative slot, NaN at later positions of a chunk, rows before position 0 and behind the last sequence."""
    hq, hkv, d, n = 2, 1, 64, 6
    k, v = (torch.zeros(2, hkv, 16, kv4.row_bytes(d), dtype=torch.uint8) for _ in range(2))
    g = torch.Generator().manual_seed(3)
    x = torch.randn(n, hkv, d, generator=g)
    kv4.write_rows(k, torch.arange(n), x)
    nan = x.clone()
    nan[4] = float("nan")
    q = torch.randn(n + 1, hq * d, generator=g)
    table = torch.tensor([[0]], dtype=torch.int32)
    i32 = dict(dtype=torch.int32)

    def run(rows, length=n):
        attn = AttnBatch(cu_q=torch.tensor([0, rows], **i32), kv_lens=torch.tensor([length], **i32), block_tables=table, num_seqs=1,
                         num_decode=0, max_q_len=rows, max_kv_len=length, num_tokens=rows)
        return ops.paged_attention(q, k, v, attn, 0.125, hq, hkv, d)

    kv4.write_rows(v, torch.arange(n), x)
    clean = run(n)
    assert not clean[n].any()
    late = run(n, 4)
    assert not late[:2].any() and bool(late[2:n].isfinite().all()) and bool(late[2:n].any(-1).all())
    kv4.write_rows(v, torch.arange(n), nan)
    out = run(n)
    assert torch.equal(out[:4], clean[:4]) and bool(out[4:n].isnan().all())
    kv4.write_rows(k, torch.tensor([0]), torch.full((1, hkv, d), float("nan")))
    rows, _ = ops.read_cache(k, v, torch.tensor([-1, 0, 1], dtype=torch.int32), d)
    assert not rows[0].any() and bool(rows[1].isnan().all()) and bool(rows[2].isfinite().all())


def test_an_extension_of_another_torch_is_built_again(tmp_path, monkeypatch):
    from xixi_vllm_b200.ops import build
    lib = tmp_path / "_xv_torch.so"
    monkeypatch.setattr(build, "TORCH_LIB", str(lib))
    runs = []

    def compiler(cmd, **kw):
        runs.append(cmd)
        mark = next(a for a in cmd if a.startswith("-DXV_BUILT_FOR=")).split('"')[1]
        with open(cmd[cmd.index("-o") + 1], "wb") as f:
            f.write(b"code " + mark.encode() + b" code")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build_torch()                                       # not there
    build.build_torch()                                       # fits
    assert len(runs) == 1
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    build.build_torch()                                       # newer than its sources, but of another torch
    build.build_torch()
    assert len(runs) == 2 and b"torch 1.0.0 " in lib.read_bytes()
    os.utime(lib, (0, 0))
    build.build_torch()                                       # older than its sources
    assert len(runs) == 3


def test_the_native_forwards_scratch_covers_every_step():
    """Over a grid of head counts, sequences, chunk and table lengths: what a launch asks for is never more than it has."""
    from xixi_vllm_b200.ops import cuda
    from xixi_vllm_b200.runtime.native_forward import kv4_scratch_bytes
    L = cuda.lib()
    split = shared = 0
    for hq, hkv in ((1, 1), (4, 2), (5, 1), (16, 1), (12, 1), (32, 8), (40, 8), (8, 8)):
        for sms in (148, 132, 20):
            for most in (1, 7, 64, 300):
                have = kv4_scratch_bytes(L, most, hq, hkv, sms)
                for n in {1, 2, most // 3 + 1, most}:
                    for reach in (16, 500, 512, 2100, 5000, 20480, 131072):
                        splits = L.xv_kv4_decode_splits(n, hkv, sms, reach)
                        assert L.xv_kv4_decode_workspace_bytes(n, hq, hkv, splits, sms) <= have
                        shared += splits == 0
                        for q in (0, 1, 63, 64, 65, 700, 4096):
                            splits = L.xv_kv4_prefill_splits(n, q, hq, hkv, reach, sms)
                            assert splits >= 1 and L.xv_kv4_prefill_workspace_bytes(n, q, hq, hkv, splits) <= have
                            split += splits > 1
    assert split > 1000 and shared > 500


# ---- the engine with kv_cache_dtype="int4" ----

def _generate(model_dir, prompts, max_tokens=8, **kw):
    from xixi_vllm_b200 import Engine, EngineConfig, SamplingParams
    base = dict(device="cpu", dtype="float32", num_kvcache_blocks=128, max_num_seqs=8, max_num_batched_tokens=64,
                context_len=256, kv_cache_dtype="int4")
    base.update(kw)
    eng = Engine(EngineConfig(model=model_dir, **base))
    try:
        seqs = [eng.add_request(p, SamplingParams(max_tokens=max_tokens, ignore_eos=True)) for p in prompts]
        while eng.has_unfinished():
            eng.step()
        return [s.token_ids[s.num_prompt_tokens:] for s in seqs]
    finally:
        eng.destroy()


def _prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1024, (n,), generator=g).tolist() for n in lens]


def test_engine_runs_on_a_4_bit_cache_and_scheduling_does_not_change_tokens(tiny_model_dir):
    """Chunked prefill, a shared prefix and preemption read pages that other steps wrote."""
    shared = _prompts([40], 5)[0]
    prompts = [shared + p for p in _prompts([9, 30, 3, 17], 6)]
    whole = _generate(tiny_model_dir, prompts, prefix_backend="none", max_num_batched_tokens=512)
    assert all(len(t) == 8 for t in whole)
    assert _generate(tiny_model_dir, prompts, prefix_backend="radix", max_num_batched_tokens=32) == whole
    assert _generate(tiny_model_dir, prompts, prefix_backend="none", num_kvcache_blocks=14) == whole
    assert _generate(tiny_model_dir, prompts, kvcache_block_size=48, async_scheduling="on") == whole


def test_engine_tp2_on_a_4_bit_cache_equals_one_rank(tiny_model_dir):
    prompts = _prompts([16, 5, 33], 7)
    assert _generate(tiny_model_dir, prompts, tp_size=2, nccl_port=29911) == _generate(tiny_model_dir, prompts)


def test_pool_sizes_and_reads_its_tokens(tiny_model_dir):
    from xixi_vllm_b200.config import load_model_config
    from xixi_vllm_b200.parallel import groups
    from xixi_vllm_b200.runtime.kv_pool import KVPool
    groups.single_process_groups()
    try:
        cfg = load_model_config(tiny_model_dir)
        pools = {t: KVPool(cfg, num_blocks=4, block_size=32, device="cpu", dtype=torch.bfloat16, cache_dtype=t)
                 for t in ("auto", "int4")}
        assert pools["auto"].bytes_per_block == 2 * 2 * 2 * 32 * 128
        assert pools["int4"].bytes_per_block == 2 * 2 * 2 * 32 * 40
        assert all(p.kv_cache.numel() * p.kv_cache.element_size() == 4 * p.bytes_per_block for p in pools.values())
        n = {t: KVPool.auto_num_blocks(cfg, block_size=32, dtype=torch.bfloat16, device="cpu", gpu_memory_utilization=0.9,
                                       cache_dtype=t) for t in pools}
        assert n["int4"] == n["auto"] * 128 // 40
        slots = torch.tensor([33, 2], dtype=torch.int32)
        x = torch.randn(2, 2, 64).bfloat16()
        for name, p in pools.items():
            for c in (p.k_cache(1), p.v_cache(1)):
                if name == "int4":
                    kv4.write_rows(c, slots, x)
                else:
                    c[slots.long() // 32, :, slots.long() % 32] = x
            k, v = p.read_tokens(1, slots)
            assert k.shape == x.shape and torch.equal(k, v)
            assert float((k - x).float().abs().max()) <= (0 if name == "auto" else 0.3)
            k, v = p.read_tokens(1, torch.tensor([-1, 33], dtype=torch.int32))
            assert not k[0].any() and not v[0].any() and bool(k[1].any())
    finally:
        groups.destroy_model_parallel()


def test_configuration_and_command_lines(tiny_model_dir, tmp_path):
    import run
    from xixi_vllm_b200 import EngineConfig
    from xixi_vllm_b200.models.synth import make_model_dir
    from xixi_vllm_b200.utils.run_utils import engine_config_from
    assert EngineConfig(model=tiny_model_dir, device="cpu").kv_cache_dtype == "auto"
    with pytest.raises(ValueError, match="kv_cache_dtype must be"):
        EngineConfig(model=tiny_model_dir, device="cpu", kv_cache_dtype="int8")
    with pytest.raises(ValueError, match="head_dim 128"):
        EngineConfig(model=tiny_model_dir, device="cuda", kv_cache_dtype="int4")      # head_dim 64
    with pytest.raises(ValueError, match="head_dim"):
        EngineConfig(model=make_model_dir(str(tmp_path), "tiny", weights=False, head_dim=40), device="cpu", kv_cache_dtype="int4")
    args = run.build_parser().parse_args(["--model", tiny_model_dir, "--device", "cpu", "--kv-cache-dtype", "int4"])
    assert engine_config_from(run.config_from_args(args), tiny_model_dir).kv_cache_dtype == "int4"


def test_the_benchmark_takes_the_caches_form(monkeypatch):
    import importlib.util
    import sys
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bench.py")
    spec = importlib.util.spec_from_file_location("bench_script", path)
    bench = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bench)
    monkeypatch.setattr(sys, "argv", ["bench.py"])
    assert bench.parse_args().kv_cache_dtype == "auto"
    monkeypatch.setattr(sys, "argv", ["bench.py", "--mode", "decode", "--kv-cache-dtype", "int4"])
    assert bench.parse_args().kv_cache_dtype == "int4"
