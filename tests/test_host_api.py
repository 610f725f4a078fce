"""Host-side contract of the drop-in wrappers (no GPU needed: these raise before any launch)."""
import pytest
import torch


def _qkv():
    q = torch.zeros(1, 4, 2, 128)
    return q, q.clone(), q.clone()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_dtype_other_than_bf16_raises(dtype):
    """The reference computes in ``dtype`` (attention.py:1134-1141); these kernels compute in
    bf16, so asking for another dtype raises rather than silently returning bf16 accuracy."""
    from lbw_amd import attention, cross_attention, exact_attention, exact_attention_chunks
    q, k, v = _qkv()
    with pytest.raises(NotImplementedError, match="bfloat16"):
        attention(q, k, v, dtype=dtype)
    with pytest.raises(NotImplementedError, match="bfloat16"):
        exact_attention(q, k, v, dtype=dtype)
    with pytest.raises(NotImplementedError, match="bfloat16"):
        exact_attention_chunks(q, [k], [v], dtype=dtype)
    with pytest.raises(NotImplementedError, match="bfloat16"):
        cross_attention(q, k, v, dtype=dtype)


def test_unsupported_options_raise():
    from lbw_amd import attention
    q, k, v = _qkv()
    with pytest.raises(NotImplementedError):
        attention(q, k, v, causal=True)
    with pytest.raises(NotImplementedError):
        attention(q, k, v, dropout_p=0.1)
    with pytest.raises(NotImplementedError):
        attention(q, k, v, window_size=(4, 4))


def test_cpu_tensors_are_rejected_loudly():
    """No CPU fallback: host tensors reach the device check and raise."""
    from lbw_amd import attention
    q, k, v = _qkv()
    with pytest.raises(RuntimeError, match="GPU tensor"):
        attention(q.to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16))


def test_bench_refuses_more_than_one_gpu():
    """bench.py measures one GPU: --gpus above 1 (or a multi-rank launch) exits with status 2 and
    says so, before touching a device."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for argv, env in ((["--gpus", "2"], {}), ([], {"WORLD_SIZE": "2"})):
        r = subprocess.run([sys.executable, os.path.join(root, "bench.py"), *argv],
                           capture_output=True, text=True, timeout=120,
                           env={**os.environ, **env})
        assert r.returncode == 2, (argv, env, r.stdout, r.stderr)
        assert "one GPU" in r.stdout + r.stderr


def _writers():
    """Op -> (its call on tensors without memory, the tensors that it writes): the write is what counts here."""
    import itertools
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="meta")  # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device="meta")  # noqa: E731
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="meta")  # noqa: E731
    x, row, w, table = bf(1, 8, 2, 128), bf(8, 256), bf(256), f32(8, 64, 2)
    part = ([f32(1, 2, 8, 128)], [f32(1, 2, 8)], [f32(1, 2, 8)])
    outs = [bf(1, 8, 2, 128) for _ in range(5)]
    rows = [bf(8, 256) for _ in range(3)]
    codes, scales = u8(1, 8, 2, 128), f32(1, 2, 1)
    ops = torch.ops.lbw
    o = iter(outs)
    calls = {
        "attention_out": lambda t: ops.attention_out(x, [x], [x], 0, -1, None, 0.0, 0, t),
        "cross_attention_out": lambda t: ops.cross_attention_out(x, x, x, None, -1, 0, -1, 0.0, t),
        "attention_fp8kv_out": lambda t: ops.attention_fp8kv_out(x, [u8(1, 8, 2, 128)], [u8(1, 8, 2, 128)], [scales],
                                                                 [scales], 0, -1, 0.0, 0, t),
        "attention_chain_out": lambda t: ops.attention_chain_out(x, [x], [x], None, None, None, 0, -1, 0.0, t),
        "attention_merge_out": lambda t: ops.attention_merge_out(*part, t),
    }
    res = {n: (f, [next(o)]) for n, f in calls.items()}
    res["qk_norm_rope_"] = (lambda a, b, c: ops.qk_norm_rope_(row, row, None, None, w, w, table, [8, 1, 1], 1e-6, 2, a,
                                                              b, row, c, 1.0, 1.0, 0), rows)
    res["kv_quant_fp8_"] = (lambda a, b: ops.kv_quant_fp8_(x, a, b), [codes, scales.clone()])
    assert len(set(map(id, itertools.chain(*(t for _, t in res.values()))))) == 10
    return res


@pytest.mark.parametrize("op", ["attention_out", "cross_attention_out", "attention_fp8kv_out", "attention_chain_out",
                                "attention_merge_out", "qk_norm_rope_", "kv_quant_fp8_"])
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_writes_are_counted(op, mode):
    """A backward pass that saved a tensor which one of these ops overwrites must be able to tell."""
    from lbw_amd import _lib
    _lib.ops()
    call, outs = _writers()[op]
    before = [t._version for t in outs]
    with mode():
        call(*outs)
    assert [t._version for t in outs] == [n + 1 for n in before]
    h = torch.zeros_like(outs[0], dtype=torch.float32).requires_grad_() * 1
    y = (h * h).sum()
    call(h.detach(), *outs[1:])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        outs = [torch.zeros_like(t) for t in outs]
        call(*outs)                               # inference tensors, which have no count
    with torch.no_grad():
        call(*outs)
