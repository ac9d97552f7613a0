"""Refusals of the paged-cache operators and their host arithmetic (no GPU needed)."""
import math

import pytest
import torch

from kyojin_mac_b200 import _lib, ops


@pytest.fixture(scope="module")
def lib():
    _lib.build()
    return _lib.lib()


def test_operators_take_cuda_tensors_only():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros((2, 2, 64), dtype=torch.float16)
    c = torch.zeros((1, 2, 16, 64), dtype=torch.float16)
    t = torch.zeros((1, 1), dtype=torch.int32)
    for call in (lambda: ops.paged_step(t, i[:1], i[:1], i, i[:1], 16, 2), lambda: ops.paged_release(t, i[:1], torch.ones(1, dtype=torch.bool), i, i[:1], 16),
                 lambda: ops.rope(x, i, torch.zeros(32)), lambda: ops.rope_append(x, x, x, i, i, torch.zeros(32), c, c), lambda: ops.paged_attention(x, c, c, t, i[:1], i, 2)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


P = 64                       # stands for an address that is 16-byte aligned; every call below is refused before anything is read


def test_step_refusals(lib):
    good = dict(lens=P, new=P, free=P, cap=10, count=P, table=P, ld=4, batch=2, cols=4, page=16, rows=5)
    call = lambda **k: lib.kyb_paged_step(*{**good, **k}.values(), P, P, P, P, P, P, P, None)
    for bad in (dict(lens=None), dict(table=None), dict(cap=0), dict(ld=3), dict(batch=0), dict(batch=1 << 24), dict(cols=0), dict(page=0), dict(page=24), dict(page=8), dict(page=512),
                dict(rows=-1), dict(rows=1 << 31)):
        assert call(**bad) == _lib.EINVAL, bad
    assert lib.kyb_paged_release(P, None, P, 4, 2, 4, 16, P, 10, P, P, None) == _lib.EINVAL
    assert lib.kyb_paged_release(P, P, P, 4, 2, 4, 20, P, 10, P, P, None) == _lib.EINVAL


def test_rope_refusals(lib):
    good = dict(q=P, q_t=128, q_h=64, k=P, k_t=64, k_h=64, v=P, v_t=64, v_h=64, pos=P, slots=P, inv=P, tokens=3, hq=2, hkv=1, d=64, rot=64, inter=0, m=1.0, dt=1, qo=P, qo_t=128, qo_h=64,
                kc=P, kc_p=1024, kc_h=1024, vc=P, vc_p=1024, vc_h=1024, pages=2, page=16)
    call = lambda **k: lib.kyb_rope_append(*{**good, **k}.values(), None)
    for bad in (dict(q=None), dict(k=None), dict(slots=None), dict(q=P + 2), dict(vc=P + 8), dict(q_t=100), dict(kc_p=1028), dict(d=60), dict(d=264), dict(rot=0), dict(rot=40), dict(rot=80),
                dict(dt=0), dict(dt=3), dict(hq=-1), dict(hq=0, hkv=0), dict(tokens=-1), dict(tokens=1 << 31), dict(pages=0), dict(page=48)):
        assert call(**bad) == _lib.EINVAL, bad
    assert call(tokens=0) == _lib.OK


def test_attention_refusals(lib):
    good = dict(q=P, q_t=128, q_h=64, k=P, k_p=1024, k_h=1024, v=P, v_p=1024, v_h=1024, pages=2, page=16, table=P, ld=3, cols=3, kv=P, cu=P, batch=1, tokens=3, max_q=3, hq=2, hkv=1, d=64,
                dt=1, scale=0.1, window=0, sinks=0, out=P, o_t=128, o_h=64, ws=P, wsn=1 << 30)
    call = lambda **k: lib.kyb_paged_attention(*{**good, **k}.values(), None)
    for bad in (dict(q=None), dict(v=None), dict(table=None), dict(out=None), dict(q=P + 2), dict(out=P + 4), dict(q_t=100), dict(k_p=1028), dict(o_h=-64), dict(pages=0), dict(pages=1 << 31),
                dict(page=8), dict(page=100), dict(ld=2), dict(cols=0), dict(cols=1 << 28, ld=1 << 28), dict(batch=0), dict(tokens=-1), dict(tokens=1 << 30), dict(max_q=-1), dict(hq=0),
                dict(hq=3, hkv=2), dict(hq=129), dict(d=96), dict(dt=0), dict(scale=math.nan), dict(scale=math.inf), dict(window=-1), dict(sinks=-1), dict(sinks=4)):
        assert call(**bad) == _lib.EINVAL, bad
    assert call(tokens=0) == _lib.OK


def test_rope_frequencies():
    inv, m = ops.rope_frequencies(64, 10000.0, device="cpu")
    assert m == 1.0 and inv.dtype == torch.float32 and torch.allclose(inv.double(), 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64), rtol=1e-7)
    lin, _ = ops.rope_frequencies(64, 10000.0, {"type": "linear", "factor": 4.0}, "cpu")
    assert torch.allclose(lin, inv / 4)
    ntk, _ = ops.rope_frequencies(64, 10000.0, {"type": "ntk", "factor": 4.0}, "cpu")
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(inv[-1]) / 4, rel_tol=1e-6)
    l3, _ = ops.rope_frequencies(128, 500000.0, {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_context": 8192}, "cpu")
    base, _ = ops.rope_frequencies(128, 500000.0, device="cpu")
    turns = 8192 * base.double() / (2 * math.pi)
    assert torch.equal(l3[turns > 4], base[turns > 4]) and torch.allclose(l3[turns < 1], base[turns < 1] / 8) and ((l3 <= base) & (l3 >= base / 8 * 0.999999)).all()
    ya, m = ops.rope_frequencies(128, 10000.0, {"type": "yarn", "factor": 16.0, "original_context": 4096}, "cpu")
    b2, _ = ops.rope_frequencies(128, 10000.0, device="cpu")
    assert math.isclose(m, 0.1 * math.log(16.0) + 1.0) and ya[0] == b2[0] and math.isclose(float(ya[-1]), float(b2[-1]) / 16, rel_tol=1e-6)
    for bad in (dict(rot=20), dict(rot=0), dict(rot=64, base=1.0), dict(rot=64, scaling={"type": "linear"}), dict(rot=64, scaling={"type": "linear", "factor": 0.5}),
                dict(rot=64, scaling={"type": "other", "factor": 2.0}),
                dict(rot=64, scaling={"type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0, "original_context": 8192})):
        with pytest.raises(ValueError):
            ops.rope_frequencies(device="cpu", **bad)
