"""Refusals of the paged-cache operators and their host arithmetic (no GPU needed)."""
import math
import os
import re

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


def _call(entry, block, good, **other):
    return entry(block.pack(*{**good, **other}.values()), None)


def test_step_refusals(lib):
    good = dict(lens=P, new=P, free=P, count=P, table=P, cu=P, kv=P, pos=P, slots=P, lens_out=P, count_out=P, refused=P, cap=10, ld=4, batch=2, cols=4, page=16, rows=5)
    for bad in (dict(lens=0), dict(table=0), dict(slots=0), dict(cap=0), dict(cap=1 << 31), dict(ld=3), dict(batch=0), dict(batch=1 << 24), dict(cols=0), dict(page=0), dict(page=24), dict(page=8),
                dict(page=512), dict(page=16 + (1 << 32)), dict(page=-16), dict(rows=-1), dict(rows=1 << 31)):
        assert _call(lib.kyb_paged_step, _lib.PAGED_STEP_ARGS, good, **bad) == _lib.EINVAL, bad
    assert lib.kyb_paged_step(None, None) == _lib.EINVAL
    assert lib.kyb_paged_release(P, None, P, 4, 2, 4, 16, P, 10, P, P, None) == _lib.EINVAL
    assert lib.kyb_paged_release(P, P, P, 4, 2, 4, 20, P, 10, P, P, None) == _lib.EINVAL


def test_rope_refusals(lib):
    good = dict(q=P, k=P, v=P, pos=P, slots=P, inv=P, qo=P, kc=P, vc=P, q_t=128, q_h=64, k_t=64, k_h=64, v_t=64, v_h=64, qo_t=128, qo_h=64, kc_p=1024, kc_h=1024, vc_p=1024, vc_h=1024, tokens=3,
                hq=2, hkv=1, d=64, rot=64, inter=0, dt=1, pages=2, page=16, m=1.0)
    for bad in (dict(q=0), dict(k=0), dict(slots=0), dict(q=P + 2), dict(vc=P + 8), dict(q_t=100), dict(kc_p=1028), dict(d=60), dict(d=264), dict(rot=0), dict(rot=40), dict(rot=80), dict(dt=0),
                dict(dt=3), dict(hq=-1), dict(hq=1 << 32), dict(hq=0, hkv=0), dict(tokens=-1), dict(tokens=1 << 31), dict(pages=0), dict(page=48)):
        assert _call(lib.kyb_rope_append, _lib.ROPE_APPEND_ARGS, good, **bad) == _lib.EINVAL, bad
    assert _call(lib.kyb_rope_append, _lib.ROPE_APPEND_ARGS, good, tokens=0) == _lib.OK and lib.kyb_rope_append(None, None) == _lib.EINVAL


def test_attention_refusals(lib):
    good = dict(q=P, k=P, v=P, table=P, kv=P, cu=P, out=P, ws=P, q_t=128, q_h=64, k_p=1024, k_h=1024, v_p=1024, v_h=1024, o_t=128, o_h=64, pages=2, page=16, ld=3, cols=3, batch=1, tokens=3,
                max_q=3, hq=2, hkv=1, d=64, dt=1, window=0, sinks=0, wsn=1 << 30, scale=0.1)
    for bad in (dict(q=0), dict(v=0), dict(table=0), dict(out=0), dict(q=P + 2), dict(out=P + 4), dict(q_t=100), dict(k_p=1028), dict(o_h=-64), dict(pages=0), dict(pages=1 << 31),
                dict(page=8), dict(page=100), dict(page=16 + (1 << 32)), dict(ld=2), dict(cols=0), dict(cols=1 << 28, ld=1 << 28), dict(batch=0), dict(tokens=-1), dict(tokens=1 << 30),
                dict(max_q=-1), dict(max_q=1 << 31), dict(hq=0), dict(hq=3, hkv=2), dict(hq=129), dict(d=96), dict(dt=0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e300),
                dict(window=-1), dict(sinks=-1), dict(sinks=4), dict(tokens=1 << 29, hq=64)):
        assert _call(lib.kyb_paged_attention, _lib.PAGED_ATTENTION_ARGS, good, **bad) == _lib.EINVAL, bad
    assert _call(lib.kyb_paged_attention, _lib.PAGED_ATTENTION_ARGS, good, tokens=0) == _lib.OK and lib.kyb_paged_attention(None, None) == _lib.EINVAL


def test_argument_blocks_match_the_header():
    """Sizes of the packed blocks against the structs of include/kyb.h: pointers, int64 and a double, 8 bytes each."""
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "kyb.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, block in (("kyb_paged_step_args", _lib.PAGED_STEP_ARGS), ("kyb_rope_append_args", _lib.ROPE_APPEND_ARGS), ("kyb_paged_attention_args", _lib.PAGED_ATTENTION_ARGS)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name, text).group(1)
        kinds = "".join(("Q" if "*" in d else "d" if d.strip().startswith("double") else "q") * (d.count(",") + 1) for d in body.split(";") if d.strip())
        assert kinds == "".join(c * int(n) for n, c in re.findall(r"(\d+)([Qq])", block.format)) + ("d" if block.format.endswith("d") else ""), name


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
