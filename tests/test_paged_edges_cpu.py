"""Host checks of the paged-cache operators at the edges of what their documentation allows (no GPU needed)."""
import itertools
import math
import os
import random
import subprocess

import pytest
import torch

from kyojin_mac_b200 import _lib, ops


# ------------------------------------------------------------------------------------------------ memory that a call reads and writes
def _places(t):
    """Element numbers of a view in its storage."""
    n = torch.zeros(1, dtype=torch.long)
    for s, st in zip(t.shape, t.stride()):
        n = (n[:, None] + torch.arange(s) * st).flatten()
    return set((n + t.storage_offset()).tolist())


def _views(buf):
    """Views of one buffer of 4096 values as callers make them: rows of a product, heads apart, transposed, shifted."""
    for off, tokens, heads, d in itertools.product((0, 8, 16, 64, 200), (1, 3, 5), (1, 2, 4), (8, 16)):
        for layout in ((heads * d, d), (96, d), (128, d), (128, 2 * d), (d, tokens * d), (64, 16), (200, d)):
            t = torch.as_strided(buf, (tokens, heads, d), (*layout, 1), off)
            if len(_places(t)) == t.numel():
                yield t


def test_overlap_is_found():
    """A pair that shares an element is never taken for one that does not; the layouts that callers use are taken."""
    buf, r = torch.zeros(4096, dtype=torch.float16), random.Random(1)
    views = list(_views(buf))
    found = taken = 0
    for _ in range(20000):
        a, b = r.choice(views), r.choice(views)
        v = ops._Views([("q", a), ("out", b)], ["out"], ("q", "out"))
        walk = lambda t: (t.storage_offset(), t.shape, [s for n, s in zip(t.shape, t.stride()) if n > 1])
        same = walk(a) == walk(b)                                            # (the stride of a dimension of one is never used)
        shared = bool(_places(a) & _places(b))
        try:
            v.check(a.data_ptr(), b.data_ptr())
            assert not shared or same
            taken += not shared
        except ValueError:
            found += shared
    assert found > 1000 and taken > 1000


def test_usual_layouts_pass():
    t, hq, hkv, d, w = 5, 4, 2, 16, 128 + 8
    buf = torch.zeros(4096, dtype=torch.float16)
    q, k, v = (torch.as_strided(buf, (t, h, d), (w, d, 1), off) for h, off in ((hq, 0), (hkv, hq * d), (hkv, (hq + hkv) * d)))
    pool = torch.zeros((3, 2, hkv, 16, d), dtype=torch.float16)              # pages outside, keys and values inside
    kc, vc = pool[:, 0], pool[:, 1]
    named = [("q", q), ("k", k), ("v", v), ("k_cache", kc), ("v_cache", vc), ("out", q)]
    ptrs = [x.data_ptr() for _, x in named]
    ops._Views(named, ["k_cache", "v_cache", "out"], ("q", "out")).check(*ptrs)
    apart = torch.zeros((t, hq, 2, d), dtype=torch.float16)                  # heads of queries and output in turn
    ops._Views([("q", apart[:, :, 0]), ("out", apart[:, :, 1])], ["out"], ("q", "out")).check(apart.data_ptr(), apart[:, :, 1].data_ptr())
    for name, other in (("out", k), ("out", torch.as_strided(buf, (t, hq, d), (w, d, 1), 8)), ("out", torch.as_strided(buf, (t, hq, d), (hq * d, d, 1), 0)), ("v_cache", kc), ("k_cache", vc)):
        bad = [(n, other if n == name else x) for n, x in named]
        with pytest.raises(ValueError, match="overlap"):
            ops._Views(bad, ["k_cache", "v_cache", "out"], ("q", "out")).check(*[x.data_ptr() for _, x in bad])
    empty = torch.zeros((0, 4, 16), dtype=torch.float16)
    ops._Views([("q", empty), ("out", empty)], ["out"], ("q", "out")).check(empty.data_ptr(), empty.data_ptr())


# ------------------------------------------------------------------------------------------------ numbers
@pytest.fixture(scope="module")
def lib():
    _lib.build()
    return _lib.lib()


P = 64                       # stands for an address that is 16-byte aligned; calls below are refused, or end for want of a device, before anything is read
ATTENTION = dict(q=P, k=P, v=P, table=P, kv=P, cu=P, out=P, ws=P, q_t=128, q_h=64, k_p=1024, k_h=1024, v_p=1024, v_h=1024, o_t=128, o_h=64, pages=2, page=16, ld=3, cols=3, batch=1, tokens=0,
                 max_q=3, hq=2, hkv=1, d=64, dt=1, window=0, sinks=0, wsn=1 << 30, scale=0.1)


def test_scale_in_powers_of_two(lib):
    """The kernels use scale * log2(e): a scale that is finite itself but not so (above 2.36e38) is refused; the largest that is passes (no tokens: nothing to do)."""
    call = lambda scale: lib.kyb_paged_attention(_lib.PAGED_ATTENTION_ARGS.pack(*{**ATTENTION, "scale": scale}.values()), None)
    for bad in (2.4e38, -2.4e38, 3.4e38, math.inf, -math.inf, math.nan):
        assert call(bad) == _lib.EINVAL, bad
    for good in (2.3e38, -2.3e38, 0.0, 1e-45, 1.0):
        assert call(good) == _lib.OK, good


# ------------------------------------------------------------------------------------------------ error texts
def test_a_driver_without_the_encoder_is_named(tmp_path):
    """Where the driver has no tensor-map encoder (as here, where there is no driver), the error says so instead of a bare number."""
    src = tmp_path / "maps.cpp"
    src.write_text("""
#include <stdarg.h>
#include <stdio.h>
#include "tc_common.cuh"
void kyb_set_error(const char* fmt, ...) { va_list a; va_start(a, fmt); vprintf(fmt, a); va_end(a); printf("\\n"); }
int main() {
    if (kyb_get_encode_tiled()) return 77;
    CUtensorMap m;
    return kyb_make_tmap_2d(&m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, (void*)256, 128, 64, 128, 64, 64) == KYB_ECUDA ? 0 : 1;
}
""")
    csrc = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")
    cuda = "/usr/local/cuda"
    if not os.path.exists(cuda + "/include/cuda.h"):
        pytest.skip("no CUDA headers")
    exe = str(tmp_path / "maps")
    subprocess.run(["g++", "-std=c++17", "-I", csrc, "-I", os.path.join(csrc, "..", "..", "include"), "-I", cuda + "/include", str(src), "-o", exe, "-L", cuda + "/lib64", "-lcudart_static", "-ldl", "-lrt",
                    "-lpthread"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    if r.returncode == 77:
        pytest.skip("this driver has the encoder")
    assert r.returncode == 0 and "not available from this driver" in r.stdout, r


@pytest.mark.parametrize("scaling", [
    {"type": "llama3", "factor": 8.0}, {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0}, {"type": "yarn", "factor": 4.0},
    {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_context": 0}, {"type": "yarn", "factor": 4.0, "original_context": 0},
    {"type": "yarn", "factor": 4.0, "original_context": -5}, {"type": "yarn", "factor": 4.0, "original_context": math.inf}, {"type": "yarn", "factor": 4.0, "original_context": 4096, "beta_slow": 0},
    {"type": "yarn", "factor": 4.0, "original_context": 4096, "beta_fast": 1, "beta_slow": 32}, {"type": "linear"}, {}])
def test_scalings_that_lack_a_number(scaling):
    """A scaling without one of its numbers, or with one that means nothing, is refused as any other argument is."""
    with pytest.raises(ValueError, match="scaling|factor"):
        ops.rope_frequencies(64, 10000.0, scaling, "cpu")


def test_base_is_finite():
    for bad in (math.inf, math.nan, 1.0, -5.0):
        with pytest.raises(ValueError, match="base"):
            ops.rope_frequencies(64, bad, device="cpu")
