"""The attention block over quantized linears (paged.AttentionBlock, paged.PagedCache) on the GPU: against the same layer in 64 bits, captured and replayed."""
import numpy as np
import pytest
import torch

import paged_reference as R
from kyojin_mac_b200 import foreign_linear as FL, foreign_pack as FP, ops, synth
from kyojin_mac_b200.host_graph import HostGraph
from kyojin_mac_b200.paged import AttentionBlock, PagedCache

pytestmark = pytest.mark.gpu

HID, HEADS, KV, D, PAGE = 512, 8, 2, 64, 16
WIDTHS = [HEADS * D, KV * D, KV * D]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _linear(n, k, rng):
    return FL.ForeignLinear(FP.to_pack("Q8_0", synth.raw_blocks("q8_0", n, k, rng), k))


def _block(rng, **more):
    return AttentionBlock(_linear(sum(WIDTHS), HID, rng), _linear(HID, HEADS * D, rng), HEADS, KV, D, rot=32, **more)


def _x(rows, g):
    return (torch.randn((rows, HID), generator=g) * 0.05).to(torch.float16).cuda()


class History:
    """What each request has sent so far, and the layer over it in 64 bits: decoded weights, fp16 at the same points (the products' outputs, the turned heads, the
    attention's output)."""

    def __init__(self, block, requests):
        self.b, self.k, self.v = block, [[] for _ in range(requests)], [[] for _ in range(requests)]
        self.wqkv = torch.cat([m.dev.dequant(torch.float32).cpu().double() for m in block.qkv])
        self.wo = block.o.dev.dequant(torch.float32).cpu().double()

    def __call__(self, x, new):
        b, x = self.b, x.cpu().double()
        inv, out, at = b.inv_freq.cpu(), [], 0
        for r, n in enumerate(new):
            y = (x[at:at + n] @ self.wqkv.T).half()
            q, k, v = (z.unflatten(1, (-1, D)) for z in y.split(WIDTHS, 1))
            p = torch.arange(n) + sum(t.shape[0] for t in self.k[r])
            q = R.turn(q, p, inv, b.interleaved, b.mscale).half()
            self.k[r].append(R.turn(k, p, inv, b.interleaved, b.mscale).half()), self.v[r].append(v)
            if n:
                pk, pv = (torch.cat(t)[None].transpose(1, 2) for t in (self.k[r], self.v[r]))
                o, _ = R.attention(q, pk, pv, torch.zeros((1, 1), dtype=torch.int32), _i32([int(p[-1]) + 1]), _i32([0, n]), D ** -0.5, b.window, b.sinks)
                out.append(o.half().double().flatten(1) @ self.wo.T)
            at += n
        return torch.cat(out)


def _near(got, want):
    """The products and their rounding points are the same on both sides, so what is left is that values next to a border of fp16 round the other way: a relative Frobenius
    distance of a few 2^-11, and never more than the linears' own bound of 1e-3 three times over (q | k | v, attention, o)."""
    d = (got.cpu().double() - want).norm() / want.norm()
    assert d < 3e-3, float(d)


@pytest.mark.parametrize("more", [dict(), dict(interleaved=True, window=24, sinks=2), dict(base=500000.0, scaling={"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                                                                                                      "high_freq_factor": 4.0, "original_context": 8192})])
def test_block_over_steps(more):
    rng, g = np.random.default_rng(5), torch.Generator().manual_seed(5)
    block = _block(rng, **more)
    cache = PagedCache(1, 24, KV, D, 3, 128, PAGE)
    layer = History(block, 3)
    for new in ([20, 0, 70], [1, 1, 1], [33, 5, 1], [1, 1, 1]):
        rows = sum(new)
        x = _x(rows + 2, g)
        s = cache.step(_i32(new), rows + 2)
        y = block(x, cache, s, max(new))
        assert s.refused.item() == 0 and torch.isfinite(y).all()             # the two rows behind the last request too
        _near(y[:rows], layer(x, new))
    cache.release(torch.tensor([True, True, True], device="cuda"))
    assert cache.free_count.item() == 24 and sorted(cache.free_pages.tolist()) == list(range(24)) and cache.lens.tolist() == [0, 0, 0]


def test_three_linears_and_a_group():
    """q, k and v as three linears, alone and as members of a same-input group, give what the fused linear gives."""
    rng, g = np.random.default_rng(6), torch.Generator().manual_seed(6)
    fused = _block(rng)
    d = fused.qkv[0].dev

    class Three(torch.nn.Module):
        def __init__(self):
            super().__init__()
            cut = np.cumsum([0] + WIDTHS)
            self.q, self.k, self.v = (FL.ForeignLinear(FL.DevPack.from_t16(d.fmt, d.t16[ops.t16_nbytes(d.fmt, int(a), HID) if a else 0:ops.t16_nbytes(d.fmt, int(b), HID)], int(b - a), HID))
                                      for a, b in zip(cut[:-1], cut[1:]))

        def forward(self, x):
            return self.q(x), self.k(x), self.v(x)
    model = Three()
    want = None
    for grouped in (False, True):
        if grouped:
            assert FL.group_same_input(model, (_x(2, g),), log=lambda *_: None)["members"] == 3
        for block in (fused, AttentionBlock((model.q, model.k, model.v), fused.o, HEADS, KV, D, rot=32)):
            cache = PagedCache(1, 8, KV, D, 2, 64, PAGE)
            x = _x(40, torch.Generator().manual_seed(7))
            y = block(x, cache, cache.step(_i32([9, 31]), 40), 31)
            want = y if want is None else want
            assert torch.equal(y, want)


def test_captured_steps_move_on():
    """A decode step captured once and replayed: lengths, pages and slots move on the device, the results are those of eager steps."""
    rng, g = np.random.default_rng(8), torch.Generator().manual_seed(8)
    block = _block(rng)
    new = _i32([1, 1])
    caches = [PagedCache(1, 12, KV, D, 2, 96, PAGE) for _ in range(2)]
    x0 = _x(50, g)
    for c in caches:
        block(x0, c, c.step(_i32([15, 35]), 50), 35)
    state = [t.clone() for t in (caches[1].table, caches[1].lens, caches[1].free_count, caches[1].keys[0], caches[1].values[0])]
    step = HostGraph(lambda x: block(x, caches[1], caches[1].step(new, 2), 1), [(2, HID)])
    for t, old in zip((caches[1].table, caches[1].lens, caches[1].free_count, caches[1].keys[0], caches[1].values[0]), state):
        t.copy_(old)                                                         # what the warm-up moved
    for _ in range(20):                                                      # across the end of a page
        x = _x(2, g)
        want = block(x, caches[0], caches[0].step(new, 2), 1)
        step.inputs[0].copy_(x)
        assert torch.equal(step()[0], want.cpu())
    assert caches[0].lens.tolist() == caches[1].lens.tolist() == [35, 55] and torch.equal(caches[0].table, caches[1].table)
    del step


def test_refused_requests_give_zeros():
    """Too few pages: the request that is not served keeps its length, its attention is zeros and the others are served."""
    rng, g = np.random.default_rng(9), torch.Generator().manual_seed(9)
    block = _block(rng)
    cache = PagedCache(1, 3, KV, D, 3, 64, PAGE)
    s = cache.step(_i32([30, 20, 4]), 54)
    y = block(_x(54, g), cache, s, 30)
    assert s.refused.item() == 2 and cache.lens.tolist() == [30, 0, 0] and cache.free_count.item() == 1
    assert (y[30:] == 0).all() and not (y[:30] == 0).all()


def test_block_refusals():
    rng = np.random.default_rng(1)
    a, o = _linear(sum(WIDTHS), HID, rng), _linear(HID, HEADS * D, rng)
    for bad in (dict(heads=HEADS, kv_heads=4, head_dim=D), dict(heads=4, kv_heads=KV, head_dim=D), dict(heads=HEADS, kv_heads=KV, head_dim=D, rot=80)):
        with pytest.raises(ValueError):
            AttentionBlock(a, o, **bad)
    block = AttentionBlock(a, o, HEADS, KV, D)
    cache = PagedCache(1, 4, KV, D, 1, 32, PAGE)
    with pytest.raises(ValueError):
        block(torch.zeros((3, HID), dtype=torch.float16, device="cuda"), cache, cache.step(_i32([2]), 2), 2)
    for bad in (dict(page=24), dict(head_dim=96), dict(requests=0), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(layers=1, pages=4, kv_heads=2, head_dim=64, requests=1, max_tokens=10), **bad})


def test_operator_refusals():
    """Shapes, types, strides and devices that the operators refuse before anything is launched; a refused call leaves the device usable."""
    q = torch.zeros((4, 4, 64), dtype=torch.float16, device="cuda")
    kc = torch.zeros((3, 2, 16, 64), dtype=torch.float16, device="cuda")
    vc, table, kv, cu = kc.clone(), _i32([[0, 1]]), _i32([4]), _i32([0, 4])
    good = dict(q=q, k_cache=kc, v_cache=vc, table=table, kv_lens=kv, cu_q=cu, max_q=4)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q[:, :3]), dict(q=q.bfloat16()), dict(q=q.transpose(1, 2)), dict(q=torch.zeros((4, 4, 96), dtype=torch.float16, device="cuda")),
                dict(k_cache=kc[:, :, :8]), dict(k_cache=kc.transpose(2, 3)), dict(v_cache=vc[:2]), dict(v_cache=vc.bfloat16()), dict(table=table.long()), dict(table=table[0]),
                dict(kv_lens=kv.long()), dict(kv_lens=_i32([4, 4])), dict(cu_q=cu[:1]), dict(max_q=-1), dict(window=-1), dict(sinks=2), dict(out=q[:3]), dict(out=q.bfloat16()),
                dict(table=table.cpu()), dict(q=q.cpu()), dict(q=q.clone().requires_grad_())):
        with pytest.raises(ValueError):
            ops.paged_attention(**{**good, **bad})
    base = torch.zeros(4 * 4 * 64 + 8, dtype=torch.float16, device="cuda")
    from kyojin_mac_b200._lib import KybError
    for n in (0, 1):                                                         # an address that is not 16-byte aligned: also when the shape has been seen before
        with pytest.raises((ValueError, KybError)):
            ops.paged_attention(**{**good, "q": base[1:1 + q.numel()].view(q.shape)})
        ops.paged_attention(**good)
    with pytest.raises((ValueError, KybError)):
        ops.paged_attention(**good, scale=float("nan"))
    inv, _ = ops.rope_frequencies(64)
    pos = _i32([0, 1, 2, 3])
    k = torch.zeros((4, 2, 64), dtype=torch.float16, device="cuda")
    rope = dict(q=q, k=k, v=k, positions=pos, slots=pos, inv_freq=inv, k_cache=kc, v_cache=vc)
    ops.rope_append(**rope)
    for bad in (dict(positions=pos.long()), dict(positions=pos[:3]), dict(slots=pos[:3]), dict(k=k[:, :1]), dict(v=k.bfloat16()), dict(inv_freq=inv.double()), dict(k_cache=kc[..., :32]),
                dict(q=q.float()), dict(out=q[:2])):
        with pytest.raises(ValueError):
            ops.rope_append(**{**rope, **bad})
    with pytest.raises((ValueError, KybError)):
        ops.rope(q, pos, ops.rope_frequencies(128)[0])                       # more values than a head has
    step = dict(table=table, lens=kv, new_lens=kv, free_pages=_i32([2]), free_count=_i32([1]), page=16, rows=4)
    for bad in (dict(table=table.float()), dict(lens=_i32([1, 2])), dict(new_lens=kv.long()), dict(free_pages=_i32([])), dict(free_count=_i32([1, 1])), dict(page=24), dict(rows=-1)):
        with pytest.raises(ValueError):
            ops.paged_step(**{**step, **bad})
    torch.cuda.synchronize()
    ops.check_device_status()
