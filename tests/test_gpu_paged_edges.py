"""Paged-cache operators at the edges of what their documentation allows: items that follow each other without a pause, dominant keys, offsets that overlap, memory that is shared."""
import random

import pytest
import torch

import paged_reference as R
from kyojin_mac_b200 import ops
from kyojin_mac_b200._lib import EINVAL, KybError

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(qn):
    return _i32([sum(qn[:i]) for i in range(len(qn) + 1)])


# ------------------------------------------------------------------------------------------------ many short items
@pytest.mark.parametrize("hq,hkv,d,lo,hi", [(8, 8, 64, 17, 60), (4, 4, 128, 17, 60), (16, 4, 64, 20, 90), (8, 8, 64, 100, 150), (6, 6, 128, 100, 280)])
def test_short_items_follow_each_other(hq, hkv, d, lo, hi):
    """Several hundred short requests: each CTA goes through dozens of items of one key tile or two, with one query tile or two, one behind the other. Every call gives the
    same, all rows are written and no wait runs out."""
    r = random.Random(hq + d + hi)
    qn = [r.randint(lo, hi) for _ in range(300)]
    k, v, table = R.pool(qn, 16, hkv, d, F16, 31)
    lens, cu = _i32(qn), _offsets(qn)
    q = torch.randn((sum(qn), hq, d), device="cuda").to(F16)
    first = ops.paged_attention(q, k, v, table, lens, cu, hi)
    for _ in range(40):
        out = torch.full_like(q, 9.0)
        assert torch.equal(ops.paged_attention(q, k, v, table, lens, cu, hi, out=out), first)
    ops.check_device_status()
    want, tol = R.attention(q, k, v, table, lens, cu, d ** -0.5, 0, 0)
    assert ((first.cpu().double() - want).abs() <= tol).all()


# ------------------------------------------------------------------------------------------------ a dominant key
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("d,qn,n,b", [(128, 1, 9000, 1), (64, 2, 5000, 300), (128, 4, 3500, 300), (128, 70, 6001, 1), (64, 300, 4100, 1)])
@pytest.mark.parametrize("at", [0, 3000])
@pytest.mark.parametrize("above", [18.0, 22.0, 25.5, 27.0])
def test_dominant_key(above, at, d, qn, n, b, dt):
    """One key takes nearly all of the mass (its score 2^above over the others' level), its value is a thousandth of theirs: what the many others add up to shows in the output.
    A weight is rounded relative to a reference that lies 2^7 at least under the row's largest, so fp16 loses 2^-32 of the largest weight per key at most, not 2^-25: the bound of
    `R.attention` with its term for that taken 2^-7 times. b requests share the pages, so that one CTA walks a whole context."""
    g = torch.Generator().manual_seed(int(above) + d)
    k, v, table = R.pool([n], 64, 1, d, torch.float32, 41, device="cpu")
    k = torch.where(torch.isnan(k), k, torch.randn(k.shape, generator=g) * 0.05)
    k[..., 0] = torch.where(torch.isnan(k[..., 0]), k[..., 0], 0.0)
    v = torch.where(torch.isnan(v), v, 1.0 + 0.25 * torch.rand(v.shape, generator=g))
    page, place = int(table[0, at // 64]), at % 64
    k[page, 0, place] = 0.0
    k[page, 0, place, 0], v[page, 0, place] = above * 0.6931 * d ** 0.5 / 16.0, 0.001
    q = torch.randn((qn, 4, d), generator=g) * 0.5
    q[..., 0] = 16.0
    q, k, v, table = q.to(dt).cuda(), k.to(dt).cuda(), v.to(dt).cuda(), table.cuda()
    got = ops.paged_attention(q.repeat(b, 1, 1), k, v, table.repeat(b, 1), _i32([n] * b), _offsets([qn] * b), qn).view(b, qn, 4, d)
    want, tol = R.attention(q, k, v, table, _i32([n]), _i32([0, qn]), d ** -0.5, 0, 0)
    if dt == F16:
        keys = (torch.arange(n - qn, n) + 1.0).double()[:, None, None]
        tol = tol - keys * 2.0 ** -25 * (1 - 2.0 ** -7) * float(v[~v.isnan()].abs().max())
    err = (got.cpu().double() - want).abs()
    assert (tol > 0).all() and (err <= tol).all(), float((err / tol).max())


# ------------------------------------------------------------------------------------------------ offsets that give the requests more rows than there are
@pytest.mark.parametrize("rows,pairs,max_q,hkv,cols", [(64, 20, 1, 2, 4), (64, 20, 64, 2, 4), (5, 300, 1, 1, 4), (20000, 2000, 1, 1, 300), (20000, 2000, 300, 1, 300), (30, 1, 30, 1, 4)])
def test_offsets_that_overlap(rows, pairs, max_q, hkv, cols):
    """Offsets 0, T, 0, T, ...: every second request would own all rows, and the sums of their key tiles could pass any bound. Nothing is written, the status word tells; calls
    with good offsets are served before and after."""
    page, d = 64, 64
    k, v = (torch.randn((3, hkv, page, d), device="cuda").to(F16) for _ in range(2))
    q = torch.randn((rows, 4 * hkv, d), device="cuda").to(F16)
    batch = 2 * pairs + 1
    table = torch.zeros((batch, cols), dtype=torch.int32, device="cuda")
    lens = torch.full((batch,), page, dtype=torch.int32, device="cuda")
    good = torch.full((batch + 1,), rows, dtype=torch.int32, device="cuda")
    good[0] = 0
    bad = torch.zeros_like(good)
    bad[1::2] = rows
    lens[0] = max(page, rows)
    want = ops.paged_attention(q, k, v, table, lens, good, max_q)
    out = torch.full_like(q, 6.0)
    lens[:] = cols * page
    ops.paged_attention(q, k, v, table, lens, bad, max_q, out=out)
    with pytest.raises(KybError, match="offsets") as e:
        ops.check_device_status()
    assert e.value.status == EINVAL
    assert (out == 6.0).all()
    lens[:] = page
    lens[0] = max(page, rows)
    assert torch.equal(ops.paged_attention(q, k, v, table, lens, good, max_q, out=out), want)
    ops.check_device_status()


# ------------------------------------------------------------------------------------------------ outputs that lie over inputs
@pytest.mark.parametrize("rows", [3, 60])
def test_overlapping_memory_is_refused(rows):
    """An output that lies over a part of the queries, keys or cache is refused, also when its shapes have been seen before; the queries' own place, and neighbours in one buffer, are
    taken."""
    hq, hkv, d, page = 8, 2, 64, 16
    buf = torch.randn(((rows + 2) * (hq + 2 * hkv) * d,), device="cuda").to(F16)
    w = (hq + 2 * hkv) * d
    prod = buf[:rows * w].view(rows, w)
    q, k, v = (x.unflatten(1, (-1, d)) for x in prod.split((hq * d, hkv * d, hkv * d), dim=1))
    pool = torch.randn((16, 2, hkv, page, d), device="cuda").to(F16)
    kc, vc = pool[:, 0], pool[:, 1]
    table, lens, cu = _i32([[0, 1, 2, 3]]), _i32([rows]), _i32([0, rows])
    attend = lambda **kw: ops.paged_attention(kw.get("q", q), kc, vc, table, lens, cu, rows, out=kw.get("out"))
    dense = q.contiguous()
    want = attend(q=dense)
    shifted = torch.empty(dense.numel() + hq * d, dtype=F16, device="cuda")
    a, b = shifted[:dense.numel()].view(dense.shape), shifted[hq * d:].view(dense.shape)
    a.copy_(dense)
    for _ in range(2):
        for bad in (dict(q=a, out=b), dict(out=buf[8:8 + dense.numel()].view(dense.shape)), dict(q=dense, out=pool.flatten()[:dense.numel()].view(dense.shape))):
            with pytest.raises(ValueError, match="overlap"):
                attend(**bad)
        assert torch.equal(attend(q=a, out=torch.empty_like(a)), want)
    assert torch.equal(attend(q=a, out=a), want)
    pos, slots = torch.arange(rows, device="cuda").to(torch.int32), torch.arange(rows, device="cuda").to(torch.int32)
    inv, _ = ops.rope_frequencies(d)
    put = lambda **kw: ops.rope_append(*(kw.get(n, t) for n, t in (("q", q), ("k", k), ("v", v))), pos, slots, inv, kw.get("kc", kc), kw.get("vc", vc), out=kw.get("out"))
    turned = put()
    wide = torch.as_strided(buf, (rows, hq, d), (w, d, 1), hkv * d)          # over the product's rows, two heads on
    for bad in (dict(out=wide), dict(vc=kc), dict(k=pool.flatten()[:rows * hkv * d].view(rows, hkv, d))):
        with pytest.raises(ValueError, match="overlap"):
            put(**bad)
    with pytest.raises(ValueError, match="overlap"):
        ops.rope(dense, pos, inv, out=torch.as_strided(dense, dense.shape, (d, rows * d, 1)))
    assert put(out=q).data_ptr() == q.data_ptr() and torch.equal(q, turned)


# ------------------------------------------------------------------------------------------------ no backward
def test_whatever_takes_part_in_differentiation_is_refused():
    """Queries, keys, values, caches, outputs and frequencies that require a gradient or carry a forward-mode tangent: also when the same shapes have passed before; without
    gradients they are taken."""
    import torch.autograd.forward_ad as fwd
    x = lambda *s: torch.randn(s, device="cuda").to(F16)
    inv, _ = ops.rope_frequencies(64)
    pos = _i32([0, 1, 2])
    rope = dict(q=x(3, 4, 64), k=x(3, 2, 64), v=x(3, 2, 64), inv_freq=inv, k_cache=x(2, 2, 16, 64), v_cache=x(2, 2, 16, 64), out=x(3, 4, 64))
    attend = dict(q=x(3, 4, 64), k_cache=x(2, 2, 16, 64), v_cache=x(2, 2, 16, 64), out=x(3, 4, 64))
    alone = dict(x=x(3, 4, 64), inv_freq=inv, out=x(3, 4, 64))
    calls = ((lambda **kw: ops.rope_append(positions=pos, slots=pos, **kw), rope), (lambda **kw: ops.rope(positions=pos, **kw), alone),
             (lambda **kw: ops.paged_attention(table=_i32([[0]]), kv_lens=_i32([3]), cu_q=_i32([0, 3]), max_q=3, **kw), attend))
    for call, good in calls:
        for turn in range(2):
            for name, t in good.items():
                leaf = t.clone().requires_grad_()
                with pytest.raises(ValueError, match="gradient"):
                    call(**{**good, name: leaf})
                with torch.no_grad():
                    call(**{**good, name: leaf})
                with fwd.dual_level():
                    call(**good)
                    with pytest.raises(ValueError, match="gradient"):
                        call(**{**good, name: fwd.make_dual(t, torch.ones_like(t))})
            call(**good)


# ------------------------------------------------------------------------------------------------ pages given back
@pytest.mark.parametrize("b,room", [(2500, 10 ** 6), (2500, 900), (2500, 0), (1024, 500), (1025, 40), (30, 11)])
def test_release_into_a_short_list(b, room):
    """A list without room for all: the requests up to the one that overflows it give their pages back, those behind it keep theirs (wherever a thousand requests end), and a request
    that holds no page is served."""
    r = random.Random(b + room)
    page, cols = 16, 5
    lens = [r.choice((0, r.randint(1, 70))) for _ in range(b)]
    need = [-(-n // page) for n in lens]
    ids = r.sample(range(10 ** 6), sum(need) + 3)
    at = [sum(need[:i]) for i in range(b)]
    table = [ids[a:a + n] + [-1] * (cols - n) for a, n in zip(at, need)]
    which = [r.random() < 0.7 for _ in range(b)]
    cap = 3 + min(room, sum(n for n, w in zip(need, which) if w))
    free, asked, refused, lens_after, table_after = ids[-3:], 0, 0, list(lens), [list(t) for t in table]
    for i in range(b):
        if not which[i]:
            continue
        asked += need[i]
        if need[i] and 3 + asked > cap:
            refused += 1
            continue
        free += table[i][:need[i]]
        lens_after[i], table_after[i] = 0, [-1] * cols
    t, ln, ct, fr = _i32(table), _i32(lens), _i32([3]), _i32(ids[-3:] + [-9] * (cap - 3))
    got = ops.paged_release(t, ln, torch.tensor(which, device="cuda"), fr, ct, page).item()
    assert got == refused and ct.item() == len(free) and fr.tolist() == free + [-9] * (cap - len(free))
    assert ln.tolist() == lens_after and t.tolist() == table_after


# ------------------------------------------------------------------------------------------------ dimensions of one
@pytest.mark.parametrize("hq", [1, 4, 40])
def test_strides_of_dimensions_of_one(hq):
    """One token of rows of an odd width, one head, one page: a stride that nothing steps by may be anything, in inputs, caches and outputs."""
    d, page = 64, 16
    x = lambda *s: torch.randn(s, device="cuda").to(F16)

    def odd(t):
        """The same values with strides of 1001 at dimensions of one."""
        return torch.as_strided(t, t.shape, [s if n > 1 else 1001 for n, s in zip(t.shape, t.stride())])
    inv, _ = ops.rope_frequencies(d)
    pos, one = _i32([5]), _i32([[0]])
    q, k, v, kc, vc = x(1, hq, d), x(1, 1, d), x(1, 1, d), x(1, 1, page, d), x(1, 1, page, d)
    attend = lambda f: ops.paged_attention(f(q), f(kc), f(vc), one, _i32([6]), _i32([0, 1]), 1, out=f(torch.zeros_like(q)))
    turn = lambda f: ops.rope(f(q), pos, inv, out=f(torch.zeros_like(q)))

    def put(f):
        c, w = kc.clone(), vc.clone()
        return ops.rope_append(f(q), f(k), f(v), pos, pos, inv, f(c), f(w), out=f(torch.zeros_like(q))), c, w
    for call in (attend, turn, put):
        for order in ((odd, lambda t: t), (lambda t: t, odd)):
            ops._passed.clear()                                              # whichever is seen first
            a, b = (call(f) for f in order)
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    many = x(30, 1, d)                                                       # several tokens of one head, and one request of one page
    a, b = (ops.paged_attention(f(many), f(x2), f(x3), _i32([[0, 0]]), _i32([30]), _i32([0, 30]), 30) for f, x2, x3 in ((odd, kc, vc), (lambda t: t, kc, vc)))
    assert torch.equal(a, b)
