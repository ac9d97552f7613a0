"""Paged-cache operators on the GPU: the step's slots, the rotary append and attention over the cache against plain 64-bit forms (tests/paged_reference.py)."""
import random

import pytest
import torch

import paged_reference as R
from kyojin_mac_b200 import ops

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ slots of a step
def _step_case(b, page, seed, hi_len, hi_new, cols_off=2, rows_off=0, count_off=5):
    r = random.Random(seed)
    lens, news = [r.randint(0, hi_len) for _ in range(b)], [r.choice((0, 1, r.randint(0, hi_new))) for _ in range(b)]
    have = [-(-n // page) for n in lens]
    want = [-(-(n + q) // page) for n, q in zip(lens, news)]
    ids = list(range(sum(want) + 50))
    r.shuffle(ids)
    cols = max(1, max(want) + cols_off)
    table, at = [], 0
    for n in have:
        table.append((ids[at:at + n] + [-1] * cols)[:max(cols, n)][:cols])
        at += n
    free = ids[at:]
    count = max(0, min(len(free), sum(want) - sum(have) + count_off))
    return lens, news, free, count, table, max(0, sum(news) + rows_off)


@pytest.mark.parametrize("b,page,hi_len,hi_new,cols_off,rows_off,count_off", [
    (1, 16, 0, 1, 0, 0, 0), (1, 64, 100, 300, 0, 0, 0), (64, 64, 2000, 1, 2, 0, 5), (64, 16, 50, 40, 0, 7, 0),
    (33, 32, 300, 60, 2, 0, -9),           # the free list runs out in the middle
    (40, 16, 300, 60, -3, 0, 5),           # some requests do not fit their row of the table
    (50, 128, 300, 60, 1, -100, 5),        # the step has too few rows
    (1500, 16, 90, 20, 1, 3, -40),         # more requests than threads
    (3000, 256, 700, 9, 0, 0, 0), (7, 16, 10, 6000, 1, 0, 2), (5, 16, 0, 0, 1, 4, 0)])
def test_step_slots(b, page, hi_len, hi_new, cols_off, rows_off, count_off):
    lens, news, free, count, table, rows = _step_case(b, page, b * 31 + page, hi_len, hi_new, cols_off, rows_off, count_off)
    want = R.step(lens, news, free, count, table, page, rows)
    t, ln, nw, fr, ct = _i32(table), _i32(lens), _i32(news), _i32(free), _i32([count])
    for turn in range(2):                                                    # the inputs stay as they are: the same call again gives the same
        s = ops.paged_step(t, ln, nw, fr, ct, page, rows)
        got = [x.tolist() for x in (s.cu_q, s.kv_lens, s.positions, s.slots, s.lens)] + [s.free_count.item(), s.refused.item(), t.tolist()]
        for name, a, w in zip(("cu_q", "kv_lens", "positions", "slots", "lens", "free_count", "refused", "table"), got, want):
            assert a == w, (turn, name)
    assert ln.tolist() == lens and ct.item() == count and fr.tolist() == free
    t2 = _i32(table)
    s = ops.paged_step(t2, ln, nw, fr, ct, page, rows, in_place=True)
    assert ln.tolist() == want[4] and ct.item() == want[5] and t2.tolist() == want[7] and s.lens.data_ptr() == ln.data_ptr()


def test_step_odd_values():
    """Negative lengths count as 0, a free count above the list as the list; a table with a wider row stride."""
    wide = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    s = ops.paged_step(wide[:, :4], _i32([-5, 0]), _i32([-3, 20]), _i32([8, 9, 10]), _i32([99]), 16, 20)
    assert s.cu_q.tolist() == [0, 0, 20] and s.kv_lens.tolist() == [0, 20] and s.free_count.item() == 1 and s.refused.item() == 0
    assert s.slots.tolist() == [10 * 16 + i for i in range(16)] + [9 * 16 + i for i in range(4)] and wide[1].tolist() == [10, 9] + [-1] * 7


def test_release_returns_pages():
    page, b = 16, 1300
    r = random.Random(4)
    lens = [r.randint(0, 70) for _ in range(b)]
    need = [-(-n // page) for n in lens]
    ids = list(range(sum(need) + 20))
    r.shuffle(ids)
    cols, at, table = 6, 0, []
    for n in need:
        table.append(ids[at:at + n] + [-1] * (cols - n))
        at += n
    which = [r.random() < 0.5 for _ in range(b)]
    cap = 20 + sum(n for n, w in zip(need, which) if w)
    free = _i32(ids[at:] + [0] * (cap - 20))
    t, ln, ct = _i32(table), _i32(lens), _i32([20])
    assert ops.paged_release(t, ln, torch.tensor(which, device="cuda"), free, ct, page).item() == 0
    back = [p for row, n, w in zip(table, need, which) if w for p in row[:n]]
    assert ct.item() == cap and free.tolist() == ids[at:] + back
    assert ln.tolist() == [0 if w else n for n, w in zip(lens, which)]
    assert t.tolist() == [[-1] * cols if w else row for row, w in zip(table, which)]
    # a list without room: the first requests in order fit, the others keep their pages
    t, ln, ct, free = _i32([[5, -1], [6, 7]]), _i32([16, 17]), _i32([1]), _i32([3, 0])
    assert ops.paged_release(t, ln, torch.tensor([True, True], device="cuda"), free, ct, page).item() == 1
    assert ct.item() == 2 and free.tolist() == [3, 5] and ln.tolist() == [0, 17] and t.tolist() == [[-1, -1], [6, 7]]


# ------------------------------------------------------------------------------------------------ rotary append
@pytest.mark.parametrize("t,hq,hkv,d,rot,inter,page,dt", [
    (1, 1, 1, 64, 64, False, 16, F16), (3, 8, 2, 128, 128, False, 64, F16), (65, 25, 5, 64, 32, True, 16, BF16), (130, 7, 1, 128, 48, False, 128, BF16),
    (300, 64, 8, 128, 128, True, 32, F16), (37, 4, 4, 256, 256, False, 256, F16), (40, 3, 3, 72, 16, False, 16, BF16), (500, 2, 1, 64, 16, True, 64, F16)])
def test_rope_append(t, hq, hkv, d, rot, inter, page, dt):
    g = torch.Generator().manual_seed(t)
    qkv = (torch.randn((t, (hq + 2 * hkv) * d + 8), generator=g) * 3).to(dt).cuda()            # rows wider than the heads
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv[:, :(hq + 2 * hkv) * d].split((hq * d, hkv * d, hkv * d), dim=1))
    pos = torch.randint(0, 1 << 20, (t,), generator=g).to(torch.int32)
    pos[0] = 0 if t > 1 else 131071
    if t > 5:
        pos[2], pos[4] = -1, 2000000000
    n = t // page + 2
    slots = torch.randperm(n * page, generator=g)[:t].to(torch.int32)
    if t > 5:
        slots[3], slots[5] = -1, n * page                                    # nowhere, and behind the cache
    inv, mscale = ops.rope_frequencies(rot, 10000.0)
    mscale = 1.25
    kc, vc = (torch.full((n, hkv, page, d), 7.0, dtype=dt, device="cuda") for _ in range(2))
    before = qkv.clone()
    out = torch.full((t, hq, d), -3.0, dtype=dt, device="cuda")
    got = ops.rope_append(q, k, v, pos.cuda(), slots.cuda(), inv, kc, vc, interleaved=inter, mscale=mscale, out=out)
    assert got is out and torch.equal(qkv, before)
    row = pos >= 0
    for x, y in ((q, out), ):
        x = x.cpu()
        want = R.turn(x, pos, inv.cpu(), inter, mscale)
        tol = R.turn_bound(x, want, inv.cpu(), inter, mscale)
        assert ((y.cpu().double() - want).abs() <= tol)[row].all()
        assert torch.equal(y.cpu()[..., rot:][row], x[..., rot:][row]) and (y.cpu()[~row] == -3.0).all()
    put = row & (slots >= 0) & (slots < n * page)
    kw = R.turn(k.cpu(), pos, inv.cpu(), inter, mscale)
    tol = R.turn_bound(k.cpu(), kw, inv.cpu(), inter, mscale)
    flat = lambda c: c.cpu().transpose(1, 2).reshape(n * page, hkv, d)       # [slot, head, d]
    at = slots[put].long()
    assert ((flat(kc)[at].double() - kw[put]).abs() <= tol[put]).all() and torch.equal(flat(vc)[at], v.cpu()[put])
    rest = torch.ones(n * page, dtype=torch.bool)
    rest[at] = False
    assert (flat(kc)[rest] == 7.0).all() and (flat(vc)[rest] == 7.0).all()
    again = ops.rope(q, pos.cuda(), inv, interleaved=inter, mscale=mscale, out=q)              # in place, without a cache
    assert again is q and torch.equal(q[row.cuda()], out[row.cuda()]) and torch.equal(k, before[:, hq * d:(hq + hkv) * d].unflatten(1, (-1, d)))


def test_rope_no_tokens():
    inv, _ = ops.rope_frequencies(64)
    x = torch.empty((0, 4, 64), dtype=F16, device="cuda")
    assert ops.rope(x, _i32([]), inv).shape == (0, 4, 64)


# ------------------------------------------------------------------------------------------------ attention
def _attend(kv, qn, hq, hkv, d, page, dt, window=0, sinks=0, seed=0, scale=None, gain=2.0, max_q=None, tail=3, views=False, stale=float("nan"), cols=None):
    """Runs a batch and holds every row to the bound; rows outside the batch keep what they held."""
    k, v, table = R.pool(kv, page, hkv, d, dt, seed, cols=cols, stale=stale)
    cu = [0]
    for n in qn:
        cu.append(cu[-1] + n)
    t = cu[-1] + tail
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn((t, hq, d), generator=g) * gain).to(dt).cuda()
    out = torch.full((t, hq, d), -5.0, dtype=dt, device="cuda")
    if views:                                                                # heads of wider rows, keys and values of one allocation
        wide = torch.zeros((t, hq * d + 40), dtype=dt, device="cuda")
        wide[:, 8:8 + hq * d] = q.flatten(1)
        q = wide[:, 8:8 + hq * d].unflatten(1, (hq, d))
        both = torch.stack((k, v), 1)
        k, v = both[:, 0], both[:, 1]
        wide_t = torch.full((table.shape[0], table.shape[1] + 3), 10 ** 9, dtype=torch.int32, device="cuda")
        wide_t[:, :table.shape[1]] = table
        table = wide_t[:, :table.shape[1]]
    got = ops.paged_attention(q, k, v, table, _i32(kv), _i32(cu), max(qn) if max_q is None else max_q, scale=scale, window=window, sinks=sinks, out=out)
    assert got is out
    want, tol = R.attention(q[:cu[-1]], k, v, table, _i32(kv), _i32(cu), d ** -0.5 if scale is None else scale, window, sinks)
    err = (out[:cu[-1]].cpu().double() - want).abs()
    assert torch.isfinite(err).all() and (err <= tol).all(), (float((err / tol).max()), int((err > tol).sum()))
    assert (out[cu[-1]:] == -5.0).all()
    ops.check_device_status()
    return out


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_decode_pages_and_types(page, d, dt):
    _attend([1, 15, 64, 65, 300, 517], [1] * 6, 8, 2, d, page, dt, seed=page + d)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (6, 2), (5, 5), (28, 4), (64, 8), (40, 2), (128, 1), (71, 1)])
def test_decode_heads(hq, hkv):
    _attend([3, 200, 129], [1, 1, 1], hq, hkv, 128, 32, F16, seed=hq)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 0), (100, 33), (128, 200), (5000, 4)])
@pytest.mark.parametrize("qn", [[1, 1, 1, 1], [2, 1, 3, 2], [1, 90, 300, 17]])
def test_window_and_sinks(window, sinks, qn):
    _attend([1, 90, 700, 333][:4] if qn[0] == 1 else [2, 90, 700, 333], qn, 8, 2, 128, 16, F16, window, sinks, seed=window)


@pytest.mark.parametrize("qn,kv", [([4, 2, 3], [4, 600, 77]), ([7], [7]), ([16], [400]), ([33, 1], [33, 900]), ([128], [128]), ([129], [1000]), ([257, 256, 255], [257, 900, 300]), ([600], [2000]),
                                   ([1, 300, 0, 5, 64], [700, 300, 55, 5, 640])])
@pytest.mark.parametrize("hq,hkv,d,dt", [(8, 1, 128, F16), (6, 2, 64, BF16), (4, 4, 128, BF16), (7, 1, 128, F16)])
def test_chunks(qn, kv, hq, hkv, d, dt):
    _attend(kv, qn, hq, hkv, d, 64 if len(qn) != 1 else 16, dt, seed=sum(kv))


@pytest.mark.parametrize("hq,hkv", [(16, 1), (24, 1), (20, 2), (3, 3), (64, 1), (128, 1)])
def test_chunk_heads(hq, hkv):
    _attend([150, 40, 391], [70, 40, 9], hq, hkv, 64, 32, F16, seed=hq)


@pytest.mark.parametrize("b,most", [(161, 1), (700, 2), (400, 40), (900, 9)])
def test_more_requests_than_threads(b, most):
    """Batches beyond what one pass of a CTA's threads over the lengths takes, requests without rows and without keys among them."""
    r = random.Random(b)
    qn = [r.choice((0, 1, 1, r.randint(1, most))) for _ in range(b)]
    qn[3] = most
    kv = [n + r.choice((0, r.randint(0, 40), r.randint(0, 200))) if r.random() < 0.9 else 0 for n in qn]
    _attend(kv, qn, 4, 1, 64, 16, F16, seed=b)


def test_long_contexts_are_split():
    _attend([9001], [1], 8, 1, 128, 64, F16, seed=1)
    _attend([6000, 5], [1, 1], 4, 2, 64, 128, BF16, seed=2)
    _attend([5003], [40], 8, 1, 128, 32, F16, seed=3)
    _attend([4000], [130], 2, 2, 128, 256, BF16, window=3000, sinks=64, seed=4)


@pytest.mark.parametrize("qn", [[1, 1, 0], [40, 200, 0]])
def test_rows_without_keys(qn):
    """kv_lens 0 and kv_lens below the number of rows: rows in front of the first key give zeros."""
    out = _attend([0, qn[1] - qn[1] // 2, 30], qn, 8, 2, 128, 16, F16, tail=5)
    assert (out[:qn[0] + qn[1] // 2] == 0).all()


@pytest.mark.parametrize("qn", [[1, 1], [60, 70]])
def test_stale_places(qn):
    """Places behind a request's end hold NaN or infinities, table entries there anything; so do pages in front of every row's window."""
    for stale in (float("nan"), float("inf"), float("-inf")):
        _attend([100, 77], qn, 8, 2, 128, 64, F16, stale=stale, cols=9)
    k, v, table = R.pool([500, 431], 32, 2, 64, F16, 3)
    lens, cu, window = _i32([500, 431]), _i32([0, qn[0], qn[0] + qn[1]]), 50
    q = torch.randn((qn[0] + qn[1], 4, 64), device="cuda").to(F16)
    want = ops.paged_attention(q, k, v, table, lens, cu, max(qn), window=window, sinks=3)
    for r, (n, c) in enumerate(zip((500, 431), qn)):
        dead = torch.arange(3, n - c - window + 1)                           # seen by no row
        for x in (k, v):
            x[table[r].long()[dead // 32].cuda(), :, (dead % 32).cuda()] = float("nan")
        table[r, 1:(n - c - window + 1) // 32] = 10 ** 6                     # whole pages there given back
    assert torch.equal(ops.paged_attention(q, k, v, table, lens, cu, max(qn), window=window, sinks=3), want)


@pytest.mark.parametrize("qn", [[1, 1], [60, 40]])
def test_entries_that_are_no_page(qn):
    """Table entries outside the pool inside the context read as tokens of zeros."""
    k, v, table = R.pool([200, 150], 16, 2, 128, F16, 5)
    table[0, 3], table[1, 0], table[1, 5] = -1, k.shape[0], 2 ** 31 - 1
    lens, cu = _i32([200, 150]), _i32([0, qn[0], sum(qn)])
    q = torch.randn((sum(qn), 8, 128), device="cuda").to(F16)
    got = ops.paged_attention(q, k, v, table, lens, cu, max(qn))
    want, tol = R.attention(q, k, v, table, lens, cu, 128 ** -0.5, 0, 0)
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_lengths_beyond_the_table():
    """kv_lens beyond the table's columns: the keys behind them are not there, positions stay."""
    k, v, table = R.pool([128, 128], 64, 1, 128, F16, 6)
    lens, cu = _i32([140, 1000]), _i32([0, 1, 41])
    q = torch.randn((41, 8, 128), device="cuda").to(F16)
    got = ops.paged_attention(q, k, v, table, lens, cu, 40)
    want, tol = R.attention(q, k, v, table, lens, cu, 128 ** -0.5, 0, 0)
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("qn", [[1, 1, 1], [3, 1, 2], [100, 1, 60]])
def test_strided_views(qn):
    _attend([300, 64, 199], qn, 8, 2, 128, 32, F16, views=True, seed=8)


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales_and_large_scores(scale):
    _attend([300, 200], [1, 2], 4, 1, 128, 32, F16, scale=scale, gain=1.0, seed=9)
    _attend([300, 200], [100, 90], 4, 1, 128, 32, F16, scale=scale, gain=1.0, seed=10)
    _attend([700], [130], 4, 1, 128, 32, F16, gain=30.0, seed=11)            # one key takes almost everything
    _attend([700], [1], 4, 1, 128, 32, F16, gain=30.0, seed=12)


@pytest.mark.parametrize("qn,said", [([1, 3, 40], 1), ([300, 2, 90], 4), ([1, 1, 2], 4000)])
def test_wrong_max_q_still_serves_every_row(qn, said):
    _attend([50 + qn[0], 400, 129], qn, 8, 1, 128, 16, F16, max_q=said, seed=13)


@pytest.mark.parametrize("qn", [[1] * 5, [2, 1, 200, 30, 1]])
def test_runs_repeat_bit_for_bit(qn):
    k, v, table = R.pool([900, 33, 512, 700, 2000], 32, 2, 128, BF16, 14)
    lens, cu = _i32([900, 33, 512, 700, 2000]), _i32([sum(qn[:i]) for i in range(6)])
    q = torch.randn((sum(qn), 16, 128), device="cuda").to(BF16)
    first = ops.paged_attention(q, k, v, table, lens, cu, max(qn))
    for _ in range(3):
        assert torch.equal(ops.paged_attention(q, k, v, table, lens, cu, max(qn)), first)


@pytest.mark.parametrize("qn", [[1, 1], [50, 128]])
def test_streams_and_graphs(qn):
    """Two captured graphs of one shape replay side by side on two streams, with new inputs each time, beside eager calls."""
    k, v, table = R.pool([3000, 1200], 64, 2, 128, F16, 15)
    lens, cu = _i32([3000, 1200]), _i32([0, qn[0], sum(qn)])
    qs = [torch.randn((sum(qn), 16, 128), device="cuda").to(F16) for _ in range(6)]
    want = [ops.paged_attention(q, k, v, table, lens, cu, max(qn)) for q in qs]
    held, graphs, outs = [qs[0].clone(), qs[1].clone()], [], []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for h, s in zip(held, streams):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            outs.append(ops.paged_attention(h, k, v, table, lens, cu, max(qn)))
        graphs.append(gr)
    for turn in range(3):
        held[0].copy_(qs[2 * turn]), held[1].copy_(qs[2 * turn + 1])
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    gr.replay()
        side = ops.paged_attention(qs[turn], k, v, table, lens, cu, max(qn))
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[2 * turn]) and torch.equal(outs[1], want[2 * turn + 1]) and torch.equal(side, want[turn])


def test_no_rows():
    k, v, table = R.pool([10], 16, 1, 64, F16, 1)
    out = ops.paged_attention(torch.empty((0, 2, 64), dtype=F16, device="cuda"), k, v, table, _i32([10]), _i32([0, 0]), 0)
    assert out.shape == (0, 2, 64)
    q = torch.randn((4, 2, 64), device="cuda").to(F16)
    keep = torch.full_like(q, 2.0)
    for max_q in (0, 1, 50):
        assert (ops.paged_attention(q, k, v, table, _i32([10]), _i32([0, 0]), max_q, out=keep) == 2.0).all()


def test_steps_in_a_row():
    """Prompt, chunks and single tokens of three requests through paged_step, rope_append and paged_attention, against attention over the whole history."""
    torch.manual_seed(3)
    b, hq, hkv, d, page, dt = 3, 8, 2, 64, 16, F16
    inv, m = ops.rope_frequencies(d, 10000.0, {"type": "yarn", "factor": 4.0, "original_context": 2048})
    kc, vc = (torch.full((40, hkv, page, d), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    table = torch.full((b, 16), -1, dtype=torch.int32, device="cuda")
    lens, free, count = _i32([0] * b), torch.randperm(40, device="cuda").to(torch.int32), _i32([40])
    hist = [([], []) for _ in range(b)]
    for new in ([40, 0, 7], [1, 60, 1], [1, 1, 1], [30, 1, 33], [1, 1, 1]):
        rows = sum(new) + 2
        s = ops.paged_step(table, lens, _i32(new), free, count, page, rows, in_place=True)
        q, k, v = (torch.randn((rows, h, d), device="cuda").to(dt) for h in (hq, hkv, hkv))
        qt = ops.rope_append(q, k, v, s.positions, s.slots, inv, kc, vc, mscale=m)
        out = ops.paged_attention(qt, kc, vc, table, s.kv_lens, s.cu_q, max(new))
        cu = s.cu_q.tolist()
        assert s.refused.item() == 0
        for r in range(b):
            at = slice(cu[r], cu[r + 1])
            pos = s.positions[at].cpu()
            hist[r][0].append(R.turn(k[at].cpu(), pos, inv.cpu(), False, m).to(dt)), hist[r][1].append(v[at].cpu())
            n = sum(len(x) for x in hist[r][0])
            if new[r] == 0:
                continue
            pk, pv = (torch.cat(x)[None].transpose(1, 2) for x in hist[r])   # one page that holds everything
            want, tol = R.attention(qt[at], pk, pv, _i32([[0]]), _i32([n]), _i32([0, new[r]]), d ** -0.5, 0, 0)
            # the cache's keys may differ from the 64-bit turn by one step where that falls between two values: scores move by scale |q| |k| 2^-10 at most
            more = 2 * (qt[at].cpu().double().abs().sum(-1, keepdim=True) * pk.double().abs().amax() * d ** -0.5 * 2.0 ** -10) * pv.double().abs().amax()
            assert ((out[at].cpu().double() - want).abs() <= tol + more).all(), (new, r)
    assert ops.paged_release(table, lens, torch.tensor([True, False, True], device="cuda"), free, count, page).item() == 0
    assert lens.tolist()[0] == 0 and count.item() == 40 - (-(-int(lens[1]) // page))


# ------------------------------------------------------------------------------------------------ layouts, large offsets, calls out of the ordinary
@pytest.mark.parametrize("qn", [[1, 2, 1], [60, 1, 33]])
def test_heads_apart_and_transposed(qn):
    """Queries and output whose heads are not neighbours: every second block of d values; heads outside, tokens inside; keys head by head over all pages."""
    kv, hq, hkv, d, page = [70, 200, 33], 8, 2, 128, 16
    k, v, table = R.pool(kv, page, hkv, d, F16, 21)
    t = sum(qn)
    q = torch.randn((t, hq, d), device="cuda").to(F16)
    lens, cu = _i32(kv), _i32([sum(qn[:i]) for i in range(4)])
    want = ops.paged_attention(q, k, v, table, lens, cu, max(qn))
    for lay in ("apart", "heads first"):
        mk = (lambda: torch.zeros((t, hq, 2, d), dtype=F16, device="cuda")[:, :, 1]) if lay == "apart" else (lambda: torch.zeros((hq, t, d), dtype=F16, device="cuda").transpose(0, 1))
        q2, out = mk(), mk()
        q2.copy_(q)
        assert torch.equal(ops.paged_attention(q2, k, v, table, lens, cu, max(qn), out=out), want)
        inv, _ = ops.rope_frequencies(d)
        pos = torch.arange(t, device="cuda").to(torch.int32)
        assert torch.equal(ops.rope(q2, pos, inv, out=mk()), ops.rope(q, pos, inv))
    k2, v2 = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))        # [head][page] in memory
    assert torch.equal(ops.paged_attention(q, k2, v2, table, lens, cu, max(qn)), want)
    for bad in (q[:1].expand(t, hq, d), q[:, :1].expand(t, hq, d)):
        with pytest.raises(ValueError, match="overlap"):
            ops.paged_attention(q, k, v, table, lens, cu, max(qn), out=bad)


@pytest.mark.parametrize("qn", [[1, 2, 1], [60, 1, 133], [7, 300, 4]])
def test_output_in_the_queries_place(qn):
    kv = [70, 900, 333]
    k, v, table = R.pool(kv, 32, 2, 128, BF16, 22)
    q = torch.randn((sum(qn) + 2, 8, 128), device="cuda").to(BF16)
    lens, cu = _i32(kv), _i32([sum(qn[:i]) for i in range(4)])
    want = ops.paged_attention(q, k, v, table, lens, cu, max(qn), out=q.clone())
    assert ops.paged_attention(q, k, v, table, lens, cu, max(qn), out=q) is q and torch.equal(q, want)


def test_cache_beyond_four_gigabytes():
    """Pages whose bytes lie behind 2^32 (and values behind 2^31): append and attention reach them."""
    page, hkv, d, n = 64, 8, 128, 40000                                      # 5.2 GB each
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("16 GB of free device memory needed")
    kc, vc = (torch.empty((n, hkv, page, d), dtype=F16, device="cuda") for _ in range(2))
    t, ids = 150, [n - 1, 5, n - 7]
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((t, h, d), generator=g).to(F16).cuda() for h in (16, hkv, hkv))
    pos = torch.arange(t)
    slots = torch.tensor([ids[p // page] * page + p % page for p in range(t)], dtype=torch.int32).cuda()
    inv, _ = ops.rope_frequencies(d)
    qt = ops.rope_append(q, k, v, pos.to(torch.int32).cuda(), slots, inv, kc, vc)
    table, small = _i32([ids]), _i32([[0, 1, 2]])
    ks, vs = (c[torch.tensor(ids, device="cuda")].clone() for c in (kc, vc))
    for lens, cu in ((_i32([t]), _i32([0, t])), (_i32([t]), _i32([0, 1]))):
        rows = int(cu[1])
        got = ops.paged_attention(qt[:rows], kc, vc, table, lens, cu, rows)
        assert torch.equal(got, ops.paged_attention(qt[:rows], ks, vs, small, lens, cu, rows))
        want, tol = R.attention(qt[:rows], ks, vs, small, lens, cu, d ** -0.5, 0, 0)
        assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("qn", [1, 40])
def test_row_offsets_out_of_order(qn):
    """Offsets that fall, are negative or lie behind the rows reach no memory outside the tensors: the kernels bring them inside. Requests with good ones are served."""
    kv = [50, 60, 70]
    k, v, table = R.pool(kv, 16, 1, 64, F16, 23)
    whole = torch.zeros((3 * qn + 6, 8, 64), dtype=F16, device="cuda")
    q = whole[3:3 * qn + 3]
    q.normal_()
    good = [0, qn, 2 * qn, 3 * qn]
    want = ops.paged_attention(q, k, v, table, _i32(kv), _i32(good), qn)
    for cu in ([0, qn, -5, -9], [0, qn, 10 ** 9, 2 ** 31 - 1], [0, qn, qn, -2 ** 31]):
        out = torch.zeros_like(whole)
        ops.paged_attention(q, k, v, table, _i32(kv), _i32(cu), qn, out=out[3:3 * qn + 3])
        assert torch.equal(out[3:3 + qn], want[:qn]) and (out[:3] == 0).all() and (out[3 * qn + 3:] == 0).all()
    out = ops.paged_attention(q, k, v, table, _i32([-4, 50 * 2 ** 20, 70]), _i32(good), qn)      # lengths that are negative or beyond any table
    assert (out[:qn] == 0).all() and torch.equal(out[2 * qn:], want[2 * qn:])
    ops.check_device_status()


@pytest.mark.parametrize("one_stream", [False, True])
def test_another_stream_and_threads(one_stream):
    """Calls on side streams, from two host threads at once (on streams of their own or on one), give what calls in a row give."""
    import threading
    k, v, table = R.pool([700, 300], 32, 2, 128, F16, 24)
    lens = _i32([700, 300])
    jobs = [(torch.randn((n * 2, 8, 128), device="cuda").to(F16), _i32([0, n, 2 * n]), n) for n in (1, 30, 2, 90)]
    want = [ops.paged_attention(q, k, v, table, lens, cu, n) for q, cu, n in jobs]
    torch.cuda.synchronize()
    got = [[None] * 4 for _ in range(2)]
    shared = torch.cuda.Stream()

    def work(who):
        with torch.cuda.stream(shared if one_stream else torch.cuda.Stream()):
            for _ in range(20):
                for i, (q, cu, n) in enumerate(jobs):
                    got[who][i] = ops.paged_attention(q, k, v, table, lens, cu, n)
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(w,)) for w in range(2)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_first_cuda_call_of_a_thread():
    """Both kernels as the first CUDA call that a host thread makes."""
    import threading
    k, v, table = R.pool([300], 32, 2, 128, F16, 25)
    lens, got = _i32([300]), {}
    jobs = {n: (torch.randn((n, 8, 128), device="cuda").to(F16), _i32([0, n])) for n in (1, 50)}
    outs = {n: torch.zeros_like(q) for n, (q, _) in jobs.items()}
    torch.cuda.synchronize()
    for n, (q, cu) in jobs.items():
        t = threading.Thread(target=lambda: got.update({n: ops.paged_attention(q, k, v, table, lens, cu, n, out=outs[n])}))
        t.start(), t.join()
        assert torch.equal(got[n], ops.paged_attention(q, k, v, table, lens, cu, n))
