"""Plain 64-bit forms of the paged-cache operators for the tests, and the bounds that their tolerances are made of."""
import math

import torch


def step(lens, news, free, count, table, page, rows):
    """Request by request on Python integers: (cu_q, kv_lens, positions, slots, lens, count, refused, table)."""
    table = [list(r) for r in table]
    cu, kv, out_lens, refused = [0], [], [], 0
    pos, slots = [-1] * rows, [-1] * rows
    first = upto = taken = 0
    for r, (n, q) in enumerate(zip(lens, news)):
        q = max(0, q)
        have, want = -(-n // page), -(-(n + q) // page)
        fits = want <= len(table[r]) and first + q <= rows
        need = want - have if fits else 0
        upto += need
        ok = fits and (need == 0 or upto <= count)
        if ok:
            for k in range(need):
                table[r][have + k] = free[count - 1 - (upto - need + k)]
            taken += need
            for i in range(q):
                p = n + i
                pos[first + i], slots[first + i] = p, table[r][p // page] * page + p % page
        refused += not ok
        kv.append(n + q if ok else 0)
        out_lens.append(n + q if ok else n)
        first += q
        cu.append(min(first, rows))
    return cu, kv, pos, slots, out_lens, count - taken, refused, table


def turn(x, pos, inv, interleaved, mscale):
    """x [T, heads, d] in 64 bits, its first 2 len(inv) values turned."""
    y, rot = x.double().clone(), 2 * inv.numel()
    ang = pos.double()[:, None, None] * inv.double()
    c, s = ang.cos() * mscale, ang.sin() * mscale
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = y[..., i].clone(), y[..., j].clone()
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y


def turn_bound(x, y, inv, interleaved, mscale):
    """|difference| allowed against `turn` (y its result): half a step of the type, and (|a| + |b|) mscale 2^-20 for the arithmetic in 32 bits: rounding the reduced
    angle (2^-22.3), sine and cosine (2^-23), three roundings of the sum (3 x 2^-24) stay below 2^-20 together."""
    rot, m = 2 * inv.numel(), x.double().abs().clone()
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    ab = m[..., i] + m[..., j]
    m = torch.zeros_like(m)
    m[..., i] = m[..., j] = ab
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    return torch.finfo(x.dtype).eps / 2 * y.abs() + m * mscale * 2.0 ** -20 + tiny


def attention(q, kc, vc, table, kv, cu, scale, window, sinks):
    """(o, bound) in 64 bits on the CPU: softmax over the visible keys of each row, and how far a kernel may be off.

    A kernel rounds the weights p to the type (u = eps / 2 relative, and 2^-25 in absolute terms where fp16 runs out of exponents: weights count from a maximum that gives
    one of them 1 at least) and the result once more; its scores carry the rounding of a sum of d products in 32 bits, (d + 2) 2^-23 of the sum of magnitudes, and
    the exponential 2^-20. Errors e of the weights move o by at most 2 e sum p |v| (numerator and denominator)."""
    u = torch.finfo(q.dtype).eps / 2
    fp16 = q.dtype == torch.float16
    q, kc, vc = q.cpu().double(), kc.cpu().double(), vc.cpu().double()
    table, kv, cu = table.cpu().long(), kv.cpu().tolist(), cu.cpu().tolist()
    page, group = kc.shape[2], q.shape[1] // kc.shape[1]
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    for r, n in enumerate(kv):
        rows = cu[r + 1] - cu[r]
        end = min(n, table.shape[1] * page)
        if rows <= 0 or n <= 0:
            continue
        ids = table[r, :-(-end // page)]
        held = (ids >= 0) & (ids < kc.shape[0])
        k, v = (torch.where(held.view(-1, 1, 1, 1), x[ids.clamp(0, kc.shape[0] - 1)], 0.0).transpose(1, 2).flatten(0, 1)[:end] for x in (kc, vc))      # [keys, heads, d]
        p = torch.arange(n - rows, n)[:, None]
        j = torch.arange(end)[None]
        see = j <= p
        if window:
            see &= (j > p - window) | (j < sinks)
        alive = see.any(0)                                                   # places no row sees may hold anything
        k, v = torch.where(alive[:, None, None], k, 0.0), torch.where(alive[:, None, None], v, 0.0)
        for h in range(q.shape[1]):
            x, kh, vh = q[cu[r]:cu[r + 1], h], k[:, h // group], v[:, h // group]
            s = (x @ kh.T * scale).masked_fill(~see, -math.inf)
            top = s.amax(1, keepdim=True)
            w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
            es = (x.abs() @ kh.abs().T * abs(scale) * (x.shape[1] + 2) * 2.0 ** -23).masked_fill(~see, 0.0).amax(1, keepdim=True)
            a = w @ vh.abs()
            o[cu[r]:cu[r + 1], h] = w @ vh
            low = see.sum(1, keepdim=True) * (2.0 ** -25 if fp16 else 0.0) * vh.abs().amax()
            tol[cu[r]:cu[r + 1], h] = u * (w @ vh).abs() + (u * (1 + u) + 2 * (es + 2.0 ** -20)) * a + low + 2.0 ** -25
    return o, tol


def pool(kv, page, hkv, d, dtype, seed, device="cuda", spare=3, cols=None, fill=None, stale=float("nan")):
    """A cache pool of random values in which request r holds kv[r] tokens in shuffled pages; places that hold none are `stale`. Returns (k, v, table)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in kv]
    n = sum(need) + spare
    ids = torch.randperm(n, generator=g)
    cols = max(max(need), 1) if cols is None else cols
    table = torch.full((len(kv), cols), -7 if fill is None else fill, dtype=torch.int32)
    k, v = (torch.randn((n, hkv, page, d), generator=g) for _ in range(2))
    at = 0
    live = torch.zeros((n, page), dtype=torch.bool)
    for r, m in enumerate(need):
        table[r, :m] = ids[at:at + m].to(torch.int32)
        t = torch.arange(kv[r])
        live[ids[at:at + m][t // page], t % page] = True
        at += m
    for x in (k, v):
        x.masked_fill_(~live[:, None, :, None], stale)
    return k.to(dtype).to(device), v.to(dtype).to(device), table.to(device)
