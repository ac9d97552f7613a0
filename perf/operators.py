"""Serving attention over a paged cache, the part of a decoder layer between its q | k | v product and its o product: the step's slots from request lengths,
rotary positions with the cache append, and attention of the step's new tokens over the cache. Each case is one pass through one operator.

A case is a dict of plain values; `prepare` makes the inputs from a seed (lengths go by the case alone, so that `work` knows them), `run` is one pass (elementary torch
operations in 32 bits, or the package's calls when `own` is set), `exact` the same outputs in 64 bits. Sizes are those of the benchmark's 32B-class layer (64 query / 8
key-value heads of 128) and generic ones."""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the bookkeeping of a decode step: 64 sequences, one new token each (latency)
        dict(name="step_decode_b64", kind="step", b=64, new_lo=1, new_hi=1, ctx_lo=100, ctx_hi=16000, page=64),
        # a busy server's step: 1000 requests with chunks of up to 120 tokens, small pages
        dict(name="step_mixed_b1000", kind="step", b=1000, new_lo=0, new_hi=120, ctx_lo=0, ctx_hi=4000, page=16),
        # positions and cache append of a decode step of 64 sequences in the benchmark's layer
        dict(name="rope_decode_t64", kind="rope", t=64, hq=64, hkv=8, d=128, rot=128, inter=False, page=64, far=32000, dtype="fp16"),
        # the same of a long prompt chunk at far positions (frequencies stretched for a long context)
        dict(name="rope_prefill_t8191", kind="rope", t=8191, hq=64, hkv=8, d=128, rot=128, inter=False, page=64, far=1000000, dtype="fp16"),
        # a model that turns part of each head, neighbours paired, bf16, an odd number of heads
        dict(name="rope_partial_t1000", kind="rope", t=1000, hq=25, hkv=5, d=64, rot=32, inter=True, page=16, far=8000, dtype="bf16"),
        # one sequence, one token, a short context: latency
        dict(name="attn_decode_b1", kind="attn", b=1, q_lo=1, q_hi=1, ctx_lo=777, ctx_hi=777, hq=64, hkv=8, d=128, page=64, window=0, sinks=0, dtype="fp16"),
        # a decode batch of the benchmark's layer over ragged contexts: cache bandwidth
        dict(name="attn_decode_b64", kind="attn", b=64, q_lo=1, q_hi=1, ctx_lo=1000, ctx_hi=16000, hq=64, hkv=8, d=128, page=64, window=0, sinks=0, dtype="fp16"),
        # two very long contexts, few rows: the work has to be split over the context
        dict(name="attn_decode_long", kind="attn", b=2, q_lo=1, q_hi=1, ctx_lo=120000, ctx_hi=131000, hq=32, hkv=4, d=128, page=128, window=0, sinks=0, dtype="fp16"),
        # a decode batch with a sliding window and four first tokens that stay visible
        dict(name="attn_decode_window", kind="attn", b=128, q_lo=1, q_hi=1, ctx_lo=3000, ctx_hi=20000, hq=32, hkv=8, d=128, page=16, window=2048, sinks=4, dtype="bf16"),
        # a prompt of 4001 tokens from its start
        dict(name="attn_prefill_t4001", kind="attn", b=1, q_lo=4001, q_hi=4001, ctx_lo=0, ctx_hi=0, hq=64, hkv=8, d=128, page=64, window=0, sinks=0, dtype="fp16"),
        # a chunk of 1024 tokens of a long prompt, 32000 of them already in the cache
        dict(name="attn_chunk_1k_on_32k", kind="attn", b=1, q_lo=1024, q_hi=1024, ctx_lo=32000, ctx_hi=32000, hq=64, hkv=8, d=128, page=64, window=0, sinks=0, dtype="fp16"),
        # decoding sequences and prompt chunks in one batch, small heads, window and sinks
        dict(name="attn_mixed_b12", kind="attn", b=12, q_lo=1, q_hi=300, ctx_lo=0, ctx_hi=3800, hq=28, hkv=4, d=64, page=32, window=1500, sinks=16, dtype="bf16"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    kind = rng.choice(("step", "rope", "rope", "decode", "decode", "decode", "chunk", "chunk", "mixed"))
    page, dtype = rng.choice((16, 32, 64, 128, 256)), rng.choice(("fp16", "fp16", "bf16"))
    if kind == "step":
        return dict(kind="step", b=_log(rng, 1, 1000), new_lo=rng.choice((0, 1)), new_hi=_log(rng, 1, 120), ctx_lo=0, ctx_hi=_log(rng, 10, 4000), page=page)
    d, hkv = rng.choice((64, 128, 128)), rng.choice((1, 2, 4, 5, 8))
    hq = hkv * rng.choice((1, 2, 3, 4, 5, 7, 8))
    if kind == "rope":
        return dict(kind="rope", t=_log(rng, 1, 8191), hq=hq, hkv=hkv, d=d, rot=rng.choice((d, d, d // 2, d // 4, 48)), inter=rng.choice((False, False, True)), page=page,
                    far=_log(rng, 100, 1000000), dtype=dtype)
    window = rng.choice((0, 0, _log(rng, 16, 8192)))
    sinks = rng.choice((0, 4, 33)) if window else 0
    more = dict(hq=hq, hkv=hkv, d=d, page=page, window=window, sinks=sinks, dtype=dtype)
    if kind == "decode":                                                     # 1 .. 4 new tokens a sequence
        b = _log(rng, 1, 128)
        hi = _log(rng, 64, max(65, min(131000, 1000000 // b)))
        q = rng.choice((1, 1, 1, 2, 4))
        return dict(kind="attn", b=b, q_lo=1, q_hi=q, ctx_lo=hi // rng.choice((1, 2, 16)), ctx_hi=hi, **more)
    if kind == "chunk":                                                      # one or a few sequences, a chunk of a prompt each
        b, q = rng.choice((1, 1, 2, 3)), _log(rng, 17, 2048)
        hi = _log(rng, 16, max(17, min(32000, 1500000000 // (b * q * hq) - q)))
        return dict(kind="attn", b=b, q_lo=max(1, q // 2), q_hi=q, ctx_lo=hi // 3, ctx_hi=hi, **more)
    b, q = _log(rng, 2, 16), _log(rng, 5, 300)                               # decoding sequences and chunks together
    hi = _log(rng, 16, max(17, min(8000, 1500000000 // (b * q * hq) - q)))
    return dict(kind="attn", b=b, q_lo=1, q_hi=q, ctx_lo=0, ctx_hi=hi, **more)


def _lengths(c):
    """(tokens already cached, new tokens) of each request of a case: by its values alone, the same for every seed."""
    r = random.Random("%s %s %s" % (c["b"], c["ctx_lo"], c["ctx_hi"]))
    lo, hi = (c["new_lo"], c["new_hi"]) if c["kind"] == "step" else (c["q_lo"], c["q_hi"])
    ctx = [r.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["b"])]
    new = [r.choice((lo, r.randint(lo, hi), hi)) for _ in range(c["b"])]
    new[0] = hi                                                              # one request has the longest chunk
    return ctx, new


def _visible(c):
    """Visible (token, key) pairs, and the keys that some token of their request sees."""
    w, s = c["window"], c["sinks"]
    pairs = keys = 0
    for n, q in zip(*_lengths(c)):
        for p in range(n, n + q):
            lo = max(0, p - w + 1) if w else 0
            pairs += p + 1 - lo + min(s, lo)
        lo = max(0, n - w + 1) if w else 0
        keys += n + q - lo + min(s, lo)
    return pairs, keys


def work(c):
    if c["kind"] == "step":
        ctx, new = _lengths(c)
        pages = sum(-(-(n + q) // c["page"]) - -(-n // c["page"]) for n, q in zip(ctx, new))
        return {"bytes": 4 * (2 * c["b"] + 2 * pages + 3 * c["b"] + 2 * sum(new)), "flops": 0}
    if c["kind"] == "rope":
        moved = 2 * 2 * c["t"] * (c["hq"] + 2 * c["hkv"]) * c["d"]
        return {"bytes": moved + 8 * c["t"], "flops": 3 * c["t"] * (c["hq"] + c["hkv"]) * c["rot"]}
    pairs, keys = _visible(c)
    tokens = sum(_lengths(c)[1])
    return {"bytes": 2 * 2 * keys * c["hkv"] * c["d"] + 2 * 2 * tokens * c["hq"] * c["d"] + 4 * keys // c["page"], "flops": 4 * pairs * c["hq"] * c["d"]}


# ------------------------------------------------------------------------------------------------ inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    page = c["page"]
    s = dict(case=c, page=page)
    if c["kind"] == "step":
        ctx, new = _lengths(c)
        have, want = [-(-n // page) for n in ctx], [-(-(n + q) // page) for n, q in zip(ctx, new)]
        ids = torch.randperm(sum(want) + 100, generator=g, device=DEV).to(torch.int32)
        cols = max(want) + 3
        flat = torch.full((c["b"] * cols,), -1, dtype=torch.int32, device=DEV)
        held = torch.cat([torch.arange(k) + r * cols for r, k in enumerate(have)]).to(DEV)
        flat[held] = ids[:held.numel()]
        free = ids[held.numel():].contiguous()
        return dict(s, table=flat.view(c["b"], cols), lens=_ints(ctx), new=_ints(new), free=free, free_count=_ints([free.numel()]), rows=sum(new))
    dt = DTYPE[c["dtype"]]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    if c["kind"] == "rope":
        t = c["t"]
        n = -(-t // page) + 2                                                # a pool with room for the tokens, in places drawn from the seed
        qkv = torch.randn((t, (hq + 2 * hkv) * d), device=DEV, generator=g).to(dt)      # the q | k | v product's output
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split((hq * d, hkv * d, hkv * d), dim=1))
        first = int(torch.randint(0, c["far"], (1,), generator=g, device=DEV))
        pos = (first + torch.arange(t, device=DEV)) if t > 128 else torch.randint(0, c["far"], (t,), generator=g, device=DEV)
        slots = torch.randperm(n * page, generator=g, device=DEV)[:t]
        inv = 500000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=DEV) / c["rot"])
        inv = torch.where(inv < 2 * math.pi / 8192, inv / 8, inv)            # slow turns stretched eightfold, as for a context longer than the one trained on
        kc, vc = (torch.zeros((n, hkv, page, d), dtype=dt, device=DEV) for _ in range(2))
        return dict(s, q=q, k=k, v=v, pos=pos.to(torch.int32), slots=slots.to(torch.int32), inv=inv.float(), kc=kc, vc=vc, stretch=1.0 + 0.1 * math.log(8))
    ctx, new = _lengths(c)
    kv = [n + q for n, q in zip(ctx, new)]
    cols = -(-max(kv) // page)
    pages = [-(-n // page) for n in kv]
    n = sum(pages) + 7
    ids = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    flat = torch.zeros((c["b"] * cols,), dtype=torch.int32, device=DEV)
    held = torch.cat([torch.arange(k) + r * cols for r, k in enumerate(pages)]).to(DEV)
    flat[held] = ids[:held.numel()]
    mk = lambda *shape: torch.randn(shape, device=DEV, generator=g, dtype=torch.float16 if dt == torch.float16 else torch.float32).to(dt)  # noqa: E731
    cu = [0]
    for q in new:
        cu.append(cu[-1] + q)
    return dict(s, q=mk(cu[-1], hq, d) * 2, kc=mk(n, hkv, page, d), vc=mk(n, hkv, page, d), table=flat.view(c["b"], cols), kv=_ints(kv), cu=_ints(cu), max_q=max(new))


# ------------------------------------------------------------------------------------------------ one pass
def _plain_step(s):
    page, lens, new, rows = s["page"], s["lens"].long(), s["new"].long(), s["rows"]
    b, cols = s["table"].shape
    cu = torch.cat((torch.zeros(1, dtype=torch.long, device=DEV), new.cumsum(0)))
    have, want = (lens + page - 1) // page, (lens + new + page - 1) // page
    fits = (want <= cols) & (cu[1:] <= rows)
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= s["free_count"].long()))
    taken = torch.where(served, need, 0)
    col = torch.arange(cols, device=DEV)[None]
    fill = served[:, None] & (col >= have[:, None]) & (col < want[:, None])
    at = s["free_count"].long() - 1 - ((upto - need - have)[:, None] + col)
    s["table"].copy_(torch.where(fill, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"]))
    t = torch.arange(rows, device=DEV)
    req = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=b - 1)
    on = served[req] & (t < cu[-1])
    pos = lens[req] + t - cu[req]
    slot = s["table"][req, (pos // page).clamp(0, cols - 1)].long() * page + pos % page
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return dict(cu_q=i32(cu.clamp(max=rows)), kv_lens=i32(torch.where(served, lens + new, 0)), positions=i32(torch.where(on, pos, -1)), slots=i32(torch.where(on, slot, -1)),
                lens=i32(torch.where(served, lens + new, lens)), free_count=i32(s["free_count"] - taken.sum()), refused=i32((~served).sum().reshape(1)), table=s["table"])


def _turn(x, cos, sin, rot, inter):
    """x [t, heads, d] in 32 bits, its first `rot` values turned by the pairs' angles."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, w), -1).flatten(-2) if inter else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_rope(s):
    c, page = s["case"], s["page"]
    angle = s["pos"].double()[:, None, None] * s["inv"].double()
    cos, sin = (angle.cos() * s["stretch"]).float(), (angle.sin() * s["stretch"]).float()
    q = _turn(s["q"].float(), cos, sin, c["rot"], c["inter"]).to(s["q"].dtype)
    k = _turn(s["k"].float(), cos, sin, c["rot"], c["inter"]).to(s["k"].dtype)
    at, off = s["slots"].long() // page, s["slots"].long() % page
    s["kc"][at, :, off] = k
    s["vc"][at, :, off] = s["v"]
    return dict(q=q, k_cache=s["kc"], v_cache=s["vc"])


def _plain_attn(s):
    c, page, dt = s["case"], s["page"], s["q"].dtype
    hkv, d, b = c["hkv"], c["d"], c["b"]
    cu, kv = s["cu"].long(), s["kv"].long()
    n = cu[1:] - cu[:-1]
    row = torch.arange(s["max_q"], device=DEV)
    at = (cu[:-1, None] + row).clamp(max=s["q"].shape[0] - 1)                # [b, q] rows of the packed tokens
    q = s["q"][at].float().view(b, s["max_q"], hkv, -1, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    key = torch.arange(s["table"].shape[1] * page, device=DEV)
    pos = (kv - n)[:, None] + row
    see = (key <= pos[..., None]) & (key < kv[:, None, None])
    if c["window"]:
        see &= (key > pos[..., None] - c["window"]) | (key < c["sinks"])
    pages = s["table"].long()
    k = s["kc"][pages].float().transpose(1, 2).reshape(b, hkv, -1, d)        # [b, h, keys, d]
    sc = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).view(b, hkv, -1, s["max_q"], key.numel())
    del k
    sc.masked_fill_(~see[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((key < kv[:, None]).view(b, 1, -1, 1), s["vc"][pages].float().transpose(1, 2).reshape(b, hkv, -1, d), 0.0)
    o = torch.matmul(p.view(b, hkv, -1, key.numel()), v).view(b, hkv, -1, s["max_q"], d)
    o = (o / torch.where(total == 0, 1.0, total)).permute(0, 3, 1, 2, 4).reshape(b, s["max_q"], -1, d)
    return o[row < n[:, None]].to(dt)


def run(s):
    kind = s["case"]["kind"]
    if own:
        from kyojin_mac_b200 import ops
        c = s["case"]
        if kind == "step":
            r = ops.paged_step(s["table"], s["lens"], s["new"], s["free"], s["free_count"], s["page"], s["rows"])
            return dict(cu_q=r.cu_q, kv_lens=r.kv_lens, positions=r.positions, slots=r.slots, lens=r.lens, free_count=r.free_count, refused=r.refused, table=s["table"])
        if kind == "rope":
            q = ops.rope_append(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["inv"], s["kc"], s["vc"], interleaved=c["inter"], mscale=s["stretch"])
            return dict(q=q, k_cache=s["kc"], v_cache=s["vc"])
        return ops.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["kv"], s["cu"], s["max_q"], window=c["window"], sinks=c["sinks"])
    return _plain_step(s) if kind == "step" else _plain_rope(s) if kind == "rope" else _plain_attn(s)


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(c, seed):
    if c["kind"] == "step":                                                  # whole numbers: nothing is rounded
        return None
    s = prepare(c, seed)
    page = c["page"]
    if c["kind"] == "rope":
        rot, half = c["rot"], c["rot"] // 2
        first, second = (range(0, rot, 2), range(1, rot, 2)) if c["inter"] else (range(half), range(half, rot))
        z = torch.polar(torch.full((), s["stretch"], dtype=torch.float64, device=DEV).expand(c["t"], half), s["pos"].double()[:, None] * s["inv"].double())[:, None]

        def turned(x):
            y = x.double().clone()
            w = torch.complex(y[..., list(first)], y[..., list(second)]) * z
            y[..., list(first)], y[..., list(second)] = w.real, w.imag
            return y
        kc, vc = s["kc"].double(), s["vc"].double()
        for store, x in ((kc, turned(s["k"])), (vc, s["v"].double())):
            flat = store.transpose(1, 2).reshape(-1, c["hkv"], c["d"])       # [slot, head, d]
            flat[s["slots"].long()] = x
            store.copy_(flat.view(-1, page, c["hkv"], c["d"]).transpose(1, 2))
        return dict(q=turned(s["q"]), k_cache=kc, v_cache=vc)
    ctx, new = _lengths(c)
    group = c["hq"] // c["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for r, (n, t) in enumerate(zip(ctx, new)):
        ids = s["table"][r, :-(-(n + t) // page)].long()
        p = torch.arange(n, n + t, device=DEV)[:, None]
        j = torch.arange(n + t, device=DEV)[None]
        hide = j > p
        if c["window"]:
            hide |= (p - j >= c["window"]) & (j >= c["sinks"])
        for h in range(c["hkv"]):
            k, v = (x[ids, h].reshape(-1, c["d"])[:n + t].double() for x in (s["kc"], s["vc"]))
            for i in range(h * group, (h + 1) * group):
                sc = s["q"][at:at + t, i].double() @ k.T / math.sqrt(c["d"])
                out[at:at + t, i] = torch.softmax(sc.masked_fill(hide, -math.inf), -1) @ v
        at += t
    return out
