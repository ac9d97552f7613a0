"""Thin torch-tensor front end of the C ABI: pointers, sizes and the current CUDA stream go straight to libkyb.so."""
from __future__ import annotations

import contextlib
import math
from typing import NamedTuple

import numpy as np
import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib, flags as F
from .layout import FMT_ID, padded_rows


# The current stream's handle without a torch.cuda.Stream object around it: every launch asks for it (3.2 us through torch.cuda.current_stream(), 0.2 us so).
_raw_stream, _cur_device = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)


def _stream() -> int:
    if _raw_stream is None or not torch.cuda.is_initialized():
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_cur_device())


def _fmt(fmt) -> int:
    if isinstance(fmt, str):
        if fmt not in FMT_ID:
            raise ValueError(f"unknown format {fmt!r}")
        return FMT_ID[fmt]
    return int(fmt)


def _need_cuda(*ts):
    for t in ts:
        if t is not None and (not isinstance(t, torch.Tensor) or not t.is_cuda):
            raise ValueError("kyojin_mac_b200 operators take CUDA tensors (there is no CPU path)")


def t16_nbytes(fmt, n: int, k: int) -> int:
    v = _lib.lib().kyb_t16_nbytes(_fmt(fmt), n, k)
    if v == 0:
        raise ValueError(f"bad T16 shape fmt={fmt} n={n} k={k} (k must be a positive multiple of 256)")
    return v


def raw_to_t16(fmt, raw: torch.Tensor, n: int, k: int) -> torch.Tensor:
    """GGUF rows uint8 [n, row_bytes] on the device -> T16 bytes on the device."""
    _need_cuda(raw)
    raw = raw.contiguous()
    out = torch.empty(t16_nbytes(fmt, n, k), dtype=torch.uint8, device=raw.device)
    _lib.check(_lib.lib().kyb_repack_raw_to_t16(_fmt(fmt), raw.data_ptr(), n, k, out.data_ptr(), _stream()))
    return out


def t16_to_raw(fmt, t16: torch.Tensor, n: int, k: int) -> torch.Tensor:
    _need_cuda(t16)
    rb = _lib.lib().kyb_raw_row_bytes(_fmt(fmt), k)
    out = torch.empty((n, rb), dtype=torch.uint8, device=t16.device)
    _lib.check(_lib.lib().kyb_repack_t16_to_raw(_fmt(fmt), t16.data_ptr(), n, k, out.data_ptr(), _stream()))
    return out


def dequant(fmt, t16: torch.Tensor, n: int, k: int, dtype=torch.float16, gscale: float = 1.0, row0: int = 0, nrows: int | None = None) -> torch.Tensor:
    """T16 -> [nrows, k] float32 (bit-equal to the reference decoder) or float16 (that value rounded, saturated)."""
    _need_cuda(t16)
    nrows = n - row0 if nrows is None else nrows
    if dtype not in (torch.float32, torch.float16):
        raise ValueError("dequant output is float32 or float16")
    out = torch.empty((nrows, k), dtype=dtype, device=t16.device)
    _lib.check(_lib.lib().kyb_dequant_t16(_fmt(fmt), t16.data_ptr(), n, k, row0, nrows, float(gscale), 0 if dtype == torch.float32 else 1,
                                          out.data_ptr(), k, _stream()))
    return out


_ws: dict = {}


def workspace(device, nbytes: int) -> torch.Tensor:
    """Grow-only scratch buffer per (device, stream): the chunk sums of the GEMV's two-launch form live here."""
    key = (device.index, _stream())
    buf = _ws.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = _ws[key] = torch.empty(max(nbytes, 4 << 20), dtype=torch.uint8, device=device)
    return buf


def release_workspaces(stream_id: int | None = None) -> None:
    """Drops the cached workspaces (of one stream id, or all): for callers that create and retire many streams."""
    for key in [k for k in _ws if stream_id is None or k[1] == stream_id]:
        del _ws[key]


def gemv(fmt, t16: torch.Tensor, n: int, k: int, x: torch.Tensor, gscale: float = 1.0, out: torch.Tensor | None = None, chained: bool = False,
         x2: torch.Tensor | None = None, limit: float | None = None) -> torch.Tensor:
    """y fp16 [m, n] = x fp16 [m, k] @ W^T for m <= 32, W in T16.
    chained: launch with programmatic stream serialization (the kernel sets up and prefetches weights while the preceding kernel of the stream drains, and waits
    for it before touching x or y): only when the weights were not written by the kernel directly before this call on the stream. Same bits either way.
    x2: gated input, the row fed to the product is fp16(silu(x row) * x2 row), formed while the rows are staged (optional clamp `limit`)."""
    _need_cuda(t16, x, x2)
    if x.dtype != torch.float16 or x.dim() != 2 or x.shape[1] != k:
        raise ValueError(f"x must be float16 [m, {k}], got {x.dtype} {tuple(x.shape)}")
    if x.stride(1) != 1:
        x = x.contiguous()
    if x2 is not None:
        if x2.dtype != torch.float16 or x2.shape != x.shape:
            raise ValueError("the gated form takes two float16 tensors of one shape")
        if x2.stride() != x.stride():
            x, x2 = x.contiguous(), x2.contiguous()
    m, fid = x.shape[0], _fmt(fmt)
    y = out if out is not None else x.new_empty((m, n))
    L = _lib.lib()
    need = L.kyb_gemv_workspace_bytes(fid, n, k, m)
    ws = workspace(x.device, need) if need else None
    wp, wn = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
    if x2 is not None:
        rc = L.kyb_gemv_glu_t16(fid, t16.data_ptr(), n, k, x.data_ptr(), x2.data_ptr(), float(limit or 0.0), m, x.stride(0), float(gscale), y.data_ptr(), y.stride(0), wp, wn,
                                1 if chained else 0, _stream())
    else:
        rc = L.kyb_gemv_t16(fid, t16.data_ptr(), n, k, x.data_ptr(), m, x.stride(0), float(gscale), y.data_ptr(), y.stride(0), wp, wn, 1 if chained else 0, _stream())
    if rc:
        _lib.check(rc)
    return y


def gemm_f16(a: torch.Tensor, b: torch.Tensor, gscale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """d fp16 [m, n] = a fp16 [m, k] @ b fp16 [n, k]^T on tcgen05 (fp32 accumulation in tensor memory, saturated fp16 result)."""
    _need_cuda(a, b)
    if a.dtype != torch.float16 or b.dtype != torch.float16 or a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"gemm_f16 takes float16 [m, k] and [n, k], got {a.dtype} {tuple(a.shape)} and {b.dtype} {tuple(b.shape)}")
    if a.stride(1) != 1:
        a = a.contiguous()
    if b.stride(1) != 1:
        b = b.contiguous()
    m, k = a.shape
    n = b.shape[0]
    d = out if out is not None else torch.empty((m, n), dtype=torch.float16, device=a.device)
    _lib.check(_lib.lib().kyb_gemm_f16_tn(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), m, n, k, float(gscale), d.data_ptr(), d.stride(0), _stream()))
    return d


def gemv_plan(fmt, n: int, k: int, m: int, workspace_bytes: int | None = None) -> dict:
    """How a decode product is launched; workspace_bytes: for a caller that brings that much scratch (None: as much as the best form wants)."""
    import ctypes
    out = (ctypes.c_int * 8)()
    L = _lib.lib()
    _lib.check(L.kyb_gemv_plan(_fmt(fmt), n, k, m, out) if workspace_bytes is None else L.kyb_gemv_plan_within(_fmt(fmt), n, k, m, workspace_bytes, out))
    return dict(zip(("nt", "aligned", "warps", "kc", "kbp", "ksplit", "smem", "grid"), list(out)))


def gemv_workspace_bytes(fmt, n: int, k: int, m: int) -> int:
    """Bytes of scratch the product needs (0: one launch; else chunk sums through the workspace and a finalize launch)."""
    return int(_lib.lib().kyb_gemv_workspace_bytes(_fmt(fmt), n, k, m))


def check_device_status() -> None:
    _lib.check(_lib.lib().kyb_check_device_status(_stream()))


def to_device_t16(fmt: str, raw_np: np.ndarray, n: int, k: int, device="cuda") -> torch.Tensor:
    """Host GGUF rows (numpy uint8 [n, row_bytes]) -> device T16, repacked on the device."""
    raw = torch.from_numpy(np.ascontiguousarray(raw_np)).to(device)
    return raw_to_t16(fmt, raw, n, k)


# ------------------------------------------------------------------------------------------------ routed experts
def _p(t):
    return None if t is None else t.data_ptr()


def moe_select(logits: torch.Tensor, E: int, K: int, norm: bool = True, has_shared: bool = False):
    """logits fp32 [T, >= E (+1)] -> (inds uint32-as-int32 [T*K], scs f32 [T*K], sgs f32 [T] or None)."""
    _need_cuda(logits)
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("router logits must be contiguous float32 [T, E(+1)]")
    T = logits.shape[0]
    inds = torch.empty(T * K, dtype=torch.int32, device=logits.device)
    scs = torch.empty(T * K, dtype=torch.float32, device=logits.device)
    sgs = torch.empty(T, dtype=torch.float32, device=logits.device) if has_shared else None
    _lib.check(_lib.lib().kyb_moe_select(logits.data_ptr(), logits.stride(0), T, E, K, int(norm), int(has_shared), inds.data_ptr(), scs.data_ptr(), _p(sgs), _stream()))
    return inds, scs, sgs


_ROUTER_PIECES: dict = {}


def _router_pieces(gw: torch.Tensor, sg: torch.Tensor | None):
    """The gate cut into three fp16 pieces per row for the tensor-core router, made once per (gate tensor, version) and kept (a few MB per gate)."""
    key = (gw.data_ptr(), gw._version, tuple(gw.shape), None if sg is None else (sg.data_ptr(), sg._version))
    hit = _ROUTER_PIECES.get(key)
    if hit is None:
        E, H = gw.shape
        rpad = int(_lib.lib().kyb_router_rpad(E, 0 if sg is None else 1))
        pieces = torch.empty((3 * rpad, H), dtype=torch.float16, device=gw.device)
        inv = torch.empty((rpad,), dtype=torch.float32, device=gw.device)
        _lib.check(_lib.lib().kyb_router_split(gw.data_ptr(), _p(sg), E, H, pieces.data_ptr(), inv.data_ptr(), _stream()))
        if len(_ROUTER_PIECES) >= 64:
            _ROUTER_PIECES.clear()
        hit = _ROUTER_PIECES[key] = (pieces, inv, rpad, gw, sg)              # the gate tensors are kept alive so that their addresses stay theirs
    return hit[0], hit[1], hit[2]


def router_logits(x: torch.Tensor, gw: torch.Tensor, sgw: torch.Tensor | None = None, tensor_cores: bool | None = None) -> torch.Tensor:
    """fp32 [T, E + 1] router logits of x [T, H] (fp32 / fp16 / bf16) on the fp32 gate gw [E, H]; column E = shared-expert gate logit (sgw [H]) or unwritten.
    tensor_cores: None = by size (fp16 activations, at least flags.ROUTER_TC_MIN_ROWS tokens: one tcgen05 GEMM on the gate cut into three fp16 pieces + a
    recombining launch; below that the fp32 kernels, whose two forms agree bit for bit); True / False force one path."""
    _need_cuda(x, gw)
    if gw.dtype != torch.float32 or x.dtype not in _DT or x.dim() != 2 or x.shape[1] != gw.shape[1]:
        raise ValueError("router_logits takes x [T, H] (fp32 / fp16 / bf16) and an fp32 gate [E, H]")
    x, gw = (x if x.stride(1) == 1 else x.contiguous()), gw.contiguous()
    sg = None if sgw is None else sgw.reshape(-1).to(torch.float32).contiguous()
    T, (E, H) = x.shape[0], gw.shape
    lg = torch.empty((T, E + 1), dtype=torch.float32, device=x.device)
    if sg is None:
        lg[:, E].zero_()                                                    # no shared expert: the column exists (fixed row pitch) and reads as 0
    if tensor_cores is None:
        tensor_cores = x.dtype == torch.float16 and T >= F.ROUTER_TC_MIN_ROWS and H % 64 == 0
    if tensor_cores:
        if x.dtype != torch.float16 or H % 64:
            raise ValueError("the tensor-core router takes float16 activations with H a multiple of 64")
        pieces, inv, rpad = _router_pieces(gw, sg)
        work = workspace(x.device, T * 3 * rpad * 4)
        _lib.check(_lib.lib().kyb_router_logits_tc(x.data_ptr(), x.stride(0), pieces.data_ptr(), inv.data_ptr(), T, E, 0 if sg is None else 1, H, work.data_ptr(), lg.data_ptr(),
                                                   lg.stride(0), _stream()))
        return lg
    _lib.check(_lib.lib().kyb_router_logits(x.data_ptr(), _DT[x.dtype], x.stride(0), gw.data_ptr(), _p(sg), T, E, H, lg.data_ptr(), lg.stride(0), _stream()))
    return lg


def dequant_rows(fmt, t16: torch.Tensor, n: int, k: int, rows: torch.Tensor, dtype=torch.float16, gscale: float = 1.0) -> torch.Tensor:
    """[len(rows), k] decoded rows of a T16 matrix, gathered by id (int tensor on the device, 0 <= id < n)."""
    _need_cuda(t16, rows)
    ids = rows.reshape(-1).to(torch.int32).contiguous()
    out = torch.empty((ids.numel(), k), dtype=dtype, device=t16.device)
    if ids.numel():
        _lib.check(_lib.lib().kyb_dequant_rows_t16(_fmt(fmt), t16.data_ptr(), n, k, ids.data_ptr(), ids.numel(), float(gscale), _DT[dtype], out.data_ptr(), k, _stream()))
    return out


def gather_flat(srcs, dsts, nbytes=None) -> None:
    """Copies srcs[i] into dsts[i] (equal byte counts, multiples of 16 bytes, 16-byte aligned) with one launch per 128 pairs. Entries are contiguous device tensors
    or raw device addresses (ints, e.g. peer-mapped pointers; then nbytes[i] gives the size)."""
    import ctypes as C
    n = len(srcs)
    if n == 0:
        return
    ptr = lambda t: t if isinstance(t, int) else t.data_ptr()
    sizes = []
    for i, (a, b) in enumerate(zip(srcs, dsts)):
        sz = None
        for t in (a, b):
            if isinstance(t, torch.Tensor):
                if not t.is_cuda or not t.is_contiguous():
                    raise ValueError("gather_flat copies contiguous CUDA tensors")
                tsz = t.numel() * t.element_size()
                if sz is not None and tsz != sz:
                    raise ValueError("gather_flat: source and destination differ in size")
                sz = tsz
        if sz is None:
            sz = int(nbytes[i])
        sizes.append(sz)
    for i in range(0, n, 128):
        m = min(128, n - i)
        S = (C.c_void_p * m)(*[ptr(t) for t in srcs[i:i + m]])
        D = (C.c_void_p * m)(*[ptr(t) for t in dsts[i:i + m]])
        B = (C.c_int64 * m)(*sizes[i:i + m])
        _lib.check(_lib.lib().kyb_gather_flat(S, D, B, m, _stream()))


def moe_plan(ids: torch.Tensor, E: int, topk: int, mt: int = 128, wts: torch.Tensor | None = None, rank: torch.Tensor | None = None):
    """Counting sort of the slots by expert. Returns dict(order, inv, tok, ids_s, wts_s, off, tb)."""
    _need_cuda(ids)
    ids = ids.reshape(-1).to(torch.int32).contiguous()
    P, dev = ids.numel(), ids.device
    mk = lambda n, dt: torch.empty(n, dtype=dt, device=dev)
    out = dict(order=mk(P, torch.int32), inv=mk(P, torch.int32), tok=mk(P, torch.int32), ids_s=mk(P, torch.int32),
               wts_s=mk(P, torch.float32) if wts is not None else None, off=mk(E + 1, torch.int32), tb=mk(E + 1, torch.int32))
    w = None if wts is None else wts.reshape(-1).to(torch.float32).contiguous()
    r = None if rank is None else rank.to(torch.int32).contiguous()
    _lib.check(_lib.lib().kyb_moe_plan(ids.data_ptr(), _p(w), _p(r), E, P, topk, mt, out["order"].data_ptr(), out["inv"].data_ptr(), out["tok"].data_ptr(),
                                       out["ids_s"].data_ptr(), _p(out["wts_s"]), out["off"].data_ptr(), out["tb"].data_ptr(), _stream()))
    return out


def gather_rows(x: torch.Tensor, src: torch.Tensor, div: int = 1, perm: torch.Tensor | None = None) -> torch.Tensor:
    """out[r] = x[src[r] // div] (fp16 rows), optional column permutation."""
    _need_cuda(x, src)
    if x.dtype != torch.float16 or x.stride(1) != 1:
        raise ValueError("gather_rows takes float16 rows")
    R, k = src.numel(), x.shape[1]
    out = torch.empty((R, k), dtype=torch.float16, device=x.device)
    _lib.check(_lib.lib().kyb_gather_rows(x.data_ptr(), x.stride(0), x.shape[0], src.data_ptr(), div, _p(perm), R, k, out.data_ptr(), k, _stream()))
    return out


def silu_mul(a: torch.Tensor, b: torch.Tensor, limit: float | None = None, perm: torch.Tensor | None = None) -> torch.Tensor:
    """fp16(silu(a) * b) computed in fp32 (optional clamp as the reference's swiglu_limit)."""
    _need_cuda(a, b)
    if a.shape != b.shape or a.dtype != torch.float16 or b.dtype != torch.float16 or a.stride() != b.stride() or a.stride(1) != 1:
        raise ValueError("silu_mul takes two float16 [rows, n] tensors of the same layout")
    rows, n = a.shape
    h = torch.empty((rows, n), dtype=torch.float16, device=a.device)
    _lib.check(_lib.lib().kyb_silu_mul(a.data_ptr(), b.data_ptr(), a.stride(0), rows, n, float(limit or 0.0), _p(perm), h.data_ptr(), n, _stream()))
    return h


def moe_combine(y: torch.Tensor, scs: torch.Tensor, K: int, sgs: torch.Tensor | None = None, shared: torch.Tensor | None = None, dtype=torch.float16) -> torch.Tensor:
    """y fp16 [T*K, H] (slot order), scs f32 [T*K] -> [T, H] weighted sum (+ gated shared expert)."""
    _need_cuda(y, scs)
    S, H = y.shape
    T = S // K
    o = torch.empty((T, H), dtype=dtype, device=y.device)
    _lib.check(_lib.lib().kyb_moe_combine(y.data_ptr(), y.stride(0), scs.data_ptr(), _p(sgs), _p(shared), 0 if shared is None else shared.stride(0), T, K, H,
                                          0 if dtype == torch.float32 else 1, o.data_ptr(), H, _stream()))
    return o


def moe_groups(eids: torch.Tensor, E: int):
    """Expert election for the gathered GEMV: slots of one expert are served 8 at a time. Returns the scratch triple (g_expert, g_slots, ngroups) that
    gemv_group takes as `groups`; one election serves every projection of a layer. Slots with an id outside [0, E) are in no group."""
    _need_cuda(eids)
    eids = eids.reshape(-1).to(torch.int32).contiguous()
    S = eids.numel()
    scratch = torch.empty(S * 9 + 1, dtype=torch.int32, device=eids.device)
    g_expert, g_slots, ngroups = scratch[:S], scratch[S:9 * S], scratch[9 * S:]
    _lib.check(_lib.lib().kyb_moe_groups(eids.data_ptr(), S, E, g_expert.data_ptr(), g_slots.data_ptr(), ngroups.data_ptr(), _stream()))
    return g_expert, g_slots, ngroups


def gemv_group(fmt, t16: torch.Tensor, n: int, k: int, E: int, x: torch.Tensor, eids: torch.Tensor, xrows: torch.Tensor | None = None, xdiv: int = 1,
               gs: torch.Tensor | None = None, out: torch.Tensor | None = None, groups=None, t16b: torch.Tensor | None = None, gsb: torch.Tensor | None = None,
               x2: torch.Tensor | None = None, limit: float | None = None) -> torch.Tensor:
    """y fp16 [S, n]: slot s = expert eids[s] applied to row xrows[s] (or s // xdiv) of x fp16 [*, k]; one weight read per expert and 8 slots.
    t16b (+ gsb): a second stack of the same shape in the same launch, y is [2 S, n] with its results in rows [S, 2 S). x2: gated input, the row fed to the
    product is fp16(silu(x row) * x2 row). groups: the election of moe_groups(eids, E) when the caller already has it."""
    _need_cuda(t16, x, eids, t16b, x2)
    if x.dtype != torch.float16 or x.stride(1) != 1 or x.shape[1] != k:
        raise ValueError(f"x must be float16 [rows, {k}]")
    if x2 is not None and (x2.dtype != torch.float16 or x2.shape != x.shape or x2.stride() != x.stride()):
        raise ValueError("the gated form takes two float16 tensors of one shape and layout")
    if t16b is not None and t16b.numel() != t16.numel():
        raise ValueError("the pair form takes two stacks of one shape and format")
    S = eids.numel()
    eids = eids.reshape(-1).to(torch.int32).contiguous()
    rows = S * (2 if t16b is not None else 1)
    y = out if out is not None else torch.empty((rows, n), dtype=torch.float16, device=x.device)
    if y.shape[0] != rows:
        raise ValueError(f"out must hold {rows} rows")
    g_expert, g_slots, ngroups = groups if groups is not None else moe_groups(eids, E)
    xr = None if xrows is None else xrows.reshape(-1).to(torch.int32).contiguous()
    _lib.check(_lib.lib().kyb_gemv_group_t16(_fmt(fmt), t16.data_ptr(), _p(t16b), n, k, E, x.data_ptr(), _p(x2), float(limit or 0.0), x.stride(0), eids.data_ptr(), _p(xr), xdiv, S,
                                             _p(gs), _p(gsb), y.data_ptr(), y.stride(0), g_expert.data_ptr(), g_slots.data_ptr(), ngroups.data_ptr(), _stream()))
    return y


def gemm_f16_grouped(a: torch.Tensor, b: torch.Tensor, n: int, E: int, tb: torch.Tensor, off: torch.Tensor, row_map: torch.Tensor | None = None,
                     gs: torch.Tensor | None = None, out: torch.Tensor | None = None, out_rows: int | None = None) -> torch.Tensor:
    """d [rows, n]: sorted rows a fp16 [s, k] of expert segments (off) times the fp16 expert stack b [E*n, k]; tile list tb (tiles of 128 rows)."""
    _need_cuda(a, b, tb, off)
    s, k = a.shape
    d = out if out is not None else torch.empty((out_rows or s, n), dtype=torch.float16, device=a.device)
    _lib.check(_lib.lib().kyb_gemm_f16_grouped(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), s, n, k, E, tb.data_ptr(), off.data_ptr(), _p(row_map), _p(gs),
                                               d.data_ptr(), d.stride(0), _stream()))
    return d


def gemm_kq(fmt, t16: torch.Tensor, n: int, k: int, a: torch.Tensor, gscale: float = 1.0, out: torch.Tensor | None = None, msub: int = 0,
            split: int | None = None) -> torch.Tensor:
    """d fp16 [m, n] = a fp16 [m, k] @ W^T with W decoded from its T16 tiles inside the GEMM (no fp16 copy of W in HBM).
    split: number of k-ranges (split-k through an fp32 workspace for products that leave most SMs idle); None = the library's suggestion when msub is 0
    and `flags.GEMM_SPLIT_K` is on, 1 = never."""
    _need_cuda(t16, a)
    if a.dtype != torch.float16 or a.dim() != 2 or a.shape[1] != k:
        raise ValueError(f"gemm_kq takes float16 [m, {k}], got {a.dtype} {tuple(a.shape)}")
    if a.stride(1) != 1:
        a = a.contiguous()
    m = a.shape[0]
    d = out if out is not None else a.new_empty((m, n))
    L = _lib.lib()
    if split is None:
        split = L.kyb_gemm_kq_split(_fmt(fmt), n, k, m) if (msub == 0 and F.GEMM_SPLIT_K) else 1
    if split > 1:
        need = L.kyb_gemm_kq_split_bytes(n, m, split)
        ws = workspace(a.device, need)
        _lib.check(L.kyb_gemm_kq_splitk(_fmt(fmt), t16.data_ptr(), n, k, a.data_ptr(), a.stride(0), m, float(gscale), d.data_ptr(), d.stride(0), split, ws.data_ptr(),
                                        ws.numel(), _stream()))
        return d
    _lib.check(L.kyb_gemm_kq(_fmt(fmt), t16.data_ptr(), n, k, a.data_ptr(), a.stride(0), m, float(gscale), d.data_ptr(), d.stride(0), msub, _stream()))
    return d


def gemm_kq_plan(fmt, n: int, k: int, m: int, split: int = 1, destinations: int = 1) -> dict:
    """The form gemm_kq (several destinations: gemm_kq_ag) takes for a shape: by CTA pairs or not, activation rows per work item, work items."""
    import ctypes
    out = (ctypes.c_int64 * 3)()
    _lib.check(_lib.lib().kyb_gemm_kq_plan(_fmt(fmt), n, k, m, split, destinations, out))
    return dict(pair=bool(out[0]), rows=out[1], items=out[2])


def gemm_kq_ag(fmt, t16: torch.Tensor, n: int, k: int, a: torch.Tensor, peer_ptrs, ldd: int, col0: int, gscale: float = 1.0, msub: int = 0) -> None:
    """gemm_kq whose epilogue stores every tile into the [m, ldd] fp16 output matrix of every rank (peer_ptrs: peer-mapped base addresses, own rank included) at
    column col0: the all-gather of an N-sharded linear happens inside the GEMM. The caller synchronises the ranks around the call."""
    _need_cuda(t16, a)
    if a.dtype != torch.float16 or a.dim() != 2 or a.shape[1] != k:
        raise ValueError(f"gemm_kq_ag takes float16 [m, {k}], got {a.dtype} {tuple(a.shape)}")
    if a.stride(1) != 1:
        a = a.contiguous()
    out = _lib.PeerOut.of(peer_ptrs)
    _lib.check(_lib.lib().kyb_gemm_kq_ag(_fmt(fmt), t16.data_ptr(), n, k, a.data_ptr(), a.stride(0), a.shape[0], float(gscale), out, ldd, col0, msub, _stream()))


def gemm_kq_grouped(fmt, t16: torch.Tensor, n: int, k: int, E: int, a: torch.Tensor, tb: torch.Tensor, off: torch.Tensor, row_map: torch.Tensor | None = None,
                    gs: torch.Tensor | None = None, out: torch.Tensor | None = None, out_rows: int | None = None, mt: int = 256) -> torch.Tensor:
    """d [rows, n]: sorted rows a fp16 [s, k] of expert segments (off) times the T16 expert stack (E * n rows), decoded inside the GEMM; tile list tb of mt-row
    tiles (moe_plan with the same mt, 128 or 256)."""
    _need_cuda(t16, a, tb, off)
    s = a.shape[0]
    d = out if out is not None else torch.empty((out_rows or s, n), dtype=torch.float16, device=a.device)
    _lib.check(_lib.lib().kyb_gemm_kq_grouped(_fmt(fmt), t16.data_ptr(), n, k, E, a.data_ptr(), a.stride(0), s, tb.data_ptr(), off.data_ptr(), _p(row_map), _p(gs),
                                              d.data_ptr(), d.stride(0), mt, _stream()))
    return d


def gemm_kq_grouped_glu(fmt, t16_gate: torch.Tensor, t16_up: torch.Tensor, n: int, k: int, E: int, a: torch.Tensor, tb: torch.Tensor, off: torch.Tensor,
                        gs_gate: torch.Tensor | None = None, gs_up: torch.Tensor | None = None, limit: float | None = None, mt: int = 256) -> torch.Tensor:
    """h fp16 [s, n] = silu(a W_gate^T) * (a W_up^T) on sorted rows, the gate and up stacks of a routed layer in ONE grouped product with the gated activation in
    its epilogue (both products rounded to fp16 first, as the separate launches would store them)."""
    _need_cuda(t16_gate, t16_up, a, tb, off)
    s = a.shape[0]
    h = torch.empty((s, n), dtype=torch.float16, device=a.device)
    _lib.check(_lib.lib().kyb_gemm_kq_grouped_glu(_fmt(fmt), t16_gate.data_ptr(), t16_up.data_ptr(), n, k, E, a.data_ptr(), a.stride(0), s, tb.data_ptr(), off.data_ptr(),
                                                  _p(gs_gate), _p(gs_up), float(limit or 0.0), h.data_ptr(), h.stride(0), mt, _stream()))
    return h


# ------------------------------------------------------------------------------------------------ NVFP4 tensor-core path
_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def nvfp4_sf_bytes(rows: int, k: int) -> int:
    return _lib.lib().kyb_nvfp4_sf_bytes(rows, k)


def nvfp4_quant_rows(x: torch.Tensor, swizzled: bool = True, plain: bool = True):
    """x fp16 / bf16 [rows, k] -> (codes uint8 [rows, k/2], plain scales uint8 [rows, k/16] or None, chunk-layout scales uint8 or None)."""
    _need_cuda(x)
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("nvfp4_quant_rows takes fp16 / bf16 [rows, k]")
    rows, k = x.shape
    codes = torch.empty((rows, k // 2), dtype=torch.uint8, device=x.device)
    sp = torch.empty((rows, k // 16), dtype=torch.uint8, device=x.device) if plain else None
    ss = torch.empty(nvfp4_sf_bytes(rows, k), dtype=torch.uint8, device=x.device) if swizzled else None
    _lib.check(_lib.lib().kyb_nvfp4_quant_rows(x.data_ptr(), _DT[x.dtype], x.stride(0), rows, k, codes.data_ptr(), _p(sp), _p(ss), _stream()))
    return codes, sp, ss


def nvfp4_unpack_rows(codes: torch.Tensor, scales: torch.Tensor, dtype=torch.float16) -> torch.Tensor:
    _need_cuda(codes, scales)
    rows, k = codes.shape[0], codes.shape[1] * 2
    out = torch.empty((rows, k), dtype=dtype, device=codes.device)
    _lib.check(_lib.lib().kyb_nvfp4_unpack_rows(codes.data_ptr(), scales.data_ptr(), rows, k, _DT[dtype], out.data_ptr(), k, _stream()))
    return out


def nvfp4_sf_swizzle(plain: torch.Tensor, k: int) -> torch.Tensor:
    """plain scale bytes [rows, k/16] -> chunk layout."""
    _need_cuda(plain)
    plain = plain.contiguous()
    rows = plain.shape[0]
    out = torch.empty(nvfp4_sf_bytes(rows, k), dtype=torch.uint8, device=plain.device)
    _lib.check(_lib.lib().kyb_nvfp4_sf_swizzle(plain.data_ptr(), rows, k, out.data_ptr(), 1, _stream()))
    return out


def nvfp4_sf_unswizzle(swz: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    out = torch.empty((rows, k // 16), dtype=torch.uint8, device=swz.device)
    _lib.check(_lib.lib().kyb_nvfp4_sf_swizzle(out.data_ptr(), rows, k, swz.data_ptr(), 0, _stream()))
    return out


def gemm_nvfp4_ag(a_codes, sfa, b_codes, sfb, m: int, n: int, k: int, peer_ptrs, ldd: int, col0: int, gscale: float = 1.0, dtype=torch.float16) -> None:
    """gemm_nvfp4 with the all-gather of an N-sharded linear folded into the epilogue (see gemm_kq_ag)."""
    _need_cuda(a_codes, sfa, b_codes, sfb)
    out = _lib.PeerOut.of(peer_ptrs)
    _lib.check(_lib.lib().kyb_gemm_nvfp4_ag(a_codes.data_ptr(), sfa.data_ptr(), b_codes.data_ptr(), sfb.data_ptr(), m, n, k, float(gscale), _DT[dtype], out, ldd, col0, _stream()))


def gemm_nvfp4(a_codes, sfa, b_codes, sfb, m: int, n: int, k: int, gscale: float = 1.0, dtype=torch.float16, out=None) -> torch.Tensor:
    """d [m, n] = gscale * dequant(A) dequant(B)^T on block-scaled tcgen05 (scales in the chunk layout)."""
    _need_cuda(a_codes, sfa, b_codes, sfb)
    d = out if out is not None else torch.empty((m, n), dtype=dtype, device=a_codes.device)
    _lib.check(_lib.lib().kyb_gemm_nvfp4(a_codes.data_ptr(), sfa.data_ptr(), b_codes.data_ptr(), sfb.data_ptr(), m, n, k, float(gscale), _DT[d.dtype], d.data_ptr(),
                                         d.stride(0), _stream()))
    return d


# ------------------------------------------------------------------------------------------------ attention over a paged cache
_NOGUARD = contextlib.nullcontext()


def _place(*ts):
    """The device guard of a call: all tensors on one CUDA device; that device current during the call."""
    dev = ts[0].device
    for t in ts:
        if not t.is_cuda:
            raise ValueError("kyojin_mac_b200 operators take CUDA tensors (there is no CPU path)")
        if t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}: one device per call")
    return _NOGUARD if _cur_device is not None and dev.index == _cur_device() else torch.cuda.device(dev)


def _i32(t, name, *shape):
    if t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise ValueError(f"{name} must be contiguous int32 [{', '.join('*' if s is None else str(s) for s in shape)}], got {t.dtype} {tuple(t.shape)}")


def _table(t, page):
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] < 1 or t.shape[1] < 1 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"the block table is int32 [batch, columns] with dense rows, got {t.dtype} {tuple(t.shape)}")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("the block table's rows overlap")
    if page not in (16, 32, 64, 128, 256):
        raise ValueError(f"{page} tokens a page: 16, 32, 64, 128 or 256")


def _no_gradient(t, name):
    """There is no backward here: a tensor that takes part in differentiation is refused rather than cut off from it."""
    if (t.requires_grad and torch.is_grad_enabled()) or (_forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None):
        raise ValueError(f"{name} requires a gradient: the paged cache serves inference (use torch.no_grad or detach)")


def _heads(t, name):
    """[tokens, heads, d] of a 16-bit type, heads dense, strides that 16-byte accesses can follow."""
    if t.dtype not in (torch.float16, torch.bfloat16) or t.dim() != 3:
        raise ValueError(f"{name} must be float16 or bfloat16 [tokens, heads, d], got {t.dtype} {tuple(t.shape)}")
    _no_gradient(t, name)
    if t.numel() and (t.stride(2) != 1 or any(s % 8 for s in _steps(t)) or t.data_ptr() % 16):
        raise ValueError(f"{name}: heads must be dense, strides multiples of 8 elements, the start 16-byte aligned; got strides {t.stride()}")


def _steps(t):
    """The two outer strides; that of a dimension of one, which may be anything, as 0."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape[:2], t.stride()))


def _own_rows(t, name):
    """An output [tokens, heads, d] whose heads do not overlap in memory."""
    (n0, s0), (n1, s1) = sorted(((t.shape[0], t.stride(0)), (t.shape[1], t.stride(1))), key=lambda p: p[1])
    if t.numel() and ((n0 > 1 and s0 < t.shape[2]) or (n1 > 1 and s1 < (s0 * n0 if n0 > 1 else t.shape[2]))):
        raise ValueError(f"{name}: heads overlap in memory, strides {t.stride()}")


def _cache(t, name, like=None):
    if t.dtype not in (torch.float16, torch.bfloat16) or t.dim() != 4 or t.shape[2] not in (16, 32, 64, 128, 256) or (like is not None and (t.shape != like.shape or t.dtype != like.dtype)):
        raise ValueError(f"{name} must be float16 or bfloat16 [pages, kv heads, 16 .. 256 (a power of two), d], keys and values alike, got {t.dtype} {tuple(t.shape)}")
    _no_gradient(t, name)
    p, h, n, d = t.shape
    if t.numel() == 0 or t.stride(3) != 1 or t.stride(2) != d or t.data_ptr() % 16 or (p > 1 and (t.stride(0) % 8 or t.stride(0) < n * d)) or (h > 1 and (t.stride(1) % 8 or t.stride(1) < n * d)):
        raise ValueError(f"{name}: the tokens of a page and head must be dense, strides multiples of 8 elements, the start 16-byte aligned; got strides {t.stride()}")


class _Views:
    """Where the tensors of a call lie relative to each other: what a call writes overlaps nothing else of it, or other blocks of the launch would read values that this one has
    written already. views: (name, tensor) of 16-bit tensors that come as addresses later; writes: names of those written; same: a pair that may be one and the same memory."""

    def __init__(self, views, writes, same):
        self.names = [n for n, _ in views]
        self.dims = [sorted(((s, n) for n, s in zip(t.shape, t.stride()) if n > 1), reverse=True) for _, t in views]
        size = [2 * self.extent(d) if t.numel() else 0 for d, (_, t) in zip(self.dims, views)]
        self.pairs = [(i, j, size[i], size[j], {a, b} == set(same) and self.dims[i] == self.dims[j]) for j, b in enumerate(self.names) for i, a in enumerate(self.names[:j])
                      if a in writes or b in writes]
        self.passed = set()                                                  # offsets of the tensors from the first that have passed

    @staticmethod
    def extent(dims):
        return sum(s * (n - 1) for s, n in dims) + 1

    @classmethod
    def disjoint(cls, a, b, offset):
        """Whether views of the dims a, b = [(stride, size), ...] (falling strides, in elements), the second starting `offset` elements behind the first, are certain to share nothing: their
        ranges lie apart, or they have outer strides in common and lie apart within those (q and k of one q | k | v product)."""
        if offset >= cls.extent(a) or -offset >= cls.extent(b):
            return True
        outer = 0
        while a and b and a[0][0] == b[0][0] > 1 and outer % a[0][0] == 0:
            outer, a, b = a[0][0], a[1:], b[1:]
            if offset % outer >= cls.extent(a) and offset % outer + cls.extent(b) <= outer:
                return True
        return False

    def check(self, first, *others):
        offsets = tuple([p - first for p in others])
        if offsets in self.passed:
            return
        ptrs = (0,) + offsets
        for i, j, m, n, same in self.pairs:
            off = ptrs[j] - ptrs[i]
            if -n < off < m and not (same and off == 0) and (off % 2 or not self.disjoint(self.dims[i], self.dims[j], off // 2)):
                raise ValueError(f"{self.names[i]} and {self.names[j]} overlap in memory")
        if len(self.passed) >= 256:
            self.passed.clear()
        self.passed.add(offsets)


# Calls whose shapes, strides, types and numbers have passed the checks (their description; nothing of their data): a decode step repeats its calls for every layer and
# token, and the checks cost more than the launch.
_passed: dict = {}


def _remember(key, value):
    if len(_passed) >= 1024:
        _passed.clear()
    _passed[key] = value
    return value


class PagedStep(NamedTuple):
    """What `paged_step` gives: int32 device tensors."""
    cu_q: torch.Tensor          # [batch + 1] first row of each request
    kv_lens: torch.Tensor       # [batch] tokens to attend over, the new ones included (0: not served)
    positions: torch.Tensor     # [rows] place of each row's token in its request (-1: not served, or a row behind the last request)
    slots: torch.Tensor         # [rows] place in the cache (-1 as above)
    lens: torch.Tensor          # [batch] tokens held after the step
    free_count: torch.Tensor    # [1] free pages left
    refused: torch.Tensor       # [1] requests that could not be served


def paged_step(table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor, page: int, rows: int,
               in_place: bool = False) -> PagedStep:
    """Slots of a step from request lengths, in one launch without a word to the host. Request r holds lens[r] tokens and brings new_lens[r] (packed in request order
    into the step's `rows` rows); the pages it lacks come from the top of free_pages[:free_count] and are entered in its row of `table` [batch, columns].
    A request is served when its pages fit the columns, its tokens the rows, and the needs of the requests up to its own the free list (one that needs no page
    is not held up); `refused` counts the others, whose lengths stay. Needs and rows count in order, served or not: a request that does not fit holds up those behind it that need a
    page, and behind more tokens than rows all are refused, those without tokens too; leave out of a step what cannot be served (new_lens 0).
    in_place: lens and free_count are updated too (a captured step that is replayed)."""
    dev = table.get_device()
    key = (dev, table.shape, table.is_contiguous() or table.stride(), table.dtype, lens.shape, lens.dtype, lens.is_contiguous(), new_lens.shape, new_lens.dtype, new_lens.is_contiguous(),
           free_pages.shape, free_pages.dtype, free_pages.is_contiguous(), free_count.shape, free_count.dtype, page, rows, in_place, lens.get_device(), new_lens.get_device(), free_pages.get_device(),
           free_count.get_device())
    known = _passed.get(key)
    if known is None:
        _place(table, lens, new_lens, free_pages, free_count)
        _table(table, page)
        b, cols = table.shape
        _i32(lens, "lens", b), _i32(new_lens, "new_lens", b), _i32(free_pages, "free_pages", None), _i32(free_count, "free_count", 1)
        if free_pages.numel() < 1 or rows < 0:
            raise ValueError("the free list is an array with room for a page at least, rows not negative")
        sizes = [b + 1, b, rows, rows, 1] + ([] if in_place else [b, 1])
        offs = [4 * sum(sizes[:i]) for i in range(len(sizes))]
        known = _remember(key, (sum(sizes), sizes, offs, _lib.PAGED_STEP_SPLIT[1].pack(free_pages.shape[0], max(table.stride(0), cols), b, cols, page, rows)))
    if dev != torch.cuda.current_device() if _cur_device is None else dev != _cur_device():
        with torch.cuda.device(dev):
            return paged_step(table, lens, new_lens, free_pages, free_count, page, rows, in_place)
    total, sizes, offs, numbers = known
    buf = lens.new_empty(total)                                              # all results side by side
    at, lens_p, count_p = buf.data_ptr(), lens.data_ptr(), free_count.data_ptr()
    cu, kv, pos, slots, refused, *more = buf.split_with_sizes(sizes)
    out_lens, out_count = (lens, free_count) if in_place else more
    out_lens_p, out_count_p = (lens_p, count_p) if in_place else (at + offs[5], at + offs[6])
    rc = _lib.lib().kyb_paged_step(_lib.PAGED_STEP_SPLIT[0].pack(lens_p, new_lens.data_ptr(), free_pages.data_ptr(), count_p, table.data_ptr(), at, at + offs[1], at + offs[2], at + offs[3],
                                                                 out_lens_p, out_count_p, at + offs[4]) + numbers, _stream())
    if rc:
        _lib.check(rc)
    return PagedStep(cu, kv, pos, slots, out_lens, out_count, refused)


def paged_release(table: torch.Tensor, lens: torch.Tensor, which: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor, page: int) -> torch.Tensor:
    """The pages of the requests with which[r] (bool [batch]) go back to the free list, in place: their lengths become 0, their table entries -1. Returns int32 [1]:
    requests whose pages, behind those of the others before them, would overflow the list (they keep them; one without pages is not held up)."""
    guard = _place(table, lens, which, free_pages, free_count)
    _table(table, page)
    b, cols = table.shape
    _i32(lens, "lens", b), _i32(free_pages, "free_pages", None), _i32(free_count, "free_count", 1)
    if which.dtype not in (torch.bool, torch.uint8) or which.shape != (b,) or not which.is_contiguous() or free_pages.numel() < 1:
        raise ValueError(f"which must be bool [{b}], the free list an array with room for a page at least")
    with guard:
        refused = lens.new_empty(1)
        _lib.check(_lib.lib().kyb_paged_release(lens.data_ptr(), which.data_ptr(), table.data_ptr(), max(table.stride(0), cols), b, cols, page, free_pages.data_ptr(), free_pages.numel(),
                                                free_count.data_ptr(), refused.data_ptr(), _stream()))
    return refused


def rope_frequencies(rot: int, base: float = 10000.0, scaling: dict | None = None, device="cuda"):
    """(inv_freq fp32 [rot / 2], mscale) of rotary positions: inv_freq[i] = base^(-2 i / rot), made in 64 bits. scaling, for contexts longer than the one trained on:
    {"type": "linear", "factor"}: all frequencies divided by the factor;
    {"type": "ntk", "factor"}: the base grown to base * factor^(rot / (rot - 2)), so that the slowest pair is divided by the factor and the fastest stays;
    {"type": "llama3", "factor", "low_freq_factor", "high_freq_factor", "original_context"}: pairs of fewer than low_freq_factor turns in the original context divided by
    the factor, of more than high_freq_factor kept, in between mixed linearly in the number of turns;
    {"type": "yarn", "factor", "original_context", "beta_fast" (32), "beta_slow" (1)}: the same with a ramp over the pair's index, and mscale = 0.1 ln(factor) + 1."""
    if rot < 16 or rot % 16:
        raise ValueError(f"rot={rot}: a multiple of 16")
    if not base > 1.0 or not math.isfinite(base):
        raise ValueError("the base is a finite number above 1")
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    inv, mscale = base ** (-i / rot), 1.0
    if scaling is not None:
        def number(name, default=None, zero=False):
            v = scaling.get(name, default)
            if v is None or not 0.0 <= float(v) < math.inf or (float(v) == 0.0 and not zero):
                raise ValueError(f"a scaling of type {kind!r} has a positive {name}, got {v}")
            return float(v)
        kind, f = scaling.get("type"), float(scaling.get("factor", 0.0))
        if not f >= 1.0 or not math.isfinite(f):
            raise ValueError("a scaling has a factor of 1 at least")
        if kind == "linear":
            inv = inv / f
        elif kind == "ntk":
            inv = (base * f ** (rot / (rot - 2))) ** (-i / rot)
        elif kind == "llama3":
            low, high, ctx = number("low_freq_factor", zero=True), number("high_freq_factor"), number("original_context")
            if not high > low:
                raise ValueError("high_freq_factor is above low_freq_factor")
            keep = ((ctx * inv / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
            inv = inv * keep + inv / f * (1 - keep)
        elif kind == "yarn":
            ctx, fast, slow = number("original_context"), number("beta_fast", 32.0), number("beta_slow", 1.0)
            if not fast > slow:
                raise ValueError("a scaling's beta_fast is above its beta_slow")
            index = lambda turns: rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))          # pair that makes so many turns in the context
            a, b = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rot - 1)
            keep = 1.0 - ((torch.arange(rot // 2, dtype=torch.float64) - a) / max(b - a, 0.001)).clamp(0.0, 1.0)
            inv, mscale = inv * keep + inv / f * (1 - keep), 0.1 * math.log(f) + 1.0
        else:
            raise ValueError(f"unknown scaling {kind!r}")
    return inv.to(torch.float32).to(device), mscale


def _rope_check(key, q, k, v, positions, slots, inv_freq, kc, vc, interleaved, mscale, out):
    _place(*(t for t in (q, k, v, positions, slots, inv_freq, kc, vc, out) if t is not None))
    _heads(q, "q"), _i32(positions, "positions", q.shape[0])
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq is contiguous float32 [rot / 2]")
    _no_gradient(inv_freq, "inv_freq")
    T, hq, d = q.shape
    if out is not None:
        _heads(out, "out"), _own_rows(out, "out")
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out has the queries' shape and type")
    ks = vs = kcs = vcs = (0, 0)
    hkv = pages = page = 0
    if k is not None:
        _heads(k, "k"), _heads(v, "v"), _cache(kc, "k_cache"), _cache(vc, "v_cache", kc), _i32(slots, "slots", T)
        if k.shape != (T, kc.shape[1], d) or v.shape != k.shape or kc.shape[3] != d or not q.dtype == k.dtype == v.dtype == kc.dtype:
            raise ValueError(f"q [T, heads, d], k and v [T, kv heads, d] and the cache go together, in one type: got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}, {tuple(kc.shape)}")
        ks, vs, kcs, vcs = _steps(k), _steps(v), _steps(kc), _steps(vc)
        pages, hkv, page = kc.shape[:3]
    os_ = (hq * d, d) if out is None else _steps(out)
    views = [(n, t) for n, t in (("q", q), ("k", k), ("v", v), ("k_cache", kc), ("v_cache", vc), ("out", out)) if t is not None]
    return _remember(key, (_lib.ROPE_APPEND_SPLIT[1].pack(*_steps(q), *ks, *vs, *os_, *kcs, *vcs, T, hq, hkv, d, 2 * inv_freq.shape[0], 1 if interleaved else 0, _DT[q.dtype], pages, page,
                                                          mscale), _Views(views, [n for n, _ in views if n in ("k_cache", "v_cache", "out")], ("q", "out"))))


def _rope_call(q, k, v, positions, slots, inv_freq, kc, vc, interleaved, mscale, out):
    """The queries turned (into `out`), keys and values into the cache where there are any."""
    dev, grad = q.get_device(), q.requires_grad or inv_freq.requires_grad or (out is not None and out.requires_grad) or _forward_ad._current_level >= 0
    if k is None:
        key = (dev, q.shape, q.stride(), q.dtype, positions.shape, positions.dtype, positions.is_contiguous(), inv_freq.shape, inv_freq.dtype, positions.get_device(), inv_freq.get_device(), interleaved,
               mscale)
    else:
        grad = grad or k.requires_grad or v.requires_grad or kc.requires_grad or vc.requires_grad
        key = (dev, q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, positions.shape, positions.dtype, positions.is_contiguous(), slots.shape, slots.dtype,
               slots.is_contiguous(), inv_freq.shape, inv_freq.dtype, kc.shape, kc.is_contiguous() or kc.stride(), kc.dtype, vc.shape, vc.is_contiguous() or vc.stride(), vc.dtype, k.get_device(),
               v.get_device(), positions.get_device(), slots.get_device(), inv_freq.get_device(), kc.get_device(), vc.get_device(), interleaved, mscale)
    if out is not None:
        key += (out.shape, out.stride(), out.dtype, out.get_device())
    known = None if grad or not inv_freq.is_contiguous() else _passed.get(key)
    if known is None:
        known = _rope_check(key, q, k, v, positions, slots, inv_freq, kc, vc, interleaved, mscale, out)
    if dev != torch.cuda.current_device() if _cur_device is None else dev != _cur_device():
        with torch.cuda.device(dev):
            return _rope_call(q, k, v, positions, slots, inv_freq, kc, vc, interleaved, mscale, out)
    numbers, views = known
    given = out is not None
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    qp, pp, ip, op = q.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), out.data_ptr()
    if k is None:
        if given:
            views.check(qp, op)
        ptrs = _lib.ROPE_APPEND_SPLIT[0].pack(qp, 0, 0, pp, 0, ip, op, 0, 0)
    else:
        kp, vp, kcp, vcp = k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr()
        if given:
            views.check(qp, kp, vp, kcp, vcp, op)
        else:
            views.check(qp, kp, vp, kcp, vcp)
        ptrs = _lib.ROPE_APPEND_SPLIT[0].pack(qp, kp, vp, pp, slots.data_ptr(), ip, op, kcp, vcp)
    rc = _lib.lib().kyb_rope_append(ptrs + numbers, _stream())
    if rc:
        _lib.check(rc)
    return out


def rope(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False, mscale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """x fp16 / bf16 [tokens, heads, d] with the first rot = 2 len(inv_freq) values of every head turned: pairs (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved, by
    positions[t] * inv_freq[i], scaled by mscale. Rows of a negative position are left as they are in `out` (x itself, or memory apart from it)."""
    return _rope_call(x, None, None, positions, None, inv_freq, None, None, interleaved, mscale, out)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, inv_freq: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                interleaved: bool = False, mscale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """`rope` of a step's queries, and in the same launch its keys (turned) and values into the cache [pages, kv heads, tokens of a page, d] at slots[t]. q [T, heads, d],
    k and v [T, kv heads, d] may be views of one q | k | v product. Returns the turned queries (in `out`: q itself, or memory apart
    from the other tensors). Rows with a negative position are left alone, a slot outside the cache
    stores nothing. The slots of a step are distinct (paged_step's are): one that two rows share holds values of either."""
    return _rope_call(q, k, v, positions, slots, inv_freq, k_cache, v_cache, interleaved, mscale, out)


def _attention_check(key, q, kc, vc, table, kv_lens, cu_q, max_q, scale, window, sinks, out):
    _place(*(t for t in (q, kc, vc, table, kv_lens, cu_q, out) if t is not None))
    _heads(q, "q"), _cache(kc, "k_cache"), _cache(vc, "v_cache", kc)
    (T, hq, d), (pages, hkv, page, dk) = q.shape, kc.shape
    _table(table, page)
    b, cols = table.shape
    _i32(kv_lens, "kv_lens", b), _i32(cu_q, "cu_q", b + 1)
    if d != dk or d not in (64, 128) or q.dtype != kc.dtype or hq % hkv or hq < hkv:
        raise ValueError(f"heads of 64 or 128, a multiple of the cache's heads, in the cache's type: got q {q.dtype} {tuple(q.shape)}, cache {kc.dtype} {tuple(kc.shape)}")
    if max_q < 0 or window < 0 or sinks < 0 or (sinks and not window):
        raise ValueError("max_q, window and sinks are not negative, sinks come with a window")
    if out is not None:
        _heads(out, "out"), _own_rows(out, "out")
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out has the queries' shape and type")
    with torch.cuda.device(q.device):
        need = _lib.lib().kyb_paged_attention_workspace_bytes(b, T, max_q, cols, page, hq, hkv, d)
    os_ = (hq * d, d) if out is None else _steps(out)
    views = None if out is None else _Views([("q", q), ("k_cache", kc), ("v_cache", vc), ("out", out)], ["out"], ("q", "out"))
    return _remember(key, (need, views, _lib.PAGED_ATTENTION_SPLIT[1].pack(*_steps(q), *_steps(kc), *_steps(vc), *os_, pages, page, max(table.stride(0), cols), cols, b, T, max_q, hq, hkv,
                                                                    d, _DT[q.dtype], window, sinks, need, d ** -0.5 if scale is None else scale)))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor, max_q: int, scale: float | None = None,
                    window: int = 0, sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's new tokens over a paged cache: q fp16 / bf16 [T, heads, d] packed by request (rows [cu_q[r], cu_q[r + 1]); the last one is token
    kv_lens[r] - 1), keys and values through the block table [batch, columns]. Causal; window > 0: the last `window` tokens only, and the first `sinks` ones.
    cu_q does not fall: where it does so far that the requests would own more than T rows, nothing is written and `check_device_status` raises.
    max_q: the largest number of new tokens of a request (chooses the kernel; requests with more are served all the same). scale: d ** -0.5 unless given.
    Keys and values that some row of a request sees are finite; other places of the cache may hold anything. A row that sees nothing (kv_lens 0) gives zeros; rows behind the last request are left as they were (undefined without `out`). `out` is q itself
    or memory apart from q and the cache. Returns out [T, heads, d]."""
    dev = q.get_device()
    key = (dev, q.shape, q.is_contiguous() or q.stride(), q.dtype, k_cache.shape, k_cache.is_contiguous() or k_cache.stride(), k_cache.dtype, v_cache.shape,
           v_cache.is_contiguous() or v_cache.stride(), v_cache.dtype, table.shape, table.is_contiguous() or table.stride(), table.dtype, kv_lens.shape, kv_lens.dtype, kv_lens.is_contiguous(),
           cu_q.shape, cu_q.dtype, cu_q.is_contiguous(), max_q, scale, window, sinks, k_cache.get_device(), v_cache.get_device(), table.get_device(), kv_lens.get_device(), cu_q.get_device(),
           None if out is None else (out.shape, out.stride(), out.dtype, out.get_device()))
    grad = q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or (out is not None and out.requires_grad) or _forward_ad._current_level >= 0
    known = None if grad else _passed.get(key)
    if known is None:
        known = _attention_check(key, q, k_cache, v_cache, table, kv_lens, cu_q, max_q, scale, window, sinks, out)
    if dev != torch.cuda.current_device() if _cur_device is None else dev != _cur_device():
        with torch.cuda.device(dev):
            return paged_attention(q, k_cache, v_cache, table, kv_lens, cu_q, max_q, scale, window, sinks, out)
    need, views, numbers = known
    qp, kp, vp = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        views.check(qp, kp, vp, out.data_ptr())
    # the call's own scratch: captured graphs that replay side by side share nothing, nor do calls of two threads on one stream, whose launches may interleave
    ws = q.new_empty((need + 1) // 2)
    rc = _lib.lib().kyb_paged_attention(_lib.PAGED_ATTENTION_SPLIT[0].pack(qp, kp, vp, table.data_ptr(), kv_lens.data_ptr(), cu_q.data_ptr(),
                                                                           out.data_ptr(), ws.data_ptr()) + numbers, _stream())
    if rc:
        _lib.check(rc)
    return out
