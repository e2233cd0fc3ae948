"""Functional torch wrappers over the C ABI (device tensors in, device tensors out).

Every function enqueues on torch's current stream and returns without
synchronising.  Weight tensors are raw GGUF bytes (``torch.uint8``) or bf16
bits (``torch.uint16``/``torch.bfloat16``/``torch.int16``) already on the GPU.
"""
from __future__ import annotations

import ctypes

import torch

from npu_amd import _lib as L
from npu_amd.gguf_types import QK, GGMLQuantizationType, block_bytes, block_weights


def _as_bf16_bits(w: torch.Tensor) -> torch.Tensor:
    if w.dtype == torch.bfloat16:
        return w.view(torch.int16)
    if w.dtype in (torch.int16, torch.uint16):
        return w
    raise TypeError(f"bf16 weights must be bfloat16/uint16/int16, got {w.dtype}")


def dequant(qtype: int, raw: torch.Tensor, n_superblocks: int | None = None) -> torch.Tensor:
    """Raw blocks (uint8, on GPU) -> fp32 [n_blocks * block weights] (256, or 32 for Q8_0)."""
    bb = block_bytes(qtype)
    if raw.dtype != torch.uint8:
        raise TypeError(f"raw must be uint8, got {raw.dtype}")
    if n_superblocks is None:
        if raw.numel() % bb:
            raise ValueError(f"{raw.numel()} bytes is not a whole number of {bb}-byte superblocks")
        n_superblocks = raw.numel() // bb
    out = torch.empty(n_superblocks * block_weights(qtype), dtype=torch.float32, device=raw.device)
    L.check(L.lib().gm_dequant_f32(int(qtype), L.ptr(raw), n_superblocks, L.ptr(out), L.stream_ptr()),
            "gm_dequant_f32")
    return out


def transcode_i8(qtype: int, raw: torch.Tensor) -> torch.Tensor:
    """Raw Q8_0 / Q4_K / Q5_K / Q6_K blocks (uint8, on GPU) -> I8 sub-blocks (uint8, 48 bytes
    per 32 weights, in weight order; ``gm_transcode_i8``)."""
    bb, bw = block_bytes(qtype), block_weights(qtype)
    if raw.dtype != torch.uint8:
        raise TypeError(f"raw must be uint8, got {raw.dtype}")
    if raw.numel() % bb:
        raise ValueError(f"{raw.numel()} bytes is not a whole number of {bb}-byte blocks")
    n = raw.numel() // bb
    out = torch.empty(n * bw // 32 * 48, dtype=torch.uint8, device=raw.device)
    L.check(L.lib().gm_transcode_i8(int(qtype), L.ptr(raw.contiguous()), n, L.ptr(out), L.stream_ptr()),
            "gm_transcode_i8")
    return out


def matvec(qtype: int, w: torch.Tensor, M: int, K: int, x: torch.Tensor) -> torch.Tensor:
    """y[..., M] = W[M, K] @ x[..., K] with W raw (IQ4_XS/IQ3_XXS) or bf16."""
    if qtype == GGMLQuantizationType.BF16:
        w = _as_bf16_bits(w)
    elif w.dtype != torch.uint8:
        raise TypeError(f"quantized weights must be uint8, got {w.dtype}")
    if x.shape[-1] != K:
        raise ValueError(f"x last dim {x.shape[-1]} != K={K}")
    xf = x.reshape(-1, K).to(torch.float32).contiguous()
    n_tok = xf.shape[0]
    y = torch.empty((n_tok, M), dtype=torch.float32, device=xf.device)
    L.check(L.lib().gm_matvec(int(qtype), L.ptr(w), M, K, L.ptr(xf), n_tok, L.ptr(y), L.stream_ptr()),
            "gm_matvec")
    return y.reshape(*x.shape[:-1], M)


def swiglu_mlp(q_gu: int, w_gate: torch.Tensor, w_up: torch.Tensor, q_down: int, w_down: torch.Tensor,
               D: int, FF: int, x: torch.Tensor) -> torch.Tensor:
    """down(silu(gate x) * up x) for x[..., D]."""
    if q_gu == GGMLQuantizationType.BF16:
        w_gate, w_up = _as_bf16_bits(w_gate), _as_bf16_bits(w_up)
    if q_down == GGMLQuantizationType.BF16:
        w_down = _as_bf16_bits(w_down)
    xf = x.reshape(-1, D).to(torch.float32).contiguous()
    n_tok = xf.shape[0]
    h = torch.empty((n_tok, FF), dtype=torch.float32, device=xf.device)
    y = torch.empty((n_tok, D), dtype=torch.float32, device=xf.device)
    L.check(L.lib().gm_swiglu_mlp(int(q_gu), L.ptr(w_gate), L.ptr(w_up), int(q_down), L.ptr(w_down), D, FF,
                                  L.ptr(xf), n_tok, L.ptr(h), L.ptr(y), L.stream_ptr()), "gm_swiglu_mlp")
    return y.reshape(*x.shape[:-1], D)


def router_topk(w_router: torch.Tensor, x: torch.Tensor, k: int, *, bias: torch.Tensor | None = None,
                w_sh_gate: torch.Tensor | None = None, norm_w: torch.Tensor | None = None,
                eps: float = 1e-6):
    """Router logits, top-k ids (int32), renormalised weights and sigmoid shared gate.

    Returns ``(ids [T,k], weights [T,k], logits [T,E], sh_gate [T] or None)``.
    """
    w = _as_bf16_bits(w_router)
    E, D = w.shape
    xf = x.reshape(-1, D).to(torch.float32).contiguous()
    T = xf.shape[0]
    dev = xf.device
    ids = torch.empty((T, k), dtype=torch.int32, device=dev)
    wts = torch.empty((T, k), dtype=torch.float32, device=dev)
    logits = torch.empty((T, E), dtype=torch.float32, device=dev)
    shg = torch.empty((T,), dtype=torch.float32, device=dev) if w_sh_gate is not None else None
    wsh = _as_bf16_bits(w_sh_gate).contiguous() if w_sh_gate is not None else None
    b = bias.to(torch.float32).contiguous() if bias is not None else None
    nw = norm_w.to(torch.float32).contiguous() if norm_w is not None else None
    L.check(L.lib().gm_router_topk(L.ptr(w.contiguous()), L.ptr(b), L.ptr(xf), T, D, E, k, L.ptr(wsh), L.ptr(nw),
                                   float(eps), L.ptr(ids), L.ptr(wts), L.ptr(logits), L.ptr(shg), L.stream_ptr()),
            "gm_router_topk")
    return ids, wts, logits, shg


def moe_dispatch(ids: torch.Tensor, E: int):
    """Expert-sorted dispatch of top-k ids [T, k]: (counts[E], offsets[E+1], sorted_pairs[T*k])."""
    ids32 = ids.to(torch.int32).contiguous()
    T, k = ids32.shape
    dev = ids32.device
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    pairs = torch.empty(T * k, dtype=torch.int32, device=dev)
    L.check(L.lib().gm_moe_dispatch(L.ptr(ids32), T, k, E, L.ptr(counts), L.ptr(offsets), L.ptr(pairs),
                                    L.stream_ptr()), "gm_moe_dispatch")
    return counts, offsets, pairs


def moe_workspace_bytes(layer: L.GmMoeLayer, T: int) -> int:
    n = L.lib().gm_moe_workspace_bytes(ctypes.byref(layer), T)
    if n == 0:
        raise ValueError(f"gm_moe_workspace_bytes: {L.last_error()}")
    return int(n)


def moe_workspace_offsets(layer: L.GmMoeLayer, T: int) -> dict[str, int]:
    o = [ctypes.c_size_t() for _ in range(4)]
    L.check(L.lib().gm_moe_workspace_offsets(ctypes.byref(layer), T, *[ctypes.byref(v) for v in o]),
            "gm_moe_workspace_offsets")
    return dict(zip(("logits", "ids", "weights", "sh_gate"), (v.value for v in o)))


def moe_forward_raw(layer: L.GmMoeLayer, x: torch.Tensor, y: torch.Tensor, ws: torch.Tensor,
                    residual: bool = False, stage: int = 0, path: str = "auto") -> None:
    """Enqueue the fused MoE block (stage 0) or one of its stages 1..3: y = moe(rmsnorm(x)) (+ x).

    path: "auto" (decode kernels for T <= 8, prefill GEMMs above), "decode" or "prefill"."""
    T = x.shape[0]
    flags = L.GM_MOE_RESIDUAL if residual else 0
    if stage == 0:
        fn = {"auto": "gm_moe_forward", "decode": "gm_moe_decode", "prefill": "gm_moe_prefill"}[path]
        rc = getattr(L.lib(), fn)(ctypes.byref(layer), L.ptr(x), L.ptr(y), T, flags, L.ptr(ws), ws.numel(),
                                  L.stream_ptr())
    else:
        rc = L.lib().gm_moe_forward_stage(ctypes.byref(layer), L.ptr(x), L.ptr(y), T, flags, L.ptr(ws),
                                          ws.numel(), stage, L.stream_ptr())
    L.check(rc, "gm_moe_forward")


def moe_chain_raw(layers, x: torch.Tensor, y: torch.Tensor, buf: torch.Tensor | None, workspaces,
                  residual: bool = False) -> None:
    """Enqueue gm_moe_chain over ``layers`` (GmMoeLayer structs) with one workspace per layer:
    x_{l+1} = moe_l(rmsnorm_l(x_l)) (+ x_l); the last layer writes y, the others alternate
    between y and buf."""
    n = len(layers)
    if n < 1 or len(workspaces) != n:
        raise ValueError("moe_chain_raw: one workspace per layer")
    arr = (L.GmMoeLayer * n)(*layers)
    wsp = (ctypes.c_void_p * n)(*[L.ptr(w) for w in workspaces])
    wsb = (ctypes.c_size_t * n)(*[w.numel() for w in workspaces])
    flags = L.GM_MOE_RESIDUAL if residual else 0
    rc = L.lib().gm_moe_chain(arr, n, L.ptr(x), L.ptr(y), L.ptr(buf) if buf is not None else None, x.shape[0],
                              flags, wsp, wsb, L.stream_ptr())
    L.check(rc, "gm_moe_chain")



def moe_chain_mode(layers, T: int) -> int:
    """gm_moe_chain's path for ``layers`` at ``T`` tokens: 1 = the accumulator-linked T = 1
    kernels (one router launch, then two launches per layer), 2 = the combine-linked T > 1
    kernels (one router launch, then four launches per layer; needs distinct workspaces per
    layer), 0 = one gm_moe_forward per layer."""
    n = len(layers)
    arr = (L.GmMoeLayer * n)(*layers)
    rc = L.lib().gm_moe_chain_fused(arr, n, T)
    if rc < 0:
        L.check(rc, "gm_moe_chain_fused")
    return int(rc)


def moe_chain_fused(layers, T: int) -> bool:
    """Whether gm_moe_chain links consecutive layers at ``T`` tokens (mode 1 or 2 above)
    rather than running one gm_moe_forward per layer."""
    return moe_chain_mode(layers, T) > 0


# ------------------------------------------------------------ serving a batch
_T16 = {torch.float16: L.GM_QTYPE_F16, torch.bfloat16: L.GM_QTYPE_BF16}
_ELEM = {torch.float32: L.GM_QTYPE_F32, **_T16}


def _elem(t: torch.Tensor, name: str, among=_ELEM) -> int:
    qtype = among.get(t.dtype)
    if qtype is None:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in among)}, got {t.dtype}")
    return qtype


def _rows(t: torch.Tensor, name: str, shape) -> tuple[int, int]:
    """The strides of t's tokens and heads; t must have the given shape [T, heads, head_dim]
    (or be pages) and contiguous rows of head_dim."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    st = t.stride()
    if st[-1] != 1:
        raise ValueError(f"{name}: the last dim must be contiguous")
    return st[:2]


def _ints(t: torch.Tensor, name: str, shape) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor):
    """(type, n_pages, page_size, n_head_kv, head_dim) of a cache."""
    ct = _elem(k_pages, "k_pages", _T16)
    if k_pages.dim() != 4:
        raise ValueError(f"k_pages must be [n_pages, page_size, n_head_kv, head_dim], got {list(k_pages.shape)}")
    if v_pages.dtype != k_pages.dtype or v_pages.shape != k_pages.shape:
        raise ValueError("v_pages must have k_pages' shape and type")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("k_pages and v_pages must be contiguous")
    return (ct, *k_pages.shape)


def _out(out: torch.Tensor | None, shape, dtype: torch.dtype, like: torch.Tensor, *inputs) -> torch.Tensor:
    """``out``, or a new tensor; one that is given must not overlap ``like`` or ``inputs``, which
    blocks read while others write."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    if out.shape != shape or out.dtype != dtype or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {list(shape)} {dtype}, got {list(out.shape)} {out.dtype}")
    lo, hi = _span(out)
    for t in (like, *inputs):
        if t is not None:
            a, b = _span(t)
            if a < hi and lo < b:
                raise ValueError("out overlaps an input")
    return out


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The addresses between t's first byte and its last."""
    if t.numel() == 0:
        return 0, 0
    p = t.data_ptr()
    return p, p + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _one_device(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    dev = first.get_device()
    if dev < 0:
        raise ValueError("tensors must be on the GPU")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
    return dev


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


# the number alone: rope_append of 8 tokens takes 12.6 us of host time, 14.2 with the stream as an object
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _enqueue(dev: int, name: str, args, ws_bytes=None) -> None:
    """Call the entry point ``name`` on the current stream of device ``dev``; with ``ws_bytes``
    (the name of its size query) it gets a workspace of its own."""
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _enqueue(dev, name, args, ws_bytes)
    lib = L.lib()
    stream = _stream_of(dev)
    if ws_bytes is None:
        rc = getattr(lib, name)(args, stream)
    else:
        n = getattr(lib, ws_bytes)(args)
        if n == 0:
            L.check(L.GM_EINVAL, name)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        rc = getattr(lib, name)(args, ws.data_ptr(), n, stream)
    L.check(rc, name)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor, *,
                axis: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
                k_norm: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The step between the projections and the attention of many sequences' new tokens:
    rotated (and, with ``q_norm`` / ``k_norm`` [head_dim] fp32, RMS-normed) q is returned, k
    and v go to the cache (``gm_rope_append``).

    q [T, n_head, head_dim], k and v [T, n_head_kv, head_dim] (one type; views into a
    projection's rows are fine); positions int32 [T] or [n_axes, T]; inv_freq fp64
    [rope_dim / 2], radians per position, and axis int32 [rope_dim / 2], the axis that turns
    each pair (``qwen_serve.build_rope_axes``); k_pages / v_pages [n_pages, page_size,
    n_head_kv, head_dim] bf16 or fp16; slots int32 [T], the cache row of each token (page
    times page_size plus row), negative for none, no row twice.  The result has the cache's
    type, or ``out_dtype``.  A packed buffer [T, n_head_kv, head_dim] viewed as one page,
    with slots 0 .. T - 1, serves where no cache is wanted."""
    in_type = _elem(q, "q")
    ct, n_pages, page, hkv, dh = _pages(k_pages, v_pages)
    if q.dim() != 3:
        raise ValueError(f"q must be [T, n_head, head_dim], got {list(q.shape)}")
    T, hq, _ = q.shape
    strides = *_rows(q, "q", (T, hq, dh)), *_rows(k, "k", (T, hkv, dh)), *_rows(v, "v", (T, hkv, dh))
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must have one type")
    n_axes = positions.shape[0] if positions.dim() == 2 else 1
    _ints(positions, "positions", (n_axes, T) if positions.dim() == 2 else (T,))
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise TypeError("inv_freq must be contiguous float64 [rope_dim / 2]")
    half = inv_freq.shape[0]
    _ints(slots, "slots", (T,))
    if axis is not None:
        _ints(axis, "axis", (half,))
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (w.dtype != torch.float32 or w.shape != (dh,) or not w.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 [{dh}]")
    if not (positions.is_contiguous() and slots.is_contiguous() and (axis is None or axis.is_contiguous())):
        raise ValueError("positions, slots and axis must be contiguous")
    dev = _one_device(q, k, v, positions, inv_freq, k_pages, v_pages, slots, axis, q_norm, k_norm, out)
    out = _out(out, (T, hq, dh), out_dtype or (k_pages.dtype if out is None else out.dtype), q, k, v, k_pages, v_pages,
               positions, slots)
    a = L.filled(L.GmRopeAppendArgs, q.data_ptr(), k.data_ptr(), v.data_ptr(), positions.data_ptr(),
                 inv_freq.data_ptr(), _ptr(axis), _ptr(q_norm), _ptr(k_norm), out.data_ptr(), k_pages.data_ptr(),
                 v_pages.data_ptr(), slots.data_ptr(), *strides, n_pages * page, eps, T, n_axes, hq, hkv, dh, 2 * half,
                 in_type, _elem(out, "out"), ct)
    _enqueue(dev, "gm_rope_append", a)
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: float | None = None, gate: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over a paged cache (``gm_paged_attention``):
    q [n_seq, n_head, head_dim] in fp32 or the cache's type, block_table int32 [n_seq, width]
    (page numbers in order; entries past a sequence's last page are not read), lengths int32
    [n_seq] with the new token counted.  ``scale`` (positive) defaults to head_dim ** -0.5; ``gate`` of
    q's shape multiplies the result by its sigmoid.  Sequences of length 0 give zeros.
    Lengths and tables are read on the device only, so the call may be captured and replayed
    with other ones."""
    qt = _elem(q, "q")
    ct, n_pages, page, hkv, dh = _pages(k_pages, v_pages)
    if q.dim() != 3:
        raise ValueError(f"q must be [n_seq, n_head, head_dim], got {list(q.shape)}")
    B, hq, _ = q.shape
    qs = _rows(q, "q", (B, hq, dh))
    _ints(lengths, "lengths", (B,))
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [n_seq, width], got {list(block_table.shape)}")
    width = block_table.shape[1]
    _ints(block_table, "block_table", (B, width))
    if (width > 1 and block_table.stride(1) != 1) or not lengths.is_contiguous():
        raise ValueError("lengths and the rows of block_table must be contiguous")
    gt, gs = 0, (0, 0)
    if gate is not None:
        gt = _elem(gate, "gate")
        gs = _rows(gate, "gate", (B, hq, dh))
    dev = _one_device(q, k_pages, v_pages, block_table, lengths, gate, out)
    out = _out(out, (B, hq, dh), q.dtype, q, k_pages, v_pages, block_table, lengths, gate)
    if B == 0:
        return out
    a = L.filled(L.GmPagedAttnArgs, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
                 lengths.data_ptr(), _ptr(gate), out.data_ptr(), *qs, *gs, block_table.stride(0) if B > 1 else width,
                 dh ** -0.5 if scale is None else scale, B, hq, hkv, dh, n_pages, page, width, qt, ct, gt)
    _enqueue(dev, "gm_paged_attention", a, "gm_paged_attention_workspace_bytes")
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, *,
                     cu_k: torch.Tensor | None = None, block_table: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None, scale: float | None = None,
                     gate: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over packed prompts (``gm_prompt_attention``): q [n_q, n_head,
    head_dim] bf16 or fp16, sequence b in rows cu_q[b] .. cu_q[b + 1] - 1 (int32 [n_seq + 1]).
    Keys and values are k, v [n_k, n_head_kv, head_dim] packed by cu_k (cu_q where it is
    None), or, with block_table [n_seq, width] and lengths [n_seq] (both int32), the first
    lengths[b] positions of cache pages k, v [n_pages, page_size, n_head_kv, head_dim].  A
    sequence's last query row sees all its keys, so a prompt may follow cached ones.  Rows
    that see no key give zeros; rows of ``out`` outside the sequences are left as they were."""
    paged = block_table is not None
    if paged != (lengths is not None) or (paged and cu_k is not None):
        raise ValueError("keys are packed (cu_k) or in pages (block_table and lengths)")
    qt = _elem(q, "q", _T16)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must have one type")
    if q.dim() != 3 or k.dim() != (4 if paged else 3):
        raise ValueError("q must be [n_q, n_head, head_dim], k and v [n_k, n_head_kv, head_dim] or pages")
    n_q, hq, dh = q.shape
    n_seq = cu_q.shape[0] - 1
    if cu_q.dim() != 1 or n_seq < 0:
        raise ValueError("cu_q must be [n_seq + 1]")
    _ints(cu_q, "cu_q", (n_seq + 1,))
    qs = _rows(q, "q", (n_q, hq, dh))
    n_k = n_pages = page = width = ts = 0
    if paged:
        _, n_pages, page, hkv, _ = _pages(k, v)
        if block_table.dim() != 2 or block_table.shape[0] != n_seq:
            raise ValueError(f"block_table must be [{n_seq}, width], got {list(block_table.shape)}")
        width = block_table.shape[1]
        _ints(block_table, "block_table", (n_seq, width))
        _ints(lengths, "lengths", (n_seq,))
        if (width > 1 and block_table.stride(1) != 1) or not lengths.is_contiguous():
            raise ValueError("lengths and the rows of block_table must be contiguous")
        ts = block_table.stride(0) if n_seq > 1 else width
    else:
        n_k, hkv, _ = k.shape
        cu_k = cu_q if cu_k is None else _ints(cu_k, "cu_k", (n_seq + 1,))
    if k.shape[-1] != dh:
        raise ValueError(f"k has head_dim {k.shape[-1]}, q {dh}")
    ks, vs = _rows(k, "k", k.shape), _rows(v, "v", k.shape)
    if paged:
        ks = vs = (0, 0)
    if not cu_q.is_contiguous() or (cu_k is not None and not cu_k.is_contiguous()):
        raise ValueError("cu_q and cu_k must be contiguous")
    gt, gs = 0, (0, 0)
    if gate is not None:
        gt = _elem(gate, "gate")
        gs = _rows(gate, "gate", (n_q, hq, dh))
    dev = _one_device(q, k, v, cu_q, cu_k, block_table, lengths, gate, out)
    out = _out(out, (n_q, hq, dh), q.dtype, q, k, v, cu_q, cu_k, block_table, lengths, gate)
    a = L.filled(L.GmPromptAttnArgs, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), _ptr(cu_k),
                 _ptr(block_table), _ptr(lengths), _ptr(gate), out.data_ptr(), *qs, *ks, *vs, *gs, ts,
                 dh ** -0.5 if scale is None else scale, n_q, n_k, n_seq, hq, hkv, dh, n_pages, page, width, qt, gt)
    _enqueue(dev, "gm_prompt_attention", a)
    return out


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
           top_k: int | torch.Tensor | None = None, top_p: float | torch.Tensor | None = None,
           min_p: float | torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of logits [n_row, vocab] (fp32, bf16 or fp16; rows may be strided)
    at the given uniform numbers u fp32 [n_row] in [0, 1): int64 [n_row] (``gm_sample``).

    Filters in this order: the top_k largest (0: all), the shortest run of the largest whose
    weight reaches top_p of theirs, the ones of at least min_p times the largest weight; the
    pick is the inverse of the running sum of what is left, in the vocabulary's order.  Each
    parameter is one value or a tensor of one per row (fp32; top_k int32).  temperature 0 is
    the argmax, lowest index first.  A row without a logit above -inf gives -1."""
    lt = _elem(logits, "logits")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [n_row, vocab], got {list(logits.shape)}")
    B, V = logits.shape
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("logits: the last dim must be contiguous")
    if u.dtype != torch.float32 or u.shape != (B,) or not u.is_contiguous():
        raise ValueError(f"u must be contiguous float32 [{B}]")
    held, alone = [], []
    for name, val, dt, none in (("temperature", temperature, torch.float32, 1.0), ("top_k", top_k, torch.int32, 0),
                                ("top_p", top_p, torch.float32, 1.0), ("min_p", min_p, torch.float32, 0.0)):
        if isinstance(val, torch.Tensor):
            if val.dtype != dt or val.shape != (B,) or not val.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dt} [{B}] or one value")
            held.append(val)
            alone.append(none)
        else:
            held.append(None)
            alone.append(none if val is None else val)
    dev = _one_device(logits, u, *held, out)
    out = _out(out, (B,), torch.int64, logits, u, *held)
    if B == 0:
        return out
    a = L.filled(L.GmSampleArgs, logits.data_ptr(), u.data_ptr(), *(_ptr(t) for t in held), out.data_ptr(),
                 logits.stride(0) if B > 1 else V, *alone, B, V, lt)
    _enqueue(dev, "gm_sample", a, "gm_sample_workspace_bytes")
    return out
