"""The serving operators of npu_amd.ops (rope_append, paged_attention, prompt_attention,
sample) against plain 64-bit implementations.

Tolerances.  A result rounded to a type is off by at most eps / 2 of it (H below; in fp16 at
least 2^-25, half the step of its smallest values).  Before
that: rotation in fp32 with an angle good to 2^-24 turns and sums of two products, 2e-6 of the
row's largest value; fp32 scores of at most 256 products in chains of at most 24 MFMAs, off by
26 x 2^-24 of sum |q k| scale (at most 16 here), and twice that of the largest |v| in an
output, 5e-5 of it; probabilities rounded to 16 bits, H of sum p |v|.  Sampled tokens are equal.
"""
import math

import pytest
import torch

from npu_amd import ops

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
H = {BF: 2.0 ** -8, HF: 2.0 ** -11, F32: 2.0 ** -24}      # half a step, relative to the value


def _g(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# ------------------------------------------------------------ rope_append
def _rope_ref(x, w, pos, inv, axis, eps):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    half = inv.shape[0]
    p = pos if pos.dim() == 2 else pos[None]
    a = p[axis.long()].t().double() * inv if axis is not None else p[0].double()[:, None] * inv
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi = x[..., :half], x[..., half:2 * half]
    return torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., 2 * half:]], -1)


def _close(got, want, tol):
    if got.dtype == HF:
        tol = tol + 2.0 ** -25                                # below 2^-14 the steps of fp16 are 2^-24
    d = (got.double() - want).abs()
    far = float((d / tol.clamp(min=1e-300)).nan_to_num(math.inf).max())
    assert far <= 1, f"off by {far:.3g} times the tolerance"


@pytest.mark.parametrize("T,hq,hkv,dh,rd,axes,dtype,ct,norm,layout", [
    (1, 16, 2, 256, 64, 3, F32, BF, True, "row"),
    (7, 16, 2, 256, 64, 1, BF, BF, False, "row"),
    (600, 4, 2, 128, 128, 3, HF, HF, True, "plain"),
    (33, 7, 1, 64, 6, 1, F32, HF, True, "odd"),
    (5, 3, 3, 64, 0, 1, BF, BF, True, "plain"),
    (130, 12, 4, 64, 64, 1, BF, HF, False, "odd"),
    (513, 24, 4, 128, 50, 3, HF, BF, True, "row"),
    (65, 1, 1, 256, 256, 1, F32, BF, False, "plain"),
])
def test_rope_append(gpu, T, hq, hkv, dh, rd, axes, dtype, ct, norm, layout):
    print(f"rope T={T} heads={hq},{hkv},{dh} rd={rd} axes={axes} {dtype} {ct} {layout}", flush=True)
    g = _g(T + rd)
    if layout == "row":                     # as a projection leaves them: [q | gate] per head, k, v
        row = _randn(g, T, (2 * hq + 2 * hkv) * dh, dtype=dtype)
        q = row[:, :2 * hq * dh].view(T, hq, 2 * dh)[..., :dh]
        k = row[:, 2 * hq * dh:(2 * hq + hkv) * dh].view(T, hkv, dh)
        v = row[:, (2 * hq + hkv) * dh:].view(T, hkv, dh)
    else:
        pad = 1 if layout == "odd" else 0   # rows that start at odd elements
        q, k, v = (_randn(g, T, n, dh + pad, dtype=dtype)[..., pad:] for n in (hq, hkv, hkv))
    pos = torch.randint(0, 2_000_000, (axes, T), generator=g, device="cuda", dtype=torch.int32)
    pos[0, 0] = 2 ** 31 - 1
    pos[-1, -1] = -12345
    if axes == 1 and T % 2:
        pos = pos[0].contiguous()
    inv = 1e7 ** (-torch.arange(rd // 2, dtype=torch.float64, device="cuda") / max(1, rd // 2))
    axis = torch.randint(0, axes, (rd // 2,), generator=g, device="cuda", dtype=torch.int32) if axes > 1 else None
    qn, kn = (1 + _randn(g, dh, scale=0.1), 1 + _randn(g, dh, scale=0.1)) if norm else (None, None)
    page = 16
    n = -(-T // page) + 2
    kp, vp = (_randn(g, n, page, hkv, dh, dtype=ct) for _ in range(2))
    slots = torch.randperm(n * page, generator=g, device="cuda")[:T].to(torch.int32)
    slots[T // 3] = -1
    if T > 4:
        slots[T // 2] = n * page            # a row behind the cache
    kw, vw = kp.double(), vp.double()
    q2 = ops.rope_append(q, k, v, pos, inv, kp, vp, slots, axis=axis, q_norm=qn, k_norm=kn, eps=1e-6)
    assert q2.dtype == ct and q2.shape == (T, hq, dh)
    want = _rope_ref(q, qn, pos, inv, axis, 1e-6)
    _close(q2, want, H[ct] * want.abs() + 2e-6 * want.abs().amax(-1, keepdim=True))
    live = (slots >= 0) & (slots < n * page)
    at = slots[live].long()
    kw.view(-1, hkv, dh)[at] = _rope_ref(k, kn, pos, inv, axis, 1e-6)[live]
    vw.view(-1, hkv, dh)[at] = v.double()[live]
    _close(kp, kw, H[ct] * kw.abs() + 2e-6 * kw.abs().amax(-1, keepdim=True))
    _close(vp, vw, H[ct] * vw.abs())
    q3 = ops.rope_append(q, k, v, pos, inv, kp, vp, slots, axis=axis, q_norm=qn, k_norm=kn, out_dtype=F32)
    _close(q3, want, 2.0 ** -24 * want.abs() + 2e-6 * want.abs().amax(-1, keepdim=True))


def test_rope_append_far_position_matches_the_near_one(gpu):
    """A whole number of turns changes nothing: positions 2^30 apart with inv_freq 2 pi / 2^10."""
    g = _g(3)
    q, k, v = (_randn(g, 4, n, 64) for n in (2, 1, 1))
    inv = torch.full((32,), 2 * math.pi / 1024, dtype=torch.float64, device="cuda")
    kp, vp = torch.zeros(2, 1, 4, 1, 64, dtype=BF, device="cuda")
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    near = torch.tensor([1, 5, 700, 1023], dtype=torch.int32, device="cuda")
    a = ops.rope_append(q, k, v, near, inv, kp, vp, slots, out_dtype=F32)
    b = ops.rope_append(q, k, v, near + 2 ** 30, inv, kp, vp, slots, out_dtype=F32)
    assert float((a - b).abs().max()) <= 2e-6 * float(a.abs().max())


# ------------------------------------------------------------ attention
def _attend_ref(q, k, v, scale, last, seen=None):
    """q [n, Hq, D], k / v [m, Hkv, D], row i sees keys 0 .. last[i] (and those in seen [m]):
    (softmax(q k) v, softmax(q k) |v|) in 64 bits, zeros where a row sees none."""
    n, hq, d = q.shape
    m, hkv, _ = k.shape
    q = q.double().view(n, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
    k, v = (t.double().permute(1, 0, 2).contiguous() for t in (k, v))
    x = torch.bmm(q, k.transpose(1, 2).contiguous()).view(hkv, hq // hkv, n, m) * scale
    live = torch.arange(m, device=q.device) <= last[:, None]
    if seen is not None:
        live = live & seen
    x = x.masked_fill(~live, -math.inf)
    p = torch.softmax(x, -1).masked_fill(~live.any(-1)[:, None], 0.0).view(hkv, -1, m)
    v = torch.where(live.any(0)[None, :, None], v, 0.0)        # what no row sees counts for nothing
    o, a = torch.bmm(p, v), torch.bmm(p, v.abs())
    return tuple(t.view(hkv, hq // hkv, n, d).permute(2, 0, 1, 3).reshape(n, hq, d) for t in (o, a))


def _tol(want, absv, v, dtype, rounded):
    return H[dtype] * want.abs() + (H[rounded] * absv if rounded != F32 else 0) + 5e-5 * v.double().abs().max()


def _paged(g, lengths, page, hkv, dh, ct, spare=2, poison=True):
    """(k, v, table): pages in any order; whatever no sequence reads is NaN."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    k, v = (_randn(g, total, page, hkv, dh, dtype=ct) for _ in range(2))
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(need) + 1
    table = torch.full((len(lengths), width), -7, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        if poison and n and lengths[b] % page:
            k[order[at - 1], lengths[b] % page:] = float("nan")
            v[order[at - 1], lengths[b] % page:] = float("inf")
    if poison:
        k[order[at:].long()] = float("nan")
        v[order[at:].long()] = float("nan")
    return k, v, table


def _keys(k, table, b, n, page):
    pages = table[b, :-(-n // page)].long()
    return k[pages].reshape(-1, *k.shape[2:])[:n]


def _check_decode(out, q, k, v, table, lengths, page, scale, gate, dtype, ct):
    for b, n in enumerate(lengths):
        if n == 0:
            assert bool((out[b] == 0).all())
            continue
        kk, vv = _keys(k, table, b, n, page), _keys(v, table, b, n, page)
        want, absv = _attend_ref(q[b:b + 1], kk, vv, scale, torch.tensor([n - 1], device="cuda"))
        if gate is not None:
            f = torch.sigmoid(gate[b:b + 1].double())
            want, absv = want * f, absv * f
        _close(out[b:b + 1], want, _tol(want, absv, vv, dtype, F32 if dtype == F32 else ct))


TYPES = [(BF, BF), (HF, HF), (F32, BF), (F32, HF)]


@pytest.mark.parametrize("dtype,ct", TYPES)
@pytest.mark.parametrize("hq,hkv,dh,page,lengths,gate", [
    (16, 2, 256, 64, [1], True),
    (16, 2, 256, 16, [0, 31, 32, 33, 0, 257, 1], False),
    (8, 8, 64, 7, [5, 200, 64, 1000], True),
    (24, 4, 128, 1, [40, 0, 3], False),
    (40, 2, 128, 128, [129, 700], True),
    (7, 1, 256, 48, [4099], False),
    (6, 2, 64, 32, [0, 0], False),
])
def test_paged_attention(gpu, dtype, ct, hq, hkv, dh, page, lengths, gate):
    print(f"decode heads={hq},{hkv},{dh} page={page} lengths={lengths} {dtype} {ct}", flush=True)
    g = _g(sum(lengths) + dh)
    k, v, table = _paged(g, lengths, page, hkv, dh, ct)
    row = _randn(g, len(lengths), hq, 2 * dh, dtype=dtype)
    q, gt = row[..., :dh], (row[..., dh:] if gate else None)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = ops.paged_attention(q, k, v, table, n, gate=gt)
    assert out.dtype == dtype
    _check_decode(out, q, k, v, table, lengths, page, dh ** -0.5, gt, dtype, ct)


@pytest.mark.parametrize("dtype,ct", TYPES)
def test_paged_attention_many_sequences(gpu, dtype, ct):
    """More sequences than blocks, most of them short, some empty, one long."""
    g = _g(5)
    lengths = torch.randint(0, 70, (300,), generator=g, device="cuda").tolist()
    lengths[17] = 5000
    lengths[299] = 0
    k, v, table = _paged(g, lengths, 16, 2, 128, ct)
    q = _randn(g, 300, 8, 128, dtype=dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = ops.paged_attention(q, k, v, table, n, scale=0.2)
    _check_decode(out, q, k, v, table, lengths, 16, 0.2, None, dtype, ct)


@pytest.mark.parametrize("dh", [64, 256])
def test_paged_attention_the_most_sequences(gpu, dh):
    """8,192 of them, the largest tables of rounds in LDS; a page of its own for each, shared by
    the first and the last."""
    g = _g(6)
    B = 8192
    lengths = torch.randint(0, 4, (B,), generator=g, device="cuda", dtype=torch.int32)
    lengths[0] = lengths[-1] = 3
    k, v = (_randn(g, B, 4, 1, dh, dtype=BF) for _ in range(2))
    table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None].clone()
    table[-1] = 0
    q = _randn(g, B, 2, dh, dtype=BF)
    out = ops.paged_attention(q, k, v, table, lengths)
    kk, vv = k[table[:, 0].long(), :, 0].double(), v[table[:, 0].long(), :, 0].double()
    x = (q.double()[:, :, None] * kk[:, None]).sum(-1) * dh ** -0.5
    dead = torch.arange(4, device="cuda") >= lengths[:, None]
    p = torch.softmax(x.masked_fill(dead[:, None], -math.inf), -1).nan_to_num(0.0)
    want, absv = ((p[..., None] * f[:, None]).sum(2) for f in (vv, vv.abs()))
    _close(out, want, _tol(want, absv, vv, BF, BF))


def test_paged_attention_one_long_sequence(gpu):
    """70,001 positions over all blocks, scores far apart, q rows at odd elements."""
    g = _g(6)
    k, v, table = _paged(g, [70_001], 64, 2, 256, BF)
    q = _randn(g, 1, 16, 257, dtype=F32, scale=4.0)[..., 1:]
    n = torch.tensor([70_001], dtype=torch.int32, device="cuda")
    out = ops.paged_attention(q, k, v, table, n)
    kk, vv = _keys(k, table, 0, 70_001, 64), _keys(v, table, 0, 70_001, 64)
    want, absv = _attend_ref(q, kk, vv, 1 / 16, n.long() - 1)
    _close(out, want, 4 * _tol(want, absv, vv, F32, F32))      # scores four times as large


def test_paged_attention_pages_that_are_none(gpu):
    """A page number outside the cache holds no keys; a length past the table counts as the table."""
    g = _g(7)
    k, v, table = _paged(g, [100, 64, 40], 16, 2, 64, BF, poison=False)
    table = table[:, :7].contiguous()
    table[0, 2], table[0, 5], table[1, :] = -1, k.shape[0], 2 ** 31 - 1
    q = _randn(g, 3, 4, 64, dtype=BF)
    n = torch.tensor([112, 64, 10_000], dtype=torch.int32, device="cuda")
    table[0, 6] = 0
    table[2, 3:] = table[0, 0]
    out = ops.paged_attention(q, k, v, table, n)
    seen = torch.ones(112, dtype=torch.bool, device="cuda")
    seen[32:48] = seen[80:96] = False
    for b, s in ((0, seen), (2, None)):
        rows = table[b].clamp(0, k.shape[0] - 1).long()
        kk, vv = k[rows].reshape(-1, 2, 64), v[rows].reshape(-1, 2, 64)
        want, absv = _attend_ref(q[b:b + 1], kk, vv, 0.125, torch.tensor([111], device="cuda"), s)
        _close(out[b:b + 1], want, _tol(want, absv, vv, BF, BF))
    assert bool((out[1] == 0).all())


def test_paged_attention_offsets_past_32_bits(gpu):
    """A cache of 2^32 bytes and more in each array: the last pages are the ones read."""
    g = _g(8)
    n_pages = 70_000
    k, v = (torch.empty(n_pages, 64, 2, 256, dtype=BF, device="cuda") for _ in range(2))
    table = torch.tensor([[69_999, 3, 69_998, 42_000]], dtype=torch.int32, device="cuda")
    for t in (k, v):
        t[table[0].long()] = _randn(g, 4, 64, 2, 256, dtype=BF)
    q = _randn(g, 1, 16, 256, dtype=F32)
    out = ops.paged_attention(q, k, v, table, torch.tensor([250], dtype=torch.int32, device="cuda"))
    kk, vv = _keys(k, table, 0, 250, 64), _keys(v, table, 0, 250, 64)
    want, absv = _attend_ref(q, kk, vv, 1 / 16, torch.tensor([249], device="cuda"))
    _close(out, want, _tol(want, absv, vv, F32, F32))
    qb = q.to(BF).expand(3, 16, 256)
    o2 = ops.prompt_attention(qb, k, v, torch.tensor([0, 3], dtype=torch.int32, device="cuda"), block_table=table,
                              lengths=torch.tensor([250], dtype=torch.int32, device="cuda"))
    want, absv = _attend_ref(qb, kk, vv, 1 / 16, torch.arange(247, 250, device="cuda"))
    _close(o2, want, _tol(want, absv, vv, BF, BF))


def test_paged_attention_large_values(gpu):
    """fp32 queries beyond what 16 bits hold, and tiny ones, against both cache types."""
    g = _g(9)
    for ct in (BF, HF):
        for scale in (1e9, 1e-9):
            k, v, table = _paged(g, [300], 16, 1, 128, ct)
            q = _randn(g, 1, 4, 128) * scale
            n = torch.tensor([300], dtype=torch.int32, device="cuda")
            out = ops.paged_attention(q, k, v, table, n, scale=0.1 / scale)
            kk, vv = _keys(k, table, 0, 300, 16), _keys(v, table, 0, 300, 16)
            want, absv = _attend_ref(q, kk, vv, 0.1 / scale, torch.tensor([299], device="cuda"))
            _close(out, want, _tol(want, absv, vv, F32, F32))


def test_paged_attention_repeats_bit_for_bit_on_two_streams(gpu):
    g = _g(10)
    lengths = [3000, 5, 0, 777]
    k, v, table = _paged(g, lengths, 32, 2, 128, BF)
    q = _randn(g, 4, 8, 128, dtype=BF)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = ops.paged_attention(q, k, v, table, n)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.paged_attention(q, k, v, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------ packed prompts
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("hq,hkv,dh,new,cached,gate", [
    (16, 2, 256, [1], [0], True),
    (16, 2, 256, [40, 0, 17, 130], [0, 5, 300, 3], False),
    (8, 8, 64, [129, 1, 64, 65], [0, 0, 63, 100], True),
    (24, 4, 128, [33, 200], [7, 0], False),
    (7, 1, 256, [95, 5], [0, 31], True),
    (6, 2, 64, [300], [0], False),
    (32, 1, 128, [21], [50], False),
    (4, 4, 128, [513], [0], True),
    (4, 2, 64, [50, 9, 3], [-20, -9, 2], False),      # fewer keys than queries, none at all
])
def test_prompt_attention(gpu, dtype, paged, hq, hkv, dh, new, cached, gate):
    print(f"prompt heads={hq},{hkv},{dh} new={new} cached={cached} {dtype} paged={paged}", flush=True)
    g = _g(sum(new) + dh)
    lengths = [a + b for a, b in zip(new, cached)]
    front, behind = 3, 5                                # rows outside the sequences
    cu = [front]
    for n in new:
        cu.append(cu[-1] + n)
    T = cu[-1] + behind
    row = _randn(g, T, hq, 2 * dh, dtype=dtype)
    q, gt = row[..., :dh], (row[..., dh:] if gate else None)
    cu_q = torch.tensor(cu, dtype=torch.int32, device="cuda")
    page = 16
    out = torch.full((T, hq, dh), 7.0, dtype=dtype, device="cuda")
    if paged:
        k, v, table = _paged(g, lengths, page, hkv, dh, dtype)
        ops.prompt_attention(q, k, v, cu_q, block_table=table, out=out, gate=gt,
                             lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        kv = [(_keys(k, table, b, n, page), _keys(v, table, b, n, page)) for b, n in enumerate(lengths)]
    else:
        ck = [2]
        for n in lengths:
            ck.append(ck[-1] + n)
        kv_row = _randn(g, ck[-1] + 1, 2, hkv, dh, dtype=dtype)
        kv_row[0], kv_row[-1] = float("nan"), float("nan")
        k, v = kv_row[:, 0], kv_row[:, 1]
        ops.prompt_attention(q, k, v, cu_q, cu_k=torch.tensor(ck, dtype=torch.int32, device="cuda"), out=out, gate=gt)
        kv = [(k[ck[b]:ck[b + 1]], v[ck[b]:ck[b + 1]]) for b in range(len(new))]
    assert bool((out[:front] == 7).all()) and bool((out[cu[-1]:] == 7).all())
    for b, n in enumerate(new):
        if n == 0:
            continue
        rows = slice(cu[b], cu[b + 1])
        kk, vv = kv[b]
        if lengths[b] == 0:
            assert bool((out[rows] == 0).all())
            continue
        last = lengths[b] - n + torch.arange(n, device="cuda")
        want, absv = _attend_ref(q[rows], kk, vv, dh ** -0.5, last)
        if gate:
            f = torch.sigmoid(gt[rows].double())
            want, absv = want * f, absv * f
        _close(out[rows], want, _tol(want, absv, vv, dtype, dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_prompt_attention_values_that_are_not_finite(gpu, dtype, dh):
    """A token whose K or V is infinite or NaN changes nothing for the tokens before it, and what
    the later ones get is infinite or NaN where the formula's is."""
    g = _g(11)
    T = 200
    q, k, v = (_randn(g, T, h, dh, dtype=dtype) for h in (4, 2, 2))
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    clean = ops.prompt_attention(q, k, v, cu)
    v[150, 0, 3], v[151, 1, 5], v[152, 1, 7] = float("inf"), float("-inf"), float("nan")
    k[180, 0, 0] = float("nan")
    out = ops.prompt_attention(q, k, v, cu)
    assert torch.equal(out[:150], clean[:150])
    assert torch.isfinite(out[150:180, 2:, 0:5]).all() and torch.equal(out[150:180, 2:, :5], clean[150:180, 2:, :5])
    assert bool((out[150:180, :2, 3] == float("inf")).all())
    assert bool((out[151:, 2:, 5] == float("-inf")).all()) and bool(out[152:, 2:, 7].isnan().all())
    assert bool(out[180:, :2].isnan().all())
    rest = torch.ones(dh, dtype=torch.bool, device="cuda")
    rest[3] = False
    assert torch.equal(out[150:180, :2][..., rest], clean[150:180, :2][..., rest])


def test_prompt_attention_pages_that_are_none(gpu):
    g = _g(12)
    k, v, table = _paged(g, [150], 16, 2, 128, HF, poison=False)
    table[0, 3], table[0, 7] = -1, 2 ** 31 - 1
    q = _randn(g, 90, 4, 128, dtype=HF)
    out = ops.prompt_attention(q, k, v, torch.tensor([0, 90], dtype=torch.int32, device="cuda"), block_table=table,
                               lengths=torch.tensor([150], dtype=torch.int32, device="cuda"))
    seen = torch.ones(160, dtype=torch.bool, device="cuda")
    seen[48:64] = seen[112:128] = False
    rows = table[0, :10].clamp(0, k.shape[0] - 1).long()
    kk, vv = k[rows].reshape(-1, 2, 128)[:150], v[rows].reshape(-1, 2, 128)[:150]
    want, absv = _attend_ref(q, kk, vv, 128 ** -0.5, 60 + torch.arange(90, device="cuda"), seen[:150])
    _close(out, want, _tol(want, absv, vv, HF, HF))


def test_prompt_attention_scores_that_grow(gpu):
    """Later keys score higher and higher, so that the running maximum moves in every tile; and
    scores near the largest that fp16 holds."""
    g = _g(13)
    for dtype, top in ((BF, 60.0), (HF, 60.0), (HF, 30_000.0)):
        q = torch.zeros(300, 2, 64, dtype=dtype, device="cuda")
        q[..., 0] = 1.0
        k = _randn(g, 300, 1, 64, dtype=dtype)
        k[:, 0, 0] = torch.linspace(0, top, 300, device="cuda").to(dtype)
        v = _randn(g, 300, 1, 64, dtype=dtype)
        cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
        out = ops.prompt_attention(q, k, v, cu, scale=1.0)
        want, absv = _attend_ref(q, k, v, 1.0, torch.arange(300, device="cuda"))
        _close(out, want, _tol(want, absv, v, dtype, dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("hq,hkv,dh,new,cached,gate", [
    (16, 2, 256, [1, 1500, 0, 2099, 600], [0, 70, 9, 1, 333], True),    # Dh 256 with enough rows for wide blocks
    (20, 1, 256, [3300], [31], False),
    (8, 2, 64, [i % 7 for i in range(100)], [(5 * i) % 41 for i in range(100)], False),     # over 64 sequences
    (16, 2, 256, [(3 * i) % 40 for i in range(150)], [0] * 150, True),
    (2, 2, 128, [0] * 70 + [300] + [0] * 70 + [129, 1], [0] * 143, False),
])
def test_prompt_attention_large(gpu, dtype, paged, hq, hkv, dh, new, cached, gate):
    test_prompt_attention(gpu, dtype, paged, hq, hkv, dh, new, cached, gate)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dh", [64, 256])
def test_prompt_attention_queries_at_odd_elements(gpu, dtype, dh):
    g = _g(16)
    T = 77
    row = _randn(g, T, 4, 2 * dh + 1, dtype=dtype)
    q, gt = row[..., 1:dh + 1], row[..., dh + 1:]
    k, v = (_randn(g, T, 2, dh, dtype=dtype) for _ in range(2))
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    out = ops.prompt_attention(q, k, v, cu, gate=gt)
    assert torch.equal(out, ops.prompt_attention(q.contiguous(), k, v, cu, gate=gt.contiguous()))
    want, absv = _attend_ref(q, k, v, dh ** -0.5, torch.arange(T, device="cuda"))
    f = torch.sigmoid(gt.double())
    _close(out, want * f, _tol(want * f, absv * f, v, dtype, dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_attention_wide_blocks_on_odd_values(gpu, dtype):
    """The Dh 256 variant for many rows: values that are not finite behind and before a token,
    and scores that grow with every key."""
    g = _g(17)
    T, hq = 4200, 16
    q, k, v = (_randn(g, T, h, 256, dtype=dtype) for h in (hq, 2, 2))
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    clean = ops.prompt_attention(q, k, v, cu)
    at = 3001
    v[at, 0, 3], v[at + 1, 1, 250] = float("inf"), float("nan")
    k[at + 500, 1, 9] = float("nan")
    out = ops.prompt_attention(q, k, v, cu)
    assert torch.equal(out[:at], clean[:at])
    h = hq // 2
    assert bool((out[at:, :h, 3] == float("inf")).all()) and torch.equal(out[at:, :h, 4:], clean[at:, :h, 4:])
    assert bool(out[at + 1:, h:, 250].isnan().all()) and bool(out[at + 500:, h:].isnan().all())
    assert torch.equal(out[at + 1:at + 500, h:, :250], clean[at + 1:at + 500, h:, :250])
    for top in (60.0, 30_000.0):
        q = torch.zeros(T, hq, 256, dtype=dtype, device="cuda")
        q[..., 0] = 1.0
        k = _randn(g, T, 1, 256, dtype=dtype)
        k[:, 0, 0] = torch.linspace(0, top, T, device="cuda").to(dtype)
        v = _randn(g, T, 1, 256, dtype=dtype)
        out = ops.prompt_attention(q, k, v, cu, scale=1.0)
        want, absv = _attend_ref(q[:, :1], k, v, 1.0, torch.arange(T, device="cuda"))
        _close(out[:, :1], want, _tol(want, absv, v, dtype, dtype))
        assert torch.equal(out, out[:, :1].expand_as(out))


def test_prompt_attention_one_token_is_paged_attention(gpu):
    """One query row per sequence: the two operators' results agree to their roundings."""
    g = _g(14)
    lengths = [70, 1, 333]
    k, v, table = _paged(g, lengths, 16, 2, 128, BF)
    q = _randn(g, 3, 8, 128, dtype=BF)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    a = ops.paged_attention(q, k, v, table, n)
    b = ops.prompt_attention(q, k, v, torch.arange(4, dtype=torch.int32, device="cuda"), block_table=table, lengths=n)
    _check_decode(b, q, k, v, table, lengths, 16, 128 ** -0.5, None, BF, BF)
    assert float((a.float() - b.float()).abs().max()) <= 4 * H[BF] * float(v.float().nan_to_num(0, 0, 0).abs().max())


# ------------------------------------------------------------ sampling
def _sample_ref(x, u, t, k, p, mp):
    """One row in 64 bits on the host, filter by filter."""
    x = x.double().cpu()
    x = torch.where(x.isnan(), -math.inf, x) + 0.0
    V = x.numel()
    y, order = torch.sort(x, descending=True, stable=True)
    if y[0] == -math.inf:
        return -1
    if not t > 0:
        return int(order[0])
    w = torch.where(y == y[0], 1.0, torch.exp((y - y[0]) / t))
    if y[0] == math.inf:
        w = (y == math.inf).double()
    w = torch.where(y == -math.inf, 0.0, w)
    keep = w > 0
    rank = torch.arange(V)
    if 0 < k < V:
        keep &= rank < k
    w = torch.where(keep, w, 0.0)
    if p < 1:
        keep &= (rank == 0) | (torch.cumsum(w, 0) - w < p * w.sum())
    if mp > 0:
        keep &= (rank == 0) | (w >= min(mp, 1.0))
    w = torch.zeros(V, dtype=torch.float64).scatter_(0, order, torch.where(keep, w, 0.0))
    run = torch.cumsum(w, 0)
    past = (run > u * run[-1]) & (w > 0)
    return int(past.to(torch.int8).argmax()) if bool(past.any()) else int(w.nonzero()[-1])


def _f32(v):
    return float(torch.tensor(v, dtype=F32))


def _logits(g, B, V, dtype, spread=2.5):
    x = _randn(g, B, V, scale=spread)
    x[:, ::97] += torch.empty_like(x[:, ::97]).exponential_(0.3, generator=g)
    return x.to(dtype)


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 20, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (1.0, 50, 0.9, 0.05), (1.3, 0, 0.9, 0.0),
           (0.8, 0, 1.0, 0.1), (1.0, 0, 0.95, 0.02), (1.0, 1, 0.5, 0.5), (0.0, 5, 0.5, 0.5), (1.0, 300, 0.99, 0.0),
           (2.0, 2000, 1.0, 0.0), (2.0, 3000, 0.9, 0.0), (1.5, 1500, 1.0, 0.001), (0.01, 0, 0.9, 0.0),
           (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1e9, 0, 0.3, 0.0), (math.inf, 7, 1.0, 0.0),
           (5.0, 0, 0.5, 1e-30), (1.0, 10 ** 6, 2.0, -1.0), (float("nan"), 0, 1.0, 0.0), (1.0, 40, 1e-9, 0.0)]


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("V", [1, 5, 511, 512, 513, 1001, 32_000, 248_320])
def test_sample_one_row_each(gpu, V, dtype):
    """Every filter with a value of its own per row (rows at odd elements), the same one by one."""
    print(f"sample V={V} {dtype}", flush=True)
    g = _g(V)
    B = len(FILTERS)
    x = torch.empty(B, V + 3, dtype=dtype, device="cuda")[:, 1:V + 1]
    x.copy_(_logits(g, B, V, dtype))
    u = torch.rand(B, generator=g, device="cuda")
    u[0] = 0.0
    u[1] = 1 - 2.0 ** -24
    t, k, p, mp = (torch.tensor(c, dtype=d, device="cuda") for c, d in
                   zip(zip(*FILTERS), (F32, torch.int32, F32, F32)))
    got = ops.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    assert got.dtype == torch.int64
    want = [_sample_ref(x[b], float(u[b]), *(_f32(f) if i != 1 else f for i, f in enumerate(FILTERS[b])))
            for b in range(B)]
    assert got.tolist() == want
    b = V % B
    tb, kb, pb, mb = FILTERS[b]
    one = ops.sample(x[b:b + 1].contiguous(), u[b:b + 1].contiguous(), temperature=tb, top_k=kb, top_p=pb, min_p=mb)
    assert one.tolist() == [want[b]]


@pytest.mark.parametrize("dtype", [F32, HF])
def test_sample_the_largest_vocabulary(gpu, dtype):
    g = _g(2)
    V = 2 ** 21
    rows = [(0.7, 50, 0.9, 0.0), (1.0, 0, 0.7, 0.0), (1.0, 5000, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0)]
    x = _randn(g, len(rows), V, scale=1.5).to(dtype)
    u = torch.rand(len(rows), generator=g, device="cuda")
    t, k, p, mp = (torch.tensor(c, dtype=d, device="cuda") for c, d in zip(zip(*rows), (F32, torch.int32, F32, F32)))
    got = ops.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    assert got.tolist() == [_sample_ref(x[b], float(u[b]), *(_f32(f) if i != 1 else f for i, f in enumerate(rows[b])))
                            for b in range(len(rows))]
    with pytest.raises(ValueError, match="vocab"):
        ops.sample(torch.empty(1, V + 1, dtype=dtype, device="cuda"), u[:1])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_sample_over_the_unit_interval(gpu, dtype):
    """One row at many u: the picks run through the kept tokens in the vocabulary's order."""
    g = _g(21)
    n = 400
    x = _logits(g, 1, 50_001, dtype).expand(n, -1)
    u = torch.linspace(0, 1 - 2.0 ** -24, n, device="cuda")
    for t, k, p, mp in ((0.7, 30, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 2500, 1.0, 0.0), (1.0, 0, 1.0, 0.0)):
        got = ops.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
        assert got.tolist() == [_sample_ref(x[0], float(v), _f32(t), k, _f32(p), mp) for v in u.tolist()]
        assert got.tolist() == sorted(got.tolist())


@pytest.mark.parametrize("V", [700, 3001, 248_320])
@pytest.mark.parametrize("t,k,p,mp", [(1.0, 0, 0.5, 0.0), (1.0, 10, 1.0, 0.0), (1.0, 2000, 1.0, 0.0),
                                      (1.0, 2000, 0.25, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.5)])
def test_sample_ties(gpu, V, t, k, p, mp):
    """Rows of one value, and of two: ties go to the lowest index, at the borders too."""
    x = torch.zeros(3, V, device="cuda")
    x[1, V // 2:] = 1.0
    x[2] = -0.0
    x[2, ::2] = 0.0
    u = torch.tensor([0.5, 0.25, 0.9999], device="cuda")
    got = ops.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    assert got.tolist() == [_sample_ref(x[b], float(u[b]), t, k, p, mp) for b in range(3)]


def test_sample_rows_that_are_masked(gpu):
    """-inf and NaN are never taken, a row of nothing else gives -1, and +inf takes everything."""
    inf, nan = float("inf"), float("nan")
    V = 2000
    x = torch.full((8, V), -inf, device="cuda")
    x[1, 777] = -3e38
    x[2] = nan
    x[3, 5:9] = torch.tensor([nan, 1.0, nan, 2.0], device="cuda")
    x[4] = torch.randn(V, generator=_g(1), device="cuda")
    x[4, [100, 900, 1500]] = inf
    x[5] = torch.finfo(F32).min
    x[6, 1999] = 0.0
    x[7] = nan
    x[7, 3] = -1e-40
    u = torch.full((8,), 0.5, device="cuda")
    for t, k, p, mp in FILTERS:
        got = ops.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
        assert got.tolist() == [_sample_ref(x[b], 0.5, _f32(t), k, _f32(p), _f32(mp)) for b in range(8)], (t, k, p, mp)


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("V", [4000, 131_072])
def test_sample_flat_rows_of_both_signs(gpu, V, dtype):
    """Thousands of values about 0 that are nearly equal in weight: the cut is found among
    their bits, where the order of the negative ones is the other way round."""
    g = _g(V)
    flat = [(1.0, V // 2, 1.0, 0.0), (1.0, 0, 0.4, 0.0), (1.0, 3 * V // 4, 0.7, 0.0), (1.0, V - 1, 1.0, 0.0),
            (1.0, 0, 1 - 2.0 ** -24, 0.0), (1.0, 0, 0.6, 0.9995), (1.0, 0, 1.0, 0.9995), (1e-4, 0, 0.9999, 0.0),
            (1e-5, V // 3, 1.0, 0.0), (1e-4, V // 3, 0.9999, 1e-12), (1e-2, 0, 0.9999999, 0.0)]
    x = _randn(g, len(flat), V, scale=1e-3).to(dtype)
    u = torch.rand(len(flat), generator=g, device="cuda")
    t, k, p, mp = (torch.tensor(c, dtype=d, device="cuda") for c, d in zip(zip(*flat), (F32, torch.int32, F32, F32)))
    got = ops.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    assert got.tolist() == [_sample_ref(x[b], float(u[b]), *(_f32(f) if i != 1 else f for i, f in enumerate(flat[b])))
                            for b in range(len(flat))]


@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_sample_filters_that_end_far_out(gpu, dtype):
    """A few tokens far above all others: the k-th value is tens to thousands of temperatures
    away, past the histogram's fine bins and past its last."""
    g = _g(77)
    V = 30_000
    rows = [(t, k, p, mp) for t in (0.5, 0.2, 0.01) for k, p, mp in
            ((40, 1.0, 0.0), (1500, 1.0, 0.0), (300, 0.999, 0.0), (0, 1 - 2.0 ** -24, 0.0), (0, 1.0, 1e-30), (5, 0.9, 0.5))]
    x = _randn(g, len(rows), V, scale=2.0)
    x[:, 17:V:4001] += 15.0
    x = x.to(dtype)
    u = torch.rand(len(rows), generator=g, device="cuda")
    u[::2] = 1 - 2.0 ** -24
    t, k, p, mp = (torch.tensor(c, dtype=d, device="cuda") for c, d in zip(zip(*rows), (F32, torch.int32, F32, F32)))
    got = ops.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    assert got.tolist() == [_sample_ref(x[b], float(u[b]), *(_f32(f) if i != 1 else f for i, f in enumerate(rows[b])))
                            for b in range(len(rows))]


# ------------------------------------------------------------ capture, a run of them together
def test_captured_and_replayed_with_other_lengths(gpu):
    """A decode step of the four operators in a graph: replayed with other positions, lengths,
    tables and numbers, eager calls in between, every replay equal to the eager result."""
    g = _g(31)
    B, hq, hkv, dh, page, V = 6, 8, 2, 128, 16, 5000
    k, v, table = _paged(g, [400] * B, page, hkv, dh, BF, poison=False)
    inv = 1e6 ** (-torch.arange(32, dtype=torch.float64, device="cuda") / 32)
    lm = _randn(g, hq * dh, V, scale=0.05)
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")

    def fresh(seed):
        h = _g(seed)
        n = torch.randint(1, 400, (B,), generator=h, device="cuda", dtype=torch.int32)
        n[2] = 1
        at = n - 1
        slot = table[torch.arange(B, device="cuda"), (at // page).long()] * page + at % page
        return {"qkv": _randn(h, B, hq + 2 * hkv, dh), "n": n, "pos": at.contiguous(), "slot": slot,
                "u": torch.rand(B, generator=h, device="cuda")}

    def step(s, kp, vp):
        q = ops.rope_append(s["qkv"][:, :hq], s["qkv"][:, hq:hq + hkv], s["qkv"][:, hq + hkv:], s["pos"], inv, kp, vp,
                            s["slot"])
        a = ops.paged_attention(q, kp, vp, table, s["n"])
        b = ops.prompt_attention(q, kp, vp, cu, block_table=table, lengths=s["n"])
        logits = a.float().view(B, -1) @ lm
        ids = ops.sample(logits, s["u"], temperature=0.9, top_p=0.9)
        return a, b, ids

    held = fresh(100)
    kg, vg = k.clone(), v.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held, kg, vg)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(held, kg, vg)
    for seed in (101, 102, 103):
        new = fresh(seed)
        for name, t in held.items():
            t.copy_(new[name])
        kg.copy_(k)
        vg.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        ke, ve = k.clone(), v.clone()
        want = step(new, ke, ve)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(kg, ke) and torch.equal(vg, ve)


def test_tensors_on_the_host_are_refused(gpu):
    x, u = torch.zeros(1, 8, device="cuda"), torch.zeros(1)
    with pytest.raises(ValueError, match="different devices"):
        ops.sample(x, u)


def test_outputs_over_inputs_and_values_out_of_range_are_refused(gpu):
    g = _g(41)
    q = _randn(g, 2, 4, 64, dtype=BF)
    k, v, table = _paged(g, [20, 9], 16, 2, 64, BF, poison=False)
    n = torch.tensor([20, 9], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        ops.paged_attention(q, k, v, table, n, out=q)
    rows = _randn(g, 3, 4, 128, dtype=BF)
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    kv = _randn(g, 3, 2, 64, dtype=BF)
    flat = rows.view(-1)[:3 * 4 * 64].view(3, 4, 64)
    with pytest.raises(ValueError, match="overlaps"):
        ops.prompt_attention(rows[..., 64:], kv, kv, cu, out=flat)
    out = torch.empty(3, 4, 64, dtype=BF, device="cuda")
    assert ops.prompt_attention(rows[..., 64:], kv, kv, cu, out=out) is out
    x, u = _randn(g, 2, 100), torch.rand(2, device="cuda")
    for kw in (dict(top_k=2 ** 40), dict(top_k=2.5)):
        with pytest.raises(ValueError, match="GmSampleArgs"):
            ops.sample(x, u, **kw)
    # past fp32's range is infinity, as in any fp32 tensor
    assert ops.sample(x, u, temperature=1e300).tolist() == ops.sample(x, u, temperature=math.inf).tolist()
    buf = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        ops.sample(x, buf.view(torch.float32)[:2], out=buf[:2])


def test_calls_on_two_streams_at_once(gpu):
    """Every operator on two streams in turn, with nothing between: each call's result is the
    one it gives alone."""
    g = _g(51)
    x, u = _logits(g, 40, 50_001, BF), torch.rand(40, generator=g, device="cuda")
    q, k, v = (_randn(g, 900, h, 128, dtype=HF) for h in (8, 2, 2))
    cu = torch.tensor([0, 200, 201, 900], dtype=torch.int32, device="cuda")
    kp, vp, table = _paged(g, [700, 3, 90], 16, 2, 128, HF, poison=False)
    n = torch.tensor([700, 3, 90], dtype=torch.int32, device="cuda")
    calls = (lambda: ops.sample(x, u, temperature=1.1, top_p=0.9), lambda: ops.sample(x, u, top_k=700, min_p=0.01),
             lambda: ops.prompt_attention(q, k, v, cu), lambda: ops.paged_attention(q[:3], kp, vp, table, n))
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        for j, f in enumerate(calls):
            with torch.cuda.stream(streams[(i + j) % 2]):
                got.append((j, f()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[j]) for j, o in got)


@pytest.mark.parametrize("dtype,ct", TYPES)
def test_paged_attention_values_that_are_not_finite(gpu, dtype, ct):
    """An infinite or NaN V that a sequence sees shows in its dim, and nowhere else."""
    g = _g(52)
    k, v, table = _paged(g, [300, 300], 16, 2, 128, ct, poison=False)
    table[1] = table[0]
    q = _randn(g, 2, 8, 128, dtype=dtype)
    n = torch.tensor([300, 40], dtype=torch.int32, device="cuda")
    clean = ops.paged_attention(q, k, v, table, n)
    page, row = int(table[0, 6]), 4                      # position 100: of the first sequence alone
    v[page, row, 0, 5], v[page, row, 1, 77] = float("inf"), float("nan")
    out = ops.paged_attention(q, k, v, table, n)
    assert torch.equal(out[1], clean[1])
    assert not torch.isfinite(out[0, :4, 5]).any() and bool(out[0, 4:, 77].isnan().all())
    out[0, :4, 5], out[0, 4:, 77] = clean[0, :4, 5], clean[0, 4:, 77]
    assert torch.equal(out, clean)


def test_prompt_attention_heads_that_are_expanded(gpu):
    g = _g(53)
    q, k, v = (_randn(g, 150, h, 64, dtype=BF) for h in (6, 1, 1))
    cu = torch.tensor([0, 31, 150], dtype=torch.int32, device="cuda")
    want = ops.prompt_attention(q, k, v, cu)
    got = ops.prompt_attention(q, k.expand(-1, 3, -1), v.expand(-1, 3, -1), cu)
    for b, (i, j) in enumerate(((0, 31), (31, 150))):
        ref, absv = _attend_ref(q[i:j], k[i:j], v[i:j], 64 ** -0.5, torch.arange(j - i, device="cuda"))
        for o in (want, got):
            _close(o[i:j], ref, _tol(ref, absv, v, BF, BF))
