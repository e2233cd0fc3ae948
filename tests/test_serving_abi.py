"""The serving operators' argument checks (no GPU: nothing is ever launched): the C entry
points' refusals and workspace sizes, and the Python wrappers' shapes and types."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

from npu_amd import _lib as L, ops

HEADER = (Path(__file__).resolve().parents[1] / "include" / "npu_amd.h").read_text()
P = 1 << 20                                       # a pointer that is aligned and never followed
BF, F16, F32 = L.GM_QTYPE_BF16, L.GM_QTYPE_F16, L.GM_QTYPE_F32


@pytest.mark.parametrize("cname,mirror", [("gm_rope_append_args", "GmRopeAppendArgs"),
                                          ("gm_paged_attn_args", "GmPagedAttnArgs"),
                                          ("gm_prompt_attn_args", "GmPromptAttnArgs"),
                                          ("gm_sample_args", "GmSampleArgs")])
def test_struct_layout_matches_header(cname, mirror):
    fields = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), HEADER, re.S).group(1)
    fields = re.sub(r"/\*.*?\*/", "", fields, flags=re.S)
    flat, types = [], []
    for decl in filter(None, (d.strip() for d in fields.split(";"))):
        kind = re.match(r"(?:const )?(\w+)(\s*\*)?", decl)
        names = decl[kind.end():].replace("*", "").split(",")
        flat += [n.strip() for n in names]
        types += ["ptr" if kind.group(2) or "*" in decl else kind.group(1)] * len(names)
    mirrored = getattr(L, mirror)._fields_
    assert flat == [f for f, _ in mirrored]
    as_c = {ctypes.c_void_p: "ptr", ctypes.c_int64: "int64_t", ctypes.c_int: "int32_t", ctypes.c_float: "float"}
    assert types == [as_c[t] for _, t in mirrored]


def _set(cls, base, kw):
    a = cls()
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


ROPE = dict(q=P, k=P, v=P, positions=P, inv_freq=P, q_out=P, k_pages=P, v_pages=P, slots=P, q_stride_t=1024,
            q_stride_h=256, k_stride_t=512, k_stride_h=256, v_stride_t=512, v_stride_h=256, n_rows=64, eps=1e-6, T=2,
            n_axes=1, n_head=4, n_head_kv=2, head_dim=256, rope_dim=64, in_type=F32, out_type=BF, cache_type=BF)


@pytest.mark.parametrize("kw,says", [
    (dict(n_head=3), "multiple of n_head_kv"), (dict(head_dim=96), "head_dim=96"), (dict(head_dim=512), "head_dim"),
    (dict(rope_dim=63), "rope_dim"), (dict(rope_dim=258), "rope_dim"), (dict(rope_dim=-2), "rope_dim"),
    (dict(in_type=L.GM_QTYPE_I8), "in_type"), (dict(cache_type=F32), "cache_type"), (dict(out_type=18), "out_type"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(n_rows=1 << 31), "n_rows"), (dict(T=-1), "T"),
    (dict(n_axes=0), "axis"), (dict(slots=0), "NULL"), (dict(inv_freq=0), "NULL"), (dict(k_pages=0), "NULL"),
    (dict(q_out=P + 8), "16-byte"), (dict(v_pages=P + 2), "16-byte"), (dict(n_head=1 << 20, n_head_kv=1), "n_head"),
])
def test_rope_append_refusals(kw, says):
    assert L.lib().gm_rope_append(ctypes.byref(_set(L.GmRopeAppendArgs, ROPE, kw)), None) == L.GM_EINVAL
    assert says in L.last_error()


def test_no_tokens_do_nothing():
    lib = L.lib()
    assert lib.gm_rope_append(ctypes.byref(_set(L.GmRopeAppendArgs, ROPE, dict(T=0, q=0, slots=0))), None) == L.GM_OK
    assert lib.gm_rope_append(None, None) == L.GM_EINVAL
    assert lib.gm_prompt_attention(ctypes.byref(_set(L.GmPromptAttnArgs, PROMPT, dict(n_q=0))), None) == L.GM_OK
    assert lib.gm_paged_attention(ctypes.byref(_set(L.GmPagedAttnArgs, PAGED, dict(n_seq=0))), None, 0, None) == L.GM_OK
    assert lib.gm_sample(ctypes.byref(_set(L.GmSampleArgs, SAMPLE, dict(n_row=0))), None, 0, None) == L.GM_OK


PAGED = dict(q=P, k_pages=P, v_pages=P, block_table=P, lengths=P, out=P, q_stride_t=1024, q_stride_h=256,
             table_stride=8, scale=0.1, n_seq=3, n_head=4, n_head_kv=2, head_dim=256, n_pages=16, page_size=16,
             table_width=8, q_type=BF, cache_type=BF, gate_type=BF)


@pytest.mark.parametrize("kw,says", [
    (dict(n_head=5), "multiple"), (dict(head_dim=80), "head_dim"), (dict(n_seq=8193), "n_seq"),
    (dict(n_pages=0), "positive"), (dict(page_size=0), "positive"), (dict(n_pages=1 << 28), "cache rows"),
    (dict(table_stride=7), "table_stride"), (dict(table_width=-1, table_stride=0), "table_stride"),
    (dict(n_seq=8000, table_width=1 << 20, table_stride=1 << 20), "positions"), (dict(cache_type=F32), "cache_type"),
    (dict(q_type=F16), "q_type"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
])
def test_paged_attention_refusals(kw, says):
    a = _set(L.GmPagedAttnArgs, PAGED, kw)
    assert L.lib().gm_paged_attention_workspace_bytes(ctypes.byref(a)) == 0
    assert L.lib().gm_paged_attention(ctypes.byref(a), P, 1 << 30, None) == L.GM_EINVAL
    assert says in L.last_error()


@pytest.mark.parametrize("kw,says", [
    (dict(block_table=0), "NULL"), (dict(lengths=0), "NULL"), (dict(out=P + 4), "16-byte"),
    (dict(k_pages=P + 8), "16-byte"), (dict(gate=P, gate_type=3), "gate_type"),
])
def test_paged_attention_pointers(kw, says):
    a = _set(L.GmPagedAttnArgs, PAGED, kw)
    assert L.lib().gm_paged_attention(ctypes.byref(a), P, 1 << 30, None) == L.GM_EINVAL
    assert says in L.last_error()


def test_workspaces():
    lib = L.lib()
    a = _set(L.GmPagedAttnArgs, PAGED, {})
    n = lib.gm_paged_attention_workspace_bytes(ctypes.byref(a))
    assert n > 0 and n % 256 == 0
    assert lib.gm_paged_attention(ctypes.byref(a), P, n - 1, None) == L.GM_EWORKSPACE
    assert lib.gm_paged_attention(ctypes.byref(a), P + 16, n, None) == L.GM_EINVAL and "256-byte" in L.last_error()
    # bounded however long the tables are
    big = _set(L.GmPagedAttnArgs, PAGED, dict(n_seq=512, table_width=8192, table_stride=8192, n_head=32))
    assert lib.gm_paged_attention_workspace_bytes(ctypes.byref(big)) < 256 << 20
    s = _set(L.GmSampleArgs, SAMPLE, {})
    n = lib.gm_sample_workspace_bytes(ctypes.byref(s))
    assert n > 0 and n % 256 == 0
    assert lib.gm_sample(ctypes.byref(s), P, n - 1, None) == L.GM_EWORKSPACE
    assert lib.gm_sample(ctypes.byref(s), P + 16, n, None) == L.GM_EINVAL and "256-byte" in L.last_error()


PROMPT = dict(q=P, k=P, v=P, cu_q=P, cu_k=P, out=P, q_stride_t=1024, q_stride_h=256, k_stride_t=512, k_stride_h=256,
              v_stride_t=512, v_stride_h=256, scale=0.1, n_q=10, n_k=10, n_seq=2, n_head=4, n_head_kv=2, head_dim=256,
              type=BF)
PAGES = dict(cu_k=0, block_table=P, lengths=P, n_pages=4, page_size=16, table_width=4, table_stride=4)


@pytest.mark.parametrize("kw,says", [
    (dict(n_head=3), "multiple"), (dict(head_dim=32), "head_dim"), (dict(type=F32), "type"), (dict(n_q=-1), "negative"),
    (dict(n_seq=9000), "n_seq"), (dict(scale=0.0), "scale"), (dict(block_table=P), "packed"), (dict(lengths=P), "packed"),
    (dict(cu_k=0), "NULL"), (dict(cu_q=0), "NULL"), (dict(k_stride_t=511), "16-byte"), (dict(v=P + 2), "16-byte"),
    (dict(out=P + 8), "16-byte"), (dict(gate=P, gate_type=7), "gate_type"), (dict(n_q=1 << 30, n_head=8), "n_q"),
    (dict(PAGES, page_size=0), "positive"), (dict(PAGES, lengths=0), "packed"), (dict(PAGES, cu_k=P), "packed"),
    (dict(PAGES, table_stride=3), "table_stride"),
])
def test_prompt_attention_refusals(kw, says):
    assert L.lib().gm_prompt_attention(ctypes.byref(_set(L.GmPromptAttnArgs, PROMPT, kw)), None) == L.GM_EINVAL
    assert says in L.last_error()


SAMPLE = dict(logits=P, u=P, ids=P, row_stride=1000, temperature_all=1.0, top_p_all=1.0, n_row=4, vocab=1000, type=F32)


@pytest.mark.parametrize("kw,says", [
    (dict(vocab=0), "vocab"), (dict(vocab=(1 << 21) + 1), "vocab"), (dict(n_row=-1), "n_row"), (dict(n_row=70_000), "n_row"),
    (dict(type=18), "type"), (dict(row_stride=-1), "row_stride"), (dict(logits=0), "NULL"), (dict(u=0), "NULL"),
    (dict(ids=0), "NULL"), (dict(logits=P + 2), "aligned"),
])
def test_sample_refusals(kw, says):
    assert L.lib().gm_sample(ctypes.byref(_set(L.GmSampleArgs, SAMPLE, kw)), P, 1 << 30, None) == L.GM_EINVAL
    assert says in L.last_error()


# ------------------------------------------------------------ the Python wrappers
def _z(*s, dt=torch.bfloat16):
    return torch.zeros(*s, dtype=dt)


def _i(*s):
    return torch.zeros(*s, dtype=torch.int32)


def _rope(**kw):
    a = dict(q=_z(3, 4, 64), k=_z(3, 2, 64), v=_z(3, 2, 64), positions=_i(3), inv_freq=torch.zeros(8, dtype=torch.float64),
             k_pages=_z(2, 4, 2, 64), v_pages=_z(2, 4, 2, 64), slots=_i(3))
    a.update(kw)
    return ops.rope_append(**a)


@pytest.mark.parametrize("kw,err", [
    ({}, ValueError),                                           # on the host
    (dict(q=_z(3, 4, 128)), ValueError), (dict(q=_z(3, 4, 64).double()), TypeError), (dict(k=_z(4, 2, 64)), ValueError),
    (dict(k=_z(3, 2, 64).float()), TypeError), (dict(q=_z(3, 64, 4).transpose(1, 2)), ValueError),
    (dict(positions=_i(3).long()), TypeError), (dict(positions=_i(2, 4)), ValueError), (dict(slots=_i(4)), ValueError),
    (dict(inv_freq=torch.zeros(8)), TypeError), (dict(axis=_i(7)), ValueError), (dict(q_norm=torch.ones(32)), ValueError),
    (dict(k_pages=_z(2, 4, 2, 64).float()), TypeError), (dict(v_pages=_z(2, 4, 2, 64).half()), ValueError),
    (dict(k_pages=_z(4, 2, 64)), ValueError), (dict(positions=_i(3, 2).t()), ValueError),
])
def test_rope_append_wrapper_refusals(kw, err):
    with pytest.raises(err):
        _rope(**kw)


def _decode(**kw):
    a = dict(q=_z(3, 4, 64), k_pages=_z(2, 4, 2, 64), v_pages=_z(2, 4, 2, 64), block_table=_i(3, 2), lengths=_i(3))
    a.update(kw)
    return ops.paged_attention(**a)


@pytest.mark.parametrize("kw,err", [
    ({}, ValueError), (dict(q=_z(3, 4, 32)), ValueError), (dict(q=_z(12, 64)), ValueError), (dict(lengths=_i(2)), ValueError),
    (dict(lengths=_i(3).long()), TypeError), (dict(block_table=_i(2, 2)), ValueError),
    (dict(block_table=_i(2, 3).t()), ValueError), (dict(gate=_z(3, 4, 32)), ValueError), (dict(lengths=_i(6)[::2]), ValueError),
    (dict(k_pages=_z(2, 2, 4, 64).transpose(1, 2)), ValueError), (dict(out=_z(3, 4, 64).float()), ValueError),
])
def test_paged_attention_wrapper_refusals(kw, err):
    with pytest.raises(err):
        _decode(**kw)


def _prompt(**kw):
    a = dict(q=_z(9, 4, 64), k=_z(9, 2, 64), v=_z(9, 2, 64), cu_q=_i(3))
    a.update(kw)
    return ops.prompt_attention(**a)


@pytest.mark.parametrize("kw,err", [
    ({}, ValueError), (dict(q=_z(9, 4, 64).float()), TypeError), (dict(k=_z(9, 2, 64).half()), TypeError),
    (dict(cu_k=_i(4)), ValueError), (dict(lengths=_i(2)), ValueError), (dict(block_table=_i(2, 2)), ValueError),
    (dict(block_table=_i(2, 2), lengths=_i(2)), ValueError), (dict(v=_z(8, 2, 64)), ValueError),
    (dict(k=_z(9, 2, 128), v=_z(9, 2, 128)), ValueError), (dict(cu_q=_i(0)), ValueError),
    (dict(cu_q=_i(3).long()), TypeError), (dict(cu_q=_i(6)[::2]), ValueError),
])
def test_prompt_attention_wrapper_refusals(kw, err):
    with pytest.raises(err):
        _prompt(**kw)


@pytest.mark.parametrize("kw,err", [
    ({}, ValueError), (dict(logits=_z(2, 0)), ValueError), (dict(logits=_z(2, 8).double()), TypeError),
    (dict(u=torch.zeros(3)), ValueError), (dict(u=torch.zeros(2).double()), ValueError),
    (dict(top_k=torch.zeros(2)), ValueError), (dict(top_p=torch.zeros(3)), ValueError),
    (dict(logits=_z(8, 2).t()), ValueError), (dict(logits=_z(8)), ValueError), (dict(min_p=_z(2)), ValueError),
])
def test_sample_wrapper_refusals(kw, err):
    a = dict(logits=_z(2, 8), u=torch.zeros(2))
    a.update(kw)
    with pytest.raises(err):
        ops.sample(**a)
