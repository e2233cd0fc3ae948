"""The paged cache's bookkeeping, on the host: pages, slots, tables and refusals."""
import pytest
import torch

from npu_amd import qwen_core as QN, qwen_serve as QS


def _cache(n_seq=3, n_pages=8, page=4, **kw):
    cfg = QN.Config(d_model=256, n_layer=2, n_head=2, n_head_kv=1, head_dim=64, is_attention=[False, True])
    return QS.PagedCache(cfg, n_seq, n_pages, page_size=page, dev=torch.device("cpu"), **kw)


def test_pages_are_given_out_once_and_come_back():
    c = _cache()
    assert c.k[0] is None and c.k[1].shape == (8, 4, 1, 64) and c.k[1].dtype == torch.bfloat16
    s = c.reserve([5, 0, 4])
    assert (s.seqs, s.counts, s.single) == ([0, 2], [5, 4], False)
    assert s.positions.tolist() == [0, 1, 2, 3, 4, 0, 1, 2, 3] and s.cu_q.tolist() == [0, 5, 9]
    assert s.lengths.tolist() == [5, 4] and s.table.shape == (2, 2) and s.table[1, 1] == -1
    assert len(set(s.slots.tolist())) == 9
    for b, row in enumerate(s.table.tolist()):
        for j, p in enumerate(s.positions[s.cu_q[b]:s.cu_q[b + 1]].tolist()):
            assert s.slots[s.cu_q[b] + j] == row[p // 4] * 4 + p % 4
    one = c.reserve([1, 1, 1])
    assert one.single and one.lengths.tolist() == [6, 1, 5] and one.positions.tolist() == [5, 0, 4]
    assert one.table[0, :2].tolist() == s.table[0].tolist()
    assert not set(one.slots.tolist()) & set(s.slots.tolist())
    used = [p for pages in c.pages for p in pages]
    assert len(used) == len(set(used)) == 8 - len(c.free)
    c.release(0)
    assert c.length == [0, 1, 5] and c.pages[0] == [] and len(c.free) == 8 - 3
    for b in (1, 2):
        c.release(b)
    assert sorted(c.free) == list(range(8))


def test_a_step_that_does_not_fit_changes_nothing():
    c = _cache(n_seq=2, n_pages=3)
    c.reserve([4, 3])
    before = (list(c.length), [list(p) for p in c.pages], list(c.free))
    with pytest.raises(MemoryError, match="2 pages needed, 1 of 3 free"):
        c.reserve([1, 2])
    assert before == (c.length, c.pages, c.free)
    assert c.reserve([0, 1]).seqs == [1] and c.reserve([0, 0]).table.shape == (0, 0)


@pytest.mark.parametrize("kw,error", [(dict(n_seq=0), ValueError), (dict(n_pages=0), ValueError),
                                      (dict(page=0), ValueError), (dict(dtype=torch.float32), TypeError),
                                      (dict(n_pages=2 ** 20, page=2 ** 11), ValueError)])
def test_caches_that_are_refused(kw, error):
    with pytest.raises(error, match="PagedCache"):
        _cache(**kw)


@pytest.mark.parametrize("counts", [[1], [1, -1, 0], [1, 2, 3, 4]])
def test_counts_that_are_refused(counts):
    with pytest.raises(ValueError, match="counts must be"):
        _cache().reserve(counts)


def test_rope_axes_turn_as_the_table_does():
    inv, axis = QS.build_rope_axes(64, 1e6, dev=torch.device("cpu"))
    cos, sin = QN.build_partial_rope_cache(64, 50, 1e6)
    a = torch.arange(50, dtype=torch.float64)[:, None] * inv
    # the table's angles are fp32: position 49 times two roundings of 2^-24, and its own
    assert axis is None and float((a.cos() - cos[:, :32]).abs().max()) <= 49 * 3 * 2.0 ** -24
    assert float((a.sin() - sin[:, 32:]).abs().max()) <= 49 * 3 * 2.0 ** -24
    assert QS.build_rope_axes(16, 1e4, (3, 1, 4), torch.device("cpu"))[1].tolist() == [0, 0, 0, 1, 2, 2, 2, 2]
    with pytest.raises(ValueError, match="do not add up"):
        QS.build_rope_axes(16, 1e4, (3, 1), torch.device("cpu"))


def test_prompts_that_are_refused():
    c = _cache()
    with pytest.raises(ValueError, match="2 prompts for 3 sequences"):
        QS.generate(None, [[1], [2]], 4, c)
    with pytest.raises(ValueError, match="needs a token"):
        QS.generate(None, [[1], [], [2]], 4, c)
    c.reserve([1, 0, 0])
    with pytest.raises(ValueError, match="must be empty"):
        QS.generate(None, [[1], [2], [3]], 4, c)
