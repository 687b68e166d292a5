"""The host side of PagedSequenceCache (no GPU): pages, lengths, refusals."""

import pytest
import torch

from mx_fbgemm.sequence_attention import PagedSequenceCache


def make(**kw):
    args = dict(pages=6, page_size=4, heads=2, head_dim=16, max_sequences=3, max_length=16, device="cpu")
    return PagedSequenceCache(**{**args, **kw})


def table_of(c, s):
    return c._rows([s])[0].tolist()


def test_pages_follow_the_lengths_and_come_back():
    c = make()
    a, b = c.add(), c.add()
    assert (a, b, c.free_pages, c.length(a)) == (0, 1, 6, 0)
    c._reserve([a, b], [5, 4])
    assert c.free_pages == 3
    rows = c._rows([a, b])
    assert rows.shape == (2, 2) and rows.data_ptr() == c._table.data_ptr()
    used = set(c._pages[a]) | set(c._pages[b])
    assert len(used) == 3 and rows[0].tolist() == c._pages[a] and rows[1].tolist() == [*c._pages[b], -1]
    assert c._rows([b, a]).tolist() == [[*c._pages[b], -1], c._pages[a]]
    c._reserve([a], [8])  # inside its second page
    assert c.free_pages == 3
    c.remove(a)
    assert c.free_pages == 5
    assert c.add() == a and c.length(a) == 0
    c._reserve([a], [16])
    assert c.free_pages == 1 and table_of(c, a) == c._pages[a] and not set(c._pages[a]) & set(c._pages[b])


def test_all_pages_or_none():
    c = make(pages=3)
    a, b = c.add(), c.add()
    with pytest.raises(RuntimeError, match="4 pages needed, 3 free"):
        c._reserve([a, b], [8, 8])
    assert c.free_pages == 3 and c._pages == {a: [], b: []}
    with pytest.raises(RuntimeError, match="max_length 16"):
        c._reserve([a], [17])


def test_refusals():
    for kw in (dict(pages=0), dict(page_size=0), dict(head_dim=12), dict(head_dim=136), dict(max_length=0),
               dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            make(**kw)
    c = make()
    a = c.add()
    k = torch.zeros((2, 2, 16), dtype=torch.bfloat16)
    with pytest.raises(KeyError):
        c.append([2], [2], k, k)
    with pytest.raises(KeyError):
        c.remove(1)
    with pytest.raises(ValueError):
        c.append([a], [1], k, k)
    with pytest.raises(ValueError):
        c.append([a, a], [1, 1], k, k)
    with pytest.raises(ValueError):
        c.append([a], [-1], k, k)
    with pytest.raises(ValueError):
        c.attend([a], k)
    c.add(), c.add()
    with pytest.raises(RuntimeError, match="in use"):
        c.add()
    c.append([], [], k[:0], k[:0])
