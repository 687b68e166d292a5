"""The rotary table that a cache object keeps."""

import torch

from mx_fbgemm.sequence_attention import PagedSequenceCache, rotary_table


def make_cache(rotary):
    return PagedSequenceCache(pages=4, page_size=4, heads=1, head_dim=32, max_sequences=2, max_length=16, device="cpu",
                              rotary=rotary)


def test_a_view_of_a_table_is_laid_out_once():
    wide = rotary_table(20, 64, device="cpu")
    view = wide[:, 8:16]
    assert not view.is_contiguous()
    kept = make_cache(view)._rotary
    assert kept.is_contiguous() and kept.data_ptr() % 16 == 0 and torch.equal(kept, view)


def test_a_contiguous_table_is_the_callers_own():
    table = rotary_table(16, 32, device="cpu")
    assert make_cache(table)._rotary is table and make_cache(None)._rotary is None
