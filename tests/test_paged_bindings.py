"""Layouts that the paged bindings take and refuse (no GPU needed)."""
import pytest
import torch


def test_the_stride_of_a_single_head_does_not_matter(capi):
    t = torch.zeros(1, 5, 8).transpose(0, 1)                  # [5 tokens, 1 head, 8], heads 40 elements apart as far as torch says
    assert t.stride() == (8, 40, 1)
    assert capi._rows(t, "q", -1) == (t.data_ptr(), 8)
    wide = torch.zeros(1, 5, 24)[:, :, 8:16].transpose(0, 1)
    assert capi._rows(wide, "q", -1) == (wide.data_ptr(), 24)


def test_heads_apart_are_refused(capi):
    for t in (torch.zeros(5, 4, 8)[:, ::2], torch.zeros(2, 5, 8).transpose(0, 1), torch.zeros(5, 2, 16)[:, :, ::2]):
        with pytest.raises(ValueError):
            capi._rows(t, "q", -1)
