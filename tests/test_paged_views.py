"""Views of queries that the paged decode's wrapper takes or refuses, without a
GPU: host tensors that say they lie on the backend's device."""
import pytest

import aigpu
from test_paged_refusals import _here


def _call(q, heads, dim=64, **kw):
    import torch
    if aigpu.available():
        pytest.skip("the tensors are the host's: no call is made beside a device")
    pages = _here(torch.zeros((4, 2, 16, dim), dtype=torch.bfloat16))
    table, lengths = _here(torch.zeros((3, 5), dtype=torch.int32)), _here(torch.zeros(3, dtype=torch.int32))
    out = _here(torch.zeros((3, heads, dim)))
    aigpu.paged_decode(_here(q), out, pages, pages, table, lengths, stream=0, **kw)


@pytest.mark.parametrize("view", ["first half", "second half", "every other head", "one column short"])
def test_a_gated_query_is_twice_dim_wide(view):
    """a head stride of 2 dim is not enough: the gate of these views would be read outside them, the last one's past
    the end of the buffer"""
    import torch
    wide = torch.zeros((3, 4, 128))
    q = {"first half": wide[..., :64], "second half": wide[..., 64:],
         "every other head": torch.zeros((3, 8, 64))[:, 1::2], "one column short": wide[..., :127]}[view]
    with pytest.raises(ValueError, match="2 dim"):
        _call(q, 4, output_gate=True)


@pytest.mark.parametrize("view", ["whole", "wider rows", "middle of a projection"])
def test_gated_queries_that_are_wide_enough(view):
    import torch
    q = {"whole": torch.zeros((3, 4, 128)), "wider rows": torch.zeros((3, 4, 200))[..., :128],
         "middle of a projection": torch.zeros((3, 12, 128))[:, 4:8]}[view]
    with pytest.raises(aigpu.AiGpuError, match="no usable gfx950 device"):
        _call(q, 4, output_gate=True)
