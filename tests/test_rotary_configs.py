"""``Rotary.of`` and the attention block's rotary, of rope configs whose rotated part of a head is odd: no whole number of
pairs, refused as the block's own rotation refuses it (on the CPU)."""
import pytest
import torch

from lagunalab_amd.attention import Attention, rope_frequencies
from lagunalab_amd.rotary import Rotary


def rope(dims):
    return {"rope_theta": 1e4, "partial_rotary_factor": dims / 128}


def block(dims, hq=2, kv=1, C=8):
    w = lambda *s: torch.zeros(s)  # noqa: E731
    return Attention(w(hq * 128, C), w(kv * 128, C), w(kv * 128, C), w(C, hq * 128), w(hq, C), w(128), w(128), hq, kv,
                     rope(dims))


@pytest.mark.parametrize("dims", [1, 11, 127])
def test_odd_parts_of_a_head(dims):
    assert rope_frequencies(128, rope(dims))[1] == dims
    with pytest.raises(ValueError, match=f"{dims} rotated dims"):
        Rotary.of(rope(dims), "cpu")
    with pytest.raises(ValueError, match=f"{dims} rotated dims"):
        block(dims)


@pytest.mark.parametrize("dims", [0, 2, 6, 64, 128])
def test_even_parts_of_a_head(dims):
    inv_freq, _, mscale = rope_frequencies(128, rope(dims))
    for r in (Rotary.of(rope(dims), "cpu"), block(dims).rotary):
        assert (r.dims, r.mscale, r.interleaved) == (dims, mscale, False) and torch.equal(r.inv_freq, inv_freq)
