"""tqk_evict_q8 as a decoding loop calls it: empty and short caches, sums kept beside lengths on the device."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tqk(cuda):
    from tailorquantkernel_b200 import tqk as t
    return t


@pytest.mark.parametrize("in_place", [True, False])
def test_lengths_above_a_max_len_of_zero_are_reported(tqk, cuda, in_place):
    """max_len 0 is a bound like any other: a length above it is clamped and reported, and nothing is written."""
    import torch
    k = torch.randint(0, 256, (2, 1, 50, 36), dtype=torch.uint8, device="cuda")
    w = torch.rand((2, 1, 50), device="cuda")
    k0, w0 = k.clone(), w.clone()
    for values, status in (([0, 0], "OK"), ([7, 0], "EDEVLEN")):
        lens = torch.tensor(values, dtype=torch.int32, device="cuda")
        out = lens if in_place else torch.full_like(lens, -1)
        tqk.evict(tqk.evict_args(k, k, 1, 32, 50, 10, weight=w, n_items=2, item_stride_blocks=50, stat_item_stride=50, lens=lens,
                                 max_len=0, lens_out=out))
        assert tqk.tqk_device_error_status(tqk.device_status(clear=True)) == getattr(tqk, status)
        assert out.tolist() == [0, 0]
    out = torch.full((2,), -1, dtype=torch.int32, device="cuda")
    tqk.evict(tqk.evict_args(k, k, 1, 32, 50, 10, weight=w, n_items=2, item_stride_blocks=50, stat_item_stride=50, lens_out=out))
    assert out.tolist() == [0, 0] and torch.equal(k, k0) and torch.equal(w, w0) and tqk.device_status() == 0
