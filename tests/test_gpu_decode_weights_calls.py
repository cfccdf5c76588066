"""tqk_decode_q8_weights as a decoding loop calls it: in place, one call after the other, on short and long caches, from
several host threads, and after a call that did not finish."""
import numpy as np
import pytest

from test_gpu_decode_weights import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tqk(cuda):
    from tailorquantkernel_b200 import tqk as t
    return t


def _bits(t):
    import torch
    return t.view(torch.int32)


@pytest.mark.parametrize("nq,nkv,hd,mt,lens,device_lens,pad,split", [
    (8, 2, 128, 131, [131, 131, 131], False, 1, 0),                    # packed; sums of neighbours share lines
    (8, 2, 128, 1000, [999, 130, 65, 800, 31], True, 3, -1),           # balanced schedule
    (7, 1, 128, 203, [203, 150, 97], False, 5, 0),                     # unpacked, odd strides
    (6, 3, 64, 97, [97, 96], False, 7, 0),                             # CUDA cores
])
def test_calls_back_to_back_add_to_each_other(tqk, cuda, nq, nkv, hd, mt, lens, device_lens, pad, split):
    """50 calls in place with nothing between them: the bits of 50 calls with a synchronisation after each."""
    import torch
    sums = []
    for wait in (True, False):
        c = Case(tqk, mt, nq, nkv, hd, mt, lens, append=False, device_lens=device_lens, pad=pad)
        a, w = c.args(split), c.wargs()
        torch.cuda.synchronize()
        for _ in range(50):
            tqk.decode_weights(a, w)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        sums.append(c.dw)
    assert torch.equal(_bits(sums[0]), _bits(sums[1]))
    got = c.item(sums[1], nkv * mt).reshape(len(lens), nkv, mt)
    for i, n in enumerate(lens):  # every call added weights that sum to the group's q heads; each addition rounds once
        added = (got[i, :, :n].astype(np.float64) - c.weight[i, :, :n]).sum(-1)
        assert np.abs(added - 50 * nq / nkv).max() < 50 * nq / nkv * 1e-5 + 50 * n * 2.0 ** -24 * got[i, :, :n].max()
