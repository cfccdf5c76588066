"""tqk_evict_q8 against a plain implementation: which rows are kept, where they go, and that nothing else is written.
Every output is compared bit for bit (the operator only moves values)."""
import numpy as np
import pytest

from _cache_ops import evict_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tqk(cuda):
    from tailorquantkernel_b200 import tqk as t
    return t


def _weights(rng, kind, shape):
    w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        w = np.floor(w) / 2
    elif kind == "equal":
        w = np.full(shape, 0.25, np.float32)
    elif kind == "odd":  # every kind of value, in a few distinct ones
        odd = np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0, -1.0, 1e-42, -1e-42, 3e38], np.float32)
        w = odd[rng.integers(0, len(odd), shape)]
    return w


def _bits(a):
    return a.view(np.uint32) if a.dtype == np.float32 else a


CASES = [  # nkv, hd, mt, lens, device lens, budget, first, recent, weights, positions
    (2, 128, 40, [40], False, 30, 2, 5, "normal", "rising"),
    (1, 32, 7, [7], False, 1, 0, 0, "normal", None),
    (1, 32, 2, [2], False, 1, 1, 0, "normal", "rising"),
    (3, 64, 200, [200, 199, 198], False, 64, 0, 64, "ties", "mixed"),
    (2, 256, 90, [90], False, 45, 20, 25, "normal", "mixed"),
    (8, 128, 600, [0, 600, 1, 300, 301, 302], True, 300, 4, 50, "ties", "mixed"),
    (2, 128, 4097, [4097], False, 4096, 4, 256, "normal", "mixed"),
    (2, 128, 9000, [9000], False, 100, 4, 32, "normal", "rising"),       # two CTAs per head
    (1, 128, 40000, [40000, 20000], True, 19999, 0, 1000, "ties", "mixed"),
    (2, 32, 70001, [70001], False, 70000, 3, 500, "equal", "mixed"),
    (1, 32, 258048, [258048], False, 1234, 4, 100, "normal", "rising"),  # the longest
    (1, 32, 250001, [250001], False, 249000, 0, 0, "ties", None),
    (2, 128, 140001, [140001], False, 50000, 4, 1000, "normal", "mixed"),
    (1, 64, 258048, [258048], False, 129000, 0, 0, "normal", None),      # as many holes as a CTA can have
    (1, 32, 258048, [258048], False, 60000, 0, 60000, "normal", "rising"),
    (16, 32, 16500, [16500, 16499], False, 9000, 4, 100, "normal", "mixed"),  # more CTAs than SMs hold alone
    (2, 64, 513, [513], False, 200, 0, 0, "odd", None),
    (2, 64, 9001, [9001], False, 4000, 10, 10, "odd", "mixed"),
    (2, 128, 1000, [1000], False, 500, 0, 0, "equal", "mixed"),
    (1, 128, 1000, [1000], False, 500, 100, 400, "normal", "same"),      # positions all equal: all rows protected alike
    (1, 128, 1000, [1000], False, 500, 0, 10, "normal", "extreme"),
    (2, 128, 64, [64, 64], False, 64, 8, 8, "normal", "rising"),         # nothing to evict
]


def _positions(rng, kind, shape):
    if kind is None:
        return None
    pos = np.cumsum(rng.integers(1, 4, shape), -1).astype(np.int32)
    if kind == "mixed":
        half = shape[-1] // 2
        pos[..., :half] = rng.permuted(pos[..., :half], axis=-1)
    elif kind == "same":
        pos[:] = 17
    elif kind == "extreme":
        pos = rng.integers(-2 ** 31, 2 ** 31 - 1, shape).astype(np.int32)
        pos[..., 3], pos[..., 5] = 2 ** 31 - 1, -2 ** 31
    return pos


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("nkv,hd,mt,lens,device_lens,budget,first,recent,weights,positions", CASES)
def test_evict(tqk, cuda, nkv, hd, mt, lens, device_lens, budget, first, recent, weights, positions, in_place):
    import torch
    rng = np.random.default_rng(mt + budget)
    items, row, pad = len(lens), hd // 32 * 36, 3
    shape = (items, nkv, mt)
    k, v = (rng.integers(0, 256, (*shape, row), dtype=np.uint8) for _ in range(2))
    w, pos = _weights(rng, weights, shape), _positions(rng, positions, shape)

    def strided(a):  # items `pad` elements apart beyond their own
        flat = np.full((items, nkv * mt + pad), 9, a.dtype)
        flat[:, :nkv * mt] = a.reshape(items, -1)
        return torch.from_numpy(flat).cuda()

    def host(t):
        a = t.cpu().numpy()
        assert (a[:, nkv * mt:] == 9).all()
        return a[:, :nkv * mt].reshape(shape)

    dk, dv, dw = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), strided(w)
    dp = strided(pos) if pos is not None else None
    dw2 = dw if in_place else strided(np.full(shape, 5.5, np.float32))
    dp2 = dp if in_place or dp is None else strided(np.full(shape, 55, np.int32))
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    lens_out = dl if in_place else torch.full_like(dl, -1)
    step = lens[1] - lens[0] if items > 1 else 0
    how = dict(lens=dl, max_len=max(lens)) if device_lens else dict(len0=lens[0], len_step=step)
    tqk.evict(tqk.evict_args(dk, dv, nkv, hd, mt, budget, weight=dw, weight_out=dw2, position=dp, position_out=dp2,
                             n_items=items, item_stride_blocks=nkv * mt * (hd // 32), stat_item_stride=nkv * mt + pad,
                             n_first=first, n_recent=recent, lens_out=lens_out, **how))
    torch.cuda.synchronize()

    k_ref, v_ref = k.copy(), v.copy()
    w_ref = w.copy() if in_place else np.full(shape, 5.5, np.float32)
    p_ref = None if pos is None else pos.copy() if in_place else np.full(shape, 55, np.int32)
    for i, n in enumerate(lens):
        for h in range(nkv):
            _, dst, src = evict_ref(w[i, h], None if pos is None else pos[i, h], n, budget, first, recent)
            k_ref[i, h, dst], v_ref[i, h, dst] = k[i, h, src], v[i, h, src]
            m = min(n, budget)
            for ref, old in ((w_ref, w), (p_ref, pos)):
                if ref is not None:
                    ref[i, h, :m] = old[i, h, :m]
                    ref[i, h, dst] = old[i, h, src]
    assert np.array_equal(dk.cpu().numpy(), k_ref) and np.array_equal(dv.cpu().numpy(), v_ref)
    assert np.array_equal(_bits(host(dw2)), _bits(w_ref))
    if pos is not None:
        assert np.array_equal(host(dp2), p_ref)
    if not in_place:
        assert np.array_equal(_bits(host(dw)), _bits(w)) and (pos is None or np.array_equal(host(dp), pos))
    assert lens_out.tolist() == [min(n, budget) for n in lens]
    assert tqk.device_status() == 0


FEW_HEADS = [  # out of place, several clusters share a head's moves
    (1, 256, 20001, [20001], False, 10000, 4, 100, "normal", "mixed"),
    (2, 128, 30000, [30000, 17000], True, 12345, 4, 100, "ties", "mixed"),      # the second: fewer moves
    (1, 128, 30000, [0, 30000, 15000, 15001], True, 15000, 0, 0, "odd", None),  # nothing, all, nothing, one row
    (4, 64, 9000, [9000], False, 4500, 4, 100, "equal", "rising"),
    (3, 32, 120000, [120000], False, 4096, 4, 100, "normal", "rising"),
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("nkv,hd,mt,lens,device_lens,budget,first,recent,weights,positions", FEW_HEADS)
def test_few_heads(tqk, cuda, nkv, hd, mt, lens, device_lens, budget, first, recent, weights, positions, in_place):
    test_evict(tqk, cuda, nkv, hd, mt, lens, device_lens, budget, first, recent, weights, positions, in_place)


def test_lengths_from_the_device_are_clamped(tqk, cuda):
    import torch
    nkv, hd, mt = 1, 32, 50
    k = torch.randint(0, 256, (2, nkv, mt, 36), dtype=torch.uint8, device="cuda")
    w = torch.rand((2, nkv, mt), device="cuda")
    k0, w0 = k.clone(), w.clone()
    lens = torch.tensor([60, -1], dtype=torch.int32, device="cuda")
    tqk.evict(tqk.evict_args(k, k.clone(), nkv, hd, mt, 10, weight=w, n_items=2, item_stride_blocks=nkv * mt,
                             stat_item_stride=nkv * mt, lens=lens, max_len=40, lens_out=lens))
    assert tqk.tqk_device_error_status(tqk.device_status(clear=True)) == tqk.EDEVLEN
    assert lens.tolist() == [10, 0]
    assert torch.equal(k[1], k0[1]) and torch.equal(k[0, :, 10:], k0[0, :, 10:])
    keep, dst, src = evict_ref(w0[0, 0].cpu().numpy(), None, 40, 10, 0, 0)
    ref = k0[0, 0].clone()
    ref[torch.from_numpy(dst).cuda()] = k0[0, 0][torch.from_numpy(src).cuda()]
    assert torch.equal(k[0, 0], ref)


def test_captured_replayed_and_on_two_streams(tqk, cuda):
    """Two captured evictions replayed side by side on restored caches give the eager results each time."""
    import torch
    nkv, hd, mt, budget = 4, 128, 20000, 5000
    runs = []
    for seed in range(2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        k = torch.randint(0, 256, (nkv, mt, 144), dtype=torch.uint8, device="cuda", generator=g)
        v = torch.randint(0, 256, (nkv, mt, 144), dtype=torch.uint8, device="cuda", generator=g)
        w = torch.rand((nkv, mt), device="cuda", generator=g)
        start = [t.clone() for t in (k, v, w)]
        a = tqk.evict_args(k, v, nkv, hd, mt, budget, weight=w, len0=mt)
        tqk.evict(a)
        want = [t.clone() for t in (k, v, w)]
        s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            tqk.evict(a)
        runs.append(((k, v, w), start, want, s, graph))
    for _ in range(3):
        for now, start, *_ in runs:
            for t, x in zip(now, start):
                t.copy_(x)
        torch.cuda.synchronize()
        for *_, s, graph in runs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for now, _, want, *_ in runs:
            assert all(torch.equal(t, x) for t, x in zip(now, want))
