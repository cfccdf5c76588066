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


@pytest.mark.parametrize("nq,nkv,hd,mt,lens,split,unit_heads", [
    (8, 4, 128, 300, [300, 300], 64, 1),           # unpacked tensor-core kernel
    (16, 4, 128, 300, [300, 200], 64, 2),          # packed: a unit is two kv heads
    (40, 2, 128, 300, [300, 300], 64, 1),          # two units per kv head: one of them is enough
    (4, 2, 64, 300, [300, 150], 64, 1),            # CUDA cores
    (8, 2, 128, 9000, [9000], -1, 2),              # balanced schedule, one unit over many CTAs
])
def test_a_decode_that_gives_up_adds_nothing(tqk, cuda, nq, nkv, hd, mt, lens, split, unit_heads):
    """A unit whose splits are never merged -- what a wait that runs out leaves behind, made here by a merge ticket that no
    split can complete -- keeps its sums and positions; the other units get theirs."""
    import torch
    c = Case(tqk, 81 + hd, nq, nkv, hd, mt, lens, device_lens=True)
    a, w = c.args(split), c.wargs()
    ws = torch.zeros(tqk.decode_weights_workspace_size(a) // 4 * 4, dtype=torch.uint8, device="cuda")
    before = c.dw.clone()
    tqk.decode_weights(a, c.wargs(c.dw.clone()), ws)   # leaves plausible scores, maxima and sums in the workspace
    c.dpos.fill_(-5)
    c.dq.copy_(torch.randn(c.dq.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    want = c.dw.clone()
    tqk.decode_weights(a, c.wargs(want), ws)
    c.dpos.fill_(-5)
    # the first ticket of the last item's last unit; 17 tickets a unit
    units = nkv // unit_heads * -(-(nq // nkv) // 16)  # 16 q heads at most in a unit of the unpacked kernels
    ws.view(torch.int32)[17 * (len(lens) * units - 1)] = 1000
    tqk.decode_weights(a, w, ws)
    torch.cuda.synchronize()
    got, kept, full = (c.item(t, nkv * mt).reshape(len(lens), nkv, mt).view(np.int32) for t in (c.dw, before, want))
    heads = slice(nkv - unit_heads, nkv)
    full[-1, heads] = kept[-1, heads]
    assert np.array_equal(got, full)
    pos = c.item(c.dpos, nkv * mt).reshape(len(lens), nkv, mt)
    assert (pos[-1, heads] == -5).all()
    assert len(lens) == 1 or pos[0, 0, lens[0] - 1] == 1000


def test_two_threads_on_their_per_thread_streams(tqk, cuda):
    """cudaStreamPerThread is one handle and a stream per thread: each thread has library buffers of its own, also while the
    other's grow."""
    import threading
    import torch
    lens = [[40], [2000], [300], [4000], [70], [900]]
    cases = [[Case(tqk, 91 + 10 * t + i, 8, 2, 128, n[0], n, append=False) for i, n in enumerate(lens)] for t in range(2)]
    want = []
    for cs in cases:
        for c in cs:
            dw = c.dw.clone()
            tqk.decode_weights(c.args(64), c.wargs(dw))
            want.append((c.out.clone(), dw))
            c.out.fill_(float("nan"))
    torch.cuda.synchronize()
    failed = []

    def work(cs):
        try:
            for _ in range(20):
                for c in cs:
                    tqk.decode_weights(c.args(64), c.wargs(c.after), stream=2)
        except Exception as e:  # seen by the test
            failed.append(e)

    for cs in cases:
        for c in cs:
            c.after = torch.full_like(c.dw, float("nan"))
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(cs,)) for cs in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for c, (out, dw) in zip(cases[0] + cases[1], want):
        assert torch.equal(c.out, out) and torch.equal(_bits(c.after), _bits(dw))


def test_a_captured_decode_keeps_its_library_workspace(tqk, cuda):
    """A graph of tqk_decode_q8 with the library's workspace, replayed after larger calls on its stream made that grow."""
    import torch
    small, large = Case(tqk, 101, 8, 2, 128, 700, [700]), Case(tqk, 102, 32, 8, 128, 3000, [3000] * 8, append=False)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    tqk.decode(small.args(64), stream=s)
    s.synchronize()
    want = small.out.clone()
    small.out.fill_(float("nan"))
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        tqk.decode(small.args(64))
        with pytest.raises(tqk.TQKError):  # no growth under capture, which goes on
            tqk.decode(large.args(64))
    tqk.decode_weights(large.args(64), large.wargs(), stream=s)   # grows
    s.synchronize()
    junk = [torch.full((1 << 18,), float("nan"), device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s):
            g.replay()
        tqk.decode_weights(large.args(64), large.wargs(), stream=s)
        s.synchronize()
        assert torch.equal(small.out, want)
        small.out.fill_(float("nan"))
        torch.cuda.synchronize()
    assert all(t.isnan().all() for t in junk)


@pytest.mark.parametrize("nq,nkv,hd,mt,lens,device_lens", [
    (8, 1, 128, 64, [64], False), (7, 1, 128, 65, [65, 64, 1], True),         # 8 rows; the limit and one above it
    (16, 1, 128, 40, [40], False), (15, 1, 128, 66, [64, 33, 0, 17], True),   # 16 rows
    (16, 1, 256, 33, [33], False), (6, 2, 256, 64, [64, 63], False),          # head_dim 256, 16 and 8 rows
    (12, 3, 128, 64, [17, 16, 15], False), (2, 2, 128, 64, [1, 2], False),
    (32, 2, 128, 50, [50, 49], False), (34, 2, 128, 50, [50, 49], False),     # one slice of 16; two slices: not fused
    (16, 4, 128, 64, [64, 64], False), (16, 4, 128, 65, [65, 65], False),     # packed
])
@pytest.mark.parametrize("append", [True, False])
def test_short_caches_add_their_weights_in_the_decode(tqk, cuda, nq, nkv, hd, mt, lens, device_lens, append):
    """Every tensor-core kernel on both sides of the length up to which it adds the weights itself."""
    import torch
    c = Case(tqk, nq * 100 + mt, nq, nkv, hd, mt, lens, append, device_lens, pad=3)
    after = c.dw.clone()
    tqk.decode_weights(c.args(), c.wargs(after))
    torch.cuda.synchronize()
    c.check(after)
    tqk.decode_weights(c.args(), c.wargs())
    assert torch.equal(_bits(c.dw), _bits(after)) and tqk.device_status() == 0


@pytest.mark.parametrize("own_workspace", [False, True])
def test_two_threads_on_one_stream(tqk, cuda, own_workspace):
    """Calls of two host threads on one stream and one workspace: neither's decode comes between the other's decode and its
    weight pass, and neither's growth takes the buffer that the other launches with."""
    import threading
    import torch
    cases = [[Case(tqk, 121 + 10 * t + i, 8, 2, 128, n, [n], append=False) for i, n in enumerate((3000, 200, 800, 5000))]
             for t in range(2)]
    every = cases[0] + cases[1]
    for c in every:
        c.want = c.dw.clone()
        tqk.decode_weights(c.args(64), c.wargs(c.want))
        c.want_out = c.out.clone()
        c.after = torch.full_like(c.dw, float("nan"))
        c.plain = torch.empty_like(c.out)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    ws = torch.zeros(max(tqk.decode_weights_workspace_size(c.args(64)) for c in every), dtype=torch.uint8,
                     device="cuda") if own_workspace else None
    torch.cuda.synchronize()
    failed = []

    def work(cs):
        try:
            for _ in range(50):
                for c in cs:
                    tqk.decode_weights(c.args(64), c.wargs(c.after), ws, stream=s)
                    c.out, keep = c.plain, c.out
                    tqk.decode(c.args(64), ws, stream=s)
                    c.out = keep
        except Exception as e:  # seen by the test
            failed.append(e)

    threads = [threading.Thread(target=work, args=(cs,)) for cs in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for c in every:
        assert torch.equal(_bits(c.after), _bits(c.want)) and torch.equal(c.out, c.want_out)
        assert (c.plain - c.want_out).abs().max() < 1e-5


def test_a_capture_elsewhere_does_not_matter(tqk, cuda):
    """While a stream that does not follow the default stream is captured, a call with the library's workspace on another
    stream goes ahead, growth included, and the capture goes on."""
    import torch
    c = Case(tqk, 141, 8, 2, 128, 700, [700], append=False)
    want = c.dw.clone()
    tqk.decode_weights(c.args(64), c.wargs(want))
    after = torch.full_like(c.dw, float("nan"))
    torch.cuda.synchronize()
    s, other, g, x = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s, capture_error_mode="relaxed"):
        x.add_(1)
        tqk.decode_weights(c.args(64), c.wargs(after), stream=other)
        x.add_(1)
    torch.cuda.synchronize()
    assert torch.equal(_bits(after), _bits(want))
    g.replay()
    torch.cuda.synchronize()
    assert x.item() == 2
