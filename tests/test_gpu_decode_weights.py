"""tqk_decode_q8_weights: the decode's output and the running sums of attention weights, against float64 attention over
the same quantised values (tests/_cache_ops.py), at the bounds derived there; the appended rows bit for bit
against tqk_decode_q8's."""
import numpy as np
import pytest

import oracle
from _cache_ops import U, attend64, scales, values, weight_bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tqk(cuda):
    from tailorquantkernel_b200 import tqk as t
    return t


class Case:
    """Caches, queries, sums and a call's argument structs, item strides padded by `pad` elements."""

    def __init__(self, tqk, seed, nq, nkv, hd, mt, lens, append=True, device_lens=False, pad=0, max_len=None):
        import torch
        rng = np.random.default_rng(seed)
        self.tqk, self.nq, self.nkv, self.hd, self.mt, self.lens, self.append = tqk, nq, nkv, hd, mt, list(lens), append
        items, nb = len(lens), hd // 32
        self.items, self.nb = items, nb
        port = oracle.Oracle("port")

        def normal(*shape):
            return rng.standard_normal(shape, dtype=np.float32)

        self.k, self.v = port.quantize_rows(normal(items, nkv, mt, hd)), port.quantize_rows(normal(items, nkv, mt, hd))
        self.q, self.kn, self.vn = normal(items, nq, hd), normal(items, nkv, hd), normal(items, nkv, hd)
        self.weight = rng.random((items, nkv, mt), dtype=np.float32)
        for i, n in enumerate(lens):  # what nothing may read: rows behind the end, and the appended slot
            end = n - 1 if append and n else n
            self.k[i, :, end:], self.v[i, :, end:] = 0xFF, 0xFF  # NaN scales
            self.weight[i, :, end:] = np.nan
        self.qq = port.quantize_rows(self.q)
        pad_blocks = 4 * ((pad + 3) // 4)  # keeps rows 16-byte aligned

        def strided(a, n, extra):
            """Items of `a` n elements apart plus `extra`, as one flat device tensor."""
            flat = np.full((items, n + extra), 77, a.dtype)
            flat[:, :n] = a.reshape(items, n)
            return torch.from_numpy(flat).cuda()

        row = nb * 36
        self.dk, self.dv = (strided(p, nkv * mt * row, pad_blocks * 36) for p in (self.k, self.v))
        self.dw = strided(self.weight, nkv * mt, pad)
        self.dpos = strided(np.full((items, nkv, mt), -5, np.int32), nkv * mt, pad)
        self.dq, self.dkn, self.dvn = (torch.from_numpy(a).cuda() for a in (self.q, self.kn, self.vn))
        self.dlens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.out = torch.full((items, nq * hd), float("nan"), device="cuda")
        self.new_pos = torch.arange(1000, 1000 + items, dtype=torch.int32, device="cuda")
        self.pad, self.pad_blocks, self.device_lens = pad, pad_blocks, device_lens
        self.max_len = max(self.lens) if max_len is None else max_len

    def args(self, split=0, **kw):
        new = dict(k_new=self.dkn, v_new=self.dvn, kv_new_item_stride=self.nkv * self.hd) if self.append else {}
        if self.device_lens:
            lens = dict(lens=self.dlens, max_len=self.max_len)
        else:
            step = self.lens[1] - self.lens[0] if self.items > 1 else 0
            assert all(n == self.lens[0] + i * step for i, n in enumerate(self.lens))
            lens = dict(len0=self.lens[0], len_step=step)
        return self.tqk.decode_args(self.dk, self.dv, self.nq, self.nkv, self.hd, self.mt, self.dq, self.out,
                                    n_items=self.items, item_stride_blocks=self.nkv * self.mt * self.nb + self.pad_blocks,
                                    q_item_stride=self.nq * self.hd, out_item_stride=self.nq * self.hd,
                                    split_tokens=split, **lens, **new, **kw)

    def wargs(self, out=None, **kw):
        if self.append and "position" not in kw:
            kw.update(position=self.dpos, new_pos=self.new_pos)
        return self.tqk.weights_args(self.dw, out, item_stride=self.nkv * self.mt + self.pad, **kw)

    def item(self, t, n):
        """The host copy of a strided device tensor, without the padding."""
        a = t.cpu().numpy()
        assert (a[:, n:] == np.array(77, a.dtype)).all(), "padding between items was written"
        return a[:, :n]

    def check(self, dw_out=None, big_out=None):
        """Output, sums, appended rows and positions against float64 and the reference quantiser."""
        items, nkv, mt, nb = self.items, self.nkv, self.mt, self.nb
        row = nb * 36
        k, v = (self.item(t, nkv * mt * row).reshape(items, nkv, mt, row) for t in (self.dk, self.dv))
        k_ref, v_ref = self.k.copy(), self.v.copy()
        if self.append:
            port = oracle.Oracle("port")
            pos = self.item(self.dpos, nkv * mt).reshape(items, nkv, mt)
            pos_ref = np.full_like(pos, -5)
            for i, n in enumerate(self.lens):
                if n:
                    k_ref[i, :, n - 1] = port.quantize_rows(self.kn[i])
                    v_ref[i, :, n - 1] = port.quantize_rows(self.vn[i])
                    pos_ref[i, :, n - 1] = 1000 + i
            assert np.array_equal(pos, pos_ref)
        assert np.array_equal(k, k_ref) and np.array_equal(v, v_ref)
        out_ref, w_ref, big = attend64(self.qq, k_ref, v_ref, self.lens)
        n = max(self.lens)
        rel = weight_bound(nb, big, n)
        got = (self.dw if dw_out is None else dw_out)
        got = self.item(got, nkv * mt).reshape(items, nkv, mt).astype(np.float64)
        for i, m in enumerate(self.lens):
            end = m - 1 if self.append and m else m
            base = self.weight[i].astype(np.float64)
            base[:, end:m] = 0.0
            total = base[:, :m] + w_ref[i, :, :m]
            # the sum over g heads rounds g times, the addition once
            bound = w_ref[i, :, :m] * (rel + self.nq // nkv * U) + 2 * U * total
            assert (np.abs(got[i, :, :m] - total) <= bound).all(), \
                f"item {i}: worst {np.max(np.abs(got[i, :, :m] - total) / bound):.2f} of the bound"
            assert np.isnan(got[i, :, m:]).all(), "sums behind the end were written"
        out = self.out.cpu().numpy().reshape(items, self.nq, self.hd)
        for i, m in enumerate(self.lens):
            if m == 0:
                assert (out[i] == 0).all()
                continue
            # each weight's error, P's split into two fp16 (2^-22 of the largest p * scale), a sum of n products in
            # chains (n / 64 steps of a 16-term product, each step truncating: two half steps) and the merges
            vmax = np.abs(values(v_ref[i, :, :m])).max()
            bound = vmax * (rel + 2.0 ** -21 + 2 * (m / 64 + 64) * U)
            assert np.abs(out[i] - out_ref[i]).max() <= bound
        return out


CASES = [  # nq, nkv, hd, mt, lens, append, device lens, pad, split
    (14, 2, 64, 40, [1], True, False, 0, 0),
    (1, 1, 32, 9, [3], False, False, 0, 0),
    (6, 2, 32, 130, [128, 65, 2], True, False, 3, 0),
    (5, 1, 64, 700, [699], True, False, 0, 64),
    (16, 16, 64, 300, [300, 299], False, False, 5, 0),
    (24, 2, 64, 200, [200], True, False, 0, 0),             # 12 q heads per kv head: two slices
    (12, 3, 128, 129, [129], True, False, 0, 0),            # 4 per kv head, odd kv heads: unpacked
    (32, 8, 128, 80, [17, 16, 15], True, False, 2, 0),      # packed
    (32, 8, 128, 1, [1], True, False, 0, 0),
    (8, 2, 128, 4097, [4097, 4097], True, False, 0, 0),     # packed, cluster merge
    (8, 2, 128, 3000, [3000], False, False, 0, 64),         # packed, two merge levels
    (8, 2, 128, 600, [0, 600, 1, 64, 63, 65], False, True, 1, 0),
    (8, 2, 128, 600, [599, 2, 1, 64, 63, 65], True, True, 1, -1),   # balanced schedule
    (8, 2, 128, 600, [0, 600, 0], False, True, 0, -1),
    (8, 1, 128, 1000, [1000, 513], True, False, 0, 0),      # 8 per kv head
    (7, 1, 128, 260, [260], True, False, 0, 64),
    (40, 2, 128, 90, [90, 80, 70], False, False, 4, 0),     # 20 per kv head: slices of 16 and 4
    (16, 1, 256, 150, [150], True, False, 0, 0),
    (3, 3, 256, 77, [76, 77], False, False, 1, 0),
    (8, 8, 128, 300, [0], False, False, 0, 0),
]


@pytest.mark.parametrize("nq,nkv,hd,mt,lens,append,device_lens,pad,split", CASES)
def test_output_and_sums(tqk, cuda, nq, nkv, hd, mt, lens, append, device_lens, pad, split):
    import torch
    c = Case(tqk, nq * 1000 + mt, nq, nkv, hd, mt, lens, append, device_lens, pad)
    # out of place first: the sums before the call stay
    before = c.dw.clone()
    after = c.dw.clone()
    tqk.decode_weights(c.args(split), c.wargs(after))
    torch.cuda.synchronize()
    out = c.check(after)
    assert torch.equal(c.dw.view(torch.int32), before.view(torch.int32))
    # in place: the same bits (the append writes the same row again)
    c.out.fill_(float("nan"))
    tqk.decode_weights(c.args(split), c.wargs())
    torch.cuda.synchronize()
    assert torch.equal(c.dw.view(torch.int32), after.view(torch.int32))
    assert np.array_equal(c.out.cpu().numpy().reshape(out.shape), out)
    assert tqk.device_status() == 0


def test_output_agrees_with_the_plain_decode(tqk, cuda):
    import torch
    c = Case(tqk, 5, 32, 8, 128, 1500, [1500, 1400, 1300])
    tqk.decode_weights(c.args(), c.wargs())
    got = c.out.clone()
    tqk.decode(c.args())
    # both are within the decode's bound of the exact value
    assert (got - c.out).abs().max() < 1e-5


def test_norm_and_rope_are_fused_as_in_the_decode(tqk, cuda):
    """The fused prologue equals tqk_qk_norm_rope before the call, bit for bit."""
    import torch
    rng = np.random.default_rng(3)
    for nq, nkv, hd in ((8, 2, 128), (6, 2, 64), (8, 8, 256)):
        a, b = (Case(tqk, 11, nq, nkv, hd, 200, [200]) for _ in range(2))
        qn, kn = (torch.from_numpy(rng.random(hd, dtype=np.float32) + 0.5).cuda() for _ in range(2))
        cs, sn = (torch.from_numpy(f(rng.random(hd // 2) * 6).astype(np.float32)).cuda() for f in (np.cos, np.sin))
        tqk.decode_weights(a.args(q_norm=qn, k_norm=kn, norm_eps=1e-5, rope_cos=cs, rope_sin=sn), a.wargs())
        tqk.qk_norm_rope(b.dq, b.dkn, 1, nq, nkv, hd, qn, kn, 1e-5, cs, sn)
        tqk.decode_weights(b.args(), b.wargs())
        assert torch.equal(a.out, b.out) and torch.equal(a.dk, b.dk) and torch.equal(a.dw.view(torch.int32), b.dw.view(torch.int32))


def test_sums_accumulate_over_tokens(tqk, cuda):
    """Ten tokens appended one by one: the sums are those of ten separate softmaxes."""
    import torch
    nq, nkv, hd, mt, n0 = 8, 2, 128, 64, 20
    c = Case(tqk, 21, nq, nkv, hd, mt, [n0])
    rng = np.random.default_rng(22)
    port = oracle.Oracle("port")
    total = c.weight.astype(np.float64)
    total[..., n0 - 1:] = 0.0
    bound = 0.0
    for step in range(10):
        n = n0 + step
        q, kn, vn = (rng.standard_normal(s, dtype=np.float32) for s in ((1, nq, hd), (1, nkv, hd), (1, nkv, hd)))
        for t, x in ((c.dq, q), (c.dkn, kn), (c.dvn, vn)):
            t.copy_(torch.from_numpy(x))
        c.lens = [n]
        tqk.decode_weights(c.args(), c.wargs(position=c.dpos, new_pos0=n - 1))
        c.k[0, :, n - 1], c.v[0, :, n - 1] = port.quantize_rows(kn[0]), port.quantize_rows(vn[0])
        _, w, big = attend64(port.quantize_rows(q), c.k, c.v, [n])
        total[..., :n] += w[..., :n]
        bound += weight_bound(4, big, n) * w.max() + 4 * U * total[..., :n].max()
    got = c.dw.cpu().numpy().reshape(nkv, mt)[:, :n]
    assert np.abs(got - total[0, :, :n]).max() <= bound
    assert np.array_equal(c.dpos.cpu().numpy().reshape(nkv, mt)[:, n0 - 1:n], np.tile(np.arange(n0 - 1, n), (nkv, 1)))


def test_nan_and_infinite_scores_follow_the_formula(tqk, cuda):
    """A NaN key inside the length makes its head's weights and output NaN, other heads stay; an infinite V scale does
    not reach the weights."""
    import torch
    for nq, nkv, hd in ((8, 2, 128), (6, 2, 64), (4, 2, 256)):
        c = Case(tqk, 31, nq, nkv, hd, 100, [90], append=False)
        row = hd // 32 * 36
        k = c.dk.view(nkv, 100, row)
        k[0, 40, :4].copy_(torch.tensor([np.nan], dtype=torch.float32).view(torch.uint8))
        v = c.dv.view(nkv, 100, row)
        v[1, 7, :4].copy_(torch.tensor([np.inf], dtype=torch.float32).view(torch.uint8))
        tqk.decode_weights(c.args(), c.wargs())
        w = c.dw.cpu().numpy().reshape(nkv, 100)
        out = c.out.cpu().numpy().reshape(nkv, -1, hd)
        assert np.isnan(w[0, :90]).all() and np.isnan(out[0]).all()
        assert np.isfinite(w[1, :90]).all() and np.isfinite(out[1, :, 32:]).all()


def test_device_lengths_are_clamped_to_max_len(tqk, cuda):
    import torch
    c = Case(tqk, 41, 8, 2, 128, 300, [100, 100], append=False, device_lens=True)
    c.dlens.copy_(torch.tensor([250, -3], dtype=torch.int32))  # the call says max_len 100
    tqk.decode_weights(c.args(), c.wargs())
    assert tqk.tqk_device_error_status(tqk.device_status(clear=True)) == tqk.EDEVLEN
    c.lens = [100, 0]
    assert (c.out[1] == 0).all()
    got = c.item(c.dw, 2 * 300).reshape(2, 2, 300)
    assert np.isnan(got[0, :, 100:]).all() and np.isfinite(got[0, :, :100]).all()
    assert np.array_equal(got[1, :, :100], c.weight[1, :, :100])


def test_caller_workspace_is_shared_with_the_decode(tqk, cuda):
    """One zeroed workspace serves decode and weight calls, with and without splits, in any order."""
    import torch
    small = Case(tqk, 51, 8, 2, 128, 50, [50])
    large = Case(tqk, 52, 8, 2, 128, 3000, [3000])
    need = max(tqk.decode_weights_workspace_size(x.args(sp)) for x in (small, large) for sp in (0, 64))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    tqk.workspace_init(ws)
    for x, sp in ((small, 0), (large, 64), (small, 0), (large, 0), (large, 64)):
        tqk.decode_weights(x.args(sp), x.wargs(x.dw.clone()), ws)
        got = x.out.clone()
        tqk.decode(x.args(sp), ws)
        assert (got - x.out).abs().max() < 1e-5
    with pytest.raises(tqk.TQKError) as e:
        tqk.decode_weights(large.args(64), large.wargs(), ws[:tqk.decode_weights_workspace_size(large.args(64)) - 1])
    assert e.value.status == tqk.EWORKSPACE
    with pytest.raises(tqk.TQKError) as e:
        tqk.decode_weights(small.args(), small.wargs(), ws[1:])
    assert e.value.status in (tqk.EALIGN, tqk.EWORKSPACE)


def test_captured_and_replayed_on_two_streams(tqk, cuda):
    """Two graphs, each with its own workspace, replayed side by side and again after the inputs changed."""
    import torch
    cs = [Case(tqk, 61 + i, 8, 2, 128, 2000, [1990, 1980]) for i in range(2)]
    want = []
    for c in cs:
        before = c.dw.clone()
        tqk.decode_weights(c.args(), c.wargs())
        want.append((c.out.clone(), c.dw.clone()))
        c.dw.copy_(before)
        c.before = before
    graphs, streams, spaces = [], [], []
    for c in cs:
        ws = torch.zeros(tqk.decode_weights_workspace_size(c.args()), dtype=torch.uint8, device="cuda")
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            tqk.decode_weights(c.args(), c.wargs(), ws)
        graphs.append(g), streams.append(s), spaces.append(ws)
    for rep in range(3):
        for c in cs:
            c.dw.copy_(c.before)
            c.out.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, (out, dw) in zip(cs, want):
            assert torch.equal(c.out, out) and torch.equal(c.dw.view(torch.int32), dw.view(torch.int32))


def test_capture_needs_a_workspace(tqk, cuda):
    import torch
    c = Case(tqk, 65, 8, 2, 128, 100, [100])
    tqk.decode_weights(c.args(), c.wargs())
    torch.cuda.synchronize()
    s, g, x = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    with torch.cuda.graph(g, stream=s):
        x.add_(1)
        with pytest.raises(tqk.TQKError) as e:
            tqk.decode_weights(c.args(), c.wargs())
        assert e.value.status == tqk.EWORKSPACE
    g.replay()
    assert x.item() == 1


def test_library_workspace_on_another_stream(tqk, cuda):
    import torch
    c = Case(tqk, 71, 32, 8, 128, 900, [900])
    before = c.dw.clone()
    tqk.decode_weights(c.args(), c.wargs())
    out, dw = c.out.clone(), c.dw.clone()
    c.dw.copy_(before)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    tqk.decode_weights(c.args(), c.wargs(), stream=s)
    s.synchronize()
    assert torch.equal(c.out, out) and torch.equal(c.dw.view(torch.int32), dw.view(torch.int32))
