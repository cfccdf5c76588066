"""tqk_process_logits against a plain implementation that rounds every step to fp32 as the operator defines it: the
outputs are compared bit for bit (NaN with NaN)."""
import numpy as np
import pytest

from _cache_ops import logits_ref, pack_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tqk(cuda):
    from tailorquantkernel_b200 import tqk as t
    return t


def _packed(rng, rows, lo, hi, vocab, wild):
    """Packed lists of token ids with their offsets; `wild` adds ids outside the vocabulary."""
    lens = rng.integers(lo, hi + 1, rows)
    lens[0], lens[-1] = hi, lo
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    ids = (rng.random(off[-1]) ** 3 * vocab).astype(np.int32)  # repeats many
    if wild and ids.size:
        ids[::7] = rng.choice([-1, vocab, vocab + 5, -2 ** 31, 2 ** 31 - 1], ids[::7].shape)
    return ids, off


CASES = [  # rows, vocab, history, biases, allowed share, penalties (repetition, frequency, presence), row padding
    (1, 1, (3, 3), (2, 2), 1.0, (1, 1, 1), 0),
    (2, 31, (0, 40), (0, 9), 0.5, (1, 1, 1), 1),
    (3, 33, (0, 5), None, 0.1, (1, 0, 0), 31),
    (1, 127, (500, 500), (64, 64), None, (0, 1, 0), 0),
    (5, 128, (0, 300), (0, 30), 0.5, (0, 0, 1), 4),
    (4, 2048, None, (0, 7), 0.3, None, 0),
    (4, 2050, (1, 2000), None, None, (1, 1, 1), 2),       # rows of 8-byte alignment
    (7, 32003, (0, 2049), (0, 11), 0.02, (1, 1, 1), 0),   # odd rows
    (3, 131072, (0, 9000), (5, 50), 0.9, (1, 1, 1), 0),   # a whole piece per CTA
    (2, 131077, (100, 100), (3, 3), 0.9, (1, 1, 1), 3),   # and some more
    (2, 300001, (0, 5000), (0, 40), 0.5, (1, 1, 1), 7),   # several pieces, unaligned
    (2, 299008, (0, 5000), (0, 40), 0.5, (1, 1, 1), 0),   # several pieces, aligned
    (3, 50257, None, None, 0.5, None, 0),
    (3, 50256, None, None, None, None, 0),
]


@pytest.mark.parametrize("mode", ["out", "in place", "choice"])
@pytest.mark.parametrize("rows,vocab,history,biases,share,penal,pad", CASES)
def test_against_the_definition(tqk, cuda, rows, vocab, history, biases, share, penal, pad, mode):
    import torch
    rng = np.random.default_rng(vocab + rows)
    x = rng.standard_normal((rows, vocab), dtype=np.float32) * 3
    special = np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-40, 3e38], np.float32)
    if vocab > 30 and share is not None:  # odd values, also in masked places
        at = rng.integers(0, vocab, 40)
        x[:, at] = special[rng.integers(0, len(special) - (rows == 1), (rows, 40))]
    kw, want_kw = {}, [dict() for _ in range(rows)]

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()

    if history:
        ids, off = _packed(rng, rows, *history, vocab, wild=vocab > 1)
        prompts = rng.integers(-1, history[1] + 2, rows).astype(np.int32)  # some beyond the history
        kw.update(tokens=dev(ids) if ids.size else dev(np.zeros(1, np.int32)), n_tokens=ids.size, token_offsets=dev(off),
                  prompt_lens=dev(prompts))
        for name, on in zip(("repetition", "frequency", "presence"), penal):
            if on:
                val = (rng.random(rows, dtype=np.float32) + (0.7 if name == "repetition" else -0.3))
                kw[name] = dev(val)
                for r in range(rows):
                    want_kw[r][name] = val[r]
        for r in range(rows):
            want_kw[r].update(tokens=ids[off[r]:off[r + 1]], prompt=int(prompts[r]))
    if biases:
        ids, off = _packed(rng, rows, *biases, min(vocab, 50), wild=vocab > 1)  # repeated tokens
        val = rng.standard_normal(ids.size, dtype=np.float32) * 5
        kw.update(bias_tokens=dev(ids) if ids.size else dev(np.zeros(1, np.int32)),
                  bias_values=dev(val) if ids.size else dev(np.zeros(1, np.float32)), n_bias=ids.size, bias_offsets=dev(off))
        for r in range(rows):
            want_kw[r]["bias"] = list(zip(ids[off[r]:off[r + 1]].tolist(), val[off[r]:off[r + 1]]))
    if share is not None:
        allowed = rng.random((rows, vocab)) < share
        if rows > 2:
            allowed[1] = False  # a grammar that leaves nothing
        kw["mask"] = dev(pack_bits(allowed))
        for r in range(rows):
            want_kw[r]["allowed"] = allowed[r]
    buf = torch.full((rows, vocab + pad), 7.0, device="cuda")
    logits = buf[:, :vocab]
    logits.copy_(torch.from_numpy(x))
    obuf = buf if mode == "in place" else torch.full((rows, vocab + pad), 7.0, device="cuda")
    choice = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    tqk.process_logits(tqk.logits_args(logits, out=None if mode == "choice" else obuf[:, :vocab], choice=choice, **kw))
    torch.cuda.synchronize()
    got = obuf.cpu().numpy()
    assert (got[:, vocab:] == 7.0).all()
    for r in range(rows):
        ref, best = logits_ref(x[r], **want_kw[r])
        if mode == "choice":
            assert (got[r] == 7.0).all()
        else:
            nan = np.isnan(ref)
            assert np.array_equal(np.isnan(got[r, :vocab]), nan)
            assert np.array_equal(got[r, :vocab][~nan].view(np.uint32), ref[~nan].view(np.uint32))
        assert choice[r].item() == best
    if mode != "in place":
        assert np.array_equal(logits.cpu().numpy().view(np.uint32), x.view(np.uint32))
    assert tqk.device_status() == 0


MANY_ROWS = [  # few CTAs per row
    (160, 20001, (0, 12000), (0, 11), 0.5, (1, 1, 1), 0),   # 2, in one or two rounds by the history
    (600, 1001, (0, 300), (0, 5), 0.9, (1, 1, 1), 3),       # 1 with a part of a chunk
    (300, 8193, (0, 9000), None, 0.5, (1, 1, 0), 0),        # 1 with a block more than a chunk
    (76, 140001, (0, 9500), (0, 30), 0.5, (1, 1, 1), 0),    # 8 with more than 16384 tokens each
    (75, 140004, (0, 9500), (0, 30), 0.5, (0, 1, 1), 0),
]


@pytest.mark.parametrize("mode", ["out", "in place", "choice"])
@pytest.mark.parametrize("rows,vocab,history,biases,share,penal,pad", MANY_ROWS)
def test_many_rows(tqk, cuda, rows, vocab, history, biases, share, penal, pad, mode):
    test_against_the_definition(tqk, cuda, rows, vocab, history, biases, share, penal, pad, mode)


def test_ties_go_to_the_lowest_token(tqk, cuda):
    import torch
    for vocab in (100, 40000, 140001):
        x = torch.zeros((3, vocab), device="cuda")
        x[0, [5, vocab // 2, vocab - 1]] = 2.0
        x[1, vocab - 1] = 2.0
        choice = torch.empty(3, dtype=torch.int32, device="cuda")
        tqk.process_logits(tqk.logits_args(x, choice=choice))
        assert choice.tolist() == [5, vocab - 1, 0]


def test_mask_rows(tqk, cuda):
    """Rows share mask rows, go without one (-1), and an index out of range allows nothing and is reported."""
    import torch
    vocab = 5000
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((5, vocab), dtype=np.float32)).cuda()
    allowed = rng.random((2, vocab)) < 0.5
    out, choice = torch.empty_like(x), torch.empty(5, dtype=torch.int32, device="cuda")
    mask = torch.from_numpy(pack_bits(allowed)).cuda()
    rows = torch.tensor([1, -1, 0, 1, -1], dtype=torch.int32, device="cuda")
    tqk.process_logits(tqk.logits_args(x, out=out, choice=choice, mask=mask, mask_rows=rows))
    for r, m in enumerate(rows.tolist()):
        ref, best = logits_ref(x[r].cpu().numpy(), allowed=allowed[m] if m >= 0 else None)
        assert np.array_equal(out[r].cpu().numpy(), ref) and choice[r].item() == best
    assert tqk.device_status() == 0
    for bad in (2, -2):
        rows[3] = bad
        tqk.process_logits(tqk.logits_args(x, out=out, choice=choice, mask=mask, mask_rows=rows))
        assert choice[3].item() == -1 and torch.isinf(out[3]).all() and choice[1].item() == int(x[1].argmax())
        assert tqk.tqk_device_error_status(tqk.device_status(clear=True)) == tqk.EDEVLEN


def test_bad_offsets_are_clamped_and_reported(tqk, cuda):
    import torch
    vocab = 1000
    x = torch.zeros((3, vocab), device="cuda")
    tokens = torch.arange(10, dtype=torch.int32, device="cuda")
    off = torch.tensor([-5, 4, 2, 100], dtype=torch.int32, device="cuda")  # before, falling, behind
    freq = torch.ones(3, device="cuda")
    out = torch.empty_like(x)
    tqk.process_logits(tqk.logits_args(x, out=out, tokens=tokens, token_offsets=off, frequency=freq))
    assert tqk.tqk_device_error_status(tqk.device_status(clear=True)) == tqk.EDEVLEN
    assert out[0].nonzero()[:, 0].tolist() == [0, 1, 2, 3]
    assert out[1].nonzero().numel() == 0
    assert out[2].nonzero()[:, 0].tolist() == list(range(2, 10))


def test_captured_with_changing_lists(tqk, cuda):
    """A captured call replays on whatever the lists and offsets then hold; two graphs side by side."""
    import torch
    vocab, rows, cap = 20000, 2, 64
    rng = np.random.default_rng(2)
    runs = []
    for i in range(2):
        x = torch.from_numpy(rng.standard_normal((rows, vocab), dtype=np.float32)).cuda()
        out, choice = torch.empty_like(x), torch.empty(rows, dtype=torch.int32, device="cuda")
        tokens, off = torch.zeros(cap, dtype=torch.int32, device="cuda"), torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
        rep = torch.full((rows,), 1.5, device="cuda")
        a = tqk.logits_args(x, out=out, choice=choice, tokens=tokens, token_offsets=off, repetition=rep)
        tqk.process_logits(a)  # sets the kernel up before the capture
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            tqk.process_logits(a)
        runs.append((x, out, choice, tokens, off, s, g, rep))
    for step in range(4):
        lists = []
        for x, out, choice, tokens, off, s, g, _ in runs:
            ids = x.topk(step + 1).indices.to(torch.int32)  # the best tokens are penalised
            tokens[:rows * (step + 1)] = ids.flatten()
            off.copy_(torch.arange(rows + 1, dtype=torch.int32) * (step + 1))
            lists.append(ids.cpu().numpy())
        torch.cuda.synchronize()
        for *_, s, g, _ in runs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (x, out, choice, *_), ids in zip(runs, lists):
            for r in range(rows):
                ref, best = logits_ref(x[r].cpu().numpy(), tokens=ids[r], repetition=1.5)
                assert np.array_equal(out[r].cpu().numpy(), ref) and choice[r].item() == best


@pytest.mark.parametrize("vocab", [9000, 70000, 131072, 300001])
def test_every_token_in_the_history(tqk, cuda, vocab):
    """More marked tokens than a warp lists at a time, and a hot token whose count passes 16 bits."""
    import torch
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((2, vocab), dtype=np.float32)
    hot = np.full(70000, 7, np.int32)
    lists = [rng.permutation(vocab).astype(np.int32), np.concatenate([hot, np.arange(0, vocab, 3, dtype=np.int32)])]
    off = np.concatenate([[0], np.cumsum([len(v) for v in lists])]).astype(np.int32)
    prompts = np.array([vocab // 2, 11], np.int32)
    allowed = rng.random((2, vocab)) < 0.7
    bias = [[(5, 1.0), (vocab - 1, 2.0)], [(7, 40000.0), (8, -1.0), (7, 0.5)]]
    dx = torch.from_numpy(x).cuda()
    out, choice = torch.empty_like(dx), torch.empty(2, dtype=torch.int32, device="cuda")

    def dev(a, t=None):
        return torch.from_numpy(np.asarray(a, t)).cuda()

    tqk.process_logits(tqk.logits_args(
        dx, out=out, choice=choice, tokens=dev(np.concatenate(lists)), token_offsets=dev(off), prompt_lens=dev(prompts),
        repetition=dev([1.25, 1.5], np.float32), frequency=dev([0.25, 0.5], np.float32), presence=dev([0.125, 0.75], np.float32),
        bias_tokens=dev([t for b in bias for t, _ in b], np.int32), bias_values=dev([v for b in bias for _, v in b], np.float32),
        bias_offsets=dev([0, 2, 5], np.int32), mask=dev(pack_bits(allowed))))
    for r in range(2):
        ref, best = logits_ref(x[r], tokens=lists[r], prompt=int(prompts[r]), repetition=[1.25, 1.5][r],
                               frequency=[0.25, 0.5][r], presence=[0.125, 0.75][r], bias=bias[r], allowed=allowed[r])
        assert np.array_equal(out[r].cpu().numpy().view(np.uint32), ref.view(np.uint32)) and choice[r].item() == best


def test_histories_at_any_address(tqk, cuda):
    """Token arrays that start 0 to 3 words into a 16-byte unit, with lists that start and end anywhere."""
    import torch
    rng = np.random.default_rng(4)
    vocab, rows = 5003, 4
    x = rng.standard_normal((rows, vocab), dtype=np.float32)
    dx, buf = torch.from_numpy(x).cuda(), torch.zeros(12000, dtype=torch.int32, device="cuda")
    for shift in range(4):
        lens = rng.integers(0, 2500, rows)
        off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        ids = rng.integers(0, vocab, off[-1]).astype(np.int32)
        tokens = buf[shift:shift + max(1, len(ids))]
        tokens[:len(ids)] = torch.from_numpy(ids).cuda()
        rep = rng.random(rows, dtype=np.float32) + 1
        out, choice = torch.empty_like(dx), torch.empty(rows, dtype=torch.int32, device="cuda")
        tqk.process_logits(tqk.logits_args(dx, out=out, choice=choice, tokens=tokens, n_tokens=len(ids),
                                           token_offsets=torch.from_numpy(off).cuda(), repetition=torch.from_numpy(rep).cuda()))
        for r in range(rows):
            ref, best = logits_ref(x[r], tokens=ids[off[r]:off[r + 1]], repetition=rep[r])
            assert np.array_equal(out[r].cpu().numpy(), ref) and choice[r].item() == best


def test_one_cta_has_all_the_work(tqk, cuda):
    """A bias list whose tokens all lie in every 16th block of 128 of the vocabulary (one CTA's share, with 16 to a row),
    each twice and far apart: its search of the list outlasts the other CTAs' work many times over."""
    import torch
    rng = np.random.default_rng(8)
    vocab, rows = 131072, 2
    x = rng.standard_normal((rows, vocab), dtype=np.float32)
    own = np.concatenate([np.arange(b, b + 128) for b in range(128, vocab, 16 * 128)]).astype(np.int32)
    ids = np.tile(np.concatenate([own, rng.permutation(own)]), rows)
    val = rng.standard_normal(ids.size, dtype=np.float32)
    val[len(own) + 5] = 100.0  # the first row's choice is among them; the second's may not be
    off = np.array([0, 2 * len(own), 4 * len(own)], np.int32)
    out, choice = torch.empty((rows, vocab), device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
    tqk.process_logits(tqk.logits_args(torch.from_numpy(x).cuda(), out=out, choice=choice, n_bias=ids.size,
                                       bias_tokens=torch.from_numpy(ids).cuda(), bias_values=torch.from_numpy(val).cuda(),
                                       bias_offsets=torch.from_numpy(off).cuda()))
    for r in range(rows):
        ref, best = logits_ref(x[r], bias=list(zip(ids[off[r]:off[r + 1]].tolist(), val[off[r]:off[r + 1]])))
        assert np.array_equal(out[r].cpu().numpy(), ref) and choice[r].item() == best
