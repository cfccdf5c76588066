"""The operators as a decoding program uses them: a small decoder whose caches hold a budget of rows per head, token by
token -- project, append and attend with running sums, evict, logits, constraints, the next token.  Every step is
compared with a float64 simulation that keeps each head's rows as a plain list; the simulation takes over the
device's sums for the choice of rows (two nearly equal sums may order either way) and the device's token."""
import numpy as np
import pytest

import oracle
from _cache_ops import U, attend64, evict_ref, logits_ref, pack_bits, values, weight_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nq,nkv,hd,in_graph", [(8, 2, 128, False), (6, 2, 64, False), (8, 2, 128, True)])
def test_decoding_loop(cuda, nq, nkv, hd, in_graph):
    import torch
    from tailorquantkernel_b200 import tqk
    layers, vocab, budget, room, prompt, steps = 2, 1003, 40, 48, 37, 30
    mt, nb, row = budget + (room - budget), hd // 32, hd // 32 * 36
    rng = np.random.default_rng(nq + hd)
    port = oracle.Oracle("port")

    def normal(*shape):
        return rng.standard_normal(shape, dtype=np.float32)

    hidden = nq * hd
    embed, head = normal(vocab, hidden) * 0.3, normal(vocab, hidden) * 0.05
    wq, wk, wv = normal(layers, hidden, nq * hd) * 0.05, normal(layers, hidden, nkv * hd) * 0.05, normal(layers, hidden, nkv * hd) * 0.05
    d_embed, d_head, d_wq, d_wk, d_wv = (torch.from_numpy(a).cuda() for a in (embed, head, wq, wk, wv))

    kp, vp = (port.quantize_rows(normal(layers, nkv, mt, hd)) for _ in range(2))  # a prompt's rows are in the caches
    weight = np.zeros((layers, nkv, mt), np.float32)
    position = np.tile(np.arange(mt, dtype=np.int32), (layers, nkv, 1))
    dk, dv, dw, dp = (torch.from_numpy(a.copy()).cuda() for a in (kp, vp, weight, position))
    lens = torch.full((layers,), prompt, dtype=torch.int32, device="cuda")  # rows in the caches
    lens_next = lens.clone()
    new_pos = torch.zeros(layers, dtype=torch.int32, device="cuda")
    q, k, v = (torch.empty((layers, n), device="cuda") for n in (nq * hd, nkv * hd, nkv * hd))
    attn = torch.empty((layers, nq * hd), device="cuda")
    logits = torch.empty((1, vocab), device="cuda")
    choice = torch.zeros(1, dtype=torch.int32, device="cuda")
    tokens, offsets = torch.zeros(steps + 1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    rep, freq = torch.full((1,), 1.3, device="cuda"), torch.full((1,), 0.2, device="cuda")
    allowed = rng.random((1, vocab)) < 0.5
    out = torch.empty_like(logits)

    a = tqk.decode_args(dk, dv, nq, nkv, hd, mt, q, attn, n_items=layers, item_stride_blocks=nkv * mt * nb, lens=lens_next,
                        max_len=mt, q_item_stride=nq * hd, out_item_stride=nq * hd, k_new=k, v_new=v,
                        kv_new_item_stride=nkv * hd)
    w = tqk.weights_args(dw, item_stride=nkv * mt, position=dp, new_pos=new_pos)
    e = tqk.evict_args(dk, dv, nkv, hd, mt, budget, n_items=layers, item_stride_blocks=nkv * mt * nb, stat_item_stride=nkv * mt,
                       lens=lens_next, max_len=mt, n_first=2, n_recent=8, weight=dw, position=dp, lens_out=lens)
    g = tqk.logits_args(logits, out=out, choice=choice, tokens=tokens, token_offsets=offsets, repetition=rep,
                        frequency=freq, mask=torch.from_numpy(pack_bits(allowed)).cuda())
    ws = torch.zeros(tqk.decode_weights_workspace_size(a), dtype=torch.uint8, device="cuda")

    def step():  # device work only, so that it can be captured
        torch.add(lens, 1, out=lens_next)
        tqk.decode_weights(a, w, ws)
        torch.mm(attn.sum(0, keepdim=True), d_head.T, out=logits)
        tqk.evict(e)
        tqk.process_logits(g)

    graph = None
    if in_graph:
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            torch.mm(attn.sum(0, keepdim=True), d_head.T, out=logits)  # the library's set-up
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        torch.cuda.synchronize()

    sim = [[dict(k=kp[i, h, :prompt].copy(), v=vp[i, h, :prompt].copy(), w=np.zeros(prompt, np.float32),
                 p=np.arange(prompt, dtype=np.int32)) for h in range(nkv)] for i in range(layers)]
    history, token = [3], 3
    tokens[0] = 3
    evicted = 0
    for n in range(steps):
        x = d_embed[token]
        for i in range(layers):
            q[i], k[i], v[i] = x @ d_wq[i], x @ d_wk[i], x @ d_wv[i]
        new_pos.fill_(prompt + n)
        offsets[1] = len(history)
        graph.replay() if graph else step()
        torch.cuda.synchronize()
        kn, vn, qn = (t.cpu().numpy() for t in (k, v, q))
        got_out, got_w, got_p = attn.cpu().numpy(), dw.cpu().numpy(), dp.cpu().numpy()
        got_k, got_v = dk.cpu().numpy(), dv.cpu().numpy()
        for i in range(layers):
            qq = port.quantize_rows(qn[i].reshape(nq, hd))
            for h in range(nkv):
                s = sim[i][h]
                s["k"] = np.concatenate([s["k"], port.quantize_rows(kn[i].reshape(nkv, hd)[h][None])])
                s["v"] = np.concatenate([s["v"], port.quantize_rows(vn[i].reshape(nkv, hd)[h][None])])
                s["p"] = np.append(s["p"], np.int32(prompt + n))
                size, grp = len(s["p"]), nq // nkv
                ref, add, big = attend64(qq[None, h * grp:(h + 1) * grp], s["k"][None, None], s["v"][None, None], [size])
                rel = weight_bound(nb, big, size)
                vmax = np.abs(values(s["v"])).max()
                bound = vmax * (rel + 2.0 ** -21 + 2 * (size / 64 + 64) * U)
                assert np.abs(got_out[i].reshape(nq, hd)[h * grp:(h + 1) * grp] - ref[0]).max() <= bound
                total = np.append(s["w"], 0.0).astype(np.float64) + add[0, 0]
                # which rows stay, by the device's sums: every kept slot's sum is on the device already
                m = min(size, budget)
                kept_pos = got_p[i, h, :m]
                order = [int(np.flatnonzero(s["p"] == p)[0]) for p in kept_pos]
                tol = add[0, 0] * (rel + grp * U) + 2 * U * total
                assert (np.abs(got_w[i, h, :m] - total[order]) <= tol[order]).all()
                if size > budget:
                    evicted += 1
                    lost = sorted(set(range(size)) - set(order))
                    assert len(lost) == 1 and len(set(order)) == budget
                    p = s["p"][lost[0]]
                    assert p >= 2 and p <= prompt + n - 8  # protected positions stay
                    free = [j for j in range(size) if s["p"][j] >= 2 and s["p"][j] <= prompt + n - 8]
                    assert total[lost[0]] <= min(total[j] + tol[j] for j in free) + tol[lost[0]]
                    # the only kept row from slot `budget` on, if any, moved into the hole; all others kept their slots
                    assert all(o == j for j, o in enumerate(order) if j != lost[0])
                sim[i][h] = dict(k=s["k"][order], v=s["v"][order], p=kept_pos.copy(), w=got_w[i, h, :m].copy())
                assert np.array_equal(got_k[i, h, :m], sim[i][h]["k"]) and np.array_equal(got_v[i, h, :m], sim[i][h]["v"])
        assert lens.tolist() == [min(prompt + n + 1, budget)] * layers
        ref, best = logits_ref(logits[0].cpu().numpy(), tokens=np.array(history, np.int32), repetition=1.3, frequency=0.2,
                               allowed=allowed[0])
        assert np.array_equal(out[0].cpu().numpy(), ref) and choice.item() == best
        token = best
        history.append(token)
        tokens[len(history) - 1] = token
    assert evicted > 0 and tqk.device_status() == 0


def test_unconstrained_choice_is_the_forward_passes(cuda):
    """tqk_process_logits without constraints agrees with the greedy choice of tqk_forward_token on its logits."""
    import torch
    from tailorquantkernel_b200 import tqk
    g = torch.Generator(device="cuda").manual_seed(1)
    nq, nkv, hd, hidden, inter, vocab, mt = 4, 2, 32, 128, 256, 515, 16

    def rows(r, c):
        return tqk.quantize_rows(torch.randn((r, c), device="cuda", generator=g) * 0.1)

    def ones(n):
        return torch.rand(n, device="cuda", generator=g) + 0.5

    lay = dict(input_norm=ones(hidden), post_norm=ones(hidden), wq=rows(nq * hd, hidden), wk=rows(nkv * hd, hidden),
               wv=rows(nkv * hd, hidden), wo=rows(hidden, nq * hd), q_norm=ones(hd), k_norm=ones(hd), wgate=rows(inter, hidden),
               wup=rows(inter, hidden), wdown=rows(hidden, inter), k_cache=tqk.empty_planes(nkv, mt, hd),
               v_cache=tqk.empty_planes(nkv, mt, hd))
    ang = torch.arange(mt, device="cuda")[:, None] * torch.logspace(0, -3, hd // 2, device="cuda")
    cfg = dict(n_layers=1, n_q_heads=nq, n_kv_heads=nkv, head_dim=hd, hidden_size=hidden, intermediate_size=inter,
               vocab_size=vocab, max_tokens=mt, rms_eps=1e-5)
    keep = (rows(vocab, hidden), ones(hidden), ang.cos().contiguous(), ang.sin().contiguous())
    m = tqk.model_struct(cfg, [lay], *keep)
    scratch = torch.empty(tqk.forward_scratch_bytes(m), dtype=torch.uint8, device="cuda")
    logits = torch.empty((1, vocab), device="cuda")
    nxt, choice = (torch.full((1,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    a = tqk.logits_args(logits, choice=choice)
    token = 5
    for pos in range(6):
        tqk.forward_token(m, token, pos, scratch, logits, nxt)
        tqk.process_logits(a)
        assert choice.item() == nxt.item()
        token = nxt.item()
