"""Measured cases of the cache-eviction and logit operators.

Three operators of a decoding loop over Q8 caches (blocks of 32 int8 values
behind one fp32 scale, 36 bytes):

  decode  decode attention that also adds every cached row's attention weight,
          summed over the q heads of its group, to a running sum per row
          (tqk.decode_weights);
  evict   for each head, keeping a budget of rows -- the first positions, the
          most recent ones and the largest sums -- and moving the kept rows of
          the tail into the slots of the evicted ones (tqk.evict);
  logits  repetition, frequency and presence penalties over each row's token
          history, token biases, grammar bit masks and the greedy choice
          (tqk.process_logits).

`own` selects who computes: False the plain torch forms below, True the
framework's entry points.
"""
import random

import numpy as np
import torch

own = False

QK = 32      # values per Q8 block
BLOCK = 36   # bytes per Q8 block: fp32 scale, 32 int8


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # the first tokens of one layer of a small model: nothing but latency
        dict(name="decode-first", op="decode", items=1, n_q=14, n_kv=2, hd=64, max_tokens=128, lo=3, hi=3, append=True),
        # one token through the 32 attention layers of the benchmark's decode workload
        dict(name="decode-layers", op="decode", items=32, n_q=32, n_kv=8, hd=128, max_tokens=4097, lo=4097, hi=4097,
             append=True),
        # the benchmark's ragged batch: 64 sequences of 512 to 8192 tokens, one layer
        dict(name="decode-ragged", op="decode", items=64, n_q=32, n_kv=8, hd=128, max_tokens=8192, lo=512, hi=8192,
             append=True),
        # the benchmark's long context: one layer of one sequence, 8 q heads on each kv head
        dict(name="decode-long", op="decode", items=1, n_q=64, n_kv=8, hd=128, max_tokens=131072, lo=131072, hi=131072,
             append=False),
        # one layer of one sequence goes back under its budget after a few tokens
        dict(name="evict-small", op="evict", items=1, n_kv=8, hd=128, max_tokens=512, lo=300, hi=300, budget=257, first=4,
             recent=32, ties=False),
        # steady state of a decoding loop: each of 32 layers is one row above its budget
        dict(name="evict-step", op="evict", items=32, n_kv=8, hd=128, max_tokens=4097, lo=4097, hi=4097, budget=4096,
             first=4, recent=256, ties=False),
        # a ragged batch is cut to a quarter after its prompts; sums with many equal values, short rows untouched
        dict(name="evict-ragged", op="evict", items=64, n_kv=8, hd=128, max_tokens=8192, lo=512, hi=8192, budget=2048,
             first=16, recent=512, ties=True),
        # one long sequence is cut to a quarter
        dict(name="evict-long", op="evict", items=1, n_kv=8, hd=128, max_tokens=131072, lo=131072, hi=131072,
             budget=32768, first=4, recent=4096, ties=False),
        # the next token of one sequence, everything on
        dict(name="logits-one", op="logits", rows=1, vocab=128256, lo=1500, hi=1500, bias=16, allowed=0.02, penal=True),
        # a small batch over an odd vocabulary, penalties and biases without a grammar
        dict(name="logits-odd", op="logits", rows=7, vocab=32003, lo=0, hi=2049, bias=5, allowed=0.0, penal=True),
        # a serving batch with penalties, biases and masks
        dict(name="logits-batch", op="logits", rows=64, vocab=128256, lo=20, hi=4000, bias=40, allowed=0.5, penal=True),
        # the largest batch, long histories
        dict(name="logits-large", op="logits", rows=256, vocab=128256, lo=500, hi=16000, bias=100, allowed=0.9, penal=True),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["decode", "evict", "logits"])
    if op == "logits":
        vocab = _log_int(rng, 1000, 152064)
        rows = _log_int(rng, 1, max(1, 256 * 128256 // vocab if vocab > 16000 else 512))
        hi = _log_int(rng, 1, 16000)
        return dict(op=op, rows=rows, vocab=vocab, lo=rng.choice([0, 1, hi // 2, hi]), hi=hi, bias=rng.choice([0, 1, 17, 100]),
                    allowed=rng.choice([0.0, 0.001, 0.3, 0.97]), penal=rng.random() < 0.8)
    hd = rng.choice([32, 64, 128, 128, 128, 256])
    n_kv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    items = _log_int(rng, 1, 64)
    # cache and products are at most those of the largest listed case
    most = 64 * 8 * 4352 * 128 // (items * n_kv * hd) * 4 // max(4, group)
    hi = _log_int(rng, 1, min(131072, most))
    lo = rng.choice([1, max(1, hi // 16), max(1, hi // 2), hi])
    max_tokens = hi + rng.choice([0, 0, 1, 13, 64])
    if op == "decode":
        append = rng.random() < 0.7
        return dict(op=op, items=items, n_q=n_kv * group, n_kv=n_kv, hd=hd, max_tokens=max_tokens,
                    lo=lo if append or rng.random() < 0.7 else 0, hi=hi, append=append)
    budget = max(1, min(max_tokens, rng.choice([hi - 1, hi // 2, hi // 4, (9 * hi) // 10, hi])))
    recent = rng.choice([0, 1, budget // 8, budget // 2])
    first = min(budget - recent, rng.choice([0, 4, 16]))
    return dict(op=op, items=items, n_kv=n_kv, hd=hd, max_tokens=max_tokens, lo=lo, hi=hi, budget=budget, first=first,
                recent=recent, ties=rng.random() < 0.5)


def _lengths(case, n):
    """n lengths from lo to hi (both among them where n > 1), the same ones for every seed."""
    if n == 1 or case["lo"] == case["hi"]:
        return [case["hi"]] * n
    got = [case["lo"] + (case["hi"] - case["lo"]) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(got)
    return got


def _ragged(case):
    return case["items"] > 1 and case["lo"] != case["hi"]


# --------------------------------------------------------------------------- inputs
def _quantize(x):
    """fp32 rows [..., n] as Q8: codes [..., n/32, 32] (int8) and scales [..., n/32], by the caches' rule:
    scale = max|x| / 127, code = x * (1 / scale) to the nearest even, each step rounded to fp32."""
    b = x.reshape(*x.shape[:-1], -1, QK)
    d = b.abs().amax(-1) / 127.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    return torch.round(b * inv[..., None]).to(torch.int8), d


def _codes(plane):
    """The int8 codes [..., nb, 32] of a plane, a view."""
    return plane.view(*plane.shape[:-1], -1, BLOCK)[..., 4:].view(torch.int8)


def _scales(plane):
    """The fp32 scales [..., nb] of a plane, a view."""
    return plane.view(torch.float32).view(*plane.shape[:-1], -1, BLOCK // 4)[..., 0]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)

    def plane():
        """A Q8 plane [items, n_kv, max_tokens, hd/32 * 36] (uint8) of N(0,1) rows, made item by item."""
        p = torch.empty((items, n_kv, mt, hd // QK * BLOCK), dtype=torch.uint8, device="cuda")
        for i in range(items):
            codes, d = _quantize(torch.randn((n_kv, mt, hd), device="cuda", generator=g))
            _codes(p)[i], _scales(p)[i] = codes, d
        return p

    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        lens = _lengths(case, rows)
        s["logits"] = torch.randn((rows, vocab), device="cuda", generator=g) * 3
        s["offsets"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
        s["n_tokens"] = int(sum(lens))
        # token frequencies fall off steeply, so histories repeat themselves
        s["tokens"] = (torch.rand(max(1, s["n_tokens"]), device="cuda", generator=g) ** 3 * vocab).to(torch.int32)
        s["prompt_lens"] = torch.tensor([n // 2 for n in lens], dtype=torch.int32, device="cuda")
        u = torch.rand((3, rows), device="cuda", generator=g)
        s["repetition"], s["frequency"], s["presence"] = 1.0 + 0.3 * u[0], 0.5 * u[1], 0.5 * u[2]
        nb = case["bias"]
        s["bias_offsets"] = torch.arange(0, rows * nb + 1, nb or 1, dtype=torch.int32, device="cuda")[:rows + 1]
        s["bias_tokens"] = torch.randint(0, vocab, (max(1, rows * nb),), device="cuda", generator=g, dtype=torch.int32)
        s["bias_values"] = torch.randn(max(1, rows * nb), device="cuda", generator=g) * 4
        words = (vocab + 31) // 32
        bits = torch.rand((rows, words, 32), device="cuda", generator=g) < case["allowed"]
        s["mask"] = (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
        s["out"] = torch.empty_like(s["logits"])
        s["choice"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        return s
    items, n_kv, hd, mt = case["items"], case["n_kv"], case["hd"], case["max_tokens"]
    lens = _lengths(case, items)
    s["k"], s["v"] = plane(), plane()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # the sums that earlier tokens left: heavy-tailed; with ties, multiples of 1/4 as few tokens leave
    w = torch.exp(2.0 * torch.randn((items, n_kv, mt), device="cuda", generator=g))
    if case.get("ties"):
        w = torch.floor(w * 4) / 4
    if case["op"] == "decode":
        w = w * (case["n_q"] / n_kv / case["hi"])  # about a token's share: what the call adds shows beside it
    s["weight"], s["weight_out"] = w, w.clone()
    # positions: increasing with gaps; the front half of the slots, where earlier evictions moved rows, is mixed
    pos = torch.cumsum(torch.randint(1, 4, (items, n_kv, mt), device="cuda", generator=g), -1)
    half = case["hi"] // 2
    if case["op"] == "evict" and half:
        mix = torch.argsort(torch.rand((items, n_kv, half), device="cuda", generator=g), -1)
        pos[..., :half] = pos[..., :half].gather(-1, mix)
    s["position"] = pos.to(torch.int32)
    s["position_out"] = s["position"].clone()
    if case["op"] == "decode":
        s["q"] = torch.randn((items, case["n_q"] * hd), device="cuda", generator=g)
        s["k_new"] = torch.randn((items, n_kv * hd), device="cuda", generator=g)
        s["v_new"] = torch.randn((items, n_kv * hd), device="cuda", generator=g)
        s["new_pos"] = torch.full((items,), 3 * mt + 1, dtype=torch.int32, device="cuda")
        s["out"] = torch.empty((items, case["n_q"] * hd), device="cuda")
    else:
        s["lens_out"] = torch.empty(items, dtype=torch.int32, device="cuda")
    return s


# --------------------------------------------------------------------------- the framework's calls
def _plan(s):
    """The argument struct of the state's call: a decoding program fills it once for its buffers and keeps it."""
    from tailorquantkernel_b200 import tqk
    if s["op"] == "logits":
        pen, bias, mask = s["penal"], s["bias"] > 0, s["mask"] if s["allowed"] else None
        return tqk.logits_args(
            s["logits"], out=s["out"], choice=s["choice"],
            tokens=s["tokens"] if pen else None, token_offsets=s["offsets"] if pen else None,
            n_tokens=s["n_tokens"] if pen else 0, prompt_lens=s["prompt_lens"] if pen else None,
            repetition=s["repetition"] if pen else None, frequency=s["frequency"] if pen else None,
            presence=s["presence"] if pen else None,
            bias_tokens=s["bias_tokens"] if bias else None, bias_values=s["bias_values"] if bias else None,
            bias_offsets=s["bias_offsets"] if bias else None, n_bias=s["rows"] * s["bias"], mask=mask)
    items, n_kv, hd, mt = s["items"], s["n_kv"], s["hd"], s["max_tokens"]
    planes = dict(n_items=items, item_stride_blocks=n_kv * mt * (hd // QK))
    lens = dict(lens=s["lens"], max_len=s["hi"]) if _ragged(s) else dict(len0=s["hi"])
    if s["op"] == "decode":
        new = dict(k_new=s["k_new"], v_new=s["v_new"], kv_new_item_stride=n_kv * hd) if s["append"] else {}
        a = tqk.decode_args(s["k"], s["v"], s["n_q"], n_kv, hd, mt, s["q"], s["out"], q_item_stride=s["n_q"] * hd,
                            out_item_stride=s["n_q"] * hd, **planes, **lens, **new)
        new = dict(position=s["position"], new_pos=s["new_pos"]) if s["append"] else {}
        return a, tqk.weights_args(s["weight"], s["weight_out"], item_stride=n_kv * mt, **new)
    return tqk.evict_args(s["k"], s["v"], n_kv, hd, mt, s["budget"], n_first=s["first"], n_recent=s["recent"],
                          weight=s["weight"], weight_out=s["weight_out"], position=s["position"],
                          position_out=s["position_out"], stat_item_stride=n_kv * mt, lens_out=s["lens_out"], **planes,
                          **lens)


def _run_own(s):
    from tailorquantkernel_b200 import tqk
    if "plan" not in s:
        s["plan"] = _plan(s)
    if s["op"] == "logits":
        tqk.process_logits(s["plan"])
        return {"out": s["out"], "choice": s["choice"]}
    if s["op"] == "decode":
        tqk.decode_weights(*s["plan"])
        return _decode_outputs(s, s["out"], s["weight_out"])
    tqk.evict(s["plan"])
    return _evict_outputs(s, s["weight_out"], s["position_out"], s["lens_out"])


def _decode_outputs(s, out, weight):
    got = {"out": out, "weight": weight}
    if s["append"]:  # the caches with the appended rows, and their positions
        got.update(k=_codes(s["k"]), kd=_scales(s["k"]), v=_codes(s["v"]), vd=_scales(s["v"]), position=s["position"])
    return got


def _evict_outputs(s, weight, position, lens):
    return {"k": _codes(s["k"]), "kd": _scales(s["k"]), "v": _codes(s["v"]), "vd": _scales(s["v"]), "weight": weight,
            "position": position, "lens": lens}


# --------------------------------------------------------------------------- plain forms
def _plain_logits(s):
    x, rows, vocab = s["logits"], s["rows"], s["vocab"]
    row = torch.arange(rows, device="cuda")
    if s["penal"]:
        at = torch.arange(s["n_tokens"], device="cuda")
        r = torch.bucketize(at, s["offsets"][1:], right=True)
        flat = r * vocab + s["tokens"][:s["n_tokens"]].long()
        fresh = (at - s["offsets"][r] >= s["prompt_lens"][r]).float()  # generated, not of the prompt
        seen = torch.zeros(rows * vocab, device="cuda").index_fill_(0, flat, 1.0).view(rows, vocab) > 0
        count = torch.zeros(rows * vocab, device="cuda").index_add_(0, flat, fresh).view(rows, vocab)
        rep = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - s["frequency"][:, None] * count
        x = torch.where(count > 0, x - s["presence"][:, None], x)
    if s["bias"]:
        flat = row.repeat_interleave(s["bias"]) * vocab + s["bias_tokens"].long()
        x = x + torch.zeros(rows * vocab, device="cuda").index_add_(0, flat, s["bias_values"]).view(rows, vocab)
    if s["allowed"]:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = torch.where(bits.view(rows, -1)[:, :vocab] > 0, x, torch.full_like(x, -torch.inf))
    top = x.amax(-1, keepdim=True)
    # the first of the largest; -1 where nothing is left
    at = torch.where(x == top, torch.arange(vocab, device="cuda", dtype=torch.int32), vocab).amin(-1)
    return {"out": x if x is not s["logits"] else x.clone(),
            "choice": torch.where(top[:, 0] > -torch.inf, at, -1).to(torch.int32)}


def _plain_decode(s):
    items, n_kv, hd, n = s["items"], s["n_kv"], s["hd"], s["hi"]
    group, lens = s["n_q"] // n_kv, s["lens"].long()
    item = torch.arange(items, device="cuda")
    if s["append"]:
        for_k, for_v = (_quantize(s[name].view(items, n_kv, hd)) for name in ("k_new", "v_new"))
        _codes(s["k"])[item, :, lens - 1], _scales(s["k"])[item, :, lens - 1] = for_k
        _codes(s["v"])[item, :, lens - 1], _scales(s["v"])[item, :, lens - 1] = for_v
        s["position"][item, :, lens - 1] = s["new_pos"][:, None]
    qc, qd = _quantize(s["q"].view(items, n_kv, group, hd))
    q = (qc * qd[..., None]).view(items, n_kv, group, hd)
    k, v = ((_codes(s[p])[:, :, :n] * _scales(s[p])[:, :, :n, :, None]).view(items, n_kv, n, hd) for p in ("k", "v"))
    slot = torch.arange(n, device="cuda")
    valid = (slot < lens[:, None])[:, None, None]
    scores = torch.where(valid, (q @ k.transpose(-1, -2)) * (1.0 / hd ** 0.5), -torch.inf)
    p = torch.where(valid, torch.exp(scores - scores.amax(-1, keepdim=True)), 0.0)
    w = torch.where(valid, p / p.sum(-1, keepdim=True), 0.0)
    weight = s["weight"].clone()
    if s["append"]:
        weight[item, :, lens - 1] = 0.0  # whatever an earlier tenant of the slot left
    weight[:, :, :n] += w.sum(2)
    return _decode_outputs(s, (w @ v).view(items, -1), weight)


def _plain_evict(s):
    items, n_kv, n, budget = s["items"], s["n_kv"], s["hi"], min(s["budget"], s["hi"])
    slot = torch.arange(n, device="cuda")
    lens = s["lens"][:, None, None]
    valid = slot < lens
    pos, w = s["position"][:, :, :n], s["weight"][:, :, :n]
    newest = torch.where(valid, pos, -1).amax(-1, keepdim=True)
    kept_always = (pos < s["first"]) | (pos > newest - s["recent"])
    key = torch.where(valid, torch.where(kept_always, torch.inf, w), -torch.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices  # equal keys: the lower slot first
    keep = torch.zeros_like(valid.expand_as(key)).scatter(-1, order[..., :budget], True) & valid
    hole, mover = valid & ~keep & (slot < budget), keep & (slot >= budget)
    # the j-th hole takes the j-th mover
    nth = torch.where(mover, mover.cumsum(-1) - 1, n)
    movers = torch.zeros(items, n_kv, n + 1, dtype=torch.long, device="cuda").scatter(-1, nth, slot.expand_as(nth))
    src = torch.where(hole, movers.gather(-1, hole.cumsum(-1).clamp(max=n) - hole.long()), slot)[..., :budget]
    item, head = torch.arange(items, device="cuda")[:, None, None], torch.arange(n_kv, device="cuda")[:, None]
    s["k"][:, :, :budget], s["v"][:, :, :budget] = s["k"][item, head, src], s["v"][item, head, src]
    weight, position = s["weight"].clone(), s["position"].clone()
    weight[:, :, :budget], position[:, :, :budget] = w.gather(-1, src), pos.gather(-1, src)
    return _evict_outputs(s, weight, position, s["lens"].clamp(max=s["budget"]))


def run(state):
    if own:
        return _run_own(state)
    return {"logits": _plain_logits, "decode": _plain_decode, "evict": _plain_evict}[state["op"]](state)


# --------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(s)
    return _exact_decode(s) if case["op"] == "decode" else _exact_evict(s)


def _exact_logits(s):
    """Row by row and list by list, in numpy float64."""
    host = {k: v.cpu().numpy() for k, v in s.items() if torch.is_tensor(v)}
    out, choice = np.empty((s["rows"], s["vocab"])), np.empty(s["rows"], np.int32)
    for r in range(s["rows"]):
        x = host["logits"][r].astype(np.float64)
        if s["penal"]:
            tokens = host["tokens"][host["offsets"][r]:host["offsets"][r + 1]]
            rep = float(host["repetition"][r])
            for t in np.unique(tokens):
                x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
            made, times = np.unique(tokens[host["prompt_lens"][r]:], return_counts=True)
            x[made] -= float(host["frequency"][r]) * times + float(host["presence"][r])
        if s["bias"]:
            at = slice(host["bias_offsets"][r], host["bias_offsets"][r + 1])
            np.add.at(x, host["bias_tokens"][at], host["bias_values"][at].astype(np.float64))
        if s["allowed"]:
            x[np.unpackbits(host["mask"][r].view(np.uint8), bitorder="little")[:s["vocab"]] == 0] = -np.inf
        out[r], choice[r] = x, np.argmax(x) if x.max() > -np.inf else -1
    return {"out": out, "choice": choice}


def _exact_decode(s):
    """Item by item, in torch float64; the quantised values are those of the caches' (fp32) rule."""
    items, n_kv, hd = s["items"], s["n_kv"], s["hd"]
    group = s["n_q"] // n_kv
    out = torch.zeros((items, s["n_q"] * hd), dtype=torch.float64, device="cuda")
    weight = s["weight"].double()

    def values(codes, scales):
        return (codes.double() * scales.double()[..., None]).flatten(-2)

    for i, n in enumerate(_lengths(s, items)):
        if n == 0:
            continue
        k, v = (values(_codes(s[p][i, :, :n]), _scales(s[p][i, :, :n])) for p in ("k", "v"))
        if s["append"]:
            k[:, -1] = values(*_quantize(s["k_new"][i].view(n_kv, hd)))
            v[:, -1] = values(*_quantize(s["v_new"][i].view(n_kv, hd)))
            weight[i, :, n - 1] = 0
        q = values(*_quantize(s["q"][i].view(n_kv, group, hd)))
        w = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / hd ** 0.5, -1)
        out[i] = torch.einsum("hgt,htd->hgd", w, v).flatten()
        weight[i, :, :n] += w.sum(1)
    got = {"out": out, "weight": weight}
    if s["append"]:  # the caches hold bytes of the fp32 rule
        got.update(k=None, kd=None, v=None, vd=None, position=None)
    return got


def _exact_evict(s):
    """Head by head, in numpy."""
    weight, position = s["weight"].double().cpu().numpy(), s["position"].cpu().numpy()
    budget = s["budget"]
    for i, n in enumerate(_lengths(s, s["items"])):
        for h in range(s["n_kv"] if n > budget else 0):
            w, p = weight[i, h, :n].copy(), position[i, h, :n].copy()
            rank = np.where((p < s["first"]) | (p > p.max() - s["recent"]), np.inf, w)
            kept = np.zeros(n, bool)
            kept[np.lexsort((np.arange(n), -rank))[:budget]] = True
            to, src = np.flatnonzero(~kept[:budget]), budget + np.flatnonzero(kept[budget:])
            weight[i, h, to], position[i, h, to] = w[src], p[src]
    return {"k": None, "kd": None, "v": None, "vd": None, "weight": weight, "position": position,
            "lens": np.minimum(s["lens"].cpu().numpy(), budget)}


def work(case):
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        n = sum(_lengths(case, rows)) if case["penal"] else 0
        return {"bytes": rows * vocab * 8 + (rows * vocab / 8 if case["allowed"] else 0) + 4 * n +
                8 * rows * case["bias"] + 4 * rows, "flops": rows * vocab}
    items, n_kv, hd = case["items"], case["n_kv"], case["hd"]
    lens, row = _lengths(case, items), hd // QK * BLOCK
    if case["op"] == "decode":
        # each K and V row once, each sum read and written, q, output and new rows
        return {"bytes": sum(lens) * n_kv * (2 * row + 8) + items * (2 * case["n_q"] + 2 * n_kv) * hd * 4,
                "flops": 4 * sum(lens) * case["n_q"] * hd}
    total = 0
    for n in lens:
        # each sum and position read, those of the kept rows written; the rows that move read and written once: the
        # recent ones, which lie in the tail, and the tail's share of the largest sums
        b, r, f = min(case["budget"], n), case["recent"] / 2, case["first"] / 2  # positions advance by 2 a row
        tail = n - b
        moved = min(r, tail) + max(0, b - f - r) * max(0, tail - r) / max(1, n - r - f)
        total += n_kv * (8 * n + 8 * b + min(moved, b, tail) * 4 * row)
    return {"bytes": total, "flops": 0}
